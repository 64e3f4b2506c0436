// Row arithmetic shared by the packed row operators: 16 bytes of storage as fp32 lanes or packed fp32 pairs, and sums over
// the threads that share a row.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "sm100_ptx.cuh"

namespace ntb200 {
namespace {

// 16 bytes of storage <-> fp32 lanes
template <int DT>
struct Vec16;
template <>
struct Vec16<NTB200_F32> {
  static constexpr int kElems = 4;
  static __device__ __forceinline__ void unpack(const uint4& r, float* f) {
    f[0] = __uint_as_float(r.x), f[1] = __uint_as_float(r.y), f[2] = __uint_as_float(r.z), f[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
  static __device__ __forceinline__ float load1(const void* p, int64_t i) { return reinterpret_cast<const float*>(p)[i]; }
  static __device__ __forceinline__ void store1(void* p, int64_t i, float v) { reinterpret_cast<float*>(p)[i] = v; }
};
template <>
struct Vec16<NTB200_F16> {
  static constexpr int kElems = 8;
  static __device__ __forceinline__ void unpack(const uint4& r, float* f) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
      f[2 * k] = t.x, f[2 * k + 1] = t.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const __half2 h = __floats2half2_rn(f[2 * k], f[2 * k + 1]);
      w[k] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ float load1(const void* p, int64_t i) { return __half2float(reinterpret_cast<const __half*>(p)[i]); }
  static __device__ __forceinline__ void store1(void* p, int64_t i, float v) { reinterpret_cast<__half*>(p)[i] = __float2half_rn(v); }
};
template <>
struct Vec16<NTB200_BF16> {
  static constexpr int kElems = 8;
  static __device__ __forceinline__ void unpack(const uint4& r, float* f) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {  // a bf16 is the upper half of an fp32
      f[2 * k] = __uint_as_float(w[k] << 16);
      f[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * k], f[2 * k + 1]);
      w[k] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ float load1(const void* p, int64_t i) {
    return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  }
  static __device__ __forceinline__ void store1(void* p, int64_t i, float v) {
    reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  }
};

// The same 16 bytes as kElems / 2 packed fp32 pairs (sm_100 adds, subtracts and multiplies two fp32 values
// held in a 64-bit register pair with one instruction: the LayerNorm kernel is otherwise bound by its issue
// slots, not by memory).
template <int DT>
__device__ __forceinline__ void unpack_pairs(const uint4& r, uint64_t* p) {
  float f[Vec16<DT>::kElems];
  Vec16<DT>::unpack(r, f);
#pragma unroll
  for (int k = 0; k < Vec16<DT>::kElems / 2; ++k) p[k] = ptx::f32x2_pack(f[2 * k], f[2 * k + 1]);
}
template <int DT>
__device__ __forceinline__ uint4 pack_pairs(const uint64_t* p) {
  float f[Vec16<DT>::kElems];
#pragma unroll
  for (int k = 0; k < Vec16<DT>::kElems / 2; ++k) ptx::f32x2_unpack(p[k], f[2 * k], f[2 * k + 1]);
  return Vec16<DT>::pack(f);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum over the GROUP threads that share a row: part of a warp (GROUP == 8, 16: neighbouring lanes), a warp
// (GROUP == 32) or the whole block.
template <int GROUP>
__device__ __forceinline__ float group_sum(float v, float* scratch) {
  if (GROUP < 32) {
#pragma unroll
    for (int o = GROUP / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
  v = warp_sum(v);
  if (GROUP == 32) return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();  // scratch may still be read from the previous reduction
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  float t = lane < GROUP / 32 ? scratch[lane] : 0.0f;
  return warp_sum(t);
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace ntb200
