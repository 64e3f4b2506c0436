// What the kernels of the attention backward pass share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace ntb200 {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxHeadDim = 256;

namespace {

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }

}  // namespace

// What every kernel of the backward pass reads and writes; strides in elements, all matrices [tokens, H * d] at head 0.
struct BwdArgs {
  const void *grad, *q, *k, *v, *out;
  const float* lse;  // [H, q_tokens]
  float* delta;      // [H, q_tokens]: D
  const uint2* top;  // [batch, H]: bits of the largest |dO_i|^2 and |V_j|^2 of the sequence and head (fp16 kernels only, else NULL)
  void *dq, *dk, *dv;
  int64_t ldq, ldk, ldv, lddq, lddk, lddv;  // grad and out are contiguous: their stride is H * d
  const int64_t *offsets_q, *offsets_k;
  int64_t row_elems_q, row_elems_k;
  int64_t batch, q_tokens;
  int H, d;
  float scaling;
};

// The device-built list of work items of one side: items[i] = (first row of the tile, valid rows in it, first row of the
// sequence's other side, its length), seq[i] = the sequence.
struct ListOut {
  int4* items;
  int* seq;
  int* count;
};

// One work item: a tile of the own side, and the other side of its sequence
struct Item {
  int64_t row0;   // first row of the tile
  int rows;       // valid rows in it
  int64_t other;  // first row of the other side
  int n_other;    // and its length
};

namespace {

__device__ __forceinline__ Item decode(const int4& w) { return {w.x, w.y, w.z, w.w}; }

// fp16 holds dS only between 2^-24 and 65504, while gradients and values come at any scale: dS is computed from dO times a power of
// two, and the product's sum is divided by it again (both exact).  With R = max |dO_i| max |V_j| over the sequence and head (2-norms),
// |dS_ij| = P_ij (1 - P_ij) |dP_ij - (mean of the other dP, weighted by P)| <= 1/4 2R.  So the factor brings R to (2^15, 2^16]: dS
// stays under 2^15, and as little as possible of it falls under fp16's normal numbers.
__device__ __forceinline__ float scale_of(const uint2& top) {
  const int e = (int)(__float_as_uint(__uint_as_float(top.x) * __uint_as_float(top.y)) >> 23);  // R^2 in [2^(e - 127), 2^(e - 126))
  if (e == 0) return 1.0f;                                                                      // nothing but zeros (or Inf and NaN)
  return __uint_as_float((unsigned)(127 + 16 - ((e - 126 + 1) >> 1)) << 23);                    // (e in 31 .. 207)
}
__device__ __forceinline__ float grad_scale(const BwdArgs& a, const int* __restrict__ seq, int64_t i, int h) {
  return a.top == nullptr ? 1.0f : scale_of(a.top[(int64_t)seq[i] * a.H + h]);
}

}  // namespace

// attention_backward_tcgen05.cu: heads of 64 and 128, fp16 / bf16; a.delta and the lists (tiles of 128 rows) are in place
bool attn_bwd_tcgen05_supported(const BwdArgs& a, int64_t k_tokens, int dtype);
int attn_bwd_tcgen05_launch(const BwdArgs& a, int64_t k_tokens, int dtype, const ListOut& kv, const ListOut& qi, int64_t kv_capacity,
                            int64_t q_capacity, cudaStream_t st);
// whole sequences as items, heads of 64: seqs lists (first key, keys, first query, queries) of every sequence with rows on either side;
// scratch: H * 64 * q_tokens floats, 16-byte aligned (unused where no sequence has more than 128 keys)
int attn_bwd_fused_launch(const BwdArgs& a, int64_t k_tokens, int dtype, const ListOut& seqs, float* scratch, cudaStream_t st);

}  // namespace ntb200
