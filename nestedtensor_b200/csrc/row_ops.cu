// Row operators on the packed token matrix [T = sum(L_i), E] of a nested tensor: the steps of a
// transformer encoder layer that sit between the projections.  All of them stream every element once
// (HBM-bound), never see padding, and keep their arithmetic in fp32 whatever the storage type.
//
//   layer_norm                    out = (x - mean) * rsqrt(var + eps) * gamma + beta          per row
//   add_bias_residual_layer_norm  the same on x + residual + bias (one pass instead of three)
//   add_bias_gelu                 out = gelu_tanh(x + bias)
//
// Replaces fastertransformer::layer_norm (nestedtensor/csrc/cuda/transformer_kernels.cu:260-335) as used by
// cuda::NestedTensor_layer_norm (nestedtensor/csrc/cuda/layernorm.cpp:14-76), add_bias_input_layernorm
// (transformer_kernels.cu:64-156, cuda_kernels.cu:114-159) and add_bias_act / add_bias_gelu
// (cuda_kernels.cu:73-104, transformer_kernels.cu:52-62).

#include "row_vec.cuh"

namespace ntb200 {
namespace {

constexpr int kLnThreads = 256;

struct RowStats {  // [rows] fp32 each, or NULL
  float *mean, *rstd;
};

// One row per GROUP threads, the row held in registers between the passes (one global read, one global
// write per element).  VPL = 16-byte vectors per thread; vector v of the row belongs to thread v % GROUP.
// Mean and variance are the two-pass forms of the reference kernel (sum, then sum of squared deviations).
// A 16-bit row without the fused additions stays in its packed form (4 registers per vector instead of 8) and is
// widened again in each pass, which is exact: half the registers, twice the rows in flight per SM.
// FULL: the row is exactly VPL * GROUP vectors (no per-vector bound test).  STATS: mean and rstd of every row are stored too,
// for a backward pass.
template <int DT, int VPL, int GROUP, bool FUSED, bool FULL, bool STATS>
__global__ void __launch_bounds__(kLnThreads, (!FUSED && FULL && DT != NTB200_F32 && VPL <= 4) ? 6 : 1)
layer_norm_kernel(const void* x, const void* __restrict__ residual, const void* __restrict__ bias,
                  const void* __restrict__ gamma, const void* __restrict__ beta, float eps, void* out, int64_t rows,
                  int cols, RowStats stats) {  // out may alias x: a thread has read all it needs of the row before it writes
  constexpr int EPV = Vec16<DT>::kElems;
  constexpr int kRowsPerBlock = kLnThreads / GROUP;
  constexpr bool RAW = !FUSED && DT != NTB200_F32;
  __shared__ float scratch[kLnThreads / 32];
  const int t = threadIdx.x % GROUP;
  const int64_t row = (int64_t)blockIdx.x * kRowsPerBlock + threadIdx.x / GROUP;
  const bool live = row < rows;  // whole groups are live or not; a warp of several short rows may hold both kinds
  if (GROUP == 32 && !live) return;
  const int nv = cols / EPV;
  const uint4* xr = reinterpret_cast<const uint4*>(x) + row * nv;
  const uint4* rr = reinterpret_cast<const uint4*>(residual) + row * nv;
  constexpr int PPV = EPV / 2;  // packed pairs per vector
  uint4 raw[RAW ? VPL : 1];
  uint64_t v[RAW ? 1 : VPL][PPV];
  if (RAW) {  // all loads of the row first
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      const int vec = t + j * GROUP;
      raw[j] = make_uint4(0u, 0u, 0u, 0u);
      if ((FULL || vec < nv) && live) raw[j] = xr[vec];
    }
  }
  uint64_t sum2 = 0;
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    const int vec = t + j * GROUP;
    if (RAW) {
      uint64_t a[PPV];
      unpack_pairs<DT>(raw[j], a);  // (vectors past the row are zero)
#pragma unroll
      for (int k = 0; k < PPV; ++k) sum2 = ptx::f32x2_add(sum2, a[k]);
    } else if ((FULL || vec < nv) && live) {
      unpack_pairs<DT>(xr[vec], v[j]);
      if (FUSED) {
        uint64_t a[PPV];
        if (residual != nullptr) {
          unpack_pairs<DT>(rr[vec], a);
#pragma unroll
          for (int k = 0; k < PPV; ++k) v[j][k] = ptx::f32x2_add(v[j][k], a[k]);
        }
        if (bias != nullptr) {
          unpack_pairs<DT>(reinterpret_cast<const uint4*>(bias)[vec], a);
#pragma unroll
          for (int k = 0; k < PPV; ++k) v[j][k] = ptx::f32x2_add(v[j][k], a[k]);
        }
      }
#pragma unroll
      for (int k = 0; k < PPV; ++k) sum2 = ptx::f32x2_add(sum2, v[j][k]);
    } else {
#pragma unroll
      for (int k = 0; k < PPV; ++k) v[j][k] = 0;
    }
  }
  // (an empty asm that "rewrites" the packed row: keeps the compiler from carrying the widened copy across the pass)
#define NTB200_LN_LAUNDER()                                                                                     \
  if (RAW) {                                                                                                    \
    _Pragma("unroll") for (int j = 0; j < VPL; ++j)                                                             \
        asm volatile("" : "+r"(raw[j].x), "+r"(raw[j].y), "+r"(raw[j].z), "+r"(raw[j].w));                      \
  }
  NTB200_LN_LAUNDER();
  float s_lo, s_hi;
  ptx::f32x2_unpack(sum2, s_lo, s_hi);
  const float mean = group_sum<GROUP>(s_lo + s_hi, scratch) / (float)cols;
  const uint64_t mean2 = ptx::f32x2_pack(mean, mean);
  uint64_t sq2 = 0;
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    if (FULL || t + j * GROUP < nv) {
      if (RAW) {
        uint64_t a[PPV];
        unpack_pairs<DT>(raw[j], a);
#pragma unroll
        for (int k = 0; k < PPV; ++k) {
          const uint64_t d = ptx::f32x2_sub(a[k], mean2);
          sq2 = ptx::f32x2_fma(d, d, sq2);
        }
      } else {
#pragma unroll
        for (int k = 0; k < PPV; ++k) {
          v[j][k] = ptx::f32x2_sub(v[j][k], mean2);  // deviations replace the values
          sq2 = ptx::f32x2_fma(v[j][k], v[j][k], sq2);
        }
      }
    }
  }
  NTB200_LN_LAUNDER();
#undef NTB200_LN_LAUNDER
  ptx::f32x2_unpack(sq2, s_lo, s_hi);
  const float rstd = rsqrtf(group_sum<GROUP>(s_lo + s_hi, scratch) / (float)cols + eps);
  if (!live) return;
  if (STATS && t == 0) {
    stats.mean[row] = mean;
    stats.rstd[row] = rstd;
  }
  const uint64_t rstd2 = ptx::f32x2_pack(rstd, rstd);
  uint4* orow = reinterpret_cast<uint4*>(out) + row * nv;
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    const int vec = t + j * GROUP;
    if (FULL || vec < nv) {
      uint64_t o[PPV], d[PPV];
      if (RAW) {
        unpack_pairs<DT>(raw[j], d);
#pragma unroll
        for (int k = 0; k < PPV; ++k) d[k] = ptx::f32x2_sub(d[k], mean2);
      } else {
#pragma unroll
        for (int k = 0; k < PPV; ++k) d[k] = v[j][k];
      }
      if (gamma != nullptr) {
        uint64_t g[PPV], b[PPV];
        unpack_pairs<DT>(reinterpret_cast<const uint4*>(gamma)[vec], g);
        unpack_pairs<DT>(reinterpret_cast<const uint4*>(beta)[vec], b);
#pragma unroll
        for (int k = 0; k < PPV; ++k) o[k] = ptx::f32x2_fma(ptx::f32x2_fma(d[k], rstd2, 0ull), g[k], b[k]);
      } else {
#pragma unroll
        for (int k = 0; k < PPV; ++k) o[k] = ptx::f32x2_fma(d[k], rstd2, 0ull);
      }
      orow[vec] = pack_pairs<DT>(o);
    }
  }
}

// Any row length and alignment: one block per row, three passes over global memory.
template <int DT>
__global__ void __launch_bounds__(kLnThreads)
layer_norm_generic_kernel(const void* x, const void* __restrict__ residual, const void* __restrict__ bias,
                          const void* __restrict__ gamma, const void* __restrict__ beta, float eps, void* out, int64_t rows,
                          int cols, RowStats stats) {
  __shared__ float scratch[kLnThreads / 32];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const int64_t base = row * cols;
    auto value = [&](int i) {
      float a = Vec16<DT>::load1(x, base + i);
      if (residual != nullptr) a += Vec16<DT>::load1(residual, base + i);
      if (bias != nullptr) a += Vec16<DT>::load1(bias, i);
      return a;
    };
    float sum = 0.0f;
    for (int i = threadIdx.x; i < cols; i += kLnThreads) sum += value(i);
    const float mean = group_sum<kLnThreads>(sum, scratch) / (float)cols;
    float sq = 0.0f;
    for (int i = threadIdx.x; i < cols; i += kLnThreads) {
      const float d = value(i) - mean;
      sq += d * d;
    }
    const float rstd = rsqrtf(group_sum<kLnThreads>(sq, scratch) / (float)cols + eps);
    if (stats.mean != nullptr && threadIdx.x == 0) {
      stats.mean[row] = mean;
      stats.rstd[row] = rstd;
    }
    for (int i = threadIdx.x; i < cols; i += kLnThreads) {
      float o = (value(i) - mean) * rstd;
      if (gamma != nullptr) o = o * Vec16<DT>::load1(gamma, i) + Vec16<DT>::load1(beta, i);
      Vec16<DT>::store1(out, base + i, o);  // out may alias x: every thread rereads only what it writes itself
    }
  }
}

// Rows that are not made of whole 16-byte vectors, with statistics for a backward pass: one row per GROUP threads, element by
// element, held in registers between the passes: 34 us for 24 000 rows of 771 bf16, bound by instruction issue (about 31 per
// element), where the generic kernel, which reads the row three times, takes 94 and the copy alone would take 11.
template <int DT, int VPL, int GROUP>
__global__ void __launch_bounds__(kLnThreads)
layer_norm_elements_kernel(const void* __restrict__ x, const void* __restrict__ gamma, const void* __restrict__ beta, float eps,
                           void* __restrict__ out, int64_t rows, int cols, RowStats stats) {
  constexpr int kRows = kLnThreads / GROUP, kWarps = GROUP / 32;
  __shared__ float scratch[kLnThreads / 32];
  const int t = threadIdx.x % GROUP, group = threadIdx.x / GROUP, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto sum = [&](float v) {
    v = warp_sum(v);
    if (kWarps == 1) return v;
    auto sync = [&]() {
      if (GROUP == kLnThreads) __syncthreads();
      else asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(GROUP) : "memory");
    };
    sync();  // scratch of the previous sum has been read
    if (lane == 0) scratch[warp] = v;
    sync();
    v = 0.0f;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) v += scratch[group * kWarps + k];
    return v;
  };
  for (int64_t row0 = (int64_t)blockIdx.x * kRows; row0 < rows; row0 += (int64_t)gridDim.x * kRows) {
    const int64_t row = row0 + group, base = row * cols;
    const bool live = row < rows;
    float v[VPL], s = 0.0f;
#pragma unroll
    for (int j = 0; j < VPL; ++j) v[j] = live && t + j * GROUP < cols ? Vec16<DT>::load1(x, base + t + j * GROUP) : 0.0f;
#pragma unroll
    for (int j = 0; j < VPL; ++j) s += v[j];
    const float mean = sum(s) / (float)cols;
    s = 0.0f;
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      v[j] -= mean;
      if (t + j * GROUP < cols) s = fmaf(v[j], v[j], s);
    }
    const float rstd = rsqrtf(sum(s) / (float)cols + eps);
    if (!live) continue;
    if (t == 0) {
      stats.mean[row] = mean;
      stats.rstd[row] = rstd;
    }
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      const int c = t + j * GROUP;
      if (c < cols) {
        float o = v[j] * rstd;
        if (gamma != nullptr) o = fmaf(o, Vec16<DT>::load1(gamma, c), Vec16<DT>::load1(beta, c));
        Vec16<DT>::store1(out, base + c, o);
      }
    }
  }
}

// tanh form of GELU, the one the reference's fused kernels use (cuda_kernels.cu:29-36)
__device__ __forceinline__ float gelu_tanh(float x) {
  return 0.5f * x * (1.0f + tanhf(0.7978845608028654f * (x + 0.044715f * x * x * x)));
}

template <int DT>
__global__ void __launch_bounds__(256)
add_bias_gelu_kernel(const void* x, const void* __restrict__ bias, void* out, int64_t n_vec,
                     int vec_per_row) {
  constexpr int EPV = Vec16<DT>::kElems;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n_vec; i += (int64_t)gridDim.x * 256) {
    float a[EPV], b[EPV];
    Vec16<DT>::unpack(reinterpret_cast<const uint4*>(x)[i], a);
    if (bias != nullptr) {
      Vec16<DT>::unpack(reinterpret_cast<const uint4*>(bias)[i % vec_per_row], b);
#pragma unroll
      for (int k = 0; k < EPV; ++k) a[k] += b[k];
    }
#pragma unroll
    for (int k = 0; k < EPV; ++k) a[k] = gelu_tanh(a[k]);
    reinterpret_cast<uint4*>(out)[i] = Vec16<DT>::pack(a);
  }
}

template <int DT>
__global__ void __launch_bounds__(256)
add_bias_gelu_scalar_kernel(const void* x, const void* __restrict__ bias, void* out, int64_t n,
                            int cols) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    float a = Vec16<DT>::load1(x, i);
    if (bias != nullptr) a += Vec16<DT>::load1(bias, i % cols);
    Vec16<DT>::store1(out, i, gelu_tanh(a));
  }
}

template <int DT, bool FUSED, bool STATS = false>
int launch_layer_norm(const void* x, const void* residual, const void* bias, const void* gamma, const void* beta, float eps,
                      void* out, int64_t rows, int64_t cols, cudaStream_t st, RowStats stats = {nullptr, nullptr}) {
  constexpr int EPV = Vec16<DT>::kElems;
  const bool vec_ok = cols % EPV == 0 && aligned16(x) && aligned16(out) && (residual == nullptr || aligned16(residual)) &&
                      (bias == nullptr || aligned16(bias)) && (gamma == nullptr || (aligned16(gamma) && aligned16(beta)));
  const int64_t nv = cols / EPV;
#define NTB200_LN_LAUNCH(VPL, GROUP)                                                                              \
  do {                                                                                                            \
    const int64_t rpb = kLnThreads / GROUP;                                                                       \
    const int64_t grid = (rows + rpb - 1) / rpb;                                                                  \
    if (grid > 0x7fffffff) return NTB200_INVALID_ARG;                                                             \
    if (nv == (int64_t)(VPL) * (GROUP))                                                                           \
      layer_norm_kernel<DT, VPL, GROUP, FUSED, true, STATS><<<(unsigned)grid, kLnThreads, 0, st>>>(x, residual, bias, gamma, beta, \
                                                                                           eps, out, rows, (int)cols, stats); \
    else                                                                                                          \
      layer_norm_kernel<DT, VPL, GROUP, FUSED, false, STATS><<<(unsigned)grid, kLnThreads, 0, st>>>(x, residual, bias, gamma, beta, \
                                                                                            eps, out, rows, (int)cols, stats); \
  } while (0)
  // Vectors per thread = ceil(nv / GROUP): widths such as 768, 1280 or 1536 get an exact fit (3, 5 or 6 vectors per
  // lane, no idle slots, the variant without bound tests) instead of the next power of two.  A packed 16-bit row
  // (no fused additions) stays on one warp up to 512 vectors: 16 loads in flight per lane, no block-wide reduction.
  constexpr bool kPacked = !FUSED && DT != NTB200_F32;
  if (vec_ok && nv <= 8) NTB200_LN_LAUNCH(1, 8);  // short rows: several rows per warp, every lane busy
  else if (vec_ok && nv <= 16) NTB200_LN_LAUNCH(1, 16);
  else if (vec_ok && nv <= 32) NTB200_LN_LAUNCH(1, 32);
  else if (vec_ok && nv <= 64) NTB200_LN_LAUNCH(2, 32);
  else if (vec_ok && nv <= 96) NTB200_LN_LAUNCH(3, 32);
  else if (vec_ok && nv <= 128) NTB200_LN_LAUNCH(4, 32);
  else if (vec_ok && nv <= 160) NTB200_LN_LAUNCH(5, 32);
  else if (vec_ok && nv <= 192) NTB200_LN_LAUNCH(6, 32);
  else if (vec_ok && nv <= 256) NTB200_LN_LAUNCH(8, 32);
  else if (vec_ok && kPacked && nv <= 512) {
    if constexpr (kPacked) {
      if (nv <= 384) NTB200_LN_LAUNCH(12, 32);
      else NTB200_LN_LAUNCH(16, 32);
    }
  } else if (vec_ok && nv <= 512) NTB200_LN_LAUNCH(2, kLnThreads);
  else if (vec_ok && nv <= 768) NTB200_LN_LAUNCH(3, kLnThreads);
  else if (vec_ok && nv <= 1024) NTB200_LN_LAUNCH(4, kLnThreads);
  else if (vec_ok && nv <= 1280) NTB200_LN_LAUNCH(5, kLnThreads);
  else if (vec_ok && nv <= 1536) NTB200_LN_LAUNCH(6, kLnThreads);
  else if (vec_ok && nv <= 2048) NTB200_LN_LAUNCH(8, kLnThreads);
  else if (STATS && !vec_ok && cols <= 4096) {
#define NTB200_LN_ELEMENTS(VPL, GROUP)                                                                                     \
  do {                                                                                                                     \
    const int64_t need = (rows + kLnThreads / (GROUP) - 1) / (kLnThreads / (GROUP));                                       \
    layer_norm_elements_kernel<DT, VPL, GROUP><<<(unsigned)(need < 148 * 32 ? need : 148 * 32), kLnThreads, 0, st>>>(      \
        x, gamma, beta, eps, out, rows, (int)cols, stats);                                                                 \
  } while (0)
    // (13 elements a thread beside 16: 24 000 rows of 515 bf16 take 33 us with 13 and 35 with 16, of 705 36 and 39, of 831 37 and 43)
    if (cols <= 128) NTB200_LN_ELEMENTS(4, 32);
    else if (cols <= 512) NTB200_LN_ELEMENTS(16, 32);
    else if (cols <= 832) NTB200_LN_ELEMENTS(13, 64);
    else if (cols <= 1024) NTB200_LN_ELEMENTS(16, 64);
    else if (cols <= 2048) NTB200_LN_ELEMENTS(16, 128);
    else NTB200_LN_ELEMENTS(16, 256);
#undef NTB200_LN_ELEMENTS
  } else {
    const int64_t grid = rows < 148 * 32 ? rows : 148 * 32;
    layer_norm_generic_kernel<DT><<<(unsigned)grid, kLnThreads, 0, st>>>(x, FUSED ? residual : nullptr,
                                                                        FUSED ? bias : nullptr, gamma, beta, eps, out, rows,
                                                                        (int)cols, stats);
  }
#undef NTB200_LN_LAUNCH
  return status_from_cuda(cudaGetLastError());
}

int layer_norm_entry(const void* x, const void* residual, const void* bias, const void* gamma, const void* beta, float eps,
                     void* out, int64_t rows, int64_t cols, int dtype, void* stream) {
  if (rows < 0 || cols < 0 || cols > 0x7fffffff || !(eps >= 0.0f)) return NTB200_INVALID_ARG;
  if ((gamma == nullptr) != (beta == nullptr)) return NTB200_INVALID_ARG;
  if (rows == 0 || cols == 0) return NTB200_OK;
  if (x == nullptr || out == nullptr) return NTB200_INVALID_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool fused = residual != nullptr || bias != nullptr;
  switch (dtype) {
    case NTB200_F32:
      return fused ? launch_layer_norm<NTB200_F32, true>(x, residual, bias, gamma, beta, eps, out, rows, cols, st)
                   : launch_layer_norm<NTB200_F32, false>(x, residual, bias, gamma, beta, eps, out, rows, cols, st);
    case NTB200_F16:
      return fused ? launch_layer_norm<NTB200_F16, true>(x, residual, bias, gamma, beta, eps, out, rows, cols, st)
                   : launch_layer_norm<NTB200_F16, false>(x, residual, bias, gamma, beta, eps, out, rows, cols, st);
    case NTB200_BF16:
      return fused ? launch_layer_norm<NTB200_BF16, true>(x, residual, bias, gamma, beta, eps, out, rows, cols, st)
                   : launch_layer_norm<NTB200_BF16, false>(x, residual, bias, gamma, beta, eps, out, rows, cols, st);
    default:
      return NTB200_UNSUPPORTED_DTYPE;
  }
}

template <int DT>
int launch_bias_gelu(const void* x, const void* bias, void* out, int64_t rows, int64_t cols, cudaStream_t st) {
  constexpr int EPV = Vec16<DT>::kElems;
  const int64_t n = rows * cols;
  if (cols % EPV == 0 && aligned16(x) && aligned16(out) && (bias == nullptr || aligned16(bias))) {
    const int64_t n_vec = n / EPV;
    int64_t grid = (n_vec + 255) / 256;
    if (grid > 148 * 64) grid = 148 * 64;
    add_bias_gelu_kernel<DT><<<(unsigned)grid, 256, 0, st>>>(x, bias, out, n_vec, (int)(cols / EPV));
  } else {
    int64_t grid = (n + 255) / 256;
    if (grid > 148 * 64) grid = 148 * 64;
    add_bias_gelu_scalar_kernel<DT><<<(unsigned)grid, 256, 0, st>>>(x, bias, out, n, (int)cols);
  }
  return status_from_cuda(cudaGetLastError());
}

}  // namespace
}  // namespace ntb200

extern "C" {

int ntb200_layer_norm(const void* x, const void* gamma, const void* beta, float eps, void* out, int64_t rows, int64_t cols,
                      int dtype, void* stream) {
  return ntb200::layer_norm_entry(x, nullptr, nullptr, gamma, beta, eps, out, rows, cols, dtype, stream);
}

int ntb200_layer_norm_train(const void* x, const void* gamma, const void* beta, float eps, void* out, float* mean, float* rstd,
                            int64_t rows, int64_t cols, int dtype, void* stream) {
  if (rows < 0 || cols < 0 || cols > 0x7fffffff || !(eps >= 0.0f)) return NTB200_INVALID_ARG;
  if ((gamma == nullptr) != (beta == nullptr)) return NTB200_INVALID_ARG;
  if (dtype != NTB200_F32 && dtype != NTB200_F16 && dtype != NTB200_BF16) return NTB200_UNSUPPORTED_DTYPE;
  if (rows == 0 || cols == 0) return NTB200_OK;
  if (x == nullptr || out == nullptr || mean == nullptr || rstd == nullptr) return NTB200_INVALID_ARG;
  using namespace ntb200;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const RowStats stats = {mean, rstd};
  switch (dtype) {
    case NTB200_F32: return launch_layer_norm<NTB200_F32, false, true>(x, nullptr, nullptr, gamma, beta, eps, out, rows, cols, st, stats);
    case NTB200_F16: return launch_layer_norm<NTB200_F16, false, true>(x, nullptr, nullptr, gamma, beta, eps, out, rows, cols, st, stats);
    default: return launch_layer_norm<NTB200_BF16, false, true>(x, nullptr, nullptr, gamma, beta, eps, out, rows, cols, st, stats);
  }
}

int ntb200_add_bias_residual_layer_norm(const void* x, const void* residual, const void* bias, const void* gamma,
                                        const void* beta, float eps, void* out, int64_t rows, int64_t cols, int dtype,
                                        void* stream) {
  return ntb200::layer_norm_entry(x, residual, bias, gamma, beta, eps, out, rows, cols, dtype, stream);
}

int ntb200_add_bias_gelu(const void* x, const void* bias, void* out, int64_t rows, int64_t cols, int dtype, void* stream) {
  if (rows < 0 || cols < 0 || cols > 0x7fffffff) return NTB200_INVALID_ARG;
  if (rows == 0 || cols == 0) return NTB200_OK;
  if (x == nullptr || out == nullptr) return NTB200_INVALID_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case NTB200_F32: return ntb200::launch_bias_gelu<NTB200_F32>(x, bias, out, rows, cols, st);
    case NTB200_F16: return ntb200::launch_bias_gelu<NTB200_F16>(x, bias, out, rows, cols, st);
    case NTB200_BF16: return ntb200::launch_bias_gelu<NTB200_BF16>(x, bias, out, rows, cols, st);
    default: return NTB200_UNSUPPORTED_DTYPE;
  }
}

}  // extern "C"
