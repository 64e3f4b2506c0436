// Gradients of LayerNorm over the rows of the packed token matrix [T = sum(L_i), E]:
//
//     n  = (x - mean) rstd        gw = g gamma
//     dx = rstd (gw - mean(gw) - n mean(gw n))      per row
//     dgamma = sum_t g n          dbeta = sum_t g   per column
//
// One pass reads x and g and writes dx (HBM-bound: 3 T E elements); mean and rstd come from the forward pass (8 bytes a row).
// A row is held in registers by the GROUP threads that share it, and the same threads always hold the same columns, so the
// column sums stay in their registers (fp32) over all rows of a persistent block; every block leaves one [2, E] partial, and a
// second, small kernel adds the partials in block order.  No atomics: the same bits on every run.
//
// Measured: 976 000 rows of 1024 bf16 in 942 us alone (6.4 TB/s, 0.97 of a copy), 1040 back to back with the forward pass; 37 000 of
// 768 fp16 in 43 us (4.0 TB/s): 18 us of that do not depend on the rows (4 700 take 19, 75 000 70, 303 000 224; the rest goes at
// 6.8 TB/s), and most of those are the column sums at the end, eight turns of a block with a barrier after each (30 % of the warps' time
// is spent at barriers, of which the rows have none); 24 000 of 771 bf16, element by element, in 56 us (2.0 TB/s, bound by
// instruction issue).  Rows that neither form holds in registers are read again: 20 000 of 8200 bf16 take 900 us (1.1 TB/s) and of
// 4100 462, where 8192 take 212.

#include "row_vec.cuh"

namespace ntb200 {
namespace {

constexpr int kBlock = 256;

// One row's access unit: EPV consecutive elements (16 bytes, or one element where rows are not made of whole vectors).
template <int DT, int EPV>
struct Unit {
  using Raw = uint4;
  static __device__ __forceinline__ Raw load(const void* p, int64_t i) { return reinterpret_cast<const uint4*>(p)[i]; }
  static __device__ __forceinline__ void unpack(const Raw& r, float* f) { Vec16<DT>::unpack(r, f); }
  static __device__ __forceinline__ void store(void* p, int64_t i, const float* f) { reinterpret_cast<uint4*>(p)[i] = Vec16<DT>::pack(f); }
  static __device__ __forceinline__ Raw zero() { return make_uint4(0u, 0u, 0u, 0u); }
};
template <int DT>
struct Unit<DT, 1> {
  using Raw = float;
  static __device__ __forceinline__ Raw load(const void* p, int64_t i) { return Vec16<DT>::load1(p, i); }
  static __device__ __forceinline__ void unpack(const Raw& r, float* f) { f[0] = r; }
  static __device__ __forceinline__ void store(void* p, int64_t i, const float* f) { Vec16<DT>::store1(p, i, f[0]); }
  static __device__ __forceinline__ Raw zero() { return 0.0f; }
};

// Sums of a and b over the GROUP neighbouring threads that share a row.  GROUP > 32: whole warps, through `scratch` and (GROUP <
// the block) a named barrier of their own.
template <int GROUP>
__device__ __forceinline__ void group_sum2(float& a, float& b, float2* scratch) {
#pragma unroll
  for (int o = (GROUP < 32 ? GROUP : 32) / 2; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  if (GROUP <= 32) return;
  constexpr int kWarps = GROUP / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = threadIdx.x / GROUP;
  auto sync = [&]() {
    if (GROUP == kBlock) __syncthreads();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(GROUP) : "memory");
  };
  sync();  // scratch of the previous row has been read
  if (lane == 0) scratch[warp] = make_float2(a, b);
  sync();
  a = b = 0.0f;
#pragma unroll
  for (int k = 0; k < kWarps; ++k) {
    const float2 v = scratch[group * kWarps + k];
    a += v.x;
    b += v.y;
  }
}

__device__ __forceinline__ void copy_async_16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// AFFINE: gamma given and column sums wanted.  nv = units per row (cols / EPV).  Rows of a warp (whole vectors) come through two
// shared-memory stages per warp, the next row's copies in flight under the current row's arithmetic: the accumulators leave
// registers for only 16 warps an SM, whose own loads did not keep the memory busy (976 000 rows of 1024 bf16: 1090 us without).
template <int DT, int EPV, int VPL, int GROUP, bool AFFINE>
__global__ void __launch_bounds__(kBlock, 2)
layer_norm_backward_kernel(const void* __restrict__ grad, const void* __restrict__ x, const float* __restrict__ mean,
                           const float* __restrict__ rstd, const void* __restrict__ gamma, void* __restrict__ dx,
                           float* __restrict__ partial, int64_t rows, int nv) {
  using U = Unit<DT, EPV>;
  constexpr int kRows = kBlock / GROUP;  // rows a block works on at a time
  // whole vectors keep gamma in shared memory (in registers it spilled at 32 columns a thread), single elements in registers
  constexpr bool kGammaSmem = AFFINE && EPV > 1;
  constexpr bool kAsync = EPV > 1 && GROUP == 32;
  extern __shared__ __align__(16) float ln_smem[];  // kAsync: stages; kGammaSmem: gamma; then [2, cols] column sums of the block's warps
  constexpr int kStageFloats = kAsync ? (kBlock / 32) * 2 * 2 * VPL * 32 * 4 : 0;
  __shared__ float2 scratch[8];
  const int t = threadIdx.x % GROUP;
  const float inv_cols = 1.0f / (float)(nv * EPV);
  typename U::Raw gam[kGammaSmem ? 1 : VPL];
  typename U::Raw* s_gam = reinterpret_cast<typename U::Raw*>(ln_smem + kStageFloats);
  float* s_cols = ln_smem + kStageFloats + (kGammaSmem ? nv * (int)(sizeof(typename U::Raw) / sizeof(float)) : 0);
  if (kGammaSmem) {
    for (int v = threadIdx.x; v < nv; v += kBlock) s_gam[v] = U::load(gamma, v);
    __syncthreads();
  }
  float acc_g[AFFINE ? VPL * EPV : 1], acc_b[AFFINE ? VPL * EPV : 1];
#pragma unroll
  for (int j = 0; j < (kGammaSmem ? 1 : VPL); ++j) {
    gam[j] = U::zero();
    if (AFFINE && !kGammaSmem && t + j * GROUP < nv) gam[j] = U::load(gamma, t + j * GROUP);
  }
#pragma unroll
  for (int k = 0; k < (AFFINE ? VPL * EPV : 1); ++k) acc_g[k] = acc_b[k] = 0.0f;

  const int64_t step = (int64_t)gridDim.x * kRows;
  // stage st of this warp: x, then g, a lane's vector j at j * 512 + lane * 16 (a lane reads only what it copied itself)
  const uint32_t stage0 = (uint32_t)__cvta_generic_to_shared(ln_smem) + (threadIdx.x >> 5) * (2 * 2 * VPL * 512) + (threadIdx.x & 31) * 16;
  float mu_next = 0.0f, rs_next = 0.0f;
  auto request = [&](int64_t row, int st) {
    if (row < rows) {
#pragma unroll
      for (int j = 0; j < VPL; ++j) {
        const int v = t + j * GROUP;
        if (v < nv) {
          copy_async_16(stage0 + (st * 2) * (VPL * 512) + j * 512, reinterpret_cast<const uint4*>(x) + row * nv + v);
          copy_async_16(stage0 + (st * 2 + 1) * (VPL * 512) + j * 512, reinterpret_cast<const uint4*>(grad) + row * nv + v);
        }
      }
      mu_next = mean[row];
      rs_next = rstd[row];
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  int st = 0;
  if constexpr (kAsync) request((int64_t)blockIdx.x * kRows + threadIdx.x / GROUP, 0);
  // (whole warps stay in the loop until their last row is done: a warp of several short rows may hold live and dead ones)
  for (int64_t row0 = (int64_t)blockIdx.x * kRows; row0 < rows; row0 += step) {
    const int64_t row = row0 + threadIdx.x / GROUP;
    const bool live = row < rows;
    const int64_t base = row * nv;
    typename U::Raw xr[VPL], gr[VPL];
    float mu = mu_next, rs = rs_next;
    if constexpr (kAsync) {
      request(row + step, st ^ 1);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
#pragma unroll
      for (int j = 0; j < VPL; ++j) {
        xr[j] = gr[j] = U::zero();
        if (live && t + j * GROUP < nv) {
          const uint32_t at = stage0 + (st * 2) * (VPL * 512) + j * 512;
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(xr[j].x), "=r"(xr[j].y), "=r"(xr[j].z), "=r"(xr[j].w) : "r"(at) : "memory");
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(gr[j].x), "=r"(gr[j].y), "=r"(gr[j].z), "=r"(gr[j].w)
                       : "r"(at + VPL * 512)
                       : "memory");
        }
      }
      st ^= 1;
    } else {
#pragma unroll
      for (int j = 0; j < VPL; ++j) {
        const int v = t + j * GROUP;
        xr[j] = gr[j] = U::zero();
        if (live && v < nv) {
          xr[j] = U::load(x, base + v);
          gr[j] = U::load(grad, base + v);
        }
      }
      mu = live ? mean[row] : 0.0f, rs = live ? rstd[row] : 0.0f;
    }
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      if (live && t + j * GROUP < nv) {
        float xf[EPV], gf[EPV], wf[EPV];
        U::unpack(xr[j], xf);
        U::unpack(gr[j], gf);
        U::unpack(kGammaSmem ? s_gam[t + j * GROUP] : gam[kGammaSmem ? 0 : j], wf);
#pragma unroll
        for (int k = 0; k < EPV; ++k) {
          const float n = (xf[k] - mu) * rs;
          const float gw = AFFINE ? gf[k] * wf[k] : gf[k];
          s1 += gw;
          s2 = fmaf(gw, n, s2);
          if (AFFINE) {
            acc_g[j * EPV + k] = fmaf(gf[k], n, acc_g[j * EPV + k]);
            acc_b[j * EPV + k] += gf[k];
          }
        }
      }
    }
    group_sum2<GROUP>(s1, s2, scratch);
    if (dx == nullptr || !live) continue;
    const float c1 = s1 * inv_cols, c2 = s2 * inv_cols;
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      const int v = t + j * GROUP;
      if (v < nv) {
        float xf[EPV], gf[EPV], wf[EPV];
        U::unpack(xr[j], xf);
        U::unpack(gr[j], gf);
        U::unpack(kGammaSmem ? s_gam[t + j * GROUP] : gam[kGammaSmem ? 0 : j], wf);
#pragma unroll
        for (int k = 0; k < EPV; ++k) {
          const float n = (xf[k] - mu) * rs;
          const float gw = AFFINE ? gf[k] * wf[k] : gf[k];
          gf[k] = rs * (gw - c1 - n * c2);
        }
        U::store(dx, base + v, gf);
      }
    }
  }

  if constexpr (AFFINE) {
    const int cols = nv * EPV;
    float* out = partial + (int64_t)blockIdx.x * 2 * cols;
    if constexpr (kRows == 1) {  // every column belongs to one thread
#pragma unroll
      for (int j = 0; j < VPL; ++j) {
        const int v = t + j * GROUP;
        if (v < nv) {
#pragma unroll
          for (int k = 0; k < EPV; ++k) {
            out[v * EPV + k] = acc_g[j * EPV + k];
            out[cols + v * EPV + k] = acc_b[j * EPV + k];
          }
        }
      }
    } else {
      // rows of one warp first (GROUP < 32), then the warps in turn
#pragma unroll
      for (int k = 0; k < VPL * EPV; ++k) {
#pragma unroll
        for (int o = 16; o >= GROUP && o > 0; o >>= 1) {
          acc_g[k] += __shfl_xor_sync(0xffffffffu, acc_g[k], o);
          acc_b[k] += __shfl_xor_sync(0xffffffffu, acc_b[k], o);
        }
      }
      const int lane = threadIdx.x & 31;
      constexpr int kTurn = GROUP < 32 ? 32 : GROUP;  // threads that add their columns at a time
      for (int w = 0; w < kBlock / kTurn; ++w) {
        if ((int)threadIdx.x / kTurn == w && (GROUP >= 32 || lane < GROUP)) {
#pragma unroll
          for (int j = 0; j < VPL; ++j) {
            const int v = t + j * GROUP;
            if (v < nv) {
#pragma unroll
              for (int k = 0; k < EPV; ++k) {
                float* g = s_cols + v * EPV + k;
                *g = (w == 0 ? 0.0f : *g) + acc_g[j * EPV + k];
                g[cols] = (w == 0 ? 0.0f : g[cols]) + acc_b[j * EPV + k];
              }
            }
          }
        }
        __syncthreads();
      }
      for (int i = threadIdx.x; i < 2 * cols; i += kBlock) out[i] = s_cols[i];
    }
  }
}

// Any row length: one block per row for dx (three passes over the row), ...
template <int DT>
__global__ void __launch_bounds__(kBlock)
layer_norm_backward_rows_kernel(const void* __restrict__ grad, const void* __restrict__ x, const float* __restrict__ mean,
                                const float* __restrict__ rstd, const void* __restrict__ gamma, void* __restrict__ dx, int64_t rows,
                                int64_t cols) {
  __shared__ float2 scratch[8];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const int64_t base = row * cols;
    const float mu = mean[row], rs = rstd[row];
    float s1 = 0.0f, s2 = 0.0f;
    for (int64_t i = threadIdx.x; i < cols; i += kBlock) {
      const float n = (Vec16<DT>::load1(x, base + i) - mu) * rs;
      const float gw = Vec16<DT>::load1(grad, base + i) * (gamma != nullptr ? Vec16<DT>::load1(gamma, i) : 1.0f);
      s1 += gw;
      s2 = fmaf(gw, n, s2);
    }
    group_sum2<kBlock>(s1, s2, scratch);
    const float c1 = s1 / (float)cols, c2 = s2 / (float)cols;
    for (int64_t i = threadIdx.x; i < cols; i += kBlock) {
      const float n = (Vec16<DT>::load1(x, base + i) - mu) * rs;
      const float gw = Vec16<DT>::load1(grad, base + i) * (gamma != nullptr ? Vec16<DT>::load1(gamma, i) : 1.0f);
      Vec16<DT>::store1(dx, base + i, rs * (gw - c1 - n * c2));
    }
  }
}

// ... and one thread per column and block of rows for the column sums.
template <int DT>
__global__ void __launch_bounds__(kBlock)
layer_norm_backward_columns_kernel(const void* __restrict__ grad, const void* __restrict__ x, const float* __restrict__ mean,
                                   const float* __restrict__ rstd, float* __restrict__ partial, int64_t rows, int64_t cols) {
  const int64_t c = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  if (c >= cols) return;
  const int64_t per = (rows + gridDim.y - 1) / gridDim.y;
  const int64_t r0 = blockIdx.y * per, r1 = r0 + per < rows ? r0 + per : rows;
  float g = 0.0f, b = 0.0f;
  for (int64_t r = r0; r < r1; ++r) {
    const float v = Vec16<DT>::load1(grad, r * cols + c);
    g = fmaf(v, (Vec16<DT>::load1(x, r * cols + c) - mean[r]) * rstd[r], g);
    b += v;
  }
  float* out = partial + (int64_t)blockIdx.y * 2 * cols;
  out[c] = g;
  out[cols + c] = b;
}

// out[c] = sum over the blocks' partials, in a fixed order: 32 running sums a column (one per warp), then those in turn.
constexpr int kReduceWarps = 32;
template <int DT>
__global__ void __launch_bounds__(kReduceWarps * 32)
layer_norm_backward_reduce_kernel(const float* __restrict__ partial, int blocks, void* __restrict__ dgamma, void* __restrict__ dbeta,
                                  int64_t cols) {
  __shared__ float s[kReduceWarps][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  float a = 0.0f;
  if (c < 2 * cols) {
#pragma unroll 8
    for (int k = warp; k < blocks; k += kReduceWarps) a += partial[(int64_t)k * 2 * cols + c];
  }
  s[warp][lane] = a;
  __syncthreads();
  if (warp != 0 || c >= 2 * cols) return;
#pragma unroll
  for (int w = 1; w < kReduceWarps; ++w) a += s[w][lane];
  if (c < cols) {
    if (dgamma != nullptr) Vec16<DT>::store1(dgamma, c, a);
  } else if (dbeta != nullptr) {
    Vec16<DT>::store1(dbeta, c - cols, a);
  }
}

constexpr int kMaxPartials = 4 * kNumSMs;  // most blocks that leave a partial

struct BwdCall {
  const void *grad, *x;
  const float *mean, *rstd;
  const void* gamma;
  void *dx, *dgamma, *dbeta;
  float* partial;
  int64_t rows, cols;
};

// the blocks that are resident at once, queried once per device and kernel
template <typename F>
int resident_blocks(F kernel, int threads, size_t smem, std::atomic<int>* cache) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return kNumSMs;
  int n = cache[dev].load(std::memory_order_relaxed);
  if (n > 0) return n;
  int per_sm = 0, sms = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, smem) != cudaSuccess || per_sm < 1) per_sm = 1;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms < 1) sms = kNumSMs;
  n = per_sm * sms;
  cache[dev].store(n, std::memory_order_relaxed);
  return n;
}

template <int DT, int EPV, int VPL, int GROUP, bool AFFINE>
int launch_rows(const BwdCall& c, int* blocks, cudaStream_t st) {
  constexpr int kRows = kBlock / GROUP;
  // the stages of the rows of warps, gamma (whole vectors) and the column sums of several rows' threads
  constexpr int kStageBytes = EPV > 1 && GROUP == 32 ? (kBlock / 32) * 2 * 2 * VPL * 512 : 0;
  constexpr int kPerUnit = (AFFINE && EPV > 1 ? 16 : 0) + (AFFINE && kRows > 1 ? 2 * EPV * (int)sizeof(float) : 0);
  constexpr int kMostSmem = kStageBytes + GROUP * VPL * kPerUnit;  // 74 KB at most
  const size_t smem = kStageBytes + (size_t)(c.cols / EPV) * kPerUnit;
  auto kernel = layer_norm_backward_kernel<DT, EPV, VPL, GROUP, AFFINE>;
  if (kMostSmem > 48 * 1024) {
    static std::atomic<int> configured[kMaxDevices];
    if (!once_per_device(configured, [] {
          return cudaFuncSetAttribute(layer_norm_backward_kernel<DT, EPV, VPL, GROUP, AFFINE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      kMostSmem) == cudaSuccess;
        }))
      return NTB200_LAUNCH_FAILED;
  }
  static std::atomic<int> cache[kMaxDevices];
  int64_t grid = resident_blocks(kernel, kBlock, kMostSmem, cache);
  if (grid > kMaxPartials) grid = kMaxPartials;
  const int64_t need = (c.rows + kRows - 1) / kRows;
  if (grid > need) grid = need;
  *blocks = (int)grid;
  kernel<<<(unsigned)grid, kBlock, smem, st>>>(c.grad, c.x, c.mean, c.rstd, c.gamma, c.dx, c.partial, c.rows, (int)(c.cols / EPV));
  return status_from_cuda(cudaGetLastError());
}

template <int DT, bool AFFINE>
int launch_backward(const BwdCall& c, int* blocks, cudaStream_t st) {
  constexpr int EPV = Vec16<DT>::kElems;
  const bool vec = c.cols % EPV == 0 && aligned16(c.grad) && aligned16(c.x) && (c.dx == nullptr || aligned16(c.dx)) &&
                   (c.gamma == nullptr || aligned16(c.gamma));
  const int64_t nv = c.cols / EPV;
  if (vec) {
    if (nv <= 8) return launch_rows<DT, EPV, 1, 8, AFFINE>(c, blocks, st);
    if (nv <= 16) return launch_rows<DT, EPV, 1, 16, AFFINE>(c, blocks, st);
    if (nv <= 32) return launch_rows<DT, EPV, 1, 32, AFFINE>(c, blocks, st);
    if (nv <= 64) return launch_rows<DT, EPV, 2, 32, AFFINE>(c, blocks, st);
    if (nv <= 96) return launch_rows<DT, EPV, 3, 32, AFFINE>(c, blocks, st);
    if (nv <= 128) return launch_rows<DT, EPV, 4, 32, AFFINE>(c, blocks, st);
    if (nv <= 192) return launch_rows<DT, EPV, 3, 64, AFFINE>(c, blocks, st);
    if (nv <= 256) return launch_rows<DT, EPV, 4, 64, AFFINE>(c, blocks, st);
    if (nv <= 384) return launch_rows<DT, EPV, 3, 128, AFFINE>(c, blocks, st);
    if (nv <= 512) return launch_rows<DT, EPV, 4, 128, AFFINE>(c, blocks, st);
    if (nv <= 768) return launch_rows<DT, EPV, 3, 256, AFFINE>(c, blocks, st);
    if (nv <= 1024) return launch_rows<DT, EPV, 4, 256, AFFINE>(c, blocks, st);
  } else {
    // (13 elements a thread beside 16: the two sums of each are registers too.  24 000 rows of 515 bf16 take 47 us with 13 and 56 with
    // 16, of 705 55 and 66, of 831 58 and 72; in fp32 the two are within 1.5 us)
    if (c.cols <= 128) return launch_rows<DT, 1, 4, 32, AFFINE>(c, blocks, st);
    if (c.cols <= 256) return launch_rows<DT, 1, 8, 32, AFFINE>(c, blocks, st);
    if (c.cols <= 512) return launch_rows<DT, 1, 8, 64, AFFINE>(c, blocks, st);
    if (c.cols <= 832) return launch_rows<DT, 1, 13, 64, AFFINE>(c, blocks, st);
    if (c.cols <= 1024) return launch_rows<DT, 1, 16, 64, AFFINE>(c, blocks, st);
    if (c.cols <= 2048) return launch_rows<DT, 1, 16, 128, AFFINE>(c, blocks, st);
    if (c.cols <= 4096) return launch_rows<DT, 1, 16, 256, AFFINE>(c, blocks, st);
  }
  if (c.dx != nullptr) {
    const int64_t grid = c.rows < kNumSMs * 8 ? c.rows : kNumSMs * 8;
    layer_norm_backward_rows_kernel<DT><<<(unsigned)grid, kBlock, 0, st>>>(c.grad, c.x, c.mean, c.rstd, c.gamma, c.dx, c.rows, c.cols);
  }
  if (AFFINE) {
    const int64_t gx = (c.cols + kBlock - 1) / kBlock;
    int64_t gy = kMaxPartials / gx;
    gy = gy < 1 ? 1 : (gy > c.rows ? c.rows : gy);
    *blocks = (int)gy;
    layer_norm_backward_columns_kernel<DT><<<dim3((unsigned)gx, (unsigned)gy), kBlock, 0, st>>>(c.grad, c.x, c.mean, c.rstd, c.partial,
                                                                                             c.rows, c.cols);
  }
  return status_from_cuda(cudaGetLastError());
}

template <int DT>
int backward(const BwdCall& c, cudaStream_t st) {
  // (without a gradient of gamma or beta to write, gamma still enters dx: the columns' sums are then made for nothing, and small)
  const bool affine = c.gamma != nullptr;
  int blocks = 0;
  if (c.rows > 0) {
    const int rc = affine ? launch_backward<DT, true>(c, &blocks, st) : launch_backward<DT, false>(c, &blocks, st);
    if (rc != NTB200_OK) return rc;
  }
  if (affine && (c.dgamma != nullptr || c.dbeta != nullptr)) {
    const int64_t grid = (2 * c.cols + 31) / 32;
    layer_norm_backward_reduce_kernel<DT><<<(unsigned)grid, kReduceWarps * 32, 0, st>>>(c.partial, blocks, c.dgamma, c.dbeta, c.cols);
  }
  return status_from_cuda(cudaGetLastError());
}

}  // namespace
}  // namespace ntb200

using namespace ntb200;

extern "C" {

size_t ntb200_layer_norm_backward_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  const int64_t blocks = rows < kMaxPartials ? rows : kMaxPartials;
  return (size_t)blocks * 2 * (size_t)cols * sizeof(float);
}

int ntb200_layer_norm_backward(const void* grad, const void* x, const float* mean, const float* rstd, const void* gamma, void* grad_x,
                               void* grad_gamma, void* grad_beta, int64_t rows, int64_t cols, int dtype, void* workspace,
                               size_t workspace_bytes, void* stream) {
  if (rows < 0 || cols < 0 || cols > 0x7fffffff - 256) return NTB200_INVALID_ARG;
  if (dtype != NTB200_F32 && dtype != NTB200_F16 && dtype != NTB200_BF16) return NTB200_UNSUPPORTED_DTYPE;
  if (gamma == nullptr && (grad_gamma != nullptr || grad_beta != nullptr)) return NTB200_INVALID_ARG;
  if (cols == 0 || (rows == 0 && grad_gamma == nullptr && grad_beta == nullptr)) return NTB200_OK;
  if (rows > 0 && (grad == nullptr || x == nullptr || mean == nullptr || rstd == nullptr)) return NTB200_INVALID_ARG;
  if (gamma != nullptr && rows > 0) {
    if (workspace == nullptr || workspace_bytes < ntb200_layer_norm_backward_workspace_bytes(rows, cols)) return NTB200_WORKSPACE_TOO_SMALL;
    if (reinterpret_cast<uintptr_t>(workspace) & 3) return NTB200_MISALIGNED;
  }
  const BwdCall c = {grad, x, mean, rstd, gamma, grad_x, grad_gamma, grad_beta, static_cast<float*>(workspace), rows, cols};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case NTB200_F32: return backward<NTB200_F32>(c, st);
    case NTB200_F16: return backward<NTB200_F16>(c, st);
    default: return backward<NTB200_BF16>(c, st);
  }
}

}  // extern "C"
