// Gradients of varlen attention on packed ragged batches.  For every sequence b and head h, with a = scaling:
//
//     P = softmax(a Q K^T)    O = P V                          (the forward pass; P is not kept)
//     dV = P^T dO             dP = dO V^T
//     D  = rowsum(dO * O)     dS = P * (dP - D)                (the softmax's Jacobian: sum_j P_ij dP_ij = dO_i . O_i)
//     dQ = a dS K             dK = a dS^T Q
//
// P is computed again from the forward pass's row statistics, P_ij = 2^(a log2(e) q_i.k_j - lse_i) with lse_i the base-2
// logarithm of the row's softmax denominator, so nothing of size L x L is ever stored.
//
// A sequence's gradients are sums over its own rows only, taken in a fixed order by one block: no atomics, the same bits on
// every run and whatever the rest of the batch holds.

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "attention_internal.cuh"
#include "attention_tiny.cuh"
#include "common.cuh"

namespace ntb200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxHeadDim = 256;

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

// What every kernel of the backward pass reads and writes; strides in elements, all matrices [tokens, H * d] at head 0.
struct BwdArgs {
  const void *grad, *q, *k, *v, *out;
  const float* lse;  // [H, q_tokens]
  float* delta;      // [H, q_tokens]: D
  void *dq, *dk, *dv;
  int64_t ldq, ldk, ldv, lddq, lddk, lddv;  // grad and out are contiguous: their stride is H * d
  const int64_t *offsets_q, *offsets_k;
  int64_t row_elems_q, row_elems_k;
  int64_t batch, q_tokens;
  int H, d;
  float scaling;
};

// ------------------------------------------------------------------ work list
// items[i] = (first row of the tile, valid rows in it, first row of the sequence's other side, its length) for every `tile`
// rows of the own side (keys for dK / dV, queries for dQ), longest other side first.  A sequence whose other side is empty
// keeps its items: their gradients are zeros, written by the kernel that walks no tile at all.  One block.
constexpr int kListThreads = 1024;
constexpr int kListBuckets = 32;

__global__ void __launch_bounds__(kListThreads)
backward_items_kernel(const int64_t* __restrict__ offsets_own, int64_t row_elems_own, const int64_t* __restrict__ offsets_other,
                      int64_t row_elems_other, int64_t batch, int tile, int4* __restrict__ items, int* __restrict__ count) {
  __shared__ int s_cnt[kListBuckets], s_base[kListBuckets];
  if (threadIdx.x < kListBuckets) s_cnt[threadIdx.x] = 0;
  __syncthreads();
  auto bucket = [&](int64_t n) {  // tiles of the other side, by powers of two beyond 16
    const int t = (int)((n + tile - 1) / tile);
    return t < 16 ? t : 16 + (27 - __clz(t) < kListBuckets - 17 ? 27 - __clz(t) : kListBuckets - 17);
  };
  for (int64_t b = threadIdx.x; b < batch; b += kListThreads) {
    const int64_t n = (offsets_own[b + 1] - offsets_own[b]) / row_elems_own, m = (offsets_other[b + 1] - offsets_other[b]) / row_elems_other;
    if (n > 0) atomicAdd(&s_cnt[bucket(m)], (int)((n + tile - 1) / tile));
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int acc = 0;
    for (int k = kListBuckets - 1; k >= 0; --k) {
      s_base[k] = acc;
      acc += s_cnt[k];
    }
    *count = acc;
  }
  __syncthreads();
  for (int64_t b = threadIdx.x; b < batch; b += kListThreads) {
    const int64_t n = (offsets_own[b + 1] - offsets_own[b]) / row_elems_own, m = (offsets_other[b + 1] - offsets_other[b]) / row_elems_other;
    if (n <= 0) continue;
    const int tiles = (int)((n + tile - 1) / tile);
    const int pos = atomicAdd(&s_base[bucket(m)], tiles);  // (the order inside a bucket decides nothing but the schedule)
    const int t0 = (int)(offsets_own[b] / row_elems_own), o0 = (int)(offsets_other[b] / row_elems_other);
    for (int t = 0; t < tiles; ++t) {
      const int64_t rows = n - (int64_t)t * tile;
      items[pos + t] = make_int4(t0 + t * tile, (int)(rows < tile ? rows : tile), o0, (int)m);
    }
  }
}

// ------------------------------------------------------------------ D = rowsum(dO * O)
template <typename T>
__global__ void __launch_bounds__(256) attn_delta_kernel(BwdArgs a) {
  const int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (w >= a.q_tokens * a.H) return;
  const int64_t t = w / a.H;
  const int h = (int)(w - t * a.H);
  const int64_t base = t * ((int64_t)a.H * a.d) + (int64_t)h * a.d;
  float s = 0.0f;
  for (int i = lane; i < a.d; i += 32)
    s = fmaf(to_f32(static_cast<const T*>(a.grad)[base + i]), to_f32(static_cast<const T*>(a.out)[base + i]), s);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) a.delta[(int64_t)h * a.q_tokens + t] = s;
}

// ------------------------------------------------------------------ tiles in 32 bits, any type and head size
// One block owns BT rows r of one side and walks the other side's rows c in tiles of BT:
//     KV:  r = keys,    A_own = K, B_own = V;   c = queries, A = Q, B = dO:   dV_r += P_cr dO_c,  dK_r += dS_cr Q_c
//     !KV: r = queries, A_own = Q, B_own = dO;  c = keys,    A = K, B = V:    dQ_r += dS_cr K_c
// with S_cr = A_own,r . A_c and dP_cr = B_own,r . B_c in both.  Everything is held in fp32 in shared memory, each thread
// computes a (BT/16) x (BT/16) patch of S and dP and keeps BT/16 rows x DP/16 columns of each gradient in registers.
template <typename T, int BT, int DP>
__device__ __forceinline__ void load_rows(float* __restrict__ s, const T* __restrict__ g, int64_t ld, int rows, int d) {
  for (int i = threadIdx.x; i < BT * DP; i += 256) {
    const int r = i / DP, c = i % DP;
    s[r * (DP + 4) + c] = (r < rows && c < d) ? to_f32(g[(int64_t)r * ld + c]) : 0.0f;
  }
}

template <int BT, int DP>
constexpr int bwd_simt_smem() { return (4 * BT * (DP + 4) + 2 * BT * (BT + 4) + 2 * BT) * 4; }

template <typename T, int BT, int DP, bool KV>
__global__ void __launch_bounds__(256)
attn_bwd_simt_kernel(BwdArgs a, const int4* __restrict__ items, const int* __restrict__ count) {
  constexpr int MI = BT / 16, LD = DP + 4, LS = BT + 4, NC = DP / 16;
  extern __shared__ __align__(16) float bwd_smem[];
  float* own_a = bwd_smem;
  float* own_b = own_a + BT * LD;
  float* oth_a = own_b + BT * LD;
  float* oth_b = oth_a + BT * LD;
  float* s_p = oth_b + BT * LD;
  float* s_ds = s_p + BT * LS;
  float* s_lse = s_ds + BT * LS;
  float* s_delta = s_lse + BT;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const int64_t n = (int64_t)*count * a.H;
  const int64_t E = (int64_t)a.H * a.d;
  const float scale = a.scaling * kLog2e;
  const int d4 = (a.d + 3) & ~3;
  for (int64_t w = blockIdx.x; w < n; w += gridDim.x) {
    const int4 it = items[w / a.H];
    const int h = (int)(w % a.H);
    const int64_t col = (int64_t)h * a.d;
    const T* ga_own = (KV ? static_cast<const T*>(a.k) + it.x * a.ldk : static_cast<const T*>(a.q) + it.x * a.ldq) + col;
    const T* gb_own = (KV ? static_cast<const T*>(a.v) + it.x * a.ldv : static_cast<const T*>(a.grad) + it.x * E) + col;
    const int64_t ld_a_own = KV ? a.ldk : a.ldq, ld_b_own = KV ? a.ldv : E;
    const int64_t ld_a = KV ? a.ldq : a.ldk, ld_b = KV ? E : a.ldv;
    const float* g_lse = a.lse + (int64_t)h * a.q_tokens;
    const float* g_delta = a.delta + (int64_t)h * a.q_tokens;
    __syncthreads();  // the previous item's tiles have been read
    load_rows<T, BT, DP>(own_a, ga_own, ld_a_own, it.y, a.d);
    load_rows<T, BT, DP>(own_b, gb_own, ld_b_own, it.y, a.d);
    if (!KV && threadIdx.x < BT) {
      const bool ok = (int)threadIdx.x < it.y && it.w > 0;  // (rows without keys have no statistics)
      s_lse[threadIdx.x] = ok ? g_lse[it.x + threadIdx.x] : INFINITY;
      s_delta[threadIdx.x] = ok ? g_delta[it.x + threadIdx.x] : 0.0f;
    }
    float acc1[KV ? MI : 1][KV ? NC : 1], acc2[MI][NC];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        acc2[i][j] = 0.0f;
        if (KV) acc1[i][j] = 0.0f;
      }
    for (int c0 = 0; c0 < it.w; c0 += BT) {
      const int nc = it.w - c0 < BT ? it.w - c0 : BT;
      const int64_t o0 = (int64_t)it.z + c0;
      __syncthreads();
      load_rows<T, BT, DP>(oth_a, (KV ? static_cast<const T*>(a.q) + o0 * a.ldq : static_cast<const T*>(a.k) + o0 * a.ldk) + col, ld_a, nc, a.d);
      load_rows<T, BT, DP>(oth_b, (KV ? static_cast<const T*>(a.grad) + o0 * E : static_cast<const T*>(a.v) + o0 * a.ldv) + col, ld_b, nc, a.d);
      if (KV && threadIdx.x < BT) {
        const bool ok = (int)threadIdx.x < nc;
        s_lse[threadIdx.x] = ok ? g_lse[o0 + threadIdx.x] : INFINITY;  // 2^(x - inf) = 0: a row past the end counts nothing
        s_delta[threadIdx.x] = ok ? g_delta[o0 + threadIdx.x] : 0.0f;
      }
      __syncthreads();
      float s[MI][MI], dp[MI][MI];
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < MI; ++j) s[i][j] = dp[i][j] = 0.0f;
      auto products = [&](const float* oth, const float* own, float (&acc)[MI][MI]) {
#pragma unroll 2
        for (int c = 0; c < d4; c += 4) {
          float4 x[MI], y[MI];
#pragma unroll
          for (int i = 0; i < MI; ++i) x[i] = *reinterpret_cast<const float4*>(oth + (ty + 16 * i) * LD + c);
#pragma unroll
          for (int j = 0; j < MI; ++j) y[j] = *reinterpret_cast<const float4*>(own + (tx + 16 * j) * LD + c);
#pragma unroll
          for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < MI; ++j) {
              acc[i][j] = fmaf(x[i].x, y[j].x, acc[i][j]);
              acc[i][j] = fmaf(x[i].y, y[j].y, acc[i][j]);
              acc[i][j] = fmaf(x[i].z, y[j].z, acc[i][j]);
              acc[i][j] = fmaf(x[i].w, y[j].w, acc[i][j]);
            }
        }
      };
      products(oth_a, own_a, s);
      products(oth_b, own_b, dp);
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < MI; ++j) {
          const int c = ty + 16 * i, r = tx + 16 * j;
          const int qi = KV ? c : r;
          // a key past the end of the sequence has no probability (its zeroed row would score 0)
          const float p = (!KV && c >= nc) ? 0.0f : exp2f(fmaf(s[i][j], scale, -s_lse[qi]));
          if (KV) s_p[c * LS + r] = p;
          s_ds[c * LS + r] = p * (dp[i][j] - s_delta[qi]);
        }
      __syncthreads();
      for (int c = 0; c < nc; ++c) {
        float ds[MI], pv[MI];
#pragma unroll
        for (int i = 0; i < MI; ++i) {
          ds[i] = s_ds[c * LS + ty * MI + i];
          if (KV) pv[i] = s_p[c * LS + ty * MI + i];
        }
#pragma unroll
        for (int m = 0; m < NC / 4; ++m) {
          const float4 x = *reinterpret_cast<const float4*>(oth_a + c * LD + tx * 4 + 64 * m);
#pragma unroll
          for (int i = 0; i < MI; ++i) {
            acc2[i][4 * m] = fmaf(ds[i], x.x, acc2[i][4 * m]);
            acc2[i][4 * m + 1] = fmaf(ds[i], x.y, acc2[i][4 * m + 1]);
            acc2[i][4 * m + 2] = fmaf(ds[i], x.z, acc2[i][4 * m + 2]);
            acc2[i][4 * m + 3] = fmaf(ds[i], x.w, acc2[i][4 * m + 3]);
          }
          if (KV) {
            const float4 y = *reinterpret_cast<const float4*>(oth_b + c * LD + tx * 4 + 64 * m);
#pragma unroll
            for (int i = 0; i < MI; ++i) {
              acc1[i][4 * m] = fmaf(pv[i], y.x, acc1[i][4 * m]);
              acc1[i][4 * m + 1] = fmaf(pv[i], y.y, acc1[i][4 * m + 1]);
              acc1[i][4 * m + 2] = fmaf(pv[i], y.z, acc1[i][4 * m + 2]);
              acc1[i][4 * m + 3] = fmaf(pv[i], y.w, acc1[i][4 * m + 3]);
            }
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int r = ty * MI + i;
      if (r >= it.y) continue;
      T* o2 = (KV ? static_cast<T*>(a.dk) + (it.x + r) * a.lddk : static_cast<T*>(a.dq) + (it.x + r) * a.lddq) + col;
      T* o1 = KV ? static_cast<T*>(a.dv) + (it.x + r) * a.lddv + col : nullptr;
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        const int c = tx * 4 + 64 * (j / 4) + j % 4;
        if (c < a.d) {
          o2[c] = from_f32<T>(acc2[i][j] * a.scaling);
          if (KV) o1[c] = from_f32<T>(acc1[i][j]);
        }
      }
    }
  }
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int64_t item_capacity(int64_t batch, int64_t tokens) { return batch + tokens / 32 + 1; }  // tiles of 32 rows or more

// delta | count, KV items | count, Q items; every part on a 16-byte boundary
struct BwdWorkspace {
  size_t delta, kv, q, bytes;
  BwdWorkspace(int64_t batch, int64_t q_tokens, int64_t k_tokens, int H) {
    delta = 0;
    kv = ((size_t)q_tokens * H * 4 + 15) / 16 * 16;
    q = kv + 16 + sizeof(int4) * (size_t)item_capacity(batch, k_tokens);
    bytes = q + 16 + sizeof(int4) * (size_t)item_capacity(batch, q_tokens);
  }
};

template <typename T, int BT, int DP>
int launch_bwd_simt(const BwdArgs& a, int64_t k_tokens, uint8_t* ws, const BwdWorkspace& at, cudaStream_t st) {
  constexpr int kSmem = bwd_simt_smem<BT, DP>();
  static std::atomic<int> configured[kMaxDevices];
  if (!once_per_device(configured, [] {
        return cudaFuncSetAttribute(attn_bwd_simt_kernel<T, BT, DP, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) == cudaSuccess &&
               cudaFuncSetAttribute(attn_bwd_simt_kernel<T, BT, DP, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) == cudaSuccess;
      }))
    return NTB200_LAUNCH_FAILED;
  int *n_kv = reinterpret_cast<int*>(ws + at.kv), *n_q = reinterpret_cast<int*>(ws + at.q);
  int4 *kv = reinterpret_cast<int4*>(ws + at.kv + 16), *qi = reinterpret_cast<int4*>(ws + at.q + 16);
  const int per_sm = 227 * 1024 / (kSmem + 1024);
  auto grid = [&](int64_t tokens) {
    const int64_t most = (a.batch + tokens / BT + 1) * a.H;
    return (unsigned)(most < (int64_t)kNumSMs * per_sm ? most : (int64_t)kNumSMs * per_sm);
  };
  if (k_tokens > 0) {
    backward_items_kernel<<<1, kListThreads, 0, st>>>(a.offsets_k, a.row_elems_k, a.offsets_q, a.row_elems_q, a.batch, BT, kv, n_kv);
    attn_bwd_simt_kernel<T, BT, DP, true><<<grid(k_tokens), 256, kSmem, st>>>(a, kv, n_kv);
  }
  if (a.q_tokens > 0) {
    backward_items_kernel<<<1, kListThreads, 0, st>>>(a.offsets_q, a.row_elems_q, a.offsets_k, a.row_elems_k, a.batch, BT, qi, n_q);
    attn_bwd_simt_kernel<T, BT, DP, false><<<grid(a.q_tokens), 256, kSmem, st>>>(a, qi, n_q);
  }
  return status_from_cuda(cudaGetLastError());
}

template <typename T>
int launch_bwd(const BwdArgs& a, int64_t k_tokens, uint8_t* ws, const BwdWorkspace& at, cudaStream_t st) {
  if (a.q_tokens > 0 && k_tokens > 0) {
    const int64_t blocks = ceil_div(a.q_tokens * a.H, 8);
    if (blocks > 0x7fffffffll) return NTB200_UNSUPPORTED_SHAPE;
    attn_delta_kernel<T><<<(unsigned)blocks, 256, 0, st>>>(a);
  }
  if (a.d <= 64) return launch_bwd_simt<T, 64, 64>(a, k_tokens, ws, at, st);
  if (a.d <= 128) return launch_bwd_simt<T, 64, 128>(a, k_tokens, ws, at, st);
  return launch_bwd_simt<T, 32, 256>(a, k_tokens, ws, at, st);
}

}  // namespace
}  // namespace ntb200

using namespace ntb200;

extern "C" {

size_t ntb200_varlen_attention_backward_workspace_bytes(int64_t batch, int64_t q_tokens, int64_t k_tokens, int num_heads, int head_dim,
                                                        int dtype) {
  (void)head_dim, (void)dtype;
  if (batch <= 0 || q_tokens < 0 || k_tokens < 0 || num_heads < 1) return 0;
  return BwdWorkspace(batch, q_tokens, k_tokens, num_heads).bytes;
}

int ntb200_varlen_attention_backward(const void* grad_out, const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv,
                                     const void* out, const float* lse, void* grad_q, int64_t ld_grad_q, void* grad_k, int64_t ld_grad_k,
                                     void* grad_v, int64_t ld_grad_v, const int64_t* offsets_q, int64_t row_elems_q,
                                     const int64_t* offsets_k, int64_t row_elems_k, int64_t batch, int64_t q_tokens, int64_t k_tokens,
                                     int num_heads, int head_dim, int64_t max_len_q, int64_t max_len_k, float scaling, int dtype, int path,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  if (batch < 0 || q_tokens < 0 || k_tokens < 0 || num_heads < 1 || head_dim < 1 || row_elems_q < 1 || row_elems_k < 1 || max_len_q < 0 ||
      max_len_k < 0 || path < 0 || path > 1)
    return NTB200_INVALID_ARG;
  if (dtype != NTB200_F32 && dtype != NTB200_F16 && dtype != NTB200_BF16) return NTB200_UNSUPPORTED_DTYPE;
  if (head_dim > kMaxHeadDim) return NTB200_UNSUPPORTED_SHAPE;
  const int64_t E = (int64_t)num_heads * head_dim;
  if (ldq < E || ldk < E || ldv < E || ld_grad_q < E || ld_grad_k < E || ld_grad_v < E) return NTB200_INVALID_ARG;
  if (batch == 0 || (q_tokens == 0 && k_tokens == 0)) return NTB200_OK;
  if (q_tokens >= (1ll << 31) - 256 || k_tokens >= (1ll << 31) - 256 || batch >= (1ll << 31) - 256) return NTB200_UNSUPPORTED_SHAPE;
  if (offsets_q == nullptr || offsets_k == nullptr || workspace == nullptr) return NTB200_INVALID_ARG;
  if (q_tokens > 0 && (grad_out == nullptr || q == nullptr || out == nullptr || lse == nullptr || grad_q == nullptr)) return NTB200_INVALID_ARG;
  if (k_tokens > 0 && (k == nullptr || v == nullptr || grad_k == nullptr || grad_v == nullptr)) return NTB200_INVALID_ARG;
  const BwdWorkspace at(batch, q_tokens, k_tokens, num_heads);
  if (workspace_bytes < at.bytes) return NTB200_WORKSPACE_TOO_SMALL;
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return NTB200_MISALIGNED;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const BwdArgs a = {grad_out, q, k, v, out, lse, reinterpret_cast<float*>(ws + at.delta), grad_q, grad_k, grad_v,
                     ldq, ldk, ldv, ld_grad_q, ld_grad_k, ld_grad_v, offsets_q, offsets_k, row_elems_q, row_elems_k,
                     batch, q_tokens, num_heads, head_dim, scaling};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case NTB200_F32: return launch_bwd<float>(a, k_tokens, ws, at, st);
    case NTB200_F16: return launch_bwd<__half>(a, k_tokens, ws, at, st);
    default: return launch_bwd<__nv_bfloat16>(a, k_tokens, ws, at, st);
  }
}

}  // extern "C"
