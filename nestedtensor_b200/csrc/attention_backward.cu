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
// A sequence's gradients are sums over its own rows only, taken in a fixed order by one block, and its kernel is chosen by its own
// lengths: no atomics, the same bits on every run and whatever the rest of the batch holds.

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cfloat>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "attention_backward.cuh"
#include "attention_internal.cuh"
#include "attention_tiny.cuh"
#include "common.cuh"
#include "row_vec.cuh"

namespace ntb200 {
namespace {

// ------------------------------------------------------------------ work lists and D = rowsum(dO * O), one launch
// Which kernel takes a sequence depends on its own lengths only, so that a batch cut in parts gives the bits of the whole.  A class
// of sequences: longest side in (over, to].
struct Class {
  int64_t over, to;
  __host__ __device__ bool any() const { return to > over; }
  __device__ __forceinline__ bool has(int64_t n, int64_t m) const {
    const int64_t l = n > m ? n : m;
    return l > over && l <= to;
  }
};

// An item for every `tile` rows of the own side (keys for dK / dV, queries for dQ) of the class's sequences, longest other side first.
// A sequence whose other side is empty keeps its items: their gradients are zeros, written by a block that walks no tile at
// all.  One block.
constexpr int kListBuckets = 32;
constexpr int kPrepThreads = 256;

__device__ __forceinline__ void build_backward_items(const int64_t* __restrict__ offsets_own, int64_t row_elems_own,
                                                     const int64_t* __restrict__ offsets_other, int64_t row_elems_other, int64_t batch,
                                                     int tile, const Class& cls, const ListOut& out) {
  __shared__ int s_cnt[kListBuckets], s_base[kListBuckets];
  if (threadIdx.x < kListBuckets) s_cnt[threadIdx.x] = 0;
  __syncthreads();
  auto bucket = [&](int64_t n) {  // tiles of the other side, by powers of two beyond 16
    const int t = (int)((n + tile - 1) / tile);
    return t < 16 ? t : 16 + (27 - __clz(t) < kListBuckets - 17 ? 27 - __clz(t) : kListBuckets - 17);
  };
  for (int64_t b = threadIdx.x; b < batch; b += kPrepThreads) {
    const int64_t n = (offsets_own[b + 1] - offsets_own[b]) / row_elems_own, m = (offsets_other[b + 1] - offsets_other[b]) / row_elems_other;
    if (n > 0 && cls.has(n, m)) atomicAdd(&s_cnt[bucket(m)], (int)((n + tile - 1) / tile));
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int acc = 0;
    for (int k = kListBuckets - 1; k >= 0; --k) {
      s_base[k] = acc;
      acc += s_cnt[k];
    }
    *out.count = acc;
  }
  __syncthreads();
  for (int64_t b = threadIdx.x; b < batch; b += kPrepThreads) {
    const int64_t n = (offsets_own[b + 1] - offsets_own[b]) / row_elems_own, m = (offsets_other[b + 1] - offsets_other[b]) / row_elems_other;
    if (n <= 0 || !cls.has(n, m)) continue;
    const int tiles = (int)((n + tile - 1) / tile);
    const int pos = atomicAdd(&s_base[bucket(m)], tiles);  // (the order inside a bucket decides nothing but the schedule)
    const int t0 = (int)(offsets_own[b] / row_elems_own), o0 = (int)(offsets_other[b] / row_elems_other);
    for (int t = 0; t < tiles; ++t) {
      const int64_t rows = n - (int64_t)t * tile;
      out.items[pos + t] = make_int4(t0 + t * tile, (int)(rows < tile ? rows : tile), o0, (int)m);
      out.seq[pos + t] = (int)b;
    }
  }
}

__global__ void __launch_bounds__(kPrepThreads) query_items_kernel(BwdArgs a, int tile, ListOut l) {
  build_backward_items(a.offsets_q, a.row_elems_q, a.offsets_k, a.row_elems_k, a.batch, tile, Class{0, INT64_MAX}, l);
}

// An item for every sequence of the class: (first key, keys, first query, queries), most tile pairs first.  One block.
__device__ __forceinline__ void build_sequence_items(const BwdArgs& a, const Class& cls, const ListOut& out) {
  __shared__ int s_cnt[kListBuckets], s_base[kListBuckets];
  if (threadIdx.x < kListBuckets) s_cnt[threadIdx.x] = 0;
  __syncthreads();
  auto lengths = [&](int64_t b) {
    const int q0 = (int)(a.offsets_q[b] / a.row_elems_q), k0 = (int)(a.offsets_k[b] / a.row_elems_k);
    return make_int4(k0, (int)(a.offsets_k[b + 1] / a.row_elems_k) - k0, q0, (int)(a.offsets_q[b + 1] / a.row_elems_q) - q0);
  };
  auto bucket = [&](const int4& l) {
    const long long t = (long long)((l.y + 127) / 128) * ((l.w + 127) / 128);
    const int n = t > 1 << 20 ? 1 << 20 : (int)t;
    return n < 16 ? n : (28 - __clz(n) + 15 < kListBuckets - 1 ? 28 - __clz(n) + 15 : kListBuckets - 1);
  };
  for (int64_t b = threadIdx.x; b < a.batch; b += kPrepThreads) {
    const int4 l = lengths(b);
    if (cls.has(l.y, l.w)) atomicAdd(&s_cnt[bucket(l)], 1);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int acc = 0;
    for (int k = kListBuckets - 1; k >= 0; --k) {
      s_base[k] = acc;
      acc += s_cnt[k];
    }
    *out.count = acc;
  }
  __syncthreads();
  for (int64_t b = threadIdx.x; b < a.batch; b += kPrepThreads) {
    const int4 l = lengths(b);
    if (!cls.has(l.y, l.w)) continue;
    const int pos = atomicAdd(&s_base[bucket(l)], 1);
    out.items[pos] = l;
    out.seq[pos] = (int)b;
  }
}

// The lists of a backward pass: tiles of the short and the long class's sequences, the sequences of the middle class.
struct Lists {
  ListOut kv, qi, long_kv, long_qi, mid;
};
struct Plan {
  Class short_, mid, long_;
  int tile;  // rows of the short class's tiles; the long class's have 128
};
constexpr int kListBlocks = 5;

// D from the rounded O is off by |dO| |O| times half a step of the 16-bit type, and that goes into every dS_ij = P_ij (dP_ij - D_i) of
// the row alike.  Over many keys it is small next to dP; a sequence of one key has dS = 0, and all of its dQ and dK would be that
// error.  So a row of up to kFewKeys keys sums D = sum_j P_ij dP_ij itself, in 32 bits.  (Relative error of bf16 dQ and dK, heads of
// 64: 2 keys 0.0039 from O, 0.0024 from P; 4 keys 0.0029; 16 keys 0.0025; 64 keys 0.0024, the rounding of dS and of the result.)
constexpr int kFewKeys = 16;

// Raises the largest squared 2-norm of a sequence and head.  A row that holds Inf or NaN does not count: no factor mends it, and the
// others' gradients are held as if it were not there.
__device__ __forceinline__ void raise_norm(unsigned* at, float m) {
  if (m <= FLT_MAX) atomicMax(at, __float_as_uint(m));
}

// Rows of V a warp takes.  One pass over V, 13 us of the launch's 46 for 34 000 tokens of 12 heads; one row a warp, each with a search
// of its own, takes 24.
constexpr int kValueRows = 8;
__host__ __device__ __forceinline__ int64_t prepare_blocks(int64_t tokens, int rows) {
  return (tokens + rows * (kPrepThreads / 32) - 1) / (rows * (kPrepThreads / 32));
}

// |V_j|^2 of the rows from t0 on, one warp, into the largest of their sequence and head
__device__ __forceinline__ void value_norms(const BwdArgs& a, uint2* __restrict__ top, int64_t k_tokens, int64_t t0) {
  if (t0 >= k_tokens) return;
  const int lane = threadIdx.x & 31, n = (int)(k_tokens - t0 < kValueRows ? k_tokens - t0 : kValueRows);
  const int nv = a.H * a.d / 8, per = a.d / 8, log_per = 31 - __clz(per);
  // lane i: the sequence of row i (-1: behind the last one)
  const int64_t e = (t0 + lane % kValueRows) * a.row_elems_k;
  const int64_t b = find_entry(a.offsets_k, 0, a.batch - 1, e);
  const int seq = e < a.offsets_k[b + 1] ? (int)b : -1;
  for (int v = lane; v < nv + lane; v += 32) {  // (the same trips for every lane: the sums are warp-wide)
    uint4 x[kValueRows];
#pragma unroll
    for (int i = 0; i < kValueRows; ++i)
      x[i] = i < n && v < nv ? reinterpret_cast<const uint4*>(static_cast<const __half*>(a.v) + (t0 + i) * a.ldv)[v] : make_uint4(0u, 0u, 0u, 0u);
    const bool writes = v < nv && (lane & (per - 1)) == 0;
    float most = 0.0f;
    int of = __shfl_sync(0xffffffffu, seq, 0);
#pragma unroll
    for (int i = 0; i < kValueRows; ++i) {
      float f[8], m = 0.0f;
      Vec16<NTB200_F16>::unpack(x[i], f);
#pragma unroll
      for (int k = 0; k < 8; ++k) m = fmaf(f[k], f[k], m);
      for (int w = per / 2; w > 0; w >>= 1) m += __shfl_xor_sync(0xffffffffu, m, w);
      const int s = __shfl_sync(0xffffffffu, seq, i);
      if (i < n && s != of) {
        if (writes && of >= 0) raise_norm(&top[(int64_t)of * a.H + (v >> log_per)].y, most);
        most = 0.0f;
        of = s;
      }
      if (i < n && m <= FLT_MAX) most = fmaxf(most, m);
    }
    if (writes && of >= 0) raise_norm(&top[(int64_t)of * a.H + (v >> log_per)].y, most);
  }
}

// The first blocks build one list each; every warp of the others takes one query token: D of all its heads, and (fp16) |dO|^2 for the
// largest of its sequence and head; behind them (fp16) the rows of V likewise.  VEC: heads of 32, 64 or 128 elements on
// 16-byte boundaries: a head on d / 8 lanes.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kPrepThreads, 4)
backward_prepare_kernel(BwdArgs a, Plan plan, Lists l, uint2* top, int64_t k_tokens) {
  switch (blockIdx.x) {  // (a class without sequences gives an empty list)
    case 0: build_backward_items(a.offsets_k, a.row_elems_k, a.offsets_q, a.row_elems_q, a.batch, plan.tile, plan.short_, l.kv); return;
    case 1: build_backward_items(a.offsets_q, a.row_elems_q, a.offsets_k, a.row_elems_k, a.batch, plan.tile, plan.short_, l.qi); return;
    case 2: if (plan.long_.any()) build_backward_items(a.offsets_k, a.row_elems_k, a.offsets_q, a.row_elems_q, a.batch, 128, plan.long_, l.long_kv); return;
    case 3: if (plan.long_.any()) build_backward_items(a.offsets_q, a.row_elems_q, a.offsets_k, a.row_elems_k, a.batch, 128, plan.long_, l.long_qi); return;
    case 4: if (plan.mid.any()) build_sequence_items(a, plan.mid, l.mid); return;
    default: break;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t block = (int64_t)blockIdx.x - kListBlocks, q_blocks = prepare_blocks(a.q_tokens, 1);
  const int64_t E = (int64_t)a.H * a.d;
  if constexpr (VEC && std::is_same<T, __half>::value) {
    if (block >= q_blocks) {
      value_norms(a, top, k_tokens, ((block - q_blocks) * (kPrepThreads / 32) + warp) * kValueRows);
      return;
    }
  }
  const int64_t t = block * (kPrepThreads / 32) + warp;
  if (t >= a.q_tokens) return;
  const T* g = static_cast<const T*>(a.grad) + t * E;
  const T* o = static_cast<const T*>(a.out) + t * E;
  constexpr bool kRounded = !std::is_same<T, float>::value;  // O has fewer bits than D
  [[maybe_unused]] constexpr int kSteps = 4;                 // steps of 256 elements whose loads are in flight together
  [[maybe_unused]] uint4 x[kSteps], y[kSteps];
  [[maybe_unused]] const int nv = (int)(E / 8);
  [[maybe_unused]] auto load = [&](int first) {
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int v = first + 32 * i;
      x[i] = y[i] = make_uint4(0u, 0u, 0u, 0u);
      if (v < nv) {
        x[i] = reinterpret_cast<const uint4*>(g)[v];
        y[i] = reinterpret_cast<const uint4*>(o)[v];
      }
    }
  };
  if constexpr (VEC) load(lane);  // (in flight while the sequence is looked up)
  int64_t b = 0, key0 = 0, keys = 0;
  bool few = false;
  if constexpr (kRounded) {
    b = find_entry_warp(a.offsets_q, 0, a.batch - 1, t * a.row_elems_q);
    if (t * a.row_elems_q >= a.offsets_q[b + 1]) return;  // behind the last sequence: nothing reads its D
    const int64_t k_first = a.offsets_k[b], k_elems = a.offsets_k[b + 1] - k_first;
    few = k_elems <= kFewKeys * a.row_elems_k;
    if (few) key0 = k_first / a.row_elems_k, keys = k_elems / a.row_elems_k;
  }
  const float scale = a.scaling * kLog2e;
  const T* q = static_cast<const T*>(a.q) + t * a.ldq;
  const T* k0 = static_cast<const T*>(a.k) + key0 * a.ldk;
  const T* v0 = static_cast<const T*>(a.v) + key0 * a.ldv;
  if constexpr (VEC) {
    constexpr int kDtype = std::is_same<T, __half>::value ? NTB200_F16 : NTB200_BF16;  // (VEC: 16-bit types)
    const int per = a.d / 8, log_per = 31 - __clz(per);  // lanes per head: 4, 8 or 16
    if (few) {
      constexpr int kAhead = 4;  // keys whose rows are in flight together
      for (int v = lane; v < nv + lane; v += 32) {  // (the same trips for every lane: the sums are warp-wide)
        const bool live = v < nv;
        const int h = live ? v >> log_per : 0;
        float xe[8], qe[8], s = 0.0f, m = 0.0f;
        Vec16<kDtype>::unpack(live ? reinterpret_cast<const uint4*>(g)[v] : make_uint4(0u, 0u, 0u, 0u), xe);
        Vec16<kDtype>::unpack(live ? reinterpret_cast<const uint4*>(q)[v] : make_uint4(0u, 0u, 0u, 0u), qe);
        const float lse = live ? a.lse[(int64_t)h * a.q_tokens + t] : 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) m = fmaf(xe[e], xe[e], m);
        for (int w = per / 2; w > 0; w >>= 1) m += __shfl_xor_sync(0xffffffffu, m, w);
        for (int j0 = 0; j0 < (int)keys; j0 += kAhead) {
          uint4 kv[kAhead], vv[kAhead];
#pragma unroll
          for (int i = 0; i < kAhead; ++i) {
            kv[i] = vv[i] = make_uint4(0u, 0u, 0u, 0u);
            if (live && j0 + i < (int)keys) {
              kv[i] = reinterpret_cast<const uint4*>(k0 + (j0 + i) * a.ldk)[v];
              vv[i] = reinterpret_cast<const uint4*>(v0 + (j0 + i) * a.ldv)[v];
            }
          }
#pragma unroll
          for (int i = 0; i < kAhead; ++i) {
            float ke[8], ve[8], sij = 0.0f, dp = 0.0f;
            Vec16<kDtype>::unpack(kv[i], ke);
            Vec16<kDtype>::unpack(vv[i], ve);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              sij = fmaf(qe[e], ke[e], sij);
              dp = fmaf(xe[e], ve[e], dp);
            }
            for (int w = per / 2; w > 0; w >>= 1) {
              sij += __shfl_xor_sync(0xffffffffu, sij, w);
              dp += __shfl_xor_sync(0xffffffffu, dp, w);
            }
            if (j0 + i < (int)keys) s = fmaf(exp2f(fmaf(sij, scale, -lse)), dp, s);
          }
        }
        if (live && (lane & (per - 1)) == 0) {
          a.delta[(int64_t)h * a.q_tokens + t] = s;
          if (top != nullptr) raise_norm(&top[b * a.H + h].x, m);
        }
      }
      return;
    }
    for (int first = lane; first < nv + lane; first += 32 * kSteps) {
      if (first != lane) load(first);
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        if (first - lane + 32 * i >= nv) break;
        float s = 0.0f, m = 0.0f, xe[8], ye[8];
        Vec16<kDtype>::unpack(x[i], xe);
        Vec16<kDtype>::unpack(y[i], ye);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          s = fmaf(xe[k], ye[k], s);
          m = fmaf(xe[k], xe[k], m);
        }
        for (int w = per / 2; w > 0; w >>= 1) {
          s += __shfl_xor_sync(0xffffffffu, s, w);
          m += __shfl_xor_sync(0xffffffffu, m, w);
        }
        const int v = first + 32 * i;
        if (v < nv && (lane & (per - 1)) == 0) {
          const int h = v >> log_per;
          a.delta[(int64_t)h * a.q_tokens + t] = s;
          if (top != nullptr) raise_norm(&top[b * a.H + h].x, m);
        }
      }
    }
  } else {
    for (int h = 0; h < a.H; ++h) {
      float s = 0.0f;
      const int64_t col = (int64_t)h * a.d;
      if (few) {
        const float lse = a.lse[(int64_t)h * a.q_tokens + t];
        for (int64_t j = 0; j < keys; ++j) {
          float sij = 0.0f, dp = 0.0f;
          for (int i = lane; i < a.d; i += 32) {
            sij = fmaf(to_f32(q[col + i]), to_f32(k0[j * a.ldk + col + i]), sij);
            dp = fmaf(to_f32(g[col + i]), to_f32(v0[j * a.ldv + col + i]), dp);
          }
#pragma unroll
          for (int w = 16; w > 0; w >>= 1) {
            sij += __shfl_xor_sync(0xffffffffu, sij, w);
            dp += __shfl_xor_sync(0xffffffffu, dp, w);
          }
          s = fmaf(exp2f(fmaf(sij, scale, -lse)), dp, s);
        }
      } else {
        for (int i = lane; i < a.d; i += 32) s = fmaf(to_f32(g[col + i]), to_f32(o[col + i]), s);
#pragma unroll
        for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
      }
      if (lane == 0) a.delta[(int64_t)h * a.q_tokens + t] = s;
    }
  }
}

// ------------------------------------------------------------------ tiles in 32 bits, any type and head size
// One block owns BT rows r of one side and walks the other side's rows c in tiles of BT:
//     KV:  r = keys,    A_own = K, B_own = V;   c = queries, A = Q, B = dO:   dV_r += P_cr dO_c,  dK_r += dS_cr Q_c
//     !KV: r = queries, A_own = Q, B_own = dO;  c = keys,    A = K, B = V:    dQ_r += dS_cr K_c
// with S_cr = A_own,r . A_c and dP_cr = B_own,r . B_c in both.  Everything is held in fp32 in shared memory, each thread
// computes a (BT/16) x (BT/16) patch of S and dP and keeps BT/16 rows x DP/16 columns of each gradient in registers.  fp32 has no
// tensor-core product of its precision, so this is bound by the FMA units and the shared-memory reads that feed them: 0.58
// GFLOP in 16 sequences of up to 200 tokens (4 heads of 64) take 57 us, two waves of items of up to four tiles; two sequences
// of up to 1400 (12 heads) 594 us, 22 TFLOP/s of its seven products (832 us before two blocks fitted an SM).
template <typename T, int BT, int DP>
__device__ __forceinline__ void load_rows(float* __restrict__ s, const T* __restrict__ g, int64_t ld, int rows, int d) {
  if constexpr (std::is_same<T, float>::value) {
    if (d % 4 == 0 && ld % 4 == 0 && (reinterpret_cast<uintptr_t>(g) & 15) == 0) {
#pragma unroll
      for (int i = threadIdx.x; i < BT * DP / 4; i += 256) {
        const int r = i / (DP / 4), c = i % (DP / 4) * 4;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (r < rows && c < d) v = *reinterpret_cast<const float4*>(g + (int64_t)r * ld + c);
        *reinterpret_cast<float4*>(s + r * (DP + 4) + c) = v;
      }
      return;
    }
  }
  for (int i = threadIdx.x; i < BT * DP; i += 256) {
    const int r = i / DP, c = i % DP;
    s[r * (DP + 4) + c] = (r < rows && c < d) ? to_f32(g[(int64_t)r * ld + c]) : 0.0f;
  }
}

// MI neighbouring values at a multiple of MI
template <int MI>
__device__ __forceinline__ void load_some(float (&v)[MI], const float* __restrict__ s) {
  if constexpr (MI == 4) {
    const float4 x = *reinterpret_cast<const float4*>(s);
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
  } else {
#pragma unroll
    for (int i = 0; i < MI; ++i) v[i] = s[i];
  }
}

template <int BT, int DP>
constexpr int bwd_simt_smem() { return (4 * BT * (DP + 4) + 2 * BT * (BT + 4) + 2 * BT) * 4; }

template <typename T, int BT, int DP, bool KV>
__device__ __forceinline__ void bwd_simt_item(const BwdArgs& a, const Item& it, int h) {
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
  const int64_t E = (int64_t)a.H * a.d;
  const float scale = a.scaling * kLog2e;
  const int d4 = (a.d + 3) & ~3;
  const int64_t col = (int64_t)h * a.d;
  const T* ga_own = (KV ? static_cast<const T*>(a.k) + it.row0 * a.ldk : static_cast<const T*>(a.q) + it.row0 * a.ldq) + col;
  const T* gb_own = (KV ? static_cast<const T*>(a.v) + it.row0 * a.ldv : static_cast<const T*>(a.grad) + it.row0 * E) + col;
  const int64_t ld_a_own = KV ? a.ldk : a.ldq, ld_b_own = KV ? a.ldv : E;
  const int64_t ld_a = KV ? a.ldq : a.ldk, ld_b = KV ? E : a.ldv;
  const float* g_lse = a.lse + (int64_t)h * a.q_tokens;
  const float* g_delta = a.delta + (int64_t)h * a.q_tokens;
  __syncthreads();  // the previous item's tiles have been read
  load_rows<T, BT, DP>(own_a, ga_own, ld_a_own, it.rows, a.d);
  load_rows<T, BT, DP>(own_b, gb_own, ld_b_own, it.rows, a.d);
  if (!KV && threadIdx.x < BT) {
    const bool ok = (int)threadIdx.x < it.rows && it.n_other > 0;  // (rows without keys have no statistics)
    s_lse[threadIdx.x] = ok ? g_lse[it.row0 + threadIdx.x] : INFINITY;
    s_delta[threadIdx.x] = ok ? g_delta[it.row0 + threadIdx.x] : 0.0f;
  }
  float acc1[KV ? MI : 1][KV ? NC : 1], acc2[MI][NC];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      acc2[i][j] = 0.0f;
      if (KV) acc1[i][j] = 0.0f;
    }
  for (int c0 = 0; c0 < it.n_other; c0 += BT) {
    const int nc = it.n_other - c0 < BT ? it.n_other - c0 : BT;
    const int64_t o0 = it.other + c0;
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
      load_some(ds, s_ds + c * LS + ty * MI);
      if (KV) load_some(pv, s_p + c * LS + ty * MI);
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
    if (r >= it.rows) continue;
    T* o2 = (KV ? static_cast<T*>(a.dk) + (it.row0 + r) * a.lddk : static_cast<T*>(a.dq) + (it.row0 + r) * a.lddq) + col;
    T* o1 = KV ? static_cast<T*>(a.dv) + (it.row0 + r) * a.lddv + col : nullptr;
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

// KV items, then Q items, in one launch: neither alone fills the GPU when the batch is small
template <typename T, int BT, int DP>
__global__ void __launch_bounds__(256, DP == 64 ? 2 : 1) attn_bwd_simt_kernel(BwdArgs a, ListOut kv, ListOut qi) {
  const int64_t n_kv = (int64_t)*kv.count * a.H, n = n_kv + (int64_t)*qi.count * a.H;
  for (int64_t w = blockIdx.x; w < n; w += gridDim.x) {
    if (w < n_kv) bwd_simt_item<T, BT, DP, true>(a, decode(kv.items[w / a.H]), (int)(w % a.H));
    else bwd_simt_item<T, BT, DP, false>(a, decode(qi.items[(w - n_kv) / a.H]), (int)((w - n_kv) % a.H));
  }
}

// The forward pass in the same tiles, for training calls that no tensor-core kernel takes: r = queries, and the online softmax over
// tiles of keys; a row's maximum and sum are kept in shared memory between tiles.
template <int BT, int DP>
constexpr int fwd_simt_smem() { return (3 * BT * (DP + 4) + BT * (BT + 4) + 3 * BT) * 4; }

template <typename T, int BT, int DP>
__global__ void __launch_bounds__(256, DP == 64 ? 2 : 1)
attn_fwd_simt_kernel(BwdArgs a, T* __restrict__ out, float* __restrict__ lse, const int4* __restrict__ items, const int* __restrict__ count) {
  constexpr int MI = BT / 16, LD = DP + 4, LS = BT + 4, NC = DP / 16;
  extern __shared__ __align__(16) float bwd_smem[];
  float* s_q = bwd_smem;
  float* s_k = s_q + BT * LD;
  float* s_v = s_k + BT * LD;
  float* s_p = s_v + BT * LD;  // [key][query]
  float* s_top = s_p + BT * LS;
  float* s_sum = s_top + BT;
  float* s_corr = s_sum + BT;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const int64_t n = (int64_t)*count * a.H;
  const int64_t E = (int64_t)a.H * a.d;
  const float scale = a.scaling * kLog2e;
  const int d4 = (a.d + 3) & ~3;
  for (int64_t w = blockIdx.x; w < n; w += gridDim.x) {
    const Item it = decode(items[w / a.H]);
    const int h = (int)(w % a.H);
    const int64_t col = (int64_t)h * a.d;
    __syncthreads();  // the previous item's tiles have been read
    load_rows<T, BT, DP>(s_q, static_cast<const T*>(a.q) + it.row0 * a.ldq + col, a.ldq, it.rows, a.d);
    if (threadIdx.x < BT) {
      s_top[threadIdx.x] = -INFINITY;
      s_sum[threadIdx.x] = 0.0f;
    }
    float acc[MI][NC];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NC; ++j) acc[i][j] = 0.0f;
    for (int c0 = 0; c0 < it.n_other; c0 += BT) {
      const int nc = it.n_other - c0 < BT ? it.n_other - c0 : BT;
      __syncthreads();
      load_rows<T, BT, DP>(s_k, static_cast<const T*>(a.k) + (it.other + c0) * a.ldk + col, a.ldk, nc, a.d);
      load_rows<T, BT, DP>(s_v, static_cast<const T*>(a.v) + (it.other + c0) * a.ldv + col, a.ldv, nc, a.d);
      __syncthreads();
      float s[MI][MI];  // key ty + 16 i, query tx + 16 j
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < MI; ++j) s[i][j] = 0.0f;
#pragma unroll 2
      for (int c = 0; c < d4; c += 4) {
        float4 x[MI], y[MI];
#pragma unroll
        for (int i = 0; i < MI; ++i) x[i] = *reinterpret_cast<const float4*>(s_k + (ty + 16 * i) * LD + c);
#pragma unroll
        for (int j = 0; j < MI; ++j) y[j] = *reinterpret_cast<const float4*>(s_q + (tx + 16 * j) * LD + c);
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int j = 0; j < MI; ++j) {
            s[i][j] = fmaf(x[i].x, y[j].x, s[i][j]);
            s[i][j] = fmaf(x[i].y, y[j].y, s[i][j]);
            s[i][j] = fmaf(x[i].z, y[j].z, s[i][j]);
            s[i][j] = fmaf(x[i].w, y[j].w, s[i][j]);
          }
      }
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < MI; ++j) s_p[(ty + 16 * i) * LS + tx + 16 * j] = s[i][j] * scale;
      __syncthreads();
      // one warp takes BT / 8 queries: 32 lanes over the tile's keys
      const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
      for (int r = 0; r < BT / 8; ++r) {
        const int q = warp * (BT / 8) + r;
        float v[BT / 32], top = s_top[q];
#pragma unroll
        for (int k = 0; k < BT / 32; ++k) {
          v[k] = lane + 32 * k < nc ? s_p[(lane + 32 * k) * LS + q] : -INFINITY;
          top = fmaxf(top, v[k]);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < BT / 32; ++k) {
          v[k] = lane + 32 * k < nc ? exp2f(v[k] - top) : 0.0f;
          sum += v[k];
          s_p[(lane + 32 * k) * LS + q] = v[k];
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) {
          const float corr = exp2f(s_top[q] - top);  // 0 on the first tile
          s_corr[q] = corr;
          s_sum[q] = s_sum[q] * corr + sum;
          s_top[q] = top;
        }
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const float corr = s_corr[ty * MI + i];
#pragma unroll
        for (int j = 0; j < NC; ++j) acc[i][j] *= corr;
      }
      for (int c = 0; c < nc; ++c) {
        float p[MI];
        load_some(p, s_p + c * LS + ty * MI);
#pragma unroll
        for (int m = 0; m < NC / 4; ++m) {
          const float4 x = *reinterpret_cast<const float4*>(s_v + c * LD + tx * 4 + 64 * m);
#pragma unroll
          for (int i = 0; i < MI; ++i) {
            acc[i][4 * m] = fmaf(p[i], x.x, acc[i][4 * m]);
            acc[i][4 * m + 1] = fmaf(p[i], x.y, acc[i][4 * m + 1]);
            acc[i][4 * m + 2] = fmaf(p[i], x.z, acc[i][4 * m + 2]);
            acc[i][4 * m + 3] = fmaf(p[i], x.w, acc[i][4 * m + 3]);
          }
        }
      }
    }
    __syncthreads();
    if (lse != nullptr && threadIdx.x < BT && (int)threadIdx.x < it.rows && it.n_other > 0)
      lse[(int64_t)h * a.q_tokens + it.row0 + threadIdx.x] = s_top[threadIdx.x] + log2f(s_sum[threadIdx.x]);
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int r = ty * MI + i;
      if (r >= it.rows) continue;
      const float inv = it.n_other > 0 ? 1.0f / s_sum[r] : 0.0f;  // no keys: zeros
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        const int c = tx * 4 + 64 * (j / 4) + j % 4;
        if (c < a.d) out[(it.row0 + r) * E + col + c] = from_f32<T>(acc[i][j] * inv);
      }
    }
  }
}

// ------------------------------------------------------------------ tensor cores (mma.sync), heads of 32, 64, 128 in 16 bits
// The same walk as the 32-bit tile kernels, a block of four warps per 64 own rows: a warp's 16 rows r are the M rows of every
// product, so S and dP come out as accumulators, become P and dS in registers and are at once the A operands of the products
// with the other side's rows (no shared-memory round trip):
//     S = A_own A_c^T,  dP = B_own B_c^T        (B operands: rows of the other side's tiles)
//     acc1 += P B_c,    acc2 += dS A_c          (B operands: the same tiles, transposed by ldmatrix)
// Other side's tiles of 64 rows come double-buffered through cp.async.  P and dS are rounded to the 16-bit type for the products
// (as the forward pass rounds P); all sums are fp32.  Bound by the ldmatrix and mma.sync issue of its 9 products, of which short
// sequences leave part empty: 10 000 tokens of lengths up to 64, 8 heads of 128, 133 us with the lists and D.
constexpr int kMmaThreads = 128, kMmaTile = 64;

template <typename T, int D>
__device__ __forceinline__ void load_tile_zfill(uint32_t dst, const T* __restrict__ g, int64_t ld, int rows) {
  constexpr int kChunks = D / 8;
#pragma unroll
  for (int i = 0; i < kMmaTile * kChunks / kMmaThreads; ++i) {
    const int idx = threadIdx.x + i * kMmaThreads;
    const int r = idx / kChunks, c = idx % kChunks;
    const bool ok = r < rows;
    cp_async_16_zfill(dst + tile_off<D>(r, c), g + (int64_t)(ok ? r : 0) * ld + c * 8, ok ? 16u : 0u);
  }
}

template <int D>
constexpr int bwd_mma_smem() { return 6 * kMmaTile * D * 2 + 4 * kMmaTile * 4; }

template <typename T, int D, bool KV>
__device__ __forceinline__ void bwd_mma_tile(const BwdArgs& a, const Item& it, float gs, int h, uint8_t* smem) {
  constexpr int KS = D / 16, NO = D / 8;
  constexpr int CW = D <= 64 ? 64 : 32;  // other rows whose S and dP are in registers at a time
  constexpr bool kKeep = D <= 64;        // own fragments in registers, or read again from shared memory
  constexpr uint32_t kBytes = kMmaTile * D * 2;
  const uint32_t s_own_a = (uint32_t)__cvta_generic_to_shared(smem), s_own_b = s_own_a + kBytes, s_oth = s_own_b + kBytes;
  float* s_lse = reinterpret_cast<float*>(smem + 6 * kBytes);  // [2][64]
  float* s_delta = s_lse + 2 * kMmaTile;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t E = (int64_t)a.H * D, col = (int64_t)h * D;
  const T* ga = (KV ? static_cast<const T*>(a.k) + it.row0 * a.ldk : static_cast<const T*>(a.q) + it.row0 * a.ldq) + col;
  const T* gb = (KV ? static_cast<const T*>(a.v) + it.row0 * a.ldv : static_cast<const T*>(a.grad) + it.row0 * E) + col;
  const T* oa = (KV ? static_cast<const T*>(a.q) + it.other * a.ldq : static_cast<const T*>(a.k) + it.other * a.ldk) + col;
  const T* ob = (KV ? static_cast<const T*>(a.grad) + it.other * E : static_cast<const T*>(a.v) + it.other * a.ldv) + col;
  const int64_t ld_oa = KV ? a.ldq : a.ldk, ld_ob = KV ? E : a.ldv;
  const float* g_lse = a.lse + (int64_t)h * a.q_tokens;
  const float* g_delta = a.delta + (int64_t)h * a.q_tokens;
  const float scale = a.scaling * kLog2e;
  const int n_tiles = (it.n_other + kMmaTile - 1) / kMmaTile;
  auto load_other = [&](int j) {
    const int st = j & 1, n = it.n_other - j * kMmaTile;
    load_tile_zfill<T, D>(s_oth + st * 2 * kBytes, oa + (int64_t)j * kMmaTile * ld_oa, ld_oa, n);
    load_tile_zfill<T, D>(s_oth + st * 2 * kBytes + kBytes, ob + (int64_t)j * kMmaTile * ld_ob, ld_ob, n);
    if (KV && threadIdx.x < kMmaTile) {
      const bool ok = (int)threadIdx.x < n;
      s_lse[st * kMmaTile + threadIdx.x] = ok ? g_lse[it.other + j * kMmaTile + threadIdx.x] : INFINITY;  // 2^(x - inf) = 0
      s_delta[st * kMmaTile + threadIdx.x] = ok ? g_delta[it.other + j * kMmaTile + threadIdx.x] * gs : 0.0f;
    }
  };
  if (n_tiles > 0) {
    load_tile_zfill<T, D>(s_own_a, ga, KV ? a.ldk : a.ldq, it.rows);
    load_tile_zfill<T, D>(s_own_b, gb, KV ? a.ldv : E, it.rows);
    load_other(0);
    cp_async_commit();
  }
  const int r0 = warp * 16 + (lane >> 2), r1 = r0 + 8;
  float lse0 = INFINITY, lse1 = INFINITY, dl0 = 0.0f, dl1 = 0.0f;
  if (!KV && n_tiles > 0) {
    if (r0 < it.rows) lse0 = g_lse[it.row0 + r0], dl0 = g_delta[it.row0 + r0] * gs;
    if (r1 < it.rows) lse1 = g_lse[it.row0 + r1], dl1 = g_delta[it.row0 + r1] * gs;
  }
  const bool active = warp * 16 < it.rows;
  float acc1[KV ? NO : 1][4], acc2[NO][4];
#pragma unroll
  for (int i = 0; i < NO; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      acc2[i][j] = 0.0f;
      if (KV) acc1[KV ? i : 0][j] = 0.0f;
    }
  uint32_t fa[kKeep ? KS : 1][4], fb[kKeep ? KS : 1][4];
  for (int j = 0; j < n_tiles; ++j) {
    if (j + 1 < n_tiles) {
      load_other(j + 1);
      cp_async_commit();
      cp_async_wait<1>();
    } else {
      cp_async_wait<0>();
    }
    __syncthreads();
    if (active) {
      const uint32_t ta = s_oth + (j & 1) * 2 * kBytes, tb = ta + kBytes;
      const float* lse_c = s_lse + (j & 1) * kMmaTile;
      const float* delta_c = s_delta + (j & 1) * kMmaTile;
      const int nc = it.n_other - j * kMmaTile < kMmaTile ? it.n_other - j * kMmaTile : kMmaTile;
      if (kKeep && j == 0) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          ldmatrix_x4(fa[kKeep ? ks : 0], s_own_a + tile_off<D>(warp * 16 + (lane & 15), ks * 2 + (lane >> 4)));
          ldmatrix_x4(fb[kKeep ? ks : 0], s_own_b + tile_off<D>(warp * 16 + (lane & 15), ks * 2 + (lane >> 4)));
        }
      }
#pragma unroll 1
      for (int c0 = 0; c0 < nc; c0 += CW) {
        const int groups = (nc - c0 + 15) / 16;  // of 16 other rows, CW / 16 at most
        float s[CW / 8][4], dp[CW / 8][4];
#pragma unroll
        for (int i = 0; i < CW / 8; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) s[i][k] = dp[i][k] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          uint32_t xa[4], xb[4];
          if (!kKeep) {
            ldmatrix_x4(xa, s_own_a + tile_off<D>(warp * 16 + (lane & 15), ks * 2 + (lane >> 4)));
            ldmatrix_x4(xb, s_own_b + tile_off<D>(warp * 16 + (lane & 15), ks * 2 + (lane >> 4)));
          }
          const uint32_t(&ua)[4] = kKeep ? fa[kKeep ? ks : 0] : xa;
          const uint32_t(&ub)[4] = kKeep ? fb[kKeep ? ks : 0] : xb;
#pragma unroll
          for (int np = 0; np < CW / 16; ++np) {
            if (np < groups) {
              uint32_t f[4];
              const uint32_t off = tile_off<D>(c0 + np * 16 + (lane & 7) + ((lane >> 4) << 3), ks * 2 + ((lane >> 3) & 1));
              ldmatrix_x4(f, ta + off);
              MmaOp<T>::mma(s[np * 2], ua, f[0], f[1]);
              MmaOp<T>::mma(s[np * 2 + 1], ua, f[2], f[3]);
              ldmatrix_x4(f, tb + off);
              MmaOp<T>::mma(dp[np * 2], ub, f[0], f[1]);
              MmaOp<T>::mma(dp[np * 2 + 1], ub, f[2], f[3]);
            }
          }
        }
        uint32_t pf[CW / 16][4], df[CW / 16][4];  // P and dS as A fragments
#pragma unroll
        for (int nt = 0; nt < CW / 8; ++nt) {
          const int c = c0 + nt * 8 + 2 * (lane & 3);
          float p[4], ds[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float l = KV ? lse_c[c + (k & 1)] : (k < 2 ? lse0 : lse1);
            const float dl = KV ? delta_c[c + (k & 1)] : (k < 2 ? dl0 : dl1);
            p[k] = exp2f(fmaf(s[nt][k], scale, -l));
            // a key past the end has no probability (its zeroed row scores 0); a query past the end has lse = inf
            if (!KV && c + (k & 1) >= nc) p[k] = 0.0f;
            ds[k] = p[k] * fmaf(dp[nt][k], gs, -dl);
          }
          pf[nt >> 1][(nt & 1) * 2] = MmaOp<T>::pack(p[0], p[1]);
          pf[nt >> 1][(nt & 1) * 2 + 1] = MmaOp<T>::pack(p[2], p[3]);
          df[nt >> 1][(nt & 1) * 2] = MmaOp<T>::pack(ds[0], ds[1]);
          df[nt >> 1][(nt & 1) * 2 + 1] = MmaOp<T>::pack(ds[2], ds[3]);
        }
#pragma unroll
        for (int ks = 0; ks < CW / 16; ++ks) {
          if (ks < groups) {
#pragma unroll
            for (int np = 0; np < NO / 2; ++np) {
              uint32_t f[4];
              const uint32_t off = tile_off<D>(c0 + ks * 16 + (lane & 7) + (((lane >> 3) & 1) << 3), np * 2 + (lane >> 4));
              ldmatrix_x4_trans(f, ta + off);
              MmaOp<T>::mma(acc2[np * 2], df[ks], f[0], f[1]);
              MmaOp<T>::mma(acc2[np * 2 + 1], df[ks], f[2], f[3]);
              if (KV) {
                ldmatrix_x4_trans(f, tb + off);
                MmaOp<T>::mma(acc1[KV ? np * 2 : 0], pf[ks], f[0], f[1]);
                MmaOp<T>::mma(acc1[KV ? np * 2 + 1 : 0], pf[ks], f[2], f[3]);
              }
            }
          }
        }
      }
    }
    __syncthreads();  // this stage is refilled next
  }
  const float f2 = a.scaling / gs;
  T* out2 = (KV ? static_cast<T*>(a.dk) + it.row0 * a.lddk : static_cast<T*>(a.dq) + it.row0 * a.lddq) + col;
  T* out1 = KV ? static_cast<T*>(a.dv) + it.row0 * a.lddv + col : nullptr;
  const int64_t ld2 = KV ? a.lddk : a.lddq;
#pragma unroll
  for (int nt = 0; nt < NO; ++nt) {
    const int c = nt * 8 + 2 * (lane & 3);
    if (r0 < it.rows) {
      *reinterpret_cast<uint32_t*>(out2 + r0 * ld2 + c) = MmaOp<T>::pack(acc2[nt][0] * f2, acc2[nt][1] * f2);
      if (KV) *reinterpret_cast<uint32_t*>(out1 + r0 * a.lddv + c) = MmaOp<T>::pack(acc1[KV ? nt : 0][0], acc1[KV ? nt : 0][1]);
    }
    if (r1 < it.rows) {
      *reinterpret_cast<uint32_t*>(out2 + r1 * ld2 + c) = MmaOp<T>::pack(acc2[nt][2] * f2, acc2[nt][3] * f2);
      if (KV) *reinterpret_cast<uint32_t*>(out1 + r1 * a.lddv + c) = MmaOp<T>::pack(acc1[KV ? nt : 0][2], acc1[KV ? nt : 0][3]);
    }
  }
}

// dK and dV of every (key tile, head), then dQ of every (query tile, head)
template <typename T, int D>
__global__ void __launch_bounds__(kMmaThreads) attn_bwd_mma_kernel(BwdArgs a, ListOut kv, ListOut qi) {
  extern __shared__ __align__(128) uint8_t mma_smem[];
  const int64_t n_kv = (int64_t)*kv.count * a.H, n = n_kv + (int64_t)*qi.count * a.H;
  for (int64_t w = blockIdx.x; w < n; w += gridDim.x) {
    const bool is_kv = w < n_kv;
    const int64_t i = (is_kv ? w : w - n_kv) / a.H;
    const int h = (int)((is_kv ? w : w - n_kv) - i * a.H);
    if (is_kv) bwd_mma_tile<T, D, true>(a, decode(kv.items[i]), grad_scale(a, kv.seq, i, h), h, mma_smem);
    else bwd_mma_tile<T, D, false>(a, decode(qi.items[i]), grad_scale(a, qi.seq, i, h), h, mma_smem);
  }
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t item_capacity(int64_t batch, int64_t tokens, int tile) { return batch + tokens / tile + 1; }

// delta | largest |dO|^2 and |V|^2 | five lists (count, items, their sequences) | dQ in fp32 (the kernel with whole sequences as items); every part
// on a 16-byte boundary
struct BwdWorkspace {
  size_t delta, top, lists[kListBlocks], seqs[kListBlocks], scratch, bytes;
  BwdWorkspace(int64_t batch, int64_t q_tokens, int64_t k_tokens, int H, size_t scratch_bytes) {
    auto up = [](size_t v) { return (v + 15) / 16 * 16; };
    const int64_t n[kListBlocks] = {item_capacity(batch, k_tokens, 32), item_capacity(batch, q_tokens, 32), item_capacity(batch, k_tokens, 128),
                                    item_capacity(batch, q_tokens, 128), batch};  // (tiles of 32 rows or more)
    delta = 0;
    top = up((size_t)q_tokens * H * 4);
    size_t at = top + up((size_t)batch * H * sizeof(uint2));
    for (int i = 0; i < kListBlocks; ++i) {
      lists[i] = at;
      seqs[i] = at + 16 + sizeof(int4) * (size_t)n[i];
      at = seqs[i] + up(4 * (size_t)n[i]);
    }
    scratch = at;
    bytes = scratch + up(scratch_bytes);
  }
  Lists make(uint8_t* ws) const {
    auto list = [&](int i) {
      return ListOut{reinterpret_cast<int4*>(ws + lists[i] + 16), reinterpret_cast<int*>(ws + seqs[i]), reinterpret_cast<int*>(ws + lists[i])};
    };
    return {list(0), list(1), list(2), list(3), list(4)};
  }
};

template <typename T, bool VEC>
int launch_prepare(const BwdArgs& a, const Plan& plan, const Lists& l, uint2* top, int64_t k_tokens, cudaStream_t st) {
  const int64_t blocks = kListBlocks + prepare_blocks(a.q_tokens, 1) + (top != nullptr ? prepare_blocks(k_tokens, kValueRows) : 0);
  if (blocks > 0x7fffffffll) return NTB200_UNSUPPORTED_SHAPE;
  if (top != nullptr && cudaMemsetAsync(top, 0, (size_t)a.batch * a.H * sizeof(uint2), st) != cudaSuccess) return NTB200_LAUNCH_FAILED;
  backward_prepare_kernel<T, VEC><<<(unsigned)blocks, kPrepThreads, 0, st>>>(a, plan, l, top, k_tokens);
  return status_from_cuda(cudaGetLastError());
}

template <typename T, int BT, int DP>
int launch_bwd_simt(const BwdArgs& a, int64_t k_tokens, const Lists& l, cudaStream_t st) {
  constexpr int kSmem = bwd_simt_smem<BT, DP>();
  static std::atomic<int> configured[kMaxDevices];
  if (!once_per_device(configured, [] {
        return cudaFuncSetAttribute(attn_bwd_simt_kernel<T, BT, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) == cudaSuccess;
      }))
    return NTB200_LAUNCH_FAILED;
  const int rc = launch_prepare<T, false>(a, Plan{{0, INT64_MAX}, {0, 0}, {0, 0}, BT}, l, nullptr, k_tokens, st);
  if (rc != NTB200_OK) return rc;
  const int per_sm = 227 * 1024 / (kSmem + 1024);
  const int64_t most = (item_capacity(a.batch, k_tokens, BT) + item_capacity(a.batch, a.q_tokens, BT)) * a.H;
  const unsigned grid = (unsigned)(most < (int64_t)kNumSMs * per_sm ? most : (int64_t)kNumSMs * per_sm);
  attn_bwd_simt_kernel<T, BT, DP><<<grid, 256, kSmem, st>>>(a, l.kv, l.qi);
  return status_from_cuda(cudaGetLastError());
}

template <typename T, int BT, int DP>
int launch_fwd_simt(const BwdArgs& a, void* out, float* lse, const ListOut& l, cudaStream_t st) {
  constexpr int kSmem = fwd_simt_smem<BT, DP>();
  static std::atomic<int> configured[kMaxDevices];
  if (!once_per_device(configured, [] {
        return cudaFuncSetAttribute(attn_fwd_simt_kernel<T, BT, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) == cudaSuccess;
      }))
    return NTB200_LAUNCH_FAILED;
  query_items_kernel<<<1, kPrepThreads, 0, st>>>(a, BT, l);
  const int per_sm = 227 * 1024 / (kSmem + 1024);
  const int64_t most = item_capacity(a.batch, a.q_tokens, BT) * a.H;
  const unsigned grid = (unsigned)(most < (int64_t)kNumSMs * per_sm ? most : (int64_t)kNumSMs * per_sm);
  attn_fwd_simt_kernel<T, BT, DP><<<grid, 256, kSmem, st>>>(a, static_cast<T*>(out), lse, l.items, l.count);
  return status_from_cuda(cudaGetLastError());
}

template <typename T>
int launch_fwd(const BwdArgs& a, void* out, float* lse, const ListOut& l, cudaStream_t st) {
  if (a.d <= 64) return launch_fwd_simt<T, 64, 64>(a, out, lse, l, st);
  if (a.d <= 128) return launch_fwd_simt<T, 64, 128>(a, out, lse, l, st);
  return launch_fwd_simt<T, 32, 256>(a, out, lse, l, st);
}

template <typename T, int D>
int launch_bwd_mma(const BwdArgs& a, int64_t k_tokens, const Lists& l, cudaStream_t st) {
  constexpr int kSmem = bwd_mma_smem<D>();
  static std::atomic<int> configured[kMaxDevices];
  if (!once_per_device(configured, [] {
        return cudaFuncSetAttribute(attn_bwd_mma_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) == cudaSuccess;
      }))
    return NTB200_LAUNCH_FAILED;
  const int64_t most = (item_capacity(a.batch, k_tokens, kMmaTile) + item_capacity(a.batch, a.q_tokens, kMmaTile)) * a.H;
  const int64_t resident = (int64_t)kNumSMs * (D == 32 ? 8 : D == 64 ? 4 : 2);
  attn_bwd_mma_kernel<T, D><<<(unsigned)(most < resident ? most : resident), kMmaThreads, kSmem, st>>>(a, l.kv, l.qi);
  return status_from_cuda(cudaGetLastError());
}

// Sequences of up to kShort tokens on both sides go to the mma.sync kernel, whose tiles have 64 rows: 21 000 tokens of lengths up to 64
// take 273 us there and 449 on the tcgen05 kernels (16 heads of 64), 10 000 take 133 and 204 (8 heads of 128); of lengths up to
// 128, 291 and 265, and 148 and 141.
constexpr int64_t kShort = 64;
// Heads of 64: sequences of up to kMid tokens as whole items (S and dP once for all three gradients): 128 sequences of 32 to 512 tokens, 12
// heads: 416 us against 445 with an item per tile; beyond, a sequence would keep its one CTA busy for long (one of 1024, 16
// heads: 217 us against 47).
constexpr int64_t kMid = 512;

Plan make_plan(int d, bool tc, int path) {
  constexpr int64_t kAll = INT64_MAX;
  if (!tc || path == 2) return {{0, kAll}, {0, 0}, {0, 0}, kMmaTile};
  if (path == 3) return {{0, 0}, {0, 0}, {0, kAll}, kMmaTile};
  if (path == 4) return {{0, 0}, {0, kAll}, {0, 0}, kMmaTile};
  if (d == 64) return {{0, kShort}, {kShort, kMid}, {kMid, kAll}, kMmaTile};
  return {{0, kShort}, {0, 0}, {kShort, kAll}, kMmaTile};
}

// fp32 sums of dQ over the key tiles of the middle class's sequences
size_t scratch_bytes(int64_t q_tokens, int64_t max_len_k, int H, int d, int dtype, int path) {
  return d == 64 && dtype != NTB200_F32 && (path == 0 || path == 4) && max_len_k > 128 ? (size_t)q_tokens * H * d * 4 : 0;
}

template <typename T>
int launch_bwd(const BwdArgs& args, int64_t k_tokens, int64_t max_len, uint8_t* ws, const BwdWorkspace& at, int path, cudaStream_t st) {
  const Lists l = at.make(ws);
  BwdArgs a = args;
  if constexpr (!std::is_same<T, float>::value) {
    constexpr int dtype = std::is_same<T, __half>::value ? NTB200_F16 : NTB200_BF16;
    const bool mma = (a.d == 32 || a.d == 64 || a.d == 128) && aligned16(a.grad) && aligned16(a.q) && aligned16(a.k) && aligned16(a.v) &&
                     aligned16(a.out) && aligned16(a.dq) && aligned16(a.dk) && aligned16(a.dv) && a.ldq % 8 == 0 && a.ldk % 8 == 0 &&
                     a.ldv % 8 == 0 && a.lddq % 8 == 0 && a.lddk % 8 == 0 && a.lddv % 8 == 0;
    const bool tc = mma && a.d >= 64 && attn_bwd_tcgen05_supported(a, k_tokens, dtype);
    if ((path == 2 && !mma) || (path >= 3 && !tc) || (path == 4 && a.d != 64)) return NTB200_UNSUPPORTED_SHAPE;
    if (mma && path != 1) {
      const Plan plan = make_plan(a.d, tc, path);
      a.top = dtype == NTB200_F16 ? reinterpret_cast<uint2*>(ws + at.top) : nullptr;
      int rc = launch_prepare<T, true>(a, plan, l, const_cast<uint2*>(a.top), k_tokens, st);
      if (rc == NTB200_OK && plan.long_.any() && max_len > plan.long_.over)
        rc = attn_bwd_tcgen05_launch(a, k_tokens, dtype, l.long_kv, l.long_qi, item_capacity(a.batch, k_tokens, 128),
                                     item_capacity(a.batch, a.q_tokens, 128), st);
      if (rc == NTB200_OK && plan.mid.any() && max_len > plan.mid.over)
        rc = attn_bwd_fused_launch(a, k_tokens, dtype, l.mid, at.bytes > at.scratch ? reinterpret_cast<float*>(ws + at.scratch) : nullptr, st);
      if (rc != NTB200_OK || !plan.short_.any()) return rc;
      if (a.d == 32) return launch_bwd_mma<T, 32>(a, k_tokens, l, st);
      if (a.d == 64) return launch_bwd_mma<T, 64>(a, k_tokens, l, st);
      return launch_bwd_mma<T, 128>(a, k_tokens, l, st);
    }
  } else if (path > 1) {
    return NTB200_UNSUPPORTED_SHAPE;
  }
  if (a.d <= 64) return launch_bwd_simt<T, 64, 64>(a, k_tokens, l, st);
  if (a.d <= 128) return launch_bwd_simt<T, 64, 128>(a, k_tokens, l, st);
  return launch_bwd_simt<T, 32, 256>(a, k_tokens, l, st);
}

}  // namespace

size_t attn_fwd_tiles_workspace_bytes(int64_t batch, int64_t q_tokens) {
  return 16 + (sizeof(int4) + sizeof(int)) * (size_t)item_capacity(batch, q_tokens, 32);
}

int attn_fwd_tiles_launch(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv, void* out, const AttnRows& rows,
                          int64_t batch, int64_t q_tokens, int H, int d, float scaling, int dtype, void* workspace, cudaStream_t st) {
  BwdArgs a = {};
  a.q = q, a.k = k, a.v = v;
  a.ldq = ldq, a.ldk = ldk, a.ldv = ldv;
  a.offsets_q = rows.offsets_q, a.offsets_k = rows.offsets_k;
  a.row_elems_q = rows.row_elems_q, a.row_elems_k = rows.row_elems_k;
  a.batch = batch, a.q_tokens = q_tokens;
  a.H = H, a.d = d, a.scaling = scaling;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const int64_t cap = item_capacity(batch, q_tokens, 32);
  const ListOut l = {reinterpret_cast<int4*>(ws + 16), reinterpret_cast<int*>(ws + 16 + sizeof(int4) * cap), reinterpret_cast<int*>(ws)};
  switch (dtype) {
    case NTB200_F32: return launch_fwd<float>(a, out, rows.lse, l, st);
    case NTB200_F16: return launch_fwd<__half>(a, out, rows.lse, l, st);
    default: return launch_fwd<__nv_bfloat16>(a, out, rows.lse, l, st);
  }
}

}  // namespace ntb200

using namespace ntb200;

extern "C" {

size_t ntb200_varlen_attention_backward_workspace_bytes(int64_t batch, int64_t q_tokens, int64_t k_tokens, int num_heads, int head_dim,
                                                        int64_t max_len_q, int64_t max_len_k, int dtype, int path) {
  (void)max_len_q;
  if (batch <= 0 || q_tokens < 0 || k_tokens < 0 || num_heads < 1 || head_dim < 1) return 0;
  return BwdWorkspace(batch, q_tokens, k_tokens, num_heads, scratch_bytes(q_tokens, max_len_k, num_heads, head_dim, dtype, path)).bytes;
}

int ntb200_varlen_attention_backward(const void* grad_out, const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv,
                                     const void* out, const float* lse, void* grad_q, int64_t ld_grad_q, void* grad_k, int64_t ld_grad_k,
                                     void* grad_v, int64_t ld_grad_v, const int64_t* offsets_q, int64_t row_elems_q,
                                     const int64_t* offsets_k, int64_t row_elems_k, int64_t batch, int64_t q_tokens, int64_t k_tokens,
                                     int num_heads, int head_dim, int64_t max_len_q, int64_t max_len_k, float scaling, int dtype, int path,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  if (batch < 0 || q_tokens < 0 || k_tokens < 0 || num_heads < 1 || head_dim < 1 || row_elems_q < 1 || row_elems_k < 1 || max_len_q < 0 ||
      max_len_k < 0 || path < 0 || path > 4 || !std::isfinite(scaling * kLog2e))
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
  const BwdWorkspace at(batch, q_tokens, k_tokens, num_heads,
                        scratch_bytes(q_tokens, max_len_k, num_heads, head_dim, dtype, path));
  if (workspace_bytes < at.bytes) return NTB200_WORKSPACE_TOO_SMALL;
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return NTB200_MISALIGNED;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const BwdArgs a = {grad_out, q, k, v, out, lse, reinterpret_cast<float*>(ws + at.delta), nullptr, grad_q, grad_k, grad_v,
                     ldq, ldk, ldv, ld_grad_q, ld_grad_k, ld_grad_v, offsets_q, offsets_k, row_elems_q, row_elems_k,
                     batch, q_tokens, num_heads, head_dim, scaling};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t max_len = max_len_q > max_len_k ? max_len_q : max_len_k;
  switch (dtype) {
    case NTB200_F32: return launch_bwd<float>(a, k_tokens, max_len, ws, at, path, st);
    case NTB200_F16: return launch_bwd<__half>(a, k_tokens, max_len, ws, at, path, st);
    default: return launch_bwd<__nv_bfloat16>(a, k_tokens, max_len, ws, at, path, st);
  }
}

}  // extern "C"
