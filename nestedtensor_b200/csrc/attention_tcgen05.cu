// Variable-length self-attention on tcgen05 tensor cores, fp16 / bf16, head_dim 64; with row statistics (the forward pass of
// training) head_dim 128 too.  What follows describes 64; Cfg<128> says what differs.
//
// One CTA = one (sequence, head, 128-query tile).  For every block of 128 keys:
//     S[128 x n]   = Q K^T          tcgen05.mma, both operands K-major in shared memory (TMA, 128-B swizzle)
//     P            = exp2(scale*log2e*S - m)   one softmax thread per query ROW (TMEM lane = row, so no
//                                   cross-thread reduction); P is written back over S as packed 16-bit
//     O[128 x 64] += P V            tcgen05.mma with A = P read from tensor memory, B = V tile as MN-major
// S / P (128 columns) and O (64 columns) live in tensor memory (256 columns per CTA, two CTAs per SM so
// one CTA's softmax overlaps the other's MMAs).  Q, K and V tiles come straight out of the packed token
// matrices through 2-D tensor maps (row = token, column = head): for self-attention the three maps are one map over
// the [T, 3E] projection output with column offsets 0 / E / 2E; for cross-attention (queries of sequence b over the
// keys / values of sequence b of another nested tensor) they are maps over the [Tq, E] query projection and the
// key / value projections.  Padded tokens are never materialised; rows past the end of a sequence belong to the next
// sequence (or are zero-filled past the end of the buffer) and are masked / cleared / never stored.
// The list of (sequence, query tile) work items is built on the device, longest sequences first.
// Every wait is bounded; a wait that runs out sets an error flag, the CTA drains and frees its TMEM.
// Replaces steps 2-8 of bt_min_mha (nestedtensor/csrc/cuda/mha.cpp:59-105).

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "attention_internal.cuh"
#include "attention_tc.cuh"
#include "attention_tiny.cuh"
#include "common.cuh"
#include "sm100_ptx.cuh"

namespace ntb200 {
namespace {

__device__ int g_attn_error = 0;  // bit 0 producer, 1 MMA issuer, 2 softmax

constexpr int kQT = 128;   // query rows per CTA (TMEM lanes)
constexpr int kKV = 128;   // keys per block
constexpr int kHalf = kQT * 64 * 2;  // 16 KB: one 128 x 64 two-byte tile, as TMA writes it
// Of the 16 key pairs of a 32-key chunk, pair 2k+1 is exponentiated by the polynomial when bit k is set
// (0xff: half of all exponentials, 0xaa: a quarter, 0: none), the others on the MUFU unit.  A quarter measured
// best on B200 at the BERT-large batch (none: +1 %, half: +6 %).  The polynomial is off by up to 1.9e-4, where rounding P costs
// 3.9e-3 in bf16 and 4.9e-4 in fp16; a training pass in fp16 does without it: the gradients compute P again from the row's
// denominator with exponentials that are right to 2^-22, and the two should agree.
template <int FMT, bool STATS>
constexpr unsigned kPolyPairs = STATS && FMT == 0 ? 0u : 0xaau;
// A row's reference maximum is raised (and its running output rescaled) only when a block's maximum exceeds it
// by more than this many powers of two.
constexpr float kLazyRescale = 8.0f;
constexpr int kTmemCols = 256;        // of each of the two CTAs of an SM
constexpr int kAttnThreads = 256;     // warps 0-3 softmax, warp 4 TMA, warp 5 MMA, warps 6-7 idle
// Register exchange of setmaxnreg.  A request for more registers than the other warps of the CTA give back blocks for
// ever (it is not one of the bounded waits), so the two counts must add up to twice the count the kernel is launched
// with: 128 at two 256-thread CTAs per SM.  With eight warps every SM sub-partition hosts one softmax warp and one
// control / idle warp of the CTA, so the exchange also balances per sub-partition.
constexpr int kRegLaunch = 65536 / (2 * kAttnThreads);
constexpr int kRegSoftmax = 208;
constexpr int kRegControl = 48;
static_assert(kRegSoftmax + kRegControl == 2 * kRegLaunch && kRegLaunch % 8 == 0, "setmaxnreg exchange must balance");

// Head dim 64: S in tensor-memory columns [0,128), P [128,192), O [192,256); Q buffers and K, V stages of 16 KB, two of each.
// Head dim 128: S [0,128) with P over its first half, O [128,256); one Q buffer and one stage of 32 KB, so that two CTAs still
// share an SM: the next QK^T waits for this PV, and the other CTA's products run meanwhile.  Two sequences of about 4500
// tokens, 8 heads, bf16: 197 us (0.83 PFLOP/s) against 564 on the mma.sync kernel; sequences of 1 to 512, 42 against 66; of
// 1 to 128, 31 against 43.  Bound by the softmax warps' issue and latency, as at 64.
template <int D>
struct Cfg {
  static constexpr bool kSepP = D == 64;  // P has columns of its own
  static constexpr int kPCol = kSepP ? 128 : 0, kOCol = kSepP ? 192 : 128;
  static constexpr int kHalves = D / 64;
  static constexpr int kTile = kHalves * kHalf;
  static constexpr int kStages = D == 64 ? 2 : 1, kQBufs = kStages;
  static constexpr int kSmem = 1024 + kTile * (kQBufs + 2 * kStages) + 256;
};

template <int kStages>
struct Ctrl {
  uint64_t full_k[kStages];   // K tile (plus Q with the first block of an item) landed
  uint64_t empty_k[kStages];  // QK^T of that stage retired: K (and the Q buffer two items back) reusable
  uint64_t full_v[kStages];
  uint64_t empty_v[kStages];  // PV of that stage retired (and the softmax warps have stored its P)
  uint64_t s_ready;
  uint64_t s_free;
  uint64_t p_ready;
  uint64_t o_ready;
  uint64_t done;
  uint32_t tmem_base;
  volatile int abort;
};

static_assert(sizeof(Ctrl<2>) <= 256, "control block exceeds its shared-memory slot");

// ------------------------------------------------------------------ work list
// items[i] = (first query token of the tile, valid query rows in the tile, first key token of the sequence, number
// of keys) for every 128-query tile, ordered by decreasing number of key blocks so that the longest items start
// first; *count = number of items.  Sequences without queries or without keys produce no item; the output rows of a
// sequence without keys are zeroed here (an empty softmax).  Sequences of at most skip_short queries and keys produce
// no item either: the caller has given them to the warp-per-(sequence, head) kernel.  One block.
constexpr int kListThreads = 1024;
constexpr int kBuckets = 9;  // key blocks 1..8+, (0 unused)

template <bool SELF>  // SELF: queries and keys are the same sequences, so none has queries without keys
__device__ __forceinline__ void build_items_block(const int64_t* __restrict__ offsets_q, const int64_t* __restrict__ offsets_k,
                                                  int64_t row_elems_q, int64_t row_elems_k, int64_t E, int64_t batch,
                                                  int4* __restrict__ items, int* __restrict__ count, int64_t capacity,
                                                  uint16_t* __restrict__ out, int skip_short) {
  const int nthreads = (int)blockDim.x;  // 1024 alone, 256 beside the short-sequence warps
  __shared__ int s_cnt[kBuckets];
  __shared__ int s_base[kBuckets];
  if (threadIdx.x < kBuckets) s_cnt[threadIdx.x] = 0;
  __syncthreads();
  for (int64_t b = threadIdx.x; b < batch; b += nthreads) {
    const int64_t Lq = (offsets_q[b + 1] - offsets_q[b]) / row_elems_q, Lk = (offsets_k[b + 1] - offsets_k[b]) / row_elems_k;
    if (Lq <= 0 || Lk <= 0 || (Lq <= skip_short && Lk <= skip_short)) continue;
    const int nq = (int)((Lq + kQT - 1) / kQT);
    int nb = (int)((Lk + kKV - 1) / kKV);
    nb = nb >= kBuckets ? kBuckets - 1 : nb;
    atomicAdd(&s_cnt[nb], nq);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int acc = 0;
    for (int k = kBuckets - 1; k >= 1; --k) {
      s_base[k] = acc;
      acc += s_cnt[k];
    }
    *count = acc < capacity ? acc : (int)capacity;
  }
  __syncthreads();
  for (int64_t b = threadIdx.x; b < batch; b += nthreads) {
    const int64_t Lq = (offsets_q[b + 1] - offsets_q[b]) / row_elems_q, Lk = (offsets_k[b + 1] - offsets_k[b]) / row_elems_k;
    if (Lq <= 0 || Lk <= 0 || (Lq <= skip_short && Lk <= skip_short)) continue;
    const int nq = (int)((Lq + kQT - 1) / kQT);
    int nb = (int)((Lk + kKV - 1) / kKV);
    nb = nb >= kBuckets ? kBuckets - 1 : nb;
    const int pos = atomicAdd(&s_base[nb], nq);
    const int tq0 = (int)(offsets_q[b] / row_elems_q), tk0 = (int)(offsets_k[b] / row_elems_k);
    for (int t = 0; t < nq; ++t) {
      const int64_t rows = Lq - (int64_t)t * kQT < kQT ? Lq - (int64_t)t * kQT : kQT;
      if (pos + t < capacity) items[pos + t] = make_int4(tq0 + t * kQT, (int)rows, tk0, (int)Lk);
    }
  }
  if (SELF) return;
  // Queries whose key sequence is empty get zeros (self-attention never has any: Lq == Lk).  The sequences are found in
  // parallel and listed in shared memory; the block then clears their rows together.
  __shared__ int s_nempty;
  __shared__ int s_empty[kListThreads];
  if (threadIdx.x == 0) s_nempty = 0;
  __syncthreads();
  for (int64_t b = threadIdx.x; b < batch; b += nthreads) {
    if (offsets_k[b + 1] > offsets_k[b] || offsets_q[b + 1] == offsets_q[b]) continue;
    const int pos = atomicAdd(&s_nempty, 1);
    if (pos < kListThreads) {
      s_empty[pos] = (int)b;
    } else {  // more than the list holds: this thread clears the rows itself
      for (int64_t e = offsets_q[b] / row_elems_q * E; e < offsets_q[b + 1] / row_elems_q * E; ++e) out[e] = 0;
    }
  }
  __syncthreads();
  const int n_listed = s_nempty < kListThreads ? s_nempty : kListThreads;
  for (int i = 0; i < n_listed; ++i) {
    const int64_t e0 = offsets_q[s_empty[i]] / row_elems_q * E, e1 = offsets_q[s_empty[i] + 1] / row_elems_q * E;
    for (int64_t e = e0 + threadIdx.x; e < e1; e += nthreads) out[e] = 0;
  }
}

__global__ void __launch_bounds__(kListThreads) build_items_kernel(const int64_t* __restrict__ offsets_q,
                                                                   const int64_t* __restrict__ offsets_k, int64_t row_elems_q,
                                                                   int64_t row_elems_k, int64_t E, int64_t batch,
                                                                   int4* __restrict__ items, int* __restrict__ count,
                                                                   int64_t capacity, uint16_t* __restrict__ out) {
  build_items_block<false>(offsets_q, offsets_k, row_elems_q, row_elems_k, E, batch, items, count, capacity, out, 0);
}

// The same list for self-attention on the default path, in one launch with the short sequences: block 0 builds the list
// without the sequences of at most kTinyMaxLen tokens, and every warp of the other blocks computes one (sequence, head)
// of those sequences by itself (attn_tiny_warp; it returns at once for a longer sequence).  The short sequences thus
// cost no launch of their own, and which kernel computes a sequence depends on its own length only.
constexpr int kPrepWarps = 8;
template <int D>
constexpr int kPrepSmem = kPrepWarps * 3 * (int)kTinyMaxLen * D * 2;  // 96 / 192 KB: Q, K, V tiles of 32 x D per warp

template <typename T, int D>
__global__ void __launch_bounds__(kPrepWarps * 32)
prepare_self_attention_kernel(const int64_t* __restrict__ offsets, int64_t row_elems, int64_t batch, int64_t E,
                              int4* __restrict__ items, int* __restrict__ count, int64_t capacity, const T* __restrict__ qkv,
                              T* __restrict__ out, int H, float scale_log2e, LseOut lse) {
  extern __shared__ __align__(128) uint8_t prep_smem[];
  if (blockIdx.x == 0) {
    build_items_block<true>(offsets, offsets, row_elems, row_elems, E, batch, items, count, capacity, reinterpret_cast<uint16_t*>(out),
                            (int)kTinyMaxLen);
    return;
  }
  const int warp = threadIdx.x >> 5;
  attn_tiny_warp<T, D, (int)kTinyMaxLen>(qkv, 3 * E, qkv + E, 3 * E, qkv + 2 * E, 3 * E, out, offsets, offsets, row_elems, row_elems,
                                           batch, H, scale_log2e, ((int64_t)blockIdx.x - 1) * kPrepWarps + warp,
                                           (uint32_t)__cvta_generic_to_shared(prep_smem) + (uint32_t)warp * (uint32_t)(kPrepSmem<D> / kPrepWarps),
                                           lse);
}

// ------------------------------------------------------------------ attention
// Persistent: CTA c works on items c, c + gridDim.x, ... of the flattened (work item, head) list.  All
// barriers run on one global block counter g (one phase per 128-key block).
//   warps 0-3  softmax warpgroup (one thread per query row; registers raised with setmaxnreg so a whole
//              128-key row of S lives in registers: S is read from tensor memory ONCE per block)
//   warp 4     TMA producer   warp 5  MMA issuer (also clears V rows past a sequence's end)   warps 6-7  idle
// Tensor memory (256 columns): S [0,128) fp32, P [128,192) packed 16-bit, O [192,256) fp32.  P has its own
// columns, so QK^T of block g+1 is issued as soon as the softmax warps have read S of block g
// (s_free), before PV of block g: the tensor pipe works under the softmax of the same CTA.
// Two 256-thread CTAs per SM at 128 registers per thread; the control warpgroup then drops to 48 and the
// softmax warpgroup rises to 208.
// The output of an item is written during the FIRST block of the next item (after that block's row maximum,
// 16 columns at a time so that it fits beside the live S row): its last PV retires while the next S is loaded
// and reduced, instead of being waited for.  The softmax warps sit at their register budget; this only pays
// because the write needs about 30 registers (it spilled, and lost 20 %, before the row sums were cut to two
// packed accumulators).
// STATS: the rows' softmax denominators are stored too (LseOut), for a backward pass.
template <int FMT, int D, bool STATS>
__global__ void __launch_bounds__(kAttnThreads, 2)
attn_tcgen05_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                    const __grid_constant__ CUtensorMap map_v, int col_q, int col_k, int col_v, void* __restrict__ out,
                    const int4* __restrict__ items, const int* __restrict__ count, int H, float scale_log2e, LseOut lse) {
  using C = Cfg<D>;
  constexpr int kStages = C::kStages, kTile = C::kTile;
  const int n_items = *count;
  if ((int64_t)blockIdx.x >= (int64_t)n_items * H) return;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Ctrl<kStages>* ctrl = reinterpret_cast<Ctrl<kStages>*>(smem + kTile * (C::kQBufs + 2 * kStages));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t E = (int64_t)H * D;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      ptx::mbar_init(ptx::smem_u32(&ctrl->full_k[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&ctrl->empty_k[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&ctrl->full_v[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&ctrl->empty_v[s]), 5);  // PV commit + the four softmax warps
    }
    ptx::mbar_init(ptx::smem_u32(&ctrl->s_ready), 1);
    ptx::mbar_init(ptx::smem_u32(&ctrl->s_free), 4);
    ptx::mbar_init(ptx::smem_u32(&ctrl->p_ready), 4);
    ptx::mbar_init(ptx::smem_u32(&ctrl->o_ready), 1);
    ptx::mbar_init(ptx::smem_u32(&ctrl->done), 1);
    ctrl->abort = 0;
    ptx::fence_barrier_init();
    ptx::prefetch_tensormap(&map_q);
    ptx::prefetch_tensormap(&map_k);
    ptx::prefetch_tensormap(&map_v);
  }
  if (warp == 5) {
    ptx::tmem_alloc(ptx::smem_u32(&ctrl->tmem_base), kTmemCols);
    ptx::tmem_relinquish();
    ptx::tc_fence_before_sync();
  }
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem_base = ctrl->tmem_base;
  const uint32_t s_q = ptx::smem_u32(smem);          // Q buffers
  const uint32_t s_k = s_q + C::kQBufs * kTile;      // K ring: stage s at s_k + s*kTile
  const uint32_t s_v = s_k + kStages * kTile;        // V ring: stage s at s_v + s*kTile

  // One 16-byte record per work item; every role fetches the record of its NEXT item while it works on
  // the current one, so the load latency never sits on a critical path.
  struct Item {
    int tq, rows, h, L, tok0, n_blk;  // first query token and valid rows of the tile; keys: first token and count
  };
  // Position in the flattened (work item, head) list; a CTA steps through it by gridDim.x without a
  // division per item.
  struct Pos {
    int item, h;
  };
  const int step_items = (int)(gridDim.x / (unsigned)H), step_heads = (int)(gridDim.x % (unsigned)H);
  const Pos first = {(int)(blockIdx.x / (unsigned)H), (int)(blockIdx.x % (unsigned)H)};
  auto next = [&](Pos p) {
    p.item += step_items;
    p.h += step_heads;
    if (p.h >= H) {
      p.h -= H;
      ++p.item;
    }
    return p;
  };
  auto fetch = [&](const Pos& p) { return p.item < n_items ? __ldg(items + p.item) : make_int4(0, 1, 0, 1); };
  auto decode = [&](const Pos& p, const int4& w) {
    Item it;
    it.h = p.h;
    it.tq = w.x;
    it.rows = w.y;
    it.tok0 = w.z;
    it.L = w.w;
    it.n_blk = (w.w + kKV - 1) / kKV;
    return it;
  };

  if (warp >= 4) {
    ptx::setmaxnreg_dec<kRegControl>();
    if (warp == 4 && ptx::elect_one()) {
      // ------------------------------------------------------------ TMA producer
      bool ok = true;
      uint32_t g = 0, n = 0;
      int4 rec = fetch(first);
      for (Pos i = first; i.item < n_items && ok; i = next(i), ++n) {
        const Item it = decode(i, rec);
        rec = fetch(next(i));
        for (int j = 0; j < it.n_blk; ++j, ++g) {
          const uint32_t s = g % kStages, ph = (g / kStages) & 1;
          // K (and Q) as soon as the QK^T that last read this stage has retired ...
          if (!wait_or_abort(ptx::smem_u32(&ctrl->empty_k[s]), ph ^ 1, &ctrl->abort)) {
            ok = false;
            break;
          }
          const uint32_t fk = ptx::smem_u32(&ctrl->full_k[s]);
          ptx::mbar_arrive_expect_tx(fk, (j == 0 ? 2 : 1) * kTile);
          // Q buffer n % kQBufs was last read by item n - kQBufs, all of whose QK^T precede the release of this stage
#pragma unroll
          for (int x = 0; x < C::kHalves; ++x) {
            if (j == 0) ptx::tma_load_2d(s_q + (n % C::kQBufs) * kTile + x * kHalf, &map_q, fk, col_q + it.h * D + x * 64, it.tq);
            ptx::tma_load_2d(s_k + s * kTile + x * kHalf, &map_k, fk, col_k + it.h * D + x * 64, it.tok0 + j * kKV);
          }
          // ... V only once the PV that last read its stage has retired
          if (!wait_or_abort(ptx::smem_u32(&ctrl->empty_v[s]), ph ^ 1, &ctrl->abort)) {
            ok = false;
            ++g;  // the K load of this block was issued: include it in the drain below
            break;
          }
          const uint32_t fv = ptx::smem_u32(&ctrl->full_v[s]);
          ptx::mbar_arrive_expect_tx(fv, kTile);
#pragma unroll
          for (int x = 0; x < C::kHalves; ++x)
            ptx::tma_load_2d(s_v + s * kTile + x * kHalf, &map_v, fv, col_v + it.h * D + x * 64, it.tok0 + j * kKV);
        }
      }
      if (!ok) {
        ctrl->abort = 1;
        atomicOr(&g_attn_error, 1);
      }
      // every issued load must land before exit (a V load that was never issued after an abort cannot
      // complete; that wait is bounded and runs out)
      const uint32_t first = g > (uint32_t)kStages ? g - kStages : 0;
      for (uint32_t k = first; k < g; ++k) {
        ptx::mbar_wait(ptx::smem_u32(&ctrl->full_k[k % kStages]), (k / kStages) & 1);
        if (ok) ptx::mbar_wait(ptx::smem_u32(&ctrl->full_v[k % kStages]), (k / kStages) & 1);
      }
    } else if (warp == 5 && ptx::elect_one()) {
      // ------------------------------------------------------------ MMA issuer
      bool ok = true;
      const uint32_t t_s = tmem_base, t_p = tmem_base + C::kPCol, t_o = tmem_base + C::kOCol;
      constexpr uint32_t idesc_pv = ptx::umma_idesc_f16(FMT, kQT, D, 0, 1);  // B = V is MN-major
      const uint64_t desc_q0 = ptx::umma_desc_kmajor_sw128(s_q);
      const uint64_t desc_k0 = ptx::umma_desc_kmajor_sw128(s_k);
      const uint64_t desc_v0 = ptx::umma_desc_mnmajor_sw128(s_v, C::kHalves > 1 ? kHalf : 16);
      // cursor A: the block whose QK^T is issued next (runs one block ahead of cursor B: PV)
      Pos ia = first;
      uint32_t ga = 0, na = 0;
      int ja = 0;
      Item a = decode(ia, fetch(ia));
      int4 rec_a = fetch(next(ia));
      auto issue_qk = [&]() -> bool {
        const uint32_t s = ga % kStages, ph = (ga / kStages) & 1;
        if (!wait_or_abort(ptx::smem_u32(&ctrl->full_k[s]), ph, &ctrl->abort)) return false;
        ptx::tc_fence_after_sync();
        int nvalid = a.L - ja * kKV;
        nvalid = nvalid > kKV ? kKV : nvalid;
        const uint32_t idesc_qk = ptx::umma_idesc_f16(FMT, kQT, (nvalid + 15) & ~15);
        const uint64_t dq = desc_q0 + (uint64_t)((na % C::kQBufs) * (kTile >> 4));
        const uint64_t dk = desc_k0 + (uint64_t)(s * (kTile >> 4));
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint64_t at = (uint64_t)((k / 4) * (kHalf >> 4) + 2 * (k % 4));
          ptx::umma_f16(t_s, dq + at, dk + at, idesc_qk, k != 0 ? 1u : 0u);
        }
        ptx::umma_commit(ptx::smem_u32(&ctrl->empty_k[s]));
        ptx::umma_commit(ptx::smem_u32(&ctrl->s_ready));
        ++ga;
        if (++ja == a.n_blk) {
          ja = 0;
          ++na;
          ia = next(ia);
          a = decode(ia, rec_a);
          rec_a = fetch(next(ia));
        }
        return true;
      };
      ok = issue_qk();
      uint32_t gb = 0;
      int4 rec_b = fetch(first);
      for (Pos ib = first; ib.item < n_items && ok; ib = next(ib)) {
        const Item b = decode(ib, rec_b);
        rec_b = fetch(next(ib));
        for (int jb = 0; jb < b.n_blk && ok; ++jb, ++gb) {
          // S of block gb is in the softmax warps' registers: the next QK^T may overwrite it
          if (C::kSepP && ia.item < n_items) {
            if (!wait_or_abort(ptx::smem_u32(&ctrl->s_free), gb & 1, &ctrl->abort)) { ok = false; break; }
            if (!issue_qk()) { ok = false; break; }
          }
          const uint32_t s = gb % kStages;
          int nvalid = b.L - jb * kKV;
          nvalid = nvalid > kKV ? kKV : nvalid;
          if ((nvalid & 15) != 0) {
            // The last 16-key step of a ragged block multiplies P (exactly zero there) with V rows that belong to the
            // NEXT sequence: 0 x NaN or 0 x Inf in such a row would reach this sequence's output.  While the softmax
            // warps are still busy with this block, this thread clears those rows of the landed V tile, so that a
            // non-finite value stays inside the sequence that holds it (the reference pads every sequence with zeros).
            if (!wait_or_abort(ptx::smem_u32(&ctrl->full_v[s]), (gb / kStages) & 1, &ctrl->abort)) { ok = false; break; }
            const int r_end = (nvalid + 15) & ~15;
            for (int r = nvalid; r < r_end; ++r) {
              const uint32_t addr = s_v + s * kTile + (uint32_t)((r >> 3) * 1024 + (r & 7) * 128);
#pragma unroll
              for (int c = 0; c < 8 * C::kHalves; ++c)
                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(addr + (c / 8) * kHalf + (c % 8) * 16), "r"(0u) : "memory");
            }
            ptx::fence_proxy_async();  // make the generic-proxy stores visible to the tensor core's reads
          }
          if (!wait_or_abort(ptx::smem_u32(&ctrl->p_ready), gb & 1, &ctrl->abort)) { ok = false; break; }
          if (!wait_or_abort(ptx::smem_u32(&ctrl->full_v[s]), (gb / kStages) & 1, &ctrl->abort)) { ok = false; break; }
          ptx::tc_fence_after_sync();
          const int ksteps = (nvalid + 15) >> 4;
          const uint64_t dv = desc_v0 + (uint64_t)(s * (kTile >> 4));
#pragma unroll
          for (int ks = 0; ks < kKV / 16; ++ks) {
            if (ks < ksteps)
              ptx::umma_f16_ts(t_o, t_p + ks * 8, dv + (uint64_t)(ks * (2048 >> 4)), idesc_pv, (jb | ks) != 0 ? 1u : 0u);
          }
          ptx::umma_commit(ptx::smem_u32(&ctrl->empty_v[s]));
          ptx::umma_commit(ptx::smem_u32(&ctrl->o_ready));
          if (!C::kSepP && ia.item < n_items) {
            // P lies over S: the next QK^T waits for this PV (the SM's other CTA works meanwhile)
            if (!wait_or_abort(ptx::smem_u32(&ctrl->o_ready), gb & 1, &ctrl->abort)) { ok = false; break; }
            if (!issue_qk()) { ok = false; break; }
          }
        }
      }
      if (!ok) {
        ctrl->abort = 1;
        atomicOr(&g_attn_error, 2);
      }
      // every MMA issued must have retired before tensor memory is freed
      ptx::umma_commit(ptx::smem_u32(&ctrl->done));
      ptx::mbar_wait(ptx::smem_u32(&ctrl->done), 0);
    }
  } else {
    // ------------------------------------------------------------ softmax, one thread per query row
    ptx::setmaxnreg_inc<kRegSoftmax>();
    const int q = warp;                              // TMEM lane quarter of this warp
    const int row = q * 32 + lane;                   // row inside the tile = TMEM lane
    const uint32_t lane_addr = (uint32_t)(q * 32) << 16;
    const uint32_t t_s = tmem_base + lane_addr, t_p = tmem_base + C::kPCol + lane_addr, t_o = tmem_base + C::kOCol + lane_addr;
    bool ok = true;
    uint32_t g = 0;

    // State of the item whose output is still to be written (by write_pending, during the next item).
    struct Pending {
      bool any;          // an item is waiting for its output
      bool warp_active;  // this warp owns valid rows of it
      float inv;         // 1 / softmax denominator of this thread's row
      int rows;          // valid rows in the tile
      int64_t out_row0;  // element offset of (first token of the tile, head) in the output
    } pend = {false, false, 0.0f, 0, 0};
    auto write_pending = [&]() {
      // each thread normalises its own row and stores it 32 bytes (one full sector) at a time, 16 accumulator
      // columns per step so that it fits beside a live S row
      if (pend.warp_active) {
        const bool live = row < pend.rows;  // (the tensor-memory loads are warp-wide: only the store is per row)
        const float inv = pend.inv;
        uint16_t* orow = reinterpret_cast<uint16_t*>(out) + pend.out_row0 + (int64_t)row * E;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          uint32_t r0[16];
          ptx::tmem_ld_32x32b_x16(t_o + c * 16, r0);
          ptx::tmem_ld_wait();
          if (live)
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(orow + c * 16),
                       "r"(pack2<FMT>(__uint_as_float(r0[0]) * inv, __uint_as_float(r0[1]) * inv)),
                       "r"(pack2<FMT>(__uint_as_float(r0[2]) * inv, __uint_as_float(r0[3]) * inv)),
                       "r"(pack2<FMT>(__uint_as_float(r0[4]) * inv, __uint_as_float(r0[5]) * inv)),
                       "r"(pack2<FMT>(__uint_as_float(r0[6]) * inv, __uint_as_float(r0[7]) * inv)),
                       "r"(pack2<FMT>(__uint_as_float(r0[8]) * inv, __uint_as_float(r0[9]) * inv)),
                       "r"(pack2<FMT>(__uint_as_float(r0[10]) * inv, __uint_as_float(r0[11]) * inv)),
                       "r"(pack2<FMT>(__uint_as_float(r0[12]) * inv, __uint_as_float(r0[13]) * inv)),
                       "r"(pack2<FMT>(__uint_as_float(r0[14]) * inv, __uint_as_float(r0[15]) * inv))
                       : "memory");
        }
      }
      pend.any = false;
    };
    int4 rec = fetch(first);
    for (Pos i = first; i.item < n_items; i = next(i)) {
      const Item it = decode(i, rec);
      rec = fetch(next(i));
      const bool warp_active = q * 32 < it.rows;  // warp-uniform
      float m = -INFINITY, l = 0.0f;
      for (int j = 0; j < it.n_blk; ++j, ++g) {
        if (ok && !wait_or_abort(ptx::smem_u32(&ctrl->s_ready), g & 1, &ctrl->abort)) ok = false;
        int nvalid = it.L - j * kKV;
        nvalid = nvalid > kKV ? kKV : nvalid;
        const int nchunks = (nvalid + 31) >> 5;
        uint32_t sv[4][32];  // the whole row of S (up to 128 keys) in registers
        if (ok && warp_active) {
          ptx::tc_fence_after_sync();
          ptx::tmem_ld_32x32b_x32(t_s, sv[0]);
          if (nchunks > 1) ptx::tmem_ld_32x32b_x32(t_s + 32, sv[1]);
          if (nchunks > 2) ptx::tmem_ld_32x32b_x32(t_s + 64, sv[2]);
          if (nchunks > 3) ptx::tmem_ld_32x32b_x32(t_s + 96, sv[3]);
          ptx::tmem_ld_wait();
        }
        // S has been consumed: the MMA warp may issue the next block's QK^T
        if (C::kSepP) {
          ptx::tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&ctrl->s_free));
        }
        float m_new = m, corr = 1.0f;
        bool any_up = false;
        if (ok && warp_active) {
          // Keys past the end of the sequence become -inf once, here, so that the maximum and the exponentials
          // below need no per-element predicate (only the last 32-key chunk of a block can be ragged).
          // (Written as a loop of zero or one trips: as a plain `if` the compiler predicates the 128 selects and
          // issues them for every block, ragged or not - about 230 cycles per block on the measured build.)
#pragma unroll 1
          for (int ragged = (nvalid & 31) != 0 ? 1 : 0; ragged > 0; --ragged) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              // (a range test, not "c == nchunks - 1": the latter is turned into a run-time index and sends the
              // row to local memory)
              if (nvalid > c * 32 && nvalid < (c + 1) * 32) {
#pragma unroll
                for (int k = 0; k < 32; ++k) sv[c][k] = (c * 32 + k >= nvalid) ? 0xff800000u : sv[c][k];
              }
            }
          }
          // row maximum, four independent chains of three-input maxima
          float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if (c < nchunks) {
#pragma unroll
              for (int k = 0; k < 32; k += 8) {
                mx0 = ptx::fmax3(mx0, __uint_as_float(sv[c][k]), __uint_as_float(sv[c][k + 1]));
                mx1 = ptx::fmax3(mx1, __uint_as_float(sv[c][k + 2]), __uint_as_float(sv[c][k + 3]));
                mx2 = ptx::fmax3(mx2, __uint_as_float(sv[c][k + 4]), __uint_as_float(sv[c][k + 5]));
                mx3 = ptx::fmax3(mx3, __uint_as_float(sv[c][k + 6]), __uint_as_float(sv[c][k + 7]));
              }
            }
          }
          const float mxs = fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3)) * scale_log2e;
          if (j == 0) {
            m_new = mxs;  // the first block of an item: O is overwritten and the row sum starts at zero
          } else {
            // Lazy rescaling: while no row of the warp exceeds its reference maximum by more than kLazyRescale, the
            // reference stays and P simply grows up to 2^kLazyRescale, which fp32 sums and 16-bit P hold without
            // loss; the final division by the row sum cancels the offset.
            any_up = __any_sync(0xffffffffu, mxs > m + kLazyRescale);
            if (any_up) {
              m_new = fmaxf(m, mxs);
              corr = ptx::ex2_approx(m - m_new);
            }
          }
        }
        // PV of the previous block must have retired before P is overwritten / O is rescaled
        if (ok && g > 0 && !wait_or_abort(ptx::smem_u32(&ctrl->o_ready), (g - 1) & 1, &ctrl->abort)) ok = false;
        if (ok && j == 0 && pend.any) {
          // Output of the previous item, written while this item's first block is already in flight: its last
          // PV retired during the work above, and this item's first PV (which overwrites O) cannot be issued
          // before these warps arrive at p_ready below.
          ptx::tc_fence_after_sync();
          write_pending();
        }
        if (ok && warp_active) {
          ptx::tc_fence_after_sync();
          if (any_up) {
            // rescale the running output (only when some row of the warp raised its reference maximum)
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {  // 16 columns at a time: the S row stays live in registers
              uint32_t r0[16];
              ptx::tmem_ld_32x32b_x16(t_o + c * 16, r0);
              ptx::tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < 16; ++k) r0[k] = __float_as_uint(__uint_as_float(r0[k]) * corr);
              ptx::tmem_st_32x32b_x16(t_o + c * 16, r0);
            }
          }
          // P = exp2(S*scale*log2e - m_new), packed two per column.  A quarter of the exponentials go through
          // a polynomial on the FMA pipe instead of the MUFU unit (16 results per clock per SM); measured at
          // the BERT-large workload a quarter beats none, three eighths and a half, because the polynomial
          // costs about five issue slots per value.  Scaling, polynomial and row sum run on packed fp32 pairs.
          const uint64_t sc2 = ptx::f32x2_pack(scale_log2e, scale_log2e);
          const uint64_t nm2 = ptx::f32x2_pack(-m_new, -m_new);
          uint64_t acc0 = 0, acc1 = 0;  // packed partial row sums (four independent chains)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if (c < nchunks) {
              uint32_t pk[16];
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const uint64_t xa = ptx::f32x2_fma(ptx::f32x2_pack(__uint_as_float(sv[c][4 * k]), __uint_as_float(sv[c][4 * k + 1])), sc2, nm2);
                const uint64_t xb = ptx::f32x2_fma(ptx::f32x2_pack(__uint_as_float(sv[c][4 * k + 2]), __uint_as_float(sv[c][4 * k + 3])), sc2, nm2);
                float a0, a1, b0, b1;
                ptx::f32x2_unpack(xa, a0, a1);
                ptx::f32x2_unpack(xb, b0, b1);
                const float p0 = ptx::ex2_approx(a0), p1 = ptx::ex2_approx(a1);
                float p2, p3;
                if ((kPolyPairs<FMT, STATS> >> k) & 1) {
                  if (STATS) {  // (the polynomial's exponent arithmetic loses a NaN: 0 x brings it back)
                    const uint64_t x = ptx::f32x2_pack(ptx::fmax_nan(b0, -126.0f), ptx::fmax_nan(b1, -126.0f));
                    ptx::ex2_poly_x2(x, p2, p3);
                    ptx::f32x2_unpack(ptx::f32x2_fma(x, ptx::f32x2_pack(0.0f, 0.0f), ptx::f32x2_pack(p2, p3)), p2, p3);
                  } else {
                    ptx::ex2_poly_x2(ptx::f32x2_pack(fmaxf(b0, -126.0f), fmaxf(b1, -126.0f)), p2, p3);
                  }
                } else {
                  p2 = ptx::ex2_approx(b0);
                  p3 = ptx::ex2_approx(b1);
                }
                acc0 = ptx::f32x2_add(acc0, ptx::f32x2_pack(p0, p1));
                acc1 = ptx::f32x2_add(acc1, ptx::f32x2_pack(p2, p3));
                pk[2 * k] = pack2<FMT>(p0, p1);
                pk[2 * k + 1] = pack2<FMT>(p2, p3);
              }
              ptx::tmem_st_32x32b_x16(t_p + c * 16, pk);
            }
          }
          float rs, rs_hi;
          ptx::f32x2_unpack(ptx::f32x2_add(acc0, acc1), rs, rs_hi);
          rs += rs_hi;
          l = l * corr + rs;
          m = m_new;
          ptx::tmem_st_wait();
        }
        ptx::tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          ptx::mbar_arrive(ptx::smem_u32(&ctrl->p_ready));
          ptx::mbar_arrive(ptx::smem_u32(&ctrl->empty_v[g % kStages]));
        }
      }
      // the output of this item is written during the next item's first block (or after the loop)
      pend.any = true;
      pend.warp_active = warp_active;
      pend.inv = 1.0f / l;
      pend.rows = it.rows;
      pend.out_row0 = (int64_t)it.tq * E + (int64_t)it.h * D;
      if (STATS && ok && row < it.rows) lse.ptr[(int64_t)it.h * lse.ld + it.tq + row] = m + log2f(l);
    }
    if (ok && pend.any) {  // the last item of this CTA
      if (!wait_or_abort(ptx::smem_u32(&ctrl->o_ready), (g - 1) & 1, &ctrl->abort)) ok = false;
      if (ok) {
        ptx::tc_fence_after_sync();
        write_pending();
      }
    }
    if (!ok && lane == 0) {
      ctrl->abort = 1;
      atomicOr(&g_attn_error, 4);
    }
  }

  ptx::tc_fence_before_sync();
  __syncthreads();
  if (warp == 5) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc(tmem_base, kTmemCols);
  }
}

template <int FMT, int D, bool STATS>
int launch(const TileSource& q, int col_q, const TileSource& k, int col_k, const TileSource& v, int col_v, void* out,
           const AttnRows& rows, int64_t batch, int64_t q_tokens, int H, float scaling, int dtype, void* workspace, cudaStream_t st,
           int skip_short) {  // skip_short > 0: self-attention only
  const int64_t E = (int64_t)H * D;
  CUtensorMap map_q, map_k, map_v;
  if (!make_tile_map(&map_q, q, dtype) || !make_tile_map(&map_k, k, dtype) || !make_tile_map(&map_v, v, dtype))
    return NTB200_LAUNCH_FAILED;
  static std::atomic<int> attr_set[kMaxDevices];
  if (!once_per_device(attr_set, [] {
        return cudaFuncSetAttribute(attn_tcgen05_kernel<FMT, D, STATS>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::kSmem) == cudaSuccess;
      }))
    return NTB200_LAUNCH_FAILED;
  const int64_t capacity = attn_tcgen05_item_capacity(batch, q_tokens);
  int* count = static_cast<int*>(workspace);
  int4* items = reinterpret_cast<int4*>(static_cast<uint8_t*>(workspace) + 16);
  if (skip_short > 0) {
    // self-attention on the default path (q, k and v are column blocks of one [T, 3E] matrix, offsets_q == offsets_k)
    using T16 = typename std::conditional<FMT == 0, __half, __nv_bfloat16>::type;
    static std::atomic<int> prep_set[kMaxDevices];
    if (!once_per_device(prep_set, [] {
          return cudaFuncSetAttribute(prepare_self_attention_kernel<T16, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, kPrepSmem<D>) ==
                 cudaSuccess;
        }))
      return NTB200_LAUNCH_FAILED;
    const int64_t blocks = 1 + (batch * H + kPrepWarps - 1) / kPrepWarps;
    if (blocks > 0x7fffffffll) return NTB200_UNSUPPORTED_SHAPE;
    prepare_self_attention_kernel<T16, D><<<(unsigned)blocks, kPrepWarps * 32, kPrepSmem<D>, st>>>(
        rows.offsets_q, rows.row_elems_q, batch, E, items, count, capacity, static_cast<const T16*>(q.base), static_cast<T16*>(out), H,
        scaling * 1.4426950408889634f, LseOut{rows.lse, q_tokens});
  } else {
    build_items_kernel<<<1, kListThreads, 0, st>>>(rows.offsets_q, rows.offsets_k, rows.row_elems_q, rows.row_elems_k, E, batch, items,
                                                   count, capacity, static_cast<uint16_t*>(out));
  }
  int dev = 0, sms = kNumSMs;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  int64_t grid = 2ll * sms;  // two resident CTAs per SM, each loops over its share of the items
  if (grid > capacity * H) grid = capacity * H;
  attn_tcgen05_kernel<FMT, D, STATS><<<(unsigned)grid, kAttnThreads, Cfg<D>::kSmem, st>>>(
      map_q, map_k, map_v, col_q, col_k, col_v, out, items, count, H, scaling * 1.4426950408889634f, LseOut{rows.lse, q_tokens});
  return status_from_cuda(cudaGetLastError());
}

}  // namespace

int64_t attn_tcgen05_item_capacity(int64_t batch, int64_t total_tokens) { return batch + total_tokens / kQT + 1; }

size_t attn_tcgen05_workspace_bytes(int64_t batch, int64_t total_tokens) {
  return 16 + sizeof(int4) * (size_t)attn_tcgen05_item_capacity(batch, total_tokens);
}

bool attn_tcgen05_supported(int64_t batch, int64_t total_tokens, int num_heads, int head_dim, int dtype, bool stats) {
  return (head_dim == 64 || (stats && head_dim == 128)) && (dtype == NTB200_F16 || dtype == NTB200_BF16) && num_heads <= 65535 &&
         total_tokens < (1ll << 31) - kQT && 3ll * num_heads * head_dim < (1ll << 31) &&
         attn_tcgen05_item_capacity(batch, total_tokens) < (1ll << 31);
}

namespace {

using LaunchFn = decltype(&launch<0, 64, false>);

LaunchFn pick(int dtype, int d, bool stats) {  // (head dim 128 comes with statistics only: attn_tcgen05_supported)
  if (dtype == NTB200_F16) return d == 128 ? launch<0, 128, true> : stats ? launch<0, 64, true> : launch<0, 64, false>;
  return d == 128 ? launch<1, 128, true> : stats ? launch<1, 64, true> : launch<1, 64, false>;
}

}  // namespace

int attn_tcgen05_launch(const void* qkv, void* out, const AttnRows& rows, int64_t batch, int64_t total_tokens, int H, int d, float scaling,
                        int dtype, void* workspace, cudaStream_t st, int skip_short) {
  const int64_t E = (int64_t)H * d;
  const TileSource src = {qkv, total_tokens, 3 * E, 3 * E};  // one map, three column offsets
  return pick(dtype, d, rows.lse != nullptr)(src, 0, src, (int)E, src, (int)(2 * E), out, rows, batch, total_tokens, H, scaling, dtype, workspace,
                                             st, skip_short);
}

int attn_tcgen05_cross_launch(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv, void* out,
                              const AttnRows& rows, int64_t batch, int64_t q_tokens, int64_t k_tokens, int H, int d, float scaling, int dtype,
                              void* workspace, cudaStream_t st) {
  const int64_t E = (int64_t)H * d;
  const TileSource sq = {q, q_tokens, E, ldq}, sk = {k, k_tokens, E, ldk}, sv = {v, k_tokens, E, ldv};
  return pick(dtype, d, rows.lse != nullptr)(sq, 0, sk, 0, sv, 0, out, rows, batch, q_tokens, H, scaling, dtype, workspace, st, 0);
}

int attn_tcgen05_error_flags_read_and_clear() {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_attn_error, sizeof(int)) != cudaSuccess) return -1;
  if (v != 0) {
    int zero = 0;
    cudaMemcpyToSymbol(g_attn_error, &zero, sizeof(int));
  }
  return v;
}

}  // namespace ntb200
