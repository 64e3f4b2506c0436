// Attention backward pass on tcgen05 tensor cores, heads of 64 and 128, fp16 / bf16 (mathematics: attention_backward.cu).
//
// A work item is (128 own rows, head) of one sequence; the other side's rows come in tiles of 128.  Own rows are keys (KV items:
// dV, dK) or queries (Q items: dQ); with A_own, B_own = K, V / Q, dO and A_c, B_c = Q, dO / K, V:
//     S  = A_own A_c^T       dP = B_own B_c^T        tcgen05.mma, all operands K-major tiles in shared memory (TMA, 128-B swizzle)
//     P  = 2^(a log2(e) S - lse)   dS = P * (dP - D)  one thread per own row and half of its columns, in registers
//     acc1 += P B_c (KV)     acc2 += dS A_c           A = P, dS from tensor memory (16-bit, packed), B = the same tiles, MN-major
// P and dS thus never pass through shared memory, and a gradient is one block's sum over its sequence in order: no atomics.
// Taking dQ in items of its own computes S and dP twice (7 products instead of 5), in exchange for fp32 sums that stay in
// tensor memory and never meet in global memory.
//
// Persistent, one CTA per SM (the accumulators of two gradients, S and dP fill most of its tensor memory); 12 warps:
//     warps 0-7   softmax: warps w and w + 4 share 32 rows, each takes every other chunk of 32 columns
//     warp 8 TMA, warp 9 MMA, warps 10-11 helpers: row statistics of KV items' queries into shared memory, and the rows of a ragged
//                 tile past the sequence's end cleared (a zero probability times a neighbour's NaN or Inf would reach the sum)
// Tensor memory: S [0,128), dP [128,256), acc1 and acc2 from 256.  Heads of 64 leave room for P and dS of their own, so the next
// tile's S and dP are computed while this tile's are still operands; at 128 P and dS take the columns of the S and dP chunks
// they come from (a thread overwrites only what it has read itself), and the next S waits for this P's product.
// All barriers count tiles g of the CTA over its items.  Every wait is bounded: a wait that runs out sets an error flag, the
// roles fall through and the CTA frees its tensor memory.

#include <type_traits>

#include "attention_backward.cuh"
#include "attention_tc.cuh"
#include "common.cuh"
#include "sm100_ptx.cuh"

namespace ntb200 {
namespace {

__device__ int g_attn_bwd_error = 0;  // bit 0 producer / helpers, 1 MMA issuer, 2 softmax

constexpr int kTR = 128;                // rows of a tile
constexpr int kHalf = kTR * 64 * 2;     // 16 KB: 128 rows x 64 columns
constexpr int kBwdThreads = 384;
constexpr int kRegSoftmax = 216, kRegControl = 72, kRegLaunch = 168;
// (setmaxnreg blocks for ever on registers nobody gives back: the shares must add up to what the block was launched with)
static_assert(2 * kRegSoftmax + kRegControl == 3 * kRegLaunch && kRegLaunch % 8 == 0 && kRegLaunch * kBwdThreads <= 65536,
              "setmaxnreg exchange must balance");

template <int D>
struct Cfg {
  static constexpr int kHalves = D / 64;
  static constexpr int kTile = kHalves * kHalf;
  static constexpr bool kSep = D == 64;           // P and dS have columns of their own
  static constexpr int kOwn = D == 64 ? 2 : 1;    // own tile pairs in shared memory
  static constexpr int kStages = D == 64 ? 4 : 2; // other tile pairs
  static constexpr int kAcc1 = 256, kAcc2 = 256 + D;
  static constexpr int kStats = 2 * kTR * 4;      // -lse and -D of a stage
  static constexpr int kSmem = 1024 + (kOwn + kStages) * 2 * kTile + kStages * kStats + 512;
  // tensor-memory columns of the packed P and dS of a chunk of 32 columns
  static __device__ __forceinline__ int p_col(int chunk) { return kSep ? 384 + 16 * chunk : 32 * chunk; }
  static __device__ __forceinline__ int ds_col(int chunk) { return kSep ? 448 + 16 * chunk : 128 + 32 * chunk; }
};

template <int D>
struct Ctrl {
  uint64_t own_full[Cfg<D>::kOwn], own_empty[Cfg<D>::kOwn];
  uint64_t full[Cfg<D>::kStages], empty[Cfg<D>::kStages], aux[Cfg<D>::kStages];
  uint64_t s_ready, s_free, p_ready, p_done, dp_ready, dp_free, ds_ready, ds_done, acc_free, done;
  uint32_t tmem_base;
  volatile int abort;
};

struct TcArgs {
  BwdArgs a;
  ListOut kv, qi;
};

template <int FMT, int D>
__global__ void __launch_bounds__(kBwdThreads, 1)
attn_bwd_tcgen05_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                        const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_g, const __grid_constant__ TcArgs t) {
  using C = Cfg<D>;
  using T = typename std::conditional<FMT == 0, __half, __nv_bfloat16>::type;
  static_assert(sizeof(Ctrl<D>) <= 512, "control block exceeds its shared-memory slot");
  const BwdArgs& a = t.a;
  const unsigned H = (unsigned)a.H;
  const unsigned n_kv = (unsigned)*t.kv.count * H, n_all = n_kv + (unsigned)*t.qi.count * H;
  if (blockIdx.x >= n_all) return;
  extern __shared__ uint8_t bwd_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(bwd_smem_raw) + 1023) & ~uintptr_t(1023));
  float* s_stats = reinterpret_cast<float*>(smem + (C::kOwn + C::kStages) * 2 * C::kTile);
  Ctrl<D>* ctrl = reinterpret_cast<Ctrl<D>*>(reinterpret_cast<uint8_t*>(s_stats) + C::kStages * C::kStats);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kOwn; ++s) {
      ptx::mbar_init(ptx::smem_u32(&ctrl->own_full[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&ctrl->own_empty[s]), 1);
    }
    for (int s = 0; s < C::kStages; ++s) {
      ptx::mbar_init(ptx::smem_u32(&ctrl->full[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&ctrl->empty[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&ctrl->aux[s]), 2);  // both helper warps
    }
    ptx::mbar_init(ptx::smem_u32(&ctrl->s_ready), 1);
    ptx::mbar_init(ptx::smem_u32(&ctrl->s_free), 8);
    ptx::mbar_init(ptx::smem_u32(&ctrl->p_ready), 8);
    ptx::mbar_init(ptx::smem_u32(&ctrl->p_done), 1);
    ptx::mbar_init(ptx::smem_u32(&ctrl->dp_ready), 1);
    ptx::mbar_init(ptx::smem_u32(&ctrl->dp_free), 8);
    ptx::mbar_init(ptx::smem_u32(&ctrl->ds_ready), 8);
    ptx::mbar_init(ptx::smem_u32(&ctrl->ds_done), 1);
    ptx::mbar_init(ptx::smem_u32(&ctrl->acc_free), 8);
    ptx::mbar_init(ptx::smem_u32(&ctrl->done), 1);
    ctrl->abort = 0;
    ptx::fence_barrier_init();
    ptx::prefetch_tensormap(&map_q);
    ptx::prefetch_tensormap(&map_k);
    ptx::prefetch_tensormap(&map_v);
    ptx::prefetch_tensormap(&map_g);
  }
  if (warp == 9) {
    ptx::tmem_alloc(ptx::smem_u32(&ctrl->tmem_base), 512);
    ptx::tmem_relinquish();
    ptx::tc_fence_before_sync();
  }
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem = ctrl->tmem_base;
  const uint32_t s_own = ptx::smem_u32(smem);                  // own pair o at s_own + o * 2 * kTile: A, then B
  const uint32_t s_oth = s_own + C::kOwn * 2 * C::kTile;       // stage s at s_oth + s * 2 * kTile: A, then B

  // Work item w: KV items first (the longer ones), then Q items; every role walks the same items and fetches the record of the
  // next one while it works on this one.
  auto fetch = [&](unsigned w) {
    if (w >= n_all) return make_int4(0, 0, 0, 0);
    return __ldg(w < n_kv ? t.kv.items + w / H : t.qi.items + (w - n_kv) / H);
  };
  auto head = [&](unsigned w) { return (int)((w < n_kv ? w : w - n_kv) % H); };
  auto tiles_of = [](const Item& it) { return (it.n_other + kTR - 1) / kTR; };
  auto wait = [&](uint64_t* bar, uint32_t parity) { return wait_or_abort(ptx::smem_u32(bar), parity, &ctrl->abort); };

  if (warp >= 8) {
    ptx::setmaxnreg_dec<kRegControl>();
    if (warp == 8 && ptx::elect_one()) {
      // ------------------------------------------------------------ TMA producer
      bool ok = true;
      uint32_t g = 0, n = 0;
      int4 rec = fetch(blockIdx.x);
      for (unsigned w = blockIdx.x; w < n_all && ok; w += gridDim.x) {
        const Item it = decode(rec);
        rec = fetch(w + gridDim.x);
        const int nt = tiles_of(it);
        if (nt == 0) continue;
        const bool kv = w < n_kv;
        const int col = head(w) * D;
        const uint32_t o = n % C::kOwn;
        if (!wait(&ctrl->own_empty[o], ((n / C::kOwn) & 1) ^ 1)) {
          ok = false;
          break;
        }
        const uint32_t bo = ptx::smem_u32(&ctrl->own_full[o]);
        ptx::mbar_arrive_expect_tx(bo, 2 * C::kTile);
#pragma unroll
        for (int x = 0; x < C::kHalves; ++x) {
          ptx::tma_load_2d(s_own + o * 2 * C::kTile + x * kHalf, kv ? &map_k : &map_q, bo, col + 64 * x, (int)it.row0);
          ptx::tma_load_2d(s_own + o * 2 * C::kTile + C::kTile + x * kHalf, kv ? &map_v : &map_g, bo, col + 64 * x, (int)it.row0);
        }
        ++n;
        for (int j = 0; j < nt; ++j, ++g) {
          const uint32_t s = g % C::kStages;
          if (!wait(&ctrl->empty[s], ((g / C::kStages) & 1) ^ 1)) {
            ok = false;
            break;
          }
          const uint32_t b = ptx::smem_u32(&ctrl->full[s]);
          ptx::mbar_arrive_expect_tx(b, 2 * C::kTile);
          const int row = (int)it.other + j * kTR;
#pragma unroll
          for (int x = 0; x < C::kHalves; ++x) {
            ptx::tma_load_2d(s_oth + s * 2 * C::kTile + x * kHalf, kv ? &map_q : &map_k, b, col + 64 * x, row);
            ptx::tma_load_2d(s_oth + s * 2 * C::kTile + C::kTile + x * kHalf, kv ? &map_g : &map_v, b, col + 64 * x, row);
          }
        }
      }
      if (!ok) {
        ctrl->abort = 1;
        atomicOr(&g_attn_bwd_error, 1);
      }
      // every issued load must land before the block exits
      for (uint32_t k = n > (uint32_t)C::kOwn ? n - C::kOwn : 0; k < n; ++k)
        ptx::mbar_wait(ptx::smem_u32(&ctrl->own_full[k % C::kOwn]), (k / C::kOwn) & 1);
      for (uint32_t k = g > (uint32_t)C::kStages ? g - C::kStages : 0; k < g; ++k)
        ptx::mbar_wait(ptx::smem_u32(&ctrl->full[k % C::kStages]), (k / C::kStages) & 1);
    } else if (warp == 9 && ptx::elect_one()) {
      // ------------------------------------------------------------ MMA issuer
      constexpr uint32_t idesc_acc = ptx::umma_idesc_f16(FMT, kTR, 64, 0, 1);  // B is MN-major, 64 columns at a time
      const uint64_t d_own = ptx::umma_desc_kmajor_sw128(s_own);
      const uint64_t d_oth = ptx::umma_desc_kmajor_sw128(s_oth);
      const uint64_t d_mn = ptx::umma_desc_mnmajor_sw128(s_oth);
      // cursor of the tile whose S and dP are issued next: one tile ahead of the products with P and dS
      unsigned wa = blockIdx.x;
      uint32_t ga = 0, na = 0;
      int ja = 0, nta = 0, n_other_a = 0;
      int4 rec_a = fetch(wa);
      auto settle = [&]() {  // to the next item that has tiles
        while (wa < n_all) {
          const Item it = decode(rec_a);
          rec_a = fetch(wa + gridDim.x);
          nta = tiles_of(it);
          n_other_a = it.n_other;
          if (nta > 0) return;
          wa += gridDim.x;
        }
      };
      settle();
      auto scores = [&](uint32_t tm, int which, uint64_t* ready) {  // which: 0 = A (S), 1 = B (dP)
        const uint32_t s = ga % C::kStages, o = na % C::kOwn;
        int nc = n_other_a - ja * kTR;
        nc = nc > kTR ? kTR : nc;
        const uint32_t idesc = ptx::umma_idesc_f16(FMT, kTR, (nc + 15) & ~15);
        const uint64_t da = d_own + (uint64_t)((o * 2 + which) * (C::kTile >> 4));
        const uint64_t db = d_oth + (uint64_t)((s * 2 + which) * (C::kTile >> 4));
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint64_t at = (uint64_t)((k / 4) * (kHalf >> 4) + 2 * (k % 4));
          ptx::umma_f16(tm, da + at, db + at, idesc, k != 0 ? 1u : 0u);
        }
        ptx::umma_commit(ptx::smem_u32(ready));
      };
      auto issue_s = [&]() -> bool {
        if (ja == 0 && !wait(&ctrl->own_full[na % C::kOwn], (na / C::kOwn) & 1)) return false;
        if (!wait(&ctrl->full[ga % C::kStages], (ga / C::kStages) & 1)) return false;
        ptx::tc_fence_after_sync();
        scores(tmem, 0, &ctrl->s_ready);
        return true;
      };
      auto issue_dp = [&]() {  // (its tiles landed before issue_s)
        ptx::tc_fence_after_sync();
        scores(tmem + 128, 1, &ctrl->dp_ready);
        ++ga;
        if (++ja == nta) {
          ptx::umma_commit(ptx::smem_u32(&ctrl->own_empty[na % C::kOwn]));
          ja = 0;
          ++na;
          wa += gridDim.x;
          settle();
        }
      };
      bool ok = true;
      if (wa < n_all) {
        ok = issue_s();
        if (ok) issue_dp();
      }
      uint32_t g = 0, n = 0;
      int4 rec = fetch(blockIdx.x);
      for (unsigned w = blockIdx.x; w < n_all && ok; w += gridDim.x) {
        const Item it = decode(rec);
        rec = fetch(w + gridDim.x);
        const int nt = tiles_of(it);
        if (nt == 0) continue;
        const bool kv = w < n_kv;
        for (int j = 0; j < nt && ok; ++j, ++g) {
          const uint32_t s = g % C::kStages;
          const bool more = wa < n_all;
          int nc = it.n_other - j * kTR;
          nc = nc > kTR ? kTR : nc;
          const int ksteps = (nc + 15) >> 4;
          auto product = [&](int acc, int which, bool is_p) {
#pragma unroll
            for (int ks = 0; ks < kTR / 16; ++ks) {
              if (ks < ksteps) {
                const uint32_t ta = tmem + (is_p ? C::p_col(ks / 2) : C::ds_col(ks / 2)) + 8 * (ks % 2);
#pragma unroll
                for (int x = 0; x < C::kHalves; ++x)
                  ptx::umma_f16_ts(tmem + acc + 64 * x, ta,
                                   d_mn + (uint64_t)((s * 2 + which) * (C::kTile >> 4) + x * (kHalf >> 4) + ks * (2048 >> 4)), idesc_acc,
                                   (j | ks) != 0 ? 1u : 0u);
              }
            }
          };
          if (C::kSep && more) {  // S of this tile is in registers: the next may overwrite it
            if (!wait(&ctrl->s_free, g & 1) || !issue_s()) { ok = false; break; }
          }
          if (!wait(&ctrl->aux[s], (g / C::kStages) & 1)) { ok = false; break; }
          if (j == 0 && n > 0 && !wait(&ctrl->acc_free, (n - 1) & 1)) { ok = false; break; }
          if (!wait(&ctrl->p_ready, g & 1)) { ok = false; break; }
          ptx::tc_fence_after_sync();
          if (kv) product(C::kAcc1, 1, true);
          ptx::umma_commit(ptx::smem_u32(&ctrl->p_done));
          if (!C::kSep && more) {  // the next S takes the columns of this P
            if (!wait(&ctrl->p_done, g & 1) || !issue_s()) { ok = false; break; }
          }
          if (C::kSep && more) {
            if (!wait(&ctrl->dp_free, g & 1)) { ok = false; break; }
            issue_dp();
          }
          if (!wait(&ctrl->ds_ready, g & 1)) { ok = false; break; }
          ptx::tc_fence_after_sync();
          product(C::kAcc2, 0, false);
          ptx::umma_commit(ptx::smem_u32(&ctrl->ds_done));
          ptx::umma_commit(ptx::smem_u32(&ctrl->empty[s]));
          if (!C::kSep && more) {
            if (!wait(&ctrl->ds_done, g & 1)) { ok = false; break; }
            issue_dp();
          }
        }
        ++n;
      }
      if (!ok) {
        ctrl->abort = 1;
        atomicOr(&g_attn_bwd_error, 2);
      }
      ptx::umma_commit(ptx::smem_u32(&ctrl->done));  // every MMA has retired before tensor memory is freed
      ptx::mbar_wait(ptx::smem_u32(&ctrl->done), 0);
    } else if (warp >= 10) {
      // ------------------------------------------------------------ helpers: warp 10 lse and A tiles, warp 11 D and B tiles
      const int me = warp - 10;
      bool ok = true;
      uint32_t g = 0;
      int4 rec = fetch(blockIdx.x);
      for (unsigned w = blockIdx.x; w < n_all && ok; w += gridDim.x) {
        const Item it = decode(rec);
        rec = fetch(w + gridDim.x);
        const int nt = tiles_of(it);
        const bool kv = w < n_kv;
        const int h = head(w);
        const float* src = (me == 0 ? a.lse : a.delta) + (int64_t)h * a.q_tokens + it.other;
        const float f = me == 0 ? -1.0f : (kv && nt > 0 ? -grad_scale(a, t.kv.seq, w / H, h) : 0.0f);
        for (int j = 0; j < nt; ++j, ++g) {
          const uint32_t s = g % C::kStages;
          int nc = it.n_other - j * kTR;
          nc = nc > kTR ? kTR : nc;
          float v[4];
          if (kv) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int c = lane + 32 * k;
              v[k] = c < nc ? src[j * kTR + c] * f : 0.0f;
            }
          }
          if (!wait(&ctrl->full[s], (g / C::kStages) & 1)) {
            ok = false;
            break;
          }
          if (kv) {
            float* dst = s_stats + s * (C::kStats / 4) + me * kTR;
#pragma unroll
            for (int k = 0; k < 4; ++k) dst[lane + 32 * k] = v[k];
          }
          const int r_end = (nc + 15) & ~15;
          for (int i = lane; i < (r_end - nc) * 8 * C::kHalves; i += 32) {
            const int r = nc + i / (8 * C::kHalves), x = i % (8 * C::kHalves);
            const uint32_t addr = s_oth + (s * 2 + me) * C::kTile + (x / 8) * kHalf + (r >> 3) * 1024 + (r & 7) * 128 + (x % 8) * 16;
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(addr), "r"(0u) : "memory");
          }
          ptx::fence_proxy_async();  // the tensor core reads the cleared rows
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&ctrl->aux[s]));
        }
      }
      if (!ok && lane == 0) {
        ctrl->abort = 1;
        atomicOr(&g_attn_bwd_error, 1);
      }
    }
  } else {
    // ------------------------------------------------------------ softmax
    ptx::setmaxnreg_inc<kRegSoftmax>();
    const int q = warp & 3, wg = warp >> 2;
    const int row = q * 32 + lane;
    const uint32_t tl = tmem + ((uint32_t)(q * 32) << 16);
    const float scale = a.scaling * kLog2e;
    const uint64_t sc2 = ptx::f32x2_pack(scale, scale);
    bool ok = true;
    uint32_t g = 0;
    auto arrive = [&](uint64_t* bar) {
      ptx::tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(bar));
    };
    int4 rec = fetch(blockIdx.x);
    for (unsigned w = blockIdx.x; w < n_all; w += gridDim.x) {
      const Item it = decode(rec);
      rec = fetch(w + gridDim.x);
      const bool kv = w < n_kv;
      const int h = head(w);
      const int nt = tiles_of(it);
      const bool live = q * 32 < it.rows;  // warp-uniform: this warp owns valid rows
      const float gs = grad_scale(a, kv ? t.kv.seq : t.qi.seq, (kv ? w : w - n_kv) / H, h);
      const uint64_t gs2 = ptx::f32x2_pack(gs, gs);
      uint64_t nl2 = 0, nd2 = 0;  // -lse and -D of this row (Q items)
      if (!kv && nt > 0 && row < it.rows) {
        const int64_t i = (int64_t)h * a.q_tokens + it.row0 + row;
        const float nl = -a.lse[i], nd = -a.delta[i] * gs;
        nl2 = ptx::f32x2_pack(nl, nl);
        nd2 = ptx::f32x2_pack(nd, nd);
      }
      for (int j = 0; j < nt; ++j, ++g) {
        const uint32_t s = g % C::kStages;
        int nc = it.n_other - j * kTR;
        nc = nc > kTR ? kTR : nc;
        const float* stats = s_stats + s * (C::kStats / 4);
        uint32_t sv[2][32];
        float p[2][32];
        // ---- P
        if (ok && !wait(&ctrl->s_ready, g & 1)) ok = false;
        if (ok && kv && !wait(&ctrl->aux[s], (g / C::kStages) & 1)) ok = false;
        if (ok && live) {
          ptx::tc_fence_after_sync();
#pragma unroll
          for (int k = 0; k < 2; ++k)
            if ((wg + 2 * k) * 32 < nc) ptx::tmem_ld_32x32b_x32(tl + (wg + 2 * k) * 32, sv[k]);
          ptx::tmem_ld_wait();
        }
        arrive(&ctrl->s_free);
        if (ok && live) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int c0 = (wg + 2 * k) * 32;
            if (c0 < nc) {
#pragma unroll
              for (int i = 0; i < 32; i += 4) {
                uint64_t n0 = nl2, n1 = nl2;
                if (kv) {
                  const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(stats + c0 + i);
                  n0 = v.x, n1 = v.y;
                }
                const uint64_t x0 = ptx::f32x2_fma(ptx::f32x2_pack(__uint_as_float(sv[k][i]), __uint_as_float(sv[k][i + 1])), sc2, n0);
                const uint64_t x1 = ptx::f32x2_fma(ptx::f32x2_pack(__uint_as_float(sv[k][i + 2]), __uint_as_float(sv[k][i + 3])), sc2, n1);
                float e0, e1, e2, e3;
                ptx::f32x2_unpack(x0, e0, e1);
                ptx::f32x2_unpack(x1, e2, e3);
                p[k][i] = ptx::ex2_approx(e0);
                p[k][i + 1] = ptx::ex2_approx(e1);
                p[k][i + 2] = ptx::ex2_approx(e2);
                p[k][i + 3] = ptx::ex2_approx(e3);
              }
              // columns past the end of the sequence: no probability, whatever was there (a loop of zero or one trips, so that
              // whole chunks do not pay for the selects)
#pragma unroll 1
              for (int ragged = nc - c0 < 32 ? 1 : 0; ragged > 0; --ragged) {
#pragma unroll
                for (int i = 0; i < 32; ++i) p[k][i] = c0 + i >= nc ? 0.0f : p[k][i];
              }
            }
          }
        }
        if (kv) {
          // the product with the previous P must have read these columns
          if (C::kSep && ok && g > 0 && !wait(&ctrl->p_done, (g - 1) & 1)) ok = false;
          if (ok && live) {
            ptx::tc_fence_after_sync();
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              if ((wg + 2 * k) * 32 < nc) {
                uint32_t pk[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) pk[i] = pack2<FMT>(p[k][2 * i], p[k][2 * i + 1]);
                ptx::tmem_st_32x32b_x16(tl + C::p_col(wg + 2 * k), pk);
              }
            }
            ptx::tmem_st_wait();
          }
        }
        arrive(&ctrl->p_ready);
        // ---- dS
        if (ok && !wait(&ctrl->dp_ready, g & 1)) ok = false;
        if (ok && live) {
          ptx::tc_fence_after_sync();
#pragma unroll
          for (int k = 0; k < 2; ++k)
            if ((wg + 2 * k) * 32 < nc) ptx::tmem_ld_32x32b_x32(tl + 128 + (wg + 2 * k) * 32, sv[k]);
          ptx::tmem_ld_wait();
        }
        arrive(&ctrl->dp_free);
        if (C::kSep && ok && g > 0 && !wait(&ctrl->ds_done, (g - 1) & 1)) ok = false;
        if (ok && live) {
          ptx::tc_fence_after_sync();
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int c0 = (wg + 2 * k) * 32;
            if (c0 < nc) {
#pragma unroll
              for (int i = 0; i < 32; i += 4) {
                uint64_t n0 = nd2, n1 = nd2;
                if (kv) {
                  const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(stats + kTR + c0 + i);
                  n0 = v.x, n1 = v.y;
                }
                const uint64_t x0 = ptx::f32x2_fma(ptx::f32x2_pack(__uint_as_float(sv[k][i]), __uint_as_float(sv[k][i + 1])), gs2, n0);
                const uint64_t x1 = ptx::f32x2_fma(ptx::f32x2_pack(__uint_as_float(sv[k][i + 2]), __uint_as_float(sv[k][i + 3])), gs2, n1);
                const uint64_t y0 = ptx::f32x2_mul(ptx::f32x2_pack(p[k][i], p[k][i + 1]), x0);
                const uint64_t y1 = ptx::f32x2_mul(ptx::f32x2_pack(p[k][i + 2], p[k][i + 3]), x1);
                ptx::f32x2_unpack(y0, p[k][i], p[k][i + 1]);
                ptx::f32x2_unpack(y1, p[k][i + 2], p[k][i + 3]);
              }
#pragma unroll 1
              for (int ragged = nc - c0 < 32 ? 1 : 0; ragged > 0; --ragged) {
#pragma unroll
                for (int i = 0; i < 32; ++i) p[k][i] = c0 + i >= nc ? 0.0f : p[k][i];
              }
              uint32_t pk[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) pk[i] = pack2<FMT>(p[k][2 * i], p[k][2 * i + 1]);
              ptx::tmem_st_32x32b_x16(tl + C::ds_col(wg + 2 * k), pk);
            }
          }
          ptx::tmem_st_wait();
        }
        arrive(&ctrl->ds_ready);
      }
      // ---- the item's gradients: KV: warps 0-3 dV, warps 4-7 dK; Q: half of dQ's columns each
      if (nt > 0 && ok && !wait(&ctrl->ds_done, (g - 1) & 1)) ok = false;
      if (ok && live) {
        ptx::tc_fence_after_sync();
        constexpr int kCols = D;
        const int cols = kv ? kCols : kCols / 2;
        const int col0 = kv ? 0 : wg * (kCols / 2);
        const int acc = kv && wg == 0 ? C::kAcc1 : C::kAcc2;
        const float f = kv && wg == 0 ? 1.0f : a.scaling / gs;
        T* out = static_cast<T*>(kv ? (wg == 0 ? a.dv : a.dk) : a.dq) + (it.row0 + row) * (kv ? (wg == 0 ? a.lddv : a.lddk) : a.lddq) +
                 (int64_t)h * D + col0;
        for (int c = 0; c < cols; c += 32) {
          uint32_t r[32];
          if (nt > 0) {
            ptx::tmem_ld_32x32b_x32(tl + acc + col0 + c, r);
            ptx::tmem_ld_wait();
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) r[i] = 0u;  // nothing on the other side: zeros
          }
          if (row < it.rows) {
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              uint4 v;
              v.x = pack2<FMT>(__uint_as_float(r[i]) * f, __uint_as_float(r[i + 1]) * f);
              v.y = pack2<FMT>(__uint_as_float(r[i + 2]) * f, __uint_as_float(r[i + 3]) * f);
              v.z = pack2<FMT>(__uint_as_float(r[i + 4]) * f, __uint_as_float(r[i + 5]) * f);
              v.w = pack2<FMT>(__uint_as_float(r[i + 6]) * f, __uint_as_float(r[i + 7]) * f);
              *reinterpret_cast<uint4*>(out + c + i) = v;
            }
          }
        }
      }
      if (nt > 0) arrive(&ctrl->acc_free);
    }
    if (!ok && lane == 0) {
      ctrl->abort = 1;
      atomicOr(&g_attn_bwd_error, 4);
    }
  }

  ptx::tc_fence_before_sync();
  __syncthreads();
  if (warp == 9) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc(tmem, 512);
  }
}

template <int FMT, int D>
int launch(const BwdArgs& a, int64_t k_tokens, int dtype, const ListOut& kv, const ListOut& qi, int64_t items, cudaStream_t st) {
  using C = Cfg<D>;
  const int64_t E = (int64_t)a.H * D;
  CUtensorMap map_q, map_k, map_v, map_g;
  if (!make_tile_map(&map_q, {a.q, a.q_tokens, E, a.ldq}, dtype) || !make_tile_map(&map_k, {a.k, k_tokens, E, a.ldk}, dtype) ||
      !make_tile_map(&map_v, {a.v, k_tokens, E, a.ldv}, dtype) || !make_tile_map(&map_g, {a.grad, a.q_tokens, E, E}, dtype))
    return NTB200_LAUNCH_FAILED;
  static std::atomic<int> configured[kMaxDevices];
  if (!once_per_device(configured, [] {
        return cudaFuncSetAttribute(attn_bwd_tcgen05_kernel<FMT, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem) == cudaSuccess;
      }))
    return NTB200_LAUNCH_FAILED;
  int dev = 0, sms = kNumSMs;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int64_t grid = items < sms ? items : sms;
  const TcArgs t = {a, kv, qi};
  attn_bwd_tcgen05_kernel<FMT, D><<<(unsigned)grid, kBwdThreads, C::kSmem, st>>>(map_q, map_k, map_v, map_g, t);
  return status_from_cuda(cudaGetLastError());
}

}  // namespace

// (both sides need rows: a tensor map over none cannot be made; the mma.sync kernel writes the zeros of that case)
bool attn_bwd_tcgen05_supported(const BwdArgs& a, int64_t k_tokens, int dtype) {
  return (a.d == 64 || a.d == 128) && (dtype == NTB200_F16 || dtype == NTB200_BF16) && a.q_tokens > 0 && k_tokens > 0 &&
         (a.batch * 2 + (a.q_tokens + k_tokens) / 128 + 4) * (int64_t)a.H < (1ll << 31) && (int64_t)a.H * a.d < (1ll << 31) &&
         a.ldq < (1ll << 38) && a.ldk < (1ll << 38) && a.ldv < (1ll << 38);
}

int attn_bwd_tcgen05_launch(const BwdArgs& a, int64_t k_tokens, int dtype, const ListOut& kv, const ListOut& qi, int64_t kv_capacity,
                            int64_t q_capacity, cudaStream_t st) {
  const int64_t items = (kv_capacity + q_capacity) * a.H;
  if (dtype == NTB200_F16) return a.d == 64 ? launch<0, 64>(a, k_tokens, dtype, kv, qi, items, st) : launch<0, 128>(a, k_tokens, dtype, kv, qi, items, st);
  return a.d == 64 ? launch<1, 64>(a, k_tokens, dtype, kv, qi, items, st) : launch<1, 128>(a, k_tokens, dtype, kv, qi, items, st);
}

int attn_bwd_tcgen05_error_flags_read_and_clear() {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_attn_bwd_error, sizeof(int)) != cudaSuccess) return -1;
  if (v != 0) {
    int zero = 0;
    cudaMemcpyToSymbol(g_attn_bwd_error, &zero, sizeof(int));
  }
  return v;
}

}  // namespace ntb200
