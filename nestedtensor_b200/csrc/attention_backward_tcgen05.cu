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
// Every step between the roles costs a warp some 150-200 cycles whether it waits or not, and eight warps hide little of that, so
// a tile takes a softmax warp only two waits (S, dP) and two arrivals (P, dS): each commit also covers the product before it.
// Measured: two sequences of about 4500 tokens, 8 heads of 128, bf16: 619 us, 0.67 PFLOP/s of the five products.  Tensor pipe 46 %,
// exponentials 20 %, issue slots 35 %: nothing is full; what a tile waits for is the latency of the chain S, P, dP, dS.  The compiler
// works within the 168 registers of the launch: heads of 128 spill 80 bytes a thread (stores; 156 loads), heads of 64 24 (52).
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
  static constexpr int kStats = 2 * kTR * 4 + 16; // -lse and -D of a stage; (fp16) dO's factor
  static constexpr int kStaging = (kOwn + kStages) * 2 * kTile + kStages * kStats + 512;  // 2 KB a softmax warp for the outputs
  static constexpr int kSmem = 1024 + kStaging + 8 * 2048;
  // tensor-memory columns of the packed P and dS of a chunk of 32 columns
  static __device__ __forceinline__ int p_col(int chunk) { return kSep ? 384 + 16 * chunk : 32 * chunk; }
  static __device__ __forceinline__ int ds_col(int chunk) { return kSep ? 448 + 16 * chunk : 128 + 32 * chunk; }
};

template <int D>
struct Ctrl {
  uint64_t own_full[Cfg<D>::kOwn], own_empty[Cfg<D>::kOwn];
  uint64_t full[Cfg<D>::kStages], empty[Cfg<D>::kStages], aux[Cfg<D>::kStages];
  uint64_t s_ready, p_ready, p_done, dp_ready, ds_ready, ds_done, item_done, acc_free, done;
  uint32_t tmem_base;
  volatile int abort;
};

// Four exponentials 2^x.  bf16: two of every eight on the FMA pipe (a polynomial, relative error 1.9e-4 where rounding P to bf16
// costs up to 3.9e-3): the 16 results per clock of the MUFU units are what the P phase waits for.  fp16 rounds to 4.9e-4, so there
// all go through MUFU.
template <int FMT, bool POLY>
__device__ __forceinline__ void ex2_four(uint64_t x0, uint64_t x1, float* p) {
  float e0, e1, e2, e3;
  ptx::f32x2_unpack(x0, e0, e1);
  p[0] = ptx::ex2_approx(e0);
  p[1] = ptx::ex2_approx(e1);
  ptx::f32x2_unpack(x1, e2, e3);
  if (FMT == 1 && POLY) {
    const uint64_t x = ptx::f32x2_pack(ptx::fmax_nan(e2, -126.0f), ptx::fmax_nan(e3, -126.0f));
    ptx::ex2_poly_x2(x, p[2], p[3]);
    // (the polynomial's exponent arithmetic loses a NaN: 0 x brings it back)
    ptx::f32x2_unpack(ptx::f32x2_fma(x, ptx::f32x2_pack(0.0f, 0.0f), ptx::f32x2_pack(p[2], p[3])), p[2], p[3]);
  } else {
    p[2] = ptx::ex2_approx(e2);
    p[3] = ptx::ex2_approx(e3);
  }
}

// Columns past the end of the sequence have no probability, whatever was in their columns (in a loop of zero or one trips, so that
// whole chunks do not pay for the selects).
__device__ __forceinline__ void cut_columns(float (&x)[32], int c0, int nc) {
#pragma unroll 1
  for (int ragged = nc - c0 < 32 ? 1 : 0; ragged > 0; --ragged) {
#pragma unroll
    for (int i = 0; i < 32; ++i) x[i] = c0 + i >= nc ? 0.0f : x[i];
  }
}

// 32 columns of 32 rows (one row per lane, packed 16-bit, 64 bytes) to global memory through the warp's 2 KB of shared memory: stored
// row by row from the lanes themselves, every 16-byte store would touch 32 lines.
__device__ __forceinline__ void store_rows(uint32_t stage, const uint4 (&v)[4], uint8_t* out, int64_t row_bytes, int rows) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4)), "r"(v[i].x), "r"(v[i].y),
                 "r"(v[i].z), "r"(v[i].w)
                 : "memory");
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = i * 8 + lane / 4, c = lane % 4;
    uint4 x;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                 : "r"(stage + r * 64 + ((c ^ ((r >> 1) & 3)) << 4))
                 : "memory");
    if (r < rows) *reinterpret_cast<uint4*>(out + r * row_bytes + c * 16) = x;
  }
  __syncwarp();
}

template <int FMT>
__device__ __forceinline__ void pack_row(const uint32_t (&r)[32], float f, uint4 (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i].x = pack2<FMT>(__uint_as_float(r[8 * i]) * f, __uint_as_float(r[8 * i + 1]) * f);
    v[i].y = pack2<FMT>(__uint_as_float(r[8 * i + 2]) * f, __uint_as_float(r[8 * i + 3]) * f);
    v[i].z = pack2<FMT>(__uint_as_float(r[8 * i + 4]) * f, __uint_as_float(r[8 * i + 5]) * f);
    v[i].w = pack2<FMT>(__uint_as_float(r[8 * i + 6]) * f, __uint_as_float(r[8 * i + 7]) * f);
  }
}

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
    ptx::mbar_init(ptx::smem_u32(&ctrl->s_ready), 3);  // the commit and both helper warps
    ptx::mbar_init(ptx::smem_u32(&ctrl->p_ready), 8);
    ptx::mbar_init(ptx::smem_u32(&ctrl->p_done), 1);
    ptx::mbar_init(ptx::smem_u32(&ctrl->dp_ready), 1);
    ptx::mbar_init(ptx::smem_u32(&ctrl->ds_ready), 8);
    ptx::mbar_init(ptx::smem_u32(&ctrl->ds_done), 1);
    ptx::mbar_init(ptx::smem_u32(&ctrl->item_done), 1);
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
  // for roles of whole warps: the lanes agree, so that none is left alone at a warp-wide instruction when a wait runs out
  auto wait_warp = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait_or_abort(ptx::smem_u32(bar), parity, &ctrl->abort)) != 0; };

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
          // p_ready: P is in place, and S has been read.  The commit behind the next S covers this product too, so that a warp that
          // finds the next S ready may overwrite P; the same holds for dP and dS.
          if (!wait(&ctrl->aux[s], (g / C::kStages) & 1)) { ok = false; break; }
          if (j == 0 && n > 0 && !wait(&ctrl->acc_free, (n - 1) & 1)) { ok = false; break; }
          if (!wait(&ctrl->p_ready, g & 1)) { ok = false; break; }
          ptx::tc_fence_after_sync();
          if (kv) product(C::kAcc1, 1, true);
          if (!C::kSep) {  // the next S takes the columns of this P
            ptx::umma_commit(ptx::smem_u32(&ctrl->p_done));
            if (more && !wait(&ctrl->p_done, g & 1)) { ok = false; break; }
          }
          if (more && !issue_s()) { ok = false; break; }
          if (!wait(&ctrl->ds_ready, g & 1)) { ok = false; break; }
          ptx::tc_fence_after_sync();
          product(C::kAcc2, 0, false);
          ptx::umma_commit(ptx::smem_u32(&ctrl->empty[s]));
          if (j == nt - 1) ptx::umma_commit(ptx::smem_u32(&ctrl->item_done));
          if (!C::kSep) {
            ptx::umma_commit(ptx::smem_u32(&ctrl->ds_done));
            if (more && !wait(&ctrl->ds_done, g & 1)) { ok = false; break; }
          }
          if (more) issue_dp();
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
      // cursor over the tiles, one ahead: its statistics are on the way while the current tile is waited for
      unsigned w = blockIdx.x;
      auto fetch_seq = [&](unsigned w) {
        if (FMT != 0 || me != 1 || w >= n_all) return 0;
        return __ldg(w < n_kv ? t.kv.seq + w / H : t.qi.seq + (w - n_kv) / H);
      };
      int4 rec = fetch(w), rec_next = fetch(w + gridDim.x);
      int seq = fetch_seq(w), seq_next = fetch_seq(w + gridDim.x);
      int j = 0, nt = 0;
      uint2 top = make_uint2(0u, 0u);
      float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      Item it = decode(rec);
      auto step = [&]() {
        w += gridDim.x;
        rec = rec_next, seq = seq_next;
        rec_next = fetch(w + gridDim.x), seq_next = fetch_seq(w + gridDim.x);
      };
      auto open = [&]() {  // the next item that has tiles
        for (; w < n_all; step()) {
          it = decode(rec);
          nt = tiles_of(it);
          if (nt > 0) break;
        }
        j = 0;
        if (FMT == 0 && me == 1 && w < n_all) top = a.top[(int64_t)seq * H + head(w)];
      };
      auto load = [&]() {
        if (w >= n_kv) return;
        const float* src = (me == 0 ? a.lse : a.delta) + (int64_t)head(w) * a.q_tokens + it.other + j * kTR;
        const int nc = it.n_other - j * kTR;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = lane + 32 * k < nc ? src[lane + 32 * k] : 0.0f;
      };
      open();
      if (w < n_all) load();
      while (w < n_all) {
        const uint32_t s = g % C::kStages;
        const bool kv = w < n_kv;
        const uint2 top_c = top;
        const float vc[4] = {v[0], v[1], v[2], v[3]};
        int nc = it.n_other - j * kTR;
        nc = nc > kTR ? kTR : nc;
        if (++j == nt) {
          step();
          open();
        }
        if (w < n_all) load();
        if (!wait_warp(&ctrl->full[s], (g / C::kStages) & 1)) {
          ok = false;
          break;
        }
        float* dst = s_stats + s * (C::kStats / 4);
        const float gs = FMT == 0 && me == 1 ? scale_of(top_c) : 1.0f;
        if (FMT == 0 && me == 1 && lane == 0) dst[2 * kTR] = gs;
        if (kv) {
#pragma unroll
          for (int k = 0; k < 4; ++k) dst[me * kTR + lane + 32 * k] = vc[k] * -gs;
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
        // the statistics count into s_ready of their tile, whose phase begins when the tile before it is ready
        if (g > 0 && !wait_warp(&ctrl->s_ready, (g - 1) & 1)) {
          ok = false;
          break;
        }
        if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&ctrl->s_ready));
        ++g;
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
    // The gradients of an item are written during the first tile of the next one (its last product retires meanwhile).
    struct Pending {
      bool any, live;
      T* out;             // of the warp's first row
      int64_t row_bytes;
      int rows, cols, acc;
      float f;
    } pend = {false, false, nullptr, 0, 0, 0, 0, 0.0f};
    const uint32_t stage = ptx::smem_u32(smem) + (uint32_t)C::kStaging + (uint32_t)warp * 2048u;
    auto write_out = [&](const Pending& o, bool zeros) {  // (whole warps: o.rows of this warp's 32 rows are valid)
      for (int c = 0; c < o.cols; c += 32) {
        uint32_t r[32];
        uint4 v[4];
        if (!zeros) {
          ptx::tmem_ld_32x32b_x32(tl + o.acc + c, r);
          ptx::tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) r[i] = 0u;
        }
        pack_row<FMT>(r, o.f, v);
        store_rows(stage, v, reinterpret_cast<uint8_t*>(o.out + c), o.row_bytes, o.rows);
      }
    };
    uint32_t n = 0;  // items with tiles whose gradients have been written
    auto flush = [&]() {
      if (!pend.any) return;
      if (ok && !wait_warp(&ctrl->item_done, n & 1)) ok = false;
      ++n;
      if (ok && pend.live) {
        ptx::tc_fence_after_sync();
        write_out(pend, false);
      }
      arrive(&ctrl->acc_free);
      pend.any = false;
    };
    // P of this thread's (up to) 64 columns, 2^(scale S - lse); lse per column (KV items, from shared memory) or per row
    auto exponentials = [&](auto is_kv, const uint32_t (&sv)[2][32], float (&p)[2][32], const float* stats, uint64_t nl, int nc) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int c0 = (wg + 2 * k) * 32;
        if (c0 < nc) {
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            ulonglong2 n = make_ulonglong2(nl, nl);
            if constexpr (decltype(is_kv)::value) n = *reinterpret_cast<const ulonglong2*>(stats + c0 + i);
            const uint64_t x0 = ptx::f32x2_fma(ptx::f32x2_pack(__uint_as_float(sv[k][i]), __uint_as_float(sv[k][i + 1])), sc2, n.x);
            const uint64_t x1 = ptx::f32x2_fma(ptx::f32x2_pack(__uint_as_float(sv[k][i + 2]), __uint_as_float(sv[k][i + 3])), sc2, n.y);
            if (i & 4) ex2_four<FMT, true>(x0, x1, p[k] + i);
            else ex2_four<FMT, false>(x0, x1, p[k] + i);
          }
          cut_columns(p[k], c0, nc);
        }
      }
    };
    // dS = P (gs dP - gs D), over P, and to tensor memory
    auto products = [&](auto is_kv, const uint32_t (&sv)[2][32], float (&p)[2][32], const float* stats, uint64_t nd, uint64_t gs2, int nc) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int c0 = (wg + 2 * k) * 32;
        if (c0 < nc) {
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            ulonglong2 n = make_ulonglong2(nd, nd);
            if constexpr (decltype(is_kv)::value) n = *reinterpret_cast<const ulonglong2*>(stats + c0 + i);
            const uint64_t x0 = ptx::f32x2_fma(ptx::f32x2_pack(__uint_as_float(sv[k][i]), __uint_as_float(sv[k][i + 1])), gs2, n.x);
            const uint64_t x1 = ptx::f32x2_fma(ptx::f32x2_pack(__uint_as_float(sv[k][i + 2]), __uint_as_float(sv[k][i + 3])), gs2, n.y);
            ptx::f32x2_unpack(ptx::f32x2_mul(ptx::f32x2_pack(p[k][i], p[k][i + 1]), x0), p[k][i], p[k][i + 1]);
            ptx::f32x2_unpack(ptx::f32x2_mul(ptx::f32x2_pack(p[k][i + 2], p[k][i + 3]), x1), p[k][i + 2], p[k][i + 3]);
          }
          cut_columns(p[k], c0, nc);
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) pk[i] = pack2<FMT>(p[k][2 * i], p[k][2 * i + 1]);
          ptx::tmem_st_32x32b_x16(tl + C::ds_col(wg + 2 * k), pk);
        }
      }
    };
    // what an item needs from memory is fetched one item ahead (its record two)
    struct Ahead {
      int4 rec;
      float lse, delta;  // of this row (Q items)
    };
    auto look = [&](unsigned w, const int4& r) {
      Ahead x = {r, 0.0f, 0.0f};
      if (w >= n_kv && w < n_all && row < r.y && r.w > 0) {
        const int64_t i = (int64_t)head(w) * a.q_tokens + r.x + row;
        x.lse = a.lse[i];
        x.delta = a.delta[i];
      }
      return x;
    };
    int4 rec2 = fetch(blockIdx.x + gridDim.x);
    Ahead next = look(blockIdx.x, fetch(blockIdx.x));
    for (unsigned w = blockIdx.x; w < n_all; w += gridDim.x) {
      const Ahead cur = next;
      next = look(w + gridDim.x, rec2);
      rec2 = fetch(w + 2 * gridDim.x);
      const Item it = decode(cur.rec);
      const bool kv = w < n_kv;
      const int h = head(w);
      const int nt = tiles_of(it);
      const bool live = q * 32 < it.rows;  // warp-uniform: this warp owns valid rows
      float gs = 1.0f;                     // (fp16) dO's factor, beside the statistics of every tile
      const uint64_t nl2 = ptx::f32x2_pack(-cur.lse, -cur.lse);  // (Q items)
      for (int j = 0; j < nt; ++j, ++g) {
        const uint32_t s = g % C::kStages;
        int nc = it.n_other - j * kTR;
        nc = nc > kTR ? kTR : nc;
        const float* stats = s_stats + s * (C::kStats / 4);
        uint32_t sv[2][32];
        float p[2][32];
        // ---- P
        if (ok && !wait_warp(&ctrl->s_ready, g & 1)) ok = false;
        if (ok && live) {
          ptx::tc_fence_after_sync();
#pragma unroll
          for (int k = 0; k < 2; ++k)
            if ((wg + 2 * k) * 32 < nc) ptx::tmem_ld_32x32b_x32(tl + (wg + 2 * k) * 32, sv[k]);
          ptx::tmem_ld_wait();
        }
        if (ok && live) {
          if (kv) exponentials(std::true_type{}, sv, p, stats, 0, nc);
          else exponentials(std::false_type{}, sv, p, nullptr, nl2, nc);
        }
        if (ok && live && kv) {
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
        arrive(&ctrl->p_ready);
        if (j == 0) flush();
        // ---- dS
        if (ok && !wait_warp(&ctrl->dp_ready, g & 1)) ok = false;
        if (ok && live) {
          ptx::tc_fence_after_sync();
#pragma unroll
          for (int k = 0; k < 2; ++k)
            if ((wg + 2 * k) * 32 < nc) ptx::tmem_ld_32x32b_x32(tl + 128 + (wg + 2 * k) * 32, sv[k]);
          ptx::tmem_ld_wait();
          if (FMT == 0) gs = stats[2 * kTR];
          const uint64_t gs2 = ptx::f32x2_pack(gs, gs);
          if (kv) products(std::true_type{}, sv, p, stats + kTR, 0, gs2, nc);
          else products(std::false_type{}, sv, p, nullptr, ptx::f32x2_pack(-cur.delta * gs, -cur.delta * gs), gs2, nc);
          ptx::tmem_st_wait();
        }
        arrive(&ctrl->ds_ready);
      }
      // ---- the item's gradients: KV: warps 0-3 dV, warps 4-7 dK; Q: half of dQ's columns each
      const int col0 = kv ? 0 : wg * (D / 2);
      Pending o;
      o.any = true;
      o.live = live;
      o.rows = it.rows - q * 32;
      o.cols = kv ? D : D / 2;
      o.acc = (kv && wg == 0 ? C::kAcc1 : C::kAcc2) + col0;
      o.f = kv && wg == 0 ? 1.0f : a.scaling / gs;
      const int64_t ld = kv ? (wg == 0 ? a.lddv : a.lddk) : a.lddq;
      o.row_bytes = ld * 2;
      o.out = static_cast<T*>(kv ? (wg == 0 ? a.dv : a.dk) : a.dq) + (it.row0 + q * 32) * ld + (int64_t)h * D + col0;
      if (nt > 0) pend = o;
      else if (ok && live) write_out(o, true);  // nothing on the other side: zeros
    }
    flush();
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

// ------------------------------------------------------------------ whole sequences: five products
// The same roles for heads of 64, with an item per (sequence, head): all key tiles of the sequence in turn, each against all query
// tiles.  S and dP are computed once for dV, dK and dQ: dS goes to shared memory as well-formed operand tiles (row = key, 64
// queries a half), read K-major for dK += dS Q and MN-major for dQ = dS^T K.  Four more warps add the dQ tiles of successive key
// tiles up in fp32 (scratch in global memory, one thread per row and always the same one: the order of the sum is fixed) and
// write them out with the last key tile; a sequence of one key tile needs no scratch.
// Half the exponentials and 5/7 of the products of the kernel above, but a sequence is one CTA's: for batches whose sequences are
// short and many (attention_backward.cu chooses).  34 000 tokens in 128 sequences of 32 to 512, 12 heads, fp16: 356 us, 0.25
// PFLOP/s of the five products; bound, like the kernel above, by the chain S, P, dP, dS, product through each softmax warp (tensor
// pipe 16 %, exponentials 12 %, issue slots 25 %, and 15 % of the time some SMs have no sequence left).  The 128 registers of the launch
// spill 226 bytes a thread in fp16 (stores; 278 loads) and 196 (248) in bf16.
constexpr int kFusedThreads = 512;
constexpr int kFusedRegSoftmax = 168, kFusedRegAdd = 96, kFusedRegControl = 80, kFusedRegLaunch = 128;
static_assert(2 * kFusedRegSoftmax + kFusedRegAdd + kFusedRegControl == 4 * kFusedRegLaunch && kFusedRegLaunch * kFusedThreads <= 65536,
              "setmaxnreg exchange must balance");

struct Fused {
  static constexpr int D = 64, kTile = kHalf, kOwn = 2, kStages = 3;
  static constexpr int kAccV = 256, kAccK = 320, kAccQ = 384, kP = 448;  // tensor-memory columns; S 0, dP 128
  static constexpr int kStats = 2 * kTR * 4 + 16;
  static constexpr int kDs = 2 * kHalf;  // dS: 128 keys x 128 queries
  static constexpr int kStaging = (kOwn + kStages) * 2 * kTile + kDs + kStages * kStats + 512;  // 2 KB a warp for the outputs
  static constexpr int kSmem = 1024 + kStaging + 12 * 2048;
  static_assert(kSmem <= 227 * 1024, "more shared memory than a block has");
};

struct FusedCtrl {
  uint64_t own_full[Fused::kOwn], own_empty[Fused::kOwn], own_aux[Fused::kOwn];
  uint64_t full[Fused::kStages], empty[Fused::kStages], aux[Fused::kStages];
  uint64_t s_ready, p_ready, dp_ready, ds_ready, dq_ready, dq_free, own_done, acc_free, done;
  uint32_t tmem_base;
  volatile int abort;
};

struct FusedArgs {
  BwdArgs a;
  ListOut seqs;     // an item per sequence: (first key, keys, first query, queries)
  float4* scratch;  // [H][16][q_tokens]: dQ in fp32 while its key tiles are added up
};

template <int FMT>
__global__ void __launch_bounds__(kFusedThreads, 1)
attn_bwd_fused_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                      const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_g, const __grid_constant__ FusedArgs t) {
  using C = Fused;
  using T = typename std::conditional<FMT == 0, __half, __nv_bfloat16>::type;
  static_assert(sizeof(FusedCtrl) <= 512, "control block exceeds its shared-memory slot");
  const BwdArgs& a = t.a;
  const unsigned H = (unsigned)a.H;
  const unsigned n_all = (unsigned)*t.seqs.count * H;
  if (blockIdx.x >= n_all) return;
  extern __shared__ uint8_t bwd_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(bwd_smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* smem_ds = smem + (C::kOwn + C::kStages) * 2 * C::kTile;
  float* s_stats = reinterpret_cast<float*>(smem_ds + C::kDs);
  FusedCtrl* ctrl = reinterpret_cast<FusedCtrl*>(reinterpret_cast<uint8_t*>(s_stats) + C::kStages * C::kStats);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kOwn; ++s) {
      ptx::mbar_init(ptx::smem_u32(&ctrl->own_full[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&ctrl->own_empty[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&ctrl->own_aux[s]), 1);
    }
    for (int s = 0; s < C::kStages; ++s) {
      ptx::mbar_init(ptx::smem_u32(&ctrl->full[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&ctrl->empty[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&ctrl->aux[s]), 2);
    }
    ptx::mbar_init(ptx::smem_u32(&ctrl->s_ready), 3);  // the commit and both helper warps
    ptx::mbar_init(ptx::smem_u32(&ctrl->p_ready), 8);
    ptx::mbar_init(ptx::smem_u32(&ctrl->dp_ready), 1);
    ptx::mbar_init(ptx::smem_u32(&ctrl->ds_ready), 8);
    ptx::mbar_init(ptx::smem_u32(&ctrl->dq_ready), 1);
    ptx::mbar_init(ptx::smem_u32(&ctrl->dq_free), 4);
    ptx::mbar_init(ptx::smem_u32(&ctrl->own_done), 1);
    ptx::mbar_init(ptx::smem_u32(&ctrl->acc_free), 8);
    ptx::mbar_init(ptx::smem_u32(&ctrl->done), 1);
    ctrl->abort = 0;
    ptx::fence_barrier_init();
    ptx::prefetch_tensormap(&map_q);
    ptx::prefetch_tensormap(&map_k);
    ptx::prefetch_tensormap(&map_v);
    ptx::prefetch_tensormap(&map_g);
  }
  if (warp == 13) {
    ptx::tmem_alloc(ptx::smem_u32(&ctrl->tmem_base), 512);
    ptx::tmem_relinquish();
    ptx::tc_fence_before_sync();
  }
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem = ctrl->tmem_base;
  const uint32_t s_own = ptx::smem_u32(smem);
  const uint32_t s_oth = s_own + C::kOwn * 2 * C::kTile;
  const uint32_t s_ds = ptx::smem_u32(smem_ds);

  auto fetch = [&](unsigned w) { return w < n_all ? __ldg(t.seqs.items + w / H) : make_int4(0, 0, 0, 0); };
  auto head = [&](unsigned w) { return (int)(w % H); };
  auto tiles = [](int n) { return (n + kTR - 1) / kTR; };
  auto wait = [&](uint64_t* bar, uint32_t parity) { return wait_or_abort(ptx::smem_u32(bar), parity, &ctrl->abort); };
  // for roles of whole warps: the lanes agree, so that none is left alone at a warp-wide instruction when a wait runs out
  auto wait_warp = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait_or_abort(ptx::smem_u32(bar), parity, &ctrl->abort)) != 0; };
  // record: x first key, y keys, z first query, w queries.  Own tiles (keys) are counted by n, tiles (own x queries) by g.

  if (warp >= 12) {
    ptx::setmaxnreg_dec<kFusedRegControl>();
    if (warp == 12 && ptx::elect_one()) {
      // ------------------------------------------------------------ TMA producer
      bool ok = true;
      uint32_t g = 0, n = 0;
      int4 rec = fetch(blockIdx.x);
      for (unsigned w = blockIdx.x; w < n_all && ok; w += gridDim.x) {
        const int4 it = rec;
        rec = fetch(w + gridDim.x);
        const int nk = tiles(it.y), nq = tiles(it.w), col = head(w) * C::D;
        if (nq == 0) continue;
        for (int kt = 0; kt < nk && ok; ++kt, ++n) {
          const uint32_t o = n % C::kOwn;
          if (!wait(&ctrl->own_empty[o], ((n / C::kOwn) & 1) ^ 1)) {
            ok = false;
            break;
          }
          const uint32_t bo = ptx::smem_u32(&ctrl->own_full[o]);
          ptx::mbar_arrive_expect_tx(bo, 2 * C::kTile);
          ptx::tma_load_2d(s_own + o * 2 * C::kTile, &map_k, bo, col, it.x + kt * kTR);
          ptx::tma_load_2d(s_own + o * 2 * C::kTile + C::kTile, &map_v, bo, col, it.x + kt * kTR);
          for (int j = 0; j < nq; ++j, ++g) {
            const uint32_t s = g % C::kStages;
            if (!wait(&ctrl->empty[s], ((g / C::kStages) & 1) ^ 1)) {
              ok = false;
              ++n;  // this own pair was issued: part of the drain below
              break;
            }
            const uint32_t b = ptx::smem_u32(&ctrl->full[s]);
            ptx::mbar_arrive_expect_tx(b, 2 * C::kTile);
            ptx::tma_load_2d(s_oth + s * 2 * C::kTile, &map_q, b, col, it.z + j * kTR);
            ptx::tma_load_2d(s_oth + s * 2 * C::kTile + C::kTile, &map_g, b, col, it.z + j * kTR);
          }
          if (!ok) break;
        }
      }
      if (!ok) {
        ctrl->abort = 1;
        atomicOr(&g_attn_bwd_error, 1);
      }
      for (uint32_t k = n > (uint32_t)C::kOwn ? n - C::kOwn : 0; k < n; ++k)
        ptx::mbar_wait(ptx::smem_u32(&ctrl->own_full[k % C::kOwn]), (k / C::kOwn) & 1);
      for (uint32_t k = g > (uint32_t)C::kStages ? g - C::kStages : 0; k < g; ++k)
        ptx::mbar_wait(ptx::smem_u32(&ctrl->full[k % C::kStages]), (k / C::kStages) & 1);
    } else if (warp == 13 && ptx::elect_one()) {
      // ------------------------------------------------------------ MMA issuer
      constexpr uint32_t idesc_acc = ptx::umma_idesc_f16(FMT, kTR, 64, 0, 1);  // A K-major (or tensor memory), B MN-major
      constexpr uint32_t idesc_dq = ptx::umma_idesc_f16(FMT, kTR, 64, 1, 1);   // A MN-major: dS transposed
      const uint64_t d_own = ptx::umma_desc_kmajor_sw128(s_own), d_oth = ptx::umma_desc_kmajor_sw128(s_oth);
      const uint64_t d_own_mn = ptx::umma_desc_mnmajor_sw128(s_own), d_oth_mn = ptx::umma_desc_mnmajor_sw128(s_oth);
      const uint64_t d_ds = ptx::umma_desc_kmajor_sw128(s_ds), d_ds_mn = ptx::umma_desc_mnmajor_sw128(s_ds, kHalf);
      // cursor of the tile whose S and dP are issued next
      unsigned wa = blockIdx.x;
      uint32_t ga = 0, na = 0;
      int ja = 0, ka = 0, nka = 0, nqa = 0, len_q = 0;
      int4 rec_a = fetch(wa);
      auto settle = [&]() {
        while (wa < n_all) {
          const int4 it = rec_a;
          rec_a = fetch(wa + gridDim.x);
          nka = tiles(it.y), nqa = tiles(it.w), len_q = it.w;
          if (nka > 0 && nqa > 0) return;
          wa += gridDim.x;
        }
      };
      settle();
      auto scores = [&](uint32_t tm, int which, uint64_t* ready) {
        const uint32_t s = ga % C::kStages, o = na % C::kOwn;
        int nc = len_q - ja * kTR;
        nc = nc > kTR ? kTR : nc;
        const uint32_t idesc = ptx::umma_idesc_f16(FMT, kTR, (nc + 15) & ~15);
        const uint64_t da = d_own + (uint64_t)((o * 2 + which) * (C::kTile >> 4)), db = d_oth + (uint64_t)((s * 2 + which) * (C::kTile >> 4));
#pragma unroll
        for (int k = 0; k < C::D / 16; ++k) ptx::umma_f16(tm, da + 2 * k, db + 2 * k, idesc, k != 0 ? 1u : 0u);
        ptx::umma_commit(ptx::smem_u32(ready));
      };
      auto issue_s = [&]() -> bool {
        if (ja == 0 && !wait(&ctrl->own_full[na % C::kOwn], (na / C::kOwn) & 1)) return false;
        if (!wait(&ctrl->full[ga % C::kStages], (ga / C::kStages) & 1)) return false;
        ptx::tc_fence_after_sync();
        scores(tmem, 0, &ctrl->s_ready);
        return true;
      };
      auto issue_dp = [&]() {
        scores(tmem + 128, 1, &ctrl->dp_ready);
        ++ga;
        if (++ja == nqa) {
          ja = 0;
          ++na;
          if (++ka == nka) {
            ka = 0;
            wa += gridDim.x;
            settle();
          }
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
        const int4 it = rec;
        rec = fetch(w + gridDim.x);
        const int nk = tiles(it.y), nq = tiles(it.w);
        if (nq == 0) continue;
        for (int kt = 0; kt < nk && ok; ++kt, ++n) {
          const uint32_t o = n % C::kOwn;
          const int rows = it.y - kt * kTR < kTR ? it.y - kt * kTR : kTR;
          for (int j = 0; j < nq && ok; ++j, ++g) {
            const uint32_t s = g % C::kStages;
            const bool more = wa < n_all;
            int nc = it.w - j * kTR;
            nc = nc > kTR ? kTR : nc;
            const int ksteps = (nc + 15) >> 4;
            if (!wait(&ctrl->aux[s], (g / C::kStages) & 1)) { ok = false; break; }
            if (j == 0 && n > 0 && !wait(&ctrl->acc_free, (n - 1) & 1)) { ok = false; break; }
            if (!wait(&ctrl->p_ready, g & 1)) { ok = false; break; }
            ptx::tc_fence_after_sync();
#pragma unroll
            for (int ks = 0; ks < kTR / 16; ++ks)  // dV += P dO
              if (ks < ksteps)
                ptx::umma_f16_ts(tmem + C::kAccV, tmem + C::kP + 8 * ks, d_oth_mn + (uint64_t)((s * 2 + 1) * (C::kTile >> 4) + ks * (2048 >> 4)),
                                 idesc_acc, (j | ks) != 0 ? 1u : 0u);
            if (more && !issue_s()) { ok = false; break; }
            if (!wait(&ctrl->ds_ready, g & 1)) { ok = false; break; }
            if (j == 0 && !wait(&ctrl->own_aux[o], (n / C::kOwn) & 1)) { ok = false; break; }
            if (g > 0 && !wait(&ctrl->dq_free, (g - 1) & 1)) { ok = false; break; }
            ptx::tc_fence_after_sync();
#pragma unroll
            for (int ks = 0; ks < kTR / 16; ++ks)  // dQ = dS^T K, over the tile's keys
              if (ks * 16 < rows)
                ptx::umma_f16(tmem + C::kAccQ, d_ds_mn + (uint64_t)(ks * (2048 >> 4)), d_own_mn + (uint64_t)(o * 2 * (C::kTile >> 4) + ks * (2048 >> 4)),
                              idesc_dq, ks != 0 ? 1u : 0u);
            ptx::umma_commit(ptx::smem_u32(&ctrl->dq_ready));
#pragma unroll
            for (int ks = 0; ks < kTR / 16; ++ks)  // dK += dS Q
              if (ks < ksteps)
                ptx::umma_f16(tmem + C::kAccK, d_ds + (uint64_t)((ks / 4) * (kHalf >> 4) + 2 * (ks % 4)),
                              d_oth_mn + (uint64_t)(s * 2 * (C::kTile >> 4) + ks * (2048 >> 4)), idesc_acc, (j | ks) != 0 ? 1u : 0u);
            ptx::umma_commit(ptx::smem_u32(&ctrl->empty[s]));
            if (j == nq - 1) {
              ptx::umma_commit(ptx::smem_u32(&ctrl->own_done));
              ptx::umma_commit(ptx::smem_u32(&ctrl->own_empty[o]));
            }
            if (more) issue_dp();
          }
        }
      }
      if (!ok) {
        ctrl->abort = 1;
        atomicOr(&g_attn_bwd_error, 2);
      }
      ptx::umma_commit(ptx::smem_u32(&ctrl->done));
      ptx::mbar_wait(ptx::smem_u32(&ctrl->done), 0);
    } else if (warp >= 14) {
      // ------------------------------------------------------------ helpers: warp 14 lse, A tiles and own keys, warp 15 D and B tiles
      const int me = warp - 14;
      auto clear = [&](uint32_t tile, int from) {  // rows of a landed tile past the sequence's end, up to the next 16
        const int to = (from + 15) & ~15;
        for (int i = lane; i < (to - from) * 8; i += 32) {
          const int r = from + i / 8;
          const uint32_t addr = tile + (r >> 3) * 1024 + (r & 7) * 128 + (i % 8) * 16;
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(addr), "r"(0u) : "memory");
        }
        ptx::fence_proxy_async();
        __syncwarp();
      };
      bool ok = true;
      uint32_t g = 0, n = 0;
      auto fetch_seq = [&](unsigned w) { return FMT == 0 && me == 1 && w < n_all ? __ldg(t.seqs.seq + w / H) : 0; };
      unsigned w = blockIdx.x;
      int4 rec = fetch(w), rec_next = fetch(w + gridDim.x);
      int seq = fetch_seq(w), seq_next = fetch_seq(w + gridDim.x);
      int j = 0, kt = 0, nk = 0, nq = 0;
      uint2 top = make_uint2(0u, 0u);
      float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      auto step = [&]() {
        w += gridDim.x;
        rec = rec_next, seq = seq_next;
        rec_next = fetch(w + gridDim.x), seq_next = fetch_seq(w + gridDim.x);
      };
      auto open = [&]() {
        for (; w < n_all; step()) {
          nk = tiles(rec.y), nq = tiles(rec.w);
          if (nk > 0 && nq > 0) break;
        }
        if (FMT == 0 && me == 1 && w < n_all) top = a.top[(int64_t)seq * H + head(w)];
      };
      auto load = [&]() {
        const float* src = (me == 0 ? a.lse : a.delta) + (int64_t)head(w) * a.q_tokens + rec.z + j * kTR;
        const int nc = rec.w - j * kTR;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = lane + 32 * k < nc ? src[lane + 32 * k] : 0.0f;
      };
      open();
      if (w < n_all) load();
      while (w < n_all) {
        const uint32_t s = g % C::kStages, o = n % C::kOwn;
        const uint2 top_c = top;
        const float vc[4] = {v[0], v[1], v[2], v[3]};
        const bool first = j == 0;
        const uint32_t own_parity = (n / C::kOwn) & 1;
        const int rows = rec.y - kt * kTR < kTR ? rec.y - kt * kTR : kTR;
        int nc = rec.w - j * kTR;
        nc = nc > kTR ? kTR : nc;
        if (++j == nq) {  // on to the next tile, whose statistics are fetched before this one's are waited for
          j = 0;
          ++n;
          if (++kt == nk) {
            kt = 0;
            step();
            open();
          }
        }
        if (w < n_all) load();
        if (me == 0 && first) {
          if (!wait_warp(&ctrl->own_full[o], own_parity)) {
            ok = false;
            break;
          }
          clear(s_own + o * 2 * C::kTile, rows);
          if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&ctrl->own_aux[o]));
        }
        if (!wait_warp(&ctrl->full[s], (g / C::kStages) & 1)) {
          ok = false;
          break;
        }
        float* dst = s_stats + s * (C::kStats / 4);
        const float gs = FMT == 0 && me == 1 ? scale_of(top_c) : 1.0f;
        if (FMT == 0 && me == 1 && lane == 0) dst[2 * kTR] = gs;
#pragma unroll
        for (int k = 0; k < 4; ++k) dst[me * kTR + lane + 32 * k] = vc[k] * -gs;
        clear(s_oth + (s * 2 + me) * C::kTile, nc);
        if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&ctrl->aux[s]));
        // the statistics count into s_ready of their tile, whose phase begins when the tile before it is ready
        if (g > 0 && !wait_warp(&ctrl->s_ready, (g - 1) & 1)) {
          ok = false;
          break;
        }
        if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&ctrl->s_ready));
        ++g;
      }
      if (!ok && lane == 0) {
        ctrl->abort = 1;
        atomicOr(&g_attn_bwd_error, 1);
      }
    }
  } else if (warp >= 8) {
    // ------------------------------------------------------------ dQ: one thread per query row of the tile
    ptx::setmaxnreg_dec<kFusedRegAdd>();
    const int row = (warp - 8) * 32 + lane;
    const uint32_t tl = tmem + ((uint32_t)((warp - 8) * 32) << 16) + C::kAccQ;
    const uint32_t stage = ptx::smem_u32(smem) + (uint32_t)C::kStaging + (uint32_t)warp * 2048u;
    bool ok = true;
    uint32_t g = 0;
    int4 rec = fetch(blockIdx.x);
    for (unsigned w = blockIdx.x; w < n_all; w += gridDim.x) {
      const int4 it = rec;
      rec = fetch(w + gridDim.x);
      const int nk = tiles(it.y), nq = tiles(it.w), h = head(w);
      if (nk == 0) {  // queries without keys: zeros
        for (int r = row; r < it.w; r += kTR) {
          uint4* o = reinterpret_cast<uint4*>(static_cast<T*>(a.dq) + ((int64_t)it.z + r) * a.lddq + (int64_t)h * C::D);
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] = make_uint4(0u, 0u, 0u, 0u);
        }
        continue;
      }
      const float f = a.scaling / grad_scale(a, t.seqs.seq, w / H, h);
      for (int kt = 0; kt < nk; ++kt) {
        for (int j = 0; j < nq; ++j, ++g) {
          // (no scratch was asked for where no sequence was to have more than one key tile: then none is touched)
          const bool live = j * kTR + row < it.w && (nk == 1 || t.scratch != nullptr), first = kt == 0, last = kt == nk - 1;
          const int64_t token = (int64_t)it.z + j * kTR + row;
          float4* sc = t.scratch + (int64_t)h * 16 * a.q_tokens + token;
          T* out = static_cast<T*>(a.dq) + (token - lane) * a.lddq + (int64_t)h * C::D;  // the warp's first row
          float4 old[8];
          if (!first && live) {
#pragma unroll
            for (int i = 0; i < 8; ++i) old[i] = sc[(int64_t)i * a.q_tokens];
          }
          if (ok && !wait_warp(&ctrl->dq_ready, g & 1)) ok = false;
          if (ok) ptx::tc_fence_after_sync();
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            uint32_t r[32];
            if (ok) {
              ptx::tmem_ld_32x32b_x32(tl + 32 * x, r);
              ptx::tmem_ld_wait();
            }
            if (x == 1) {
              ptx::tc_fence_before_sync();
              __syncwarp();
              if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&ctrl->dq_free));
            }
            if (!ok) continue;
            if (!first && live) {
              if (x == 1) {
#pragma unroll
                for (int i = 0; i < 8; ++i) old[i] = sc[(int64_t)(8 + i) * a.q_tokens];
              }
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                r[4 * i] = __float_as_uint(__uint_as_float(r[4 * i]) + old[i].x);
                r[4 * i + 1] = __float_as_uint(__uint_as_float(r[4 * i + 1]) + old[i].y);
                r[4 * i + 2] = __float_as_uint(__uint_as_float(r[4 * i + 2]) + old[i].z);
                r[4 * i + 3] = __float_as_uint(__uint_as_float(r[4 * i + 3]) + old[i].w);
              }
            }
            if (last) {
              uint4 v[4];
              pack_row<FMT>(r, f, v);
              store_rows(stage, v, reinterpret_cast<uint8_t*>(out + 32 * x), a.lddq * 2, it.w - j * kTR - (warp - 8) * 32);
            } else if (live) {
#pragma unroll
              for (int i = 0; i < 8; ++i)
                sc[(int64_t)(8 * x + i) * a.q_tokens] = make_float4(__uint_as_float(r[4 * i]), __uint_as_float(r[4 * i + 1]),
                                                                    __uint_as_float(r[4 * i + 2]), __uint_as_float(r[4 * i + 3]));
            }
          }
        }
      }
    }
    if (!ok && lane == 0) {
      ctrl->abort = 1;
      atomicOr(&g_attn_bwd_error, 4);
    }
  } else {
    // ------------------------------------------------------------ softmax, one thread per key row and half of the columns
    ptx::setmaxnreg_inc<kFusedRegSoftmax>();
    const int q = warp & 3, wg = warp >> 2;
    const int row = q * 32 + lane;
    const uint32_t tl = tmem + ((uint32_t)(q * 32) << 16);
    const float scale = a.scaling * kLog2e;
    const uint64_t sc2 = ptx::f32x2_pack(scale, scale);
    bool ok = true;
    uint32_t g = 0, n = 0;
    auto arrive = [&](uint64_t* bar) {
      ptx::tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(bar));
    };
    struct Pending {
      bool any, live;
      T* out;  // of the warp's first row
      int rows;
      float f;
    } pend = {false, false, nullptr, 0, 0.0f};
    const uint32_t stage = ptx::smem_u32(smem) + (uint32_t)C::kStaging + (uint32_t)warp * 2048u;
    const int64_t row_bytes = (wg == 0 ? a.lddv : a.lddk) * 2;
    auto write_out = [&](const Pending& o, bool zeros) {  // warps 0-3: dV, warps 4-7: dK
#pragma unroll
      for (int c = 0; c < C::D; c += 32) {
        uint32_t r[32];
        uint4 v[4];
        if (!zeros) {
          ptx::tmem_ld_32x32b_x32(tl + (wg == 0 ? C::kAccV : C::kAccK) + c, r);
          ptx::tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) r[i] = 0u;
        }
        pack_row<FMT>(r, o.f, v);
        store_rows(stage, v, reinterpret_cast<uint8_t*>(o.out + c), row_bytes, o.rows);
      }
    };
    auto flush = [&]() {
      if (!pend.any) return;
      if (ok && !wait_warp(&ctrl->own_done, n & 1)) ok = false;
      ++n;
      if (ok && pend.live) {
        ptx::tc_fence_after_sync();
        write_out(pend, false);
      }
      arrive(&ctrl->acc_free);
      pend.any = false;
    };
    int4 rec = fetch(blockIdx.x);
    for (unsigned w = blockIdx.x; w < n_all; w += gridDim.x) {
      const int4 it = rec;
      float gs = 1.0f;  // (fp16) dO's factor, beside the statistics of every tile
      rec = fetch(w + gridDim.x);
      const int nk = tiles(it.y), nq = tiles(it.w), h = head(w);
      for (int kt = 0; kt < nk; ++kt) {
        const int rows = it.y - kt * kTR < kTR ? it.y - kt * kTR : kTR;
        const bool live = q * 32 < rows, whole = q * 32 + 32 <= rows;  // warp-uniform
        for (int j = 0; j < nq; ++j, ++g) {
          const uint32_t s = g % C::kStages;
          int nc = it.w - j * kTR;
          nc = nc > kTR ? kTR : nc;
          const float* stats = s_stats + s * (C::kStats / 4);
          float p[2][32];
          // ---- P
          if (ok && !wait_warp(&ctrl->s_ready, g & 1)) ok = false;
          if (ok && live) {
            ptx::tc_fence_after_sync();
#pragma unroll
            for (int k = 0; k < 2; ++k) {  // (a chunk at a time: both with P do not fit the registers)
              const int c0 = (wg + 2 * k) * 32;
              if (c0 < nc) {
                uint32_t sv[32], pk[16];
                ptx::tmem_ld_32x32b_x32(tl + c0, sv);
                ptx::tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                  const ulonglong2 nl = *reinterpret_cast<const ulonglong2*>(stats + c0 + i);
                  const uint64_t x0 = ptx::f32x2_fma(ptx::f32x2_pack(__uint_as_float(sv[i]), __uint_as_float(sv[i + 1])), sc2, nl.x);
                  const uint64_t x1 = ptx::f32x2_fma(ptx::f32x2_pack(__uint_as_float(sv[i + 2]), __uint_as_float(sv[i + 3])), sc2, nl.y);
                  if (i & 4) ex2_four<FMT, true>(x0, x1, p[k] + i);
                  else ex2_four<FMT, false>(x0, x1, p[k] + i);
                }
                cut_columns(p[k], c0, nc);
#pragma unroll
                for (int i = 0; i < 16; ++i) pk[i] = pack2<FMT>(p[k][2 * i], p[k][2 * i + 1]);
                ptx::tmem_st_32x32b_x16(tl + C::kP + 16 * (wg + 2 * k), pk);
              }
            }
            ptx::tmem_st_wait();
          }
          arrive(&ctrl->p_ready);
          if (j == 0) flush();
          // ---- dS
          if (ok && !wait_warp(&ctrl->dp_ready, g & 1)) ok = false;
          if (ok && live) {
            ptx::tc_fence_after_sync();
            if (FMT == 0) gs = stats[2 * kTR];
            const uint64_t gs2 = ptx::f32x2_pack(gs, gs);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int chunk = wg + 2 * k, c0 = chunk * 32;
              if (c0 < nc) {
                uint32_t sv[32];
                ptx::tmem_ld_32x32b_x32(tl + 128 + c0, sv);
                ptx::tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                  const ulonglong2 nd = *reinterpret_cast<const ulonglong2*>(stats + kTR + c0 + i);
                  const uint64_t x0 = ptx::f32x2_fma(ptx::f32x2_pack(__uint_as_float(sv[i]), __uint_as_float(sv[i + 1])), gs2, nd.x);
                  const uint64_t x1 = ptx::f32x2_fma(ptx::f32x2_pack(__uint_as_float(sv[i + 2]), __uint_as_float(sv[i + 3])), gs2, nd.y);
                  ptx::f32x2_unpack(ptx::f32x2_mul(ptx::f32x2_pack(p[k][i], p[k][i + 1]), x0), p[k][i], p[k][i + 1]);
                  ptx::f32x2_unpack(ptx::f32x2_mul(ptx::f32x2_pack(p[k][i + 2], p[k][i + 3]), x1), p[k][i + 2], p[k][i + 3]);
                }
                cut_columns(p[k], c0, nc);
                uint32_t pk[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) pk[i] = pack2<FMT>(p[k][2 * i], p[k][2 * i + 1]);
                // keys past the end are summed over by dQ: zeros (again in a loop of zero or one trips)
#pragma unroll 1
                for (int ragged = whole ? 0 : 1; ragged > 0; --ragged) {
#pragma unroll
                  for (int i = 0; i < 16; ++i) pk[i] = row < rows ? pk[i] : 0u;
                }
                // row = key, 64 queries a half, 128-byte swizzle: eight rows' 16-byte pieces fall into different banks
                const uint32_t base = s_ds + (chunk >> 1) * kHalf + (row >> 3) * 1024 + (row & 7) * 128;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const uint32_t addr = base + ((((chunk & 1) * 4 + i) ^ (row & 7)) << 4);
                  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(pk[4 * i]), "r"(pk[4 * i + 1]), "r"(pk[4 * i + 2]),
                               "r"(pk[4 * i + 3])
                               : "memory");
                }
              }
            }
            ptx::fence_proxy_async();  // the tensor core reads dS
          }
          arrive(&ctrl->ds_ready);
        }
        Pending o;
        o.any = true;
        o.live = live;
        o.rows = rows - q * 32;
        o.f = wg == 0 ? 1.0f : a.scaling / gs;
        o.out = static_cast<T*>(wg == 0 ? a.dv : a.dk) + ((int64_t)it.x + kt * kTR + q * 32) * (wg == 0 ? a.lddv : a.lddk) + (int64_t)h * C::D;
        if (nq > 0) pend = o;
        else if (ok && live) write_out(o, true);  // keys without queries: zeros
      }
    }
    flush();
    if (!ok && lane == 0) {
      ctrl->abort = 1;
      atomicOr(&g_attn_bwd_error, 4);
    }
  }

  ptx::tc_fence_before_sync();
  __syncthreads();
  if (warp == 13) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc(tmem, 512);
  }
}

template <int FMT>
int launch_fused(const BwdArgs& a, int64_t k_tokens, int dtype, const ListOut& seqs, float* scratch, cudaStream_t st) {
  using C = Fused;
  const int64_t E = (int64_t)a.H * C::D;
  CUtensorMap map_q, map_k, map_v, map_g;
  if (!make_tile_map(&map_q, {a.q, a.q_tokens, E, a.ldq}, dtype) || !make_tile_map(&map_k, {a.k, k_tokens, E, a.ldk}, dtype) ||
      !make_tile_map(&map_v, {a.v, k_tokens, E, a.ldv}, dtype) || !make_tile_map(&map_g, {a.grad, a.q_tokens, E, E}, dtype))
    return NTB200_LAUNCH_FAILED;
  static std::atomic<int> configured[kMaxDevices];
  if (!once_per_device(configured, [] {
        return cudaFuncSetAttribute(attn_bwd_fused_kernel<FMT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem) == cudaSuccess;
      }))
    return NTB200_LAUNCH_FAILED;
  int dev = 0, sms = kNumSMs;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int64_t grid = a.batch * a.H < sms ? a.batch * a.H : sms;
  const FusedArgs t = {a, seqs, reinterpret_cast<float4*>(scratch)};
  attn_bwd_fused_kernel<FMT><<<(unsigned)grid, kFusedThreads, C::kSmem, st>>>(map_q, map_k, map_v, map_g, t);
  return status_from_cuda(cudaGetLastError());
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

int attn_bwd_fused_launch(const BwdArgs& a, int64_t k_tokens, int dtype, const ListOut& seqs, float* scratch, cudaStream_t st) {
  return dtype == NTB200_F16 ? launch_fused<0>(a, k_tokens, dtype, seqs, scratch, st) : launch_fused<1>(a, k_tokens, dtype, seqs, scratch, st);
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
