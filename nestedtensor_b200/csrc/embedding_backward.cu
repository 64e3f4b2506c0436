// Gradient of a scaled embedding lookup, out[t] = scale * weight[index[t]], as the dense table
//
//     dW[v] = scale * sum over { t : index[t] = v } of g[t]        (zeros for tokens that do not occur, and for padding_idx)
//
// 1. The tokens are sorted by index, stable: the positions of one index follow one another in their own order.
// 2. A warp takes 32 consecutive sorted positions, gathers their gradient rows and adds the runs of equal indices in fp32
//    registers.  A run that lies inside the warp's 32 is written to dW once; the two that may cross its ends leave fp32
//    partial rows.  Warps beside them write the rows of the absent tokens.
// 3. Runs over more than one warp are added up from their partials in a fixed order.
// Every gradient row is read once and every row of dW written once (HBM-bound: T E + V E elements); the sums' order depends on
// the indices alone (no floating-point atomics), so the same inputs give the same bits.
//
// Measured at 150 000 tokens of a table of 50 000 x 1024 bf16, frequencies falling as 1 / rank: sort 34 us (two passes of 8 bits, each
// a count and a scatter that wait on one another, far from any rate), sums 74 us (0.41 GB: 5.5 TB/s), runs over several
// warps 24 us (most tokens belong to a few hundred indices, whose partial rows are read again).  Up to a few thousand tokens the
// launches one after another are the time: 310 tokens of 256 fp32 columns take 24 us in three kernels.

#include "row_vec.cuh"

namespace ntb200 {
namespace {

constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMaxDigit = 9;           // bits of a digit: 32 warps x 512 counters = 64 KB of shared memory
constexpr int64_t kSingleBlock = 4096; // up to this many tokens one block sorts alone, in one launch
constexpr int kChunk = 32;             // sorted positions per warp

// index -> sort key: what has no gradient row (padding, out of range) sorts behind the table
template <typename IDX>
__device__ __forceinline__ uint32_t key_of(IDX i, int64_t vocab, int64_t padding) {
  return (i < 0 || (int64_t)i >= vocab || (int64_t)i == padding) ? (uint32_t)vocab : (uint32_t)i;
}

// Where a pass finds its input: the index tensor (first pass) or the previous pass's (key, position) arrays.
template <typename IDX>
struct PassIn {
  const IDX* index;
  const uint32_t *keys, *pos;
  int64_t vocab, padding;
  bool first;
  __device__ __forceinline__ uint32_t key(int64_t t) const { return first ? key_of(index[t], vocab, padding) : keys[t]; }
  __device__ __forceinline__ uint32_t position(int64_t t) const { return first ? (uint32_t)t : pos[t]; }
};

__device__ __forceinline__ uint32_t digit_of(uint32_t key, int shift, int bits) { return (key >> shift) & ((1u << bits) - 1u); }

constexpr int kGroupTiles = 8;  // tiles whose counts one block makes, and their sum

// counts of every digit: hist[tile][digit], and group[block][digit] over the block's kGroupTiles tiles
template <typename IDX>
__global__ void __launch_bounds__(kSortThreads)
radix_count_kernel(PassIn<IDX> in, int64_t tokens, int tile, int tiles, int shift, int bits, uint32_t* __restrict__ hist,
                   uint32_t* __restrict__ group) {
  __shared__ uint32_t cnt[kGroupTiles << kMaxDigit];
  const int bins = 1 << bits;
  for (int i = threadIdx.x; i < kGroupTiles * bins; i += kSortThreads) cnt[i] = 0;
  __syncthreads();
  const int64_t t0 = (int64_t)blockIdx.x * kGroupTiles * tile;
  const int64_t t1 = t0 + (int64_t)kGroupTiles * tile < tokens ? t0 + (int64_t)kGroupTiles * tile : tokens;
  for (int64_t t = t0 + threadIdx.x; t < t1; t += kSortThreads)
    atomicAdd(&cnt[(int)(t - t0) / tile * bins + digit_of(in.key(t), shift, bits)], 1u);
  __syncthreads();
  for (int i = threadIdx.x; i < kGroupTiles * bins; i += kSortThreads) {
    const int64_t tl = (int64_t)blockIdx.x * kGroupTiles + i / bins;
    if (tl < tiles) hist[tl * bins + i % bins] = cnt[i];
  }
  if ((int)threadIdx.x < bins) {
    uint32_t sum = 0;
    for (int k = 0; k < kGroupTiles; ++k) sum += cnt[k * bins + threadIdx.x];
    group[(int64_t)blockIdx.x * bins + threadIdx.x] = sum;
  }
}

// One stable pass over the tile [t0, t1), number `blk`: every warp owns a contiguous part of it.  hist == NULL: the tile is the
// whole input.  smem: [kSortWarps][bins] counters.
template <typename IDX>
__device__ __forceinline__ void radix_scatter_tile(const PassIn<IDX>& in, int64_t t0, int64_t t1, int shift, int bits,
                                                   const uint32_t* __restrict__ hist, const uint32_t* __restrict__ group, int blk,
                                                   int groups, uint32_t* wcnt,
                                                   uint32_t* __restrict__ keys_out, uint32_t* __restrict__ pos_out) {
  __shared__ uint32_t s_below[1 << kMaxDigit], s_total[1 << kMaxDigit], s_warp[kSortWarps];
  const int bins = 1 << bits, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kSortWarps * bins; i += kSortThreads) wcnt[i] = 0;
  if ((int)threadIdx.x < bins) s_below[threadIdx.x] = s_total[threadIdx.x] = 0;
  __syncthreads();
  const int64_t per = ((t1 - t0 + kSortThreads - 1) / kSortThreads) * 32;  // whole groups of 32 per warp
  const int64_t w0 = t0 + warp * per, w1 = w0 + per < t1 ? w0 + per : t1;
  for (int64_t t = w0 + lane; t < w1; t += 32) atomicAdd(&wcnt[warp * bins + digit_of(in.key(t), shift, bits)], 1u);
  __syncthreads();
  if (hist != nullptr) {
    // every digit's count over the tiles before this one (whole groups, then this group's), and over all
    const int bin = threadIdx.x % bins, part = threadIdx.x / bins, parts = kSortThreads / bins;
    const int mine = blk / kGroupTiles;
    uint32_t below = 0, total = 0;
#pragma unroll 8
    for (int k = part; k < groups; k += parts) {
      const uint32_t c = group[(int64_t)k * bins + bin];
      total += c;
      below += k < mine ? c : 0u;
    }
    for (int k = mine * kGroupTiles + part; k < blk; k += parts) below += hist[(int64_t)k * bins + bin];
    atomicAdd(&s_below[bin], below);
    atomicAdd(&s_total[bin], total);
  } else if ((int)threadIdx.x < bins) {
    uint32_t total = 0;
    for (int w = 0; w < kSortWarps; ++w) total += wcnt[w * bins + threadIdx.x];
    s_total[threadIdx.x] = total;
  }
  __syncthreads();
  // exclusive scan of the totals over the digits (bins <= 512 < threads)
  uint32_t v = (int)threadIdx.x < bins ? s_total[threadIdx.x] : 0u, incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) s_warp[warp] = incl;
  __syncthreads();
  if ((int)threadIdx.x < bins) {
    uint32_t run = incl - v + s_below[threadIdx.x];
    for (int w = 0; w < warp; ++w) run += s_warp[w];
    for (int w = 0; w < kSortWarps; ++w) {
      const uint32_t c = wcnt[w * bins + threadIdx.x];
      wcnt[w * bins + threadIdx.x] = run;
      run += c;
    }
  }
  __syncthreads();
  for (int64_t g = w0; g < w1; g += 32) {  // (uniform over the warp)
    const int64_t t = g + lane;
    const bool live = t < w1;
    const uint32_t key = live ? in.key(t) : 0u, pos = live ? in.position(t) : 0u;
    const uint32_t d = live ? digit_of(key, shift, bits) : 0xffffffffu;
    const unsigned same = __match_any_sync(0xffffffffu, d);
    const uint32_t rank = __popc(same & ((1u << lane) - 1u));
    uint32_t at = 0;
    if (live) at = wcnt[warp * bins + d] + rank;
    __syncwarp();
    if (live && rank == 0) wcnt[warp * bins + d] += __popc(same);
    __syncwarp();
    if (live) {
      keys_out[at] = key;
      pos_out[at] = pos;
    }
  }
}

template <typename IDX>
__global__ void __launch_bounds__(kSortThreads)
radix_scatter_kernel(PassIn<IDX> in, int64_t tokens, int tile, int shift, int bits, const uint32_t* __restrict__ hist,
                     const uint32_t* __restrict__ group, int groups, uint32_t* __restrict__ keys_out, uint32_t* __restrict__ pos_out,
                     int* __restrict__ n_long) {
  extern __shared__ uint32_t sort_smem[];
  if (blockIdx.x == 0 && threadIdx.x < 2) n_long[threadIdx.x] = 0;
  const int64_t t0 = (int64_t)blockIdx.x * tile, t1 = t0 + tile < tokens ? t0 + tile : tokens;
  radix_scatter_tile(in, t0, t1, shift, bits, hist, group, (int)blockIdx.x, groups, sort_smem, keys_out, pos_out);
}

// All passes in one block; the result is in keys[passes & 1 ? 0 : 1] ... (see launch).
template <typename IDX>
__global__ void __launch_bounds__(kSortThreads)
radix_single_kernel(PassIn<IDX> in, int64_t tokens, int passes, int bits, uint32_t* __restrict__ ka, uint32_t* __restrict__ pa,
                    uint32_t* __restrict__ kb, uint32_t* __restrict__ pb, int* __restrict__ n_long) {
  extern __shared__ uint32_t sort_smem[];
  if (threadIdx.x < 2) n_long[threadIdx.x] = 0;
  for (int p = 0; p < passes; ++p) {
    radix_scatter_tile<IDX>(in, 0, tokens, p * bits, bits, nullptr, nullptr, 0, 0, sort_smem, ka, pa);
    __syncthreads();  // the pass's output is read by the whole block, its counters cleared
    in.first = false;
    in.keys = ka, in.pos = pa;
    uint32_t *tk = ka, *tp = pa;
    ka = kb, pa = pb;
    kb = tk, pb = tp;
  }
}

// ------------------------------------------------------------------ sums of the sorted rows
template <int DT, int EPV>
struct RowUnit {
  using Raw = uint4;
  static __device__ __forceinline__ Raw load(const void* p, int64_t i) { return reinterpret_cast<const uint4*>(p)[i]; }
  static __device__ __forceinline__ void add(float* a, const Raw& r) {
    float f[EPV];
    Vec16<DT>::unpack(r, f);
#pragma unroll
    for (int k = 0; k < EPV; ++k) a[k] += f[k];
  }
  static __device__ __forceinline__ void store(void* p, int64_t i, const float* f) { reinterpret_cast<uint4*>(p)[i] = Vec16<DT>::pack(f); }
};
template <int DT>
struct RowUnit<DT, 1> {
  using Raw = float;
  static __device__ __forceinline__ Raw load(const void* p, int64_t i) { return Vec16<DT>::load1(p, i); }
  static __device__ __forceinline__ void add(float* a, const Raw& r) { a[0] += r; }
  static __device__ __forceinline__ void store(void* p, int64_t i, const float* f) { Vec16<DT>::store1(p, i, f[0]); }
};

struct SumArgs {
  const void* grad;
  const uint32_t *keys, *pos;  // sorted
  void* dw;
  float* partial;  // [chunks][2][cols]: sums of the chunk's first run (begun before it) and of its last run (not ended in it)
  // chunks whose last run begins there and goes on: n_long[0] of them at the front of long_list; those whose run covers the next
  // kFar chunks, n_long[1] of them, at its back
  int *n_long, *long_list;
  int64_t chunks;
  int64_t tokens, vocab, cols;
  float scale;
};

constexpr int kSumWarps = 8;
constexpr int kAhead = 4;  // rows loaded before they are added
constexpr int kFar = 31;   // chunks after the first that one warp of embedding_long_runs_kernel adds up

template <int DT, int EPV, int VPL>
__global__ void __launch_bounds__(kSumWarps * 32, 2)
embedding_sum_kernel(SumArgs a, int slabs, int64_t sum_warps) {
  using U = RowUnit<DT, EPV>;
  const int lane = threadIdx.x & 31;
  int64_t w = (int64_t)blockIdx.x * kSumWarps + (threadIdx.x >> 5);
  const int nv = (int)(a.cols / EPV);
  if (w >= sum_warps) {
    // 32 rows of the table: those whose token does not occur are zeros
    w -= sum_warps;
    const int64_t v = w * 32 + lane;
    bool absent = v < a.vocab;
    if (absent) {
      int64_t lo = 0, hi = a.tokens;  // first position with a key >= v
      while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (a.keys[mid] < (uint32_t)v) lo = mid + 1;
        else hi = mid;
      }
      absent = lo == a.tokens || a.keys[lo] != (uint32_t)v;
    }
    float zeros[EPV];
#pragma unroll
    for (int k = 0; k < EPV; ++k) zeros[k] = 0.0f;
    unsigned todo = __ballot_sync(0xffffffffu, absent);
    while (todo != 0) {
      const int64_t row = w * 32 + (__ffs(todo) - 1);
      todo &= todo - 1;
      for (int u = lane; u < nv; u += 32) U::store(a.dw, row * nv + u, zeros);
    }
    return;
  }
  const int64_t chunk = w / slabs;
  const int u0 = (int)(w % slabs) * (32 * VPL) + lane;
  const int64_t t0 = chunk * kChunk;
  const uint32_t vocab = (uint32_t)a.vocab;
  uint32_t key = vocab, pos = 0;
  if (t0 + lane < a.tokens) {
    key = a.keys[t0 + lane];
    pos = a.pos[t0 + lane];
  }
  const uint32_t before = t0 > 0 ? a.keys[t0 - 1] : vocab;  // (vocab: no run)
  const uint32_t after = t0 + kChunk < a.tokens ? a.keys[t0 + kChunk] : vocab;
  const int n = __popc(__ballot_sync(0xffffffffu, key != vocab));  // sorted: the rows that count come first
  if (n == 0) return;
  float acc[VPL * EPV];
#pragma unroll
  for (int k = 0; k < VPL * EPV; ++k) acc[k] = 0.0f;
  bool begun_here = __shfl_sync(0xffffffffu, key, 0) != before;
  uint32_t run = __shfl_sync(0xffffffffu, key, 0);
  auto flush = [&](bool goes_on) {
    if (begun_here && !goes_on) {
#pragma unroll
      for (int j = 0; j < VPL; ++j) {
        if (u0 + 32 * j < nv) {
#pragma unroll
          for (int k = 0; k < EPV; ++k) acc[j * EPV + k] *= a.scale;
          U::store(a.dw, (int64_t)run * nv + u0 + 32 * j, acc + j * EPV);
        }
      }
    } else {
      float* p = a.partial + (chunk * 2 + (begun_here ? 1 : 0)) * a.cols;
#pragma unroll
      for (int j = 0; j < VPL; ++j) {
        if (u0 + 32 * j < nv) {
#pragma unroll
          for (int k = 0; k < EPV; ++k) p[(int64_t)(u0 + 32 * j) * EPV + k] = acc[j * EPV + k];
        }
      }
      if (begun_here && w % slabs == 0 && lane == 0) {
        const int64_t far = t0 + (int64_t)(kFar + 1) * kChunk;
        if (far < a.tokens && a.keys[far] == run) a.long_list[a.chunks - 1 - atomicAdd(a.n_long + 1, 1)] = (int)chunk;
        else a.long_list[atomicAdd(a.n_long, 1)] = (int)chunk;
      }
    }
  };
  // (loads are clamped to the last row and unit instead of predicated: all of a step's are in flight together; what a lane past
  // the row's end adds up is never stored)
  int unit[VPL];
#pragma unroll
  for (int j = 0; j < VPL; ++j) unit[j] = u0 + 32 * j < nv ? u0 + 32 * j : nv - 1;
  for (int e0 = 0; e0 < n; e0 += kAhead) {
    typename U::Raw rows[kAhead][VPL];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int64_t base = (int64_t)__shfl_sync(0xffffffffu, pos, e0 + i < n ? e0 + i : n - 1) * nv;
#pragma unroll
      for (int j = 0; j < VPL; ++j) rows[i][j] = U::load(a.grad, base + unit[j]);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (e0 + i < n) {
        const uint32_t k = __shfl_sync(0xffffffffu, key, e0 + i);
        if (k != run) {
          flush(false);
          run = k;
          begun_here = true;
#pragma unroll
          for (int c = 0; c < VPL * EPV; ++c) acc[c] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < VPL; ++j) U::add(acc + j * EPV, rows[i][j]);
      }
    }
  }
  flush(n == kChunk && after == run);
}

// The runs over several chunks: the partial of the chunk where the run begins, then those of the chunks whose first key is the
// run's, in order.  Columns in blocks of 128.  Runs of at most kFar + 1 chunks: one warp each; longer ones first, a block each: its
// warps in turn, and their sums in order.
template <int DT>
__global__ void __launch_bounds__(256) embedding_long_runs_kernel(SumArgs a, int col_blocks) {
  __shared__ float s[8][128];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t n_far = (int64_t)a.n_long[1] * col_blocks, n_near = (int64_t)a.n_long[0] * col_blocks;
  for (int64_t i = blockIdx.x; i < n_far; i += gridDim.x) {
    const int64_t c = a.long_list[a.chunks - 1 - i / col_blocks];
    const int64_t col0 = (i % col_blocks) * 128;
    const uint32_t run = a.keys[c * kChunk + kChunk - 1];
    // last chunk whose first key is the run's (first keys are sorted; chunk c + 1's is): 32 probes per step
    int64_t lo = c + 1, hi = a.chunks - 1;
    while (hi > lo) {
      const int64_t step = (hi - lo + 31) / 32;
      int64_t probe = lo + step * (lane + 1);
      probe = probe > hi ? hi : probe;
      const unsigned le = __ballot_sync(0xffffffffu, a.keys[probe * kChunk] <= run);
      if (le == 0) {
        hi = lo + step - 1;
      } else {
        const int top = 31 - __clz(le);
        int64_t nlo = lo + step * (top + 1);
        nlo = nlo > hi ? hi : nlo;
        const int64_t nhi = nlo + step - 1;
        lo = nlo;
        hi = nhi > hi ? hi : nhi;
      }
    }
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int64_t k = c + warp; k <= lo; k += 8) {
      const float* p = a.partial + (k * 2 + (k == c ? 1 : 0)) * a.cols + col0;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (col0 + lane + 32 * j < a.cols) acc[j] += p[lane + 32 * j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) s[warp][lane + 32 * j] = acc[j];
    __syncthreads();
    if (threadIdx.x < 128 && col0 + threadIdx.x < a.cols) {
      float t = s[0][threadIdx.x];
#pragma unroll
      for (int wv = 1; wv < 8; ++wv) t += s[wv][threadIdx.x];
      Vec16<DT>::store1(a.dw, (int64_t)run * a.cols + col0 + threadIdx.x, t * a.scale);
    }
  }
  for (int64_t i = (int64_t)blockIdx.x * 8 + warp; i < n_near; i += (int64_t)gridDim.x * 8) {
    const int64_t c = a.long_list[i / col_blocks];
    const int64_t col0 = (i % col_blocks) * 128;
    const uint32_t run = a.keys[c * kChunk + kChunk - 1];
    // lane k: does chunk c + 1 + k begin with the run?  (sorted: the ones that do come first; at most kFar)
    const unsigned on = __ballot_sync(0xffffffffu, c + 1 + lane < a.chunks && a.keys[(c + 1 + lane) * kChunk] == run);
    const int m = __popc(on);
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int k = 0; k <= m; ++k) {
      const float* p = a.partial + ((c + k) * 2 + (k == 0 ? 1 : 0)) * a.cols + col0;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (col0 + lane + 32 * j < a.cols) acc[j] += p[lane + 32 * j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (col0 + lane + 32 * j < a.cols) Vec16<DT>::store1(a.dw, (int64_t)run * a.cols + col0 + lane + 32 * j, acc[j] * a.scale);
  }
}

struct EmbWorkspace {
  size_t k0, p0, k1, p1, hist, group, n_long, list, partial, bytes;
  int64_t chunks, blocks, groups;
  int tile;
  EmbWorkspace(int64_t tokens, int64_t cols) {
    auto up = [](size_t v) { return (v + 15) / 16 * 16; };
    chunks = (tokens + kChunk - 1) / kChunk;
    // tiles of whole kSortThreads so that at most 2 * 148 blocks share the table of counts
    const int64_t per = (tokens + 2 * kNumSMs - 1) / (2 * kNumSMs);
    tile = (int)((per + kSortThreads - 1) / kSortThreads * kSortThreads);
    if (tile < kSortThreads) tile = kSortThreads;
    blocks = (tokens + tile - 1) / tile;
    const size_t arr = up((size_t)tokens * 4);
    k0 = 0, p0 = k0 + arr, k1 = p0 + arr, p1 = k1 + arr;
    hist = p1 + arr;
    groups = (blocks + kGroupTiles - 1) / kGroupTiles;
    group = hist + (tokens > kSingleBlock ? up((size_t)blocks * (1 << kMaxDigit) * 4) : 0);
    n_long = group + (tokens > kSingleBlock ? up((size_t)groups * (1 << kMaxDigit) * 4) : 0);
    list = n_long + 16;
    partial = list + up((size_t)chunks * 4);
    bytes = partial + (size_t)chunks * 2 * (size_t)cols * 4;
  }
};

template <typename IDX>
int sort_tokens(const IDX* index, int64_t tokens, int64_t vocab, int64_t padding, uint8_t* ws, const EmbWorkspace& at, const uint32_t** keys,
                const uint32_t** pos, cudaStream_t st) {
  int bits = 1;  // of the largest key, vocab itself
  while (bits < 32 && (uint64_t)vocab >> bits) ++bits;
  const int passes = (bits + kMaxDigit - 1) / kMaxDigit;
  const int digit = (bits + passes - 1) / passes;
  uint32_t* k[2] = {reinterpret_cast<uint32_t*>(ws + at.k0), reinterpret_cast<uint32_t*>(ws + at.k1)};
  uint32_t* p[2] = {reinterpret_cast<uint32_t*>(ws + at.p0), reinterpret_cast<uint32_t*>(ws + at.p1)};
  uint32_t* hist = reinterpret_cast<uint32_t*>(ws + at.hist);
  uint32_t* group = reinterpret_cast<uint32_t*>(ws + at.group);
  int* n_long = reinterpret_cast<int*>(ws + at.n_long);
  const size_t smem = (size_t)kSortWarps * (1u << digit) * 4;
  static std::atomic<int> configured[kMaxDevices];
  if (!once_per_device(configured, [] {
        const int most = kSortWarps * (1 << kMaxDigit) * 4;
        return cudaFuncSetAttribute(radix_scatter_kernel<IDX>, cudaFuncAttributeMaxDynamicSharedMemorySize, most) == cudaSuccess &&
               cudaFuncSetAttribute(radix_single_kernel<IDX>, cudaFuncAttributeMaxDynamicSharedMemorySize, most) == cudaSuccess;
      }))
    return NTB200_LAUNCH_FAILED;
  PassIn<IDX> in = {index, nullptr, nullptr, vocab, padding, true};
  if (tokens <= kSingleBlock) {
    radix_single_kernel<IDX><<<1, kSortThreads, smem, st>>>(in, tokens, passes, digit, k[0], p[0], k[1], p[1], n_long);
  } else {
    for (int i = 0; i < passes; ++i) {
      radix_count_kernel<IDX><<<(unsigned)at.groups, kSortThreads, 0, st>>>(in, tokens, at.tile, (int)at.blocks, i * digit, digit, hist, group);
      radix_scatter_kernel<IDX><<<(unsigned)at.blocks, kSortThreads, smem, st>>>(in, tokens, at.tile, i * digit, digit, hist, group,
                                                                                 (int)at.groups, k[i & 1], p[i & 1], n_long);
      in.first = false;
      in.keys = k[i & 1], in.pos = p[i & 1];
    }
  }
  *keys = k[(passes - 1) & 1];
  *pos = p[(passes - 1) & 1];
  return status_from_cuda(cudaGetLastError());
}

template <int DT, int EPV, int VPL>
int launch_sums(const SumArgs& a, cudaStream_t st) {
  const int64_t nv = a.cols / EPV, slabs = (nv + 32 * VPL - 1) / (32 * VPL);
  const int64_t sum_warps = (a.tokens + kChunk - 1) / kChunk * slabs, zero_warps = (a.vocab + 31) / 32;
  const int64_t grid = (sum_warps + zero_warps + kSumWarps - 1) / kSumWarps;
  if (grid > 0x7fffffff) return NTB200_UNSUPPORTED_SHAPE;
  embedding_sum_kernel<DT, EPV, VPL><<<(unsigned)grid, kSumWarps * 32, 0, st>>>(a, (int)slabs, sum_warps);
  if (a.tokens > kChunk) {
    const int64_t col_blocks = (a.cols + 127) / 128;
    int64_t g = (a.tokens + kChunk - 1) / kChunk * col_blocks;
    if (g > 8 * kNumSMs) g = 8 * kNumSMs;
    embedding_long_runs_kernel<DT><<<(unsigned)g, 256, 0, st>>>(a, (int)col_blocks);
  }
  return status_from_cuda(cudaGetLastError());
}

template <int DT>
int sums(const SumArgs& a, cudaStream_t st) {
  constexpr int EPV = Vec16<DT>::kElems;
  // (four 16-byte vectors a lane, over 96 of them a row, spill 36 bytes beside the four rows in flight)
  if (a.cols % EPV == 0 && aligned16(a.grad) && aligned16(a.dw)) {
    const int64_t nv = a.cols / EPV;
    if (nv <= 32) return launch_sums<DT, EPV, 1>(a, st);
    if (nv <= 64) return launch_sums<DT, EPV, 2>(a, st);
    if (nv <= 96) return launch_sums<DT, EPV, 3>(a, st);
    return launch_sums<DT, EPV, 4>(a, st);
  }
  // Single elements, several slabs of columns for wide rows.  Twelve a lane: four rows of them are in flight beside the sums, and 16
  // spill (394 bytes stored; 12: 128).  15 000 tokens, fp32, 16 and 12 a lane: 131 columns 32 and 16 us, 333 41 and 19, 513 42 and 20,
  // 1001 50 and 30, 2055 75 and 65; bf16: 29 and 23, 32 and 25, 33 and 26, 36 and 30, 56 and 56.
  if (a.cols <= 128) return launch_sums<DT, 1, 4>(a, st);
  return launch_sums<DT, 1, 12>(a, st);
}

}  // namespace
}  // namespace ntb200

using namespace ntb200;

extern "C" {

size_t ntb200_embedding_backward_workspace_bytes(int64_t tokens, int64_t embed_dim) {
  if (tokens <= 0 || embed_dim <= 0 || tokens >= (1ll << 31) - 1) return 0;
  return EmbWorkspace(tokens, embed_dim).bytes;
}

int ntb200_embedding_backward(const void* grad, const void* index, int index_bytes, void* grad_weight, int64_t tokens, int64_t vocab,
                              int64_t embed_dim, int64_t padding_idx, float scale, int dtype, void* workspace, size_t workspace_bytes,
                              void* stream) {
  if (tokens < 0 || vocab < 0 || embed_dim < 0 || (index_bytes != 4 && index_bytes != 8)) return NTB200_INVALID_ARG;
  if (dtype != NTB200_F32 && dtype != NTB200_F16 && dtype != NTB200_BF16) return NTB200_UNSUPPORTED_DTYPE;
  if (vocab == 0 || embed_dim == 0) return NTB200_OK;
  if (tokens >= (1ll << 31) - 1 || vocab >= (1ll << 31) - 1 || embed_dim >= (1ll << 31) - 1) return NTB200_UNSUPPORTED_SHAPE;
  if (grad_weight == nullptr) return NTB200_INVALID_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  SumArgs a = {grad, nullptr, nullptr, grad_weight, nullptr, nullptr, nullptr, (tokens + kChunk - 1) / kChunk, tokens, vocab, embed_dim, scale};
  if (tokens > 0) {
    if (grad == nullptr || index == nullptr) return NTB200_INVALID_ARG;
    const EmbWorkspace at(tokens, embed_dim);
    if (workspace == nullptr || workspace_bytes < at.bytes) return NTB200_WORKSPACE_TOO_SMALL;
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return NTB200_MISALIGNED;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    const int rc = index_bytes == 8
                       ? sort_tokens(static_cast<const int64_t*>(index), tokens, vocab, padding_idx, ws, at, &a.keys, &a.pos, st)
                       : sort_tokens(static_cast<const int32_t*>(index), tokens, vocab, padding_idx, ws, at, &a.keys, &a.pos, st);
    if (rc != NTB200_OK) return rc;
    a.partial = reinterpret_cast<float*>(ws + at.partial);
    a.n_long = reinterpret_cast<int*>(ws + at.n_long);
    a.long_list = reinterpret_cast<int*>(ws + at.list);
  }
  switch (dtype) {
    case NTB200_F32: return sums<NTB200_F32>(a, st);
    case NTB200_F16: return sums<NTB200_F16>(a, st);
    default: return sums<NTB200_BF16>(a, st);
  }
}

}  // extern "C"
