// kd_embedding.hip -- surface_embedding: a table of embeddings (a row per face or vertex) looked
// up at an index image or at the faces' corners, and the table's gradient.
//
//   forward    out[i] = T(scale * E[key_i]),  0 where index[i] lies outside [0, rows)
//   backward   dE[k]  = T(scale * sum_{i : key_i = k} g[i])
// with key_i = batch(i) * rows + index[i] for a table per batch entry.  Products and sums are held
// in 32 bits (64 for fp64 data) and rounded once to T.
//
// Forward: one pass, a thread per 16 bytes of output; reads 8 n bytes of indices and the rows that
// are looked at, writes n * D * sizeof(T).
//
// Backward: no atomics on values, so the result does not depend on timing.  The tokens that name a row
// are sorted by key with a stable least-significant-digit radix sort (up to 10 bits a pass, 8 bytes a
// token), so a row's tokens stand together in token order; then each group of G lanes (one row of the
// gradient, 16 bytes a lane) walks a run of sorted tokens and adds their gradient rows in registers.
// Runs that cross a group's border are joined in LDS by the group in which they begin, runs that cross
// a workgroup's border by a second launch or, where the workgroups are few, by the last one.  The split
// of the walk over groups goes by position and not by key, so one face that fills the image costs no
// more than any other.
#include "kd_capi.hpp"
#include "kd_common.hpp"
#include "kd_float16.hpp"

#include <algorithm>
#include <type_traits>

namespace kd {

constexpr int kMaxBits = 10;                // of a sort digit: 16-bit keys take two passes, 20-bit ones too
constexpr int kDigits = 1 << kMaxBits;
constexpr int kFewCounts = 32768;           // up to so many counts (tiles x digits) need no scan launch
constexpr int kSortOne = 16384;             // up to so many tokens one workgroup sorts in one launch
constexpr int kJoinHere = 32;               // up to so many workgroups the last one joins the borders
constexpr int kJoinRounds = 4;              // (in so many rounds of its groups)
constexpr int kMaxChannels = 1 << 20;

// ------------------------------------------------------------------------------------------------
// forward
// ------------------------------------------------------------------------------------------------
// WHOLE: rows are whole 16-byte vectors, 16-byte aligned.  The output is written past the caches: it
// is larger than they are where its time counts, and the table's rows are what they should hold.  Bound
// by the bytes written: 2,097,152 tokens of 64 channels in bf16 (268 MB out, 17 MB of indices) 51 us,
// 5.6 TB/s; 8,388,608 of 32 channels in fp16 136 us, 4.4 TB/s (averages of six calls, as all times of one
// kernel here).
template <typename T, bool WHOLE>
__global__ __launch_bounds__(kBlock) void kd_embed_gather(
    int64_t n, uint32_t per_batch, int64_t rows, int D, int rows_per_block,
    const int64_t *__restrict__ index, const T *__restrict__ table, typename Wide<T>::type scale,
    T *__restrict__ out) {
  constexpr int V = 16 / sizeof(T);
  constexpr int U = 4;  // in flight per thread: the index, then the row, then the store
  const int64_t r0 = block_id() * rows_per_block;
  if (r0 >= n) return;
  const uint32_t nrow = (uint32_t)min((int64_t)rows_per_block, n - r0);
  const uint32_t vpr = (uint32_t)(D + V - 1) / V, total = nrow * vpr;
  for (uint32_t v0 = threadIdx.x; v0 < total; v0 += U * kBlock) {
    uint32_t lr[U], c[U];
    int64_t k[U];
    Pack<T, V> o[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t v = min(v0 + u * kBlock, total - 1);
      lr[u] = v / vpr;
      c[u] = (v - lr[u] * vpr) * V;
      k[u] = index[r0 + lr[u]];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (k[u] >= 0 && k[u] < rows) {
        const int64_t row =
            per_batch ? (int64_t)((uint32_t)(r0 + lr[u]) / per_batch) * rows + k[u] : k[u];
        o[u] = load_pack<T, V>(table + row * D + c[u], WHOLE ? V : D - (int)c[u]);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) o[u].v[j] = (T)0.f;
        k[u] = -1;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (v0 + u * kBlock >= total) break;
      if (k[u] >= 0) {
#pragma unroll
        for (int j = 0; j < V; ++j) o[u].v[j] = from_wide<T>(to_wide(o[u].v[j]) * scale);
      }
      T *to = out + (r0 + lr[u]) * D + c[u];
      if constexpr (WHOLE) {
        typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
        __builtin_nontemporal_store(__builtin_bit_cast(u32x4, o[u]), (u32x4 *)to);
      } else {
        store_pack<T, V>(to, o[u], D - (int)c[u]);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------
// stable radix sort of (key, token)
// ------------------------------------------------------------------------------------------------
struct SortKeys {
  const int64_t *index;  // first pass: keys from the indices, tokens that name no row left out
  const uint2 *pairs;    // later: (key, token)
  const uint32_t *kept;  // later: how many
  uint32_t n, per_batch;
  int64_t rows;
  __device__ __forceinline__ uint32_t count() const { return index ? n : *kept; }
  __device__ __forceinline__ bool get(uint32_t i, uint32_t m, uint2 &kt) const {
    if (i >= m) return false;
    if (!index) {
      kt = pairs[i];
      return true;
    }
    const int64_t k = index[i];
    kt.x = (uint32_t)((per_batch ? (int64_t)(i / per_batch) * rows : 0) + k);
    kt.y = i;
    return k >= 0 && k < rows;
  }
};

// rows that no token names: zeros
__device__ __forceinline__ void embed_fill(uint32_t block, uint32_t nblocks, int64_t bytes,
                                           void *p) {
  const int64_t head = min(bytes, (int64_t)((16 - ((uintptr_t)p & 15)) & 15));
  const int64_t body = (bytes - head) / 16, i0 = (int64_t)block * blockDim.x + threadIdx.x;
  uint4 *q = (uint4 *)((char *)p + head);
  for (int64_t i = i0; i < body; i += (int64_t)nblocks * blockDim.x) q[i] = make_uint4(0, 0, 0, 0);
  if (block == 0) {  // the two ends, 2 bytes at a time
    uint16_t *a = (uint16_t *)p, *z = (uint16_t *)(q + body);
    const int na = (int)(head / 2), nz = (int)((bytes - head - body * 16) / 2);
    if ((int)threadIdx.x < na) a[threadIdx.x] = 0;
    if ((int)threadIdx.x < nz) z[threadIdx.x] = 0;
  }
}

// Tokens a thread takes in a tile of kBlock times as many.  Small tiles fill the chip and shorten the
// chain of ranks in a workgroup, large ones leave fewer counts to sum and longer runs to write.  Both
// passes of 262,144 tokens take 31 us with 4 tokens a thread and 50 with 16, of 600,000 46, 46 and 58
// with 4, 8 and 16, of 2,097,152 57, 51 and 58, of 8,388,608 153, 121 and 120.
inline int sort_iters(int64_t n) { return n <= (1 << 19) ? 4 : n <= (1 << 22) ? 8 : 16; }

// Per tile the count of each digit; the blocks behind the tiles clear the gradient.
// few: a tile's counts stand together, else a digit's.
template <int ITERS>
__global__ __launch_bounds__(kBlock) void kd_embed_hist(SortKeys s, int shift, uint32_t mask,
                                                        int ntile, bool few, uint32_t *__restrict__ hist,
                                                        int64_t fill_bytes, void *fill) {
  if ((int)blockIdx.x >= ntile) {
    embed_fill(blockIdx.x - ntile, gridDim.x - ntile, fill_bytes, fill);
    return;
  }
  __shared__ uint32_t cnt[kDigits];
  for (uint32_t d = threadIdx.x; d <= mask; d += kBlock) cnt[d] = 0;
  __syncthreads();
  const uint32_t base = blockIdx.x * (uint32_t)(ITERS * kBlock), m = s.count();
  if (base < m) {
#pragma unroll
    for (int it = 0; it < ITERS; ++it) {
      uint2 kt;
      if (s.get(base + it * kBlock + threadIdx.x, m, kt)) atomicAdd(&cnt[(kt.x >> shift) & mask], 1u);
    }
  }
  __syncthreads();
  for (uint32_t d = threadIdx.x; d <= mask; d += kBlock)
    hist[few ? (int64_t)blockIdx.x * (mask + 1) + d : (int64_t)d * ntile + blockIdx.x] = cnt[d];
}

// Inclusive sum over the workgroup's N threads; total in every thread.
template <int N = kBlock>
__device__ __forceinline__ uint32_t wg_scan(uint32_t x, uint32_t *s_w, uint32_t &total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const uint32_t y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  if (lane == 63) s_w[w] = x;
  __syncthreads();
  uint32_t off = 0;
  total = 0;
#pragma unroll
  for (int k = 0; k < N / kWave; ++k) {
    if (k < w) off += s_w[k];
    total += s_w[k];
  }
  __syncthreads();
  return x + off;
}

// One workgroup per digit: its per-tile counts become exclusive offsets, the sum its total.
__global__ __launch_bounds__(kBlock) void kd_embed_scan(int ntile, uint32_t *__restrict__ hist,
                                                        uint32_t *__restrict__ totals) {
  __shared__ uint32_t s_w[kBlock / kWave];
  uint32_t *h = hist + (int64_t)blockIdx.x * ntile;
  uint32_t run = 0;
  for (int b = 0; b < ntile; b += kBlock) {
    const int i = b + threadIdx.x;
    const uint32_t c = i < ntile ? h[i] : 0u;
    uint32_t tot;
    const uint32_t inc = wg_scan(c, s_w, tot);
    if (i < ntile) h[i] = run + inc - c;
    run += tot;
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = run;
}

// A wave's rank of its ITERS x 64 consecutive tokens (kt, those of `in`), 64 at a time: the lanes that hold
// the same digit are found with one ballot per digit bit, a lane's rank is the number of lower ones among
// them plus the wave's count of that digit so far.  The order within a digit is the tokens' order: stable.
template <int ITERS>
__device__ __forceinline__ void embed_rank(const uint2 (&kt)[ITERS], uint32_t in, int iters, int shift,
                                           int bits, uint32_t *cnt, uint32_t (&rank)[ITERS]) {
  const uint32_t mask = (1u << bits) - 1u;
#pragma unroll
  for (int it = 0; it < ITERS; ++it) {
    if (it < iters) {
      const bool have = (in >> it) & 1u;
      const uint32_t d = (kt[it].x >> shift) & mask;
      uint64_t same = __ballot(have);
      for (int b = 0; b < bits; ++b) {
        const uint64_t set = __ballot((d >> b) & 1u);
        same &= ((d >> b) & 1u) ? set : ~set;
      }
      const int below = __builtin_amdgcn_mbcnt_hi((uint32_t)(same >> 32),
                                                  __builtin_amdgcn_mbcnt_lo((uint32_t)same, 0));
      uint32_t r = 0;
      if (have) {
        r = cnt[d];
        rank[it] = r + below;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (have && below == 0) cnt[d] = r + (uint32_t)__popcll(same);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  }
}

// Bound by latency and the scattered 8-byte writes: of 8,388,608 tokens the 4,217,024 that name one of
// 50,000 rows are written in 47 us, and in the second pass in 28 us, behind 17 us of counting; of
// 2,097,152 in 15 and 12 us behind 8.5.
// few: each workgroup adds up all tiles' counts itself, 16 bytes a thread and a share of the tiles: both
// passes of 262,144 tokens take 30 us in four launches against 26 in six, a call whose launches are its
// time 104 us against 109.
template <int ITERS>
__global__ __launch_bounds__(kBlock) void kd_embed_scatter(
    SortKeys s, int shift, int bits, int ntile, bool few, const uint32_t *__restrict__ hist,
    const uint32_t *__restrict__ totals, uint32_t *__restrict__ kept, uint2 *__restrict__ out) {
  constexpr int kWaves = kBlock / kWave;
  __shared__ uint32_t wcnt[kWaves][kDigits];
  __shared__ uint4 s_all[kBlock], s_before[kBlock];
  __shared__ uint32_t s_w[kWaves];
  const uint32_t mask = (1u << bits) - 1u, m = s.count();
  if (blockIdx.x * (uint32_t)(ITERS * kBlock) >= m && blockIdx.x > 0) return;
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (uint32_t d = threadIdx.x; d <= mask; d += kBlock) {
#pragma unroll
    for (int k = 0; k < kWaves; ++k) wcnt[k][d] = 0;
  }
  const uint32_t base = blockIdx.x * (uint32_t)(ITERS * kBlock) + w * (ITERS * kWave) + lane;
  uint2 kt[ITERS];
  uint32_t rank[ITERS], in = 0;
#pragma unroll
  for (int it = 0; it < ITERS; ++it)
    if (s.get(base + it * kWave, m, kt[it])) in |= 1u << it;
  const int quads = (int)(mask + 1) / 4, shares = kBlock / quads;  // (two bits or more)
  if (few) {
    uint4 all = make_uint4(0, 0, 0, 0), before = all;
#pragma unroll 8
    for (int k = (int)threadIdx.x / quads; k < ntile; k += shares) {
      const uint4 c = ((const uint4 *)hist)[k * quads + (int)threadIdx.x % quads];
      const bool b = k < (int)blockIdx.x;
      all.x += c.x, all.y += c.y, all.z += c.z, all.w += c.w;
      before.x += b ? c.x : 0u, before.y += b ? c.y : 0u;
      before.z += b ? c.z : 0u, before.w += b ? c.w : 0u;
    }
    s_all[threadIdx.x] = all;
    s_before[threadIdx.x] = before;
    for (int h = shares / 2; h >= 1; h >>= 1) {
      __syncthreads();
      if ((int)threadIdx.x < h * quads) {
        const uint4 c = s_all[threadIdx.x + h * quads], b = s_before[threadIdx.x + h * quads];
        uint4 &x = s_all[threadIdx.x], &y = s_before[threadIdx.x];
        x.x += c.x, x.y += c.y, x.z += c.z, x.w += c.w;
        y.x += b.x, y.y += b.y, y.z += b.z, y.w += b.w;
      }
    }
  }
  __syncthreads();
  embed_rank<ITERS>(kt, in, ITERS, shift, bits, wcnt[w], rank);
  __syncthreads();
  // where each digit begins among all tokens, and this tile's part of it
  // (a thread takes kDigits / kBlock digits in a row, as the sum over the digits needs)
  constexpr int kPer = kDigits / kBlock;
  uint32_t all[kPer], before[kPer], mine = 0, tot;
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    const uint32_t d = threadIdx.x * kPer + q;
    all[q] = before[q] = 0;
    if (d > mask) continue;
    if (few) {
      all[q] = ((const uint32_t *)s_all)[d];
      before[q] = ((const uint32_t *)s_before)[d];
    } else {
      all[q] = totals[d];
      before[q] = hist[(int64_t)d * ntile + blockIdx.x];
    }
    mine += all[q];
  }
  uint32_t begin = wg_scan(mine, s_w, tot) - mine;
  if (blockIdx.x == 0 && threadIdx.x == 0 && kept) {
    kept[0] = tot;
    kept[1] = 0;
  }
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    const uint32_t d = threadIdx.x * kPer + q;
    if (d > mask) continue;
    uint32_t off = begin + before[q];
    begin += all[q];
#pragma unroll
    for (int k = 0; k < kWaves; ++k) {
      const uint32_t c = wcnt[k][d];
      wcnt[k][d] = off;
      off += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int it = 0; it < ITERS; ++it)
    if ((in >> it) & 1u) out[wcnt[w][(kt[it].x >> shift) & mask] + rank[it]] = kt[it];
}

// All passes for few tokens in one workgroup, in the place of two launches a pass (bound by the latency
// of its loads, ranks and stores: 9,680 tokens and 6,335 rows 22 us against 39 us for the four launches,
// 16,000 tokens 43 us against 43).  The blocks behind the first clear the gradient.
constexpr int kOneThreads = 1024, kOneIters = kSortOne / kOneThreads;
static_assert(kOneThreads == kDigits, "a thread a digit");
__global__ __launch_bounds__(kOneThreads) void kd_embed_sort(SortKeys s, int bits, int passes,
                                                             uint32_t *kept, uint2 *even, uint2 *odd,
                                                             int64_t fill_bytes, void *fill) {
  if (blockIdx.x > 0) {
    embed_fill(blockIdx.x - 1, gridDim.x - 1, fill_bytes, fill);
    return;
  }
  constexpr int kWaves = kOneThreads / kWave;
  __shared__ uint32_t wcnt[kWaves][kDigits];
  __shared__ uint32_t s_w[kWaves];
  const uint32_t mask = (1u << bits) - 1u, d = threadIdx.x;
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  uint32_t m = s.n;
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * bits, iters = (int)((m + kOneThreads - 1) / kOneThreads);
    if (d <= mask) {
#pragma unroll
      for (int k = 0; k < kWaves; ++k) wcnt[k][d] = 0;
    }
    const uint32_t base = (uint32_t)(w * iters * kWave + lane);
    uint2 kt[kOneIters];
    uint32_t rank[kOneIters], in = 0;
#pragma unroll
    for (int it = 0; it < kOneIters; ++it) {
      if (it < iters && s.get(base + it * kWave, m, kt[it])) in |= 1u << it;
    }
    __syncthreads();
    embed_rank<kOneIters>(kt, in, iters, shift, bits, wcnt[w], rank);
    __syncthreads();
    uint32_t mine = 0, tot;
    if (d <= mask) {
#pragma unroll
      for (int k = 0; k < kWaves; ++k) mine += wcnt[k][d];
    }
    uint32_t off = wg_scan<kOneThreads>(mine, s_w, tot) - mine;
    if (d <= mask) {
#pragma unroll
      for (int k = 0; k < kWaves; ++k) {
        const uint32_t c = wcnt[k][d];
        wcnt[k][d] = off;
        off += c;
      }
    }
    __syncthreads();
    uint2 *out = pass & 1 ? odd : even;
#pragma unroll
    for (int it = 0; it < kOneIters; ++it) {
      if ((in >> it) & 1u) out[wcnt[w][(kt[it].x >> shift) & mask] + rank[it]] = kt[it];
    }
    m = tot;
    s.index = nullptr;
    s.pairs = out;
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    kept[0] = m;
    kept[1] = 0;
  }
}

// ------------------------------------------------------------------------------------------------
// sums over the runs of equal keys
// ------------------------------------------------------------------------------------------------
// Bound by the gathered gradient rows, which are as long as a memory access or shorter: 1,054,304 rows
// of 128 bytes 50 us, 2.9 TB/s; 4,217,024 rows of 64 bytes 124 us, 2.5 TB/s.
constexpr int kHasHead = 1;   // the first run began before this range
constexpr int kHasTail = 2;   // the last run goes on behind this range
constexpr int kThrough = 4;   // one run covers the range and both borders (its sum is the head's)

struct SegArgs {
  uint32_t *kept;          // sorted tokens; behind it the workgroups that are done
  int D, glog, per_group;  // lanes per gradient row (log2), sorted tokens per group
  const uint2 *pairs;
  int *flags;              // per workgroup
};

template <typename T, int V>
__device__ __forceinline__ void embed_store(T *out, int D, uint32_t key, int col,
                                            const typename Wide<T>::type *acc,
                                            typename Wide<T>::type scale) {
  Pack<T, V> o;
#pragma unroll
  for (int j = 0; j < V; ++j) o.v[j] = from_wide<T>(acc[j] * scale);
  store_pack<T, V>(out + (int64_t)key * D + col, o, D - col);
}

template <typename T>
__device__ __forceinline__ void embed_segments(const SegArgs &a, const T *__restrict__ grad,
                                               typename Wide<T>::type scale, T *out,
                                               typename Wide<T>::type *head,
                                               typename Wide<T>::type *tail) {
  using A = typename Wide<T>::type;
  constexpr int V = 16 / sizeof(T), U = 4;  // channels of a lane, gradient rows in flight
  __shared__ A s_head[kBlock * V];
  __shared__ int s_kind[kBlock];
  const uint32_t n = *a.kept;
  const int G = 1 << a.glog, NG = kBlock >> a.glog;
  const int g = threadIdx.x >> a.glog, gl = threadIdx.x & (G - 1);
  const int col = ((int)blockIdx.y * G + gl) * V;
  const bool live = col < a.D;
  if ((uint64_t)blockIdx.x * NG * (uint64_t)a.per_group >= n) {  // behind the last token
    if (threadIdx.x == 0 && blockIdx.y == 0) a.flags[blockIdx.x] = 0;
    return;
  }
  const uint64_t s64 = ((uint64_t)blockIdx.x * NG + g) * (uint64_t)a.per_group;
  const uint32_t s = (uint32_t)min(s64, (uint64_t)n);
  const uint32_t e = (uint32_t)min(s64 + a.per_group, (uint64_t)n);
  int kind = 0;
  A acc[V];
#pragma unroll
  for (int j = 0; j < V; ++j) acc[j] = (A)0;
  if (s < e) {
    const uint32_t none = 0xffffffffu;  // (keys are below 2^31)
    const uint32_t prev = s > 0 ? a.pairs[s - 1].x : none;
    const uint32_t next = e < n ? a.pairs[e].x : none;
    uint32_t cur = a.pairs[s].x;
    bool from_prev = cur == prev;
    for (uint32_t i = s; i < e; i += U) {
      uint2 kt[U];
      Pack<T, V> row[U];
#pragma unroll
      for (int u = 0; u < U; ++u) kt[u] = a.pairs[min(i + u, e - 1)];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (live && i + u < e) row[u] = load_pack<T, V>(grad + (int64_t)kt[u].y * a.D + col, a.D - col);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i + u >= e) break;
        if (kt[u].x != cur) {  // the run ends inside this group's range
          if (from_prev) {
            kind |= kHasHead;
#pragma unroll
            for (int j = 0; j < V; ++j) s_head[threadIdx.x * V + j] = acc[j];
          } else if (live) {
            embed_store<T, V>(out, a.D, cur, col, acc, scale);
          }
          cur = kt[u].x;
          from_prev = false;
#pragma unroll
          for (int j = 0; j < V; ++j) acc[j] = (A)0;
        }
        if (live) {
#pragma unroll
          for (int j = 0; j < V; ++j) acc[j] += to_wide(row[u].v[j]);
        }
      }
    }
    const bool on = next == cur;
    if (from_prev) {
      kind |= kHasHead | (on ? kThrough : 0);
#pragma unroll
      for (int j = 0; j < V; ++j) s_head[threadIdx.x * V + j] = acc[j];
    } else if (on) {
      kind |= kHasTail;  // (its sum stays in registers)
    } else if (live) {
      embed_store<T, V>(out, a.D, cur, col, acc, scale);
    }
  }
  if (gl == 0) s_kind[g] = kind;
  __syncthreads();
  const int64_t wcol = (int64_t)gridDim.y * G * V;  // a partial's channels
  if (kind & kHasTail) {  // the run's owner: add the heads behind it
    int q = g + 1;
    bool open = true;
    for (; q < NG && open; ++q) {
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] += s_head[((q << a.glog) + gl) * V + j];
      open = s_kind[q] & kThrough;
    }
    if (!open) {
      if (live) embed_store<T, V>(out, a.D, a.pairs[e - 1].x, col, acc, scale);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) tail[(int64_t)blockIdx.x * wcol + col + j] = acc[j];
    }
  }
  if (g == 0) {
    int f = 0;
    if (kind & kHasHead) {  // the run that began in an earlier workgroup
      f = kHasHead;
      A h[V];
#pragma unroll
      for (int j = 0; j < V; ++j) h[j] = s_head[threadIdx.x * V + j];
      bool open = kind & kThrough;
      for (int q = 1; q < NG && open; ++q) {
#pragma unroll
        for (int j = 0; j < V; ++j) h[j] += s_head[((q << a.glog) + gl) * V + j];
        open = s_kind[q] & kThrough;
      }
      if (open) f |= kThrough;
#pragma unroll
      for (int j = 0; j < V; ++j) head[(int64_t)blockIdx.x * wcol + col + j] = h[j];
    }
    // a run that is open at the end of the workgroup began in it unless it runs through
    for (int q = NG - 1; q >= 0; --q) {
      if (s_kind[q] & kHasTail) f |= kHasTail;
      if (!(s_kind[q] & kThrough)) break;
    }
    if (gl == 0 && blockIdx.y == 0) a.flags[blockIdx.x] = f;
  }
}

// The runs that cross a workgroup's border, each added up where it begins: a group of lanes takes one
// border and joins the two sides; the few runs that go on through whole workgroups are left to all
// groups together, one after the other, in a fixed order.
template <typename T>
__device__ __forceinline__ void embed_join(const SegArgs &a, int bx, int by, int gy, int nwg,
                                           typename Wide<T>::type scale,
                                           const typename Wide<T>::type *head,
                                           const typename Wide<T>::type *tail, T *out) {
  using A = typename Wide<T>::type;
  constexpr int V = 16 / sizeof(T);
  __shared__ int s_end;
  __shared__ uint8_t s_long[kBlock];
  __shared__ A s_sum[kBlock * V];
  const int G = 1 << a.glog, NG = kBlock >> a.glog;
  const int g = threadIdx.x >> a.glog, gl = threadIdx.x & (G - 1);
  const int col = (by * G + gl) * V;
  const int64_t wcol = (int64_t)gy * G * V;
  // a run that is open at the end of workgroup w goes on behind it: the position is inside
  auto store = [&](int w, const A *acc) {
    const uint64_t end = (uint64_t)(w + 1) * NG * a.per_group;
    if (col < a.D) embed_store<T, V>(out, a.D, a.pairs[end - 1].x, col, acc, scale);
  };
  bool far = false;
  {
    const int w = bx * NG + g;
    if (w < nwg - 1 && (a.flags[w] & kHasTail)) {
      far = a.flags[w + 1] & kThrough;
      if (!far) {
        A acc[V];
#pragma unroll
        for (int j = 0; j < V; ++j)
          acc[j] = tail[(int64_t)w * wcol + col + j] + head[(int64_t)(w + 1) * wcol + col + j];
        store(w, acc);
      }
    }
    if (gl == 0) s_long[g] = far;
  }
  if (!__syncthreads_or(far)) return;
  for (int q0 = 0; q0 < NG; ++q0) {
    if (!s_long[q0]) continue;  // (the same for the whole workgroup)
    const int w = bx * NG + q0;
    if (threadIdx.x == 0) s_end = nwg;
    __syncthreads();
    // the first workgroup behind w through which the run does not go on
    for (int b = w + 1; b < nwg; b += kBlock) {
      const int q = b + threadIdx.x;
      if (q < nwg && !(a.flags[q] & kThrough)) atomicMin(&s_end, q);
      __syncthreads();
      const bool found = s_end < nwg;
      __syncthreads();
      if (found) break;
    }
    const int last = min(s_end, nwg - 1);
    A acc[V];
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] = g == 0 ? tail[(int64_t)w * wcol + col + j] : (A)0;
    for (int q = w + 1 + g; q <= last; q += NG) {
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] += head[(int64_t)q * wcol + col + j];
    }
#pragma unroll
    for (int j = 0; j < V; ++j) s_sum[threadIdx.x * V + j] = acc[j];
    __syncthreads();
    if (g == 0) {
      for (int q = 1; q < NG; ++q) {
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] += s_sum[((q << a.glog) + gl) * V + j];
      }
      store(w, acc);
    }
    __syncthreads();
  }
}

template <typename T>
__global__ __launch_bounds__(kBlock) void kd_embed_join(SegArgs a, int nwg,
                                                        typename Wide<T>::type scale,
                                                        const typename Wide<T>::type *__restrict__ head,
                                                        const typename Wide<T>::type *__restrict__ tail,
                                                        T *__restrict__ out) {
  embed_join<T>(a, (int)blockIdx.x, (int)blockIdx.y, (int)gridDim.y, nwg, scale, head, tail, out);
}

// JOIN: the workgroup that is done last joins the borders of all, where there are few workgroups: the
// time is that of a second launch (4,000 tokens 18.5 us against 8.7 and 8.6), without the launch.  Each
// workgroup's fence costs 0.2 us, one after the other: with 196 of them 44 us against 11.
template <typename T, bool JOIN>
__global__ __launch_bounds__(kBlock) void kd_embed_segments(SegArgs a, const T *__restrict__ grad,
                                                            typename Wide<T>::type scale, T *out,
                                                            typename Wide<T>::type *head,
                                                            typename Wide<T>::type *tail) {
  embed_segments<T>(a, grad, scale, out, head, tail);
  if constexpr (JOIN) {
    __shared__ bool s_last;
    const int nwg = (int)gridDim.x, gy = (int)gridDim.y, per = kBlock >> a.glog;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) s_last = atomicAdd(a.kept + 1, 1u) == gridDim.x * gridDim.y - 1;
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    for (int y = 0; y < gy; ++y)
      for (int x = 0; x * per < nwg; ++x) {
        embed_join<T>(a, x, y, gy, nwg, scale, head, tail, out);
        __syncthreads();
      }
  }
}

// ------------------------------------------------------------------------------------------------
// host
// ------------------------------------------------------------------------------------------------
struct EmbedPlan {
  int glog, gy, per_group, nwg, iters, ntile, passes, bits;
  size_t pairs, hist, part, flags, total;  // workspace parts in bytes
};

static size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

static EmbedPlan embed_plan(int64_t n, int64_t nkeys, int D, int esize) {
  EmbedPlan p;
  const int V = 16 / esize, cols = (D + V - 1) / V;
  p.glog = 0;
  while (p.glog < 6 && (1 << p.glog) < cols) ++p.glog;
  p.gy = (cols + (1 << p.glog) - 1) >> p.glog;
  const int64_t ng = kBlock >> p.glog;
  // tokens per group: long walks write less at the borders, short ones fill the chip
  p.per_group = 64;
  while (p.per_group > 8 && (n + ng * p.per_group - 1) / (ng * p.per_group) < 4096) p.per_group >>= 1;
  p.nwg = (int)((n + ng * p.per_group - 1) / (ng * p.per_group));
  p.iters = sort_iters(n);
  p.ntile = (int)((n + p.iters * kBlock - 1) / (p.iters * kBlock));
  int kb = 1;
  while (kb < 32 && ((nkeys - 1) >> kb) != 0) ++kb;  // keys 0 .. nkeys - 1
  p.passes = (kb + kMaxBits - 1) / kMaxBits;
  p.bits = std::max((kb + p.passes - 1) / p.passes, 2);
  const int asize = esize == 8 ? 8 : 4;
  p.pairs = up256(8 * (size_t)n);
  p.hist = up256(4 * (size_t)kDigits * (size_t)p.ntile + 4 * kDigits + 8);
  p.part = up256((size_t)p.nwg * (size_t)p.gy * (size_t)(V << p.glog) * (size_t)asize);
  p.flags = up256(4 * (size_t)p.nwg);
  p.total = 2 * p.pairs + p.hist + 2 * p.part + p.flags;
  return p;
}

static int embed_check(int64_t n, int64_t batch, int64_t rows, int D, const void *index,
                       const void *x) {
  KD_CHECK_ARG(n >= 0 && n < ((int64_t)1 << 31), "surface_embedding: need 0 <= indices < 2^31");
  KD_CHECK_ARG(batch >= 1 && rows >= 0 && rows < ((int64_t)1 << 31) &&
                   batch < ((int64_t)1 << 31) && batch * rows < ((int64_t)1 << 31),
               "surface_embedding: need batch >= 1 and batch * rows < 2^31");
  KD_CHECK_ARG(n % batch == 0, "surface_embedding: the indices do not split over the batch");
  KD_CHECK_ARG(D >= 0 && D <= kMaxChannels, "surface_embedding: need 0 <= channels <= 2^20");
  KD_CHECK_ARG(n == 0 || index, "surface_embedding: index is NULL");
  KD_CHECK_ARG(n == 0 || D == 0 || x, "surface_embedding: NULL input");
  return KD_OK;
}

template <typename T>
static int embed_forward(int64_t n, int64_t batch, int64_t rows, int D, const int64_t *index,
                         const T *table, double scale, T *out, hipStream_t stream) {
  const int rc = embed_check(n, batch, rows, D, index, out);
  if (rc != KD_OK) return rc;
  KD_CHECK_ARG(rows == 0 || D == 0 || n == 0 || table, "surface_embedding: embeddings is NULL");
  if (n == 0 || D == 0) return KD_OK;
  using A = typename Wide<T>::type;
  constexpr int V = 16 / (int)sizeof(T);
  const int rpb = std::max(1, kBlock * 4 / ((D + V - 1) / V));
  const dim3 grid = grid_of((n + rpb - 1) / rpb);
  const uint32_t pb = batch > 1 ? (uint32_t)(n / batch) : 0u;
  {
    ProfScope prof(K_EMBED_FWD, stream);
    if (D % V == 0 && (((uintptr_t)table | (uintptr_t)out) & 15u) == 0)
      hipLaunchKernelGGL((kd_embed_gather<T, true>), grid, dim3(kBlock), 0, stream, n, pb, rows,
                         D, rpb, index, table, (A)scale, out);
    else
      hipLaunchKernelGGL((kd_embed_gather<T, false>), grid, dim3(kBlock), 0, stream, n, pb,
                         rows, D, rpb, index, table, (A)scale, out);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(KD_ERR_LAUNCH, "surface_embedding: %s", hipGetErrorString(e));
  return KD_OK;
}

template <typename T>
static int embed_backward(int64_t n, int64_t batch, int64_t rows, int D, const int64_t *index,
                          const T *grad, double scale, T *out, void *ws, size_t wsb,
                          hipStream_t stream) {
  const int rc = embed_check(n, batch, rows, D, index, grad);
  if (rc != KD_OK) return rc;
  const int64_t nkeys = batch * rows, nout = nkeys * D;
  if (nout == 0) return KD_OK;
  KD_CHECK_ARG(out, "surface_embedding: grad_embeddings is NULL");
  using A = typename Wide<T>::type;
  const int64_t fill = nout * (int64_t)sizeof(T);
  const unsigned fblocks = (unsigned)std::min<int64_t>((fill / 16 + kBlock) / kBlock, 2048);
  ProfScope prof(K_EMBED_BWD, stream);
  if (n == 0) {
    hipLaunchKernelGGL(kd_embed_hist<4>, dim3(fblocks), dim3(kBlock), 0, stream, SortKeys{}, 0, 0u, 0,
                       false, (uint32_t *)nullptr, fill, (void *)out);
  } else {
    const EmbedPlan p = embed_plan(n, nkeys, D, (int)sizeof(T));
    if (wsb < p.total || !ws)
      return set_error(KD_ERR_WORKSPACE, "workspace too small: %zu < %zu", wsb, p.total);
    KD_CHECK_ARG(((uintptr_t)ws & 255u) == 0,
                 "surface_embedding: the workspace must be aligned to 256 bytes");
    char *c = (char *)ws;
    uint2 *buf[2] = {(uint2 *)c, (uint2 *)(c + p.pairs)};
    c += 2 * p.pairs;
    uint32_t *hist = (uint32_t *)c, *totals = hist + (size_t)kDigits * p.ntile;
    uint32_t *kept = totals + kDigits;
    c += p.hist;
    A *head = (A *)c, *tail = (A *)(c + p.part);
    int *flags = (int *)(c + 2 * p.part);
    SortKeys s;
    s.index = index;
    s.pairs = nullptr;
    s.kept = kept;
    s.n = (uint32_t)n;
    s.per_batch = batch > 1 ? (uint32_t)(n / batch) : 0u;
    s.rows = rows;
    if (n <= kSortOne) {
      hipLaunchKernelGGL(kd_embed_sort, dim3(1 + (unsigned)std::min<int64_t>(fblocks, 512)),
                         dim3(kOneThreads), 0, stream, s, p.bits, p.passes, kept, buf[0], buf[1], fill,
                         (void *)out);
      s.pairs = buf[(p.passes - 1) & 1];
    } else {
      const uint32_t mask = (1u << p.bits) - 1u;
      const unsigned nt = (unsigned)p.ntile;
      const bool few = (int64_t)p.ntile * (mask + 1) <= kFewCounts;
      for (int q = 0; q < p.passes; ++q) {
        const int shift = q * p.bits;
        const unsigned extra = q == 0 ? fblocks : 0u;  // the first launch clears the gradient too
        uint32_t *first = q == 0 ? kept : nullptr;
        auto pass = [&](auto iters) {
          constexpr int I = decltype(iters)::value;
          hipLaunchKernelGGL(kd_embed_hist<I>, dim3(nt + extra), dim3(kBlock), 0, stream, s, shift, mask,
                             p.ntile, few, hist, fill, (void *)out);
          if (!few)
            hipLaunchKernelGGL(kd_embed_scan, dim3(mask + 1), dim3(kBlock), 0, stream, p.ntile, hist,
                               totals);
          hipLaunchKernelGGL(kd_embed_scatter<I>, dim3(nt), dim3(kBlock), 0, stream, s, shift, p.bits,
                             p.ntile, few, hist, totals, first, buf[q & 1]);
        };
        if (p.iters == 4)
          pass(std::integral_constant<int, 4>{});
        else if (p.iters == 8)
          pass(std::integral_constant<int, 8>{});
        else
          pass(std::integral_constant<int, 16>{});
        s.index = nullptr;
        s.pairs = buf[q & 1];
      }
    }
    SegArgs a;
    a.kept = kept;
    a.D = D;
    a.glog = p.glog;
    a.per_group = p.per_group;
    a.pairs = s.pairs;
    a.flags = flags;
    const dim3 grid((unsigned)p.nwg, (unsigned)p.gy);
    const int per = kBlock >> p.glog;
    if (p.nwg > 1 && p.nwg <= kJoinHere && p.gy * ((p.nwg + per - 1) / per) <= kJoinRounds) {
      hipLaunchKernelGGL((kd_embed_segments<T, true>), grid, dim3(kBlock), 0, stream, a, grad, (A)scale,
                         out, head, tail);
    } else {
      hipLaunchKernelGGL((kd_embed_segments<T, false>), grid, dim3(kBlock), 0, stream, a, grad,
                         (A)scale, out, head, tail);
      if (p.nwg > 1)
        hipLaunchKernelGGL(kd_embed_join<T>, dim3((unsigned)((p.nwg + per - 1) / per), (unsigned)p.gy),
                           dim3(kBlock), 0, stream, a, p.nwg, (A)scale, (const A *)head,
                           (const A *)tail, out);
    }
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    return set_error(KD_ERR_LAUNCH, "surface_embedding bwd: %s", hipGetErrorString(e));
  return KD_OK;
}

}  // namespace kd

using namespace kd;

extern "C" {

size_t kd_surface_embedding_workspace_size(int64_t num_indices, int64_t batch, int64_t rows,
                                           int channels, int element_size) {
  if (num_indices <= 0 || num_indices >= ((int64_t)1 << 31) || batch < 1 || rows < 1 ||
      rows >= ((int64_t)1 << 31) || batch >= ((int64_t)1 << 31) ||
      batch * rows >= ((int64_t)1 << 31) || channels < 1 || channels > kMaxChannels ||
      (element_size != 2 && element_size != 4 && element_size != 8))
    return 0;
  return embed_plan(num_indices, batch * rows, channels, element_size).total;
}

#define KD_EMBED(SFX, T)                                                                          \
  int kd_surface_embedding_forward_##SFX(int64_t n, int64_t batch, int64_t rows, int channels,    \
                                         const int64_t *index, const void *embeddings,            \
                                         double scale, void *out, void *stream) {                 \
    return embed_forward<T>(n, batch, rows, channels, index, (const T *)embeddings, scale,        \
                            (T *)out, (hipStream_t)stream);                                       \
  }                                                                                               \
  int kd_surface_embedding_backward_##SFX(                                                        \
      int64_t n, int64_t batch, int64_t rows, int channels, const int64_t *index,                 \
      const void *grad_out, double scale, void *grad_embeddings, void *workspace,                 \
      size_t workspace_bytes, void *stream) {                                                     \
    return embed_backward<T>(n, batch, rows, channels, index, (const T *)grad_out, scale,         \
                             (T *)grad_embeddings, workspace, workspace_bytes,                    \
                             (hipStream_t)stream);                                                \
  }

KD_EMBED(f32, float)
KD_EMBED(f64, double)
KD_EMBED(f16, half_t)
KD_EMBED(bf16, bfloat_t)

}  // extern "C"
