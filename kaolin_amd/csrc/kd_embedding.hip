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
// Backward: no atomics on values, so the result does not depend on timing.  The tokens are sorted
// by key with a stable least-significant-digit radix sort (two to four passes over 8 bytes a
// token), so a row's tokens stand together in token order; then each group of G lanes (one row of
// the gradient, 16 bytes a lane) walks a run of sorted tokens and adds their gradient rows in
// registers.  Runs that cross a group's border are joined in LDS by the group in which they begin,
// runs that cross a workgroup's border by a second launch.  The split of the walk over groups goes
// by position and not by key, so one face that fills the image costs no more than any other.
#include "kd_capi.hpp"
#include "kd_common.hpp"
#include "kd_float16.hpp"

#include <algorithm>

namespace kd {

constexpr int kSortTile = 4096;             // tokens per sort workgroup (16 per thread)
constexpr int kSortIters = kSortTile / kBlock;
constexpr int kDigits = 256;
constexpr int kMaxChannels = 1 << 20;

// ------------------------------------------------------------------------------------------------
// forward
// ------------------------------------------------------------------------------------------------
template <typename T, int VEC>
__global__ __launch_bounds__(kBlock) void kd_embed_gather(
    int64_t n, uint32_t per_batch, int64_t rows, int D, int rows_per_block,
    const int64_t *__restrict__ index, const T *__restrict__ table, typename Wide<T>::type scale,
    T *__restrict__ out) {
  using A = typename Wide<T>::type;
  const int64_t r0 = (int64_t)blockIdx.x * rows_per_block;
  const uint32_t nrow = (uint32_t)min((int64_t)rows_per_block, n - r0);
  const uint32_t vpr = (uint32_t)(D / VEC), total = nrow * vpr;
  for (uint32_t v = threadIdx.x; v < total; v += kBlock) {
    const uint32_t lr = v / vpr, c = (v - lr * vpr) * VEC;
    const int64_t i = r0 + lr;
    const int64_t k = index[i];
    Pack<T, VEC> o;
    if (k >= 0 && k < rows) {
      const int64_t row = per_batch ? (int64_t)((uint32_t)i / per_batch) * rows + k : k;
      const Pack<T, VEC> e = *(const Pack<T, VEC> *)(table + row * D + c);
#pragma unroll
      for (int j = 0; j < VEC; ++j) o.v[j] = from_wide<T>(to_wide(e.v[j]) * scale);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) o.v[j] = from_wide<T>((A)0);
    }
    *(Pack<T, VEC> *)(out + i * D + c) = o;
  }
}

// ------------------------------------------------------------------------------------------------
// stable radix sort of (key, token)
// ------------------------------------------------------------------------------------------------
struct SortKeys {
  const int64_t *index;  // first pass: keys from the indices
  const uint32_t *keys, *toks;
  uint32_t n, per_batch, nkeys;
  int64_t rows;
  __device__ __forceinline__ uint32_t key(uint32_t i) const {
    if (!index) return keys[i];
    const int64_t k = index[i];
    if (k < 0 || k >= rows) return nkeys;  // no row: sorted behind every row
    return (uint32_t)((per_batch ? (int64_t)(i / per_batch) * rows : 0) + k);
  }
  __device__ __forceinline__ uint32_t tok(uint32_t i) const { return index ? i : toks[i]; }
};

__global__ __launch_bounds__(kBlock) void kd_embed_hist(SortKeys s, int shift, uint32_t mask,
                                                        int ntile, uint32_t *__restrict__ hist) {
  __shared__ uint32_t cnt[kDigits];
  cnt[threadIdx.x] = 0;
  __syncthreads();
  const uint32_t base = blockIdx.x * (uint32_t)kSortTile;
#pragma unroll 4
  for (int it = 0; it < kSortIters; ++it) {
    const uint32_t i = base + it * kBlock + threadIdx.x;
    if (i < s.n) atomicAdd(&cnt[(s.key(i) >> shift) & mask], 1u);
  }
  __syncthreads();
  if (threadIdx.x <= mask) hist[(int64_t)threadIdx.x * ntile + blockIdx.x] = cnt[threadIdx.x];
}

// Inclusive sum over the workgroup's threads; total in every thread.
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
  for (int k = 0; k < kBlock / kWave; ++k) {
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

// Each wave ranks its 1024 consecutive tokens 64 at a time: the lanes that hold the same digit are
// found with one ballot per digit bit, a lane's rank is the number of lower ones among them plus
// the wave's count of that digit so far.  The order within a digit is the tokens' order: stable.
__global__ __launch_bounds__(kBlock) void kd_embed_scatter(
    SortKeys s, int shift, int bits, int ntile, const uint32_t *__restrict__ hist,
    const uint32_t *__restrict__ totals, uint32_t *__restrict__ okeys,
    uint32_t *__restrict__ otoks) {
  constexpr int kWaves = kBlock / kWave;
  __shared__ uint32_t wcnt[kWaves][kDigits];
  __shared__ uint32_t s_w[kWaves];
  const uint32_t mask = (1u << bits) - 1u;
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
  for (int k = 0; k < kWaves; ++k) wcnt[k][threadIdx.x] = 0;
  // where each digit begins among all tokens
  uint32_t tot;
  const uint32_t mine = threadIdx.x <= mask ? totals[threadIdx.x] : 0u;
  const uint32_t begin = wg_scan(mine, s_w, tot) - mine;  // (barriers inside)
  const uint32_t base = blockIdx.x * (uint32_t)kSortTile + w * (kSortTile / kWaves) + lane;
  uint32_t key[kSortIters], rank[kSortIters];
#pragma unroll
  for (int it = 0; it < kSortIters; ++it) {
    const uint32_t i = base + it * kWave;
    key[it] = i < s.n ? s.key(i) : 0u;
  }
#pragma unroll
  for (int it = 0; it < kSortIters; ++it) {
    const bool in = base + it * kWave < s.n;
    const uint32_t d = (key[it] >> shift) & mask;
    uint64_t same = __ballot(in);
    for (int b = 0; b < bits; ++b) {
      const uint64_t m = __ballot((d >> b) & 1u);
      same &= ((d >> b) & 1u) ? m : ~m;
    }
    const int below = __builtin_amdgcn_mbcnt_hi((uint32_t)(same >> 32),
                                                __builtin_amdgcn_mbcnt_lo((uint32_t)same, 0));
    uint32_t r = 0;
    if (in) {
      r = wcnt[w][d];
      rank[it] = r + below;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (in && below == 0) wcnt[w][d] = r + (uint32_t)__popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  __syncthreads();
  if (threadIdx.x <= mask) {
    uint32_t off = begin + hist[(int64_t)threadIdx.x * ntile + blockIdx.x];
#pragma unroll
    for (int k = 0; k < kWaves; ++k) {
      const uint32_t c = wcnt[k][threadIdx.x];
      wcnt[k][threadIdx.x] = off;
      off += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int it = 0; it < kSortIters; ++it) {
    const uint32_t i = base + it * kWave;
    if (i < s.n) {
      const uint32_t p = wcnt[w][(key[it] >> shift) & mask] + rank[it];
      okeys[p] = key[it];
      otoks[p] = s.tok(i);
    }
  }
}

// ------------------------------------------------------------------------------------------------
// sums over the runs of equal keys
// ------------------------------------------------------------------------------------------------
constexpr int kHasHead = 1;   // the first run began before this range
constexpr int kHasTail = 2;   // the last run goes on behind this range
constexpr int kThrough = 4;   // one run covers the range and both borders (its sum is the head's)

struct SegArgs {
  uint32_t n, nkeys;
  int D, glog, per_group;  // lanes per gradient row (log2), sorted tokens per group
  const uint32_t *keys, *toks;
  int *flags;              // per workgroup
};

template <typename T>
__global__ __launch_bounds__(kBlock) void kd_embed_fill(int64_t n, T *__restrict__ p) {
  for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * kBlock)
    p[i] = (T)0;
}

template <typename T, int VEC>
__device__ __forceinline__ void embed_store(T *out, int D, uint32_t key, int col,
                                            const typename Wide<T>::type *acc,
                                            typename Wide<T>::type scale) {
  Pack<T, VEC> o;
#pragma unroll
  for (int j = 0; j < VEC; ++j) o.v[j] = from_wide<T>(acc[j] * scale);
  *(Pack<T, VEC> *)(out + (int64_t)key * D + col) = o;
}

template <typename T, int VEC>
__global__ __launch_bounds__(kBlock) void kd_embed_segments(SegArgs a, const T *__restrict__ grad,
                                                            typename Wide<T>::type scale,
                                                            T *__restrict__ out,
                                                            typename Wide<T>::type *__restrict__ head,
                                                            typename Wide<T>::type *__restrict__ tail) {
  using A = typename Wide<T>::type;
  constexpr int U = 4;  // gradient rows in flight per lane
  __shared__ A s_head[kBlock * VEC], s_tail[kBlock * VEC];
  __shared__ int s_kind[kBlock];
  const int G = 1 << a.glog, NG = kBlock >> a.glog;
  const int g = threadIdx.x >> a.glog, gl = threadIdx.x & (G - 1);
  const int col = ((int)blockIdx.y * G + gl) * VEC;
  const bool live = col < a.D;
  const uint64_t s64 = ((uint64_t)blockIdx.x * NG + g) * (uint64_t)a.per_group;
  const uint32_t s = (uint32_t)min(s64, (uint64_t)a.n);
  const uint32_t e = (uint32_t)min(s64 + a.per_group, (uint64_t)a.n);
  int kind = 0;
  A acc[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) acc[j] = (A)0;
  if (s < e) {
    const uint32_t none = 0xffffffffu;
    const uint32_t prev = s > 0 ? a.keys[s - 1] : none;
    const uint32_t next = e < a.n ? a.keys[e] : none;
    uint32_t cur = a.keys[s];
    bool from_prev = cur == prev;
    for (uint32_t i = s; i < e; i += U) {
      uint32_t k[U];
      Pack<T, VEC> row[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        k[u] = i + u < e ? a.keys[i + u] : none;
        if (k[u] < a.nkeys && live)
          row[u] = *(const Pack<T, VEC> *)(grad + (int64_t)a.toks[i + u] * a.D + col);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i + u >= e || cur >= a.nkeys) break;
        if (k[u] != cur) {  // the run ends inside this group's range
          if (from_prev) {
            kind |= kHasHead;
#pragma unroll
            for (int j = 0; j < VEC; ++j) s_head[threadIdx.x * VEC + j] = acc[j];
          } else if (live) {
            embed_store<T, VEC>(out, a.D, cur, col, acc, scale);
          }
          cur = k[u];
          from_prev = false;
#pragma unroll
          for (int j = 0; j < VEC; ++j) acc[j] = (A)0;
          if (cur >= a.nkeys) break;  // tokens without a row: nothing behind them either
        }
        if (live) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) acc[j] += to_wide(row[u].v[j]);
        }
      }
    }
    if (cur < a.nkeys) {
      const bool on = next == cur;
      if (from_prev) {
        kind |= kHasHead | (on ? kThrough : 0);
#pragma unroll
        for (int j = 0; j < VEC; ++j) s_head[threadIdx.x * VEC + j] = acc[j];
      } else if (on) {
        kind |= kHasTail;
#pragma unroll
        for (int j = 0; j < VEC; ++j) s_tail[threadIdx.x * VEC + j] = acc[j];
      } else if (live) {
        embed_store<T, VEC>(out, a.D, cur, col, acc, scale);
      }
    }
  }
  if (gl == 0) s_kind[g] = kind;
  __syncthreads();
  const int64_t wcol = (int64_t)gridDim.y * G * VEC;  // a partial's channels
  if (kind & kHasTail) {  // the run's owner: add the heads behind it
    int q = g + 1;
    bool open = true;
    for (; q < NG && open; ++q) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] += s_head[((q << a.glog) + gl) * VEC + j];
      open = s_kind[q] & kThrough;
    }
    if (!open) {
      if (live) embed_store<T, VEC>(out, a.D, a.keys[e - 1], col, acc, scale);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) tail[(int64_t)blockIdx.x * wcol + col + j] = acc[j];
    }
  }
  if (g == 0) {
    int f = 0;
    if (kind & kHasHead) {  // the run that began in an earlier workgroup
      f = kHasHead;
      A h[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) h[j] = s_head[threadIdx.x * VEC + j];
      bool open = kind & kThrough;
      for (int q = 1; q < NG && open; ++q) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) h[j] += s_head[((q << a.glog) + gl) * VEC + j];
        open = s_kind[q] & kThrough;
      }
      if (open) f |= kThrough;
#pragma unroll
      for (int j = 0; j < VEC; ++j) head[(int64_t)blockIdx.x * wcol + col + j] = h[j];
    }
    // a run that is open at the end of the workgroup began in it unless it runs through
    for (int q = NG - 1; q >= 0; --q) {
      if (s_kind[q] & kHasTail) f |= kHasTail;
      if (!(s_kind[q] & kThrough)) break;
    }
    if (gl == 0 && blockIdx.y == 0) a.flags[blockIdx.x] = f;
  }
}

// The runs that cross a workgroup's border: the workgroup in which such a run begins adds up its
// own part and the heads of the workgroups behind it, split over the groups of lanes in a fixed
// order.
template <typename T, int VEC>
__global__ __launch_bounds__(kBlock) void kd_embed_join(SegArgs a, int nwg,
                                                        typename Wide<T>::type scale,
                                                        const typename Wide<T>::type *__restrict__ head,
                                                        const typename Wide<T>::type *__restrict__ tail,
                                                        T *__restrict__ out) {
  using A = typename Wide<T>::type;
  const int w = blockIdx.x;
  if (!(a.flags[w] & kHasTail)) return;
  __shared__ int s_end;
  __shared__ A s_sum[kBlock * VEC];
  const int G = 1 << a.glog, NG = kBlock >> a.glog;
  const int g = threadIdx.x >> a.glog, gl = threadIdx.x & (G - 1);
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
  const int col = ((int)blockIdx.y * G + gl) * VEC;
  const int64_t wcol = (int64_t)gridDim.y * G * VEC;
  A acc[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) acc[j] = g == 0 ? tail[(int64_t)w * wcol + col + j] : (A)0;
  for (int q = w + 1 + g; q <= last; q += NG) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] += head[(int64_t)q * wcol + col + j];
  }
#pragma unroll
  for (int j = 0; j < VEC; ++j) s_sum[threadIdx.x * VEC + j] = acc[j];
  __syncthreads();
  if (g == 0 && col < a.D) {
    for (int q = 1; q < NG; ++q) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] += s_sum[((q << a.glog) + gl) * VEC + j];
    }
    const uint64_t end = (uint64_t)(w + 1) * NG * a.per_group;  // <= n: a run goes on behind it
    embed_store<T, VEC>(out, a.D, a.keys[end - 1], col, acc, scale);
  }
}

// ------------------------------------------------------------------------------------------------
// host
// ------------------------------------------------------------------------------------------------
struct EmbedPlan {
  int vec, glog, gy, per_group, nwg, ntile, passes, bits;
  size_t pairs, hist, part, flags, total;  // workspace parts in bytes
};

static size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

static EmbedPlan embed_plan(int64_t n, int64_t nkeys, int D, int esize, bool vec) {
  EmbedPlan p;
  p.vec = vec ? 16 / esize : 1;
  const int cols = D / p.vec;
  p.glog = 0;
  while (p.glog < 6 && (1 << p.glog) < cols) ++p.glog;
  p.gy = (cols + (1 << p.glog) - 1) >> p.glog;
  const int ng = kBlock >> p.glog;
  // tokens per group: long walks read less at the borders, short ones fill the chip
  p.per_group = 64;
  while (p.per_group > 8 && (n + (int64_t)ng * p.per_group - 1) / ((int64_t)ng * p.per_group) < 2048)
    p.per_group >>= 1;
  p.nwg = (int)((n + (int64_t)ng * p.per_group - 1) / ((int64_t)ng * p.per_group));
  p.ntile = (int)((n + kSortTile - 1) / kSortTile);
  int kb = 1;
  while (kb < 32 && (nkeys >> kb) != 0) ++kb;  // keys 0 .. nkeys
  p.passes = (kb + 7) / 8;
  p.bits = (kb + p.passes - 1) / p.passes;
  const int asize = esize == 8 ? 8 : 4;
  p.pairs = up256(4 * (size_t)n);
  p.hist = up256(4 * (size_t)kDigits * (size_t)p.ntile + 4 * kDigits);
  // the workspace query does not know the pointers' alignment: the larger of both layouts
  p.part = up256((size_t)p.nwg * (size_t)p.gy * (size_t)(p.vec << p.glog) * (size_t)asize);
  p.flags = up256(4 * (size_t)p.nwg);
  p.total = 4 * p.pairs + p.hist + 2 * p.part + p.flags;
  return p;
}

static size_t embed_workspace(int64_t n, int64_t nkeys, int D, int esize) {
  size_t t = embed_plan(n, nkeys, D, esize, false).total;
  if (D % (16 / esize) == 0) t = std::max(t, embed_plan(n, nkeys, D, esize, true).total);
  return t;
}

static bool embed_aligned(const void *p) { return ((uintptr_t)p & 15u) == 0; }

static int embed_check(int64_t n, int64_t batch, int64_t rows, int D, const void *index,
                       const void *x, const void *y) {
  KD_CHECK_ARG(n >= 0 && n < ((int64_t)1 << 31), "surface_embedding: need 0 <= indices < 2^31");
  KD_CHECK_ARG(batch >= 1 && rows >= 0 && rows < ((int64_t)1 << 31) &&
                   batch * rows < ((int64_t)1 << 31),
               "surface_embedding: need batch >= 1 and batch * rows < 2^31");
  KD_CHECK_ARG(n % batch == 0, "surface_embedding: the indices do not split over the batch");
  KD_CHECK_ARG(D >= 0 && D <= kMaxChannels, "surface_embedding: need 0 <= channels <= 2^20");
  KD_CHECK_ARG(n == 0 || index, "surface_embedding: index is NULL");
  KD_CHECK_ARG(n == 0 || D == 0 || x, "surface_embedding: NULL input");
  (void)y;
  return KD_OK;
}

template <typename T>
static int embed_forward(int64_t n, int64_t batch, int64_t rows, int D, const int64_t *index,
                         const T *table, double scale, T *out, hipStream_t stream) {
  const int rc = embed_check(n, batch, rows, D, index, out, nullptr);
  if (rc != KD_OK) return rc;
  KD_CHECK_ARG(rows == 0 || D == 0 || n == 0 || table, "surface_embedding: embeddings is NULL");
  if (n == 0 || D == 0) return KD_OK;
  using A = typename Wide<T>::type;
  constexpr int V = 16 / (int)sizeof(T);
  const bool vec = D % V == 0 && embed_aligned(table) && embed_aligned(out);
  const int vpr = vec ? D / V : D;
  const int rpb = std::max(1, kBlock * 4 / vpr);
  const unsigned grid = (unsigned)((n + rpb - 1) / rpb);
  const uint32_t pb = batch > 1 ? (uint32_t)(n / batch) : 0u;
  {
    ProfScope prof(K_EMBED_FWD, stream);
    if (vec)
      hipLaunchKernelGGL((kd_embed_gather<T, V>), dim3(grid), dim3(kBlock), 0, stream, n, pb, rows,
                         D, rpb, index, table, (A)scale, out);
    else
      hipLaunchKernelGGL((kd_embed_gather<T, 1>), dim3(grid), dim3(kBlock), 0, stream, n, pb, rows,
                         D, rpb, index, table, (A)scale, out);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(KD_ERR_LAUNCH, "surface_embedding: %s", hipGetErrorString(e));
  return KD_OK;
}

template <typename T, int VEC>
static void embed_segments(const EmbedPlan &p, const SegArgs &a, const T *grad,
                           typename Wide<T>::type scale, T *out, void *head, void *tail,
                           hipStream_t stream) {
  using A = typename Wide<T>::type;
  const dim3 grid((unsigned)p.nwg, (unsigned)p.gy);
  hipLaunchKernelGGL((kd_embed_segments<T, VEC>), grid, dim3(kBlock), 0, stream, a, grad, scale,
                     out, (A *)head, (A *)tail);
  if (p.nwg > 1)
    hipLaunchKernelGGL((kd_embed_join<T, VEC>), grid, dim3(kBlock), 0, stream, a, p.nwg, scale,
                       (const A *)head, (const A *)tail, out);
}

template <typename T>
static int embed_backward(int64_t n, int64_t batch, int64_t rows, int D, const int64_t *index,
                          const T *grad, double scale, T *out, void *ws, size_t wsb,
                          hipStream_t stream) {
  const int rc = embed_check(n, batch, rows, D, index, grad, nullptr);
  if (rc != KD_OK) return rc;
  const int64_t nkeys = batch * rows, nout = nkeys * D;
  if (nout == 0) return KD_OK;
  KD_CHECK_ARG(out, "surface_embedding: grad_embeddings is NULL");
  using A = typename Wide<T>::type;
  constexpr int V = 16 / (int)sizeof(T);
  const bool vec = D % V == 0 && embed_aligned(grad) && embed_aligned(out);
  const EmbedPlan p = embed_plan(n, nkeys, D, (int)sizeof(T), vec);
  if (n > 0 && (wsb < p.total || !ws))
    return set_error(KD_ERR_WORKSPACE, "workspace too small: %zu < %zu", wsb, p.total);
  ProfScope prof(K_EMBED_BWD, stream);
  {  // rows that no token names
    const int64_t words = (nout * (int64_t)sizeof(T)) / 4;
    const bool even = (nout * (int64_t)sizeof(T)) % 4 == 0 && ((uintptr_t)out & 3u) == 0;
    const int64_t m = even ? words : nout;
    const unsigned blocks = (unsigned)std::min<int64_t>((m + kBlock - 1) / kBlock, 4096);
    if (even)
      hipLaunchKernelGGL(kd_embed_fill<uint32_t>, dim3(blocks), dim3(kBlock), 0, stream, m,
                         (uint32_t *)out);
    else
      hipLaunchKernelGGL(kd_embed_fill<uint16_t>, dim3(blocks), dim3(kBlock), 0, stream, m,
                         (uint16_t *)out);
  }
  if (n > 0) {
    char *c = (char *)ws;
    uint32_t *buf[4];
    for (int i = 0; i < 4; ++i) buf[i] = (uint32_t *)(c + (size_t)i * p.pairs);
    c += 4 * p.pairs;
    uint32_t *hist = (uint32_t *)c, *totals = hist + (size_t)kDigits * p.ntile;
    c += p.hist;
    void *head = c, *tail = c + p.part;
    int *flags = (int *)(c + 2 * p.part);
    SortKeys s;
    s.n = (uint32_t)n;
    s.per_batch = batch > 1 ? (uint32_t)(n / batch) : 0u;
    s.nkeys = (uint32_t)nkeys;
    s.rows = rows;
    s.keys = s.toks = nullptr;
    s.index = index;
    const uint32_t mask = (1u << p.bits) - 1u;
    int cur = 0;
    for (int q = 0; q < p.passes; ++q) {
      const int shift = q * p.bits;
      hipLaunchKernelGGL(kd_embed_hist, dim3(p.ntile), dim3(kBlock), 0, stream, s, shift, mask,
                         p.ntile, hist);
      hipLaunchKernelGGL(kd_embed_scan, dim3(mask + 1), dim3(kBlock), 0, stream, p.ntile, hist,
                         totals);
      hipLaunchKernelGGL(kd_embed_scatter, dim3(p.ntile), dim3(kBlock), 0, stream, s, shift, p.bits,
                         p.ntile, hist, totals, buf[2 * cur], buf[2 * cur + 1]);
      s.index = nullptr;
      s.keys = buf[2 * cur];
      s.toks = buf[2 * cur + 1];
      cur ^= 1;
    }
    SegArgs a;
    a.n = (uint32_t)n;
    a.nkeys = (uint32_t)nkeys;
    a.D = D;
    a.glog = p.glog;
    a.per_group = p.per_group;
    a.keys = s.keys;
    a.toks = s.toks;
    a.flags = flags;
    if (vec)
      embed_segments<T, V>(p, a, grad, (A)scale, out, head, tail, stream);
    else
      embed_segments<T, 1>(p, a, grad, (A)scale, out, head, tail, stream);
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
      rows >= ((int64_t)1 << 31) || batch * rows >= ((int64_t)1 << 31) || channels < 1 ||
      channels > kMaxChannels || (element_size != 2 && element_size != 4 && element_size != 8))
    return 0;
  return embed_workspace(num_indices, batch * rows, channels, element_size);
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
