// kd_xent.hpp -- surface_cross_entropy: softmax cross entropy of pixel features against every row
// of a table of embeddings, without keeping the logits, and both gradients.
//
//   z_iv = scale x_i . e_v,   loss_i = log sum_v exp z_iv - z_iy,   y = labels[i]
// over the rows i whose label names a row of the table (0 <= y < V); the others take no part.
// Everything is written with the label's own term left out of the sums:
//   L'_i = log sum_{v != y} exp z_iv,   w_i = 1 - p_iy = sigmoid(L'_i - z_iy)
//   loss_i = softplus(L'_i - z_iy)
//   dX_i = g_i scale w_i (m_i - e_y),   m_i = sum_{v != y} exp(z_iv - L'_i) e_v
//   dE_v = scale sum_i g_i q_iv x_i,    q_iv = p_iv (v != y),  -w_i (v = y)
// so that nothing cancels where p_iy is next to 1 (a trained network), in the loss or in p - 1.
//
// Forward: rows with a label are listed (in order) and packed with the table into the matrix
// instructions' operand layout; kd_xent_rows holds a block of rows in registers and walks the
// table once: 32 x 32 logits at a time, a running maximum and sum (32 bits), and, if dX is wanted,
// the weighted sum of the table's rows (32 bits) -- the logits never leave registers.  When there
// are few rows the table is split over workgroups and kd_xent_combine joins the parts.
// Backward: kd_xent_table holds a block of table rows and walks the pixels; the logits are computed
// again from the packed operands with the saved log sums, split over the pixels when the table is
// small and joined in a fixed order.  No atomics on values: results do not depend on timing.
//
// 16-bit data multiply exactly into 32-bit sums.  The probabilities enter their product with the
// table (or the features) rounded to the data's type, at most 2^-8 (bf16) or 2^-11 (fp16, scaled so
// that small ones stay normal) of each term, like the operands themselves (up to 32 channels and
// for few rows in two parts, see walk_parts); the sums L' use the unrounded values, the weights of dX's mean add up to 1
// as they are rounded (see walk_norm).  What dE keeps of it, with more rows than kFewRows: where
// thousands of pixels have the same probabilities to 2^-9 (an untrained table, logits of 1e-3), a part that
// all features have in common is off by up to 2^-9 of it.  32-bit data are split into three bf16 parts (8 + 8 + 8 bits, the whole significand) and multiplied as the six products above 2^-24:
// the fp32 matrix instructions run at 1/16 of the bf16 rate, six bf16 products at 1/6.
// Losses are 32-bit numbers for every type, gradients of the data's type, rounded once.
#pragma once

#include "kd_capi.hpp"
#include "kd_common.hpp"
#include "kd_float16.hpp"

#include <cfloat>

#include <algorithm>
#include <type_traits>

namespace kd {
namespace xent {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef half_t half8 __attribute__((ext_vector_type(8)));
typedef bfloat_t bfloat8 __attribute__((ext_vector_type(8)));

// How data of type T are multiplied: the operand type H, its 8-vector, the number of parts
// (planes), and the power of two by which probabilities are scaled in the products.
template <typename T>
struct Form;
template <>
struct Form<bfloat_t> {
  using H = bfloat_t;
  using H8 = bfloat8;
  static constexpr int np = 1;
  static constexpr float shift = 0.f, slack = 8.f, shift_table = 0.f;
};
template <>
struct Form<half_t> {
  using H = half_t;
  using H8 = half8;
  static constexpr int np = 1;
  // exp2(z - max + shift) <= 2^(shift + slack) stays below 65504
  static constexpr float shift = 10.f, slack = 5.f, shift_table = 14.f;
};
template <>
struct Form<float> {
  using H = bfloat_t;
  using H8 = bfloat8;
  static constexpr int np = 3;
  static constexpr float shift = 0.f, slack = 8.f, shift_table = 0.f;
};

__device__ __forceinline__ f32x16 mfma(half8 a, half8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma(bfloat8 a, bfloat8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ f32x4 mfma16(half8 a, half8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(bfloat8 a, bfloat8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// x as three bf16, each the nearest to what is left (exact: what the first two leave, at most 2^-18 x,
// has 8 bits).  Parts by truncation would all have the sign of x, and so would the three small
// products that are not formed: 4e-8 of every logit, a gradient of the table 8e-7 off where rounded
// parts leave 4e-9 (60,000 pixels, 59 rows, 3 channels, scale 24).
__device__ __forceinline__ void split3(float x, uint16_t &a, uint16_t &b, uint16_t &c) {
  const uint32_t cut = __float_as_uint(x) & 0xffff0000u;  // (the nearest to these is infinite)
  const bfloat_t h =
      fabsf(x) < 0x1.ffp127f ? (bfloat_t)x : __builtin_bit_cast(bfloat_t, (uint16_t)(cut >> 16));
  const float r = x - (float)h;
  const bfloat_t m = (bfloat_t)r;
  a = __builtin_bit_cast(uint16_t, h);
  b = __builtin_bit_cast(uint16_t, m);
  c = __builtin_bit_cast(uint16_t, (bfloat_t)(r - (float)m));
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kSlots = 64, kSlotPad = 16;  // maxima of the table, 64 bytes apart
constexpr int kRowPad = 256;  // packed rows are padded with zeros to a multiple of this
constexpr int kMapChunk = 2048;   // pixels listed at a time
constexpr int kListChunks = 4;    // up to so many chunks one workgroup lists them all
constexpr int kSumChunks = 4096;  // up to so many chunks a workgroup adds up the counts before its own

// The work of one call.  Packed operands of a matrix M (rows padded to kRowPad, channels to DP),
// in tiles of 32 rows, each tile NP planes, 16 bytes a lane:
//   straight   [tile][plane][k step of 16 channels][lane][8] = M[lane % 32][16 step + 8 (lane / 32) + j]
//   transposed [tile][plane][row half s][32 channels t][lane][8] =
//       M[16 s + 8 (j / 4) + 4 (lane / 32) + j % 4][32 t + lane % 32]
// The transposed order of rows is the order in which a 32 x 32 product leaves its result in a
// lane's registers, so a block of probabilities goes into the next product as it stands.
struct Args {
  int64_t n, npad;  // pixels, padded
  int V, vpad, D, dp;
  float c2, c2l;    // |scale| log2(e), and what its rounding left
  float scale;
  int reduction;    // 0 none, 1 mean, 2 sum
  // state kept from forward to backward
  int *count;       // pixels with a label
  int *rowid, *lab; // listed pixel -> pixel, its label
  int *far;         // 1: logits beyond kFar
  float *lse, *rl;  // exponent of a probability but its logit, factor of the exponential
  float *w;         // its complement negated (scaled)
  float *xn;        // squared sizes of the pixels' features
  uint32_t *emax, *xmax;  // the largest squared sizes of rows and pixels (their bits), kSlots of each
  uint32_t *ticket; // workgroups that have added up their losses
  uint16_t *xs, *xt, *es;
  float *raw;       // (n, D): w (m - e_y)
  // scratch
  int *blk;
  uint16_t *et;
  float *pm, *pl, *pz, *po;  // a part's maximum, sum, label's logit (or -inf), weighted sum
  float *pq;                 // and the sum of the probabilities as they enter the weighted sum
  float *lrow;
  double *part;
  float *grow, *gfac, *pe;  // a pixel's incoming gradient, and times its factor
  uint32_t *gmax;
};

// ------------------------------------------------------------------------------------------------
// listing the pixels with a label
// ------------------------------------------------------------------------------------------------
static __global__ __launch_bounds__(kBlock) void kd_xent_count(int64_t n, int64_t V,
                                                               const int64_t *__restrict__ labels,
                                                               int *__restrict__ blk) {
  __shared__ int s_c[kBlock / kWave];
  const int64_t b = (int64_t)blockIdx.x * kMapChunk;
  int c = 0;
#pragma unroll
  for (int k = 0; k < kMapChunk / kBlock; ++k) {
    const int64_t i = b + k * kBlock + threadIdx.x;
    const int64_t y = i < n ? labels[i] : -1;
    c += __popcll(__ballot(y >= 0 && y < V));
  }
  if ((threadIdx.x & 63) == 0) s_c[threadIdx.x >> 6] = c;
  __syncthreads();
  if (threadIdx.x == 0) blk[blockIdx.x] = s_c[0] + s_c[1] + s_c[2] + s_c[3];
}

// The sum of the threads' values, in every thread.
__device__ __forceinline__ int wg_total(int x, int *s_x) {
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) x += __shfl_xor(x, s);
  if ((threadIdx.x & 63) == 0) s_x[threadIdx.x >> 6] = x;
  __syncthreads();
  const int t = s_x[0] + s_x[1] + s_x[2] + s_x[3];
  __syncthreads();
  return t;
}

// One workgroup: the chunks' counts become offsets (for more chunks than a workgroup adds up itself).
static __global__ __launch_bounds__(kBlock) void kd_xent_scan(int nblk, int *__restrict__ blk) {
  __shared__ int s_w[kBlock / kWave];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int run = 0;
  for (int b = 0; b < nblk; b += kBlock) {
    const int i = b + threadIdx.x;
    const int c = i < nblk ? blk[i] : 0;
    int x = c;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const int y = __shfl_up(x, d);
      if (lane >= d) x += y;
    }
    if (lane == 63) s_w[w] = x;
    __syncthreads();
    int off = 0, tot = 0;
#pragma unroll
    for (int k = 0; k < kBlock / kWave; ++k) {
      if (k < w) off += s_w[k];
      tot += s_w[k];
    }
    __syncthreads();
    if (i < nblk) blk[i] = run + off + x - c;
    run += tot;
  }
}

// The pixels without a label cost a walk as much as the others, so the walks take a list (in order) of
// those with one; counts and list read the labels twice: 2,097,152 in 6.9 and 7.7 us, 2.4 TB/s
// (averages of six calls, as all times of one kernel here; cards and their
// clocks differ by up to 6 %).
// Lists the pixels of `chunks` chunks a workgroup: blk holds the chunks' counts, or their offsets
// (scanned), or is not needed (one workgroup lists all).  Losses of pixels without a label are 0.
static __global__ __launch_bounds__(kBlock) void kd_xent_map(Args a, int chunks, bool scanned,
                                                             const int64_t *__restrict__ labels,
                                                             float *__restrict__ loss) {
  __shared__ int s_c[4];
  int run = 0;
  if (chunks == 1 && scanned) {
    run = a.blk[blockIdx.x];
  } else if (chunks == 1) {
    int c = 0;
    for (int k = threadIdx.x; k < (int)blockIdx.x; k += kBlock) c += a.blk[k];
    run = wg_total(c, s_c);
  }
  for (int q = 0; q < chunks; ++q) {
    const int64_t b = ((int64_t)blockIdx.x * chunks + q) * kMapChunk;
    if (b >= a.n) break;
    int64_t y[kMapChunk / kBlock];
#pragma unroll
    for (int k = 0; k < kMapChunk / kBlock; ++k) {
      const int64_t i = b + k * kBlock + threadIdx.x;
      y[k] = i < a.n ? labels[i] : -1;
    }
#pragma unroll
    for (int k = 0; k < kMapChunk / kBlock; ++k) {
      const int64_t i = b + k * kBlock + threadIdx.x;
      int total;
      const int p = wg_compact(y[k] >= 0 && y[k] < a.V, s_c, total);
      if (p >= 0) {
        a.rowid[run + p] = (int)i;
        a.lab[run + p] = (int)y[k];
      } else if (a.reduction == 0 && i < a.n) {
        loss[i] = 0.f;
      }
      run += total;
    }
  }
  if (blockIdx.x == gridDim.x - 1) {
    if (threadIdx.x < kSlots) a.emax[threadIdx.x * kSlotPad] = a.xmax[threadIdx.x * kSlotPad] = 0u;
    if (threadIdx.x == 0) {
      *a.count = run;
      *a.far = 0;
      *a.ticket = 0u;
    }
  }
}

// ------------------------------------------------------------------------------------------------
// packing
// ------------------------------------------------------------------------------------------------
// A tile of 32 rows goes through LDS, 16 bytes a lane in and out.  Once per call, so that the walks,
// which read every tile hundreds of times, copy it as it is.  Bound by bytes: 1,054,304 pixels and 50,000
// rows of 128 channels in bf16 125 us, 4.5 TB/s.
template <typename T, int DP>
__global__ __launch_bounds__(kBlock) void kd_xent_pack(Args a, int xtiles,
                                                       const T *__restrict__ features,
                                                       const T *__restrict__ table) {
  using F = Form<T>;
  constexpr int V = 16 / sizeof(T);
  constexpr int kPitch = DP + V;  // rows 16 bytes apart over the banks
  constexpr int kLanes = DP / V < kWave ? DP / V : kWave;  // that hold a row
  __shared__ __align__(16) T s_m[32 * kPitch];
  __shared__ uint32_t s_top[kBlock / kWave];
  uint32_t top = 0;
  const int64_t bid = block_id();
  const bool is_x = bid < xtiles;
  const int64_t tile = is_x ? bid : bid - xtiles;
  if (tile >= a.vpad / 32 && !is_x) return;
  const int count = *a.count;
  const int64_t r0 = tile * 32;
  if (is_x && r0 >= ((int64_t)count + kRowPad - 1) / kRowPad * kRowPad) return;
  const bool flip = is_x && a.scale < 0.f;
#pragma unroll
  for (int q = 0; q * kBlock < 32 * DP / V; ++q) {
    const int e = q * kBlock + threadIdx.x, r = e / (DP / V), d = e % (DP / V) * V;
    if (r >= 32) break;  // (whole waves)
    const int64_t i = r0 + r;
    Pack<T, V> x;
#pragma unroll
    for (int j = 0; j < V; ++j) x.v[j] = (T)0.f;
    if (d < a.D) {
      if (is_x) {
        if (i < count) x = load_pack<T, V>(features + (int64_t)a.rowid[i] * a.D + d, a.D - d);
      } else if (i < a.V) {
        x = load_pack<T, V>(table + i * a.D + d, a.D - d);
      }
    }
    // the row's squared size (DP / V lanes hold it), no less than it is where the squares leave the range
    float size = 0x1p-100f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      size = fmaf((float)x.v[j], (float)x.v[j], size);
      if (flip) x.v[j] = (T)(-(float)x.v[j]);
    }
    *(uint4 *)&s_m[r * kPitch + d] = __builtin_bit_cast(uint4, x);
#pragma unroll
    for (int k = kLanes / 2; k >= 1; k >>= 1) size += __shfl_xor(size, k);
    if (is_x && d == 0) a.xn[i] = size;
    top = max(top, __float_as_uint(size));
  }
#pragma unroll
  for (int k = 32; k >= kLanes; k >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, k));
  if ((threadIdx.x & 63) == 0) s_top[threadIdx.x >> 6] = top;
  if (is_x && threadIdx.x < 32 && r0 + threadIdx.x >= count) {
    a.lab[r0 + threadIdx.x] = -1;
    a.lse[r0 + threadIdx.x] = -INFINITY;  // its probabilities are 0
    a.rl[r0 + threadIdx.x] = 0.f;
    a.w[r0 + threadIdx.x] = 0.f;
  }
  __syncthreads();
  if (threadIdx.x == 0)  // spread over the slots: they would queue at one address
    atomicMax((is_x ? a.xmax : a.emax) + tile % kSlots * kSlotPad,
              max(max(s_top[0], s_top[1]), max(s_top[2], s_top[3])));
  constexpr int kGroups = 32 * DP / 8;  // 16-byte groups per plane and layout
  uint16_t *straight = (is_x ? a.xs : a.es) + tile * F::np * 32 * DP;
  uint16_t *transposed = is_x ? a.xt : a.et;
  auto put = [&](uint16_t *to, int g, const T *x) {
    Pack<uint16_t, 8> o[F::np];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (F::np == 1)
        o[0].v[j] = __builtin_bit_cast(uint16_t, x[j]);
      else
        split3(x[j], o[0].v[j], o[1].v[j], o[2].v[j]);
    }
#pragma unroll
    for (int p = 0; p < F::np; ++p)
      *(uint4 *)(to + (int64_t)p * 32 * DP + g * 8) = __builtin_bit_cast(uint4, o[p]);
  };
  for (int g = threadIdx.x; g < kGroups; g += kBlock) {
    const int lane = g & 63, r = lane & 31, d = 16 * (g >> 6) + 8 * (lane >> 5);
    T x[8];
    *(uint4 *)x = *(const uint4 *)&s_m[r * kPitch + d];
    if constexpr (sizeof(T) == 4) *(uint4 *)(x + 4) = *(const uint4 *)&s_m[r * kPitch + d + 4];
    put(straight, g, x);
  }
  if (!transposed) return;
  transposed += tile * F::np * 32 * DP;
  for (int g = threadIdx.x; g < kGroups; g += kBlock) {
    constexpr int kT = DP / 32;
    const int lane = g & 63, blkid = g >> 6;
    const int r = 16 * (blkid / kT) + 4 * (lane >> 5), d = 32 * (blkid % kT) + (lane & 31);
    T x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = s_m[(r + 8 * (j >> 2) + (j & 3)) * kPitch + d];
    put(transposed, g, x);
  }
}

// ------------------------------------------------------------------------------------------------
// shared pieces of the two walks
// ------------------------------------------------------------------------------------------------
// acc += the i-th of the planes' products of a . b, the large one last.  SWAP: the order that the same
// product has with a and b exchanged, so that the logits of both walks have the same roundings.
template <int NP, bool SWAP = false, typename H8>
__device__ __forceinline__ f32x16 product(int i, const H8 *a, const H8 *b, f32x16 c) {
  if constexpr (NP == 1) {
    return mfma(a[0], b[0], c);
  } else {
    constexpr int ka[6] = {0, 2, 1, 0, 1, 0}, kb[6] = {2, 0, 1, 1, 0, 0};
    return mfma(a[SWAP ? kb[i] : ka[i]], b[SWAP ? ka[i] : kb[i]], c);
  }
}

// log2 of a term: the logit times the factor, in two parts for 32-bit data (a factor off by 2^-25
// would be a bias that no averaging takes out), and an offset (first, where the sum becomes small).
template <typename T>
__device__ __forceinline__ float exponent(float s, float c2, float c2l, float offset) {
  const float e = fmaf(s, c2, offset);
  if constexpr (sizeof(T) == 4) return fmaf(s, c2l, e);
  return e;
}

// Logits that may be larger than this (in log2, by the largest sizes of the pixels and the rows) take
// walks of their own, tile by tile, in which a term's log2 is the logit times the factor, rounded, the
// same number in both walks.  In the others that product is not rounded: an offset of its size is off by
// half a step of it, which an exponential turns into 2^-25 of the logit, relative.  In 16 bits, whose
// other walks hold the offset log2 of the sum in one number, that is 2^-15 here for fp16 and 2^-13 for
// bf16, a sixteenth of half a step each; without a limit all types' gradients were 0.8 % off at logits of
// 8e4, wrong at 1e7 and not finite at 1e9.  With 32-bit data the offset is two numbers, a whole one (exact
// up to 2^24) and a factor of the exponential.
// Measured (loss; loss and both gradients), bounded / with the running maximum / large logits: bf16, 64
// channels, 263,576 pixels x 50,000 rows 2.4 / 2.7 / 3.4 ms; 7.1 / 7.7 / 11.3 ms; 256 channels, 131,788 x
// 10,000 0.65 / 0.68 / 0.72; 3.2 / 3.4 / 4.8; fp16, 64 channels, 131,072 x 10,000 0.40 / 0.40 / 0.47; 0.95 /
// 0.92 / 1.42; fp32, 64 channels, 131,712 x 10,000 0.87 / 0.89 / 0.97; 3.52 / 3.65 / 3.54.
template <typename T>
constexpr float kFar = std::is_same_v<T, float> ? 0x1p22f : std::is_same_v<T, half_t> ? 0x1p10f : 0x1p12f;

// the largest of a kind of sizes, squared (NaN if there is one: its bits are above infinity's)
__device__ __forceinline__ float largest(const uint32_t *slots) {
  uint32_t big = slots[(threadIdx.x & 63) * kSlotPad];
#pragma unroll
  for (int k = 32; k >= 1; k >>= 1) big = max(big, (uint32_t)__shfl_xor((int)big, k));
  return __uint_as_float(big);
}

// the upper halves of two words as one
__device__ __forceinline__ uint32_t upper2(uint32_t lo, uint32_t hi) {
  return __builtin_amdgcn_perm(hi, lo, 0x07060302u);
}

// Two probabilities of a lane as elements 2 i and 2 i + 1 of an operand (its words, part by part).
template <typename T, int PP>
__device__ __forceinline__ void pack_pair(float p0, float p1, int i, uint4 *o) {
  using H = typename Form<T>::H;
  if constexpr (Form<T>::np == 1) {
    typedef H h2 __attribute__((ext_vector_type(2)));
    h2 v;
    v[0] = (H)p0;
    v[1] = (H)p1;
    ((uint32_t *)o)[i] = __builtin_bit_cast(uint32_t, v);
    if constexpr (PP == 2) {
      h2 r;
      r[0] = (H)(p0 - (float)v[0]);
      r[1] = (H)(p1 - (float)v[1]);
      ((uint32_t *)&o[1])[i] = __builtin_bit_cast(uint32_t, r);
    }
  } else {
    // (by truncation, which is cheaper: the other operand's parts are rounded, so what is left out has
    // either sign all the same)
    uint32_t u[3][2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float p = k ? p1 : p0;
      const uint32_t a = __float_as_uint(p);
      const float r = p - __uint_as_float(a & 0xffff0000u);
      const uint32_t b = __float_as_uint(r);
      u[0][k] = a;
      u[1][k] = b;
      u[2][k] = __float_as_uint(r - __uint_as_float(b & 0xffff0000u));
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) ((uint32_t *)&o[k])[i] = upper2(u[k][0], u[k][1]);
  }
}

// How a walk is laid out (KIND 0: over the table, loss only; 1: over the table with dX; 2: over the
// pixels, dE; 3: the same for few rows, see walk_parts), for np planes and dp channels.
// Blocks of 32 rows that a wave holds.  Every operand read from LDS feeds one product per block; with
// one block a product, 32 clocks on each of four SIMDs, takes all that LDS delivers (4 x 1 KiB), so
// 16-bit data take two where two waves a SIMD have the registers: losses at 256 channels of 527,000
// pixels and 10,000 rows 2.43 -> 2.07 ms (33,000 and 2,000: 47 and 48 us).  Not the sums at 128
// channels, where two blocks leave one wave a SIMD: dE of 527,000 pixels 2.98 -> 2.87 ms, but of 33,000
// pixels and 2,000 rows 55 -> 65 us, dX of 132,000 0.64 -> 0.69 ms.
constexpr int walk_blocks(int np, int dp, int kind) {
  return np == 1 && kind != 3 && (dp <= 64 || kind == 0) ? 2 : 1;
}
// Waves per SIMD: one where the held operands, the sums and the blocks of logits need more than 256
// registers.
constexpr int walk_waves(int np, int dp, int kind) {
  return (np == 1 ? dp == 256 && kind > 0 : dp >= (kind > 0 ? 128 : 256)) ? 1 : 2;
}
// Into how many column ranges the sums are cut, over workgroups that each form the logits: two where
// the operands of all columns would not fit LDS twice.
constexpr int walk_columns(int np, int dp, int kind) {
  return np == 3 && dp == 256 && kind > 0 ? 2 : 1;
}
// Parts of a probability in its product with the table's rows or the pixels' features.  Rounded once
// to bf16 or fp16 (half a step, 2^-8 or 2^-11 of the probability, which averages out over rows that
// differ), the error stays whole where few channels make the rows alike: one channel and tens of rows
// had gradients 2e-3 to 4e-3 off in bf16, where one rounding of the result is 1.7e-3.  Up to 32
// channels, where the exponentials take longer than the products, a second part carries what the first
// left out.
// Tables of few rows too, for dE: an error that is the same for many pixels stays whole there, as each row
// has many of them (100,000 pixels that are alike, 8 rows, bf16: 7.7e-2 of the gradient, 1.6e-3 in two
// parts), and the time of such a call is in the pixels' bytes: 500,000 pixels of 64 channels, both
// gradients, 10 rows 349 -> 341 us, 100 rows 373 -> 371, but 300 rows 444 -> 485 and 1,000 662 -> 804.
constexpr int kFewRows = 256;
constexpr int walk_parts(int np, int dp, int kind) {
  return np == 3 ? 3 : (dp == 32 || kind == 3 ? 2 : 1);
}
constexpr int walk_table(int np, int dp, int V) { return np == 1 && dp > 32 && V <= kFewRows ? 3 : 2; }
// The weighted sum's weights are the rounded probabilities over their own sum: over the sum of the
// unrounded ones they would not add up to 1, and a direction that all likely rows have in common would be
// off by 2^-9 of it, many times the differences that the gradient is made of (8 rows whose common part is
// 30 times their spread: 1.7e-2 of the gradient in bf16, 1.8e-3 with this, where one rounding of the
// result is 1.7e-3).  Two products of 16 x 16 x 32 a block and tile: 1.6 % of a call of 263,576 pixels x
// 50,000 rows x 64 channels with both gradients.
constexpr bool walk_norm(int np, int kind) {
  return kind == 1 && np == 1;
}
constexpr int walk_rows(int np, int dp, int kind) { return 128 * walk_blocks(np, dp, kind); }
// Workgroups: as many as run at once on 256 compute units.
constexpr int walk_workers(int np, int dp, int kind) {
  return 256 * walk_waves(np, dp, kind) / walk_columns(np, dp, kind);
}

template <typename T, int DP, int KIND>
struct Walk {
  static constexpr int np = Form<T>::np;
  static constexpr int rb = walk_blocks(np, DP, KIND);
  static constexpr int waves = walk_waves(np, DP, KIND);
  static constexpr int cs = walk_columns(np, DP, KIND);
  static constexpr int pp = walk_parts(np, DP, KIND);
  static constexpr bool norm = walk_norm(np, KIND);
  static constexpr int rows = walk_rows(np, DP, KIND);  // held by a workgroup
  static constexpr int workers = walk_workers(np, DP, KIND);
  static constexpr int tile_bytes = np * 32 * DP * 2;  // a tile's operands: a multiple of 1024
  static constexpr int sum_bytes = tile_bytes / cs;    // of the weighted sum
};

// How the work is dealt to the workgroups that run at once: `blocks` blocks of held rows, each walked
// over `pairs` pairs of tiles.  Every workgroup takes the same number of whole blocks, all of them
// walking in step so that they read the same tiles at the same time; the blocks that are left over
// are dealt evenly by pairs, across their borders.  So no round is left half empty, with few blocks
// as with many, and the count of pixels with a label need not be known on the host.
// A block's parts (one, or those of the left-over deal) stand in consecutive slots.
struct Deal {
  int pairs, full, rem, nw;  // whole blocks a worker, blocks left over, workers that share those
  int64_t units;
  int workers;
  __device__ __forceinline__ Deal(int64_t blocks, int pairs_, int workers_)
      : pairs(pairs_), workers(workers_) {
    full = (int)(blocks / workers);
    rem = (int)(blocks - (int64_t)full * workers);
    units = (int64_t)rem * pairs;
    nw = (int)min((int64_t)workers, units);
  }
  __device__ __forceinline__ int64_t begin(int w) const { return units * w / nw; }
  // the slots of a block's parts
  __device__ __forceinline__ void parts(int64_t block, int64_t &slot, int &n) const {
    const int64_t whole = (int64_t)full * workers;
    if (block < whole) {
      slot = block;
      n = 1;
    } else if (units == 0) {
      slot = 0;
      n = 0;
    } else {
      const int64_t t = block - whole;
      const int64_t w0 = ((t * pairs + 1) * nw - 1) / units;
      const int64_t w1 = ((t + 1) * pairs * nw - 1) / units;
      slot = whole + w0 + t;
      n = (int)(w1 - w0) + 1;
    }
  }
  // calls f(block, first pair, last pair, slot) for worker w's share
  template <typename F>
  __device__ __forceinline__ void each(int w, F f) const {
    int64_t u = 0, end = 0;
    if (w < nw) {
      u = begin(w);
      end = begin(w + 1);
    }
    for (int k = 0;; ++k) {  // (one call: the walks are long)
      int64_t block = (int64_t)k * workers + w, slot = block;
      int p0 = 0, p1 = pairs;
      if (k >= full) {
        if (u >= end) break;
        const int t = (int)(u / pairs);
        p0 = (int)(u - (int64_t)t * pairs);
        p1 = (int)min((int64_t)pairs, p0 + (end - u));
        u += p1 - p0;
        block = (int64_t)full * workers + t;
        slot = block + w;
      }
      f(block, p0, p1, slot);
    }
  }
};
inline int64_t deal_slots(int64_t rows, int np, int dp, int kind) {
  return rows / walk_rows(np, dp, kind) + walk_workers(np, dp, kind) + 1;
}

// The waves that share a SIMD take different priorities (by their slot): waves of the same priority
// fall into step, all in their products and then all in their exponentials, and leave one of the two
// pipes idle; with one ahead the other fills the pipe that it leaves free.
__device__ __forceinline__ void stagger() {
  const uint32_t slot = __builtin_amdgcn_s_getreg(4 | (3 << 11));  // the wave's slot in its SIMD
  if (slot & 1)
    __builtin_amdgcn_s_setprio(1);
  else
    __builtin_amdgcn_s_setprio(0);
}

// Copies `bytes` from global memory to LDS without registers: 1 KB a wave and instruction, waited
// for with arrive().
template <int BYTES>
__device__ __forceinline__ void fetch(uint4 *dst, const uint16_t *src) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  static_assert(BYTES % 1024 == 0, "a wave copies 1 KB at a time");
#pragma unroll
  for (int c = 0; c < BYTES / 1024; c += 4) {
    if (BYTES % 4096 != 0 && c + wave >= BYTES / 1024) break;
    const int k = c + wave;
    __builtin_amdgcn_global_load_lds(
        (const __attribute__((address_space(1))) void *)(src + k * 512 + lane * 8),
        (__attribute__((address_space(3))) void *)(dst + k * 64), 16, 0, 0);
  }
}

// The transposed operands of a tile for the column range z (see Walk::cs).
template <typename W>
__device__ __forceinline__ void fetch_sum(uint4 *dst, const uint16_t *src, int z) {
  if constexpr (W::cs == 1) {
    fetch<W::sum_bytes>(dst, src);
  } else {
    constexpr int kBlocks = 2 * W::np, kPart = W::sum_bytes / kBlocks;  // per plane and row half
#pragma unroll
    for (int k = 0; k < kBlocks; ++k)
      fetch<kPart>(dst + k * (kPart / 16), src + (k * W::cs + z) * (kPart / 2));
  }
}

__device__ __forceinline__ void arrive() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// One step of a walk: the matrix pipe's work on the tiles i - 1 (weighted sum) and i + 1 (logits), and
// the vector pipe's on tile i (exponentials) in the products' shadow, so that a wave keeps both pipes
// busy by itself.  s holds the logits of tile i and then of i + 1, q the operands of i - 1 and then
// of i.
template <typename T, int DP, int KIND>
struct Step {
  using F = Form<T>;
  using H8 = typename F::H8;
  using W = Walk<T, DP, KIND>;
  static constexpr bool SUM = KIND > 0;
  static constexpr int NP = F::np, RB = W::rb, PP = W::pp, KS = DP / 16, DT = DP / 32 / W::cs;
  // Three parts of 256 channels and their sums do not fit the registers: the held rows' second and third
  // parts, which three of six products take, are read again for every tile, by the vector cache, which
  // is free for them (held, 500 bytes a lane are spilled: 27,000 pixels x 56,506 rows of 235 channels take
  // 48.9 ms for both gradients, with two parts held 37.6, with one 28.3).
  static constexpr bool kLean = NP == 3 && DP == 256 && SUM;
  static constexpr int HP = kLean ? 1 : NP;
  H8 held[RB][KS][HP];
  const uint16_t *low;
  f32x16 s[RB];
  f32x16 o[SUM ? RB : 1][SUM ? DT : 1];
  uint4 q[RB][2][PP];
  // The sums of q (see walk_norm), by the matrix pipe: the operand of a 32 x 32 x 16 product, 32 pixels in
  // two halves of the lanes, taken as one of 16 x 16 x 32 has pixels c and c + 16 in the even and odd
  // groups of 16 lanes.  Rows of ones and zeros keep them apart, and lane l gets pixel l % 32's sum.
  // (finite values only: 0 times another pixel's NaN)
  static constexpr bool NORM = W::norm;
  f32x4 sum_q[NORM ? RB : 1];
  H8 pick;

  __device__ __forceinline__ void hold(const uint16_t *packed, int64_t row0) {
    const int lane = threadIdx.x & 63;
    low = packed + ((row0 >> 5) * NP + HP) * KS * 512 + lane * 8;
#pragma unroll
    for (int b = 0; b < RB; ++b) {
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int p = 0; p < HP; ++p)
          held[b][k][p] =
              *(const H8 *)(packed + ((((row0 >> 5) + b) * NP + p) * KS + k) * 512 + lane * 8);
      if constexpr (SUM) {
#pragma unroll
        for (int t = 0; t < DT; ++t) o[b][t] = (f32x16)(0.f);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int p = 0; p < PP; ++p) q[b][h][p] = make_uint4(0, 0, 0, 0);
      if constexpr (NORM) sum_q[b] = (f32x4)(0.f);
    }
    if constexpr (NORM) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        pick[j] = ((lane >> 2) & 1) == ((lane >> 4) & 1) ? (typename F::H)1.f : (typename F::H)0.f;
    }
  }

  // The products of a step, one after the other, with between(i) behind the i-th: the weighted sum's
  // (if ADD) and the logits' (if LOGITS).  Operands are read from LDS a few products ahead; the fences
  // keep the compiler from gathering the products and the vector work apart.
  template <bool ADD, bool LOGITS, typename Between>
  __device__ __forceinline__ void products(const uint4 *straight, const uint4 *transposed,
                                           f32x16 *next, Between between) {
    if constexpr (NP == 3) {
      products3<ADD, LOGITS>(straight, transposed, next[0], between);
      return;
    }
    constexpr int kAdd = ADD ? 2 * DT : 0, kOps = kAdd + (LOGITS ? KS : 0);
    constexpr int kAhead = RB == 2 ? 3 : 5;
    const int lane = threadIdx.x & 63;
    H8 a[kOps];
    auto load = [&](int n) {
      a[n] = n < kAdd ? *(const H8 *)&transposed[n * 64 + lane]
                      : *(const H8 *)&straight[(n - kAdd) * 64 + lane];
    };
#pragma unroll
    for (int n = 0; n < (kAhead < kOps ? kAhead : kOps); ++n) load(n);
    between(0);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (LOGITS) {
#pragma unroll
      for (int b = 0; b < RB; ++b) next[b] = (f32x16)(0.f);
    }
    int done = 1;
#pragma unroll
    for (int n = 0; n < kOps; ++n) {
      if (n + kAhead < kOps) load(n + kAhead);
      if constexpr (NORM) {
        if (n < kAdd && n % DT == 0) {
#pragma unroll
          for (int b = 0; b < RB; ++b)
#pragma unroll
            for (int p = PP - 1; p >= 0; --p)
              sum_q[b] = mfma16(pick, __builtin_bit_cast(H8, q[b][n / DT][p]), sum_q[b]);
        }
      }
#pragma unroll
      for (int p = PP - 1; p >= 0; --p) {  // (the small part first)
        if (n >= kAdd && p > 0) continue;
#pragma unroll
        for (int b = 0; b < RB; ++b) {
          if (n < kAdd)
            o[b][n % DT] = mfma(a[n], __builtin_bit_cast(H8, q[b][n / DT][p]), o[b][n % DT]);
          else
            next[b] = mfma(a[n], held[b][n - kAdd][0], next[b]);
          between(done++);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  }

  // The same for operands of three parts.  A product rounds its sum with every term, so the five small
  // products of all terms go first, at 2^-8 of the sum's size, and then the large ones: as many
  // roundings as a sum of 32-bit products has.  A tile's weighted sum is formed by itself and added as
  // a whole, one rounding a tile.
  template <bool ADD, bool LOGITS, typename Between>
  __device__ __forceinline__ void products3(const uint4 *straight, const uint4 *transposed,
                                            f32x16 &next, Between between) {
    const int lane = threadIdx.x & 63;
    constexpr int kAdd = ADD ? 2 * DT : 0;                    // groups of the weighted sum
    constexpr int kSmall = LOGITS ? KS : 0;                   // groups of small products
    constexpr int kLast = LOGITS ? (KS < 4 ? 1 : KS / 4) : 0;  // groups of large ones
    constexpr int kPer = KS < 4 ? KS : 4;
    constexpr int kGroups = kAdd + kSmall + kLast;
    H8 a[2][4];  // a group's operands: three planes, or the first planes of kPer steps
    H8 first;    // the first plane of the other row half
    // groups that the parts read again are ahead: 500 clocks, as a load from L2 takes (0: 10 % slower)
    constexpr int kDeep = 2, kRing = kDeep + 2;
    H8 rest[kLean ? kRing : 1][kLean ? NP - HP : 1];
    const uint16_t *again = low;
    if constexpr (kLean) asm volatile("" : "+v"(again));  // (not read once before the walk)
    auto load = [&](int g) {
      H8 *to = a[g & 1];
      if (g < kAdd) {  // group 2 d + h
#pragma unroll
        for (int p = 0; p < 3; ++p)
          to[p] = *(const H8 *)&transposed[((p * 2 + (g & 1)) * DT + g / 2) * 64 + lane];
      } else if (g < kAdd + kSmall) {
#pragma unroll
        for (int p = 0; p < 3; ++p) to[p] = *(const H8 *)&straight[(p * KS + g - kAdd) * 64 + lane];
      } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j)
          to[j] = *(const H8 *)&straight[((g - kAdd - kSmall) * kPer + j) * 64 + lane];
      }
    };
    auto read_again = [&](int k) {
      if constexpr (kLean) {
        if (k < 0 || k >= kSmall) return;
#pragma unroll
        for (int p = HP; p < 3; ++p)
          rest[k % kRing][p - HP] = *(const H8 *)(again + ((p - HP) * KS + k) * 512);
      }
    };
    load(0);
#pragma unroll
    for (int k = 0; k <= kDeep - kAdd; ++k) read_again(k);
    int done = 0;
    auto slot = [&] {
      between(done++);
      __builtin_amdgcn_sched_barrier(0);
    };
    slot();
    f32x16 tmp[2];
    if constexpr (LOGITS) next = (f32x16)(0.f);
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      if (g + 1 < kGroups) load(g + 1);
      read_again(g + 1 + kDeep - kAdd);
      const H8 *x = a[g & 1];
      if (g < kAdd) {
        const int d = g / 2, h = g & 1;
        H8 w[3], w0;
#pragma unroll
        for (int p = 0; p < 3; ++p) w[p] = __builtin_bit_cast(H8, q[0][h][p]);
        w0 = __builtin_bit_cast(H8, q[0][0][0]);
        if (h == 0) {
          tmp[d & 1] = (f32x16)(0.f);
          first = x[0];
        }
#pragma unroll
        for (int i = 0; i < 5; ++i) {
          tmp[d & 1] = product<3>(i, x, w, tmp[d & 1]);
          slot();
        }
        if (h == 1) {
          tmp[d & 1] = mfma(first, w0, tmp[d & 1]);
          slot();
          tmp[d & 1] = mfma(x[0], w[0], tmp[d & 1]);
          slot();
        }
      } else if (g < kAdd + kSmall) {
        H8 y[3];
#pragma unroll
        for (int p = 0; p < HP; ++p) y[p] = held[0][g - kAdd][p];
        if constexpr (kLean) {
#pragma unroll
          for (int p = HP; p < 3; ++p) y[p] = rest[(g - kAdd) % kRing][p - HP];
        }
#pragma unroll
        for (int i = 0; i < 5; ++i) {
          next = product<3, (KIND >= 2)>(i, x, y, next);
          slot();
        }
      } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          next = mfma(x[j], held[0][(g - kAdd - kSmall) * kPer + j][0], next);
          slot();
        }
      }
      // the sum of the columns before, once its products are through
      if (ADD && g >= 2 && g <= kAdd && g % 2 == 0) {
        o[0][g / 2 - 1] += tmp[(g / 2 - 1) & 1];
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if constexpr (ADD && !LOGITS) o[0][DT - 1] += tmp[(DT - 1) & 1];
  }

  __device__ __forceinline__ void logits(const uint4 *straight) {
    products<false, true>(straight, straight, s, [](int) {});
  }

  // Operands of three parts: an infinite element's second and third parts are NaN, and so are its
  // logits.  The products of the first parts alone give the infinity (or NaN) that they are.
  __device__ __forceinline__ void infinities(const uint4 *straight) {
    if constexpr (NP == 3) {
      bool odd = false;
#pragma unroll
      for (int i = 0; i < 16; ++i) odd |= !(fabsf(s[0][i]) < INFINITY);
      if (!__any(odd)) return;
      const int lane = threadIdx.x & 63;
      f32x16 large = (f32x16)(0.f);
#pragma unroll
      for (int k = 0; k < KS; ++k)
        large = mfma(*(const H8 *)&straight[k * 64 + lane], held[0][k][0], large);
#pragma unroll
      for (int i = 0; i < 16; ++i) s[0][i] = fabsf(s[0][i]) < INFINITY ? s[0][i] : large[i];
    }
  }

  __device__ __forceinline__ void add(const uint4 *transposed) {
    products<true, false>(transposed, transposed, s, [](int) {});
  }

  // pair(b, i, z0, z1): the probabilities 2 i and 2 i + 1 of block b in place of their logits
  template <typename Pair>
  __device__ __forceinline__ void step(const uint4 *straight, const uint4 *transposed, Pair pair) {
    constexpr int kSlots =
        NP == 3 ? 6 * (KS + (SUM ? 2 * DT : 0)) + 1 : RB * (KS + (SUM ? 2 * DT * PP : 0)) + 1;
    constexpr int kPairs = RB * 8;
    f32x16 next[RB];
    uint4 fresh[RB][2][PP];
    // split operands: behind the weighted sum, whose operands' registers the new ones take over
    constexpr int kFirst = NP == 3 && SUM ? 12 * DT : 0;
    products<SUM, true>(straight, transposed, next, [&](int slot) {
      if (slot < kFirst) return;
      const int k0 = (slot - kFirst) * kPairs / (kSlots - kFirst);
      const int k1 = (slot + 1 - kFirst) * kPairs / (kSlots - kFirst);
#pragma unroll
      for (int k = k0; k < k1; ++k) {
        const int b = k / 8, i = k % 8;
        float p0 = s[b][2 * i], p1 = s[b][2 * i + 1];
        pair(b, i, p0, p1);
        if constexpr (SUM) {
          pack_pair<T, PP>(p0, p1, i & 3, fresh[b][i >> 2]);
          // (stays in its slot: the compiler would move it behind the products)
#pragma unroll
          for (int p = 0; p < PP; ++p)
            asm volatile("" : "+v"(((uint32_t *)&fresh[b][i >> 2][p])[i & 3]));
        }
      }
    });
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      s[b] = next[b];
      if constexpr (SUM) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int p = 0; p < PP; ++p) q[b][h][p] = fresh[b][h][p];
      }
    }
  }

  // the sums, lane = held row, to [row][DP] from column c0 on
  __device__ __forceinline__ void store(float *out, int64_t row0, int c0) const {
    const int lane = threadIdx.x & 63, half = lane >> 5;
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f32x4 v;
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = o[b][d][4 * i + j];
          *(f32x4 *)(out + (row0 + 32 * b + (lane & 31)) * DP + c0 + 32 * d + 8 * i + 4 * half) =
              v;
        }
  }
};

// ------------------------------------------------------------------------------------------------
// the walk over the table
// ------------------------------------------------------------------------------------------------
// exp2 of logits up to this size needs no maximum: 2^60 a term leaves room for the sum and for the
// smallest term, 2^-60, in 32 bits (and in bf16), if the table's rows are no larger than 2^20 and the
// largest no smaller than 2^-20.
constexpr float kSafeLogit = 60.f, kSafeRow = 0x1p40f;  // (the latter squared)

template <typename T, int DP, bool SUM>
struct RowsWalk : Step<T, DP, SUM ? 1 : 0> {
  using B = Step<T, DP, SUM ? 1 : 0>;
  using F = Form<T>;
  using H8 = typename F::H8;
  static constexpr int RB = B::RB, DT = B::DT, PP = B::PP;
  int lab[RB];
  float m[RB], l[RB][2], t[RB][2], zy[RB];  // l + t: the sum of the probabilities in four terms
  float far_q[RB];                          // a lane's part of the sum of q, of a walk of large logits
  int V;
  float c2, c2l;

  // the label's own column and the table's padding take no part
  __device__ __forceinline__ void mask(int v0) {
    bool near = false;
#pragma unroll
    for (int b = 0; b < RB; ++b) near |= (uint32_t)(lab[b] - v0) < 32u;
    if (v0 + 32 > V || __any(near)) {
      int first = 4 * ((threadIdx.x & 63) >> 5);
      asm volatile("" : "+v"(first));  // its sums stay in here and out of the loop's registers
      first += v0;
#pragma unroll
      for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int v = first + 8 * (i >> 2) + (i & 3);
          zy[b] = v == lab[b] ? this->s[b][i] : zy[b];
          this->s[b][i] = v == lab[b] || v >= V ? -INFINITY : this->s[b][i];
        }
    }
  }

  // the running maximum over the new logits: a power of two apart from the last one, so that what is
  // summed up already (q too) changes exactly
  __device__ __forceinline__ void raise() {
    float top[RB];
    bool up = false;
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      top[b] = fmaxf(this->s[b][0], this->s[b][1]);
#pragma unroll
      for (int i = 2; i < 16; i += 2)
        top[b] = fmaxf(fmaxf(top[b], this->s[b][i]), this->s[b][i + 1]);
      top[b] *= c2;
      up |= top[b] > m[b] + F::slack;
    }
    if (__any(up)) {  // rarely after the first tiles
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        const float mn = fmaxf(m[b], ceilf(fmaxf(top[b], __shfl_xor(top[b], 32))));
        const float f = __builtin_amdgcn_exp2f(m[b] - mn);
        m[b] = mn;
        l[b][0] *= f;
        l[b][1] *= f;
        t[b][0] *= f;
        t[b][1] *= f;
        far_q[b] *= f;
        if constexpr (B::NORM) this->sum_q[b] *= f;
        if constexpr (SUM) {
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) this->o[b][d][i] *= f;
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int p = 0; p < PP; ++p)
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                typename F::H *e = (typename F::H *)&this->q[b][h][p] + j;
                *e = (typename F::H)((float)*e * f);
              }
        }
      }
    }
  }

  template <bool ONLINE>
  __device__ __forceinline__ void ready(int v0) {
    mask(v0);
    if constexpr (ONLINE) raise();
  }

  // a tile of large logits (see kFar), with no other's work beside it.  The power of two by which
  // probabilities are scaled in the products stays out of the maximum, which may be too large for it.
  __device__ __forceinline__ void far_tile(const uint4 *s_e, const uint4 *s_t, int v0) {
    B::logits(s_e);
    B::infinities(s_e);
    mask(v0);
    raise();
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p0 = __builtin_amdgcn_exp2f(this->s[b][2 * i] * c2 - m[b]);
        const float p1 = __builtin_amdgcn_exp2f(this->s[b][2 * i + 1] * c2 - m[b]);
        t[b][0] += p0;
        t[b][1] += p1;
        if constexpr (SUM) {
          constexpr float f = F::shift == 0.f ? 1.f : 0x1p10f;
          pack_pair<T, PP>(p0 * f, p1 * f, i & 3, this->q[b][i >> 2]);
          if constexpr (B::NORM) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const float p = (k ? p1 : p0) * f, large = (float)(typename F::H)p;
              far_q[b] += PP == 1 ? large : large + (float)(typename F::H)(p - large);
            }
          }
        }
      }
    fold();
    if constexpr (SUM) B::add(s_t);
  }

  // The sums of the last tiles (one of 32-bit data, two of 16-bit data) to those before: a walk of
  // 150,000 rows would be 40,000 additions a lane, whose roundings leave 3e-6 of the sum.  With 32-bit
  // data l[b][1] holds what the last addition lost; with 16-bit data that takes 1.5 % of the time, and
  // a rounding every 16 probabilities is little beside the operands'.
  __device__ __forceinline__ void fold() {
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      if constexpr (sizeof(T) == 4) {
        const float y = l[b][1] + (t[b][0] + t[b][1]), sum = l[b][0] + y;
        l[b][1] = y - (sum - l[b][0]);
        l[b][0] = sum;
      } else {
        l[b][0] += t[b][0];
        l[b][1] += t[b][1];
      }
      t[b][0] = t[b][1] = 0.f;
    }
  }

  template <bool ONLINE>
  __device__ __forceinline__ void next(const uint4 *s_e, const uint4 *s_t) {
    B::step(s_e, s_t, [&](int b, int, float &p0, float &p1) {
      if constexpr (ONLINE || sizeof(T) == 4) {
        const float shift = ONLINE ? F::shift - m[b] : 0.f;
        p0 = __builtin_amdgcn_exp2f(exponent<T>(p0, c2, c2l, shift));
        p1 = __builtin_amdgcn_exp2f(exponent<T>(p1, c2, c2l, shift));
      } else {
        p0 = __builtin_amdgcn_exp2f(p0 * c2);
        p1 = __builtin_amdgcn_exp2f(p1 * c2);
      }
      t[b][0] += p0;
      t[b][1] += p1;
      asm volatile("" : "+v"(t[b][0]), "+v"(t[b][1]));  // (stays in its slot)
    });
    if constexpr (sizeof(T) == 4) fold();
  }
};

// Bound by the matrix pipe, with the exponentials (16 a lane and 32 x 32 logits, 8 clocks each) partly
// beside it.  Measured: 64 channels, bf16, 263,576 pixels x 50,000 rows with dX: 3.81 ms, 0.89 PFLOP/s;
// 128 channels, losses of 1,054,304 pixels: 12.7 ms, 1.06 PFLOP/s (a bf16 library product of 8192^3
// reaches 1.17); 256 channels, 131,788 x 10,000 with dX: 1.61 ms, 0.84 PFLOP/s, where one block of
// rows a wave waits for LDS; fp32, 64 channels, 131,712 x 10,000: 1.83 ms, 0.18 PFLOP/s counted once,
// 1.1 of bf16 products (a fp32 library product reaches 0.13).
template <typename T, int DP, bool SUM>
__global__ __launch_bounds__(kBlock, (Walk<T, DP, SUM ? 1 : 0>::waves)) void kd_xent_rows(Args a) {
  using F = Form<T>;
  using W = Walk<T, DP, SUM ? 1 : 0>;
  constexpr int RB = W::rb, kBytes = W::tile_bytes;
  __shared__ uint4 s_e0[kBytes / 16], s_e1[kBytes / 16];
  __shared__ uint4 s_t0[SUM ? W::sum_bytes / 16 : 1], s_t1[SUM ? W::sum_bytes / 16 : 1];
  const int z = blockIdx.z;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const Deal deal(((int64_t)*a.count + W::rows - 1) / W::rows, (a.V + 63) / 64, W::workers);
  stagger();
  const float size2 = largest(a.emax), size = a.c2 * sqrtf(size2);
  const bool fits = F::shift == 0.f && size2 < kSafeRow && size2 > 1.f / kSafeRow;
  const bool far = !(size * sqrtf(largest(a.xmax)) < kFar<T>);  // (a NaN too)
  if (far && blockIdx.x == 0 && z == 0 && threadIdx.x == 0) *a.far = 1;
  const uint16_t *es = a.es, *et = a.et;
  constexpr int64_t kTile = kBytes / 2;
  // (the whole share in one way, so that the registers of one are not those of the other)
  auto share = [&](auto is_far) {
    constexpr bool FAR = decltype(is_far)::value;
    RowsWalk<T, DP, SUM> w;
    w.V = a.V;
    w.c2 = a.c2;
    w.c2l = a.c2l;
    deal.each(blockIdx.x, [&](int64_t block, int p0, int p1, int64_t slot) {
      const int64_t row0 = block * W::rows + wave * (32 * RB);
      bool general = true;
      if constexpr (!FAR) {
        // |logit| <= |x| |e| scale, over the kRowPad rows about this wave's (so that the choice does not
        // depend on how many of them a wave holds); a NaN size takes the general way
        bool safe = fits;
#pragma unroll
        for (int k = 0; k < kRowPad / kWave; ++k)
          safe &= size * sqrtf(a.xn[row0 / kRowPad * kRowPad + k * kWave + lane]) < kSafeLogit;
        general = !__all(safe);
      }
      w.hold(a.xs, row0);
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        w.lab[b] = a.lab[row0 + 32 * b + (lane & 31)];
        w.m[b] = general ? -FLT_MAX : 0.f;
        w.l[b][0] = w.l[b][1] = w.t[b][0] = w.t[b][1] = w.far_q[b] = 0.f;
        w.zy[b] = -INFINITY;
      }
      const int t0 = 2 * p0, t1 = 2 * p1;
      auto walk = [&](auto online) {
        constexpr bool ONLINE = decltype(online)::value;
        fetch<kBytes>(s_e0, es + t0 * kTile);
        arrive();
        fetch<kBytes>(s_e1, es + (t0 + 1) * kTile);
        if constexpr (SUM) fetch_sum<W>(s_t1, et + t0 * kTile, z);  // (times zeros)
        w.logits(s_e0);
        w.template ready<ONLINE>(t0 * 32);
        arrive();
        for (int t = t0; t < t1; t += 2) {
          const int t2 = min(t + 2, t1 - 1), t3 = min(t + 3, t1 - 1);  // behind the end: not used
          fetch<kBytes>(s_e0, es + t2 * kTile);
          if constexpr (SUM) fetch_sum<W>(s_t0, et + t * kTile, z);
          w.template next<ONLINE>(s_e1, s_t1);
          w.template ready<ONLINE>((t + 1) * 32);
          arrive();
          fetch<kBytes>(s_e1, es + t3 * kTile);
          if constexpr (SUM) fetch_sum<W>(s_t1, et + (t + 1) * kTile, z);
          w.template next<ONLINE>(s_e0, s_t0);
          if constexpr (sizeof(T) == 2) w.fold();
          w.template ready<ONLINE>(t2 * 32);
          arrive();
        }
        if constexpr (SUM) w.add(s_t1);
      };
      if constexpr (FAR) {
        for (int t = t0; t < t1; ++t) {
          fetch<kBytes>(s_e0, es + t * kTile);
          if constexpr (SUM) fetch_sum<W>(s_t0, et + t * kTile, z);
          arrive();
          w.far_tile(s_e0, s_t0, t * 32);
          __syncthreads();
        }
        if constexpr (SUM && F::shift != 0.f) {
#pragma unroll
          for (int b = 0; b < RB; ++b)
#pragma unroll
            for (int d = 0; d < RowsWalk<T, DP, SUM>::DT; ++d) w.o[b][d] *= 0x1p-10f;
        }
      } else if (general) {
        walk(std::true_type{});
      } else {
        walk(std::false_type{});
      }
      const int64_t out = slot * W::rows + wave * (32 * RB);
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        const int64_t r = out + 32 * b + (lane & 31);
        float l = w.l[b][0] + w.l[b][1];
        l += __shfl_xor(l, 32);
        const float other = __shfl_xor(w.zy[b], 32);  // one of the halves has met the label, or none
        float q = 0.f;
        if constexpr (W::norm) {
          q = w.sum_q[b][0];
          if constexpr (FAR) q = (w.far_q[b] + __shfl_xor(w.far_q[b], 32)) * (F::shift != 0.f ? 0x1p-10f : 1.f);
        }
        if (half == 0 && z == 0) {
          if constexpr (W::norm) a.pq[r] = q;
          a.pz[r] = w.zy[b] == -INFINITY ? other : w.zy[b];
          a.pm[r] = FAR ? w.m[b] : w.m[b] - F::shift;
          a.pl[r] = l;
        }
      }
      if constexpr (SUM) w.store(a.po, out, z * (DP / W::cs));
    });
  };
  if (far)
    share(std::true_type{});
  else
    share(std::false_type{});
}

// ------------------------------------------------------------------------------------------------
// joining the parts: G lanes per listed pixel; with RAW, four channels of dX a lane
// ------------------------------------------------------------------------------------------------
// Bound by the bytes of the parts' sums (32 bits) and of dX before its gradient: 131,788 pixels of 256
// channels 100 us, 2.7 TB/s, in the time of 3 ms.
constexpr int kFewParts = 16;

// A pixel's loss softplus(L' - z_y) from the maximum (log2) and the sum over the rows but its label's
// and from the label's logit; w: 1 - p_y, base + rest: log2 of the whole sum (far: see kFar), base a
// whole number and the larger of the two sides, so that rest is small.
__device__ __forceinline__ float pixel_loss(float m, float l, float z, bool far, const Args &a,
                                            float &w, float &base, float &rest) {
  const float z2 = z * a.c2;
  // log2 of the sum less z_y, both near the whole number m + k: the difference is formed where it is
  // small (m is a whole number), the sum's logarithm next to 1 if the loss is neither large nor small
  float k = fminf(fmaxf(rintf(z2 - m), -1e9f), 1e9f);
  const float mk = m + k;
  if (far) k = mk - m;  // (as far as m + k was rounded)
  const float d = far ? z2 - mk : fmaf(z, a.c2, -mk) + z * a.c2l;
  const float fits = fminf(fmaxf(k, -40.f), 40.f);  // (sums reach from 2^-60 to 2^91)
  const float part = log2f(l * __builtin_amdgcn_exp2f(-fits)), g = part - (k - fits);
  float u = (g - d) * kLn2;  // -inf when the label is the only row
  if (z2 == INFINITY) u = NAN;  // as infinity less infinity
  const float t = expf(-fabsf(u)), more = log1pf(t);
  const bool others = u > 0.f;
  w = u != u ? u : (others ? 1.f : t) / (1.f + t);
  base = u != u ? u : others ? m : far ? z2 : mk;  // (never infinite, as that of padding is)
  rest = fmaf(more, kLog2e, others ? part + fits : far ? 0.f : d);
  return u != u ? u : fmaxf(u, 0.f) + more;
}

template <typename T, int DP, int G, bool RAW>
__global__ __launch_bounds__(kBlock) void kd_xent_combine(Args a, const T *__restrict__ table,
                                                          float *__restrict__ loss) {
  const int gl = threadIdx.x & (G - 1);
  const int64_t r = block_id() * (kBlock / G) + threadIdx.x / G;
  const int count = *a.count;
  if (r >= count) return;
  const int64_t i = a.rowid[r];
  using W = Walk<T, DP, RAW ? 1 : 0>;
  int64_t slot;
  int n;
  Deal(((int64_t)count + W::rows - 1) / W::rows, (a.V + 63) / 64, W::workers)
      .parts(r / W::rows, slot, n);
  const int64_t first = slot * W::rows + r % W::rows;
  const int d = 4 * gl, left = a.D - d;  // (D <= 4 G)
  Pack<T, 4> e;
  f32x4 o = (f32x4)(0.f);
  if (RAW && left > 0) {
    e = load_pack<T, 4>(table + (int64_t)a.lab[r] * a.D + d, left);
    if (n == 1) o = *(const f32x4 *)(a.po + first * DP + d);
  }
  const bool few = n < kFewParts;  // every lane goes through them all

  const int s0 = few ? 0 : gl, ds = few ? 1 : G;
  float m = -FLT_MAX, z = -INFINITY;
#pragma unroll 4
  for (int s = s0; s < n; s += ds) {
    const int64_t q = first + (int64_t)s * W::rows;
    const float part = a.pz[q];
    m = fmaxf(m, a.pm[q]);
    z = part == -INFINITY ? z : part;  // (a NaN stays)
  }
  if (!few) {
#pragma unroll
    for (int s = G / 2; s >= 1; s >>= 1) {
      const float part = __shfl_xor(z, s);
      m = fmaxf(m, __shfl_xor(m, s));
      z = part == -INFINITY ? z : part;
    }
  }
  float l = 0.f, lq = 0.f;  // (lq: see walk_norm)
#pragma unroll 4
  for (int s = s0; s < n; s += ds) {
    const int64_t q = first + (int64_t)s * W::rows;
    const float f = __builtin_amdgcn_exp2f(a.pm[q] - m);
    l += a.pl[q] * f;
    if constexpr (W::norm) lq += a.pq[q] * f;
  }
  if (!few) {
#pragma unroll
    for (int s = G / 2; s >= 1; s >>= 1) {
      l += __shfl_xor(l, s);
      if constexpr (W::norm) lq += __shfl_xor(lq, s);
    }
  }
  if constexpr (!W::norm) lq = l;
  float wn, base, rest;
  const bool far = *a.far;
  const float out = pixel_loss(m, l, z, far, a, wn, base, rest);
  if (gl == 0) {
    if (far) {
      a.rl[r] = exp2f(-rest);
    } else if (sizeof(T) == 4) {
      const float whole = floorf(rest);
      base += whole;
      a.rl[r] = exp2f(whole - rest);
    } else {
      base += rest - Form<T>::shift_table;  // (no factor)
    }
    a.lse[r] = -base;
    a.w[r] = -wn * exp2f(Form<T>::shift_table);
    if (a.reduction == 0)
      loss[i] = out;
    else
      a.lrow[r] = out;
  }
  if constexpr (RAW) {
    if (left <= 0) return;
    const float inv = lq > 0.f ? 1.f / lq : (lq == 0.f ? 0.f : lq);
    if (n > 1) {
#pragma unroll 4
      for (int s = 0; s < n; ++s) {
        const int64_t q = first + (int64_t)s * W::rows;
        o += *(const f32x4 *)(a.po + q * DP + d) * __builtin_amdgcn_exp2f(a.pm[q] - m);
      }
    }
    Pack<float, 4> v;
#pragma unroll
    for (int j = 0; j < 4; ++j) v.v[j] = wn * (o[j] * inv - (float)e.v[j]);
    store_pack<float, 4>(a.raw + i * a.D + d, v, left);
  }
}

// ------------------------------------------------------------------------------------------------
// the loss of a few pixels
// ------------------------------------------------------------------------------------------------
// Up to kFewPixels pixels and no gradients (a query at a clicked pixel): the table is read once as it
// stands, straight into the products' operands, and nothing is listed, packed or kept.  Each wave
// takes tiles of 32 table rows in turn; the workgroup's parts are joined in LDS, all of them by a
// second launch of one workgroup.  Bound by the table's bytes: one pixel, 200,000 rows of 256
// channels in bf16 29.4 us, 3.5 TB/s, and 8 us for the join.
constexpr int kFewPixels = 64, kFewWorkers = 512;

// 8 channels of a row
template <typename T>
struct Chunk {
  T x[8];
  // `left` of them inside the row, no read behind it
  __device__ __forceinline__ void load(const T *row, int left) {
    constexpr int V = 16 / sizeof(T);
#pragma unroll
    for (int k = 0; k < 8; k += V) {
      const Pack<T, V> p = left > k ? load_pack<T, V>(row + k, left - k) : Pack<T, V>{};
#pragma unroll
      for (int j = 0; j < V; ++j) x[k + j] = p.v[j];
    }
  }
  // all 8, whatever they are
  __device__ __forceinline__ void load_any(const T *p) {
    const Pack<T, 8> v = *(const Pack<T, 8> *)p;
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = v.v[j];
  }
  __device__ __forceinline__ void clear_behind(int left) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = j < left ? x[j] : (T)0.f;
  }
  __device__ __forceinline__ void operand(uint4 *o) const {
    Pack<uint16_t, 8> u[Form<T>::np];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (Form<T>::np == 1)
        u[0].v[j] = __builtin_bit_cast(uint16_t, x[j]);
      else
        split3(x[j], u[0].v[j], u[1].v[j], u[2].v[j]);
    }
#pragma unroll
    for (int p = 0; p < Form<T>::np; ++p) o[p] = __builtin_bit_cast(uint4, u[p]);
  }
};

template <typename T, int DP>
__global__ __launch_bounds__(kBlock) void kd_xent_few(Args a, const T *__restrict__ features,
                                                      const T *__restrict__ table,
                                                      const int64_t *__restrict__ labels) {
  using F = Form<T>;
  using H8 = typename F::H8;
  constexpr int NP = F::np, KS = DP / 16, kTimes = NP == 3 ? 6 : 1;
  constexpr int kChunk = NP == 3 ? (KS < 4 ? KS : 4) : (KS < 16 ? KS : 16);  // operands in flight
  __shared__ float s_p[3][kBlock / kWave][32];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const int64_t i = (int64_t)blockIdx.y * 32 + (lane & 31);  // this lane's pixel
  uint4 x[KS][NP];
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    const int d = 16 * k + 8 * half;
    Chunk<T> f;
    f.load(features + i * a.D + d, i < a.n ? a.D - d : 0);
    if (a.scale < 0.f) {
#pragma unroll
      for (int j = 0; j < 8; ++j) f.x[j] = (T)(-(float)f.x[j]);
    }
    f.operand(x[k]);
  }
  const int64_t y = i < a.n ? labels[i] : -1;
  float m = -FLT_MAX, l = 0.f, zy = -INFINITY;
  const int ntile = (a.V + 31) / 32;
  for (int t = blockIdx.x * (kBlock / kWave) + wave; t < ntile; t += gridDim.x * (kBlock / kWave)) {
    const int64_t v0 = (int64_t)t * 32, v = v0 + (lane & 31);
    f32x16 s = (f32x16)(0.f), low = (f32x16)(0.f);
    // all the tile's loads at once, with no branch between them: the chunks that cross a row's end
    // read on into the next row, which the last tiles of the table have not
    const bool inside = (v0 + 32) * a.D + 7 <= (int64_t)a.V * a.D;
#pragma unroll
    for (int c = 0; c < KS; c += kChunk) {
      Chunk<T> e[kChunk];
      if (inside) {
#pragma unroll
        for (int k = 0; k < kChunk; ++k)
          e[k].load_any(table + v * a.D + min(16 * (c + k) + 8 * half, a.D - 1));
        if (a.D < 16 * (c + kChunk)) {
#pragma unroll
          for (int k = 0; k < kChunk; ++k) e[k].clear_behind(a.D - (16 * (c + k) + 8 * half));
        }
      } else {
#pragma unroll
        for (int k = 0; k < kChunk; ++k) {
          const int d = 16 * (c + k) + 8 * half;
          e[k].load(table + v * a.D + d, v < a.V ? a.D - d : 0);
        }
      }
#pragma unroll
      for (int k = 0; k < kChunk; ++k) {
        uint4 ew[NP];
        H8 ea[NP], xb[NP];
        e[k].operand(ew);
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          ea[p] = __builtin_bit_cast(H8, ew[p]);
          xb[p] = __builtin_bit_cast(H8, x[c + k][p]);
        }
        // (the small products by themselves: see products3)
#pragma unroll
        for (int q = 0; q < kTimes - 1; ++q) low = product<NP>(q, ea, xb, low);
        s = product<NP>(kTimes - 1, ea, xb, s);
      }
    }
    if constexpr (NP == 3) {
#pragma unroll
      for (int j = 0; j < 16; ++j)  // (an infinite element's small products are NaN)
        s[j] = fabsf(s[j]) < INFINITY ? s[j] + low[j] : s[j];
    }
    if (v0 + 32 > a.V || __any((uint64_t)(y - v0) < 32u)) {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int64_t r = v0 + 8 * (j >> 2) + 4 * half + (j & 3);
        zy = r == y ? s[j] : zy;
        s[j] = r == y || r >= a.V ? -INFINITY : s[j];
      }
    }
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 16; ++j) top = fmaxf(top, s[j]);
    top = ceilf(top * a.c2);  // (whole numbers: see pixel_loss)
    if (top > m) {  // (a lane by itself: the halves of a pixel are joined at the end)
      l *= __builtin_amdgcn_exp2f(m - top);
      m = top;
    }
    float sum = 0.f;
    const bool far = !(fabsf(m) < kFar<T>);
#pragma unroll
    for (int j = 0; j < 16; ++j)
      sum += __builtin_amdgcn_exp2f(far ? s[j] * a.c2 - m : exponent<T>(s[j], a.c2, a.c2l, -m));
    l += sum;
  }
  // the two halves, then the waves
  {
    const float mo = __shfl_xor(m, 32), lo = __shfl_xor(l, 32), zo = __shfl_xor(zy, 32);
    const float mn = fmaxf(m, mo);
    l = l * __builtin_amdgcn_exp2f(m - mn) + lo * __builtin_amdgcn_exp2f(mo - mn);
    m = mn;
    zy = zy == -INFINITY ? zo : zy;
  }
  if (half == 0) {
    s_p[0][wave][lane] = m;
    s_p[1][wave][lane] = l;
    s_p[2][wave][lane] = zy;
  }
  __syncthreads();
  if (threadIdx.x >= 32) return;
#pragma unroll
  for (int w = 1; w < kBlock / kWave; ++w) {
    const float mo = s_p[0][w][lane], zo = s_p[2][w][lane];
    const float mn = fmaxf(m, mo);
    l = l * __builtin_amdgcn_exp2f(m - mn) + s_p[1][w][lane] * __builtin_amdgcn_exp2f(mo - mn);
    m = mn;
    zy = zy == -INFINITY ? zo : zy;
  }
  const int64_t q = (int64_t)blockIdx.x * kFewPixels + i;
  a.pm[q] = m;
  a.pl[q] = l;
  a.pz[q] = zy;
}

template <typename T>
__global__ __launch_bounds__(1024) void kd_xent_few_join(Args a, int nparts,
                                                                const int64_t *__restrict__ labels,
                                                                float *__restrict__ loss) {
  constexpr int kLanes = 1024 / kFewPixels;
  __shared__ float s_m[kLanes][kFewPixels], s_l[kLanes][kFewPixels], s_z[kLanes][kFewPixels];
  const int i = threadIdx.x % kFewPixels, j = threadIdx.x / kFewPixels;
  float m = -FLT_MAX, l = 0.f, z = -INFINITY;
  if (i < a.n) {
#pragma unroll 4
    for (int p = j; p < nparts; p += kLanes) {
      const int q = p * kFewPixels + i;
      const float mo = a.pm[q], zo = a.pz[q], mn = fmaxf(m, mo);
      l = l * __builtin_amdgcn_exp2f(m - mn) + a.pl[q] * __builtin_amdgcn_exp2f(mo - mn);
      m = mn;
      z = zo == -INFINITY ? z : zo;
    }
  }
  s_m[j][i] = m;
  s_l[j][i] = l;
  s_z[j][i] = z;
  __syncthreads();
  if (j) return;  // one wave is left, a lane a pixel
#pragma unroll
  for (int k = 1; k < kLanes; ++k) {
    const float mo = s_m[k][i], zo = s_z[k][i], mn = fmaxf(m, mo);
    l = l * __builtin_amdgcn_exp2f(m - mn) + s_l[k][i] * __builtin_amdgcn_exp2f(mo - mn);
    m = mn;
    z = zo == -INFINITY ? z : zo;
  }
  const int64_t y = i < a.n ? labels[i] : -1;
  const bool in = y >= 0 && y < a.V;
  const bool far = !(fmaxf(fabsf(m), fabsf(z * a.c2)) < kFar<T>);
  float w, base, rest;
  const float out = in ? pixel_loss(m, l, z, far, a, w, base, rest) : 0.f;
  if (a.reduction == 0) {
    if (i < a.n) loss[i] = out;
    return;
  }
  double sum = (double)out;
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) sum += __shfl_xor(sum, s);
  const int count = __popcll(__ballot(in));
  if (i == 0) *loss = (float)(a.reduction == 1 ? sum / (double)(count > 0 ? count : 1) : sum);
}

// ------------------------------------------------------------------------------------------------
// the loss
// ------------------------------------------------------------------------------------------------
constexpr int kReduceBlocks = 256;

__device__ __forceinline__ double wg_sum(double x, double *s_x) {
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) x += __shfl_xor(x, s);
  if ((threadIdx.x & 63) == 0) s_x[threadIdx.x >> 6] = x;
  __syncthreads();
  return s_x[0] + s_x[1] + s_x[2] + s_x[3];
}

// Each workgroup adds up its share; the one that finishes last adds up the shares, in their order.
static __global__ __launch_bounds__(kBlock) void kd_xent_sum(Args a, float *__restrict__ loss) {
  __shared__ double s_x[kBlock / kWave];
  __shared__ bool s_last;
  const int count = *a.count;
  double x = 0.0;
  for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < count;
       i += (int64_t)gridDim.x * kBlock)
    x += (double)a.lrow[i];
  x = wg_sum(x, s_x);
  if (threadIdx.x == 0) {
    a.part[blockIdx.x] = x;
    __threadfence();
    s_last = atomicAdd(a.ticket, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  double y = 0.0;
  if (threadIdx.x < gridDim.x)
    y = __hip_atomic_load(&a.part[threadIdx.x], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  y = wg_sum(y, s_x);
  if (threadIdx.x == 0)
    *loss = (float)(a.reduction == 1 ? y / (double)(count > 0 ? count : 1) : y);
}

// ------------------------------------------------------------------------------------------------
// backward
// ------------------------------------------------------------------------------------------------
// The listed pixels' gradients of a loss per pixel, and the largest of their sizes per workgroup of
// grad_steps() x kBlock pixels: few in a row are short of latency (26,000 pixels 5 us with 4 against 12
// with 16), many leave fewer sizes to look through.
__host__ __device__ inline int grad_steps(int64_t npad) { return npad <= (1 << 20) ? 4 : 16; }
__host__ __device__ inline int grad_blocks(int64_t npad) {
  const int64_t chunk = (int64_t)grad_steps(npad) * kBlock;
  return (int)((npad + chunk - 1) / chunk);
}

// factors: of 32-bit data, the others have them only with large logits
static __global__ __launch_bounds__(kBlock) void kd_xent_rowgrad(Args a, bool factors,
                                                                 const float *__restrict__ grad) {
  __shared__ uint32_t s_m[kBlock / kWave];
  const int count = *a.count;
  const int steps = grad_steps(a.npad);
  uint32_t top = 0;
#pragma unroll 4
  for (int k = 0; k < steps; ++k) {
    const int64_t r = ((int64_t)blockIdx.x * steps + k) * kBlock + threadIdx.x;
    const float g = r < count ? grad[a.rowid[r]] : 0.f;
    if (r < a.npad) {
      a.grow[r] = g;
      if (factors || *a.far) a.gfac[r] = r < count ? g * a.rl[r] : 0.f;
    }
    top = max(top, __float_as_uint(fabsf(g)));
  }
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, s));
  if ((threadIdx.x & 63) == 0) s_m[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x == 0) a.gmax[blockIdx.x] = max(max(s_m[0], s_m[1]), max(s_m[2], s_m[3]));
}

// The power of two that brings the largest gradient into [1, 2): the products' operands stay in
// range whatever the incoming gradient's scale.  No larger than 2^112, so that its inverse and 2^14
// times it are normal numbers; gradients below 2^-112 are then less than 1.
__device__ __forceinline__ float grad_unit(const Args &a) {
  __shared__ uint32_t s_u[kBlock / kWave];
  const int nblk = grad_blocks(a.npad);
  uint32_t top = 0;
  for (int k = threadIdx.x; k < nblk; k += kBlock) top = max(top, a.gmax[k]);
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, s));
  if ((threadIdx.x & 63) == 0) s_u[threadIdx.x >> 6] = top;
  __syncthreads();
  const uint32_t e = max(max(s_u[0], s_u[1]), max(s_u[2], s_u[3])) >> 23;
  if (e == 255) return 1.f;  // infinite or NaN
  return e == 254 ? 0x1p-127f : __uint_as_float(min(254u - e, 239u) << 23);
}

// The walk over the pixels: kd_xent_rows with the sides exchanged, the logits formed a second time
// (2 n V D more operations; kept, they would be n V values written and read, 26 GB at the sizes below
// in 16 bits, 10 ms).  Bound as there.  Measured: 64 channels, bf16, 263,576 pixels x 50,000 rows 3.43 ms,
// 0.98 PFLOP/s; 256 channels, 131,788 x 10,000 1.79 ms, 0.75 PFLOP/s; fp32, 64 channels, 131,712 x
// 10,000 1.95 ms.
// A lane's 16 pixels of a tile are 8 i + 4 (lane / 32) + j: their exponents (and factors) are read one step
// ahead, of 32-bit data by way of LDS and a pair at a time (held in registers they cost 6 to 11 %).
template <typename T, int DP, bool ROWG, int KIND>
struct TableWalk : Step<T, DP, KIND> {
  using B = Step<T, DP, KIND>;
  using F = Form<T>;
  static constexpr int NP = B::NP, RB = B::RB, PP = B::PP;
  static constexpr bool FAC = ROWG || sizeof(T) == 4;  // exponentials have a factor
  int v0, near;  // near: this lane's pixel's label
  float c2, c2l, unit;
  f32x4 lse[NP == 1 ? 4 : 1], g[NP == 1 && FAC ? 4 : 1];
  const float *plse, *pw, *pg, *pf;  // pg: incoming gradients, pf: factors
  const int *plab;

  // the exponents and factors of a lane's pixels 8 i + 4 (lane / 32) + k .., of those of a tile
  template <typename VEC>
  __device__ __forceinline__ void rows(const float *tile_lse, const float *tile_f, int i, int k, VEC &l,
                                       VEC &f) {
    const int r = 8 * i + 4 * ((threadIdx.x & 63) >> 5) + k;
    l = *(const VEC *)(tile_lse + r);
    if (FAC) f = *(const VEC *)(tile_f + r);
    // (before the probabilities: unit times one of them can leave the range where g is small)
    if (ROWG) f *= unit;
  }
  // 32-bit data: tile t's by way of LDS, 64 x 4 bytes
  __device__ __forceinline__ void fetch_rows(float *s_r, int t) {
    const int lane = threadIdx.x & 63;
    if (NP == 1 || threadIdx.x >= kWave) return;
    __builtin_amdgcn_global_load_lds(
        (const __attribute__((address_space(1))) void *)((lane < 32 ? plse : pf - 32) +
                                                         (int64_t)t * 32 + lane),
        (__attribute__((address_space(3))) void *)s_r, 4, 0, 0);
  }
  __device__ __forceinline__ int label(int t) { return plab[(int64_t)t * 32 + (threadIdx.x & 31)]; }

  // 16-bit data: what the next step needs
  __device__ __forceinline__ void ahead(int t, f32x4 *l, f32x4 *f, int &y) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      rows(plse + (int64_t)t * 32, pf + (int64_t)t * 32, i, 0, l[i], f[FAC ? i : 0]);
    y = label(t);
  }

  // tile t is stepped over (s_r: its exponents and factors), t1 the next one's values
  __device__ __forceinline__ void next(const uint4 *s_x, const uint4 *s_t, const float *s_r, int t,
                                       int t1) {
    f32x4 l1[NP == 1 ? 4 : 1], g1[NP == 1 && FAC ? 4 : 1];
    f32x2 l2[2], g2[2];
    int near1;
    // one step ahead; where registers are short, from LDS, one pair ahead
    if constexpr (NP == 1) {
      ahead(t1, l1, g1, near1);
    } else {
      rows(s_r, s_r + 32, 0, 0, l2[0], g2[0]);
      near = label(t);
    }
    B::step(s_x, s_t, [&](int, int i, float &p0, float &p1) {
      f32x2 l, f = {1.f, 1.f};
      if constexpr (NP == 1) {
        const int j = 2 * (i & 1);
        l[0] = lse[i / 2][j], l[1] = lse[i / 2][j + 1];
        if (FAC) f[0] = g[i / 2][j], f[1] = g[i / 2][j + 1];
      } else {
        if (i < 7) rows(s_r, s_r + 32, (i + 1) / 2, 2 * ((i + 1) & 1), l2[(i + 1) & 1], g2[(i + 1) & 1]);
        l = l2[i & 1];
        f = g2[i & 1];
      }
      p0 = __builtin_amdgcn_exp2f(exponent<T>(p0, c2, c2l, l[0]));
      p1 = __builtin_amdgcn_exp2f(exponent<T>(p1, c2, c2l, l[1]));
      if (FAC) {
        p0 *= f[0];
        p1 *= f[1];
      }
    });
    labelled(t);
    if constexpr (NP == 1) {
      near = near1;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        lse[i] = l1[i];
        if (FAC) g[i] = g1[i];
      }
    }
  }

  // a tile of large logits (see kFar), with no other's work beside it
  __device__ __forceinline__ void far_tile(const uint4 *s_x, const uint4 *s_t, int t) {
    const int lane = threadIdx.x & 63;
    near = label(t);
    B::logits(s_x);
    B::infinities(s_x);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t r = (int64_t)t * 32 + 8 * i + 4 * (lane >> 5);
      const f32x4 l = *(const f32x4 *)(plse + r);
      f32x4 f = *(const f32x4 *)(pf + r) * unit;
      if constexpr (F::shift_table != 0.f) f *= 0x1p14f;
#pragma unroll
      for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          float p[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            p[k] = __builtin_amdgcn_exp2f(this->s[b][4 * i + j + k] * c2 + l[j + k]) * f[j + k];
            if (l[j + k] == -INFINITY) p[k] = 0.f;  // (padding, whatever the row holds)
          }
          pack_pair<T, PP>(p[0], p[1], 2 * (i & 1) + j / 2, this->q[b][i >> 1]);
        }
    }
    labelled(t);
    B::add(s_t);
  }

  // pixels of tile t labelled with these rows: p - 1 = -(1 - p) in the place of p
  __device__ __forceinline__ void labelled(int t) {
    const int lane = threadIdx.x & 63, half = lane >> 5;
    if (__any((uint32_t)(near - v0) < 32u * RB)) {
      int64_t r = (int64_t)t * 32 + 4 * half;
      asm volatile("" : "+v"(r));  // its sums stay in here and out of the loop's registers
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int64_t k = r + 16 * h + 8 * (j >> 2) + (j & 3);
          const int y = plab[k] - v0 - (lane & 31);
          const float neg = ROWG ? pw[k] * (pg[k] * unit) : pw[k];
          uint16_t part[3] = {0, 0, 0};
          if constexpr (NP == 1) {
            const typename F::H large = (typename F::H)neg;
            part[0] = __builtin_bit_cast(uint16_t, large);
            part[1] = __builtin_bit_cast(uint16_t, (typename F::H)(neg - (float)large));
          } else
            split3(neg, part[0], part[1], part[2]);
#pragma unroll
          for (int b = 0; b < RB; ++b)
#pragma unroll
            for (int p = 0; p < PP; ++p) {
              uint16_t *e = (uint16_t *)&this->q[b][h][p] + j;
              *e = y == 32 * b ? part[p] : *e;
            }
        }
    }
  }
};

template <typename T, int DP, bool ROWG, int KIND>
__global__ __launch_bounds__(kBlock, (Walk<T, DP, KIND>::waves)) void kd_xent_table(Args a) {
  using W = Walk<T, DP, KIND>;
  constexpr int RB = W::rb, kBytes = W::tile_bytes;
  __shared__ uint4 s_x0[kBytes / 16], s_x1[kBytes / 16];
  __shared__ uint4 s_t0[W::sum_bytes / 16], s_t1[W::sum_bytes / 16];
  __shared__ float s_r0[W::np == 1 ? 1 : kWave], s_r1[W::np == 1 ? 1 : kWave];
  const int z = blockIdx.z;
  const int wave = threadIdx.x >> 6;
  const Deal deal((a.V + W::rows - 1) / W::rows, (int)(((int64_t)*a.count + 63) / 64), W::workers);
  stagger();
  const float unit = ROWG ? grad_unit(a) : 1.f;
  const bool far = *a.far;
  const uint16_t *xs = a.xs, *xt = a.xt;
  constexpr int64_t kTile = kBytes / 2;
  auto share = [&](auto is_far) {  // (see kd_xent_rows)
    constexpr bool FAR = decltype(is_far)::value;
    TableWalk<T, DP, ROWG, KIND> w;
    w.c2 = a.c2;
    w.c2l = a.c2l;
    w.unit = unit;
    w.plse = a.lse;
    w.pw = a.w;
    w.pg = a.grow;
    w.pf = !ROWG ? a.rl : FAR || sizeof(T) == 4 ? a.gfac : a.grow;
    w.plab = a.lab;
    deal.each(blockIdx.x, [&](int64_t block, int p0, int p1, int64_t slot) {
      w.v0 = (int)(block * W::rows) + wave * (32 * RB);
      w.hold(a.es, w.v0);
      const int t0 = 2 * p0, t1 = 2 * p1;
      if constexpr (FAR) {
        for (int t = t0; t < t1; ++t) {
          fetch<kBytes>(s_x0, xs + t * kTile);
          fetch_sum<W>(s_t0, xt + t * kTile, z);
          arrive();
          w.far_tile(s_x0, s_t0, t);
          __syncthreads();
        }
      } else if (t0 < t1) {
        fetch<kBytes>(s_x0, xs + t0 * kTile);
        if constexpr (W::np == 1) w.ahead(t0, w.lse, w.g, w.near);
        w.fetch_rows(s_r0, t0);
        arrive();
        fetch<kBytes>(s_x1, xs + (t0 + 1) * kTile);
        fetch_sum<W>(s_t1, xt + t0 * kTile, z);  // (times zeros)
        w.logits(s_x0);
        arrive();
        for (int t = t0; t < t1; t += 2) {
          const int t2 = min(t + 2, t1 - 1), t3 = min(t + 3, t1 - 1);  // behind the end: not used
          fetch<kBytes>(s_x0, xs + t2 * kTile);
          fetch_sum<W>(s_t0, xt + t * kTile, z);
          w.fetch_rows(s_r1, t + 1);
          w.next(s_x1, s_t1, s_r0, t, t + 1);
          arrive();
          fetch<kBytes>(s_x1, xs + t3 * kTile);
          fetch_sum<W>(s_t1, xt + (t + 1) * kTile, z);
          w.fetch_rows(s_r0, t2);
          w.next(s_x0, s_t0, s_r1, t + 1, t2);
          arrive();
        }
        w.add(s_t1);
      }
      w.store(a.pe, slot * W::rows + wave * (32 * RB), z * (DP / W::cs));
    });
  };
  if (far)
    share(std::true_type{});
  else
    share(std::false_type{});
}

// The gradient's common factor: the incoming scalar, over the count for the mean.
__device__ __forceinline__ float grad_factor(const Args &a, const float *grad) {
  float g = *grad;
  if (a.reduction == 1) {
    const int count = *a.count;
    g /= (float)(count > 0 ? count : 1);
  }
  return g;
}

// The first `xblocks` workgroups scale dX, the others join the parts of dE: four channels a thread.
template <typename T, int DP, int KIND>
__global__ __launch_bounds__(kBlock) void kd_xent_grads(Args a, int64_t xblocks, int vpr,
                                                        const int64_t *__restrict__ labels,
                                                        const float *__restrict__ grad,
                                                        T *__restrict__ gx, T *__restrict__ ge) {
  const int64_t bid = block_id();
  const bool is_x = bid < xblocks;
  const int64_t q = (is_x ? bid : bid - xblocks) * kBlock + threadIdx.x;
  const int64_t r = q <= 0xffffffffll ? (int64_t)((uint32_t)q / (uint32_t)vpr) : q / vpr;
  const int d = (int)(q - r * vpr) * 4, left = a.D - d;
  float f = 1.f;
  if (!is_x && a.reduction == 0)
    f = 1.f / grad_unit(a);  // (the workgroup as a whole)
  else if (a.reduction != 0)
    f = grad_factor(a, grad);
  Pack<T, 4> o;
#pragma unroll
  for (int j = 0; j < 4; ++j) o.v[j] = (T)0.f;
  if (is_x) {
    if (r >= a.n) return;
    const int64_t y = labels[r];
    if (y >= 0 && y < a.V) {
      if (a.reduction == 0) f = grad[r];
      const Pack<float, 4> x = load_pack<float, 4>(a.raw + r * a.D + d, left);
#pragma unroll
      for (int j = 0; j < 4; ++j) o.v[j] = (T)(x.v[j] * (a.scale * f));
    }
    store_pack<T, 4>(gx + r * a.D + d, o, left);
  } else {
    if (r >= a.V) return;
    f32x4 x = (f32x4)(0.f);
    using W = Walk<T, DP, KIND>;
    int64_t slot;
    int n;
    Deal((a.V + W::rows - 1) / W::rows, (int)(((int64_t)*a.count + 63) / 64), W::workers)
        .parts(r / W::rows, slot, n);
    const float *part = a.pe + (slot * W::rows + r % W::rows) * DP + d;
#pragma unroll 8
    for (int s = 0; s < n; ++s) x += *(const f32x4 *)(part + (int64_t)s * W::rows * DP);
    const float g = exp2f(-Form<T>::shift_table) * fabsf(a.scale) * f;
#pragma unroll
    for (int j = 0; j < 4; ++j) o.v[j] = (T)(x[j] * g);
    store_pack<T, 4>(ge + r * a.D + d, o, left);
  }
}

// ------------------------------------------------------------------------------------------------
// host
// ------------------------------------------------------------------------------------------------
inline int padded_channels(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 128 ? 128 : 256; }

struct Space {
  char *base;
  size_t used;
  template <typename U>
  U *take(size_t n) {
    U *p = base ? (U *)(base + used) : nullptr;
    used += (n * sizeof(U) + 255) & ~(size_t)255;
    return p;
  }
};

inline Args shape(int64_t n, int64_t V, int D, int np, double scale, int reduction) {
  Args a = {};
  a.n = n;
  a.npad = (n + kRowPad - 1) / kRowPad * kRowPad;
  a.V = (int)V;
  a.vpad = (int)((V + kRowPad - 1) / kRowPad * kRowPad);
  a.D = D;
  a.dp = padded_channels(D);
  a.scale = (float)scale;
  // never 0: a masked logit, -inf, stays -inf (a scale of 0 makes every logit next to 0 all the same)
  const double c2 = std::max(fabs(scale) * 1.4426950408889634, 1e-30);
  a.c2 = (float)c2;
  if (np == 3 && (double)a.c2 > c2) a.c2 = nextafterf(a.c2, 0.f);
  // positive too, for the same reason; 16-bit data are multiplied by c2 alone, all of them
  a.c2l = np == 3 ? std::max((float)(c2 - (double)a.c2), 1.2e-38f) : 1.2e-38f;
  a.reduction = reduction;
  return a;
}

// Few enough pixels, and no gradients: see kd_xent_few, which needs no state and a part a workgroup.
inline bool few_pixels(const Args &a, bool need_x, bool need_e) {
  return a.n > 0 && a.n <= kFewPixels && !need_x && !need_e;
}

inline size_t lay_state(Args &a, int np, bool need_x, bool need_e, void *base) {
  Space s{(char *)base, 0};
  if (few_pixels(a, need_x, need_e)) return 1;
  const size_t xe = (size_t)a.npad * a.dp * np, ee = (size_t)a.vpad * a.dp * np;
  a.count = s.take<int>(64);
  a.far = s.take<int>(64);
  a.emax = s.take<uint32_t>(kSlots * kSlotPad);
  a.xmax = s.take<uint32_t>(kSlots * kSlotPad);
  a.ticket = s.take<uint32_t>(64);
  a.rowid = s.take<int>(a.npad);
  a.lab = s.take<int>(a.npad);
  a.lse = s.take<float>(a.npad);
  a.rl = s.take<float>(a.npad);
  a.w = s.take<float>(a.npad);
  a.xn = s.take<float>(a.npad);
  a.xs = s.take<uint16_t>(xe);
  a.xt = need_e ? s.take<uint16_t>(xe) : nullptr;
  a.es = s.take<uint16_t>(ee);
  a.raw = need_x ? s.take<float>((size_t)a.n * a.D) : nullptr;
  return s.used;
}

inline size_t lay_forward(Args &a, int np, bool need_x, bool need_e, void *base) {
  Space s{(char *)base, 0};
  if (few_pixels(a, need_x, need_e)) {
    for (float **p : {&a.pm, &a.pl, &a.pz}) *p = s.take<float>(kFewWorkers * kFewPixels);
    return s.used;
  }
  a.blk = s.take<int>((size_t)((a.n + kMapChunk - 1) / kMapChunk));
  a.et = need_x ? s.take<uint16_t>((size_t)a.vpad * a.dp * np) : nullptr;
  const int kind = need_x ? 1 : 0;
  const size_t part =
      (size_t)deal_slots(a.npad, np, a.dp, kind) * (size_t)walk_rows(np, a.dp, kind);
  a.pm = s.take<float>(part);
  a.pl = s.take<float>(part);
  a.pz = s.take<float>(part);
  a.pq = walk_norm(np, kind) ? s.take<float>(part) : nullptr;
  a.po = need_x ? s.take<float>(part * a.dp) : nullptr;
  a.lrow = s.take<float>(a.npad);
  a.part = s.take<double>(kReduceBlocks);
  return s.used;
}

inline size_t lay_backward(Args &a, int np, bool need_e, void *base) {
  Space s{(char *)base, 0};
  a.gmax = s.take<uint32_t>((size_t)grad_blocks(a.npad) + 1);
  a.grow = s.take<float>(a.npad);
  a.gfac = s.take<float>(a.npad);
  const int kind = walk_table(np, a.dp, a.V);
  const size_t part =
      (size_t)deal_slots(a.vpad, np, a.dp, kind) * (size_t)walk_rows(np, a.dp, kind);
  a.pe = need_e ? s.take<float>(part * a.dp) : nullptr;
  return s.used;
}

inline int check(int64_t n, int64_t V, int D, double scale, int reduction) {
  KD_CHECK_ARG(n >= 0 && n < ((int64_t)1 << 31) - kRowPad,
               "surface_cross_entropy: need 0 <= pixels < 2^31 - 256");
  KD_CHECK_ARG(V >= 1 && V < ((int64_t)1 << 31) - kRowPad,
               "surface_cross_entropy: need 1 <= embeddings < 2^31 - 256");
  KD_CHECK_ARG(D >= 1 && D <= 256, "surface_cross_entropy: need 1 <= channels <= 256");
  KD_CHECK_ARG(scale - scale == 0.0 && fabs(scale) < 1e30,
               "surface_cross_entropy: scale must be finite");
  KD_CHECK_ARG(reduction >= 0 && reduction <= 2, "surface_cross_entropy: unknown reduction");
  return KD_OK;
}

template <typename T, int DP, int KIND>
dim3 walk_grid() {
  return dim3(Walk<T, DP, KIND>::workers, 1, Walk<T, DP, KIND>::cs);
}

template <typename T, int DP>
void launch_few(const Args &a, const T *features, const T *table, const int64_t *labels, float *loss,
                hipStream_t stream) {
  const int wgs = std::min((a.V + 127) / 128, kFewWorkers);
  hipLaunchKernelGGL((kd_xent_few<T, DP>), dim3(wgs, (unsigned)((a.n + 31) / 32)), dim3(kBlock), 0,
                     stream, a, features, table, labels);
  hipLaunchKernelGGL(kd_xent_few_join<T>, dim3(1), dim3(1024), 0, stream, a, wgs, labels, loss);
}

template <typename T, int DP>
void launch_forward(const Args &a, bool need_x, const T *features, const T *table, float *loss,
                    hipStream_t stream) {
  const int xtiles = (int)(a.npad / 32), etiles = a.vpad / 32;
  hipLaunchKernelGGL((kd_xent_pack<T, DP>), grid_of((int64_t)xtiles + etiles), dim3(kBlock), 0,
                     stream, a, xtiles, features, table);
  if (need_x)
    hipLaunchKernelGGL((kd_xent_rows<T, DP, true>), (walk_grid<T, DP, 1>()), dim3(kBlock), 0,
                       stream, a);
  else
    hipLaunchKernelGGL((kd_xent_rows<T, DP, false>), (walk_grid<T, DP, 0>()), dim3(kBlock), 0,
                       stream, a);
  auto combine = [&](auto lanes, auto raw) {
    constexpr int G = decltype(lanes)::value, per = kBlock / G;  // listed pixels a workgroup joins
    hipLaunchKernelGGL((kd_xent_combine<T, DP, G, decltype(raw)::value>),
                       grid_of((a.n + per - 1) / per), dim3(kBlock), 0, stream, a, table, loss);
  };
  if (need_x)
    combine(std::integral_constant<int, DP / 4>{}, std::true_type{});
  else if (a.npad / Walk<T, DP, 0>::rows * kFewParts <= Walk<T, DP, 0>::workers)  // many parts
    combine(std::integral_constant<int, DP / 4>{}, std::false_type{});
  else
    combine(std::integral_constant<int, 1>{}, std::false_type{});
}

inline int64_t blocks(int64_t n) { return (n + kBlock - 1) / kBlock; }

template <typename T, int DP, int KIND>
void launch_table(const Args &a, const int64_t *labels, const float *grad, T *gx, T *ge,
                  hipStream_t stream) {
  if (ge && a.reduction == 0)
    hipLaunchKernelGGL((kd_xent_table<T, DP, true, KIND>), (walk_grid<T, DP, KIND>()), dim3(kBlock), 0,
                       stream, a);
  else if (ge)
    hipLaunchKernelGGL((kd_xent_table<T, DP, false, KIND>), (walk_grid<T, DP, KIND>()), dim3(kBlock), 0,
                       stream, a);
  const int vpr = (a.D + 3) / 4;
  const int64_t xb = gx ? blocks(a.n * vpr) : 0, eb = ge ? blocks((int64_t)a.V * vpr) : 0;
  if (xb + eb > 0)
    hipLaunchKernelGGL((kd_xent_grads<T, DP, KIND>), grid_of(xb + eb), dim3(kBlock), 0, stream, a, xb,
                       vpr, labels, grad, gx, ge);
}

template <typename T, int DP>
void launch_backward(const Args &a, const int64_t *labels, const float *grad, T *gx, T *ge,
                     hipStream_t stream) {
  if constexpr (walk_table(Form<T>::np, DP, 1) == 3) {
    if (walk_table(Form<T>::np, DP, a.V) == 3) {
      launch_table<T, DP, 3>(a, labels, grad, gx, ge, stream);
      return;
    }
  }
  launch_table<T, DP, 2>(a, labels, grad, gx, ge, stream);
}

template <typename T>
int forward(int64_t n, int64_t V, int D, const T *features, const T *table, const int64_t *labels,
            double scale, int reduction, int need_x, int need_e, float *loss, void *state,
            size_t state_bytes, void *scratch, size_t scratch_bytes, hipStream_t stream) {
  const int rc = check(n, V, D, scale, reduction);
  if (rc != KD_OK) return rc;
  KD_CHECK_ARG(loss || (n == 0 && reduction == 0), "surface_cross_entropy: loss is NULL");
  KD_CHECK_ARG(table && (n == 0 || (features && labels)), "surface_cross_entropy: NULL input");
  Args a = shape(n, V, D, Form<T>::np, scale, reduction);
  const size_t ns = lay_state(a, Form<T>::np, need_x, need_e, state);
  const size_t nw = lay_forward(a, Form<T>::np, need_x, need_e, scratch);
  if (!state || state_bytes < ns || !scratch || scratch_bytes < nw)
    return set_error(KD_ERR_WORKSPACE, "workspace too small: %zu < %zu or %zu < %zu", state_bytes,
                     ns, scratch_bytes, nw);
  KD_CHECK_ARG((((uintptr_t)state | (uintptr_t)scratch) & 255u) == 0,
               "surface_cross_entropy: state and scratch must be aligned to 256 bytes");
  ProfScope prof(K_XENT_FWD, stream);
  if (few_pixels(a, need_x, need_e)) {
    switch (a.dp) {
      case 32: launch_few<T, 32>(a, features, table, labels, loss, stream); break;
      case 64: launch_few<T, 64>(a, features, table, labels, loss, stream); break;
      case 128: launch_few<T, 128>(a, features, table, labels, loss, stream); break;
      default: launch_few<T, 256>(a, features, table, labels, loss, stream); break;
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess)
      return set_error(KD_ERR_LAUNCH, "surface_cross_entropy: %s", hipGetErrorString(e));
    return KD_OK;
  }
  const int nblk = (int)((n + kMapChunk - 1) / kMapChunk);
  if (nblk <= kListChunks) {  // one workgroup lists them all in less time than two launches take
    hipLaunchKernelGGL(kd_xent_map, dim3(1), dim3(kBlock), 0, stream, a, kListChunks, false, labels,
                       loss);
  } else {
    hipLaunchKernelGGL(kd_xent_count, dim3(nblk), dim3(kBlock), 0, stream, n, V, labels, a.blk);
    const bool scan = nblk > kSumChunks;
    if (scan) hipLaunchKernelGGL(kd_xent_scan, dim3(1), dim3(kBlock), 0, stream, nblk, a.blk);
    hipLaunchKernelGGL(kd_xent_map, dim3(nblk), dim3(kBlock), 0, stream, a, 1, scan, labels, loss);
  }
  if (n > 0) {
    switch (a.dp) {
      case 32: launch_forward<T, 32>(a, need_x, features, table, loss, stream); break;
      case 64: launch_forward<T, 64>(a, need_x, features, table, loss, stream); break;
      case 128: launch_forward<T, 128>(a, need_x, features, table, loss, stream); break;
      default: launch_forward<T, 256>(a, need_x, features, table, loss, stream); break;
    }
  }
  if (reduction != 0)
    hipLaunchKernelGGL(kd_xent_sum, dim3(n > 16 * kBlock ? kReduceBlocks : 1), dim3(kBlock), 0,
                       stream, a, loss);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    return set_error(KD_ERR_LAUNCH, "surface_cross_entropy: %s", hipGetErrorString(e));
  return KD_OK;
}

template <typename T>
int backward(int64_t n, int64_t V, int D, const int64_t *labels, double scale, int reduction,
             int need_x, int need_e, const float *grad, T *gx, T *ge, void *state,
             size_t state_bytes, void *scratch, size_t scratch_bytes, hipStream_t stream) {
  const int rc = check(n, V, D, scale, reduction);
  if (rc != KD_OK) return rc;
  KD_CHECK_ARG(grad || (n == 0 && reduction == 0), "surface_cross_entropy: grad_loss is NULL");
  KD_CHECK_ARG(n == 0 || labels, "surface_cross_entropy: NULL input");
  KD_CHECK_ARG((!gx || need_x) && (!ge || need_e),
               "surface_cross_entropy: a gradient that the forward call did not prepare");
  Args a = shape(n, V, D, Form<T>::np, scale, reduction);
  const size_t ns = lay_state(a, Form<T>::np, need_x, need_e, state);
  const size_t nw = lay_backward(a, Form<T>::np, ge != nullptr, scratch);
  if (!state || state_bytes < ns || !scratch || scratch_bytes < nw)
    return set_error(KD_ERR_WORKSPACE, "workspace too small: %zu < %zu or %zu < %zu", state_bytes,
                     ns, scratch_bytes, nw);
  KD_CHECK_ARG((((uintptr_t)state | (uintptr_t)scratch) & 255u) == 0,
               "surface_cross_entropy: state and scratch must be aligned to 256 bytes");
  ProfScope prof(K_XENT_BWD, stream);
  if (ge && reduction == 0)
    hipLaunchKernelGGL(kd_xent_rowgrad,
                       dim3((unsigned)std::max(grad_blocks(a.npad), 1)),
                       dim3(kBlock), 0, stream, a, sizeof(T) == 4, grad);
  switch (a.dp) {
    case 32: launch_backward<T, 32>(a, labels, grad, gx, ge, stream); break;
    case 64: launch_backward<T, 64>(a, labels, grad, gx, ge, stream); break;
    case 128: launch_backward<T, 128>(a, labels, grad, gx, ge, stream); break;
    default: launch_backward<T, 256>(a, labels, grad, gx, ge, stream); break;
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    return set_error(KD_ERR_LAUNCH, "surface_cross_entropy bwd: %s", hipGetErrorString(e));
  return KD_OK;
}

}  // namespace xent
}  // namespace kd

#define KD_XENT(SFX, T)                                                                           \
  extern "C" int kd_surface_xent_forward_##SFX(                                                   \
      int64_t n, int64_t rows, int channels, const void *features, const void *embeddings,        \
      const int64_t *labels, double scale, int reduction, int need_features, int need_embeddings, \
      float *loss, void *state, size_t state_bytes, void *scratch, size_t scratch_bytes,          \
      void *stream) {                                                                             \
    return kd::xent::forward<T>(n, rows, channels, (const T *)features, (const T *)embeddings,    \
                                labels, scale, reduction, need_features, need_embeddings, loss,   \
                                state, state_bytes, scratch, scratch_bytes, (hipStream_t)stream); \
  }                                                                                               \
  extern "C" int kd_surface_xent_backward_##SFX(                                                  \
      int64_t n, int64_t rows, int channels, const int64_t *labels, double scale, int reduction,  \
      int need_features, int need_embeddings, const float *grad_loss, void *grad_features,        \
      void *grad_embeddings, void *state, size_t state_bytes, void *scratch,                      \
      size_t scratch_bytes, void *stream) {                                                       \
    return kd::xent::backward<T>(n, rows, channels, labels, scale, reduction, need_features,      \
                                 need_embeddings, grad_loss, (T *)grad_features,                  \
                                 (T *)grad_embeddings, state, state_bytes, scratch,               \
                                 scratch_bytes, (hipStream_t)stream);                             \
  }
