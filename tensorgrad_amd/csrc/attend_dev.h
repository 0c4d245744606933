// Device code shared by the attention kernels (k_attend.hip, k_attend_grad.hip, k_attend_small.hip).
//
// Products of f32 operands run on the f16 matrix instructions: a value times a power of two that puts its tile's (or row's)
// largest at 2^14 is split as hi + lo of 11 bits each, and a b = hi hi + hi lo + lo hi, accumulated in f32. The product
// left out and the two residues are at most 3 * 2^-22 of |a b|; a value 2^-15 of the largest and below loses bits of its
// lo part, an error of 2^-40 of the largest. Three products at the f16 rate stand for one f32 product: 443 TFLOP/s of a
// measured 1329, where the f32 matrix instruction reaches 154.
//
// Fragments of a 16 x 16 x 32 product: lane l holds row (A) or column (B) l % 16 and k = 8 g + 0..7, g = l / 16; a result's
// register r holds row 4 g + r of column l % 16. One fragment of a wavefront is 1 KiB. A wavefront's own 16 rows (queries, or
// keys) are the columns, so that a lane's results belong to ONE of them: running maxima and sums are lane arithmetic and two
// exchanges. Two blocks of scores, tile rows 0..15 and 16..31, are the next product's B fragment as they stand, if its A
// fragments take their k in the same order: rows 4 g + 0..3, then 16 + 4 g + 0..3.
//
// 32 columns a wavefront (32 x 32 x 16) would read fragments from LDS half as often, but their operands and results take the
// registers of a SIMD's one or two wavefronts, which then wait for every product: measured slower in every case but the
// gradients of head size 32 without documents (4 %); those of head size 128 took half as long again.
#pragma once
#include "kernels.h"
#include "sequence.h"

namespace tgk {
namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 32;          // rows of a tile
constexpr int kFrag = 512;         // halves of a fragment (1 KiB)
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kNone = -INFINITY, kLowest = -0x1.fffffep127f;

// What the kernels need to know of a packed tile. One power of two serves all its rows, that of the largest, unless they
// differ by more than 2^12 (uneven): then every row has its own, and what was multiplied by it takes the row's `rel`, the
// tile's over the row's, afterwards. So a row keeps its precision whatever its neighbours are. odd: infinities, NaN or rows
// 2^90 apart: blocks that walk such a tile, or have such rows of their own, run in plain f32.
struct TileInfo {
  float scale, inv;                // power of two on the largest row's values, and its inverse
  int uneven, odd;
  int dmin, dmax;                  // documents of its rows (>= 0 ones; none: dmin > dmax)
  int same;                        // all rows have one document
  int pad;
};

// What a block needs of each row of a tile it walks, 32 values each (integers as bits), 2 KiB that come with the fragments
// into LDS: of queries and of keys. Row S_INFO: the TileInfo of the first operand (q, k) and eight words on the second's (dy,
// v). From LDS, because a load from memory inside the loop would wait for the next tile's fragments, which are ahead of it.
// QS_DOT: dot(dy, y) share; QS_BELOW: sees keys below.
enum { QS_TOP, QS_SHARE, QS_DOT, QS_POS, QS_SLOPE, QS_BELOW, QS_DOC, QS_RELQ, QS_RELG, S_INFO, kSide = 16 };
enum { KS_DOC, KS_RELK, KS_RELV };
constexpr int kSideFrags = kSide * kTile * 4 / 1024;

__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(min(max(e, -126), 127) + 127) << 23); }
__device__ __forceinline__ int exponent(float x) { return (int)((__float_as_uint(x) >> 23) & 255) - 127; }   // floor(log2 |x|)
// A product that is rounded before it is added to.
__device__ __forceinline__ float rounded_mul(float x, float y) {
#pragma clang fp contract(off)
  return x * y;
}
// What a score is made of: the queries' values take the factor `part` (0.5 to 1, rounded once, wherever they are split), so that
// the sum of products times 2^exp is q.k scale log2(e), or q.k scale / cap, without a rounding. That makes a score the same
// number in every walk, forward and backward (but for low parts below f16's steps, 2^-27 of a row's largest), and its distance
// to the row's largest exact: with a rounded factor inside a fused multiply-add that distance would be off by half a step of the
// largest, a factor of 2^128 for scores of 2^32.
struct Score {
  float part;
  int exp;
};
__device__ __forceinline__ Score score_parts(const AttendDesc& a) {
  const float c = a.cap > 0 ? a.scale / a.cap : a.scale * kLog2e;
  return {__builtin_amdgcn_frexp_mantf(c), __builtin_amdgcn_frexp_expf(c)};
}
// The score of x (sum of products, or its tanh) for f, in log2.
__device__ __forceinline__ float score_of(bool slopes, float x, float f, float slope, int far) {
  return slopes ? fmaf(x, f, -rounded_mul(slope, fabsf((float)far))) : rounded_mul(x, f);
}
// 2^e of a sum of products. Rows of 1e-19, or of 1e25, take it out of f32's range: kept within (pow2), it leaves such scores next
// to 0, or past f32's range, and a sum of 0 or a hidden key's minus infinity as they are.
__device__ __forceinline__ float score_unit(const Score& s, int e) { return pow2(s.exp + e); }
// The same of dP: a sum of 0 stays 0.
__device__ __forceinline__ float dot_unit(int e) { return __builtin_amdgcn_ldexpf(1.0f, min(e, 127)); }

// hi and lo of two values.
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  const f32x2 v = {x, y};
  hi = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, half2v));
  float rx, ry;
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(rx) : "v"(hi), "v"(x));
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(ry) : "v"(hi), "v"(y));
  const f32x2 r = {rx, ry};
  lo = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, half2v));
}
__device__ __forceinline__ void split8(const float* x, half8& hi, half8& lo) {
  u32x4 a, b;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t p, q;
    split2(x[2 * i], x[2 * i + 1], p, q);
    a[i] = p;
    b[i] = q;
  }
  hi = __builtin_bit_cast(half8, a);
  lo = __builtin_bit_cast(half8, b);
}

__device__ __forceinline__ f32x4 mfma(half8 a, half8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// tanh. Up to kFlat by an odd polynomial (least squares in the relative error: 0.16 * 2^-24 off, 1.4 with f32's roundings);
// above by 1 - e^-2x, which does not cancel there.
constexpr float kFlat = 0.625f;
__device__ __forceinline__ float tanh_flat(float x) {
  const float q = x * x;
  const float r = fmaf(q, fmaf(q, fmaf(q, fmaf(q, -0.00570404f, 0.02063786f), -0.05373916f), 0.13331432f), -0.33333281f);
  return fmaf(x * q, r, x);
}
__device__ __forceinline__ float tanh_of(float x) {
  const float z = fabsf(x), e = __builtin_amdgcn_exp2f(-2 * kLog2e * z);
  const float far = copysignf((1 - e) * __builtin_amdgcn_rcpf(1 + e), x);
  return z < kFlat ? tanh_flat(x) : far;
}
// What the queries of one batch entry see, wave-uniform.
struct Sight {
  int n, first, prefix;            // keys that are there; position of query 0; keys every query sees
  const int32_t* doc;
  bool causal, positional;
};
__device__ __forceinline__ Sight sight(const AttendDesc& a, int b) {
  Sight s;
  s.n = a.lengths ? min(max(a.lengths[b], 0), a.Tk) : a.Tk;
  s.first = s.n - a.Tq;
  s.prefix = a.prefix ? a.prefix[b] : 0;
  s.doc = a.documents ? a.documents + (int64_t)b * a.Tk : nullptr;
  s.causal = a.causal;
  s.positional = a.positional;
  return s;
}
// A query at position p sees the keys below this, of its document.
__device__ __forceinline__ int sees_below(const Sight& s, int p) {
  if (s.positional && p < 0) return 0;
  return s.causal ? min(s.n, max(p + 1, s.prefix)) : s.n;
}
__device__ __forceinline__ int doc_at(const Sight& s, int p) { return s.doc && p >= 0 ? s.doc[p] : -1; }   // negative: sees nothing
// Does it see any: then, where positions matter, the key at its own. From the masks, not from sums or maxima, which NaN and
// minus infinities in what is seen empty as well.
__device__ __forceinline__ bool sees_any(const Sight& s, int below, int doc) { return below > 0 && (!s.doc || doc >= 0); }
// A row's softmax for its gradients, two values: P = exp2(score - top) share. top is the logarithm of the sum, and share what its
// rounding leaves (close to 1), up to 2^24, where its steps reach 2; above, top is the largest score itself and share 1 / sum. A row
// that sees nothing: exp2(score - inf) = 0.
__device__ __forceinline__ void write_stats(const AttendDesc& a, int64_t row, bool none, float m, float sum) {
  const float l = __builtin_amdgcn_logf(sum), lse = m + l;
  const bool far = fabsf(m) >= 0x1p24f;
  a.stats[2 * row] = none ? INFINITY : far ? m : lse;
  a.stats[2 * row + 1] = none ? 1.0f : far ? 1.0f / sum : __builtin_amdgcn_exp2f((lse - m) - l);
}

// Rows [lo, hi] of positions against keys [j0, j0 + 32): does any pair see, do all.
struct Span {
  int pmin, pmax, dmin, dmax;      // positions and documents (>= 0) of the rows
  bool same;                       // one document
};
__device__ __forceinline__ bool any_seen(const Sight& s, const Span& q, const TileInfo& k, int j0) {
  if (j0 >= s.n || (s.positional && q.pmax < 0)) return false;
  if (s.causal && j0 > q.pmax && j0 >= s.prefix) return false;
  return !s.doc || (k.dmin <= q.dmax && q.dmin <= k.dmax);
}
__device__ __forceinline__ bool all_seen(const Sight& s, const Span& q, const TileInfo& k, int j0) {
  if (j0 + kTile > s.n || (s.positional && q.pmin < 0)) return false;
  if (s.causal && j0 + kTile - 1 > q.pmin && j0 + kTile > s.prefix) return false;
  return !s.doc || (k.same && q.same && k.dmin == q.dmin);
}

// N fragments from memory straight into LDS (lane l's 16 bytes land at base + 16 l) by eight wavefronts, wavefront w's at src
// and lds + 1024 w. In inline assembly, so that the compiler does not drain every load before the next LDS read; the kernels
// wait (vmcnt) and meet (barrier) themselves.
__device__ __forceinline__ void frag_to_lds(const char* src, uint32_t lds, uint32_t lane16) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(lane16), "s"(src), "{m0}"(lds));
}
template <int N>
__device__ __forceinline__ void frags_to_lds(const char* src, uint32_t lds, uint32_t lane16, int w) {
#pragma unroll
  for (int f = 0; f < N / 8; ++f) frag_to_lds(src + f * 8192, lds + f * 8192, lane16);
  if (N % 8 && w < N % 8) frag_to_lds(src + N / 8 * 8192, lds + N / 8 * 8192, lane16);
}
__device__ __forceinline__ void loads_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}

__device__ __forceinline__ float finite_abs(float x) {
  x = fabsf(x);
  return x < INFINITY ? x : 0.0f;
}

// Sums over several tiles in one accumulator: the weights (f16 parts of x 2^e) times a tile packed at 2^t are in units of
// 2^-(e + t), which must be the accumulator's 2^-c. A lane's c only falls, when a tile's largest weight `big` would pass
// 2^14, or e f32's exponents (weights below 2^-113 of large rows): what comes later and is smaller is rounded like the largest
// of the sum (2^-37 of it), what was hidden has weight 0 and counts for nothing. c starts at kUnset, the accumulator at 0.
// Returns e; *change: the accumulator's factor.
constexpr int kUnset = 1000;
__device__ __forceinline__ int fit_unit(int& c, float big, int t, float* change) {
  int e = c - t;
  if (big > 0 && e > min(14 - exponent(big), 127)) {
    e = min(12 - exponent(big), 125);
    *change *= __builtin_amdgcn_ldexpf(1.0f, e + t - c);   // 0 where acc no longer counts
    c = e + t;
  }
  return e;
}
__device__ __forceinline__ half8 frag(const _Float16* L, int f) { return *(const half8*)(L + f * kFrag + (threadIdx.x & 63) * 8); }
// Over the four lanes l % 16 + 0, 16, 32, 48 of a column.
__device__ __forceinline__ float groups_max(float x) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float groups_sum(float x) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// B fragments of 16 rows times `mul` (lane l: row l % 16), each row with its own power of two; returns its exponent. *infinite:
// the row holds an infinity, which has no hi and lo parts.
template <int N>
__device__ __forceinline__ int load_rows(const float* row, bool valid, int n, bool wide, float mul, half8 (&hi)[N], half8 (&lo)[N],
                                         bool* infinite = nullptr) {
  const int g = (threadIdx.x >> 4) & 3;
  float x[N][8], m = 0;
#pragma unroll
  for (int c = 0; c < N; ++c) {
    const int d = 32 * c + 8 * g;
    if (wide) {
      f32x4 u = {}, w = {};
      if (valid && d < n) {
        u = *(const f32x4*)(row + d);
        w = *(const f32x4*)(row + d + 4);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) { x[c][i] = u[i]; x[c][4 + i] = w[i]; }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[c][i] = valid && d + i < n ? row[d + i] : 0.0f;
    }
  }
#pragma unroll
  for (int c = 0; c < N; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(x[c][i] * mul));
  m = groups_max(m);
  if (infinite) *infinite = m == INFINITY;
  const int e = m > 0 ? min(14 - exponent(m), 126) : 0;
  const float s = pow2(e);
#pragma unroll
  for (int c = 0; c < N; ++c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[c][i] = x[c][i] * mul * s;
    split8(x[c], hi[c], lo[c]);
  }
  return e;
}
// x = A fragments (N chunks of 32 features, two blocks of 16 rows each, from fragment f0) times B fragments; a chunk's
// fragments are read while the chunk before is multiplied. Queries against keys or keys against queries (KQ), the products are
// added in the same order: k lo q hi, k hi q lo, k hi q hi.
template <bool KQ, int N>
__device__ __forceinline__ void scores(const _Float16* L, int f0, const half8 (&bh)[N], const half8 (&bl)[N], float (&x)[8]) {
  f32x4 z[2] = {};
  half8 a[2][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) a[0][i] = frag(L, f0 + i);
#pragma unroll
  for (int c = 0; c < N; ++c) {
    const half8* u = a[c & 1];
    if (c + 1 < N)
#pragma unroll
      for (int i = 0; i < 4; ++i) a[(c + 1) & 1][i] = frag(L, f0 + 4 * c + 4 + i);
    z[0] = KQ ? mfma(u[1], bh[c], z[0]) : mfma(u[0], bl[c], z[0]);
    z[1] = KQ ? mfma(u[3], bh[c], z[1]) : mfma(u[2], bl[c], z[1]);
    z[0] = KQ ? mfma(u[0], bl[c], z[0]) : mfma(u[1], bh[c], z[0]);
    z[1] = KQ ? mfma(u[2], bl[c], z[1]) : mfma(u[3], bh[c], z[1]);
    z[0] = mfma(u[0], bh[c], z[0]);
    z[1] = mfma(u[2], bh[c], z[1]);
    __builtin_amdgcn_sched_barrier(0);
  }
#pragma unroll
  for (int q = 0; q < 8; ++q) x[q] = z[q / 4][q % 4];
}
// Both products of a pair, step by step in turn.
template <bool KQ, int N>
__device__ __forceinline__ void pair(const _Float16* L, int f0, const half8 (&bh)[N], const half8 (&bl)[N], float (&x)[8], int f1,
                                       const half8 (&ch)[N], const half8 (&cl)[N], float (&y)[8]) {
  f32x4 z[4] = {};
  half8 a[2][8];
  auto read = [&](int c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[c & 1][i] = frag(L, f0 + 4 * c + i);
      a[c & 1][4 + i] = frag(L, f1 + 4 * c + i);
    }
  };
  read(0);
#pragma unroll
  for (int c = 0; c < N; ++c) {
    const half8* u = a[c & 1];
    if (c + 1 < N) read(c + 1);
    z[0] = KQ ? mfma(u[1], bh[c], z[0]) : mfma(u[0], bl[c], z[0]);
    z[1] = KQ ? mfma(u[3], bh[c], z[1]) : mfma(u[2], bl[c], z[1]);
    z[2] = mfma(u[5], ch[c], z[2]);
    z[3] = mfma(u[7], ch[c], z[3]);
    z[0] = KQ ? mfma(u[0], bl[c], z[0]) : mfma(u[1], bh[c], z[0]);
    z[1] = KQ ? mfma(u[2], bl[c], z[1]) : mfma(u[3], bh[c], z[1]);
    z[2] = mfma(u[4], cl[c], z[2]);
    z[3] = mfma(u[6], cl[c], z[3]);
    z[0] = mfma(u[0], bh[c], z[0]);
    z[1] = mfma(u[2], bh[c], z[1]);
    z[2] = mfma(u[4], ch[c], z[2]);
    z[3] = mfma(u[6], ch[c], z[3]);
    __builtin_amdgcn_sched_barrier(0);
  }
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    x[q] = z[q / 4][q % 4];
    y[q] = z[2 + q / 4][q % 4];
  }
}
// acc += A fragments (N blocks of 16 features, from fragment f0) times the split of x * scale, read as above.
template <int N>
__device__ __forceinline__ void accumulate(f32x4 (&acc)[N], const float (&x)[8], float scale, const _Float16* L, int f0) {
  half8 a[2][4], bh, bl;
#pragma unroll
  for (int i = 0; i < 4; ++i) a[0][i] = frag(L, f0 + i);
  float z[8];
#pragma unroll
  for (int q = 0; q < 8; ++q) z[q] = x[q] * scale;
  split8(z, bh, bl);
#pragma unroll
  for (int d = 0; d < N; d += 2) {
    const half8* u = a[d / 2 & 1];
    if (d + 2 < N)
#pragma unroll
      for (int i = 0; i < 4; ++i) a[(d / 2 + 1) & 1][i] = frag(L, f0 + 2 * d + 4 + i);
    acc[d] = mfma(u[1], bh, acc[d]);
    acc[d + 1] = mfma(u[3], bh, acc[d + 1]);
    acc[d] = mfma(u[0], bl, acc[d]);
    acc[d + 1] = mfma(u[2], bl, acc[d + 1]);
    acc[d] = mfma(u[0], bh, acc[d]);
    acc[d + 1] = mfma(u[2], bh, acc[d + 1]);
    __builtin_amdgcn_sched_barrier(0);
  }
}
template <int N>
__device__ __forceinline__ void rescale(f32x4 (&acc)[N], float change) {
  if (__builtin_expect(!__any(change != 1), 1)) return;   // the hint keeps the moves for it out of the common path
#pragma unroll
  for (int d = 0; d < N; ++d)
#pragma unroll
    for (int q = 0; q < 4; ++q) acc[d][q] *= change;
}
__device__ __forceinline__ void per_row(float (&x)[8], const float* rel, int g) {
#pragma unroll
  for (int q = 0; q < 8; ++q) x[q] *= rel[16 * (q / 4) + 4 * g + q % 4];
}
__device__ __forceinline__ float largest(const float (&x)[8]) {
  float m = 0;
#pragma unroll
  for (int q = 0; q < 8; ++q) m = fmaxf(m, fabsf(x[q]));
  return groups_max(m);
}
// x = tanh(x u), all 8; the polynomial alone where no lane needs more
__device__ __forceinline__ void tanh_all(float (&x)[8], float u) {
  float m = 0;
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    x[q] *= u;
    m = fmaxf(m, fabsf(x[q]));
  }
  if (__any(m >= kFlat)) {
#pragma unroll
    for (int q = 0; q < 8; ++q) x[q] = tanh_of(x[q]);
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q) x[q] = tanh_flat(x[q]);
  }
}
template <int N>
__device__ __forceinline__ void store_row(float* row, const f32x4 (&acc)[N], int c, float scale, int n, bool wide, int g) {
#pragma unroll
  for (int d = 0; d < N; ++d) {
    const int at = 16 * d + 4 * g;
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = __builtin_amdgcn_ldexpf(acc[d][e], -c) * scale;
    if (wide) {
      if (at < n) *(f32x4*)(row + at) = v;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) if (at + e < n) row[at + e] = v[e];
    }
  }
}

// Operand x's (0 or 1) TileInfo from a side block, wave-uniform.
__device__ __forceinline__ TileInfo side_info(const float* side, int x) {
  const int* p = (const int*)(side + S_INFO * kTile + 8 * x);
  auto u = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
  return {__int_as_float(u(p[0])), __int_as_float(u(p[1])), u(p[2]), u(p[3]), u(p[4]), u(p[5]), u(p[6]), 0};
}
// Does a query with these bounds see key z of the tile at j0. Without branches: with the document read behind the other
// conditions, `if (!seen) x[q] = 0` comes out of the compiler wrong (right in its IR; in the machine code the block for keys of
// other documents is empty, their 0 written before a copy of the whole vector undoes it), and hidden keys keep their values.
__device__ __forceinline__ bool key_seen(const Sight& s, const float* side, int j0, int z, int below, int doc) {
  const int id = __float_as_int(side[KS_DOC * kTile + z]);
  return (j0 + z < below) & (!s.doc | ((doc >= 0) & (id == doc)));
}
// First and one past the last of the tiles [t0, t1) whose documents meet [lo, hi] (all of them without documents); odd: one
// of those is, or the block's own rows are (`own`, of each lane). By the whole block.
struct Range {
  int t0, t1;
  bool odd;
};
__device__ __forceinline__ Range tile_range(const Sight& s, int t0, int t1, const TileInfo* docs, const TileInfo* x, const TileInfo* y,
                                            int dmin, int dmax, bool own, int (&buf)[5]) {
  const int tid = threadIdx.x;
  if (tid < 5) buf[tid] = tid == 0 || tid == 2 ? INT32_MAX : tid == 4 ? 0 : INT32_MIN;
  __syncthreads();
  if ((tid & 63) == 0 && s.doc) {
    atomicMin(&buf[0], dmin);
    atomicMax(&buf[1], dmax);
  }
  if (own) atomicOr(&buf[4], 1);
  __syncthreads();
  const int lo = buf[0], hi = buf[1];
  int first = INT32_MAX, end = INT32_MIN, odd = 0;
  for (int t = t0 + tid; t < t1; t += 256) {
    if (s.doc && !(docs[t].dmin <= hi && lo <= docs[t].dmax)) continue;
    first = min(first, t);
    end = max(end, t + 1);
    odd |= x[t].odd | y[t].odd;
  }
  if (first != INT32_MAX) {
    atomicMin(&buf[2], first);
    atomicMax(&buf[3], end);
    if (odd) atomicOr(&buf[4], 1);
  }
  __syncthreads();
  Range r;
  r.t0 = __builtin_amdgcn_readfirstlane(buf[2]);
  r.t1 = __builtin_amdgcn_readfirstlane(buf[3]);
  r.odd = __builtin_amdgcn_readfirstlane(buf[4]) != 0;
  if (r.t0 >= r.t1) r.t0 = r.t1 = 0;
  return r;
}

// ---- plain f32, for blocks that walk an odd tile: a wavefront takes one row at a time, a lane a pair ----

struct PlainPair {
  float score, slack;              // log2; 1 - tanh^2
};
__device__ __forceinline__ float plain_dot(const float* x, const float* y, int n) {
  float s = 0;
#pragma unroll 1
  for (int d = 0; d < n; ++d) s = fmaf(x[d], y[d], s);
  return s;
}
__device__ __forceinline__ PlainPair plain_score(const AttendDesc& a, float dot, float slope, int far) {
  PlainPair r;
  float x = dot * a.scale, t = 0;
  if (a.cap > 0) {
    t = tanh_of(x / a.cap);
    x = a.cap * t;
  }
  r.score = fmaf(-slope, fabsf((float)far), x * kLog2e);
  r.slack = fmaf(-t, t, 1.0f);
  return r;
}
// acc[e] += w of each lane k times rows(k)[64 e + lane], lanes of weight 0 left out
template <class RowOf>
__device__ __forceinline__ void plain_add(float (&acc)[2], float w, RowOf row_of, int n) {
  const int lane = threadIdx.x & 63;
#pragma unroll 1
  for (int k = 0; k < 64; ++k) {
    const float x = __shfl(w, k);
    if (x == 0) continue;
    const float* r = row_of(k);
#pragma unroll
    for (int e = 0; e < 2; ++e) if (64 * e + lane < n) acc[e] = fmaf(x, r[64 * e + lane], acc[e]);
  }
}

// A block's slab (batch entry and key head) and its item of the slab's, in the order that blocks start. Hardware deals block
// ids to the 8 XCDs in turn; a slab stays on one XCD (or 2, 4, 8 of them where there are fewer slabs), whose L2 then holds
// its packed tiles, and every XCD gets long and short items alike.
__device__ __forceinline__ void place(uint32_t id, uint32_t slabs, int& slab, int& item) {
  const uint32_t x = id % 8, k = id / 8;
  if (slabs % 8 == 0) {
    slab = x + 8 * (k % (slabs / 8));
    item = k / (slabs / 8);
  } else if (8 % slabs == 0) {
    slab = x % slabs;
    item = k * (8 / slabs) + x / slabs;
  } else {
    slab = id % slabs;
    item = id / slabs;
  }
}
}  // namespace

// ---- packing -----------------------------------------------------------------------------------

// One operand as tiles of 32 rows: row fragments (k = features) and / or column fragments (k = rows).
struct PackJob {
  Rows x;
  int n, G, rows, tiles;           // features; heads that share a key head; rows = positions * G; tiles
  _Float16 *rowf, *colf;           // [slab][tile][D padded / 8][512], or null
  TileInfo* info;                  // [slab][tile]
  bool query;                      // rows are queries, else keys
  float* side;                     // [slab][tile][kSide][32]: what a block needs of each row of the tile, see below
  int rel;                         // where this operand's rel goes
  bool second;                     // and its info
  bool ids;                        // this job also writes the rows' documents and the rest
  bool score;                      // queries: the row fragments take their factor (score_parts)
  Rows y;                          // of the gradient dy (ids of queries, times their share): y's rows for its dot products
};
// The attention's operands as packed for one pass, in the workspace.
struct Packs {
  int n;
  int Hk, tiles;                   // tiles: the most of any job
  bool wide;                       // every operand's rows are 16-byte aligned and whole 16-byte pieces
  PackJob job[4];
  AttendDesc a;
};
void attend_pack(Packs p, int DP, hipStream_t st);
// Blocks for `items` of each slab: those of place() beyond the last item end at once.
inline unsigned place_grid(int64_t slabs, int64_t items) {
  return (unsigned)(slabs % 8 != 0 && 8 % slabs == 0 ? (items + 8 / slabs - 1) / (8 / slabs) * 8 : slabs * items);
}
inline int attend_dp(const AttendDesc& a) { return (max(a.D, a.Dv) + 31) / 32 * 32; }
// Rows that k_attend_small.hip holds (query rows of a key head, and keys); 0: not for it.
inline int attend_small_rows(const AttendDesc& a) {
  const int64_t n = max((int64_t)(a.H / a.Hk) * a.Tq, (int64_t)a.Tk);
  const int dp = attend_dp(a);
  return n <= 32 && dp <= 64 ? 32 : n <= 64 && dp <= 32 ? 64 : 0;
}
void attend_small_forward(const AttendDesc& a, hipStream_t st);
void attend_small_grad(const AttendGradDesc& g, hipStream_t st);
inline bool attend_wide(const Rows& x, int n) {
  return ((uintptr_t)x.p & 15) == 0 && x.b % 4 == 0 && x.h % 4 == 0 && x.t % 4 == 0 && n % 8 == 0;
}

}  // namespace tgk
