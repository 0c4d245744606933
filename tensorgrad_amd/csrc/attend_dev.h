// Device code shared by the attention kernels (k_attend.hip, k_attend_grad.hip).
//
// Products of f32 operands run on the f16 matrix instructions: a value times a power of two that puts its tile's (or row's)
// largest at 2^14 is split as hi + lo of 11 bits each, and a b = hi hi + hi lo + lo hi, accumulated in f32. The product
// left out and the two residues are at most 3 * 2^-22 of |a b|; a value 2^-15 of the largest and below loses bits of its
// lo part, an error of 2^-40 of the largest. Three products at the f16 rate stand for one f32 product: 443 TFLOP/s of a
// measured 1329, where the f32 matrix instruction reaches 154.
//
// Fragments of a 32 x 32 x 16 product: lane l holds row (A) or column (B) l % 32 and k = 8 (l / 32) + 0..7; a result's
// register r holds row 8 (r / 4) + 4 (l / 32) + r % 4 of column l % 32. One fragment of a wavefront is 1 KiB. The scores'
// registers 8 s .. 8 s + 7 are the B fragment of the next product's k step s as they stand, if that product's A fragments
// take their k in the same order: rows 16 s + 4 h + 0..3 and 16 s + 8 + 4 h + 0..3 for lane half h.
#pragma once
#include "kernels.h"
#include "sequence.h"

namespace tgk {
namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 32;          // rows of a tile
constexpr int kFrag = 512;         // halves of a fragment (1 KiB)
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr float kNone = -INFINITY;

// What the kernels need to know of a packed tile. irregular: it holds infinities, NaN or rows whose largest values differ
// by more than 2^20, so that one scale cannot serve it: it is multiplied in f32, value by value.
struct TileInfo {
  float scale;                     // power of two on the packed values
  int norm;                        // 2^norm bounds the rows' 2-norms
  int irregular;
  int dmin, dmax;                  // documents of its rows (>= 0 ones; none: dmin > dmax)
  int same;                        // all rows have one document
  int pad[2];
};

__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(min(max(e, -126), 127) + 127) << 23); }
__device__ __forceinline__ int exponent(float x) { return (int)((__float_as_uint(x) >> 23) & 255) - 127; }   // floor(log2 |x|)

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

__device__ __forceinline__ f32x16 mfma(half8 a, half8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// Over lanes l and l ^ 32, which hold the two halves of a row.
__device__ __forceinline__ float halves_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// tanh, to a few units of its own last place: an odd rational form (continued fraction to x^5) where 1 - e^-2x would
// cancel, else that. The rational form is off by less than 2^-25 of the value up to 0.625.
__device__ __forceinline__ float tanh_of(float x) {
  const float z = fabsf(x), q = x * x;
  const float e = __builtin_amdgcn_exp2f(-2 * kLog2e * z);
  const bool small = z < 0.625f;
  const float num = small ? z * fmaf(q, fmaf(q, 1.0f, 105.0f), 945.0f) : 1 - e;
  const float den = small ? fmaf(q, fmaf(q, 15.0f, 420.0f), 945.0f) : 1 + e;
  const float r = __builtin_amdgcn_rcpf(den);
  return copysignf(num * r, x);
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

// 1 KiB fragments from memory straight into LDS: lane l's 16 bytes land at base + 16 l. In inline assembly, so that the
// compiler does not drain every load before the next LDS read; the kernels wait (vmcnt) and meet (barrier) themselves.
__device__ __forceinline__ void frag_to_lds(const _Float16* src, uint32_t lds, uint32_t lane16) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(lane16), "s"(src), "{m0}"(lds));
}
__device__ __forceinline__ void loads_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}

// Row r of tile-ordered rows: r = i G + g is position i of the g-th query head that shares the key head (keys: G = 1).
struct RowMap {
  const float* p;                  // of (b, first head)
  int64_t h, t;
  FastDiv group;
  __device__ __forceinline__ const float* row(int r) const {
    const uint32_t i = fastdiv((uint32_t)r, group), g = (uint32_t)r - i * group.d;
    return p + g * h + i * t;
  }
};
__device__ __forceinline__ RowMap row_map(const Rows& x, int b, int head, const FastDiv& group) {
  return {x.p + b * x.b + head * x.h, x.h, x.t, group};
}

// An exponent that bounds a 2-norm: values of at most `top`, whose squares relative to it sum to sq.
__device__ __forceinline__ int norm_exponent(float top, float sq) {
  return top > 0 ? exponent(top) + 1 + (exponent(sq) + 2) / 2 : -126;
}
__device__ __forceinline__ float finite_abs(float x) {
  x = fabsf(x);
  return x < INFINITY ? x : 0.0f;
}

// B fragments of 32 rows (lane l: row l % 32), each row with its own power of two; returns its exponent, and in *norm a bound
// on its 2-norm. wide: rows are 16-byte aligned and n a multiple of 8.
template <int KC>
__device__ __forceinline__ int load_rows(const float* row, bool valid, int n, bool wide, half8 (&hi)[KC], half8 (&lo)[KC],
                                         int* norm = nullptr) {
  const int h = (threadIdx.x >> 5) & 1;
  float x[KC][8];
#pragma unroll
  for (int c = 0; c < KC; ++c) {
    const int d = 16 * c + 8 * h;
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
  float m = 0;
#pragma unroll
  for (int c = 0; c < KC; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, finite_abs(x[c][i]));   // the others stay what they are
  m = halves_max(m);
  if (norm) {
    float sq = 0;
    const float inv = m > 0 ? 1.0f / fmaxf(m, 1e-37f) : 0.0f;
#pragma unroll
    for (int c = 0; c < KC; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float z = finite_abs(x[c][i]) * inv;
        sq = fmaf(z, z, sq);
      }
    *norm = norm_exponent(m, halves_sum(sq));
  }
  const int e = m > 0 ? min(14 - exponent(m), 126) : 0;
  const float s = pow2(e);
#pragma unroll
  for (int c = 0; c < KC; ++c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[c][i] *= s;
    split8(x[c], hi[c], lo[c]);
  }
  return e;
}

// Products in f32, value by value, for tiles that one scale cannot serve (rare, so small code rather than fast).
// s[r] = row(8 (r / 4) + 4 h + r % 4 of the tile) . mine, for n features.
template <class RowOf>
__device__ __forceinline__ void plain_scores(f32x16& s, RowOf row_of, int rows, const float* mine, bool valid, int n) {
  const int h = (threadIdx.x >> 5) & 1;
#pragma unroll 1
  for (int q = 0; q < 16; ++q) {
    const int j = 8 * (q / 4) + 4 * h + q % 4;
    float x = 0;
    if (valid && j < rows) {
      const float* a = row_of(j);
#pragma unroll 1
      for (int d = 0; d < n; ++d) x = fmaf(a[d], mine[d], x);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = r == q ? x : s[r];
  }
}
// Sums over several tiles in one accumulator: the weights (f16 parts of x 2^e) times a tile packed at 2^t are in units of
// 2^-(e + t), which must be the accumulator's 2^-c. A lane's c only falls, when a tile's largest weight `big` would pass
// 2^14: what comes later and is smaller is rounded like the largest of the sum (2^-37 of it), what was hidden has weight 0
// and counts for nothing. c starts at kUnset, the accumulator at 0. Returns e; *change: the accumulator's factor.
constexpr int kUnset = 1000;
__device__ __forceinline__ int fit_unit(int& c, float big, int t, float* change) {
  int e = c - t;
  if (big > 0 && e > 14 - exponent(big)) {
    e = min(12 - exponent(big), 110);
    *change *= __builtin_amdgcn_ldexpf(1.0f, e + t - c);   // 0 where acc no longer counts
    c = e + t;
  }
  return e;
}
template <int DB>
__device__ __forceinline__ void rescale(f32x16 (&acc)[DB], float change) {
  if (!__any(change != 1)) return;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int q = 0; q < 16; ++q) acc[d][q] *= change;
}
// acc (columns: lanes, rows: features) += sum over the tile's rows j of row(j) * w[j] in f32, rows of weight 0 left out. The
// values go in as they are, so acc leaves its unit for the sum, and returns to it unless they are too large for it.
template <int DB, class RowOf>
__device__ __forceinline__ void plain_accumulate(f32x16 (&acc)[DB], int& c, const f32x16& w, RowOf row_of, int rows, int n) {
  const int lane = threadIdx.x & 63, h = lane >> 5;
  rescale<DB>(acc, __builtin_amdgcn_ldexpf(1.0f, c == kUnset ? 0 : -c));
#pragma unroll 1
  for (int j = 0; j < min(rows, kTile); ++j) {
    const int at = 4 * (j / 8) + j % 4;
    float x = 0;
#pragma unroll
    for (int r = 0; r < 16; ++r) x = r == at ? w[r] : x;
    x = __shfl(x, (lane & 31) + 32 * ((j / 4) & 1));
    const float* a = row_of(j);
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int d = 32 * b + 8 * (r / 4) + 4 * h + r % 4;
        if (d < n && x != 0) acc[b][r] = fmaf(x, a[d], acc[b][r]);
      }
  }
  float m = 0;
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) m = fmaxf(m, finite_abs(acc[b][r]));
  m = halves_max(m);
  if (m > 0) c = min(min(c == kUnset ? 26 - exponent(m) : c, 110 - exponent(m)), 120);
  rescale<DB>(acc, pow2(c == kUnset ? 0 : c));
}

// acc += A fragments (feature blocks x two k steps, from fragment f0 of L) times the split of x * scale
template <int DB>
__device__ __forceinline__ void accumulate(f32x16 (&acc)[DB], const f32x16& x, float scale, const _Float16* L, int f0) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    float z[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) z[q] = x[8 * ks + q] * scale;
    half8 bh, bl;
    split8(z, bh, bl);
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      const half8 ah = *(const half8*)(L + (f0 + (d * 2 + ks) * 2) * kFrag + lane * 8);
      const half8 al = *(const half8*)(L + (f0 + (d * 2 + ks) * 2 + 1) * kFrag + lane * 8);
      acc[d] = mfma(al, bh, acc[d]);
      acc[d] = mfma(ah, bl, acc[d]);
      acc[d] = mfma(ah, bh, acc[d]);
    }
  }
}
// A fragments (KC k steps, from fragment f0 of L) times B fragments
template <int KC>
__device__ __forceinline__ f32x16 scores(const _Float16* L, int f0, const half8 (&bh)[KC], const half8 (&bl)[KC]) {
  const int lane = threadIdx.x & 63;
  f32x16 x = {};
#pragma unroll
  for (int c = 0; c < KC; ++c) {
    const half8 ah = *(const half8*)(L + (f0 + 2 * c) * kFrag + lane * 8), al = *(const half8*)(L + (f0 + 2 * c + 1) * kFrag + lane * 8);
    x = mfma(al, bh[c], x);
    x = mfma(ah, bl[c], x);
    x = mfma(ah, bh[c], x);
  }
  return x;
}
__device__ __forceinline__ float largest(const f32x16& x) {   // magnitude, over a row's two lane halves
  float m = 0;
#pragma unroll
  for (int q = 0; q < 16; ++q) m = fmaxf(m, fabsf(x[q]));
  return halves_max(m);
}

// Blocks of one slab (batch entry and key head) on one XCD, whose L2 then holds its packed tiles: hardware deals block ids
// to the 8 XCDs in turn.
__device__ __forceinline__ uint32_t xcd_order(uint32_t id, uint32_t total) {
  const uint32_t per = total / 8;
  return id < per * 8 ? (id % 8) * per + id / 8 : id;
}

}  // namespace

// ---- packing -----------------------------------------------------------------------------------

// One operand as tiles of 32 rows: row fragments (k = features) and / or column fragments (k = rows).
struct PackJob {
  Rows x;
  int n, G, rows, tiles;           // features; heads that share a key head; rows = positions * G; tiles
  _Float16 *rowf, *colf;           // [slab][tile][2 KC][512], [slab][tile][4 DB][512], or null
  TileInfo* info;                  // [slab][tile]
  bool query;                      // rows are queries: their documents are those at their positions
  // of the gradient dy: y's rows for its dot products, and what the key blocks need of each row, else null
  Rows y;
  float* rowinfo;                  // [slab][tile][kRowInfo][32]
};
enum { RI_LSE, RI_DOT, RI_POS, RI_SLOPE, RI_BELOW, RI_DOC, kRowInfo = 8 };   // dot(dy, y); sees keys below; ints as bits
// The attention's operands as packed for one pass, in the workspace.
struct Packs {
  int n;
  int Hk;
  bool wide;                       // every operand's rows are 16-byte aligned and whole 16-byte pieces
  PackJob job[4];
  AttendDesc a;
};
void attend_pack(const Packs& p, int DP, hipStream_t st);
inline int attend_dp(const AttendDesc& a) { return (max(a.D, a.Dv) + 31) / 32 * 32; }
inline bool attend_wide(const Rows& x, int n) {
  return ((uintptr_t)x.p & 15) == 0 && x.b % 4 == 0 && x.h % 4 == 0 && x.t % 4 == 0 && n % 8 == 0;
}

}  // namespace tgk
