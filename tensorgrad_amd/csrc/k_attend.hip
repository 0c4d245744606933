// Masked attention for gfx950: y = softmax(scores) v, one pass over the keys with a running maximum and sum, so that no
// score reaches memory. Two ways, by the number of query rows that share a key head (G query heads times Tq):
//  * many rows: k and v are packed once into f16 hi / lo fragments (pack_tiles), then blocks of 8 wavefronts with 16 rows
//    each walk the visible key tiles (attend_tiles), four wavefronts a SIMD, so that one's products run beside the others'
//    vector work. Scores are computed transposed (keys x queries);
//  * few rows (one new token against a cache): the keys are read once, in f32, by all heads that share them (attend_few);
//    bound by memory, so split over the keys until the card is full. Without a gradient: the gradients compute scores as the
//    tiles do.
// Both split a long key axis when there are few rows (attend_join). A few dozen positions in all: k_attend_small.hip.
#include "attend_dev.h"

namespace tgk {
namespace {

// ---- packing -------------------------------------------------------------------------------------

// A block packs one tile of 32 rows: reads them once, finds their scales, writes its fragments. Rows that see nothing and
// are seen by nothing are packed as zeros, whatever they hold. Bound by memory: the seven operands of a gradient over 4096
// rows of 16 query and 4 key heads of 128 are 51 us (117 MB read, 159 MB written: 5.4 TB/s).
template <int DP>
__global__ __launch_bounds__(256) void pack_tiles(Packs p) {
  constexpr int DB = DP / 32, LD = DP + 4;
  __shared__ float x[kTile * LD];
  __shared__ float top[kTile], own[kTile];
  __shared__ int doc[kTile];
  const PackJob j = p.job[blockIdx.y];
  const int tile = blockIdx.x % p.tiles, slab = blockIdx.x / p.tiles, b = slab / p.Hk, hk = slab % p.Hk;
  if (tile >= j.tiles) return;
  const Sight s = sight(p.a, b);
  const int tid = threadIdx.x, row = tid / 8, sub = tid % 8, r = tile * kTile + row;
  const int i = r / j.G, g = r - i * j.G, pos = j.query ? s.first + i : r;
  const int id = r < j.rows ? doc_at(s, pos) : -1;
  const bool in = r < j.rows && (!s.doc || id >= 0) && (j.query ? !s.positional || pos >= 0 : pos < s.n);
  const int64_t at = b * j.x.b + (int64_t)(hk * j.G + g) * j.x.h + (int64_t)i * j.x.t;
  const bool dots = j.ids && j.query;
  const int64_t stat = 2 * (((int64_t)b * p.a.H + hk * j.G + g) * p.a.Tq + i);
  const float mul = dots && in ? p.a.stats[stat + 1] : 1.0f;
  float m = 0, dot = 0;
  bool odd = false;
#pragma unroll
  for (int c = 0; c < DB; ++c) {
    const int d = 4 * (sub + 8 * c);
    f32x4 u = {};
    if (in) {
      if (p.wide && d < j.n) u = *(const f32x4*)(j.x.p + at + d);
      if (!p.wide)
#pragma unroll
        for (int q = 0; q < 4; ++q) u[q] = d + q < j.n ? j.x.p[at + d + q] : 0.0f;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      u[q] *= mul;
      odd |= !(fabsf(u[q]) < INFINITY);
      m = fmaxf(m, finite_abs(u[q]));
    }
    *(f32x4*)(x + row * LD + d) = u;
    if (dots && in) {
      const int64_t ay = b * j.y.b + (int64_t)(hk * j.G + g) * j.y.h + (int64_t)i * j.y.t;
#pragma unroll
      for (int q = 0; q < 4; ++q) if (d + q < j.n) dot = fmaf(u[q], j.y.p[ay + d + q], dot);
    }
  }
#pragma unroll
  for (int o = 1; o < 8; o *= 2) {
    m = fmaxf(m, __shfl_xor(m, o));
    dot += __shfl_xor(dot, o);
    odd = __shfl_xor((int)odd, o) || odd;
  }
  float* side = j.side + ((int64_t)slab * j.tiles + tile) * (kSide * kTile);
  if (sub == 0) {
    top[row] = odd ? INFINITY : m;
    doc[row] = id;
    if (dots) {
      const AttendDesc& a = p.a;
      const int h = hk * j.G + g;
      side[QS_TOP * kTile + row] = in ? a.stats[stat] : INFINITY;
      side[QS_SHARE * kTile + row] = mul;
      side[QS_DOT * kTile + row] = in ? dot : 0.0f;
      side[QS_POS * kTile + row] = __int_as_float(pos);
      side[QS_SLOPE * kTile + row] = in && a.slopes ? a.slopes[h] * kLog2e : 0.0f;
      side[QS_BELOW * kTile + row] = __int_as_float(in ? sees_below(s, pos) : 0);
      side[QS_DOC * kTile + row] = __int_as_float(id);
    } else if (j.ids) {
      side[KS_DOC * kTile + row] = __int_as_float(id);
    }
  }
  __syncthreads();
  const int lane = tid & 63, w = tid >> 6, l = lane & 31;
  const float mine = top[l];
  float hi = mine, lo = mine > 0 ? mine : INFINITY;
  int dmin = doc[l] >= 0 ? doc[l] : INT32_MAX, dmax = doc[l] >= 0 ? doc[l] : INT32_MIN;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    hi = fmaxf(hi, __shfl_xor(hi, o));
    lo = fminf(lo, __shfl_xor(lo, o));
    dmin = min(dmin, __shfl_xor(dmin, o));
    dmax = max(dmax, __shfl_xor(dmax, o));
  }
  const bool bad = !(hi < INFINITY) || (hi > 0 && exponent(hi) - exponent(lo) > 90);
  const bool uneven = !bad && hi > 0 && exponent(hi) - exponent(lo) > 12, same = dmin == dmax && !__any(doc[l] < 0);
  const int e = bad || hi == 0 ? 0 : min(14 - exponent(hi), 126);
  const int64_t slot = (int64_t)slab * j.tiles + tile;
  if (tid == 0) {
    const TileInfo t = {pow2(e), pow2(-e), uneven, bad, dmin, dmax, same, 0};
    j.info[slot] = t;
    *(TileInfo*)(side + S_INFO * kTile + 8 * j.second) = t;
  }
  if (tid < kTile) {
    const int mye = uneven && mine > 0 ? min(14 - exponent(mine), 126) : e;
    own[l] = pow2(mye);
    side[j.rel * kTile + l] = pow2(e - mye);
  }
  if (bad) return;
  __syncthreads();
  const int g4 = lane >> 4, l16 = lane & 15;
  const float part = j.score ? score_parts(p.a).part : 1.0f;
  if (j.rowf)
    for (int c = w; c < 2 * DB; c += 4) {   // 32 features c / 2 of 16 rows c % 2
      const int r = 16 * (c % 2) + l16;
      float z[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) z[q] = x[r * LD + 32 * (c / 2) + 8 * g4 + q] * part * own[r];
      half8 a, f;
      split8(z, a, f);
      half8* o = (half8*)(j.rowf + (slot * 2 * DB + c) * 2 * kFrag) + lane;
      o[0] = a;
      o[kFrag / 8] = f;
    }
  if (j.colf)
    for (int c = w; c < 2 * DB; c += 4) {   // 16 features c of all rows
      float z[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const int k = 16 * (q / 4) + 4 * g4 + q % 4;
        z[q] = x[k * LD + 16 * c + l16] * own[k];
      }
      half8 a, f;
      split8(z, a, f);
      half8* o = (half8*)(j.colf + (slot * 2 * DB + c) * 2 * kFrag) + lane;
      o[0] = a;
      o[kFrag / 8] = f;
    }
}

// ---- many rows -----------------------------------------------------------------------------------

struct TilesArgs {
  AttendDesc a;
  const _Float16 *kf, *vf;         // k's row fragments, v's column fragments
  const TileInfo *ki, *vi;
  const float* side;
  FastDiv group;                   // G
  int M, blocks, splits;           // rows of a slab, row blocks, parts of the key axis
  bool wide;
  float* part;                     // parts: [split][slab][M][Dv], of sums of weights 1
  f32x2* psum;                     // their largest scores and sums: [split][slab][M]
};

// Where a row's result goes, and its largest score and sum. A part that has no such score says f32's lowest, and a part whose
// weights are all 0 has a sum and a result of 0.
__device__ __forceinline__ float* result_row(const TilesArgs& A, int split, int slab, int b, int head, int r, int i, float m, float sum, bool none,
                                             bool writes) {
  const AttendDesc& a = A.a;
  if (A.splits > 1) {
    const int64_t at = ((int64_t)split * a.B * a.Hk + slab) * A.M + r;
    if (writes) A.psum[at] = f32x2{fmaxf(m, kLowest), sum};
    return A.part + at * a.Dv;
  }
  if (writes && a.stats) write_stats(a, ((int64_t)b * a.H + head) * a.Tq + i, none, m, sum);
  return a.y.p ? a.y.p + b * a.y.b + head * a.y.h + (int64_t)i * a.y.t : nullptr;
}

// A wavefront's rows [row0, row0 + 16) over keys [j0, j1) in plain f32.
__device__ __forceinline__ void plain_rows(const TilesArgs& A, const Sight& s, int split, int slab, int b, int hk, int row0, int j0, int j1) {
  const AttendDesc& a = A.a;
  const int lane = threadIdx.x & 63, G = (int)A.group.d;
  const float* k = a.k.p + b * a.k.b + hk * a.k.h;
  const float* v = a.v.p + b * a.v.b + hk * a.v.h;
#pragma unroll 1
  for (int r = row0; r < min(row0 + 16, A.M); ++r) {
    const int i = r / G, head = hk * G + r % G, p = s.first + i, doc = doc_at(s, p), end = min(j1, sees_below(s, p));
    const float* q = a.q.p + b * a.q.b + head * a.q.h + (int64_t)i * a.q.t;
    const float slope = a.slopes ? a.slopes[head] * kLog2e : 0.0f;
    auto shown = [&](int j) { return j < end && (!s.doc || (doc >= 0 && s.doc[j] == doc)); };
    auto score = [&](int j) { return plain_score(a, plain_dot(k + j * a.k.t, q, a.D), slope, p - j).score; };
    float m = kNone;
#pragma unroll 1
    for (int j = j0 + lane; j < end; j += 64)
      if (shown(j)) m = fmaxf(m, score(j));
#pragma unroll
    for (int o = 1; o < 64; o *= 2) m = fmaxf(m, __shfl_xor(m, o));
    const bool none = !sees_any(s, sees_below(s, p), doc);
    if (m == kNone) m = 0;         // nothing, NaN alone, or minus infinities
    float sum = 0, acc[2] = {0, 0};
#pragma unroll 1
    for (int c = j0; c < end; c += 64) {
      const int j = c + lane;
      const float w = shown(j) ? __builtin_amdgcn_exp2f(score(j) - m) : 0.0f;
      sum += w;
      plain_add(acc, w, [&](int z) { return v + min(c + z, a.Tk - 1) * a.v.t; }, a.Dv);
    }
#pragma unroll
    for (int o = 1; o < 64; o *= 2) sum += __shfl_xor(sum, o);
    float* y = result_row(A, split, slab, b, head, r, i, m, sum, none, lane == 0);
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (y && 64 * e + lane < a.Dv) y[64 * e + lane] = (A.splits > 1 ? sum == 0 : none) ? 0.0f : acc[e] / sum;
  }
}

// Bound by the issue of products and vector work together, which overlap only between wavefronts: 4096 x 4096 pairs without
// masks, 8 heads of 128: 204 us, 337 TFLOP/s of the 443 that three f16 products for one allow; capped and causal: 156 us. k and
// v come two tiles in turn: the next one travels while this one is multiplied.
template <int DP, bool CAP, bool SLOPES>
__global__ __launch_bounds__(512, 4) void attend_tiles(TilesArgs A) {
  constexpr int N = DP / 32, F = 4 * N, F_V = F, F_SIDE = 2 * F, NF = F_SIDE + kSideFrags;
  __shared__ __align__(16) _Float16 lds[2 * NF * kFrag];
  __shared__ int range[5];
  const AttendDesc& a = A.a;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), g4 = lane >> 4, l = lane & 15;
  int slab, item;
  place(blockIdx.x, a.B * a.Hk, slab, item);
  if (item >= A.blocks * A.splits) return;
  const int split = item % A.splits, blk = A.blocks - 1 - item / A.splits;   // the last rows see the most keys: first
  const int b = slab / a.Hk, hk = slab % a.Hk, G = (int)A.group.d;
  const Sight s = sight(a, b);
  const int tiles = (a.Tk + kTile - 1) / kTile;

  // this lane's query
  const int row0 = blk * 128 + w * 16, r = row0 + l;
  const bool valid = r < A.M;
  const int i = (int)fastdiv((uint32_t)min(r, A.M - 1), A.group), g = min(r, A.M - 1) - i * G, head = hk * G + g;
  const int p = s.first + i, doc = doc_at(s, p), below = sees_below(s, p);

  // the wavefront's rows, and the block's key tiles
  Span me;
  me.pmin = s.first + (int)fastdiv((uint32_t)min(row0, A.M - 1), A.group);
  me.pmax = s.first + (int)fastdiv((uint32_t)min(row0 + 15, A.M - 1), A.group);
  me.dmin = valid && doc >= 0 ? doc : INT32_MAX;
  me.dmax = valid && doc >= 0 ? doc : INT32_MIN;
  if (s.doc) {
#pragma unroll
    for (int o = 1; o < 16; o *= 2) {
      me.dmin = min(me.dmin, __shfl_xor(me.dmin, o));
      me.dmax = max(me.dmax, __shfl_xor(me.dmax, o));
    }
  }
  me.dmin = __builtin_amdgcn_readfirstlane(me.dmin);
  me.dmax = __builtin_amdgcn_readfirstlane(me.dmax);
  me.same = !__any(valid && doc < 0) && me.dmin == me.dmax;
  const TileInfo* ki = A.ki + (int64_t)slab * tiles;
  const TileInfo* vi = A.vi + (int64_t)slab * tiles;
  const int last = s.first + (int)fastdiv((uint32_t)min(blk * 128 + 127, A.M - 1), A.group);   // of the block
  half8 qh[N], ql[N];
  bool infinite;
  const Score sc = score_parts(a);
  const int qe = load_rows<N>(a.q.p + b * a.q.b + head * a.q.h + (int64_t)i * a.q.t, valid, a.D, A.wide, sc.part, qh, ql, &infinite);
  int t0 = 0, t1 = s.n;
  if (s.causal) t1 = min(t1, max(last + 1, s.prefix));
  if (s.positional && last < 0) t1 = 0;
  const Range range_ = tile_range(s, 0, (t1 + kTile - 1) / kTile, ki, ki, vi, me.dmin, me.dmax,
                                  infinite && sees_any(s, below, doc), range);
  t0 = range_.t0;
  t1 = range_.t1;
  if (A.splits > 1) {
    const int n = t1 - t0, each = (n + A.splits - 1) / A.splits;
    t0 = min(t0 + split * each, t1);
    t1 = min(t0 + each, t1);
  }
  if (__builtin_expect(range_.odd, 0)) {
    plain_rows(A, s, split, slab, b, hk, row0, t0 * kTile, t1 * kTile);
    return;
  }

  const float slope = SLOPES ? a.slopes[head] * kLog2e : 0.0f;
  const int64_t tile0 = (int64_t)slab * tiles + t0;
  const uint32_t base = lds_address(lds) + w * 1024, lane16 = lane * 16;
  const char* kf = (const char*)(A.kf + tile0 * (F * kFrag)) + w * 1024;
  const char* vf = (const char*)(A.vf + tile0 * (F * kFrag)) + w * 1024;
  const char* side_p = (const char*)(A.side + tile0 * (kSide * kTile)) + w * 1024;
  auto fetch = [&](int buf) {      // the next tile
    const uint32_t to = base + buf * (NF * 1024);
    frags_to_lds<F>(kf, to, lane16, w);
    frags_to_lds<F>(vf, to + F_V * 1024, lane16, w);
    frags_to_lds<kSideFrags>(side_p, to + F_SIDE * 1024, lane16, w);
    kf += F * 1024;
    vf += F * 1024;
    side_p += kSide * kTile * 4;
  };

  f32x4 acc[2 * N];
#pragma unroll
  for (int d = 0; d < 2 * N; ++d) acc[d] = f32x4{};
  float m = kNone, sum = 0;        // running maximum (log2) and this lane's part of the sum
  int ce = kUnset;                 // acc is in units of 2^-ce
  if (t0 < t1) fetch(0);
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1, j0 = t * kTile;
    loads_done();
    __syncthreads();
    if (t + 1 < t1) fetch(buf ^ 1);
    const _Float16* L = lds + buf * (NF * kFrag);
    const float* side = (const float*)(L + F_SIDE * kFrag);
    const TileInfo kt = side_info(side, 0), vt = side_info(side, 1);
    if (__builtin_expect(!any_seen(s, me, kt, j0), 0)) continue;
    float x[8];                    // transposed: element q of this lane is key j0 + 16 (q / 4) + 4 g4 + q % 4
    scores<true, N>(L, 0, qh, ql, x);
    if (__builtin_expect(kt.uneven, 0)) per_row(x, side + KS_RELK * kTile, g4);
    float f = score_unit(sc, exponent(kt.inv) - qe);   // the score is f x, in log2
    if (CAP) {
      tanh_all(x, f);
      f = a.cap * kLog2e;
    }
    if (CAP || SLOPES) {
#pragma unroll
      for (int q = 0; q < 8; ++q) x[q] = score_of(SLOPES, x[q], f, slope, p - (j0 + 16 * (q / 4) + 4 * g4 + q % 4));
      f = 1;
    }
    if (__builtin_expect(!all_seen(s, me, kt, j0), 0)) {
#pragma unroll
      for (int q = 0; q < 8; ++q) x[q] = key_seen(s, side, j0, 16 * (q / 4) + 4 * g4 + q % 4, below, doc) ? x[q] : kNone;
    }
    float top = x[0];
#pragma unroll
    for (int q = 1; q < 8; ++q) top = fmaxf(top, x[q]);
    top = groups_max(top) * f;
    // The running maximum moves only when it grows by more than 2^8 (or from nothing), so that most tiles leave acc alone:
    // weights then reach 2^8 instead of 1.
    const bool up = top > m + 8 || (m == kNone && top > kNone);
    const float to = up ? top : m, keep = up ? __builtin_amdgcn_exp2f(m - to) : 1.0f;
    m = to;
    // what acc held has shrunk: so may its unit
    const int shrunk = up && keep > 0 && ce != kUnset ? min(-exponent(keep) - 1, 100) : 0;
    float change = keep * pow2(shrunk), part = 0;
    ce += shrunk;
    const float off = m == kNone ? 0.0f : m;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      x[q] = __builtin_amdgcn_exp2f(fmaf(x[q], f, -off));
      part += x[q];
    }
    sum = fmaf(sum, keep, part);
    float big = __builtin_amdgcn_exp2f(top - off);
    if (__builtin_expect(vt.uneven, 0)) {
      per_row(x, side + KS_RELV * kTile, g4);
      big = largest(x);
    }
    const int e = fit_unit(ce, big, exponent(vt.scale), &change);
    rescale(acc, change);
    accumulate(acc, x, pow2(e), L, F_V);
  }

  sum = groups_sum(sum);
  if (!valid) return;
  const bool none = !sees_any(s, below, doc);
  const float out = (A.splits > 1 ? sum == 0 : none) ? 0.0f : 1.0f / sum;
  float* y = result_row(A, split, slab, b, head, r, i, m, sum, none, g4 == 0);
  if (y) store_row(y, acc, ce, out, a.Dv, A.splits > 1 ? a.Dv % 4 == 0 : A.wide, g4);
}

// ---- few rows --------------------------------------------------------------------------------------

struct FewArgs {
  AttendDesc a;
  int M, splits, each;             // keys of a part
  float* part;
  f32x2* psum;
};

// Eight lanes share a key row: each reads E of its features as 16-byte pieces (8 rows of 128 bytes a load instruction) and
// multiplies them with the same features of all R query rows, which it keeps. Every group of eight lanes carries a running
// maximum, sum and result of its own (the maximum from f32's lowest on, so that weights of scores of minus infinity are 0
// whatever came before); the 32 groups of a block are joined once at its end. A part is the same number of keys
// for every batch entry, so that blocks past a short one end at once and those that work are alike. 8 caches of up to 16000
// keys, 4 key heads of 128, 16 query heads: 67 to 68 us, 5.8 TB/s.
template <int E, int R, bool WIDE>
__global__ __launch_bounds__(256) void attend_few(FewArgs A) {
  const AttendDesc& a = A.a;
  const int tid = threadIdx.x, sub = tid & 7, grp = tid >> 3;
  const int split = blockIdx.x % A.splits, slab = blockIdx.x / A.splits, b = slab / a.Hk, hk = slab % a.Hk, G = a.H / a.Hk;
  const Sight s = sight(a, b);
  auto feature = [&](int e) { return WIDE ? 4 * (sub + 8 * (e / 4)) + e % 4 : sub + 8 * e; };
  auto load = [&](const float* row, int n, float (&x)[E]) {
    if (WIDE) {
#pragma unroll
      for (int e = 0; e < E; e += 4) {
        f32x4 u = {};
        if (feature(e) < n) u = *(const f32x4*)(row + feature(e));
#pragma unroll
        for (int q = 0; q < 4; ++q) x[e + q] = u[q];
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = feature(e) < n ? row[feature(e)] : 0.0f;
    }
  };
  float q[R][E], acc[R][E], m[R], sum[R];
  int p[R], doc[R], below[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int rr = min(r, A.M - 1), i = rr / G, head = hk * G + rr % G;
    load(a.q.p + b * a.q.b + head * a.q.h + i * a.q.t, a.D, q[r]);
    p[r] = s.first + i;
    doc[r] = doc_at(s, p[r]);
    below[r] = sees_below(s, p[r]);
    m[r] = kLowest;
    sum[r] = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[r][e] = 0;
  }
  const int pmin = p[0], pmax = p[R - 1];
  int n = s.n;
  if (s.causal) n = min(n, max(pmax + 1, s.prefix));
  if (s.positional && pmax < 0) n = 0;
  const int begin = min((int64_t)split * A.each, (int64_t)n), end = min((int64_t)begin + A.each, (int64_t)n);
  const float* k = a.k.p + b * a.k.b + hk * a.k.h;
  const float* v = a.v.p + b * a.v.b + hk * a.v.h;
  float kn[E], vn[E];
  bool on = begin + grp < end;
  if (on) {
    load(k + (begin + grp) * a.k.t, a.D, kn);
    load(v + (begin + grp) * a.v.t, a.Dv, vn);
  }
  for (int j0 = begin; j0 < end; j0 += 32) {
    const int j = j0 + grp;
    float kx[E], vx[E];
#pragma unroll
    for (int e = 0; e < E; ++e) { kx[e] = kn[e]; vx[e] = vn[e]; }
    const bool here = on;
    on = j + 32 < end;
    if (on) {                      // the next rows travel while these are multiplied
      load(k + (j + 32) * a.k.t, a.D, kn);
      load(v + (j + 32) * a.v.t, a.Dv, vn);
    }
    if (!here) continue;
    const bool all = !s.doc && (!s.causal || j <= pmin) && !(s.positional && pmin < 0);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float x = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) x = fmaf(q[r][e], kx[e], x);
      x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0xB1, 15, 15, true));   // lane ^ 1
      x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x4E, 15, 15, true));   // lane ^ 2
      x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x141, 15, 15, true));  // 7 - lane
      x *= a.scale;
      if (a.cap > 0) x = a.cap * tanh_of(x / a.cap);
      if (a.slopes) x -= a.slopes[hk * G + min(r, A.M - 1) % G] * fabsf((float)(p[r] - j));
      x = rounded_mul(x, kLog2e);
      if (!all && (j >= below[r] || (s.doc && (doc[r] < 0 || s.doc[j] != doc[r])))) continue;
      if (x > m[r] + 8) {
        const float top = x < INFINITY ? x : m[r] == kLowest ? 0.0f : m[r];   // an infinite score shows in the weight
        const float keep = __builtin_amdgcn_exp2f(m[r] - top);
        m[r] = top;
        sum[r] *= keep;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[r][e] *= keep;
      }
      const float w = __builtin_amdgcn_exp2f(x - m[r]);
      sum[r] += w;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[r][e] = fmaf(w, vx[e], acc[r][e]);
    }
  }
  // the eight groups of a wavefront, then the four wavefronts
#pragma unroll
  for (int o = 8; o < 64; o *= 2)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float other = __shfl_xor(m[r], o), top = fmaxf(m[r], other);
      const float here = __builtin_amdgcn_exp2f(m[r] - top), there = __builtin_amdgcn_exp2f(other - top);
      m[r] = top;
      sum[r] = fmaf(__shfl_xor(sum[r], o), there, sum[r] * here);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[r][e] = fmaf(__shfl_xor(acc[r][e], o), there, acc[r][e] * here);
    }
  __shared__ float sm[4][R], ss[4][R], sa[4][R][8 * E];
  if (grp % 8 == 0) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (sub == 0) {
        sm[grp / 8][r] = m[r];
        ss[grp / 8][r] = sum[r];
      }
#pragma unroll
      for (int e = 0; e < E; ++e) sa[grp / 8][r][feature(e)] = acc[r][e];
    }
  }
  __syncthreads();
  for (int z = tid; z < min(R, A.M) * (8 * E); z += 256) {
    const int r = z / (8 * E), d = z % (8 * E), i = r / G, head = hk * G + r % G;
    float top = kLowest, all = 0, o = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) top = fmaxf(top, sm[u][r]);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float f = __builtin_amdgcn_exp2f(sm[u][r] - top);
      all = fmaf(ss[u][r], f, all);
      o = fmaf(sa[u][r][d], f, o);
    }
    const bool none = !sees_any(s, sees_below(s, s.first + i), doc_at(s, s.first + i));
    o = (A.splits > 1 ? all == 0 : none) ? 0.0f : o / all;
    const int64_t at = ((int64_t)split * a.B * a.Hk + slab) * A.M + r;
    if (d < a.Dv) {
      if (A.splits > 1) A.part[at * a.Dv + d] = o;
      else if (a.y.p) a.y.p[b * a.y.b + head * a.y.h + i * a.y.t + d] = o;
    }
    if (d == 0 && A.splits > 1) A.psum[at] = f32x2{top, all};
  }
}

// ---- joining the parts ---------------------------------------------------------------------------

// Parts at most, and blocks that are wanted: one round of the card. 512 blocks of attend_few read 8 sequences of up to 16000
// keys (4 heads of 128, 16 query heads) in 66 us, 1024 in 74, 2048 in 83, and 256 leave compute units idle (89). attend_tiles
// over 32 slabs of 777 rows of 96: 33 us and 10 to join, 46 with 256. Rows enough for 512 blocks are not cut: 1024 gain 16 of
// 289 us at 4096 causal rows of 128 and lose 19 of 36 in documents.
constexpr int kMostParts = 512;
constexpr int kJoinFew = 16;       // parts of a row that 32 threads join

struct JoinArgs {
  AttendDesc a;
  int M, splits;
  const float* part;
  const f32x2* psum;
};
// Bound by memory (24864 rows of 2 parts of 96: 11 us). L threads join a row: its weights first, then every 32 threads an
// L / 32nd of the parts. 32 threads take a row with few parts and a block one with many (a long cache read by one token: 16
// parts by 32 threads or 64 by a block, 8 or 7 us; one thread a feature took 33). A sum of NaN makes the row NaN.
template <int L>
__global__ __launch_bounds__(256) void attend_join(JoinArgs A) {
  constexpr int W = L < 64 ? L : 64, P = L / 32, PER = 256 / L;
  const AttendDesc& a = A.a;
  __shared__ float weight[PER * (L == 256 ? kMostParts : kJoinFew)];
  __shared__ f32x4 sums[P > 1 ? 256 : 1];
  const int tid = threadIdx.x, own = tid / L, t = tid % L, unit = t % 32, d = 4 * unit;
  const int64_t rows = (int64_t)a.B * a.Hk * A.M, row = (int64_t)blockIdx.x * PER + own, at = min(row, rows - 1);
  const int r = (int)(at % A.M), slab = (int)(at / A.M), b = slab / a.Hk, hk = slab % a.Hk, G = a.H / a.Hk;
  const int i = r / G, head = hk * G + r % G;
  const Sight s = sight(a, b);
  const bool none = !sees_any(s, sees_below(s, s.first + i), doc_at(s, s.first + i));
  float top = kLowest, all = 0;
  for (int z = t % W; z < A.splits; z += W) top = fmaxf(top, A.psum[at + z * rows].x);
#pragma unroll
  for (int o = 1; o < W; o *= 2) top = fmaxf(top, __shfl_xor(top, o));
  for (int z = t % W; z < A.splits; z += W) {
    const f32x2 e = A.psum[at + z * rows];
    const float w = __builtin_amdgcn_exp2f(e.x - top) * e.y;
    if (t < W) weight[own * A.splits + z] = w;
    all += w;
  }
#pragma unroll
  for (int o = 1; o < W; o *= 2) all += __shfl_xor(all, o);
  __syncthreads();
  f32x4 x = {};
  const float* part = A.part + at * a.Dv + d;
#pragma unroll 4
  for (int z = t / 32; z < A.splits; z += P) {
    const float w = weight[own * A.splits + z];
    f32x4 u = {};
    if (a.Dv % 4 == 0) {
      if (d < a.Dv) u = *(const f32x4*)(part + z * rows * a.Dv);
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) if (d + q < a.Dv) u[q] = part[z * rows * a.Dv + q];
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) x[q] = fmaf(w, u[q], x[q]);
  }
  if constexpr (P > 1) {
    sums[tid] = x;
    __syncthreads();
    if (tid >= 32) return;
#pragma unroll
    for (int z = 1; z < P; ++z) x += sums[32 * z + tid];
  }
  if (row >= rows) return;
  if (a.y.p) {
    float* y = a.y.p + b * a.y.b + head * a.y.h + (int64_t)i * a.y.t + d;
#pragma unroll
    for (int q = 0; q < 4; ++q) if (d + q < a.Dv) y[q] = none ? 0.0f : x[q] / all;
  }
  if (a.stats && t == 0) write_stats(a, ((int64_t)b * a.H + head) * a.Tq + i, none, top, all);
}

// ---- plans -----------------------------------------------------------------------------------------

struct Plan {
  int DP, M, G, tiles, blocks, splits, slabs, each;
  bool few;
  int64_t kf, vf, ki, vi, side, part, psum, bytes;   // byte offsets into the workspace
};
constexpr int64_t kAlign = 256;
inline int64_t take(int64_t& at, int64_t bytes) {
  const int64_t b = at;
  at += (bytes + kAlign - 1) / kAlign * kAlign;
  return b;
}
// Rows that attend_few keeps in registers: 16 E floats a lane of queries and results.
inline int few_rows(int DP) { return DP <= 32 ? 16 : DP <= 64 ? 8 : 4; }

Plan plan(const AttendDesc& a) {
  Plan p{};
  p.DP = attend_dp(a);
  p.G = a.H / a.Hk;
  p.M = p.G * a.Tq;
  p.slabs = a.B * a.Hk;
  p.tiles = (a.Tk + kTile - 1) / kTile;
  p.few = !a.stats && p.M <= few_rows(p.DP) && (p.M <= 2 || a.Tk >= 32 * p.M);
  if (p.few) {
    p.blocks = 1;
    const int64_t want = std::max<int64_t>(1, kMostParts / p.slabs);
    p.each = (int)std::max<int64_t>(128, ((a.Tk + want - 1) / want + 31) / 32 * 32);
    p.splits = std::max(1, (a.Tk - 1) / p.each + 1);
  } else {
    p.blocks = (p.M + 127) / 128;
    const int64_t have = (int64_t)p.slabs * p.blocks;
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(kMostParts / have, p.tiles / 8));
  }
  int64_t at = 0;
  if (!p.few) {
    const int64_t frag = (int64_t)p.slabs * p.tiles * p.DP * kTile * 4;
    p.kf = take(at, frag);
    p.vf = take(at, frag);
    p.ki = take(at, (int64_t)p.slabs * p.tiles * sizeof(TileInfo));
    p.vi = take(at, (int64_t)p.slabs * p.tiles * sizeof(TileInfo));
    p.side = take(at, (int64_t)p.slabs * p.tiles * kSide * kTile * 4);
  }
  if (p.splits > 1) {
    p.part = take(at, (int64_t)p.splits * p.slabs * p.M * a.Dv * 4);
    p.psum = take(at, (int64_t)p.splits * p.slabs * p.M * 8);
  }
  p.bytes = at;
  return p;
}

template <int DP>
void run_tiles(const TilesArgs& t, unsigned grid, hipStream_t st) {
  if (t.a.cap > 0 && t.a.slopes) klaunch(attend_tiles<DP, true, true>, dim3(grid), dim3(512), 0, st, t);
  else if (t.a.cap > 0) klaunch(attend_tiles<DP, true, false>, dim3(grid), dim3(512), 0, st, t);
  else if (t.a.slopes) klaunch(attend_tiles<DP, false, true>, dim3(grid), dim3(512), 0, st, t);
  else klaunch(attend_tiles<DP, false, false>, dim3(grid), dim3(512), 0, st, t);
}
template <int E, int R>
void run_few(const FewArgs& f, bool wide, int slabs, hipStream_t st) {
  if (wide) klaunch(attend_few<E, R, true>, dim3(f.splits * slabs), dim3(256), 0, st, f);
  else klaunch(attend_few<E, R, false>, dim3(f.splits * slabs), dim3(256), 0, st, f);
}
template <int E>
void run_few_rows(const FewArgs& f, bool wide, int slabs, hipStream_t st) {
  if (f.M <= 1) run_few<E, 1>(f, wide, slabs, st);
  else if (f.M <= 2) run_few<E, 2>(f, wide, slabs, st);
  else if (f.M <= 4) run_few<E, 4>(f, wide, slabs, st);
  else if constexpr (E <= 8) {
    if (E > 4 || f.M <= 8) run_few<E, 8>(f, wide, slabs, st);
    else if constexpr (E <= 4) run_few<E, 16>(f, wide, slabs, st);
  }
}

}  // namespace

void attend_pack(Packs p, int DP, hipStream_t st) {
  p.tiles = 0;
  for (int i = 0; i < p.n; ++i) p.tiles = std::max(p.tiles, p.job[i].tiles);
  const dim3 grid((unsigned)p.tiles * p.a.B * p.Hk, p.n);
  if (DP == 32) klaunch(pack_tiles<32>, grid, dim3(256), 0, st, p);
  else if (DP == 64) klaunch(pack_tiles<64>, grid, dim3(256), 0, st, p);
  else if (DP == 96) klaunch(pack_tiles<96>, grid, dim3(256), 0, st, p);
  else klaunch(pack_tiles<128>, grid, dim3(256), 0, st, p);
}

int64_t attend_workspace_bytes(const AttendDesc& a) { return attend_small_rows(a) ? 0 : plan(a).bytes; }

void attend(const AttendDesc& a, void* work, hipStream_t st) {
  if (attend_small_rows(a)) return attend_small_forward(a, st);
  const Plan p = plan(a);
  char* w = (char*)work;
  float* part = p.splits > 1 ? (float*)(w + p.part) : nullptr;
  f32x2* psum = p.splits > 1 ? (f32x2*)(w + p.psum) : nullptr;
  const bool wide = attend_wide(a.q, a.D) && attend_wide(a.k, a.D) && attend_wide(a.v, a.Dv) && (!a.y.p || attend_wide(a.y, a.Dv));
  if (p.few) {
    const FewArgs f{a, p.M, p.splits, p.each, part, psum};
    if (p.DP == 32) run_few_rows<4>(f, wide, p.slabs, st);
    else if (p.DP == 64) run_few_rows<8>(f, wide, p.slabs, st);
    else if (p.DP == 96) run_few_rows<12>(f, wide, p.slabs, st);
    else run_few_rows<16>(f, wide, p.slabs, st);
  } else {
    Packs k{};
    k.n = 2;
    k.Hk = a.Hk;
    k.wide = wide;
    k.a = a;
    float* side = (float*)(w + p.side);
    k.job[0] = {a.k, a.D, 1, a.Tk, p.tiles, (_Float16*)(w + p.kf), nullptr, (TileInfo*)(w + p.ki), false, side, KS_RELK, false, true, false, {}};
    k.job[1] = {a.v, a.Dv, 1, a.Tk, p.tiles, nullptr, (_Float16*)(w + p.vf), (TileInfo*)(w + p.vi), false, side, KS_RELV, true, false, false, {}};
    attend_pack(k, p.DP, st);
    const TilesArgs t{a, (_Float16*)(w + p.kf), (_Float16*)(w + p.vf), (TileInfo*)(w + p.ki), (TileInfo*)(w + p.vi), side,
                      make_fastdiv(p.G), p.M, p.blocks, p.splits, wide, part, psum};
    const unsigned grid = place_grid(p.slabs, (int64_t)p.blocks * p.splits);
    if (p.DP == 32) run_tiles<32>(t, grid, st);
    else if (p.DP == 64) run_tiles<64>(t, grid, st);
    else if (p.DP == 96) run_tiles<96>(t, grid, st);
    else run_tiles<128>(t, grid, st);
  }
  if (p.splits > 1) {
    const JoinArgs j{a, p.M, p.splits, part, psum};
    const int64_t rows = (int64_t)p.slabs * p.M;
    if (p.splits <= kJoinFew) klaunch(attend_join<32>, dim3((rows + 7) / 8), dim3(256), 0, st, j);
    else klaunch(attend_join<256>, dim3(rows), dim3(256), 0, st, j);
  }
}

}  // namespace tgk
