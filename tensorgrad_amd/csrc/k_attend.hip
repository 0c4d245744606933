// Masked attention for gfx950: y = softmax(scores) v, one pass over the keys with a running maximum and sum, so that no
// score reaches memory. Three kernels, by the number of query rows that share a key head (G query heads times Tq):
//  * many rows: k and v are packed once into f16 hi / lo fragments (attend_pack), then blocks of 4 wavefronts with 32 rows
//    each walk the visible key tiles (attend_tiles). Scores are computed transposed (keys x queries), so that a lane holds
//    half the keys of ONE query: maximum and sum are lane arithmetic and one exchange between lane halves, and the
//    probabilities are the next product's B fragment as they stand;
//  * few rows (one new token against a cache): the keys are read once, in f32, by all heads that share them (attend_few);
//    bound by memory, so split over the keys until the card is full.
// Both split a long key axis when there are few rows, and join the parts (attend_join).
#include "attend_dev.h"

namespace tgk {
namespace {

// ---- packing -------------------------------------------------------------------------------------

// A block packs one tile of 32 rows: reads them once, finds the tile's scale, writes its fragments.
template <int DP>
__global__ __launch_bounds__(256) void pack_tiles(Packs p) {
  constexpr int KC = DP / 16, DB = DP / 32, LD = DP + 4;
  __shared__ float x[kTile * LD];
  __shared__ float top[kTile];
  __shared__ int norm[kTile], doc[kTile];
  const PackJob j = p.job[blockIdx.z];
  const int tile = blockIdx.x, slab = blockIdx.y, b = slab / p.Hk, hk = slab % p.Hk;
  if (tile >= j.tiles) return;
  const int tid = threadIdx.x, row = tid / 8, sub = tid % 8, r = tile * kTile + row;
  const bool in = r < j.rows;
  const int i = r / j.G, g = r - i * j.G;
  const int64_t at = b * j.x.b + (int64_t)(hk * j.G + g) * j.x.h + (int64_t)i * j.x.t;
  float m = 0, dot = 0;
  bool odd = false;
  float v[DP / 8];
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
      odd |= !(fabsf(u[q]) < INFINITY);
      m = fmaxf(m, finite_abs(u[q]));
      v[4 * c + q] = u[q];
    }
    *(f32x4*)(x + row * LD + d) = u;
    if (j.rowinfo && in) {
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
  // the 2-norm, from values relative to the largest so that nothing overflows: 2^norm >= it
  float sq = 0;
  const float inv = m > 0 ? 1.0f / fmaxf(m, 1e-37f) : 0.0f;
#pragma unroll
  for (int q = 0; q < DP / 8; ++q) {
    const float z = finite_abs(v[q]) * inv;
    sq = fmaf(z, z, sq);
  }
#pragma unroll
  for (int o = 1; o < 8; o *= 2) sq += __shfl_xor(sq, o);
  if (sub == 0) {
    const Sight s = sight(p.a, b);
    const int pos = j.query ? s.first + i : r;
    top[row] = odd ? INFINITY : m;
    norm[row] = norm_exponent(m, sq);
    doc[row] = in ? doc_at(s, pos) : -1;
    if (j.rowinfo) {
      const AttendDesc& a = p.a;
      const int h = hk * j.G + g;
      float* o = j.rowinfo + ((int64_t)slab * j.tiles + tile) * (kRowInfo * kTile) + row;
      o[RI_LSE * kTile] = in ? a.lse[((int64_t)b * a.H + h) * a.Tq + i] : INFINITY;
      o[RI_DOT * kTile] = in ? dot : 0.0f;
      o[RI_POS * kTile] = __int_as_float(pos);
      o[RI_SLOPE * kTile] = in && a.slopes ? a.slopes[h] * kLog2e : 0.0f;
      o[RI_BELOW * kTile] = __int_as_float(in ? sees_below(s, pos) : 0);
      o[RI_DOC * kTile] = __int_as_float(doc[row]);
    }
  }
  __syncthreads();
  const int lane = tid & 63, w = tid >> 6, h = lane >> 5, l = lane & 31;
  float hi = top[l], lo = hi > 0 ? hi : INFINITY;
  int nm = norm[l], dmin = doc[l] >= 0 ? doc[l] : INT32_MAX, dmax = doc[l] >= 0 ? doc[l] : INT32_MIN;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    hi = fmaxf(hi, __shfl_xor(hi, o));
    lo = fminf(lo, __shfl_xor(lo, o));
    nm = max(nm, __shfl_xor(nm, o));
    dmin = min(dmin, __shfl_xor(dmin, o));
    dmax = max(dmax, __shfl_xor(dmax, o));
  }
  bool bad = !(hi < INFINITY);
  const bool same = dmin == dmax && !__any(doc[l] < 0);
  bad |= lo * 1048576.0f < hi;
  const float scale = bad || hi == 0 ? 1.0f : pow2(min(14 - exponent(hi), 126));
  const int64_t slot = (int64_t)slab * j.tiles + tile;
  if (tid == 0) {
    TileInfo t{};
    t.scale = scale;
    t.norm = nm;
    t.irregular = bad;
    t.dmin = dmin;
    t.dmax = dmax;
    t.same = same;
    j.info[slot] = t;
  }
  if (bad) return;
  if (j.rowf)
    for (int c = w; c < KC; c += 4) {
      float z[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) z[q] = x[l * LD + 16 * c + 8 * h + q] * scale;
      half8 a, e;
      split8(z, a, e);
      half8* o = (half8*)(j.rowf + (slot * KC + c) * 2 * kFrag) + lane;
      o[0] = a;
      o[kFrag / 8] = e;
    }
  if (j.colf)
    for (int c = w; c < 2 * DB; c += 4) {   // feature block c / 2, k step c % 2
      float z[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) z[q] = x[(16 * (c % 2) + 8 * (q / 4) + 4 * h + q % 4) * LD + 32 * (c / 2) + l] * scale;
      half8 a, e;
      split8(z, a, e);
      half8* o = (half8*)(j.colf + (slot * 2 * DB + c) * 2 * kFrag) + lane;
      o[0] = a;
      o[kFrag / 8] = e;
    }
}

// ---- many rows -----------------------------------------------------------------------------------

struct TilesArgs {
  AttendDesc a;
  const _Float16 *kf, *vf;         // k's row fragments, v's column fragments
  const TileInfo *ki, *vi;
  FastDiv group;                   // G
  int M, blocks, splits;           // rows of a slab, row blocks, parts of the key axis
  bool wide;
  float *part, *plse;              // parts: [split][slab][M][Dv], [split][slab][M]
};

template <int DP, bool RICH>       // RICH: capped scores or slopes
__global__ __launch_bounds__(256, 2) void attend_tiles(TilesArgs A) {
  constexpr int KC = DP / 16, DB = DP / 32, NF = 2 * KC + 4 * DB;
  __shared__ __align__(16) _Float16 lds[2][NF * kFrag];
  __shared__ int range[4];
  const AttendDesc& a = A.a;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, l = lane & 31;
  const uint32_t id = xcd_order(blockIdx.x, gridDim.x);
  const uint32_t per = (uint32_t)A.blocks * A.splits;
  const int slab = id / per, split = id % per % A.splits;
  const int blk = A.blocks - 1 - (int)(id % per / A.splits);       // the last rows see the most keys: first
  const int b = slab / a.Hk, hk = slab % a.Hk, G = (int)A.group.d;
  const Sight s = sight(a, b);
  const int tiles = (a.Tk + kTile - 1) / kTile;

  // this lane's query
  const int row0 = blk * 128 + w * kTile, r = row0 + l;
  const bool valid = r < A.M;
  const int i = (int)fastdiv((uint32_t)min(r, A.M - 1), A.group), g = min(r, A.M - 1) - i * G, head = hk * G + g;
  const int p = s.first + i, doc = doc_at(s, p), below = sees_below(s, p);
  const float* qrow = a.q.p + b * a.q.b + head * a.q.h + (int64_t)i * a.q.t;
  half8 qh[KC], ql[KC];
  const int qe = load_rows<KC>(qrow, valid, a.D, A.wide, qh, ql);
  const float slope = RICH && a.slopes ? a.slopes[head] * kLog2e : 0.0f;

  // the wavefront's rows, and the block's key tiles
  Span me;
  me.pmin = s.first + (int)fastdiv((uint32_t)min(row0, A.M - 1), A.group);
  me.pmax = s.first + (int)fastdiv((uint32_t)min(row0 + kTile - 1, A.M - 1), A.group);
  me.dmin = valid && doc >= 0 ? doc : INT32_MAX;
  me.dmax = valid && doc >= 0 ? doc : INT32_MIN;
  if (s.doc) {
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
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
  int t0 = 0, t1 = s.n;
  if (s.causal) t1 = min(t1, max(last + 1, s.prefix));
  if (s.positional && last < 0) t1 = 0;
  t1 = (t1 + kTile - 1) / kTile;
  if (s.doc) {
    if (tid < 4) range[tid] = tid & 1 ? INT32_MIN : INT32_MAX;
    __syncthreads();
    if (lane == 0) {
      atomicMin(&range[0], me.dmin);
      atomicMax(&range[1], me.dmax);
    }
    __syncthreads();
    const int lo = range[0], hi = range[1];
    int first = INT32_MAX, end = INT32_MIN;
    for (int t = tid; t < t1; t += 256)
      if (ki[t].dmin <= hi && lo <= ki[t].dmax) {
        first = min(first, t);
        end = max(end, t + 1);
      }
    atomicMin(&range[2], first);
    atomicMax(&range[3], end);
    __syncthreads();
    t0 = range[2];
    t1 = range[3];
    if (t0 >= t1) t0 = t1 = 0;
  }
  if (A.splits > 1) {
    const int n = t1 - t0, each = (n + A.splits - 1) / A.splits;
    t0 = min(t0 + split * each, t1);
    t1 = min(t0 + each, t1);
  }
  t0 = __builtin_amdgcn_readfirstlane(t0);
  t1 = __builtin_amdgcn_readfirstlane(t1);

  const _Float16* kf = A.kf + (int64_t)slab * tiles * (2 * KC * kFrag);
  const _Float16* vf = A.vf + (int64_t)slab * tiles * (4 * DB * kFrag);
  const uint32_t base = lds_address(lds), lane16 = lane * 16;
  auto fetch = [&](int t, int buf) {
#pragma unroll
    for (int f = 0; f < NF / 4; ++f) {
      const int q = f * 4 + w;
      const _Float16* src = q < 2 * KC ? kf + ((int64_t)t * (2 * KC) + q) * kFrag : vf + ((int64_t)t * (4 * DB) + q - 2 * KC) * kFrag;
      frag_to_lds(src, base + (buf * NF + q) * (kFrag * 2), lane16);
    }
  };

  f32x16 acc[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) acc[d] = f32x16{};
  float m = kNone, sum = 0;        // running maximum (log2) and this lane half's sum
  int ce = kUnset;                 // acc is in units of 2^-ce
  if (t0 < t1) fetch(t0, 0);
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1, j0 = t * kTile;
    loads_done();
    __syncthreads();
    if (t + 1 < t1) fetch(t + 1, buf ^ 1);
    const TileInfo kt = ki[t], vt = vi[t];
    if (!any_seen(s, me, kt, j0)) continue;
    const _Float16* L = lds[buf];
    // scores, transposed: register r of this lane is key j0 + 8 (r / 4) + 4 h + r % 4
    f32x16 x = {};
    float unit;
    if (kt.irregular) {
      const float* k = a.k.p + b * a.k.b + hk * a.k.h + (int64_t)j0 * a.k.t;
      plain_scores(x, [&](int j) { return k + j * a.k.t; }, a.Tk - j0, qrow, valid, a.D);
      unit = a.scale;
    } else {
      x = scores<KC>(L, 0, qh, ql);
      unit = a.scale * pow2(-qe) * (1.0f / kt.scale);
    }
    float f = 1;                   // exponent of 2 = f x (plain) or x (RICH)
    if (RICH) {
      if (a.cap > 0) {
        const float u = unit / a.cap, c = a.cap * kLog2e;
#pragma unroll
        for (int q = 0; q < 16; ++q) x[q] = c * tanh_of(x[q] * u);
      } else {
        const float u = unit * kLog2e;
#pragma unroll
        for (int q = 0; q < 16; ++q) x[q] *= u;
      }
      if (a.slopes)
#pragma unroll
        for (int q = 0; q < 16; ++q) x[q] -= slope * fabsf((float)(p - (j0 + 8 * (q / 4) + 4 * h + q % 4)));
    } else {
      f = unit * kLog2e;
    }
    if (!all_seen(s, me, kt, j0)) {
      if (s.doc) {
        int dj[16];
#pragma unroll
        for (int q = 0; q < 16; ++q) dj[q] = s.doc[min(j0 + 8 * (q / 4) + 4 * h + q % 4, a.Tk - 1)];
#pragma unroll
        for (int q = 0; q < 16; ++q) x[q] = dj[q] == doc && doc >= 0 ? x[q] : kNone;
      }
#pragma unroll
      for (int q = 0; q < 16; ++q) x[q] = j0 + 8 * (q / 4) + 4 * h + q % 4 < below ? x[q] : kNone;
    }
    float top = x[0];
#pragma unroll
    for (int q = 1; q < 16; ++q) top = fmaxf(top, x[q]);
    top = halves_max(top) * f;
    // The maximum moves only when it grows by more than 2^8 (or from nothing), so that most tiles leave acc alone: weights
    // then reach 2^8 instead of 1.
    float keep = 1;
    if (top > m + 8 || (m == kNone && top > kNone)) {
      keep = __builtin_amdgcn_exp2f(m - top);
      m = top;
      sum *= keep;
    }
    const float off = m == kNone ? 0.0f : m;
#pragma unroll
    for (int q = 0; q < 16; ++q) x[q] = __builtin_amdgcn_exp2f(fmaf(x[q], f, -off));
    float part = 0;
#pragma unroll
    for (int q = 0; q < 16; ++q) part += x[q];
    sum += part;
    float change = keep;
    if (vt.irregular) {
      const float* v = a.v.p + b * a.v.b + hk * a.v.h + (int64_t)j0 * a.v.t;
      rescale<DB>(acc, change);
      plain_accumulate<DB>(acc, ce, x, [&](int j) { return v + j * a.v.t; }, a.Tk - j0, a.Dv);
      continue;
    }
    // what acc held has shrunk by `keep`: so may its unit
    if (keep < 1 && ce != kUnset) {
      const int shrunk = keep > 0 ? min(-exponent(keep) - 1, 100) : 0;
      change *= pow2(shrunk);
      ce += shrunk;
    }
    const int e = fit_unit(ce, __builtin_amdgcn_exp2f(top - off), exponent(vt.scale), &change);
    rescale<DB>(acc, change);
    accumulate<DB>(acc, x, pow2(e), L, 2 * KC);
  }

  sum = halves_sum(sum);
  if (!valid) return;
  const bool none = sum == 0;      // not m: a visible NaN leaves no maximum
  const float lse = none ? (A.splits > 1 ? kNone : INFINITY) : m + __builtin_amdgcn_logf(sum);
  const float out = none ? 0.0f : 1.0f / sum;
  float* y;
  if (A.splits > 1) {
    const int64_t at = ((int64_t)split * a.B * a.Hk + slab) * A.M + r;
    if (h == 0) A.plse[at] = lse;
    y = A.part + at * a.Dv;
  } else {
    if (h == 0 && a.lse) a.lse[((int64_t)b * a.H + head) * a.Tq + i] = lse;
    y = a.y.p + b * a.y.b + head * a.y.h + (int64_t)i * a.y.t;
    if (!a.y.p) return;
  }
  const bool wide = A.splits > 1 ? a.Dv % 4 == 0 : A.wide;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int at = 32 * d + 8 * q + 4 * h;
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = none ? 0.0f : __builtin_amdgcn_ldexpf(acc[d][4 * q + e], -ce) * out;
      if (wide) {
        if (at < a.Dv) *(f32x4*)(y + at) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) if (at + e < a.Dv) y[at + e] = v[e];
      }
    }
}

// ---- few rows --------------------------------------------------------------------------------------

struct FewArgs {
  AttendDesc a;
  int M, splits;
  float *part, *plse;
};

// Eight lanes share a key row: each reads E of its features as 16-byte pieces (8 rows of 128 bytes a load instruction) and
// multiplies them with the same features of all R query rows, which it keeps. Every group of eight lanes carries a running
// maximum, sum and result of its own; the 32 groups of a block are joined once at its end.
template <int E, int R, bool WIDE>
__global__ __launch_bounds__(256) void attend_few(FewArgs A) {
  const AttendDesc& a = A.a;
  const int tid = threadIdx.x, sub = tid & 7, grp = tid >> 3;
  const int split = blockIdx.x, slab = blockIdx.y, b = slab / a.Hk, hk = slab % a.Hk, G = a.H / a.Hk;
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
    m[r] = kNone;
    sum[r] = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[r][e] = 0;
  }
  const int pmin = p[0], pmax = p[R - 1];
  int n = s.n;
  if (s.causal) n = min(n, max(pmax + 1, s.prefix));
  if (s.positional && pmax < 0) n = 0;
  const int each = ((n + A.splits - 1) / A.splits + 31) / 32 * 32;
  const int begin = min((int64_t)split * each, (int64_t)n), end = min(begin + each, n);
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
      x *= kLog2e;
      if (!all && (j >= below[r] || (s.doc && (doc[r] < 0 || s.doc[j] != doc[r])))) continue;
      if (x > m[r] + 8 || m[r] == kNone) {
        const float top = __builtin_isfinite(x) ? x : m[r] == kNone ? 0.0f : m[r];   // an infinite score shows in the weight
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
  // the block's 32 groups, row by row
  __shared__ float sm[32], ss[32], sa[32][8 * E + 1];
  for (int r = 0; r < min(R, A.M); ++r) {
    float mr = 0, sr = 0;
#pragma unroll
    for (int z = 0; z < R; ++z) if (z == r) { mr = m[z]; sr = sum[z]; }
    if (sub == 0) { sm[grp] = mr; ss[grp] = sr; }
#pragma unroll
    for (int z = 0; z < R; ++z)
      if (z == r)
#pragma unroll
        for (int e = 0; e < E; ++e) sa[grp][feature(e)] = acc[z][e];
    __syncthreads();
    float top = kNone, all = 0;
    for (int z = 0; z < 32; ++z) top = fmaxf(top, sm[z]);
    const int i = r / G, head = hk * G + r % G;
    if (top != kNone) for (int z = 0; z < 32; ++z) all += ss[z] * __builtin_amdgcn_exp2f(sm[z] - top);
    if (tid < a.Dv) {
      float o = 0;
      if (top != kNone) {
        for (int z = 0; z < 32; ++z) if (sm[z] != kNone) o = fmaf(sa[z][tid], __builtin_amdgcn_exp2f(sm[z] - top), o);
        o /= all;
      }
      if (A.splits > 1) A.part[(((int64_t)split * a.B * a.Hk + slab) * A.M + r) * a.Dv + tid] = o;
      else if (a.y.p) a.y.p[b * a.y.b + head * a.y.h + i * a.y.t + tid] = o;
    }
    if (tid == 0) {
      const float lse = top == kNone ? kNone : top + __builtin_amdgcn_logf(all);
      if (A.splits > 1) A.plse[((int64_t)split * a.B * a.Hk + slab) * A.M + r] = lse;
      else if (a.lse) a.lse[((int64_t)b * a.H + head) * a.Tq + i] = top == kNone ? INFINITY : lse;
    }
    __syncthreads();
  }
}

// ---- joining the parts ---------------------------------------------------------------------------

struct JoinArgs {
  AttendDesc a;
  int M, splits;
  const float *part, *plse;
};
__global__ __launch_bounds__(128) void attend_join(JoinArgs A) {
  const AttendDesc& a = A.a;
  const int r = blockIdx.x, slab = blockIdx.y, b = slab / a.Hk, hk = slab % a.Hk, G = a.H / a.Hk;
  const int i = r / G, head = hk * G + r % G, tid = threadIdx.x;
  const int64_t at = (int64_t)slab * A.M + r, step = (int64_t)a.B * a.Hk * A.M;
  float top = kNone, all = 0, o = 0;
  for (int z = 0; z < A.splits; ++z) top = fmaxf(top, A.plse[at + z * step]);
  if (top != kNone)
    for (int z = 0; z < A.splits; ++z) {
      const float e = A.plse[at + z * step];
      if (e == kNone) continue;
      const float w = __builtin_amdgcn_exp2f(e - top);
      all += w;
      if (tid < a.Dv) o = fmaf(w, A.part[(at + z * step) * a.Dv + tid], o);
    }
  if (a.y.p && tid < a.Dv) a.y.p[b * a.y.b + head * a.y.h + (int64_t)i * a.y.t + tid] = top == kNone ? 0.0f : o / all;
  if (a.lse && tid == 0) a.lse[((int64_t)b * a.H + head) * a.Tq + i] = top == kNone ? INFINITY : top + __builtin_amdgcn_logf(all);
}

// ---- plans -----------------------------------------------------------------------------------------

struct Plan {
  int DP, M, G, tiles, blocks, splits, slabs;
  bool few;
  int64_t kf, vf, ki, vi, part, plse, bytes;   // byte offsets into the workspace
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
  p.few = p.M <= few_rows(p.DP) && (p.M <= 2 || a.Tk >= 32 * p.M);
  if (p.few) {
    p.blocks = 1;
    const int64_t want = (2048 + p.slabs - 1) / p.slabs, most = (a.Tk + 127) / 128;
    p.splits = (int)std::max<int64_t>(1, std::min(want, most));
  } else {
    p.blocks = (p.M + 127) / 128;
    const int64_t have = (int64_t)p.slabs * p.blocks;
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(512 / have, p.tiles / 8));
  }
  int64_t at = 0;
  if (!p.few) {
    const int64_t frag = (int64_t)p.slabs * p.tiles * p.DP * kTile * 4;
    p.kf = take(at, frag);
    p.vf = take(at, frag);
    p.ki = take(at, (int64_t)p.slabs * p.tiles * sizeof(TileInfo));
    p.vi = take(at, (int64_t)p.slabs * p.tiles * sizeof(TileInfo));
  }
  if (p.splits > 1) {
    p.part = take(at, (int64_t)p.splits * p.slabs * p.M * a.Dv * 4);
    p.plse = take(at, (int64_t)p.splits * p.slabs * p.M * 4);
  }
  p.bytes = at;
  return p;
}

template <int DP>
void run_tiles(const TilesArgs& t, int64_t grid, hipStream_t st) {
  if (t.a.cap > 0 || t.a.slopes) klaunch(attend_tiles<DP, true>, dim3((unsigned)grid), dim3(256), 0, st, t);
  else klaunch(attend_tiles<DP, false>, dim3((unsigned)grid), dim3(256), 0, st, t);
}
template <int E, int R>
void run_few(const FewArgs& f, bool wide, int slabs, hipStream_t st) {
  if (wide) klaunch(attend_few<E, R, true>, dim3(f.splits, slabs), dim3(256), 0, st, f);
  else klaunch(attend_few<E, R, false>, dim3(f.splits, slabs), dim3(256), 0, st, f);
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

void attend_pack(const Packs& p, int DP, hipStream_t st) {
  int tiles = 0;
  for (int i = 0; i < p.n; ++i) tiles = std::max(tiles, p.job[i].tiles);
  const dim3 grid(tiles, p.a.B * p.Hk, p.n);
  if (DP == 32) klaunch(pack_tiles<32>, grid, dim3(256), 0, st, p);
  else if (DP == 64) klaunch(pack_tiles<64>, grid, dim3(256), 0, st, p);
  else if (DP == 96) klaunch(pack_tiles<96>, grid, dim3(256), 0, st, p);
  else klaunch(pack_tiles<128>, grid, dim3(256), 0, st, p);
}

int64_t attend_workspace_bytes(const AttendDesc& a) { return plan(a).bytes; }

void attend(const AttendDesc& a, void* work, hipStream_t st) {
  const Plan p = plan(a);
  char* w = (char*)work;
  float* part = p.splits > 1 ? (float*)(w + p.part) : nullptr;
  float* plse = p.splits > 1 ? (float*)(w + p.plse) : nullptr;
  const bool wide = attend_wide(a.q, a.D) && attend_wide(a.k, a.D) && attend_wide(a.v, a.Dv) && (!a.y.p || attend_wide(a.y, a.Dv));
  if (p.few) {
    const FewArgs f{a, p.M, p.splits, part, plse};
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
    k.job[0] = {a.k, a.D, 1, a.Tk, p.tiles, (_Float16*)(w + p.kf), nullptr, (TileInfo*)(w + p.ki), false, {}, nullptr};
    k.job[1] = {a.v, a.Dv, 1, a.Tk, p.tiles, nullptr, (_Float16*)(w + p.vf), (TileInfo*)(w + p.vi), false, {}, nullptr};
    attend_pack(k, p.DP, st);
    const TilesArgs t{a, (_Float16*)(w + p.kf), (_Float16*)(w + p.vf), (TileInfo*)(w + p.ki), (TileInfo*)(w + p.vi),
                      make_fastdiv(p.G), p.M, p.blocks, p.splits, wide, part, plse};
    const int64_t grid = (int64_t)p.slabs * p.blocks * p.splits;
    if (p.DP == 32) run_tiles<32>(t, grid, st);
    else if (p.DP == 64) run_tiles<64>(t, grid, st);
    else if (p.DP == 96) run_tiles<96>(t, grid, st);
    else run_tiles<128>(t, grid, st);
  }
  if (p.splits > 1) klaunch(attend_join, dim3(p.M, p.slabs), dim3(128), 0, st, JoinArgs{a, p.M, p.splits, part, plse});
}

}  // namespace tgk
