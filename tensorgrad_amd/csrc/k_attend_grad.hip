// Gradients of masked attention for gfx950. With P = exp(score - top) share, D_i = dy_i . y_i, dP_ij = dy_i . v_j,
//   ds = P (dP - D) (1 - tanh^2),  dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i P_ij dy_i
// (sums over i run over the query heads that share the key head). Two kernels, each with the whole of its own sums, so that
// nothing is added by atomics and results repeat bit for bit; scores and dP are computed in both (7 products instead of 5):
//  * attend_grad_kv: a wavefront keeps 16 keys, k and v in registers, and walks the query rows; scores are computed as
//    queries x keys, so that P and ds are the B fragments of dv and dk as they stand;
//  * attend_grad_q: a wavefront keeps 16 query rows and walks the keys, scores transposed as in the forward pass.
// The walked operands are packed once (attend_pack, k_attend.hip); top and D come with them. A row's share is a factor of all
// that is linear in its dy: dy is packed, and D made, with it.
#include "attend_dev.h"

namespace tgk {
namespace {

struct GradArgs {
  AttendGradDesc g;
  const _Float16 *qr, *qc, *gr, *gc, *kr, *kc, *vr;   // row / column fragments of q, dy, k, v
  const TileInfo *qi, *gi, *ki, *vi;
  const float *qside, *kside;
  FastDiv group;
  int M, qtiles, ktiles, blocks, splits, qsplits, least;   // splits: parts of the query rows, of `least` tiles; qsplits: of the keys
  bool wide;
  float *pk, *pv, *pq;                                // parts: of dk, dv [split][slab][Tk][D or Dv], of dq [qsplit][slab][M][D]
  int* parts;                                         // with documents or a window: parts of dk and dv that were written, [slab][blocks]
};

// ---- dk, dv --------------------------------------------------------------------------------------

// Query tiles [from, to) that the masks by position let see any of the keys [k0, k0 + 128).
__device__ __forceinline__ void seeing_tiles(const GradArgs& A, const Sight& s, int k0, int& from, int& to) {
  int64_t i0 = 0;                  // first position index that sees any: a prefix shows its keys to all
  if (s.causal && k0 >= s.prefix) i0 = (int64_t)k0 - s.first;
  if (s.positional) i0 = max(i0, (int64_t)-s.first);
  from = (int)min(max(i0, (int64_t)0) * A.group.d / kTile, (int64_t)A.qtiles);
  to = k0 < s.n ? A.qtiles : 0;
  if (s.window && k0 >= s.stay) {  // the last of the keys leaves the window
    const int64_t i1 = (int64_t)k0 + 127 + s.window - s.first;
    to = (int)min((int64_t)to, (max(i1, (int64_t)0) * A.group.d + kTile - 1) / kTile);
  }
}
// Those of part `split`, equal stretches of all rows, so that blocks that run together walk the same ones. False: none, which
// the join finds again and does not read. With documents or a window the stretch that sees a key block is short: there its tiles are
// cut into equal parts, of 8 at least (few rows with a window: 3), when they are known (8 x 1000 positions, 2 key heads of 64:
// documents of 50 take 47 us and 10 to join instead of 121 uncut, of 170 66 and 11 instead of 165, one document 120 and 13 instead
// of 282; 4096 rows of 4 slabs, head size 128, a window of 512 and 4 sinks, 80 tiles a block: 257 and 36, in parts of 20 at least
// 369 and 28, by equal stretches of all rows 409). With a window the long walks, of keys that stay, start first.
__device__ __forceinline__ bool part_rows(const GradArgs& A, const Sight& s, int k0, int split, int& from, int& to) {
  seeing_tiles(A, s, k0, from, to);
  if (A.splits == 1 || s.doc || s.window) return true;
  const int each = (A.qtiles + A.splits - 1) / A.splits;
  from = max(from, split * each);
  to = min(to, (split + 1) * each);
  return from < to;
}

__device__ __forceinline__ bool own_part(const GradArgs& A, const Sight& s, int split, int slab, int blk, int& t0, int& t1) {
  if (!(s.doc || s.window) || A.splits == 1) return true;
  const int each = max((t1 - t0 + A.splits - 1) / A.splits, A.least);
  if (split == 0 && threadIdx.x == 0) A.parts[slab * A.blocks + blk] = (t1 - t0 + each - 1) / each;
  t0 += split * each;
  t1 = min(t0 + each, t1);
  return t0 < t1;
}

// Where dk and dv of key j go.
__device__ __forceinline__ float* dk_row(const GradArgs& A, int split, int slab, int b, int hk, int j) {
  if (!A.g.dk.p) return nullptr;
  if (A.splits > 1) return A.pk + (((int64_t)split * A.g.a.B * A.g.a.Hk + slab) * A.g.a.Tk + j) * A.g.a.D;
  return A.g.dk.p + b * A.g.dk.b + hk * A.g.dk.h + (int64_t)j * A.g.dk.t;
}
__device__ __forceinline__ float* dv_row(const GradArgs& A, int split, int slab, int b, int hk, int j) {
  if (!A.g.dv.p) return nullptr;
  if (A.splits > 1) return A.pv + (((int64_t)split * A.g.a.B * A.g.a.Hk + slab) * A.g.a.Tk + j) * A.g.a.Dv;
  return A.g.dv.p + b * A.g.dv.b + hk * A.g.dv.h + (int64_t)j * A.g.dv.t;
}

// A wavefront's keys [j0, j0 + 16) over query rows [r0, r1) in plain f32.
template <int WHAT>
__device__ __forceinline__ void plain_keys(const GradArgs& A, const Sight& s, int split, int slab, int b, int hk, int j0, int r0, int r1) {
  const AttendDesc& a = A.g.a;
  const int lane = threadIdx.x & 63, G = (int)A.group.d;
  r1 = min(r1, A.M);
  auto row = [&](const Rows& x, int r) { return x.p + b * x.b + (hk * G + r % G) * x.h + (int64_t)(r / G) * x.t; };
#pragma unroll 1
  for (int j = j0; j < min(j0 + 16, a.Tk); ++j) {
    const float* k = a.k.p + b * a.k.b + hk * a.k.h + (int64_t)j * a.k.t;
    const float* v = a.v.p + b * a.v.b + hk * a.v.h + (int64_t)j * a.v.t;
    const int doc = s.doc ? s.doc[j] : 0;
    float dk[2] = {0, 0}, dv[2] = {0, 0};
#pragma unroll 1
    for (int c = r0; c < r1; c += 64) {
      const int r = c + lane;
      float p = 0, ds = 0;
      if (r < r1) {
        const float* side = A.qside + ((int64_t)slab * A.qtiles + r / kTile) * (kSide * kTile) + r % kTile;
        if (j < __float_as_int(side[QS_BELOW * kTile]) && (j >= sees_from(s, __float_as_int(side[QS_POS * kTile])) || j < s.stay) &&
            (!s.doc || (doc >= 0 && __float_as_int(side[QS_DOC * kTile]) == doc))) {
          const PlainPair z = plain_score(a, plain_dot(row(a.q, r), k, a.D), side[QS_SLOPE * kTile], __float_as_int(side[QS_POS * kTile]) - j);
          const float share = side[QS_SHARE * kTile], w = __builtin_amdgcn_exp2f(z.score - side[QS_TOP * kTile]);
          p = w * share;
          ds = w * fmaf(plain_dot(row(A.g.dy, r), v, a.Dv), share, -side[QS_DOT * kTile]) * z.slack;
        }
      }
      if (WHAT & 2) plain_add(dv, p, [&](int z) { return row(A.g.dy, min(c + z, A.M - 1)); }, a.Dv);
      if (WHAT & 1) plain_add(dk, ds, [&](int z) { return row(a.q, min(c + z, A.M - 1)); }, a.D);
    }
    float* ok = dk_row(A, split, slab, b, hk, j);
    float* ov = dv_row(A, split, slab, b, hk, j);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (WHAT & 1 && ok && 64 * e + lane < a.D) ok[64 * e + lane] = dk[e] * a.scale;
      if (WHAT & 2 && ov && 64 * e + lane < a.Dv) ov[64 * e + lane] = dv[e];
    }
  }
}

// Eight wavefronts of 16 keys. WHAT: 1 for dk, 2 for dv, 3 for both in one walk. Up to head size 64 two blocks share a CU. Both
// gradients of 4096 capped causal rows of 16 heads of 128: 679 us (by 32 keys 990, in walks of their own); of 8 heads of 64:
// 194 us (205); of 8 x 1000 rows of 8 heads of 64 in documents of 170: 66 us (81); of 32 without documents: 87 us.
template <int DP, bool RICH, int WHAT, bool WIN>
__global__ __launch_bounds__(512, DP <= 64 ? 4 : 2) void attend_grad_kv(GradArgs A) {
  constexpr int N = DP / 32, F = 4 * N;                      // chunks of 32 features; fragments of an operand
  constexpr bool DK = WHAT & 1, DV = WHAT & 2;
  constexpr int F_GR = F, F_QC = F_GR + (DK ? F : 0), F_GC = F_QC + (DK ? F : 0), F_SIDE = F_GC + (DV ? F : 0), NF = F_SIDE + kSideFrags;
  __shared__ __align__(16) _Float16 lds[2 * NF * kFrag];
  __shared__ int range[5];
  const AttendDesc& a = A.g.a;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, l = lane & 15;
  int slab, item;
  place(blockIdx.x, a.B * a.Hk, slab, item);
  if (item >= A.blocks * A.splits) return;
  // blocks that start together walk the same rows; with a window, those of the first keys start first
  const int split = WIN ? item % A.splits : A.splits - 1 - item / A.blocks, blk = WIN ? item / A.splits : item % A.blocks;
  const int b = slab / a.Hk, hk = slab % a.Hk;
  const Sight s = sight<WIN>(a, b);
  const int j0 = blk * 128 + w * 16, jt = j0 / kTile * kTile, j = j0 + l;   // masks are judged by whole tiles of keys
  const bool valid = j < a.Tk;
  const int doc = s.doc && valid ? s.doc[j] : -1;
  const int64_t kt = (int64_t)slab * A.ktiles + min(jt / kTile, A.ktiles - 1);
  TileInfo mine = A.ki[kt];
  const bool own = jt < a.Tk && (mine.odd || (DK && A.vi[kt].odd));
  if (jt >= a.Tk) {
    mine.dmin = INT32_MAX;
    mine.dmax = INT32_MIN;
  }
  const TileInfo* qi = A.qi + (int64_t)slab * A.qtiles;
  const TileInfo* gi = A.gi + (int64_t)slab * A.qtiles;
  int from, to;
  if (!part_rows(A, s, blk * 128, split, from, to)) return;   // nothing, and the join knows
  const Range range_ = tile_range(s, from, to, gi, qi, gi, mine.dmin, mine.dmax, own, range);
  int t0 = range_.t0, t1 = range_.t1;
  if (!own_part(A, s, split, slab, blk, t0, t1)) return;
  if (__builtin_expect(range_.odd, 0)) {
    plain_keys<WHAT>(A, s, split, slab, b, hk, j0, t0 * kTile, t1 * kTile);
    return;
  }

  half8 kh[N], kl[N], vh[DK ? N : 1], vl[DK ? N : 1];
  const int ke = load_rows<N>(a.k.p + b * a.k.b + hk * a.k.h + (int64_t)min(j, a.Tk - 1) * a.k.t, valid, a.D, A.wide, 1.0f, kh, kl);
  int ve = 0;
  if constexpr (DK) ve = load_rows<N>(a.v.p + b * a.v.b + hk * a.v.h + (int64_t)min(j, a.Tk - 1) * a.v.t, valid, a.Dv, A.wide, 1.0f, vh, vl);
  const int64_t tile0 = (int64_t)slab * A.qtiles + t0;
  const uint32_t base = lds_address(lds) + w * 1024, lane16 = lane * 16;
  const char* qr = (const char*)(A.qr + tile0 * (F * kFrag)) + w * 1024;
  const char* gr = (const char*)(A.gr + tile0 * (F * kFrag)) + w * 1024;
  const char* qc = (const char*)(A.qc + tile0 * (F * kFrag)) + w * 1024;
  const char* gc = (const char*)(A.gc + tile0 * (F * kFrag)) + w * 1024;
  const char* side_p = (const char*)(A.qside + tile0 * (kSide * kTile)) + w * 1024;
  auto fetch = [&](int buf) {      // the next tile
    const uint32_t to = base + buf * (NF * 1024);
    frags_to_lds<F>(qr, to, lane16, w);
    qr += F * 1024;
    if (DK) {
      frags_to_lds<F>(gr, to + F_GR * 1024, lane16, w);
      frags_to_lds<F>(qc, to + F_QC * 1024, lane16, w);
      gr += F * 1024;
      qc += F * 1024;
    }
    if (DV) {
      frags_to_lds<F>(gc, to + F_GC * 1024, lane16, w);
      gc += F * 1024;
    }
    frags_to_lds<kSideFrags>(side_p, to + F_SIDE * 1024, lane16, w);
    side_p += kSide * kTile * 4;
  };

  f32x4 dk[2 * N], dv[2 * N];
#pragma unroll
  for (int d = 0; d < 2 * N; ++d) dk[d] = dv[d] = f32x4{};
  int ck = kUnset, cv = kUnset;
  const Score sc = score_parts(a);
  if (t0 < t1) fetch(0);
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1, r0 = t * kTile;
    loads_done();
    __syncthreads();
    if (t + 1 < t1) fetch(buf ^ 1);
    const _Float16* L = lds + buf * (NF * kFrag);
    const float* side = (const float*)(L + F_SIDE * kFrag);
    const TileInfo qt = side_info(side, 0), gt = side_info(side, 1);
    Span rows;
    rows.pmin = s.first + (int)fastdiv((uint32_t)r0, A.group);
    rows.pmax = s.first + (int)fastdiv((uint32_t)min(r0 + kTile - 1, A.M - 1), A.group);
    rows.dmin = gt.dmin;
    rows.dmax = gt.dmax;
    rows.same = gt.same;
    if (__builtin_expect(j0 >= a.Tk || !any_seen(s, rows, mine, jt), 0)) continue;
    // element q: row r0 + 16 (q / 4) + 4 g + q % 4
    float x[8], y[8] = {};
    if constexpr (DK && N == 2) {  // the pair in turn would spill registers here
      scores<false, N>(L, 0, kh, kl, x);
      scores<false, N>(L, F_GR, vh, vl, y);
    } else if constexpr (DK) pair<false, N>(L, 0, kh, kl, x, F_GR, vh, vl, y);
    else {
      scores<false, N>(L, 0, kh, kl, x);
    }
    if (__builtin_expect(qt.uneven, 0)) per_row(x, side + QS_RELQ * kTile, g);
    if (DK && __builtin_expect(gt.uneven, 0)) per_row(y, side + QS_RELG * kTile, g);
    const float yunit = dot_unit(exponent(gt.inv) - ve);
    float f = score_unit(sc, exponent(qt.inv) - ke);
    if (RICH && a.cap > 0) {
      tanh_all(x, f);
      f = a.cap * kLog2e;
    }
    const bool all = A.M - r0 >= kTile && all_seen(s, rows, mine, jt);
#pragma unroll
    for (int q4 = 0; q4 < 2; ++q4) {
      const int at = 16 * q4 + 4 * g;
      const f32x4 top = *(const f32x4*)(side + QS_TOP * kTile + at), dot = *(const f32x4*)(side + QS_DOT * kTile + at);
      f32x4 less;                  // score less top
      if (RICH && a.slopes) {
        const f32x4 pos = *(const f32x4*)(side + QS_POS * kTile + at), slope = *(const f32x4*)(side + QS_SLOPE * kTile + at);
#pragma unroll
        for (int e = 0; e < 4; ++e) less[e] = score_of(true, x[4 * q4 + e], f, slope[e], __float_as_int(pos[e]) - j) - top[e];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) less[e] = RICH ? rounded_mul(x[4 * q4 + e], f) - top[e] : fmaf(x[4 * q4 + e], f, -top[e]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int q = 4 * q4 + e;
        const float p = __builtin_amdgcn_exp2f(less[e]);
        if (DK) {
          y[q] = p * fmaf(y[q], yunit, -dot[e]);
          if (RICH && a.cap > 0) y[q] *= fmaf(-x[q], x[q], 1.0f);   // 1 - tanh^2
        }
        x[q] = p;
      }
      if (__builtin_expect(!all, 0)) {
        const f32x4 below = *(const f32x4*)(side + QS_BELOW * kTile + at), rdoc = *(const f32x4*)(side + QS_DOC * kTile + at);
        const f32x4 pos = *(const f32x4*)(side + QS_POS * kTile + at);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool ok = (j < __float_as_int(below[e])) & ((j >= sees_from(s, __float_as_int(pos[e]))) | (j < s.stay)) &
                          (!s.doc | ((doc >= 0) & (__float_as_int(rdoc[e]) == doc)));
          x[4 * q4 + e] = ok ? x[4 * q4 + e] : 0.0f;
          y[4 * q4 + e] = ok ? y[4 * q4 + e] : 0.0f;
        }
      }
    }
    if (DV) {
      if (__builtin_expect(gt.uneven, 0)) per_row(x, side + QS_RELG * kTile, g);
      float change = 1;
      const int e = fit_unit(cv, largest(x), exponent(gt.scale), &change);
      rescale(dv, change);
      accumulate(dv, x, pow2(e), L, F_GC);
    }
    if (DK) {
      if (__builtin_expect(qt.uneven, 0)) per_row(y, side + QS_RELQ * kTile, g);
      float change = 1;
      const int e = fit_unit(ck, largest(y), exponent(qt.scale), &change);
      rescale(dk, change);
      accumulate(dk, y, pow2(e), L, F_QC);
    }
  }

  if (!valid) return;
  float* ok = dk_row(A, split, slab, b, hk, j);
  float* ov = dv_row(A, split, slab, b, hk, j);
  if (DK && ok) store_row(ok, dk, ck, a.scale, a.D, A.splits > 1 ? a.D % 4 == 0 : A.wide, g);
  if (DV && ov) store_row(ov, dv, cv, 1.0f, a.Dv, A.splits > 1 ? a.Dv % 4 == 0 : A.wide, g);
}

// The parts of dk, dv and dq in order: a block takes 32 keys of the 128 that the parts were split for, or 32 query rows.
__global__ __launch_bounds__(256) void attend_grad_join(GradArgs A) {
  const AttendDesc& a = A.g.a;
  const int what = blockIdx.y, n = what == 1 ? a.Dv : a.D, G = what == 2 ? (int)A.group.d : 1, T = what == 2 ? A.M : a.Tk;
  const Rows& o = what == 0 ? A.g.dk : what == 1 ? A.g.dv : A.g.dq;
  if (!o.p || (what == 2 ? A.qsplits : A.splits) == 1) return;
  const int tiles = max(A.ktiles, A.qtiles), slab = (int)(blockIdx.x / (unsigned)tiles), r0 = (int)(blockIdx.x % (unsigned)tiles) * kTile;
  if (r0 >= T) return;
  const int b = slab / a.Hk, hk = slab % a.Hk;
  const Sight s = sight(a, b);
  int first = 0, last = A.qsplits - 1;   // parts that were written
  if (what < 2 && (s.doc || s.window)) {
    last = A.parts[slab * A.blocks + r0 / 128] - 1;
  } else if (what < 2) {
    first = A.splits;
    last = -1;
    for (int z = threadIdx.x & 63; z < A.splits; z += 64) {
      int from, to;
      if (part_rows(A, s, r0 / 128 * 128, z, from, to)) {
        first = min(first, z);
        last = max(last, z);
      }
    }
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
      first = min(first, __shfl_xor(first, o));
      last = max(last, __shfl_xor(last, o));
    }
  }
  const int64_t all = (int64_t)a.B * a.Hk * T * n;
  const float* part = (what == 0 ? A.pk : what == 1 ? A.pv : A.pq) + ((int64_t)slab * T + r0) * n;
  auto to = [&](int r) { return o.p + b * o.b + (hk * G + r % G) * o.h + (int64_t)(r / G) * o.t; };
  const int end = min(kTile, T - r0) * n;
  const bool wide = n % 4 == 0, aligned = A.wide;
  for (int e = 4 * threadIdx.x; e < end; e += 1024) {
    f32x4 x = {};
#pragma unroll 4
    for (int z = first; z <= last; ++z) {
      const float* from = part + z * all + e;
      if (wide) x += *(const f32x4*)from;
      else
#pragma unroll
        for (int q = 0; q < 4; ++q) if (e + q < end) x[q] += from[q];
    }
    if (wide && aligned) {
      *(f32x4*)(to(r0 + e / n) + e % n) = x;
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) if (e + q < end) to(r0 + (e + q) / n)[(e + q) % n] = x[q];
    }
  }
}

// ---- dq --------------------------------------------------------------------------------------------

// Where dq of row r of a slab goes.
__device__ __forceinline__ float* dq_row(const GradArgs& A, int split, int slab, int b, int head, int r, int i) {
  if (A.qsplits > 1) return A.pq + (((int64_t)split * A.g.a.B * A.g.a.Hk + slab) * A.M + r) * A.g.a.D;
  return A.g.dq.p + b * A.g.dq.b + head * A.g.dq.h + (int64_t)i * A.g.dq.t;
}
// A wavefront's rows [row0, row0 + 16) over keys [j0, j1) in plain f32.
__device__ __forceinline__ void plain_dq(const GradArgs& A, const Sight& s, int split, int slab, int b, int hk, int row0, int j0, int j1) {
  const AttendDesc& a = A.g.a;
  const int lane = threadIdx.x & 63, G = (int)A.group.d;
  const float* k = a.k.p + b * a.k.b + hk * a.k.h;
  const float* v = a.v.p + b * a.v.b + hk * a.v.h;
#pragma unroll 1
  for (int r = row0; r < min(row0 + 16, A.M); ++r) {
    const int i = r / G, head = hk * G + r % G;
    const float* q = a.q.p + b * a.q.b + head * a.q.h + (int64_t)i * a.q.t;
    const float* dy = A.g.dy.p + b * A.g.dy.b + head * A.g.dy.h + (int64_t)i * A.g.dy.t;
    const float* side = A.qside + ((int64_t)slab * A.qtiles + r / kTile) * (kSide * kTile) + r % kTile;
    const int p = __float_as_int(side[QS_POS * kTile]), doc = __float_as_int(side[QS_DOC * kTile]);
    const int end = min(j1, __float_as_int(side[QS_BELOW * kTile])), from = sees_from(s, p);
    float dq[2] = {0, 0};
#pragma unroll 1
    for (int c = j0; c < end; c += 64) {
      const int j = c + lane;
      float ds = 0;
      if (j < end && (j >= from || j < s.stay) && (!s.doc || (doc >= 0 && s.doc[j] == doc))) {
        const PlainPair z = plain_score(a, plain_dot(k + j * a.k.t, q, a.D), side[QS_SLOPE * kTile], p - j);
        ds = __builtin_amdgcn_exp2f(z.score - side[QS_TOP * kTile]) *
             fmaf(plain_dot(v + j * a.v.t, dy, a.Dv), side[QS_SHARE * kTile], -side[QS_DOT * kTile]) * z.slack;
      }
      plain_add(dq, ds, [&](int z) { return k + min(c + z, a.Tk - 1) * a.k.t; }, a.D);
    }
    float* o = dq_row(A, split, slab, b, head, r, i);
#pragma unroll
    for (int e = 0; e < 2; ++e) if (64 * e + lane < a.D) o[64 * e + lane] = dq[e] * a.scale;
  }
}

// Eight wavefronts of 16 query rows. 4096 capped causal rows of 16 heads of 128: 374 us (470 by 32 rows); 8 x 1000 rows of 8
// heads of 64 in documents of 170: 42 us (57).
template <int DP, bool RICH, bool WIN>
__global__ __launch_bounds__(512) void attend_grad_q(GradArgs A) {
  constexpr int N = DP / 32, F = 4 * N, F_V = F, F_KC = 2 * F, F_SIDE = 3 * F, NF = F_SIDE + kSideFrags;
  __shared__ __align__(16) _Float16 lds[2 * NF * kFrag];
  __shared__ int range[5];
  const AttendDesc& a = A.g.a;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), g4 = lane >> 4, l = lane & 15;
  const int rblocks = (A.M + 127) / 128;
  int slab, item;
  place(blockIdx.x, a.B * a.Hk, slab, item);
  if (item >= rblocks * A.qsplits) return;
  const int split = item % A.qsplits, blk = rblocks - 1 - item / A.qsplits;
  const int b = slab / a.Hk, hk = slab % a.Hk, G = (int)A.group.d;
  const Sight s = sight<WIN>(a, b);
  const int row0 = blk * 128 + w * 16, r = row0 + l, rr = min(r, A.M - 1);
  const bool valid = r < A.M;
  const int i = (int)fastdiv((uint32_t)rr, A.group), g = rr - i * G, head = hk * G + g;
  const int p = s.first + i, doc = doc_at(s, p), below = sees_below(s, p), from = sees_from(s, p);
  const int qt = min(row0 / kTile, A.qtiles - 1), rt = row0 / kTile * kTile;   // masks are judged by whole tiles of rows
  const float* mine = A.qside + ((int64_t)slab * A.qtiles + qt) * (kSide * kTile) + row0 % kTile + l;
  const float top = mine[QS_TOP * kTile], share = mine[QS_SHARE * kTile], dot = mine[QS_DOT * kTile];
  const TileInfo gt = A.gi[(int64_t)slab * A.qtiles + qt];
  const bool own = rt < A.M && (gt.odd || A.qi[(int64_t)slab * A.qtiles + qt].odd);
  Span me;
  me.pmin = s.first + (int)fastdiv((uint32_t)min(rt, A.M - 1), A.group);
  me.pmax = s.first + (int)fastdiv((uint32_t)min(rt + kTile - 1, A.M - 1), A.group);
  me.dmin = rt < A.M ? gt.dmin : INT32_MAX;
  me.dmax = rt < A.M ? gt.dmax : INT32_MIN;
  me.same = gt.same;

  const TileInfo* ki = A.ki + (int64_t)slab * A.ktiles;
  const TileInfo* vi = A.vi + (int64_t)slab * A.ktiles;
  const int last = s.first + (int)fastdiv((uint32_t)min(blk * 128 + 127, A.M - 1), A.group);
  int end = s.n;
  if (s.causal) end = min(end, max(last + 1, s.prefix));
  if (s.positional && last < 0) end = 0;
  const Gap gap = gap_before(s, max(s.first + (int)fastdiv((uint32_t)(blk * 128), A.group), 0));
  const Range range_ = tile_range(s, 0, (end + kTile - 1) / kTile, ki, ki, vi, me.dmin, me.dmax, own, range, gap);
  const Walk walk = walk_part<WIN>(range_.t0, range_.t1, gap, split, A.qsplits);
  const int t0 = walk.t0, t1 = walk.t1;
  if (__builtin_expect(range_.odd, 0)) {
    plain_dq(A, s, split, slab, b, hk, row0, t0 * kTile, t1 * kTile);
    return;
  }

  half8 qh[N], ql[N], gh[N], gl[N];
  const Score sc = score_parts(a);
  const int qe = load_rows<N>(a.q.p + b * a.q.b + head * a.q.h + (int64_t)i * a.q.t, valid, a.D, A.wide, sc.part, qh, ql);
  const int ge = load_rows<N>(A.g.dy.p + b * A.g.dy.b + head * A.g.dy.h + (int64_t)i * A.g.dy.t, valid, a.Dv, A.wide, share, gh, gl);
  const float slope = RICH && a.slopes ? a.slopes[head] * kLog2e : 0.0f;
  const int64_t tile0 = (int64_t)slab * A.ktiles + t0;
  const uint32_t base = lds_address(lds) + w * 1024, lane16 = lane * 16;
  const char* kr = (const char*)(A.kr + tile0 * (F * kFrag)) + w * 1024;
  const char* vr = (const char*)(A.vr + tile0 * (F * kFrag)) + w * 1024;
  const char* kc = (const char*)(A.kc + tile0 * (F * kFrag)) + w * 1024;
  const char* side_p = (const char*)(A.kside + tile0 * (kSide * kTile)) + w * 1024;
  auto fetch = [&](int buf, int step) {   // the tile `step` ahead of the last
    const uint32_t to = base + buf * (NF * 1024);
    kr += (int64_t)step * (F * 1024);
    vr += (int64_t)step * (F * 1024);
    kc += (int64_t)step * (F * 1024);
    side_p += (int64_t)step * (kSide * kTile * 4);
    frags_to_lds<F>(kr, to, lane16, w);
    frags_to_lds<F>(vr, to + F_V * 1024, lane16, w);
    frags_to_lds<F>(kc, to + F_KC * 1024, lane16, w);
    frags_to_lds<kSideFrags>(side_p, to + F_SIDE * 1024, lane16, w);
  };

  f32x4 dq[2 * N];
#pragma unroll
  for (int d = 0; d < 2 * N; ++d) dq[d] = f32x4{};
  int cq = kUnset;
  const bool cap = RICH && a.cap > 0;
  if (t0 < t1) fetch(0, 0);
  for (int t = t0, next, buf = 0; t < t1; t = next, buf ^= 1) {
    const int j0 = t * kTile;
    next = WIN ? walk.after(t) : t + 1;
    loads_done();
    __syncthreads();
    if (next < t1) fetch(buf ^ 1, next - t);
    const _Float16* L = lds + buf * (NF * kFrag);
    const float* side = (const float*)(L + F_SIDE * kFrag);
    const TileInfo kt = side_info(side, 0), vt = side_info(side, 1);
    if (__builtin_expect(!any_seen(s, me, kt, j0), 0)) continue;
    // element q: key j0 + 16 (q / 4) + 4 g4 + q % 4
    float x[8], y[8];
    pair<true, N>(L, 0, qh, ql, x, F_V, gh, gl, y);
    if (__builtin_expect(kt.uneven, 0)) per_row(x, side + KS_RELK * kTile, g4);
    if (__builtin_expect(vt.uneven, 0)) per_row(y, side + KS_RELV * kTile, g4);
    const float yunit = dot_unit(exponent(vt.inv) - ge);
    float f = score_unit(sc, exponent(kt.inv) - qe);
    if (cap) {
      tanh_all(x, f);
      f = a.cap * kLog2e;
    }
    float less[8];                 // score less top
    if (RICH && a.slopes) {
#pragma unroll
      for (int q = 0; q < 8; ++q) less[q] = score_of(true, x[q], f, slope, p - (j0 + 16 * (q / 4) + 4 * g4 + q % 4)) - top;
    } else {
#pragma unroll
      for (int q = 0; q < 8; ++q) less[q] = RICH ? rounded_mul(x[q], f) - top : fmaf(x[q], f, -top);
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      y[q] = __builtin_amdgcn_exp2f(less[q]) * fmaf(y[q], yunit, -dot);
      if (cap) y[q] *= fmaf(-x[q], x[q], 1.0f);
    }
    if (__builtin_expect(!all_seen(s, me, kt, j0), 0)) {
#pragma unroll
      for (int q = 0; q < 8; ++q) y[q] = key_seen(s, side, j0, 16 * (q / 4) + 4 * g4 + q % 4, below, from, doc) ? y[q] : 0.0f;
    }
    if (__builtin_expect(kt.uneven, 0)) per_row(y, side + KS_RELK * kTile, g4);
    float change = 1;
    const int e = fit_unit(cq, largest(y), exponent(kt.scale), &change);
    rescale(dq, change);
    accumulate(dq, y, pow2(e), L, F_KC);
  }
  if (valid)
    store_row(dq_row(A, split, slab, b, head, r, i), dq, cq, a.scale, a.D, A.qsplits > 1 ? a.D % 4 == 0 : A.wide, g4);
}

// ---- plan --------------------------------------------------------------------------------------------

struct GradPlan {
  int DP, M, G, qtiles, ktiles, blocks, splits, qsplits, least, slabs;
  int64_t qr, qc, gr, gc, kr, kc, vr, qi, gi, ki, vi, qside, kside, pk, pv, pq, parts, bytes;
};
GradPlan grad_plan(const AttendGradDesc& g) {
  const AttendDesc& a = g.a;
  GradPlan p{};
  p.DP = attend_dp(a);
  p.G = a.H / a.Hk;
  p.M = p.G * a.Tq;
  p.slabs = a.B * a.Hk;
  p.qtiles = (p.M + kTile - 1) / kTile;
  p.ktiles = (a.Tk + kTile - 1) / kTile;
  p.blocks = (a.Tk + 127) / 128;
  const int64_t have = (int64_t)p.slabs * p.blocks;
  // About 1024 blocks, two to four rounds of the card: 512 leave it to the longest (4096 causal rows of 4 slabs, head size 128:
  // 832 us and 21 to join, instead of 677 and 31), 2048 write and join twice the parts (624 and 58).
  // Of a window's few rows parts of 3 tiles; training steps by those and by 8: 19 slabs of 7 heads, 81 positions, head size 128 (38
  // parts of 8) 85 us and 96, 16 of 4 heads, 300 x 64 (192) 80 and 88, 8 of 2, 700 x 128 (240) 112 and 111, 8 of 1, 1000 x 64 (256) 74
  // and 80; from there on those of 8, but for the least work: 8 of 4, 600 x 96 (360) 155 and 123, 16 of 4, 512 x 64 (512) 114 and 107.
  p.least = a.window && have * (p.qtiles / 8) < 256 ? 3 : 8;
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>((1024 + have - 1) / have, p.qtiles / p.least));
  // dq in parts only where its blocks leave compute units idle: 224 of them (32 slabs of 777 rows, head size 96) take 55 us, in
  // two parts 52 and 6 to join.
  p.qsplits = (int)std::max<int64_t>(1, std::min<int64_t>(256 / ((int64_t)p.slabs * ((p.M + 127) / 128)), p.ktiles / 8));
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t b = at;
    at += (bytes + 255) / 256 * 256;
    return b;
  };
  const int64_t q = (int64_t)p.slabs * p.qtiles, k = (int64_t)p.slabs * p.ktiles, tile = (int64_t)p.DP * kTile * 4;
  p.qr = take(q * tile);
  p.qc = take(q * tile);
  p.gr = take(q * tile);
  p.gc = take(q * tile);
  p.kr = take(k * tile);
  p.kc = take(k * tile);
  p.vr = take(k * tile);
  p.qi = take(q * sizeof(TileInfo));
  p.gi = take(q * sizeof(TileInfo));
  p.ki = take(k * sizeof(TileInfo));
  p.vi = take(k * sizeof(TileInfo));
  p.qside = take(q * kSide * kTile * 4);
  p.kside = take(k * kSide * kTile * 4);
  if (p.splits > 1) {
    p.pk = take((int64_t)p.splits * p.slabs * a.Tk * a.D * 4);
    p.pv = take((int64_t)p.splits * p.slabs * a.Tk * a.Dv * 4);
    p.parts = take(have * 4);
  }
  if (p.qsplits > 1) p.pq = take((int64_t)p.qsplits * p.slabs * p.M * a.D * 4);
  p.bytes = at;
  return p;
}

template <int DP, bool RICH, bool WIN>
void run_grad(const GradArgs& A, int slabs, hipStream_t st) {
  const AttendGradDesc& g = A.g;
  const dim3 keys(place_grid(slabs, (int64_t)A.blocks * A.splits));
  if (g.dk.p && g.dv.p) klaunch(attend_grad_kv<DP, RICH, 3, WIN>, keys, dim3(512), 0, st, A);
  else if (g.dk.p) klaunch(attend_grad_kv<DP, RICH, 1, WIN>, keys, dim3(512), 0, st, A);
  else if (g.dv.p) klaunch(attend_grad_kv<DP, RICH, 2, WIN>, keys, dim3(512), 0, st, A);
  if (g.dq.p)
    klaunch(attend_grad_q<DP, RICH, WIN>, dim3(place_grid(slabs, (int64_t)((A.M + 127) / 128) * A.qsplits)), dim3(512), 0, st, A);
}
template <int DP>
void run_grad(const GradArgs& A, int slabs, hipStream_t st) {
  const bool rich = A.g.a.cap > 0 || A.g.a.slopes;
  if (rich && A.g.a.window) run_grad<DP, true, true>(A, slabs, st);
  else if (rich) run_grad<DP, true, false>(A, slabs, st);
  else if (A.g.a.window) run_grad<DP, false, true>(A, slabs, st);
  else run_grad<DP, false, false>(A, slabs, st);
}

}  // namespace

int64_t attend_grad_workspace_bytes(const AttendGradDesc& g) { return attend_small_rows(g.a) ? 0 : grad_plan(g).bytes; }

void attend_grad(const AttendGradDesc& g, void* work, hipStream_t st) {
  if (attend_small_rows(g.a)) return attend_small_grad(g, st);
  const GradPlan p = grad_plan(g);
  const AttendDesc& a = g.a;
  char* w = (char*)work;
  auto half = [&](int64_t at) { return (_Float16*)(w + at); };
  auto info = [&](int64_t at) { return (TileInfo*)(w + at); };
  const bool wide = attend_wide(a.q, a.D) && attend_wide(a.k, a.D) && attend_wide(a.v, a.Dv) && attend_wide(g.dy, a.Dv) &&
                    (!g.dq.p || attend_wide(g.dq, a.D)) && (!g.dk.p || attend_wide(g.dk, a.D)) && (!g.dv.p || attend_wide(g.dv, a.Dv));
  Packs k{};
  k.n = 4;
  k.Hk = a.Hk;
  k.wide = wide;
  k.a = a;
  float *qs = (float*)(w + p.qside), *ks = (float*)(w + p.kside);
  k.job[0] = {a.q, a.D, p.G, p.M, p.qtiles, half(p.qr), half(p.qc), info(p.qi), true, qs, QS_RELQ, false, false, true, {}};
  k.job[1] = {g.dy, a.Dv, p.G, p.M, p.qtiles, half(p.gr), half(p.gc), info(p.gi), true, qs, QS_RELG, true, true, false, a.y};
  k.job[2] = {a.k, a.D, 1, a.Tk, p.ktiles, half(p.kr), half(p.kc), info(p.ki), false, ks, KS_RELK, false, true, false, {}};
  k.job[3] = {a.v, a.Dv, 1, a.Tk, p.ktiles, half(p.vr), nullptr, info(p.vi), false, ks, KS_RELV, true, false, false, {}};
  attend_pack(k, p.DP, st);
  const GradArgs A{g, half(p.qr), half(p.qc), half(p.gr), half(p.gc), half(p.kr), half(p.kc), half(p.vr),
                   info(p.qi), info(p.gi), info(p.ki), info(p.vi), qs, ks, make_fastdiv(p.G), p.M, p.qtiles,
                   p.ktiles, p.blocks, p.splits, p.qsplits, p.least, wide, (float*)(w + p.pk), (float*)(w + p.pv), (float*)(w + p.pq),
                   (int*)(w + p.parts)};
  if (p.DP == 32) run_grad<32>(A, p.slabs, st);
  else if (p.DP == 64) run_grad<64>(A, p.slabs, st);
  else if (p.DP == 96) run_grad<96>(A, p.slabs, st);
  else run_grad<128>(A, p.slabs, st);
  if ((p.splits > 1 && (g.dk.p || g.dv.p)) || (p.qsplits > 1 && g.dq.p))
    klaunch(attend_grad_join, dim3((unsigned)((int64_t)p.slabs * std::max(p.ktiles, p.qtiles)), 3), dim3(256), 0, st, A);
}

}  // namespace tgk
