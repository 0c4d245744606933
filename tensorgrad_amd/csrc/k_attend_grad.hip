// Gradients of masked attention for gfx950. With P = exp(score - lse), D_i = dy_i . y_i, dP_ij = dy_i . v_j,
//   ds = P (dP - D) (1 - tanh^2),  dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i P_ij dy_i
// (sums over i run over the query heads that share the key head). Two kernels, each with the whole of its own sums, so that
// nothing is added by atomics and results repeat bit for bit; scores and dP are computed in both (7 products instead of 5):
//  * attend_grad_kv: a wavefront keeps 32 keys, k and v in registers, and walks the query rows; scores are computed as
//    queries x keys, so that P and ds are the B fragments of dv and dk as they stand;
//  * attend_grad_q: a wavefront keeps 32 query rows and walks the keys, scores transposed as in the forward pass.
// The walked operands are packed once (attend_pack, k_attend.hip); lse and D come with them.
#include "attend_dev.h"

namespace tgk {
namespace {

struct GradArgs {
  AttendGradDesc g;
  const _Float16 *qr, *qc, *gr, *gc, *kr, *kc, *vr;   // row / column fragments of q, dy, k, v
  const TileInfo *qi, *gi, *ki, *vi;
  const float* rowinfo;
  FastDiv group;
  int M, qtiles, ktiles, blocks, splits;
  bool wide;
  float *pk, *pv;                                     // parts of dk, dv: [split][slab][Tk][D or Dv]
};

// This lane's column of acc (features), in units of 2^-c, to a row in memory.
template <int DB>
__device__ __forceinline__ void store_row(float* row, const f32x16 (&acc)[DB], int c, float scale, int n, bool wide) {
  const int h = (threadIdx.x >> 5) & 1;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int at = 32 * d + 8 * q + 4 * h;
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = __builtin_amdgcn_ldexpf(acc[d][4 * q + e], -c) * scale;
      if (wide) {
        if (at < n) *(f32x4*)(row + at) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) if (at + e < n) row[at + e] = v[e];
      }
    }
}

// ---- dk, dv --------------------------------------------------------------------------------------

template <int DP, bool RICH>
__global__ __launch_bounds__(256, DP <= 64 ? 2 : 1) void attend_grad_kv(GradArgs A) {
  constexpr int KC = DP / 16, DB = DP / 32;
  constexpr int F_GR = 2 * KC, F_QC = 4 * KC, F_GC = F_QC + 4 * DB, F_INFO = F_GC + 4 * DB, NF = F_INFO + 1;
  __shared__ __align__(16) _Float16 lds[2 * NF * kFrag];
  const AttendDesc& a = A.g.a;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, l = lane & 31;
  const uint32_t id = xcd_order(blockIdx.x, gridDim.x);
  const uint32_t per = (uint32_t)A.blocks * A.splits;
  const int slab = id / per, split = id % per % A.splits, blk = id % per / A.splits;   // the first keys are seen by most
  const int b = slab / a.Hk, hk = slab % a.Hk;
  const Sight s = sight(a, b);
  const int j0 = blk * 128 + w * kTile, j = j0 + l, kt = min(j0 / kTile, A.ktiles - 1);
  const bool valid = j < a.Tk;
  const float* krow = a.k.p + b * a.k.b + hk * a.k.h + (int64_t)min(j, a.Tk - 1) * a.k.t;
  const float* vrow = a.v.p + b * a.v.b + hk * a.v.h + (int64_t)min(j, a.Tk - 1) * a.v.t;
  half8 kh[KC], kl[KC], vh[KC], vl[KC];
  int vnorm;
  const int ke = load_rows<KC>(krow, valid, a.D, A.wide, kh, kl);
  const int ve = load_rows<KC>(vrow, valid, a.Dv, A.wide, vh, vl, &vnorm);
  const int doc = s.doc && valid ? s.doc[j] : -1;
  const TileInfo mine = A.ki[(int64_t)slab * A.ktiles + kt];

  // the query tiles that see any of the block's keys: from its first key's position on, unless a prefix shows it to all
  const TileInfo* qi = A.qi + (int64_t)slab * A.qtiles;
  const TileInfo* gi = A.gi + (int64_t)slab * A.qtiles;
  const int k0 = blk * 128;
  int t0 = 0, t1 = A.qtiles;
  if (k0 >= s.n) t1 = 0;
  int64_t i0 = 0;                  // first position index that sees anything here
  if (s.causal && k0 >= s.prefix) i0 = (int64_t)k0 - s.first;
  if (s.positional) i0 = max(i0, (int64_t)-s.first);
  t0 = (int)min(max(i0, (int64_t)0) * A.group.d / kTile, (int64_t)t1);
  if (s.doc) {
    __shared__ int range[4];
    if (tid < 4) range[tid] = tid & 1 ? INT32_MIN : INT32_MAX;
    __syncthreads();
    if (lane == 0 && j0 < a.Tk) {
      atomicMin(&range[0], mine.dmin);
      atomicMax(&range[1], mine.dmax);
    }
    __syncthreads();
    const int lo = range[0], hi = range[1];
    int first = INT32_MAX, end = INT32_MIN;
    for (int t = t0 + tid; t < t1; t += 256)
      if (gi[t].dmin <= hi && lo <= gi[t].dmax) {
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
    const int n = max(t1 - t0, 0), each = (n + A.splits - 1) / A.splits;
    t0 = min(t0 + split * each, t1);
    t1 = min(t0 + each, t1);
  }
  t0 = __builtin_amdgcn_readfirstlane(t0);
  t1 = __builtin_amdgcn_readfirstlane(t1);

  const int64_t tile0 = (int64_t)slab * A.qtiles;
  const uint32_t base = lds_address(lds), lane16 = lane * 16;
  auto fetch = [&](int t, int buf) {
#pragma unroll
    for (int f = 0; f < (NF + 3) / 4; ++f) {
      const int q = f * 4 + w;
      const _Float16* src;
      if (q < F_GR) src = A.qr + ((tile0 + t) * (2 * KC) + q) * kFrag;
      else if (q < F_QC) src = A.gr + ((tile0 + t) * (2 * KC) + q - F_GR) * kFrag;
      else if (q < F_GC) src = A.qc + ((tile0 + t) * (4 * DB) + q - F_QC) * kFrag;
      else if (q < F_INFO) src = A.gc + ((tile0 + t) * (4 * DB) + q - F_GC) * kFrag;
      else src = (const _Float16*)(A.rowinfo + (tile0 + t) * (kRowInfo * kTile));
      if (q < NF) frag_to_lds(src, base + (buf * NF + q) * (kFrag * 2), lane16);
    }
  };

  f32x16 dk[DB], dv[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) dk[d] = dv[d] = f32x16{};
  int ck = kUnset, cv = kUnset;
  const RowMap qmap = row_map(a.q, b, hk * (int)A.group.d, A.group), gmap = row_map(A.g.dy, b, hk * (int)A.group.d, A.group);
  if (t0 < t1) fetch(t0, 0);
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1, r0 = t * kTile;
    loads_done();
    __syncthreads();
    if (t + 1 < t1) fetch(t + 1, buf ^ 1);
    const TileInfo qt = qi[t], gt = gi[t];
    Span rows;
    rows.pmin = s.first + (int)fastdiv((uint32_t)r0, A.group);
    rows.pmax = s.first + (int)fastdiv((uint32_t)min(r0 + kTile - 1, A.M - 1), A.group);
    rows.dmin = gt.dmin;
    rows.dmax = gt.dmax;
    rows.same = gt.same;
    if (j0 >= a.Tk || !any_seen(s, rows, mine, j0)) continue;
    const _Float16* L = lds + buf * NF * kFrag;
    const float* info = (const float*)(L + F_INFO * kFrag);
    const bool odd = qt.irregular || gt.irregular;
    const int left = A.M - r0;
    // register r: row r0 + 8 (r / 4) + 4 h + r % 4
    f32x16 x, y;
    float unit, yunit;
    if (odd) {
      plain_scores(x, [&](int i) { return qmap.row(r0 + i); }, left, krow, valid, a.D);
      plain_scores(y, [&](int i) { return gmap.row(r0 + i); }, left, vrow, valid, a.Dv);
      unit = a.scale;
      yunit = 1;
    } else {
      x = scores<KC>(L, 0, kh, kl);
      y = scores<KC>(L, F_GR, vh, vl);
      unit = a.scale * pow2(-ke) * (1.0f / qt.scale);
      yunit = pow2(-ve) * (1.0f / gt.scale);
    }
    f32x16 slack;                  // 1 - tanh^2
    if (RICH) {
      if (a.cap > 0) {
        const float u = unit / a.cap, c = a.cap * kLog2e;
#pragma unroll
        for (int q = 0; q < 16; ++q) {
          const float th = tanh_of(x[q] * u);
          slack[q] = fmaf(-th, th, 1.0f);
          x[q] = c * th;
        }
      } else {
#pragma unroll
        for (int q = 0; q < 16; ++q) {
          x[q] *= unit * kLog2e;
          slack[q] = 1;
        }
      }
    }
    const float f = RICH ? 1.0f : unit * kLog2e;
    const bool all = left >= kTile && all_seen(s, rows, mine, j0);
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      const int at = 8 * q4 + 4 * h;
      const f32x4 lse = *(const f32x4*)(info + RI_LSE * kTile + at), dot = *(const f32x4*)(info + RI_DOT * kTile + at);
      f32x4 pos, slope, below, rdoc;
      if (RICH && a.slopes) {
        pos = *(const f32x4*)(info + RI_POS * kTile + at);
        slope = *(const f32x4*)(info + RI_SLOPE * kTile + at);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * q4 + e] -= slope[e] * fabsf((float)(__float_as_int(pos[e]) - j));
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int q = 4 * q4 + e;
        const float p = __builtin_amdgcn_exp2f(fmaf(x[q], f, -lse[e]));
        float ds = p * fmaf(y[q], yunit, -dot[e]);
        if (RICH) ds *= slack[q];
        x[q] = p;
        y[q] = ds;
      }
      if (!all) {
        below = *(const f32x4*)(info + RI_BELOW * kTile + at);
        rdoc = *(const f32x4*)(info + RI_DOC * kTile + at);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool ok = j < __float_as_int(below[e]) && (!s.doc || (doc >= 0 && __float_as_int(rdoc[e]) == doc));
          x[4 * q4 + e] = ok ? x[4 * q4 + e] : 0.0f;
          y[4 * q4 + e] = ok ? y[4 * q4 + e] : 0.0f;
        }
      }
    }
    if (odd) {
      plain_accumulate<DB>(dv, cv, x, [&](int i) { return gmap.row(r0 + i); }, left, a.Dv);
      plain_accumulate<DB>(dk, ck, y, [&](int i) { return qmap.row(r0 + i); }, left, a.D);
      continue;
    }
    float change = 1;
    int e = fit_unit(cv, largest(x), exponent(gt.scale), &change);
    rescale<DB>(dv, change);
    accumulate<DB>(dv, x, pow2(e), L, F_GC);
    change = 1;
    e = fit_unit(ck, largest(y), exponent(qt.scale), &change);
    rescale<DB>(dk, change);
    accumulate<DB>(dk, y, pow2(e), L, F_QC);
  }

  if (!valid) return;
  const bool parts = A.splits > 1;
  const int64_t at = ((int64_t)split * a.B * a.Hk + slab) * a.Tk + j;
  if (A.g.dk.p) {
    float* o = parts ? A.pk + at * a.D : A.g.dk.p + b * A.g.dk.b + hk * A.g.dk.h + (int64_t)j * A.g.dk.t;
    store_row<DB>(o, dk, ck, a.scale, a.D, parts ? a.D % 4 == 0 : A.wide);
  }
  if (A.g.dv.p) {
    float* o = parts ? A.pv + at * a.Dv : A.g.dv.p + b * A.g.dv.b + hk * A.g.dv.h + (int64_t)j * A.g.dv.t;
    store_row<DB>(o, dv, cv, 1.0f, a.Dv, parts ? a.Dv % 4 == 0 : A.wide);
  }
}

// The parts of dk and dv in order.
__global__ __launch_bounds__(256) void attend_grad_join(GradArgs A) {
  const AttendDesc& a = A.g.a;
  const bool v = blockIdx.y;
  const int n = v ? a.Dv : a.D;
  const Rows& o = v ? A.g.dv : A.g.dk;
  const float* part = v ? A.pv : A.pk;
  if (!o.p) return;
  const int64_t all = (int64_t)a.B * a.Hk * a.Tk * n, at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= all) return;
  float x = 0;
  for (int z = 0; z < A.splits; ++z) x += part[at + z * all];
  const int64_t row = at / n;
  const int d = (int)(at - row * n), j = (int)(row % a.Tk), slab = (int)(row / a.Tk);
  o.p[slab / a.Hk * o.b + slab % a.Hk * o.h + (int64_t)j * o.t + d] = x;
}

// ---- dq --------------------------------------------------------------------------------------------

template <int DP, bool RICH>
__global__ __launch_bounds__(256, DP <= 64 ? 2 : 1) void attend_grad_q(GradArgs A) {
  constexpr int KC = DP / 16, DB = DP / 32;
  constexpr int F_V = 2 * KC, F_KC = 4 * KC, NF = F_KC + 4 * DB;
  __shared__ __align__(16) _Float16 lds[2 * NF * kFrag];
  const AttendDesc& a = A.g.a;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, l = lane & 31;
  const uint32_t id = xcd_order(blockIdx.x, gridDim.x);
  const int rblocks = (A.M + 127) / 128;
  const int slab = id / rblocks, blk = rblocks - 1 - (int)(id % rblocks);
  const int b = slab / a.Hk, hk = slab % a.Hk, G = (int)A.group.d;
  const Sight s = sight(a, b);
  const int row0 = blk * 128 + w * kTile, r = row0 + l, rr = min(r, A.M - 1);
  const bool valid = r < A.M;
  const int i = (int)fastdiv((uint32_t)rr, A.group), g = rr - i * G, head = hk * G + g;
  const int p = s.first + i, doc = doc_at(s, p), below = sees_below(s, p);
  const float* qrow = a.q.p + b * a.q.b + head * a.q.h + (int64_t)i * a.q.t;
  const float* grow = A.g.dy.p + b * A.g.dy.b + head * A.g.dy.h + (int64_t)i * A.g.dy.t;
  half8 qh[KC], ql[KC], gh[KC], gl[KC];
  const int qe = load_rows<KC>(qrow, valid, a.D, A.wide, qh, ql);
  const int ge = load_rows<KC>(grow, valid, a.Dv, A.wide, gh, gl);
  const float slope = RICH && a.slopes ? a.slopes[head] * kLog2e : 0.0f;
  const int qt = min(row0 / kTile, A.qtiles - 1);
  const float* info = A.rowinfo + ((int64_t)slab * A.qtiles + qt) * (kRowInfo * kTile) + l;
  const float lse = info[RI_LSE * kTile], dot = info[RI_DOT * kTile];
  const TileInfo mine = A.gi[(int64_t)slab * A.qtiles + qt];
  Span me;
  me.pmin = s.first + (int)fastdiv((uint32_t)min(row0, A.M - 1), A.group);
  me.pmax = s.first + (int)fastdiv((uint32_t)min(row0 + kTile - 1, A.M - 1), A.group);
  me.dmin = mine.dmin;
  me.dmax = mine.dmax;
  me.same = mine.same;

  const TileInfo* ki = A.ki + (int64_t)slab * A.ktiles;
  const TileInfo* vi = A.vi + (int64_t)slab * A.ktiles;
  const int last = s.first + (int)fastdiv((uint32_t)min(blk * 128 + 127, A.M - 1), A.group);
  int t0 = 0, t1 = s.n;
  if (s.causal) t1 = min(t1, max(last + 1, s.prefix));
  if (s.positional && last < 0) t1 = 0;
  t1 = (t1 + kTile - 1) / kTile;
  if (s.doc) {
    __shared__ int range[4];
    if (tid < 4) range[tid] = tid & 1 ? INT32_MIN : INT32_MAX;
    __syncthreads();
    if (lane == 0 && row0 < A.M) {
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
  t0 = __builtin_amdgcn_readfirstlane(t0);
  t1 = __builtin_amdgcn_readfirstlane(t1);

  const int64_t tile0 = (int64_t)slab * A.ktiles;
  const uint32_t base = lds_address(lds), lane16 = lane * 16;
  auto fetch = [&](int t, int buf) {
#pragma unroll
    for (int f = 0; f < NF / 4; ++f) {
      const int q = f * 4 + w;
      const _Float16* src;
      if (q < F_V) src = A.kr + ((tile0 + t) * (2 * KC) + q) * kFrag;
      else if (q < F_KC) src = A.vr + ((tile0 + t) * (2 * KC) + q - F_V) * kFrag;
      else src = A.kc + ((tile0 + t) * (4 * DB) + q - F_KC) * kFrag;
      frag_to_lds(src, base + (buf * NF + q) * (kFrag * 2), lane16);
    }
  };

  f32x16 dq[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) dq[d] = f32x16{};
  int cq = kUnset;
  if (t0 < t1) fetch(t0, 0);
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1, j0 = t * kTile;
    loads_done();
    __syncthreads();
    if (t + 1 < t1) fetch(t + 1, buf ^ 1);
    const TileInfo kt = ki[t], vt = vi[t];
    if (!any_seen(s, me, kt, j0)) continue;
    const _Float16* L = lds + buf * NF * kFrag;
    const bool odd = kt.irregular || vt.irregular;
    const float* k = a.k.p + b * a.k.b + hk * a.k.h + (int64_t)j0 * a.k.t;
    const float* v = a.v.p + b * a.v.b + hk * a.v.h + (int64_t)j0 * a.v.t;
    f32x16 x, y;
    float unit, yunit;
    if (odd) {
      plain_scores(x, [&](int j) { return k + j * a.k.t; }, a.Tk - j0, qrow, valid, a.D);
      plain_scores(y, [&](int j) { return v + j * a.v.t; }, a.Tk - j0, grow, valid, a.Dv);
      unit = a.scale;
      yunit = 1;
    } else {
      x = scores<KC>(L, 0, qh, ql);
      y = scores<KC>(L, F_V, gh, gl);
      unit = a.scale * pow2(-qe) * (1.0f / kt.scale);
      yunit = pow2(-ge) * (1.0f / vt.scale);
    }
    const bool all = all_seen(s, me, kt, j0);
    const float u = RICH && a.cap > 0 ? unit / a.cap : unit * kLog2e, c = a.cap * kLog2e;
#pragma unroll
    for (int q = 0; q < 16; ++q) {
      const int j = j0 + 8 * (q / 4) + 4 * h + q % 4;
      float z = x[q] * u, slack = 1;
      if (RICH && a.cap > 0) {
        z = tanh_of(z);
        slack = fmaf(-z, z, 1.0f);
        z *= c;
      }
      if (RICH && a.slopes) z -= slope * fabsf((float)(p - j));
      const float w = __builtin_amdgcn_exp2f(RICH ? z - lse : fmaf(x[q], u, -lse));
      y[q] = w * fmaf(y[q], yunit, -dot);
      if (RICH) y[q] *= slack;
    }
    if (!all) {
      if (s.doc) {
        int dj[16];
#pragma unroll
        for (int q = 0; q < 16; ++q) dj[q] = s.doc[min(j0 + 8 * (q / 4) + 4 * h + q % 4, a.Tk - 1)];
#pragma unroll
        for (int q = 0; q < 16; ++q) y[q] = dj[q] == doc && doc >= 0 ? y[q] : 0.0f;
      }
#pragma unroll
      for (int q = 0; q < 16; ++q) y[q] = j0 + 8 * (q / 4) + 4 * h + q % 4 < below ? y[q] : 0.0f;
    }
    if (odd) {
      plain_accumulate<DB>(dq, cq, y, [&](int j) { return k + j * a.k.t; }, a.Tk - j0, a.D);
      continue;
    }
    float change = 1;
    const int e = fit_unit(cq, largest(y), exponent(kt.scale), &change);
    rescale<DB>(dq, change);
    accumulate<DB>(dq, y, pow2(e), L, F_KC);
  }
  if (valid)
    store_row<DB>(A.g.dq.p + b * A.g.dq.b + head * A.g.dq.h + (int64_t)i * A.g.dq.t, dq, cq, a.scale, a.D, A.wide);
}

// ---- plan --------------------------------------------------------------------------------------------

struct GradPlan {
  int DP, M, G, qtiles, ktiles, blocks, splits, slabs;
  int64_t qr, qc, gr, gc, kr, kc, vr, qi, gi, ki, vi, rowinfo, pk, pv, bytes;
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
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(512 / have, p.qtiles / 8));
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
  p.rowinfo = take(q * kRowInfo * kTile * 4);
  if (p.splits > 1) {
    p.pk = take((int64_t)p.splits * p.slabs * a.Tk * a.D * 4);
    p.pv = take((int64_t)p.splits * p.slabs * a.Tk * a.Dv * 4);
  }
  p.bytes = at;
  return p;
}

template <int DP, bool RICH>
void run_grad(const GradArgs& A, int slabs, hipStream_t st) {
  const AttendGradDesc& g = A.g;
  if (g.dk.p || g.dv.p)
    klaunch(attend_grad_kv<DP, RICH>, dim3((unsigned)(slabs * A.blocks * A.splits)), dim3(256), 0, st, A);
  if (g.dq.p)
    klaunch(attend_grad_q<DP, RICH>, dim3((unsigned)(slabs * ((A.M + 127) / 128))), dim3(256), 0, st, A);
}
template <int DP>
void run_grad(const GradArgs& A, int slabs, hipStream_t st) {
  if (A.g.a.cap > 0 || A.g.a.slopes) run_grad<DP, true>(A, slabs, st);
  else run_grad<DP, false>(A, slabs, st);
}

}  // namespace

int64_t attend_grad_workspace_bytes(const AttendGradDesc& g) { return grad_plan(g).bytes; }

void attend_grad(const AttendGradDesc& g, void* work, hipStream_t st) {
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
  k.job[0] = {a.q, a.D, p.G, p.M, p.qtiles, half(p.qr), half(p.qc), info(p.qi), true, {}, nullptr};
  k.job[1] = {g.dy, a.Dv, p.G, p.M, p.qtiles, half(p.gr), half(p.gc), info(p.gi), true, a.y, (float*)(w + p.rowinfo)};
  k.job[2] = {a.k, a.D, 1, a.Tk, p.ktiles, half(p.kr), half(p.kc), info(p.ki), false, {}, nullptr};
  k.job[3] = {a.v, a.Dv, 1, a.Tk, p.ktiles, half(p.vr), nullptr, info(p.vi), false, {}, nullptr};
  attend_pack(k, p.DP, st);
  const GradArgs A{g, half(p.qr), half(p.qc), half(p.gr), half(p.gc), half(p.kr), half(p.kc), half(p.vr),
                   info(p.qi), info(p.gi), info(p.ki), info(p.vi), (const float*)(w + p.rowinfo), make_fastdiv(p.G), p.M, p.qtiles,
                   p.ktiles, p.blocks, p.splits, wide, (float*)(w + p.pk), (float*)(w + p.pv)};
  if (p.DP == 32) run_grad<32>(A, p.slabs, st);
  else if (p.DP == 64) run_grad<64>(A, p.slabs, st);
  else if (p.DP == 96) run_grad<96>(A, p.slabs, st);
  else run_grad<128>(A, p.slabs, st);
  if (p.splits > 1 && (g.dk.p || g.dv.p)) {
    const int64_t most = (int64_t)a.B * a.Hk * a.Tk * std::max(a.D, a.Dv);
    klaunch(attend_grad_join, dim3((unsigned)((most + 255) / 256), 2), dim3(256), 0, st, A);
  }
}

}  // namespace tgk
