// Linear attention with a decay for each head for gfx950. Positions are cut into segments of kSeg. Within one, results are sums
// over pairs of positions; what comes in from the positions before is one product with the state at the segment's border:
//
//   S[t] = r_t lam S[t-1] + k_t v_t^T                         (r_t: 0 where a document begins)
//   y_i  = scale (sum_{j <= i} w_ij (q_i.k_j) v_j + c_i S_in^T q_i),                  w_ij = lam^(i-j) in one document, else 0
//   dq_i = scale (sum_{j <= i} w_ij (dy_i.v_j) k_j + c_i S_in dy_i),                  c_i = lam^(i-s0+1) where S_in still counts
//   dk_j = sum_{i >= j} scale w_ij (v_j.dy_i) q_i + e_j G_out v_j,                    e_j = lam^(last-j) where j still counts
//   dv_j = sum_{i >= j} scale w_ij (k_j.q_i) dy_i + e_j G_out^T k_j
//   S_out = f S_in + sum_j e_j k_j v_j^T,    G_in = f G_out + sum_i scale c_i q_i dy_i^T,    f = lam^(rows of the segment) or 0
//
// G: the gradient of the state. All four results have one form, out_r = sum_s w (row_r.X_s) Z_s + coef_r M row_r, and both
// states another, so there are three kernels: sums over a segment (linear_sums), states from sums (linear_join), results from
// pairs and states (linear_pairs). Nothing is added by atomics.
#include <algorithm>

#include "kernels.h"
#include "sequence.h"

namespace tgk {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kSeg = 256;          // positions of a segment
constexpr int kRows = 64;          // rows of a block
constexpr int kTile = 32;          // rows of a tile in LDS
constexpr int kNever = INT32_MAX;

__device__ __forceinline__ f32x4 mfma(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
__device__ __forceinline__ float power(float rate, int n) { return __builtin_amdgcn_exp2f(rate * (float)n); }

// What the positions of one batch entry are, and those of one segment.
struct Marks {
  const int32_t *documents, *lengths;
  int T;
};
__device__ __forceinline__ int count_of(const Marks& m, int b) { return m.lengths ? min(max(m.lengths[b], 0), m.T) : m.T; }

// since[t - s0] for the positions of the segment at s0: the first one, in the segment, of the document they belong to; -1 where
// that began before (or the state that came in counts); kNever for positions that are not there. By 256 threads; ends at a barrier.
__device__ __forceinline__ void mark(const Marks& m, int b, int s0, int n, int* since, int* waves) {
  const int tid = threadIdx.x, t = s0 + tid, lane = tid & 63, w = tid >> 6;
  if (!m.documents) {
    if (tid < kSeg) since[tid] = t < n ? -1 : kNever;
    __syncthreads();
    return;
  }
  const int32_t* doc = m.documents + (int64_t)b * m.T;
  const bool here = tid < kSeg && t < n;
  const int id = here ? doc[t] : -1;
  int first = here && t > 0 && doc[t - 1] != id ? t : -1;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const int z = __shfl_up(first, o);
    if (lane >= o) first = max(first, z);
  }
  if (lane == 63) waves[w] = first;
  __syncthreads();
  for (int k = 0; k < w; ++k) first = max(first, waves[k]);
  if (tid < kSeg) since[tid] = here && id >= 0 ? first : kNever;
  __syncthreads();
}
// The segment's last position that is there; what a position leaves of itself there, and of what came in.
struct Ends {
  int last, since;                 // last < s0: none
};
__device__ __forceinline__ Ends ends(const int* since, int s0, int n) {
  const int last = min(s0 + kSeg, n) - 1;
  return {last, last >= s0 ? since[last - s0] : kNever};
}
__device__ __forceinline__ float leaves(const Ends& e, const int* since, int s0, int j, float rate) {
  return j <= e.last && since[j - s0] != kNever && j >= e.since ? power(rate, e.last - j) : 0.0f;
}
__device__ __forceinline__ float comes(const int* since, int s0, int i, float rate) {
  return since[i - s0] == -1 ? power(rate, i - s0 + 1) : 0.0f;
}
__device__ __forceinline__ float stays(const Ends& e, int s0, float rate) {
  return e.last < s0 ? 1.0f : e.since == -1 ? power(rate, e.last - s0 + 1) : 0.0f;
}

// Rows [r0, r0 + 32) of x as a tile of LD floats a row, zero where keep(t) says that a row does not count and past its n
// features. Returns whether this thread met infinities or NaN.
template <int DP, class Keep>
__device__ __forceinline__ bool stage(float* tile, const float* x, int64_t stride, int r0, int T, int n, bool wide, Keep keep) {
  constexpr int LD = DP + 4, Q = DP / 4;
  bool odd = false;
  for (int e = threadIdx.x; e < kTile * Q; e += 256) {
    const int r = e / Q, d = e % Q * 4, t = r0 + r;
    f32x4 u = {};
    if (t < T && keep(t)) {
      const float* p = x + (int64_t)t * stride + d;
      if (wide) {
        if (d < n) u = *(const f32x4*)p;
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) if (d + q < n) u[q] = p[q];
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) odd |= !(fabsf(u[q]) < INFINITY);
    *(f32x4*)(tile + r * LD + d) = u;
  }
  return odd;
}

// ---- sums over a segment -----------------------------------------------------------------------------

struct SumsArgs {
  Marks m;
  Rows x, y;                       // x: k or q, y: v or dy
  int H, share, segs, n, ny;       // query heads, those that share a row of x and y (1: none); features
  bool back, wide;                 // back: of q and dy, weights c, else of k and v, weights e
  float scale;
  const float* rate;
  float *sums, *stay;              // [segs][B * H][n][ny], [segs][B * H]
};
template <int DP>
__global__ __launch_bounds__(256) void linear_sums(SumsArgs A) {
  constexpr int LD = DP + 4, NB = DP / 16, PER = NB * NB / 4;
  __shared__ __align__(16) float xs[kTile * LD], ys[kTile * LD];
  __shared__ int since[kSeg], waves[4];
  __shared__ float weight[kSeg];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 4, l = lane & 15;
  const int seg = blockIdx.x % A.segs, bh = blockIdx.x / A.segs, b = bh / A.H, h = bh % A.H, s0 = seg * kSeg;
  const int n = count_of(A.m, b);
  mark(A.m, b, s0, n, since, waves);
  const Ends e = ends(since, s0, n);
  const float rate = A.rate[h];
  weight[tid] = s0 + tid > e.last ? 0.0f : A.back ? A.scale * comes(since, s0, s0 + tid, rate) : leaves(e, since, s0, s0 + tid, rate);
  const float* x = A.x.p + b * A.x.b + (h / A.share) * A.x.h;
  const float* y = A.y.p + b * A.y.b + (h / A.share) * A.y.h;
  auto counts = [&](int t) { return weight[t - s0] != 0; };
  f32x4 acc[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) acc[i] = f32x4{};
  const int stop = A.y.p ? e.last : s0 - 1;
  for (int t0 = s0; t0 <= stop; t0 += kTile) {
    __syncthreads();
    stage<DP>(xs, x, A.x.t, t0, A.m.T, A.n, A.wide, counts);
    stage<DP>(ys, y, A.y.t, t0, A.m.T, A.ny, A.wide, counts);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kTile; k += 4) {       // positions t0 + k + g
      const float c = weight[t0 - s0 + k + g];
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int id = w * PER + i, dx = id / NB, dy = id % NB;
        acc[i] = mfma(xs[(k + g) * LD + 16 * dx + l] * c, ys[(k + g) * LD + 16 * dy + l], acc[i]);
      }
    }
  }
  const int64_t at = (int64_t)seg * (gridDim.x / A.segs) + bh;
  float* out = A.sums + at * A.n * A.ny;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int id = w * PER + i, d = 16 * (id / NB) + 4 * g, c = 16 * (id % NB) + l;
#pragma unroll
    for (int q = 0; q < 4; ++q) if (d + q < A.n && c < A.ny) out[(d + q) * A.ny + c] = acc[i][q];
  }
  if (tid == 0) A.stay[at] = stays(e, s0, rate);
}

// ---- states at the segments' borders -------------------------------------------------------------------

struct JoinArgs {
  float* sums;                     // [segs][rows][each]: replaced by the state that comes in (back: goes out)
  const float *stay, *first;       // first: [rows][each] or null
  float* last;                     // or null
  int segs;
  int64_t rows, each;
  bool back;
};
__global__ __launch_bounds__(256) void linear_join(JoinArgs A) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, all = A.rows * A.each;
  if (id >= all) return;
  const int64_t row = id / A.each;
  float s = A.first ? A.first[id] : 0.0f;
#pragma unroll 4
  for (int i = 0; i < A.segs; ++i) {
    const int64_t seg = A.back ? A.segs - 1 - i : i;
    float* at = A.sums + seg * all + id;
    const float add = *at, f = A.stay[seg * A.rows + row];
    *at = s;
    s = f == 0 ? add : fmaf(f, s, add);
  }
  if (A.last) A.last[id] = s;
}

// ---- results from pairs and states -----------------------------------------------------------------------

struct Pairs {
  Rows rows, x, z, out;            // row r with x_s, weights on z_s
  int heads, group, share;         // heads of `rows`; those of x and z that a row meets in turn; rows' heads that share one of x
  int n, nz;                       // features of rows and x; of z and out
  bool back, transposed;           // back: pairs with later positions; transposed: m is [nz][n], else [n][nz]
  const float *m, *edge;           // states [segs][B * H][.], or null; at the first segment (back: last) this one, or null
  float pairs, states;             // factors of both parts
};
struct PairsArgs {
  Marks m;
  int B, H, segs, blocks;
  bool wide;
  const float* rate;
  Pairs p[3];
};
template <int DP>
__global__ __launch_bounds__(256) void linear_pairs(PairsArgs A) {
  constexpr int LD = DP + 4, C = DP / 16;
  __shared__ __align__(16) float xs[kTile * LD], zs[kTile * LD];
  __shared__ int since[kSeg], waves[4];
  const Pairs p = A.p[blockIdx.y];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 4, l = lane & 15;
  const int blk = blockIdx.x % A.blocks, bh = blockIdx.x / A.blocks, b = bh / p.heads, head = bh % p.heads;
  if (b >= A.B) return;
  const int T = A.m.T, r0 = blk * kRows, seg = r0 / kSeg, s0 = seg * kSeg, n = count_of(A.m, b);
  mark(A.m, b, s0, n, since, waves);
  const Ends end = ends(since, s0, n);
  const int r = r0 + 16 * w + l;
  const bool here = p.rows.p && r < T && since[r - s0] != kNever;
  auto there = [&](int t) { return since[t - s0] != kNever; };
  float row[C][4];
  {
    const float* at = p.rows.p + b * p.rows.b + head * p.rows.h + (int64_t)min(r, T - 1) * p.rows.t;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int d = 16 * c + 4 * g;
      f32x4 u = {};
      if (here) {
        if (A.wide) {
          if (d < p.n) u = *(const f32x4*)(at + d);
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q) if (d + q < p.n) u[q] = at[d + q];
        }
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) row[c][q] = u[q];
    }
  }
  f32x4 acc[C];
#pragma unroll
  for (int c = 0; c < C; ++c) acc[c] = f32x4{};
  // x[k][q]: weight of tile row 16 k + 4 g + q on this lane's row. odd: the tile has infinities or NaN, which must not reach the
  // rows whose weight on them is 0.
  auto add = [&](const float (&x)[2][4], bool odd) {
    if (__builtin_expect(odd, 0)) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll 1
          for (int o = 0; o < 4; ++o) {
            const float f = __shfl(x[k][q], 16 * o + l);
            if (f == 0) continue;
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[c][e] = fmaf(f, zs[(16 * k + 4 * o + q) * LD + 16 * c + 4 * g + e], acc[c][e]);
          }
      return;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int c = 0; c < C; ++c) acc[c] = mfma(zs[(16 * k + 4 * g + q) * LD + 16 * c + l], x[k][q], acc[c]);
  };
  for (int gi = 0; gi < p.group; ++gi) {
    const int h = p.back ? head * p.group + gi : head, hx = h / p.share;
    const float rate = A.rate[h];
    const bool border = p.back ? seg == A.segs - 1 : seg == 0;
    const float* m = border ? p.edge : p.m + ((int64_t)seg * A.B * A.H) * p.n * p.nz;
    if (m) {
      m += ((int64_t)b * A.H + h) * p.n * p.nz;
      float coef = 0;
      if (here) coef = p.states * (p.back ? leaves(end, since, s0, r, rate) : comes(since, s0, r, rate));
      for (int e0 = 0; e0 < p.n; e0 += kTile) {
        __syncthreads();
        bool odd = false;
        for (int e = tid; e < kTile * DP; e += 256) {
          const int i = p.transposed ? e % kTile : e / DP, d = p.transposed ? e / kTile : e % DP;
          float u = 0;
          if (e0 + i < p.n && d < p.nz) u = p.transposed ? m[d * p.n + e0 + i] : m[(e0 + i) * p.nz + d];
          odd |= !(fabsf(u) < INFINITY);
          zs[i * LD + d] = u;
        }
        odd = __syncthreads_or(odd);
        float x[2][4];
#pragma unroll
        for (int c = 0; c < C; c += 2) {
          if (16 * c != e0) continue;
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int q = 0; q < 4; ++q) x[k][q] = coef == 0 ? 0.0f : row[c + k][q] * coef;
        }
        add(x, odd);
      }
    }
    const float* px = p.x.p + b * p.x.b + hx * p.x.h;
    const float* pz = p.z.p + b * p.z.b + hx * p.z.h;
    const int from = p.back ? r0 : s0, to = p.x.p && p.z.p ? min(p.back ? s0 + kSeg : r0 + kRows, n) : 0;
    for (int t0 = from; t0 < to; t0 += kTile) {
      __syncthreads();
      stage<DP>(xs, px, p.x.t, t0, T, p.n, A.wide, there);
      const bool odd = __syncthreads_or(stage<DP>(zs, pz, p.z.t, t0, T, p.nz, A.wide, there));
      const int w0 = r0 + 16 * w;
      if (p.back ? t0 + kTile <= w0 : t0 > w0 + 15) continue;
      f32x4 s[2] = {};
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const f32x4 u = *(const f32x4*)(xs + (16 * k + l) * LD + 16 * c + 4 * g);
#pragma unroll
          for (int q = 0; q < 4; ++q) s[k] = mfma(u[q], row[c][q], s[k]);
        }
      float x[2][4];
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int t = t0 + 16 * k + 4 * g + q, i = p.back ? t : r, j = p.back ? r : t;
          const bool seen = here && t < n && j <= i && j >= since[i - s0];
          x[k][q] = seen ? s[k][q] * power(rate, i - j) * p.pairs : 0.0f;
        }
      add(x, odd);
    }
  }
  if (r >= T) return;
  float* out = p.out.p + b * p.out.b + head * p.out.h + (int64_t)r * p.out.t;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int d = 16 * c + 4 * g;
    const f32x4 u = here ? acc[c] : f32x4{};
    if (A.wide) {
      if (d < p.nz) *(f32x4*)(out + d) = u;
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) if (d + q < p.nz) out[d + q] = u[q];
    }
  }
}

// ---- plans -------------------------------------------------------------------------------------------------

inline bool wide_rows(const Rows& x, int n) { return ((uintptr_t)x.p & 15) == 0 && x.b % 4 == 0 && x.h % 4 == 0 && x.t % 4 == 0 && n % 4 == 0; }
inline int segments(const LinearDesc& a) { return (a.T + kSeg - 1) / kSeg; }
inline int padded(const LinearDesc& a) { return (std::max(a.D, a.Dv) + 31) / 32 * 32; }
inline int64_t sums_bytes(const LinearDesc& a) {
  const int64_t n = (int64_t)segments(a) * a.B * a.H;
  return n * a.D * a.Dv * 4 + (n * 4 + 255) / 256 * 256;
}
inline Marks marks(const LinearDesc& a) { return {a.documents, a.lengths, a.T}; }

// States at the borders of all segments (in place of the sums), and the one at the end.
void states(const LinearDesc& a, const Rows& x, const Rows& y, bool back, const float* first, float* last, float* sums, hipStream_t st) {
  SumsArgs s{};
  s.m = marks(a);
  s.x = x;
  s.y = y;
  s.H = a.H;
  s.share = back ? 1 : a.H / a.Hk;
  s.segs = segments(a);
  s.n = a.D;
  s.ny = a.Dv;
  s.back = back;
  s.wide = wide_rows(x, a.D) && wide_rows(y, a.Dv);
  s.scale = a.scale;
  s.rate = a.rate;
  s.sums = sums;
  const int64_t rows = (int64_t)a.B * a.H, each = (int64_t)a.D * a.Dv;
  s.stay = sums + s.segs * rows * each;
  const dim3 grid((unsigned)(rows * s.segs));
  switch (padded(a)) {
    case 32: klaunch(linear_sums<32>, grid, dim3(256), 0, st, s); break;
    case 64: klaunch(linear_sums<64>, grid, dim3(256), 0, st, s); break;
    case 96: klaunch(linear_sums<96>, grid, dim3(256), 0, st, s); break;
    default: klaunch(linear_sums<128>, grid, dim3(256), 0, st, s);
  }
  const JoinArgs j{sums, s.stay, first, last, s.segs, rows, each, back};
  klaunch(linear_join, dim3((unsigned)((rows * each + 255) / 256)), dim3(256), 0, st, j);
}
void pairs(PairsArgs& p, const LinearDesc& a, int jobs, hipStream_t st) {
  p.m = marks(a);
  p.B = a.B;
  p.H = a.H;
  p.segs = segments(a);
  p.blocks = (a.T + kRows - 1) / kRows;
  p.rate = a.rate;
  p.wide = true;
  for (int i = 0; i < jobs; ++i)
    p.wide = p.wide && wide_rows(p.p[i].rows, p.p[i].n) && wide_rows(p.p[i].x, p.p[i].n) && wide_rows(p.p[i].z, p.p[i].nz) &&
             wide_rows(p.p[i].out, p.p[i].nz);
  const dim3 grid((unsigned)((int64_t)p.blocks * a.B * a.H), jobs);
  switch (padded(a)) {
    case 32: klaunch(linear_pairs<32>, grid, dim3(256), 0, st, p); break;
    case 64: klaunch(linear_pairs<64>, grid, dim3(256), 0, st, p); break;
    case 96: klaunch(linear_pairs<96>, grid, dim3(256), 0, st, p); break;
    default: klaunch(linear_pairs<128>, grid, dim3(256), 0, st, p);
  }
}

}  // namespace

int64_t linear_workspace_bytes(const LinearDesc& a) { return sums_bytes(a); }

void linear(const LinearDesc& a, void* work, hipStream_t st) {
  float* sums = (float*)work;
  const int G = a.H / a.Hk;
  if (a.last || (a.y.p && segments(a) > 1)) states(a, a.k, a.v, false, a.state, a.last, sums, st);
  if (!a.y.p) return;
  PairsArgs p{};
  p.p[0] = {a.q, a.k, a.v, a.y, a.H, 1, G, a.D, a.Dv, false, false, sums, a.state, a.scale, a.scale};
  pairs(p, a, 1, st);
}

int64_t linear_grad_workspace_bytes(const LinearGradDesc& g) { return 2 * sums_bytes(g.a); }

void linear_grad(const LinearGradDesc& g, void* work, hipStream_t st) {
  const LinearDesc& a = g.a;
  float *S = (float*)work, *Gs = (float*)((char*)work + sums_bytes(a));
  const bool several = segments(a) > 1;
  const int G = a.H / a.Hk;
  if (g.dq.p && several) states(a, a.k, a.v, false, a.state, nullptr, S, st);
  if (g.dfirst || ((g.dk.p || g.dv.p) && several)) states(a, a.q, g.dy, true, g.dstate, g.dfirst, Gs, st);
  PairsArgs p{};
  int jobs = 0;
  if (g.dq.p) p.p[jobs++] = {g.dy, a.v, a.k, g.dq, a.H, 1, G, a.Dv, a.D, false, true, S, a.state, a.scale, a.scale};
  if (g.dk.p) p.p[jobs++] = {a.v, g.dy, a.q, g.dk, a.Hk, G, 1, a.Dv, a.D, true, true, Gs, g.dstate, a.scale, 1.0f};
  if (g.dv.p) p.p[jobs++] = {a.k, a.q, g.dy, g.dv, a.Hk, G, 1, a.D, a.Dv, true, false, Gs, g.dstate, a.scale, 1.0f};
  if (jobs) pairs(p, a, jobs, st);
}

}  // namespace tgk
