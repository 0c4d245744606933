// Attention over a few dozen positions (sample-sized models), forward and gradients, in plain f32: a block takes a key head
// and its G Tq query rows whole, in LDS, one launch a direction. Bound by launches and by the latency of a block's phases
// (loads, products, softmax): for 256 key heads of 16 positions and head size 16 a training step is 6.4 + 8.3 us of kernels,
// 19 us as called; packing, tiles and the two gradient walks were five launches and 32. 64 positions, head size 32: 39 us
// instead of 49, and the same (38) for 8 key heads, which is where longer ones are left to the tiles.
#include "attend_dev.h"

namespace tgk {
namespace {

// A key head's rows: N of each at most, W features at most, 256 threads as 16 x 16. A thread has the results i = ti + 16 a,
// j = tj + 16 b of a product: LD is odd, so that 16 rows of a column lie in 16 banks.
template <int N, int W>
struct Small {
  static constexpr int LD = W + 1, LP = N + 1, I = N / 16, T = 256 / N;
  static_assert(N % 16 == 0 && W % 16 == 0 && T <= 64);
};

// x[i][d] = row i of n, zero past the end. Loads go out together: past the end they read a value that is there.
template <int N, int W>
struct Loaded {
  float x[N * W / 256];
};
template <int N, int W, class RowOf>
__device__ __forceinline__ Loaded<N, W> load_all(int rows, int n, RowOf row_of) {
  Loaded<N, W> l;
#pragma unroll
  for (int u = 0; u < N * W / 256; ++u) {
    const int e = threadIdx.x + 256 * u;
    l.x[u] = row_of(min(e / W, max(rows, 1) - 1))[min(e % W, n - 1)];
  }
  return l;
}
template <int N, int W>
__device__ __forceinline__ void keep_all(float* x, int rows, int n, const Loaded<N, W>& l) {
#pragma unroll
  for (int u = 0; u < N * W / 256; ++u) {
    const int e = threadIdx.x + 256 * u, i = e / W, d = e % W;
    x[i * (W + 1) + d] = i < rows && d < n ? l.x[u] : 0.0f;
  }
}
// o[a][b] = sum over k < n of fa(ti + 16 a, k) fb(tj + 16 b, k). MASKED: weights of 0 count for nothing, whatever they meet.
template <bool MASKED, int A, int B, class FA, class FB>
__device__ __forceinline__ void product(float (&o)[A][B], int n, FA fa, FB fb) {
  const int ti = threadIdx.x / 16, tj = threadIdx.x % 16;
#pragma unroll
  for (int i = 0; i < A; ++i)
#pragma unroll
    for (int j = 0; j < B; ++j) o[i][j] = 0;
#pragma unroll 4
  for (int k = 0; k < n; ++k) {
    float x[A], y[B];
#pragma unroll
    for (int i = 0; i < A; ++i) x[i] = fa(ti + 16 * i, k);
#pragma unroll
    for (int j = 0; j < B; ++j) y[j] = fb(tj + 16 * j, k);
#pragma unroll
    for (int i = 0; i < A; ++i)
#pragma unroll
      for (int j = 0; j < B; ++j) o[i][j] = MASKED && x[i] == 0 ? o[i][j] : fmaf(x[i], y[j], o[i][j]);
  }
}

// Row r of a slab: its query index, head, position, and what it sees.
struct Row {
  int i, head, p, doc, below;
};
__device__ __forceinline__ Row row_at(const AttendDesc& a, const Sight& s, int hk, int G, int r) {
  Row x;
  x.i = r / G;
  x.head = hk * G + r % G;
  x.p = s.first + x.i;
  x.doc = doc_at(s, x.p);
  x.below = sees_below(s, x.p);
  return x;
}
__device__ __forceinline__ bool sees(const Sight& s, const Row& x, int j) {
  return j < x.below && (!s.doc || (x.doc >= 0 && s.doc[j] == x.doc));
}
__device__ __forceinline__ float* at(const Rows& x, int b, int head, int t) { return x.p + b * x.b + head * x.h + (int64_t)t * x.t; }

template <int N, int W>
__global__ __launch_bounds__(256) void attend_small(AttendDesc a) {
  using Z = Small<N, W>;
  __shared__ float q[N * Z::LD], k[N * Z::LD], v[N * Z::LD], p[N * Z::LP], total[N];
  const int slab = blockIdx.x, b = slab / a.Hk, hk = slab % a.Hk, G = a.H / a.Hk, M = G * a.Tq;
  const int tid = threadIdx.x, ti = tid / 16, tj = tid % 16;
  const Sight s = sight(a, b);
  const auto lq = load_all<N, W>(M, a.D, [&](int r) { return at(a.q, b, hk * G + r % G, r / G); });
  const auto lk = load_all<N, W>(s.n, a.D, [&](int j) { return at(a.k, b, hk, j); });
  const auto lv = load_all<N, W>(s.n, a.Dv, [&](int j) { return at(a.v, b, hk, j); });
  keep_all<N, W>(q, M, a.D, lq);
  keep_all<N, W>(k, s.n, a.D, lk);
  keep_all<N, W>(v, s.n, a.Dv, lv);
  __syncthreads();
  float x[Z::I][Z::I];
  product<false>(x, a.D, [&](int r, int d) { return q[r * Z::LD + d]; }, [&](int j, int d) { return k[j * Z::LD + d]; });
#pragma unroll
  for (int i = 0; i < Z::I; ++i) {
    const int r = ti + 16 * i;
    if (r >= M) break;
    const Row w = row_at(a, s, hk, G, r);
    const float slope = a.slopes ? a.slopes[w.head] * kLog2e : 0.0f;
#pragma unroll
    for (int e = 0; e < Z::I; ++e) p[r * Z::LP + tj + 16 * e] = plain_score(a, x[i][e], slope, w.p - (tj + 16 * e)).score;
  }
  __syncthreads();
  const int r = tid / Z::T, sub = tid % Z::T;      // Z::T threads a row
  if (r < M) {
    const Row w = row_at(a, s, hk, G, r);
    float m = kNone, sum = 0;
    bool any = false;
    for (int j = sub; j < a.Tk; j += Z::T)
      if (sees(s, w, j)) {
        m = fmaxf(m, p[r * Z::LP + j]);
        any = true;
      }
#pragma unroll
    for (int o = 1; o < Z::T; o *= 2) {
      m = fmaxf(m, __shfl_xor(m, o));
      any = __shfl_xor((int)any, o) || any;
    }
    if (m == kNone) m = 0;         // nothing, NaN alone, or minus infinities
    for (int j = sub; j < a.Tk; j += Z::T) {
      const float e = sees(s, w, j) ? __builtin_amdgcn_exp2f(p[r * Z::LP + j] - m) : 0.0f;
      p[r * Z::LP + j] = e;
      sum += e;
    }
#pragma unroll
    for (int o = 1; o < Z::T; o *= 2) sum += __shfl_xor(sum, o);
    if (sub == 0) {
      total[r] = any ? sum : INFINITY;             // a row that sees nothing is 0
      if (a.stats) write_stats(a, ((int64_t)b * a.H + w.head) * a.Tq + w.i, !any, m, sum);
    }
  }
  if (!a.y.p) return;
  __syncthreads();
  float y[Z::I][W / 16];
  product<true>(y, a.Tk, [&](int r, int j) { return p[r * Z::LP + j]; }, [&](int d, int j) { return v[j * Z::LD + d]; });
#pragma unroll
  for (int i = 0; i < Z::I; ++i) {
    const int r = ti + 16 * i;
    if (r >= M) break;
    float* to = at(a.y, b, hk * G + r % G, r / G);
#pragma unroll
    for (int e = 0; e < W / 16; ++e) if (tj + 16 * e < a.Dv) to[tj + 16 * e] = y[i][e] / total[r];
  }
}

template <int N, int W>
__global__ __launch_bounds__(256) void attend_grad_small(AttendGradDesc g) {
  using Z = Small<N, W>;
  const AttendDesc& a = g.a;
  __shared__ float q[N * Z::LD], k[N * Z::LD], v[N * Z::LD], dy[N * Z::LD], p[N * Z::LP], ds[N * Z::LP], dots[N];
  const int slab = blockIdx.x, b = slab / a.Hk, hk = slab % a.Hk, G = a.H / a.Hk, M = G * a.Tq;
  const int tid = threadIdx.x, ti = tid / 16, tj = tid % 16;
  const Sight s = sight(a, b);
  const auto lq = load_all<N, W>(M, a.D, [&](int r) { return at(a.q, b, hk * G + r % G, r / G); });
  const auto lg = load_all<N, W>(M, a.Dv, [&](int r) { return at(g.dy, b, hk * G + r % G, r / G); });
  const auto lk = load_all<N, W>(s.n, a.D, [&](int j) { return at(a.k, b, hk, j); });
  const auto lv = load_all<N, W>(s.n, a.Dv, [&](int j) { return at(a.v, b, hk, j); });
  keep_all<N, W>(q, M, a.D, lq);
  keep_all<N, W>(dy, M, a.Dv, lg);
  keep_all<N, W>(k, s.n, a.D, lk);
  keep_all<N, W>(v, s.n, a.Dv, lv);
  __syncthreads();
  {
    const int r = tid / Z::T, sub = tid % Z::T;
    float dot = 0;
    if (r < M) {
      const float* y = at(a.y, b, hk * G + r % G, r / G);
      for (int d = sub; d < a.Dv; d += Z::T) dot = fmaf(dy[r * Z::LD + d], y[d], dot);
    }
#pragma unroll
    for (int o = 1; o < Z::T; o *= 2) dot += __shfl_xor(dot, o);
    if (sub == 0) dots[r] = dot;
  }
  __syncthreads();
  float x[Z::I][Z::I], z[Z::I][Z::I];
  product<false>(x, a.D, [&](int r, int d) { return q[r * Z::LD + d]; }, [&](int j, int d) { return k[j * Z::LD + d]; });
  product<false>(z, a.Dv, [&](int r, int d) { return dy[r * Z::LD + d]; }, [&](int j, int d) { return v[j * Z::LD + d]; });
#pragma unroll
  for (int i = 0; i < Z::I; ++i) {
    const int r = ti + 16 * i;
    if (r >= M) break;
    const Row w = row_at(a, s, hk, G, r);
    const float slope = a.slopes ? a.slopes[w.head] * kLog2e : 0.0f;
    const float* stats = a.stats + 2 * (((int64_t)b * a.H + w.head) * a.Tq + w.i);
    const float top = stats[0], share = stats[1];
#pragma unroll
    for (int e = 0; e < Z::I; ++e) {
      const int j = tj + 16 * e;
      const PlainPair c = plain_score(a, x[i][e], slope, w.p - j);
      const bool shown = sees(s, w, j);
      const float weight = shown ? __builtin_amdgcn_exp2f(c.score - top) * share : 0.0f;
      p[r * Z::LP + j] = weight;
      ds[r * Z::LP + j] = shown ? weight * (z[i][e] - dots[r]) * c.slack : 0.0f;
    }
  }
  __syncthreads();
  float o[Z::I][W / 16];
  if (g.dq.p) {
    product<true>(o, a.Tk, [&](int r, int j) { return ds[r * Z::LP + j]; }, [&](int d, int j) { return k[j * Z::LD + d]; });
#pragma unroll
    for (int i = 0; i < Z::I; ++i) {
      const int r = ti + 16 * i;
      if (r >= M) break;
      float* to = at(g.dq, b, hk * G + r % G, r / G);
#pragma unroll
      for (int e = 0; e < W / 16; ++e) if (tj + 16 * e < a.D) to[tj + 16 * e] = o[i][e] * a.scale;
    }
  }
  auto keys = [&](const Rows& out, const float* weights, const float* rows, int n, float scale) {
    product<true>(o, M, [&](int j, int r) { return weights[r * Z::LP + j]; }, [&](int d, int r) { return rows[r * Z::LD + d]; });
#pragma unroll
    for (int i = 0; i < Z::I; ++i) {
      const int j = ti + 16 * i;
      if (j >= a.Tk) break;
      float* to = at(out, b, hk, j);
#pragma unroll
      for (int e = 0; e < W / 16; ++e) if (tj + 16 * e < n) to[tj + 16 * e] = o[i][e] * scale;
    }
  };
  if (g.dk.p) keys(g.dk, ds, q, a.D, a.scale);
  if (g.dv.p) keys(g.dv, p, dy, a.Dv, 1.0f);
}

template <int N, int W>
void run(const AttendDesc& a, hipStream_t st) { klaunch(attend_small<N, W>, dim3(a.B * a.Hk), dim3(256), 0, st, a); }
template <int N, int W>
void run(const AttendGradDesc& g, hipStream_t st) { klaunch(attend_grad_small<N, W>, dim3(g.a.B * g.a.Hk), dim3(256), 0, st, g); }
template <class Desc>
void run(const Desc& d, const AttendDesc& a, hipStream_t st) {
  if (attend_small_rows(a) == 64) run<64, 32>(d, st);
  else if (attend_dp(a) == 32) run<32, 32>(d, st);
  else run<32, 64>(d, st);
}

}  // namespace

void attend_small_forward(const AttendDesc& a, hipStream_t st) { run(a, a, st); }
void attend_small_grad(const AttendGradDesc& g, hipStream_t st) { run(g, g.a, st); }

}  // namespace tgk
