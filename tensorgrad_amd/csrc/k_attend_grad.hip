// Gradients of masked attention for gfx950: a block per row, plain f32.
#include "attend_dev.h"

namespace tgk {
namespace {

constexpr int kThreads = 256;

// x / cap's tanh t and the score.
__device__ __forceinline__ float score(const AttendDesc& a, const Sight& s, int h, int i, int j, float dot, float& t) {
  float x = a.scale * dot;
  t = 0;
  if (a.cap > 0) {
    t = tanhf(x / a.cap);
    x = a.cap * t;
  }
  if (a.slopes) x -= a.slopes[h] * fabsf((float)(s.first + i - j));
  return x;
}

__device__ __forceinline__ float dot(const float* x, const float* y, int n) {
  float s = 0;
  for (int d = 0; d < n; ++d) s = fmaf(x[d], y[d], s);
  return s;
}

// p and ds of one pair.
__device__ __forceinline__ bool pair(const AttendGradDesc& g, const Sight& s, int b, int h, int hk, int i, int j, float& p, float& ds) {
  const AttendDesc& a = g.a;
  p = ds = 0;
  if (!sees(s, s.first + i, doc_at(s, s.first + i), j)) return false;
  const float* q = a.q.p + b * a.q.b + h * a.q.h + i * a.q.t;
  const float* y = a.y.p + b * a.y.b + h * a.y.h + i * a.y.t;
  const float* dy = g.dy.p + b * g.dy.b + h * g.dy.h + i * g.dy.t;
  const float* k = a.k.p + b * a.k.b + hk * a.k.h + j * a.k.t;
  const float* v = a.v.p + b * a.v.b + hk * a.v.h + j * a.v.t;
  float t;
  const float x = score(a, s, h, i, j, dot(q, k, a.D), t);
  p = exp2f(x * kLog2e - a.lse[((int64_t)b * a.H + h) * a.Tq + i]);
  ds = p * (dot(dy, v, a.Dv) - dot(dy, y, a.Dv)) * (1 - t * t) * a.scale;
  return true;
}

__global__ __launch_bounds__(kThreads) void attend_grad_q(AttendGradDesc g) {
  __shared__ float pd[kThreads];
  const AttendDesc& a = g.a;
  const int i = blockIdx.x, h = blockIdx.y, b = blockIdx.z, hk = h / (a.H / a.Hk), tid = threadIdx.x;
  const Sight s = sight(a, b);
  const float* k = a.k.p + b * a.k.b + hk * a.k.h;
  float acc = 0;
  for (int j0 = 0; j0 < a.Tk; j0 += kThreads) {
    float p, ds = 0;
    const bool on = j0 + tid < a.Tk && pair(g, s, b, h, hk, i, j0 + tid, p, ds);
    __syncthreads();
    pd[tid] = on ? ds : 0;
    __syncthreads();
    if (tid < a.D)
      for (int jj = 0; jj < kThreads && j0 + jj < a.Tk; ++jj)
        if (pd[jj] != 0) acc = fmaf(pd[jj], k[(j0 + jj) * a.k.t + tid], acc);
  }
  if (tid < a.D) g.dq.p[b * g.dq.b + h * g.dq.h + i * g.dq.t + tid] = acc;
}

__global__ __launch_bounds__(kThreads) void attend_grad_kv(AttendGradDesc g) {
  __shared__ float pp[kThreads], pd[kThreads];
  const AttendDesc& a = g.a;
  const int j = blockIdx.x, hk = blockIdx.y, b = blockIdx.z, group = a.H / a.Hk, tid = threadIdx.x;
  const Sight s = sight(a, b);
  float ak = 0, av = 0;
  for (int h = hk * group; h < (hk + 1) * group; ++h) {
    const float* q = a.q.p + b * a.q.b + h * a.q.h;
    const float* dy = g.dy.p + b * g.dy.b + h * g.dy.h;
    for (int i0 = 0; i0 < a.Tq; i0 += kThreads) {
      float p = 0, ds = 0;
      if (i0 + tid < a.Tq) pair(g, s, b, h, hk, i0 + tid, j, p, ds);
      __syncthreads();
      pp[tid] = p;
      pd[tid] = ds;
      __syncthreads();
      for (int ii = 0; ii < kThreads && i0 + ii < a.Tq; ++ii) {
        if (pd[ii] != 0 && tid < a.D) ak = fmaf(pd[ii], q[(i0 + ii) * a.q.t + tid], ak);
        if (pp[ii] != 0 && tid < a.Dv) av = fmaf(pp[ii], dy[(i0 + ii) * g.dy.t + tid], av);
      }
    }
  }
  if (g.dk.p && tid < a.D) g.dk.p[b * g.dk.b + hk * g.dk.h + j * g.dk.t + tid] = ak;
  if (g.dv.p && tid < a.Dv) g.dv.p[b * g.dv.b + hk * g.dv.h + j * g.dv.t + tid] = av;
}

}  // namespace

int64_t attend_grad_workspace_bytes(const AttendGradDesc&) { return 0; }

void attend_grad(const AttendGradDesc& g, void*, hipStream_t st) {
  const AttendDesc& a = g.a;
  if (g.dq.p) klaunch(attend_grad_q, dim3(a.Tq, a.H, a.B), dim3(kThreads), 0, st, g);
  if (g.dk.p || g.dv.p) klaunch(attend_grad_kv, dim3(a.Tk, a.Hk, a.B), dim3(kThreads), 0, st, g);
}

}  // namespace tgk
