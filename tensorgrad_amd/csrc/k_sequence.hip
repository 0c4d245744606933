// Rotary positions of several axes and the gated linear recurrence for gfx950.
#include "kernels.h"
#include "sequence.h"

namespace tgk {
namespace {

// A thread turns one pair of one row (b, t) in every head of every tensor.
__global__ __launch_bounds__(256) void rope_pairs(RopeDesc r) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int units = r.D - r.half;            // pairs, then features that pass
  if (id >= (int64_t)r.B * r.T * units) return;
  const int u = (int)(id % units);
  const int t = (int)(id / units % r.T), b = (int)(id / units / r.T);
  float c = 1, s = 0;
  const bool turn = u < r.half;
  if (turn) {
    const RopePair p = r.pairs[u];
    double sd, cd;
    sincos((double)r.positions[((int64_t)p.axis * r.B + b) * r.T + t] * p.freq, &sd, &cd);
    c = (float)cd;
    s = (float)sd;
  }
  for (int i = 0; i < r.n; ++i) {
    const float sg = r.inverse[i] ? -s : s;
    for (int h = 0; h < r.heads[i]; ++h) {
      const float* x = r.x[i].p + b * r.x[i].b + h * r.x[i].h + t * r.x[i].t;
      float* y = r.y[i].p + b * r.y[i].b + h * r.y[i].h + t * r.y[i].t;
      if (turn) {
        const float x1 = x[u], x2 = x[u + r.half];
        y[u] = x1 * c - x2 * sg;
        y[u + r.half] = x2 * c + x1 * sg;
      } else {
        y[u + r.half] = x[u + r.half];
      }
    }
  }
}

__global__ __launch_bounds__(64) void scan_channels(ScanDesc s) {
  const int64_t c = (int64_t)blockIdx.x * 64 + threadIdx.x, b = blockIdx.y;
  if (c >= s.C) return;
  float h = s.h0 ? s.h0[b * s.C + c] : 0;
  for (int64_t t = 0; t < s.T; ++t) {
    const int64_t at = (b * s.T + t) * s.C + c;
    h = fmaf(s.a[at], h, s.x[at]);
    s.h[at] = h;
  }
}

__global__ __launch_bounds__(64) void scan_grad_channels(ScanGradDesc s) {
  const int64_t c = (int64_t)blockIdx.x * 64 + threadIdx.x, b = blockIdx.y;
  if (c >= s.C) return;
  float carry = 0;
  for (int64_t t = s.T - 1; t >= 0; --t) {
    const int64_t at = (b * s.T + t) * s.C + c;
    const float g = s.dh[at] + carry;
    const float before = t > 0 ? s.h[at - s.C] : s.h0 ? s.h0[b * s.C + c] : 0;
    if (s.da) s.da[at] = g * before;
    if (s.dx) s.dx[at] = g;
    carry = s.a[at] * g;
  }
  if (s.dh0) s.dh0[b * s.C + c] = carry;
}

}  // namespace

void rope(const RopeDesc& r, hipStream_t st) {
  const int64_t n = (int64_t)r.B * r.T * (r.D - r.half);
  klaunch(rope_pairs, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, r);
}

int64_t scan_workspace_bytes(int64_t, int64_t, int64_t) { return 0; }
void scan(const ScanDesc& s, void*, hipStream_t st) {
  klaunch(scan_channels, dim3((unsigned)((s.C + 63) / 64), (unsigned)s.B), dim3(64), 0, st, s);
}
void scan_grad(const ScanGradDesc& s, void*, hipStream_t st) {
  klaunch(scan_grad_channels, dim3((unsigned)((s.C + 63) / 64), (unsigned)s.B), dim3(64), 0, st, s);
}

}  // namespace tgk
