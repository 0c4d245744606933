// Host-side launch wrappers of the sequence operators: masked attention (k_attend.hip), rotary positions of several axes
// and the gated linear recurrence (k_sequence.hip). Values are f32, indices i32; strides count elements.
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>

namespace tgk {

// Rows of [B, heads, T, D] read through strides; the last axis is contiguous.
struct Rows {
  float* p;
  int64_t b, h, t;
};

// y = attention(q, k, v), see ops.py: score = cap tanh(scale q.k / cap) - slope |p - j| (cap 0: scale q.k), p = n - Tq + i
// for the n keys of a batch entry. y or stats may be absent (null).
struct AttendDesc {
  int B, H, Hk, Tq, Tk, D, Dv;
  Rows q, k, v, y;
  float* stats;              // [B, H, Tq, 2], for the gradients: P = exp2(score log2(e) - stats[0]) stats[1]
  const int32_t* documents;  // [B, Tk] or null
  const int32_t* prefix;     // [B] or null
  const int32_t* lengths;    // [B] or null
  const float* slopes;       // [H] or null
  float scale, cap;
  bool causal, positional;   // positional: a query before position 0 sees nothing
};
struct AttendGradDesc {
  AttendDesc a;              // a.y and a.stats: the forward's results, read
  Rows dy, dq, dk, dv;       // dq, dk, dv may be absent (null)
};
constexpr int kAttendMaxHead = 128;
int64_t attend_workspace_bytes(const AttendDesc& a);
void attend(const AttendDesc& a, void* work, hipStream_t st);
int64_t attend_grad_workspace_bytes(const AttendGradDesc& g);
void attend_grad(const AttendGradDesc& g, void* work, hipStream_t st);

// Rotary positions: up to kRopeMax tensors turned by the same positions in one launch.
struct RopePair {
  double freq;               // angle = position * freq
  int32_t axis, pad;
};
constexpr int kRopeMax = 8;
struct RopeDesc {
  int B, T, D, half, n;      // half: pairs; features from 2 half on are copied
  const int32_t* positions;  // [A, B, T]
  const RopePair* pairs;     // [half]
  Rows x[kRopeMax], y[kRopeMax];
  int heads[kRopeMax];
  bool inverse[kRopeMax];
};
void rope(const RopeDesc& r, hipStream_t st);

// h[b, t, c] = a h[b, t-1, c] + x, all [B, T, C] contiguous, h0 [B, C] or null (zeros).
struct ScanDesc {
  int64_t B, T, C;
  const float *a, *x, *h0;
  float* h;
};
struct ScanGradDesc {
  int64_t B, T, C;
  const float *a, *h, *dh, *h0;
  float *da, *dx, *dh0;      // each may be absent (null)
};
int64_t scan_workspace_bytes(int64_t B, int64_t T, int64_t C);
void scan(const ScanDesc& s, void* work, hipStream_t st);
void scan_grad(const ScanGradDesc& s, void* work, hipStream_t st);

}  // namespace tgk
