// Rotary positions of several axes and the gated linear recurrence for gfx950.
#include <algorithm>

#include "kernels.h"
#include "sequence.h"

namespace tgk {
namespace {

// ---- rotary positions ------------------------------------------------------------------------------
//
// Bound by memory: every value is read once and written once. A thread finds the angle of one pair of one row (b, t) and
// turns that pair in `each` heads, all tensors' heads counted through, so that the angle costs little. Few rows: fewer heads
// a thread, so that there are threads for the whole card. 4 x 4096 positions, 20 heads of 128, there and back: 671 MB in 122 us,
// 5.5 TB/s.

// cos and sin of position * freq. The product is taken in 64 bits and brought to r in [-pi/4, pi/4] by the nearest multiple
// of pi/2 (in two parts, 2^-106 in all), where the Taylor series to r^9 and r^10 are off by less than 2^-28. Up to some 2^50: the
// multiple must come out right to a half (bases below 2^-16 are refused).
__device__ __forceinline__ void angle(int position, double freq, float& c, float& s) {
  const double x = (double)position * freq, n = rint(x * 0.63661977236758134308);
  const float r = (float)fma(-n, 6.123233995736766e-17, fma(-n, 1.5707963267948966, x));
  const float q = r * r;
  const float sr = fmaf(r * q, fmaf(q, fmaf(q, fmaf(q, 1.0f / 362880, -1.0f / 5040), 1.0f / 120), -1.0f / 6), r);
  const float cr = fmaf(q, fmaf(q, fmaf(q, fmaf(q, fmaf(q, -1.0f / 3628800, 1.0f / 40320), -1.0f / 720), 1.0f / 24), -0.5f), 1.0f);
  const int k = (int)((long long)n & 3);
  c = k & 1 ? sr : cr;
  s = k & 1 ? cr : sr;
  if (k == 1 || k == 2) c = -c;
  if (k >= 2) s = -s;
}

struct RopeArgs {
  RopeDesc d;
  FastDiv units, T;
  int total, each;                 // heads of all tensors; heads a thread
};
__global__ __launch_bounds__(256) void rope_pairs(RopeArgs R) {
  const RopeDesc& r = R.d;
  const uint32_t id = blockIdx.x * 256 + threadIdx.x, row = fastdiv(id, R.units), u = id - row * R.units.d;
  if (row >= (uint32_t)(r.B * r.T)) return;
  const int b = fastdiv(row, R.T), t = row - b * R.T.d;
  const bool turn = (int)u < r.half;         // a pair, else a feature that passes
  float c = 1, s = 0;
  if (turn) {
    const RopePair p = r.pairs[u];
    angle(r.positions[((int64_t)p.axis * r.B + b) * r.T + t], p.freq, c, s);
  }
  const int from = blockIdx.y * R.each, to = min(from + R.each, R.total);
  int first = 0;                             // heads before this tensor
  for (int i = 0; i < r.n; first += r.heads[i], ++i) {
    const int h0 = max(from - first, 0), h1 = min(to - first, r.heads[i]);
    const float sg = r.inverse[i] ? -s : s;
    const float* x = r.x[i].p + b * r.x[i].b + t * r.x[i].t;
    float* y = r.y[i].p + b * r.y[i].b + t * r.y[i].t;
    for (int h = h0; h < h1; h += 4) {
      float x1[4], x2[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float* xh = x + min(h + e, h1 - 1) * r.x[i].h;
        x1[e] = turn ? xh[u] : 0.0f;
        x2[e] = xh[u + r.half];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (h + e >= h1) break;
        float* yh = y + (h + e) * r.y[i].h;
        if (turn) yh[u] = x1[e] * c - x2[e] * sg;
        yh[u + r.half] = turn ? x2[e] * c + x1[e] * sg : x2[e];
      }
    }
  }
}

// ---- gated linear recurrence -----------------------------------------------------------------------
//
// Bound by memory: a and x are read once and h written once (a, h, dh read, da, dx written). Channels alone do not fill the
// card, so time is cut into chunks, and a chunk keeps its values in registers while it waits for what comes in:
//  * a block holds 64 channels x 4 S steps, S steps a wavefront, a channel a lane. Each wavefront folds its steps into
//    (A, H), h_out = A h_in + H; the block joins its four and publishes its own pair;
//  * what comes in is joined from the pairs of the chunks before, in a fixed order whatever the timing (so results repeat bit
//    for bit): first those of whole groups of kGroup chunks, which the last block of each group joins and publishes, then
//    those of its own group;
//  * then the steps are run again from registers, now with the true state, and stored.
// 4 x 8192 x 1024: forward 403 MB in 87 us (4.6 TB/s), backward 671 MB in 132 us (5.1 TB/s); a large copy reaches 5.0.
// A state of 1e30 may fall to an ordinary value by a product of gates that f32 does not hold, so products are held as
// s = A 2^100: A is exact to f32's roundings down to 2^-226, and what is lost below is at most 2^-250 of h_in, under 2^-122.
// Gates above 1 in magnitude can take a product out of the range upwards (from 2^28 on) while no state is (h_in = 0, or a small
// gate later), or bring back what fell out of it. A block with such products waits for the true state, runs its steps in order
// and publishes (NaN, its state), which replaces any state; a group with one, likewise. s is 0 only after a gate of 0: a state
// that is infinite stays so through smaller products.
// A pair is one 64-bit word, stored and loaded whole at device scope; all ones mean "not there yet". A block takes its place
// from a counter as it starts, and waits only for blocks of lower places: those are running, and publish their own pair
// after waiting for lower places at most, a group's pair too. So every wait ends.

typedef unsigned long long word;
constexpr int kGroup = 8;
constexpr word kEmpty = ~0ull;
constexpr float kSet = __builtin_nanf("");   // a product that replaces the state

__device__ __forceinline__ word look(const word* at) { return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ float gates(word v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float value(word v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ void publish(word* at, float A, float H) {
  word v = (word)__float_as_uint(H) << 32 | __float_as_uint(A);
  if (v == kEmpty) v = kEmpty - 1;             // a NaN either way
  __hip_atomic_store(at, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
constexpr float kOne = 0x1p100f, kPerOne = 0x1p-100f;   // s of A = 1
__device__ __forceinline__ float not_zero(float s) { return s == 0 ? copysignf(0x1p-149f, s) : s; }
// A state through a product of gates, A state + H: the smaller factor takes the power of two, where nothing of it is lost that
// the product would keep.
__device__ __forceinline__ float through(float s, float state, float H) {
  const bool large = fabsf(s) >= 1;
  const float h = fmaf(large ? s * kPerOne : s, large ? state : state * kPerOne, H);
  return s != s ? H : h;
}
__device__ __forceinline__ float product(float s, float z) {
  const bool large = fabsf(s) >= fabsf(z);
  const float p = (large ? s : z) * kPerOne * (large ? z : s);
  return s == 0 || z == 0 ? p : not_zero(p);
}
// Whether a product of gates, seen factor by factor, can be used: it must not have left the range upwards (then s is infinite,
// or NaN), nor downwards where a factor above 1 may have brought it back.
struct Reach {
  float least = kOne, gate = 0;
  __device__ __forceinline__ void see(float s, float g) {
    least = fminf(least, fabsf(s));
    gate = fmaxf(gate, fabsf(g));
  }
  __device__ __forceinline__ bool out(float s) const { return !(fabsf(s) < INFINITY) || (gate > 1 && least < 0x1p-126f); }
};
// (A, H) followed by n pairs, `step` words apart, in order. Loads go out together; what is not there yet is asked for again.
__device__ __forceinline__ void follow(float& A, float& H, Reach& reach, const word* at, int64_t step, int n) {
  for (int k0 = 0; k0 < n; k0 += kGroup) {
    word v[kGroup];
#pragma unroll
    for (int k = 0; k < kGroup; ++k) v[k] = look(at + min(k0 + k, n - 1) * step);
#pragma unroll
    for (int k = 0; k < kGroup; ++k) {
      if (k0 + k >= n) break;
      while (v[k] == kEmpty) {
        __builtin_amdgcn_s_sleep(2);
        v[k] = look(at + (k0 + k) * step);
      }
      H = through(gates(v[k]), H, value(v[k]));
      A = product(A, gates(v[k]));
      reach.see(A, gates(v[k]) * kPerOne);
    }
  }
}

struct ScanPlan {
  int S, chunks, cblocks;          // steps a wavefront; chunks of 4 S steps; blocks of 64 channels over all batch entries
  int64_t words;                   // pairs: of the chunks, then of the groups, [.][cblocks * 64]; then the place counter
};
ScanPlan scan_plan(int64_t B, int64_t T, int64_t C) {
  ScanPlan p{};
  p.cblocks = (int)(B * ((C + 63) / 64));
  p.S = 32;
  while (p.S > 4 && (T <= 2 * p.S || p.cblocks * ((T + 4 * p.S - 1) / (4 * p.S)) < 256)) p.S /= 2;
  p.chunks = (int)((T + 4 * p.S - 1) / (4 * p.S));
  p.words = p.chunks > 1 ? (int64_t)(p.chunks + p.chunks / kGroup) * p.cblocks * 64 + 1 : 0;
  return p;
}

__global__ __launch_bounds__(256) void scan_clear(word* w, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n) w[i] = i == n - 1 ? 0 : kEmpty;   // the last word is the place counter
}

// Forward and backward in one form: step u = 0, 1, .. is t = u or t = T - 1 - u, state = gate * state + in. Backward the
// state g[t + 1] comes in to step t through its gate a[t + 1].
struct ScanArgs {
  int64_t T, C;
  int chunks, cblocks, per;        // per: channel blocks of a batch entry
  const float *a, *in, *h0, *h;    // h: backward
  float *out, *da, *dh0;           // out: h, or dx; each may be null backward
  word* words;
};

template <int S, bool BACK>
__global__ __launch_bounds__(256) void scan_chunks(ScanArgs s) {
  __shared__ float fold[4][2][64], came[64];
  __shared__ unsigned place;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int64_t row = (int64_t)s.cblocks * 64;
  unsigned id = blockIdx.x;
  if (s.chunks > 1) {
    if (tid == 0) place = atomicAdd((unsigned*)(s.words + (s.chunks + s.chunks / kGroup) * row), 1u);
    __syncthreads();
    id = place;
  }
  const int chunk = id / s.cblocks, cb = id % s.cblocks, b = cb / s.per;
  const int64_t c = (int64_t)(cb % s.per) * 64 + lane, cc = min(c, s.C - 1);
  const int64_t u0 = ((int64_t)chunk * 4 + w) * S, base = (int64_t)b * s.T * s.C + cc;
  const float h0 = s.h0 ? s.h0[(int64_t)b * s.C + cc] : 0.0f;
  float g[S], x[S], before[BACK ? S : 1];
#pragma unroll
  for (int k = 0; k < S; ++k) {    // past the end: any value that is there, put right below
    const int64_t u = min(u0 + k, s.T - 1), t = BACK ? s.T - 1 - u : u;
    x[k] = s.in[base + t * s.C];
    g[k] = s.a[base + (BACK ? min(t + 1, s.T - 1) : t) * s.C];
    if (BACK) before[k] = s.da ? s.h[base + max(t - 1, (int64_t)0) * s.C] : 0.0f;
  }
#pragma unroll
  for (int k = 0; k < S; ++k) {    // there the state goes on as it is
    const int64_t u = u0 + k;
    if (BACK && u == 0) g[k] = 0;  // nothing comes in to the last step
    if (BACK && u == s.T - 1) before[k] = h0;
    if (u >= s.T) {
      x[k] = 0;
      g[k] = 1;
    }
  }
  float A = kOne, H = 0, gate = 1;   // gate: the smallest
  Reach own;
#pragma unroll
  for (int k = 0; k < S; ++k) {
    H = fmaf(g[k], H, x[k]);
    A *= g[k];
    own.see(A, g[k]);
    gate = fminf(gate, fabsf(g[k]));
  }
  if (gate > 0) A = not_zero(A);
  fold[w][0][lane] = A;
  fold[w][1][lane] = H;
  const bool apart = __syncthreads_or(own.out(A));   // the wavefronts' products cannot be used
  word* pairs = s.words + (int64_t)cb * 64 + lane;
  word* groups = pairs + s.chunks * row;
  const int group = chunk / kGroup, in_group = chunk % kGroup;
  const bool closes = in_group == kGroup - 1;
  float state = BACK ? 0.0f : h0, skip = kOne;
  Reach none;
  if (!apart) {
    if (s.chunks > 1) {
      if (w == 0) {
        float a4 = kOne, h4 = 0;
        Reach reach;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float f = fold[k][0][lane];
          h4 = through(f, h4, fold[k][1][lane]);
          a4 = product(a4, f);
          reach.see(a4, f * kPerOne);
        }
        const bool serial = __any(reach.out(a4));     // nor their product
        if (!serial) publish(pairs + chunk * row, a4, h4);
        float ga = kOne, gh = 0;
        follow(ga, gh, reach, pairs + (int64_t)group * kGroup * row, row, in_group);   // the group's chunks before this one
        const float all = product(ga, a4);                // the group's product
        reach.see(all, a4 * kPerOne);
        const bool whole = !__any(reach.out(all));
        if (whole && closes) publish(groups + group * row, all, through(a4, gh, h4));
        follow(skip, state, none, groups, row, group);
        if (whole) state = through(ga, state, gh);
        else follow(skip, state, none, pairs + (int64_t)group * kGroup * row, row, in_group);
        came[lane] = state;
        if (!whole) {
#pragma unroll
          for (int k = 0; k < 4; ++k) state = through(fold[k][0][lane], state, fold[k][1][lane]);
          if (serial) publish(pairs + chunk * row, kSet, state);
          if (closes) publish(groups + group * row, kSet, state);
        }
      }
      __syncthreads();
      state = came[lane];
    }
    for (int k = 0; k < w; ++k) state = through(fold[k][0][lane], state, fold[k][1][lane]);
  } else {
    if (w == 0) {
      if (s.chunks > 1) {
        follow(skip, state, none, groups, row, group);
        follow(skip, state, none, pairs + (int64_t)group * kGroup * row, row, in_group);
      }
      came[lane] = state;
    }
    float mine = 0;                // the state that comes to this wavefront
    for (int k = 0; k < 4; ++k) {
      __syncthreads();
      if (w == k) {
        float h = mine = came[lane];
#pragma unroll
        for (int e = 0; e < S; ++e) h = fmaf(g[e], h, x[e]);
        came[lane] = h;
      }
    }
    __syncthreads();
    if (s.chunks > 1 && w == 0) {
      publish(pairs + chunk * row, kSet, came[lane]);
      if (closes) publish(groups + group * row, kSet, came[lane]);
    }
    state = mine;
  }
  if (c >= s.C) return;
#pragma unroll
  for (int k = 0; k < S; ++k) {
    const int64_t u = u0 + k, t = BACK ? s.T - 1 - u : u;
    if (u >= s.T) break;
    state = fmaf(g[k], state, x[k]);
    if (!BACK || s.out) s.out[base + t * s.C] = state;
    if (BACK && s.da) s.da[base + t * s.C] = state * before[k];
  }
  if (BACK && s.dh0 && u0 < s.T && u0 + S >= s.T) s.dh0[(int64_t)b * s.C + c] = state * s.a[base];
}

}  // namespace

void rope(const RopeDesc& r, hipStream_t st) {
  RopeArgs R{r, make_fastdiv((uint32_t)(r.D - r.half)), make_fastdiv((uint32_t)r.T), 0, 0};
  for (int i = 0; i < r.n; ++i) R.total += r.heads[i];
  const int64_t threads = (int64_t)r.B * r.T * (r.D - r.half);
  // 2^19 threads fill the card (256 CUs of 32 wavefronts); beyond, a thread takes all heads
  R.each = (int)std::min<int64_t>(R.total, std::max<int64_t>((R.total + 65534) / 65535, threads * R.total >> 19));
  klaunch(rope_pairs, dim3((unsigned)((threads + 255) / 256), (unsigned)((R.total + R.each - 1) / R.each)), dim3(256), 0, st, R);
}

int64_t scan_workspace_bytes(int64_t B, int64_t T, int64_t C) { return scan_plan(B, T, C).words * 8; }

namespace {
template <bool BACK>
void run_scan(ScanArgs s, int64_t B, void* work, hipStream_t st) {
  const ScanPlan p = scan_plan(B, s.T, s.C);
  s.chunks = p.chunks;
  s.cblocks = p.cblocks;
  s.per = (int)((s.C + 63) / 64);
  s.words = (word*)work;
  if (p.words) klaunch(scan_clear, dim3((unsigned)((p.words + 255) / 256)), dim3(256), 0, st, s.words, p.words);
  const dim3 grid((unsigned)((int64_t)p.chunks * p.cblocks));
  if (p.S == 32) klaunch(scan_chunks<32, BACK>, grid, dim3(256), 0, st, s);
  else if (p.S == 16) klaunch(scan_chunks<16, BACK>, grid, dim3(256), 0, st, s);
  else if (p.S == 8) klaunch(scan_chunks<8, BACK>, grid, dim3(256), 0, st, s);
  else klaunch(scan_chunks<4, BACK>, grid, dim3(256), 0, st, s);
}
}  // namespace

void scan(const ScanDesc& d, void* work, hipStream_t st) {
  ScanArgs s{};
  s.T = d.T;
  s.C = d.C;
  s.a = d.a;
  s.in = d.x;
  s.h0 = d.h0;
  s.out = d.h;
  run_scan<false>(s, d.B, work, st);
}

void scan_grad(const ScanGradDesc& d, void* work, hipStream_t st) {
  ScanArgs s{};
  s.T = d.T;
  s.C = d.C;
  s.a = d.a;
  s.in = d.dh;
  s.h0 = d.h0;
  s.h = d.h;
  s.out = d.dx;
  s.da = d.da;
  s.dh0 = d.dh0;
  run_scan<true>(s, d.B, work, st);
}

}  // namespace tgk
