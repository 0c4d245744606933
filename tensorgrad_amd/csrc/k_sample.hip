// Choice of the next token for gfx950: temperature, top-k, top-p and min-p from a given random number, see ops.py.
//
// Every limit keeps a first part of the tokens ordered by (falling logit, rising index), so no sort is needed: a border (key,
// ties) is found by counting and weighing tokens in bins of their logit's bits. Weights are whole numbers, exp(z) times 2^unit
// with z = (logit - largest) / temperature in 64 bits and 62 bits for the sum of all: sums do not depend on their order, so
// counts, borders and the choice agree with each other and repeat, and a weight is off by 2^(-unit-1) of the largest at most.
#include <algorithm>

#include "kernels.h"
#include "sequence.h"

namespace tgk {
namespace {

typedef unsigned long long u64;
constexpr int kThreads = 1024, kWaves = kThreads / 64, kBins = 2048;
constexpr uint32_t kNoKey = 0xffffffffu;   // minus infinity and NaN: never chosen

// Ascending in falling logits; -0 and 0 are equal.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (!(x > -INFINITY)) return kNoKey;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b & 0x80000000u ? b : ~b & 0x7fffffffu;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key : ~key & 0x7fffffffu); }

struct Row {
  float top;                       // largest logit
  double per;                      // 1 / temperature
  int unit;
};
__device__ __forceinline__ double weight(const Row& r, float x) {   // of the largest
  if (x == r.top) return 1;
  return exp(((double)x - (double)r.top) * r.per);
}
__device__ __forceinline__ u64 whole(const Row& r, double w) { return (u64)rint(ldexp(w, r.unit)); }

__device__ __forceinline__ u64 wave_sum(u64 x) {
#pragma unroll
  for (int o = 1; o < 64; o *= 2) x += __shfl_xor(x, o);
  return x;
}
__device__ __forceinline__ u64 wave_scan(u64 x) {   // inclusive
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const u64 z = __shfl_up(x, o);
    if ((int)(threadIdx.x & 63) >= o) x += z;
  }
  return x;
}

// The first tokens of the order: those of a key below `key`, and the first `ties` of that key.
struct Border {
  uint32_t key;
  u64 ties;
};

struct Bins {
  u64 mass[kBins];
  uint32_t count[kBins];
  u64 sums[kWaves];
  u64 found[4];
};

// A border of the order before the border `within`: where the count reaches `most`, or the mass `target` (a token is kept while
// what stands before it weighs less). *total: the mass of what is kept. Three levels of bits of the key.
template <bool COUNT>
__device__ Border find_border(const float* x, int V, const Row& r, Border within, u64 most, double target, Bins& bins, u64* total) {
  const int tid = threadIdx.x;
  uint32_t lo = 0;                 // keys of the bin that the border lies in: lo ...
  int shift = 32;                  // ... and its first 32 - shift bits
  u64 before = 0, mass_before = 0;
  for (int level = 0; level < 3; ++level) {
    const int bits = level < 2 ? 11 : 10, next = shift - bits;
    for (int i = tid; i < kBins; i += kThreads) {
      bins.mass[i] = 0;
      bins.count[i] = 0;
    }
    __syncthreads();
    for (int i = tid; i < V; i += kThreads) {
      const uint32_t k = key_of(x[i]);
      if (k == kNoKey || k > within.key || (shift < 32 && (k >> shift) != (lo >> shift))) continue;
      const uint32_t bin = (k >> next) & ((1u << bits) - 1);
      atomicAdd(&bins.count[bin], 1u);
      if (k < within.key) atomicAdd(&bins.mass[bin], whole(r, weight(r, x[i])));
    }
    __syncthreads();
    if (tid == 0) {                // the last key's ties that count
      if (within.key != kNoKey && (shift == 32 || (within.key >> shift) == (lo >> shift))) {
        const uint32_t bin = (within.key >> next) & ((1u << bits) - 1);
        bins.mass[bin] += within.ties * whole(r, weight(r, value_of(within.key)));
      }
      u64 c = before, m = mass_before;
      int at = 0, last = -1;
      u64 lc = c, lm = m;
      for (; at < 1 << bits; ++at) {
        if (!bins.count[at]) continue;
        last = at;
        lc = c;
        lm = m;
        c += bins.count[at];
        m += bins.mass[at];
        if (COUNT ? c >= most : !((double)m < target)) break;
      }
      bins.found[0] = last;        // the bin of the border, or the last one that holds any
      bins.found[1] = lc;
      bins.found[2] = lm;
      bins.found[3] = last >= 0 ? bins.count[last] : 0;
    }
    __syncthreads();
    lo |= (uint32_t)bins.found[0] << next;
    before = bins.found[1];
    mass_before = bins.found[2];
    shift = next;
    __syncthreads();
  }
  const u64 w = whole(r, weight(r, value_of(lo)));
  u64 ties = bins.found[3];        // of key lo, all there are
  if (lo == within.key) ties = min(ties, within.ties);
  if (COUNT) {
    ties = min(ties, most - before);
  } else {
    u64 keep = 0;                  // those with mass before them below the target
    if (w == 0) keep = (double)mass_before < target ? ties : 0;
    else {
      const double room = (target - (double)mass_before) / (double)w;
      keep = room > 0 ? (u64)fmin(ceil(room), (double)ties) : 0;
      while (keep > 0 && !((double)(mass_before + (keep - 1) * w) < target)) --keep;
      while (keep < ties && (double)(mass_before + keep * w) < target) ++keep;
    }
    ties = keep;
  }
  *total = mass_before + ties * w;
  return {lo, ties};
}

// One block a row, several passes over it.
__global__ __launch_bounds__(kThreads) void sample_rows(SampleDesc s) {
  __shared__ Bins bins;
  __shared__ uint32_t tops[kWaves];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const float* x = s.logits + row * s.V;
  uint32_t top = kNoKey;
  for (int i = tid; i < s.V; i += kThreads) top = min(top, key_of(x[i]));
#pragma unroll
  for (int o = 1; o < 64; o *= 2) top = min(top, (uint32_t)__shfl_xor((int)top, o));
  if (lane == 0) tops[w] = top;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kWaves; ++k) top = min(top, tops[k]);
  if (top == kNoKey) {
    if (tid == 0) s.token[row] = -1;
    return;
  }
  Row r;
  r.top = value_of(top);
  const double heat = s.temperature ? (double)s.temperature[row] : s.temperature1;
  const bool greedy = !(heat > 0);
  r.per = greedy ? 1 : 1 / heat;
  r.unit = 62 - (s.V > 1 ? 32 - __clz(s.V - 1) : 0);
  const int32_t most = s.top_k ? s.top_k[row] : s.top_k1;
  const double p = s.top_p ? (double)s.top_p[row] : s.top_p1, least = s.min_p ? (double)s.min_p[row] : s.min_p1, u = s.u[row];
  Border kept = {kNoKey, 0};
  u64 total = 0;
  if (greedy) kept = {top, 1};
  else {
    if (most > 0 && most < s.V) kept = find_border<true>(x, s.V, r, kept, most, 0, bins, &total);
    if (p < 1) {
      if (kept.key == kNoKey) {    // the mass of all
        u64 m = 0;
        for (int i = tid; i < s.V; i += kThreads) if (key_of(x[i]) != kNoKey) m += whole(r, weight(r, x[i]));
        m = wave_sum(m);
        __syncthreads();
        if (lane == 0) bins.sums[w] = m;
        __syncthreads();
        for (int k = 0; k < kWaves; ++k) total += bins.sums[k];
      }
      kept = find_border<false>(x, s.V, r, kept, 0, p > 0 ? p * (double)total : 1.0, bins, &total);
    }
  }
  // each wavefront takes one stretch of the row, 64 tokens a step
  const int each = ((s.V + kWaves - 1) / kWaves + 63) / 64 * 64, from = min(w * each, s.V), to = min(from + each, s.V);
  int limit = INT32_MAX;           // tokens of the border's key count below this index
  if (kept.key != kNoKey) {
    u64 ties = 0;
    for (int i = from + lane; i < to; i += 64) ties += key_of(x[i]) == kept.key;
    ties = wave_sum(ties);
    __syncthreads();
    if (lane == 0) bins.sums[w] = ties;
    if (tid == 0) bins.found[0] = s.V;
    __syncthreads();
    u64 before = 0;
    for (int k = 0; k < w; ++k) before += bins.sums[k];
    if (before <= kept.ties && kept.ties < before + ties) {
      for (int i0 = from; i0 < to; i0 += 64) {
        const int i = i0 + lane;
        const bool tie = i < to && key_of(x[i]) == kept.key;
        const u64 mask = __ballot(tie);
        const u64 at = before + __popcll(mask & ((1ull << lane) - 1));
        if (tie && at == kept.ties) bins.found[0] = i;
        before += __popcll(mask);
        if (before > kept.ties) break;
      }
    }
    __syncthreads();
    limit = (int)bins.found[0];
  }
  auto weigh = [&](int i) -> u64 {
    if (i >= to) return 0;
    const float v = x[i];
    const uint32_t k = key_of(v);
    if (k == kNoKey || k > kept.key || (k == kept.key && i >= limit)) return 0;
    const double m = weight(r, v);
    return m >= least || k == top ? whole(r, m) : 0;
  };
  u64 mine = 0;
  for (int i = from + lane; i - lane < to; i += 64) mine += weigh(i);
  mine = wave_sum(mine);
  __syncthreads();
  if (lane == 0) bins.sums[w] = mine;
  __syncthreads();
  u64 before = 0, all = 0;
  for (int k = 0; k < kWaves; ++k) {
    if (k < w) before += bins.sums[k];
    all += bins.sums[k];
  }
  // passed: sum > u all, as whole numbers; u in [0, 1) leaves the last token's sum, all, to pass
  const u64 goal = min((u64)fmax(u * (double)all, 0.0), all - 1);
  if (!(before <= goal && goal < before + mine)) return;
  for (int i0 = from; i0 < to; i0 += 64) {
    const u64 m = weigh(i0 + lane), sum = before + wave_scan(m);
    const u64 passed = __ballot(sum > goal);
    if (passed) {
      if (lane == __ffsll(passed) - 1) s.token[row] = i0 + lane;
      return;
    }
    before = __shfl(sum, 63);
  }
}

}  // namespace

int64_t sample_workspace_bytes(const SampleDesc&) { return 0; }
void sample(const SampleDesc& s, void*, hipStream_t st) { klaunch(sample_rows, dim3((unsigned)s.rows), dim3(kThreads), 0, st, s); }

}  // namespace tgk
