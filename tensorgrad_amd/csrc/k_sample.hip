// Choice of the next token for gfx950: temperature, top-k, top-p and min-p from a given random number, see ops.py.
//
// Every limit keeps a first part of the tokens ordered by (falling logit, rising index), so the row is not sorted. Tokens are
// counted and weighed in bins of their distance to the largest logit; the bins that a limit's border may lie in are found by sums
// over bins, their tokens alone are listed and sorted, and what is kept is told by one bound on (logit, index). The weights of what
// is kept are summed by stretches of the vocabulary, and the stretch where the sum passes u of all is walked once more.
//
// Weights are whole numbers, exp(-z) times 2^unit with z = (largest - logit) / temperature in 64 bits and 62 bits for the sum of
// all: sums do not depend on their order, so counts, borders and the choice agree with each other and repeat. A weight is off by
// 2^(-unit-1) of the largest from being a whole number, and by 2^-50 of it at most from its own arithmetic: z / ln 2 = t by five
// roundings, 5 ln(2) t 2^-t <= 1.9 times 2^-53, the series 2, its last steps 1.4. Beyond some 32 to 43 in z they are 0. A
// temperature of 0 is a top-k of 1.
//
// A row is read three times, the first time from memory, and a stretch of it once more: for its largest logit; into bins, with
// weights of 32 bits that tell where top_p's border is to be looked for; for the list, with the weights of 64 bits that decide. Many
// rows: a block takes one, in one launch (sample_one; sample_short, which sorts all). Few rows of many tokens: several blocks a row,
// in four launches (sample_tops, _bins, _list, _choice).
#include <algorithm>
#include <cfloat>

#include "kernels.h"
#include "sequence.h"

namespace tgk {
namespace {

typedef unsigned long long u64;
constexpr int kBins = 2048;
constexpr int kList = 2048;                // tokens that are sorted, at most
constexpr uint32_t kNoKey = 0xffffffffu;   // minus infinity and NaN: never chosen
constexpr u64 kAll = ~0ull;

// Ascending in falling logits; -0 and 0 are equal.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (!(x > -INFINITY)) return kNoKey;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b & 0x80000000u ? b : ~b & 0x7fffffffu;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key : ~key & 0x7fffffffu); }
__device__ __forceinline__ u64 order_of(uint32_t key, int i) { return (u64)key << 32 | (uint32_t)i; }

// A row, its limits and its largest logit.
struct Row {
  const float* x;
  int V, most, unit;
  float top;                       // largest logit
  float shrink, shrunk;            // 1 or, where differences of logits may pass f32, 1 / 2; top times it
  float per_bin, per1;             // of differences times `shrink`: bins for 1; per in 32 bits
  double per, p, least, u;         // log2(e) / temperature; top_p; min_p times 2^unit; the random number
  bool by_count, by_mass;          // what limits
};
constexpr double kLn2 = 0.693147180559945309417;
__device__ __forceinline__ Row row_of(const SampleDesc& s, int64_t row, float top) {
  Row r;
  r.x = s.logits + row * s.V;
  r.V = s.V;
  r.top = top;
  const double heat = s.temperature ? (double)s.temperature[row] : s.temperature1;
  const double share = s.min_p ? (double)s.min_p[row] : s.min_p1;
  const bool greedy = !(heat > 0) || !(share <= 1);   // the first of the order alone; by NaN too
  const double per = greedy ? 1 : 1 / fmin(heat, FLT_MAX);
  r.unit = 62 - (s.V > 1 ? 32 - __clz(s.V - 1) : 0);
  r.per = per * (1 / kLn2);
  const bool vast = top > 0x1p100f;          // up to there f32 holds the distance of any x
  r.shrink = vast ? 0.5f : 1.0f;
  r.shrunk = top * r.shrink;
  r.per1 = (float)(vast ? 2 * r.per : r.per);
  r.per_bin = (float)((vast ? 2 * per : per) * (kBins / (1.001 * kLn2 * (r.unit + 1))));
  r.most = greedy ? 1 : s.top_k ? s.top_k[row] : s.top_k1;
  r.p = s.top_p ? (double)s.top_p[row] : s.top_p1;
  r.least = greedy ? 0 : __builtin_amdgcn_ldexp(share, r.unit);
  r.u = s.u[row];
  r.by_count = r.most > 0 && r.most < s.V;
  r.by_mass = r.p < 1 && !greedy;
  return r;
}
// A token's weight times 2^unit, 0 far from the top: 2^-t = 2^-n 2^f by the series of 2^f for |f| <= 1 / 2, 2^-52 off at most. Of
// a logit that is there. t is a number for infinite logits too. Three-operand instructions with the coefficient in scalar registers:
// the compiler's own choice copies every coefficient first.
struct Series {
  double c[13];
  constexpr Series() : c() {
    c[0] = 1;
    for (int k = 1; k < 13; ++k) c[k] = c[k - 1] * kLn2 / k;
  }
};
__device__ __forceinline__ double weight(const Row& r, float x) {
  constexpr Series s;
  const double t = fmin(fmax(((double)r.top - (double)x) * r.per, 0.0), 4000.0), n = rint(t), f = n - t;
  double e = s.c[12];
#pragma unroll
  for (int k = 11; k > 0; --k) asm("v_fma_f64 %0, %1, %2, %3" : "=v"(e) : "v"(e), "v"(f), "s"(s.c[k]));
  return __builtin_amdgcn_ldexp(fma(e, f, 1.0), r.unit - (int)n);
}
__device__ __forceinline__ u64 whole(double w) { return (u64)rint(w); }
// per_bin or per1 times how far a logit is from the largest. None where it is the largest: the factor may be infinite, or both logits.
__device__ __forceinline__ float distance(const Row& r, float x, float per) {
  return x == r.top ? 0.0f : fmaf(-x, r.shrink, r.shrunk) * per;
}
// A token's bin, rising with the distance to the top in equal steps; kBins: so far that its weight is 0, or not there.
__device__ __forceinline__ int bin_of(const Row& r, float x) {
  const float b = distance(r, x, r.per_bin);
  return b < kBins ? (int)b : kBins;
}

// The same from 32 bits, 2^-17 of it off at most (and 1): what finds where a border is to be looked for.
constexpr double kSlack = 0x1p-16;         // of a part of the sum: both sums off
__device__ __forceinline__ u64 about(const Row& r, float x) {
  return (u64)__builtin_amdgcn_exp2f((float)r.unit - distance(r, x, r.per1));
}

// Lanes' values without LDS: of a 64-bit number, by rows of 16 lanes (0 where there is none).
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ u64 moved(u64 x) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(x >> 32), CTRL, ROWS, 0xf, false);
  return (u64)hi << 32 | lo;
}
// Lane ^ half's value.
template <int HALF>
__device__ __forceinline__ u64 other_lane(u64 x) {
  if constexpr (HALF == 1) return moved<0xB1>(x);                 // [1, 0, 3, 2] of 4
  else if constexpr (HALF == 2) return moved<0x4E>(x);            // [2, 3, 0, 1]
  else if constexpr (HALF == 4) return moved<0x1B>(moved<0x141>(x));   // 8 mirrored, then 4
  else if constexpr (HALF == 8) return moved<0x128>(x);           // 16 turned by 8
  else {
    const uint32_t lo = (uint32_t)x, hi = (uint32_t)(x >> 32);
    const auto l = HALF == 16 ? __builtin_amdgcn_permlane16_swap(lo, lo, false, false) : __builtin_amdgcn_permlane32_swap(lo, lo, false, false);
    const auto h = HALF == 16 ? __builtin_amdgcn_permlane16_swap(hi, hi, false, false) : __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
    const int k = threadIdx.x & HALF ? 0 : 1;
    return (u64)h[k] << 32 | l[k];
  }
}
__device__ __forceinline__ u64 wave_scan(u64 x) {   // inclusive
  x += moved<0x111>(x);
  x += moved<0x112>(x);
  x += moved<0x114>(x);
  x += moved<0x118>(x);
  x += moved<0x142, 0xa>(x);       // a row's last to the next, for rows 1 and 3; then lane 31's to rows 2 and 3
  x += moved<0x143, 0xc>(x);
  return x;
}
__device__ __forceinline__ u64 lane_value(u64 x, int lane) {
  return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)x, lane);
}
__device__ __forceinline__ u64 wave_sum(u64 x) { return lane_value(wave_scan(x), 63); }
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int o = 1; o < 64; o *= 2) x = fmaxf(x, __shfl_xor(x, o));
  return x;
}

struct Bins {
  u64 mass[kBins];                         // about
  uint32_t count[kBins];
};
// What a block shares while it finds a row's borders and its choice.
template <int LIST>
struct Work {
  u64 list[LIST];
  u64 sums[2][16];
  u64 found[8];
  uint32_t listed;
};

// f(i, x[i]) for a thread's i of [from, to), `step` apart; 8 loads at once.
template <class F>
__device__ __forceinline__ void each_token(const float* x, int from, int to, int step, F f) {
  constexpr int N = 8;
  for (int i = from; i < to; i += N * step) {
    float v[N];
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = x[min(i + e * step, to - 1)];
#pragma unroll
    for (int e = 0; e < N; ++e) if (i + e * step < to) f(i + e * step, v[e]);
  }
}

// The largest logit of [from, to); NaN is none.
template <int THREADS, class Work>
__device__ __forceinline__ float block_top(const float* x, int from, int to, Work& w) {
  float top = -INFINITY;
  each_token(x, from + (int)threadIdx.x, to, THREADS, [&](int, float v) { top = fmaxf(top, v); });
  top = wave_max(top);
  if ((threadIdx.x & 63) == 0) w.sums[0][threadIdx.x >> 6] = __float_as_uint(top);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < THREADS / 64; ++k) top = fmaxf(top, __uint_as_float((uint32_t)w.sums[0][k]));
  return top;
}
// Counts and weighs [from, to) in bins. A few tokens at most are kept by their count alone: then all of them are listed.
constexpr int kFew = 1024;
__device__ __forceinline__ bool few(const Row& r) { return r.by_count && r.most <= kFew; }
template <int THREADS>
__device__ __forceinline__ void clear_bins(Bins& b) {
  for (int i = threadIdx.x; i < kBins; i += THREADS) {
    b.mass[i] = 0;
    b.count[i] = 0;
  }
}
template <int THREADS>
__device__ __forceinline__ void fill_bins(const Row& r, int from, int to, Bins& b) {
  const bool weigh = r.by_mass && !few(r);
  each_token(r.x, from + (int)threadIdx.x, to, THREADS, [&](int, float x) {
    const int bin = bin_of(r, x);
    if (bin == kBins) return;
    atomicAdd(&b.count[bin], 1u);
    if (weigh) atomicAdd(&b.mass[bin], about(r, x));
  });
}
// Sums over the bins before this thread's first (it has kBins / THREADS of them), and over all.
template <int THREADS, class Work>
__device__ __forceinline__ void bin_sums(const Bins& b, Work& w, u64& count, u64& mass, u64& all_count, u64& all_mass) {
  constexpr int N = kBins / THREADS;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  u64 c = 0, m = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    c += b.count[tid * N + i];
    m += b.mass[tid * N + i];
  }
  const u64 cs = wave_scan(c), ms = wave_scan(m);
  __syncthreads();
  if (lane == 63) {
    w.sums[0][wave] = cs;
    w.sums[1][wave] = ms;
  }
  __syncthreads();
  count = cs - c;
  mass = ms - m;
  all_count = all_mass = 0;
#pragma unroll
  for (int k = 0; k < THREADS / 64; ++k) {
    if (k < wave) {
      count += w.sums[0][k];
      mass += w.sums[1][k];
    }
    all_count += w.sums[0][k];
    all_mass += w.sums[1][k];
  }
}

// What the bins say: the bins [b0, b1] hold every border, `count` tokens stand before b0 and `size` are in them. whole: top_p is a
// part of the mass of all tokens, else of those up to b1 that top_k keeps.
struct Borders {
  int b0, b1;
  u64 count, size;
  bool whole;
};
constexpr Borders kNoBorder = {kBins, kBins - 1, 0, 0, false};
template <int THREADS, class Work>
__device__ __forceinline__ Borders borders(const Row& r, const Bins& b, Work& w) {
  constexpr int N = kBins / THREADS;
  const int tid = threadIdx.x;
  u64 c0, m0, all_c, all_m;
  bin_sums<THREADS>(b, w, c0, m0, all_c, all_m);
  if (tid < 8) w.found[tid] = 0;
  __syncthreads();
  const bool counted = r.by_count && all_c > (u64)r.most;
  // calls f(bin, sums before it, sums with it) for this thread's bins
  auto each = [&](auto f) {
    u64 c = c0, m = m0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const u64 c1 = c + b.count[tid * N + i], m1 = m + b.mass[tid * N + i];
      f(tid * N + i, c, m, c1, m1);
      c = c1;
      m = m1;
    }
  };
  if (counted) {
    each([&](int bin, u64 c, u64 m, u64 c1, u64 m1) {
      if (c < (u64)r.most && (u64)r.most <= c1) {
        w.found[0] = bin;
        w.found[1] = m;
        w.found[2] = c1;
        w.found[3] = c;
      }
    });
    __syncthreads();
  }
  const int kbin = (int)w.found[0];
  const u64 through = counted ? w.found[2] : all_c;
  if (few(r)) return {0, counted ? kbin : kBins - 1, 0, through, false};   // all that top-k keeps, or all there are
  if (!r.by_mass) return counted ? Borders{kbin, kbin, w.found[3], through - w.found[3], false} : kNoBorder;
  // the sum that top_p is a part of: top-k's border bin is not resolved yet
  const double least = r.p > 0 ? r.p * (1 - kSlack) * (double)(counted ? w.found[1] : all_m) : 0;
  const double most = r.p > 0 ? r.p * (1 + kSlack) * (double)all_m : 0;
  each([&](int bin, u64 c, u64 m, u64 c1, u64 m1) {
    if (((double)m < least || bin == 0) && !((double)m1 < least)) {
      w.found[4] = bin;
      w.found[5] = c;
    }
    if (((double)m < most || bin == 0) && (!((double)m1 < most) || bin == kBins - 1)) {
      w.found[6] = bin;
      w.found[7] = c1;
    }
  });
  __syncthreads();
  const int b0 = (int)w.found[4];
  const u64 count = w.found[5];
  if (counted) return {b0, kbin, count, through - count, false};
  return {b0, (int)w.found[6], count, w.found[7] - count, true};
}

// Lists the tokens of a stretch in the border's bins, and sums weights of the others, by a wavefront.
struct Sums {
  u64 all, before, kept;           // of all (`whole`); of the bins before the border's; of those of them that min_p keeps
};
template <class Push>
__device__ __forceinline__ Sums list_and_sum(const Row& r, const Borders& o, int from, int to, Push push) {
  Sums s = {};
  const int weigh = o.whole ? kBins : o.b0;
  each_token(r.x, from + (int)(threadIdx.x & 63), to, 64, [&](int i, float x) {
    const int bin = bin_of(r, x);
    if (bin >= o.b0 && bin <= o.b1) push(order_of(key_of(x), i));
    if (bin < weigh) {
      const double w = weight(r, x);
      const u64 m = whole(w);
      s.all += m;
      if (bin < o.b0) {
        s.before += m;
        s.kept += w >= r.least ? m : 0;
      }
    }
  });
  return {wave_sum(s.all), wave_sum(s.before), wave_sum(s.kept)};
}

// One step of a bitonic sort between lanes, straight: a branch a step cost 300 ns of latency instead of 40.
template <int HALF>
__device__ __forceinline__ void lane_step(u64& x, int i, int size) {
  const u64 y = other_lane<HALF>(x);
  const bool low = ((i & HALF) == 0) == ((i & size) == 0);   // takes the smaller
  x = (y < x) == low ? y : x;
}
template <int HALF>
__device__ __forceinline__ void lane_steps(u64& x, int i, int size) {
  lane_step<HALF>(x, i, size);
  if constexpr (HALF > 1) lane_steps<HALF / 2>(x, i, size);
}
// Sorts the first n of w.list: bitonic, a thread having every THREADS-th token. Steps of 1 to 32 places are exchanges of lanes, those of
// THREADS and more a thread's own; the rest go through LDS, 10 of 55 steps for 1024 tokens of 1024 threads.
template <int THREADS, int LIST>
__device__ __forceinline__ void sort_list(int n, Work<LIST>& w) {
  constexpr int N = LIST / THREADS;
  const int tid = threadIdx.x, uniform = __builtin_amdgcn_readfirstlane(n);
  int n2 = 64;
  while (n2 < uniform) n2 *= 2;
  u64 x[N];
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const int i = e * THREADS + tid;
    x[e] = i < n ? w.list[i] : kAll;
    if (e * THREADS >= n2) continue;
    lane_steps<1>(x[e], i, 2);
    lane_steps<2>(x[e], i, 4);
    lane_steps<4>(x[e], i, 8);
    lane_steps<8>(x[e], i, 16);
    lane_steps<16>(x[e], i, 32);
    lane_steps<32>(x[e], i, 64);
  }
  auto keep = [&](int e, u64 other, int size, int half) {
    const int i = e * THREADS + tid;
    const bool low = ((i & half) == 0) == ((i & size) == 0);
    x[e] = (other < x[e]) == low ? other : x[e];
  };
  for (int size = 128; size <= n2; size *= 2) {
    for (int half = size / 2; half >= 64; half /= 2) {
      if (half >= THREADS) {
#pragma unroll
        for (int d = 1; d < N; d *= 2)
          if (half == d * THREADS)
#pragma unroll
            for (int e = 0; e < N; ++e)
              if ((e & d) == 0) {
                const u64 a = x[e], b = x[e + d];
                keep(e, b, size, half);
                keep(e + d, a, size, half);
              }
      } else {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < N; ++e) if (e * THREADS < n2) w.list[e * THREADS + tid] = x[e];
        __syncthreads();
#pragma unroll
        for (int e = 0; e < N; ++e) if (e * THREADS < n2) keep(e, w.list[e * THREADS + (tid ^ half)], size, half);
      }
    }
#pragma unroll
    for (int e = 0; e < N; ++e) if (e * THREADS < n2) lane_steps<32>(x[e], e * THREADS + tid, size);
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < N; ++e) if (e * THREADS < n2) w.list[e * THREADS + tid] = x[e];
  __syncthreads();
}

// The bound of what is kept (an order, inclusive) from the n tokens of the border's bins in w.list and the mass of the others; calls
// add(token, weight) for those of them that are kept, by min_p too. ok: the border does lie in these bins.
template <int THREADS, int LIST, class Add>
__device__ __forceinline__ u64 bound_of_list(const Row& r, const Borders& o, int n, u64 before_all, u64 all, Work<LIST>& w, bool& ok, Add add) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  sort_list<THREADS, LIST>(n, w);
  // a thread has N neighbours; those that top-k keeps
  constexpr int N = LIST / THREADS;
  const int kept = r.by_count ? (int)min((u64)n, (u64)r.most - min((u64)r.most, o.count)) : n;
  double m[N];
  u64 sum = 0;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const int i = tid * N + e;
    const uint32_t key = i < kept ? (uint32_t)(w.list[i] >> 32) : kNoKey;
    m[e] = key == kNoKey ? 0 : weight(r, value_of(key));
    sum += whole(m[e]);
  }
  const u64 scan = wave_scan(sum);
  if (lane == 63) w.sums[0][wave] = scan;
  __syncthreads();
  u64 before = before_all + scan - sum, through = before_all;
#pragma unroll
  for (int k = 0; k < THREADS / 64; ++k) {
    if (k < wave) before += w.sums[0][k];
    through += w.sums[0][k];
  }
  if (tid == 0) w.found[0] = 0;
  __syncthreads();
  const double target = r.by_mass ? (r.p > 0 ? r.p * (double)(o.whole ? all : through) : 1.0) : (double)INFINITY;
  ok = (o.b0 == 0 || (double)before_all < target) && (!o.whole || o.b1 == kBins - 1 || !((double)through < target));
  int mine = 0;                    // what a wavefront keeps: in all, a first part of the list
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const int i = tid * N + e;
    const u64 u = whole(m[e]);
    const bool in = i < kept && (double)before < target;
    mine += __popcll(__ballot(in));
    if (in && m[e] >= r.least) add((int)(uint32_t)w.list[i], u);
    before += u;
  }
  if (lane == 0 && mine) atomicAdd(&w.found[0], (u64)mine);
  __syncthreads();
  const int end = (int)w.found[0];
  return end > 0 ? w.list[end - 1] : n > 0 ? w.list[0] - 1 : kAll;
}

// The same bound without a list, for more tokens than it holds in the border's bins: three levels of the key's bits, each a walk
// over the row. `within`: of what stands up to this key, and the first `ties` of that key.
struct Border {
  uint32_t key;
  u64 ties;
};
template <int THREADS, bool COUNT, class Work>
__device__ __forceinline__ Border find_border(const Row& r, Border within, double target, Bins& b, Work& w, u64* total) {
  constexpr int N = kBins / THREADS;
  const int tid = threadIdx.x;
  uint32_t lo = 0;                 // keys of the bin that the border lies in: lo ...
  int shift = 32;                  // ... and its first 32 - shift bits
  u64 before = 0, mass_before = 0;
#pragma unroll 1
  for (int level = 0; level < 3; ++level) {
    const int bits = level < 2 ? 11 : 10, next = shift - bits;
    __syncthreads();
    for (int i = tid; i < kBins; i += THREADS) {
      b.mass[i] = 0;
      b.count[i] = 0;
    }
    __syncthreads();
    for (int i = tid; i < r.V; i += THREADS) {
      const float v = r.x[i];
      const uint32_t k = key_of(v);
      if (k == kNoKey || k > within.key || (shift < 32 && (k >> shift) != (lo >> shift))) continue;
      const uint32_t bin = (k >> next) & ((1u << bits) - 1);
      atomicAdd(&b.count[bin], 1u);
      if (k < within.key) atomicAdd(&b.mass[bin], whole(weight(r, v)));
    }
    __syncthreads();
    // the last key's ties that count
    if (tid == 0 && within.key != kNoKey && (shift == 32 || (within.key >> shift) == (lo >> shift)))
      b.mass[(within.key >> next) & ((1u << bits) - 1)] += within.ties * whole(weight(r, value_of(within.key)));
    if (tid == 0) w.found[0] = kBins;
    __syncthreads();
    u64 c, m, all_c, all_m;
    bin_sums<THREADS>(b, w, c, m, all_c, all_m);
    u64 c1 = c, m1 = m;
    int last = -1;                 // the last bin that holds any, and the first that reaches the border
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int bin = tid * N + i;
      c1 += b.count[bin];
      m1 += b.mass[bin];
      if (!b.count[bin]) continue;
      last = bin;
      if (COUNT ? before + c1 >= (u64)r.most : !((double)(mass_before + m1) < target)) {
        atomicMin(&w.found[0], (u64)bin);
        break;
      }
    }
    if (tid == 0) w.found[1] = 0;
    __syncthreads();
    if (last >= 0) atomicMax(&w.found[1], (u64)last);
    __syncthreads();
    const int border = w.found[0] < kBins ? (int)w.found[0] : (int)w.found[1];
    __syncthreads();
    if (border / N == tid) {
      for (int i = 0; i < border % N; ++i) {
        c += b.count[tid * N + i];
        m += b.mass[tid * N + i];
      }
      w.found[2] = c;
      w.found[3] = m;
      w.found[4] = b.count[border];
    }
    __syncthreads();
    lo |= (uint32_t)border << next;
    before += w.found[2];
    mass_before += w.found[3];
    shift = next;
  }
  const u64 one = whole(weight(r, value_of(lo)));
  u64 ties = w.found[4];           // of key lo, all there are
  if (lo == within.key) ties = min(ties, within.ties);
  if (COUNT) {
    ties = min(ties, (u64)r.most - before);
  } else {                         // those with mass before them below the target
    u64 keep = 0;
    if (one == 0) keep = (double)mass_before < target ? ties : 0;
    else {
      const double room = (target - (double)mass_before) / (double)one;
      keep = room > 0 ? (u64)fmin(ceil(room), (double)ties) : 0;
      while (keep > 0 && !((double)(mass_before + (keep - 1) * one) < target)) --keep;
      while (keep < ties && (double)(mass_before + keep * one) < target) ++keep;
    }
    ties = keep;
  }
  *total = mass_before + ties * one;
  return {lo, ties};
}
template <int THREADS, class Work>
__device__ __forceinline__ u64 bound_by_walks(const Row& r, Bins& b, Work& w) {
  u64 all_mass = 0;
  if (r.by_mass && !r.by_count) {
    u64 sum = 0;
    for (int i = threadIdx.x; i < r.V; i += THREADS)
      if (key_of(r.x[i]) != kNoKey) sum += whole(weight(r, r.x[i]));
    sum = wave_sum(sum);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) w.sums[0][threadIdx.x >> 6] = sum;
    __syncthreads();
    for (int k = 0; k < THREADS / 64; ++k) all_mass += w.sums[0][k];
    __syncthreads();
  }
  Border kept = {kNoKey, 0};
  u64 total = all_mass;
  if (r.by_count) kept = find_border<THREADS, true>(r, kept, 0, b, w, &total);
  if (r.by_mass) kept = find_border<THREADS, false>(r, kept, r.p > 0 ? r.p * (double)total : 1.0, b, w, &total);
  if (kept.ties == 0) return order_of(kept.key, 0) - 1;
  // the index of the last tie that is kept: a wavefront takes a stretch
  constexpr int W = THREADS / 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, each = ((r.V + W - 1) / W + 63) / 64 * 64;
  const int from = min(wave * each, r.V), to = min(from + each, r.V);
  u64 ties = 0;
  for (int i = from + lane; i < to; i += 64) ties += key_of(r.x[i]) == kept.key;
  ties = wave_sum(ties);
  __syncthreads();
  if (lane == 0) w.sums[0][wave] = ties;
  if (tid == 0) w.found[0] = r.V;
  __syncthreads();
  u64 before = 0;
  for (int k = 0; k < wave; ++k) before += w.sums[0][k];
  if (before < kept.ties && kept.ties <= before + ties) {
    for (int i0 = from; i0 < to; i0 += 64) {
      const int i = i0 + lane;
      const bool tie = i < to && key_of(r.x[i]) == kept.key;
      const u64 mask = __ballot(tie);
      if (tie && before + __popcll(mask & ((1ull << lane) - 1)) + 1 == kept.ties) w.found[0] = i;
      before += __popcll(mask);
    }
  }
  __syncthreads();
  return order_of(kept.key, (int)w.found[0]);
}

// The weight that token i has in the choice.
__device__ __forceinline__ u64 kept_weight(const Row& r, u64 bound, int i, float x) {
  if (!(x > -INFINITY) || x < value_of((uint32_t)(bound >> 32)) || order_of(key_of(x), i) > bound) return 0;
  const double w = weight(r, x);
  return w >= r.least ? whole(w) : 0;
}
// Sum of the weights of [from, to), by a wavefront.
__device__ __forceinline__ u64 stretch_sum(const Row& r, u64 bound, int from, int to) {
  u64 sum = 0;
  each_token(r.x, from + (int)(threadIdx.x & 63), to, 64, [&](int i, float x) { sum += kept_weight(r, bound, i, x); });
  return wave_sum(sum);
}
// The token of [from, to) where the sum of weights passes `goal`, by a block: a thread sums N neighbours.
template <int THREADS, class Work>
__device__ __forceinline__ void choose(const Row& r, u64 bound, int from, int to, u64 goal, Work& w, int32_t* token) {
  constexpr int N = 4;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int i0 = from; i0 < to; i0 += N * THREADS) {
    u64 m[N], sum = 0;
    float v[N];
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = r.x[min(i0 + N * tid + e, to - 1)];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int i = i0 + N * tid + e;
      m[e] = i < to ? kept_weight(r, bound, i, v[e]) : 0;
      sum += m[e];
    }
    const u64 scan = wave_scan(sum);
    __syncthreads();
    if (lane == 63) w.sums[0][wave] = scan;
    __syncthreads();
    u64 before = scan - sum, all = 0;
#pragma unroll
    for (int k = 0; k < THREADS / 64; ++k) {
      if (k < wave) before += w.sums[0][k];
      all += w.sums[0][k];
    }
    if (goal < all) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        if (before <= goal && goal < before + m[e]) *token = i0 + N * tid + e;
        before += m[e];
      }
      return;
    }
    goal -= all;
  }
}
// Passed: sum > u all, as whole numbers; at most all - 1, which the last token's sum passes. Clamped before it is a whole number, too.
__device__ __forceinline__ u64 goal_of(const Row& r, u64 all) {
  return min((u64)fmin(fmax(r.u * (double)all, 0.0), (double)all), all - 1);
}

// ---- a block a row -------------------------------------------------------------------------------------

// At most 256 tokens, all of them sorted by a single wavefront: no bins. Bound by latency: the sort's dependent steps (64 rows of 65
// tokens 8 us).
constexpr int kShort = 256;
__global__ __launch_bounds__(64) void sample_short(SampleDesc s) {
  constexpr int THREADS = 64, N = kShort / THREADS;
  __shared__ Work<kShort> w;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  const float* x = s.logits + row * s.V;
  float v[N];
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = x[min(e * THREADS + tid, s.V - 1)];
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const int i = e * THREADS + tid;
    w.list[i] = i < s.V ? order_of(key_of(v[e]), i) : kAll;
  }
  const float top = block_top<THREADS>(x, 0, s.V, w);
  if (top == -INFINITY) {
    if (tid == 0) s.token[row] = -1;
    return;
  }
  const Row r = row_of(s, row, top);
  bool ok;
  const u64 bound =
      r.by_count || r.by_mass ? bound_of_list<THREADS, kShort>(r, {0, kBins - 1, 0, 0, false}, s.V, 0, 0, w, ok, [](int, u64) {}) : kAll;
  u64 mine = 0;
#pragma unroll
  for (int e = 0; e < N; ++e) if (e * THREADS + tid < s.V) mine += kept_weight(r, bound, e * THREADS + tid, v[e]);
  choose<THREADS>(r, bound, 0, s.V, goal_of(r, wave_sum(mine)), w, s.token + row);
}

// 1024 threads a row, so that 256 rows fill the card, or 256. Bound by the weights in 64 bits, some 60 instructions of 4 to 8 cycles
// a token, which every token up to a border needs once (256 rows of 50001, 51 MB: no limit 38 us, top-k of 50 34, top_p 0.9 53;
// limits of their own in each row 54, 0.95 TB/s). More than 2048 tokens in the border's bins send a row to bound_by_walks: 256 rows of
// 50001 equal logits 434 us; several blocks a row, 4 rows of 128000 rounded to quarters 312 (28 unrounded), 32 of 200000 as good as
// flat 475.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void sample_one(SampleDesc s) {
  constexpr int W = THREADS / 64;
  __shared__ Bins bins;
  __shared__ Work<kList> w;
  __shared__ u64 stretch[W], total[2];   // what is kept of a wavefront's stretch; mass of all, and before the border's bins
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  clear_bins<THREADS>(bins);
  if (tid == 0) w.listed = 0;
  if (tid < 2) total[tid] = 0;
  const float top = block_top<THREADS>(s.logits + row * s.V, 0, s.V, w);
  if (top == -INFINITY) {
    if (tid == 0) s.token[row] = -1;
    return;
  }
  const Row r = row_of(s, row, top);
  Borders o = kNoBorder;
  if (r.by_count || r.by_mass) {
    fill_bins<THREADS>(r, 0, s.V, bins);
    __syncthreads();
    o = borders<THREADS>(r, bins, w);
  }
  const int each = ((s.V + W - 1) / W + 63) / 64 * 64, from = min(wave * each, s.V), to = min(from + each, s.V);
  u64 bound = kAll;
  bool ok = o.size <= kList;
  if (ok) {
    const Sums mine = list_and_sum(r, o, from, to, [&](u64 x) { w.list[atomicAdd(&w.listed, 1u)] = x; });
    if (lane == 0) {
      stretch[wave] = mine.kept;
      atomicAdd(&total[0], mine.all);
      atomicAdd(&total[1], mine.before);
    }
    __syncthreads();
    if (o.b1 >= o.b0)
      bound = bound_of_list<THREADS, kList>(r, o, (int)w.listed, total[1], total[0], w, ok, [&](int i, u64 m) { atomicAdd(&stretch[i / each], m); });
  }
  if (__builtin_expect(!ok, 0)) {
    bound = bound_by_walks<THREADS>(r, bins, w);
    const u64 mine = stretch_sum(r, bound, from, to);
    __syncthreads();
    if (lane == 0) stretch[wave] = mine;
  }
  __syncthreads();
  u64 all = 0;
#pragma unroll
  for (int k = 0; k < W; ++k) all += stretch[k];
  u64 goal = goal_of(r, all);
  int k = 0;
  while (k < W - 1 && goal >= stretch[k]) goal -= stretch[k++];
  choose<THREADS>(r, bound, min(k * each, s.V), min((k + 1) * each, s.V), goal, w, s.token + row);
}

// ---- several blocks a row ------------------------------------------------------------------------------
//
// Parts of 4096 tokens or more, 1024 threads each: with 256 threads the rows' bins, joined by atomics on whole numbers, took 16 us
// instead of 11. 32 rows of 200000 tokens (25.6 MB), temperature 1.6, top_p 0.95: largest logits 6 us, bins 11, list and weights 20
// (bound by the weights in 64 bits), choice 16 (a sort of some 800 tokens 5, the rest dependent steps). 4 rows of 128000, top-k of 50:
// 3, 4, 8 and 9: latency.

constexpr int kPartThreads = 1024, kPartWaves = kPartThreads / 64, kParts = 256;   // parts: at most
constexpr int kStretches = 4;      // of a part: what is kept is summed for each
struct RowSpace {                  // of a row in the workspace
  Bins bins;
  u64 list[kList];
  u64 listed;
  Borders borders;
};
struct PartArgs {
  SampleDesc s;
  int parts, each;                 // tokens of a part, a multiple of 64 a wavefront
  RowSpace* rows;
  float* tops;                     // [rows][parts]
  Sums* sums;                      // [rows][parts * kStretches]
};
// The row's largest logit; minus infinity: none.
__device__ __forceinline__ float top_of(const PartArgs& a, int64_t row) {
  float top = -INFINITY;
  for (int k = threadIdx.x & 63; k < a.parts; k += 64) top = fmaxf(top, a.tops[row * a.parts + k]);
  return wave_max(top);
}
__global__ __launch_bounds__(kPartThreads) void sample_tops(PartArgs a) {
  __shared__ Work<64> w;
  const int part = blockIdx.x;
  const int64_t row = blockIdx.y;
  const int tid = threadIdx.x, from = part * a.each, to = min(from + a.each, a.s.V);
  const float top = block_top<kPartThreads>(a.s.logits + row * a.s.V, from, to, w);
  if (tid == 0) a.tops[row * a.parts + part] = top;
  RowSpace& sp = a.rows[row];
  for (int i = part * kPartThreads + tid; i < kBins; i += a.parts * kPartThreads) {
    sp.bins.mass[i] = 0;
    sp.bins.count[i] = 0;
  }
  if (part == 0 && tid == 0) sp.listed = 0;
}
__global__ __launch_bounds__(kPartThreads) void sample_bins(PartArgs a) {
  __shared__ Bins bins;
  const int part = blockIdx.x, tid = threadIdx.x, from = part * a.each, to = min(from + a.each, a.s.V);
  const int64_t row = blockIdx.y;
  const float top = top_of(a, row);
  const Row r = row_of(a.s, row, top);
  if (top == -INFINITY || !(r.by_count || r.by_mass)) return;
  clear_bins<kPartThreads>(bins);
  __syncthreads();
  fill_bins<kPartThreads>(r, from, to, bins);
  __syncthreads();
  RowSpace& sp = a.rows[row];
  for (int i = tid; i < kBins; i += kPartThreads)
    if (bins.count[i]) {
      atomicAdd(&sp.bins.count[i], bins.count[i]);
      if (bins.mass[i]) atomicAdd(&sp.bins.mass[i], bins.mass[i]);
    }
}
// Lists the tokens of the border's bins, in LDS first, so that a block takes its places in the row's list at once; sums the others.
__global__ __launch_bounds__(kPartThreads) void sample_list(PartArgs a) {
  __shared__ Work<kList> w;
  __shared__ Sums sums[kPartWaves];
  const int part = blockIdx.x, tid = threadIdx.x, wave = tid >> 6;
  const int64_t row = blockIdx.y;
  const float top = top_of(a, row);
  const Row r = row_of(a.s, row, top);
  if (top == -INFINITY) return;
  RowSpace& sp = a.rows[row];
  if (tid == 0) w.listed = 0;
  Borders o = kNoBorder;
  if (r.by_count || r.by_mass) o = borders<kPartThreads>(r, sp.bins, w);
  if (part == 0 && tid == 0) sp.borders = o;
  if (o.size > kList) return;
  __syncthreads();
  const int each = a.each / kPartWaves, from = min(part * a.each + wave * each, a.s.V), to = min(from + each, a.s.V);
  const Sums mine = list_and_sum(r, o, from, to, [&](u64 x) { w.list[atomicAdd(&w.listed, 1u)] = x; });
  if ((tid & 63) == 0) sums[wave] = mine;
  __syncthreads();
  const int n = (int)w.listed;
  if (tid < kStretches) {
    constexpr int W = kPartWaves / kStretches;
    Sums all = {};
#pragma unroll
    for (int k = 0; k < W; ++k) {
      all.all += sums[tid * W + k].all;
      all.before += sums[tid * W + k].before;
      all.kept += sums[tid * W + k].kept;
    }
    a.sums[(row * a.parts + part) * kStretches + tid] = all;
    if (tid == 0 && n > 0) w.found[0] = atomicAdd(&sp.listed, (u64)n);
  }
  __syncthreads();
  for (int i = tid; i < n; i += kPartThreads) sp.list[w.found[0] + i] = w.list[i];
}
// The bound of what is kept, and the choice, a block a row.
__global__ __launch_bounds__(1024) void sample_choice(PartArgs a) {
  __shared__ Work<kList> w;
  __shared__ Bins bins;
  __shared__ u64 stretch[kParts * kStretches], total[2];
  static_assert(kParts * kStretches == 1024);
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float top = top_of(a, row);
  if (top == -INFINITY) {
    if (tid == 0) a.s.token[row] = -1;
    return;
  }
  const Row r = row_of(a.s, row, top);
  RowSpace& sp = a.rows[row];
  const Borders o = sp.borders;
  const int n = a.parts * kStretches, each = a.each / kStretches;
  u64 bound = kAll;
  bool ok = o.size <= kList;
  if (ok) {
    if (tid < 2) total[tid] = 0;
    for (int i = tid; i < (int)o.size; i += 1024) w.list[i] = sp.list[i];
    __syncthreads();
    const Sums s = tid < n ? a.sums[row * n + tid] : Sums{};
    stretch[tid] = s.kept;
    if (wave * 64 < n) {
      const u64 all = wave_sum(s.all), before = wave_sum(s.before);
      if (lane == 0) {
        atomicAdd(&total[0], all);
        atomicAdd(&total[1], before);
      }
    }
    __syncthreads();
    if (o.b1 >= o.b0)
      bound = bound_of_list<1024, kList>(r, o, (int)o.size, total[1], total[0], w, ok, [&](int i, u64 m) { atomicAdd(&stretch[i / each], m); });
  }
  if (__builtin_expect(!ok, 0)) {
    bound = bound_by_walks<1024>(r, bins, w);
    __syncthreads();
    for (int k = wave; k < n; k += 16) {
      const u64 sum = stretch_sum(r, bound, min(k * each, a.s.V), min((k + 1) * each, a.s.V));
      if (lane == 0) stretch[k] = sum;
    }
  }
  __syncthreads();
  // every wavefront finds the stretch
  u64 all = 0;
  for (int k = lane; k < n; k += 64) all += stretch[k];
  all = wave_sum(all);
  u64 goal = goal_of(r, all), before = 0;
  for (int k0 = 0; k0 < n; k0 += 64) {
    const u64 m = k0 + lane < n ? stretch[k0 + lane] : 0, sum = before + wave_scan(m), passed = __ballot(sum > goal);
    if (passed) {
      const int l = __ffsll(passed) - 1, from = min((k0 + l) * each, a.s.V);
      goal -= lane_value(sum - m, l);
      choose<1024>(r, bound, from, min(from + each, a.s.V), goal, w, a.s.token + row);
      return;
    }
    before = lane_value(sum, 63);
  }
}

struct SamplePlan {
  int parts, each;                 // 1 part: a block a row
  int64_t tops, sums, bytes;
};
SamplePlan sample_plan(const SampleDesc& s) {
  SamplePlan p{};
  p.parts = 1;
  // Several blocks a row where rows alone leave half of the card idle and are long enough for four launches (top_p 0.9: a row of
  // 20000 tokens 24 us, in one block 26; of 9000 24 and 19; 64 rows of 50001 37 and 48, 127 of them 47 and 49).
  if (s.rows <= 128 && s.V > 24576) p.parts = (int)std::min<int64_t>((s.V + 4095) / 4096, std::max<int64_t>(kParts / s.rows, 1));
  p.each = ((s.V + p.parts - 1) / p.parts + kPartThreads - 1) / kPartThreads * kPartThreads;
  p.parts = (s.V + p.each - 1) / p.each;
  if (p.parts > 1) {
    p.tops = s.rows * (int64_t)sizeof(RowSpace);
    p.sums = p.tops + (s.rows * p.parts * 4 + 7) / 8 * 8;
    p.bytes = p.sums + s.rows * p.parts * kStretches * (int64_t)sizeof(Sums);
  }
  return p;
}

}  // namespace

int64_t sample_workspace_bytes(const SampleDesc& s) { return sample_plan(s).bytes; }

void sample(const SampleDesc& s, void* work, hipStream_t st) {
  const SamplePlan p = sample_plan(s);
  const dim3 rows((unsigned)s.rows), grid((unsigned)p.parts, (unsigned)s.rows), block(kPartThreads);
  if (p.parts == 1) {
    // 256 threads where a row is short, or more rows than compute units are not long: top-k of 50 of 512 rows of 4000 tokens 18 us, by
    // 1024 threads 29, of 300 rows of 8000 22 and 28; of 4 rows of 8000 19 and 14, of 512 of 20000 41 and 38
    if (s.V <= kShort) klaunch(sample_short, rows, dim3(64), 0, st, s);
    else if (s.V <= 4096 || (s.rows > 256 && s.V <= 16384)) klaunch(sample_one<256>, rows, dim3(256), 0, st, s);
    else klaunch(sample_one<1024>, rows, dim3(1024), 0, st, s);
    return;
  }
  char* w = (char*)work;
  const PartArgs a{s, p.parts, p.each, (RowSpace*)w, (float*)(w + p.tops), (Sums*)(w + p.sums)};
  const bool limits = s.temperature || s.min_p || s.top_k || s.top_p || !(s.temperature1 > 0) || (s.top_k1 > 0 && s.top_k1 < s.V) ||
                      s.top_p1 < 1;
  klaunch(sample_tops, grid, block, 0, st, a);
  if (limits) klaunch(sample_bins, grid, block, 0, st, a);
  klaunch(sample_list, grid, block, 0, st, a);
  klaunch(sample_choice, rows, dim3(1024), 0, st, a);
}

}  // namespace tgk
