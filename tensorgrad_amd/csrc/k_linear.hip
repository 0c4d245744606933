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
// G: the gradient of the state. y, dq, dk and dv have one form, out_r = sum_s w (row_r.X_s) Z_s + coef_r M row_r, and both states
// another, so there are three kernels: sums over a segment (linear_sums), states from sums (linear_join), results from pairs and
// states (linear_tiles). A few positions are walked one after another (linear_steps). Nothing is added by atomics.
//
// Products run on the f32 matrix instructions: no scales for operands of any size, and the work is bound by memory about as much.
// Fragments of a 16 x 16 x 4 product: lane l holds row (A) or column (B) l % 16 and k = g = l / 16; a result's register q holds row
// 4 g + q of column l % 16. A wavefront's own 16 rows are the columns of every product. A tile of 32 rows lies in LDS in f32: read
// by 16 bytes, four steps of a product over features (k of step q is feature 4 g + q of 16), or by columns, a product over rows
// whose k of step q is row 4 g + q, which is where the weights stand as they come out of the first product.
//
// What a row does not see has weight 0, and 0 times an infinity or NaN is NaN; a dot product may be infinite where no state is: rows
// whose result is not finite are computed again pair by pair in 64 bits, from what they see alone. So are rows of which weights below
// f32's range, 2^-126, may lose something that counts: under a decay whose weights in a segment fall below 2^-100, where 2^-126 times
// the largest products that a block's operands allow is above 2^-60 and above 2^-30 of a result of theirs.
#include <algorithm>
#include <cmath>

#include "kernels.h"
#include "lds_dev.h"
#include "sequence.h"

namespace tgk {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kSeg = kLinearSegment;   // positions of a segment
constexpr int kTile = 32;          // rows of a tile in LDS
constexpr int kNever = INT32_MAX;

__device__ __forceinline__ f32x4 mfma(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
__device__ __forceinline__ float power(float rate, int n) { return __builtin_amdgcn_exp2f(rate * (float)n); }
__device__ __forceinline__ float scalar(float x) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(x))); }

struct Marks {
  const int32_t *documents, *lengths;
  int T;
};
__device__ __forceinline__ int count_of(const Marks& m, int b) { return m.lengths ? min(max(m.lengths[b], 0), m.T) : m.T; }

// since[t - s0] for the positions of the segment at s0: the first one, in the segment, of the document they belong to; -1 where
// that began before (or the state that came in counts); kNever for positions that are not there. Ends at a barrier.
__device__ __forceinline__ void mark(const Marks& m, int b, int s0, int n, int* since) {
  const int tid = threadIdx.x;
  if (!m.documents) {
    for (int i = tid; i < kSeg; i += blockDim.x) since[i] = s0 + i < n ? -1 : kNever;
  } else if (tid < 64) {
    const int32_t* doc = m.documents + (int64_t)b * m.T;
    int before = -1;
    for (int i = tid; i < kSeg; i += 64) {
      const int t = s0 + i;
      const bool here = t < n;
      const int id = here ? doc[t] : -1;
      int first = here && t > 0 && doc[t - 1] != id ? t : -1;
#pragma unroll
      for (int o = 1; o < 64; o *= 2) {
        const int z = __shfl_up(first, o);
        if (tid >= o) first = max(first, z);
      }
      first = max(first, before);
      before = __shfl(first, 63);
      since[i] = here && id >= 0 ? first : kNever;
    }
  }
  __syncthreads();
}
// The segment's last position that is there; and how often the decay applies, none (-1) where the weight is 0 by a mask: to what a
// position leaves of itself there, to what came in at a position, and to what is left of it at the end.
struct Ends {
  int last, since;                 // last < s0: none
};
__device__ __forceinline__ Ends ends(const int* since, int s0, int n) {
  const int last = min(s0 + kSeg, n) - 1;
  return {last, last >= s0 ? since[last - s0] : kNever};
}
__device__ __forceinline__ int leaves(const Ends& e, const int* since, int s0, int j) {
  return j <= e.last && since[j - s0] != kNever && j >= e.since ? e.last - j : -1;
}
__device__ __forceinline__ int comes(const int* since, int s0, int i) { return since[i - s0] == -1 ? i - s0 + 1 : -1; }
__device__ __forceinline__ int stays(const Ends& e, int s0) { return e.last < s0 ? 0 : e.since == -1 ? e.last - s0 + 1 : -1; }

// 2^(rate n) as a product, so that a state counts where its weight alone is below f32's range: down to 2^-226 together, and exactly
// `near` down to 2^-100. A negative `near` stands for a weight that a mask makes 0.
struct Weight {
  float near, far;
};
__device__ __forceinline__ Weight weight_of(float rate, int n) {
  const float e = rate * (float)n;
  return n < 0 ? Weight{-1.0f, 0.0f} : Weight{__builtin_amdgcn_exp2f(fmaxf(e, -100.0f)), __builtin_amdgcn_exp2f(fminf(e + 100.0f, 0.0f))};
}
// The same as a factor above 1 / 2 and a power of 2, by which a state is multiplied: no decay above 0 forgets an infinity or NaN.
struct Decay {
  float factor;
  int shift;
};
__device__ __forceinline__ Decay decay_of(float e) {   // of 2^e
  const float whole = ceilf(e);
  return {__builtin_amdgcn_exp2f(e - whole), (int)whole};
}
__device__ __forceinline__ bool is_number(float x) { return fabsf(x) < INFINITY; }
// Weights of 64 bits, for what is computed again: no operand or product of f32 values leaves their range, and an infinity times one of
// them stays.
__device__ __forceinline__ double power64(float rate, int n) {
  const double e = (double)rate * n, k = floor(e);
  return __builtin_amdgcn_ldexp((double)__builtin_amdgcn_exp2f((float)(e - k)), max((int)k, -1000));
}

// ---- tiles in LDS --------------------------------------------------------------------------------------
//
// A row has PITCH floats, in pieces of 16 bytes; piece c of row r lies at place c ^ swizzle(r), so that 16 rows' same piece, and 4
// rows' 4 pieces, lie in different banks.

template <int DP>
struct Tile {
  static constexpr int PITCH = DP == 96 ? 128 : DP, PIECES = PITCH / 4, FLOATS = kTile * PITCH;
  static __device__ __forceinline__ int swizzle(int r) { return DP == 32 ? (r >> 1) & 7 : r & 15; }
  static __device__ __forceinline__ int place(int r, int piece) { return r * PITCH + 4 * (piece ^ swizzle(r)); }
  // Fragments. An opaque lane keeps the compiler from holding every place's address through a loop over tiles (142 registers
  // instead of 121 for 128 features); where pieces are told apart by 4 c ^ .., what c's upper bits add is a constant of the instruction.
  static __device__ __forceinline__ int opaque(int lane) {
    asm volatile("" : "+v"(lane));
    return lane;
  }
  // at[c % 4] + far(c): piece 4 c + g of row l
  static __device__ __forceinline__ void by_piece(int (&at)[4], int lane) {
    const int l = lane & 15, g = lane >> 4;
#pragma unroll
    for (int c = 0; c < 4; ++c) at[c] = place(l, (4 * c + g) % PIECES);
  }
  // row[q] + column[c % 4] + far(c): feature 16 c + l of row 4 g + q
  static __device__ __forceinline__ void by_column(int (&row)[4], int (&column)[4], int lane) {
    static_assert(DP > 32);
    const int l = lane & 15, g = lane >> 4;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      row[q] = (4 * g + q) * PITCH + 4 * ((l >> 2) ^ q) + (l & 3);
      column[q] = 16 * (q ^ g);
    }
  }
  static __device__ __forceinline__ constexpr int far(int c) { return c / 4 * 64; }
};

// Rows [r0, r0 + 32) of x from memory straight into LDS, by WAVES wavefronts: 16 bytes a lane, or (not WIDE: rows that are not whole
// 16-byte pieces) 4, with addresses of 64 bits. Nothing is masked: rows past the last and features past the n-th are others that are
// there. The kernels wait (vmcnt) and meet (barrier) themselves.
template <int DP, int WAVES, bool WIDE>
__device__ __forceinline__ void tile_to_lds(const float* x, int64_t stride, int r0, int rows, int n, uint32_t lds, int w) {
  constexpr int PIECES = Tile<DP>::PIECES, PITCH = Tile<DP>::PITCH, N = kTile * PITCH / (WIDE ? 256 : 64);
  const int lane = Tile<DP>::opaque(threadIdx.x & 63), left = rows - 1 - r0;
  const float* base = x + (int64_t)r0 * stride;
#pragma unroll
  for (int i = 0; i < (N + WAVES - 1) / WAVES; ++i) {
    const int k = w + i * WAVES;
    if (N % WAVES && k >= N) break;
    if constexpr (WIDE) {
      const int r = k * (64 / PIECES) + lane / PIECES, c = (lane % PIECES) ^ Tile<DP>::swizzle(r);
      const uint32_t off = (uint32_t)min(r, left) * (uint32_t)(4 * stride) + (4 * c < n ? 16 * c : 0);
      load16_to_lds(base, off, lds + k * 1024);
    } else {
      const int e = k * 64 + lane, r = e / PITCH, c = (e % PITCH / 4) ^ Tile<DP>::swizzle(r);
      const float* at = base + min(r, left) * stride + min(4 * c + e % 4, n - 1);
      load4_to_lds(at, lds + k * 256);
    }
  }
}

// ---- sums over a segment -----------------------------------------------------------------------------
//
// A block sums k v^T of a segment, four wavefronts a quarter of the product each, over tiles of 32 positions of which the next one
// is on its way. Bound by memory: 64 heads of 4096 positions, 128 x 128 features, read 268 MB and write 134 MB of states in 115 us
// (3.5 TB/s). Segments of 128: a state of 128 features then weighs as much as a segment's keys do; in longer ones the states'
// bytes fall and the pairs, bound by the matrix instructions, rise.

struct SumsArgs {
  Marks m;
  Rows x, y;                       // x: k or q, y: v or dy
  int H, share, segs, n, ny;       // query heads, those that share a row of x and y (1: none); features
  bool back;                       // back: of q and dy, weights c, else of k and v, weights e
  float scale;
  const float* rate;
  float* sums;                     // [segs][B * H][n][ny]
  float* stay;                     // [segs][B * H]: log2 of what stays of the state that came in; 1: nothing
};
template <int DX, int DY, bool WIDE>
__global__ __launch_bounds__(256) void linear_sums(SumsArgs A) {
  using LX = Tile<DX>;
  using LY = Tile<DY>;
  constexpr int BX = DX / 32, BY = DY / 32;   // a wavefront takes a quarter of the sums
  __shared__ __align__(16) float xs[2][LX::FLOATS], ys[2][LY::FLOATS];
  __shared__ int since[kSeg];
  __shared__ Weight weight[kSeg];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, l = lane & 15;
  const int seg = blockIdx.x % A.segs, bh = blockIdx.x / A.segs, b = bh / A.H, h = bh % A.H, s0 = seg * kSeg;
  const int n = count_of(A.m, b);
  const float* x = A.x.p + b * A.x.b + (h / A.share) * A.x.h;
  const float* y = A.y.p + b * A.y.b + (h / A.share) * A.y.h;
  const int stop = A.y.p ? min(s0 + kSeg, n) : s0;
  auto fetch = [&](int t0, int buf) {
    tile_to_lds<DX, 4, WIDE>(x, A.x.t, t0, A.m.T, A.n, lds_address(xs[buf]), w);
    tile_to_lds<DY, 4, WIDE>(y, A.y.t, t0, A.m.T, A.ny, lds_address(ys[buf]), w);
  };
  const float rate = scalar(A.rate[h]);
  mark(A.m, b, s0, n, since);
  const Ends e = ends(since, s0, n);
  if (s0 < stop) fetch(s0, 0);
  auto times = [&](int t) { return A.back ? comes(since, s0, t) : leaves(e, since, s0, t); };
  if (tid < kSeg) {
    Weight c = weight_of(rate, s0 + tid > e.last ? -1 : times(s0 + tid));
    if (A.back && c.near > 0) (c.near * A.scale >= 0x1p-110f ? c.near : c.far) *= A.scale;   // where it keeps both in range
    weight[tid] = c;
  }
  const int dx = (w >> 1) * BX, dy = (w & 1) * BY;
  f32x4 acc[BX][BY];
#pragma unroll
  for (int i = 0; i < BX; ++i)
#pragma unroll
    for (int j = 0; j < BY; ++j) acc[i][j] = f32x4{};
  // `far` is not 1 only where the decay is fast or the scale small; the loop with it takes 3 % longer
  auto walk = [&](auto far) {
    constexpr bool FAR = far.value;
    for (int t0 = s0, buf = 0; t0 < stop; t0 += kTile, buf ^= 1) {
      loads_done();
      __syncthreads();
      if (t0 + kTile < stop) fetch(t0 + kTile, buf ^ 1);
      const float *X = xs[buf], *Y = ys[buf];
      float u[2][BX], v[2][BY];
      auto read = [&](int k) {       // positions t0 + 4 k + g, ahead of their use by one step; 0 where masked, whatever they hold
        const int r = 4 * k + g;
        const Weight c = weight[t0 - s0 + r];
#pragma unroll
        for (int i = 0; i < BX; ++i) {
          const float a = X[LX::place(r, 4 * (dx + i) + l / 4) + l % 4];
          u[k & 1][i] = c.near < 0 ? 0.0f : a * c.near;
        }
#pragma unroll
        for (int j = 0; j < BY; ++j) {
          const float z = Y[LY::place(r, 4 * (dy + j) + l / 4) + l % 4];
          v[k & 1][j] = c.near < 0 ? 0.0f : FAR ? z * c.far : z;
        }
      };
      read(0);
#pragma unroll
      for (int k = 0; k < kTile / 4; ++k) {
        if (k + 1 < kTile / 4) read(k + 1);
#pragma unroll
        for (int i = 0; i < BX; ++i)
#pragma unroll
          for (int j = 0; j < BY; ++j) acc[i][j] = mfma(u[k & 1][i], v[k & 1][j], acc[i][j]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  if (rate * kSeg < -100.0f || (A.back && A.scale < 0x1p-10f)) walk(std::true_type());
  else walk(std::false_type());
  const int64_t at = (int64_t)seg * (gridDim.x / A.segs) + bh;
  float* out = A.sums + at * A.n * A.ny;
  float bad = 0;                   // NaN for infinities and NaN
#pragma unroll
  for (int i = 0; i < BX; ++i)
#pragma unroll
    for (int j = 0; j < BY; ++j) {
      const int d = 16 * (dx + i) + 4 * g, c = 16 * (dy + j) + l;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        bad = fmaf(acc[i][j][q], 0.0f, bad);
        if (d + q < A.n && c < A.ny) out[(d + q) * A.ny + c] = acc[i][j][q];
      }
    }
  if (tid == 0) A.stay[at] = stays(e, s0) < 0 ? 1.0f : rate * (float)stays(e, s0);
  if (__builtin_expect(!__any(bad != bad), 1)) return;
  // again in 64 bits, a lane its own entries: an infinity times a weight that is 0 in 32 bits is an infinity
  loads_done();                    // they are written before they are written again
#pragma unroll 1
  for (int i = 0; i < 4 * BX * BY; ++i) {
    const int d = 16 * (dx + i / (4 * BY)) + 4 * g + i % 4, c = 16 * (dy + i / 4 % BY) + l;
    if (d >= A.n || c >= A.ny) continue;
    double sum = 0;
#pragma unroll 1
    for (int t = s0; t < min(stop, e.last + 1); ++t)
      if (times(t) >= 0) sum += (double)x[(int64_t)t * A.x.t + d] * y[(int64_t)t * A.y.t + c] * power64(rate, times(t));
    out[d * A.ny + c] = (float)(A.back ? sum * A.scale : sum);
  }
}

// ---- states at the segments' borders -------------------------------------------------------------------

struct JoinArgs {
  float* sums;                     // [segs][rows][each]: replaced by the state that comes in (back: goes out)
  const float* stay;               // [segs][rows]
  const float* first;              // [rows][each] or null
  float* last;                     // or null
  int segs;
  int64_t rows, each;
  bool back;
};
// A thread walks one value of a state through all segments. Bound by memory (the same 134 MB read and written: 42 us, 6.4 TB/s, out
// of the last-level cache).
__global__ __launch_bounds__(256) void linear_join(JoinArgs A) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, all = A.rows * A.each;
  if (id >= all) return;
  const int64_t row = id / A.each;
  float s = A.first ? A.first[id] : 0.0f;
#pragma unroll 4
  for (int i = 0; i < A.segs; ++i) {
    const int64_t seg = A.back ? A.segs - 1 - i : i;
    float* at = A.sums + seg * all + id;
    const float add = *at;
    const float e = A.stay[seg * A.rows + row];
    const Decay f = decay_of(e);
    *at = s;
    s = e > 0 ? add : fmaf(f.factor, __builtin_amdgcn_ldexpf(s, f.shift), add);
  }
  if (A.last) A.last[id] = s;
}

// ---- results from pairs and states -----------------------------------------------------------------------

// One sum of the form above.
struct Sum {
  Rows rows, out, x, z;            // rows, x and z may be absent (null): zeros, no pairs
  int n, nz;                       // features of rows and x; of out and z
  bool across;                     // M's rows are out's features, else rows' features
};
struct PairsArgs {
  Marks m;
  Sum sum[2];
  int sums, B, H, segs, blocks;    // blocks: of a head
  int heads, group, share;         // heads of `out`; back: those of x and z that a row meets in turn; else rows' heads that share one of x
  int keys;                        // heads of `out` that share one of `rows`
  const float *states, *edge;      // [segs][B * H][D][Dv]; at the first segment (back: last) this one, or null
  int D, Dv;
  float by_pair, by_state;         // factors of both parts
  float fast, large;               // a decay's log2 below which operands are looked at; the size below which they lose nothing that counts
  const float *rate, *any;         // any: an address with a feature (wide: 4), for rows that are absent
};
__device__ __forceinline__ const float* row_at(const Rows& x, int b, int head, int t) { return x.p + b * x.b + head * x.h + (int64_t)t * x.t; }

// What one block computes: rows [r0, ..) of a head.
struct Place {
  int b, head, r0, seg, s0, n;     // n: positions that are there
  int h0, group;                   // the first head of x and z, and how many
  const float* M;                  // state of h0, or null
  int from, to;                    // positions of x and z
};
template <bool BACK>
__device__ __forceinline__ Place place_of(const PairsArgs& p, const Sum& s, int unit, int rows) {
  Place o;
  const int blk = unit % p.blocks, bh = unit / p.blocks;
  o.b = bh / p.heads;
  o.head = bh % p.heads;
  o.r0 = blk * rows;
  o.seg = o.r0 / kSeg;
  o.s0 = o.seg * kSeg;
  o.n = count_of(p.m, o.b);
  o.h0 = BACK ? o.head * p.group : o.head;
  o.group = BACK ? p.group : 1;
  const bool border = BACK ? o.seg == p.segs - 1 : o.seg == 0;
  const int64_t each = (int64_t)p.D * p.Dv;
  o.M = border ? p.edge : p.states + (int64_t)o.seg * p.B * p.H * each;
  if (o.M) o.M += ((int64_t)o.b * p.H + o.h0) * each;
  o.from = BACK ? o.r0 : o.s0;
  o.to = s.x.p && s.z.p ? min(BACK ? o.s0 + kSeg : o.r0 + rows, o.n) : 0;
  return o;
}

// A wavefront's rows [w0, w0 + 16) pair by pair in 64 bits, a lane a pair or one or two features of the result. What is not finite goes
// where the states would carry it: a pair's X_e Z_d is a term of the state's entry (e, d), which row_e then multiplies. A row's own
// infinities therefore meet whole entries; other features are taken through dot products.
template <bool BACK>
__device__ __forceinline__ void plain_rows(const PairsArgs& p, const Sum& s, const Place& o, int w0, const int* since) {
  const int lane = threadIdx.x & 63;
#pragma unroll 1
  for (int r = w0; r < min(w0 + 16, p.m.T); ++r) {
    const int mine = since[r - o.s0];
    if (mine == kNever || !s.rows.p) continue;
    const float* row = row_at(s.rows, o.b, o.head / p.keys, r);
    auto seen = [&](int t) {
      const int from = since[t - o.s0], i = BACK ? t : r, j = BACK ? r : t;
      return from != kNever && j <= i && j >= (BACK ? from : mine);
    };
    const int by = BACK ? leaves(ends(since, o.s0, o.n), since, o.s0, r) : comes(since, o.s0, r);
    const bool some = (o.M && by >= 0) || o.from < o.to;   // else it sees nothing at all
    double acc[2] = {0, 0};
    bool nan = false;              // then every feature is
#pragma unroll 1
    for (int e = 0; e < s.n; ++e) nan |= some && row[e] != row[e];
#pragma unroll 1
    for (int gi = 0; gi < (some && !nan ? o.group : 0); ++gi) {
      const int h = o.h0 + gi, hx = BACK ? h : h / p.share;
      const float rate = p.rate[h];
      const double coef = by < 0 ? 0.0 : p.by_state * power64(rate, by);
      const float* M = o.M && by >= 0 ? o.M + (int64_t)gi * p.D * p.Dv : nullptr;
      auto state = [&](int e, int d) { return M ? coef * (s.across ? M[d * p.Dv + e] : M[e * p.Dv + d]) : 0.0; };
      auto weight = [&](int t) { return power64(rate, BACK ? t - r : r - t) * p.by_pair; };
#pragma unroll 1
      for (int e = 0; e < s.n; ++e)
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          const int d = 64 * a + lane;
          if (d >= s.nz) continue;
          double entry = state(e, d);
          if (!is_number(row[e]))
#pragma unroll 1
            for (int t = o.from; t < o.to; ++t)
              if (seen(t)) entry += weight(t) * row_at(s.x, o.b, hx, t)[e] * row_at(s.z, o.b, hx, t)[d];
          acc[a] += row[e] * entry;
        }
#pragma unroll 1
      for (int c = o.from; c < o.to; c += 64) {
        const int t = c + lane;
        const bool in = t < o.to && seen(t);
        double f = 0;
        if (in) {
          const float* x = row_at(s.x, o.b, hx, t);
#pragma unroll 1
          for (int e = 0; e < s.n; ++e) if (is_number(row[e])) f += (double)x[e] * row[e];
          f *= weight(t);
        }
        uint64_t left = __ballot(in);
#pragma unroll 1
        while (left) {
          const int z = __ffsll((unsigned long long)left) - 1;
          left &= left - 1;
          const double w = __shfl(f, z);
          const float *X = row_at(s.x, o.b, hx, c + z), *Z = row_at(s.z, o.b, hx, c + z);
#pragma unroll
          for (int a = 0; a < 2; ++a) {
            if (64 * a + lane >= s.nz) continue;
            const float u = Z[64 * a + lane];
            if (is_number(u)) acc[a] += w * u;
            else
#pragma unroll 1
              for (int e = 0; e < s.n; ++e) if (is_number(row[e])) acc[a] += (double)X[e] * row[e] * u;
          }
        }
      }
    }
    float* out = s.out.p + o.b * s.out.b + o.head * s.out.h + (int64_t)r * s.out.t;
#pragma unroll
    for (int a = 0; a < 2; ++a) if (64 * a + lane < s.nz) out[64 * a + lane] = nan ? NAN : (float)acc[a];
  }
}

// A wavefront's 16 rows: B fragments, and results. A fragment is read one step ahead of its use.
template <int DN, int DZ, bool WIDE>   // features, padded: of the rows, of the results
struct Own {
  using LN = Tile<DN>;
  using LZ = Tile<DZ>;
  static constexpr int CN = DN / 16, CZ = DZ / 16;
  float row[CN][4];
  f32x4 acc[CZ];
  __device__ __forceinline__ void load(const float* at, int n, int g) {
#pragma unroll
    for (int c = 0; c < CN; ++c) {
      const int d = 16 * c + 4 * g;
      if (WIDE) {
        const f32x4 u = *(const f32x4*)(at + (d < n ? d : 0));
#pragma unroll
        for (int q = 0; q < 4; ++q) row[c][q] = u[q];
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) row[c][q] = at[min(d + q, n - 1)];
      }
    }
  }
  // Zero for rows that are not there and past the features. Waits for the rows here: left to the compiler, the wait stands in the
  // loop over tiles, and there it waits for the next tiles too.
  __device__ __forceinline__ void start(bool here, int n, int g) {
#pragma unroll
    for (int c = 0; c < CN; ++c)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        row[c][q] = here && 16 * c + 4 * g + (WIDE ? 0 : q) < n ? row[c][q] : 0.0f;
        asm volatile("" : "+v"(row[c][q]));
      }
#pragma unroll
    for (int c = 0; c < CZ; ++c) acc[c] = f32x4{};
  }
  // Of a lane's part of a row's features, and of its results.
  __device__ __forceinline__ float largest() const {
    float top = 0;
#pragma unroll
    for (int c = 0; c < CN; ++c)
#pragma unroll
      for (int q = 0; q < 4; ++q) top = fmaxf(top, fabsf(row[c][q]));
    return top;
  }
  __device__ __forceinline__ float smallest(int n, int g) const {
    float least = INFINITY;
#pragma unroll
    for (int c = 0; c < CZ; ++c)
#pragma unroll
      for (int q = 0; q < 4; ++q) if (16 * c + 4 * g + q < n) least = fminf(least, fabsf(acc[c][q]));
    return least;
  }
  // tile rows times own rows: x[q] of tile row 16 (q / 4) + 4 g + q % 4
  __device__ __forceinline__ void dots(const float* tile, float (&x)[8], int g, int l) const {
    f32x4 s[2] = {}, u[2];
    int at[4];
    LN::by_piece(at, LN::opaque(16 * g + l));
    auto read = [&](int i) { u[i & 1] = *(const f32x4*)(tile + at[i / 2 % 4] + (16 * (i & 1) * LN::PITCH + LN::far(i / 2))); };
    read(0);
#pragma unroll
    for (int i = 0; i < 2 * CN; ++i) {
      if (i + 1 < 2 * CN) read(i + 1);
#pragma unroll
      for (int q = 0; q < 4; ++q) s[i & 1] = mfma(u[i & 1][q], row[i / 2][q], s[i & 1]);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) x[q] = s[q / 4][q % 4];
  }
  // acc += weights x on the tile's rows
  __device__ __forceinline__ void add(const float* tile, const float (&x)[8], int g, int l) {
    constexpr int PART = CZ % 4 == 0 ? 4 : CZ % 3 == 0 ? 3 : CZ, PARTS = CZ / PART;   // MFMAs a step
    float u[2][PART];
    int row_[4], column[4];
    if constexpr (DZ > 32) LZ::by_column(row_, column, LZ::opaque(16 * g + l));
    auto read = [&](int step) {
      const int i = step / PARTS;
#pragma unroll
      for (int e = 0; e < PART; ++e) {
        const int c = step % PARTS * PART + e;
        if constexpr (DZ > 32) u[step & 1][e] = tile[row_[i % 4] + column[c % 4] + (16 * (i / 4) * LZ::PITCH + LZ::far(c))];
        else u[step & 1][e] = tile[16 * (i / 4) * LZ::PITCH + LZ::place(4 * g + i % 4, 4 * c + l / 4) + l % 4];
      }
    };
    read(0);
#pragma unroll
    for (int step = 0; step < 8 * PARTS; ++step) {
      if (step + 1 < 8 * PARTS) read(step + 1);
#pragma unroll
      for (int e = 0; e < PART; ++e) {
        const int c = step % PARTS * PART + e;
        acc[c] = mfma(u[step & 1][e], x[step / PARTS], acc[c]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  // acc += what the rows [32 c, 32 c + 32) of M in the tile give: ACROSS, these features of the result, else these features' weights
  template <bool ACROSS>
  __device__ __forceinline__ void state(const float* tile, int c, float coef, int g, int l) {
    float x[8];
    if constexpr (ACROSS) {
      dots(tile, x, g, l);
#pragma unroll
      for (int q = 0; q < 8; ++q) acc[2 * c + q / 4][q % 4] = fmaf(coef, x[q], acc[2 * c + q / 4][q % 4]);
    } else {
#pragma unroll
      for (int q = 0; q < 8; ++q) x[q] = row[2 * c + q / 4][q % 4] * coef;
      add(tile, x, g, l);
    }
  }
  // Stores the rows; whether they are all finite.
  __device__ __forceinline__ bool store(float* out, bool in, bool here, int n, int g) const {
    float bad = 0;                 // NaN for infinities and NaN
#pragma unroll
    for (int c = 0; c < CZ; ++c) {
      const int d = 16 * c + 4 * g;
#pragma unroll
      for (int q = 0; q < 4; ++q) bad = fmaf(acc[c][q], 0.0f, bad);
      const f32x4 u = here ? acc[c] : f32x4{};
      if (!in) continue;
      if (WIDE) {
        if (d < n) *(f32x4*)(out + d) = u;
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) if (d + q < n) out[d + q] = u[q];
      }
    }
    return !__any(bad != bad);
  }
};
// Weights of the pairs of row r and tile rows t0 + 16 (q / 4) + 4 g + q % 4, -1 where masked; mine: r's mark.
template <bool BACK>
__device__ __forceinline__ void weights(float (&x)[8], const PairsArgs& p, const Place& o, float rate, int w0, int r, int t0, int mine,
                                        const int* since, int g) {
  const int far = BACK ? t0 + 4 * g - r : r - t0 - 4 * g;
#pragma unroll
  for (int q = 0; q < 8; ++q) x[q] = power(rate, BACK ? far + 16 * (q / 4) + q % 4 : far - 16 * (q / 4) - q % 4) * p.by_pair;
  // all pairs count where there are no documents and the tile is on one side of the rows
  if (p.m.documents || (BACK ? t0 < w0 + 15 || t0 + kTile > o.n : t0 + kTile - 1 > w0) || w0 + 16 > o.n) {
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int t = t0 + 16 * (q / 4) + 4 * g + q % 4, i = BACK ? t : r, j = BACK ? r : t;
      const int from = since[t - o.s0];
      const bool seen = (from != kNever) & (j <= i) & (j >= (BACK ? from : mine));
      x[q] = seen ? x[q] : -1.0f;
    }
  }
}

// W wavefronts of 16 rows. Bound by the f32 matrix instructions: 64 heads of 4096 positions, 128 x 128 features, keep them busy for
// 66 % of the cycles (y or dq 217 us, dk and dv 427; 19 GFLOP a result with the masked halves of tiles); what is lost is wavefronts
// of early rows, which wait for the tiles of late ones. LDS has no conflicts. The tiles of M, then those of the pairs, one after
// another; the next one travels to the other half of LDS while this one is multiplied, so that a tile costs one barrier. A wavefront
// walks the tiles that it has nothing to do with in loops of their own: with a branch around the work the compiler copied all 32
// registers of results for every tile, and had none left for a second block on the CU.
template <int DA, int DB>
struct Ring {
  float tile[2][Tile<DA>::FLOATS + Tile<DB>::FLOATS];
};
// Where a wavefront has a size from `large` on: the larger of `most` (a size's bits, in LDS) and its sizes.
__device__ __forceinline__ void join_max(uint32_t& most, float size, float large) {
  if (!__any(size >= large)) return;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) size = fmaxf(size, __shfl_xor(size, o));
  if ((threadIdx.x & 63) == 0) atomicMax(&most, __float_as_uint(size));
}
template <int DN, int DZ, int W, bool BACK, bool WIDE, bool LOOK, bool ACROSS>
__device__ __forceinline__ void walk_tiles(const PairsArgs& p, const Sum& s, int unit, float* ring, int (&since)[kSeg], uint32_t (&most)[2]) {
  constexpr int FZ = Tile<DZ>::FLOATS, HALF = FZ + Tile<DN>::FLOATS, FM = ACROSS ? FZ : 0;   // M's tile: as wide as its rows are
  const Place o = place_of<BACK>(p, s, unit, 16 * W);
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, l = lane & 15;
  const int T = p.m.T, w0 = o.r0 + 16 * w, r = w0 + l;
  const int mtiles = o.M ? (p.D + kTile - 1) / kTile : 0, count = mtiles + (o.from < o.to ? (o.to - o.from + kTile - 1) / kTile : 0);
  const int hx = BACK ? o.h0 : o.h0 / p.share;
  const float *M = o.M, *X = row_at(s.x, o.b, hx, 0), *Z = row_at(s.z, o.b, hx, 0);
  const uint32_t base = lds_address(ring);
  int left = count * o.group, next = 0, into = 0;   // tiles to fetch; the next one of its head (of M, then of pairs), and where to
  auto fetch = [&]() {
    if (left == 0) return;
    --left;
    const uint32_t to = base + into * (4 * HALF);
    if (next < mtiles) {
      tile_to_lds<ACROSS ? DN : DZ, W, WIDE>(M, p.Dv, next * kTile, p.D, p.Dv, to + 4 * FM, w);
    } else {
      const int t0 = o.from + (next - mtiles) * kTile;
      tile_to_lds<DZ, W, WIDE>(Z, s.z.t, t0, T, s.nz, to, w);
      tile_to_lds<DN, W, WIDE>(X, s.x.t, t0, T, s.n, to + 4 * FZ, w);
    }
    into ^= 1;
    if (++next == count) {
      next = 0;
      if (BACK) {
        M += (int64_t)p.D * p.Dv;
        X += s.x.h;
        Z += s.z.h;
      }
    }
  };
  fetch();
  Own<DN, DZ, WIDE> own;
  own.load(s.rows.p ? row_at(s.rows, o.b, o.head / p.keys, min(r, T - 1)) : p.any, s.rows.p ? s.n : 1, g);
  if (LOOK && tid < 2) most[tid] = 0;
  mark(p.m, o.b, o.s0, o.n, since);
  const Ends end = ends(since, o.s0, o.n);
  const int mine = r < T ? since[r - o.s0] : kNever;
  const bool here = mine != kNever;
  own.start(here && s.rows.p, s.n, g);
  if (LOOK) join_max(most[1], own.largest(), p.large);
  int buf = 1;
  bool fast = false, looked = false;   // LOOK: this head's decay is, one was
  float top = 0;                   // the largest operand under a fast decay, a thread a share of each tile
  auto arrive = [&](int from, int to) {   // the next tile is there, [from, to) of `buf`, and the one after it on its way
    loads_done();
    __syncthreads();
    fetch();
    buf ^= 1;
    if (!LOOK || !fast) return;
#pragma unroll 2
    for (int i = from + 4 * tid; i < to; i += 256 * W) {
      const f32x4 u = *(const f32x4*)(ring + buf * HALF + i);
      top = fmaxf(top, fmaxf(fmaxf(fabsf(u[0]), fabsf(u[1])), fmaxf(fabsf(u[2]), fabsf(u[3]))));
    }
  };
  for (int gi = 0; gi < o.group; ++gi) {
    const float rate = scalar(p.rate[o.h0 + gi]);
    if (LOOK) {
      fast = rate < p.fast;
      looked |= fast;
    }
    const int by = here ? BACK ? leaves(end, since, o.s0, r) : comes(since, o.s0, r) : -1;
    const float coef = by < 0 ? 0.0f : p.by_state * power(rate, by);
#pragma unroll
    for (int c = 0; c < (ACROSS ? DZ : DN) / 32; ++c)
      if (c < mtiles) {
        arrive(FM, FM + (ACROSS ? Tile<DN>::FLOATS : FZ));
        own.template state<ACROSS>(ring + buf * HALF + FM, c, coef, g, l);
      }
    int t0 = o.from;
    if (BACK)
      for (; t0 < min(o.to, w0 - kTile + 1); t0 += kTile) arrive(0, HALF);
    for (const int stop = BACK ? o.to : min(o.to, w0 + 16); t0 < stop; t0 += kTile) {
      arrive(0, HALF);
      float x[8], f[8];
      own.dots(ring + buf * HALF + FZ, x, g, l);
      __builtin_amdgcn_sched_barrier(0);
      weights<BACK>(f, p, o, rate, w0, r, t0, mine, since, g);
#pragma unroll
      for (int q = 0; q < 8; ++q) x[q] = f[q] < 0 ? 0.0f : x[q] * f[q];
      __builtin_amdgcn_sched_barrier(0);
      own.add(ring + buf * HALF, x, g, l);
    }
    for (; t0 < o.to; t0 += kTile) arrive(0, HALF);
  }
  bool lossy = false;
  if (looked) {
    join_max(most[0], top, p.large);
    __syncthreads();
    if (__builtin_expect((most[0] | most[1]) != 0, 0)) {
      // of 128 pairs: a dot product times two more operands at most (the state's products are fewer and have one)
      const double row = fmaxf(p.large, __uint_as_float(most[1])), x = fmaxf(fmaxf(p.large, 1.0f), __uint_as_float(most[0]));
      const double lost = 0x1p-126 * kSeg * fmax(s.n * row, 1.0) * x * x * fmaxf(1.0f, p.by_pair);
      lossy = __any(lost > 0x1p-60 && own.smallest(s.nz, g) < lost * 0x1p30);
    }
  }
  const bool fine = own.store(s.out.p + o.b * s.out.b + o.head * s.out.h + (int64_t)r * s.out.t, r < T, here && s.rows.p, s.nz, g);
  if (__builtin_expect(!fine || lossy, 0)) {
    loads_done();                  // the rows are written before they are written again
    plain_rows<BACK>(p, s, o, w0, since);
  }
}
// Features of keys and of values, padded. LOOK: a head's decay is fast (kernels of their own: the look in all of them took 2 to 5 % of
// layers of 32 and 64 features without fast decays).
template <int DK, int DV, int W, bool BACK, bool WIDE, bool LOOK>
__global__ __launch_bounds__(64 * W, W == 8 || DK + DV <= 128 ? 4 : 2) void linear_tiles(PairsArgs p) {
  __shared__ __align__(16) Ring<DK, DV> ring;
  __shared__ int since[kSeg];
  __shared__ uint32_t most[2];     // sizes of tiles' and of rows' operands
  // both sums of a place run one after the other on one XCD (blocks go to the 8 XCDs in turn), whose L2 then has their tiles
  const int id = blockIdx.x / 8, unit = (id / p.sums) * 8 + blockIdx.x % 8;
  if (unit >= p.blocks * p.B * p.heads) return;
  const Sum& s = p.sum[id % p.sums];
  if (s.across) walk_tiles<DV, DK, W, BACK, WIDE, LOOK, true>(p, s, unit, ring.tile[0], since, most);
  else walk_tiles<DK, DV, W, BACK, WIDE, LOOK, false>(p, s, unit, ring.tile[0], since, most);
}

// Sums of what each query head gave a key head's rows, in the heads' order. Bound by memory (38 MB in 10 us).
struct FoldArgs {
  const float* parts[2];           // [B][Hk * group][T][n]
  Rows out[2];
  int n[2];
  int Hk, group, T;
  int64_t rows;                    // B * Hk * T
};
__global__ __launch_bounds__(256) void linear_fold(FoldArgs A) {
  const int n = A.n[blockIdx.y];
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, row = id / n;
  if (row >= A.rows) return;
  const int d = (int)(id % n), t = (int)(row % A.T), h = (int)(row / A.T % A.Hk);
  const int64_t b = row / A.T / A.Hk, head = (int64_t)A.T * n;
  const float* part = A.parts[blockIdx.y] + ((b * A.Hk + h) * A.group) * head + (int64_t)t * n + d;
  float s = part[0];
  for (int i = 1; i < A.group; ++i) s += part[i * head];
  const Rows& out = A.out[blockIdx.y];
  out.p[b * out.b + h * out.h + t * out.t + d] = s;
}

// ---- a few positions ---------------------------------------------------------------------------------------

constexpr int kSteps = 8;          // at most

// A block keeps one head's state: a thread four columns of every RG-th row. Bound by memory: the state is read and written once (1024
// heads of 128 x 128: 136 MB in 23 us, 5.9 TB/s).
struct StepsArgs {
  LinearDesc a;
  bool wide;                       // of the states
};
template <int DP>
__global__ __launch_bounds__(256) void linear_steps(StepsArgs A) {
  constexpr int CQ = DP <= 32 ? 8 : DP <= 64 ? 16 : 32, RG = 256 / CQ, R = (DP + RG - 1) / RG;
  __shared__ float qs[kSteps][DP], ks[kSteps][DP];
  __shared__ __align__(16) float vs[kSteps][4 * CQ], part[4][kSteps][4 * CQ];   // by 16 bytes
  const LinearDesc& a = A.a;
  const int tid = threadIdx.x, cq = tid % CQ, rg = tid / CQ, w = tid >> 6, b = blockIdx.x / a.H, h = blockIdx.x % a.H, hk = h / (a.H / a.Hk);
  const int n = count_of({a.documents, a.lengths, a.T}, b);
  const int64_t state = (int64_t)blockIdx.x * a.D * a.Dv;
  f32x4 S[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int d = rg + RG * i;
    S[i] = f32x4{};
    if (!a.state || d >= a.D) continue;
    const float* p = a.state + state + (int64_t)d * a.Dv + 4 * cq;
    if (A.wide) {
      if (4 * cq < a.Dv) S[i] = *(const f32x4*)p;
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) if (4 * cq + q < a.Dv) S[i][q] = p[q];
    }
  }
  const int32_t* doc = a.documents ? a.documents + (int64_t)b * a.T : nullptr;
  for (int e = tid; e < a.T * DP; e += 256) {
    const int t = e / DP, d = e % DP;
    const bool here = t < n && (!doc || doc[t] >= 0);
    qs[t][d] = here && d < a.D ? a.q.p[b * a.q.b + h * a.q.h + t * a.q.t + d] : 0.0f;
    ks[t][d] = here && d < a.D ? a.k.p[b * a.k.b + hk * a.k.h + t * a.k.t + d] : 0.0f;
  }
  for (int e = tid; e < a.T * 4 * CQ; e += 256) {
    const int t = e / (4 * CQ), c = e % (4 * CQ);
    vs[t][c] = t < n && (!doc || doc[t] >= 0) && c < a.Dv ? a.v.p[b * a.v.b + hk * a.v.h + t * a.v.t + c] : 0.0f;
  }
  __syncthreads();
  const Decay decay = decay_of(a.rate[h]);
  for (int t = 0; t < n; ++t) {
    const bool fresh = doc && (doc[t] < 0 || (t > 0 && doc[t] != doc[t - 1]));
    const f32x4 v = *(const f32x4*)&vs[t][4 * cq];
    f32x4 y = {};
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int d = min(rg + RG * i, DP - 1);
      const float kd = ks[t][d], qd = qs[t][d];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        S[i][q] = fmaf(kd, v[q], fresh ? 0.0f : __builtin_amdgcn_ldexpf(decay.factor * S[i][q], decay.shift));
        y[q] = fmaf(qd, rg + RG * i < a.D ? S[i][q] : 0.0f, y[q]);
      }
    }
#pragma unroll
    for (int o = CQ; o < 64; o *= 2)
#pragma unroll
      for (int q = 0; q < 4; ++q) y[q] += __shfl_xor(y[q], o);
    if ((tid & 63) < CQ) *(f32x4*)&part[w][t][4 * cq] = y;
  }
  if (a.last) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int d = rg + RG * i;
      if (d >= a.D) continue;
      float* p = a.last + state + (int64_t)d * a.Dv + 4 * cq;
      if (A.wide) {
        if (4 * cq < a.Dv) *(f32x4*)p = S[i];
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) if (4 * cq + q < a.Dv) p[q] = S[i][q];
      }
    }
  }
  if (!a.y.p) return;
  __syncthreads();
  for (int e = tid; e < a.T * a.Dv; e += 256) {
    const int t = e / a.Dv, c = e % a.Dv;
    const bool here = t < n && (!doc || doc[t] >= 0);
    a.y.p[b * a.y.b + h * a.y.h + t * a.y.t + c] = here ? a.scale * ((part[0][t][c] + part[1][t][c]) + (part[2][t][c] + part[3][t][c])) : 0.0f;
  }
}

// ---- plans -------------------------------------------------------------------------------------------------

// Whole 16-byte pieces, and 32 rows within 32-bit offsets.
inline bool wide_rows(const Rows& x) { return ((uintptr_t)x.p & 15) == 0 && x.b % 4 == 0 && x.h % 4 == 0 && x.t % 4 == 0 && x.t < (1 << 24); }
inline int segments(const LinearDesc& a) { return (a.T + kSeg - 1) / kSeg; }
inline int padded(const LinearDesc& a) { return (std::max(a.D, a.Dv) + 31) / 32 * 32; }
inline int64_t states_bytes(const LinearDesc& a) { return ((int64_t)segments(a) * a.B * a.H * a.D * a.Dv * 4 + 255) / 256 * 256; }
inline int64_t stay_bytes(const LinearDesc& a) { return ((int64_t)segments(a) * a.B * a.H * 4 + 255) / 256 * 256; }

// f(keys' features, values' features), padded, as constants. Values of another size than keys have kernels of their own (14 sequences
// of 617, 8 heads of 128 and 16 features: forward 64 us, a training step 190; padded to the larger size 114 and 341; of 64 and 32: 42
// and 127 instead of 54 and 161); 96 features go with 96, or count as 128.
template <class F>
void by_sizes(const LinearDesc& a, F f) {
  int k = (a.D + 31) / 32 * 32, v = (a.Dv + 31) / 32 * 32;
  if (k == 96 || v == 96) k = v = std::max(k, v);
  auto values = [&](auto K) {
    if (v == 32) f(K, std::integral_constant<int, 32>());
    else if (v == 64) f(K, std::integral_constant<int, 64>());
    else f(K, std::integral_constant<int, 128>());
  };
  if (v == 96) f(std::integral_constant<int, 96>(), std::integral_constant<int, 96>());
  else if (k == 32) values(std::integral_constant<int, 32>());
  else if (k == 64) values(std::integral_constant<int, 64>());
  else values(std::integral_constant<int, 128>());
}
// f(the larger of both, padded).
template <class F>
void by_larger(const LinearDesc& a, F f) {
  switch (padded(a)) {
    case 32: return f(std::integral_constant<int, 32>());
    case 64: return f(std::integral_constant<int, 64>());
    case 96: return f(std::integral_constant<int, 96>());
    default: return f(std::integral_constant<int, 128>());
  }
}
// States at the borders of all segments (in place of the sums), and the one at the end.
void states(const LinearDesc& a, const Rows& x, const Rows& y, bool back, const float* first, float* last, float* at, float* stay, hipStream_t st) {
  SumsArgs s{};
  s.m = {a.documents, a.lengths, a.T};
  s.x = x;
  s.y = y;
  s.H = a.H;
  s.share = back ? 1 : a.H / a.Hk;
  s.segs = segments(a);
  s.n = a.D;
  s.ny = a.Dv;
  s.back = back;
  s.scale = a.scale;
  s.rate = a.rate;
  s.sums = at;
  const int64_t rows = (int64_t)a.B * a.H, each = (int64_t)a.D * a.Dv;
  s.stay = stay;
  const bool wide = a.D % 4 == 0 && a.Dv % 4 == 0 && wide_rows(x) && wide_rows(y);
  const dim3 grid((unsigned)(rows * s.segs));
  if (wide) by_sizes(a, [&](auto K, auto V) { klaunch(linear_sums<K.value, V.value, true>, grid, dim3(256), 0, st, s); });
  else by_larger(a, [&](auto P) { klaunch(linear_sums<P.value, P.value, false>, grid, dim3(256), 0, st, s); });
  const JoinArgs j{at, s.stay, first, last, s.segs, rows, each, back};
  klaunch(linear_join, dim3((unsigned)((rows * each + 255) / 256)), dim3(256), 0, st, j);
}

template <bool BACK>
void pairs(PairsArgs p, const LinearDesc& a, const float* at, const float* edge, hipStream_t st) {
  p.m = {a.documents, a.lengths, a.T};
  p.B = a.B;
  p.H = a.H;
  p.segs = segments(a);
  p.share = a.H / a.Hk;
  if (!p.heads) {
    p.heads = BACK ? a.Hk : a.H;
    p.group = p.share;
    p.keys = 1;
  }
  p.states = at;
  p.edge = edge;
  p.D = a.D;
  p.Dv = a.Dv;
  p.by_pair = a.scale;
  p.by_state = BACK ? 1.0f : a.scale;
  p.fast = (-100 - std::min(0.0f, std::log2(a.scale))) / kSeg;
  p.large = 0x1p17f / std::cbrt(std::max(1.0f, a.scale));   // 128 pairs of 128 products of three of them: 2^-60 lost at most
  p.rate = a.rate;
  p.any = a.q.p;
  bool wide = a.D % 4 == 0 && a.Dv % 4 == 0 && wide_rows(a.q) && (((uintptr_t)at | (uintptr_t)edge) & 15) == 0;
  for (int i = 0; i < p.sums; ++i) {
    const Sum& s = p.sum[i];
    wide = wide && wide_rows(s.rows) && wide_rows(s.out) && wide_rows(s.x) && wide_rows(s.z);
  }
  // 64 rows a block where 128 would be fewer than the card has compute units (8 heads of 4000 positions, 256 blocks of 128: a training
  // step 93 us, of 64 99)
  const int rows = a.T > 64 && (int64_t)((a.T + 127) / 128) * p.B * p.heads * p.sums >= 256 ? 128 : 64;
  p.blocks = (a.T + rows - 1) / rows;
  const int64_t units = (int64_t)p.blocks * p.B * p.heads;
  const dim3 grid((unsigned)((units + 7) / 8 * 8 * p.sums));
  auto launch = [&](auto K, auto V, auto wide, auto look) {
    if (rows == 64) klaunch(linear_tiles<K.value, V.value, 4, BACK, wide.value, look.value>, grid, dim3(256), 0, st, p);
    else klaunch(linear_tiles<K.value, V.value, 8, BACK, wide.value, look.value>, grid, dim3(512), 0, st, p);
  };
  auto sized = [&](auto look) {
    if (wide) by_sizes(a, [&](auto K, auto V) { launch(K, V, std::true_type(), look); });
    else by_larger(a, [&](auto P) { launch(P, P, std::false_type(), look); });
  };
  if (a.least < p.fast) sized(std::true_type());
  else sized(std::false_type());
}

}  // namespace

int64_t linear_workspace_bytes(const LinearDesc& a) {
  if (a.T <= kSteps && !a.borders) return 0;
  return stay_bytes(a) + (a.borders ? 0 : states_bytes(a));
}

void linear(const LinearDesc& a, void* work, hipStream_t st) {
  if (a.T <= kSteps && !a.borders) {   // the steps make no states at borders
    const StepsArgs s{a, a.Dv % 4 == 0 && ((uintptr_t)a.state & 15) == 0 && ((uintptr_t)a.last & 15) == 0};
    return by_larger(a, [&](auto P) { klaunch(linear_steps<P.value>, dim3((unsigned)(a.B * a.H)), dim3(256), 0, st, s); });
  }
  float *stay = (float*)work, *at = a.borders ? a.borders : (float*)((char*)work + stay_bytes(a));
  if (a.last || a.borders || (a.y.p && segments(a) > 1)) states(a, a.k, a.v, false, a.state, a.last, at, stay, st);
  if (!a.y.p) return;
  PairsArgs p{};
  p.sum[p.sums++] = {a.q, a.y, a.k, a.v, a.D, a.Dv, false};
  pairs<false>(p, a, at, a.state, st);
}

// Key heads that several query heads share: a block takes all of those in turn, or one where all of them would leave the card half
// empty, and what they give is summed after (3 sequences of 1777, 8 heads on 2 of 96 and 80 features: 96 us in turn, 64 + 11 apart).
// Training steps, apart and in turn: 336 blocks of 64 rows in turn 197 us and 218, 448 of them 221 and 223; 512, of 64 features, 148 and
// 142, of 128 183 and 169; 1024 260 and 239. Seven query heads a key head lose by turns longer (540 blocks 251 and 295).
static bool split_heads(const LinearGradDesc& g) {
  const LinearDesc& a = g.a;
  const int sums = (g.dk.p != nullptr) + (g.dv.p != nullptr);
  return a.H > a.Hk && (int64_t)((a.T + 63) / 64) * a.B * a.Hk * sums < 512;
}
static int64_t part_bytes(const LinearDesc& a, int n) { return ((int64_t)a.B * a.H * a.T * n * 4 + 255) / 256 * 256; }
int64_t linear_grad_workspace_bytes(const LinearGradDesc& g) {
  const int64_t parts = split_heads(g) ? (g.dk.p ? part_bytes(g.a, g.a.D) : 0) + (g.dv.p ? part_bytes(g.a, g.a.Dv) : 0) : 0;
  return stay_bytes(g.a) + (g.borders ? 1 : 2) * states_bytes(g.a) + parts;
}

void linear_grad(const LinearGradDesc& g, void* work, hipStream_t st) {
  const LinearDesc& a = g.a;
  float *stay = (float*)work, *G = (float*)((char*)work + stay_bytes(a)), *S = (float*)((char*)G + states_bytes(a));
  const bool several = segments(a) > 1;
  if (g.dq.p && several && !g.borders) states(a, a.k, a.v, false, a.state, nullptr, S, stay, st);
  if (g.dfirst || ((g.dk.p || g.dv.p) && several)) states(a, a.q, g.dy, true, g.dstate, g.dfirst, G, stay, st);
  if (g.dq.p) {
    PairsArgs p{};
    p.sum[p.sums++] = {g.dy, g.dq, a.v, a.k, a.Dv, a.D, true};
    pairs<false>(p, a, g.borders ? g.borders : S, a.state, st);
  }
  PairsArgs p{};
  if (g.dk.p) p.sum[p.sums++] = {a.v, g.dk, g.dy, a.q, a.Dv, a.D, true};
  if (g.dv.p) p.sum[p.sums++] = {a.k, g.dv, a.q, g.dy, a.D, a.Dv, false};
  if (!p.sums) return;
  if (!split_heads(g)) return pairs<true>(p, a, G, g.dstate, st);
  FoldArgs f{};
  char* part = (char*)S + (g.borders ? 0 : states_bytes(a));
  f.Hk = a.Hk;
  f.group = a.H / a.Hk;
  f.T = a.T;
  f.rows = (int64_t)a.B * a.Hk * a.T;
  for (int i = 0; i < p.sums; ++i) {
    const int n = p.sum[i].nz;
    f.parts[i] = (const float*)part;
    f.out[i] = p.sum[i].out;
    f.n[i] = n;
    p.sum[i].out = {(float*)part, (int64_t)a.H * a.T * n, (int64_t)a.T * n, n};
    part += part_bytes(a, n);
  }
  p.heads = a.H;
  p.group = 1;
  p.keys = f.group;
  pairs<true>(p, a, G, g.dstate, st);
  klaunch(linear_fold, dim3((unsigned)((f.rows * std::max(f.n[0], f.n[1]) + 255) / 256), p.sums), dim3(256), 0, st, f);
}

}  // namespace tgk
