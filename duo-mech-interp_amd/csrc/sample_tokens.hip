// Tokens drawn from softmax(logits / temperature) cut by top-k, top-p and min-p, from given random numbers, and the cut itself
// (probabilities, or logits with what is cut at -inf).
//
// Tokens are ordered by logit, ties by index. Each cut keeps a first part of that order:
//   top-k   the first k
//   top-p   of these, while the sum of the weights ahead is below p of their whole sum
//   min-p   of these, while the weight is at least m of the first one's
// and the draw is the first kept token whose running sum exceeds u of the kept ones' sum. So all that is ever asked is where in
// one order a running count or sum reaches a target. The first token always stays; temperature 0 is top-k 1.
//
// Weights w = exp((x - max) / T) are formed in 64 bits, to 2e-12 of themselves, and held as whole numbers of 2^-S of the largest (S =
// 62 - log2 V, at most 50: the sum fits), so that sums depend on no order. Half a unit a token: a sum, and with it a border of top-p
// or a draw, is known to V 2^-(S + 1) of the largest weight and 2e-12 of itself (150 K tokens: 2^-28, and fp32's own step next to 1 is
// 2^-24; 2^22 tokens: 2^-19, where a tail of weights below 2^-41 each counts as nothing). min-p is a border of logits, to 64 bits.
//
//   sample_max_kernel    the largest value of each group of 16 and of each chunk of 4096
//   sample_hist_kernel   counts and sums of weights of the row in 2048 bins by distance from the maximum, from LDS into the
//                        row's bins by integer atomics. Rows of a small top-k need none of it
//   sample_pick_kernel   one block a row: the bins' running sums give the bin of each border; the groups whose largest value
//                        reaches that bin are fetched, and the bin's few tokens put in order. For a small top-k it forms the
//                        bins itself, of the groups that reach the k-th largest group's bin: all larger tokens are in them
//                        Of rows of up to 16 K tokens it is also what the two above are
//   sample_write_kernel  probabilities or cut logits, where they are asked for
//
// Rows of 151,936 logits (a copy runs at 5.2 TB/s): three of top-k 20 13.4 us, a chain of two launches and, in the second, of
// a dozen dependent steps of one block; 256 of top-p 0.9 120 us: the maximum 29 (5.4 TB/s), the histogram 43 (26 operations a
// token, most of 64 bits, and an atomic in LDS), the pick 51, whose one block a row reads what reaches the border's bin at a CU's
// 50 GB/s, most of the row where the nucleus is large; 160 of top-p 0.95 and min-p 0.02 cut into logits 94 us: 22, 33, 12, and 29
// for the write; the same of top-k 50 and top-p 0.95, which need no histogram, 63. 250,000 logits: three rows of top-k 20 18.0 us, 32 of
// top-p 0.9 80 (8, 19, 55; 151,936: 59). 1024 rows of 16,000 take one block each, one a CU for its LDS, four turns of them: 76 us with
// logits that fall with rank^-1.5, 100 where every row falls with a power of its own, from 1.1 to 3.
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "token_weights.h"

namespace q35 {

typedef unsigned long long u64;
constexpr int kSBins = 2048, kSFine = 1536;
constexpr int kSChunk = 1024;    // quads of a block of the maximum and the write kernel: 256 groups of 4 neighbouring ones
constexpr int kSFew = 1024;      // the largest top-k whose rows need no histogram
constexpr int kSThreads = 1024;  // of the pick kernel
constexpr int kSShort = 4;       // chunks of a row that the pick kernel takes alone
constexpr int kSHeld = 10;       // groups' maxima that one of its threads holds: rows of up to 163,840 tokens; further ones are read again
constexpr int kSSort = kSThreads;  // tokens that it sorts
constexpr int kSWaves = kSThreads / 64, kSSeg = 512;  // tokens that each of its waves can list
constexpr int64_t kSMaxV = 1 << 22;

enum SampleOut : int { kSampleNone = 0, kSampleProbs = 1, kSampleLogits = 2 };

// What is kept of a row: the tokens up to (x, idx) in the order; none where idx is -1 and x infinite.
struct SampleCut {
  double scale;  // probability of a weight of 1
  float max, x;
  int idx;
  int pad;
};
struct SampleArgs {
  const float* x;
  int64_t xb, xp;  // strides of a row and of a position
  int P;           // positions per row: they share its settings
  const float *temps, *top_ps, *min_ps;
  const int32_t* top_ks;
  float temp, top_p, min_p;
  int top_k;
  const float* u;
  int64_t ub;
  int V, C, R;  // chunks of the maximum kernel, blocks per row of the histogram kernel
  int S;        // weights are whole numbers of 2^-S
  float* cmax;  // [rows][C]
  float* gmax;  // [rows][C 256]
  u64* mass;    // [rows][kSBins]
  uint32_t* count;
  SampleCut* cut;
  int32_t* tokens;
  float* out;  // [rows][V]
};

constexpr double kSFar = 1100.0 * kVTab;  // 1/32 octaves from where on a weight is 0
struct SampleRow {
  const float* x;
  double inv_t;  // 32 log2(e) / T
  float t, p, m;
  int k;     // 0: all
  bool few;  // a small top-k
};
__device__ __forceinline__ float s_setting(const float* v, float one, int b) {
  return v ? __int_as_float(load_uniform(reinterpret_cast<const int32_t*>(v) + b)) : one;
}
__device__ __forceinline__ SampleRow s_row(const SampleArgs& a, int row) {
  const int b = row / a.P;
  SampleRow r;
  r.x = a.x + b * a.xb + (row - b * a.P) * a.xp;
  r.t = s_setting(a.temps, a.temp, b);
  r.k = a.top_ks ? load_uniform(a.top_ks + b) : a.top_k;
  r.p = s_setting(a.top_ps, a.top_p, b);
  r.m = s_setting(a.min_ps, a.min_p, b);
  if (!(r.t > 0.f)) {
    r.t = 1.f;
    r.k = 1;
  }
  if (r.m > 1.f) {  // more than any weight: the first token alone, whatever equals it
    r.m = 0.f;
    r.k = 1;
  }
  if (r.k <= 0 || r.k >= a.V) r.k = 0;
  r.few = r.k > 0 && r.k <= kSFew;
  r.inv_t = fmax(32.0 * 1.4426950408889634074 / (double)r.t, 1e-300);
  return r;
}

// The distance of x from the maximum M in 1/32 octaves of the weight, and the weight in units of 2^-S: 2^(-z / 32) by the series
// of exp2_neg, with S in the exponent, and both conversions to whole numbers by adding a power of two (fp64 has no other short
// one): 26 operations a token where rint, conversions and a comparison with an infinite maximum took 34 (256 rows of 151,936
// 49 -> 43 us).
struct SampleWeight {
  int n;
  u64 w;
};
struct SampleDistance {
  int n;
  double r;  // distance less n
};
__device__ __forceinline__ SampleDistance s_distance(float x, float M, const SampleRow& r) {
  constexpr double kRound = 0x1.8p52;
  // (an infinite maximum is the largest number, from which the finite ones are as far as from any)
  const double m = fmin((double)M, DBL_MAX), z = fmin((m - fmin((double)x, DBL_MAX)) * r.inv_t, kSFar), t = z + kRound;
  return {(int)(uint32_t)__builtin_bit_cast(u64, t), z - (t - kRound)};
}
__device__ __forceinline__ SampleWeight s_weight(float x, float M, const SampleRow& row, int S, const double* tab) {
  constexpr double c1 = -0.69314718055994530942 / kVTab, c2 = c1 * c1 / 2.0, c3 = c1 * c2 / 3.0, c4 = c1 * c3 / 4.0;
  const SampleDistance z = s_distance(x, M, row);
  const double e = __builtin_fma(__builtin_fma(__builtin_fma(__builtin_fma(c4, z.r, c3), z.r, c2), z.r, c1), z.r, 1.0);
  const int k = -z.n;
  const double w = __builtin_ldexp(e * tab[k & (kVTab - 1)], (k >> 5) + S) + 0x1p52;
  return {z.n, __builtin_bit_cast(u64, w) & 0xFFFFFFFFFFFFFull};
}
// The bin of a distance: 1/32 octave each for 48 octaves, then an octave each. Never larger for a larger x.
__device__ __forceinline__ int s_bin(int n) {
  return min(min(n, kSFine - (kSFine >> 5) + (n >> 5)), kSBins - 1);
}
__device__ __forceinline__ int s_bin(float x, float M, const SampleRow& r) { return s_bin(s_distance(x, M, r).n); }
// Order-preserving bits (-0 as +0; no NaN).
__device__ __forceinline__ uint32_t s_key(float x) {
  const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float s_unkey(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

// A row in quads that lie on 16 bytes: quad q holds elements 4 q - ahead .. + 3 (ahead < 4: how far the row's start is past 16
// bytes), those outside 0 .. V - 1 as -inf.
struct SampleQuads {
  const float* base;
  int ahead, V;
  __device__ __forceinline__ SampleQuads(const float* row, int V_) : V(V_) {
    ahead = (int)(((uintptr_t)row >> 2) & 3);
    base = row - ahead;
  }
  __device__ __forceinline__ int n() const { return (ahead + V + 3) >> 2; }
  // the quads that lie in the row whole
  __device__ __forceinline__ int whole_first() const { return ahead ? 1 : 0; }
  __device__ __forceinline__ int whole_last() const { return (ahead + V) >> 2; }
  __device__ __forceinline__ f32x4 whole(int q) const {
    f32x4 v = *reinterpret_cast<const f32x4*>(base + 4 * (int64_t)q);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = v_clean(v[e]);
    return v;
  }
  __device__ __forceinline__ f32x4 load(int q) const {
    const int i = 4 * q - ahead;
    f32x4 v;
    if (i >= 0 && i + 3 < V) {
      v = *reinterpret_cast<const f32x4*>(base + 4 * (int64_t)q);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = i + e >= 0 && i + e < V ? base[4 * (int64_t)q + e] : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = v_clean(v[e]);
    return v;
  }
};
// f(value) of the row's quads first, first + step, ... below last.
template <typename F>
__device__ __forceinline__ void s_for_row(const SampleQuads& s, int first, int step, int last, F&& f) {
  constexpr int U = 4;
  const int w0 = s.whole_first(), w1 = min(last, s.whole_last());
  int q = first < w0 ? first + step : first;
  for (; q + (U - 1) * step < w1; q += U * step) {
    f32x4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = s.whole(q + u * step);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) f(v[u][e]);
  }
  for (; q < w1; q += step) {
    const f32x4 v = s.whole(q);
#pragma unroll
    for (int e = 0; e < 4; ++e) f(v[e]);
  }
  // the row's ends, in quads that others share
  for (int e = 0; e < 2; ++e) {
    const int k = e ? s.whole_last() : 0;
    if (k < last && k >= first && (k - first) % step == 0 && (e ? s.n() > s.whole_last() && (k > 0 || w0 == 0) : w0 == 1)) {
      const f32x4 v = s.load(k);
      for (int i = 0; i < 4; ++i)
        if (4 * k - s.ahead + i >= 0 && 4 * k - s.ahead + i < s.V) f(v[i]);
    }
  }
}

__global__ __launch_bounds__(256) void sample_max_kernel(SampleArgs a) {
  const int tid = threadIdx.x, row = blockIdx.y, c = blockIdx.x;
  const SampleRow r = s_row(a, row);
  const SampleQuads s(r.x, a.V);
  if (!r.few) {  // the row's bins, cleared for the next kernel
    const int per = (kSBins + a.C - 1) / a.C;
    for (int i = c * per + tid; i < min((c + 1) * per, kSBins); i += 256) {
      a.mass[(size_t)row * kSBins + i] = 0;
      a.count[(size_t)row * kSBins + i] = 0;
    }
  }
  const int last = min((c + 1) * kSChunk, s.n());
  float m = -INFINITY, mine = -INFINITY;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int q = c * kSChunk + tid + 256 * u;
    float mq = -INFINITY;
    if (q < last) {
      const f32x4 v = s.load(q);
      mq = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
    }
    m = fmaxf(mq, m);
    // a group's quads lie in four lanes, of which lane u keeps the u-th one's
    mq = fmaxf(mq, __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(mq), 0xB1, 0xF, 0xF, false)));
    mq = fmaxf(mq, __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(mq), 0x4E, 0xF, 0xF, false)));
    if ((tid & 3) == u) mine = mq;
  }
  a.gmax[((size_t)row * a.C + c) * 256 + 64 * (tid & 3) + (tid >> 2)] = mine;
  m = wave_max_f32(m);
  __shared__ float sm[4];
  if ((tid & 63) == 0) sm[tid >> 6] = m;
  __syncthreads();
  if (tid == 0) a.cmax[(size_t)row * a.C + c] = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
}

// The row's maximum from its chunks', by every wave.
__device__ __forceinline__ float s_max(const SampleArgs& a, int row) {
  float m = -INFINITY;
  for (int c = threadIdx.x & 63; c < a.C; c += 64) m = fmaxf(m, a.cmax[(size_t)row * a.C + c]);
  return wave_max_f32(m);
}

__global__ __launch_bounds__(256) void sample_hist_kernel(SampleArgs a) {
  const int tid = threadIdx.x, row = blockIdx.y;
  const SampleRow r = s_row(a, row);
  if (r.few) return;
  const SampleQuads s(r.x, a.V);
  __shared__ u64 mass[kSBins];
  __shared__ uint32_t count[kSBins];
  __shared__ double tab[kVTab];
  exp2_table(tab, tid);
  for (int i = tid; i < kSBins; i += 256) {
    mass[i] = 0;
    count[i] = 0;
  }
  const float M = s_max(a, row);
  __syncthreads();
  const int nq = s.n(), per = (nq + a.R - 1) / a.R, first = blockIdx.x * per;
  auto add = [&](float x, bool counts) {
    const SampleWeight w = s_weight(x, M, r, a.S, tab);
    const int b = s_bin(w.n);
    if (counts) atomicAdd(&count[b], 1u);
    atomicAdd(&mass[b], w.w);
  };
  if (r.k > 0) s_for_row(s, first + tid, 256, min(first + per, nq), [&](float x) { add(x, true); });
  else s_for_row(s, first + tid, 256, min(first + per, nq), [&](float x) { add(x, false); });
  __syncthreads();
  for (int i = tid; i < kSBins; i += 256) {
    if (count[i]) __hip_atomic_fetch_add(a.count + (size_t)row * kSBins + i, count[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (mass[i]) __hip_atomic_fetch_add(a.mass + (size_t)row * kSBins + i, mass[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}

// ---------------------------------------------------------------------------------------------------------------
struct SamplePick {
  u64 mass[kSBins];  // of each bin, then sums up to and with it
  uint32_t count[kSBins];
  u64 list[kSWaves][kSSeg];  // tokens, each wave's own: bits that sort as the order, above the index
  u64 sort[kSSort];
  uint16_t group[kSHeld * kSThreads];  // groups that reach a value, from a first one on
  u64 hmass[256];
  uint32_t hcount[256];
  u64 wmass[kSWaves];
  uint32_t wcount[kSWaves];
  float wmax[kSWaves];
  double tab[kVTab];
  int groups;  // of the list
  int n;       // tokens to be sorted
  int full;    // whether a wave's list was
  int bin;     // of a target
  u64 sum, to_mass;
  uint32_t digit;
};

// Lane exchanges on the vector ALU. A ds_bpermute takes 100 cycles, a scan or a step of a sort of 64-bit values two of them: the
// pick of three rows of top-k 20 16.2 -> 12.7 us.
template <int CTRL, int ROWS> __device__ __forceinline__ u64 s_dpp_or_0(u64 v) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (uint32_t)v, CTRL, ROWS, 0xF, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (uint32_t)(v >> 32), CTRL, ROWS, 0xF, true);
  return ((u64)hi << 32) | lo;
}
// Sums up to and with each lane.
__device__ __forceinline__ u64 s_wave_scan(u64 v) {
  v += s_dpp_or_0<0x111, 0xF>(v);  // row_shr:1
  v += s_dpp_or_0<0x112, 0xF>(v);
  v += s_dpp_or_0<0x114, 0xF>(v);
  v += s_dpp_or_0<0x118, 0xF>(v);
  v += s_dpp_or_0<0x142, 0xA>(v);  // row_bcast:15 into rows 1 and 3
  v += s_dpp_or_0<0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
  return v;
}
__device__ __forceinline__ uint32_t s_wave_scan(uint32_t v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, true);
  return v;
}
__device__ __forceinline__ u64 s_lane(u64 v, int lane) {  // of a uniform lane
  return ((u64)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(v >> 32), lane) << 32) |
         (uint32_t)__builtin_amdgcn_readlane((uint32_t)v, lane);
}
// The value J lanes apart (lane ^ J).
template <int J> __device__ __forceinline__ uint32_t s_xor(uint32_t v, int lane) {
  if constexpr (J == 1) return __builtin_amdgcn_mov_dpp(v, 0xB1, 0xF, 0xF, false);        // quad_perm [1,0,3,2]
  else if constexpr (J == 2) return __builtin_amdgcn_mov_dpp(v, 0x4E, 0xF, 0xF, false);   // quad_perm [2,3,0,1]
  else if constexpr (J == 4) {  // row_shl:4 into banks 0 and 2, row_shr:4 into banks 1 and 3
    const uint32_t up = __builtin_amdgcn_update_dpp(v, v, 0x104, 0xF, 0x5, false);
    return __builtin_amdgcn_update_dpp(up, v, 0x114, 0xF, 0xA, false);
  } else if constexpr (J == 8) return __builtin_amdgcn_mov_dpp(v, 0x128, 0xF, 0xF, false);  // row_ror:8
  else if constexpr (J == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return lane & 16 ? r[0] : r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return lane & 32 ? r[0] : r[1];
  }
}
// One step of a bitonic sort over J lanes: the smaller of the two stays in the lower lane where `up`.
template <int J> __device__ __forceinline__ u64 s_sort_step(u64 v, bool up, int lane) {
  const u64 o = ((u64)s_xor<J>((uint32_t)(v >> 32), lane) << 32) | s_xor<J>((uint32_t)v, lane);
  return (o < v) == (((lane & J) == 0) == up) ? o : v;
}
__device__ __forceinline__ u64 s_sort_steps(u64 v, int from, bool up, int lane) {
  if (from >= 32) v = s_sort_step<32>(v, up, lane);
  if (from >= 16) v = s_sort_step<16>(v, up, lane);
  if (from >= 8) v = s_sort_step<8>(v, up, lane);
  if (from >= 4) v = s_sort_step<4>(v, up, lane);
  if (from >= 2) v = s_sort_step<2>(v, up, lane);
  return s_sort_step<1>(v, up, lane);
}

// x[e] of four in registers
template <typename X> __device__ __forceinline__ auto pick4(const X& x, int e) { return e < 2 ? (e ? x[1] : x[0]) : e == 2 ? x[2] : x[3]; }

// Whether a token is kept: up to (x, idx) in the order.
struct SampleKept {
  float x;
  uint32_t idx;
  __device__ __forceinline__ bool has(float v, int i) const { return v > x || (v == x && (uint32_t)i <= idx); }
};

// SHORT: a row of up to 1024 groups, whose maxima and bins the block forms as well.
template <bool SHORT>
__global__ __launch_bounds__(kSThreads) void sample_pick_kernel(SampleArgs a) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.x;
  const SampleRow r = s_row(a, row);
  const SampleQuads s(r.x, a.V);
  __shared__ SamplePick g;
  const int G = a.C * 256;
  float* gmax = a.gmax + (size_t)row * G;
  exp2_table(g.tab, tid);
  float M = -INFINITY;
  if constexpr (SHORT) {
#pragma unroll
    for (int j = 0; j < kSShort; ++j) {
      const int q = tid + kSThreads * j;
      float m = -INFINITY;
      if (q < s.n()) {
        const f32x4 v = s.load(q);
        m = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
      }
      M = fmaxf(M, m);
      m = fmaxf(m, __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(m), 0xB1, 0xF, 0xF, false)));
      m = fmaxf(m, __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(m), 0x4E, 0xF, 0xF, false)));
      if (j < a.C && (tid & 3) == 0) gmax[q >> 2] = m;
    }
    M = wave_max_f32(M);
    if (lane == 0) g.wmax[wave] = M;
    __syncthreads();
    M = wave_max_f32(g.wmax[lane & (kSWaves - 1)]);
  } else {
    M = s_max(a, row);
    __syncthreads();  // (the table; above, the barrier of the maxima)
  }
  float held[kSHeld];  // the maxima of groups tid + 1024 i
#pragma unroll
  for (int i = 0; i < kSHeld; ++i)
    held[i] = (i == 0 || !SHORT) && tid + kSThreads * i < G ? gmax[tid + kSThreads * i] : -INFINITY;
  if (!(M > -INFINITY)) {  // nothing above -inf: token 0, nothing kept
    if (tid == 0) {
      a.cut[row] = {0.0, M, INFINITY, -1, 0};
      if (a.tokens) a.tokens[row] = 0;
    }
    return;
  }
  // ---- f(in, index, values) by whole waves, for quads of the row, in[e] for tokens of lo to hi: of the groups whose maximum reaches
  // lo, or, where most of them do, of all. False, and not all of them seen, as soon as more than `most` groups do.
  // Loads in flight of a wave: D in a pass over all (150 K tokens are otherwise a chain of their latencies), L of listed groups.
  auto traverse = [&](auto loads, auto still_held, float lo, float hi, int most, auto&& f) __attribute__((always_inline)) -> bool {
    constexpr int D = decltype(loads)::value, L = D > 1 ? 4 : 1;
    auto quad = [&](auto whole, bool there, int q, const f32x4& v) __attribute__((always_inline)) {
      const int i = 4 * q - s.ahead;
      bool in[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        in[e] = v[e] >= lo && v[e] <= hi;
        if constexpr (!decltype(whole)::value) in[e] = in[e] && there && i + e >= 0 && i + e < a.V;
      }
      if (__builtin_amdgcn_ballot_w64(in[0] | in[1] | in[2] | in[3])) f(in, i, v);
    };
    int seen = 0;
    for (int g0 = 0; g0 < G; g0 += kSHeld * kSThreads) {
      if (tid == 0) g.groups = 0;
      __syncthreads();
      uint32_t mine = 0;
#pragma unroll
      for (int i = 0; i < kSHeld; ++i) {
        const int at = g0 + tid + kSThreads * i;
        const float m = decltype(still_held)::value && g0 == 0 ? held[i] : at < G ? gmax[at] : -INFINITY;
        mine |= (at < G && m >= lo ? 1u : 0u) << i;
      }
      const uint32_t sum = s_wave_scan((uint32_t)__builtin_popcount(mine));
      int base = 0;
      if (lane == 63 && sum) base = atomicAdd(&g.groups, (int)sum);
      int put = __builtin_amdgcn_readlane(base, 63) + (int)sum - __builtin_popcount(mine);
#pragma unroll
      for (int i = 0; i < kSHeld; ++i)
        if (mine >> i & 1) g.group[put++] = (uint16_t)(tid + kSThreads * i);
      __syncthreads();
      const int listed = g.groups, nq = s.n(), here = min(G - g0, kSHeld * kSThreads);
      seen += listed;
      if (seen > most) {
        __syncthreads();
        return false;
      }
      if (4 * listed < here) {
        for (int k0 = 64 * wave; k0 < 4 * listed; k0 += L * kSThreads) {
          f32x4 v[L];
          int q[L];
#pragma unroll
          for (int u = 0; u < L; ++u) {
            const int k = k0 + lane + u * kSThreads, gr = k < 4 * listed ? g0 + g.group[k >> 2] : 0;
            q[u] = k < 4 * listed ? 4 * gr + (k & 3) : nq;
            v[u] = q[u] < nq ? s.load(q[u]) : zero4();
          }
#pragma unroll
          for (int u = 0; u < L; ++u) quad(std::false_type{}, q[u] < nq, q[u], v[u]);
        }
      } else {
        const int last = min(4 * (g0 + here), nq);
        for (int q0 = 4 * g0 + 64 * wave; q0 < last; q0 += D * kSThreads) {
          f32x4 v[D];
          if (q0 >= s.whole_first() && q0 + 63 + (D - 1) * kSThreads < min(last, s.whole_last())) {
#pragma unroll
            for (int u = 0; u < D; ++u) v[u] = s.whole(q0 + lane + u * kSThreads);
#pragma unroll
            for (int u = 0; u < D; ++u) quad(std::true_type{}, true, q0 + lane + u * kSThreads, v[u]);
          } else {
#pragma unroll 1
            for (int u = 0; u < D; ++u) {
              const int q = q0 + lane + u * kSThreads;
              quad(std::false_type{}, q < last, q, q < last ? s.load(q) : zero4());
            }
          }
        }
      }
      __syncthreads();
    }
    return true;
  };
  // The tokens of lo to hi into the waves' lists (mine_n of this one's), only those whose bits are first to last where `exact`;
  // false where they do not fit, or traverse() gave up.
  int mine_n = 0;
  auto collect = [&](auto still_held, float lo, float hi, bool exact, u64 first, u64 last, int most) __attribute__((always_inline)) -> bool {
    mine_n = 0;
    if (tid == 0) g.full = 0;
    const bool all = traverse(std::integral_constant<int, 6>{}, still_held, lo, hi, most, [&](bool (&in)[4], int i, const f32x4& v) __attribute__((always_inline)) {
      if (!decltype(still_held)::value && exact) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const u64 bits = ((u64)~s_key(v[e]) << 32) | (uint32_t)(i + e);
          in[e] = in[e] && bits >= first && bits <= last;
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const u64 mask = __builtin_amdgcn_ballot_w64(in[e]);
        if (!mask) continue;
        const int to = __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, mine_n));
        if (in[e] && to < kSSeg) g.list[wave][to] = ((u64)__float_as_uint(v[e]) << 32) | (uint32_t)(i + e);
        mine_n += __popcll(mask);
      }
    });
    if (lane == 0 && mine_n > kSSeg) g.full = 1;
    __syncthreads();
    const bool fits = all && !g.full;
    __syncthreads();
    return fits;
  };
  auto listed = [&](int l) __attribute__((always_inline)) -> u64 {
    const u64 t = g.list[wave][l];
    return ((u64)~s_key(__uint_as_float((uint32_t)(t >> 32))) << 32) | (uint32_t)t;
  };
  // Of the waves' lists those whose bits are first to last, together, to be sorted: how many (the first kSSort are there).
  auto gather = [&](u64 first, u64 last) __attribute__((always_inline)) -> int {
    if (tid == 0) g.n = 0;
    __syncthreads();
    for (int l0 = 0; l0 < mine_n; l0 += 64) {
      const u64 bits = l0 + lane < mine_n ? listed(l0 + lane) : 0;
      const bool in = l0 + lane < mine_n && bits >= first && bits <= last;
      const u64 mask = __builtin_amdgcn_ballot_w64(in);
      int base = 0;
      if (lane == 0 && mask) base = atomicAdd(&g.n, __popcll(mask));
      const int to = __builtin_amdgcn_readfirstlane(base) +
                     __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
      if (in && to < kSSort) g.sort[to] = bits;
    }
    __syncthreads();
    const int n = g.n;
    __syncthreads();
    return n;
  };
  // ---- the list (n tokens of it, up to kSSort) sorted, and its running sum of weights, token i in thread i; up to 64 tokens by
  // every wave for itself
  u64 v = 0, run = 0;
  int at = 0;       // this thread's place
  bool one = true;  // (every wave for itself)
  auto sort = [&](int n) __attribute__((always_inline)) {
    one = n <= 64;
    at = one ? lane : tid;
    v = at < n ? g.sort[at] : ~0ull;
    int P = 2;
    while (P < n) P <<= 1;
    for (int k = 2; k <= P; k <<= 1) {
      const bool up = (at & k) == 0;
      for (int j = k >> 1; j >= 64; j >>= 1) {
        __syncthreads();
        g.sort[tid] = v;
        __syncthreads();
        const u64 o = g.sort[tid ^ j];
        v = (o < v) == (((tid & j) == 0) == up) ? o : v;
      }
      v = s_sort_steps(v, min(k >> 1, 32), up, lane);
    }
    run = s_wave_scan(at < n ? s_weight(s_unkey(~(uint32_t)(v >> 32)), M, r, a.S, g.tab).w : 0ull);
    if (!one) {
      __syncthreads();
      if (lane == 63) g.wmass[wave] = run;
      __syncthreads();
      const u64 w = s_wave_scan(lane < 16 ? g.wmass[lane] : 0ull);
      if (wave) run += s_lane(w, wave - 1);
    }
  };
  // what thread i of the sorted list holds; the first place of it whose running sum reaches a target (or the last asked)
  auto of_place = [&](u64 mine, int i) __attribute__((always_inline)) -> u64 {
    if (one) return s_lane(mine, i);
    __syncthreads();
    if (tid == i) g.sum = mine;
    __syncthreads();
    return g.sum;
  };
  auto place_of = [&](u64 target, int most) __attribute__((always_inline)) -> int {
    const u64 in = __builtin_amdgcn_ballot_w64(at < most && run >= target);
    if (one) return in ? __builtin_ctzll(in) : most - 1;
    if (tid == 0) g.bin = most - 1;
    __syncthreads();
    if (in && lane == __builtin_ctzll(in)) atomicMin(&g.bin, tid);
    __syncthreads();
    const int i = g.bin;
    __syncthreads();
    return i;
  };
  const float u = a.tokens ? a.u[(int64_t)(row / a.P) * a.ub] : 0.f;
  auto p_target = [&](u64 Z) __attribute__((always_inline)) -> u64 {
    const double goal = ceil((double)fmaxf(r.p, 0.f) * (double)Z);
    return goal < 1.0 ? 1 : min((u64)goal, Z);
  };
  auto u_target = [&](u64 Z) __attribute__((always_inline)) -> u64 {
    const double goal = floor(fmax((double)u, 0.0) * (double)Z);
    return goal >= (double)Z ? Z : min((u64)goal + 1, Z);
  };
  // The smallest value of weight m or more: exp((x - max) / T) >= m where x >= max + T ln m, in 64 bits. (Not by the weights of values
  // next to it: their series is 2e-12 off, and next to 0 fp32 has any number of values within 2e-12 T. 2^-54 less: what rounds to 1
  // weighs 1, at an infinite temperature every finite logit.)
  float least = -INFINITY;
  if (r.m > 0.f) {
    const double border = __builtin_fma(log((double)r.m) - 0x1p-54, (double)r.t, (double)M);
    if (!(fabsf(M) < INFINITY)) {
      least = M;
    } else if (border >= -(double)FLT_MAX) {
      least = (float)border;
      if ((double)least < border) least = s_unkey(s_key(least) + 1);
    }
  }
  // ---- the row's bins, and their running sums: two a thread
  auto clear = [&]() __attribute__((always_inline)) {
    for (int i = tid; i < kSBins; i += kSThreads) {
      g.mass[i] = 0;
      g.count[i] = 0;
    }
    __syncthreads();
  };
  auto scan = [&](bool from_row) __attribute__((always_inline)) {
    u64 m[2];
    uint32_t c[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      m[i] = from_row ? a.mass[(size_t)row * kSBins + 2 * tid + i] : g.mass[2 * tid + i];
      c[i] = from_row ? a.count[(size_t)row * kSBins + 2 * tid + i] : g.count[2 * tid + i];
    }
    u64 im = s_wave_scan(m[0] + m[1]);
    uint32_t ic = s_wave_scan(c[0] + c[1]);
    if (lane == 63) {
      g.wmass[wave] = im;
      g.wcount[wave] = ic;
    }
    __syncthreads();
    const u64 wm = s_wave_scan(lane < 16 ? g.wmass[lane] : 0ull);
    const uint32_t wc = s_wave_scan(lane < 16 ? g.wcount[lane] : 0u);
    if (wave) {
      im += s_lane(wm, wave - 1);
      ic += __builtin_amdgcn_readlane(wc, wave - 1);
    }
    g.mass[2 * tid + 1] = im;
    g.mass[2 * tid] = im - m[1];
    g.count[2 * tid + 1] = ic;
    g.count[2 * tid] = ic - c[1];
    __syncthreads();
  };
  auto mass_below = [&](int b) __attribute__((always_inline)) -> u64 { return b > 0 ? g.mass[b - 1] : 0; };
  auto count_below = [&](int b) __attribute__((always_inline)) -> uint32_t { return b > 0 ? g.count[b - 1] : 0; };
  auto bin_of_mass = [&](u64 target) __attribute__((always_inline)) -> int {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (g.mass[2 * tid + i] >= target && mass_below(2 * tid + i) < target) g.bin = 2 * tid + i;
    __syncthreads();
    const int b = g.bin;
    __syncthreads();
    return b;
  };
  auto bin_of_count = [&](uint32_t target) __attribute__((always_inline)) -> int {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (g.count[2 * tid + i] >= target && count_below(2 * tid + i) < target) g.bin = 2 * tid + i;
    __syncthreads();
    const int b = g.bin;
    __syncthreads();
    return b;
  };
  // no token of the bins up to b is smaller (d: its distance in 1/32 octaves)
  auto bound = [&](int b) __attribute__((always_inline)) -> float {
    if (b >= kSBins - 1) return -INFINITY;
    if (!(fabsf(M) < INFINITY)) return M;
    const double d = b < kSFine ? b + 1.0 : kSFine + 32.0 * (b - kSFine + 1) + 1.0;
    return (float)((double)M - d / r.inv_t - 1e-6 * fabs((double)M)) - 1e-37f;
  };

  // ---- Where all that is kept is among few tokens: these are sorted, and the rest is looked up in the running sum. For a small
  // top-k the k-th largest token is no further than the k-th largest group's bin (fewer groups than k: than any), in bins of
  // its own that take no 64-bit operations.
  float floor_x = -INFINITY;
  bool bounded = true;
  u64 Z_row = 0;
  if (r.few) {
    for (int i = tid; i < kSBins; i += kSThreads) g.count[i] = 0;
    __syncthreads();
    const float per = fminf((float)r.inv_t, 1e30f);
    auto bin = [&](float x) __attribute__((always_inline)) {
      const float y = (M - x) * per;
      return x == M ? 0 : y < (float)(kSBins - 1) ? (int)y : kSBins - 1;
    };
#pragma unroll
    for (int i = 0; i < kSHeld; ++i)
      if (tid + kSThreads * i < G) atomicAdd(&g.count[bin(held[i])], 1u);
    for (int i = tid + kSHeld * kSThreads; i < G; i += kSThreads) atomicAdd(&g.count[bin(gmax[i])], 1u);
    __syncthreads();
    if (G >= r.k) {
      const uint32_t c0 = g.count[2 * tid], c1 = g.count[2 * tid + 1];
      uint32_t ic = s_wave_scan(c0 + c1);
      if (lane == 63) g.wcount[wave] = ic;
      __syncthreads();
      const uint32_t wc = s_wave_scan(lane < 16 ? g.wcount[lane] : 0u);
      if (wave) ic += __builtin_amdgcn_readlane(wc, wave - 1);
      if (ic >= (uint32_t)r.k && ic - c0 - c1 < (uint32_t)r.k) g.bin = ic - c1 >= (uint32_t)r.k ? 2 * tid : 2 * tid + 1;
      __syncthreads();
      const int b = g.bin;
      if (b < kSBins - 1)
        floor_x = fabsf(M) < INFINITY ? (float)((double)M - (b + 1.001) / (double)per - 1e-6 * fabs((double)M)) - 1e-37f : M;
      __syncthreads();
    }
  } else {
    if constexpr (SHORT) {
      clear();
#pragma unroll 1
      for (int j = 0; j < kSShort; ++j) {
        const int q = tid + kSThreads * j, i = 4 * q - s.ahead;
        if (q >= s.n()) break;
        const f32x4 x = s.load(q);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (i + e < 0 || i + e >= a.V) continue;
          const SampleWeight w = s_weight(x[e], M, r, a.S, g.tab);
          const int b = s_bin(w.n);
          if (r.k > 0) atomicAdd(&g.count[b], 1u);
          atomicAdd(&g.mass[b], w.w);
        }
      }
      __syncthreads();
    }
    scan(!SHORT);
    Z_row = g.mass[kSBins - 1];
    if (r.k > 0) floor_x = bound(bin_of_count((uint32_t)r.k));
    else if (r.p < 1.f) floor_x = bound(bin_of_mass(p_target(Z_row)));
    else bounded = false;
  }
  if (least > floor_x && !(r.k > 0 && r.p < 1.f)) {  // (top-p of top-k takes all of top-k's sum)
    floor_x = least;
    bounded = true;
  }
  if (bounded) {
    const int n = collect(std::true_type{}, floor_x, M, false, 0, ~0ull, kSSort) ? gather(0, ~0ull) : kSSort + 1;
    if (n <= kSSort) {
      sort(n);
      int K = r.k > 0 ? min(r.k, n) : n;
      if (r.p < 1.f) K = place_of(p_target(r.k > 0 ? of_place(run, K - 1) : Z_row), K) + 1;
      if (r.m > 0.f) {  // (sorted: those of at least `least` come first)
        int c = __popcll(__builtin_amdgcn_ballot_w64(at < K && s_unkey(~(uint32_t)(v >> 32)) >= least));
        if (!one) {
          if (tid == 0) g.n = 0;
          __syncthreads();
          if (lane == 0) atomicAdd(&g.n, c);
          __syncthreads();
          c = g.n;
        }
        K = max(c, 1);
      }
      const u64 Z = of_place(run, K - 1);
      if (tid == K - 1) a.cut[row] = {__builtin_ldexp(1.0, a.S) / (double)Z, M, s_unkey(~(uint32_t)(v >> 32)), (int)(uint32_t)v, 0};
      if (a.tokens) {
        const int i = place_of(u_target(Z), K);
        if (tid == i) a.tokens[row] = (int)(uint32_t)v;
      }
      return;
    }
    if (r.few) {  // many tokens of about one value: the bins, of the tokens themselves
      clear();
      traverse(std::integral_constant<int, 1>{}, std::false_type{}, floor_x, M, G, [&](bool (&in)[4], int, const f32x4& x) __attribute__((always_inline)) {
#pragma unroll 1
        for (int e = 0; e < 4; ++e) {
          if (!pick4(in, e)) continue;
          const SampleWeight w = s_weight(pick4(x, e), M, r, a.S, g.tab);
          const int b = s_bin(w.n);
          atomicAdd(&g.count[b], 1u);
          atomicAdd(&g.mass[b], w.w);
        }
      });
      scan(false);
    }
  }

  // ---- Otherwise the bin of each border, and its tokens. The smallest value of a bin up to b: six bits a step, a lane each
  auto smallest = [&](int b) __attribute__((always_inline)) -> float {
    uint32_t key = s_key(-INFINITY);  // the largest known to be below
    const uint32_t top = s_key(M);
    if (s_bin(-INFINITY, M, r) <= b) return -INFINITY;
    for (int sh = 26; sh > -6; sh -= 6) {
      const uint32_t step = sh >= 0 ? 1u << sh : 1u;
      const u64 at64 = (u64)key + (u64)(lane + 1) * step;
      const uint32_t to = (uint32_t)(at64 < top ? at64 : top);
      const u64 in = __builtin_amdgcn_ballot_w64(s_bin(s_unkey(to), M, r) <= b);
      const u64 below = (u64)key + (u64)__builtin_ctzll(in) * step;  // (the last lane's value is inside)
      key = (uint32_t)(below < top ? below : top - 1);
    }
    return s_unkey(key + 1);
  };
  float lo = 0.f, hi = 0.f;  // bin b's smallest and largest value
  auto in_bin = [&](int b) __attribute__((always_inline)) {
    lo = smallest(b);
    hi = b > 0 ? s_unkey(s_key(smallest(b - 1)) - 1) : M;
  };
  auto value_of = [&](u64 bits) __attribute__((always_inline)) -> float { return s_unkey(~(uint32_t)(bits >> 32)); };
  // What is kept so far: the tokens up to these bits (as listed), and their mass. Top-k, top-p, then (behind min-p) the draw: each
  // the token of a bin at which the running count or mass reaches a target.
  u64 kept = ~0ull, Z = g.mass[kSBins - 1];
  // (three copies: as a loop it held what they share in registers, more than there are)
  auto cut = [&](auto step_of) __attribute__((always_inline)) {
    constexpr int step = decltype(step_of)::value;
    int b;
    u64 target;
    const bool by_mass = step > 0;
    if (step == 0) {
      if (r.k <= 0 || g.count[kSBins - 1] < (uint32_t)r.k) return;  // (fewer than that are of weight m)
      b = bin_of_count((uint32_t)r.k);
      target = (uint32_t)r.k - count_below(b);
    } else if (step == 1) {
      if (!(r.p < 1.f)) return;
      target = p_target(Z);
      b = bin_of_mass(target);
      target -= mass_below(b);
    } else {
      const u64 enough = least > -INFINITY ? ((u64)~s_key(least) << 32) | 0xFFFFFFFFu : ~0ull;  // all of weight m
      if (enough < kept) {
        b = s_bin(least, M, r);
        if (tid == 0) g.to_mass = 0;
        in_bin(b);
        traverse(std::integral_constant<int, 1>{}, std::false_type{}, fmaxf(lo, least), hi, G, [&](bool (&in)[4], int, const f32x4& x) __attribute__((always_inline)) {
#pragma unroll 1
          for (int e = 0; e < 4; ++e)
            if (pick4(in, e)) atomicAdd(&g.to_mass, s_weight(pick4(x, e), M, r, a.S, g.tab).w);
        });
        kept = enough;
        Z = mass_below(b) + g.to_mass;
        __syncthreads();
      }
      if (tid == 0)
        a.cut[row] = {__builtin_ldexp(1.0, a.S) / (double)Z, M, kept == ~0ull ? -INFINITY : value_of(kept), (int)(uint32_t)kept, 0};
      if (!a.tokens) return;
      target = u_target(Z);
      b = bin_of_mass(target);
      target -= mass_below(b);
    }
    u64 token = 0;
    in_bin(b);
    u64 first = (u64)~s_key(hi) << 32, last = min(((u64)~s_key(lo) << 32) | 0xFFFFFFFFu, kept), ahead = 0, aheadw = 0;
    bool lists = false;  // whether the waves' lists hold what is first to last
    // (each turn takes 8 of the 64 bits, and 512 neighbouring ones fit any list: done in 9 turns, and bounded in any case)
    for (int turn = 0; turn < 10; ++turn) {
      // narrowed by 256 (a digit's running sums; ahead, aheadw: count or mass, and mass, in front) until the rest can be sorted
      if (!lists) lists = collect(std::false_type{}, value_of(last), value_of(first), turn > 0, first, last, G);
      const int n = lists ? gather(first, last) : kSSort + 1;
      if (n <= kSSort) {
        sort(n);
        const int i = by_mass ? place_of(target - ahead, n) : (int)(target - ahead) - 1;
        token = of_place(v, i);
        Z = mass_below(b) + aheadw + of_place(run, i);
        __syncthreads();
        break;
      }
      const int shift = max(56 - __builtin_clzll((last - first) | 1), 0);
      for (int i = tid; i < 256; i += kSThreads) {
        g.hmass[i] = 0;
        g.hcount[i] = 0;
      }
      __syncthreads();
      auto count = [&](u64 bits) __attribute__((always_inline)) {
        if (bits < first || bits > last) return;
        atomicAdd(&g.hcount[(bits - first) >> shift], 1u);
        atomicAdd(&g.hmass[(bits - first) >> shift], s_weight(value_of(bits), M, r, a.S, g.tab).w);
      };
      if (lists) {
        for (int l = lane; l < mine_n; l += 64) count(listed(l));
        __syncthreads();
      } else {
        traverse(std::integral_constant<int, 1>{}, std::false_type{}, value_of(last), value_of(first), G, [&](bool (&in)[4], int i, const f32x4& x) __attribute__((always_inline)) {
#pragma unroll 1
          for (int e = 0; e < 4; ++e)
            if (pick4(in, e)) count(((u64)~s_key(pick4(x, e)) << 32) | (uint32_t)(i + e));
        });
      }
      if (wave == 0) {
        u64 t[4], w[4], st = 0, sw = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[e] = g.hmass[4 * lane + e];
          t[e] = by_mass ? w[e] : g.hcount[4 * lane + e];
          st += t[e];
          sw += w[e];
        }
        u64 upto = ahead + s_wave_scan(st) - st, uptow = aheadw + s_wave_scan(sw) - sw;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (upto < target && upto + t[e] >= target) {
            g.digit = 4 * lane + e;
            g.sum = upto;
            g.to_mass = uptow;
          }
          upto += t[e];
          uptow += w[e];
        }
      }
      __syncthreads();
      ahead = g.sum;
      aheadw = g.to_mass;
      first = min(first + ((u64)(g.digit & 255) << shift), last);
      last = min(last, first + (((u64)1 << shift) - 1));
      __syncthreads();
    }
    if (step == 2 && tid == 0) a.tokens[row] = (int)(uint32_t)token;
    kept = token;
  };
  cut(std::integral_constant<int, 0>{});
  cut(std::integral_constant<int, 1>{});
  cut(std::integral_constant<int, 2>{});
}

template <int OUT>
__global__ __launch_bounds__(256) void sample_write_kernel(SampleArgs a) {
  const int tid = threadIdx.x, row = blockIdx.y;
  const SampleRow r = s_row(a, row);
  const SampleQuads s(r.x, a.V);
  const SampleCut c = a.cut[row];
  const SampleKept kept{c.x, (uint32_t)c.idx};
  __shared__ double tab[kVTab];
  if (OUT == kSampleProbs) {
    exp2_table(tab, tid);
    __syncthreads();
  }
  float* o = a.out + (int64_t)row * a.V;
  const bool vec = (((uintptr_t)o - 4 * (uintptr_t)s.ahead) & 15) == 0;
#pragma unroll
  for (int u = 0; u < kSChunk / 256; ++u) {
    const int q = blockIdx.x * kSChunk + tid + 256 * u;
    if (q >= s.n()) continue;
    const f32x4 x = s.load(q);
    const int i = 4 * q - s.ahead;
    bool in[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) in[e] = kept.has(x[e], i + e);
    f32x4 y;
    if constexpr (OUT == kSampleLogits) {
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = in[e] ? x[e] : -INFINITY;
    } else {
      y = zero4();
      if (in[0] || in[1] || in[2] || in[3]) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (in[e]) y[e] = (float)(v_weight(x[e], c.max, r.inv_t, tab) * c.scale);
      }
    }
    if (vec && i >= 0 && i + 3 < a.V) {
      *reinterpret_cast<f32x4*>(o + i) = y;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e >= 0 && i + e < a.V) o[i + e] = y[e];
    }
  }
}

static int64_t s_chunks(int64_t V) { return ((V + 3) / 4 + 1 + kSChunk - 1) / kSChunk; }

}  // namespace q35

extern "C" size_t q35_sample_tokens_workspace_bytes(int64_t B, int64_t P, int64_t V) {
  using namespace q35;
  if (B <= 0 || P <= 0 || V <= 0 || B > 65535 || P > 65535 || B * P > 65535 || V > kSMaxV) return 0;
  const size_t rows = (size_t)B * P;
  return rows * (kSBins * (sizeof(u64) + sizeof(uint32_t)) + sizeof(SampleCut) + s_chunks(V) * 257 * sizeof(float));
}

extern "C" int q35_sample_tokens(const float* logits, int64_t l_sb, int64_t l_sp, const float* u, int64_t u_sb,
                                 const float* temperatures, float temperature, const int32_t* top_ks, int64_t top_k,
                                 const float* top_ps, float top_p, const float* min_ps, float min_p, int32_t* tokens, int out_kind,
                                 float* out, int64_t B, int64_t P, int64_t V, void* workspace, size_t workspace_bytes,
                                 q35_stream_t stream) {
  using namespace q35;
  if (!logits || B <= 0 || P <= 0 || V <= 0 || (!tokens && !out)) return Q35_EINVAL;
  if (tokens && (!u || P != 1)) return Q35_EINVAL;
  if (out_kind < kSampleNone || out_kind > kSampleLogits || (out_kind != kSampleNone) != (out != nullptr)) return Q35_EINVAL;
  if (l_sb < 0 || u_sb < 0 || (P > 1 && l_sp < V)) return Q35_EINVAL;
  if (!(temperature >= 0.f) || top_p != top_p || min_p != min_p) return Q35_EINVAL;
  const size_t need = q35_sample_tokens_workspace_bytes(B, P, V);
  if (need == 0) return Q35_EUNSUPPORTED;
  if (!workspace || workspace_bytes < need || (uintptr_t)workspace & 15) return Q35_EWORKSPACE;
  const size_t rows = (size_t)B * P;
  SampleArgs a{};
  a.x = logits, a.xb = l_sb, a.xp = l_sp, a.P = (int)P;
  a.temps = temperatures, a.top_ps = top_ps, a.min_ps = min_ps, a.top_ks = top_ks;
  a.temp = temperature, a.top_p = top_p, a.min_p = min_p, a.top_k = (int)(top_k <= 0 || top_k >= V ? 0 : top_k);
  a.u = u, a.ub = u_sb, a.V = (int)V, a.C = (int)s_chunks(V);
  int bits = 0;
  while (((int64_t)1 << bits) < V) ++bits;
  a.S = std::min(62 - bits, 50);
  a.mass = (u64*)workspace;
  a.count = (uint32_t*)(a.mass + rows * kSBins);
  a.cut = (SampleCut*)(a.count + rows * kSBins);
  a.cmax = (float*)(a.cut + rows);
  a.gmax = a.cmax + rows * a.C;
  a.tokens = tokens, a.out = out;
  const int64_t nq = (V + 3) / 4 + 1;
  a.R = (int)std::max<int64_t>(1, std::min<int64_t>((1024 + rows - 1) / rows, (nq + 1023) / 1024));
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const dim3 chunks(a.C, (unsigned)rows);
  // A short row's maximum and bins take its one block less than the launches of the two kernels (top-p 0.9, with them and
  // without: one row of 4000 21.4 and 15.5 us, 256 of 2000 21.2 and 15.3, of 16000 30.9 and 20.1, 1024 of 16000 87 and 76)
  const bool brief = a.C <= kSShort;
  if (!brief) hipLaunchKernelGGL(sample_max_kernel, chunks, dim3(256), 0, st, a);
  // (none of its blocks has work where one small top-k holds for all rows, or the argmax)
  const int64_t k = temperature > 0.f && (min_ps || !(min_p > 1.f)) ? top_k : 1;  // (as s_row has it)
  if (!brief && (temperatures || top_ks || k <= 0 || k >= V || k > kSFew))
    hipLaunchKernelGGL(sample_hist_kernel, dim3(a.R, (unsigned)rows), dim3(256), 0, st, a);
  if (brief) hipLaunchKernelGGL(sample_pick_kernel<true>, dim3((unsigned)rows), dim3(kSThreads), 0, st, a);
  else hipLaunchKernelGGL(sample_pick_kernel<false>, dim3((unsigned)rows), dim3(kSThreads), 0, st, a);
  if (out_kind == kSampleProbs) hipLaunchKernelGGL(sample_write_kernel<kSampleProbs>, chunks, dim3(256), 0, st, a);
  else if (out_kind == kSampleLogits) hipLaunchKernelGGL(sample_write_kernel<kSampleLogits>, chunks, dim3(256), 0, st, a);
  return hipGetLastError() == hipSuccess ? Q35_OK : Q35_ELAUNCH;
}
