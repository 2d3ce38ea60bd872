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
// Weights w = exp((x - max) / T) are formed in 64 bits and held as whole numbers of 2^-S (S = 62 - log2 V: the sum fits), so
// that sums depend on no order and a border lies where 64 bits put it: 2^-44 of the largest weight for 150 K tokens.
//
//   sample_max_kernel    the row's maximum, by chunks of 4096
//   sample_hist_kernel   counts and sums of weights of the row in 2048 bins by distance from the maximum (1/50 nat of the
//                        scaled logit for 30.7 nats, 1/2 nat behind them), from LDS into the row's bins by integer atomics
//   sample_pick_kernel   one block a row: the bins' running sums give the bin of each border; its few tokens are fetched and
//                        ordered
//   sample_write_kernel  probabilities or cut logits, where they are asked for
#include <algorithm>

#include "token_weights.h"

namespace q35 {

typedef unsigned long long u64;
constexpr int kSBins = 2048, kSFine = 1536;
constexpr int kSChunk = 1024;  // quads of a block of the maximum and the write kernel
constexpr int kSList = 2048;   // tokens of a bin that are held in LDS
constexpr int64_t kSMaxV = 1 << 22;

enum SampleOut : int { kSampleNone = 0, kSampleProbs = 1, kSampleLogits = 2 };

// What is kept of a row: bins below b, and of bin b the tokens up to (key, idx) in the order.
struct SampleCut {
  double scale;  // probability of a weight of 1
  float max;
  int b;
  uint32_t key;
  int idx;
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
  double unit;  // 2^S
  float* cmax;  // [rows][C]
  u64* mass;    // [rows][kSBins]
  uint32_t* count;
  SampleCut* cut;
  int32_t* tokens;
  float* out;  // [rows][V]
};

struct SampleRow {
  const float* x;
  double inv_t;  // 32 log2(e) / T
  float bins;    // bins per unit of the logit
  float t, p, m;
  int k;  // 0: all
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
  if (r.k <= 0 || r.k >= a.V) r.k = 0;
  r.inv_t = fmax(32.0 * 1.4426950408889634074 / (double)r.t, 1e-300);
  r.bins = 50.f / r.t;
  return r;
}

// The bin of x under the maximum M: the same in every kernel (no contraction), never larger for a larger x.
__device__ __forceinline__ int s_bin(float x, float M, float bins) {
#pragma clang fp contract(off)
  if (x == M) return 0;
  const float y = (M - x) * bins;
  if (y < (float)kSFine) return (int)y;
  const float z = (y - (float)kSFine) * 0.04f;
  return z < (float)(kSBins - 1 - kSFine) ? kSFine + (int)z : kSBins - 1;  // (NaN: an infinite temperature and -inf)
}
// Order-preserving bits (-0 as +0; no NaN).
__device__ __forceinline__ uint32_t s_key(float x) {
  const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float s_unkey(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}
__device__ __forceinline__ u64 s_mass(float x, float M, double inv_t, double unit, const double* tab) {
  return (u64)(v_weight(x, M, inv_t, tab) * unit + 0.5);
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
// f(index, value) of the row's quads first, first + step, ... below last; elements outside the row are left out.
template <typename F>
__device__ __forceinline__ void s_for_row(const SampleQuads& s, int first, int step, int last, F&& f) {
  constexpr int U = 4;
  for (int q = first; q < last; q += U * step) {
    f32x4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      v[u] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      if (q + u * step < last) v[u] = s.load(q + u * step);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (q + u * step >= last) break;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = 4 * (q + u * step) - s.ahead + e;
        if (i >= 0 && i < s.V) f(i, v[u][e]);
      }
    }
  }
}

__global__ __launch_bounds__(256) void sample_max_kernel(SampleArgs a) {
  const int tid = threadIdx.x, row = blockIdx.y, c = blockIdx.x;
  const SampleRow r = s_row(a, row);
  const SampleQuads s(r.x, a.V);
  // the row's bins, cleared for the next kernel
  const int per = (kSBins + a.C - 1) / a.C;
  for (int i = c * per + tid; i < min((c + 1) * per, kSBins); i += 256) {
    a.mass[(size_t)row * kSBins + i] = 0;
    a.count[(size_t)row * kSBins + i] = 0;
  }
  const int last = min((c + 1) * kSChunk, s.n());
  float m = -INFINITY;
#pragma unroll
  for (int u = 0; u < kSChunk / 256; ++u) {
    const int q = c * kSChunk + tid + 256 * u;
    if (q < last) {
      const f32x4 v = s.load(q);
      m = fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), m);
    }
  }
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
  s_for_row(s, first + tid, 256, min(first + per, nq), [&](int, float x) {
    const int b = s_bin(x, M, r.bins);
    const u64 w = s_mass(x, M, r.inv_t, a.unit, tab);
    atomicAdd(&count[b], 1u);
    if (w) atomicAdd(&mass[b], w);
  });
  __syncthreads();
  for (int i = tid; i < kSBins; i += 256) {
    if (count[i]) __hip_atomic_fetch_add(a.count + (size_t)row * kSBins + i, count[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (mass[i]) __hip_atomic_fetch_add(a.mass + (size_t)row * kSBins + i, mass[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}

// ---------------------------------------------------------------------------------------------------------------
constexpr int kSThreads = 1024;

struct SamplePick {
  u64 mass[kSBins];  // sums up to and with each bin
  uint32_t count[kSBins];
  float lx[kSList];  // the tokens of a bin
  int li[kSList];
  u64 hmass[256];
  uint32_t hcount[256];
  u64 wmass[16];
  uint32_t wcount[16];
  double tab[kVTab];
  int n;            // tokens of the bin
  int bin;          // of a target
  uint32_t key;     // the border: key, index, and count and mass up to and with it
  int idx;
  u64 to_mass, sum;
  uint32_t digit;
};

__device__ __forceinline__ u64 s_wave_scan(u64 v, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 w = __shfl_up(v, o);
    if (lane >= o) v += w;
  }
  return v;
}

// What is in the row, kept by a cut, as f(index, value).
struct SampleKept {
  int b;
  uint32_t key;
  int idx;
  __device__ __forceinline__ bool has(int bin, float x, int i) const {
    if (bin != b) return bin < b;
    const uint32_t k = s_key(x);
    return k > key || (k == key && i <= idx);
  }
};

__global__ __launch_bounds__(kSThreads) void sample_pick_kernel(SampleArgs a) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.x;
  const SampleRow r = s_row(a, row);
  const SampleQuads s(r.x, a.V);
  __shared__ SamplePick g;
  exp2_table(g.tab, tid);
  const float M = s_max(a, row);
  if (!(M > -INFINITY)) {  // nothing above -inf: token 0, nothing kept
    if (tid == 0) {
      a.cut[row] = {0.0, M, -1, 0, 0};
      if (a.tokens) a.tokens[row] = 0;
    }
    return;
  }
  // ---- running sums of the bins: two a thread
  {
    u64 m[2];
    uint32_t c[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      m[i] = a.mass[(size_t)row * kSBins + 2 * tid + i];
      c[i] = a.count[(size_t)row * kSBins + 2 * tid + i];
    }
    const u64 im = s_wave_scan(m[0] + m[1], lane);
    const uint32_t ic = (uint32_t)s_wave_scan(c[0] + c[1], lane);
    if (lane == 63) {
      g.wmass[wave] = im;
      g.wcount[wave] = ic;
    }
    __syncthreads();
    u64 bm = 0;
    uint32_t bc = 0;
    for (int w = 0; w < wave; ++w) {
      bm += g.wmass[w];
      bc += g.wcount[w];
    }
    g.mass[2 * tid + 1] = bm + im;
    g.mass[2 * tid] = bm + im - m[1];
    g.count[2 * tid + 1] = bc + ic;
    g.count[2 * tid] = bc + ic - c[1];
    __syncthreads();
  }
  auto mass_below = [&](int b) -> u64 { return b > 0 ? g.mass[b - 1] : 0; };
  auto count_below = [&](int b) -> uint32_t { return b > 0 ? g.count[b - 1] : 0; };
  auto bin_of_mass = [&](u64 target) -> int {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (g.mass[2 * tid + i] >= target && mass_below(2 * tid + i) < target) g.bin = 2 * tid + i;
    __syncthreads();
    const int b = g.bin;
    __syncthreads();
    return b;
  };
  auto bin_of_count = [&](uint32_t target) -> int {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (g.count[2 * tid + i] >= target && count_below(2 * tid + i) < target) g.bin = 2 * tid + i;
    __syncthreads();
    const int b = g.bin;
    __syncthreads();
    return b;
  };
  // ---- the tokens of bin b that a cut keeps: into the list; their number (the list holds the first kSList that came)
  auto collect = [&](int b, const SampleKept& kept) -> int {
    if (tid == 0) g.n = 0;
    __syncthreads();
    s_for_row(s, tid, kSThreads, s.n(), [&](int i, float x) {
      if (s_bin(x, M, r.bins) == b && kept.has(b, x, i)) {
        const int at = atomicAdd(&g.n, 1);
        if (at < kSList) {
          g.lx[at] = x;
          g.li[at] = i;
        }
      }
    });
    __syncthreads();
    return g.n;
  };
  // f(index, value) of these n tokens, from the list or, where it does not hold them, from the row
  auto for_bin = [&](int b, int n, const SampleKept& kept, auto&& f) {
    if (n <= kSList) {
      for (int i = tid; i < n; i += kSThreads) f(g.li[i], g.lx[i]);
    } else {
      s_for_row(s, tid, kSThreads, s.n(), [&](int i, float x) {
        if (s_bin(x, M, r.bins) == b && kept.has(b, x, i)) f(i, x);
      });
    }
  };
  // ---- the token of bin b at which the running count or mass reaches target: (g.key, g.idx), with the bin's mass up to and
  // with it in g.to_mass
  auto border = [&](int b, const SampleKept& kept, u64 target, bool by_mass) {
    const int n = collect(b, kept);
    if (n <= 64) {
      if (wave == 0) {
        const bool there = lane < n;
        const float x = there ? g.lx[lane] : 0.f;
        const u64 me = there ? ((u64)~s_key(x) << 32) | (uint32_t)g.li[lane] : ~0ull;
        const u64 w = there ? s_mass(x, M, r.inv_t, a.unit, g.tab) : 0, t = by_mass ? w : (there ? 1 : 0);
        u64 run = 0, runw = 0;
        for (int j = 0; j < n; ++j) {
          const bool le = __shfl(me, j) <= me;
          const u64 wj = __shfl(w, j);
          run += le ? (by_mass ? wj : 1) : 0;
          runw += le ? wj : 0;
        }
        if (there && run >= target && run - t < target) {
          g.key = s_key(x);
          g.idx = g.li[lane];
          g.to_mass = runw;
        }
      }
      __syncthreads();
      return;
    }
    // digits of 8 bits: four of the key, from the largest, then three of the index, from the smallest
    u64 ahead = 0, aheadw = 0;
    uint32_t key = 0, idx = 0;
    for (int level = 0; level < 7; ++level) {
      for (int i = tid; i < 256; i += kSThreads) {
        g.hmass[i] = 0;
        g.hcount[i] = 0;
      }
      __syncthreads();
      for_bin(b, n, kept, [&](int i, float x) {
        const uint32_t d = ~s_key(x);
        uint32_t at;
        if (level < 4) {
          if (level > 0 && (d >> (32 - 8 * level)) != key) return;
          at = (d >> (24 - 8 * level)) & 255;
        } else {
          const int l = level - 4;
          if (d != key || (l > 0 && ((uint32_t)i >> (24 - 8 * l)) != idx)) return;
          at = ((uint32_t)i >> (16 - 8 * l)) & 255;
        }
        atomicAdd(&g.hcount[at], 1u);
        atomicAdd(&g.hmass[at], s_mass(x, M, r.inv_t, a.unit, g.tab));
      });
      __syncthreads();
      if (wave == 0) {
        u64 t[4], w[4], st = 0, sw = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[e] = g.hmass[4 * lane + e];
          t[e] = by_mass ? w[e] : g.hcount[4 * lane + e];
          st += t[e];
          sw += w[e];
        }
        u64 run = ahead + s_wave_scan(st, lane) - st, runw = aheadw + s_wave_scan(sw, lane) - sw;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (run < target && run + t[e] >= target) {
            g.digit = 4 * lane + e;
            g.sum = run;
            g.to_mass = level == 6 ? runw + w[e] : runw;
          }
          run += t[e];
          runw += w[e];
        }
      }
      __syncthreads();
      ahead = g.sum;
      aheadw = g.to_mass;
      if (level < 4) key = (key << 8) | g.digit;
      else idx = (idx << 8) | g.digit;
      __syncthreads();
    }
    if (tid == 0) {
      g.key = ~key;
      g.idx = (int)idx;
    }
    __syncthreads();
  };

  SampleKept kept{kSBins - 1, 0, 0x7fffffff};
  u64 Z = g.mass[kSBins - 1];
  if (r.k > 0) {
    const int b = bin_of_count((uint32_t)r.k);
    if (g.count[b] == (uint32_t)r.k) {
      kept.b = b;
      Z = g.mass[b];
    } else {
      border(b, kept, (uint32_t)r.k - count_below(b), false);
      kept = {b, g.key, g.idx};
      Z = mass_below(b) + g.to_mass;
      __syncthreads();
    }
  }
  if (r.p < 1.f) {
    const double goal = ceil((double)fmaxf(r.p, 0.f) * (double)Z);
    const u64 target = goal < 1.0 ? 1 : min((u64)goal, Z);
    const int b = bin_of_mass(target);
    if (b < kept.b && count_below(b) + 1 == g.count[b]) {
      kept = {b, 0, 0x7fffffff};
      Z = g.mass[b];
    } else {
      border(b, kept, target - mass_below(b), true);
      kept = {b, g.key, g.idx};
      Z = mass_below(b) + g.to_mass;
      __syncthreads();
    }
  }
  if (r.m > 0.f) {
    // the smallest value of weight m or more: next to max + T ln m, found among its neighbours (more than 1: the largest value)
    const float guess = fminf((float)((double)M + log((double)r.m) * (double)r.t), M);
    uint32_t key = s_key(M);
    if (fabsf(M) < INFINITY && guess > -INFINITY) {
      const uint32_t mine = min(s_key(guess) + (uint32_t)lane - 32u, key);
      const u64 in = __builtin_amdgcn_ballot_w64(v_weight(s_unkey(mine), M, r.inv_t, g.tab) >= (double)r.m);
      if (in) key = __shfl(mine, __builtin_ctzll(in));
    } else if (fabsf(M) < INFINITY) {
      key = 0;
    }
    const int b = key ? s_bin(s_unkey(key), M, r.bins) : kSBins;
    if (b < kept.b || (b == kept.b && key > kept.key)) {
      const int n = g.count[b] == count_below(b) ? 0 : collect(b, kept);
      if (tid == 0) g.sum = 0;
      __syncthreads();
      if (n)
        for_bin(b, n, kept, [&](int, float x) {
          if (s_key(x) >= key) atomicAdd(&g.sum, s_mass(x, M, r.inv_t, a.unit, g.tab));
        });
      __syncthreads();
      kept = {b, key, b == kept.b && key == kept.key ? kept.idx : 0x7fffffff};
      Z = mass_below(b) + g.sum;
      __syncthreads();
    }
  }
  if (tid == 0) a.cut[row] = {a.unit / (double)Z, M, kept.b, kept.key, kept.idx};
  if (!a.tokens) return;
  const float u = a.u[(int64_t)(row / a.P) * a.ub];
  const double goal = floor(fmax((double)u, 0.0) * (double)Z);
  const u64 target = goal >= (double)Z ? Z : min((u64)goal + 1, Z);
  const int b = bin_of_mass(target);
  border(b, kept, target - mass_below(b), true);
  if (tid == 0) a.tokens[row] = g.idx;
}

template <int OUT>
__global__ __launch_bounds__(256) void sample_write_kernel(SampleArgs a) {
  const int tid = threadIdx.x, row = blockIdx.y;
  const SampleRow r = s_row(a, row);
  const SampleQuads s(r.x, a.V);
  const SampleCut c = a.cut[row];
  const SampleKept kept{c.b, c.key, c.idx};
  __shared__ double tab[kVTab];
  exp2_table(tab, tid);
  __syncthreads();
  float* o = a.out + (int64_t)row * a.V;
  const bool vec = (((uintptr_t)o - 4 * (uintptr_t)s.ahead) & 15) == 0;
#pragma unroll
  for (int u = 0; u < kSChunk / 256; ++u) {
    const int q = blockIdx.x * kSChunk + tid + 256 * u;
    if (q >= s.n()) continue;
    const f32x4 x = s.load(q);
    const int i = 4 * q - s.ahead;
    f32x4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool in = kept.has(s_bin(x[e], c.max, r.bins), x[e], i + e);
      if (OUT == kSampleLogits) y[e] = in ? x[e] : -INFINITY;
      else y[e] = in ? (float)(v_weight(x[e], c.max, r.inv_t, tab) * c.scale) : 0.f;
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
  return rows * (kSBins * (sizeof(u64) + sizeof(uint32_t)) + sizeof(SampleCut) + ((s_chunks(V) + 3) & ~3) * sizeof(float));
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
  a.unit = __builtin_ldexp(1.0, 62 - bits);
  a.mass = (u64*)workspace;
  a.count = (uint32_t*)(a.mass + rows * kSBins);
  a.cut = (SampleCut*)(a.count + rows * kSBins);
  a.cmax = (float*)(a.cut + rows);
  a.tokens = tokens, a.out = out;
  const int64_t nq = (V + 3) / 4 + 1;
  a.R = (int)std::max<int64_t>(1, std::min<int64_t>((1024 + rows - 1) / rows, (nq + 1023) / 1024));
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const dim3 chunks(a.C, (unsigned)rows);
  hipLaunchKernelGGL(sample_max_kernel, chunks, dim3(256), 0, st, a);
  hipLaunchKernelGGL(sample_hist_kernel, dim3(a.R, (unsigned)rows), dim3(256), 0, st, a);
  hipLaunchKernelGGL(sample_pick_kernel, dim3((unsigned)rows), dim3(kSThreads), 0, st, a);
  if (out_kind == kSampleProbs) hipLaunchKernelGGL(sample_write_kernel<kSampleProbs>, chunks, dim3(256), 0, st, a);
  else if (out_kind == kSampleLogits) hipLaunchKernelGGL(sample_write_kernel<kSampleLogits>, chunks, dim3(256), 0, st, a);
  return hipGetLastError() == hipSuccess ? Q35_OK : Q35_ELAUNCH;
}
