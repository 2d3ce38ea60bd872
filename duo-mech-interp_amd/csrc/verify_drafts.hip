// Verification of drafted tokens against the target's probabilities, from given random numbers (the step behind a
// multi-token decode call; with no drafts it draws one token from the target's softmax).
//
//   p_i = softmax(logits[b, i] / temperature), q_i the draft's probabilities (1 at the draft when it has none)
//   draft i is kept while u[b, i] q_i(x_i) < p_i(x_i); the first refusal, at i = n, ends the row's drafts
//   one token more, from r = max(p_n - q_n, 0) behind a refusal and from p_n otherwise: the lowest index whose running
//   sum of r exceeds u[b, K] sum(r)
// Which token a number falls on is a comparison of running sums over the vocabulary, so exponentials and sums are formed
// in 64 bits (a flat distribution over 150 K tokens puts one draw in a hundred on the wrong side in 32); fp64
// multiply-adds run at the fp32 rate here. Temperature 0 is the argmax (lowest index, NaN never wins).
//
// Spread over the vocabulary in chunks of 4096. verify_stats_kernel leaves each chunk's maximum and sum, without the
// weight of the position's own draft: what is left of p behind a refused certain draft is then a sum of its own and not a
// difference. verify_draw_kernel, one block per row, folds the chunks of all positions, finds n, the chunk in which the
// random number falls and the token in it. A refusal with draft probabilities needs the sums of max(p - q, 0), which
// depend on n: verify_mass_kernel between the two forms them (every block of a row finds the same n, from the same numbers
// in the same order). Nothing depends on the order in which blocks run.
//
// Measured, V = 151,936: three rows of 4 certain drafts 11 us (statistics 5.3, draw 6.9: a launch and a chain of dependent
// loads each); 32 rows of 0 .. 8 drafts with probabilities 45 us (statistics 27 for 97 MB, 3.6 TB/s; mass 12; draw 8). Chunks
// of 8192, or several positions a block, measured slower: the statistics kernel hides its loads by many short blocks.
#include "q35_common.h"
#include "q35hip.h"

namespace q35 {

constexpr int kVChunk = 4096, kVPer = kVChunk / 256;
constexpr int kVMaxK = 255;

struct VStat {
  double sum;  // of exp((x - max) / temperature), without the draft's
  float max;   // over all values
  int idx;     // lowest index of the maximum
};
struct VerifyArgs {
  const float* x;
  int64_t xb, xp;  // strides of a row and of a position
  const int32_t* ids;
  int64_t idb;
  const float* q;
  int64_t qb, qp;
  const float* u;
  int64_t ub;
  const int32_t* lens;
  const float* temps;
  float temp;
  int K, V, C;
  VStat* st;
  float2* dv;    // [B][K + 1]: the draft's logit (NaN as -inf) and probability, where the draft is a token
  double* mass;  // [B][C], with draft probabilities: sums of max(p_n - q_n, 0) behind a refusal
  int32_t *n_out, *tokens;
};

__device__ __forceinline__ int v_len(const VerifyArgs& p, int b) {
  return p.lens ? min(max(load_uniform(p.lens + b), 0), p.K) : p.K;
}
// 32 log2(e) / temperature, 0 for the argmax (an infinite temperature leaves the tokens above -inf alike)
__device__ __forceinline__ double v_inv_temp(const VerifyArgs& p, int b) {
  const float t = p.temps ? __int_as_float(load_uniform(reinterpret_cast<const int32_t*>(p.temps) + b)) : p.temp;
  return t > 0.f ? fmax(32.0 * 1.4426950408889634074 / (double)t, 1e-300) : 0.0;
}
// The position's draft when it is a token, else -1
__device__ __forceinline__ int v_draft(const VerifyArgs& p, int b, int i, int len) {
  if (i >= len) return -1;
  const int id = p.ids[b * p.idb + i];
  return id >= 0 && id < p.V ? id : -1;
}

// 2^(z / 32) for z <= 0 to 2e-12 relative: z = 32 n + j + r with |r| <= 1/2, as 2^n 2^(j / 32) 2^(r / 32): a table in LDS (32
// entries of 8 bytes, one pair of banks each: no conflicts) and the Taylor series of e^(r ln 2 / 32) to r^4 (the rest is
// below (ln 2 / 64)^5 / 5! = 1.3e-12; z's own rounding adds 2^-53 |z| / 32). 11 operations of 64 bits where a series over
// |f| <= 1/2 to f^9 takes 14: they come on top of the loads in the passes over the vocabulary (statistics of 32 rows of up to
// 8 drafts: 28.7 us with 14, 26.3 with 11, 19.3 with one).
constexpr int kVTab = 32;
__device__ __forceinline__ double exp2_neg(double z, const double* tab) {
  constexpr double c1 = 0.69314718055994530942 / kVTab, c2 = c1 * c1 / 2.0, c3 = c1 * c2 / 3.0, c4 = c1 * c3 / 4.0;
  z = fmax(z, -1100.0 * kVTab);  // 0 from there on, also for -inf
  const double n = __builtin_rint(z), r = z - n;
  const int k = (int)n;
  const double e = __builtin_fma(__builtin_fma(__builtin_fma(__builtin_fma(c4, r, c3), r, c2), r, c1), r, 1.0);
  return __builtin_ldexp(e * tab[k & (kVTab - 1)], k >> 5);
}
// Threads 0 .. 31 fill the table (a barrier before its use is the caller's): the series of 2^f to f^13, |f| <= 1/2.
__device__ __forceinline__ void exp2_table(double* tab, int tid) {
  if (tid >= kVTab) return;
  constexpr double L = 0.69314718055994530942;
  const bool up = 2 * tid > kVTab;
  const double f = (double)(up ? tid - kVTab : tid) * (L / kVTab);
  double e = 1.0;
#pragma unroll
  for (int k = 13; k > 0; --k) e = __builtin_fma(e * (1.0 / k), f, 1.0);
  tab[tid] = up ? 2.0 * e : e;
}
// exp((x - m) / T) for x <= m (no NaN), inv_t = 32 log2(e) / T: 1 at the maximum, also an infinite one.
__device__ __forceinline__ double v_weight(float x, float m, double inv_t, const double* tab) {
  return x == m ? 1.0 : exp2_neg(((double)x - (double)m) * inv_t, tab);
}
// A NaN counts as -inf.
__device__ __forceinline__ float v_clean(float x) { return fmaxf(x, -INFINITY); }

__device__ __forceinline__ int wave_min_i32(int v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = min(v, __shfl_xor(v, o));
  return v;
}

// This thread's values of a chunk: element 4 (tid + 256 u) + e; `fill` past the end.
__device__ __forceinline__ void v_load_chunk(const float* row, int base, int V, int tid, float (&x)[kVPer],
                                             float fill) {
  if (base + kVChunk <= V && ((uintptr_t)row & 15) == 0) {
#pragma unroll
    for (int u = 0; u < kVPer / 4; ++u) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(row + base + 4 * (tid + 256 * u));
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * u + e] = v[e];
    }
  } else {
#pragma unroll
    for (int u = 0; u < kVPer / 4; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = base + 4 * (tid + 256 * u) + e;
        x[4 * u + e] = i < V ? row[i] : fill;
      }
  }
}
__device__ __forceinline__ int v_index(int base, int tid, int k) { return base + 4 * (tid + 256 * (k >> 2)) + (k & 3); }

__global__ __launch_bounds__(256) void verify_stats_kernel(VerifyArgs p) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int c = blockIdx.x, b = blockIdx.y / (p.K + 1), i = blockIdx.y % (p.K + 1), base = c * kVChunk;
  const int len = v_len(p, b);
  if (i > len) return;
  const double inv_t = v_inv_temp(p, b);
  const int draft = v_draft(p, b, i, len);
  const bool mine = draft >= base && draft < base + kVChunk;
  if (mine && tid == 0)
    p.dv[blockIdx.y] = {v_clean(p.x[b * p.xb + i * p.xp + draft]), p.q ? p.q[b * p.qb + i * p.qp + draft] : 1.f};
  float x[kVPer];
  v_load_chunk(p.x + b * p.xb + i * p.xp, base, p.V, tid, x, -INFINITY);
  __shared__ float sm[4];
  __shared__ int si[4];
  __shared__ double ss[4], tab[kVTab];
  exp2_table(tab, tid);
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < kVPer; ++k) {
    x[k] = v_clean(x[k]);
    m = fmaxf(m, x[k]);
  }
  m = wave_max_f32(m);
  if (lane == 0) sm[wave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  int idx = 0x7fffffff;
  double s = 0.0;
  if (inv_t > 0.0) {
    if (mine) {  // the draft's weight is no part of its chunk's sum
#pragma unroll
      for (int k = 0; k < kVPer; ++k)
        if (v_index(base, tid, k) == draft) x[k] = -INFINITY;
    }
    if (fabsf(m) < INFINITY) {
#pragma unroll
      for (int k = 0; k < kVPer; ++k) s += exp2_neg(((double)x[k] - (double)m) * inv_t, tab);
    } else {
#pragma unroll
      for (int k = 0; k < kVPer; ++k) s += x[k] == m ? 1.0 : 0.0;
    }
    s = wave_sum64(s);
  } else {
#pragma unroll
    for (int k = kVPer - 1; k >= 0; --k)
      if (x[k] == m) idx = v_index(base, tid, k);
    idx = wave_min_i32(idx);
  }
  if (lane == 0) {
    ss[wave] = s;
    si[wave] = idx;
  }
  __syncthreads();
  if (tid == 0) {
    const VStat r = {ss[0] + ss[1] + ss[2] + ss[3], m, min(min(si[0], si[1]), min(si[2], si[3]))};
    p.st[(size_t)blockIdx.y * p.C + c] = r;
  }
}

// The chunks of each position of row b folded: the maximum, its index, 1 / sum, and whether the draft is kept. The chunks
// of as many positions as fit are fetched together with the positions' drafts and what is asked of those, whatever the row's
// length (which arrives with them: no load waits for another), then one wave folds a position. Returns n once every thread
// has them.
constexpr int kVFold = 1024;  // chunks held at a time, and the most that a position may have
struct VFold {
  VStat st[kVFold];
  double inv_z[kVMaxK + 1];
  float max[kVMaxK + 1], x[kVMaxK + 1], q[kVMaxK + 1], u[kVMaxK + 1];
  int idx[kVMaxK + 1], keep[kVMaxK + 1], draft[kVMaxK + 1];
  double tab[kVTab];
};
template <int THREADS>
__device__ __forceinline__ int v_fold(const VerifyArgs& p, int b, int len, double inv_t, int tid, VFold& f) {
  const int lane = tid & 63, wave = tid >> 6, per = max(kVFold / p.C, 1);
  exp2_table(f.tab, tid);
  if (tid < p.K) {
    const int id = p.ids[b * p.idb + tid];
    const float2 d = p.dv[(size_t)b * (p.K + 1) + tid];
    f.x[tid] = d.x;
    f.q[tid] = d.y;
    f.u[tid] = p.u[b * p.ub + tid];
    f.draft[tid] = id >= 0 && id < p.V ? id : -1;
  }
  int i0 = 0;
  do {
    const int there = min(per, p.K + 1 - i0) * p.C;
    const VStat* src = p.st + ((size_t)b * (p.K + 1) + i0) * p.C;
    for (int k = tid; k < there; k += THREADS) f.st[k] = src[k];
    const int n = min(per, len + 1 - i0);
    __syncthreads();
    for (int j = wave; j < n; j += THREADS / 64) {
      const int i = i0 + j, draft = i < len ? f.draft[i] : -1;
      const VStat* st = f.st + j * p.C;
      float M = -INFINITY;
      for (int k = lane; k < p.C; k += 64) M = fmaxf(M, st[k].max);
      M = wave_max_f32(M);
      double z = 0.0;
      int idx = 0x7fffffff;
      for (int k = lane; k < p.C; k += 64) {
        const VStat s = st[k];
        if (s.max > -INFINITY) z += s.sum * v_weight(s.max, M, inv_t, f.tab);
        if (s.max == M) idx = min(idx, s.idx);
      }
      z = wave_sum64(z);
      if (!(inv_t > 0.0)) idx = wave_min_i32(idx);
      const double wd = draft >= 0 && M > -INFINITY ? v_weight(f.x[i], M, inv_t, f.tab) : 0.0;
      z += wd;
      if (lane == 0) {
        const double pr = inv_t > 0.0 ? wd / z : draft == idx ? 1.0 : 0.0;
        f.inv_z[i] = 1.0 / z;
        f.max[i] = M;
        f.idx[i] = idx;
        f.keep[i] = draft >= 0 && M > -INFINITY && (double)f.u[i] * (double)f.q[i] < pr;
      }
    }
    __syncthreads();
    i0 += per;
  } while (i0 <= len);
  int n = 0;
  while (n < len && f.keep[n]) ++n;
  return n;
}

// (One chunk a block, each with a fold of its own: four chunks to a block of 1024 threads that share one measured 19.4 us
// against 13.5 for 32 rows of up to eight drafts.)
__global__ __launch_bounds__(256) void verify_mass_kernel(VerifyArgs p) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int c = blockIdx.x, b = blockIdx.y, len = v_len(p, b), base = c * kVChunk;
  const double inv_t = v_inv_temp(p, b);
  if (!(inv_t > 0.0) || len == 0) return;
  __shared__ VFold f;
  const int n = v_fold<256>(p, b, len, inv_t, tid, f);
  const float M = f.max[n];
  if (n == len || !(M > -INFINITY)) return;  // nothing was refused: the draw takes the chunks' own sums
  const double inv_z = f.inv_z[n];
  float x[kVPer], q[kVPer];
  v_load_chunk(p.x + b * p.xb + n * p.xp, base, p.V, tid, x, -INFINITY);
  v_load_chunk(p.q + b * p.qb + n * p.qp, base, p.V, tid, q, 0.f);
  double s = 0.0;
#pragma unroll
  for (int k = 0; k < kVPer; ++k) s += fmax(v_weight(v_clean(x[k]), M, inv_t, f.tab) * inv_z - (double)q[k], 0.0);
  s = wave_sum64(s);
  __shared__ double ss[4];
  if (lane == 0) ss[wave] = s;
  __syncthreads();
  if (tid == 0) p.mass[(size_t)b * p.C + c] = ss[0] + ss[1] + ss[2] + ss[3];
}

__global__ __launch_bounds__(1024) void verify_draw_kernel(VerifyArgs p) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, b = blockIdx.x;
  const int len = v_len(p, b);
  const double inv_t = v_inv_temp(p, b);
  __shared__ VFold f;
  __shared__ double pre[16], chunk_w[kVFold];
  __shared__ int s_token, s_last;
  const float us = p.u[b * p.ub + p.K];
  const int n = v_fold<1024>(p, b, len, inv_t, tid, f);
  const float M = f.max[n];
  const bool refused = n < len;
  const int draft = refused ? f.draft[n] : -1;
  int token = M > -INFINITY ? f.idx[n] : 0;
  if (inv_t > 0.0 && M > -INFINITY) {
    const double inv_z = f.inv_z[n];
    const VStat* st = p.st + ((size_t)b * (p.K + 1) + n) * p.C;
    // Weight of each chunk into LDS: kind 0 of max(p - q, 0), kind 1 of p without the draft, kind 2 of p
    const bool here = (len + 1) * p.C <= kVFold;  // the position's chunks are still in LDS
    auto weights = [&](int kind) {
      for (int k = tid; k < p.C; k += 1024) {
        double w;
        if (kind == 0) {
          w = p.mass[(size_t)b * p.C + k];
        } else {
          const VStat s = here ? f.st[n * p.C + k] : st[k];
          w = s.max > -INFINITY ? s.sum * v_weight(s.max, M, inv_t, f.tab) : 0.0;
          if (kind == 2 && draft >= 0 && k == draft / kVChunk) w += v_weight(f.x[n], M, inv_t, f.tab);
          w *= inv_z;
        }
        chunk_w[k] = w;
      }
      __syncthreads();
    };
    int kind = !refused ? 2 : p.q ? 0 : 1;
    weights(kind);
    double tot = 0.0;
    for (int k0 = 0; k0 < p.C; k0 += 64) tot += wave_sum64(k0 + lane < p.C ? chunk_w[k0 + lane] : 0.0);
    if (!(tot > 0.0)) {  // (the same for all waves) nothing is left behind the refusal, q = p to the last bit: p itself
      kind = 2;
      __syncthreads();
      weights(kind);
      tot = 0.0;
      for (int k0 = 0; k0 < p.C; k0 += 64) tot += wave_sum64(k0 + lane < p.C ? chunk_w[k0 + lane] : 0.0);
    }
    // every wave finds the chunk
    const double all = (double)us * tot;
    double run = 0.0, before = 0.0;
    int chunk = -1, last_chunk = 0;
    for (int k0 = 0; k0 < p.C && chunk < 0; k0 += 64) {
      const double w = k0 + lane < p.C ? chunk_w[k0 + lane] : 0.0, inc = wave_scan64(w);
      const unsigned long long over = __builtin_amdgcn_ballot_w64(w > 0.0 && run + inc > all);
      const unsigned long long some = __builtin_amdgcn_ballot_w64(w > 0.0);
      if (some) last_chunk = k0 + 63 - __builtin_clzll(some);
      if (over) {
        const int l = __builtin_ctzll(over);
        chunk = k0 + l;
        before = run + __shfl(inc - w, l);
      }
      run += __shfl(inc, 63);
    }
    const double target = chunk >= 0 ? all - before : INFINITY;  // in no chunk: the last token with weight
    if (tid == 0) {
      s_token = 0x7fffffff;
      s_last = 0;
    }
    constexpr int PER = kVChunk / 1024;
    const int base = (chunk >= 0 ? chunk : last_chunk) * kVChunk + tid * PER;
    const float* xr = p.x + b * p.xb + n * p.xp;
    const float* qr = kind == 0 ? p.q + b * p.qb + n * p.qp : nullptr;
    double w[PER], sum = 0.0;
    int last = -1;
    float xv[PER], qv[PER] = {0.f, 0.f, 0.f, 0.f};
    static_assert(PER == 4, "one vector a thread");
    auto quad = [&](const float* row, float fill, float (&v)[PER]) {
      if (base + PER <= p.V && ((uintptr_t)row & 15) == 0) {
        const f32x4 w = *reinterpret_cast<const f32x4*>(row + base);
#pragma unroll
        for (int k = 0; k < PER; ++k) v[k] = w[k];
      } else {
#pragma unroll
        for (int k = 0; k < PER; ++k) v[k] = base + k < p.V ? row[base + k] : fill;
      }
    };
    quad(xr, -INFINITY, xv);
    if (kind == 0) quad(qr, 0.f, qv);
#pragma unroll
    for (int k = 0; k < PER; ++k) xv[k] = v_clean(xv[k]);
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      double v = v_weight(xv[k], M, inv_t, f.tab) * inv_z;
      if (kind == 0) v = fmax(v - (double)qv[k], 0.0);
      if (kind == 1 && base + k == draft) v = 0.0;
      w[k] = v;
      sum += v;
      if (v > 0.0) last = base + k;
    }
    // sums before this thread's values: a scan within the wave, then over the waves
    const double inc = wave_scan64(sum);
    if (lane == 63) pre[wave] = inc;
    __syncthreads();
    run = inc - sum;
    for (int k = 0; k < wave; ++k) run += pre[k];
    int hit = 0x7fffffff;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      run += w[k];
      if (run > target && w[k] > 0.0) hit = min(hit, base + k);
    }
    // the wave's first hit and last weight are those of its first and last such lane (1024 atomics on one word took 8 us)
    const unsigned long long hits = __builtin_amdgcn_ballot_w64(hit != 0x7fffffff);
    const unsigned long long some = __builtin_amdgcn_ballot_w64(last >= 0);
    if (hits && lane == __builtin_ctzll(hits)) atomicMin(&s_token, hit);
    if (some && lane == 63 - __builtin_clzll(some)) atomicMax(&s_last, last);
    __syncthreads();
    token = s_token != 0x7fffffff ? s_token : s_last;
  }
  if (tid == 0) p.n_out[b] = n;
  for (int i = tid; i <= p.K; i += 1024)
    p.tokens[(size_t)b * (p.K + 1) + i] = i < n ? p.ids[b * p.idb + i] : i == n ? token : -1;
}

static int64_t v_chunks(int64_t V) { return (V + kVChunk - 1) / kVChunk; }

}  // namespace q35

extern "C" size_t q35_verify_drafts_workspace_bytes(int64_t B, int64_t K, int64_t V) {
  using namespace q35;
  if (B <= 0 || K < 0 || V <= 0 || B > 65535 || K > kVMaxK || V > (int64_t)kVFold * kVChunk || B * (K + 1) > 65535) return 0;
  const size_t C = v_chunks(V);
  return (size_t)B * (K + 1) * C * sizeof(VStat) + (size_t)B * C * sizeof(double) + (size_t)B * (K + 1) * sizeof(float2);
}

extern "C" int q35_verify_drafts(const float* logits, int64_t l_sb, int64_t l_sp, const int32_t* draft_ids, int64_t d_sb,
                                 const float* draft_probs, int64_t p_sb, int64_t p_sp, const float* u, int64_t u_sb,
                                 const int32_t* lens, const float* temperatures, float temperature,
                                 int32_t* n_accept, int32_t* tokens, int64_t B, int64_t K, int64_t V, void* workspace,
                                 size_t workspace_bytes, q35_stream_t stream) {
  using namespace q35;
  if (!logits || !u || !n_accept || !tokens || B <= 0 || K < 0 || V <= 0) return Q35_EINVAL;
  if (K > 0 && !draft_ids) return Q35_EINVAL;
  if (l_sb < 0 || d_sb < 0 || p_sb < 0 || u_sb < 0 || (K > 0 && l_sp < V) || (draft_probs && K > 1 && p_sp < V))
    return Q35_EINVAL;
  if (!(temperature >= 0.f)) return Q35_EINVAL;
  const size_t need = q35_verify_drafts_workspace_bytes(B, K, V);
  if (need == 0) return Q35_EUNSUPPORTED;
  if (!workspace || workspace_bytes < need || (uintptr_t)workspace & 15) return Q35_EWORKSPACE;
  const int C = (int)v_chunks(V);
  VStat* st = (VStat*)workspace;
  double* mass = (double*)(st + (size_t)B * (K + 1) * C);
  float2* dv = (float2*)(mass + (size_t)B * C);
  const VerifyArgs a{logits, l_sb, l_sp, draft_ids, d_sb, K > 0 ? draft_probs : nullptr, p_sb, p_sp, u, u_sb, lens,
                     temperatures, temperature, (int)K, (int)V, C, st, dv, mass, n_accept, tokens};
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(verify_stats_kernel, dim3(C, (unsigned)(B * (K + 1))), dim3(256), 0, s, a);
  if (a.q) hipLaunchKernelGGL(verify_mass_kernel, dim3(C, (unsigned)B), dim3(256), 0, s, a);
  hipLaunchKernelGGL(verify_draw_kernel, dim3((unsigned)B), dim3(1024), 0, s, a);
  return hipGetLastError() == hipSuccess ? Q35_OK : Q35_ELAUNCH;
}
