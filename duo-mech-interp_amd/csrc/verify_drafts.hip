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
// Three launches, each spread over the vocabulary in chunks of 4096: chunk maxima and sums of every position that a row
// has; then each block of a row folds those of all its positions, finds n (every block the same, from the same numbers in
// the same order) and sums its chunk of r; then one block per row finds the chunk and the token. Nothing depends on the
// order in which blocks run.
#include "q35_common.h"
#include "q35hip.h"

namespace q35 {

constexpr int kVChunk = 4096, kVPer = kVChunk / 256;
constexpr int kVMaxK = 255;

struct VStat {
  double sum;  // of exp((x - max) / temperature)
  float max;
  int idx;     // lowest index of the maximum
};
struct VRow {
  double inv_z;
  float max;
  int n, idx, refused;
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
  double* mass;  // [B][C][2]: sums of r behind a refusal (left) and of p
  VRow* row;
  int32_t *n_out, *tokens;
};

__device__ __forceinline__ int v_len(const VerifyArgs& p, int b) {
  return p.lens ? min(max(p.lens[b], 0), p.K) : p.K;
}
// 1 / temperature, 0 for the argmax
__device__ __forceinline__ double v_inv_temp(const VerifyArgs& p, int b) {
  const float t = p.temps ? p.temps[b] : p.temp;
  return t > 0.f ? 1.0 / (double)t : 0.0;
}
// exp((x - m) / T): 1 at the maximum (also an infinite one), 0 for NaN
__device__ __forceinline__ double v_weight(float x, float m, double inv_t) {
  return x == m ? 1.0 : x < m ? exp(((double)x - (double)m) * inv_t) : 0.0;
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ float wave_max_f32(float v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}
__device__ __forceinline__ int wave_min_i32(int v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = min(v, __shfl_xor(v, o));
  return v;
}

// This thread's values of a chunk: element 4 (tid + 256 u) + e; -inf past the end.
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

__global__ __launch_bounds__(256) void verify_stats_kernel(VerifyArgs p) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int c = blockIdx.x, b = blockIdx.y / (p.K + 1), i = blockIdx.y % (p.K + 1);
  if (i > v_len(p, b)) return;
  const double inv_t = v_inv_temp(p, b);
  float x[kVPer];
  v_load_chunk(p.x + b * p.xb + i * p.xp, c * kVChunk, p.V, tid, x, -INFINITY);
  __shared__ float sm[4];
  __shared__ int si[4];
  __shared__ double ss[4];
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < kVPer; ++k) m = fmaxf(m, x[k]);
  m = wave_max_f32(m);
  if (lane == 0) sm[wave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  int idx = 0x7fffffff;
  double s = 0.0;
  if (inv_t > 0.0) {
#pragma unroll
    for (int k = 0; k < kVPer; ++k) s += v_weight(x[k], m, inv_t);
  } else {
#pragma unroll
    for (int k = kVPer - 1; k >= 0; --k)
      if (x[k] == m) idx = c * kVChunk + 4 * (tid + 256 * (k >> 2)) + (k & 3);
  }
  s = wave_sum_f64(s);
  idx = wave_min_i32(idx);
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

// r at one value: behind a refusal (left) and without one
__device__ __forceinline__ double v_left(double w, float q, bool has_q, bool is_draft) {
  return fmax(w - (has_q ? (double)q : is_draft ? 1.0 : 0.0), 0.0);
}

__global__ __launch_bounds__(256) void verify_mass_kernel(VerifyArgs p) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int c = blockIdx.x, b = blockIdx.y, len = v_len(p, b);
  const double inv_t = v_inv_temp(p, b);
  __shared__ double iz[kVMaxK + 1];
  __shared__ float mx[kVMaxK + 1];
  __shared__ int ix[kVMaxK + 1], keep[kVMaxK + 1];
  for (int i = wave; i <= len; i += 4) {
    const VStat* st = p.st + ((size_t)b * (p.K + 1) + i) * p.C;
    float M = -INFINITY;
    for (int k = lane; k < p.C; k += 64) M = fmaxf(M, st[k].max);
    M = wave_max_f32(M);
    double z = 0.0;
    int idx = 0x7fffffff;
    for (int k = lane; k < p.C; k += 64) {
      const VStat s = st[k];
      if (s.max > -INFINITY) z += s.sum * v_weight(s.max, M, inv_t);
      if (s.max == M) idx = min(idx, s.idx);
    }
    z = wave_sum_f64(z);
    idx = wave_min_i32(idx);
    int ok = 0;
    if (i < len) {
      const int id = p.ids[b * p.idb + i];
      if (id >= 0 && id < p.V && M > -INFINITY) {
        const double pr = inv_t > 0.0 ? v_weight(p.x[b * p.xb + i * p.xp + id], M, inv_t) / z : id == idx ? 1.0 : 0.0;
        const double q = p.q ? (double)p.q[b * p.qb + i * p.qp + id] : 1.0;
        ok = (double)p.u[b * p.ub + i] * q < pr;
      }
    }
    if (lane == 0) {
      iz[i] = 1.0 / z;
      mx[i] = M;
      ix[i] = idx;
      keep[i] = ok;
    }
  }
  __syncthreads();
  int n = 0;
  while (n < len && keep[n]) ++n;
  const bool refused = n < len;
  const float M = mx[n];
  const double inv_z = iz[n];
  if (c == 0 && tid == 0) {
    const VRow r = {inv_z, M, n, M > -INFINITY ? ix[n] : 0, refused};
    p.row[b] = r;
  }
  if (!(inv_t > 0.0) || !(M > -INFINITY)) return;
  float x[kVPer], q[kVPer];
  v_load_chunk(p.x + b * p.xb + n * p.xp, c * kVChunk, p.V, tid, x, -INFINITY);
  const bool has_q = refused && p.q;
  if (has_q) v_load_chunk(p.q + b * p.qb + n * p.qp, c * kVChunk, p.V, tid, q, 0.f);
  const int draft = refused && !p.q ? p.ids[b * p.idb + n] : -1;
  double sl = 0.0, sp = 0.0;
#pragma unroll
  for (int k = 0; k < kVPer; ++k) {
    const double w = v_weight(x[k], M, inv_t) * inv_z;
    sp += w;
    sl += v_left(w, has_q ? q[k] : 0.f, has_q, c * kVChunk + 4 * (tid + 256 * (k >> 2)) + (k & 3) == draft);
  }
  sl = wave_sum_f64(sl);
  sp = wave_sum_f64(sp);
  __shared__ double s2[4][2];
  if (lane == 0) {
    s2[wave][0] = sl;
    s2[wave][1] = sp;
  }
  __syncthreads();
  if (tid < 2) p.mass[((size_t)b * p.C + c) * 2 + tid] = s2[0][tid] + s2[1][tid] + s2[2][tid] + s2[3][tid];
}

__global__ __launch_bounds__(256) void verify_draw_kernel(VerifyArgs p) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, b = blockIdx.x;
  const VRow r = p.row[b];
  const double inv_t = v_inv_temp(p, b);
  __shared__ double pre[256];
  __shared__ double s_target;
  __shared__ int s_chunk, s_kind, s_token, s_last;
  int token = r.idx;
  if (inv_t > 0.0 && r.max > -INFINITY) {
    const double* ms = p.mass + (size_t)b * p.C * 2;
    if (tid == 0) {
      // sums over the chunks in order; what is left behind a refusal may be nothing (q = p to the last bit): then p
      double tot = 0.0, all = 0.0;
      for (int k = 0; k < p.C; ++k) {
        tot += ms[2 * k];
        all += ms[2 * k + 1];
      }
      const int kind = r.refused && tot > 0.0 ? 0 : 1;
      const double target = (double)p.u[b * p.ub + p.K] * (kind ? all : tot);
      double run = 0.0;
      int chunk = -1, last = 0;
      for (int k = 0; k < p.C; ++k) {
        const double m = ms[2 * k + kind];
        if (m > 0.0) last = k;
        if (chunk < 0) {
          if (run + m > target) chunk = k;
          else run += m;
        }
      }
      if (chunk < 0) {
        chunk = last;
        run = 0.0;
        s_target = INFINITY;  // none of them: its last value with weight
      } else {
        s_target = target - run;
      }
      s_chunk = chunk;
      s_kind = kind;
      s_token = 0x7fffffff;
      s_last = 0;
    }
    __syncthreads();
    const int base = s_chunk * kVChunk + tid * kVPer;
    const bool left = s_kind == 0, has_q = left && p.q;
    const int draft = left && !p.q ? p.ids[b * p.idb + r.n] : -1;
    const float* xr = p.x + b * p.xb + r.n * p.xp;
    const float* qr = has_q ? p.q + b * p.qb + r.n * p.qp : nullptr;
    double w[kVPer], sum = 0.0;
    int last = -1;
#pragma unroll
    for (int k = 0; k < kVPer; ++k) {
      const int i = base + k;
      double v = i < p.V ? v_weight(xr[i], r.max, inv_t) * r.inv_z : 0.0;
      if (left && i < p.V) v = v_left(v, has_q ? qr[i] : 0.f, has_q, i == draft);
      w[k] = v;
      sum += v;
      if (v > 0.0) last = i;
    }
    // sums before this thread's values: a scan within the wave, then over the waves
    double inc = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double v = __shfl_up(inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 63) pre[wave] = inc;
    __syncthreads();
    double run = inc - sum;
    for (int k = 0; k < wave; ++k) run += pre[k];
    const double target = s_target;
    int hit = 0x7fffffff;
#pragma unroll
    for (int k = 0; k < kVPer; ++k) {
      run += w[k];
      if (run > target && w[k] > 0.0) hit = min(hit, base + k);
    }
    if (hit != 0x7fffffff) atomicMin(&s_token, hit);
    if (last >= 0) atomicMax(&s_last, last);
    __syncthreads();
    token = s_token != 0x7fffffff ? s_token : s_last;
  }
  if (tid == 0) p.n_out[b] = r.n;
  for (int i = tid; i <= p.K; i += 256)
    p.tokens[(size_t)b * (p.K + 1) + i] = i < r.n ? p.ids[b * p.idb + i] : i == r.n ? token : -1;
}

static int64_t v_chunks(int64_t V) { return (V + kVChunk - 1) / kVChunk; }

}  // namespace q35

extern "C" size_t q35_verify_drafts_workspace_bytes(int64_t B, int64_t K, int64_t V) {
  using namespace q35;
  if (B <= 0 || K < 0 || V <= 0 || B > 65535 || K > kVMaxK || V > 0x7fff0000 || B * (K + 1) > 65535) return 0;
  const size_t C = v_chunks(V);
  return (size_t)B * (K + 1) * C * sizeof(VStat) + (size_t)B * C * 2 * sizeof(double) + (size_t)B * sizeof(VRow);
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
  VRow* row = (VRow*)(mass + (size_t)B * C * 2);
  const VerifyArgs a{logits, l_sb, l_sp, draft_ids, d_sb, K > 0 ? draft_probs : nullptr, p_sb, p_sp, u, u_sb, lens,
                     temperatures, temperature, (int)K, (int)V, C, st, mass, row, n_accept, tokens};
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(verify_stats_kernel, dim3(C, (unsigned)(B * (K + 1))), dim3(256), 0, s, a);
  hipLaunchKernelGGL(verify_mass_kernel, dim3(C, (unsigned)B), dim3(256), 0, s, a);
  hipLaunchKernelGGL(verify_draw_kernel, dim3((unsigned)B), dim3(256), 0, s, a);
  return hipGetLastError() == hipSuccess ? Q35_OK : Q35_ELAUNCH;
}
