// Products in 8-bit integers with one scale per token and one per output channel, and the rows in 8 bits that they take.
//
//   s[m] = fp32(max_k |x[m, k]| / 127), q[m, k] = rint(x[m, k] / s[m]) (half to even)
//   y[m, n] = (sum_k q[m, k] W[n, k]) s[m] ws[n]
//
// The sum is exact (int32, K up to 65536), so it depends on no order and every kernel here gives the same bits. A code is a
// rounding decision: quotient and norm are formed in 64 bits, whatever the order of a sum.
#include "gemm_common.h"

namespace q35 {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

// ---------------------------------------------------------------------------------------------------------------
// Rows in 8 bits, one block a row, held in registers: PER quads of values a thread.

// rint(x / s), half to even: x, s exact, |x / s| <= 127.5. The remainder settles what the product with 1 / s left undecided.
__device__ __forceinline__ int i8_code(double x, double s, double inv) {
  double t = __builtin_rint(x * inv);
  const double r = __builtin_fma(-t, s, x), a = fabs(r) * 2.0;  // exact: t has 8 bits, s 24
  if (a > s || (a == s && ((int)t & 1))) t += r > 0.0 ? 1.0 : -1.0;
  return (int)fmin(fmax(t, -127.0), 127.0);
}

template <typename Tx, bool NORM, int PER>
__global__ __launch_bounds__(256) void rows_i8_kernel(Tx* __restrict__ x, int64_t ldx, const float* __restrict__ y,
                                                      int64_t ldy, const float* __restrict__ w, int8_t* __restrict__ q,
                                                      float* __restrict__ s, int K, float eps) {
  const int64_t m = blockIdx.x;
  const int tid = threadIdx.x;
  Tx* xr = x + m * ldx;
  double v[PER][4];
  double ss = 0.0;
  float mx = 0.f;
  bool odd = false;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int c = 4 * (tid + 256 * i);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[i][e] = 0.0;
    if (c < K) {
      f32x4 f;
      if constexpr (sizeof(Tx) == 4) {
        f = *reinterpret_cast<const f32x4*>(xr + c);
      } else {
        const u32x2 r = *reinterpret_cast<const u32x2*>(xr + c);
        f = f32x4{bf16lo(r.x), bf16hi(r.x), bf16lo(r.y), bf16hi(r.y)};
      }
      if constexpr (NORM) {
        if (y) {
          const f32x4 a = *reinterpret_cast<const f32x4*>(y + m * ldy + c);
#pragma unroll
          for (int e = 0; e < 4; ++e) f[e] += a[e];
          *reinterpret_cast<f32x4*>(xr + c) = f;
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[i][e] = f[e];
        if constexpr (NORM) ss += v[i][e] * v[i][e];
      }
    }
  }
  __shared__ double red[4];
  __shared__ float redm[4];
  __shared__ int redo[4];
  if constexpr (NORM) {
    ss = wave_sum64(ss);
    if ((tid & 63) == 0) red[tid >> 6] = ss;
    __syncthreads();
    const double r = 1.0 / sqrt((red[0] + red[1] + red[2] + red[3]) / (double)K + (double)eps);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = 4 * (tid + 256 * i);
      if (c < K) {
        const f32x4 wv = *reinterpret_cast<const f32x4*>(w + c);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[i][e] = v[i][e] * r * (1.0 + (double)wv[e]);
      }
    }
  }
  double md = 0.0;
#pragma unroll
  for (int i = 0; i < PER; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      odd |= !(fabs(v[i][e]) < INFINITY);
      md = fmax(md, fabs(v[i][e]));
    }
  // the scale of the largest: fp32(max / 127) is monotone, so the maximum of the rounded quotients
  mx = wave_max_f32((float)(md / 127.0));
  const bool any = __builtin_amdgcn_ballot_w64(odd) != 0;
  if ((tid & 63) == 0) {
    redm[tid >> 6] = mx;
    redo[tid >> 6] = any;
  }
  __syncthreads();
  // a row that holds a value that is not finite has the scale NaN, and its products are NaN
  const float sc = fmaxf(fmaxf(redm[0], redm[1]), fmaxf(redm[2], redm[3]));
  const bool bad = redo[0] | redo[1] | redo[2] | redo[3] || !(sc < INFINITY);
  if (tid == 0) s[m] = bad ? __int_as_float(0x7fc00000) : sc;
  const bool none = bad || !(sc > 0.f);
  const double sd = none ? 1.0 : (double)sc, inv = 1.0 / sd;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int c = 4 * (tid + 256 * i);
    if (c < K) {
      uint32_t o = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) o |= (uint32_t)(uint8_t)(none ? 0 : i8_code(v[i][e], sd, inv)) << (8 * e);
      *reinterpret_cast<uint32_t*>(q + m * K + c) = o;
    }
  }
}

template <typename Tx, bool NORM>
static int rows_i8_launch(Tx* x, int64_t ldx, const float* y, int64_t ldy, const float* w, int8_t* q, float* s, int64_t M,
                          int64_t K, float eps, hipStream_t st) {
#define Q35_ROWS(PER)                                                                                                   \
  hipLaunchKernelGGL((rows_i8_kernel<Tx, NORM, PER>), dim3((unsigned)M), dim3(256), 0, st, x, ldx, y, ldy, w, q, s, (int)K, eps)
  if (K <= 1024) Q35_ROWS(1);
  else if (K <= 2048) Q35_ROWS(2);
  else if (K <= 4096) Q35_ROWS(4);
  else if (K <= 8192) Q35_ROWS(8);
  else Q35_ROWS(16);
#undef Q35_ROWS
  return hipGetLastError() == hipSuccess ? Q35_OK : Q35_ELAUNCH;
}

// ---------------------------------------------------------------------------------------------------------------
// Tiles of BM x BN outputs, a wave 32 MT x 32 NT of them. Rows of q and W go to LDS by DMA in stages of 64 inputs (rows of 64
// bytes, 16-byte chunk c at c ^ ((row >> 2) & 3): 16 consecutive lanes of a fragment read fall in distinct slots).
constexpr int kIK = 64, kINS = 4;

struct GemmI8Args {
  const int8_t* q;
  int64_t ldq;
  const float* qs;
  const int8_t* W;
  const float* ws;
  float* y;
  int64_t ldy;
  int M, N, K;
  const q35_push* pushes;
  int npush, T;
  GemmCap cap;
};

// lane of a 1 KB copy of 16 rows -> its row and 16-byte chunk
__device__ __forceinline__ int i8_copy_row(int lane) { return lane >> 2; }
__device__ __forceinline__ int i8_copy_chunk(int lane) { return (lane & 3) ^ ((lane >> 4) & 3); }

template <int MT, int NT, int WR, int WC, int EPI>
__global__ __launch_bounds__(64 * WR * WC) void gemm_i8_kernel(GemmI8Args p) {
  constexpr int BM = 32 * MT * WR, BN = 32 * NT * WC, NW = WR * WC;
  constexpr int UA = BM / 16, U = (BM + BN) / 16 / NW;  // copies of a stage's q, copies per wave
  constexpr int SB = (BM + BN) * kIK;
  static_assert((BM + BN) / 16 % NW == 0, "copies are dealt evenly");
  __shared__ __attribute__((aligned(16))) char smem[kINS * SB];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wv / WC, wc = wv % WC, l32 = lane & 31, lh = lane >> 5;
  const int nbn = (p.N + BN - 1) / BN, ntiles = nbn * ((p.M + BM - 1) / BM);
  const int xj = (int)(blockIdx.x & 7), xq = ntiles >> 3, xr = ntiles & 7;
  const int tile = xj * xq + min(xj, xr) + (int)(blockIdx.x >> 3);
  const int bm = tile / nbn, bn = tile - bm * nbn;
  const int m0 = bm * BM, n0 = bn * BN, KT = p.K / kIK;

  const int8_t* qb = p.q + (int64_t)m0 * p.ldq;
  const int8_t* wb = p.W + (int64_t)n0 * p.K;
  uint32_t src[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int u = wv + NW * i, row = 16 * (u < UA ? u : u - UA) + i8_copy_row(lane);
    src[i] = (u < UA ? (uint32_t)min(row, p.M - 1 - m0) * (uint32_t)p.ldq : (uint32_t)min(row, p.N - 1 - n0) * (uint32_t)p.K) +
             16 * i8_copy_chunk(lane);
  }
  const uint32_t lds0 = gemm_lds_u32(smem);
  auto issue = [&](int s) {
    const uint32_t base = lds0 + (s % kINS) * SB;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int u = wv + NW * i;
      gemm_dma16s((u < UA ? qb : wb) + (int64_t)s * kIK, src[i], base + u * 1024);
    }
  };
  const int ra = wr * 32 * MT + l32, rb = wc * 32 * NT + l32;
  uint32_t ao[2], bo[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int ch = ((2 * lh + j) ^ ((l32 >> 2) & 3)) << 4;
    ao[j] = ra * kIK + ch;
    bo[j] = (BM + rb) * kIK + ch;
  }
  i32x16 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;

  for (int s = 0; s < kINS - 1; ++s)
    if (s < KT) issue(s);
  for (int s = 0; s < KT; ++s) {
    const int ahead = min(KT - 1 - s, kINS - 2);
    if (ahead >= 2) gemm_wait_vm<2 * U>();
    else if (ahead == 1) gemm_wait_vm<U>();
    else gemm_wait_vm<0>();
    lds_barrier();
    if (s + kINS - 1 < KT) issue(s + kINS - 1);
    const char* st = smem + (s % kINS) * SB;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      i32x4 a[MT], b[NT];
#pragma unroll
      for (int i = 0; i < MT; ++i) a[i] = *reinterpret_cast<const i32x4*>(st + ao[j] + i * 32 * kIK);
#pragma unroll
      for (int i = 0; i < NT; ++i) b[i] = *reinterpret_cast<const i32x4*>(st + bo[j] + i * 32 * kIK);
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int k = 0; k < NT; ++k) acc[i][k] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[i], b[k], acc[i][k], 0, 0, 0);
    }
  }

  // The results leave through LDS, a wave's 32 rows at a time in an area of its own, so that a store holds whole runs of a row:
  // a lane takes CL columns of a row (gate and up of a neuron meet in it).
  constexpr int CW = 32 * NT, LD = CW + 4, CL = EPI == kGemmSwiglu ? 8 : 4, LR = CW / CL, RS = 64 / LR;
  static_assert(NW * 32 * LD * 4 <= kINS * SB, "the stages hold the waves' areas");
  lds_barrier();  // every wave has read its last fragments
  float* t = reinterpret_cast<float*>(smem) + wv * 32 * LD;
  const int c = CL * (lane % LR), n = n0 + wc * CW + c;
  float sn[CL];
#pragma unroll
  for (int e = 0; e < CL; ++e) sn[e] = p.ws[min(n + e, p.N - 1)];
  const bool pushes_here = EPI == kGemmSwiglu && gemm_pushes_touch(p.pushes, p.npush, n0 >> 1, (n0 + BN) >> 1);
  const bool vec = (p.ldy & 3) == 0 && ((uintptr_t)p.y & 15) == 0;
#pragma unroll
  for (int i = 0; i < MT; ++i) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) t[(8 * (r >> 2) + (r & 3) + 4 * lh) * LD + 32 * j + l32] = (float)acc[i][j][r];
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    const int mb = m0 + (wr * MT + i) * 32 + lane / LR;
    for (int k = 0; k < 32 / RS; ++k) {
      const int m = mb + RS * k;
      if (m >= p.M) break;
      const float sm = p.qs[m];
      float v[CL];
#pragma unroll
      for (int q = 0; q < CL / 4; ++q) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(t + (lane / LR + RS * k) * LD + c + 4 * q);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * q + e] = x[e] * sm * sn[4 * q + e];
      }
      if constexpr (EPI == kGemmSwiglu) {
        const int neuron = n >> 1, I = p.N >> 1;
        f32x4 a;
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = silu_f(v[2 * e]) * v[2 * e + 1];
        if (pushes_here) {
          const int row = gemm_push_row(m, p.T);
          for (int k2 = 0; k2 < p.npush; ++k2)
#pragma unroll
            for (int e = 0; e < 4; ++e) a[e] = gemm_push(p.pushes + k2, neuron + e, row, a[e]);
        }
        float* dst = p.y + (int64_t)m * p.ldy + neuron;
        if (vec && neuron + 4 <= I) {
          *reinterpret_cast<f32x4*>(dst) = a;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (neuron + e < I) dst[e] = a[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (neuron + e < I) gemm_capture(p.cap, m, p.T, neuron + e, a[e]);
      } else {
        float* dst = p.y + (int64_t)m * p.ldy + n;
        if (vec && n + 4 <= p.N) {
          f32x4 o = {v[0], v[1], v[2], v[3]};
          if constexpr (EPI == kGemmAccumulate) {
            const f32x4 old = *reinterpret_cast<const f32x4*>(dst);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] += old[e];
          }
          *reinterpret_cast<f32x4*>(dst) = o;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < p.N) dst[e] = EPI == kGemmAccumulate ? dst[e] + v[e] : v[e];
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
}

template <int MT, int NT, int WR, int WC>
static void gemm_i8_launch(const GemmI8Args& a, int epilogue, hipStream_t st) {
  constexpr int BM = 32 * MT * WR, BN = 32 * NT * WC;
  const dim3 grid((unsigned)(((a.M + (int64_t)BM - 1) / BM) * ((a.N + (int64_t)BN - 1) / BN))), block(64 * WR * WC);
  if (epilogue == kGemmStore) hipLaunchKernelGGL((gemm_i8_kernel<MT, NT, WR, WC, kGemmStore>), grid, block, 0, st, a);
  else if (epilogue == kGemmAccumulate) hipLaunchKernelGGL((gemm_i8_kernel<MT, NT, WR, WC, kGemmAccumulate>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((gemm_i8_kernel<MT, NT, WR, WC, kGemmSwiglu>), grid, block, 0, st, a);
}

}  // namespace q35

extern "C" int q35_quantize_rows_i8(const void* x, int64_t ldx, int dtype, int8_t* q, float* s, int64_t M, int64_t K,
                                    q35_stream_t stream) {
  using namespace q35;
  if (!x || !q || !s || M <= 0 || K <= 0 || ldx < K) return Q35_EINVAL;
  if (dtype != Q35_F32 && dtype != Q35_BF16) return Q35_EUNSUPPORTED;
  if ((K & 3) || K > 16384 || (ldx & 3) || M > 0x7fffffff || (uintptr_t)x & (dtype == Q35_F32 ? 15 : 7) || (uintptr_t)q & 3)
    return Q35_EUNSUPPORTED;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == Q35_F32)
    return rows_i8_launch<const float, false>((const float*)x, ldx, nullptr, 0, nullptr, q, s, M, K, 0.f, st);
  return rows_i8_launch<const __bf16, false>((const __bf16*)x, ldx, nullptr, 0, nullptr, q, s, M, K, 0.f, st);
}

extern "C" int q35_add_rmsnorm_i8(float* x, int64_t ldx, const float* y, int64_t ldy, const float* w, int8_t* q, float* s,
                                  int64_t M, int64_t K, float eps, q35_stream_t stream) {
  using namespace q35;
  if (!x || !w || !q || !s || M <= 0 || K <= 0 || ldx < K || (y && ldy < K)) return Q35_EINVAL;
  if ((K & 3) || K > 16384 || (ldx & 3) || (y && (ldy & 3)) || M > 0x7fffffff || ((uintptr_t)x | (uintptr_t)y | (uintptr_t)w) & 15 ||
      (uintptr_t)q & 3)
    return Q35_EUNSUPPORTED;
  return rows_i8_launch<float, true>(x, ldx, y, ldy, w, q, s, M, K, eps, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int q35_gemm_i8(const int8_t* q, int64_t ldq, const float* q_scale, const int8_t* W, const float* w_scale, float* y,
                           int64_t ldy, int64_t M, int64_t N, int64_t K, int epilogue, const q35_push* pushes, int64_t npush,
                           int64_t T, float* cap, int64_t ld_cap, int64_t ld_cap_row, q35_stream_t stream) {
  using namespace q35;
  if (!q || !q_scale || !W || !w_scale || !y || M <= 0 || N <= 0 || K <= 0 || T <= 0) return Q35_EINVAL;
  if (epilogue < kGemmStore || epilogue > kGemmSwiglu) return Q35_EINVAL;
  if (npush < 0 || (npush > 0 && !pushes) || npush > 64) return Q35_EINVAL;
  if (epilogue == kGemmSwiglu ? (N % 2 != 0 || ldy < N / 2) : ldy < N) return Q35_EINVAL;
  if (cap && (epilogue != kGemmSwiglu || ld_cap < N / 2 || ld_cap_row < N / 2 || ((uintptr_t)cap & 3))) return Q35_EINVAL;
  if (ldq < K) return Q35_EINVAL;
  if (K % kIK || K > 65536 || ldq % 16 || ldq > (1 << 23) || ((uintptr_t)q | (uintptr_t)W) & 15) return Q35_EUNSUPPORTED;
  if (M > (1 << 30) || N > (1 << 30) || T > 0x7fffffff) return Q35_EUNSUPPORTED;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const GemmI8Args a{q, ldq, q_scale, W, w_scale, y, ldy, (int)M, (int)N, (int)K, pushes, (int)npush, (int)T, {cap, ld_cap, ld_cap_row}};
  const int64_t cus = device_cus();
  if (((M + 63) / 64) * ((N + 63) / 64) > 0x7fffffff) return Q35_EUNSUPPORTED;
  if (((M + 255) / 256) * ((N + 255) / 256) >= cus) gemm_i8_launch<4, 2, 2, 4>(a, epilogue, st);
  else if (((M + 127) / 128) * ((N + 127) / 128) >= cus) gemm_i8_launch<2, 2, 2, 2>(a, epilogue, st);
  else gemm_i8_launch<1, 1, 2, 2>(a, epilogue, st);
  return hipGetLastError() == hipSuccess ? Q35_OK : Q35_ELAUNCH;
}
