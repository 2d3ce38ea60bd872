// Products in 8-bit integers with one scale per token and one per output channel, and the rows in 8 bits that they take.
//
//   s[m] = fp32(max_k |x[m, k]| / 127), q[m, k] = rint(x[m, k] / s[m]) (half to even), -127 .. 127
//   y[m, n] = (sum_k q[m, k] W[n, k]) s[m] ws[n]
//
// The sum is exact (int32, K up to 65536), so it depends on no order and every kernel here gives the same bits. A code is a
// rounding decision: quotient and norm are formed in 64 bits, whatever the order of a sum.
#include "gemm_common.h"

namespace q35 {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

// ---------------------------------------------------------------------------------------------------------------
// Rows in 8 bits, one block a row, held in registers: PER quads of values a thread, so that memory is passed over once. 16384
// rows of 3584 fp32 values take 54 us, 5.4 TB/s of the 294 MB read and written (a large copy reaches 5.2), of bf16 values 40 to 45
// (176 MB). 6144 rows of 1024 normed take 11.4 to 13.3 us (31 MB; 32 % of the vector ALU, in 64 bits), with an added y 18 (82 MB).

// rint(x / s), half to even, in -127 .. 127: x, s exact. The remainder settles what the product with 1 / s left undecided. |x / s| is
// 127 to fp32's rounding of s; where s is subnormal that rounding is up to a third of it (190 2^-149 / 127 is 2^-149 then: a quotient
// of 190), and the largest code stands for less than the value.
__device__ __forceinline__ int i8_code(double x, double s, double inv) {
  double t = __builtin_rint(x * inv);
  const double r = __builtin_fma(-t, s, x), a = fabs(r) * 2.0;  // exact: t has 8 bits, s 24
  if (a > s || (a == s && ((int)t & 1))) t += r > 0.0 ? 1.0 : -1.0;
  return (int)fmin(fmax(t, -127.0), 127.0);
}

// Values and quotients are formed in fp32 first, 2^-21 of themselves: an element whose quotient is then within 2^-12 of a half,
// or whose factors leave fp32's middle range, is formed again in 64 bits, and so are those within 2^-19 of the largest, for
// the scale. A row whose scale is far from 1 is formed in 64 bits as a whole. (All elements in 64 bits: three times the
// operations, 68 us for those 16384 rows.)
constexpr float kI8Far = 0x1p100f;

template <typename Tx, bool NORM, int NW, int PER>
__global__ __launch_bounds__(64 * NW) void rows_i8_kernel(Tx* __restrict__ x, int64_t ldx, const float* __restrict__ y,
                                                      int64_t ldy, const float* __restrict__ w, int8_t* __restrict__ q,
                                                      float* __restrict__ s, int K, float eps) {
  const int64_t m = blockIdx.x;
  const int tid = threadIdx.x;
  Tx* xr = x + m * ldx;
  f32x4 f[PER], v[NORM ? PER : 1], w1;
  double ss = 0.0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int c = 4 * (tid + 64 * NW * i);
    f[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (c < K) {
      if constexpr (sizeof(Tx) == 4) {
        f[i] = *reinterpret_cast<const f32x4*>(xr + c);
      } else {
        const u32x2 r = *reinterpret_cast<const u32x2*>(xr + c);
        f[i] = f32x4{bf16lo(r.x), bf16hi(r.x), bf16lo(r.y), bf16hi(r.y)};
      }
      if constexpr (NORM) {
        v[i] = w1 = *reinterpret_cast<const f32x4*>(w + c);
        if (y) {
          const f32x4 a = *reinterpret_cast<const f32x4*>(y + m * ldy + c);
#pragma unroll
          for (int e = 0; e < 4; ++e) f[i][e] += a[e];
          *reinterpret_cast<f32x4*>(xr + c) = f[i];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) ss = __builtin_fma((double)f[i][e], (double)f[i][e], ss);
      }
    }
  }
  __shared__ double red[NW];
  __shared__ float redm[2][NW];
  __shared__ int redo[NW];
  const int wave = tid >> 6;
  double r = 1.0;
  if constexpr (NORM) {
    ss = wave_sum64(ss);
    if constexpr (NW > 1) {
      if ((tid & 63) == 0) red[wave] = ss;
      __syncthreads();
      ss = red[0] + red[1] + red[2] + red[3];
    }
    r = 1.0 / sqrt(ss / (double)K + (double)eps);
  }
  // one quad a thread: all of them in 64 bits for the scale, for one barrier less (32 rows of 1024: 3.3 us, 4.1 with it)
  constexpr bool kAll = NORM && NW > 1 && PER == 1;
  auto exact = [&](int i, int e) -> double {
    if constexpr (!NORM) return (double)f[i][e];
    return (double)f[i][e] * r * (1.0 + (double)(PER == 1 ? w1[e] : w[4 * (tid + 64 * NW * i) + e]));
  };
  // v: the values in fp32, NaN where these cannot be relied on
  bool odd = false;
  float mx = 0.f;
  if constexpr (NORM) {
    const float rf = (float)r;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const bool in = 4 * (tid + 64 * NW * i) < K;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float g = rf * (1.f + v[i][e]), t = f[i][e] * g;
        const bool good = fabsf(g) > 1.f / kI8Far && fabsf(g) < kI8Far && fabsf(t) < kI8Far;
        v[i][e] = in ? (good ? t : NAN) : 0.f;
        mx = fmaxf(mx, v[i][e] == v[i][e] ? fabsf(v[i][e]) : 0.f);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        odd |= !(fabsf(f[i][e]) < INFINITY);
        mx = fmaxf(mx, fabsf(f[i][e]));
      }
  }
  if constexpr (!kAll) mx = wave_max_f32(mx);
  if constexpr (NORM) {
    if constexpr (!kAll && NW > 1) {
      if ((tid & 63) == 0) redm[0][wave] = mx;
      __syncthreads();
      mx = fmaxf(fmaxf(redm[0][0], redm[0][1]), fmaxf(redm[0][2], redm[0][3]));
    }
    const float near = !kAll && mx > 1.f / kI8Far ? mx * (1.f - 0x1p-19f) : 0.f;
    double md = 0.0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      bool any = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) any |= !(fabsf(v[i][e]) < near);
      if (any && 4 * (tid + 64 * NW * i) < K) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const double d = fabs(exact(i, e));
          odd |= !(d < INFINITY);
          md = fmax(md, d);
        }
      }
    }
    // the scale of the largest: fp32(max / 127) is monotone, so the maximum of the rounded quotients
    mx = wave_max_f32((float)(md / 127.0));
  }
  bool bad = __builtin_amdgcn_ballot_w64(odd) != 0;
  if constexpr (NW > 1) {
    if ((tid & 63) == 0) {
      redm[1][wave] = mx;
      redo[wave] = bad;
    }
    __syncthreads();
    mx = fmaxf(fmaxf(redm[1][0], redm[1][1]), fmaxf(redm[1][2], redm[1][3]));
    bad = redo[0] | redo[1] | redo[2] | redo[3];
  }
  // a row that holds a value that is not finite has the scale NaN, and its products are NaN
  const float sc = NORM ? mx : (float)((double)mx / 127.0);
  bad |= !(sc < INFINITY);
  if (tid == 0) s[m] = bad ? __int_as_float(0x7fc00000) : sc;
  const bool none = bad || !(sc > 0.f), all = !(sc > 1.f / kI8Far && sc < kI8Far);
  const double sd = none ? 1.0 : (double)sc, inv = 1.0 / sd;
  const float invf = (float)inv;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int c = 4 * (tid + 64 * NW * i);
    if (c < K) {
      uint32_t o = 0;
      bool again = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float t = (NORM ? v[i][e] : f[i][e]) * invf, n = __builtin_rintf(t);
        again |= !(fabsf(t - n) < 0.5f - 0x1p-12f);
        o |= (uint32_t)(uint8_t)(int)n << (8 * e);
      }
      if (again || all) {
        o = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) o |= (uint32_t)(uint8_t)i8_code(exact(i, e), sd, inv) << (8 * e);
      }
      *reinterpret_cast<uint32_t*>(q + m * K + c) = none ? 0 : o;
    }
  }
}

template <typename Tx, bool NORM>
static int rows_i8_launch(Tx* x, int64_t ldx, const float* y, int64_t ldy, const float* w, int8_t* q, float* s, int64_t M,
                          int64_t K, float eps, hipStream_t st) {
#define Q35_ROWS(NW, PER)                                                                                                \
  hipLaunchKernelGGL((rows_i8_kernel<Tx, NORM, NW, PER>), dim3((unsigned)M), dim3(64 * NW), 0, st, x, ldx, y, ldy, w, q, s, \
                     (int)K, eps)
  // one wave a row of up to 1024 values where there are rows for all CUs to hold eight (normed rows of 1024 by one wave and by
  // four: 6144 rows 10.8 and 14.1 us, 2048 6.6 and 6.9, 1024 6.2 and 4.8, 32 4.9 and 3.3)
  if (K <= 256) Q35_ROWS(1, 1);
  else if (K <= 512) Q35_ROWS(1, 2);
  else if (K <= 1024 && M >= 2048) Q35_ROWS(1, 4);
  else if (K <= 1024) Q35_ROWS(4, 1);
  else if (K <= 2048) Q35_ROWS(4, 2);
  else if (K <= 4096) Q35_ROWS(4, 4);
  else if (K <= 8192) Q35_ROWS(4, 8);
  else Q35_ROWS(4, 16);
#undef Q35_ROWS
  return hipGetLastError() == hipSuccess ? Q35_OK : Q35_ELAUNCH;
}

// ---------------------------------------------------------------------------------------------------------------
// Tiles of BM x BN outputs, a wave 32 MT x 32 NT of them. Rows of q and W go to LDS by DMA in stages of 128 inputs, whole cache
// lines (rows of 128 bytes, 16-byte chunk c at c ^ ((row >> 1) & 7): 16 consecutive lanes of a fragment read fall in distinct
// slots). Stages of 64 inputs fetched half lines and took 1.4 times as long.
//
// 16384 rows of 3584 inputs by 1024 outputs, tiles of 256 x 256 (8 waves of 128 x 64): 65 us alone, 1.86 P operations a second (a
// library product of 8192^3 reaches 2.07), 71 behind the rows' kernel, 73 added to what is there; the matrix units bound it, then the
// 64 MB of results, which leave at the end as all blocks run in step. 6144 rows of 1024 inputs by 7168 outputs with SwiGLU: 70 us,
// 1.29 P; 672 tiles are 2.6 a CU, and 88 MB leave. 333 rows of 3584 by 1024 (352 tiles of 32): 7.2 us; 32 rows of 1024 by 5120 3.2 us: latency of a stage from memory.
constexpr int kIK = 128;  // inputs of a stage

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

// What becomes of CL scaled sums of row m from column n on (CL even columns are CL / 2 gate and up pairs).
template <int EPI, int CL>
__device__ __forceinline__ void gemm_i8_finish(const GemmI8Args& p, int m, int n, const float (&v)[CL], bool vec, bool pushes_here) {
  if constexpr (EPI == kGemmSwiglu) {
    constexpr int NA = CL / 2;
    typedef float fvec __attribute__((ext_vector_type(NA)));
    const int neuron = n >> 1, I = p.N >> 1;
    fvec a;
#pragma unroll
    for (int e = 0; e < NA; ++e) a[e] = silu_f(v[2 * e]) * v[2 * e + 1];
    if (pushes_here) {
      const int row = gemm_push_row(m, p.T);
      for (int k = 0; k < p.npush; ++k)
#pragma unroll
        for (int e = 0; e < NA; ++e) a[e] = gemm_push(p.pushes + k, neuron + e, row, a[e]);
    }
    float* dst = p.y + (int64_t)m * p.ldy + neuron;
    if (vec && neuron + NA <= I) {
      *reinterpret_cast<fvec*>(dst) = a;
    } else {
#pragma unroll
      for (int e = 0; e < NA; ++e)
        if (neuron + e < I) dst[e] = a[e];
    }
#pragma unroll
    for (int e = 0; e < NA; ++e)
      if (neuron + e < I) gemm_capture(p.cap, m, p.T, neuron + e, a[e]);
  } else {
    static_assert(CL == 4, "one store");
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

// The tile of a block: each XCD takes a run of neighbouring tiles, down the rows of q where these are the fewer bytes, else along
// W's, so that its L2 holds the smaller operand and a run of the other.
__device__ __forceinline__ void gemm_i8_tile(const GemmI8Args& p, int nbm, int nbn, int& bm, int& bn) {
  const int ntiles = nbm * nbn, xj = (int)(blockIdx.x & 7), xq = ntiles >> 3, xr = ntiles & 7;
  const int tile = xj * xq + min(xj, xr) + (int)(blockIdx.x >> 3);
  if (p.M < p.N) {
    bn = tile / nbm;
    bm = tile - bn * nbm;
  } else {
    bm = tile / nbn;
    bn = tile - bm * nbn;
  }
}

template <int MT, int NT, int WR, int WC, int NS, int EPI>
__global__ __launch_bounds__(64 * WR * WC, MT * NT > 8 ? 1 : 2) void gemm_i8_kernel(GemmI8Args p) {
  constexpr int BM = 32 * MT * WR, BN = 32 * NT * WC, NW = WR * WC;
  constexpr int UA = BM / 8, U = (BM + BN) / 8 / NW;  // 1 KB copies (8 rows) of a stage's q, copies per wave
  constexpr int SB = (BM + BN) * kIK;
  static_assert((BM + BN) / 8 % NW == 0, "copies are dealt evenly");
  __shared__ __attribute__((aligned(16))) char smem[NS * SB];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wv / WC, wc = wv % WC, l32 = lane & 31, lh = lane >> 5;
  int bm, bn;
  gemm_i8_tile(p, (p.M + BM - 1) / BM, (p.N + BN - 1) / BN, bm, bn);
  const int m0 = bm * BM, n0 = bn * BN, KT = (p.K + kIK - 1) / kIK;

  const int8_t* qb = p.q + (int64_t)m0 * p.ldq;
  const int8_t* wb = p.W + (int64_t)n0 * p.K;
  // a copy's lane: row lane / 8 of its eight, slot lane % 8. K may end in the middle of a stage: then no more than its first half
  // is multiplied, and the other half's lanes copy that again.
  const int half_end = p.K % kIK ? KT - 1 : KT;
  uint32_t src[U], tail[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int u = wv + NW * i, row = 8 * (u < UA ? u : u - UA) + (lane >> 3), c = (lane & 7) ^ ((row >> 1) & 7);
    const uint32_t at = u < UA ? (uint32_t)min(row, p.M - 1 - m0) * (uint32_t)p.ldq : (uint32_t)min(row, p.N - 1 - n0) * (uint32_t)p.K;
    src[i] = at + 16 * c;
    tail[i] = at + 16 * (c & 3);
  }
  const uint32_t lds0 = gemm_lds_u32(smem);
  auto issue = [&](int s) {
    const uint32_t base = lds0 + (s % NS) * SB;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int u = wv + NW * i;
      gemm_dma16s((u < UA ? qb : wb) + (int64_t)s * kIK, s < half_end ? src[i] : tail[i], base + u * 1024);
    }
  };
  const int ra = wr * 32 * MT + l32, rb = wc * 32 * NT + l32;
  uint32_t ao[4], bo[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int ch = ((2 * j + lh) ^ ((l32 >> 1) & 7)) << 4;
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

  // The fragments of 32 inputs are read ahead of the products of the 32 before, so that the one runs beside the other: the
  // barrier that hands a stage's buffer on stands before its last products, when all of it has been read.
  i32x4 fa[2][MT], fb[2][NT];
  auto read = [&](int s, int j) {
    const char* st = smem + (s % NS) * SB;
#pragma unroll
    for (int i = 0; i < MT; ++i) fa[j & 1][i] = *reinterpret_cast<const i32x4*>(st + ao[j] + i * 32 * kIK);
#pragma unroll
    for (int i = 0; i < NT; ++i) fb[j & 1][i] = *reinterpret_cast<const i32x4*>(st + bo[j] + i * 32 * kIK);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto multiply = [&](int j) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int k = 0; k < NT; ++k)
        acc[i][k] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[j & 1][i], fb[j & 1][k], acc[i][k], 0, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto wait = [&](int s) {  // stage s has landed, with up to NS - 2 behind it in flight; all waves are past their earlier reads
    const int behind = min(KT - 1 - s, NS - 2);
    if (NS == 4 && behind >= 2) gemm_wait_vm<2 * U>();
    else if (NS == 4 && behind == 1) gemm_wait_vm<U>();
    else gemm_wait_vm<0>();
    lds_barrier();
  };
  static_assert(NS == 2 || NS == 4, "wait()");
  for (int s = 0; s < NS - 1; ++s)
    if (s < KT) issue(s);
  wait(0);
  if (NS - 1 < KT) issue(NS - 1);
  read(0, 0);
  for (int s = 0; s < KT; ++s) {
    read(s, 1);
    multiply(0);
    if (s < half_end) {
      read(s, 2);
      multiply(1);
      read(s, 3);
      multiply(2);
    }
    if (s + 1 < KT) {
      wait(s + 1);
      if (s + NS < KT) issue(s + NS);
      read(s + 1, 0);
    }
    multiply(1);
  }

  // The results leave through LDS, a wave's 32 rows at a time in an area of its own, so that a store holds whole runs of a row:
  // a lane takes CL columns of a row (gate and up of a neuron meet in it).
  constexpr int CW = 32 * NT, LD = CW + 4, CL = EPI == kGemmSwiglu ? 8 : 4, LR = CW / CL, RS = 64 / LR;
  static_assert(NW * 32 * LD * 4 <= NS * SB, "the stages hold the waves' areas");
  lds_barrier();  // every wave has read its last fragments
  float* t = reinterpret_cast<float*>(smem) + wv * 32 * LD;
  const int c = CL * (lane % LR), n = n0 + wc * CW + c;
  float sn[CL];
#pragma unroll
  for (int e = 0; e < CL; ++e) sn[e] = p.ws[min(n + e, p.N - 1)];
  const bool pushes_here = EPI == kGemmSwiglu && gemm_pushes_touch(p.pushes, p.npush, n0 >> 1, (n0 + BN) >> 1);
  const bool vec = (p.ldy & 3) == 0 && ((uintptr_t)p.y & 15) == 0;
  // (all rows' scales at once: a load for each row's turn was a third of the time of a tile of 1024 inputs)
  float sm[MT][32 / RS];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int k = 0; k < 32 / RS; ++k) sm[i][k] = p.qs[min(m0 + (wr * MT + i) * 32 + lane / LR + RS * k, p.M - 1)];
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
#pragma unroll
    for (int k = 0; k < 32 / RS; ++k) {
      const int m = mb + RS * k;
      if (m >= p.M) continue;
      float v[CL];
#pragma unroll
      for (int q = 0; q < CL / 4; ++q) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(t + (lane / LR + RS * k) * LD + c + 4 * q);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * q + e] = x[e] * sm[i][k] * sn[4 * q + e];
      }
      gemm_i8_finish<EPI, CL>(p, m, n, v, vec, pushes_here);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
}

// Few tiles: 32 x 32 outputs a block, its four waves a quarter of the stages each (wave w takes w, w + 4, ...), with no barrier
// between them before the four sums meet in LDS.
template <int EPI>
__global__ __launch_bounds__(256, 2) void gemm_i8_few_kernel(GemmI8Args p) {
  constexpr int SB = 64 * kIK, NS = 2, LD = 36;  // a stage's 32 rows of q, then of W; LD: a row of sums
  __shared__ __attribute__((aligned(16))) char smem[4 * NS * SB];
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, lh = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  int bm, bn;
  gemm_i8_tile(p, (p.M + 31) / 32, (p.N + 31) / 32, bm, bn);
  const int m0 = bm * 32, n0 = bn * 32, KT = (p.K + kIK - 1) / kIK, half_end = p.K % kIK ? KT - 1 : KT;
  const int8_t* qb = p.q + (int64_t)m0 * p.ldq;
  const int8_t* wb = p.W + (int64_t)n0 * p.K;
  uint32_t src[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = 8 * (i & 3) + (lane >> 3);
    src[i] = i < 4 ? (uint32_t)min(row, p.M - 1 - m0) * (uint32_t)p.ldq : (uint32_t)min(row, p.N - 1 - n0) * (uint32_t)p.K;
  }
  const uint32_t lds0 = gemm_lds_u32(smem) + wv * NS * SB;
  auto issue = [&](int s) {  // the last stage may be half a one, as above
    const uint32_t base = lds0 + ((s >> 2) % NS) * SB;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = (lane & 7) ^ (((8 * (i & 3) + (lane >> 3)) >> 1) & 7);
      gemm_dma16s((i < 4 ? qb : wb) + (int64_t)s * kIK, src[i] + 16 * (s < half_end ? c : c & 3), base + i * 1024);
    }
  };
  i32x16 acc;
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[r] = 0;
  if (wv < KT) issue(wv);
  if (wv + 4 < KT) issue(wv + 4);
  for (int s = wv; s < KT; s += 4) {
    if (s + 4 < KT) gemm_wait_vm<8>();
    else gemm_wait_vm<0>();
    const char* st = smem + (wv * NS + (s >> 2) % NS) * SB;
    i32x4 a[4], b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int at = l32 * kIK + (((2 * j + lh) ^ ((l32 >> 1) & 7)) << 4);
      a[j] = *reinterpret_cast<const i32x4*>(st + at);
      b[j] = *reinterpret_cast<const i32x4*>(st + 32 * kIK + at);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage has been read
    if (s + 8 < KT) issue(s + 8);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < 2 || s < half_end) acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[j], b[j], acc, 0, 0, 0);
  }
  // the sums of a wave to where its first stage was: nobody else reads or writes there
  int* t = reinterpret_cast<int*>(smem);
  constexpr int AW = NS * SB / 4;
  static_assert(AW >= 32 * LD, "an area each");
#pragma unroll
  for (int r = 0; r < 16; ++r) t[wv * AW + (8 * (r >> 2) + (r & 3) + 4 * lh) * LD + l32] = acc[r];
  __syncthreads();
  const int row = tid >> 3, c = 4 * (tid & 7), m = m0 + row, n = n0 + c;
  if (m >= p.M || n >= p.N) return;
  const bool pushes_here = EPI == kGemmSwiglu && gemm_pushes_touch(p.pushes, p.npush, n0 >> 1, (n0 + 32) >> 1);
  constexpr int al = EPI == kGemmSwiglu ? 2 : 4;
  const bool vec = (p.ldy & (al - 1)) == 0 && ((uintptr_t)p.y & (4 * al - 1)) == 0;
  i32x4 sum = {0, 0, 0, 0};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const i32x4 x = *reinterpret_cast<const i32x4*>(t + k * AW + row * LD + c);
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] += x[e];
  }
  const float sm = p.qs[m];
  float v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = (float)sum[e] * sm * p.ws[min(n + e, p.N - 1)];
  gemm_i8_finish<EPI, 4>(p, m, n, v, vec, pushes_here);
}

template <int MT, int NT, int WR, int WC, int NS>
static void gemm_i8_launch(const GemmI8Args& a, int epilogue, hipStream_t st) {
  constexpr int BM = 32 * MT * WR, BN = 32 * NT * WC;
  const dim3 grid((unsigned)(((a.M + (int64_t)BM - 1) / BM) * ((a.N + (int64_t)BN - 1) / BN))), block(64 * WR * WC);
  if (epilogue == kGemmStore) hipLaunchKernelGGL((gemm_i8_kernel<MT, NT, WR, WC, NS, kGemmStore>), grid, block, 0, st, a);
  else if (epilogue == kGemmAccumulate)
    hipLaunchKernelGGL((gemm_i8_kernel<MT, NT, WR, WC, NS, kGemmAccumulate>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((gemm_i8_kernel<MT, NT, WR, WC, NS, kGemmSwiglu>), grid, block, 0, st, a);
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
  if (K % 64 || K > 65536 || ldq % 16 || ldq > (1 << 23) || ((uintptr_t)q | (uintptr_t)W) & 15) return Q35_EUNSUPPORTED;
  if (M > (1 << 30) || N > (1 << 30) || T > 0x7fffffff) return Q35_EUNSUPPORTED;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const GemmI8Args a{q, ldq, q_scale, W, w_scale, y, ldy, (int)M, (int)N, (int)K, pushes, (int)npush, (int)T, {cap, ld_cap, ld_cap_row}};
  const int64_t cus = device_cus();
  const auto tiles = [&](int64_t b) { return ((M + b - 1) / b) * ((N + b - 1) / b); };
  if (tiles(256) > 0x7fffffff) return Q35_EUNSUPPORTED;
  // The smallest tile of which the chip takes all blocks at once, two to a CU; a larger one beyond, which reads each operand
  // less often. Where the next larger has few tiles, its CUs wait for their own reads: 1024 outputs of 3584 inputs take, in us,
  // with tiles of 32 / 64 / 128 / 256, 4.3 / 10.4 / 18.6 / 42 for 32 rows, 8.0 / 11.2 / 19.9 / 44 for 512 (512 tiles of 32), 23.4
  // / 16.1 / 23.1 / 46 for 2048 (512 of 64), 43 / 29 / 26 / 48 for 4096; 7168 outputs of 1024 inputs 32 / 21 / 15 / 22 for 1024
  // rows (448 of 128), 150 / 79 / 48 / 44 for 4096.
  if (tiles(32) <= 2 * cus) {
    const dim3 grid((unsigned)tiles(32)), block(256);
    if (epilogue == kGemmStore) hipLaunchKernelGGL((gemm_i8_few_kernel<kGemmStore>), grid, block, 0, st, a);
    else if (epilogue == kGemmAccumulate) hipLaunchKernelGGL((gemm_i8_few_kernel<kGemmAccumulate>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((gemm_i8_few_kernel<kGemmSwiglu>), grid, block, 0, st, a);
  } else if (tiles(64) <= 2 * cus) {
    gemm_i8_launch<1, 1, 2, 2, 4>(a, epilogue, st);
  } else if (tiles(128) <= 2 * cus) {
    gemm_i8_launch<2, 2, 2, 2, 2>(a, epilogue, st);
  } else {
    gemm_i8_launch<4, 2, 2, 4, 2>(a, epilogue, st);
  }
  return hipGetLastError() == hipSuccess ? Q35_OK : Q35_ELAUNCH;
}
