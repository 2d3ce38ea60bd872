// Gated causal grouped attention of T new tokens per row over a paged KV cache in bf16 or 4 bits.
//
//   token t of row b sits at position p = pos[b] + t; q' = rope_p(q rsqrt(mean q^2 + eps) (1 + w)), and per query head
//   out = sum_j softmax_j(q' . k_j scale) v_j * sigmoid(gate) over the cached keys j <= p (HF:656-698 with a cache; WGSL
//   attention, engine/kernels_qwen35.js:73-123). The new tokens' keys are in the pages already.
//
// A block takes 16 NR query rows (row r = t G + head of the group, G = Hq / Hkv) of one kv head against one run of the
// row's keys; its four waves (or eight) take 32 keys each in turn. Both products run with the keys on the matrix core's row side:
//   S^T [keys x rows]  = K Q^T   A: 16 keys of K as they lie in the page, B: Q from LDS
//   O^T [dims x rows] += V^T P^T A: V^T formed in registers, B: the exponentials, which S^T's layout hands over as they
//                                are (lane: row l % 16, keys 4 (l / 16) + r of two 16-key tiles)
// so that no score or probability crosses lanes except for a row's maximum (two exchanges) and, at the end, its sum.
// Sums, maxima and accumulators are fp32. What is rounded to fewer bits, because the matrix core takes no fp32 operands and
// parts of them (hi + lo) double a product: the exponentials to bf16 (at most 2^-8 of each weight, with the value's scale
// already in it), in both formats and for either output; Q, against bf16 keys as bf16 hi + lo (two products, 2^-16 of q),
// against 4-bit codes, whose vector work leaves no room for a second one, as fp16, each row scaled by a power of two to a
// largest value of 16 to 32 (2^-11 of q). In the norm of the output this is 1.1e-3 to 1.7e-3 of 64 bits (fp32 output, 100 to
// 4000 keys), against 1.6e-3 of the dense decode kernel, which rounds q to bf16, and 2.8e-3 of the dense prefill over the
// cache; a bf16 output's own rounding is 1.65e-3 and makes it 2.0e-3 to 2.4e-3.
//
// 4 bits: a code n enters the products as a small whole number that the operand type holds exactly, its bits or-ed into the
// mantissa of a power of two: keys 1024 + n and, from the nibble above, 1024 + 16 n in fp16 (Q / 16 against it), 5
// operations for 8 values; values 16 + n in bf16 (fp16 would not hold weight times scale). The offsets leave again: the
// keys' products start from minus the offsets' part of the sum, formed from the same rounded Q; the values' by the sum of
// the rounded weights times -24, which a product of its own collects for all four groups (row r of its A operand is -24
// where r % 4 is the group). Scales apply outside the codes: a key's to its group's partial score (fp32), a value's to the
// exponential before its rounding. What bounds the 4-bit form is the vector ALU's issue: about 570 operations beside 72
// matrix products for 32 rows x 32 keys, two fifths of them unpacking, so masks and constants are kept where one v_and_or_b32
// takes both, scales and offsets come from LDS in the form in which they are used, and what only masked rounds or scales
// that are not finite need stays behind branches.
//
// Measured (8 query and 2 key heads; a 1 GiB copy runs at 5.2 TB/s, a large bf16 product at 1380 TFLOP/s): one token for 32
// rows of up to 8192 bf16 keys 93 to 96 us (5.1 TB/s), 4-bit keys 37 (3.5 TB/s); up to five tokens a row against 4-bit keys 45 to
// 49 us (2.8 TB/s), bf16 104 (4.7 TB/s); 512 tokens of one row behind 16 K 4-bit keys 115 us (528 TFLOP/s), bf16 165; one token
// of three rows of 8192 4-bit keys 14 us.
//
// A row's keys are dealt over S blocks in runs of whole 128-key rounds by the row's own length, read on the device: the
// grid is sized by the table's capacity, the work by what is cached. With S > 1 the blocks leave (max, sum, acc) and a
// second kernel merges them; blocks whose run is empty leave nothing and are not read.
#include <algorithm>

#include "paged_kv.h"

namespace q35 {

struct PagedAttnArgs {
  const void *q, *gate;
  int64_t qb, qt, qh, gb, gt, gh;  // strides of q and gate, in elements
  const float *qw, *cos_t, *sin_t;
  float eps, scale;
  int rot, q_f32, out_f32;
  PagedTable pt;
  const int32_t *pos, *lens;
  const void *kp, *vp;
  const __bf16 *ks, *vs;
  void* out;
  float *part, *ml;  // S > 1: O [B][Hkv][T G][S][256], (max, sum) [B][Hkv][T G][S][2]
  int T, Hkv, G, S, RB;
};

typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 bf16x2;
typedef __attribute__((__vector_size__(8 * sizeof(_Float16)))) _Float16 f16x8;
typedef __attribute__((__vector_size__(2 * sizeof(float)))) float f32x2;

constexpr int kRound = 128;     // keys per round of the four waves
constexpr int kORow = kPgD + 4; // LDS row of a wave's result

// Keys that token t of row b sees: 0 .. n - 1. 0 for a token that is not there.
__device__ __forceinline__ int keys_seen(const PagedAttnArgs& p, int64_t pos, int len, int t) {
  const int64_t at = pos + t;
  return t < len && at >= 0 && at < p.pt.capacity() ? (int)at + 1 : 0;
}
// Keys of row b's run over S blocks, from the keys its last token sees: a multiple of a round.
__device__ __forceinline__ int run_keys(int n, int S) {
  const int rounds = (n + kRound - 1) / kRound;
  return (rounds + S - 1) / S * kRound;
}

template <bool I4> struct KTile;
template <> struct KTile<true> {
  u32x4 c[2];  // codes: dword 2 g + u
};
template <> struct KTile<false> {
  bf16x8 c[8];
};
template <bool I4> struct VTile;
template <> struct VTile<true> {
  u32x2 c[4];  // key 4 a + r: 16 bits per group
};
template <> struct VTile<false> {
  u32x4 c[4][2];  // key 4 a + r: dims 8 c .. and 128 + 8 c ..
};

__device__ __forceinline__ f32x4 mfma16h(const u32x4& a, const f16x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), b, c, 0, 0, 0);
}
__device__ __forceinline__ uint32_t cvt2(float a, float b) {
  const f32x2 v = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}

__device__ __forceinline__ float row16_sum(float v) {
  v += lane_dpp<0xB1>(v);
  v += lane_dpp<0x4E>(v);
  v += lane_dpp<0x141>(v);
  return v + lane_dpp<0x140>(v);
}
// A row of Q, 16 lanes of 16 dims (x[q][e] of lane j: dim 64 q + 4 j + e, scaled for base-2 exponentials), as column `col` of
// the scores' B operands: bf16 hi + lo, or fp16 with its power of two in *fac and what the codes' offsets add to each
// group's product, negated, in off[][col].
template <bool I4>
__device__ __forceinline__ void q_store(const f32x4 (&x)[4], int j, int col, u32x4* qf, f32x4 (*off)[16], float* fac) {
  if constexpr (I4) {
    // dim 64 g + 16 a + 8 u + k is step 2 g + u of lane group a; a dword's nibbles leave it in pairs (k, k + 4), those of
    // odd k times 16
    float m = 0.f;
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e) m = fmaxf(m, fabsf(x[q][e]));
    const int ex = __builtin_amdgcn_frexp_expf(row16_max_f32(m));  // (0 for 0 and for what is not finite)
    _Float16* qe = reinterpret_cast<_Float16*>(qf) + (((j >> 1) & 1) * 64 + 16 * (j >> 2) + col) * 8 + (j & 1);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float o = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const _Float16 hq = (_Float16)ldexpf(x[q][e], 5 - ex - 4 * (e & 1));
        qe[q * 1024 + 2 * e] = hq;
        o -= (e & 1 ? 1152.f : 1032.f) * (float)hq;
      }
      o = row16_sum(o);
      if (j == 0) off[q][col] = f32x4{o, o, o, o};
    }
    if (j == 0) *fac = ldexpf(1.f, ex - 5);
  } else {
    // dim 32 step + 8 a + k in order
    __bf16* qe = reinterpret_cast<__bf16*>(qf) + ((j >> 3) * 64 + 16 * ((j >> 1) & 3) + col) * 8 + 4 * (j & 1);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      bf16x4 hi, lo;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bf16_hl hl = bf16_split(x[q][e]);
        hi[e] = hl.hi;
        lo[e] = hl.lo;
      }
      *reinterpret_cast<bf16x4*>(qe + q * 1024) = hi;
      *reinterpret_cast<bf16x4*>(qe + 8 * 64 * 8 + q * 1024) = lo;
    }
  }
}
// A lane's accumulators of its row into o[256], dims in order.
template <bool I4>
__device__ __forceinline__ void o_store(const f32x4 (&acc)[16], const f32x4& corr, float* o, int a) {
  if constexpr (I4) {
#pragma unroll
    for (int g = 0; g < kPgNG; ++g)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[4 * g + e][r] + corr[g];
        *reinterpret_cast<f32x4*>(o + 64 * g + 16 * a + 4 * r) = v;
      }
  } else {
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[4 * w + e][r];
        *reinterpret_cast<f32x4*>(o + 128 * (w >> 1) + 8 * (4 * a + r) + 4 * (w & 1)) = v;
      }
  }
}
__device__ __forceinline__ f32x4 gate_load(const PagedAttnArgs& p, int b, int t, int h, int d0) {
  if (!p.gate) return zero4();
  const int64_t o = b * p.gb + t * p.gt + h * p.gh + d0;
  return p.q_f32 ? load_quad<float>((const float*)p.gate + o) : load_quad<__bf16>((const __bf16*)p.gate + o);
}
// Four values of an fp32 or bf16 tensor as they lie in memory, and what they are.
__device__ __forceinline__ u32x4 quad_raw(const void* p, bool f32, int64_t at) {
  if (f32) return *reinterpret_cast<const u32x4*>((const float*)p + at);
  const u32x2 r = *reinterpret_cast<const u32x2*>((const __bf16*)p + at);
  return u32x4{r.x, r.y, 0, 0};
}
__device__ __forceinline__ f32x4 quad_value(const u32x4& r, bool f32) {
  const f32x4 h = {bf16lo(r.x), bf16hi(r.x), bf16lo(r.y), bf16hi(r.y)};
  return f32 ? __builtin_bit_cast(f32x4, r) : h;
}
// out = O / L sigmoid(gate); zeros for a row that sees nothing
__device__ __forceinline__ void out_store(const PagedAttnArgs& p, const f32x4& O, float L, bool sees, const f32x4& g,
                                          int b, int t, int h, int d0) {
  f32x4 v = zero4();
  if (sees && L != 0.f) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = O[e] / L * (p.gate ? sigmoidf_(g[e]) : 1.f);
  }
  const int64_t oi = (((int64_t)b * p.T + t) * p.Hkv * p.G + h) * kPgD + d0;
  if (p.out_f32) {
    *reinterpret_cast<f32x4*>((float*)p.out + oi) = v;
  } else {
    const bf16x4 w = {(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
    *reinterpret_cast<bf16x4*>((__bf16*)p.out + oi) = w;
  }
}

template <bool I4, int NR, int W>
__global__ __launch_bounds__(64 * W, 2) void paged_attn_kernel(PagedAttnArgs p) {
  constexpr int ROWS = 16 * NR, KEYS = 32 * W, QP = I4 ? 1 : 2, QF = 8 * 64;  // parts of Q, 16-byte operands of one
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, a = lane >> 4;
  const int s = blockIdx.x, kvh = blockIdx.y % p.Hkv, rb = blockIdx.y / p.Hkv, b = blockIdx.z;
  const int R = p.T * p.G, r0 = rb * ROWS;

  constexpr int kQBytes = NR * QP * QF * 16, kOBytes = W * 16 * kORow * 4;
  __shared__ __attribute__((aligned(16))) char lds[kQBytes > kOBytes ? kQBytes : kOBytes];
  __shared__ f32x4 qoff[NR][kPgNG][16];  // what the codes' offsets add to a group's product, negated (four times: a C operand)
  __shared__ float qfac[ROWS];           // the power of two taken out of a row of Q
  __shared__ float mls[W][16][2];
  __shared__ __attribute__((aligned(16))) float sbuf[I4 ? W : 1][2][kPgNG][32];  // scales of a wave's keys and values
  __shared__ u32x4 m24[7];  // -24 eight times between zeros
  u32x4* qf = reinterpret_cast<u32x4*>(lds);  // [NR][hi, lo][8 steps][64 lanes]
  float* ob = reinterpret_cast<float*>(lds);  // [W waves][16][kORow], once Q has been used

  // ---- Q's rows, 16 lanes each, four waves a tile: row 4 (wave % 4) + lane / 16 of it, token r / G, head r % G of the group. Their loads and the norm
  // weight's go out before anything is known of the row's position, raw, so that nothing waits for them yet (16 rows of 16 bf16
  // tokens 25.4 -> 23.4 us, 512 tokens behind 16 K keys 117.4 -> 115.3).
  const int half = p.rot >> 1, qj = lane & 15, qcol = 4 * (wave & 3) + (lane >> 4);
  constexpr int QT = W == 4 ? NR : 1;  // tiles that a wave prepares: all, or tile wave / 4 where there is one
  const int q0 = W == 4 ? 0 : wave >> 2;
  u32x4 qx[QT][4], qp[QT][4];
  f32x4 wx[4], wp[4];
  auto pair_of = [&](int d) { return d >= p.rot ? d : d < half ? d + half : d - half; };
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    const int r = r0 + 16 * (q0 + i) + qcol, t = r / p.G, h = kvh * p.G + r - t * p.G;
    const int64_t o = b * p.qb + t * p.qt + h * p.qh;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      qx[i][q] = qp[i][q] = u32x4{0, 0, 0, 0};
      if (r < R && q0 + i < NR) {
        const int d = 64 * q + 4 * qj;
        qx[i][q] = quad_raw(p.q, p.q_f32, o + d);
        if (d < p.rot) qp[i][q] = quad_raw(p.q, p.q_f32, o + pair_of(d));
      }
    }
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    wx[q] = wp[q] = zero4();
    if (p.qw) {
      wx[q] = load_quad<float>(p.qw + 64 * q + 4 * qj);
      wp[q] = load_quad<float>(p.qw + pair_of(64 * q + 4 * qj));
    }
  }
  __builtin_amdgcn_sched_barrier(0);

  const int64_t pos = load_uniform(p.pos + b);
  const int len = p.lens ? min(max(load_uniform(p.lens + b), 0), p.T) : p.T;
  // the row's keys: those of its last token that is there (a later one sees more)
  int n_row = 0;
  if (len > 0) n_row = (int)min(max(pos + len, (int64_t)0), p.pt.capacity());
  const int t0 = r0 / p.G, t1 = (min(r0 + ROWS, R) - 1) / p.G;
  // what this block's rows see at most and at least
  int n_max = 0;
  if (t0 < len) n_max = (int)min(max(pos + min(t1, len - 1) + 1, (int64_t)0), p.pt.capacity());
  const int run = run_keys(n_row, p.S);
  const int k0 = s * run, k1 = min(k0 + run, n_max);
  const bool work = k0 < k1;
  if (!work && p.S > 1) return;  // the merge does not read empty runs' slots

  const int n_min = keys_seen(p, pos, len, t0), n_last = n_max - 1, pmask = (1 << p.pt.shift) - 1;
  // 16 keys from key0 on: the page (that of the last key for a tile past it, whose keys are masked) and the row in it.
  // Bases are scalar, a lane's part of the address 32 bits.
  struct Tile {
    size_t slot;
    bool ok;
  };
  auto tile_at = [&](int key0) -> Tile {
    const int page = p.pt.page_uniform(b, min(key0, n_last) >> p.pt.shift);
    return {(((size_t)max(page, 0) * p.Hkv + kvh) << p.pt.shift) + (key0 & pmask), page >= 0};
  };
  const uint32_t k_off = I4 ? 128 * c + 32 * a : 512 * c + 16 * a;
  const uint32_t v_off = I4 ? 128 * 4 * a + 8 * c : 16 * c;
  // (the empty asm keeps a base in scalar registers: folded with a lane's offset it would take two vector ones; the pointer
  // is made a global one again behind it, a generic one would make flat loads, which LDS waits count too)
  typedef const __attribute__((address_space(1))) char* gptr;
  auto base_of = [](const void* pages, size_t bytes) {
    uintptr_t src = (uintptr_t)pages + bytes;
    asm("" : "+s"(src));
    return (gptr)src;
  };
  // The scales of a wave's 32 keys are 256 bytes, a dword a lane: they pass through LDS, as fp32, to the lanes that need
  // them, four keys' of a tile at a time (loaded by these lanes they took 32 registers and 64 operations a round more).
  auto s_load = [&](const __bf16* pages, const Tile (&t)[2]) -> uint32_t {
    if constexpr (!I4) return 0;
    const gptr s0 = base_of(pages, t[0].slot * 8), s1 = base_of(pages, t[1].slot * 8);
    return *(const __attribute__((address_space(1))) uint32_t*)((lane < 32 ? s0 : s1) + 4 * (lane & 31));
  };
  auto s_share = [&](uint32_t mine, float (*buf)[32]) {
    buf[2 * (lane & 1)][lane >> 1] = bf16lo(mine);
    buf[2 * (lane & 1) + 1][lane >> 1] = bf16hi(mine);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  };
  struct Scales {  // of keys 4 a + r of two tiles, one group
    f32x4 s[2];
  };
  auto s_read = [&](const float (*buf)[32], int g) -> Scales {
    return {{*reinterpret_cast<const f32x4*>(&buf[g][4 * a]), *reinterpret_cast<const f32x4*>(&buf[g][16 + 4 * a])}};
  };
  auto k_load = [&](const Tile& t, KTile<I4>& k) {
    const gptr src = base_of(p.kp, t.slot * (I4 ? 128 : 512));
    if constexpr (I4) {
      k.c[0] = *(const __attribute__((address_space(1))) u32x4*)(src + k_off);
      k.c[1] = *(const __attribute__((address_space(1))) u32x4*)(src + (k_off + 16));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) k.c[i] = *(const __attribute__((address_space(1))) bf16x8*)(src + (k_off + 64 * i));
    }
  };
  // 32 rows against bf16: K's and V's operands share 64 registers (at two waves per SIMD there are 256, 136 of them
  // accumulators). As the scores release K's, V's are loaded, and the next K's as the sums release V's (512 tokens behind 16 K
  // keys 165 us; with registers for both, at one wave per SIMD, 185).
  constexpr bool kTurns = !I4 && NR == 2;
  auto v_load = [&](const Tile& t, VTile<I4>& v, int key0) {
    const gptr src = base_of(p.vp, t.slot * (I4 ? 128 : 512));
    if constexpr (I4) {
#pragma unroll
      for (int r = 0; r < 4; ++r) v.c[r] = *(const __attribute__((address_space(1))) u32x2*)(src + (v_off + 128 * r));
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        // rows past the last key may hold anything, and 0 times infinity is NaN: read the last key's row instead
        const uint32_t row = max(min(4 * a + r, n_last - key0), 0);
        v.c[r][0] = *(const __attribute__((address_space(1))) u32x4*)(src + (v_off + 512 * row));
        v.c[r][1] = *(const __attribute__((address_space(1))) u32x4*)(src + (v_off + 512 * row + 256));
      }
    }
  };
  auto k_part = [&](const Tile& t, KTile<I4>& k, int st) {
    if constexpr (kTurns)
      k.c[st] = *(const __attribute__((address_space(1))) bf16x8*)(base_of(p.kp, t.slot * 512) + (k_off + 64 * st));
  };
  auto v_part = [&](const Tile& t, VTile<I4>& v, int key0, int a4, int w, int r) {
    if constexpr (kTurns) {
      const uint32_t row = max(min(a4 + r, n_last - key0), 0);
      v.c[r][w] = *(const __attribute__((address_space(1))) u32x4*)(base_of(p.vp, t.slot * 512) + (v_off + 512 * row + 256 * w));
    }
  };

  // the rows' angles, ahead of the keys: loads return in order (the second tile's against bf16 when the first is done: there
  // are no registers for both beside the keys)
  constexpr int kAngles = kTurns ? 1 : QT;
  f32x4 co[kAngles][4], si[kAngles][4];
  auto angles = [&](int i, f32x4 (&co)[4], f32x4 (&si)[4]) {
    const int tk = (r0 + 16 * (q0 + i) + qcol) / p.G;
    const bool there = r0 + 16 * (q0 + i) + qcol < R && q0 + i < NR && keys_seen(p, pos, len, tk) > 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int d = 64 * q + 4 * qj, pj = d < half ? d : d - half;
      co[q] = si[q] = zero4();
      if (there && d < p.rot) {
        co[q] = load_quad<float>(p.cos_t + (pos + tk) * half + pj);
        si[q] = load_quad<float>(p.sin_t + (pos + tk) * half + pj);
      }
    }
  };
#pragma unroll
  for (int i = 0; i < kAngles; ++i) angles(i, co[i], si[i]);
  __builtin_amdgcn_sched_barrier(0);

  // ---- the first round's tiles, in flight while Q is prepared. The next round's tiles are loaded while this one's are
  // used, and their pages a round earlier still. A wave's last round loads its own tiles once more (from the cache) rather
  // than nothing: with no branch around the loads every wait counts how many of them may stay in flight.
  KTile<I4> kt[2];
  VTile<I4> vt[2];
  bool okv[2] = {true, true};
  int key = k0 + 32 * wave, next = key;
  Tile nt[2] = {{0, true}, {0, true}}, vt_at[2] = {{0, true}, {0, true}};
  uint32_t ks_mine = 0, vs_mine = 0;
  if (key < k1) {
#pragma unroll
    for (int u = 0; u < 2; ++u) nt[u] = tile_at(key + 16 * u);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      okv[u] = nt[u].ok;
      k_load(nt[u], kt[u]);
    }
    ks_mine = s_load(p.ks, nt);
    if constexpr (!kTurns) {
#pragma unroll
      for (int u = 0; u < 2; ++u) v_load(nt[u], vt[u], key + 16 * u);
    }
    vt_at[0] = nt[0];
    vt_at[1] = nt[1];
    vs_mine = s_load(p.vs, nt);
    if (key + KEYS < k1) next = key + KEYS;
#pragma unroll
    for (int u = 0; u < 2; ++u) nt[u] = tile_at(next + 16 * u);
  }
  __builtin_amdgcn_sched_barrier(0);

  // ---- Q: norm, rotation, scale log2(e), the split into hi + lo or the power of two, into LDS as B operands (rows that are
  // not there: zeros)
  if (work && q0 < NR) {
#pragma unroll
    for (int i = 0; i < QT; ++i) {
      const int tk = (r0 + 16 * (q0 + i) + qcol) / p.G, ia = i < kAngles ? i : 0;
      const bool there = r0 + 16 * (q0 + i) + qcol < R && keys_seen(p, pos, len, tk) > 0;
      if (i >= kAngles) angles(i, co[0], si[0]);
      f32x4 x[4], px[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        x[q] = there ? quad_value(qx[i][q], p.q_f32) : zero4();
        px[q] = there ? quad_value(qp[i][q], p.q_f32) : zero4();
      }
      float rr = 1.f;
      if (p.qw) {
        float ss = 0.f;
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int e = 0; e < 4; ++e) ss += x[q][e] * x[q][e];
        rr = rsqrtf(row16_sum(ss) * (1.f / kPgD) + p.eps);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int d = 64 * q + 4 * qj;
        const float sg = d < half ? -1.f : 1.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = x[q][e] * rr * (1.f + wx[q][e]);
          if (d < p.rot) v = v * co[ia][q][e] + sg * (px[q][e] * rr * (1.f + wp[q][e])) * si[ia][q][e];
          x[q][e] = v * (p.scale * 1.4426950408889634f);
        }
      }
      q_store<I4>(x, qj, qcol, qf + (size_t)(q0 + i) * QP * QF, qoff[q0 + i], &qfac[16 * (q0 + i) + qcol]);
    }
  }

  int seen[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    // rows that are not there are not stored: let them see what the others do, so that they ask for no mask
    const int r = r0 + 16 * i + c;
    seen[i] = r < R ? keys_seen(p, pos, len, r / p.G) : n_max;
  }
  f32x4 acc[NR][16];
  f32x4 corr[NR];  // 4 bits: -24 times the sum of the weights, of groups 0 .. 3
  float m_run[NR], l_run[NR], fac[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) {
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[i][e] = zero4();
    corr[i] = zero4();
    m_run[i] = -INFINITY;
    l_run[i] = 0.f;
  }
  // constants of the unpacking: the masks in scalar, the or-ed values in vector registers (one v_and_or_b32 takes both)
  uint32_t mk0 = 0x000F000Fu, mk1 = 0x00F000F0u, mv = 0x00780078u, ck = 0x64006400u, cv = 0x41804180u;
  asm("" : "+s"(mk0), "+s"(mk1), "+s"(mv), "+v"(ck), "+v"(cv));
  if (I4 && tid < 7) m24[tid] = tid == 3 ? u32x4{0xC1C0C1C0u, 0xC1C0C1C0u, 0xC1C0C1C0u, 0xC1C0C1C0u} : u32x4{0, 0, 0, 0};
  lds_barrier();
#pragma unroll
  for (int i = 0; i < NR; ++i) fac[i] = I4 ? qfac[16 * i + c] : 1.f;
  // 16 rows against codes: Q's operands and the offsets stay in registers
  constexpr bool kQReg = I4 && NR == 1;
  u32x4 qreg[kQReg ? 8 : 1];
  f32x4 zreg[kQReg ? kPgNG : 1];
  if constexpr (kQReg) {
#pragma unroll
    for (int k = 0; k < 8; ++k) qreg[k] = qf[64 * k + lane];
#pragma unroll
    for (int g = 0; g < kPgNG; ++g) zreg[g] = qoff[0][g][c];
  }

  while (key < k1) {
    int a4 = 4 * a;
    if constexpr (kTurns) asm volatile("" : "+v"(a4));  // (else 4 a + r are four more registers through the loop)
    // ---- scores, two tiles of 16 keys against each 16 rows
    f32x4 sc[2][NR];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < NR; ++i) sc[u][i] = zero4();
    if constexpr (I4) {
      s_share(ks_mine, sbuf[wave][0]);
#pragma unroll
      for (int g = 0; g < kPgNG; ++g) {
        const Scales ks = s_read(sbuf[wave][0], g);
        u32x4 ka[2][2];  // [tile][u]
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const uint32_t x = kt[u].c[g >> 1][2 * (g & 1) + w], y = x >> 8;
            ka[u][w] = u32x4{(x & mk0) | ck, (x & mk1) | ck, (y & mk0) | ck, (y & mk1) | ck};
          }
#pragma unroll
        for (int i = 0; i < NR; ++i) {
          f16x8 h0, h1;
          f32x4 z;
          if constexpr (kQReg) {
            h0 = __builtin_bit_cast(f16x8, qreg[2 * g]);
            h1 = __builtin_bit_cast(f16x8, qreg[2 * g + 1]);
            z = zreg[g];
          } else {
            const u32x4* qi = qf + (size_t)i * QF + 2 * g * 64 + lane;
            h0 = __builtin_bit_cast(f16x8, qi[0]);
            h1 = __builtin_bit_cast(f16x8, qi[64]);
            z = qoff[i][g][c];
          }
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            f32x4 d = mfma16h(ka[u][0], h0, z);
            d = mfma16h(ka[u][1], h1, d);
#pragma unroll
            for (int r = 0; r < 4; ++r) sc[u][i][r] += ks.s[u][r] * d[r];
          }
        }
        if constexpr (NR > 1) __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int st = 0; st < 8; ++st)
#pragma unroll
        for (int i = 0; i < NR; ++i) {
          const u32x4* qi = qf + (size_t)i * 2 * QF + st * 64 + lane;
          const bf16x8 hi = __builtin_bit_cast(bf16x8, qi[0]), lo = __builtin_bit_cast(bf16x8, qi[QF]);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            sc[u][i] = mfma16(kt[u].c[st], hi, sc[u][i]);
            sc[u][i] = mfma16(kt[u].c[st], lo, sc[u][i]);
          }
          if (!kTurns && (st & 1)) __builtin_amdgcn_sched_barrier(0);
          if (kTurns && i == NR - 1) {
            __builtin_amdgcn_sched_barrier(0);
            v_part(vt_at[0], vt[0], key, a4, st >> 2, st & 3);
            v_part(vt_at[1], vt[1], key + 16, a4, st >> 2, st & 3);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
    }
    if constexpr (!kTurns) {
      k_load(nt[0], kt[0]);
      k_load(nt[1], kt[1]);
    }
    ks_mine = s_load(p.ks, nt);
    const int after = next + KEYS < k1 ? next + KEYS : next;
    const Tile nn[2] = {tile_at(after), tile_at(after + 16)};
    __builtin_amdgcn_sched_barrier(0);
    // ---- masks, only where some row does not see every key of the two tiles
    const bool masked = key + 32 > n_min || !okv[0] || !okv[1];
    if (masked) {
#pragma unroll
      for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (key + 16 * u + a4 + r >= seen[i] || !okv[u]) sc[u][i][r] = -INFINITY;
    }
    // ---- running maximum (with a slack of 2^8 before the accumulators are rescaled) and the exponentials
    float pr[NR][8], mx[NR];
    bool up = false;
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      float m = -INFINITY;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) m = fmaxf(m, sc[u][i][r]);
      const lane_pair q = lane_swap<16>(m);
      m = max_xor32(fmaxf(q.a, q.b)) * fac[i];
      mx[i] = m;
      up |= m > m_run[i] + 8.f || (m_run[i] == -INFINITY && m > -INFINITY);
    }
    if (__builtin_amdgcn_ballot_w64(up) != 0) {
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        const float mn = fmaxf(m_run[i], mx[i]);
        const float f = m_run[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run[i] - mn);
        m_run[i] = mn;
        l_run[i] *= f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][e][r] *= f;
          __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (I4) {
#pragma unroll
          for (int g = 0; g < kPgNG; ++g) corr[i][g] *= f;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const float ms = m_run[i] == -INFINITY ? 0.f : m_run[i];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[u][i][r], fac[i], -ms));
          pr[i][4 * u + r] = e;
          l_run[i] += e;
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    // ---- P V
    if constexpr (I4) {
      s_share(vs_mine, sbuf[wave][1]);
      // a scale that is not finite or may make a weight so (2^118 and more)
      const bool wild = __builtin_amdgcn_ballot_w64((((vs_mine & 0x7F807F80u) + 0x05800580u) & 0x80008000u) != 0) != 0;
#pragma unroll
      for (int g = 0; g < kPgNG; ++g) {
        const Scales vs = s_read(sbuf[wave][1], g);
        float w[NR][8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
          for (int i = 0; i < NR; ++i) w[i][k] = pr[i][k] * vs.s[k >> 2][k & 3];
        if (wild && masked) {
          // a key that a row does not see weighs nothing there, whatever its scale is
#pragma unroll
          for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              asm volatile("" : "+v"(pr[i][k]));  // (keeps the comparisons inside the branch)
              if (pr[i][k] == 0.f) w[i][k] = 0.f;
            }
        }
        bf16x8 pg[NR];
#pragma unroll
        for (int i = 0; i < NR; ++i) {
          u32x4 pw;
#pragma unroll
          for (int k = 0; k < 4; ++k) pw[k] = cvt2(w[i][2 * k], w[i][2 * k + 1]);
          pg[i] = __builtin_bit_cast(bf16x8, pw);
        }
        uint32_t x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          x[k] = __builtin_amdgcn_perm(vt[k >> 1].c[2 * (k & 1) + 1][g >> 1], vt[k >> 1].c[2 * (k & 1)][g >> 1],
                                       g & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          u32x4 y;
#pragma unroll
          for (int k = 0; k < 4; ++k) y[k] = ((e == 0 ? x[k] << 3 : x[k] >> (4 * e - 3)) & mv) | cv;
          const bf16x8 va = __builtin_bit_cast(bf16x8, y);
#pragma unroll
          for (int i = 0; i < NR; ++i) acc[i][4 * g + e] = mfma16(va, pg[i], acc[i][4 * g + e]);
        }
        if (wild) {
          // (not finite: has reached its own group's sums, and must not the other groups')
#pragma unroll
          for (int i = 0; i < NR; ++i) {
            u32x4 pw = __builtin_bit_cast(u32x4, pg[i]);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if ((pw[k] & 0x7F80u) == 0x7F80u) pw[k] &= 0xFFFF0000u;
              if ((pw[k] & 0x7F800000u) == 0x7F800000u) pw[k] &= 0xFFFFu;
            }
            pg[i] = __builtin_bit_cast(bf16x8, pw);
          }
        }
        const bf16x8 off = __builtin_bit_cast(bf16x8, m24[(c & 3) + 3 - g]);  // -24 in the rows of group g
#pragma unroll
        for (int i = 0; i < NR; ++i) corr[i] = mfma16(off, pg[i], corr[i]);
        if constexpr (NR > 1) __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      bool odd = false;  // a value that is not finite, next to a weight of 0
      if (masked) {
        uint32_t any = 0;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
              for (int k = 0; k < 4; ++k) any |= ((vt[u].c[r][w][k] & 0x7F807F80u) + 0x00800080u) & 0x80008000u;
        odd = __builtin_amdgcn_ballot_w64(any != 0) != 0;
      }
      if (odd) {
        // What is not finite must not meet a weight of 0 in a product: it is taken out of the values here and added by
        // whether any weight meets it, +inf, -inf or both (NaN)
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int hl = 0; hl < 2; ++hl) {
              u32x4 up4 = {0, 0, 0, 0}, dn4 = {0, 0, 0, 0};
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const uint32_t word = vt[j >> 2].c[j & 3][w][k];
                const uint32_t v = (word >> (16 * hl)) & 0xFFFFu;
                uint32_t one = 0x3F80u << (16 * (j & 1)), rest = word & ~(0xFFFFu << (16 * hl));
                asm volatile("" : "+v"(one), "+v"(rest));  // (no register of theirs outside this branch)
                const bool bad = (v & 0x7F80u) == 0x7F80u;
                up4[j >> 1] |= bad && v != 0xFF80u ? one : 0u;
                dn4[j >> 1] |= bad && v != 0x7F80u ? one : 0u;
                vt[j >> 2].c[j & 3][w][k] = bad ? rest : word;
              }
#pragma unroll
              for (int i = 0; i < NR; ++i) {
                u32x4 on;
#pragma unroll
                for (int n = 0; n < 4; ++n)
                  on[n] = (pr[i][2 * n] != 0.f ? 0x3F80u : 0u) | (pr[i][2 * n + 1] != 0.f ? 0x3F800000u : 0u);
                const f32x4 cu = mfma16(__builtin_bit_cast(bf16x8, up4), __builtin_bit_cast(bf16x8, on), zero4());
                const f32x4 cd = mfma16(__builtin_bit_cast(bf16x8, dn4), __builtin_bit_cast(bf16x8, on), zero4());
                const int e = 8 * w + 2 * k + hl;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                  if (cu[r] > 0.f) acc[i][e][r] += INFINITY;
                  if (cd[r] > 0.f) acc[i][e][r] -= INFINITY;
                }
              }
              __builtin_amdgcn_sched_barrier(0);
            }
      }
      bf16x8 pg[NR];
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        u32x4 pw;
#pragma unroll
        for (int k = 0; k < 4; ++k) pw[k] = cvt2(pr[i][2 * k], pr[i][2 * k + 1]);
        pg[i] = __builtin_bit_cast(bf16x8, pw);
      }
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
#pragma unroll
          for (int hl = 0; hl < 2; ++hl) {
            const int e = 8 * w + 2 * k + hl;  // dim 128 w + 8 c + 2 k + hl
            u32x4 y;
#pragma unroll
            for (int n = 0; n < 4; ++n)
              y[n] = __builtin_amdgcn_perm(vt[n >> 1].c[2 * (n & 1) + 1][w][k], vt[n >> 1].c[2 * (n & 1)][w][k],
                                           hl ? 0x07060302u : 0x05040100u);
            const bf16x8 va = __builtin_bit_cast(bf16x8, y);
#pragma unroll
            for (int i = 0; i < NR; ++i) acc[i][e] = mfma16(va, pg[i], acc[i][e]);
          }
          __builtin_amdgcn_sched_barrier(0);
          if (kTurns && k == 3) {
#pragma unroll
            for (int st = 4 * w; st < 4 * w + 4; ++st) {
              k_part(nt[0], kt[0], st);
              k_part(nt[1], kt[1], st);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
        }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if constexpr (!kTurns) v_load(nt[u], vt[u], next + 16 * u);
      vt_at[u] = nt[u];
      okv[u] = nt[u].ok;
    }
    vs_mine = s_load(p.vs, nt);
    nt[0] = nn[0];
    nt[1] = nn[1];
    key += KEYS;
    next = after;
  }

  // ---- 16 rows at a time: each wave's rows (those that are there) into LDS, dims in order, then the waves joined, one
  // wave per row: the result, or the run's partial
  const int le = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)), ce = le & 15, ae = le >> 4, de = 4 * le;
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    float l = l_run[i];
    lane_pair q = lane_swap<16>(l);
    l = add_xor<32>(q.a + q.b);
    lds_barrier();  // Q, or the rows before these, have been used
    if (r0 + 16 * i + ce < R) {
      o_store<I4>(acc[i], corr[i], ob + ((size_t)wave * 16 + ce) * kORow, ae);
      if (ae == 0) {
        // (scores that are all NaN leave no maximum: their sum is joined all the same)
        mls[wave][ce][0] = m_run[i] == -INFINITY && l != l ? 0.f : m_run[i];
        mls[wave][ce][1] = l;
      }
    }
    lds_barrier();
#pragma unroll
    for (int jj = 0; jj < 16 / W; ++jj) {
      const int j = W * jj + wave;
      if (r0 + 16 * i + j >= R) break;
      const int r = r0 + 16 * i + j, t = r / p.G, h = kvh * p.G + r - t * p.G;
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < W; ++w) M = fmaxf(M, mls[w][j][0]);
      float L = 0.f;
      f32x4 O = zero4();
      if (M > -INFINITY) {
#pragma unroll
        for (int w = 0; w < W; ++w) {
          if (mls[w][j][0] == -INFINITY) continue;  // nothing seen
          const float f = __builtin_amdgcn_exp2f(mls[w][j][0] - M);
          L += mls[w][j][1] * f;
          const f32x4 v = *reinterpret_cast<const f32x4*>(ob + ((size_t)w * 16 + j) * kORow + de);
#pragma unroll
          for (int e = 0; e < 4; ++e) O[e] += v[e] * f;
        }
      }
      if (p.S > 1) {
        const size_t slot = (((size_t)b * p.Hkv + kvh) * R + r) * p.S + s;
        *reinterpret_cast<f32x4*>(p.part + slot * kPgD + de) = O;
        if (le < 2) p.ml[2 * slot + le] = le ? L : M;
      } else {
        out_store(p, O, L, keys_seen(p, pos, len, t) > 0, gate_load(p, b, t, h, de), b, t, h, de);
      }
    }
  }
}

// The runs of a query row (of batch row blockIdx.y) joined, U runs' loads in flight: by one wave, four rows a block, while
// that takes one go, else by the block's four waves, wave w folding runs w, w + 4, ... (512 tokens of 8 heads in 4 runs 5.4 us
// by one wave a row, 12.4 by four; 32 rows of five tokens in 8 runs 4.2 and 6.0).
template <int W, int U>
__global__ __launch_bounds__(256) void paged_attn_merge_kernel(PagedAttnArgs p) {
  const int lane = threadIdx.x & 63, d0 = 4 * lane;
  const int wave = W == 1 ? 0 : threadIdx.x >> 6;
  const int row = W == 1 ? 4 * (int)blockIdx.x + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : (int)blockIdx.x;
  const int kvh = row % p.Hkv, r = row / p.Hkv, b = blockIdx.y;
  const int R = p.T * p.G, t = r / p.G, h = kvh * p.G + r - t * p.G;
  if (W == 1 && r >= R) return;
  const int64_t pos = load_uniform(p.pos + b);
  const int len = p.lens ? min(max(load_uniform(p.lens + b), 0), p.T) : p.T;
  const int seen = keys_seen(p, pos, len, t);
  int n_row = 0;
  if (len > 0) n_row = (int)min(max(pos + len, (int64_t)0), p.pt.capacity());
  const int run = run_keys(n_row, p.S);
  // runs that hold keys this row sees (its block wrote them: the block's rows see at least as much)
  const int n = seen > 0 ? (seen + run - 1) / run : 0;
  const size_t base = (((size_t)b * p.Hkv + kvh) * R + r) * p.S;
  float M = -INFINITY, L = 0.f;
  f32x4 O = zero4();
  // the first runs are loaded without knowing n (slots of the workspace, whatever they hold), the gate with them
  f32x4 pv[U];
  float m[U], l[U];
  auto load = [&](int s0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const size_t s = base + min(s0 + W * u, p.S - 1);
      pv[u] = *reinterpret_cast<const f32x4*>(p.part + s * kPgD + d0);
      m[u] = p.ml[2 * s];
      l[u] = p.ml[2 * s + 1];
    }
  };
  load(wave);
  const f32x4 g = gate_load(p, b, t, h, d0);
  __builtin_amdgcn_sched_barrier(0);
  for (int s0 = wave; s0 < n; s0 += W * U) {
    if (s0 != wave) load(s0);
    // (selects, not branches, so that all loads are in flight together; a slot past n may hold anything)
    float mn = M;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      m[u] = s0 + W * u < n ? m[u] : -INFINITY;
      mn = fmaxf(mn, m[u]);
    }
    const float c0 = M > -INFINITY ? __builtin_amdgcn_exp2f(M - mn) : 0.f;
    L *= c0;
#pragma unroll
    for (int e = 0; e < 4; ++e) O[e] *= c0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = m[u] > -INFINITY;
      const float c1 = in ? __builtin_amdgcn_exp2f(m[u] - mn) : 0.f;
      L += in ? l[u] * c1 : 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) O[e] += in ? pv[u][e] * c1 : 0.f;
    }
    M = mn;
  }
  if constexpr (W == 1) {
    out_store(p, O, L, true, g, b, t, h, d0);
    return;
  }
  __shared__ float gm[4], gl[4];
  __shared__ f32x4 go[4][64];
  if (lane == 0) {
    gm[wave] = M;
    gl[wave] = L;
  }
  go[wave][lane] = O;
  __syncthreads();
  if (wave) return;
  float Mx = fmaxf(fmaxf(gm[0], gm[1]), fmaxf(gm[2], gm[3]));
  L = 0.f;
  O = zero4();
  if (Mx > -INFINITY) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (gm[w] == -INFINITY) continue;
      const float f = __builtin_amdgcn_exp2f(gm[w] - Mx);
      L += gl[w] * f;
#pragma unroll
      for (int e = 0; e < 4; ++e) O[e] += go[w][lane][e] * f;
    }
  }
  out_store(p, O, L, true, g, b, t, h, d0);
}

// Query rows per block, in 16s: two, which halves the unpacking and the LDS reads per row, but one where all rows fit in it
// (32 rows of up to 8192 keys, one token of four heads: bf16 95.9 us against 102.6, 4 bits 37.7 against 43.3) and for three
// 16s against codes, a quarter of whose work would be for rows that are not there (nine tokens of four heads: 64.6 against
// 70.7; 512 tokens, where none are: 150 against 123, bf16 303 against 165; five tokens, two 16s: 52.8 against 49.3).
// Runs per row: two blocks per CU, but one where that leaves a block no more than two
// rounds (three rows of 8192 4-bit keys: 64 runs 16.1 us, 32 runs 14.1, 16 runs 16.7). A table of two rounds is not split
// (256 keys, one row: 11.9 us against 12.5 for two runs and their merge, 4 bits 9.9 against 11.2; four rounds 16.4 against
// 12.7, 4 bits 12.6 against 11.3).
// Eight waves to a block, at one block per CU, for tables of two to four rounds that then need no merge either: up to three
// rounds of codes (one row of 384 keys 10.1 us against 10.6 for three runs, 32 rows 10.7 against 11.4; four rounds, 32 rows:
// 12.3 against 11.8) and two of bf16 for 32 query rows (18.4 against 19.5; one token's 16: 15.2 against 13.4: one CU then
// loads what two share); and all of them, but one token's two of bf16, where 65 to 256 blocks would be dealt to the CUs
// unevenly (80 rows of 384 keys: 19.2 us against 23.8, 4 bits 11.8 against 16.2).
struct PagedPlan {
  int NR, RB, S, W;
};
static PagedPlan paged_plan(int64_t B, int64_t T, int64_t Hkv, int64_t G, int64_t capacity, int64_t splits, int fmt) {
  const int64_t R = T * G, tiles = (R + 15) / 16;
  const int NR = tiles == 1 || (tiles == 3 && fmt == Q35_I4_G64) ? 1 : 2;
  const int64_t RB = (R + 16 * NR - 1) / (16 * NR), base = B * Hkv * RB;
  const int64_t most = (capacity + kRound - 1) / kRound;
  const bool i4 = fmt == Q35_I4_G64;
  const bool eight = base <= 256 && most > 1 && most <= 4 &&
                     (base > 64 ? i4 || NR == 2 || most > 2 : i4 ? most <= 3 : NR == 2 && most == 2);
  int64_t S = splits;
  if (S <= 0) {
    S = (512 + base - 1) / base;
    if (most <= 2 * S) S = (256 + base - 1) / base;
    if (most <= 2 || eight) S = 1;
  }
  if (S > most) S = most;
  if (S > 1024) S = 1024;
  if (S < 1) S = 1;
  return {NR, (int)RB, (int)S, S == 1 && eight ? 8 : 4};
}

}  // namespace q35

extern "C" size_t q35_gated_attn_paged_workspace_bytes(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                                                       int64_t n_blocks, int64_t page_size, int64_t splits) {
  using namespace q35;
  if (B <= 0 || T <= 0 || Hq <= 0 || Hkv <= 0 || D != kPgD || Hq % Hkv || n_blocks <= 0 || page_size <= 0 ||
      B > 65535 || T > (1 << 24) || Hq > 4096 || n_blocks > (1 << 26) || page_size > 1024)
    return 0;
  int S = 0;  // the larger of the two formats'
  for (const int fmt : {(int)Q35_BF16, (int)Q35_I4_G64})
    S = std::max(S, paged_plan(B, T, Hkv, Hq / Hkv, n_blocks * page_size, splits, fmt).S);
  if (S == 1) return 256;
  return (size_t)B * T * Hq * S * (kPgD + 2) * sizeof(float);
}

extern "C" int q35_gated_attn_paged(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* gate,
                                    int64_t g_sb, int64_t g_st, int64_t g_sh, int dtype, const float* q_norm_w,
                                    float eps, const float* cos, const float* sin, int64_t rot, const void* k_pages,
                                    const void* v_pages, const void* k_scale, const void* v_scale, int fmt,
                                    int64_t n_pages, int64_t page_size, const int32_t* table, int64_t ld_table,
                                    int64_t n_blocks, const int32_t* pos, const int32_t* lens, void* out,
                                    int out_dtype, int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                                    float scale, int64_t splits, void* workspace, size_t workspace_bytes,
                                    q35_stream_t stream) {
  using namespace q35;
  int shift = 0;
  int chk = paged_check(k_pages, v_pages, k_scale, v_scale, fmt, table, ld_table, n_blocks, n_pages, page_size, pos, B,
                        T, Hkv, D, &shift);
  if (chk == Q35_OK) chk = view_check(q, dtype, q_sb, q_st, q_sh);
  if (chk == Q35_OK && gate) chk = view_check(gate, dtype, g_sb, g_st, g_sh);
  if (chk != Q35_OK) return chk;
  if (!out || Hq <= 0 || Hq % Hkv || rot < 0 || rot > D || (rot & 1) || (rot > 0 && (!cos || !sin))) return Q35_EINVAL;
  if (out_dtype != Q35_BF16 && out_dtype != Q35_F32) return Q35_EUNSUPPORTED;
  if (rot % 8 || (uintptr_t)q_norm_w & 15 || (rot > 0 && ((uintptr_t)cos | (uintptr_t)sin) & 15) ||
      (uintptr_t)out & 15)
    return Q35_EUNSUPPORTED;
  const int64_t G = Hq / Hkv;
  if (Hq > 4096 || T * G > (1 << 24)) return Q35_EUNSUPPORTED;
  const PagedPlan pl = paged_plan(B, T, Hkv, G, n_blocks * page_size, splits, fmt);
  if (Hkv * pl.RB > 65535 || T * Hq > 0x7fffffff) return Q35_EUNSUPPORTED;
  const size_t rows = (size_t)B * T * Hq * pl.S;
  if (pl.S > 1 && (!workspace || workspace_bytes < rows * (kPgD + 2) * sizeof(float) || (uintptr_t)workspace & 15))
    return Q35_EWORKSPACE;
  PagedAttnArgs a{};
  a.q = q;
  a.gate = gate;
  a.qb = q_sb, a.qt = q_st, a.qh = q_sh, a.gb = g_sb, a.gt = g_st, a.gh = g_sh;
  a.qw = q_norm_w, a.cos_t = cos, a.sin_t = sin;
  a.eps = eps, a.scale = scale;
  a.rot = (int)rot, a.q_f32 = dtype == Q35_F32, a.out_f32 = out_dtype == Q35_F32;
  a.pt = {table, ld_table, (int)n_blocks, (int)n_pages, shift};
  a.pos = pos, a.lens = lens;
  a.kp = k_pages, a.vp = v_pages, a.ks = (const __bf16*)k_scale, a.vs = (const __bf16*)v_scale;
  a.out = out;
  a.part = (float*)workspace;
  a.ml = a.part ? a.part + rows * kPgD : nullptr;
  a.T = (int)T, a.Hkv = (int)Hkv, a.G = (int)G, a.S = pl.S, a.RB = pl.RB;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid(pl.S, (unsigned)(Hkv * pl.RB), (unsigned)B), block(256);
#define Q35_PAGED(I4, NR)                                                                            \
  do {                                                                                               \
    if (pl.W == 8) hipLaunchKernelGGL((paged_attn_kernel<I4, NR, 8>), grid, dim3(512), 0, st, a);    \
    else hipLaunchKernelGGL((paged_attn_kernel<I4, NR, 4>), grid, block, 0, st, a);                  \
  } while (0)
  if (fmt == Q35_BF16) {
    if (pl.NR == 1) Q35_PAGED(false, 1); else Q35_PAGED(false, 2);
  } else {
    if (pl.NR == 1) Q35_PAGED(true, 1); else Q35_PAGED(true, 2);
  }
#undef Q35_PAGED
  const unsigned n = (unsigned)(T * Hq);
  if (pl.S > 8) hipLaunchKernelGGL((paged_attn_merge_kernel<4, 8>), dim3(n, (unsigned)B), block, 0, st, a);
  else if (pl.S > 4) hipLaunchKernelGGL((paged_attn_merge_kernel<1, 8>), dim3((n + 3) / 4, (unsigned)B), block, 0, st, a);
  else if (pl.S > 1) hipLaunchKernelGGL((paged_attn_merge_kernel<1, 4>), dim3((n + 3) / 4, (unsigned)B), block, 0, st, a);
  return hipGetLastError() == hipSuccess ? Q35_OK : Q35_ELAUNCH;
}
