// New keys and values into a paged KV cache, and rows of one read back.
//
// paged_append_kernel: per (token, kv head) k' = rope_p(k rsqrt(mean k^2 + eps) (1 + w)) and v, written at the token's
// position p = pos[b] + t (HF:667-680; WGSL attnPrep, engine/kernels_qwen35.js:18-69, on pages). One wave per row of 256
// values, four dims a lane: the row's sum of squares is one wave sum, a group of 64 dims one row of 16 lanes.
//   bf16 pages: the arithmetic of attn_prep_kernel (fp32, then one rounding), bit for bit the rows it writes.
//   4-bit pages: per group s = bf16(fp32(max |x| / 7)), code = 8 + clamp(rint(x / s), -7, 7). A code is a rounding decision, so
//   norm, rotation and quotient are formed in 64 bits: which code a value gets then depends on the inputs alone and not on
//   the order of a sum (in 32 bits about one value in 10^6 falls on the other side). fp64 multiply-adds run at the fp32
//   rate here. A group that holds a value that is not finite gets the scale NaN: it reads back as NaN.
#include "paged_kv.h"

namespace q35 {

// The value of the lane that DPP control CTRL names, for 64-bit values.
template <int CTRL> __device__ __forceinline__ double dpp64(double v) {
  const u32x2 w = __builtin_bit_cast(u32x2, v);
  u32x2 r;
  r.x = __builtin_amdgcn_mov_dpp(w.x, CTRL, 0xF, 0xF, false);
  r.y = __builtin_amdgcn_mov_dpp(w.y, CTRL, 0xF, 0xF, false);
  return __builtin_bit_cast(double, r);
}
template <int OFF> __device__ __forceinline__ double swap_add64(double v) {
  const u32x2 w = __builtin_bit_cast(u32x2, v);
  const auto lo = OFF == 32 ? __builtin_amdgcn_permlane32_swap(w.x, w.x, false, false)
                            : __builtin_amdgcn_permlane16_swap(w.x, w.x, false, false);
  const auto hi = OFF == 32 ? __builtin_amdgcn_permlane32_swap(w.y, w.y, false, false)
                            : __builtin_amdgcn_permlane16_swap(w.y, w.y, false, false);
  u32x2 a, b;
  a.x = lo[0];
  a.y = hi[0];
  b.x = lo[1];
  b.y = hi[1];
  return __builtin_bit_cast(double, a) + __builtin_bit_cast(double, b);
}
__device__ __forceinline__ double wave_sum64(double v) {
  v += dpp64<0xB1>(v);
  v += dpp64<0x4E>(v);
  v += dpp64<0x141>(v);
  v += dpp64<0x140>(v);
  return swap_add64<32>(swap_add64<16>(v));
}
__device__ __forceinline__ double row16_max64(double v) {
  v = fmax(v, dpp64<0xB1>(v));
  v = fmax(v, dpp64<0x4E>(v));
  v = fmax(v, dpp64<0x141>(v));
  return fmax(v, dpp64<0x140>(v));
}

// Codes of four values (low nibble first) and their group's scale; a group is 16 lanes.
__device__ __forceinline__ uint32_t quantize_quad(const double (&x)[4], __bf16* s_out) {
  double m = fmax(fmax(fabs(x[0]), fabs(x[1])), fmax(fabs(x[2]), fabs(x[3])));
  // x - x is 0 for every finite x: any lane of the group that holds another value makes m infinite
  const double bad = (x[0] - x[0]) + (x[1] - x[1]) + (x[2] - x[2]) + (x[3] - x[3]);
  if (!(bad == 0.0)) m = INFINITY;
  m = row16_max64(m);
  // rounded to fp32, then to bf16: one of the two alone would give some groups near a tie another scale
  float s32 = (float)(m / 7.0);
  asm volatile("" : "+v"(s32));
  const __bf16 sb = (__bf16)s32;
  const double s = (double)(float)sb;
  uint32_t q = 0;
  if (s > 0.0 && s < INFINITY) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const double n = fmin(fmax(__builtin_rint(x[e] / s), -7.0), 7.0);
      q |= (uint32_t)((int)n + 8) << (4 * e);
    }
  } else {
    q = 0x8888;
  }
  *s_out = s < INFINITY ? sb : (__bf16)__builtin_nanf("");
  return q;
}

struct AppendArgs {
  const void *k, *v;
  int64_t kb, kt, kh, vb, vt, vh;
  const float *kw, *cos_t, *sin_t;
  float eps;
  int rot;
  PagedTable pt;
  const int32_t *pos, *lens;
  void *kp, *vp;
  __bf16 *ks, *vs;
  int T, Hkv;
  int64_t jobs;
};

// Job g = ((b T + t) Hkv + h) 2 + (0: key, 1: value), one wave each.
template <typename Tin, bool I4>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendArgs p) {
  const int lane = threadIdx.x & 63;
  const int64_t g = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (g >= p.jobs) return;
  const bool val = g & 1;
  const int64_t th = g >> 1, m = th / p.Hkv;
  const int h = (int)(th - m * p.Hkv), b = (int)(m / p.T), t = (int)(m - (int64_t)b * p.T);
  const int d0 = 4 * lane, half = p.rot >> 1;
  const Tin* src = val ? (const Tin*)p.v + b * p.vb + t * p.vt + h * p.vh
                       : (const Tin*)p.k + b * p.kb + t * p.kt + h * p.kh;
  const f32x4 x = load_quad<Tin>(src + d0);
  const int64_t at = (int64_t)p.pos[b] + t;
  if (at < 0 || at >= p.pt.capacity() || (p.lens && t >= p.lens[b])) return;
  const int page = p.pt.page(b, (int)(at >> p.pt.shift));
  if (page < 0) return;
  const int row = (int)at & ((1 << p.pt.shift) - 1);
  const size_t slot = (((size_t)page * p.Hkv + h) << p.pt.shift) + row;

  // The key's rotation partner and its table row (lanes past rot keep their values)
  f32x4 px = x, wx = zero4(), wp = zero4(), co = zero4(), si = zero4();
  const bool turns = !val && d0 < p.rot;
  const float sg = d0 < half ? -1.f : 1.f;
  if (!val && p.kw) wx = load_quad<float>(p.kw + d0);
  if (turns) {
    const int pd = d0 < half ? d0 + half : d0 - half, j = d0 < half ? d0 : d0 - half;
    px = load_quad<Tin>(src + pd);
    if (p.kw) wp = load_quad<float>(p.kw + pd);
    co = load_quad<float>(p.cos_t + at * half + j);
    si = load_quad<float>(p.sin_t + at * half + j);
  }
  if constexpr (!I4) {
    f32x4 r = x;
    if (!val) {
      f32x4 xn = x, pn = px;
      if (p.kw) {
        const float ss = wave_sum(x[0] * x[0] + x[1] * x[1] + x[2] * x[2] + x[3] * x[3]);
        const float rr = rsqrtf(ss * (1.f / kPgD) + p.eps);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          xn[e] = x[e] * rr * (1.f + wx[e]);
          pn[e] = px[e] * rr * (1.f + wp[e]);
        }
      }
      r = xn;
      if (turns) {
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = xn[e] * co[e] + sg * pn[e] * si[e];
      }
    }
    bf16x4 o = {(__bf16)r[0], (__bf16)r[1], (__bf16)r[2], (__bf16)r[3]};
    *reinterpret_cast<bf16x4*>((__bf16*)(val ? p.vp : p.kp) + slot * kPgD + d0) = o;
  } else {
    double r[4] = {x[0], x[1], x[2], x[3]};
    if (!val) {
      double pn[4] = {px[0], px[1], px[2], px[3]};
      if (p.kw) {
        const double ss = wave_sum64(r[0] * r[0] + r[1] * r[1] + r[2] * r[2] + r[3] * r[3]);
        const double rr = 1.0 / sqrt(ss * (1.0 / kPgD) + (double)p.eps);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          r[e] = r[e] * rr * (1.0 + (double)wx[e]);
          pn[e] = pn[e] * rr * (1.0 + (double)wp[e]);
        }
      }
      if (turns) {
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = r[e] * (double)co[e] + (double)sg * pn[e] * (double)si[e];
      }
    }
    __bf16 s;
    const uint32_t q = quantize_quad(r, &s);
    char* dst = (char*)(val ? p.vp : p.kp) + slot * (kPgD / 2);
    *reinterpret_cast<uint16_t*>(dst + (val ? v_quad_byte(lane) : k_quad_byte(lane))) = (uint16_t)q;
    if ((lane & 15) == 0) (val ? p.vs : p.ks)[slot * kPgNG + (lane >> 4)] = s;
  }
}

struct RowsArgs {
  const void *kp, *vp;
  const __bf16 *ks, *vs;
  PagedTable pt;
  const int32_t *pos, *lens;
  __bf16 *ko, *vo;
  int T, Hkv;
  int64_t n;  // threads: B Hkv T rows of keys and of values, 32 threads each
};

// Thread i: dims 8 m .. 8 m + 7 (m = i % 32) of one row: out row (b Hkv + h) T + t, keys first, then values.
template <bool I4>
__global__ __launch_bounds__(256) void paged_rows_kernel(RowsArgs p) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= 2 * p.n) return;
  const bool val = i >= p.n;
  const int64_t r = (val ? i - p.n : i) >> 5, bh = r / p.T;
  const int m = (int)(i & 31), t = (int)(r - bh * p.T);
  const int b = (int)(bh / p.Hkv), h = (int)(bh - (int64_t)b * p.Hkv);
  u32x4 out = {0, 0, 0, 0};
  const int64_t at = (int64_t)p.pos[b] + t;
  if (at >= 0 && at < p.pt.capacity() && (!p.lens || t < p.lens[b])) {
    const int page = p.pt.page(b, (int)(at >> p.pt.shift));
    if (page >= 0) {
      const size_t slot = (((size_t)page * p.Hkv + h) << p.pt.shift) + ((int)at & ((1 << p.pt.shift) - 1));
      if constexpr (!I4) {
        out = *reinterpret_cast<const u32x4*>((const __bf16*)(val ? p.vp : p.kp) + slot * kPgD + 8 * m);
      } else {
        const char* src = (const char*)(val ? p.vp : p.kp) + slot * (kPgD / 2);
        uint32_t w;
        if (val)
          w = *reinterpret_cast<const uint16_t*>(src + v_quad_byte(2 * m)) |
              (uint32_t)*reinterpret_cast<const uint16_t*>(src + v_quad_byte(2 * m + 1)) << 16;
        else
          w = *reinterpret_cast<const uint32_t*>(src + k_quad_byte(2 * m));
        const float s = (float)(val ? p.vs : p.ks)[slot * kPgNG + (m >> 3)];
        bf16x8 o;
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = (__bf16)((float)((int)(w >> (4 * j) & 15) - 8) * s);
        out = __builtin_bit_cast(u32x4, o);
      }
    }
  }
  *reinterpret_cast<u32x4*>((val ? p.vo : p.ko) + r * kPgD + 8 * m) = out;
}

}  // namespace q35

extern "C" int q35_paged_kv_append(const void* k, int64_t k_sb, int64_t k_st, int64_t k_sh, const void* v,
                                   int64_t v_sb, int64_t v_st, int64_t v_sh, int dtype, const float* k_norm_w,
                                   float eps, const float* cos, const float* sin, int64_t rot, const int32_t* table,
                                   int64_t ld_table, int64_t n_blocks, const int32_t* pos, const int32_t* lens,
                                   void* k_pages, void* v_pages, void* k_scale, void* v_scale, int fmt,
                                   int64_t n_pages, int64_t page_size, int64_t B, int64_t T, int64_t Hkv, int64_t D,
                                   q35_stream_t stream) {
  using namespace q35;
  int shift = 0;
  int chk = paged_check(k_pages, v_pages, k_scale, v_scale, fmt, table, ld_table, n_blocks, n_pages, page_size, pos, B,
                        T, Hkv, D, &shift);
  if (chk == Q35_OK) chk = view_check(k, dtype, k_sb, k_st, k_sh);
  if (chk == Q35_OK) chk = view_check(v, dtype, v_sb, v_st, v_sh);
  if (chk != Q35_OK) return chk;
  if (rot < 0 || rot > D || (rot & 1) || (rot > 0 && (!cos || !sin))) return Q35_EINVAL;
  if (rot % 8 || (uintptr_t)k_norm_w & 15 || (rot > 0 && ((uintptr_t)cos | (uintptr_t)sin) & 15))
    return Q35_EUNSUPPORTED;
  const int64_t jobs = B * T * Hkv * 2;
  if ((jobs + 3) / 4 > 0x7fffffff) return Q35_EUNSUPPORTED;
  const AppendArgs a{k,     v,    k_sb,    k_st,    k_sh,          v_sb,          v_st,   v_sh,     k_norm_w, cos, sin, eps,
                     (int)rot, {table, ld_table, (int)n_blocks, (int)n_pages, shift}, pos, lens, k_pages, v_pages,
                     (__bf16*)k_scale, (__bf16*)v_scale, (int)T, (int)Hkv, jobs};
  const dim3 grid((unsigned)((jobs + 3) / 4)), block(256);
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == Q35_F32) {
    if (fmt == Q35_BF16) hipLaunchKernelGGL((paged_append_kernel<float, false>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((paged_append_kernel<float, true>), grid, block, 0, st, a);
  } else {
    if (fmt == Q35_BF16) hipLaunchKernelGGL((paged_append_kernel<__bf16, false>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((paged_append_kernel<__bf16, true>), grid, block, 0, st, a);
  }
  return hipGetLastError() == hipSuccess ? Q35_OK : Q35_ELAUNCH;
}

extern "C" int q35_paged_kv_rows(const void* k_pages, const void* v_pages, const void* k_scale, const void* v_scale,
                                 int fmt, int64_t n_pages, int64_t page_size, const int32_t* table, int64_t ld_table,
                                 int64_t n_blocks, const int32_t* pos, const int32_t* lens, void* k_out, void* v_out,
                                 int64_t B, int64_t T, int64_t Hkv, int64_t D, q35_stream_t stream) {
  using namespace q35;
  int shift = 0;
  const int chk = paged_check(k_pages, v_pages, k_scale, v_scale, fmt, table, ld_table, n_blocks, n_pages, page_size,
                              pos, B, T, Hkv, D, &shift);
  if (chk != Q35_OK) return chk;
  if (!k_out || !v_out) return Q35_EINVAL;
  if (((uintptr_t)k_out | (uintptr_t)v_out) & 15) return Q35_EUNSUPPORTED;
  const int64_t n = B * Hkv * T * 32;
  if ((2 * n + 255) / 256 > 0x7fffffff) return Q35_EUNSUPPORTED;
  const RowsArgs a{k_pages, v_pages, (const __bf16*)k_scale, (const __bf16*)v_scale,
                   {table, ld_table, (int)n_blocks, (int)n_pages, shift}, pos, lens, (__bf16*)k_out, (__bf16*)v_out,
                   (int)T, (int)Hkv, n};
  const dim3 grid((unsigned)((2 * n + 255) / 256)), block(256);
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (fmt == Q35_BF16) hipLaunchKernelGGL(paged_rows_kernel<false>, grid, block, 0, st, a);
  else hipLaunchKernelGGL(paged_rows_kernel<true>, grid, block, 0, st, a);
  return hipGetLastError() == hipSuccess ? Q35_OK : Q35_ELAUNCH;
}
