// New keys and values into a paged KV cache, and rows of one read back.
//
// paged_append_kernel: per (token, kv head) k' = rope_p(k rsqrt(mean k^2 + eps) (1 + w)) and v, written at the token's
// position p = pos[b] + t (HF:667-680; WGSL attnPrep, engine/kernels_qwen35.js:18-69, on pages). One wave per row of 256
// values, four dims a lane: the row's sum of squares is one wave sum, a group of 64 dims one row of 16 lanes.
//   bf16 pages: the arithmetic of attn_prep_kernel (fp32, then one rounding), bit for bit the rows it writes.
//   4-bit pages: per group s = bf16(fp32(max |x| / 7)), code = 8 + clamp(rint(x / s), -7, 7). A code is a rounding decision, so
//   norm, rotation and quotient are those of 64 bits: which code a value gets then depends on the inputs alone and not on
//   the order of a sum (in 32 bits about one value in 10^6 falls on the other side). They are formed in fp32 first, and
//   again in 64 bits only where a rounding lies closer to a tie than fp32 can tell (one row of 256 in a hundred): 6144
//   tokens of two heads, columns of an fp32 projection, 11.0 us (29 MB, 2.6 TB/s) against 17 in 64 bits throughout. A group
//   that holds a value that is not finite gets the scale NaN: it reads back as NaN.
//   Few tokens are a launch and one chain of loads: three of two heads 2.3 us, 32 rows of up to five 3.2; 6144
//   tokens into bf16 pages 9.6 us (38 MB, 3.9 TB/s).
//
// paged_rows_kernel: (code - 8) s, or the bf16 row, per 8 dims a thread. Bounded by memory: 8 rows of up to 8192 4-bit tokens
// of two heads 26.5 us (153 MB, most of it the bf16 rows written; a 1 GiB copy runs at 5.2 TB/s), bf16 rows 49 (5.0 TB/s).
#include "paged_kv.h"

namespace q35 {

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

// The same from fp32 values, where they settle it: x[e] within 2^-20 of a[e] (at least |x[e]|) of the 64-bit value (12 half
// steps of fp32: the sum of squares 5, its root 2, the products 3, the rotation 2; the tables may hold any size). Sets
// *sure false in a lane that finds its scale's or a code's rounding within that error (with 2^-19 taken for it, which also
// covers the quotient's) of a tie, or a maximum outside 1e-30 .. 1e30.
__device__ __forceinline__ uint32_t quantize_quad_f32(const f32x4& x, const f32x4& a, bool turned, __bf16* s_out,
                                                      bool* sure) {
  const float m = row16_max_f32(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))));
  // (what was not rotated is its own bound)
  const float am = turned ? row16_max_f32(fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3]))) : m;
  const float s32 = m * (1.f / 7.f), off = am * (0x1p-19f / 7.f);
  const __bf16 sb = (__bf16)s32;
  const float s = (float)sb, inv = __builtin_amdgcn_rcpf(s), wide = inv * 0x1p-19f;
  float far = 0.f;  // the largest distance from a code, with its error
  uint32_t q = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float t = x[e] * inv, n = __builtin_rintf(t);
    far = fmaxf(far, __builtin_fmaf(a[e], wide, fabsf(t - n)));
    q |= (uint32_t)(__builtin_amdgcn_fmed3f(n, -7.f, 7.f) + 8.f) << (4 * e);
  }
  *s_out = sb;
  const float sum = x[0] + x[1] + x[2] + x[3];  // (a maximum passes over a NaN, a sum does not)
  *sure = sum == sum && m > 1e-30f && am < 1e30f && far < 0.5f && (float)(__bf16)(s32 - off) == s &&
          (float)(__bf16)(s32 + off) == s;
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
};

// Wave: one token's row of head blockIdx.y / 2, its keys (even blockIdx.y) or values, of row blockIdx.z. What bounds a long
// prompt is latency: a wave has one row in flight, and its position, page, angles, reductions and store follow each other (the
// vector ALU is 37 % busy with about 150 operations a row). Several rows a wave, with their loads ahead, measured an eighth
// slower all the same (four a wave, 6144 tokens of two heads).
template <typename Tin, bool I4>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendArgs p) {
  const int lane = threadIdx.x & 63, b = blockIdx.z, h = blockIdx.y >> 1;
  const int t = (int)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool val = blockIdx.y & 1;
  const int len = p.lens ? min(load_uniform(p.lens + b), p.T) : p.T;
  const int64_t at = (int64_t)load_uniform(p.pos + b) + t;
  if (t >= p.T) return;
  const int d0 = 4 * lane, half = p.rot >> 1;
  const bool turns = !val && d0 < p.rot;  // lanes past rot keep their values
  const int pd = !turns ? d0 : d0 < half ? d0 + half : d0 - half;
  const Tin* src = val ? (const Tin*)p.v + (b * p.vb + h * p.vh + t * p.vt) : (const Tin*)p.k + (b * p.kb + h * p.kh + t * p.kt);
  const f32x4 x = load_quad<Tin>(src + d0);
  f32x4 px = x, wx = zero4(), wp = zero4(), co = zero4(), si = zero4();
  if (!val) {
    px = load_quad<Tin>(src + pd);
    if (p.kw) {
      wx = load_quad<float>(p.kw + d0);
      wp = load_quad<float>(p.kw + pd);
    }
  }
  if (t >= len || at < 0 || at >= p.pt.capacity()) return;
  const int page = p.pt.page_uniform(b, (int)(at >> p.pt.shift));
  if (page < 0) return;
  if (turns) {
    const int j = d0 < half ? d0 : d0 - half;
    co = load_quad<float>(p.cos_t + at * half + j);
    si = load_quad<float>(p.sin_t + at * half + j);
  }
  const size_t slot = (((size_t)page * p.Hkv + h) << p.pt.shift) + ((int)at & ((1 << p.pt.shift) - 1));
  const float sg = d0 < half ? -1.f : 1.f;
  // in fp32 (what bf16 pages hold, rounded); big: the terms' magnitudes, which bound the error
  f32x4 r = x, big;
  bool norm_ok = true;
#pragma unroll
  for (int e = 0; e < 4; ++e) big[e] = fabsf(x[e]);
  if (!val) {
    f32x4 xn = x, pn = px;
    if (p.kw) {
      const float ss = wave_sum(x[0] * x[0] + x[1] * x[1] + x[2] * x[2] + x[3] * x[3]);
      const float ms = ss * (1.f / kPgD) + p.eps, rr = rsqrtf(ms);
      norm_ok = ms > 1e-30f;  // (smaller squares lose bits)
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
#pragma unroll
    for (int e = 0; e < 4; ++e) big[e] = turns ? fabsf(xn[e] * co[e]) + fabsf(pn[e] * si[e]) : fabsf(xn[e]);
  }
  if constexpr (!I4) {
    bf16x4 o = {(__bf16)r[0], (__bf16)r[1], (__bf16)r[2], (__bf16)r[3]};
    *reinterpret_cast<bf16x4*>((__bf16*)(val ? p.vp : p.kp) + slot * kPgD + d0) = o;
  } else {
    __bf16 s;
    bool sure;
    uint32_t q = quantize_quad_f32(r, big, !val && p.rot > 0, &s, &sure);
    if (__builtin_amdgcn_ballot_w64(!(sure && norm_ok)) != 0) {
      double d[4] = {x[0], x[1], x[2], x[3]};
      if (!val) {
        double pn[4] = {px[0], px[1], px[2], px[3]};
        if (p.kw) {
          const double ss = wave_sum64(d[0] * d[0] + d[1] * d[1] + d[2] * d[2] + d[3] * d[3]);
          const double rr = 1.0 / sqrt(ss * (1.0 / kPgD) + (double)p.eps);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            d[e] = d[e] * rr * (1.0 + (double)wx[e]);
            pn[e] = pn[e] * rr * (1.0 + (double)wp[e]);
          }
        }
        if (turns) {
#pragma unroll
          for (int e = 0; e < 4; ++e) d[e] = d[e] * (double)co[e] + (double)sg * pn[e] * (double)si[e];
        }
      }
      q = quantize_quad(d, &s);
    }
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
};

// Block: 32 tokens of row blockIdx.z, head blockIdx.y / 2, its keys (even blockIdx.y) or values; thread: dims 8 m .. 8 m + 7 (m = tid % 32) of four of
// them, all loaded before the first is stored.
template <bool I4>
__global__ __launch_bounds__(256) void paged_rows_kernel(RowsArgs p) {
  const int m = threadIdx.x & 31, h = blockIdx.y >> 1, b = blockIdx.z;
  const bool val = blockIdx.y & 1;
  const int len = p.lens ? min(load_uniform(p.lens + b), p.T) : p.T;
  const int64_t pos = load_uniform(p.pos + b);
  const int t0 = (int)blockIdx.x * 32 + (threadIdx.x >> 5);
  const char* src = (const char*)(val ? p.vp : p.kp);
  const __bf16* scale = val ? p.vs : p.ks;
  size_t slot[4];
  bool there[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int t = t0 + 8 * u;
    const int64_t at = pos + t;
    there[u] = t < len && at >= 0 && at < p.pt.capacity();
    const int page = there[u] ? p.pt.page(b, (int)(at >> p.pt.shift)) : -1;
    there[u] = page >= 0;
    slot[u] = there[u] ? (((size_t)page * p.Hkv + h) << p.pt.shift) + ((int)at & ((1 << p.pt.shift) - 1)) : 0;
  }
  u32x4 out[4];
  if constexpr (!I4) {
#pragma unroll
    for (int u = 0; u < 4; ++u) out[u] = *reinterpret_cast<const u32x4*>(src + slot[u] * (2 * kPgD) + 16 * m);
  } else {
    uint32_t w[4];
    float s[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const char* row = src + slot[u] * (kPgD / 2);
      if (val)
        w[u] = *reinterpret_cast<const uint16_t*>(row + v_quad_byte(2 * m)) |
               (uint32_t)*reinterpret_cast<const uint16_t*>(row + v_quad_byte(2 * m + 1)) << 16;
      else
        w[u] = *reinterpret_cast<const uint32_t*>(row + k_quad_byte(2 * m));
      s[u] = (float)scale[slot[u] * kPgNG + (m >> 3)];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      bf16x8 o;
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = (__bf16)((float)((int)(w[u] >> (4 * j) & 15) - 8) * s[u]);
      out[u] = __builtin_bit_cast(u32x4, o);
    }
  }
  __bf16* dst = (val ? p.vo : p.ko) + (((size_t)b * p.Hkv + h) * p.T + t0) * kPgD + 8 * m;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const u32x4 zero = {0, 0, 0, 0};
    if (t0 + 8 * u < p.T)
      __builtin_nontemporal_store(there[u] ? out[u] : zero, reinterpret_cast<u32x4*>(dst + (size_t)8 * u * kPgD));
  }
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
  const AppendArgs a{k,     v,    k_sb,    k_st,    k_sh,          v_sb,          v_st,   v_sh,     k_norm_w, cos, sin, eps,
                     (int)rot, {table, ld_table, (int)n_blocks, (int)n_pages, shift}, pos, lens, k_pages, v_pages,
                     (__bf16*)k_scale, (__bf16*)v_scale, (int)T, (int)Hkv};
  const dim3 grid((unsigned)((T + 3) / 4), (unsigned)(2 * Hkv), (unsigned)B), block(256);
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
  const RowsArgs a{k_pages, v_pages, (const __bf16*)k_scale, (const __bf16*)v_scale,
                   {table, ld_table, (int)n_blocks, (int)n_pages, shift}, pos, lens, (__bf16*)k_out, (__bf16*)v_out,
                   (int)T, (int)Hkv};
  const dim3 grid((unsigned)((T + 31) / 32), (unsigned)(2 * Hkv), (unsigned)B), block(256);
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (fmt == Q35_BF16) hipLaunchKernelGGL(paged_rows_kernel<false>, grid, block, 0, st, a);
  else hipLaunchKernelGGL(paged_rows_kernel<true>, grid, block, 0, st, a);
  return hipGetLastError() == hipSuccess ? Q35_OK : Q35_ELAUNCH;
}
