// Paged KV cache: what the append, the read-back and the attention kernels share.
//
// Pages: k, v [n_pages, Hkv, page_size, ...] with page_size a power of two of at least 16 tokens, so that a 16-key tile
// lies inside one page. Token position p of row b sits in page table[b * ld_table + p / page_size], at row p % page_size.
// A table entry outside 0 .. n_pages - 1 names no page: nothing is written there and its keys are not attended to.
//
// Rows of 256 values: bf16 in order (512 bytes), or 4 bits (Q35_I4_G64, 128 bytes + 4 bf16 scales). Of the 4-bit form,
// code n in 0 .. 15 of group g (dims 64 g .. 64 g + 63) stands for (n - 8) s_g. The nibbles of a row lie in the order in
// which the attention kernel's lanes take them, so that each lane's part is one run of bytes:
//   keys    dim 64 g + 16 a + 8 u + j  at nibble 64 a + 16 g + 8 u + j  (g, a < 4, u < 2, j < 8): lane group a of a
//           16x16x32 MFMA's A operand reads 32 bytes, dword 2 g + u of them is its 8 dims of step (g, u)
//   values  dim 64 g + 4 c + e         at nibble 16 c + 4 g + e         (g, e < 4, c < 16): lane c of the A operand of
//           V^T reads 8 bytes, 16 bits per group
#pragma once
#include "q35_common.h"
#include "q35hip.h"

namespace q35 {

constexpr int kPgD = 256;     // head dim
constexpr int kPgGroup = 64;  // dims per scale of the 4-bit form
constexpr int kPgNG = kPgD / kPgGroup;

struct PagedTable {
  const int32_t* table;
  int64_t ld;
  int n_blocks, n_pages, shift;  // page size 1 << shift

  // The page of block `blk` (0 .. n_blocks - 1) of row b, or -1.
  __device__ __forceinline__ int page(int b, int blk) const {
    const int p = table[(int64_t)b * ld + blk];
    return p >= 0 && p < n_pages ? p : -1;
  }
  // The same for arguments that a whole wave shares.
  __device__ __forceinline__ int page_uniform(int b, int blk) const {
    const int p = load_uniform(table + (int64_t)b * ld + blk);
    return p >= 0 && p < n_pages ? p : -1;
  }
  __device__ __forceinline__ int64_t capacity() const { return (int64_t)n_blocks << shift; }
};

// Byte of the quad of codes of dims 4 l .. 4 l + 3 in a row.
__device__ __forceinline__ int k_quad_byte(int l) { return 32 * ((l & 15) >> 2) + 8 * (l >> 4) + 2 * (l & 3); }
__device__ __forceinline__ int v_quad_byte(int l) { return 8 * (l & 15) + 2 * (l >> 4); }

// Host checks of the page arguments shared by the entry points.
inline int paged_check(const void* k_pages, const void* v_pages, const void* k_scale, const void* v_scale, int fmt,
                       const int32_t* table, int64_t ld_table, int64_t n_blocks, int64_t n_pages, int64_t page_size,
                       const int32_t* pos, int64_t B, int64_t T, int64_t Hkv, int64_t D, int* shift) {
  if (!k_pages || !v_pages || !table || !pos) return Q35_EINVAL;
  if (B <= 0 || T <= 0 || Hkv <= 0 || D <= 0 || n_blocks <= 0 || n_pages <= 0 || page_size <= 0) return Q35_EINVAL;
  if (B > 1 && ld_table < n_blocks && ld_table != 0) return Q35_EINVAL;  // (0: one table for all rows)
  if (fmt != Q35_BF16 && fmt != Q35_I4_G64) return Q35_EUNSUPPORTED;
  if (fmt == Q35_I4_G64 && (!k_scale || !v_scale)) return Q35_EINVAL;
  if (D != kPgD || page_size < 16 || page_size > 1024 || (page_size & (page_size - 1))) return Q35_EUNSUPPORTED;
  if (B > 65535 || Hkv > 4096 || T > (1 << 24) || n_pages > 0x7fffffff || n_blocks > (1 << 26) ||
      n_blocks * page_size > (1 << 30))
    return Q35_EUNSUPPORTED;
  if (((uintptr_t)k_pages | (uintptr_t)v_pages) & 15) return Q35_EUNSUPPORTED;
  if (fmt == Q35_I4_G64 && (((uintptr_t)k_scale | (uintptr_t)v_scale) & 15)) return Q35_EUNSUPPORTED;
  int s = 4;
  while ((int64_t(1) << s) < page_size) ++s;
  *shift = s;
  return Q35_OK;
}

// A [B, T, H, 256] view of fp32 or bf16 whose quads of 4 values are read as one vector.
inline int view_check(const void* p, int dtype, int64_t sb, int64_t st, int64_t sh) {
  if (!p) return Q35_EINVAL;
  if (dtype != Q35_F32 && dtype != Q35_BF16) return Q35_EUNSUPPORTED;
  if (sb < 0 || st < 0 || sh < 0) return Q35_EINVAL;
  if ((sb | st | sh) & 3 || (uintptr_t)p & (dtype == Q35_F32 ? 15 : 7)) return Q35_EUNSUPPORTED;
  return Q35_OK;
}

template <typename T> __device__ __forceinline__ f32x4 load_quad(const T* p);
template <> __device__ __forceinline__ f32x4 load_quad<float>(const float* p) {
  return *reinterpret_cast<const f32x4*>(p);
}
template <> __device__ __forceinline__ f32x4 load_quad<__bf16>(const __bf16* p) {
  const u32x2 r = *reinterpret_cast<const u32x2*>(p);
  f32x4 o = {bf16lo(r.x), bf16hi(r.x), bf16lo(r.y), bf16hi(r.y)};
  return o;
}

}  // namespace q35
