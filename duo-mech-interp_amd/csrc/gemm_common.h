// What the int8-weight GEMMs share (gemm_q8.hip, gemm_i8.hip): epilogue codes, neuron pushes and the activation capture of the
// SwiGLU epilogues, copies from global memory to LDS.
#pragma once
#include "q35_common.h"
#include "q35hip.h"

namespace q35 {

enum GemmEpi : int { kGemmStore = 0, kGemmAccumulate = 1, kGemmSwiglu = 2, kGemmSwigluSplit = 3 };

// Whether any of the push records can touch neurons nlo .. nhi - 1 (a record for every neuron, or for one in the
// range): a block whose neurons no record touches skips the per-output push loop (the model passes a fixed number of
// records, unused ones matching no neuron). Uniform: the records are read with scalar loads.
__device__ __forceinline__ bool gemm_pushes_touch(const q35_push* ps, int npush, int nlo, int nhi) {
  bool any = false;
  for (int p0 = 0; p0 < npush; p0 += 8) {  // eight records' loads in flight
    int pn[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) pn[i] = ps[min(p0 + i, npush - 1)].neuron;
#pragma unroll
    for (int i = 0; i < 8; ++i) any |= pn[i] < 0 || (pn[i] >= nlo && pn[i] < nhi);
  }
  return any;
}
// the batch row of token row m (rows of T tokens each), min(m / T, 3), without a division
__device__ __forceinline__ int gemm_push_row(int m, int T) {
  return (int)(m >= T) + (int)((int64_t)m >= 2 * (int64_t)T) + (int)((int64_t)m >= 3 * (int64_t)T);
}

// SwiGLU activation capture (p may be NULL): the activation of neuron n of global row m goes to
// p[(m / T) ldcr + (m % T) ldc + n], fp32, whatever the layout of y
struct GemmCap {
  float* p;
  int64_t ldc, ldcr;
};
__device__ __forceinline__ void gemm_capture(const GemmCap& c, int m, int T, int n, float a) {
  if (c.p) c.p[(int64_t)(m / T) * c.ldcr + (int64_t)(m % T) * c.ldc + n] = a;
}

__device__ __forceinline__ float gemm_push(const q35_push* ps, int n, int row, float a) {
  const int pn = ps->neuron;
  if (pn != n && pn >= 0) return a;
  const float v = ps->vals[row];
  return ps->mode ? a * v : a + v;
}

__device__ __forceinline__ uint32_t gemm_lds_u32(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}
// 16 bytes per lane from global memory to LDS (lane i's bytes land at M0 + 16 i), from a uniform 64-bit base (moved
// to scalar registers) and a 32-bit per-lane byte offset; no registers hold the data. Inline asm, so that the
// compiler neither moves LDS accesses across it nor waits for it: completion is awaited with explicit vmcnt counts,
// and the K loop issues no other vector memory load.
__device__ __forceinline__ void gemm_dma16s(const void* sbase, uint32_t voff, uint32_t lds_dst) {
  const uint64_t a = reinterpret_cast<uint64_t>(sbase);
  const uint64_t u = ((uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(a >> 32)) << 32) |
                     (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)a);
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds_dst), "v"(voff),
               "s"(reinterpret_cast<const void*>(u))
               : "memory", "m0");
}
template <int N> __device__ __forceinline__ void gemm_wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

}  // namespace q35
