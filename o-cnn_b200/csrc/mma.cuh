// Small products on the warp's matrix instruction (m16n8k16, 16-bit operands, fp32 sums), for kernels that are bound by what
// they read: operands by ldmatrix from rows in shared memory.
#pragma once

#include "common.cuh"

namespace ocnn {
namespace {

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
// This lane's row for ldmatrix4 of 16 rows x 16 channels as a B operand whose n is the row (products over channels): words 0, 1
// are rows 0-7, words 2, 3 rows 8-15.  Channel 16 k is 32 k bytes on.
__device__ __forceinline__ uint32_t rows_frag(uint32_t base, int pitch) {
  const int lane = threadIdx.x & 31;
  return base + ((lane & 7) + ((lane >> 4) & 1) * 8) * pitch + ((lane >> 3) & 1) * 16;
}
// For ldmatrix4t, as a B operand whose n is the channel (products over the 16 rows): words 0, 1 are channels 0-7, words 2, 3
// channels 8-15.
__device__ __forceinline__ uint32_t columns_frag(uint32_t base, int pitch) {
  const int lane = threadIdx.x & 31;
  return base + ((lane & 7) + ((lane >> 3) & 1) * 8) * pitch + ((lane >> 4) & 1) * 16;
}

template <bool HALF>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (HALF)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

}  // namespace
}  // namespace ocnn
