// Warp-level pieces of the attention kernels that read a cache (decode_kernel.cuh, tree_mma_kernel.cuh, tree_umma_kernel.cuh): m16n8k16 MMAs, their
// operands from shared memory, probabilities kept to 16 bits, merging of partial results.
#pragma once
#include <math_constants.h>
#include <stdint.h>

#include "ptx.cuh"

namespace intra {

__device__ __forceinline__ void mma_m16n8k16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// Byte offset of 16-byte piece `piece` of key row `row` in a block: the piece index is xor-ed with the row so
// that eight rows' pieces of one column lie in different banks.
__device__ __forceinline__ uint32_t row_piece(int row, int piece) { return row * 256 + ((piece ^ (row & 7)) << 4); }
// Two probabilities as a bf16 pair and the pair of their rounding errors.
__device__ __forceinline__ void split_bf16(float p0, float p1, uint32_t& hi, uint32_t& lo) {
  hi = ptx::pack_bf16(p0, p1);
  lo = ptx::pack_bf16(p0 - __uint_as_float(hi << 16), p1 - __uint_as_float(hi & 0xffff0000u));
}
// Sum of the results of P's high and low parts. An infinite value row makes the high one infinite (or NaN, where
// infinities meet); the low one, a rounding error of either sign or zero times infinity, must not turn it into NaN.
__device__ __forceinline__ float join_parts(float hi, float lo) { return fabsf(hi) < CUDART_INF_F ? hi + lo : hi; }
// Factor that brings a partial result taken against maximum m to maximum m_all (0 for an empty one).
__device__ __forceinline__ float merge_weight(float m, float m_all) {
  return m == -CUDART_INF_F ? 0.f : ptx::ex2(m - m_all);
}

}  // namespace intra
