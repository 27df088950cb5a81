// Products of a large matrix with at most eight rows, for kernels that stream the matrix: a warp multiplies 16 rows of the
// matrix with the eight rows (columns of the instruction) on mma.sync, the weights straight from global memory into the
// instruction's registers. The order of k inside an instruction does not matter as long as both operands agree: lane
// (g, t) = (lane >> 2, lane & 3) loads 16 neighbouring bytes of matrix rows g and g + 8 and the same k of row g of X.
#pragma once
#include "common.cuh"
#include "mx4.cuh"

namespace few {
constexpr int COLUMNS = 8;

__device__ __forceinline__ void mma(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Eight bfloat16 values of a row from element k on, zeros from element n on; wide: the row is whole 16-byte pieces.
__device__ __forceinline__ uint4 load8(const __nv_bfloat16* row, int k, int n, bool wide) {
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (!row || k >= n) return v;
    if (wide) return *reinterpret_cast<const uint4*>(row + k);
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (k + i < n) w[i >> 1] |= (uint32_t)__bfloat16_as_ushort(row[k + i]) << (16 * (i & 1));
    return v;
}

// X times 2^64: the other operand's elements are times 2^-126, and the products must stay clear of float32's smallest numbers.
// |x| has to be below 2^63 (beyond it the result is not finite); sums below 2^-64 may be lost.
constexpr float MX4_BACK = 4.611686018427387904e18f;         // 2^62: what is left of both factors
__device__ __forceinline__ uint32_t lift(uint32_t pair) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(pair), "r"(0x5F805F80u));
    return r;
}
}  // namespace few
