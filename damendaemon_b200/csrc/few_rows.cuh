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

namespace few {
// ---------------------------------------------------------------- a warp's share of a product, 16 rows of W by eight rows of X
// W bfloat16: steps of 32 k, two instructions each. w0, w1: rows g and g + 8 of W; x: row g of X (null: zeros); with TERMS = 2 X
// is the sum of two bfloat16 rows, x and x2 (a float32 row to 16 bits). Adds steps from .. to - 1 to acc.
template <int TERMS>
__device__ __forceinline__ void stream_bf16(const __nv_bfloat16* w0, const __nv_bfloat16* w1, const __nv_bfloat16* x, const __nv_bfloat16* x2,
                                            int K, int from, int to, bool w_wide, bool x_wide, float* acc) {
    constexpr int U = 4;
    const int t8 = (threadIdx.x & 3) * 8;
    for (; from < to; from += U) {
        uint4 a0[U], a1[U], b[U], c[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = from + u < to ? (from + u) * 32 + t8 : K;       // past the share: zeros
            a0[u] = load8(w0, k, K, w_wide);
            a1[u] = load8(w1, k, K, w_wide);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = from + u < to ? (from + u) * 32 + t8 : K;
            b[u] = load8(x, k, K, x_wide);
            if (TERMS == 2) c[u] = load8(x2, k, K, x_wide);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            mma(acc, a0[u].x, a1[u].x, a0[u].y, a1[u].y, b[u].x, b[u].y);
            mma(acc, a0[u].z, a1[u].z, a0[u].w, a1[u].w, b[u].z, b[u].w);
            if (TERMS == 2) {
                mma(acc, a0[u].x, a1[u].x, a0[u].y, a1[u].y, c[u].x, c[u].y);
                mma(acc, a0[u].z, a1[u].z, a0[u].w, a1[u].w, c[u].z, c[u].w);
            }
        }
    }
}

// W in 4 bits: steps of a group of 128 k. A block of 32 elements goes through two instructions into an accumulator of its own,
// which is added, times the block's scale, to the float32 sums: the elements need no multiplication. The sums are times
// 1 / MX4_BACK. w0, w1: a lane's 16 bytes of the first group of rows g and g + 8; s0, s1: these rows' scales.
template <int TERMS>
__device__ __forceinline__ void stream_mx4(const uint4* w0, const uint4* w1, const uint32_t* s0, const uint32_t* s1, const __nv_bfloat16* x,
                                           const __nv_bfloat16* x2, int K, int from, int to, bool x_wide, float* acc) {
    constexpr int U = 2;
    const int t8 = (threadIdx.x & 3) * 8;
    for (; from < to; from += U) {
        uint4 a0[U], a1[U];
        uint32_t f0[U], f1[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = min(from + u, to - 1);
            a0[u] = __ldg(w0 + at * 4); a1[u] = __ldg(w1 + at * 4);
            f0[u] = __ldg(s0 + at); f1[u] = __ldg(s1 + at);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (from + u >= to) break;
            uint4 b[4], c[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int k = (from + u) * mx4::GROUP + i * mx4::BLOCK + t8;
                b[i] = load8(x, k, K, x_wide);
                if (TERMS == 2) c[i] = load8(x2, k, K, x_wide);
            }
            const uint32_t* r0 = reinterpret_cast<const uint32_t*>(&a0[u]);
            const uint32_t* r1 = reinterpret_cast<const uint32_t*>(&a1[u]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t v0[4], v1[4];
                mx4::pairs(r0[i], v0);
                mx4::pairs(r1[i], v1);
                float d[4] = {0.f, 0.f, 0.f, 0.f};
                mma(d, v0[0], v1[0], v0[1], v1[1], lift(b[i].x), lift(b[i].y));
                mma(d, v0[2], v1[2], v0[3], v1[3], lift(b[i].z), lift(b[i].w));
                if (TERMS == 2) {
                    mma(d, v0[0], v1[0], v0[1], v1[1], lift(c[i].x), lift(c[i].y));
                    mma(d, v0[2], v1[2], v0[3], v1[3], lift(c[i].z), lift(c[i].w));
                }
                const float by0 = mx4::scale(f0[u], i), by1 = mx4::scale(f1[u], i);
                acc[0] = fmaf(by0, d[0], acc[0]);
                acc[1] = fmaf(by0, d[1], acc[1]);
                acc[2] = fmaf(by1, d[2], acc[2]);
                acc[3] = fmaf(by1, d[3], acc[3]);
            }
        }
    }
}

// ---------------------------------------------------------------- float32: multiply-adds, R rows of W by T rows of X
__device__ __forceinline__ float4 load4(const float* row, int k, int n, bool wide) {
    if (k >= n) return make_float4(0.f, 0.f, 0.f, 0.f);
    if (wide) return *reinterpret_cast<const float4*>(row + k);
    return make_float4(row[k], k + 1 < n ? row[k + 1] : 0.f, k + 2 < n ? row[k + 2] : 0.f, k + 3 < n ? row[k + 3] : 0.f);
}
// Steps of 128 k, four neighbours a lane; row t of X is x + t * ldx where bit t of `live` is set, the others are passed over.
constexpr int F32_ROWS = 4;
template <int T>
__device__ __forceinline__ void stream_f32(const float* const* w, const float* x, size_t ldx, uint32_t live, int K, int from, int to,
                                           bool w_wide, bool x_wide, float (*acc)[T]) {
    constexpr int U = 2;
    const int l4 = (threadIdx.x & 31) * 4;
    for (; from < to; from += U) {
        float4 a[U][F32_ROWS];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < F32_ROWS; ++r) a[u][r] = load4(w[r], from + u < to ? (from + u) * 128 + l4 : K, K, w_wide);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int t = 0; t < T; ++t) {
                if (!(live >> t & 1)) continue;
                const float4 b = load4(x + t * ldx, from + u < to ? (from + u) * 128 + l4 : K, K, x_wide);
#pragma unroll
                for (int r = 0; r < F32_ROWS; ++r) {
                    acc[r][t] = fmaf(a[u][r].x, b.x, acc[r][t]);
                    acc[r][t] = fmaf(a[u][r].y, b.y, acc[r][t]);
                    acc[r][t] = fmaf(a[u][r].z, b.z, acc[r][t]);
                    acc[r][t] = fmaf(a[u][r].w, b.w, acc[r][t]);
                }
            }
    }
}
// N values a lane -> lane l holds the warp's sum of value l * N / 32 (N a power of two, at most 32).
template <int N>
__device__ __forceinline__ float warp_sums(float* v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int n = N / 2, o = 16; o > 0; n >>= 1, o >>= 1) {
        if (n > 0) {
            const bool upper = lane & o;
#pragma unroll
            for (int j = 0; j < n; ++j) {
                const float give = upper ? v[j] : v[j + n], keep = upper ? v[j + n] : v[j];
                v[j] = keep + __shfl_xor_sync(0xffffffffu, give, o);
            }
        } else {
            v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
        }
    }
    return v[0];
}
}  // namespace few
