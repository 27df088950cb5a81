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

__device__ __forceinline__ void mma_f16(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Eight bfloat16 values of a row from element k on, zeros from element n on; wide: the row is whole 16-byte pieces. (The element by
// element form is a call: inlined, it would lie between the instructions of every user.)
static __device__ __noinline__ uint4 load8_slow(const __nv_bfloat16* row, int k, int n) {
    uint32_t e[8], w[4];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = k + i < n ? __bfloat16_as_ushort(row[k + i]) : 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = e[2 * i] | e[2 * i + 1] << 16;
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 load8(const __nv_bfloat16* row, int k, int n, bool wide) {
    if (!row || k >= n) return make_uint4(0u, 0u, 0u, 0u);
    if (!wide) return load8_slow(row, k, n);
    return *reinterpret_cast<const uint4*>(row + k);
}

// ---------------------------------------------------------------- a warp's share of a product, 16 rows of W by eight rows of X
// W bfloat16: steps of 32 k, two instructions each, AHEAD steps requested at a time. w0, w1: rows g and g + 8 of W; x: row g of X
// (whole 16-byte pieces). `have` holds what Ahead::load fetched of the first steps, before X was there. (For matrices of a few rows, which
// come from L2; the large ones go through rings.)
struct Ahead {
    static constexpr int STEPS = 6;
    uint4 a0[STEPS], a1[STEPS];
    __device__ __forceinline__ void load(const __nv_bfloat16* w0, const __nv_bfloat16* w1, int K, int from, int to, bool wide) {
        const int t8 = (threadIdx.x & 3) * 8;
#pragma unroll
        for (int u = 0; u < STEPS; ++u) {
            const int k = from + u < to ? (from + u) * 32 + t8 : K;       // past the share: zeros
            a0[u] = load8(w0, k, K, wide);
            a1[u] = load8(w1, k, K, wide);
        }
    }
};
__device__ __forceinline__ void stream_bf16(const __nv_bfloat16* w0, const __nv_bfloat16* w1, const __nv_bfloat16* x, int K, int from, int to,
                                            bool w_wide, Ahead& have, float* acc) {
    const int t8 = (threadIdx.x & 3) * 8;
    while (from < to) {
        uint4 b[Ahead::STEPS];
#pragma unroll
        for (int u = 0; u < Ahead::STEPS; ++u) b[u] = load8(x, from + u < to ? (from + u) * 32 + t8 : K, K, true);
#pragma unroll
        for (int u = 0; u < Ahead::STEPS; ++u) {
            mma(acc, have.a0[u].x, have.a1[u].x, have.a0[u].y, have.a1[u].y, b[u].x, b[u].y);
            mma(acc, have.a0[u].z, have.a1[u].z, have.a0[u].w, have.a1[u].w, b[u].z, b[u].w);
        }
        from += Ahead::STEPS;
        if (from < to) have.load(w0, w1, K, from, to, w_wide);
    }
}

// A block of 32 elements of rows g and g + 8 of a 4-bit W (a lane's word of each) by its eight elements of X, into an accumulator
// of its own; add_block adds that, times the block's scales, to the float32 sums: the elements need no scale of their own.
__device__ __forceinline__ void block_product(const uint32_t* v0, const uint32_t* v1, uint4 x, float* d) {
    mma(d, v0[0], v1[0], v0[1], v1[1], x.x, x.y);
    mma(d, v0[2], v1[2], v0[3], v1[3], x.z, x.w);
}
__device__ __forceinline__ void add_block(float by0, float by1, const float* d, float* acc) {
    acc[0] = fmaf(by0, d[0], acc[0]);
    acc[1] = fmaf(by0, d[1], acc[1]);
    acc[2] = fmaf(by1, d[2], acc[2]);
    acc[3] = fmaf(by1, d[3], acc[3]);
}

// ---------------------------------------------------------------- float32: multiply-adds, R rows of W by T rows of X
// Two multiply-adds in one instruction: a sum of even and one of odd k.
__device__ __forceinline__ void fma_pair(unsigned long long& acc, float ax, float ay, float bx, float by) {
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %2};\n\tmov.b64 b, {%3, %4};\n\tfma.rn.f32x2 %0, a, b, %0;\n\t}"
        : "+l"(acc) : "f"(ax), "f"(ay), "f"(bx), "f"(by));
}
__device__ __forceinline__ float pair_sum(unsigned long long acc) {
    float x, y;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(acc));
    return x + y;
}
static __device__ __noinline__ float4 load4_slow(const float* row, int k, int n) {
    return make_float4(row[k], k + 1 < n ? row[k + 1] : 0.f, k + 2 < n ? row[k + 2] : 0.f, k + 3 < n ? row[k + 3] : 0.f);
}
__device__ __forceinline__ float4 load4(const float* row, int k, int n, bool wide) {
    if (k >= n) return make_float4(0.f, 0.f, 0.f, 0.f);
    if (!wide) return load4_slow(row, k, n);
    return *reinterpret_cast<const float4*>(row + k);
}
// Steps of 128 k, four neighbours a lane; row t of X is x + t * ldx where bit t of `live` is set, the others are passed over.
constexpr int F32_ROWS = 4;
template <int T>
__device__ __forceinline__ void stream_f32(const float* const* w, const float* x, size_t ldx, uint32_t live, int K, int from, int to,
                                           bool w_wide, bool x_wide, unsigned long long (*acc)[T]) {
    constexpr int U = 1;
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
                    fma_pair(acc[r][t], a[u][r].x, a[u][r].y, b.x, b.y);
                    fma_pair(acc[r][t], a[u][r].z, a[u][r].w, b.z, b.w);
                }
            }
    }
}
// ---------------------------------------------------------------- shared memory by address
__device__ __forceinline__ uint4 lds16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void sts16(uint32_t at, uint4 v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
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
