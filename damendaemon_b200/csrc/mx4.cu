// Microscaled 4-bit matrices (mx4.cuh): quantisation, the values back, and the product for few rows.
#include "few_rows.cuh"

namespace {
constexpr int THREADS = 256;

// ---------------------------------------------------------------- quantisation
// Per block of 32: s - 127 = floor(log2(max |x|)) - 2, which the largest's exponent bits give (the largest element then lies
// in [4, 8)), x 2^(127 - s) is exact, and the conversion rounds to the nearest of the sixteen numbers, ties to the even
// mantissa, sizes above 6 to 6. A block with an infinity or a NaN gets s = 255. Sixteen lanes own a group, four a block, one
// eight neighbours: 32 or 16 bytes in, four bytes out, no shared memory. Bound by its bytes.
// The kernels after this one start when it has ended, not before, with its stores fenced: the products of gemm_tcgen05.cu fetch their
// weights before they wait for the kernel before them, unless they are told that it makes them (gemm_mx4 tells them).
template <typename T>
__device__ __forceinline__ void load_row8(const T* row, int k, int n, bool wide, float* x) {
    if (wide && k < n) {
        if (sizeof(T) == 4) {
            const float4 a = *reinterpret_cast<const float4*>(row + k), b = *reinterpret_cast<const float4*>(row + k + 4);
            x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
        } else {
            const uint4 v = *reinterpret_cast<const uint4*>(row + k);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[2 * i] = __uint_as_float(w[i] << 16);
                x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = k + i < n ? dd_to_f32(row[k + i]) : 0.f;
}

// (UNROLL groups of a row's neighbours, or of the next row, in flight a thread: with one 6,400 x 1,600 took twice as long)
constexpr int UNROLL = 4;

template <typename T>
__global__ void __launch_bounds__(THREADS)
quantize_kernel(const T* x, long long ldx, int width, int groups, long long n_groups, uint32_t* codes, uint32_t* scales, int wide) {
    dd_grid_wait();
    const int lane = threadIdx.x & 15, b = lane >> 2, t = lane & 3;
    const unsigned mask = 0xffffu << (threadIdx.x & 16);
    const long long first = (((long long)blockIdx.x * THREADS + threadIdx.x) >> 4) * UNROLL;
    long long row = first / groups;
    int group = (int)(first - row * groups);
    float v[UNROLL][8];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        if (first + u < n_groups) load_row8(x + row * ldx, group * mx4::GROUP + b * mx4::BLOCK + t * 8, width, wide, v[u]);
        if (++group == groups) { group = 0; ++row; }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        if (first + u >= n_groups) break;
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[u][i]) & 0x7fffffffu);
        top = max(top, __shfl_xor_sync(mask, top, 1));
        top = max(top, __shfl_xor_sync(mask, top, 2));
        const uint32_t exponent = top >> 23;
        const uint32_t s = exponent == 255 ? 255u : exponent > 2 ? exponent - 2 : 0u;
        const float by = __uint_as_float((s == 255 ? 127u : 254u - s) << 23);       // 2^(127 - s)
        uint32_t word = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {           // byte i: two elements of one parity; the second operand is the lower half
            const int e = i < 2 ? 4 * i : 4 * (i - 2) + 1;
            uint16_t byte;
            asm("{\n\t.reg .b8 q;\n\tcvt.rn.satfinite.e2m1x2.f32 q, %1, %2;\n\tcvt.u16.u8 %0, q;\n\t}"
                : "=h"(byte) : "f"(v[u][e + 2] * by), "f"(v[u][e] * by));
            word |= (uint32_t)byte << (8 * i);
        }
        codes[(first + u) * 16 + 4 * t + b] = s == 255 ? 0u : word;
        uint32_t four = s << (8 * b);
        four |= __shfl_xor_sync(mask, four, 4);
        four |= __shfl_xor_sync(mask, four, 8);
        if (lane == 0) scales[first + u] = four;
    }
    __threadfence();
}

// ---------------------------------------------------------------- the values back
// (Nor may the kernels after this one start before it has ended, as above.)
template <typename T>
__global__ void __launch_bounds__(THREADS)
values_kernel(const uint32_t* codes, const uint32_t* scales, int width, int groups, long long n_groups, T* out, int wide) {
    dd_grid_wait();
    const int lane = threadIdx.x & 15, b = lane >> 2, t = lane & 3;
    const long long first = (((long long)blockIdx.x * THREADS + threadIdx.x) >> 4) * UNROLL;
    uint32_t word[UNROLL], four[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        word[u] = first + u < n_groups ? codes[(first + u) * 16 + 4 * t + b] : 0u;
        four[u] = first + u < n_groups ? scales[first + u] : 0u;
    }
    long long row = first / groups;
    int group = (int)(first - row * groups);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const int k = group * mx4::GROUP + b * mx4::BLOCK + t * 8;
        T* to = out + row * width + k;
        if (++group == groups) { group = 0; ++row; }
        if (first + u >= n_groups || k >= width) continue;
        const uint32_t s = (four[u] >> (8 * b)) & 255u;
        const float by = __uint_as_float(s == 255 ? 0x7fc00000u : s == 0 ? 0x00400000u : s << 23);
        uint32_t pair[4];
        mx4::pairs(word[u], pair);
        __align__(16) T v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {           // the pair's element is times 2^-126
            const float e = __uint_as_float(i & 1 ? pair[i >> 1] & 0xffff0000u : pair[i >> 1] << 16) * 8.507059173023462e37f;
            v[i] = dd_from_f32<T>(e * by);
        }
        if (wide) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(v) / 16; ++i) reinterpret_cast<uint4*>(to)[i] = reinterpret_cast<const uint4*>(v)[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (k + i < width) to[i] = v[i];
        }
    }
    __threadfence();
}

// ---------------------------------------------------------------- the product, few rows
struct RowsParams {
    const uint32_t* codes;       // [N][groups][16]
    const uint32_t* scales;      // [N][groups]
    const __nv_bfloat16* X;      // [M, ldx]
    const float* bias;           // [N] or null
    const float* residual;       // [M, ldr] or null; may be out
    void* out;                   // [M, ldo]
    int M, N, K, groups, ldx, ldr, ldo, act, out_dtype, wide;
    int settled;                 // no kernel that is still running writes codes or scales
};

// Y^T = W X^T: a warp owns 16 rows of W, NT x 8 rows of X and a share of the groups; KW warps of the block share K, the other
// RW = 8 / KW have rows of their own. A block of 32 elements goes through two instructions into an accumulator of its own, which
// is added, times the block's scale, to the float32 sums: the elements need no multiplication.
template <int NT, int KW>
__global__ void __launch_bounds__(THREADS)
gemm_mx4_rows_kernel(const RowsParams p) {
    constexpr int RW = 8 / KW, U = NT == 1 ? 4 : 2;
    __shared__ float red[8][16][NT * 8 + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rw = warp / KW, kw = warp % KW;
    const int n0 = (blockIdx.x * RW + rw) * 16, m0 = blockIdx.y * NT * 8;
    const int first = p.groups * kw / KW, last = p.groups * (kw + 1) / KW;
    const size_t r0 = (size_t)min(n0 + g, p.N - 1) * p.groups, r1 = (size_t)min(n0 + g + 8, p.N - 1) * p.groups;
    const uint4* w0 = reinterpret_cast<const uint4*>(p.codes) + r0 * 4 + t;
    const uint4* w1 = reinterpret_cast<const uint4*>(p.codes) + r1 * 4 + t;
    const uint32_t* s0 = p.scales + r0;
    const uint32_t* s1 = p.scales + r1;
    uint4 c0[U], c1[U];
    uint32_t f0[U], f1[U];
    auto fetch = [&](int from) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = min(from + u, p.groups - 1);       // groups past the share are not used
            c0[u] = w0[at * 4]; c1[u] = w1[at * 4];
            f0[u] = s0[at]; f1[u] = s1[at];
        }
    };
    dd_launch_dependents();
    // A settled matrix is read while the kernel before this one ends, one that this kernel may have made behind its end, with the rows
    // (6,400 x 1,600, one row, in a graph: 4.65 us settled, 4.85 not; from memory 4.9 and 5.4. Asking L2 for the first codes before the wait instead
    // takes longer than either, 5.7).
    if (p.settled) fetch(first);
    dd_grid_wait();
    if (!p.settled) fetch(first);
    const __nv_bfloat16* x[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) x[j] = m0 + j * 8 + g < p.M ? p.X + (size_t)(m0 + j * 8 + g) * p.ldx : nullptr;
    float acc[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] = 0.f;
    for (int from = first; from < last; from += U) {
        if (from > first) fetch(from);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (from + u >= last) break;
            const int k = (from + u) * mx4::GROUP + t * 8;
            const uint32_t* a0 = reinterpret_cast<const uint32_t*>(&c0[u]);
            const uint32_t* a1 = reinterpret_cast<const uint32_t*>(&c1[u]);
            uint4 xv[NT][4];
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int b = 0; b < 4; ++b) xv[j][b] = few::load8(x[j], k + b * mx4::BLOCK, p.K, p.wide);
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                uint32_t v0[4], v1[4];
                mx4::whole_pairs(a0[b], v0);
                mx4::whole_pairs(a1[b], v1);
                const float by0 = mx4::scale(f0[u], b), by1 = mx4::scale(f1[u], b);
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    float d[4] = {0.f, 0.f, 0.f, 0.f};
                    few::block_product(v0, v1, xv[j][b], d);
                    few::add_block(by0, by1, d, acc[j]);
                }
            }
        }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[warp][g + 8 * (i >> 1)][j * 8 + 2 * t + (i & 1)] = acc[j][i];
    __syncthreads();
    for (int i = threadIdx.x; i < RW * 16 * NT * 8; i += THREADS) {
        const int row = i % (RW * 16), m = m0 + i / (RW * 16), n = blockIdx.x * RW * 16 + row;
        if (m >= p.M || n >= p.N) continue;
        float sum = 0.f;
#pragma unroll
        for (int s = 0; s < KW; ++s) sum += red[(row >> 4) * KW + s][row & 15][i / (RW * 16)];
        float v = dd_activation(sum + (p.bias ? p.bias[n] : 0.f), p.act);
        if (p.residual) v += p.residual[(size_t)m * p.ldr + n];
        if (p.out_dtype == DD_BF16) reinterpret_cast<__nv_bfloat16*>(p.out)[(size_t)m * p.ldo + n] = __float2bfloat16_rn(v);
        else reinterpret_cast<float*>(p.out)[(size_t)m * p.ldo + n] = v;
    }
}

template <int NT>
void launch_rows(const RowsParams& p, int kw, cudaStream_t s) {
    const dim3 grid(dd_ceil_div(p.N, 16 * (8 / kw)), dd_ceil_div(p.M, 8 * NT));
    if (kw == 2) dd_launch(gemm_mx4_rows_kernel<NT, 2>, grid, dim3(THREADS), 0, s, p);
    else if (kw == 4) dd_launch(gemm_mx4_rows_kernel<NT, 4>, grid, dim3(THREADS), 0, s, p);
    else dd_launch(gemm_mx4_rows_kernel<NT, 8>, grid, dim3(THREADS), 0, s, p);
}

// out[M, width] = the rows of X and zeros behind them, a thread eight neighbours: rows that are no whole 16-byte pieces, as TMA wants them.
__global__ void __launch_bounds__(THREADS)
pad_rows_kernel(const __nv_bfloat16* X, long long ldx, int K, int width, long long pieces, uint4* out) {
    dd_launch_dependents();
    dd_grid_wait();
    const int per_row = width / 8;
    for (long long i = (long long)blockIdx.x * THREADS + threadIdx.x; i < pieces; i += (long long)gridDim.x * THREADS) {
        const long long row = i / per_row;
        out[i] = few::load8(X + row * ldx, (int)(i - row * per_row) * 8, K, false);
    }
}

bool rows_of_16_bytes(const void* base, long long ld, int width, int element) {
    return !((uintptr_t)base & 15) && ld * element % 16 == 0 && width % 8 == 0;
}
}  // namespace

// x [rows, width] float32 or bfloat16 with row stride ldx; codes [rows][groups][16] words, scales [rows][groups] words of four
// bytes, groups = ceil(width / 128).
DD_API int dd_mx4_quantize(const void* x, long long ldx, long long rows, int width, void* codes, void* scales, int dtype, void* stream) {
    if (rows <= 0 || width <= 0) return 0;
    const int groups = dd_ceil_div(width, mx4::GROUP);
    const long long n = rows * groups;
    const long long blocks = (n + THREADS / 16 * UNROLL - 1) / (THREADS / 16 * UNROLL);
    if (blocks > 0x7fffffffll) return dd_fail("dd_mx4: %lld rows of %d are too many", rows, width);
    const dim3 grid((unsigned)blocks);
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == DD_F32)
        dd_launch(quantize_kernel<float>, grid, dim3(THREADS), 0, s, (const float*)x, ldx, width, groups, n, (uint32_t*)codes,
                  (uint32_t*)scales, (int)rows_of_16_bytes(x, ldx, width, 4));
    else if (dtype == DD_BF16)
        dd_launch(quantize_kernel<__nv_bfloat16>, grid, dim3(THREADS), 0, s, (const __nv_bfloat16*)x, ldx, width, groups, n,
                  (uint32_t*)codes, (uint32_t*)scales, (int)rows_of_16_bytes(x, ldx, width, 2));
    else
        return dd_fail("dd_mx4_quantize: unknown dtype %d", dtype);
    return dd_check_launch("dd_mx4_quantize");
}

// out [rows, width] contiguous, float32 or bfloat16 (exact in both).
DD_API int dd_mx4_values(const void* codes, const void* scales, long long rows, int width, void* out, int dtype, void* stream) {
    if (rows <= 0 || width <= 0) return 0;
    const int groups = dd_ceil_div(width, mx4::GROUP);
    const long long n = rows * groups;
    const long long blocks = (n + THREADS / 16 * UNROLL - 1) / (THREADS / 16 * UNROLL);
    if (blocks > 0x7fffffffll) return dd_fail("dd_mx4: %lld rows of %d are too many", rows, width);
    const dim3 grid((unsigned)blocks);
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == DD_F32)
        dd_launch(values_kernel<float>, grid, dim3(THREADS), 0, s, (const uint32_t*)codes, (const uint32_t*)scales, width, groups, n,
                  (float*)out, (int)rows_of_16_bytes(out, width, width, 4));
    else if (dtype == DD_BF16)
        dd_launch(values_kernel<__nv_bfloat16>, grid, dim3(THREADS), 0, s, (const uint32_t*)codes, (const uint32_t*)scales, width, groups, n,
                  (__nv_bfloat16*)out, (int)rows_of_16_bytes(out, width, width, 2));
    else
        return dd_fail("dd_mx4_values: unknown dtype %d", dtype);
    return dd_check_launch("dd_mx4_values");
}

// out [rows, width] bfloat16: the rows of X [rows, K] (row stride ldx), then zeros; width: K rounded up to a multiple of 8.
DD_API int dd_mx4_pad_rows(const void* X, long long ldx, long long rows, int K, int width, void* out, void* stream) {
    if (rows <= 0 || K <= 0) return 0;
    if (width % 8 || width < K || ((uintptr_t)out & 15)) return dd_fail("dd_mx4_pad_rows: rows of %d elements as rows of %d", K, width);
    const long long pieces = rows * (width / 8), blocks = (pieces + THREADS - 1) / THREADS;
    dd_launch(pad_rows_kernel, dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(THREADS), 0, (cudaStream_t)stream, (const __nv_bfloat16*)X, ldx, K,
              width, pieces, (uint4*)out);
    return dd_check_launch("dd_mx4_pad_rows");
}

// out[M, N] = act(X . W^T + bias) (+ residual), X bfloat16 [M, ldx], W the 4-bit matrix [N, K]. settled: no kernel ahead on the stream
// that may still be running writes W, whose first elements are then read before that kernel's end.
DD_API int dd_gemm_mx4_rows(const void* X, int ldx, const void* codes, const void* scales, const float* bias, const float* residual,
                            int ldr, void* out, int ldo, int M, int N, int K, int act, int out_dtype, int settled, void* stream) {
    if (M <= 0 || N <= 0) return 0;
    if (K <= 0) return dd_fail("dd_gemm_mx4_rows: K=%d", K);
    if (out_dtype != DD_BF16 && out_dtype != DD_F32) return dd_fail("dd_gemm_mx4_rows: unknown output dtype %d", out_dtype);
    if (((uintptr_t)codes & 15) || ((uintptr_t)scales & 3)) return dd_fail("dd_gemm_mx4_rows: the 4-bit matrix must be 16-byte aligned");
    if (M > 65535 * 16) return dd_fail("dd_gemm_mx4_rows: %d rows", M);
    RowsParams p;
    p.codes = (const uint32_t*)codes; p.scales = (const uint32_t*)scales; p.X = (const __nv_bfloat16*)X; p.bias = bias;
    p.residual = residual; p.out = out; p.M = M; p.N = N; p.K = K; p.groups = dd_ceil_div(K, mx4::GROUP); p.ldx = ldx; p.ldr = ldr;
    p.ldo = ldo; p.act = act; p.out_dtype = out_dtype; p.wide = rows_of_16_bytes(X, ldx, K, 2); p.settled = settled;
    const int kw = p.groups <= 4 ? 2 : p.groups <= 16 ? 4 : 8;
    cudaStream_t s = (cudaStream_t)stream;
    if (M <= 8) launch_rows<1>(p, kw, s);
    else if (M <= 16) launch_rows<2>(p, kw, s);
    else launch_rows<4>(p, kw, s);
    return dd_check_launch("dd_gemm_mx4_rows");
}
