// Products with microscaled 4-bit matrices (mx4.cuh) for many rows, on the 5th-generation tensor cores:
//
//     out[r, n] = act(scale[r] * sum_k X[r, k] W[group(tile of r)][n, k] + bias[n]) (+ residual[r, n])
//
// X bfloat16 in row tiles, W one matrix or a stack of them of which a tile meets one; or, PAIRED, the gated unit of two such products
// (N gate rows, then N up rows a group), as gemm_grouped_tcgen05.cu does it for bfloat16 matrices.
//
// An element times its block's scale is a bfloat16 number exactly, so the weights become bfloat16 on their way to the tensor
// cores and lose nothing: computed transposed, D^T = W X^T, 128 weight rows are the lanes of the accumulator, and W is the operand
// that tcgen05.mma reads from tensor memory. A thread owns a row: it takes 128 elements (64 bytes, fetched by TMA) and their
// four scales, and stores 64 pairs into its lane's columns; eight warps do nothing else until the epilogue. Two elements cost two
// shifts, two masks and a multiplication, 2.4 operations an element with the store: 128 x 128 elements take four schedulers about
// 400 clocks, the matrix instructions that use them 4 T for a tile of T rows. The decoding of a matrix for every tile of rows is what
// these kernels cost beside a bfloat16 product; they are for rows that meet different matrices (grouped by expert) and for up to a few
// hundred rows, where it hides behind the codes' way from memory.
//
// The gated unit (PAIRED): a block has 64 features, and the lanes of the accumulator are gate rows and up rows by turns of sixteen, so that
// a gate value and its up value meet by one exchange within a warp. (As two accumulators of 128 features each, the sets of
// warps taking the gate's and the up rows: 26.7 us instead of 22.8 for 17 tiles of 16 rows of 3,200 x 1,600, 24.9 and 14.9 for 11: half
// as many blocks of twice the length.)
//
// Rings: X (64 k a stage, TMA -> MMA), codes (128 k, TMA -> the eight warps), W in tensor memory (64 k, warps -> MMA). The two sets of
// four warps take groups of 128 k in turn. Sets that take turns need stages whose phases they cannot miss, since a wait for the phase
// after one that has not ended yet passes at once: codes lie in rings whose length the sets divide, so that a stage is always one
// set's; so does W in its ring of four, and in its ring of three a set that turns to half h (of 64 k) has waited for the products of half h - 6
// already (its half before that was h - 1 or h - 3, which waited for h - 4 or h - 6), so the phase it asks for is the present one or past.
// Every wait is
// bounded, and a warp's lanes decide alike.
#include "common.cuh"
#include "mx4.cuh"
#include "tcgen05.cuh"
#include <limits.h>

namespace {
constexpr int BM = 128, XK = 64, UMMA_K = 16;
constexpr int CODE_BYTES = BM * mx4::GROUP_BYTES;

struct Mx4Params {
    const uint32_t* scales;      // [groups * rows_per_group][K groups]
    const int* tile_group;       // [row tiles] or null (group 0)
    const float* bias;           // [N] or null
    const float* residual;       // [rows, ldr] or null; may be out
    const float* row_scale;      // [rows] or null
    void* out;                   // [rows, ldo]
    int* error_flag;
    int rows, N, K, k_groups, groups, rows_per_group, ldr, ldo, out_dtype, act, form;
    float limit, alpha;
    mx4::Shifts shifts;
};

// The matrix of a tile of rows, or -1: skipped on purpose, or no such matrix (an error, and nothing is read or written).
__device__ __forceinline__ int matrix_of(const Mx4Params& p, int tile) {
    const int group = p.tile_group ? p.tile_group[tile] : 0;
    if (group < p.groups) return group;
    atomicOr(p.error_flag, 1);
    return -1;
}

// SPLIT: the blocks of a cluster share K (tiles of 64 rows that are too few for the GPU otherwise).
template <int T, bool SPLIT = false> struct Mx4Config {
    static constexpr int SETS = 2;                                   // of four warps that turn codes into rows
    static constexpr int DEQUANT_WARPS = 4 * SETS, THREADS = (DEQUANT_WARPS + 2) * 32;
    static constexpr int X_BYTES = T * XK * 2;
    static constexpr int W_BYTES = CODE_BYTES;
    static constexpr int W_STAGES = 4;                               // (a set always meets the same stages: see the rings)
    static constexpr int ACC_COLS = T;
    static constexpr int A_STAGES = T <= 32 ? 3 : 4;                 // of 32 columns (64 k)
    static constexpr int A_COLS = A_STAGES * 32;
    static constexpr int TMEM_COLS = ACC_COLS + A_COLS <= 128 ? 128 : 256;
    static constexpr int BLOCKS = TMEM_COLS == 128 ? 3 : 2;          // an SM
    static constexpr int RED_BYTES = SPLIT ? BM * T * 4 : 0;         // the cluster's partial sums of this block's columns
    static constexpr int X_FIT = ((BLOCKS == 2 ? 108 : 72) * 1024 - W_STAGES * W_BYTES - RED_BYTES) / X_BYTES;
    static constexpr int X_STAGES = X_FIT < 8 ? X_FIT : 8;
    static constexpr int BARRIERS = 2 * (X_STAGES + W_STAGES + A_STAGES) + 1;
    static constexpr int SMEM_BYTES = X_STAGES * X_BYTES + W_STAGES * W_BYTES + RED_BYTES + 1024 + BARRIERS * 8 + 16;
    static_assert(W_STAGES % SETS == 0 && ACC_COLS + A_COLS <= TMEM_COLS && SMEM_BYTES <= 227 * 1024, "tensor or shared memory");
};

__device__ __forceinline__ uint32_t mul_pair(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// gelu_new(u) = u sigmoid(2 sqrt(2 / pi) (u + 0.044715 u^3)), for results that are rounded to bfloat16.
__device__ __forceinline__ float gelu_new_fast(float u) {
    return __fdividef(u, 1.0f + __expf(-1.5957691216057308f * (u + 0.044715f * u * u * u)));
}
// The factor of a block's pairs (mx4::pairs): 2^126 * 2^(s - 127), twice in a register; above 2^127 what is missing comes later.
__device__ __forceinline__ uint32_t pair_factor(uint32_t s) {
    const uint32_t bits = s == 255 ? 0x7fc0u : (min(s, 128u) + 126u) << 7;
    return bits | (bits << 16);
}

// A wait by all lanes of a warp: they decide alike.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
    return __all_sync(0xffffffffu, tc::mbar_wait(bar, parity, abort_flag));
}

template <int A> struct Act { static constexpr int value = A; };
template <typename T> struct As { using Type = T; };

// A thread's 128 elements of a row: word 4 t + b as words[t][b]. A row is 64 bytes under the 64-byte swizzle: 16-byte piece t lies at
// t ^ (row / 2 % 4).
__device__ __forceinline__ void read_codes(const uint8_t* tile, int row, uint32_t (*words)[4]) {
    const uint4* from = reinterpret_cast<const uint4*>(tile + row * mx4::GROUP_BYTES);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const uint4 v = from[t ^ ((row >> 1) & 3)];
        words[t][0] = v.x; words[t][1] = v.y; words[t][2] = v.z; words[t][3] = v.w;
    }
}
// Half of them (64 k, two blocks) as bfloat16 pairs in the order of k, times their scales. Scales of 0 .. 127 (all blocks but those whose
// largest element passes 8) need no case of their own.
__device__ __forceinline__ void half_of(const uint32_t (*words)[4], const mx4::Shifts& shifts, uint32_t four, int half, uint32_t* r) {
    const bool easy = (four & 0x80808080u) == 0;
    uint32_t scale[2], factor[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        scale[b] = (four >> (16 * half + 8 * b)) & 255u;
        factor[b] = scale[b] * 0x00800080u + 0x3F003F00u;                    // pair_factor(scale[b])
    }
    if (!easy) {
        factor[0] = pair_factor(scale[0]);
        factor[1] = pair_factor(scale[1]);
    }
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            mx4::pairs(words[t][2 * half + b], shifts, r + b * 16 + t * 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) r[b * 16 + t * 4 + j] = mul_pair(r[b * 16 + t * 4 + j], factor[b]);
        }
    if (!easy)
#pragma unroll
        for (int b = 0; b < 2; ++b)
            if (scale[b] > 128 && scale[b] < 255) {
                const uint32_t more = ((scale[b] - 1) << 7) * 0x10001u;      // 2^(s - 128)
#pragma unroll
                for (int j = 0; j < 16; ++j) r[b * 16 + j] = mul_pair(r[b * 16 + j], more);
            }
}
// Results of feature n, rows r .. r + count - 1 (at most MOST), from their sums; what the product's epilogue has is chosen outside of the
// loop over them.
template <bool PAIRED, int MOST = 8>
__device__ __forceinline__ void finish(const Mx4Params& p, int n, float bias, int r, int count, const float* g, const float* u) {
    auto columns = [&](auto act, auto type) {
        using Out = typename decltype(type)::Type;
        Out* out = reinterpret_cast<Out*>(p.out) + (size_t)r * p.ldo + n;
        const float* residual = p.residual ? p.residual + (size_t)r * p.ldr + n : nullptr;
#pragma unroll
        for (int j = 0; j < MOST; ++j) {
            if (j >= count) break;
            float v = g[j];
            if (PAIRED) v = dd_gated_value<DdType<Out>::id == DD_BF16>(v, u[j], p.form, p.limit, p.alpha);
            else {
                if (p.row_scale) v *= p.row_scale[r + j];
                v += bias;
                if (decltype(act)::value == DD_ACT_GELU_NEW) v = gelu_new_fast(v);
                else if (decltype(act)::value != DD_ACT_NONE) v = dd_activation(v, p.act);
            }
            if (residual) v += residual[(size_t)j * p.ldr];
            out[(size_t)j * p.ldo] = dd_from_f32<Out>(v);
        }
    };
    // (the fast form is for results that are rounded to bfloat16; 'tanh' stands for every other activation)
    if (p.out_dtype == DD_BF16) {
        if (p.act == DD_ACT_NONE) columns(Act<DD_ACT_NONE>{}, As<__nv_bfloat16>{});
        else if (p.act == DD_ACT_GELU_NEW) columns(Act<DD_ACT_GELU_NEW>{}, As<__nv_bfloat16>{});
        else columns(Act<DD_ACT_TANH>{}, As<__nv_bfloat16>{});
    } else if (p.act == DD_ACT_NONE) columns(Act<DD_ACT_NONE>{}, As<float>{});
    else columns(Act<DD_ACT_TANH>{}, As<float>{});
}

// The features of a block, and where a thread finds its own: lane `quarter * 32 + lane` of the accumulator is that feature's row, or,
// PAIRED, lanes
// 0 .. 15 of a quarter are the gate rows of sixteen features and 16 .. 31 their up rows (in the stage: 64 gate rows, then 64 up rows).
template <bool PAIRED> constexpr int features = PAIRED ? BM / 2 : BM;
struct Place {
    int feature, staged;
    bool up;
    __device__ __forceinline__ Place(int quarter, int lane, bool paired) {
        up = paired && lane >= 16;
        feature = paired ? quarter * 16 + (lane & 15) : quarter * 32 + lane;
        staged = feature + (up ? BM / 2 : 0);
    }
};
__device__ __forceinline__ size_t matrix_row(const Mx4Params& p, int group, int n0, const Place& at) {
    return (size_t)group * p.rows_per_group + (at.up ? p.N : 0) + min(n0 + at.feature, p.N - 1);
}
// The results of a lane's eight columns, rows r .. r + count - 1. PAIRED: a gate lane and its up lane exchange halves, and finish four
// rows each.
template <bool PAIRED>
__device__ __forceinline__ void finish_eight(const Mx4Params& p, int n, bool live, float bias, int r, int count, const float* v) {
    if (PAIRED) {
        const bool up = threadIdx.x & 16;
        float g[4], u[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float other = __shfl_xor_sync(0xffffffffu, up ? v[j] : v[4 + j], 16);
            g[j] = up ? other : v[j];
            u[j] = up ? v[4 + j] : other;
        }
        if (live) finish<true, 4>(p, n, 0.f, up ? r + 4 : r, up ? count - 4 : count, g, u);
    } else if (live)
        finish<false>(p, n, bias, r, count, v, nullptr);
}

template <int T, bool PAIRED, bool SPLIT>
__global__ void __launch_bounds__((Mx4Config<T, SPLIT>::THREADS), (Mx4Config<T, SPLIT>::BLOCKS))
gemm_mx4_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Mx4Params p) {
    using C = Mx4Config<T, SPLIT>;
    constexpr int DEQUANT_WARPS = C::DEQUANT_WARPS, SETS = C::SETS;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* x_tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* w_tiles = x_tiles + C::X_STAGES * C::X_BYTES;
    float* partial = reinterpret_cast<float*>(w_tiles + C::W_STAGES * C::W_BYTES);      // [rank][T / splits columns][BM]
    uint64_t* x_full = reinterpret_cast<uint64_t*>(w_tiles + C::W_STAGES * C::W_BYTES + C::RED_BYTES);
    uint64_t* x_empty = x_full + C::X_STAGES;
    uint64_t* w_full = x_empty + C::X_STAGES;
    uint64_t* w_empty = w_full + C::W_STAGES;
    uint64_t* a_full = w_empty + C::W_STAGES;
    uint64_t* a_empty = a_full + C::A_STAGES;
    uint64_t* acc_bar = a_empty + C::A_STAGES;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_bar + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::X_STAGES; ++s) { tc::mbar_init(&x_full[s], 1); tc::mbar_init(&x_empty[s], 1); }
        for (int s = 0; s < C::W_STAGES; ++s) { tc::mbar_init(&w_full[s], 1); tc::mbar_init(&w_empty[s], 4); }
        for (int s = 0; s < C::A_STAGES; ++s) { tc::mbar_init(&a_full[s], 4); tc::mbar_init(&a_empty[s], 1); }
        tc::mbar_init(acc_bar, 1);
        *abort_flag = 0;
        tc::fence_barrier_init();
        tc::fence_proxy_async();
    }
    if (warp == DEQUANT_WARPS + 1) {
        tc::tmem_alloc(tmem_slot, C::TMEM_COLS);
        tc::tmem_relinquish();
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = *tmem_slot, tmem_a = tmem + C::ACC_COLS;
    dd_launch_dependents();
    if (SPLIT) tc::cluster_arrive();             // (a block's shared memory may be written once it runs; waited for before the first write)
    dd_grid_wait();              // the tile's group and the rows are earlier kernels' results

    const int splits = SPLIT ? (int)tc::cluster_size() : 1, rank = SPLIT ? (int)tc::cluster_rank() : 0;
    const int n0 = blockIdx.x / splits * features<PAIRED>, row0 = blockIdx.y * T;
    const int group = matrix_of(p, blockIdx.y);
    // this block's groups of 128 k, and its blocks of 64 (h counts from the first of them)
    const int k_first = p.k_groups * rank / splits, kgroups = p.k_groups * (rank + 1) / splits - k_first;
    const int kblocks = min(2 * kgroups, (p.K + XK - 1) / XK - 2 * k_first);
    if (group >= 0) {
        if (warp == DEQUANT_WARPS) {
            if (tc::elect_one()) {
                tc::prefetch_tensormap(&map_w);
                tc::prefetch_tensormap(&map_x);
                const int w_row = group * p.rows_per_group + n0;
                bool ok = true;
                for (int i = 0; i < kgroups && ok; ++i) {
                    const int s = i % C::W_STAGES;
                    if (!tc::mbar_wait(&w_empty[s], ((i / C::W_STAGES) & 1) ^ 1, abort_flag)) break;
                    tc::mbar_expect_tx(&w_full[s], C::W_BYTES);
                    tc::tma_load_2d(w_tiles + s * C::W_BYTES, &map_w, (k_first + i) * mx4::GROUP_BYTES, w_row, &w_full[s]);
                    if (PAIRED) tc::tma_load_2d(w_tiles + s * C::W_BYTES + CODE_BYTES / 2, &map_w, (k_first + i) * mx4::GROUP_BYTES, w_row + p.N, &w_full[s]);
                    for (int h = 2 * i; h < min(2 * i + 2, kblocks); ++h) {
                        const int x = h % C::X_STAGES;
                        if (!tc::mbar_wait(&x_empty[x], ((h / C::X_STAGES) & 1) ^ 1, abort_flag)) { ok = false; break; }
                        tc::mbar_expect_tx(&x_full[x], C::X_BYTES);
                        tc::tma_load_2d(x_tiles + x * C::X_BYTES, &map_x, (2 * k_first + h) * XK, row0, &x_full[x]);
                    }
                }
            }
        } else if (warp == DEQUANT_WARPS + 1) {
            if (tc::elect_one()) {
                constexpr uint32_t idesc = tc::idesc_bf16_f32(BM, T);
                bool ok = true;
                for (int h = 0; h < kblocks; ++h) {
                    const int x = h % C::X_STAGES, a = h % C::A_STAGES;
                    if (!tc::mbar_wait(&x_full[x], (h / C::X_STAGES) & 1, abort_flag) ||
                        !tc::mbar_wait(&a_full[a], (h / C::A_STAGES) & 1, abort_flag)) { ok = false; break; }
                    tc::fence_after_sync();
                    const uint32_t x_addr = tc::smem_u32(x_tiles + x * C::X_BYTES);
                    const uint32_t from = tmem_a + a * 32;
#pragma unroll
                    for (int k = 0; k < XK / UMMA_K; ++k) {
                        const uint64_t dx = tc::smem_desc_sw128(x_addr + k * UMMA_K * 2);
                        tc::mma_bf16_a_tmem(tmem, from + k * (UMMA_K / 2), dx, idesc, (h > 0 || k > 0) ? 1u : 0u);
                    }
                    tc::mma_commit(&x_empty[x]);
                    tc::mma_commit(&a_empty[a]);
                }
                if (ok) tc::mma_commit(acc_bar);
            }
        } else {
            // warp w may touch lanes 32 * (w % 4) .. + 31 of tensor memory; a thread owns a row of the matrix
            const int quarter = warp & 3, set = warp >> 2, row = quarter * 32 + lane;
            const uint32_t lane_part = (uint32_t)(quarter * 32) << 16;
            const Place at(quarter, lane, PAIRED);
            const uint32_t* scales = p.scales + matrix_row(p, group, n0, at) * p.k_groups + k_first;
            constexpr int STEP = SETS;
            const int first = set;
            uint32_t four = first < kgroups ? scales[first] : 0u, next = first + STEP < kgroups ? scales[first + STEP] : 0u;
            bool ok = true;
            for (int i = first; i < kgroups && ok; i += STEP) {
                const uint32_t by = four;
                four = next;
                if (i + 2 * STEP < kgroups) next = scales[i + 2 * STEP];
                const int s = i % C::W_STAGES;
                if (!warp_wait(&w_full[s], (i / C::W_STAGES) & 1, abort_flag)) break;
                uint32_t words[4][4];
                read_codes(w_tiles + s * C::W_BYTES, at.staged, words);
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&w_empty[s]);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int h = 2 * i + half, a = h % C::A_STAGES;
                    if (h >= kblocks) break;
                    uint32_t r[32];
                    half_of(words, p.shifts, by, half, r);
                    if (!warp_wait(&a_empty[a], ((h / C::A_STAGES) & 1) ^ 1, abort_flag)) { ok = false; break; }
                    tc::fence_after_sync();
                    tc::tmem_st_x32(tmem_a + lane_part + a * 32, r);
                    tc::tmem_st_wait();
                    tc::fence_before_sync();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&a_full[a]);
                }
            }
            const int n = n0 + at.feature;
            const float bias = p.bias && n < p.N ? p.bias[n] : 0.f;
            const bool live = n < p.N;
            // epilogue: the sets share the columns
            const bool done = warp_wait(acc_bar, 0, abort_flag);
            tc::fence_after_sync();
            if (SPLIT) tc::cluster_wait();       // (every thread of the block waits here or below)
            if (done)
#pragma unroll 1
                for (int c0 = set * (T / SETS); c0 < (set + 1) * (T / SETS); c0 += 8) {
                    uint32_t g[8];
                    tc::tmem_ld_x8(tmem + lane_part + c0, g);
                    tc::tmem_ld_wait();
                    if (SPLIT) {                 // to the block that finishes these columns
                        const int width = T / splits, owner = c0 / width;
                        const uint32_t to = tc::map_to_rank(&partial[(rank * width + c0 - owner * width) * BM + row], owner);
#pragma unroll
                        for (int j = 0; j < 8; ++j) tc::st_cluster_f32(to + j * BM * 4, __uint_as_float(g[j]));
                    } else
                        finish_eight<PAIRED>(p, n, live, bias, row0 + c0, p.rows - row0 - c0, reinterpret_cast<const float*>(g));
                }
            if (SPLIT) {
                tc::cluster_arrive();
                tc::cluster_wait();
                const int width = T / splits;
#pragma unroll 1
                for (int c = set; c < width; c += SETS) {
                    float sum = 0.f;
#pragma unroll 1
                    for (int s = 0; s < splits; ++s) sum += partial[(s * width + c) * BM + row];      // in rank order
                    const int r = row0 + rank * width + c;
                    if (live && r < p.rows) finish<false>(p, n, bias, r, 1, &sum, nullptr);
                }
            }
        }
    }
    // the warps without an epilogue take part in the cluster's barriers
    if (SPLIT && warp >= DEQUANT_WARPS) {
        __syncwarp();
        tc::cluster_wait();
        tc::cluster_arrive();
        tc::cluster_wait();
    }
    tc::fence_before_sync();
    __syncthreads();
    if (threadIdx.x == 0 && *abort_flag) atomicOr(p.error_flag, 8);
    if (warp == DEQUANT_WARPS + 1) {
        tc::fence_after_sync();
        tc::tmem_dealloc(tmem, C::TMEM_COLS);
    }
}

// The same for tiles of 128 rows of which there are more than SMs: a block an SM that takes tile after tile, with two accumulators, so
// that the epilogue of a tile (eight warps of its own) runs under the products of the next. 4,096 rows of sixteen experts of 2,048 x 2,048 in
// tiles of 128 rows, float32 results: 52 us, a block a tile 65. What holds it: X, which every block reads for 128 features (L2 gives
// 12 TB/s), then the instructions of decoding and epilogue.
template <int T> struct LoopConfig {
    static constexpr int SETS = 4, DEQUANT_WARPS = 16, EPILOGUE_WARPS = 8, THREADS = (DEQUANT_WARPS + EPILOGUE_WARPS + 2) * 32;
    static constexpr int X_BYTES = T * XK * 2, W_STAGES = 2 * SETS;
    static constexpr int A_STAGES = (512 - 2 * T) / 32 < 8 ? (512 - 2 * T) / 32 : 8;
    static constexpr int X_FIT = (210 * 1024 - W_STAGES * CODE_BYTES) / X_BYTES, X_STAGES = X_FIT < 8 ? X_FIT : 8;
    static constexpr int BARRIERS = 2 * (X_STAGES + W_STAGES + A_STAGES + 2);
    static constexpr int SMEM_BYTES = X_STAGES * X_BYTES + W_STAGES * CODE_BYTES + 1024 + BARRIERS * 8 + 16;
    static_assert(W_STAGES % SETS == 0 && A_STAGES % (2 * SETS) == 0 && 2 * T + A_STAGES * 32 <= 512 && SMEM_BYTES <= 227 * 1024, "tensor or shared memory");
};

template <int T, bool PAIRED>
__global__ void __launch_bounds__(LoopConfig<T>::THREADS, 1)
gemm_mx4_loop_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Mx4Params p) {
    using C = LoopConfig<T>;
    constexpr int TMA_WARP = C::DEQUANT_WARPS, MMA_WARP = TMA_WARP + 1;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* x_tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* w_tiles = x_tiles + C::X_STAGES * C::X_BYTES;
    uint64_t* x_full = reinterpret_cast<uint64_t*>(w_tiles + C::W_STAGES * CODE_BYTES);
    uint64_t* x_empty = x_full + C::X_STAGES;
    uint64_t* w_full = x_empty + C::X_STAGES;
    uint64_t* w_empty = w_full + C::W_STAGES;
    uint64_t* a_full = w_empty + C::W_STAGES;
    uint64_t* a_empty = a_full + C::A_STAGES;
    uint64_t* acc_full = a_empty + C::A_STAGES;
    uint64_t* acc_empty = acc_full + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::X_STAGES; ++s) { tc::mbar_init(&x_full[s], 1); tc::mbar_init(&x_empty[s], 1); }
        for (int s = 0; s < C::W_STAGES; ++s) { tc::mbar_init(&w_full[s], 1); tc::mbar_init(&w_empty[s], 4); }
        for (int s = 0; s < C::A_STAGES; ++s) { tc::mbar_init(&a_full[s], 4); tc::mbar_init(&a_empty[s], 1); }
        for (int s = 0; s < 2; ++s) { tc::mbar_init(&acc_full[s], 1); tc::mbar_init(&acc_empty[s], C::EPILOGUE_WARPS); }
        *abort_flag = 0;
        tc::fence_barrier_init();
        tc::fence_proxy_async();
        tc::prefetch_tensormap(&map_w);
        tc::prefetch_tensormap(&map_x);
    }
    if (warp == MMA_WARP) {
        tc::tmem_alloc(tmem_slot, 512);
        tc::tmem_relinquish();
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = *tmem_slot, tmem_a = tmem + 2 * T;
    dd_launch_dependents();
    dd_grid_wait();              // the tiles' groups and the rows are earlier kernels' results

    constexpr int FEATURES = features<PAIRED>;
    const int n_tiles = (p.N + FEATURES - 1) / FEATURES, total = n_tiles * ((p.rows + T - 1) / T);
    // (both halves of the last group, also where K ends in the first: a set then always meets the same stages; zeros by zeros)
    const int kgroups = p.k_groups, kblocks = 2 * kgroups;
    // Every role walks the same tiles; the number of a stage counts on over them. w: groups of 128 k, h: blocks of 64, n: tiles.
    auto group_of = [&](int tile) { return matrix_of(p, tile / n_tiles); };
    if (warp == TMA_WARP) {
        if (tc::elect_one()) {
            int w = 0, h = 0;
            bool ok = true;
            for (int tile = blockIdx.x; tile < total && ok; tile += gridDim.x) {
                const int group = group_of(tile), n0 = tile % n_tiles * FEATURES, row0 = tile / n_tiles * T, w_row = group * p.rows_per_group + n0;
                if (group < 0) continue;
                for (int i = 0; i < kgroups && ok; ++i, ++w) {
                    const int s = w % C::W_STAGES;
                    if (!tc::mbar_wait(&w_empty[s], ((w / C::W_STAGES) & 1) ^ 1, abort_flag)) { ok = false; break; }
                    tc::mbar_expect_tx(&w_full[s], CODE_BYTES);
                    tc::tma_load_2d(w_tiles + s * CODE_BYTES, &map_w, i * mx4::GROUP_BYTES, w_row, &w_full[s]);
                    if (PAIRED) tc::tma_load_2d(w_tiles + s * CODE_BYTES + CODE_BYTES / 2, &map_w, i * mx4::GROUP_BYTES, w_row + p.N, &w_full[s]);
                    for (int half = 2 * i; half < 2 * i + 2; ++half, ++h) {
                        const int x = h % C::X_STAGES;
                        if (!tc::mbar_wait(&x_empty[x], ((h / C::X_STAGES) & 1) ^ 1, abort_flag)) { ok = false; break; }
                        tc::mbar_expect_tx(&x_full[x], C::X_BYTES);
                        tc::tma_load_2d(x_tiles + x * C::X_BYTES, &map_x, half * XK, row0, &x_full[x]);
                    }
                }
            }
        }
    } else if (warp == MMA_WARP) {
        if (tc::elect_one()) {
            constexpr uint32_t idesc = tc::idesc_bf16_f32(BM, T);
            int h = 0, n = 0;
            bool ok = true;
            for (int tile = blockIdx.x; tile < total && ok; tile += gridDim.x) {
                if (group_of(tile) < 0) continue;
                const uint32_t acc = tmem + (n & 1) * T;
                if (!tc::mbar_wait(&acc_empty[n & 1], ((n >> 1) & 1) ^ 1, abort_flag)) break;
                tc::fence_after_sync();
                for (int i = 0; i < kblocks; ++i, ++h) {
                    const int x = h % C::X_STAGES, a = h % C::A_STAGES;
                    if (!tc::mbar_wait(&x_full[x], (h / C::X_STAGES) & 1, abort_flag) ||
                        !tc::mbar_wait(&a_full[a], (h / C::A_STAGES) & 1, abort_flag)) { ok = false; break; }
                    tc::fence_after_sync();
                    const uint32_t x_addr = tc::smem_u32(x_tiles + x * C::X_BYTES);
#pragma unroll
                    for (int k = 0; k < XK / UMMA_K; ++k)
                        tc::mma_bf16_a_tmem(acc, tmem_a + a * 32 + k * (UMMA_K / 2), tc::smem_desc_sw128(x_addr + k * UMMA_K * 2), idesc,
                                            (i > 0 || k > 0) ? 1u : 0u);
                    tc::mma_commit(&x_empty[x]);
                    tc::mma_commit(&a_empty[a]);
                }
                if (ok) tc::mma_commit(&acc_full[n & 1]);
                ++n;
            }
        }
    } else if (warp < C::DEQUANT_WARPS) {
        const int quarter = warp & 3, set = warp >> 2;
        const uint32_t lane_part = (uint32_t)(quarter * 32) << 16;
        const Place at(quarter, lane, PAIRED);
        int w0 = 0, h0 = 0;                      // of the tile's first group and block
        bool ok = true;
        for (int tile = blockIdx.x; tile < total && ok; tile += gridDim.x) {
            const int group = group_of(tile), n0 = tile % n_tiles * FEATURES;
            if (group < 0) continue;
            const uint32_t* scales = p.scales + matrix_row(p, group, n0, at) * kgroups;
            const int first = (set - w0 % C::SETS + C::SETS) % C::SETS;
            uint32_t four = first < kgroups ? scales[first] : 0u;
            for (int i = first; i < kgroups && ok; i += C::SETS) {
                const uint32_t by = four;
                if (i + C::SETS < kgroups) four = scales[i + C::SETS];
                const int w = w0 + i, s = w % C::W_STAGES;
                if (!warp_wait(&w_full[s], (w / C::W_STAGES) & 1, abort_flag)) { ok = false; break; }
                uint32_t words[4][4];
                read_codes(w_tiles + s * CODE_BYTES, at.staged, words);
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&w_empty[s]);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int h = h0 + 2 * i + half, a = h % C::A_STAGES;
                    uint32_t r[32];
                    half_of(words, p.shifts, by, half, r);
                    if (!warp_wait(&a_empty[a], ((h / C::A_STAGES) & 1) ^ 1, abort_flag)) { ok = false; break; }
                    tc::fence_after_sync();
                    tc::tmem_st_x32(tmem_a + lane_part + a * 32, r);
                    tc::tmem_st_wait();
                    tc::fence_before_sync();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&a_full[a]);
                }
            }
            w0 += kgroups;
            h0 += kblocks;
        }
    } else {
        const int quarter = warp & 3;
        const uint32_t lane_part = (uint32_t)(quarter * 32) << 16;
        const Place at(quarter, lane, PAIRED);
        int number = 0;
        for (int tile = blockIdx.x; tile < total; tile += gridDim.x) {
            if (group_of(tile) < 0) continue;
            const int n = tile % n_tiles * FEATURES + at.feature, row0 = tile / n_tiles * T;
            const float bias = p.bias && n < p.N ? p.bias[n] : 0.f;
            if (!warp_wait(&acc_full[number & 1], (number >> 1) & 1, abort_flag)) break;
            tc::fence_after_sync();
            // two warps a quarter of the lanes, half of the columns each
            const int half = (warp - MMA_WARP - 1) >> 2, count = min(T, p.rows - row0);
#pragma unroll 1
            for (int c0 = half * (T / 2); c0 < min(count, (half + 1) * (T / 2)); c0 += 16) {
                uint32_t g[16];
                tc::tmem_ld_x16(tmem + (number & 1) * T + lane_part + c0, g);
                tc::tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 16; j += 8)
                    if (c0 + j < count) finish_eight<PAIRED>(p, n, n < p.N, bias, row0 + c0 + j, count - c0 - j, reinterpret_cast<const float*>(g + j));
                __syncwarp();
            }
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&acc_empty[number & 1]);
            ++number;
        }
    }
    tc::fence_before_sync();
    __syncthreads();
    if (threadIdx.x == 0 && *abort_flag) atomicOr(p.error_flag, 8);
    if (warp == MMA_WARP) {
        tc::fence_after_sync();
        tc::tmem_dealloc(tmem, 512);
    }
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int mx4_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, long long rows, long long width, long long row_bytes, int box_width,
            int box_rows, CUtensorMapSwizzle swizzle, const char* what) {
    static EncodeTiled enc = nullptr;
    if (!enc) {
        void* sym = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            enc = reinterpret_cast<EncodeTiled>(sym);
    }
    if (!enc) return dd_fail("dd_gemm_mx4: cuTensorMapEncodeTiled is not available from this driver");
    cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)row_bytes};
    cuuint32_t box[2] = {(cuuint32_t)box_width, (cuuint32_t)box_rows};
    cuuint32_t elem[2] = {1, 1};
    CUresult r = enc(map, type, 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return dd_fail("dd_gemm_mx4: cannot describe %s to TMA (driver error %d)", what, (int)r);
    return 0;
}

template <int T, bool PAIRED, bool SPLIT = false>
int launch_mx4(const CUtensorMap& mw, const CUtensorMap& mx, const Mx4Params& p, int sms, cudaStream_t s, int splits = 1) {
    using C = Mx4Config<T, SPLIT>;
    // Three blocks an SM only where two would come in turns (275 blocks: 13.9 us, 18.7 where some SMs took three of them at once; 425: 22.4 and
    // 19.7): more shared memory keeps the third out.
    const long long blocks = (long long)dd_ceil_div(p.N, features<PAIRED>) * splits * dd_ceil_div(p.rows, T);
    constexpr int TWO_FIT = 80 * 1024, MOST = C::BLOCKS == 3 && TWO_FIT > C::SMEM_BYTES ? TWO_FIT : C::SMEM_BYTES;
    const int bytes = C::BLOCKS == 3 && blocks <= 2 * sms ? TWO_FIT : C::SMEM_BYTES;
    cudaError_t e = dd_allow_shared<gemm_mx4_kernel<T, PAIRED, SPLIT>>(MOST);
    if (e != cudaSuccess) return dd_fail("dd_gemm_mx4: shared memory of %d bytes refused: %s", MOST, cudaGetErrorString(e));
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(dd_ceil_div(p.N, features<PAIRED>) * splits, dd_ceil_div(p.rows, T));
    config.blockDim = dim3(C::THREADS);
    config.dynamicSmemBytes = bytes;
    config.stream = s;
    cudaLaunchAttribute attrs[2];
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = dd_pdl_enabled ? 1 : 0;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = splits;
    attrs[1].val.clusterDim.y = 1;
    attrs[1].val.clusterDim.z = 1;
    config.attrs = attrs;
    config.numAttrs = SPLIT ? 2 : 1;
    e = cudaLaunchKernelEx(&config, gemm_mx4_kernel<T, PAIRED, SPLIT>, mw, mx, p);
    if (e != cudaSuccess) return dd_fail("dd_gemm_mx4 (clusters of %d): %s", splits, cudaGetErrorString(e));
    return dd_check_launch("dd_gemm_mx4");
}
template <int T, bool PAIRED>
int launch_loop(const CUtensorMap& mw, const CUtensorMap& mx, const Mx4Params& p, int sms, cudaStream_t s) {
    using C = LoopConfig<T>;
    const cudaError_t e = dd_allow_shared<gemm_mx4_loop_kernel<T, PAIRED>>(C::SMEM_BYTES);
    if (e != cudaSuccess) return dd_fail("dd_gemm_mx4: shared memory of %d bytes refused: %s", C::SMEM_BYTES, cudaGetErrorString(e));
    const int tiles = dd_ceil_div(p.N, features<PAIRED>) * dd_ceil_div(p.rows, T);
    dd_launch(gemm_mx4_loop_kernel<T, PAIRED>, dim3(tiles < sms ? tiles : sms), dim3(C::THREADS), (size_t)C::SMEM_BYTES, s, mw, mx, p);
    return dd_check_launch("dd_gemm_mx4");
}
}  // namespace

// X [rows, K] bf16 (row stride ldx) in tiles of `tile` rows (16, 32, 64, 128); codes, scales: `groups` 4-bit matrices of rows_per_group
// rows of K; tile_group: device array [rows / tile] (a negative group's tile is skipped, so is one out of range, with error bit 1), or
// null: one matrix for
// all rows, of which the last tile may hold fewer. dual == 0: rows_per_group == N, act(row_scale * sum + bias) + residual; dual != 0:
// rows_per_group == 2 N, the gated unit. out: [rows, N] bf16 or f32, row stride ldo.
DD_API int dd_gemm_mx4(const void* X, int ldx, const void* codes, const void* scales, int groups, int rows_per_group, const int* tile_group,
                       const float* bias, const float* residual, int ldr, const float* row_scale, void* out, int ldo, int rows, int N, int K,
                       int tile, int dual, float limit, float alpha, int form, int act, int out_dtype, int sms, int* error_flag, void* stream) {
    if (rows <= 0 || N <= 0) return 0;
    if (K <= 0 || K % 8 || ldx % 8) return dd_fail("dd_gemm_mx4: K=%d and the row stride %d must be multiples of 8 (TMA needs 16-byte rows)", K, ldx);
    if (((uintptr_t)X & 15) || ((uintptr_t)codes & 15) || ((uintptr_t)scales & 3)) return dd_fail("dd_gemm_mx4: operands must be 16-byte aligned");
    if (out_dtype != DD_BF16 && out_dtype != DD_F32) return dd_fail("dd_gemm_mx4: unknown output dtype %d", out_dtype);
    if (tile <= 0 || (tile_group && rows % tile) || dd_ceil_div(rows, tile) > 65535) return dd_fail("dd_gemm_mx4: %d rows in tiles of %d", rows, tile);
    if (groups <= 0 || (groups > 1 && !tile_group) || rows_per_group != (dual ? 2 * N : N))
        return dd_fail("dd_gemm_mx4: %d groups of %d rows do not fit N=%d", groups, rows_per_group, N);
    if ((long long)groups * rows_per_group > INT_MAX) return dd_fail("dd_gemm_mx4: %d groups of %d rows pass 32 bits", groups, rows_per_group);
    Mx4Params p;
    p.scales = (const uint32_t*)scales; p.tile_group = tile_group; p.bias = bias; p.residual = residual; p.row_scale = row_scale; p.out = out;
    p.error_flag = error_flag; p.rows = rows; p.N = N; p.K = K; p.k_groups = dd_ceil_div(K, mx4::GROUP); p.groups = groups; p.rows_per_group = rows_per_group;
    p.ldr = ldr; p.ldo = ldo; p.out_dtype = out_dtype; p.act = act; p.form = form; p.limit = limit; p.alpha = alpha; p.shifts = mx4::SHIFTS;
    const long long row_bytes = (long long)p.k_groups * mx4::GROUP_BYTES;
    CUtensorMap mw, mx;
    if (int e = mx4_map(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, (long long)groups * rows_per_group, row_bytes, row_bytes, mx4::GROUP_BYTES, dual ? BM / 2 : BM,
                        CU_TENSOR_MAP_SWIZZLE_64B, "the codes")) return e;
    if (int e = mx4_map(&mx, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, X, rows, K, (long long)ldx * 2, XK, tile, CU_TENSOR_MAP_SWIZZLE_128B, "the rows"))
        return e;
    cudaStream_t s = (cudaStream_t)stream;
    // Tiles of 64 rows that would leave most of the GPU idle share K among two, four or eight blocks, as long as each keeps two groups
    // and all fit at once (two an SM).
    int splits = 1;
    const int tiles = dd_ceil_div(N, dual ? BM / 2 : BM) * dd_ceil_div(rows, tile);
    while (tile == 64 && !dual && !tile_group && splits < 8 && tiles * splits * 2 <= 296 && p.k_groups >= splits * 4) splits *= 2;
    if (splits > 1) return launch_mx4<64, false, true>(mw, mx, p, sms, s, splits);
    if (tile == 128 && tiles > sms) return dual ? launch_loop<128, true>(mw, mx, p, sms, s) : launch_loop<128, false>(mw, mx, p, sms, s);      // more tiles than SMs
#define DD_MX4(T) \
    case T: return dual ? launch_mx4<T, true>(mw, mx, p, sms, s) : launch_mx4<T, false>(mw, mx, p, sms, s);
    switch (tile) {
        DD_MX4(16)
        DD_MX4(32)
        DD_MX4(64)
        DD_MX4(128)
    }
#undef DD_MX4
    return dd_fail("dd_gemm_mx4: tile %d is not one of 16, 32, 64, 128", tile);
}
