// A whole expert layer for one to eight tokens, in two kernels:
//
//     out[t] = residual[t] + sum over the chosen experts of weight_e * W_down_e u(W_gate_e y[t], W_up_e y[t])
//              + gate[t] * shared unit of y[t] + sum over the chosen identity outputs of weight * y[t]
//
// (or, with the weights on the inputs, of W_down_e act(weight_e W_up_e y[t])). What it cannot do without is reading the chosen
// experts' matrices once; everything here is arranged so that nothing else takes time of its own.
//
// up_kernel: every cluster of blocks routes for itself (the router's rows are few and come from L2): its blocks share the router's
// columns, send their partial logits to one another, and each block then chooses the tokens' experts, a warp a token, and
// lists the distinct ones. The experts' gate and up rows are dealt out over the blocks of the whole grid, tiles of 8 + 8 rows (16 for plain
// units); a block's warps share K. The unit's value, times the token's weight, is kept as float32 or as the sum of two bfloat16
// numbers (16 bits: a hidden row rounded to one would be the layer's largest error by far).
// down_kernel: a block owns 16 output rows and walks the chosen experts one after the other as one long sum; a token that does not use
// an expert meets it with zeros. The blocks of a cluster share that sum. No atomics: a token's sums are added in a fixed order.
//
// The streams are those of few_rows.cuh: weights straight into the registers of mma.sync (float32: multiply-adds).
#include "few_rows.cuh"
#include "route_choice.cuh"
#include "tcgen05.cuh"

// The layer's tensors and options, laid out as the Python side fills it (kernels.py: _ExpertLayer).
struct DdExpertLayer {
    const void *gate_up, *gate_up_scales, *down, *down_scales;
    const void *shared_gate_up, *shared_gate_up_scales, *shared_down, *shared_down_scales;
    const void* router;          // [experts + identity (+ 1), width], or null: by table
    const int* table;            // [vocab, top]
    const float* correction;
    int kind;                    // 0 float32, 1 bfloat16, 2 bfloat16 with 4-bit matrices
    int width, inner, experts, top, vocab, identity;
    int gated, form, act;        // gated unit (form) or plain unit (act)
    int softmax, groups, keep, renormalize, weight_input;
    int shared_inner, shared_form, shared_gate, router_stride;
    float limit, alpha, shared_limit, shared_alpha, weight_scale;
};

namespace {
constexpr int THREADS = 256, WARPS = 8, MAX_TOKENS = 8, MAX_TOP = 16, MAX_UNITS = MAX_TOKENS * MAX_TOP, MAX_OUTPUTS = 256;
enum Kind { F32 = 0, BF16 = 1, MX4 = 2 };

// What up_kernel tells down_kernel.
struct Plan {
    int n_units, pad[3];
    float own[MAX_TOKENS];       // the weight of a token's own row (identity outputs)
    int expert[MAX_UNITS];       // the distinct experts, ascending
    uint32_t tokens[MAX_UNITS];  // which tokens use them
};

struct Call {
    DdExpertLayer l;
    const void* y;               // [T, ldy]
    const float* residual;       // [T, ldr] or null
    float* out;                  // [T, ldo]
    const int* ids;              // [T] (by table)
    Plan* plan;
    uint8_t* hidden;             // [units][T][row], the shared unit's rows behind them
    int* error_flag;
    int T, ldy, ldr, ldo, max_units;
    int row, shared_row;         // elements of a hidden row (two of them a token with bfloat16)
    int w_wide, inner_wide, shared_wide, y_wide, cluster;
};

struct Tile { float sum[16][few::COLUMNS + 1]; };

// A warp's share (steps from .. to - 1) of 16 rows of a matrix [.., K] by all tokens, into dst.
// row(i): the matrix row of the tile's row i. Kinds BF16 and MX4.
template <bool FOUR_BITS, int TERMS, typename Row>
__device__ __forceinline__ void tile_product(const void* w, const void* scales, int K, Row row, const __nv_bfloat16* x, const __nv_bfloat16* x2,
                                             int from, int to, bool w_wide, bool x_wide, float* acc) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const size_t r0 = row(g), r1 = row(g + 8);
    if (FOUR_BITS) {
        const size_t groups = (K + mx4::GROUP - 1) / mx4::GROUP;
        few::stream_mx4<TERMS>(reinterpret_cast<const uint4*>(w) + r0 * groups * 4 + t, reinterpret_cast<const uint4*>(w) + r1 * groups * 4 + t,
                               reinterpret_cast<const uint32_t*>(scales) + r0 * groups, reinterpret_cast<const uint32_t*>(scales) + r1 * groups,
                               x, x2, K, from, to, x_wide, acc);
    } else {
        const __nv_bfloat16* m = reinterpret_cast<const __nv_bfloat16*>(w);
        few::stream_bf16<TERMS>(m + r0 * K, m + r1 * K, x, x2, K, from, to, w_wide, x_wide, acc);
    }
}
__device__ __forceinline__ void put_tile(Tile& dst, const float* acc, float back) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int i = 0; i < 4; ++i) dst.sum[g + 8 * (i >> 1)][2 * t + (i & 1)] = acc[i] * back;
}
// float32: four rows of the tile at a time, sums across the warp, into dst.
template <int T>
__device__ __forceinline__ void put_four(Tile& dst, int r0, float (*acc)[T]) {
    float v[few::F32_ROWS * T];
#pragma unroll
    for (int r = 0; r < few::F32_ROWS; ++r)
#pragma unroll
        for (int t = 0; t < T; ++t) v[r * T + t] = acc[r][t];
    const float sum = few::warp_sums<few::F32_ROWS * T>(v);
    const int lane = threadIdx.x & 31, i = lane * (few::F32_ROWS * T) / 32;
    if (lane % (32 / (few::F32_ROWS * T)) == 0) dst.sum[r0 + i / T][i % T] = sum;
}

__device__ __forceinline__ int steps_of(int kind, int K) { return kind == BF16 ? (K + 31) / 32 : (K + 127) / 128; }

// ---------------------------------------------------------------- routing, by every cluster for itself
struct Routing {
    int chosen[MAX_TOKENS][MAX_TOP];
    float weight[MAX_TOKENS][MAX_TOP];
    float gate[MAX_TOKENS];                      // the shared unit's
    uint32_t users[MAX_OUTPUTS];                 // per output: which tokens chose it
    int count[WARPS];
    int n_units;
    int expert[MAX_UNITS];
};

// The logits of this block's share of the columns for all tokens, added over the warps that share them: part[row][token]
template <int KIND, int T>
__device__ void partial_logits(const Call& c, int rows, int from, int to, Tile* parts) {
    const int warp = threadIdx.x >> 5;
    const int tiles = (rows + 15) / 16, shares = max(1, WARPS / tiles), items = tiles * shares;
    for (int item = warp; item < items; item += WARPS) {
        const int tile = item % tiles, share = item / tiles;
        const int a = from + (to - from) * share / shares, b = from + (to - from) * (share + 1) / shares;
        auto row = [&](int i) { return (size_t)min(tile * 16 + i, rows - 1); };
        if constexpr (KIND == F32) {
            const float* m = reinterpret_cast<const float*>(c.l.router);
            for (int r0 = 0; r0 < 16; r0 += few::F32_ROWS) {
                const float* w[few::F32_ROWS];
                float acc[few::F32_ROWS][T];
#pragma unroll
                for (int r = 0; r < few::F32_ROWS; ++r) {
                    w[r] = m + row(r0 + r) * c.l.router_stride;
#pragma unroll
                    for (int t = 0; t < T; ++t) acc[r][t] = 0.f;
                }
                few::stream_f32<T>(w, reinterpret_cast<const float*>(c.y), c.ldy, (1u << c.T) - 1, c.l.width, a, b, c.w_wide, c.y_wide, acc);
                put_four<T>(parts[item], r0, acc);
            }
        } else {
            const int lane = threadIdx.x & 31, g = lane >> 2;
            const __nv_bfloat16* m = reinterpret_cast<const __nv_bfloat16*>(c.l.router);
            const __nv_bfloat16* x = g < c.T ? reinterpret_cast<const __nv_bfloat16*>(c.y) + (size_t)g * c.ldy : nullptr;
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
            few::stream_bf16<1>(m + row(g) * c.l.router_stride, m + row(g + 8) * c.l.router_stride, x, nullptr, c.l.width, a, b, c.w_wide,
                                c.y_wide, acc);
            put_tile(parts[item], acc, 1.f);
        }
    }
}

template <int KIND, int T>
__device__ void route(const Call& c, Routing& r, float* scratch) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int outputs = c.l.experts + c.l.identity;
    for (int e = threadIdx.x; e < MAX_OUTPUTS; e += THREADS) r.users[e] = 0;
    if (c.l.router) {
        const int rows = outputs + c.l.shared_gate, tiles = (rows + 15) / 16, shares = max(1, WARPS / tiles);
        const int n = tiles * 16 * MAX_TOKENS;                          // logits, a row of eight an output
        const int rank = c.cluster > 1 ? (int)tc::cluster_rank() : 0;
        Tile* parts = reinterpret_cast<Tile*>(scratch);
        float* sums = scratch + (sizeof(Tile) / 4) * tiles * shares;     // [cluster][n]: what every block of the cluster found
        const int steps = steps_of(KIND == F32 ? F32 : BF16, c.l.width);
        partial_logits<KIND, T>(c, rows, steps * rank / c.cluster, steps * (rank + 1) / c.cluster, parts);
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += THREADS) {
            const int row = i / MAX_TOKENS, t = i % MAX_TOKENS;
            float z = 0.f;
            if (t < c.T)
                for (int s = 0; s < shares; ++s) z += parts[s * tiles + row / 16].sum[row % 16][t];
            if (c.cluster == 1) sums[i] = z;
            else
                for (int to = 0; to < c.cluster; ++to) tc::st_cluster_f32(tc::map_to_rank(&sums[rank * n + i], to), z);
        }
        if (c.cluster > 1) {
            tc::cluster_arrive();
            tc::cluster_wait();
        } else __syncthreads();
        float* value = sums + c.cluster * n;                            // [T][outputs]
        float* score = value + MAX_TOKENS * outputs;
        float* worth = score + MAX_TOKENS * outputs;
        for (int i = threadIdx.x; i < rows * MAX_TOKENS; i += THREADS) {
            const int e = i / MAX_TOKENS, t = i % MAX_TOKENS;
            float z = 0.f;
            for (int s = 0; s < c.cluster; ++s) z += sums[s * n + i];
            if (e >= outputs) r.gate[t] = 1.0f / (1.0f + expf(-z));
            else if (c.l.softmax) value[t * outputs + e] = z;
            else dd_sigmoid_score(z, e, c.l.correction, c.l.groups, value + t * outputs, score + t * outputs);
        }
        if (!c.l.shared_gate && threadIdx.x < MAX_TOKENS) r.gate[threadIdx.x] = 1.f;
        __syncthreads();
        if (warp < c.T)
            dd_choose_experts(score + warp * outputs, value + warp * outputs, worth + warp * c.l.groups, outputs, c.l.top, c.l.groups, c.l.keep,
                              c.l.weight_scale, c.l.softmax, c.l.correction, c.l.renormalize, r.chosen[warp], r.weight[warp]);
    } else {
        for (int i = threadIdx.x; i < c.T * c.l.top; i += THREADS) {
            const int t = i / c.l.top, k = i % c.l.top, id = c.ids[t];
            const int e = id >= 0 && id < c.l.vocab ? c.l.table[(size_t)id * c.l.top + k] : -1;
            r.chosen[t][k] = e;
            r.weight[t][k] = c.l.weight_scale;
        }
        if (threadIdx.x < MAX_TOKENS) r.gate[threadIdx.x] = 1.f;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < c.T * c.l.top; i += THREADS) {
        const int t = i / c.l.top, e = r.chosen[t][i % c.l.top];
        if (e >= 0 && e < outputs) atomicOr(&r.users[e], 1u << t);
        else if (blockIdx.x == 0) atomicOr(c.error_flag, 1);           // an expert out of range: left out, and reported
    }
    __syncthreads();
    // the distinct experts, ascending (a thread an expert)
    const bool used = (int)threadIdx.x < c.l.experts && r.users[threadIdx.x];
    const uint32_t votes = __ballot_sync(0xffffffffu, used);
    if (lane == 0) r.count[warp] = __popc(votes);
    __syncthreads();
    int at = __popc(votes & ((1u << lane) - 1));
    for (int w = 0; w < warp; ++w) at += r.count[w];
    if (used) r.expert[at] = threadIdx.x;
    if (threadIdx.x == 0) {
        int total = 0;
        for (int w = 0; w < WARPS; ++w) total += r.count[w];
        r.n_units = total;
    }
    __syncthreads();
}
// A token's weight on an expert: its choices of it (a table may name one twice), in their order.
__device__ __forceinline__ float weight_of(const Call& c, const Routing& r, int t, int e) {
    float w = 0.f;
    for (int k = 0; k < c.l.top; ++k)
        if (r.chosen[t][k] == e) w += r.weight[t][k];
    return w;
}

template <int KIND, int T>
__global__ void __launch_bounds__(THREADS, 2)
up_kernel(const __grid_constant__ Call c) {
    extern __shared__ __align__(16) float scratch[];
    __shared__ Routing r;
    __shared__ Tile red[2][WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    dd_launch_dependents();
    if (c.cluster > 1) {                          // a block's shared memory may be written once it runs
        tc::cluster_arrive();
        tc::cluster_wait();
    }
    dd_grid_wait();
    route<KIND, T>(c, r, scratch);
    if (blockIdx.x == 0) {
        for (int u = threadIdx.x; u < r.n_units; u += THREADS) {
            c.plan->expert[u] = r.expert[u];
            c.plan->tokens[u] = r.users[r.expert[u]];
        }
        if (threadIdx.x == 0) c.plan->n_units = r.n_units;
        if (threadIdx.x < c.T) {
            float own = 0.f;
            for (int k = 0; k < c.l.top; ++k)
                if (r.chosen[threadIdx.x][k] >= c.l.experts && r.chosen[threadIdx.x][k] < c.l.experts + c.l.identity) own += r.weight[threadIdx.x][k];
            c.plan->own[threadIdx.x] = own;
        }
    }
    const int tile_rows = c.l.gated ? 8 : 16;
    const int per_unit = (c.l.inner + tile_rows - 1) / tile_rows, for_shared = (c.l.shared_inner + 7) / 8;
    const int total = r.n_units * per_unit + for_shared;
    const int steps = steps_of(KIND, c.l.width);
    int turn = 0;
    for (int task = blockIdx.x; task < total; task += gridDim.x, turn ^= 1) {
        const int unit = task < r.n_units * per_unit ? task / per_unit : -1;         // -1: the shared one
        const int tile = unit >= 0 ? task % per_unit : task - r.n_units * per_unit;
        const int inner = unit >= 0 ? c.l.inner : c.l.shared_inner;
        const bool gated = unit < 0 || c.l.gated;
        const size_t base = unit >= 0 ? (size_t)r.expert[unit] * inner * (gated ? 2 : 1) : 0;
        const int first = tile * (gated ? 8 : 16);
        // rows 0..7 are gate rows and 8..15 the same features' up rows; plain: sixteen neighbours
        auto row = [&](int i) { return gated ? base + (i < 8 ? 0 : inner) + min(first + (i & 7), inner - 1) : base + min(first + i, inner - 1); };
        const void* w = unit >= 0 ? c.l.gate_up : c.l.shared_gate_up;
        const void* scales = unit >= 0 ? c.l.gate_up_scales : c.l.shared_gate_up_scales;
        const int from = steps * warp / WARPS, to = steps * (warp + 1) / WARPS;
        Tile* parts = red[turn];
        if constexpr (KIND == F32) {
            for (int r0 = 0; r0 < 16; r0 += few::F32_ROWS) {
                const float* rows[few::F32_ROWS];
                float acc[few::F32_ROWS][T];
#pragma unroll
                for (int i = 0; i < few::F32_ROWS; ++i) {
                    rows[i] = reinterpret_cast<const float*>(w) + row(r0 + i) * c.l.width;
#pragma unroll
                    for (int t = 0; t < T; ++t) acc[i][t] = 0.f;
                }
                few::stream_f32<T>(rows, reinterpret_cast<const float*>(c.y), c.ldy, (1u << c.T) - 1, c.l.width, from, to, c.w_wide, c.y_wide, acc);
                put_four<T>(parts[warp], r0, acc);
            }
        } else {
            const int g = lane >> 2;
            const __nv_bfloat16* x = g < c.T ? reinterpret_cast<const __nv_bfloat16*>(c.y) + (size_t)g * c.ldy : nullptr;
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
            tile_product<KIND == MX4, 1>(w, scales, c.l.width, row, x, nullptr, from, to, c.w_wide, c.y_wide, acc);
            put_tile(parts[warp], acc, KIND == MX4 ? few::MX4_BACK : 1.f);
        }
        __syncthreads();          // (the other set of tiles is written next: one barrier a task is enough)
        const int rows = gated ? 8 : 16;
        for (int i = threadIdx.x; i < rows * MAX_TOKENS; i += THREADS) {
            const int t = i / rows, f = i % rows, feature = first + f;
            const int hidden_row = unit >= 0 ? c.row : c.shared_row;
            if (t >= c.T || feature >= hidden_row || (unit >= 0 && !(r.users[r.expert[unit]] >> t & 1))) continue;
            float v = 0.f;                        // (zeros between the last feature and the end of the row)
            if (feature < inner) {
                float a = 0.f, b = 0.f;
#pragma unroll
                for (int s = 0; s < WARPS; ++s) a += parts[s].sum[f][t];
                if (gated)
#pragma unroll
                    for (int s = 0; s < WARPS; ++s) b += parts[s].sum[f + 8][t];
                const float by = unit >= 0 ? weight_of(c, r, t, r.expert[unit]) : r.gate[t];
                if (unit < 0) v = by * dd_gated_value<false>(a, b, c.l.shared_form, c.l.shared_limit, c.l.shared_alpha);
                else if (gated) v = by * dd_gated_value<false>(a, b, c.l.form, c.l.limit, c.l.alpha);
                else v = c.l.weight_input ? dd_activation(by * a, c.l.act) : by * dd_activation(a, c.l.act);
            }
            const size_t slot = unit >= 0 ? (size_t)unit * c.T + t : (size_t)t;
            if constexpr (KIND == F32) {
                float* h = reinterpret_cast<float*>(c.hidden) + (unit >= 0 ? 0 : (size_t)c.max_units * c.T * c.row);
                h[slot * hidden_row + feature] = v;
            } else {
                __nv_bfloat16* h = reinterpret_cast<__nv_bfloat16*>(c.hidden) + (unit >= 0 ? 0 : (size_t)c.max_units * c.T * c.row * 2);
                const __nv_bfloat16 hi = __float2bfloat16_rn(v);
                h[slot * 2 * hidden_row + feature] = hi;
                h[(slot * 2 + 1) * hidden_row + feature] = __float2bfloat16_rn(v - __bfloat162float(hi));
            }
        }
    }
}

template <int KIND, int T>
__global__ void __launch_bounds__(THREADS, 2)
down_kernel(const __grid_constant__ Call c) {
    __shared__ Tile red[WARPS];
    __shared__ float others[7][16][MAX_TOKENS];          // the sums of the cluster's other blocks
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int cluster = c.cluster, rank = cluster > 1 ? (int)tc::cluster_rank() : 0;
    dd_launch_dependents();
    if (cluster > 1) {
        tc::cluster_arrive();
        tc::cluster_wait();
    }
    dd_grid_wait();
    const int n0 = blockIdx.x / cluster * 16;
    const int n_units = c.plan->n_units;
    const int per_unit = steps_of(KIND, c.l.inner), for_shared = c.l.shared_inner ? steps_of(KIND, c.l.shared_inner) : 0;
    const int total = n_units * per_unit + for_shared;
    const int index = rank * WARPS + warp, sharers = cluster * WARPS;
    const int from = (int)((long long)total * index / sharers), to = (int)((long long)total * (index + 1) / sharers);
    auto each_run = [&](auto run) {              // the runs of steps of one unit in this warp's share
        for (int at = from; at < to;) {
            const int unit = at < n_units * per_unit ? at / per_unit : n_units;
            const int begin = unit * per_unit, end = min(to, unit < n_units ? begin + per_unit : total);
            run(unit, at - begin, end - begin);
            at = end;
        }
    };
    if constexpr (KIND == F32) {
        for (int r0 = 0; r0 < 16; r0 += few::F32_ROWS) {
            float acc[few::F32_ROWS][T];
#pragma unroll
            for (int i = 0; i < few::F32_ROWS; ++i)
#pragma unroll
                for (int t = 0; t < T; ++t) acc[i][t] = 0.f;
            each_run([&](int unit, int a, int b) {
                const bool shared = unit == n_units;
                const int K = shared ? c.l.shared_inner : c.l.inner, ld = shared ? c.shared_row : c.row;
                const float* w = reinterpret_cast<const float*>(shared ? c.l.shared_down : c.l.down) +
                                 (shared ? 0 : (size_t)c.plan->expert[unit] * c.l.width * K);
                const float* h = reinterpret_cast<const float*>(c.hidden) + (size_t)(shared ? c.max_units : unit) * c.T * c.row;
                const float* rows[few::F32_ROWS];
#pragma unroll
                for (int i = 0; i < few::F32_ROWS; ++i) rows[i] = w + (size_t)min(n0 + r0 + i, c.l.width - 1) * K;
                few::stream_f32<T>(rows, h, ld, shared ? (1u << c.T) - 1 : c.plan->tokens[unit], K, a, b, shared ? c.shared_wide : c.inner_wide,
                                   true, acc);
            });
            put_four<T>(red[warp], r0, acc);
        }
    } else {
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        const int g = lane >> 2;
        each_run([&](int unit, int a, int b) {
            const bool shared = unit == n_units;
            const int K = shared ? c.l.shared_inner : c.l.inner, ld = shared ? c.shared_row : c.row;
            const bool live = g < c.T && (shared || (c.plan->tokens[unit] >> g & 1));
            const __nv_bfloat16* h = reinterpret_cast<const __nv_bfloat16*>(c.hidden) + (size_t)(shared ? c.max_units : unit) * c.T * c.row * 2 +
                                     (size_t)g * 2 * ld;
            const size_t base = shared ? 0 : (size_t)c.plan->expert[unit] * c.l.width;
            auto row = [&](int i) { return base + min(n0 + i, c.l.width - 1); };
            float part[4] = {0.f, 0.f, 0.f, 0.f};
            tile_product<KIND == MX4, 2>(shared ? c.l.shared_down : c.l.down, shared ? c.l.shared_down_scales : c.l.down_scales, K, row,
                                         live ? h : nullptr, live ? h + ld : nullptr, a, b, shared ? c.shared_wide : c.inner_wide, true, part);
            // (only into the tokens that use the expert: zero times a weight that is not finite would reach the others)
            const uint32_t users = shared ? 0xffu : c.plan->tokens[unit];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (users >> (2 * (lane & 3) + (i & 1)) & 1) acc[i] += part[i];
        });
        put_tile(red[warp], acc, KIND == MX4 ? few::MX4_BACK : 1.f);
    }
    __syncthreads();
    const int f = threadIdx.x % 16, t = threadIdx.x / 16;
    float sum = 0.f;
    if (t < c.T)
#pragma unroll
        for (int s = 0; s < WARPS; ++s) sum += red[s].sum[f][t];
    if (cluster > 1) {
        if (rank > 0 && t < c.T) tc::st_cluster_f32(tc::map_to_rank(&others[rank - 1][f][t], 0), sum);
        tc::cluster_arrive();
        tc::cluster_wait();
        if (rank > 0) return;
        if (t < c.T)
            for (int s = 1; s < cluster; ++s) sum += others[s - 1][f][t];
    }
    const int n = n0 + f;
    if (t >= c.T || n >= c.l.width) return;
    if (c.l.identity) {
        const size_t at = (size_t)t * c.ldy + n;
        const float y = KIND == F32 ? reinterpret_cast<const float*>(c.y)[at] : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(c.y)[at]);
        sum = fmaf(c.plan->own[t], y, sum);
    }
    c.out[(size_t)t * c.ldo + n] = sum + (c.residual ? c.residual[(size_t)t * c.ldr + n] : 0.f);
}

template <typename K>
int launch_clusters(K* kernel, int blocks, int cluster, size_t smem, cudaStream_t s, const Call& c, const char* what) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(blocks);
    config.blockDim = dim3(THREADS);
    config.dynamicSmemBytes = smem;
    config.stream = s;
    cudaLaunchAttribute attrs[2];
    attrs[0].id = cudaLaunchAttributeClusterDimension;
    attrs[0].val.clusterDim.x = cluster;
    attrs[0].val.clusterDim.y = 1;
    attrs[0].val.clusterDim.z = 1;
    attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[1].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attrs;
    config.numAttrs = dd_pdl_enabled ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&config, kernel, c);
    if (e != cudaSuccess) return dd_fail("dd_moe_tokens (%s, clusters of %d): %s", what, cluster, cudaGetErrorString(e));
    return dd_check_launch("dd_moe_tokens");
}

template <int KIND, int T>
int launch_both(Call& c, int sms, cudaStream_t s) {
    const int outputs = c.l.experts + c.l.identity, rows = outputs + c.l.shared_gate;
    // a router of up to 64 KB is read by every block for itself, a larger one shared by a cluster's blocks
    const size_t router_bytes = c.l.router ? (size_t)rows * c.l.width * (KIND == F32 ? 4 : 2) : 0;
    c.cluster = router_bytes <= (64 << 10) ? 1 : router_bytes <= (256 << 10) ? 4 : 8;
    const int tiles = (rows + 15) / 16, shares = tiles < WARPS ? WARPS / tiles : 1;
    const size_t smem = !c.l.router ? 0 : sizeof(Tile) * tiles * shares + sizeof(float) * (c.cluster * tiles * 16 * MAX_TOKENS +
                                                                                             MAX_TOKENS * (2 * outputs + c.l.groups));
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(up_kernel<KIND, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return dd_fail("dd_moe_tokens: shared memory of %d bytes refused: %s", (int)smem, cudaGetErrorString(e));
    }
    const int tile_rows = c.l.gated ? 8 : 16;
    const long long tasks = (long long)c.max_units * ((c.l.inner + tile_rows - 1) / tile_rows) + (c.l.shared_inner + 7) / 8;
    const int most = sms * 2 / c.cluster * c.cluster;
    int blocks = tasks < most ? (int)((tasks + c.cluster - 1) / c.cluster * c.cluster) : most;
    if (int e = launch_clusters(up_kernel<KIND, T>, blocks, c.cluster, smem, s, c, "up")) return e;
    const int rows16 = dd_ceil_div(c.l.width, 16);
    c.cluster = rows16 >= 2 * sms ? 1 : rows16 >= sms ? 2 : 4;
    return launch_clusters(down_kernel<KIND, T>, rows16 * c.cluster, c.cluster, 0, s, c, "down");
}

int hidden_row(int inner) { return (inner + 7) / 8 * 8; }
size_t hidden_bytes(const DdExpertLayer& l, int T, int max_units) {
    return (size_t)T * 4 * ((size_t)max_units * hidden_row(l.inner) + hidden_row(l.shared_inner));
}
int units_of(const DdExpertLayer& l, int T) { return T * l.top < l.experts ? T * l.top : l.experts; }
}  // namespace

// Bytes of scratch that a call of T tokens needs (16-byte aligned).
DD_API long long dd_moe_tokens_scratch(const DdExpertLayer* l, int T) {
    return (long long)(sizeof(Plan) + hidden_bytes(*l, T, units_of(*l, T)));
}

// y [T, ldy] (float32 or bfloat16, by the layer's kind), residual [T, ldr] float32 or null, out [T, ldo] float32 (may be
// residual), ids [T] with a table. An expert or a token id out of range sets error bit 1 and is left out.
DD_API int dd_moe_tokens(const DdExpertLayer* l, const void* y, int ldy, const float* residual, int ldr, float* out, int ldo, const int* ids,
                         int T, void* scratch, int sms, int* error_flag, void* stream) {
    if (T <= 0) return 0;
    const int outputs = l->experts + l->identity;
    if (T > MAX_TOKENS || l->top <= 0 || l->top > MAX_TOP || l->experts <= 0 || outputs + l->shared_gate > MAX_OUTPUTS || l->top > outputs)
        return dd_fail("dd_moe_tokens: %d tokens (at most %d), %d of %d experts (at most %d of %d)", T, MAX_TOKENS, l->top, outputs, MAX_TOP,
                       MAX_OUTPUTS);
    if (!l->router == !l->table || (l->table && !ids)) return dd_fail("dd_moe_tokens: a router, or a table with token ids");
    if (l->groups <= 0 || outputs % l->groups || l->keep <= 0 || l->keep > l->groups || l->width <= 0 || l->inner <= 0)
        return dd_fail("dd_moe_tokens: %d experts in %d groups of which %d stay, width %d, inner %d", outputs, l->groups, l->keep, l->width, l->inner);
    Call c;
    c.l = *l; c.y = y; c.residual = residual; c.out = out; c.ids = ids; c.error_flag = error_flag; c.T = T; c.ldy = ldy; c.ldr = ldr; c.ldo = ldo;
    c.max_units = units_of(*l, T);
    c.row = hidden_row(l->inner); c.shared_row = hidden_row(l->shared_inner);
    c.plan = (Plan*)scratch;
    c.hidden = (uint8_t*)scratch + sizeof(Plan);
    const int piece = l->kind == F32 ? 4 : 8;
    auto aligned = [](const void* p) { return !((uintptr_t)p & 15); };
    c.w_wide = l->width % piece == 0 && aligned(l->gate_up) && aligned(l->shared_gate_up) && aligned(l->router) &&
               (!l->router || l->router_stride % piece == 0);
    c.inner_wide = l->inner % piece == 0 && aligned(l->down);
    c.shared_wide = l->shared_inner % piece == 0 && aligned(l->shared_down);
    c.y_wide = l->width % piece == 0 && ldy % piece == 0 && aligned(y);
    cudaStream_t s = (cudaStream_t)stream;
    if (l->kind == BF16) return launch_both<BF16, 8>(c, sms, s);
    if (l->kind == MX4) return launch_both<MX4, 8>(c, sms, s);
    if (l->kind != F32) return dd_fail("dd_moe_tokens: unknown kind %d", l->kind);
    if (T == 1) return launch_both<F32, 1>(c, sms, s);
    if (T == 2) return launch_both<F32, 2>(c, sms, s);
    if (T <= 4) return launch_both<F32, 4>(c, sms, s);
    return launch_both<F32, 8>(c, sms, s);
}
