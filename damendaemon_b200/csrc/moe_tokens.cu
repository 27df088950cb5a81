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
// units). The unit's value, times the token's weight, is kept as float32 or as the sum of three bfloat16 numbers (24 bits, a float32's:
// a hidden row rounded to one would be the layer's largest error by far, and two leave 2e-6 where float32 leaves 2e-7).
// down_kernel: a block owns 16 output rows (float32: 4) and walks the chosen experts one after the other as one long sum, which its
// warps share; a token that does not use an expert is passed over. No atomics: a token's sums are added in a fixed order.
//
// A token's bits do not depend on what is beside it, nor on how many tokens are: a row of a matrix is cut into parts by the layer alone
// (DdExpertLayer: up_shift, unit_part, shared_part), a part is one sum from its first product to its last, and the parts' sums are
// added in one order, whichever warps had them. How many parts a warp of down_kernel takes is free to follow the step's work.
//
// Weights go to mma.sync (float32: to multiply-adds) through a ring of TMA boxes that every warp has for itself and that runs ahead
// over the ends of its tiles: a warp waits for nobody but its own weights, and one lane asks for them (with cp.async, a lane's
// address arithmetic for every 16 bytes kept the schedulers busy half of the time, and the streams at 4 TB/s). The shared unit's matrices
// are asked into L2 while the tokens are being routed. mma.sync multiplies by eight columns: in up_kernel the tokens, in down_kernel
// the terms of the tokens that use the expert, mostly one or two of them, so that one pass over them is enough.
#include "few_rows.cuh"
#include "route_choice.cuh"
#include "tcgen05.cuh"
#include <limits.h>

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
    int settled;                 // no kernel that is still running writes the router
    int up_shift;                // a gate or up row's sum: 2^up_shift parts, each of a warp of its own
    int unit_part, shared_part;  // a down row's: steps of a part (the last may have fewer), of an expert's and of the shared unit's
    float limit, alpha, shared_limit, shared_alpha, weight_scale;
};

namespace {
constexpr int UP_THREADS = 512, UP_WARPS = 16, TERMS = 3, MAX_TOKENS = 8, MAX_TOP = 16, MAX_UNITS = MAX_TOKENS * MAX_TOP, MAX_OUTPUTS = 256;
enum Kind { F32 = 0, BF16 = 1, MX4 = 2 };

// What up_kernel tells down_kernel. A token's units have places of their own among its choices (its slots), in the order of the experts.
struct Unit {                    // a distinct expert; they ascend
    uint32_t what;               // the expert, and from bit 8 on which tokens use it
    uint32_t slots;              // a token's slot, four bits a token
};
struct Plan {
    int n_units, pad[3];
    float own[MAX_TOKENS];       // the weight of a token's own row (identity outputs)
    uint32_t slots[MAX_TOKENS];  // which slots of a token are in use
    Unit unit[MAX_UNITS];
};

// What the warps of down_kernel's blocks take: the shared unit's steps, then those of every chosen expert, in whole parts.
// (A float's quotient of whole numbers below 2^21, half a step off the border, is on the right side of it.)
__host__ __device__ __forceinline__ int quotient(int a, float inverse) { return (int)(((float)a + 0.5f) * inverse); }
struct Shares {
    int shared_steps, unit_steps, shared_part, unit_part;
    int weight;                  // of a step of the shared unit, in quarters of an expert's
    float by_weight, by_unit, by_shared_part, by_unit_part;      // inverses
    // where warp w of W begins: the start of a part that is nearest to that share of the work
    template <int W> __host__ __device__ __forceinline__ int begin(int w, int units) const {
        const int shared = shared_steps * weight, at = (shared + units * unit_steps * 4) * w / W;
        const bool in_shared = at < shared;
        const int step = in_shared ? quotient(at, by_weight) : (at - shared) >> 2, unit = in_shared ? 0 : quotient(step, by_unit);
        const int steps = in_shared ? shared_steps : unit_steps, part = in_shared ? shared_part : unit_part, base = unit * unit_steps;
        const int near = quotient(step - base + part / 2, in_shared ? by_shared_part : by_unit_part) * part;
        return (in_shared ? 0 : shared_steps + base) + (near < steps ? near : steps);
    }
};
inline Shares shares_of(const DdExpertLayer& l, int step, int weight) {
    Shares s;
    s.shared_steps = (l.shared_inner + step - 1) / step;
    s.unit_steps = (l.inner + step - 1) / step;
    s.shared_part = l.shared_part; s.unit_part = l.unit_part; s.weight = weight;
    s.by_weight = 1.0f / weight; s.by_unit = 1.0f / s.unit_steps; s.by_shared_part = 1.0f / l.shared_part; s.by_unit_part = 1.0f / l.unit_part;
    return s;
}

struct Call {
    DdExpertLayer l;
    const void* y;               // [T, ldy]
    const float* residual;       // [T, ldr] or null
    float* out;                  // [T, ldo]
    const int* ids;              // [T] (by table)
    Plan* plan;
    uint8_t* hidden;             // [units][T][terms][row], the shared unit's rows behind them
    int* error_flag;
    int T, ldy, ldr, ldo, max_units;
    int row, shared_row;         // elements of a hidden row: whole steps, zeros behind the last feature
    int y_wide, router_wide, w_wide, inner_wide;        // rows of whole 16-byte pieces (w: all matrices that meet y, inner: all down)
    int router_tiles, share_shift, cluster_shift;                    // of the routing: rows by 16, warps and blocks that share columns (log2)
    int cluster, y_pitch, stages;                                    // y_pitch: bytes of a token's row in up_kernel's shared memory
    Shares shares;
    int unit_parts, shared_parts;                                    // of a down row
};
struct Maps { CUtensorMap gate_up, shared_gate_up, down, shared_down; };

struct Tile { float sum[16][few::COLUMNS + 1]; };
template <int N> struct Count { static constexpr int value = N; };

// What a warp multiplies at a time, a tile: 16 rows of a matrix on mma.sync, 4 with multiply-adds. A stage of its ring is one TMA box
// of a tile, gate and up rows together (a copy has a cost of its own: eight tokens with eight each of 64 experts of 2 x 1,024 x 2,048, 4 bits:
// up_kernel 37 us, 44 with two boxes a stage). Four stages: with five and six one token in bfloat16 takes 38.5 us instead of 32.1, eight 109
// and 111 instead of 108.
template <int KIND> struct Stream {
    static constexpr int ROWS = KIND == F32 ? few::F32_ROWS : 16, HALF = ROWS / 2;
    static constexpr int STEP = KIND == BF16 ? 64 : KIND == F32 ? 128 : 256;         // k
    static constexpr int SUB = KIND == MX4 ? 2 : 1;                                  // groups of 128 in it
    static constexpr int BOX_ROW = KIND == F32 ? 512 : 128, STAGE_BYTES = ROWS * BOX_ROW;
    static constexpr int ELEMENT = KIND == F32 ? 4 : 2;
    static constexpr int MOST_STAGES = 4;
};
template <int KIND> __host__ __device__ __forceinline__ int parts_of(int K, int part) {       // of a down row
    return K ? ((K + Stream<KIND>::STEP - 1) / Stream<KIND>::STEP + part - 1) / part : 0;
}
__host__ __device__ constexpr int step_of(int kind) { return kind == BF16 ? 64 : kind == F32 ? 128 : 256; }

// The boxes of a stage without TMA (rows that are no whole 16-byte pieces), in the layout that TMA gives them.
template <int KIND>
__device__ __forceinline__ void fill_stage(uint32_t slot, const void* matrix, size_t row_a, size_t row_b, size_t rows, int K, int step) {
    using S = Stream<KIND>;
    const int lane = threadIdx.x & 31;
    __syncwarp();
    for (int i = lane; i < S::STAGE_BYTES / 16; i += 32) {
        const int r = i / (S::BOX_ROW / 16), piece = i % (S::BOX_ROW / 16);
        const size_t row = min(r < S::HALF ? row_a + r : row_b + r - S::HALF, rows - 1);
        if constexpr (KIND == F32) {
            const float4 v = few::load4(reinterpret_cast<const float*>(matrix) + row * K, step * S::STEP + piece * 4, K, false);
            few::sts16(slot + i * 16, make_uint4(__float_as_uint(v.x), __float_as_uint(v.y), __float_as_uint(v.z), __float_as_uint(v.w)));
        } else
            few::sts16(slot + r * S::BOX_ROW + (piece ^ (r & 7)) * 16,
                       few::load8(reinterpret_cast<const __nv_bfloat16*>(matrix) + row * K, step * S::STEP + piece * 8, K, false));
    }
    __syncwarp();
}

// A warp's ring. The fetching lane asks for stage after stage; every lane waits for them in the same order.
template <int KIND> struct Ring {
    using S = Stream<KIND>;
    uint64_t* bars;
    uint32_t base;
    int stages, asked = 0, taken = 0;            // stage numbers; their phase follows from how often they wrapped
    uint32_t phase = 0;
    __device__ __forceinline__ Ring(uint64_t* b, uint32_t at, int n) : bars(b), base(at), stages(n) {}
    __device__ __forceinline__ void ask(const CUtensorMap* map, int step, int row, int matrix) {
        uint64_t* bar = &bars[asked];
        uint8_t* slot = reinterpret_cast<uint8_t*>(__cvta_shared_to_generic(base + asked * S::STAGE_BYTES));
        tc::mbar_expect_tx(bar, S::STAGE_BYTES);
        tc::tma_load_3d(slot, map, step * (KIND == MX4 ? S::BOX_ROW : S::STEP), row, matrix, bar);
    }
    __device__ __forceinline__ void next_asked() { asked = asked + 1 == stages ? 0 : asked + 1; }
    // the address of the next stage to read; `here`: it has been asked for
    __device__ __forceinline__ uint32_t take(bool here, volatile int* gave_up) {
        if (here) tc::mbar_wait(&bars[taken], phase, gave_up);
        const uint32_t at = base + taken * S::STAGE_BYTES;
        if (++taken == stages) { taken = 0; phase ^= 1; }
        return at;
    }
};

// What a warp multiplies without a pause: 64 k of a bfloat16 matrix, a group of 128 of a 4-bit one. 16-byte pieces of the other operand
// that a lane reads for one column, and where: on mma.sync lane (g, t) takes for row g and g + 8 of the matrix the pieces 2 t and
// 2 t + 1 of 64 bfloat16 numbers (under TMA's 128-byte swizzle eight lanes then meet in no bank), or the t-th eighth of every block of a
// 4-bit group.
template <int KIND> constexpr int PIECES = KIND == MX4 ? 4 : 2;
template <int KIND> constexpr int PART = KIND == MX4 ? 128 : 64;
template <int KIND>
__device__ __forceinline__ void take_column(uint4* b, const __nv_bfloat16* x, int part) {
    const int t = threadIdx.x & 3;
    const uint4* from = reinterpret_cast<const uint4*>(x + part * PART<KIND>);
#pragma unroll
    for (int i = 0; i < PIECES<KIND>; ++i) b[i] = from[KIND == MX4 ? 4 * i + t : 2 * t + i];
}
// The row of a tile's half that lane (g, t) has: 4-bit rows in another order, so that eight lanes' pieces of a group, under TMA's 128-byte
// swizzle, meet in no bank (rows r and r + 4 side by side).
template <int KIND> __device__ __forceinline__ int row_of(int g) { return KIND == MX4 ? g >> 1 | (g & 1) << 2 : g; }
// The scales of sixteen 4-bit groups of rows g and g + 8 (row_of): lane (g, t) holds those of groups 4 t .. 4 t + 3, and asks for them a
// stretch of sixteen ahead.
struct Scales {
    static constexpr int STRETCH = 16;
    uint32_t a[4], b[4];
    __device__ __forceinline__ void load(const uint32_t* rows, size_t row_a, size_t row_b, size_t last, int groups, int from, int to) {
        const int lane = threadIdx.x & 31, first = from + (lane & 3) * 4;
        const uint32_t *p = rows + min(row_a + row_of<MX4>(lane >> 2), last) * groups, *q = rows + min(row_b + row_of<MX4>(lane >> 2), last) * groups;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            a[j] = first + j < to ? p[first + j] : 0u;
            b[j] = first + j < to ? q[first + j] : 0u;
        }
    }
    // those of group number i of the stretch
    __device__ __forceinline__ void get(int i, uint32_t& four_a, uint32_t& four_b) const {
        const int from = (threadIdx.x & 28) | (i >> 2);
        four_a = __shfl_sync(0xffffffffu, i & 2 ? (i & 1 ? a[3] : a[2]) : (i & 1 ? a[1] : a[0]), from);
        four_b = __shfl_sync(0xffffffffu, i & 2 ? (i & 1 ? b[3] : b[2]) : (i & 1 ? b[1] : b[0]), from);
    }
};

// A part of a tile (its sub-th in the stage) by P times eight columns. four0, four1: the scales of a 4-bit group of rows g and g + 8.
// F16: the other operand is float16 (in the order of mx4::pairs_f16), not bfloat16.
template <int KIND, int P, bool F16 = false>
__device__ __forceinline__ void mma_step(uint32_t slot, int sub, uint32_t four0, uint32_t four1, const uint4 (*b)[PIECES<KIND>], float (*d)[4]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    if constexpr (KIND == MX4) {
        const int row = row_of<KIND>(g);
        const uint32_t at = slot + row * 128 + ((4 * sub + t) ^ row) * 16;            // [half][row][group]
        const uint4 a0 = few::lds16(at), a1 = few::lds16(at + 1024);
        const uint32_t r0[4] = {a0.x, a0.y, a0.z, a0.w}, r1[4] = {a1.x, a1.y, a1.z, a1.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t v0[4], v1[4];
            if (F16) { mx4::pairs_f16(r0[i], v0); mx4::pairs_f16(r1[i], v1); }
            else { mx4::whole_pairs(r0[i], v0); mx4::whole_pairs(r1[i], v1); }
            const float by0 = mx4::scale(four0, i), by1 = mx4::scale(four1, i);
#pragma unroll
            for (int p = 0; p < P; ++p) {
                float e[4] = {0.f, 0.f, 0.f, 0.f};
                if (F16) {
                    few::mma_f16(e, v0[0], v1[0], v0[1], v1[1], b[p][i].x, b[p][i].y);
                    few::mma_f16(e, v0[2], v1[2], v0[3], v1[3], b[p][i].z, b[p][i].w);
                } else few::block_product(v0, v1, b[p][i], e);
                few::add_block(by0, by1, e, d[p]);
            }
        }
    } else {
        // (the tensor cores cut off where they add: a sum of 64 products starts from nothing and is added rounded)
        float e[P][4];
#pragma unroll
        for (int p = 0; p < P; ++p) e[p][0] = e[p][1] = e[p][2] = e[p][3] = 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t at = slot + g * 128 + ((2 * t + i) ^ g) * 16;
            const uint4 a0 = few::lds16(at), a1 = few::lds16(at + 1024);
#pragma unroll
            for (int p = 0; p < P; ++p) {
                few::mma(e[p], a0.x, a1.x, a0.y, a1.y, b[p][i].x, b[p][i].y);
                few::mma(e[p], a0.z, a1.z, a0.w, a1.w, b[p][i].z, b[p][i].w);
            }
        }
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int j = 0; j < 4; ++j) d[p][j] += e[p][j];
    }
}
template <int KIND>
__device__ __forceinline__ void put_tile(Tile& to, const float* d) {
    const int lane = threadIdx.x & 31, g = row_of<KIND>(lane >> 2), t = lane & 3;
#pragma unroll
    for (int i = 0; i < 4; ++i) to.sum[g + 8 * (i >> 1)][2 * t + (i & 1)] = d[i];
}

// Up to eight token numbers, ascending, four bits each.
__device__ __forceinline__ uint32_t list_of(uint32_t users) {
    uint32_t list = 0;
    for (int shift = 0; users; users &= users - 1, shift += 4) list |= (uint32_t)(__ffs(users) - 1) << shift;
    return list;
}
__device__ __forceinline__ int listed(uint32_t list, int i) { return list >> (4 * i) & 7; }

// float32: a step of four rows by N tokens of a list; row t of the other operand: x + t * ld. Four tokens at a time: registers.
template <int N> constexpr int AT_ONCE = N < 4 ? N : 4;
template <int N>
__device__ __forceinline__ void take_rows(float4* b, const float* x, size_t ld, uint32_t list, int step, int h) {
#pragma unroll
    for (int i = 0; i < AT_ONCE<N>; ++i) b[i] = *reinterpret_cast<const float4*>(x + listed(list, h + i) * ld + step * 128 + (threadIdx.x & 31) * 4);
}
template <int N>
__device__ __forceinline__ void fma_rows(uint32_t slot, const float4* b, int h, unsigned long long (*d)[N]) {
#pragma unroll
    for (int r = 0; r < few::F32_ROWS; ++r) {
        const uint4 v = few::lds16(slot + r * 512 + (threadIdx.x & 31) * 16);
#pragma unroll
        for (int i = 0; i < AT_ONCE<N>; ++i) {
            few::fma_pair(d[r][h + i], __uint_as_float(v.x), __uint_as_float(v.y), b[i].x, b[i].y);
            few::fma_pair(d[r][h + i], __uint_as_float(v.z), __uint_as_float(v.w), b[i].z, b[i].w);
        }
    }
}
template <int N>
__device__ __forceinline__ void fma_step(uint32_t slot, const float* x, size_t ld, uint32_t list, int step, unsigned long long (*d)[N]) {
#pragma unroll
    for (int h = 0; h < N; h += AT_ONCE<N>) {
        float4 b[AT_ONCE<N>];
        take_rows<N>(b, x, ld, list, step, h);
        fma_rows<N>(slot, b, h, d);
    }
}
// The warp's sums of four rows by N tokens, one a lane: lane l has that of row (l * 4 N / 32) / N and the token of the list at
// (l * 4 N / 32) % N; lanes in between have none of their own (owns_sum).
template <int N>
__device__ __forceinline__ float row_sums(unsigned long long (*d)[N]) {
    float v[few::F32_ROWS * N];
#pragma unroll
    for (int r = 0; r < few::F32_ROWS; ++r)
#pragma unroll
        for (int i = 0; i < N; ++i) v[r * N + i] = few::pair_sum(d[r][i]);
    return few::warp_sums<few::F32_ROWS * N>(v);
}
template <int N> __device__ __forceinline__ bool owns_sum(int n) {
    const int lane = threadIdx.x & 31;
    return lane % (32 / (few::F32_ROWS * N)) == 0 && lane * (few::F32_ROWS * N) / 32 % N < n;
}
// ... of rows r0 .. r0 + 3 and the first n tokens of a list, set in `to`.
template <int N>
__device__ __forceinline__ void put_rows(Tile& to, int r0, uint32_t list, int n, float sum) {
    const int at = (threadIdx.x & 31) * (few::F32_ROWS * N) / 32;
    if (owns_sum<N>(n)) to.sum[r0 + at / N][listed(list, at % N)] = sum;
}
// f(Count<N>) with N tokens at a time, N at least n.
template <typename F> __device__ __forceinline__ void by_count(int n, F f) {
    if (n == 1) f(Count<1>{});
    else if (n == 2) f(Count<2>{});
    else if (n <= 4) f(Count<4>{});
    else f(Count<8>{});
}

// ---------------------------------------------------------------- routing, by every cluster for itself
struct Routing {
    int chosen[MAX_TOKENS][MAX_TOP];
    float weight[MAX_TOKENS][MAX_TOP];
    float gate[MAX_TOKENS];                      // the shared unit's
    uint32_t y_top[MAX_TOKENS];                  // bits of a token's largest |y| (4-bit matrices)
    float y_back[MAX_TOKENS];                    // what its float16 row has to be multiplied with
    uint32_t users[MAX_OUTPUTS];                 // per output: which tokens chose it
    int count[UP_WARPS];
    int n_units;
    int expert[MAX_UNITS];
    uint8_t unit_of[MAX_OUTPUTS];
    float unit_weight[MAX_UNITS][MAX_TOKENS];    // a token's weight on a unit
    uint32_t unit_slots[MAX_UNITS], slots[MAX_TOKENS];      // as in Plan (of the block that writes it)
    uint64_t arrived;                            // the cluster's partial logits
};

// Which rows and columns of the router a warp multiplies: items of 16 rows by a share of this block's columns.
struct RouterItem {
    int tile, from, to;
    __device__ __forceinline__ RouterItem(const Call& c, int kind, int item) {
        const int steps = (c.l.width + (kind == F32 ? 127 : 31)) / (kind == F32 ? 128 : 32), rank = c.cluster_shift ? (int)tc::cluster_rank() : 0;
        const int begin = steps * rank >> c.cluster_shift, end = steps * (rank + 1) >> c.cluster_shift;
        int share = 0;
        for (tile = item; tile >= c.router_tiles; tile -= c.router_tiles) ++share;
        from = begin + ((end - begin) * share >> c.share_shift);
        to = begin + ((end - begin) * (share + 1) >> c.share_shift);
    }
};
__device__ __forceinline__ const __nv_bfloat16* router_row(const Call& c, int tile, int i) {
    return reinterpret_cast<const __nv_bfloat16*>(c.l.router) +
           (size_t)min(tile * 16 + i, c.l.experts + c.l.identity + c.l.shared_gate - 1) * c.l.router_stride;
}

// The logits of the block's columns for all tokens, by item. ahead: the first item's first steps.
template <int KIND>
__device__ void partial_logits(const Call& c, const uint8_t* y, int items, Tile* parts, few::Ahead& ahead) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2;
    // (float32: four rows of an item a warp)
    constexpr int PARTS = KIND == F32 ? 16 / few::F32_ROWS : 1;
    for (int work = warp; work < items * PARTS; work += UP_WARPS) {
        const int item = work / PARTS;
        const RouterItem it(c, KIND, item);
        if constexpr (KIND == F32) {
            const int last = c.l.experts + c.l.identity + c.l.shared_gate - 1, r0 = work % PARTS * few::F32_ROWS;
            const float* w[few::F32_ROWS];
            unsigned long long acc[few::F32_ROWS][MAX_TOKENS] = {};
#pragma unroll
            for (int r = 0; r < few::F32_ROWS; ++r)
                w[r] = reinterpret_cast<const float*>(c.l.router) + (size_t)min(it.tile * 16 + r0 + r, last) * c.l.router_stride;
            few::stream_f32<MAX_TOKENS>(w, reinterpret_cast<const float*>(y), c.y_pitch / 4, (1u << c.T) - 1, c.l.width, it.from, it.to, c.router_wide,
                                        true, acc);
            put_rows<MAX_TOKENS>(parts[item], r0, 0x76543210u, MAX_TOKENS, row_sums<MAX_TOKENS>(acc));
        } else {
            const __nv_bfloat16* x = reinterpret_cast<const __nv_bfloat16*>(y + min(g, c.T - 1) * c.y_pitch);
            const __nv_bfloat16 *w0 = router_row(c, it.tile, g), *w1 = router_row(c, it.tile, g + 8);
            if (work != warp) ahead.load(w0, w1, c.l.width, it.from, it.to, c.router_wide);
            float d[4] = {0.f, 0.f, 0.f, 0.f};
            few::stream_bf16(w0, w1, x, c.l.width, it.from, it.to, c.router_wide, ahead, d);
            put_tile<BF16>(parts[item], d);
        }
    }
}

template <int KIND>
__device__ void route(const Call& c, const uint8_t* y, Routing& r, float* scratch, few::Ahead& ahead, volatile int* gave_up) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int outputs = c.l.experts + c.l.identity;
    if (threadIdx.x < MAX_OUTPUTS) r.users[threadIdx.x] = 0;
    if (threadIdx.x < MAX_UNITS) r.unit_slots[threadIdx.x] = 0;
    if (threadIdx.x < MAX_TOKENS) r.slots[threadIdx.x] = 0;
    if (c.l.router) {
        const int rows = outputs + c.l.shared_gate, tiles = c.router_tiles, shares = 1 << c.share_shift;
        const int n = tiles * 16 * MAX_TOKENS;                          // logits, a row of eight an output
        const int rank = c.cluster > 1 ? (int)tc::cluster_rank() : 0;
        Tile* parts = reinterpret_cast<Tile*>(scratch);
        float* sums = scratch + (sizeof(Tile) / 4) * tiles * shares;     // [cluster][n]: what every block of the cluster found
        partial_logits<KIND>(c, y, tiles * shares, parts, ahead);
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += UP_THREADS) {
            const int row = i / MAX_TOKENS, t = i % MAX_TOKENS;
            float z = 0.f;
            if (t < c.T)
#pragma unroll 1
                for (int s = 0; s < shares; ++s) z += parts[s * tiles + row / 16].sum[row % 16][t];
            if (c.cluster == 1) sums[i] = z;
            else
#pragma unroll 1
                for (int to = 0; to < c.cluster; ++to) tc::st_async_f32(tc::map_to_rank(&sums[rank * n + i], to), z, tc::map_to_rank(&r.arrived, to));
        }
        if (c.cluster > 1) {
            if (threadIdx.x == 0) tc::mbar_expect_tx(&r.arrived, c.cluster * n * 4);
            tc::mbar_wait(&r.arrived, 0, gave_up);
        } else __syncthreads();
        float* value = sums + c.cluster * n;                            // [T][outputs]
        float* score = value + MAX_TOKENS * outputs;
        float* worth = score + MAX_TOKENS * outputs;
        for (int i = threadIdx.x; i < rows * MAX_TOKENS; i += UP_THREADS) {
            const int e = i / MAX_TOKENS, t = i % MAX_TOKENS;
            float z = 0.f;
#pragma unroll 1
            for (int s = 0; s < c.cluster; ++s) z += sums[s * n + i];
            if (e >= outputs) r.gate[t] = 1.0f / (1.0f + expf(-z));
            else if (c.l.softmax) value[t * outputs + e] = z;
            else dd_sigmoid_score(z, e, c.l.correction, c.l.groups, value + t * outputs, score + t * outputs);
        }
        if (!c.l.shared_gate && threadIdx.x < MAX_TOKENS) r.gate[threadIdx.x] = 1.f;
        __syncthreads();
        if (warp < c.T) {
            float *sc = score + warp * outputs, *v = value + warp * outputs, *wo = worth + warp * max(c.l.groups, MAX_TOP);
            if (outputs <= 32)
                dd_choose_few<1>(sc, v, wo, outputs, c.l.top, c.l.groups, c.l.keep, c.l.weight_scale, c.l.softmax, c.l.correction, c.l.renormalize,
                                 r.chosen[warp], r.weight[warp]);
            else if (outputs <= 64)
                dd_choose_few<2>(sc, v, wo, outputs, c.l.top, c.l.groups, c.l.keep, c.l.weight_scale, c.l.softmax, c.l.correction, c.l.renormalize,
                                 r.chosen[warp], r.weight[warp]);
            else
                dd_choose_few<MAX_OUTPUTS / 32>(sc, v, wo, outputs, c.l.top, c.l.groups, c.l.keep, c.l.weight_scale, c.l.softmax, c.l.correction,
                                                c.l.renormalize, r.chosen[warp], r.weight[warp]);
        }
    } else {
        const int t = threadIdx.x / MAX_TOP, k = threadIdx.x % MAX_TOP;
        if (t < c.T && k < c.l.top) {
            const int id = c.ids[t];
            r.chosen[t][k] = id >= 0 && id < c.l.vocab ? c.l.table[(size_t)id * c.l.top + k] : -1;
            r.weight[t][k] = c.l.weight_scale;
        }
        if (threadIdx.x < MAX_TOKENS) r.gate[threadIdx.x] = 1.f;
    }
    __syncthreads();
    const int pair_t = threadIdx.x / MAX_TOP, pair_k = threadIdx.x % MAX_TOP;        // a thread a (token, choice)
    const bool pair = pair_t < c.T && pair_k < c.l.top;
    const int pair_e = pair ? r.chosen[pair_t][pair_k] : -1;
    if (pair) {
        if (pair_e >= 0 && pair_e < outputs) atomicOr(&r.users[pair_e], 1u << pair_t);
        else if (blockIdx.x == 0) atomicOr(c.error_flag, 1);           // an expert out of range: left out, and reported
    }
    __syncthreads();
    // the distinct experts, ascending (a thread an expert)
    const bool used = (int)threadIdx.x < c.l.experts && r.users[threadIdx.x];
    const uint32_t votes = __ballot_sync(0xffffffffu, used);
    if (lane == 0) r.count[warp] = __popc(votes);
    __syncthreads();
    int at = __popc(votes & ((1u << lane) - 1)), total = 0;
#pragma unroll 1
    for (int w = 0; w < MAX_OUTPUTS / 32; ++w) {
        if (w < warp) at += r.count[w];
        total += r.count[w];
    }
    if (used) {
        r.expert[at] = threadIdx.x;
        r.unit_of[threadIdx.x] = (uint8_t)at;
    }
    if (threadIdx.x == 0) r.n_units = total;
    __syncthreads();
    if (pair_e >= 0 && pair_e < c.l.experts) {    // a token's choices of an expert (a table may name one twice), by the first of them
        float w = 0.f;
        bool first = true;
        int slot = 0;
#pragma unroll 1
        for (int i = 0; i < c.l.top; ++i) {
            const int e = r.chosen[pair_t][i];
            slot += e >= 0 && e < pair_e;
            if (e == pair_e) {
                w += r.weight[pair_t][i];
                if (i < pair_k) first = false;
            }
        }
        if (first) {
            r.unit_weight[r.unit_of[pair_e]][pair_t] = w;
            if (blockIdx.x == gridDim.x - 1) {
                atomicOr(&r.unit_slots[r.unit_of[pair_e]], (uint32_t)slot << (4 * pair_t));
                atomicOr(&r.slots[pair_t], 1u << slot);
            }
        }
    }
    __syncthreads();
}

// Asks for a matrix in L2, shared out over the grid's threads (4 KB each time).
__device__ __forceinline__ void ask_for(const void* base, size_t bytes) {
    constexpr size_t PIECE = 4096;
    const size_t n = bytes / PIECE, threads = (size_t)gridDim.x * blockDim.x;
    for (size_t i = (size_t)threadIdx.x * gridDim.x + blockIdx.x; i < n; i += threads)
        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(reinterpret_cast<const uint8_t*>(base) + i * PIECE), "r"((uint32_t)PIECE) : "memory");
}
__device__ __forceinline__ size_t matrix_bytes(int kind, size_t rows, int K) {
    return kind == MX4 ? rows * ((K + mx4::GROUP - 1) / mx4::GROUP) * mx4::GROUP_BYTES : rows * K * (kind == F32 ? 4 : 2);
}

// The barriers of a block's rings, and whether one of its waits ran out.
template <int W> struct Barriers {
    uint64_t full[W][8];
    int gave_up;
    __device__ __forceinline__ void init() {
        for (int i = threadIdx.x; i < W * 8; i += W * 32) tc::mbar_init(&full[i / 8][i % 8], 1);
        if (threadIdx.x == 0) gave_up = 0;
        tc::fence_barrier_init();
        tc::fence_proxy_async();
    }
};
// The terms of a value beyond bfloat16's largest number: an infinity is the first term alone, a number begins with the largest.
constexpr float BF16_MAX = 3.38953138925153547590e38f;       // 2^128 - 2^120
__device__ __noinline__ void put_terms_of_ends(__nv_bfloat16* h, int row, float v) {
    const __nv_bfloat16 first = isfinite(v) ? __float2bfloat16_rn(copysignf(BF16_MAX, v)) : __float2bfloat16_rn(v);
    const float rest = isfinite(v) ? v - __bfloat162float(first) : 0.f;
    const __nv_bfloat16 second = __float2bfloat16_rn(rest);
    h[0] = first;
    h[row] = second;
    h[2 * row] = __float2bfloat16_rn(rest - __bfloat162float(second));
    static_assert(TERMS == 3, "the terms above");
}
// A unit's value, in float32, as its hidden row keeps it.
template <int KIND>
__device__ __forceinline__ void put_hidden(const Call& c, bool shared, int unit, int t, int feature, float v) {
    const int row = shared ? c.shared_row : c.row;
    const size_t slot = shared ? (size_t)t : (size_t)unit * c.T + t, before = shared ? (size_t)c.max_units * c.T * c.row : 0;
    if constexpr (KIND == F32) reinterpret_cast<float*>(c.hidden)[before + slot * row + feature] = v;
    else {
        __nv_bfloat16* h = reinterpret_cast<__nv_bfloat16*>(c.hidden) + before * TERMS + slot * TERMS * row + feature;
        if (!(fabsf(v) <= BF16_MAX)) return put_terms_of_ends(h, row, v);
#pragma unroll
        for (int i = 0; i < TERMS; ++i) {
            const __nv_bfloat16 term = __float2bfloat16_rn(v);
            h[i * row] = term;
            v -= __bfloat162float(term);
        }
    }
}
// (Not inlined: the kernel is read from L2 once for every launch, and its instructions are what a small layer waits for.)
__device__ __noinline__ float unit_value(const Call& c, bool shared, float a, float b, float by) {
    if (shared) return by * dd_gated_value<false>(a, b, c.l.shared_form, c.l.shared_limit, c.l.shared_alpha);
    if (c.l.gated) return by * dd_gated_value<false>(a, b, c.l.form, c.l.limit, c.l.alpha);
    return c.l.weight_input ? dd_activation(by * a, c.l.act) : by * dd_activation(a, c.l.act);
}

template <int KIND>
__global__ void __launch_bounds__(UP_THREADS, 1)
up_kernel(const __grid_constant__ Call c, const __grid_constant__ Maps maps) {
    using S = Stream<KIND>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ Routing r;
    __shared__ Tile red[2][UP_WARPS];
    __shared__ Barriers<UP_WARPS> bars;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, width = c.l.width;
    dd_launch_dependents();
    if (c.l.shared_inner && c.w_wide) ask_for(c.l.shared_gate_up, matrix_bytes(KIND, (size_t)2 * c.l.shared_inner, width));
    // The warp's first item of the router: of a settled layer it is read while the kernel before this one ends, of another one behind the
    // wait (one token, sixteen experts of 1,600 x 1,600: 24.6 us settled, 25.3 not).
    few::Ahead ahead;
    auto read_router = [&] {
        const RouterItem it(c, KIND, warp);
        if (it.from < it.to) ahead.load(router_row(c, it.tile, lane >> 2), router_row(c, it.tile, (lane >> 2) + 8), width, it.from, it.to, c.router_wide);
    };
    if (KIND != F32 && c.l.router && c.l.settled) read_router();
    bars.init();
    if (threadIdx.x == 0) {
        if (c.w_wide) tc::prefetch_tensormap(&maps.gate_up);
        if (c.w_wide && c.l.shared_inner) tc::prefetch_tensormap(&maps.shared_gate_up);
        tc::mbar_init(&r.arrived, 1);
        tc::fence_barrier_init();
    }
    if (c.cluster > 1) {                          // a block's shared memory may be written once it runs and has its barrier
        tc::cluster_arrive();
        tc::cluster_wait();
    }
    dd_grid_wait();
    if (KIND != F32 && c.l.router && !c.l.settled) read_router();
    // the tokens' rows with zeros behind them; a row starts 16 bytes (4-bit matrices: 64) off the one before it, modulo 128, so that
    // eight lanes' pieces of two rows meet in no bank
    uint8_t* y = smem + UP_WARPS * c.stages * S::STAGE_BYTES;
    {
        const int pieces = c.y_pitch / 128 * 8, in = 16 / S::ELEMENT;
        const int by = c.T > 4 ? 2 : c.T > 2 ? 4 : c.T > 1 ? 8 : 16, t = warp / by;          // warps a token
        constexpr int FLIGHT = 4;                 // pieces that a lane asks for at a time
        if (t < c.T)
#pragma unroll 1
            for (int at = (warp % by) * 32 + lane; at < pieces; at += by * 32 * FLIGHT) {
                uint4 v[FLIGHT];
#pragma unroll
                for (int i = 0; i < FLIGHT; ++i) {
                    const int piece = at + i * by * 32;          // (behind the row: zeros, and no load)
                    if constexpr (KIND == F32) {
                        const float4 f = few::load4(reinterpret_cast<const float*>(c.y) + (size_t)t * c.ldy, piece * in, width, c.y_wide);
                        v[i] = make_uint4(__float_as_uint(f.x), __float_as_uint(f.y), __float_as_uint(f.z), __float_as_uint(f.w));
                    } else v[i] = few::load8(reinterpret_cast<const __nv_bfloat16*>(c.y) + (size_t)t * c.ldy, piece * in, width, c.y_wide);
                }
#pragma unroll
                for (int i = 0; i < FLIGHT; ++i)
                    if (at + i * by * 32 < pieces) *reinterpret_cast<uint4*>(y + t * c.y_pitch + (at + i * by * 32) * 16) = v[i];
            }
    }
    __syncthreads();
    // 4-bit matrices meet the rows as float16 (their elements become that in one instruction): times a power of two that brings a
    // row's largest element to 2^14, every bfloat16 of more than 2^-31 of it is kept exactly, what is below to 2^-39 of it
    uint8_t* x_rows = y;
    if constexpr (KIND == MX4) {
        x_rows = y + c.T * c.y_pitch;
        const int pieces = c.y_pitch / 128 * 8, by = c.T > 4 ? 2 : c.T > 2 ? 4 : c.T > 1 ? 8 : 16, t = warp / by;
        if (threadIdx.x < MAX_TOKENS) r.y_top[threadIdx.x] = 0;
        __syncthreads();
        if (t < c.T) {
            uint32_t top = 0;
#pragma unroll 1
            for (int at = (warp % by) * 32 + lane; at < pieces; at += by * 32) {
                const uint4 v = *reinterpret_cast<const uint4*>(y + t * c.y_pitch + at * 16);
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) top = max(top, max(w[i] << 16 & 0x7fff0000u, w[i] & 0x7fff0000u));
            }
            top = __reduce_max_sync(0xffffffffu, top);
            if (lane == 0) atomicMax(&r.y_top[t], top);
        }
        __syncthreads();
        if (t < c.T) {
            // times 2^up (where the largest is no number, so far down that no number becomes an infinity beside it)
            const int up = min(126, 141 - (int)(r.y_top[t] >> 23));
            const float times = __uint_as_float((uint32_t)(up + 127) << 23);
            if (warp % by == 0 && lane == 0) r.y_back[t] = __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll 1
            for (int at = (warp % by) * 32 + lane; at < pieces; at += by * 32) {
                const uint4 v = *reinterpret_cast<const uint4*>(y + t * c.y_pitch + at * 16);
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                uint32_t even[2], odd[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(even[i]) : "f"(__uint_as_float(w[2 * i + 1] << 16) * times), "f"(__uint_as_float(w[2 * i] << 16) * times));
                    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(odd[i]) : "f"(__uint_as_float(w[2 * i + 1] & 0xffff0000u) * times),
                        "f"(__uint_as_float(w[2 * i] & 0xffff0000u) * times));
                }
                *reinterpret_cast<uint4*>(x_rows + t * c.y_pitch + at * 16) = make_uint4(even[0], even[1], odd[0], odd[1]);
            }
        }
    }
    route<KIND>(c, y, r, reinterpret_cast<float*>(x_rows + c.T * c.y_pitch), ahead, &bars.gave_up);
    if (blockIdx.x == gridDim.x - 1) {            // (it has the fewest tiles)
        for (int u = threadIdx.x; u < r.n_units; u += UP_THREADS) c.plan->unit[u] = {(uint32_t)r.expert[u] | r.users[r.expert[u]] << 8, r.unit_slots[u]};
        if (threadIdx.x == 0) c.plan->n_units = r.n_units;
        if (threadIdx.x < c.T) {
            float own = 0.f;
            for (int k = 0; k < c.l.top && c.l.identity; ++k)
                if (r.chosen[threadIdx.x][k] >= c.l.experts && r.chosen[threadIdx.x][k] < c.l.experts + c.l.identity) own += r.weight[threadIdx.x][k];
            c.plan->own[threadIdx.x] = own;
            c.plan->slots[threadIdx.x] = r.slots[threadIdx.x];
        }
    }
    // tiles: the shared unit's, then every chosen expert's
    const int features = c.l.gated ? S::HALF : S::ROWS;
    const int per_unit = (c.l.inner + features - 1) / features, for_shared = (c.l.shared_inner + S::HALF - 1) / S::HALF;
    const int total = for_shared + r.n_units * per_unit;
    const float per_unit_inverse = 1.0f / (float)per_unit;
    // `share` warps share a tile's columns (choose_parts; a tile alone in a warp needs no barrier of the block)
    const int share = 1 << c.l.up_shift, slots = UP_WARPS >> c.l.up_shift, slot = warp >> c.l.up_shift, part = warp & (share - 1), stride = gridDim.x * slots;
    const int steps = (width + S::STEP - 1) / S::STEP, from = steps * part >> c.l.up_shift, to = steps * (part + 1) >> c.l.up_shift;
    // a tile: its unit (-1: the shared one), first feature, matrix of the stack (gate and up are two), and the rows where its halves begin:
    // gate rows and the same features' up rows; plain: neighbours
    struct Place { int unit, first, matrix, row_a, row_b; };
    auto place_of = [&](int tile) {
        Place p;
        // (a float's quotient of whole numbers below 2^21, half a step off the border, is on the right side of it)
        p.unit = tile < for_shared ? -1 : (int)(((float)(tile - for_shared) + 0.5f) * per_unit_inverse);
        const bool gated = p.unit < 0 || c.l.gated;
        const int inner = p.unit < 0 ? c.l.shared_inner : c.l.inner;
        p.first = p.unit < 0 ? tile * S::HALF : (tile - for_shared - p.unit * per_unit) * features;
        p.matrix = p.unit < 0 ? 0 : r.expert[p.unit] * (gated ? 2 : 1);
        p.row_a = p.matrix * inner + p.first;
        p.row_b = p.row_a + (gated ? inner : S::HALF);
        return p;
    };
    Ring<KIND> ring(bars.full[warp], tc::smem_u32(smem) + warp * c.stages * S::STAGE_BYTES, c.stages);
    // the ring's fetching end
    int f_tile = slot * gridDim.x + blockIdx.x, f_step = from;
    Place f = {};
    if (f_tile < total) f = place_of(f_tile);
    auto fetch = [&] {
        if (f_tile >= total || from >= to) return;
        if (c.w_wide && lane == 0) ring.ask(f.unit < 0 ? &maps.shared_gate_up : &maps.gate_up, f_step, f.first, f.matrix);
        ring.next_asked();
        if (++f_step == to) {
            f_step = from;
            f_tile += stride;
            if (f_tile < total) f = place_of(f_tile);
        }
    };
#pragma unroll 1
    for (int i = 0; i < c.stages - 1; ++i) fetch();
    Scales have, soon;
    const int groups = (width + mx4::GROUP - 1) / mx4::GROUP;
    auto ask_scales = [&](int tile, int at) {
        const Place p = place_of(tile);
        const bool shared = p.unit < 0;
        soon.load(reinterpret_cast<const uint32_t*>(shared ? c.l.shared_gate_up_scales : c.l.gate_up_scales), p.row_a, p.row_b,
                  (shared ? (size_t)2 * c.l.shared_inner : (size_t)c.l.experts * c.l.inner * (c.l.gated ? 2 : 1)) - 1, groups, at * S::SUB,
                  min(to * S::SUB, groups));
    };
    if (KIND == MX4 && slot * gridDim.x + blockIdx.x < total && from < to) ask_scales(slot * gridDim.x + blockIdx.x, from);
    // (columns beyond the tokens read the last one's row; nobody looks at them)
    const __nv_bfloat16* x = reinterpret_cast<const __nv_bfloat16*>(x_rows + min(lane >> 2, c.T - 1) * c.y_pitch);
    // (with shared tiles every warp of the block takes part in every round's barrier)
    for (int turn = 0, round = blockIdx.x; round < total; round += stride, turn ^= 1) {
        const int tile = round + slot * gridDim.x;
        const bool mine = tile < total;
        const Place p = place_of(mine ? tile : 0);
        const bool shared = p.unit < 0;
        const uint32_t users = shared ? (1u << c.T) - 1 : r.users[r.expert[p.unit]];
        const void* matrix = shared ? c.l.shared_gate_up : c.l.gate_up;
        const size_t matrix_rows = shared ? (size_t)2 * c.l.shared_inner : (size_t)c.l.experts * c.l.inner * (c.l.gated ? 2 : 1);
        auto next = [&](int s) {
            const uint32_t at = ring.take(c.w_wide, &bars.gave_up);
            if (!c.w_wide) fill_stage<KIND>(at, matrix, p.row_a, p.row_b, matrix_rows, width, s);
            return at;
        };
        if constexpr (KIND == F32) {
            if (mine)
                by_count(__popc(users), [&](auto count) {
                    constexpr int N = decltype(count)::value;
                    const uint32_t list = list_of(users);         // (what it lacks to N names token 0 again, and is dropped)
                    unsigned long long d[few::F32_ROWS][N] = {};
                    for (int s = from; s < to; ++s) {
                        fma_step<N>(next(s), reinterpret_cast<const float*>(y), c.y_pitch / 4, list, s, d);
                        __syncwarp();
                        fetch();          // into the stage before this one, which the warp has read
                    }
                    put_rows<N>(red[turn][warp], 0, list, __popc(users), row_sums<N>(d));
                });
            if (share > 1) __syncthreads();          // (the other set is written next: one barrier a round is enough)
            else __syncwarp();
            if (mine && part == 0) {
                const int n = shared || c.l.gated ? S::HALF : S::ROWS;
                for (int i = lane; i < n * c.T; i += 32) {
                    const int t = i / n, k = i % n, feature = p.first + k;
                    if (feature >= (shared ? c.l.shared_inner : c.l.inner) || !(users >> t & 1)) continue;
                    const Tile* have = &red[turn][warp];
                    const int other = n == S::HALF ? k + S::HALF : k;         // (of a plain unit nobody looks at b)
                    float a = have->sum[k][t], b = have->sum[other][t];
#pragma unroll 1
                    for (int s = 1; s < share; ++s) {
                        a += have[s].sum[k][t];
                        b += have[s].sum[other][t];
                    }
                    put_hidden<KIND>(c, shared, p.unit, t, feature, unit_value(c, shared, a, b, shared ? r.gate[t] : r.unit_weight[p.unit][t]));
                }
            }
        } else {
            float d[1][4] = {};
            if (mine) {
                for (int s = from; s < to; ++s) {
                    const uint32_t at = next(s);
#pragma unroll
                    for (int sub = 0; sub < S::SUB; ++sub) {
                        uint32_t four0 = 0, four1 = 0;
                        if (KIND == MX4) {
                            const int i = ((s - from) * S::SUB + sub) % Scales::STRETCH, then = s + Scales::STRETCH / S::SUB;
                            if (i == 0) {         // this stretch's have come; the next one's, of this tile or the warp's next, are asked for
                                have = soon;
                                if (then < to) ask_scales(tile, then);
                                else if (tile + stride < total) ask_scales(tile + stride, from);
                            }
                            have.get(i, four0, four1);
                        }
                        uint4 b[1][PIECES<KIND>];
                        take_column<KIND>(b[0], x, s * S::SUB + sub);
                        mma_step<KIND, 1, KIND == MX4>(at, sub, four0, four1, b, d);
                    }
                    __syncwarp();
                    fetch();
                }
            }
            if (share > 1) {                      // the first of the sharers adds up
                if (part) put_tile<KIND>(red[turn][warp], d[0]);
                __syncthreads();
                if (mine && part == 0) {
                    const int g = row_of<KIND>(lane >> 2), t = lane & 3;
#pragma unroll 1
                    for (int s = 1; s < share; ++s)          // (its own part's are still here)
#pragma unroll
                        for (int i = 0; i < 4; ++i) d[0][i] += red[turn][warp + s].sum[g + 8 * (i >> 1)][2 * t + (i & 1)];
                }
            }
            if (mine && part == 0) {
                // lane (g, t): features g (and g + 8 of a plain unit) of tokens 2 t and 2 t + 1
                const int inner = shared ? c.l.shared_inner : c.l.inner, g = row_of<KIND>(lane >> 2);
                const bool gated = shared || c.l.gated;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int t = 2 * (lane & 3) + (i & 1), feature = p.first + g + (i >> 1) * S::HALF;
                    if ((gated && i > 1) || feature >= inner || !(users >> t & 1)) continue;
                    const float back = KIND == MX4 ? r.y_back[t] : 1.f;
                    put_hidden<KIND>(c, shared, p.unit, t, feature, unit_value(c, shared, d[0][i] * back, d[0][i | 2] * back, shared ? r.gate[t] : r.unit_weight[p.unit][t]));
                }
            }
        }
        // behind the last feature: zeros to the end of the row
        const int inner = shared ? c.l.shared_inner : c.l.inner, row = shared ? c.shared_row : c.row;
        if (mine && part == 0 && p.first + (shared ? S::HALF : features) >= inner)
            for (int i = lane; i < (row - inner) * c.T; i += 32)
                if (users >> (i % c.T) & 1) put_hidden<KIND>(c, shared, p.unit, i % c.T, inner + i / c.T, 0.f);
    }
    if (bars.gave_up && lane == 0) atomicOr(c.error_flag, 8);
}

// A step of the shared unit, which every token uses, takes longer than an expert's, in quarters of which this is: in bfloat16 layers with three
// times eight columns, whose pieces there are no registers to ask for ahead (eight tokens, 2,048 x 2,048 and a shared unit, 4: 92.0 us, 12: 74.3),
// in float32 ones with more than four tokens, for the same reason (1,600 x 1,600 and a shared unit, 4: 113.6 us, 16: 103.0).
__host__ __device__ constexpr int shared_weight(int kind, int T) {
    const int columns = (T * TERMS + few::COLUMNS - 1) / few::COLUMNS;
    return kind == F32 ? (T == 1 ? 4 : T == 2 ? 5 : T <= 4 ? 8 : 16) : kind == BF16 ? (columns == 1 ? 4 : columns == 2 ? 6 : 12) : columns < 3 ? 4 : 6;
}

// The sums of a part's columns on their way from the instruction's registers to their tokens.
struct Columns { float sum[16][TERMS * MAX_TOKENS + 1]; };

template <int KIND, int W>
__global__ void __launch_bounds__(W * 32, 16 / W)
down_kernel(const __grid_constant__ Call c, const __grid_constant__ Maps maps) {
    using S = Stream<KIND>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ Columns columns[KIND == F32 ? 1 : W];
    __shared__ Plan plan;
    __shared__ Barriers<W> bars;
    constexpr int STAGES = S::MOST_STAGES;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2;
    dd_launch_dependents();
    if (c.l.shared_inner && c.inner_wide) ask_for(c.l.shared_down, matrix_bytes(KIND, c.l.width, c.l.shared_inner));
    bars.init();
    if (threadIdx.x == 0 && c.inner_wide) {
        tc::prefetch_tensormap(&maps.down);
        if (c.l.shared_inner) tc::prefetch_tensormap(&maps.shared_down);
    }
    dd_grid_wait();
    // (all of it at once, used or not)
    for (int i = threadIdx.x; i < (int)(sizeof(Plan) / 4); i += W * 32) reinterpret_cast<uint32_t*>(&plan)[i] = reinterpret_cast<const uint32_t*>(c.plan)[i];
    __syncthreads();
    const int n0 = blockIdx.x * S::ROWS;
    // the result's row and column of this thread, and what the sum is added to
    const int f = threadIdx.x % S::ROWS, t = threadIdx.x / S::ROWS, column = n0 + f;
    const bool live = t < c.T && column < c.l.width;
    float result = live && c.residual ? c.residual[(size_t)t * c.ldr + column] : 0.f;
    if (live && c.l.identity) {
        const size_t at = (size_t)t * c.ldy + column;
        const float y = KIND == F32 ? reinterpret_cast<const float*>(c.y)[at] : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(c.y)[at]);
        result = fmaf(plan.own[t], y, result);
    }
    // the parts' sums: [token][its units in their order][part][row], then [token][the shared unit's part][row]
    float* sums = reinterpret_cast<float*>(smem + W * STAGES * S::STAGE_BYTES);
    const int unit_parts = c.unit_parts, shared_parts = c.shared_parts;
    float* shared_sums = sums + c.T * c.l.top * unit_parts * S::ROWS;
    const int for_shared = c.shares.shared_steps, per_unit = c.shares.unit_steps;
    const int mine = c.shares.template begin<W>(warp + (lane & 1), plan.n_units);
    const int from = __shfl_sync(0xffffffffu, mine, 0), to = __shfl_sync(0xffffffffu, mine, 1);
    // step -> unit (-1: the shared one), its first step and its end
    auto unit_of = [&](int at) { return at < for_shared ? -1 : quotient(at - for_shared, c.shares.by_unit); };
    auto begin_of = [&](int unit) { return unit < 0 ? 0 : for_shared + unit * per_unit; };
    auto matrix_of = [&](int unit) { return unit < 0 ? 0 : (int)(plan.unit[unit].what & 255u); };
    Ring<KIND> ring(bars.full[warp], tc::smem_u32(smem) + warp * STAGES * S::STAGE_BYTES, STAGES);
    int f_at = from, f_begin = 0, f_end = from, f_matrix = 0;
    bool f_shared = false;
    auto fetch = [&] {
        if (f_at >= to) return;
        if (f_at == f_end) {
            const int unit = unit_of(f_at);
            f_shared = unit < 0;
            f_begin = begin_of(unit);
            f_end = begin_of(unit + 1);
            f_matrix = matrix_of(unit);
        }
        if (c.inner_wide && lane == 0)
            ring.ask(f_shared ? &maps.shared_down : &maps.down, f_at - f_begin, n0, f_matrix);
        ring.next_asked();
        ++f_at;
    };
#pragma unroll 1
    for (int i = 0; i < STAGES - 1; ++i) fetch();
    Scales have, soon;
    auto ask_scales = [&](int unit, int at) {     // of a unit, from step `at` on
        const bool shared = unit < 0;
        const int begin = begin_of(unit);
        const int row = matrix_of(unit) * c.l.width + n0, groups = ((shared ? c.l.shared_inner : c.l.inner) + mx4::GROUP - 1) / mx4::GROUP;
        soon.load(reinterpret_cast<const uint32_t*>(shared ? c.l.shared_down_scales : c.l.down_scales), row, row + S::HALF,
                  (size_t)(shared ? 1 : c.l.experts) * c.l.width - 1, groups, (at - begin) * S::SUB, min((min(to, begin_of(unit + 1)) - begin) * S::SUB, groups));
    };
    if (KIND == MX4 && from < to) ask_scales(unit_of(from), from);
    for (int at = from; at < to;) {               // the runs of steps of one unit
        const int unit = unit_of(at), begin = begin_of(unit), end = min(to, begin_of(unit + 1));
        const bool shared = unit < 0;
        const int K = shared ? c.l.shared_inner : c.l.inner, ld = shared ? c.shared_row : c.row;
        const uint32_t users = shared ? (1u << c.T) - 1 : plan.unit[unit].what >> 8, list = list_of(users), slots = shared ? 0u : plan.unit[unit].slots;
        const int n = __popc(users);
        const size_t hidden = (size_t)(shared ? c.max_units : unit) * c.T * c.row, matrix_rows = (size_t)(shared ? 1 : c.l.experts) * c.l.width;
        const void* matrix = shared ? c.l.shared_down : c.l.down;
        const int first_row = matrix_of(unit) * c.l.width + n0;
        // where the sums of part j of token number i of the list go
        auto place_of = [&](int i, int j) {
            const int token = listed(list, i);
            return (shared ? shared_sums + (token * shared_parts + j) * S::ROWS
                           : sums + ((token * c.l.top + (int)(slots >> (4 * token) & 15u)) * unit_parts + j) * S::ROWS);
        };
        // the parts of the run: their length, the first one's number and end
        const int part = shared ? c.l.shared_part : c.l.unit_part, first_j = quotient(at - begin, shared ? c.shares.by_shared_part : c.shares.by_unit_part);
        auto next = [&](int s) {
            const uint32_t place = ring.take(c.inner_wide, &bars.gave_up);
            if (!c.inner_wide) fill_stage<KIND>(place, matrix, first_row, first_row + S::HALF, matrix_rows, K, s - begin);
            return place;
        };
        if constexpr (KIND == F32)
            by_count(n, [&](auto count) {
                constexpr int N = decltype(count)::value;
                const float* x = reinterpret_cast<const float*>(c.hidden) + hidden;
                float4 b[AT_ONCE<N>];             // up to four rows' next step (they come from L2)
                if constexpr (N <= 4) take_rows<N>(b, x, ld, list, at - begin, 0);
                const int which = lane * (few::F32_ROWS * N) / 32;
                const bool owner = owns_sum<N>(n);
                float* own_sum = place_of(owner ? which % N : 0, first_j) + which / N;
                for (int s = at; s < end; own_sum += S::ROWS) {
                    unsigned long long d[few::F32_ROWS][N] = {};
                    for (const int stop = min(s + part, end); s < stop; ++s) {
                        if constexpr (N <= 4) {
                            float4 now[AT_ONCE<N>];
#pragma unroll
                            for (int i = 0; i < AT_ONCE<N>; ++i) now[i] = b[i];
                            if (s + 1 < end) take_rows<N>(b, x, ld, list, s + 1 - begin, 0);
                            fma_rows<N>(next(s), now, 0, d);
                        } else fma_step<N>(next(s), x, ld, list, s - begin, d);
                        __syncwarp();
                        fetch();
                    }
                    const float sum = row_sums<N>(d);
                    if (owner) *own_sum = sum;
                }
            });
        else {
            const __nv_bfloat16* h = reinterpret_cast<const __nv_bfloat16*>(c.hidden) + hidden * TERMS;
            // columns: the terms of the first token of the list, of the second, ...
            auto columns_by = [&](auto count) {
                constexpr int P = decltype(count)::value, Q = PIECES<KIND>;
                // (columns beyond the last term read the first one; nobody looks at them)
                const __nv_bfloat16* x[P];
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    const int q = p * few::COLUMNS + g < n * TERMS ? p * few::COLUMNS + g : 0;
                    x[p] = h + (size_t)(listed(list, q / TERMS) * TERMS + q % TERMS) * ld;
                }
                // pieces of the columns are requested some pieces ahead, as far as there are registers for it
                constexpr int AHEAD = P == 1 ? (KIND == BF16 ? 3 : 1) : KIND == BF16 && P == 2 ? 1 : 0, UN = AHEAD + 1 > S::SUB ? AHEAD + 1 : S::SUB;
                const int first = (at - begin) * S::SUB, pieces = (end - at) * S::SUB;
                int j = first_j, part_end = min(part * S::SUB, pieces);
                float* own_sum = place_of(min(lane & 3, n - 1), 0) + row_of<KIND>(g);         // (P == 1)
                static_assert(TERMS == 3, "a token's terms");
                float d[P][4] = {};
                uint4 b[AHEAD + 1][P][Q];
#pragma unroll
                for (int u = 0; u < AHEAD; ++u)
#pragma unroll
                    for (int p = 0; p < P; ++p) take_column<KIND>(b[u][p], x[p], first + min(u, pieces - 1));
                uint32_t place = 0;
                for (int q = 0; q < pieces; q += UN)
#pragma unroll
                    for (int u = 0; u < UN; ++u) {
                        if (q + u >= pieces) break;
                        if (u % S::SUB == 0) place = next(at + (q + u) / S::SUB);
                        if (q + u + AHEAD < pieces) {
#pragma unroll
                            for (int p = 0; p < P; ++p) take_column<KIND>(b[(u + AHEAD) % (AHEAD + 1)][p], x[p], first + q + u + AHEAD);
                        }
                        uint32_t four0 = 0, four1 = 0;
                        if (KIND == MX4) {
                            const int i = (q + u) % Scales::STRETCH, then = at + (q + u + Scales::STRETCH) / S::SUB;
                            if (i == 0) {         // the next stretch: of this run, or of the next one
                                have = soon;
                                if (then < end) ask_scales(unit, then);
                                else if (end < to) ask_scales(unit + 1, end);
                            }
                            have.get(i, four0, four1);
                        }
                        mma_step<KIND, P>(place, u % S::SUB, four0, four1, b[u % (AHEAD + 1)], d);
                        if (u % S::SUB != S::SUB - 1) continue;
                        __syncwarp();
                        fetch();
                        if (q + u + 1 < part_end) continue;
                        // A part's end: its terms' sums, added up token by token (the tokens that do not use the expert are not touched: zero
                        // times a weight that is not finite is no zero).
                        if constexpr (P == 1) {
                            // lane (g, 0) has a row's first token's first two terms, (g, 1) its third and the second token's first
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const float a = d[0][2 * h], b = d[0][2 * h + 1];
                                const float next_a = __shfl_down_sync(0xffffffffu, a, 1), next_b = __shfl_down_sync(0xffffffffu, b, 1);
                                if ((lane & 3) < n) own_sum[j * S::ROWS + h * S::HALF] = lane & 1 ? b + next_a + next_b : a + b + next_a;
                            }
                        } else {
                            const int row = row_of<KIND>(g);
#pragma unroll
                            for (int p = 0; p < P; ++p)
#pragma unroll
                                for (int i = 0; i < 4; ++i) columns[warp].sum[row + 8 * (i >> 1)][p * few::COLUMNS + 2 * (lane & 3) + (i & 1)] = d[p][i];
                            __syncwarp();
                            for (int i = lane >> 4; i < n; i += 2) {
                                const float* terms = &columns[warp].sum[lane & 15][i * TERMS];
                                place_of(i, j)[lane & 15] = terms[0] + terms[1] + terms[2];
                            }
                            __syncwarp();
                        }
#pragma unroll
                        for (int p = 0; p < P; ++p) d[p][0] = d[p][1] = d[p][2] = d[p][3] = 0.f;
                        ++j;
                        part_end = min(part_end + part * S::SUB, pieces);
                    }
            };
            if (n * TERMS <= few::COLUMNS) columns_by(Count<1>{});
            else if (n * TERMS <= 2 * few::COLUMNS) columns_by(Count<2>{});
            else columns_by(Count<3>{});
        }
        at = end;
    }
    __syncthreads();
    if (bars.gave_up && threadIdx.x == 0) atomicOr(c.error_flag, 8);
    if (!live) return;
    float sum = 0.f;
#pragma unroll 4
    for (int j = 0; j < shared_parts; ++j) sum += shared_sums[(t * shared_parts + j) * S::ROWS + f];
    for (uint32_t used = plan.slots[t]; used; used &= used - 1) {
        const float* from_here = sums + (t * c.l.top + __ffs(used) - 1) * unit_parts * S::ROWS + f;
#pragma unroll 4
        for (int j = 0; j < unit_parts; ++j) sum += from_here[j * S::ROWS];
    }
    c.out[(size_t)t * c.ldo + column] = sum + result;
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Matrices of the layer as TMA boxes of their kind (Stream): a stack of `matrices` of rows x K, boxes of box_rows rows out of box_matrices
// neighbours (a gate's and the up matrix behind it). Rows that are no whole 16-byte pieces have none.
template <int KIND>
int layer_map(CUtensorMap* map, const void* base, long long matrices, long long rows, int K, int box_matrices) {
    using S = Stream<KIND>;
    const long long row_bytes = KIND == MX4 ? (long long)dd_ceil_div(K, mx4::GROUP) * mx4::GROUP_BYTES : (long long)K * S::ELEMENT;
    if (!base || rows <= 0 || row_bytes % 16 || ((uintptr_t)base & 15)) return 0;
    static EncodeTiled enc = nullptr;
    if (!enc) {
        void* sym = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            enc = reinterpret_cast<EncodeTiled>(sym);
    }
    if (!enc) return dd_fail("dd_moe_tokens: cuTensorMapEncodeTiled is not available from this driver");
    // k (of 4-bit rows: bytes), row, matrix
    cuuint64_t dims[3] = {(cuuint64_t)(KIND == MX4 ? row_bytes : K), (cuuint64_t)rows, (cuuint64_t)matrices};
    cuuint64_t strides[2] = {(cuuint64_t)row_bytes, (cuuint64_t)(row_bytes * rows)};
    cuuint32_t box[3] = {(cuuint32_t)(KIND == MX4 ? S::BOX_ROW : S::STEP), (cuuint32_t)(S::ROWS / box_matrices), (cuuint32_t)box_matrices};
    cuuint32_t elem[3] = {1, 1, 1};
    const CUresult r = enc(map, KIND == F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : KIND == BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8,
                           3, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           KIND == F32 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return dd_fail("dd_moe_tokens: cannot describe %lld matrices of %lld x %d to TMA (driver error %d)", matrices, rows, K, (int)r);
    return 0;
}
template <int KIND>
int layer_maps(Maps* m, const DdExpertLayer& l) {
    const int halves = l.gated ? 2 : 1;
    if (int e = layer_map<KIND>(&m->gate_up, l.gate_up, (long long)l.experts * halves, l.inner, l.width, halves)) return e;
    if (int e = layer_map<KIND>(&m->down, l.down, l.experts, l.width, l.inner, 1)) return e;
    if (int e = layer_map<KIND>(&m->shared_gate_up, l.shared_gate_up, 2, l.shared_inner, l.width, 2)) return e;
    return layer_map<KIND>(&m->shared_down, l.shared_down, 1, l.width, l.shared_inner, 1);
}

// Dynamic shared memory of up_kernel, at most: less the static part.
constexpr size_t MOST_SHARED = 227 * 1024 - 32 * 1024;
template <int KIND>
int launch_up(const Call& c, const Maps& m, int blocks, size_t smem, cudaStream_t s) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(blocks);
    config.blockDim = dim3(UP_THREADS);
    config.dynamicSmemBytes = smem;
    config.stream = s;
    cudaLaunchAttribute attrs[2];
    attrs[0].id = cudaLaunchAttributeClusterDimension;
    attrs[0].val.clusterDim.x = c.cluster;
    attrs[0].val.clusterDim.y = 1;
    attrs[0].val.clusterDim.z = 1;
    attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[1].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attrs;
    config.numAttrs = dd_pdl_enabled ? 2 : 1;
    cudaError_t e = dd_allow_shared<up_kernel<KIND>>((int)MOST_SHARED);
    if (e == cudaSuccess) e = cudaLaunchKernelEx(&config, up_kernel<KIND>, c, m);
    if (e != cudaSuccess) return dd_fail("dd_moe_tokens (clusters of %d, %d bytes of shared memory): %s", c.cluster, (int)smem, cudaGetErrorString(e));
    return dd_check_launch("dd_moe_tokens");
}
// What the parts' sums of eight tokens may take of down_kernel's shared memory, so that the blocks of an SM fit beside their rings.
__host__ constexpr int sums_fit(int warps) { return (warps == 16 ? 64 : warps == 8 ? 30 : 14) * 1024; }
template <int KIND> int sums_bytes(const DdExpertLayer& l, int T) {
    return T * (l.top * parts_of<KIND>(l.inner, l.unit_part) + parts_of<KIND>(l.shared_inner, l.shared_part)) * Stream<KIND>::ROWS * 4;
}
// A block a tile; as many warps on it as let all blocks run at once.
template <int KIND> int down_warps(const DdExpertLayer& l, int sms) {
    const int tiles = dd_ceil_div(l.width, Stream<KIND>::ROWS);
    return tiles <= sms ? 16 : tiles <= 2 * sms ? 8 : 4;
}
template <int KIND, int W>
int launch_down(const Call& c, const Maps& m, cudaStream_t s) {
    constexpr int RINGS = W * Stream<KIND>::MOST_STAGES * Stream<KIND>::STAGE_BYTES + 1024;
    const cudaError_t e = dd_allow_shared<down_kernel<KIND, W>>(RINGS + sums_fit(W));
    if (e != cudaSuccess) return dd_fail("dd_moe_tokens: shared memory of %d bytes refused: %s", RINGS + sums_fit(W), cudaGetErrorString(e));
    dd_launch(down_kernel<KIND, W>, dim3(dd_ceil_div(c.l.width, Stream<KIND>::ROWS)), dim3(W * 32), (size_t)(RINGS + sums_bytes<KIND>(c.l, c.T)), s, c, m);
    return dd_check_launch("dd_moe_tokens");
}

// How up_kernel shares its routing and its shared memory out.
struct UpPlan { int tiles, shares, cluster, y_pitch; size_t fixed, stage; };
template <int KIND>
UpPlan plan_up(const DdExpertLayer& l, int T) {
    using S = Stream<KIND>;
    UpPlan u;
    const int outputs = l.experts + l.identity, rows = outputs + l.shared_gate;
    // a router of up to 64 KB is read by every block for itself, a larger one shared by a cluster's blocks
    // (128 outputs and more leave no room for what eight blocks send)
    const size_t router_bytes = l.router ? (size_t)rows * l.width * S::ELEMENT : 0;
    u.tiles = (rows + 15) / 16;
    u.shares = u.tiles >= 9 ? 1 : u.tiles >= 5 ? 2 : u.tiles >= 3 ? 4 : u.tiles == 2 ? 8 : 16;       // warps of which a tile's columns are
    if (KIND == F32) u.shares = u.shares > 4 ? u.shares / 4 : 1;                                       // (four by its rows)
    u.cluster = router_bytes <= (64 << 10) ? 1 : router_bytes <= (256 << 10) || u.tiles > 8 ? 4 : 8;
    const size_t scratch = !l.router ? 0 : sizeof(Tile) * u.tiles * u.shares + sizeof(float) * (u.cluster * u.tiles * 16 * MAX_TOKENS +
                                                                              MAX_TOKENS * (2 * outputs + (l.groups > MAX_TOP ? l.groups : MAX_TOP)));
    u.y_pitch = dd_ceil_div((long long)l.width, S::STEP) * S::STEP * S::ELEMENT + (KIND == MX4 ? 64 : 16);
    u.fixed = scratch + (size_t)T * u.y_pitch * (KIND == MX4 ? 2 : 1) + 1024;
    u.stage = UP_WARPS * S::STAGE_BYTES;
    return u;
}
// up_kernel's tiles, at most, in a call of T tokens: they, and the matrices' rows, are counted in fewer than 32 bits.
int units_of(const DdExpertLayer& l, int T) { return T * l.top < l.experts ? T * l.top : l.experts; }
template <int KIND> long long most_tiles(const DdExpertLayer& l, int T) {
    using S = Stream<KIND>;
    const int features = l.gated ? S::HALF : S::ROWS;
    return (long long)units_of(l, T) * ((l.inner + features - 1) / features) + (l.shared_inner + S::HALF - 1) / S::HALF;
}
template <int KIND> bool counts_fit(const DdExpertLayer& l, int T) {
    return most_tiles<KIND>(l, T) <= (1 << 21) && (long long)l.experts * l.inner * 2 <= INT_MAX && (long long)l.experts * l.width <= INT_MAX;
}
template <int KIND>
int most_tokens(const DdExpertLayer& l) {        // with two stages a ring
    for (int T = MAX_TOKENS; T > 0; --T) {
        const UpPlan u = plan_up<KIND>(l, T);
        if (u.fixed + 2 * u.stage <= MOST_SHARED && counts_fit<KIND>(l, T)) return T;
    }
    return 0;
}

// The blocks of up_kernel that the GPU holds at once, one an SM (a second wave of blocks would double the time): a B200's SMs take 33
// clusters of four, 15 of eight.
int up_blocks(int cluster, int sms) { return sms >= 148 ? (cluster == 1 ? sms : cluster == 4 ? 132 : 120) : sms / 2 / cluster * cluster; }

template <int KIND>
int launch_both(Call& c, const Maps& m, int sms, cudaStream_t s) {
    using S = Stream<KIND>;
    const UpPlan u = plan_up<KIND>(c.l, c.T);
    if (u.fixed + 2 * u.stage > MOST_SHARED)
        return dd_fail("dd_moe_tokens: %d rows of %d elements are more than a block's shared memory holds beside its rings", c.T, c.l.width);
    c.cluster = u.cluster; c.y_pitch = u.y_pitch; c.router_tiles = u.tiles;
    c.share_shift = u.shares == 16 ? 4 : u.shares / 2 - (u.shares == 8);
    c.cluster_shift = u.cluster == 8 ? 3 : u.cluster / 2;
    c.stages = (int)((MOST_SHARED - u.fixed) / u.stage);
    if (c.stages > S::MOST_STAGES) c.stages = S::MOST_STAGES;
    const int most = up_blocks(c.cluster, sms);
    if (!counts_fit<KIND>(c.l, c.T)) return dd_fail("dd_moe_tokens: %d experts of %d x %d are too large", c.l.experts, c.l.inner, c.l.width);
    const long long at_most = most_tiles<KIND>(c.l, c.T);
    const int blocks = at_most < most ? (int)((at_most + c.cluster - 1) / c.cluster * c.cluster) : most;
    if (int e = launch_up<KIND>(c, m, blocks, u.fixed + c.stages * u.stage, s)) return e;
    c.shares = shares_of(c.l, S::STEP, shared_weight(KIND, c.T));
    c.unit_parts = parts_of<KIND>(c.l.inner, c.l.unit_part);
    c.shared_parts = parts_of<KIND>(c.l.shared_inner, c.l.shared_part);
    const int warps = down_warps<KIND>(c.l, sms);
    return warps == 16 ? launch_down<KIND, 16>(c, m, s) : warps == 8 ? launch_down<KIND, 8>(c, m, s) : launch_down<KIND, 4>(c, m, s);
}

// How many parts the sums of a row are cut into, by the layer alone. up_kernel: as few warps on a tile as give at least three eighths of the
// grid's warps one in a step of one token (one token and eight of 1,600 x 1,600, two of sixteen experts and a shared unit: 21.2 and 49.8 us with
// two warps, 24.9 and 51.9 with one, 22.9 and 51.2 with four; one and eight of 64 4-bit experts, eight a token, 27.7 and 80.9 with one, 27.2 and 86.5
// with two). down_kernel: the lengths of parts, of a unit and of the shared unit, that on average leave the warps of a block the least to do
// one after the other in steps of one to eight tokens (with as many experts as so many tokens choose on average), counting what a part costs
// beside its steps: its sums go through shared memory. Of eleven layers timed at 1, 2, 4 and 8 tokens with other lengths the ones taken are
// within 1.5 % of the best on average. (Cut by a step's own work, a token's bits would depend on its neighbours' experts; one token of
// 1,600 x 1,600 24.7 us, now 22.6; eight, 2,048 x 2,048 and a shared unit, 70.0 and 68.4; five of the float32 layer of plain units 49.8 and 50.0.)
template <int KIND>
void choose_parts(DdExpertLayer& l, int sms) {
    using S = Stream<KIND>;
    const int features = l.gated ? S::HALF : S::ROWS, least = l.top < l.experts ? l.top : l.experts;
    const long long tiles = (l.shared_inner + S::HALF - 1) / S::HALF + (long long)least * ((l.inner + features - 1) / features);
    const int warps = up_blocks(plan_up<KIND>(l, 1).cluster, sms) * UP_WARPS, steps = dd_ceil_div(l.width, S::STEP);
    l.up_shift = 0;
    while ((UP_WARPS >> l.up_shift) > 1 && (2 << l.up_shift) <= steps && (tiles << l.up_shift) * 8 < warps * 3) ++l.up_shift;

    const int W = down_warps<KIND>(l, sms), unit_steps = dd_ceil_div(l.inner, S::STEP), shared_steps = dd_ceil_div(l.shared_inner, S::STEP);
    const int beside = KIND == MX4 ? 1 : 2;      // quarters of a step
    double best = 1e30;
    for (int p = 32, last_p = 0; p > 0; --p) {    // (about) that many parts of a unit, q of the shared one
        DdExpertLayer with = l;
        with.unit_part = dd_ceil_div(unit_steps, p);
        if (with.unit_part == last_p) continue;
        last_p = with.unit_part;
        for (int q = shared_steps ? 32 : 1, last_q = 0; q > 0; --q) {
            with.shared_part = shared_steps ? dd_ceil_div(shared_steps, q) : 1;
            if (with.shared_part == last_q) continue;
            last_q = with.shared_part;
            if (p + q > 2 && sums_bytes<KIND>(with, MAX_TOKENS) > sums_fit(W)) continue;
            double cost = 0.0, left_out = 1.0;
            for (int T = 1; T <= MAX_TOKENS; ++T) {
                left_out *= 1.0 - (double)least / l.experts;
                const int most_units = (int)(l.experts * (1.0 - left_out) + 0.5), units = most_units > least ? most_units : least;
                const Shares shares = shares_of(with, S::STEP, shared_weight(KIND, T));
                auto begin = [&](int w) { return W == 16 ? shares.begin<16>(w, units) : W == 8 ? shares.begin<8>(w, units) : shares.begin<4>(w, units); };
                int most = 0;
                for (int w = 0, from = 0, to; w < W; ++w, from = to) {
                    to = begin(w + 1);
                    const int of_shared = (to < shared_steps ? to : shared_steps) - (from < shared_steps ? from : shared_steps), of_units = to - from - of_shared;
                    const int parts = dd_ceil_div(of_shared, with.shared_part) + dd_ceil_div(of_units, with.unit_part);
                    const int work = of_shared * shares.weight + of_units * 4 + parts * beside;
                    if (work > most) most = work;
                }
                cost += (double)most * W / (shared_steps * shares.weight + units * unit_steps * 4);
            }
            if (cost < best - 1e-9) {
                best = cost;
                l.unit_part = with.unit_part;
                l.shared_part = with.shared_part;
            }
        }
    }
}

int hidden_row(int kind, int inner) { return (inner + step_of(kind) - 1) / step_of(kind) * step_of(kind); }
size_t hidden_bytes(const DdExpertLayer& l, int T, int max_units) {
    return (size_t)T * (l.kind == F32 ? 4 : 2 * TERMS) * ((size_t)max_units * hidden_row(l.kind, l.inner) + hidden_row(l.kind, l.shared_inner));
}
}  // namespace

// Bytes of scratch that a call of T tokens needs (16-byte aligned).
DD_API long long dd_moe_tokens_scratch(const DdExpertLayer* l, int T) {
    return (long long)(sizeof(Plan) + hidden_bytes(*l, T, units_of(*l, T)));
}
// The most tokens that a call with this layer can take (its rows have to fit into shared memory beside the rings, its tiles to be
// counted); 0: the layer is for the kernels of larger steps.
DD_API int dd_moe_tokens_most(const DdExpertLayer* l) {
    return l->kind == F32 ? most_tokens<F32>(*l) : l->kind == BF16 ? most_tokens<BF16>(*l) : most_tokens<MX4>(*l);
}
// Before a layer's first call: chooses its parts, and writes the matrices as TMA takes them: 512 bytes, 64-byte aligned, which every call
// copies. They hold while the matrices lie where they are.
DD_API int dd_moe_tokens_prepare(DdExpertLayer* l, void* maps, int sms) {
    static_assert(sizeof(Maps) == 512, "four tensor maps");
    Maps* m = (Maps*)maps;
    if (l->width <= 0 || l->inner <= 0 || l->experts <= 0 || l->top <= 0 || sms <= 0)
        return dd_fail("dd_moe_tokens: %d of %d experts of %d x %d on %d SMs", l->top, l->experts, l->inner, l->width, sms);
    if (l->kind == F32) choose_parts<F32>(*l, sms);
    else if (l->kind == BF16) choose_parts<BF16>(*l, sms);
    else choose_parts<MX4>(*l, sms);
    return l->kind == F32 ? layer_maps<F32>(m, *l) : l->kind == BF16 ? layer_maps<BF16>(m, *l) : layer_maps<MX4>(m, *l);
}

// y [T, ldy] (float32 or bfloat16, by the layer's kind), residual [T, ldr] float32 or null, out [T, ldo] float32 (may be
// residual), ids [T] with a table. An expert or a token id out of range sets error bit 1 and is left out.
DD_API int dd_moe_tokens(const DdExpertLayer* l, const void* maps, const void* y, int ldy, const float* residual, int ldr, float* out, int ldo,
                         const int* ids, int T, void* scratch, int sms, int* error_flag, void* stream) {
    if (T <= 0) return 0;
    const int outputs = l->experts + l->identity;
    if (T > MAX_TOKENS || l->top <= 0 || l->top > MAX_TOP || l->experts <= 0 || outputs + l->shared_gate > MAX_OUTPUTS || l->top > outputs)
        return dd_fail("dd_moe_tokens: %d tokens (at most %d), %d of %d experts (at most %d of %d)", T, MAX_TOKENS, l->top, outputs, MAX_TOP,
                       MAX_OUTPUTS);
    if (l->kind == MX4) {
        const void* codes[4] = {l->gate_up, l->down, l->shared_gate_up, l->shared_down};
        const void* scales[4] = {l->gate_up_scales, l->down_scales, l->shared_gate_up_scales, l->shared_down_scales};
        for (int i = 0; i < 4; ++i)
            if (((uintptr_t)codes[i] & 15) || ((uintptr_t)scales[i] & 3)) return dd_fail("dd_moe_tokens: 4-bit matrices must be 16-byte aligned");
    }
    if (l->up_shift < 0 || l->unit_part <= 0 || l->shared_part <= 0)
        return dd_fail("dd_moe_tokens: the layer has not been prepared");
    if (!l->router == !l->table || (l->table && !ids)) return dd_fail("dd_moe_tokens: a router, or a table with token ids");
    if (l->groups <= 0 || outputs % l->groups || l->keep <= 0 || l->keep > l->groups || l->width <= 0 || l->inner <= 0)
        return dd_fail("dd_moe_tokens: %d experts in %d groups of which %d stay, width %d, inner %d", outputs, l->groups, l->keep, l->width, l->inner);
    Call c;
    c.l = *l; c.y = y; c.residual = residual; c.out = out; c.ids = ids; c.error_flag = error_flag; c.T = T; c.ldy = ldy; c.ldr = ldr; c.ldo = ldo;
    c.max_units = units_of(*l, T);
    c.row = hidden_row(l->kind, l->inner); c.shared_row = hidden_row(l->kind, l->shared_inner);
    c.plan = (Plan*)scratch;
    c.hidden = (uint8_t*)scratch + sizeof(Plan);
    const int piece = l->kind == F32 ? 4 : 8;
    auto aligned = [](const void* p) { return !((uintptr_t)p & 15); };
    const bool four = l->kind == MX4;            // (whose rows always are whole pieces)
    c.router_wide = l->width % piece == 0 && aligned(l->router) && l->router_stride % piece == 0;
    c.w_wide = four || (l->width % piece == 0 && aligned(l->gate_up) && aligned(l->shared_gate_up));
    c.inner_wide = four || (l->inner % piece == 0 && l->shared_inner % piece == 0 && aligned(l->down) && aligned(l->shared_down));
    c.y_wide = l->width % piece == 0 && ldy % piece == 0 && aligned(y);
    cudaStream_t s = (cudaStream_t)stream;
    const Maps& m = *(const Maps*)maps;
    if (l->kind == BF16) return launch_both<BF16>(c, m, sms, s);
    if (l->kind == MX4) return launch_both<MX4>(c, m, sms, s);
    if (l->kind == F32) return launch_both<F32>(c, m, sms, s);
    return dd_fail("dd_moe_tokens: unknown kind %d", l->kind);
}
