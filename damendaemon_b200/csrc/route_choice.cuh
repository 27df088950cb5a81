// A token's experts from its router's logits: what the routing kernel (moe.cu) and the expert layers for a few tokens
// (moe_tokens.cu) share.
#pragma once
#include "common.cuh"

// Logit z of expert e of a router without softmax: what a chosen expert weighs, and what the choice looks at.
__device__ __forceinline__ void dd_sigmoid_score(float z, int e, const float* correction, int groups, float* value, float* score) {
    const float s = 1.0f / (1.0f + expf(-z));
    value[e] = s;
    // where nothing is added to the scores the logits choose: their order is the scores', which run together near one
    score[e] = correction ? s + correction[e] : (groups > 1 ? s : z);
}

// One warp, one token. value: the experts' weights (softmax: their logits, which become scores here), score: what the choice
// looks at (softmax: written here), worth: [groups] scratch; all in shared memory. The worthiest runs and then the best experts by
// repeated arg-max over the warp, the lowest index winning a tie; -1 where fewer were eligible.
__device__ __forceinline__ void dd_choose_experts(float* score, float* value, float* worth, int n_experts, int top, int groups, int keep,
                                                  float weight_scale, int softmax, const float* correction, int renormalize, int* chosen,
                                                  float* pair_weight) {
    const int lane = threadIdx.x & 31;
    constexpr float NONE = -3.0e38f;             // below every score: struck out
    if (softmax) {
        float top_z = NONE, total = 0.f;
        for (int e = lane; e < n_experts; e += 32) top_z = fmaxf(top_z, value[e]);
        top_z = dd_warp_max(top_z);
        for (int e = lane; e < n_experts; e += 32) total += expf(value[e] - top_z);
        total = dd_warp_sum(total);
        for (int e = lane; e < n_experts; e += 32) {
            const float s = expf(value[e] - top_z) / total;
            value[e] = s;
            score[e] = correction ? s + correction[e] : s;
        }
        __syncwarp();
    }
    const int per = n_experts / groups;
    if (groups > 1) {
        for (int g = lane; g < groups; g += 32) {
            float best = NONE, second = NONE;
            for (int i = 0; i < per; ++i) {
                const float s = score[g * per + i];
                if (s > best) { second = best; best = s; }
                else if (s > second) second = s;
            }
            worth[g] = best + (per > 1 ? second : 0.f);
        }
        __syncwarp();
        // keep the worthiest runs: the others' scores are struck out
        // (a kept run's worth becomes infinite and is passed over from then on)
        for (int round = 0; round < keep; ++round) {
            float best = -INFINITY;
            int at = 0x7fffffff;
            for (int g = lane; g < groups; g += 32)
                if (worth[g] > best && worth[g] < INFINITY) { best = worth[g]; at = g; }
            for (int o = 16; o > 0; o >>= 1) {
                const float ob = __shfl_xor_sync(0xffffffffu, best, o);
                const int oa = __shfl_xor_sync(0xffffffffu, at, o);
                if (ob > best || (ob == best && oa < at)) { best = ob; at = oa; }
            }
            if (lane == 0 && at < groups) worth[at] = INFINITY;     // marked as kept
            __syncwarp();
        }
        for (int e = lane; e < n_experts; e += 32)
            if (worth[e / per] != INFINITY) score[e] = NONE;
        __syncwarp();
    }
    float sum = 0.f;                             // of the chosen scores, in the order of the choice (lane 0)
    for (int k = 0; k < top; ++k) {
        float best = NONE;
        int at = 0x7fffffff;
        for (int e = lane; e < n_experts; e += 32)
            if (score[e] > best) { best = score[e]; at = e; }
        for (int o = 16; o > 0; o >>= 1) {
            const float ob = __shfl_xor_sync(0xffffffffu, best, o);
            const int oa = __shfl_xor_sync(0xffffffffu, at, o);
            if (ob > best || (ob == best && oa < at)) { best = ob; at = oa; }
        }
        if (lane == 0) {
            chosen[k] = at < n_experts ? at : -1;
            const float s = at < n_experts ? value[at] : 0.f;
            pair_weight[k] = s * weight_scale;
            sum += s;
            if (at < n_experts) score[at] = NONE;
        }
        __syncwarp();
    }
    if (renormalize && lane == 0)
        for (int k = 0; k < top; ++k) pair_weight[k] /= sum + 1e-20f;
}

// float32 -> uint32 that orders like the floats (both zeros alike); 0: struck out, below every score, or no number.
__device__ __forceinline__ uint32_t dd_score_key(float score) {
    if (!(score > -3.0e38f)) return 0u;
    const uint32_t u = __float_as_uint(score + 0.0f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
// The largest key of the warp and the lowest index that has it; lane l holds keys of indices l, l + 32, ...
template <int N>
__device__ __forceinline__ uint32_t dd_best_key(const uint32_t* key, int* at) {
    const int lane = threadIdx.x & 31;
    uint32_t best = key[0];
#pragma unroll
    for (int i = 1; i < N; ++i) best = max(best, key[i]);
    best = __reduce_max_sync(0xffffffffu, best);
    uint32_t first = 0x7fffffffu;
#pragma unroll
    for (int i = N - 1; i >= 0; --i)
        if (key[i] == best) first = lane + 32 * i;
    *at = (int)__reduce_min_sync(0xffffffffu, first);
    return best;
}
// dd_choose_experts for at most 32 N experts: the same choice and the same weights, with the scores in registers (two of sixteen in
// 0.7 us). worth: max(groups, top) numbers of scratch.
template <int N>
__device__ __forceinline__ void dd_choose_few(float* score, float* value, float* worth, int n_experts, int top, int groups, int keep, float weight_scale,
                                              int softmax, const float* correction, int renormalize, int* chosen, float* pair_weight) {
    const int lane = threadIdx.x & 31;
    float s[N];
    if (softmax) {
        float top_z = -3.0e38f, total = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) top_z = fmaxf(top_z, lane + 32 * i < n_experts ? value[lane + 32 * i] : -3.0e38f);
        top_z = dd_warp_max(top_z);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            s[i] = lane + 32 * i < n_experts ? expf(value[lane + 32 * i] - top_z) : 0.f;
            total += s[i];
        }
        total = dd_warp_sum(total);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int e = lane + 32 * i;
            if (e >= n_experts) continue;
            s[i] = s[i] / total;
            value[e] = s[i];
            if (correction) s[i] += correction[e];
            if (groups > 1) score[e] = s[i];
        }
        __syncwarp();
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = lane + 32 * i < n_experts ? score[lane + 32 * i] : 0.f;
    }
    uint32_t key[N];
#pragma unroll
    for (int i = 0; i < N; ++i) key[i] = lane + 32 * i < n_experts ? dd_score_key(s[i]) : 0u;
    if (groups > 1) {
        const int per = n_experts / groups;
        uint32_t run[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int g = lane + 32 * i;
            run[i] = 0u;
            if (g >= groups) continue;
            float best = -3.0e38f, second = -3.0e38f;
#pragma unroll 1
            for (int j = 0; j < per; ++j) {
                const float v = score[g * per + j];
                if (v > best) { second = best; best = v; }
                else if (v > second) second = v;
            }
            run[i] = max(dd_score_key(best + (per > 1 ? second : 0.f)), 1u);
            worth[g] = 0.f;
        }
        __syncwarp();
        for (int round = 0; round < keep; ++round) {
            int at;
            const uint32_t best = dd_best_key<N>(run, &at);
            if (best == 0u) break;
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (lane + 32 * i == at) { run[i] = 0u; worth[at] = 1.f; }
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (lane + 32 * i < n_experts && worth[(lane + 32 * i) / per] == 0.f) key[i] = 0u;
    }
    float sum = 0.f;                             // of the chosen scores, in the order of the choice
    if (N <= 2) {
        // an expert's place is the number of better ones: no reduction waits for the one before it
        int place[N] = {};
#pragma unroll 4
        for (int from = 0; from < min(32, n_experts); ++from)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const uint32_t other = __shfl_sync(0xffffffffu, key[j], from);
                const int at = from + 32 * j;
#pragma unroll
                for (int i = 0; i < N; ++i) place[i] += other > key[i] || (other == key[i] && at < lane + 32 * i);
            }
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (place[i] < top) {                // (there may be fewer eligible ones than places)
                chosen[place[i]] = key[i] ? lane + 32 * i : -1;
                pair_weight[place[i]] = key[i] ? value[lane + 32 * i] * weight_scale : 0.f;
                worth[place[i]] = key[i] ? value[lane + 32 * i] : 0.f;
            }
        __syncwarp();
        if (renormalize && lane == 0)
#pragma unroll 1
            for (int k = 0; k < top; ++k) sum += worth[k];
    } else
        for (int k = 0; k < top; ++k) {
            int at;
            const uint32_t best = dd_best_key<N>(key, &at);
            const float v = best ? value[at] : 0.f;
            if (lane == 0) {
                chosen[k] = best ? at : -1;
                pair_weight[k] = v * weight_scale;
            }
            sum += v;
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (best && lane + 32 * i == at) key[i] = 0u;
        }
    if (renormalize && lane == 0)
        for (int k = 0; k < top; ++k) pair_weight[k] /= sum + 1e-20f;
}
