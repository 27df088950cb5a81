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
