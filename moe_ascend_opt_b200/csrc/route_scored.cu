// Routing to experts by scores (moe_route_scored, include/moe_b200.h): softmax or sigmoid
// scores, a balance bias, expert groups, top-k, renormalised and scaled weights.
#include <cmath>

#include "common.cuh"
#include "status.h"

using namespace moe;

namespace {

constexpr int kRouteWarps = 4;
constexpr int kRouteMaxTopk = 32, kRouteMaxGroups = 32, kRouteMaxExperts = 1024;

struct RouteScoredParams {
    const void* logits;
    const float* bias;
    int64_t T;
    int E, K, dtype, score, groups, topk_groups, group_top, renorm;
    float scale;
    int32_t* ids;
    float* w;
};

MOE_DEV float load_logit(const void* p, int64_t i, int dtype) {
    return dtype == MOE_F32 ? reinterpret_cast<const float*>(p)[i] : act_to_f32(p, i, dtype == MOE_BF16);
}

// The largest value over the warp, ties to the lower index; index 0x7fffffff means none.
MOE_DEV void warp_argmax(double& v, int& i) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const double ov = __shfl_xor_sync(0xffffffffu, v, o);
        const int oi = __shfl_xor_sync(0xffffffffu, i, o);
        if (ov > v || (ov == v && oi < i)) { v = ov; i = oi; }
    }
}

// One warp per token; lane l holds experts l, l + 32, ...  The order of the scores is formed
// in 64 bits (near ties of 32-bit scores would depend on the rounding of exp), or, without a
// bias, by the logits themselves, which have the scores' order exactly.
template <int NPL>
__global__ void __launch_bounds__(kRouteWarps * 32) route_scored_kernel(const RouteScoredParams p) {
    const int64_t t = (int64_t)blockIdx.x * kRouteWarps + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (t >= p.T) return;
    const int E = p.E, per = E / p.groups;
    const int64_t base = t * E;
    float l[NPL];
    bool any = false;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
        const int e = i * 32 + lane;
        l[i] = e < E ? load_logit(p.logits, base + e, p.dtype) : -INFINITY;
        if (!(l[i] > -INFINITY)) l[i] = -INFINITY;  // NaN: masked
        l[i] = fminf(l[i], 3.402823466e38f);
        top = fmaxf(top, l[i]);
        any |= l[i] > -INFINITY;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    // softmax denominator
    double den = 1.0;
    if (p.score == MOE_SCORE_SOFTMAX && (p.bias || !p.renorm || (p.groups > 1 && p.group_top > 1))) {
        den = 0.0;
#pragma unroll
        for (int i = 0; i < NPL; ++i)
            if (l[i] > -INFINITY) den += exp((double)l[i] - (double)top);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) den += __shfl_xor_sync(0xffffffffu, den, o);
    }
    auto score_of = [&](float v) -> double {
        return p.score == MOE_SCORE_SIGMOID ? 1.0 / (1.0 + exp(-(double)v)) : exp((double)v - (double)top) / den;
    };
    // what experts are chosen by (key) and what a group's sum is made of (part)
    double key[NPL];
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
        const int e = i * 32 + lane;
        key[i] = -INFINITY;
        if (l[i] > -INFINITY) {
            key[i] = (double)l[i];
            if (p.bias) {
                const float b = p.bias[e];  // -infinity or NaN: never chosen
                key[i] = b > -INFINITY ? score_of(l[i]) + (double)fminf(b, 3.402823466e38f) : -INFINITY;
            }
        }
    }
    if (p.groups > 1) {
        double total = -INFINITY;  // of group `lane`
        for (int g = 0; g < p.groups; ++g) {
            double sum = -INFINITY;
            int taken = 0x7fffffff;
            for (int r = 0; r < p.group_top; ++r) {
                double bv = -INFINITY;
                int bi = 0x7fffffff;
#pragma unroll
                for (int i = 0; i < NPL; ++i) {
                    const int e = i * 32 + lane;
                    if (e / per == g && e != taken && key[i] > bv) { bv = key[i]; bi = e; }
                }
                warp_argmax(bv, bi);
                if (bi == 0x7fffffff) break;
                taken = bi;
                if (!p.bias && p.group_top > 1) bv = score_of((float)bv);
                sum = r == 0 ? bv : sum + bv;
            }
            if (lane == g) total = sum;
        }
        uint32_t keep = 0;
        for (int r = 0; r < p.topk_groups; ++r) {
            double bv = (lane < p.groups && !((keep >> lane) & 1u)) ? total : -INFINITY;
            int bi = bv > -INFINITY ? lane : 0x7fffffff;
            warp_argmax(bv, bi);
            if (bi == 0x7fffffff) break;
            keep |= 1u << bi;
        }
#pragma unroll
        for (int i = 0; i < NPL; ++i) {
            const int e = i * 32 + lane;
            if (e >= E || !((keep >> (e / per)) & 1u)) key[i] = -INFINITY;
        }
    }
    int mine = -1;  // lane k: the k-th choice
    for (int k = 0; k < p.K; ++k) {
        double bv = -INFINITY;
        int bi = 0x7fffffff;
#pragma unroll
        for (int i = 0; i < NPL; ++i)
            if (key[i] > bv) { bv = key[i]; bi = i * 32 + lane; }
        warp_argmax(bv, bi);
        if (bi == 0x7fffffff) break;  // nothing is left: id -1, weight 0
        if (lane == k) mine = bi;
#pragma unroll
        for (int i = 0; i < NPL; ++i)
            if (i * 32 + lane == bi) key[i] = -INFINITY;
    }
    double s = 0.0;
    if (mine >= 0) s = score_of(fminf(load_logit(p.logits, base + mine, p.dtype), 3.402823466e38f));
    if (p.renorm) {
        double sum = s;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        s = s / (sum + 1e-20);
    }
    if (lane < p.K) {
        p.ids[t * p.K + lane] = mine;
        p.w[t * p.K + lane] = (float)(s * (double)p.scale);
    }
}

}  // namespace

extern "C" int moe_route_scored(const void* logits, int32_t dtype, const float* bias, int64_t T, int64_t E, int64_t K,
                                int32_t score, int64_t num_groups, int64_t topk_groups, int32_t group_top,
                                int32_t renormalize, float scale, int32_t* ids, float* w, void* stream) {
    if (dtype != MOE_F16 && dtype != MOE_BF16 && dtype != MOE_F32)
        return fail(MOE_ERR_INVALID, "logits must be f16, bf16 or f32");
    if (T < 0 || T > (int64_t)1 << 31) return fail(MOE_ERR_INVALID, "num_tokens must be in [0, 2^31]");
    if (E <= 0 || E > kRouteMaxExperts) return fail(MOE_ERR_INVALID, "need 1 <= num_experts <= 1024");
    if (score != MOE_SCORE_SOFTMAX && score != MOE_SCORE_SIGMOID)
        return fail(MOE_ERR_INVALID, "score must be 0 (softmax) or 1 (sigmoid)");
    if (num_groups <= 0 || num_groups > kRouteMaxGroups || E % num_groups != 0)
        return fail(MOE_ERR_INVALID, "num_groups must be in [1, 32] and divide num_experts");
    if (topk_groups <= 0 || topk_groups > num_groups)
        return fail(MOE_ERR_INVALID, "need 1 <= topk_groups <= num_groups");
    if (group_top != 1 && group_top != 2) return fail(MOE_ERR_INVALID, "group_top must be 1 or 2");
    if (K <= 0 || K > kRouteMaxTopk || K > topk_groups * (E / num_groups))
        return fail(MOE_ERR_INVALID, "need 1 <= top_k <= min(32, the experts of topk_groups groups)");
    if (!std::isfinite(scale)) return fail(MOE_ERR_INVALID, "scale must be finite");
    if (T == 0) return MOE_OK;
    if (!logits || !ids || !w) return fail(MOE_ERR_INVALID, "null pointer");
    RouteScoredParams p{logits, bias, T, (int)E, (int)K, dtype, score, (int)num_groups, (int)topk_groups,
                        group_top, renormalize, scale, ids, w};
    const unsigned grid = (unsigned)((T + kRouteWarps - 1) / kRouteWarps);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int npl = (int)((E + 31) / 32);
    if (npl <= 2) route_scored_kernel<2><<<grid, kRouteWarps * 32, 0, st>>>(p);
    else if (npl <= 4) route_scored_kernel<4><<<grid, kRouteWarps * 32, 0, st>>>(p);
    else if (npl <= 8) route_scored_kernel<8><<<grid, kRouteWarps * 32, 0, st>>>(p);
    else if (npl <= 16) route_scored_kernel<16><<<grid, kRouteWarps * 32, 0, st>>>(p);
    else route_scored_kernel<32><<<grid, kRouteWarps * 32, 0, st>>>(p);
    CUDA_TRY(cudaGetLastError());
    return MOE_OK;
}
