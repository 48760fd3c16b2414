// Routing to experts by scores (moe_route_scored, include/moe_b200.h): softmax or sigmoid
// scores, a balance bias, expert groups, top-k, renormalised and scaled weights.
#include <cmath>

#include "common.cuh"
#include "status.h"

using namespace moe;

namespace {

constexpr int kRouteWarps = 4;
constexpr float kMostFloat = 3.402823466e38f;
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

// A row by the definition in 64 bits; lane l holds experts l, l + 32, ...  For rows whose order
// 32 bits do not settle, and for group sizes that the kernel below has no lane layout for.
template <int NPL>
__device__ __noinline__ void route_row_exact(const RouteScoredParams& p, int64_t t) {
    const int lane = threadIdx.x & 31;
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
        l[i] = fminf(l[i], kMostFloat);
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
                key[i] = b > -INFINITY ? score_of(l[i]) + (double)fminf(b, kMostFloat) : -INFINITY;
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
    if (mine >= 0) s = score_of(fminf(load_logit(p.logits, base + mine, p.dtype), kMostFloat));
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


// Floats as unsigned integers of the same order; 0 is below all of them.  -0 falls below +0: callers have none.
MOE_DEV uint32_t ordered(float v) {
    const uint32_t b = __float_as_uint(v);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
MOE_DEV float unordered(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// Whether approximate choices a >= b are in this order for certain: scores off by less than tol / 2,
// sums with the bias by 6e-8 of themselves, keys without their lowest bits by `cut` of themselves.
MOE_DEV bool apart(float a, float b, float tol, float cut) {
    return a - b > tol + (2.4e-7f + cut) * fmaxf(fabsf(a), fabsf(b));
}

// Descending order of N (a power of two) keys: Batcher's odd-even merge sort.
template <int N>
MOE_DEV void sort_keys(uint32_t (&k)[N]) {
#pragma unroll
    for (int p = 1; p < N; p *= 2)
#pragma unroll
        for (int q = p; q >= 1; q /= 2)
#pragma unroll
            for (int j = q % p; j + q < N; j += 2 * q)
#pragma unroll
                for (int i = 0; i < q; ++i)
                    if (i + j + q < N && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
                        const uint32_t a = k[i + j], b = k[i + j + q];
                        k[i + j] = max(a, b);
                        k[i + j + q] = min(a, b);
                    }
}

// One warp per token, lane l holding the NPL neighbouring experts from l * NPL on (wide loads; the
// lower lane is the lower index, so that a ballot breaks ties).  An expert's key is its choice as a
// 32-bit integer of the same order, the lowest log2(NPL) bits replaced by its place in the lane.
// Each lane sorts its keys once; a round of the top-k is then redux.sync over the lanes' heads, a
// ballot for the owner, and the owner's step to its next.  Two rounds more than top_k show
// whether the order is certain: neighbouring choices that the keys do not settle (scores are 32-bit
// approximations, keys lack their last bits) are compared exactly by two lanes, groups at the border of the
// kept ones by their lanes' exact pairs, and what that does not settle (three in a row, a softmax with a
// bias) goes to route_row_exact.  Of 256 sigmoid scores with a bias about two rows in a hundred have such a
// pair.  Without a bias the logits decide, which have the scores' order; 16-bit ones lose nothing in the keys.
//
// Bound: the instructions, 1,040 a row of 256 experts with sigmoid, bias and groups, issued at 71 % (the rounds are
// a serial chain, 7 warps a scheduler): 16384 such rows take 22.5 us (their 9.4 MB would take 1.5 us).  All groups settled exactly where any was at the border, and
// one kernel for all types, took 31 us.
template <int NPL, int DT, bool sigmoid>
__global__ void __launch_bounds__(kRouteWarps * 32) route_scored_kernel(const __grid_constant__ RouteScoredParams p) {
    constexpr uint32_t kPlace = NPL - 1;
    constexpr float kCut = NPL * 1.2e-7f;
    const int64_t t = (int64_t)blockIdx.x * kRouteWarps + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (t >= p.T) return;
    const int E = p.E, per = E / p.groups, e0 = lane * NPL;
    const int64_t base = t * E;
    float l[NPL];
    constexpr int esz = DT == MOE_F32 ? 4 : 2;
    const bool wide = NPL >= 4 && E % 4 == 0;
    if (wide && (reinterpret_cast<uintptr_t>(p.logits) & 15) == 0) {
#pragma unroll
        for (int i = 0; i < NPL; i += 4) {
            float v[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            if (e0 + i < E) {
                const uint8_t* q = static_cast<const uint8_t*>(p.logits) + (base + e0 + i) * esz;
                if (DT == MOE_F32) {
                    const float4 a = __ldg(reinterpret_cast<const float4*>(q));
                    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
                } else {
                    const uint2 a = __ldg(reinterpret_cast<const uint2*>(q));
                    const uint32_t w[2] = {a.x, a.y};
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[j] = scale_to_f32((uint16_t)(w[j / 2] >> (16 * (j & 1))), DT == MOE_BF16);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) l[(i + j) % NPL] = v[j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < NPL; ++i) l[i] = e0 + i < E ? load_logit(p.logits, base + e0 + i, DT) : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < NPL; ++i) l[i] = l[i] > -INFINITY ? fminf(l[i] + 0.f, kMostFloat) : -INFINITY;  // NaN: masked; -0 is 0
    const bool sums = p.groups > 1 && p.group_top > 1, scored = p.bias || sums;
    float top = 0.f, den = 1.f;
    if (!sigmoid) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < NPL; ++i) m = max(m, l[i] > -INFINITY ? ordered(l[i]) : 0u);
        m = __reduce_max_sync(0xffffffffu, m);
        top = m ? unordered(m) : 0.f;
        if (scored || !p.renorm) {
            den = 0.f;
#pragma unroll
            for (int i = 0; i < NPL; ++i) den += l[i] > -INFINITY ? expf(l[i] - top) : 0.f;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) den += __shfl_xor_sync(0xffffffffu, den, o);
        }
    }
    // keys of the choices; with `sums` and no bias the scores first, for the groups
    uint32_t key[NPL];
    float tol = 0.f;
    if (scored) {
        const float r = 1.f / den;
        float most = 0.f;  // largest score
        float bias[NPL];
        if (!p.bias) {
#pragma unroll
            for (int i = 0; i < NPL; ++i) bias[i] = 0.f;
        } else if (wide && (reinterpret_cast<uintptr_t>(p.bias) & 15) == 0) {
#pragma unroll
            for (int i = 0; i < NPL; i += 4) {
                const float4 a = e0 + i < E ? __ldg(reinterpret_cast<const float4*>(p.bias + e0 + i)) : make_float4(0.f, 0.f, 0.f, 0.f);
                bias[i % NPL] = a.x; bias[(i + 1) % NPL] = a.y; bias[(i + 2) % NPL] = a.z; bias[(i + 3) % NPL] = a.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < NPL; ++i) bias[i] = e0 + i < E ? __ldg(p.bias + e0 + i) : 0.f;
        }
#pragma unroll
        for (int i = 0; i < NPL; ++i) {
            // exp's result loses 2.4e-7 of e, its argument's rounding more where that is large; the reciprocal 1.2e-7 of s
            float s, e;
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"((sigmoid ? -l[i] : l[i] - top) * 1.44269504f));
            if (sigmoid) asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.f + e));
            else s = e * r;
            const bool live = l[i] > -INFINITY && bias[i] > -INFINITY;  // a bias of -infinity or NaN: never chosen
            most = fmaxf(most, live ? s : 0.f);
            key[i] = live ? (ordered(fminf(s + fminf(bias[i], kMostFloat), kMostFloat)) & ~kPlace) | (kPlace - i) : 0u;
        }
        most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
        // what two scores may be off by, of the largest: 2 x 4.2e-7 and the argument's rounding, 7.3e-8 |l| of a score
        // (softmax, of a difference: 1.33e-7), for the largest at most -log(most) times that and for smaller ones no
        // more; a softmax's sum adds 6e-8 a term of its lane and 7.4e-7.  Below 1e-30, where approximations
        // become zero, nothing is certain.
        constexpr float base = sigmoid ? 1.4e-6f : 1.9e-6f + NPL * 6e-8f, slope = sigmoid ? 1.5e-7f : 2.7e-7f;
        tol = most > 1e-30f ? most * (base - slope * __logf(most)) : INFINITY;
    } else {
#pragma unroll
        for (int i = 0; i < NPL; ++i) key[i] = l[i] > -INFINITY ? (ordered(l[i]) & ~kPlace) | (kPlace - i) : 0u;
    }
    sort_keys(key);
    bool settled = true;
    const bool exact_keys = !p.bias && DT != MOE_F32;  // of the logits
    if (p.groups > 1) {
        // a lane's experts are of one group, which is held by 2^n neighbouring lanes
        const int lanes = per / NPL;
        uint32_t a = key[0], b = NPL > 1 ? key[NPL > 1] : 0u;  // the group's two largest
        for (int o = 1; o < lanes; o <<= 1) {
            const uint32_t oa = __shfl_xor_sync(0xffffffffu, a, o), ob = __shfl_xor_sync(0xffffffffu, b, o);
            b = max(max(b, ob), min(a, oa));
            a = max(a, oa);
        }
        uint32_t total = a & ~kPlace;  // in every lane of the group
        if (sums && a && b) total = ordered(unordered(a & ~kPlace) + unordered(b & ~kPlace));
        if (e0 >= E) total = 0;
        // rank of this lane's group among the groups (0 the best), ties to the lower index
        const int group = lane / lanes;
        int rank = 0;
        for (int d = 1; d < p.groups; ++d) {
            const int other = group + d < p.groups ? group + d : group + d - p.groups;
            const uint32_t t2 = __shfl_sync(0xffffffffu, total, (other * lanes) & 31);
            rank += t2 > total || (t2 == total && other < group);
        }
        bool kept = total && rank < p.topk_groups;
        if ((scored || !exact_keys) && p.topk_groups < p.groups) {
            // the last group that is kept and the first that is left out
            const uint32_t in = __ballot_sync(0xffffffffu, rank == p.topk_groups - 1 && e0 < E);
            const uint32_t out = __ballot_sync(0xffffffffu, rank == p.topk_groups && e0 < E);
            const uint32_t last = __shfl_sync(0xffffffffu, total, __ffs(in) - 1), next = __shfl_sync(0xffffffffu, total, __ffs(out) - 1);
            if (next && !apart(unordered(last), unordered(next), 2.f * tol, 2.f * kCut)) {
                // in 64 bits: each lane's two best exactly (if a third is as near as the second, or a softmax has a
                // bias, the whole row is), the groups' from them, and their ranks again
                double c[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t k = key[j < NPL ? j : 0];
                    const int i = kPlace - (k & kPlace);
                    float v = 0.f;
#pragma unroll
                    for (int n = 0; n < NPL; ++n)
                        if (n == i) v = l[n];
                    c[j] = -INFINITY;
                    if (k && j < NPL) {
                        c[j] = (double)v;
                        if (scored) c[j] = sigmoid ? 1.0 / (1.0 + exp(-(double)v)) : exp((double)v - (double)top);
                        if (p.bias) c[j] += (double)fminf(p.bias[e0 + i], kMostFloat);
                    }
                }
                const uint32_t second = NPL > 1 ? key[NPL > 1] : 0u, third = NPL > 2 ? key[NPL > 2 ? 2 : 0] : 0u;
                const bool sure = !third || apart(unordered(second & ~kPlace), unordered(third & ~kPlace), tol, kCut);
                if (!__all_sync(0xffffffffu, sure) || (p.bias && !sigmoid)) settled = false;
                double x = fmax(c[0], c[1]), y = fmin(c[0], c[1]);
                for (int o = 1; o < lanes; o <<= 1) {
                    const double ox = __shfl_xor_sync(0xffffffffu, x, o), oy = __shfl_xor_sync(0xffffffffu, y, o);
                    y = fmax(fmax(y, oy), fmin(x, ox));
                    x = fmax(x, ox);
                }
                const double sum = sums && y > -INFINITY ? x + y : x;
                rank = 0;
                for (int d = 1; d < p.groups; ++d) {
                    const int other = group + d < p.groups ? group + d : group + d - p.groups;
                    const double s2 = __shfl_sync(0xffffffffu, sum, (other * lanes) & 31);
                    rank += s2 > sum || (s2 == sum && other < group);
                }
                kept = total && rank < p.topk_groups;
            }
        }
        if (sums && !p.bias) {  // the logits decide within the groups
#pragma unroll
            for (int i = 0; i < NPL; ++i) key[i] = l[i] > -INFINITY ? (ordered(l[i]) & ~kPlace) | (kPlace - i) : 0u;
            sort_keys(key);
        }
        if (!kept) {
#pragma unroll
            for (int i = 0; i < NPL; ++i) key[i] = 0;
        }
    }
    uint32_t owner_of = 1;  // lane k: holders and key of the k-th choice
    int count = 0;
    const uint32_t below = (1u << lane) - 1u;
    uint32_t key_of = 0;
    const int rounds = p.K + (exact_keys ? 0 : 2);
    for (; count < rounds; ++count) {
        const uint32_t head = key[0] & ~kPlace, best = __reduce_max_sync(0xffffffffu, head);
        if (best == 0) break;  // nothing is left: id -1, weight 0
        const uint32_t holders = __ballot_sync(0xffffffffu, head == best);
        const bool owns = head == best && (holders & below) == 0;  // the lowest of them
        const uint32_t k = __shfl_sync(0xffffffffu, key[0], __ffs(holders) - 1);
        const bool here = lane == count;
        owner_of = here ? holders : owner_of;
        key_of = here ? k : key_of;
#pragma unroll
        for (int i = 0; i + 1 < NPL; ++i) key[i] = owns ? key[i + 1] : key[i];
        key[NPL - 1] = owns ? 0u : key[NPL - 1];
    }
    int mine = lane < count ? (__ffs(owner_of) - 1) * NPL + (int)(kPlace - (key_of & kPlace)) : -1;
    uint32_t near = 0;  // bit k: choices k and k + 1 are not settled
    if (!exact_keys) {
        const float c = unordered(key_of & ~kPlace), next = __shfl_down_sync(0xffffffffu, c, 1);
        near = __ballot_sync(0xffffffffu, lane + 1 < count && !apart(c, next, p.bias ? tol : 0.f, kCut));
    }
    float v = mine >= 0 ? fminf(load_logit(p.logits, base + mine, DT), kMostFloat) : 0.f;
    if (near) {
        if ((near & near >> 1) || (p.bias && !sigmoid)) {
            settled = false;
        } else {
            double c = (double)v;
            if (p.bias && mine >= 0) c = 1.0 / (1.0 + exp(-c)) + (double)fminf(p.bias[mine], kMostFloat);
            const bool first = near >> lane & 1u, second = lane > 0 && (near >> (lane - 1) & 1u);
            const int other = lane + (first ? 1 : 0) - (second ? 1 : 0);
            const double oc = __shfl_sync(0xffffffffu, c, other);
            const int oe = __shfl_sync(0xffffffffu, mine, other);
            const float ov = __shfl_sync(0xffffffffu, v, other);
            const bool less = c < oc || (c == oc && mine > oe);
            if ((first && less) || (second && !less)) {
                mine = oe;
                v = ov;
            }
        }
    }
    if (!settled) {
        route_row_exact<NPL>(p, t);
        return;
    }
    if (lane >= p.K) mine = -1;
    float s = 0.f;
    if (mine >= 0) s = sigmoid ? 1.f / (1.f + expf(-v)) : expf(v - top) / den;
    if (p.renorm) {
        float sum = s;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        s = s / (sum + 1e-20f);
    }
    if (lane < p.K) {
        p.ids[t * p.K + lane] = mine;
        p.w[t * p.K + lane] = s * p.scale;
    }
}

// The rows of a call whose groups do not fall on 2^n whole lanes, or whose top_k takes every lane: 16384 rows of 160
// experts in 8 groups 96 us with sigmoid, bias and two a group (256 experts in 8 groups above: 22), of 60 in 4 33.
template <int NPL>
__global__ void __launch_bounds__(kRouteWarps * 32) route_scored_exact_kernel(const __grid_constant__ RouteScoredParams p) {
    const int64_t t = (int64_t)blockIdx.x * kRouteWarps + (threadIdx.x >> 5);
    if (t < p.T) route_row_exact<NPL>(p, t);
}

template <int NPL, int DT>
void route_launch_as(const RouteScoredParams& p, unsigned grid, cudaStream_t st) {
    if (p.score == MOE_SCORE_SIGMOID) route_scored_kernel<NPL, DT, true><<<grid, kRouteWarps * 32, 0, st>>>(p);
    else route_scored_kernel<NPL, DT, false><<<grid, kRouteWarps * 32, 0, st>>>(p);
}

template <int NPL>
void route_launch(const RouteScoredParams& p, cudaStream_t st) {
    const unsigned grid = (unsigned)((p.T + kRouteWarps - 1) / kRouteWarps);
    const int per = p.E / p.groups, lanes = per / NPL;
    // the two rounds past top_k need a lane each
    if (p.K > 30 || (p.groups > 1 && (per % NPL != 0 || (lanes & (lanes - 1)) != 0)))
        route_scored_exact_kernel<NPL><<<grid, kRouteWarps * 32, 0, st>>>(p);
    else if (p.dtype == MOE_F32) route_launch_as<NPL, MOE_F32>(p, grid, st);
    else if (p.dtype == MOE_BF16) route_launch_as<NPL, MOE_BF16>(p, grid, st);
    else route_launch_as<NPL, MOE_F16>(p, grid, st);
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
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (E <= 32) route_launch<1>(p, st);
    else if (E <= 64) route_launch<2>(p, st);
    else if (E <= 128) route_launch<4>(p, st);
    else if (E <= 256) route_launch<8>(p, st);
    else if (E <= 512) route_launch<16>(p, st);
    else route_launch<32>(p, st);
    CUDA_TRY(cudaGetLastError());
    return MOE_OK;
}
