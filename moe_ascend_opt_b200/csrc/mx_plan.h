// How a call of the MXFP4 expert layer runs and what its workspace holds: host arithmetic, free of CUDA.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include <algorithm>

namespace moe {
namespace mx {
constexpr int kFusedPairs = 8;     // routed pairs of the calls whose two kernels route for themselves
constexpr int kFusedStages = 32;   // depth of fused calls, in stages of 256 elements: their A buffers hold it whole
constexpr int kPrepSelf = 4096;    // pairs up to which each CTA of the token kernel counts all of them itself
constexpr int kFusedRows = 8, kSlimRows = 32, kWideRows = 128;  // rows of an m tile
}  // namespace mx

namespace layer {

constexpr int64_t kMaxPairs = 1 << 18;  // routed pairs of one pass; longer calls run in slices of tokens

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct LayerShape {
    int64_t E, H, I;
    int64_t all = 0;  // experts that the call's pairs are spread over, of which this engine holds E (0: no others)
};

// How a call of T tokens runs.  Fused: two kernels that route for themselves, where the launches and
// their latencies are what counts; slim or wide tiles after a kernel that places the token rows, by the
// rows that an expert can expect: the call's pairs over the experts of the whole layer, since a call on a part
// of them is given the pairs of the others too.
enum Plan { kPlanFused, kPlanSlim, kPlanWide };
constexpr int64_t kWideExpert = 56;  // wide tiles from this many rows an expert on
inline Plan plan_of(const LayerShape& s, int64_t T, int64_t K) {
    const int64_t P = T * K;
    if (P <= mx::kFusedPairs && ceil_div(s.H, 256) <= mx::kFusedStages) return kPlanFused;
    return P >= kWideExpert * std::max(s.E, s.all) ? kPlanWide : kPlanSlim;
}

// Tokens of one CTA of the token kernel: runs of 256 pairs or more and at most 512 runs in long
// calls (every CTA reads all runs' counts), a CTA for each SM in a short call.
inline int64_t prep_tokens(int64_t T, int64_t K, int sms) {
    const int64_t P = T * K;
    if (P <= mx::kPrepSelf) return ceil_div(T, sms);
    return std::max<int64_t>(ceil_div(256, K), ceil_div(T, 512));
}
// A bound of the runs of a long call that, unlike their number, does not fall as T grows.
inline int64_t runs_bound(int64_t T, int64_t K) { return std::min<int64_t>(512, ceil_div(T, ceil_div(256, K))); }

// Offsets of a call's workspace.  Its size does not fall as T grows while the plan stays the same.
struct Layout {
    Plan plan;
    int tile;    // rows of an m tile
    int64_t mt;  // bound of the number of m tiles
    size_t hq, hs, part, mt_list, ppos, counts, xq, xs, bytes;
};
inline Layout layout_of(const LayerShape& s, int64_t T, int64_t K) {
    Layout w{};
    const int64_t P = T * K, kb1 = ceil_div(s.H, 128), kb2 = ceil_div(s.I, 128);
    w.plan = plan_of(s, T, K);
    w.tile = w.plan == kPlanWide ? mx::kWideRows : (w.plan == kPlanFused ? mx::kFusedRows : mx::kSlimRows);
    w.mt = w.plan == kPlanFused ? P : P / w.tile + std::min(P, s.E);
    const int64_t rows = w.mt * w.tile;
    auto take = [&](int64_t n) {
        const size_t at = w.bytes;
        w.bytes += (size_t)(n + 1023) / 1024 * 1024;
        return at;
    };
    w.hq = take(rows * (s.I / 2));
    w.hs = take(w.mt * kb2 * 512);
    w.part = take((w.plan == kPlanFused ? P : rows) * s.H * 4);
    if (w.plan != kPlanFused) {
        w.mt_list = take(w.mt * 8);
        w.ppos = take(P * 4);
        w.counts = take(P > mx::kPrepSelf ? runs_bound(T, K) * s.E * 4 : 0);
        w.xq = take(rows * (s.H / 2));
        w.xs = take(w.mt * kb1 * 512);
    }
    return w;
}

inline int64_t slice_tokens(int64_t T, int64_t K) { return std::min(T, std::max<int64_t>(1, kMaxPairs / K)); }

// Bytes for a call of T tokens: of its slices, the last of which may be shorter and take another plan.
inline size_t call_bytes(const LayerShape& s, int64_t T, int64_t K) {
    const int64_t S = slice_tokens(T, K), tail = T % S;
    const size_t bytes = layout_of(s, S, K).bytes;
    return tail ? std::max(bytes, layout_of(s, tail, K).bytes) : bytes;
}

// Bytes for every call of 1 to T tokens, the longest of each plan: routed ones, and dense ones, whose pairs are
// all this engine's.
inline size_t reserve_bytes(LayerShape s, int64_t T, int64_t K) {
    size_t bytes = 0;
    for (int dense = 0; dense < 2; ++dense) {
        const int64_t k = dense ? 1 : K, S = slice_tokens(T, k);
        if (dense) s.all = 0;
        for (int64_t t : {S, mx::kFusedPairs / k, (kWideExpert * std::max(s.E, s.all) - 1) / k})
            bytes = std::max(bytes, layout_of(s, std::min(S, std::max<int64_t>(1, t)), k).bytes);
    }
    return bytes;
}

}  // namespace layer
}  // namespace moe
