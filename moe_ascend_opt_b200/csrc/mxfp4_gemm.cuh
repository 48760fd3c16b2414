// Products of MXFP4 matrices on the tensor cores (tcgen05.mma kind::mxf4, block scales applied
// by the MMA): the dense product a b^T, and the gate_up and down products of the expert layer.
//
// One persistent, warp-specialised kernel: its CTAs walk over the (128 x NT) output tiles.
//   warp 0      TMA producer: a stage is 256 elements of K, i.e. 128 bytes (one swizzle atom) of
//               each of the 128 rows of A and NT rows of B, and their scale tiles (512 bytes hold
//               128 rows x 128 elements);
//   warp 1      copies the stage's scales to TMEM (tcgen05.cp) and issues its MMAs (K = 64 each),
//               fp32 accumulators in TMEM;
//   warps 4-    epilogue, a thread per row of the tile and NT or NT / 2 columns; it takes its
//               accumulators to registers and gives the TMEM back at once, so that its arithmetic
//               and stores overlap the products of the next tile.
// The rows of A are tokens, so a thread of the epilogue holds whole 32-blocks of its token: the
// gate_up epilogue forms SiLU(gate) * up and quantises it without a word to other threads.
// gate_up weights lie in 64-row groups of 32 gate rows and the 32 up rows of the same units.
//
// Large dense products run in pairs of CTAs (clusters of two): each fetches its 128 rows of A, half of B's rows
// and its scales, all counted by CTA 0's barriers, and CTA 0 issues the MMAs of both (cta_group::2).  A thread
// of CTA 1 that forwarded its stages to CTA 0 cost more than the sharing gave (64 us against 52 at
// 8192 x 4096 x 4096).
//
// What bounds it: at many rows the ring's round trip, an MMA's end to the next data's arrival (about 1 us and a
// load's latency for four to six stages), then the single accumulator's hand-over, about 1 us a tile; at few
// rows the weights' stream.  Layers of H = 2048, I = 768, 128 experts, top-8: T = 4096 gate_up 77 us, down 65 us
// (309 GFLOP of MMAs: 47 us at four times the measured bf16 rate); T = 201 of 64 experts gate_up 26, down 15 us
// alone, 51 with the kernels around them, which overlap.
//
// All waits are bounded; one that runs out sets the error word, and every role leaves its loop.
#pragma once
#include <cuda.h>

#include "mx_plan.h"
#include "mxfp4.cuh"

namespace moe {
namespace mx {

enum Mode { kDense = 0, kGateUp = 1, kDown = 2 };
constexpr int kStageK = 256;

struct GemmParams {
    int M, N, K;         // dense: rows of a; N rows of b (of one expert); depth
    int kb;              // scale tiles along K
    int nt_count, mt_count;
    const uint8_t* sfa;  // [m tiles][kb][512]
    const uint8_t* sfb;  // dense [ceil(N / 128)][kb][512]; experts [experts][ceil(N / 256)][stages][kPanelScales]
    const int2* mt_list;       // experts: expert and rows of each m tile; rows 0 ends it
    void* out;           // dense [M][N] (out_dtype); down [m tile rows][N] fp32 parts
    int out_dtype;
    int tma_out;         // dense, wide tiles: store through the map (rows of a multiple of 16 bytes)
    int I;               // gate_up: hq [m tile rows][I / 2], hs tiles with hkb tiles along I
    int hkb;
    uint8_t* hq;
    uint8_t* hs;
    int32_t* err;
    // fused calls: the routing, the tokens, and down's weighted sum
    const void* x;
    const int32_t* ids;
    const float* tw;
    int T, topk, E, e_off, emap_n, act_bf16;
    const int32_t* emap;
    void* y;
    int y_dtype;
    unsigned int* cnt;   // down parts finished per column tile, zero between calls
};

// A kernel's shape: NT columns and TM rows of a tile (the MMA always takes 128 rows; of a tile of fewer it
// reads whatever lies behind them in shared memory, and those lanes are never read back), STAGES of the
// ring, EPI epilogue warps, CTAS per SM, ACC accumulators, BUFS staging buffers of a wide tile's epilogue warp.
// PAIR: the two CTAs of a cluster share a tile of 256 rows, 128 rows (TM) each, and each fetches half of B.
template <int NT_, int TM_, int STAGES_, int EPI_, int CTAS_, int ACC_, bool FUSED_ = false, int BUFS_ = 1, bool PAIR_ = false>
struct Shape {
    static constexpr int NT = NT_, TM = TM_, STAGES = STAGES_, kEpiWarps = EPI_, kCtas = CTAS_;
    static constexpr bool FUSED = FUSED_, PAIR = PAIR_;
    static constexpr bool EARLY = TM == 32;  // gate_up fetches its first weights while the tokens are prepared
    static constexpr int BUFS = BUFS_;  // staging buffers of an epilogue warp
    static constexpr int kSfTiles = (NT + 127) / 128;  // scale tiles (128 rows) that cover a stage's B rows
    static constexpr int kA = TM * 128, kB = NT * 128 / (PAIR ? 2 : 1);
    static constexpr int kTileRows = PAIR ? 256 : TM;
    static constexpr int kSfaKg = TM == 8 ? 128 : 512;  // scales of A for 128 elements: those of 8 rows, or a tile
    static constexpr int kSfbBytes = 1024 * kSfTiles;
    // A stage of the ring: A | B | scales of B | scales of A, the first and the last not where the kernel
    // writes A itself (WA): A and its scales for the whole depth then lie in two buffers before the ring.
    __host__ __device__ static constexpr int off_b(bool wa) { return wa ? 0 : kA; }
    __host__ __device__ static constexpr int off_sfb(bool wa) { return off_b(wa) + kB; }
    __host__ __device__ static constexpr int off_sfa(bool wa) { return off_sfb(wa) + kSfbBytes; }
    __host__ __device__ static constexpr int stage(bool wa) { return (off_sfa(wa) + (wa ? 0 : 2 * kSfaKg) + 1023) / 1024 * 1024; }
    __host__ __device__ static constexpr int a_buffer(int stages) { return stages * kA + (stages * 2 * kSfaKg + 1023) / 1024 * 1024; }
    static constexpr int kSfCols = 8 * (1 + kSfTiles);  // TMEM columns of a stage's scales
    static constexpr int kAcc = ACC_;
    static constexpr int kCols = NT / (kEpiWarps / 4);  // columns of an epilogue thread of a 128-row tile
    static constexpr int kThreads = 128 + 32 * kEpiWarps;
    // wide tiles leave through shared memory: 32 rows x 64 bytes per epilogue warp, stored by TMA
    static constexpr int kStaging = NT >= 256 ? kEpiWarps * BUFS * 2048 : 0;
    // tiles of few rows pass through shared memory too, from the one warp that can read their TMEM lanes to all
    static constexpr int kRowPitch = NT + 4;  // floats: 16-byte accesses of neighbouring rows meet no bank twice
    static constexpr int kRows = TM < 128 ? TM * kRowPitch * 4 : 0;
    // Dynamic shared memory for `stages` of depth.  The MMA's 128 rows of the last A stay inside, so do
    // the 512 bytes that a copy of its scales takes.
    __host__ __device__ static constexpr int tail(bool wa) {
        return wa || stage(wa) >= 16384 + 512 ? 0 : (16384 + 512 - stage(wa) + 1023) / 1024 * 1024;
    }
    __host__ __device__ static constexpr int smem(bool wa, int stages) {
        const int ring = STAGES * stage(wa), buffers = wa ? 2 * a_buffer(stages) : 0;
        return buffers + ring + tail(wa) + kStaging + (kRows + 1023) / 1024 * 1024;
    }
};

// Descriptor of a 512-byte scale tile for tcgen05.cp: no swizzle, 8-row groups of 128 bytes.
MOE_DEV uint64_t sf_desc(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)1 << 16 | (uint64_t)(128u >> 4) << 32 | (uint64_t)1 << 46;
}

// Instruction descriptor, kind::mxf4: A and B e2m1 (bits 7-9 and 10-11 = 1), both K-major,
// N >> 3 (bits 17-22), scales ue8m0 (bit 23), M >> 4 (bits 24-28); the scale bytes of B and A
// within a 32-bit word are chosen by bits 4-5 and 29-30 (0 or 2).
__host__ __device__ constexpr uint32_t idesc_mxf4(int M, int N) {
    return (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(M >> 4) << 24);
}

// PAIR: one instruction for the two CTAs of a cluster, 256 rows; each holds its 128 rows of A, its half of
// B's rows, and its accumulators, at the same addresses.
template <bool PAIR>
MOE_DEV void mma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, bool accumulate) {
    if (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"((uint32_t)accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"((uint32_t)accumulate)
            : "memory");
}

template <bool PAIR>
MOE_DEV void cp_scales(uint32_t taddr, uint64_t desc) {
    if (PAIR) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
    else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// Arrival on a barrier (PAIR: on that of both CTAs) when the MMAs issued so far are complete.
template <bool PAIR>
MOE_DEV void commit(uint64_t* bar) {
    if (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                         smem_u32(bar)),
                     "h"((uint16_t)3)
                     : "memory");
    else
        gemm::tc_commit(bar);
}

// Shared memory of CTA 0 of the cluster at the place of this CTA's `addr`, and an arrival there.  tcgen05's own
// fences order the accumulators' reads before it, so it carries no release (which took about a microsecond).
MOE_DEV uint32_t in_leader(uint32_t addr) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(addr));
    return a;
}
MOE_DEV void arrive_leader(uint64_t* bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(in_leader(smem_u32(bar))) : "memory");
}
MOE_DEV void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// One lane of a converged warp.
MOE_DEV bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}

MOE_DEV void tma_2d(uint32_t dst, const CUtensorMap* m, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(m), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
// PAIR: into this CTA's shared memory, counted by a barrier of CTA 0 of the cluster.
MOE_DEV void tma_2d_pair(uint32_t dst, const CUtensorMap* m, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(m), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
MOE_DEV void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
                 "r"(bytes), "r"(bar)
                 : "memory");
}
// 32 rows x 64 bytes of shared memory (64-byte swizzle) to global memory; what lies outside the map is dropped.
MOE_DEV void tma_store_2d(const CUtensorMap* m, uint32_t src, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(m), "r"(x), "r"(y), "r"(src)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// As mbar_try_wait, for arrivals from the other CTA of the cluster (arrive_leader).
MOE_DEV bool mbar_try_wait_cluster(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.relaxed.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
// Bounded wait that also ends when another role of the CTA has given up.
template <bool CLUSTER>
MOE_DEV bool wait_or_fail(uint64_t* bar, uint32_t parity, volatile int* failed) {
    for (uint32_t it = 0; it < kSpinLimit; ++it) {
        if (CLUSTER ? mbar_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity)) return true;
        if ((it & 15u) == 15u && *failed) return false;
        if (it > 8192) __nanosleep(128);
    }
    *failed = 1;
    return false;
}

// The same by a whole warp, which goes on or leaves together.
template <bool CLUSTER = false>
MOE_DEV bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* failed) {
    return __all_sync(0xffffffffu, wait_or_fail<CLUSTER>(bar, parity, failed));
}

// N consecutive fp32 columns of this thread's TMEM lane.
template <int N>
MOE_DEV void load_columns(uint32_t taddr, float (&v)[N]) {
    uint32_t r[N];
#pragma unroll
    for (int c = 0; c < N; c += 16)
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
            : "=r"(r[c]), "=r"(r[c + 1]), "=r"(r[c + 2]), "=r"(r[c + 3]), "=r"(r[c + 4]), "=r"(r[c + 5]), "=r"(r[c + 6]),
              "=r"(r[c + 7]), "=r"(r[c + 8]), "=r"(r[c + 9]), "=r"(r[c + 10]), "=r"(r[c + 11]), "=r"(r[c + 12]),
              "=r"(r[c + 13]), "=r"(r[c + 14]), "=r"(r[c + 15])
            : "r"(taddr + c));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    // the registers hold their values from the wait on: tie every use to it
#pragma unroll
    for (int c = 0; c < N; ++c) asm volatile("" : "+r"(r[c]));
#pragma unroll
    for (int c = 0; c < N; ++c) v[c] = __uint_as_float(r[c]);
}

template <int DT>
MOE_DEV uint32_t pack16(float a, float b) {
    if (DT == MOE_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// 32 columns of a row to global memory; n of them exist.  Rows whose pitch is a multiple of 16
// bytes take 16-byte stores (n is then a multiple of a store's elements).
template <int DT>
MOE_DEV void store_row(void* out, int64_t at, const float* v, int n, bool vec) {
    if (DT == MOE_F32) {
        float* o = reinterpret_cast<float*>(out) + at;
        if (vec) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (4 * j < n) reinterpret_cast<float4*>(o)[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
        } else {
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (j < n) o[j] = v[j];
        }
    } else {
        uint16_t* o = reinterpret_cast<uint16_t*>(out) + at;
        uint32_t w[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) w[j] = pack16<DT>(v[2 * j], v[2 * j + 1]);
        if (vec) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (8 * j < n) reinterpret_cast<uint4*>(o)[j] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
        } else {
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (j < n) o[j] = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
        }
    }
}

// SiLU(g) * u.  exp(-g) = 2^t (1 + r ln 2) with t = -g log2(e) rounded and r what the rounding and
// the constant lost, so that a large |g| costs no accuracy.  Past g = 128 exp(-g) adds nothing to 1, and t of the
// largest g would be infinite; below g = -88 exp overflows, and SiLU, less than 6e-37, counts as 0.
MOE_DEV float silu_up(float g, float u) {
    const float c = fminf(g, 128.f);
    const float t = -1.44269502f * c;
    const float r = fmaf(c, -1.92596299e-8f, fmaf(c, -1.44269502f, -t));
    float e;
    asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(t));
    e = g < -88.f ? INFINITY : fmaf(e, 0.693147181f * r, e);
    float q;
    asm("rcp.approx.f32 %0, %1;" : "=f"(q) : "f"(1.f + e));
    return g * q * u;
}

// Routing of a fused call by the CTA itself: a piece per expert, in the order of their first pairs, the pairs
// of a piece (at most 8, a tile's rows) in their own order.
struct FusedRoute {
    int np;
    int e[kFusedPairs];                  // local expert of each pair, -1: another engine's
    int rank[kFusedPairs];               // among the pairs of its expert
    int piece_e[kFusedPairs], rows[kFusedPairs];
    uint8_t pair[kFusedPairs * kFusedPairs];  // pair of each row
};

template <bool FUSED>
struct RouteStore {
    using type = int;
};
template <>
struct RouteStore<true> {
    using type = FusedRoute;
};

MOE_DEV void fused_route(FusedRoute& f, const GemmParams& p, int threads) {
    const int P = p.T * p.topk, tid = threadIdx.x;
    for (int i = tid; i < P; i += threads) {
        f.e[i] = local_expert(__ldcg(p.ids + i), p.e_off, p.E, p.emap, p.emap_n, i, p.topk);
        f.rows[i] = 0;
    }
    if (tid == 0) f.np = 0;
    __syncthreads();
    for (int i = tid; i < P; i += threads) {
        const int e = f.e[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < i; ++j) rank += f.e[j] == e;
        f.rank[i] = e >= 0 ? rank : -1;
    }
    __syncthreads();
    for (int i = tid; i < P; i += threads) {
        const int e = f.e[i], rank = f.rank[i];
        if (e < 0) continue;
        int heads = 0, piece = 0;
#pragma unroll 8
        for (int j = 0; j <= i; ++j) {  // the piece's first pair comes at or before i
            const int rj = f.rank[j];
            if (f.e[j] == e && rj == 0) piece = heads;
            heads += rj == 0;
        }
        f.pair[piece * kFusedPairs + rank] = (uint8_t)i;
        atomicMax(&f.rows[piece], rank + 1);
        if (rank == 0) {
            f.piece_e[piece] = e;
            atomicAdd(&f.np, 1);
        }
    }
    __syncthreads();
}

// Columns [n0, n0 + 128) of y from the parts of every pair, 4 columns a lane, in the order of a token's
// pairs; tokens first, first + step, ...
template <int DT>
MOE_DEV void fused_combine(const FusedRoute& f, const GemmParams& p, int n0, int first, int step) {
    const int n = n0 + (threadIdx.x & 31) * 4, K = p.topk;
    const float* part = static_cast<const float*>(p.out);
    if (n >= p.N) return;
    for (int t = first; t < p.T; t += step) {
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        float4 v[kFusedPairs];
        float w[kFusedPairs];
#pragma unroll
        for (int k = 0; k < kFusedPairs; ++k) {
            const int i = t * K + k;
            const bool have = k < K && f.e[min(i, p.T * p.topk - 1)] >= 0;
            v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            w[k] = 0.f;
            if (have) {
                v[k] = __ldcg(reinterpret_cast<const float4*>(part + (int64_t)i * p.N + n));
                w[k] = __ldg(p.tw + i);
            }
        }
#pragma unroll
        for (int k = 0; k < kFusedPairs; ++k) {
            a.x = fmaf(w[k], v[k].x, a.x);
            a.y = fmaf(w[k], v[k].y, a.y);
            a.z = fmaf(w[k], v[k].z, a.z);
            a.w = fmaf(w[k], v[k].w, a.w);
        }
        const int64_t at = (int64_t)t * p.N + n;
        if (DT == MOE_F32) *reinterpret_cast<float4*>(static_cast<float*>(p.y) + at) = a;
        else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.y) + at) = make_uint2(pack16<DT>(a.x, a.y), pack16<DT>(a.z, a.w));
    }
}

template <int MODE, class S>
__global__ void __launch_bounds__(S::kThreads, S::kCtas)
    mx_gemm_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb,
                   const __grid_constant__ CUtensorMap ta32, const __grid_constant__ CUtensorMap to,
                   const __grid_constant__ CUtensorMap tfa, const __grid_constant__ CUtensorMap tfb,
                   const __grid_constant__ GemmParams p) {
    constexpr int NT = S::NT, TM = S::TM, STAGES = S::STAGES;
    constexpr bool PAIR = S::PAIR;
    static_assert(!PAIR || MODE == kDense, "pairs take dense products");
    static_assert(MODE != kDown || TM < 128 || S::kStaging > 0, "down's tiles of 128 rows leave through shared memory");
    static_assert(!S::FUSED || TM == kFusedPairs, "all pairs of a fused call fit a tile");
    constexpr bool FUSED = S::FUSED, WRITE_A = FUSED && MODE == kGateUp;  // A from the token rows, by warps 2 and 3
    constexpr int kSfBase = S::kAcc * NT;  // TMEM: the accumulators, then each stage's scales
    constexpr int kTmemCols = kSfBase + STAGES * S::kSfCols <= 256 ? 256 : 512;
    static_assert(kSfBase + STAGES * S::kSfCols <= 512 && kTmemCols * S::kCtas <= 512, "TMEM");
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    constexpr int kStage = S::stage(WRITE_A), oB = S::off_b(WRITE_A), oSfB = S::off_sfb(WRITE_A), oSfA = S::off_sfa(WRITE_A);
    uint8_t* abuf = smem_raw;
    const int nstages = (p.K + kStageK - 1) / kStageK, k64 = (p.K + 63) / 64;
    uint8_t* smem = abuf + (WRITE_A ? 2 * S::a_buffer(nstages) : 0);  // the ring
    __shared__ __align__(8) uint64_t s_full[STAGES], s_empty[STAGES], s_accfull[2], s_accempty[2], s_afull[2], s_aempty[2], s_done;
    __shared__ uint32_t s_tmem;
    __shared__ int s_failed, s_go, s_last;
    __shared__ typename RouteStore<FUSED>::type s_route;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (smem_u32(smem_raw) & 1023) {  // the swizzled tiles rely on it; in every CTA or in none
        if (tid == 0) set_err(p.err, kErrFullWait);
        return;
    }

    if (tid == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&s_full[s], 1);
            mbar_init(&s_empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&s_accfull[a], 1);
            mbar_init(&s_accempty[a], TM < 128 ? 1 : S::kEpiWarps * (PAIR ? 2 : 1));
            mbar_init(&s_afull[a], 2);
            mbar_init(&s_aempty[a], 1);
        }
        mbar_init(&s_done, 1);
        s_failed = 0;
        fence_barrier_init();
    }
    if (warp == 2) {
        if (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "n"(kTmemCols)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "n"(kTmemCols)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    gemm::tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();  // the peer's barriers are ready
    gemm::tc_fence_after();
    const uint32_t tmem = s_tmem;
    volatile int* failed = &s_failed;
    // down: the routing (ids, or the tiles' list) was complete before gate_up passed its own wait and let
    // this kernel start, so the weights are fetched before the wait for gate_up's output.  So does gate_up of a
    // short call behind the token kernel, which let it start when the ids were there: it counts them itself to
    // find its first tile's expert (a layer of T = 2 19.7 -> 18.2 us, 8 33 -> 32, 128 66.7 -> 65.3; H = 2048, I = 768,
    // 128 experts, top-8, in graphs).
    const bool ahead_of_list = MODE == kGateUp && S::EARLY && p.ids != nullptr;
    int first_e = -1;
    if (ahead_of_list) {
        int* const hist = reinterpret_cast<int*>(smem + STAGES * kStage + S::tail(WRITE_A));  // the rows' place, idle so far
        for (int e = tid; e < p.E; e += S::kThreads) hist[e] = 0;
        __syncthreads();
        const int P = p.T * p.topk;
        for (int i = tid; i < P; i += S::kThreads) {
            const int e = local_expert(__ldcg(p.ids + i), p.e_off, p.E, p.emap, p.emap_n, i, p.topk);
            if (e >= 0) atomicAdd(&hist[e], 1);
        }
        __syncthreads();
        if (warp == 0) {
            const int mt0 = (int)(blockIdx.x / p.nt_count);
            int before = 0;
            for (int e0 = 0; e0 < p.E && first_e < 0; e0 += 32) {
                const int n = e0 + lane < p.E ? (hist[e0 + lane] + TM - 1) / TM : 0;
                int incl = n;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int v = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += v;
                }
                const unsigned past = __ballot_sync(0xffffffffu, before + incl > mt0);
                if (past) first_e = e0 + __ffs(past) - 1;
                before += __shfl_sync(0xffffffffu, incl, 31);
            }
        }
        __syncthreads();  // the rows' place is free
    }
    if (MODE != kDown && !(ahead_of_list && warp == 0)) asm volatile("griddepcontrol.wait;" ::: "memory");
    if (!(ahead_of_list && warp == 0)) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    FusedRoute& route = reinterpret_cast<FusedRoute&>(s_route);  // an int where nothing is fused, never read
    if (FUSED) fused_route(route, p, S::kThreads);
    // the producer alone goes ahead of gate_up's end: the bounded waits of the others must not count its time
    if (MODE == kDown && warp != 0) asm volatile("griddepcontrol.wait;" ::: "memory");

    const int mt_count = FUSED ? route.np : p.mt_count;  // of an expert list its bound
    const int64_t tiles = (int64_t)mt_count * p.nt_count;
    const int rank = PAIR ? (int)(blockIdx.x & 1) : 0;  // in the cluster
    const int first = PAIR ? blockIdx.x >> 1 : blockIdx.x, step = PAIR ? gridDim.x >> 1 : gridDim.x;
    const int nb128 = (p.N + 127) / 128;
    auto tile_of = [&](int mt) {  // expert, rows; no rows: past the list's end
        if (FUSED) return make_int2(route.piece_e[mt], route.rows[mt]);
        return MODE == kDense ? make_int2(0, min(S::kTileRows, p.M - mt * S::kTileRows)) : __ldcg(p.mt_list + mt);
    };

    if (warp == 0) {
        // As for the MMAs: the warp walks the loop with uniform operands and one elected lane issues (a
        // copy issued under a lane test, with operands that could differ by lane, takes about 100 ns).
        const uint32_t usmem = __shfl_sync(0xffffffffu, smem_u32(smem), 0);
        const bool issue = elect_one();
        bool ok = true;
        uint32_t it = 0, st = 0, parity = 1;  // stages so far; stage and phase of the ring
        // the A rows of a stage and their scales: all rows of the tile in one copy, or, of a tile of 128
        // rows that is not full, 32 rows a copy
        auto load_a = [&](uint32_t to_st, int mt, int s, int copies) {
            const uint32_t base = usmem + to_st * kStage, bar = smem_u32(&s_full[to_st]);
            if (TM < 128 || MODE == kDense || copies == 4) {
                tma_2d(base, &ta, s * 128, mt * TM, bar);
            } else {
                for (int c = 0; c < copies; ++c) tma_2d(base + c * 4096, &ta32, s * 128, mt * TM + c * 32, bar);
            }
            bulk_copy(base + oSfA, p.sfa + ((int64_t)mt * p.kb + 2 * s) * S::kSfaKg, min(2, p.kb - 2 * s) * S::kSfaKg, bar);
        };
        // a pair's stage: both CTAs' copies count on CTA 0's barrier; the second 128 rows may not exist
        auto load_pair = [&](int mt, int nt, int s) {
            const bool both = p.M - mt * 256 > 128;
            const uint32_t base = usmem + st * kStage, bar = in_leader(smem_u32(&s_full[st]));
            if (rank == 0)
                mbar_arrive_expect_tx(&s_full[st], (both ? 2 : 1) * (S::kA + 2 * S::kSfaKg) + 2 * (S::kB + S::kSfbBytes));
            tma_2d_pair(base + oB, &tb, s * 128, nt * NT + rank * (NT / 2), bar);
            tma_2d_pair(base + oSfB, &tfb, s * 256, nt * NT / 128, bar);
            if (rank == 0 || both) {
                tma_2d_pair(base, &ta, s * 128, mt * 256 + rank * 128, bar);
                tma_2d_pair(base + oSfA, &tfa, s * 256, mt * 2 + rank, bar);
            }
        };
        // of a first tile whose list is not there yet only the expert is known, and that it has rows
        int2 next = ahead_of_list ? make_int2(first_e, first_e >= 0) : first < tiles ? tile_of((int)(first / p.nt_count)) : make_int2(0, 0);
        for (int64_t tile = first; ok && tile < tiles; tile += step) {
            const int mt = (int)(tile / p.nt_count), nt = (int)(tile - (int64_t)mt * p.nt_count);
            const int2 of = next;
            const bool early = (MODE == kDown || ahead_of_list) && it == 0;
            if (tile + step < tiles && !(ahead_of_list && early)) next = tile_of((int)((tile + step) / p.nt_count));  // a tile ahead of its use
            const int e = __shfl_sync(0xffffffffu, of.x, 0), rows = __shfl_sync(0xffffffffu, of.y, 0);
            if (rows == 0) break;
            const int copies = MODE == kDense || TM < 128 ? 4 : (rows + 31) >> 5;  // quarters of a 128-row tile
            // B's scales: of an expert one contiguous piece a stage, of a dense product a piece per 128 rows
            const int sft = MODE == kDense ? min(S::kSfTiles, nb128 - nt * NT / 128) : 1;
            // B's rows: of an expert those of a panel, whose stages follow one another
            const int64_t panel0 = ((int64_t)e * ((p.N + kPanelRows - 1) / kPanelRows) + nt * NT / kPanelRows) * nstages;
            const int in_panel = nt * NT % kPanelRows;
            const uint8_t* sfb = MODE == kDense ? p.sfb + (int64_t)(nt * NT / 128) * p.kb * 512
                                                : p.sfb + panel0 * kPanelScales + in_panel / 128 * 1024;
            const int ahead = early ? min(STAGES, nstages) : 0;
            for (int s = 0; s < nstages; ++s, ++it) {
                if (!warp_wait(&s_empty[st], parity, failed)) { ok = false; break; }
                const uint32_t base = usmem + st * kStage, bar = smem_u32(&s_full[st]);
                const int kgs = min(2, p.kb - 2 * s), sfn = kgs * 512;
                if (PAIR) {
                    if (issue) load_pair(mt, nt, s);
                } else if (issue) {
                    const int sfbytes = MODE == kDense ? sfn * sft : S::kSfbBytes;
                    mbar_arrive_expect_tx(&s_full[st], (WRITE_A ? 0 : copies * (S::kA / 4) + kgs * S::kSfaKg) + S::kB + sfbytes);
                    if (MODE == kDense) {
                        tma_2d(base + oB, &tb, s * 128, nt * NT, bar);
#pragma unroll
                        for (int b = 0; b < S::kSfTiles; ++b)
                            if (b < sft) bulk_copy(base + oSfB + 1024 * b, sfb + ((int64_t)b * p.kb + 2 * s) * 512, sfn, bar);
                    } else {
                        tma_2d(base + oB, &tb, 0, (int)((panel0 + s) * kPanelRows) + in_panel, bar);
                        bulk_copy(base + oSfB, sfb + (int64_t)s * kPanelScales, S::kSfbBytes, bar);
                    }
                    if (!WRITE_A && s >= ahead) load_a(st, mt, s, copies);
                }
                __syncwarp();
                if (!WRITE_A && s < ahead && s == ahead - 1) {
                    asm volatile("griddepcontrol.wait;" ::: "memory");
                    if (ahead_of_list && tile + step < tiles) next = tile_of((int)((tile + step) / p.nt_count));
                    if (issue)
                        for (int a = 0; a < ahead; ++a) load_a(a, mt, a, copies);
                    __syncwarp();
                }
                if (++st == STAGES) {
                    st = 0;
                    parity ^= 1;
                }
            }
        }
        if ((MODE == kDown || ahead_of_list) && it == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
        // leave only when the copies have landed: a later owner of this shared memory must not be hit
        if (issue) {
            for (uint32_t b = 0; b < STAGES && b < it; ++b) {
                const uint32_t j = it - 1 - b;
                bool in = false;
                // a pair's are complete when its MMAs have read them, which also leaves no arrival to come
                uint64_t* const bar = PAIR ? &s_empty[j % STAGES] : &s_full[j % STAGES];
                for (uint32_t n = 0; n < kSpinLimit && !in; ++n) in = mbar_try_wait(bar, j / STAGES & 1);
                if (!in) *failed = 1;
            }
        }
        __syncwarp();
    } else if (warp == 1 && rank == 0) {  // of a pair, CTA 0 issues for both
        // The whole warp walks the loop, so that addresses and descriptors stay in uniform
        // registers, and one elected lane issues.
        constexpr uint32_t idesc = idesc_mxf4(PAIR ? 256 : 128, NT);
        const uint32_t utmem = __shfl_sync(0xffffffffu, tmem, 0), usmem = __shfl_sync(0xffffffffu, smem_u32(smem), 0);
        const uint32_t uabuf = __shfl_sync(0xffffffffu, smem_u32(abuf), 0);
        const bool issue = elect_one();
        uint32_t n = 0, st = 0, parity = 0;  // tiles so far; stage and phase of the ring
        bool ok = true;
        int next = first < tiles ? tile_of((int)(first / p.nt_count)).y : 0;
        for (int64_t tile = first; ok && tile < tiles; tile += step, ++n) {
            const uint32_t acc = n % S::kAcc, d = utmem + acc * NT;
            if (MODE != kDense && !FUSED) {
                const int rows = next;
                if (tile + step < tiles) next = tile_of((int)((tile + step) / p.nt_count)).y;
                if (__shfl_sync(0xffffffffu, rows, 0) == 0) break;
            }
            // half a scale tile (NT = 64): its rows' columns are 0-1 or 2-3 of the tile's four
            const uint32_t half = NT == 64 ? (uint32_t)(tile % p.nt_count & 1) * 2 : 0;
            if (!warp_wait<PAIR>(&s_accempty[acc], (n / S::kAcc & 1) ^ 1, failed)) break;
            if (WRITE_A && !warp_wait(&s_afull[n & 1], n >> 1 & 1, failed)) break;
            gemm::tc_fence_after();
            for (int s = 0; s < nstages; ++s) {
                if (!warp_wait(&s_full[st], parity, failed)) { ok = false; break; }
                gemm::tc_fence_after();
                const uint32_t ring = usmem + st * kStage, buf = uabuf + (n & 1) * S::a_buffer(nstages);
                const uint32_t sa = WRITE_A ? buf + s * S::kA : ring;
                const uint32_t sfa = WRITE_A ? buf + nstages * S::kA + s * 2 * S::kSfaKg : ring + oSfA;
                const uint64_t da = gemm::tc_desc_sw128(sa), db = gemm::tc_desc_sw128(ring + oB);
                const uint64_t dsa = sf_desc(sfa), dsb = sf_desc(ring + oSfB);
                const uint32_t tsa = utmem + kSfBase + st * S::kSfCols, tsb = tsa + 8;
                constexpr int kColsB = 4 * S::kSfTiles;  // TMEM columns of B's scales per 128 elements
                const int nkb = min(2, p.kb - 2 * s), nk = min(4, k64 - 4 * s);
                if (issue) {
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        if (i < nkb) {
                            cp_scales<PAIR>(tsa + 4 * i, dsa + S::kSfaKg / 16 * i);
#pragma unroll
                            for (int b = 0; b < S::kSfTiles; ++b) cp_scales<PAIR>(tsb + kColsB * i + 4 * b, dsb + 64 * b + 32 * i);
                        }
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (j < nk)  // 64 elements are 32 bytes inside the swizzle atom
                            mma_mxf4<PAIR>(d, da + 2 * j, db + 2 * j, idesc | (uint32_t)(j & 1) * 2 << 4 | (uint32_t)(j & 1) * 2 << 29,
                                     tsa + 4 * (j >> 1), tsb + kColsB * (j >> 1) + half, s > 0 || j > 0);
                    commit<PAIR>(&s_empty[st]);
                }
                __syncwarp();
                if (++st == STAGES) {
                    st = 0;
                    parity ^= 1;
                }
            }
            if (ok && issue) {
                if (WRITE_A) commit<false>(&s_aempty[n & 1]);
                commit<PAIR>(&s_accfull[acc]);
            }
            __syncwarp();
        }
        if (*failed && issue) {  // the MMAs in flight end before the accumulators are given back
            if (PAIR)
                asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(&s_done)) : "memory");
            else
                gemm::tc_commit(&s_done);
            for (uint32_t w = 0; w < kSpinLimit && !mbar_try_wait(&s_done, 0); ++w) {}
        }
        __syncwarp();
    } else if (WRITE_A && warp < 4) {
        // The rows of each tile's piece, quantised for the whole depth into one of the two buffers while the
        // MMAs read the other; a thread takes 8 elements, four loads in flight.
        constexpr int kFly = 4;
        const int t64 = tid - 64;
        uint32_t n = 0;
        for (int64_t tile = first; tile < tiles; tile += step, ++n) {
            const int mt = (int)(tile / p.nt_count);
            if (n >= 2 && !warp_wait(&s_aempty[n & 1], (n - 2) >> 1 & 1, failed)) break;
            uint8_t* codes = abuf + (n & 1) * S::a_buffer(nstages);
            uint8_t* scales = codes + nstages * S::kA;
            const int per = nstages * 32, units = route.rows[mt] * per;  // a multiple of 32: a warp is in or out as a whole
            for (int u0 = t64; u0 - (t64 & 31) < units; u0 += 64 * kFly) {
                uint4 q[kFly];
#pragma unroll
                for (int f = 0; f < kFly; ++f) {
                    const int u = u0 + 64 * f, r = u / per, k = (u - r * per) * 8;
                    q[f] = make_uint4(0u, 0u, 0u, 0u);
                    if (u < units && k < p.K) {
                        const int64_t t = route.pair[mt * kFusedPairs + r] / p.topk;
                        q[f] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.x) + t * p.K + k));
                    }
                }
#pragma unroll
                for (int f = 0; f < kFly; ++f) {
                    const int u = u0 + 64 * f, r = u / per, i = u - r * per;  // element 8 i of row r
                    if (u >= units) break;
                    float v[8];
                    const uint32_t w4[4] = {q[f].x, q[f].y, q[f].z, q[f].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        v[2 * j] = scale_to_f32((uint16_t)(w4[j] & 0xffffu), p.act_bf16);
                        v[2 * j + 1] = scale_to_f32((uint16_t)(w4[j] >> 16), p.act_bf16);
                    }
                    uint32_t sc;
                    const uint32_t c = quant8(v, sc);
                    const int st = i >> 5, piece = i >> 2 & 7;  // 16-byte piece of the stage's 128 bytes
                    *reinterpret_cast<uint32_t*>(codes + st * S::kA + r * 128 + ((piece ^ r) << 4) + (i & 3) * 4) = c;
                    if ((i & 3) == 0) scales[(st * 2 + (piece >> 2)) * S::kSfaKg + r * 16 + (piece & 3)] = (uint8_t)sc;
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_afull[n & 1]);
        }
    } else if (TM < 128 && warp >= 4) {
        // Few rows: warp 4 reads their TMEM lanes into shared memory, and all epilogue threads share the
        // arithmetic: 8 threads a 32-block of a row (gate_up), a warp a row (down).
        float* rows = reinterpret_cast<float*>(smem + STAGES * kStage + S::tail(WRITE_A));
        const int et = tid - 128;
        constexpr int kEt = 32 * S::kEpiWarps;
        uint32_t n = 0;
        int2 of = first < tiles ? tile_of((int)(first / p.nt_count)) : make_int2(0, 0);
        for (int64_t tile = first; tile < tiles && of.y; tile += step, ++n) {
            const int mt = (int)(tile / p.nt_count), nt = (int)(tile - (int64_t)mt * p.nt_count), mrows = of.y;
            const uint32_t acc = n % S::kAcc;
            if (tile + step < tiles) of = tile_of((int)((tile + step) / p.nt_count));
            if (warp == 4) {
                const bool go = warp_wait(&s_accfull[acc], n / S::kAcc & 1, failed);
                gemm::tc_fence_after();
                if (go) {
#pragma unroll
                    for (int c = 0; c < NT; c += 32) {
                        float v[32];
                        load_columns<32>(tmem + acc * NT + c, v);
                        if (lane < mrows)
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                *reinterpret_cast<float4*>(rows + lane * S::kRowPitch + c + 4 * j) =
                                    make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                    }
                }
                gemm::tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&s_accempty[acc]);
                    s_go = go;
                }
            }
            named_bar_sync(1, kEt);
            if (!*reinterpret_cast<volatile int*>(&s_go)) break;
            if (MODE == kGateUp) {
                for (int i = et >> 3; i < mrows * (NT / 64); i += kEt / 8) {
                    const int r = i / (NT / 64), b = i % (NT / 64), i0 = (nt * NT) / 2 + b * 32, j = et & 7;
                    const float* src = rows + r * S::kRowPitch + 64 * b + 4 * j;
                    const float4 g = *reinterpret_cast<const float4*>(src), u = *reinterpret_cast<const float4*>(src + 32);
                    const float h[4] = {silu_up(g.x, u.x), silu_up(g.y, u.y), silu_up(g.z, u.z), silu_up(g.w, u.w)};
                    uint32_t m = 0;
#pragma unroll
                    for (int k = 0; k < 4; ++k) m = max(m, __float_as_uint(h[k]) & 0x7fffffffu);
                    const uint32_t octet = 0xffu << (lane & 24);
#pragma unroll
                    for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(octet, m, o));
                    if (i0 >= p.I) continue;
                    const uint32_t sc = scale_of_amax(m);
                    const float k = inv_scale(sc);
                    const int64_t row = (int64_t)mt * TM + r;
                    *reinterpret_cast<uint16_t*>(p.hq + row * (p.I / 2) + i0 / 2 + 2 * j) =
                        (uint16_t)(cvt_e2m1x2(h[0] * k, h[1] * k) | cvt_e2m1x2(h[2] * k, h[3] * k) << 8);
                    if (j == 0) {
                        uint8_t* hs = p.hs + (TM == 8 ? ((int64_t)mt * p.hkb + (i0 >> 7)) * 128 + r * 16 + (i0 >> 5 & 3)
                                                      : tile_row_at(mt, r, i0 >> 5, p.hkb));
                        hs[0] = (uint8_t)sc;
                        // the MMAs take K in steps of 64: the scale behind an odd last block must be a number
                        if (i0 + 32 == p.I && (p.I & 32)) hs[1] = 0;
                    }
                }
            } else {
                for (int r = warp - 4; r < mrows; r += S::kEpiWarps) {
                    const int64_t row = FUSED ? (int64_t)route.pair[mt * kFusedPairs + r] : (int64_t)mt * TM + r;  // fused parts lie by pair
#pragma unroll
                    for (int c = lane * 4; c < NT; c += 128)
                        if (nt * NT + c < p.N)  // rows are multiples of 32
                            *reinterpret_cast<float4*>(static_cast<float*>(p.out) + row * p.N + nt * NT + c) =
                                *reinterpret_cast<const float4*>(rows + r * S::kRowPitch + c);
                }
            }
            named_bar_sync(1, kEt);  // the rows are read (and a part is written) before warp 4 goes on
            if (FUSED && MODE == kDown) {
                // the CTA that finishes a column tile's last part sums them
                if (et == 0) {
                    __threadfence();
                    const bool last = atomicAdd(p.cnt + nt, 1u) + 1 == (unsigned int)mt_count;
                    __threadfence();
                    if (last) p.cnt[nt] = 0;
                    s_last = last;
                }
                named_bar_sync(1, kEt);
                if (*reinterpret_cast<volatile int*>(&s_last)) {
                    if (p.y_dtype == MOE_F32) fused_combine<MOE_F32>(route, p, nt * NT, warp - 4, S::kEpiWarps);
                    else if (p.y_dtype == MOE_BF16) fused_combine<MOE_BF16>(route, p, nt * NT, warp - 4, S::kEpiWarps);
                    else fused_combine<MOE_F16>(route, p, nt * NT, warp - 4, S::kEpiWarps);
                }
            }
        }
        if (FUSED && MODE == kDown && mt_count == 0)  // no pair is this engine's
            for (int nt = blockIdx.x; nt < p.nt_count; nt += gridDim.x) {
                if (p.y_dtype == MOE_F32) fused_combine<MOE_F32>(route, p, nt * NT, warp - 4, S::kEpiWarps);
                else if (p.y_dtype == MOE_BF16) fused_combine<MOE_BF16>(route, p, nt * NT, warp - 4, S::kEpiWarps);
                else fused_combine<MOE_F16>(route, p, nt * NT, warp - 4, S::kEpiWarps);
            }
    } else if (warp >= 4) {
        const int r = (warp & 3) * 32 + lane, c0 = ((warp - 4) >> 2) * S::kCols;
        const uint32_t quarter = (uint32_t)((warp & 3) * 32);
        uint8_t* const staging0 = smem + STAGES * kStage + (warp - 4) * S::BUFS * 2048;  // wide tiles only: no tail
        uint8_t* staging = staging0;
        uint32_t stores = 0;
        // this lane's 64 bytes of the staging area, its four 16-byte pieces swizzled as the map says
        auto stage_row = [&](const uint32_t (&w)[16]) {
            staging = staging0 + stores++ % S::BUFS * 2048;
            asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(S::BUFS - 1) : "memory");  // lane 0's store from here is done
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<uint4*>(staging + lane * 64 + ((j ^ (lane >> 1 & 3)) << 4)) =
                    make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
        };
        uint32_t n = 0;
        for (int64_t tile = first; tile < tiles; tile += step, ++n) {
            const int mt = (int)(tile / p.nt_count), nt = (int)(tile - (int64_t)mt * p.nt_count);
            const uint32_t acc = n % S::kAcc;
            const int all_rows = tile_of(mt).y;
            if (all_rows == 0) break;
            const int mrows = PAIR ? min(TM, max(0, all_rows - rank * TM)) : all_rows;
            if (!warp_wait(&s_accfull[acc], n / S::kAcc & 1, failed)) break;
            gemm::tc_fence_after();
            float v[S::kCols];
            const bool any = (int)quarter < mrows;  // rows of this warp's quarter exist
            if (any) load_columns<S::kCols>(tmem + acc * NT + c0 + (quarter << 16), v);
            gemm::tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (PAIR) arrive_leader(&s_accempty[acc]);
                else mbar_arrive(&s_accempty[acc]);
            }
            const int64_t row = (int64_t)mt * S::kTileRows + rank * TM + r;
            if (MODE == kGateUp) {
                if (r >= mrows) continue;
#pragma unroll
                for (int b = 0; b < S::kCols / 64; ++b) {
                    const int i0 = (nt * NT + c0) / 2 + b * 32;
                    if (i0 >= p.I) break;
                    float h[32];
                    uint32_t m = 0;
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        h[j] = silu_up(v[64 * b + j], v[64 * b + 32 + j]);
                        m = max(m, __float_as_uint(h[j]) & 0x7fffffffu);
                    }
                    const uint32_t sc = scale_of_amax(m);
                    const float k = inv_scale(sc);
                    uint32_t q[4];
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        q[w] = 0;
#pragma unroll
                        for (int j = 0; j < 4; ++j) q[w] |= cvt_e2m1x2(h[8 * w + 2 * j] * k, h[8 * w + 2 * j + 1] * k) << (8 * j);
                    }
                    *reinterpret_cast<uint4*>(p.hq + row * (p.I / 2) + i0 / 2) = make_uint4(q[0], q[1], q[2], q[3]);
                    uint8_t* hs = p.hs + tile_row_at(mt, r, i0 >> 5, p.hkb);
                    hs[0] = (uint8_t)sc;
                    // the MMAs take K in steps of 64: the scale behind an odd last block must be a number
                    if (i0 + 32 == p.I && (p.I & 32)) hs[1] = 0;
                }
                continue;
            }
            if (S::kStaging && any && (MODE == kDown || p.tma_out)) {
                const int y0 = mt * S::kTileRows + rank * TM + (int)quarter;
                auto store_fp32 = [&](const float* f, int n0) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (n0 + 16 * h >= p.N) break;
                        uint32_t w[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) w[j] = __float_as_uint(f[16 * h + j]);
                        stage_row(w);
                        if (lane == 0) tma_store_2d(&to, smem_u32(staging), n0 + 16 * h, y0);
                    }
                };
#pragma unroll
                for (int c = 0; c < S::kCols; c += 32) {
                    const int n0 = nt * NT + c0 + c;
                    if (n0 >= p.N) break;
                    if constexpr (MODE == kDown) {
                        store_fp32(v + c, n0);
                    } else if (p.out_dtype == MOE_F32) {
                        store_fp32(v + c, n0);
                    } else {
                        uint32_t w[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            w[j] = p.out_dtype == MOE_BF16 ? pack16<MOE_BF16>(v[c + 2 * j], v[c + 2 * j + 1])
                                                           : pack16<MOE_F16>(v[c + 2 * j], v[c + 2 * j + 1]);
                        stage_row(w);
                        if (lane == 0) tma_store_2d(&to, smem_u32(staging), n0, y0);
                    }
                }
                continue;
            }
            if (MODE == kDense && r < mrows) {
                const int esz = p.out_dtype == MOE_F32 ? 4 : 2;
                const bool vec = (int64_t)p.N * esz % 16 == 0;
#pragma unroll
                for (int c = 0; c < S::kCols; c += 32) {
                    const int n0 = nt * NT + c0 + c, left = min(32, p.N - n0);
                    if (left <= 0) break;
                    if (p.out_dtype == MOE_F32) store_row<MOE_F32>(p.out, row * p.N + n0, v + c, left, vec);
                    else if (p.out_dtype == MOE_BF16) store_row<MOE_BF16>(p.out, row * p.N + n0, v + c, left, vec);
                    else store_row<MOE_F16>(p.out, row * p.N + n0, v + c, left, vec);
                }
            }
        }
    }
    if (S::kStaging && warp >= 4 && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncthreads();
    if (s_failed && tid == 0) set_err(p.err, kErrFullWait);
    gemm::tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();  // the peer's MMAs, reads and arrivals are over
    if (warp == 2) {
        gemm::tc_fence_after();
        if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kTmemCols) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kTmemCols) : "memory");
    }
}

// ------------------------------------------------------------------ expert layer: tokens
// Routed pairs in a stable order by expert, each expert's in tiles of 32 or 128 rows; the token rows
// quantised into the rows of their pairs.  A CTA takes a run of `tokens` tokens.  It needs, per
// expert, the pairs before its run and the pairs in all: for short calls it counts all pairs
// itself, for long ones the runs' counts come from mx_count_kernel.
// T = 4096, H = 2048, top-8: 22 us (its 52 MB would take 8),
// the counts 3.6 us; T = 201: 7.5 us.  A token is quantised once and written to the row of each of its pairs.
constexpr int kPrepThreads = 512, kPrepWarps = kPrepThreads / 32;

struct PrepParams {
    const void* x;
    const int32_t* ids;
    int T, K, H, E, e_off, emap_n, tokens;
    int tile_log2;  // rows of an m tile: 32 or 128
    const int32_t* emap;
    const int32_t* counts;  // [runs][E], or null: at most kPrepSelf pairs
    int2* mt_list;  // expert and rows of each m tile, then rows 0 up to the bound
    int mt_bound;
    int32_t* ppos;  // row of each pair, -1 for pairs of other engines
    uint8_t* xq;    // [rows][H / 2]
    uint8_t* xs;    // scale tiles, kb along H
    int kb;
};

// Pairs of each expert in a run of tokens.
__global__ void __launch_bounds__(kPrepThreads) mx_count_kernel(const PrepParams p, int32_t* counts) {
    extern __shared__ int32_t csm[];
    for (int e = threadIdx.x; e < p.E; e += kPrepThreads) csm[e] = 0;
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int i0 = blockIdx.x * p.tokens * p.K, i1 = min(p.T * p.K, i0 + p.tokens * p.K);
    for (int i = i0 + threadIdx.x; i < i1; i += kPrepThreads) {
        const int e = local_expert(p.ids[i], p.e_off, p.E, p.emap, p.emap_n, i, p.K);
        if (e >= 0) atomicAdd(&csm[e], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.E; e += kPrepThreads) counts[(int64_t)blockIdx.x * p.E + e] = csm[e];
}

// A block of 16-bit values -> its codes, and the scale.
template <int DT>
MOE_DEV uint32_t quant32(const uint4 (&raw)[4], uint4& codes) {
    uint32_t w[16];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        w[4 * j] = raw[j].x;
        w[4 * j + 1] = raw[j].y;
        w[4 * j + 2] = raw[j].z;
        w[4 * j + 3] = raw[j].w;
    }
    uint32_t m = 0;  // both types order by their bits, sign apart
#pragma unroll
    for (int j = 0; j < 16; ++j) m = __vmaxu2(m, w[j] & 0x7fff7fffu);
    const uint16_t top = (uint16_t)max(m & 0xffffu, m >> 16);
    const uint32_t sc = scale_of_amax(__float_as_uint(scale_to_f32(top, DT == MOE_BF16)));
    const float k = inv_scale(sc);
    uint32_t q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        q[j] = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            q[j] |= cvt_e2m1x2(scale_to_f32((uint16_t)(w[4 * j + i] & 0xffffu), DT == MOE_BF16) * k,
                               scale_to_f32((uint16_t)(w[4 * j + i] >> 16), DT == MOE_BF16) * k) << (8 * i);
    }
    codes = make_uint4(q[0], q[1], q[2], q[3]);
    return sc;
}

template <int DT>
__global__ void __launch_bounds__(kPrepThreads) mx_prep_kernel(const PrepParams p) {
    // [warps][E] pairs of each warp's share, then their first rows | [E] first tile | rows of the run's pairs
    extern __shared__ int32_t psm[];
    __shared__ int32_t s_sum[kPrepWarps];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, E = p.E;
    int32_t* first = psm + kPrepWarps * E;
    int32_t* pos = first + E;
    for (int e = tid; e < kPrepWarps * E; e += kPrepThreads) psm[e] = 0;
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int t0 = blockIdx.x * p.tokens, t1 = min(p.T, t0 + p.tokens), TK = p.T * p.K;
    // The token rows: a lane takes a block, a warp `group` (1 or 2) times 32 blocks of a token; the first are
    // fetched before the routing.
    const int nb = p.H >> 5, chunks = (nb + 31) >> 5, group = (t1 - t0) * chunks >= 2 * kPrepWarps ? 2 : 1;
    const int groups = (chunks + group - 1) / group, items = (t1 - t0) * groups;
    uint4 raw[2][4];
    auto fetch = [&](int item) {
        const int t = item / groups, b0 = (item - t * groups) * 32 * group + lane;
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.x) + (int64_t)(t0 + t) * p.H) + b0 * 4;
#pragma unroll
        for (int f = 0; f < 2; ++f)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                raw[f][j] = f < group && b0 + 32 * f < nb ? __ldg(src + 128 * f + j) : make_uint4(0u, 0u, 0u, 0u);
    };
    if (warp < items) fetch(warp);
    // the pairs whose order this CTA works out: all (short calls) or its own run's
    const int a0 = p.counts ? t0 * p.K : 0, a1 = p.counts ? t1 * p.K : TK;
    const int share = ((a1 - a0 + kPrepWarps - 1) / kPrepWarps + 31) / 32 * 32;
    const int i0 = min(a1, a0 + warp * share), i1 = min(a1, i0 + share);
    int32_t* hist = psm + warp * E;
    constexpr int kIds = kPrepSelf / kPrepThreads;  // a lane's ids in short calls; longer runs reload
    int mine[kIds];
#pragma unroll
    for (int f = 0; f < kIds; ++f) {
        const int i = i0 + f * 32 + lane;
        mine[f] = i < i1 ? p.ids[i] : -1;
    }
    for (int i = i0 + lane, f = 0; i - lane < i1; i += 32, ++f) {
        int id = -1;
#pragma unroll
        for (int g = 0; g < kIds; ++g)
            if (g == f) id = mine[g];
        if (f >= kIds && i < i1) id = p.ids[i];
        const int e = i < i1 ? local_expert(id, p.e_off, E, p.emap, p.emap_n, i, p.K) : -1;
        const unsigned peers = __match_any_sync(0xffffffffu, e);
        const int rank = __popc(peers & ((1u << lane) - 1u));
        const int before = e >= 0 ? hist[e] : 0;
        __syncwarp();
        if (i < i1) pos[i - a0] = e >= 0 ? (before + rank) << 10 | e : -1;  // rank within the warp's share
        if (e >= 0 && rank == 0) hist[e] = before + __popc(peers);
        __syncwarp();
    }
    __syncthreads();
    // the runs' counts, before this run and in all: groups of threads take every G-th run
    int32_t* before = pos + (a1 - a0);  // [2][E]
    if (p.counts) {
        for (int e = tid; e < 2 * E; e += kPrepThreads) before[e] = 0;
        __syncthreads();
        const int pad = (E + 31) & ~31, G = max(1, kPrepThreads / pad), runs = gridDim.x;
        for (int u = tid; u < G * pad || u < pad; u += kPrepThreads) {
            const int g = u / pad, e = u - g * pad;
            if (e >= E) continue;
            int base = 0, total = 0;
#pragma unroll 8
            for (int c = g; c < runs; c += G) {
                const int n = __ldcg(p.counts + (int64_t)c * E + e);
                if (c < (int)blockIdx.x) base += n;
                total += n;
            }
            atomicAdd(&before[e], base);
            atomicAdd(&before[E + e], total);
        }
        __syncthreads();
    }
    // per expert: rows before each warp's share, tiles; scan of the tiles over the experts
    int carry = 0;
    for (int e0 = 0; e0 < E; e0 += kPrepThreads) {
        const int e = e0 + tid;
        int base = 0, total = 0;
        if (e < E) {
            if (p.counts) {
                base = before[e];
                total = before[E + e];
            }
            int run = base;
            for (int w = 0; w < kPrepWarps; ++w) {
                const int n = psm[w * E + e];
                psm[w * E + e] = run;
                run += n;
            }
            if (!p.counts) total = run;
        }
        const int tile_rows = 1 << p.tile_log2, nt = (total + tile_rows - 1) >> p.tile_log2;
        int incl = nt;
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) s_sum[warp] = incl;
        __syncthreads();
        int all = 0;
        for (int w = 0; w < kPrepWarps; ++w) {
            if (w < warp) incl += s_sum[w];
            all += s_sum[w];
        }
        __syncthreads();
        const int tile = carry + incl - nt;
        if (e < E) {
            first[e] = tile << p.tile_log2;
            if (blockIdx.x == 0)
                for (int m = 0; m < nt; ++m) p.mt_list[tile + m] = make_int2(e, min(tile_rows, total - (m << p.tile_log2)));
        }
        carry += all;
    }
    if (blockIdx.x == 0)
        for (int m = carry + tid; m < p.mt_bound; m += kPrepThreads) p.mt_list[m] = make_int2(0, 0);
    __syncthreads();
    for (int i = i0 + lane; i < i1; i += 32) {
        const int v = pos[i - a0], e = v & 1023;
        pos[i - a0] = v < 0 ? -1 : first[e] + hist[e] + (v >> 10);
    }
    __syncthreads();
    pos += t0 * p.K - a0;  // the run's own pairs
    for (int i = tid; i < (t1 - t0) * p.K; i += kPrepThreads) p.ppos[t0 * p.K + i] = pos[i];
    for (int item = warp; item < items; item += kPrepWarps) {
        const int t = item / groups, b0 = (item - t * groups) * 32 * group + lane;
        uint4 codes[2];
        uint32_t words[2];
#pragma unroll
        for (int f = 0; f < 2; ++f) {
            const uint32_t sc = quant32<DT>(raw[f], codes[f]);
            words[f] = sc | __shfl_down_sync(0xffffffffu, sc, 1, 4) << 8;  // the scales of four lanes' blocks
            words[f] |= __shfl_down_sync(0xffffffffu, words[f], 2, 4) << 16;
        }
        if (item + kPrepWarps < items) fetch(item + kPrepWarps);
        for (int k = 0; k < p.K; ++k) {
            const int row = pos[t * p.K + k];
            if (row < 0) continue;
            uint4* to = reinterpret_cast<uint4*>(p.xq + (int64_t)row * (p.H / 2)) + b0;
            uint8_t* sc = p.xs + tile_row_at(row >> p.tile_log2, row & ((1 << p.tile_log2) - 1), b0, p.kb);
#pragma unroll
            for (int f = 0; f < 2; ++f) {
                if (f >= group) break;
                if (b0 + 32 * f < nb) to[32 * f] = codes[f];
                if ((lane & 3) == 0 && (b0 >> 2) + 8 * f < p.kb) *reinterpret_cast<uint32_t*>(sc + 4096 * f) = words[f];
            }
        }
    }
}

// y[t] = sum over the token's pairs, in their order, of w * part[row].  A warp takes 256 columns of a
// token, a lane 8 of them; lane k holds the k-th pair's row and weight, and 8 parts are in flight.
// T = 4096, H = 2048, top-8: 45 us for 285 MB, 6.3 TB/s.  (Parts of 16 bits with an exponent per 32 columns took 31,
// but lost a column beside one a few hundred times larger more than the output's rounding does.)
template <int DT>
__global__ void __launch_bounds__(256, 2) mx_combine_kernel(const float* part, const int32_t* ppos, const float* tw, int T, int K, int H,
                                                            void* y) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    constexpr int kFly = 8;
    const int lane = threadIdx.x & 31, chunks = (H + 255) >> 8;
    const int64_t total = (int64_t)T * chunks;
    for (int64_t i = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 5; i < total; i += (int64_t)gridDim.x * blockDim.x >> 5) {
        const int64_t t = i / chunks;
        const int n = ((int)(i - t * chunks) << 8) + lane * 8;
        const bool in = n < H;
        const int at8 = in ? n : 0;
        float a[8] = {};
        for (int k0 = 0; k0 < K; k0 += 32) {
            const int mypos = k0 + lane < K ? __ldg(ppos + t * K + k0 + lane) : -1;
            const float myw = k0 + lane < K ? __ldg(tw + t * K + k0 + lane) : 0.f;
            for (int k1 = 0; k1 < min(32, K - k0); k1 += kFly) {
                // no branch stands between the loads: of an absent pair row 0 is read, and weighs nothing
                float4 q[kFly][2];
                int pos[kFly];
#pragma unroll
                for (int f = 0; f < kFly; ++f) {
                    pos[f] = __shfl_sync(0xffffffffu, mypos, k1 + f);
                    const float4* src = reinterpret_cast<const float4*>(part + (int64_t)max(pos[f], 0) * H + at8);
                    q[f][0] = __ldcs(src);
                    q[f][1] = __ldcs(src + 1);
                }
#pragma unroll
                for (int f = 0; f < kFly; ++f) {
                    float w = __shfl_sync(0xffffffffu, myw, k1 + f);
                    if (pos[f] < 0) {
                        w = 0.f;
                        q[f][0] = q[f][1] = make_float4(0.f, 0.f, 0.f, 0.f);
                    }
                    const float v[8] = {q[f][0].x, q[f][0].y, q[f][0].z, q[f][0].w, q[f][1].x, q[f][1].y, q[f][1].z, q[f][1].w};
#pragma unroll
                    for (int j = 0; j < 8; ++j) a[j] = fmaf(w, v[j], a[j]);
                }
            }
        }
        if (!in) continue;
        const int64_t at = (t * H + n) >> 3;
        if (DT == MOE_F32) {
            float4* d = reinterpret_cast<float4*>(y) + 2 * at;
            d[0] = make_float4(a[0], a[1], a[2], a[3]);
            d[1] = make_float4(a[4], a[5], a[6], a[7]);
        } else {
            reinterpret_cast<uint4*>(y)[at] = make_uint4(pack16<DT>(a[0], a[1]), pack16<DT>(a[2], a[3]), pack16<DT>(a[4], a[5]),
                                                         pack16<DT>(a[6], a[7]));
        }
    }
}

}  // namespace mx
}  // namespace moe
