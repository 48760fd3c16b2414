// Products of MXFP4 matrices on the tensor cores (tcgen05.mma kind::mxf4, block scales applied
// by the MMA): the dense product a b^T, and the gate_up and down products of the expert layer.
//
// One persistent, warp-specialised kernel: a CTA per SM walks over the (128 x NT) output tiles.
//   warp 0      TMA producer: a stage is 256 elements of K, i.e. 128 bytes (one swizzle atom) of
//               each of the 128 rows of A and NT rows of B, and their scale tiles (512 bytes hold
//               128 rows x 128 elements);
//   warp 1      one thread copies the stage's scales to TMEM (tcgen05.cp) and issues its MMAs
//               (K = 64 each), fp32 accumulators in TMEM, two of them so that the epilogue of a
//               tile overlaps the products of the next;
//   warps 4-7   epilogue, a thread per row of the tile.
// The rows of A are tokens, so a thread of the epilogue holds whole 32-blocks of its token: the
// gate_up epilogue forms SiLU(gate) * up and quantises it without a word to other threads.
// gate_up weights lie in 64-row groups of 32 gate rows and the 32 up rows of the same units.
//
// All waits are bounded; one that runs out sets the error word, and every role leaves its loop.
#pragma once
#include <cuda.h>

#include "mxfp4.cuh"

namespace moe {
namespace mx {

enum Mode { kDense = 0, kGateUp = 1, kDown = 2 };
constexpr int kTileM = 128, kStageK = 256, kGemmThreads = 256;

struct GemmParams {
    int M, N, K;         // dense: rows of a; N rows of b (of one expert); depth
    int kb;              // scale tiles along K
    int nt_count, mt_count;
    const uint8_t* sfa;  // [m tiles][kb][512]
    const uint8_t* sfb;  // [experts][ceil(N / 128)][kb][512]
    const int32_t* mtiles;     // experts: number of m tiles, then expert and rows of each
    const int32_t* mt_expert;
    const int32_t* mt_rows;
    const int32_t* rowtok;     // token of each row of the m tiles
    void* out;           // dense [M][N] (out_dtype); down fp32 [m tiles * 128][N]
    int out_dtype;
    int I;               // gate_up: hq [m tiles * 128][I / 2], hs tiled with hkb tiles along I
    int hkb;
    uint8_t* hq;
    uint8_t* hs;
    int32_t* err;
};

template <int NT>
struct Shape {
    static constexpr int kA = kTileM * 128, kB = NT * 128;
    static constexpr int kSfB = (NT + 127) / 128 * 1024;
    static constexpr int kStage = kA + kB + 1024 + kSfB;
    static constexpr int kSfCols = 8 + kSfB / 128;  // TMEM columns of a stage's scales
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

MOE_DEV void mma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"((uint32_t)accumulate)
        : "memory");
}

MOE_DEV void cp_scales(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

MOE_DEV void tma_2d(uint32_t dst, const CUtensorMap* m, int x, int y, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(m), "r"(x), "r"(y), "r"(smem_u32(bar))
        : "memory");
}
MOE_DEV void tma_3d(uint32_t dst, const CUtensorMap* m, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(m), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}
// Four rows (the map's box is one row), 128 bytes of each.
MOE_DEV void tma_gather4(uint32_t dst, const CUtensorMap* m, int x, int4 r, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
        ::"r"(dst), "l"(m), "r"(x), "r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w), "r"(smem_u32(bar))
        : "memory");
}

// Bounded wait that also ends when another role of the CTA has given up.
MOE_DEV bool wait_or_fail(uint64_t* bar, uint32_t parity, volatile int* failed) {
    for (uint32_t it = 0; it < kSpinLimit; ++it) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((it & 15u) == 15u && *failed) return false;
        if (it > 8192) __nanosleep(128);
    }
    *failed = 1;
    return false;
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
MOE_DEV void store_row(void* out, int64_t at, const float (&v)[32], int n, bool vec) {
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

template <int MODE, int NT, int STAGES>
__global__ void __launch_bounds__(kGemmThreads, 1) mx_gemm_kernel(const __grid_constant__ CUtensorMap ta,
                                                                  const __grid_constant__ CUtensorMap tb,
                                                                  const GemmParams p) {
    using S = Shape<NT>;
    constexpr int kSfBase = 2 * NT;  // TMEM: two accumulators, then each stage's scales
    constexpr int kTmemCols = kSfBase + STAGES * S::kSfCols <= 256 ? 256 : 512;
    static_assert(kSfBase + STAGES * S::kSfCols <= 512, "TMEM");
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ __align__(8) uint64_t s_full[STAGES], s_empty[STAGES], s_accfull[2], s_accempty[2], s_done;
    __shared__ uint32_t s_tmem;
    __shared__ int s_failed;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&s_full[s], 1);
            mbar_init(&s_empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&s_accfull[a], 1);
            mbar_init(&s_accempty[a], 4);
        }
        mbar_init(&s_done, 1);
        s_failed = 0;
        fence_barrier_init();
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "n"(kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    gemm::tc_fence_before();
    __syncthreads();
    gemm::tc_fence_after();
    const uint32_t tmem = s_tmem;
    volatile int* failed = &s_failed;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    const int mt_count = MODE == kDense ? p.mt_count : p.mtiles[0];
    const int64_t tiles = (int64_t)mt_count * p.nt_count;
    const int nstages = (p.K + kStageK - 1) / kStageK, k64 = (p.K + 63) / 64;
    const int nb128 = (p.N + 127) / 128;
    uint32_t it = 0;  // stages so far (producer and MMA thread)

    if (warp == 0) {
        bool ok = true;
        for (int64_t tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x) {
            const int mt = (int)(tile / p.nt_count), nt = (int)(tile - (int64_t)mt * p.nt_count);
            const int e = MODE == kDense ? 0 : p.mt_expert[mt];
            const int mrows = MODE == kDense ? kTileM : p.mt_rows[mt];
            int copies = 1, abytes = S::kA;
            int4 rows = make_int4(0, 0, 0, 0);
            if (MODE == kGateUp) {  // 4 rows a copy; rows past the tile's last repeat it
                copies = (mrows + 3) >> 2;
                abytes = copies * 512;
                const int32_t* rt = p.rowtok + (int64_t)mt * kTileM;
                rows.x = rt[min(4 * lane, mrows - 1)];
                rows.y = rt[min(4 * lane + 1, mrows - 1)];
                rows.z = rt[min(4 * lane + 2, mrows - 1)];
                rows.w = rt[min(4 * lane + 3, mrows - 1)];
            } else if (MODE == kDown) {  // 16 rows a copy
                copies = (mrows + 15) >> 4;
                abytes = copies * 2048;
            }
            const uint8_t* sfa = p.sfa + (int64_t)mt * p.kb * 512;
            const uint8_t* sfb = p.sfb + ((int64_t)e * nb128 + (int64_t)nt * NT / 128) * p.kb * 512;
            for (int s = 0; s < nstages; ++s, ++it) {
                const int st = it % STAGES;
                if (!wait_or_fail(&s_empty[st], (it / STAGES & 1) ^ 1, failed)) { ok = false; break; }
                uint8_t* base = smem + (size_t)st * S::kStage;
                const int sfn = min(2, p.kb - 2 * s) * 512;
                if (lane == 0) {
                    mbar_arrive_expect_tx(&s_full[st], abytes + S::kB + sfn * (1 + S::kSfB / 1024));
                    tma_3d(smem_u32(base + S::kA), &tb, s * 128, nt * NT, e, &s_full[st]);
                    uint8_t* sf = base + S::kA + S::kB;
                    bulk_g2s(sf, sfa + (int64_t)s * 1024, sfn, &s_full[st]);
#pragma unroll
                    for (int b = 0; b < S::kSfB / 1024; ++b)
                        bulk_g2s(sf + 1024 + b * 1024, sfb + ((int64_t)b * p.kb + 2 * s) * 512, sfn, &s_full[st]);
                    if (MODE == kDense) tma_2d(smem_u32(base), &ta, s * 128, mt * kTileM, &s_full[st]);
                }
                __syncwarp();
                if (MODE == kGateUp && lane < copies) tma_gather4(smem_u32(base) + lane * 512, &ta, s * 128, rows, &s_full[st]);
                if (MODE == kDown && lane < copies)
                    tma_2d(smem_u32(base) + lane * 2048, &ta, s * 128, mt * kTileM + lane * 16, &s_full[st]);
                __syncwarp();
            }
        }
        // leave only when the copies have landed: a later owner of this shared memory must not be hit
        if (lane == 0 && it > 0) {
            for (uint32_t b = 0; b < STAGES && b < it; ++b) {
                const uint32_t j = it - 1 - b;
                bool in = false;
                for (uint32_t n = 0; n < kSpinLimit && !in; ++n) in = mbar_try_wait(&s_full[j % STAGES], j / STAGES & 1);
                if (!in) *failed = 1;
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc = idesc_mxf4(kTileM, NT);
            uint32_t n = 0;  // tiles so far
            bool ok = true;
            for (int64_t tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x, ++n) {
                const uint32_t acc = n & 1, d = tmem + acc * NT;
                if (!wait_or_fail(&s_accempty[acc], (n >> 1 & 1) ^ 1, failed)) break;
                gemm::tc_fence_after();
                for (int s = 0; s < nstages; ++s, ++it) {
                    const int st = it % STAGES;
                    if (!wait_or_fail(&s_full[st], it / STAGES & 1, failed)) { ok = false; break; }
                    gemm::tc_fence_after();
                    const uint32_t sa = smem_u32(smem + (size_t)st * S::kStage), sb = sa + S::kA, sf = sb + S::kB;
                    const uint32_t tsa = tmem + kSfBase + st * S::kSfCols, tsb = tsa + 8;
                    const int nkb = min(2, p.kb - 2 * s);
                    for (int i = 0; i < nkb; ++i) {
                        cp_scales(tsa + 4 * i, sf_desc(sf + 512 * i));
#pragma unroll
                        for (int b = 0; b < S::kSfB / 1024; ++b)
                            cp_scales(tsb + (S::kSfB / 256) * i + 4 * b, sf_desc(sf + 1024 + 1024 * b + 512 * i));
                    }
                    const int nk = min(4, k64 - 4 * s);
                    for (int j = 0; j < nk; ++j) {
                        const uint32_t id = (uint32_t)(j & 1) * 2;
                        mma_mxf4(d, gemm::tc_desc_sw128(sa + 32 * j), gemm::tc_desc_sw128(sb + 32 * j),
                                 idesc | id << 4 | id << 29, tsa + 4 * (j >> 1), tsb + (S::kSfB / 256) * (j >> 1), s > 0 || j > 0);
                    }
                    gemm::tc_commit(&s_empty[st]);
                }
                if (ok) gemm::tc_commit(&s_accfull[acc]);
            }
            if (*failed) {  // the MMAs in flight end before the accumulators are given back
                gemm::tc_commit(&s_done);
                for (uint32_t w = 0; w < kSpinLimit && !mbar_try_wait(&s_done, 0); ++w) {}
            }
        }
        __syncwarp();
    } else if (warp >= 4) {
        const int r = (warp & 3) * 32 + lane;
        uint32_t n = 0;
        for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++n) {
            const int mt = (int)(tile / p.nt_count), nt = (int)(tile - (int64_t)mt * p.nt_count);
            const uint32_t acc = n & 1;
            if (!wait_or_fail(&s_accfull[acc], n >> 1 & 1, failed)) break;
            gemm::tc_fence_after();
            const uint32_t taddr = tmem + acc * NT + ((uint32_t)((warp & 3) * 32) << 16);
            const int mrows = MODE == kDense ? p.M - mt * kTileM : p.mt_rows[mt];
            const bool live = r < mrows;
            const int64_t row = (int64_t)mt * kTileM + r;
            if (MODE == kGateUp) {
#pragma unroll
                for (int b = 0; b < NT / 64; ++b) {
                    const int i0 = nt * (NT / 2) + b * 32;
                    if (i0 >= p.I) break;
                    float g[32], u[32];
                    gemm::tc_ld32(taddr + 64 * b, g);
                    gemm::tc_ld32(taddr + 64 * b + 32, u);
                    uint32_t m = 0;
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        g[j] = silu_mul(g[j], u[j]);
                        m = max(m, __float_as_uint(g[j]) & 0x7fffffffu);
                    }
                    const uint32_t sc = scale_of_amax(m);
                    const float k = inv_scale(sc);
                    uint32_t q[4];
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        q[w] = 0;
#pragma unroll
                        for (int j = 0; j < 4; ++j) q[w] |= cvt_e2m1x2(g[8 * w + 2 * j] * k, g[8 * w + 2 * j + 1] * k) << (8 * j);
                    }
                    if (live) {
                        *reinterpret_cast<uint4*>(p.hq + row * (p.I / 2) + i0 / 2) = make_uint4(q[0], q[1], q[2], q[3]);
                        p.hs[tiled_at(row, i0 >> 5, p.hkb)] = (uint8_t)sc;
                        // the MMAs take K in steps of 64: the scale behind an odd last block must be a number
                        if (i0 + 32 == p.I && (p.I & 32)) p.hs[tiled_at(row, (i0 >> 5) + 1, p.hkb)] = 0;
                    }
                }
            } else {
                const int esz = MODE == kDown || p.out_dtype == MOE_F32 ? 4 : 2;
                const bool vec = (int64_t)p.N * esz % 16 == 0;
#pragma unroll
                for (int c = 0; c < NT; c += 32) {
                    const int n0 = nt * NT + c;
                    if (n0 >= p.N) break;
                    float v[32];
                    gemm::tc_ld32(taddr + c, v);
                    if (!live) continue;
                    const int left = min(32, p.N - n0);
                    if (MODE == kDown || p.out_dtype == MOE_F32) store_row<MOE_F32>(p.out, row * p.N + n0, v, left, vec);
                    else if (p.out_dtype == MOE_BF16) store_row<MOE_BF16>(p.out, row * p.N + n0, v, left, vec);
                    else store_row<MOE_F16>(p.out, row * p.N + n0, v, left, vec);
                }
            }
            gemm::tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_accempty[acc]);
        }
    }
    __syncthreads();
    if (s_failed && tid == 0) set_err(p.err, kErrFullWait);
    gemm::tc_fence_before();
    __syncthreads();
    if (warp == 2) {
        gemm::tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kTmemCols) : "memory");
    }
}

// ------------------------------------------------------------------ expert layer: routing
// Stable order of the routed pairs by expert, in tiles of 128 rows, by one CTA of 32 warps: each
// warp counts its run of pairs per expert, the counts are summed over the warps and scanned over
// the experts, and each warp places its run (ranks by __match_any_sync).
struct RouteParams {
    const int32_t* ids;
    int TK, K, E, e_off, emap_n;
    const int32_t* emap;
    int32_t* mtiles;
    int32_t* mt_expert;
    int32_t* mt_rows;
    int32_t* rowtok;
    int32_t* ppos;  // row of each pair, -1 for pairs of other engines
};

__global__ void __launch_bounds__(1024) mx_route_kernel(const RouteParams p) {
    extern __shared__ int32_t rsm[];  // [32][E] counts | [32] warp sums
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, E = p.E;
    int32_t* hist = rsm + warp * E;
    int32_t* sums = rsm + 32 * E;
    for (int e = lane; e < E; e += 32) hist[e] = 0;
    __syncwarp();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int run = ((p.TK + 31) / 32 + 31) / 32 * 32;
    const int i0 = min(p.TK, warp * run), i1 = min(p.TK, i0 + run);
    for (int i = i0 + lane; i - lane < i1; i += 32) {
        const int e = i < i1 ? local_expert(p.ids[i], p.e_off, E, p.emap, p.emap_n, i, p.K) : -1;
        const unsigned peers = __match_any_sync(0xffffffffu, e);
        if (e >= 0 && (peers & ((1u << lane) - 1u)) == 0) hist[e] += __popc(peers);
        __syncwarp();
    }
    __syncthreads();
    int cnt = 0;
    if (tid < E)
        for (int w = 0; w < 32; ++w) {
            const int c = rsm[w * E + tid];
            rsm[w * E + tid] = cnt;
            cnt += c;
        }
    const int nt = (cnt + kTileM - 1) / kTileM;
    int incl = nt;
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 31) sums[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        int v = sums[lane];
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        sums[lane] = v;
    }
    __syncthreads();
    const int first = incl - nt + (warp ? sums[warp - 1] : 0);
    if (tid < E) {
        for (int m = 0; m < nt; ++m) {
            p.mt_expert[first + m] = tid;
            p.mt_rows[first + m] = min(kTileM, cnt - m * kTileM);
        }
        for (int w = 0; w < 32; ++w) rsm[w * E + tid] += first * kTileM;
    }
    if (tid == 0) p.mtiles[0] = sums[31];
    __syncthreads();
    for (int i = i0 + lane; i - lane < i1; i += 32) {
        const int e = i < i1 ? local_expert(p.ids[i], p.e_off, E, p.emap, p.emap_n, i, p.K) : -1;
        const unsigned peers = __match_any_sync(0xffffffffu, e);
        const int rank = __popc(peers & ((1u << lane) - 1u));
        const int base = e >= 0 ? hist[e] : 0;
        __syncwarp();
        if (i < i1) {
            p.ppos[i] = e >= 0 ? base + rank : -1;
            if (e >= 0) p.rowtok[base + rank] = i / p.K;
        }
        if (e >= 0 && rank == 0) hist[e] = base + __popc(peers);
        __syncwarp();
    }
}

// Token rows -> codes [T][H / 2], and each block's scale to the scale tiles of the rows that hold
// the token: a CTA per token.
template <int DT>
__global__ void __launch_bounds__(256) mx_tokens_kernel(const void* x, int H, int K, const int32_t* ppos, uint8_t* xq,
                                                        uint8_t* xs, int kb) {
    __shared__ int32_t s_pos[64];
    const int64_t t = blockIdx.x;
    const int tid = threadIdx.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    for (int k = tid; k < K; k += blockDim.x) s_pos[k] = ppos[t * K + k];
    __syncthreads();
    const int n = H >> 3, nb = H >> 5;
    for (int i0 = 0; i0 < n; i0 += blockDim.x) {
        const int i = i0 + tid;
        float v[8] = {};
        if (i < n) load8<DT>(x, t * H + i * 8, v);
        uint32_t sc;
        const uint32_t c = quant8(v, sc);
        // the four blocks of a scale word lie in 16 neighbouring lanes
        uint32_t w = sc;
        w |= __shfl_down_sync(0xffffffffu, sc, 4, 16) << 8;
        w |= __shfl_down_sync(0xffffffffu, sc, 8, 16) << 16;
        w |= __shfl_down_sync(0xffffffffu, sc, 12, 16) << 24;
        if (i < n) {
            reinterpret_cast<uint32_t*>(xq + t * (H / 2))[i] = c;
            if ((i & 15) == 0) {
                const int b = i >> 2, left = nb - b;
                if (left < 4) w &= (1u << (8 * left)) - 1u;
                for (int k = 0; k < K; ++k)
                    if (s_pos[k] >= 0) *reinterpret_cast<uint32_t*>(xs + tiled_at(s_pos[k], b, kb)) = w;
            }
        }
    }
}

// y[t] = sum over the token's pairs, in their order, of w * part[row]
template <int DT>
__global__ void __launch_bounds__(256) mx_combine_kernel(const float* part, const int32_t* ppos, const float* tw, int T, int K,
                                                         int H, void* y) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int64_t total = (int64_t)T * (H / 4);
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t t = i / (H / 4);
        const int n = (int)(i - t * (H / 4)) * 4;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k = 0; k < K; ++k) {
            const int pos = __ldg(ppos + t * K + k);
            if (pos < 0) continue;
            const float w = __ldg(tw + t * K + k);
            const float4 v = __ldcg(reinterpret_cast<const float4*>(part + (int64_t)pos * H + n));
            a.x = fmaf(w, v.x, a.x);
            a.y = fmaf(w, v.y, a.y);
            a.z = fmaf(w, v.z, a.z);
            a.w = fmaf(w, v.w, a.w);
        }
        if (DT == MOE_F32) reinterpret_cast<float4*>(y)[i] = a;
        else reinterpret_cast<uint2*>(y)[i] = make_uint2(pack16<DT>(a.x, a.y), pack16<DT>(a.z, a.w));
    }
}

}  // namespace mx
}  // namespace moe
