// MXFP4: blocks of 32 elements along a row, each element 4-bit e2m1 (0, .5, 1, 1.5, 2, 3, 4, 6 and
// their negatives), each block one e8m0 scale 2^(s - 127) (255: NaN).
//
// Quantisation of a block with largest magnitude amax (the OCP Microscaling rule):
//   s - 127 = floor(log2(amax)) - 2, at least -127;  q = round-to-nearest-even(x / 2^(s - 127)),
// magnitudes above 6 become 6.  floor(log2) is the exponent field of amax, the division is an
// exact multiplication by a power of two, so the result is exact in 32 bits whatever the order.
// A block with an infinity or a NaN gets scale 255: every value of it decodes to NaN.
//
// Codes are packed two a byte, the even element in the low half.  Scales are row-major
// [rows][K / 32], or tiled for the tensor cores: 128 rows x 4 blocks in 512 bytes, byte
// 16 (r % 32) + 4 (r / 32) + k, tiles [ceil(rows / 128)][ceil(K / 128)], padding zero.
#pragma once
#include "tcgen05.cuh"

namespace moe {
namespace mx {

// Exponent byte of a block from the bits of its largest magnitude.
MOE_DEV uint32_t scale_of_amax(uint32_t amax_bits) {
    const uint32_t e = amax_bits >> 23;
    return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}
// 2^(127 - s): what a block is multiplied by (s = 255 only for blocks that decode to NaN).
MOE_DEV float inv_scale(uint32_t s) { return __uint_as_float((s < 253u ? 254u - s : 1u) << 23); }
// 2^(s - 127)
MOE_DEV float scale_value(uint32_t s) {
    return s == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(s ? s << 23 : 1u << 22);
}

// Two values -> two codes, `lo` in the low half (round to nearest even, saturating).
MOE_DEV uint32_t cvt_e2m1x2(float lo, float hi) {
    uint32_t r;
    asm("{\n\t.reg .b8 b;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %2, %1;\n\tcvt.u32.u8 %0, b;\n\t}" : "=r"(r) : "f"(lo), "f"(hi));
    return r;
}
// Two codes -> two halves (exact), the low code in .x.
MOE_DEV __half2 cvt_f16x2(uint32_t byte) {
    uint32_t r;
    asm("{\n\t.reg .b8 b;\n\tcvt.u8.u32 b, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b;\n\t}" : "=r"(r) : "r"(byte));
    return *reinterpret_cast<__half2*>(&r);
}

// Byte of the scale of (row, block) in the tiled layout with kb tiles along K.
MOE_DEV int64_t tiled_at(int64_t row, int64_t block, int64_t kb) {
    return ((row >> 7) * kb + (block >> 2)) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3);
}

// Expert weights lie in panels of 256 rows x 256 elements (128 bytes), one stage of a wide product, so that
// a stage is one contiguous copy whatever the matrix's row pitch; a slim product takes 128 rows of a
// panel.  [ceil(rows / 256)][stages] panels; what lies past the matrix is zero.  Their scales: 2048 bytes a
// panel, two scale tiles (256 elements) for rows 0-127, two for rows 128-255.
constexpr int kPanelRows = 256, kPanel = kPanelRows * 128, kPanelScales = 2048;
MOE_DEV int64_t panel_code_at(int64_t row, int64_t byte, int64_t stages) {
    return ((row >> 8) * stages + (byte >> 7)) * kPanel + (row & 255) * 128 + (byte & 127);
}
MOE_DEV int64_t panel_scale_at(int64_t row, int64_t block, int64_t stages) {
    return ((row >> 8) * stages + (block >> 3)) * kPanelScales + (row >> 7 & 1) * 1024 + (block >> 2 & 1) * 512 + (row & 31) * 16 +
           (row >> 5 & 3) * 4 + (block & 3);
}

// tiled_at for row r (below 128) of scale tile row `tile`, which need not be full.
MOE_DEV int64_t tile_row_at(int64_t tile, int r, int64_t block, int64_t kb) {
    return (tile * kb + (block >> 2)) * 512 + (r & 31) * 16 + (r >> 5) * 4 + (block & 3);
}

template <int DT>  // MOE_F16 / MOE_BF16 / MOE_F32: 8 consecutive values, 16-byte aligned
MOE_DEV void load8(const void* x, int64_t i, float (&v)[8]) {
    if (DT == MOE_F32) {
        const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(x) + i);
        const float4 a = __ldg(p), b = __ldg(p + 1);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 r = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(x) + i));
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[2 * j] = scale_to_f32((uint16_t)(w[j] & 0xffffu), DT == MOE_BF16);
            v[2 * j + 1] = scale_to_f32((uint16_t)(w[j] >> 16), DT == MOE_BF16);
        }
    }
}

// The 8 codes of this thread's quarter of a block, and the block's scale: four neighbouring
// lanes hold a block.
MOE_DEV uint32_t quant8(const float (&v)[8], uint32_t& scale) {
    uint32_t m = 0;  // magnitudes as bits: ordered as integers, NaN above infinity
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    scale = scale_of_amax(m);
    const float k = inv_scale(scale);
    uint32_t q = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) q |= cvt_e2m1x2(v[2 * j] * k, v[2 * j + 1] * k) << (8 * j);
    return q;
}

// Rows -> codes and scales.  A thread takes 8 elements (16 or 32 bytes), so that loads and
// stores of a warp are contiguous; four threads a block share its largest magnitude by shuffles.  The bound is
// the memory traffic: 24577 x 768 fp32 (85 MB) take 14.1 us, 6.1 TB/s; a few rows a launch's latency.
template <int DT, bool TILED>
__global__ void __launch_bounds__(256) quantize_kernel(const void* x, int64_t rows, int cols, uint8_t* q, uint8_t* s) {
    const int64_t n = rows * (cols >> 3);  // a multiple of 4: a quad is in or out as a whole
    const int nb = cols >> 5;
    const int64_t kb = (nb + 3) >> 2;
    for (int64_t i0 = (int64_t)blockIdx.x * blockDim.x; i0 < n; i0 += (int64_t)gridDim.x * blockDim.x) {
        const int64_t i = i0 + threadIdx.x;
        float v[8] = {};
        if (i < n) load8<DT>(x, i * 8, v);
        uint32_t sc;
        const uint32_t c = quant8(v, sc);
        if (i >= n) continue;
        reinterpret_cast<uint32_t*>(q)[i] = c;
        if ((i & 3) == 0) {
            const int64_t b = i >> 2;
            if (TILED) {
                const int64_t r = b / nb;
                const int k = (int)(b - r * nb);
                s[tiled_at(r, k, kb)] = (uint8_t)sc;
                if (k == nb - 1)  // the padding behind the row's last block
                    for (int j = nb; j < 4 * kb; ++j) s[tiled_at(r, j, kb)] = 0;
            } else {
                s[b] = (uint8_t)sc;
            }
        }
    }
    if (TILED) {  // the padding below the last row, a word of 4 blocks a thread
        const int64_t m = (((rows + 127) >> 7) * 128 - rows) * kb;
        for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < m; i += (int64_t)gridDim.x * blockDim.x)
            *reinterpret_cast<uint32_t*>(s + tiled_at(rows + i / kb, 4 * (i % kb), kb)) = 0u;
    }
}

// Row-major scales -> tiled (one thread a word of 4 blocks).
__global__ void tile_scales_kernel(const uint8_t* s, int64_t rows, int nb, uint8_t* out) {
    const int64_t kb = (nb + 3) >> 2, n = ((rows + 127) >> 7) * 128 * kb;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t r = i / kb, k = i - r * kb;
        uint32_t w = 0;
        if (r < rows)
            for (int j = 0; j < 4; ++j)
                if (4 * k + j < nb) w |= (uint32_t)s[r * nb + 4 * k + j] << (8 * j);
        *reinterpret_cast<uint32_t*>(out + tiled_at(r, 4 * k, kb)) = w;
    }
}

// Codes and scales -> rows, 8 elements a thread; memory traffic again: 24577 x 768 to bf16 (48 MB, most of it
// written) take 10.5 us, 4.6 TB/s, with one load in flight a thread.
template <int DT, bool TILED>
__global__ void __launch_bounds__(256) dequantize_kernel(const uint8_t* q, const uint8_t* s, int64_t rows, int cols, void* y) {
    const int64_t n = rows * (cols >> 3);
    const int nb = cols >> 5;
    const int64_t kb = (nb + 3) >> 2;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
        const uint32_t c = __ldg(reinterpret_cast<const uint32_t*>(q) + i);
        const int64_t b = i >> 2;
        uint32_t sc;
        if (TILED) {
            const int64_t r = b / nb;
            sc = __ldg(s + tiled_at(r, b - r * nb, kb));
        } else {
            sc = __ldg(s + b);
        }
        const float k = scale_value(sc);
        float v[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = __half22float2(cvt_f16x2((c >> (8 * j)) & 0xffu));
            v[2 * j] = f.x * k;
            v[2 * j + 1] = f.y * k;
        }
        if (DT == MOE_F32) {
            float4* d = reinterpret_cast<float4*>(reinterpret_cast<float*>(y) + i * 8);
            d[0] = make_float4(v[0], v[1], v[2], v[3]);
            d[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (DT == MOE_BF16) {
                    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
                    w[j] = *reinterpret_cast<const uint32_t*>(&h);
                } else {
                    const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
                    w[j] = *reinterpret_cast<const uint32_t*>(&h);
                }
            }
            reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(y))[i] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

}  // namespace mx
}  // namespace moe
