// MXFP4 entry points (include/moe_b200.h) and the MXFP4 expert layer of the engine.
#include <algorithm>
#include <atomic>
#include <mutex>
#include <new>

#include "mx_layer.h"
#include "mxfp4_gemm.cuh"
#include "status.h"

using namespace moe;

namespace {

using layer::ceil_div;

// ------------------------------------------------------------------ tensor maps
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int encoder(EncodeFn* out) {
    static std::atomic<EncodeFn> fn{nullptr};
    EncodeFn f = fn.load(std::memory_order_acquire);
    if (!f) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        CUDA_TRY(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q));
        if (!p || q != cudaDriverEntryPointSuccess) return fail(MOE_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
        f = reinterpret_cast<EncodeFn>(p);
        fn.store(f, std::memory_order_release);
    }
    *out = f;
    return MOE_OK;
}

int encode_map(CUtensorMap* m, CUtensorMapDataType type, CUtensorMapSwizzle swizzle, const void* base, int64_t esz, int64_t cols,
               int64_t rows, int box_cols, int box_rows) {
    EncodeFn fn;
    if (int rc = encoder(&fn)) return rc;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)(cols * esz)};
    const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows}, ones[2] = {1, 1};
    const CUresult r = fn(m, type, 2, const_cast<void*>(base), dims, strides, box, ones,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(MOE_ERR_CUDA, "cuTensorMapEncodeTiled failed with " + std::to_string((int)r));
    return MOE_OK;
}

// Scales as rows of `words` 32-bit words, boxes of 1 KB (a stage's scales of 128 rows) x box_rows.
int encode_scales(CUtensorMap* m, const void* base, int64_t words, int64_t rows, int box_rows) {
    return encode_map(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, CU_TENSOR_MAP_SWIZZLE_NONE, base, 4, words, rows, 256, box_rows);
}

// Codes as bytes [rows][pitch], boxes of 128 bytes x box_rows, 128-byte swizzle; what lies outside
// reads as zero.
int encode(CUtensorMap* m, const void* base, int64_t pitch, int64_t rows, int box_rows) {
    return encode_map(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, CU_TENSOR_MAP_SWIZZLE_128B, base, 1, pitch, rows, 128, box_rows);
}

// An output [rows][cols] of 2- or 4-byte elements, stored in boxes of 32 rows x 64 bytes.
int encode_out(CUtensorMap* m, void* base, int64_t esz, int64_t cols, int64_t rows) {
    return encode_map(m, esz == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, CU_TENSOR_MAP_SWIZZLE_64B, base,
                      esz, cols, rows, (int)(64 / esz), 32);
}

// ------------------------------------------------------------------ launches
// Opt-in shared memory of a kernel, once per device (a bit each).
int allow_smem(const void* fn, int bytes, std::atomic<uint64_t>& devices) {
    int dev = 0;
    CUDA_TRY(cudaGetDevice(&dev));
    const uint64_t bit = dev < 64 ? (uint64_t)1 << dev : 0;
    if (devices.load(std::memory_order_acquire) & bit) return MOE_OK;
    CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    devices.fetch_or(bit, std::memory_order_release);
    return MOE_OK;
}

template <int CLUSTER = 1, typename... P, typename... A>
int launch(void (*fn)(P...), unsigned grid, unsigned block, size_t smem, bool pdl, cudaStream_t st, A&&... args) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
    if (CLUSTER > 1) {
        cudaLaunchAttribute& a = attr[cfg.numAttrs++];
        a.id = cudaLaunchAttributeClusterDimension;
        a.val.clusterDim.x = CLUSTER;
        a.val.clusterDim.y = a.val.clusterDim.z = 1;
    }
    CUDA_TRY(cudaLaunchKernelEx(&cfg, fn, P(args)...));
    return MOE_OK;
}

int sm_count(int dev, int* out) {
    static std::atomic<int> n[64] = {};
    if (dev < 64 && (*out = n[dev].load(std::memory_order_relaxed))) return MOE_OK;
    CUDA_TRY(cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, dev));
    if (dev < 64) n[dev].store(*out, std::memory_order_relaxed);
    return MOE_OK;
}

// Kernel shapes, and the rules that choose between them (times in us; layers have H = 2048, I = 768, 128
// experts, top-8, and run in graphs).
// Dense products.  Pair: 256 x 256 tiles of two CTAs, whose 35 KB a stage and CTA let six stages be in flight:
// the ring's round trip (about 1 us plus a load's time) bounds wide tiles, so bytes per product count.  One-CTA
// tiles of 128 x 256 (51 KB, four stages) took 59 at 8192 x 4096 x 4096 where pairs take 50 (5.5 PFLOP/s; both with operands in L2, 60 without).
// Narrow: 128 x 64, two CTAs per SM, for products whose narrow tiles all run at once:
//   narrow | pairs: 1 x 4096 x 2048 5.5 | 7.5, 512 x 4096 x 4096 9.5 | 10.5, 1024 x 4096 x 4096 15.4 | 11.0.
// Layers.  Wide: 128 x 256, from 56 rows an expert on; down has few stages a tile and many stores, so three
// stages and four staging buffers.  Slim: 32 x 128, for fewer rows, where the weights' stream from memory
// bounds the kernel; two CTAs per SM with four stages each, so that down's first CTAs, and their weights, come in
// as gate_up's leave (one CTA with nine stages: T = 4 27.1, 64 66.5, 256 76.8, now 24.6, 62.4, 72.6).  An MMA of 64
// columns takes as long as one of 128, and 32 x 64 tiles were held up by them.
//   slim | wide, by rows an expert: 16 70 | 86, 32 87 | 100, 48 109 | 111, 56 119 | 114, 64 131 | 118, 96 169 | 135;
//   16 of the 128 experts, an eighth of the pairs: 7 20.7 | 26.8, 32 32 | 34, 56 36.9 | 39.8, 80 43.5 | 44.5, 96 48.5 | 47.5.
//   (Pairs, with 16-bit parts: 32 115, 128 148 | 138 wide, 256 198 | 193, 512 333 | 343: not worth their kernels here.)
// Fused: 8 x 128 and at most 8 pairs, small enough for a CTA of each kernel on an SM, so that down's first
// weights arrive while gate_up runs; two launches instead of four, which is what an eager call pays for.
//   fused | slim: eager T = 1 23.3 | 25.6, T = 2 29.1 | 27.8; in graphs 15.8 | 15.3, 22.1 | 19.8.
using Wide = mx::Shape<256, 128, 4, 8, 1, 1>;
using WideDown = mx::Shape<256, 128, 3, 8, 1, 1, false, 4>;
using Pair = mx::Shape<256, 128, 6, 8, 1, 1, false, 1, true>;
using Narrow = mx::Shape<64, 128, 4, 4, 2, 2>;
using Slim = mx::Shape<128, 32, 4, 4, 2, 1>;
using FusedUp = mx::Shape<128, 8, 7, 4, 2, 1, true>;
using FusedDown = mx::Shape<128, 8, 3, 4, 2, 1, true>;

static_assert(FusedUp::TM == mx::kFusedRows && FusedDown::TM == mx::kFusedRows && Slim::TM == mx::kSlimRows &&
                  Wide::TM == mx::kWideRows && WideDown::TM == mx::kWideRows,
              "the workspace is laid out for these tiles");

template <int MODE, class S>
int launch_gemm(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& ta32, const CUtensorMap& to, const CUtensorMap& tfa,
                const CUtensorMap& tfb, mx::GemmParams& p, int64_t m_tiles, int sms, bool pdl, cudaStream_t st) {
    auto fn = mx::mx_gemm_kernel<MODE, S>;
    constexpr bool WA = S::FUSED && MODE == mx::kGateUp;
    const int smem = S::smem(WA, (int)ceil_div(p.K, mx::kStageK));
    static std::atomic<uint64_t> devices{0};
    if (int rc = allow_smem(reinterpret_cast<const void*>(fn), S::smem(WA, mx::kFusedStages), devices)) return rc;
    p.nt_count = (int)ceil_div(p.N, S::NT);
    const int64_t at_once = S::PAIR ? sms / 2 : sms * (S::FUSED ? 1 : S::kCtas);  // tiles
    const unsigned grid = (unsigned)(std::min(m_tiles * p.nt_count, at_once) * (S::PAIR ? 2 : 1));
    return launch<S::PAIR ? 2 : 1>(fn, grid, S::kThreads, smem, pdl, st, ta, tb, ta32, to, tfa, tfb, p);
}

bool dtype_ok(int32_t t) { return t == MOE_F16 || t == MOE_BF16 || t == MOE_F32; }
bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Error word of the products that run without an engine: one per device, in mapped host memory, whose
// address is the same on both sides.
int product_error_word(int dev, int32_t** word) {
    static std::mutex mu;
    static std::atomic<int32_t*> words[64] = {};
    if (dev < 0 || dev >= 64) return fail(MOE_ERR_INVALID, "device ordinal out of range");
    int32_t* w = words[dev].load(std::memory_order_acquire);
    if (!w) {
        std::lock_guard<std::mutex> lk(mu);
        w = words[dev].load();
        if (!w) {
            cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;  // the first call may be a captured one
            CUDA_TRY(cudaThreadExchangeStreamCaptureMode(&mode));
            cudaError_t e = cudaHostAlloc(reinterpret_cast<void**>(&w), 64, cudaHostAllocMapped | cudaHostAllocPortable);
            cudaThreadExchangeStreamCaptureMode(&mode);
            void* d = nullptr;
            if (e == cudaSuccess) e = cudaHostGetDevicePointer(&d, w, 0);
            if (e == cudaSuccess && d != w) e = cudaErrorNotSupported;
            if (e != cudaSuccess) return fail(MOE_ERR_CUDA, std::string("error word: ") + cudaGetErrorString(e));
            *reinterpret_cast<volatile int32_t*>(w) = 0;
            words[dev].store(w, std::memory_order_release);
        }
    }
    *word = w;
    return MOE_OK;
}

template <int DT>
int quantize_launch(const void* x, int64_t rows, int64_t cols, uint8_t* q, uint8_t* s, bool tiled, int sms, cudaStream_t st) {
    const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(rows * (cols / 8), 256), (int64_t)sms * 16);
    if (tiled) mx::quantize_kernel<DT, true><<<grid, 256, 0, st>>>(x, rows, (int)cols, q, s);
    else mx::quantize_kernel<DT, false><<<grid, 256, 0, st>>>(x, rows, (int)cols, q, s);
    CUDA_TRY(cudaGetLastError());
    return MOE_OK;
}

int quantize(const void* x, int32_t dtype, int64_t rows, int64_t cols, uint8_t* q, uint8_t* s, bool tiled, cudaStream_t st) {
    int dev = 0, sms = 0;
    CUDA_TRY(cudaGetDevice(&dev));
    if (int rc = sm_count(dev, &sms)) return rc;
    return dtype == MOE_F32    ? quantize_launch<MOE_F32>(x, rows, cols, q, s, tiled, sms, st)
           : dtype == MOE_BF16 ? quantize_launch<MOE_BF16>(x, rows, cols, q, s, tiled, sms, st)
                               : quantize_launch<MOE_F16>(x, rows, cols, q, s, tiled, sms, st);
}

template <int DT>
int dequantize_launch(const uint8_t* q, const uint8_t* s, int64_t rows, int64_t cols, void* y, bool tiled, int sms, cudaStream_t st) {
    const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(rows * (cols / 8), 256), (int64_t)sms * 16);
    if (tiled) mx::dequantize_kernel<DT, true><<<grid, 256, 0, st>>>(q, s, rows, (int)cols, y);
    else mx::dequantize_kernel<DT, false><<<grid, 256, 0, st>>>(q, s, rows, (int)cols, y);
    CUDA_TRY(cudaGetLastError());
    return MOE_OK;
}

int check_rows(int64_t rows, int64_t cols) {
    if (rows < 0 || cols <= 0 || cols % 32 != 0) return fail(MOE_ERR_INVALID, "cols must be a positive multiple of 32");
    if (cols > (int64_t)1 << 30 || rows > (int64_t)1 << 31) return fail(MOE_ERR_INVALID, "rows or cols too large");
    return MOE_OK;
}

}  // namespace

// ------------------------------------------------------------------ C ABI
extern "C" int moe_quantize_rows_mxfp4(const void* x, int32_t dtype, int64_t rows, int64_t cols, int32_t tiled_scales,
                                       uint8_t* q, uint8_t* scales, void* stream) {
    if (int rc = check_rows(rows, cols)) return rc;
    if (!dtype_ok(dtype)) return fail(MOE_ERR_INVALID, "bad dtype");
    if (rows == 0) return MOE_OK;
    if (!x || !q || !scales) return fail(MOE_ERR_INVALID, "null pointer");
    if (!aligned(x, 16) || !aligned(q, 16) || (tiled_scales && !aligned(scales, 16)))
        return fail(MOE_ERR_INVALID, "x, the codes and tiled scales must be 16-byte aligned");
    return quantize(x, dtype, rows, cols, q, scales, tiled_scales != 0, static_cast<cudaStream_t>(stream));
}

extern "C" int moe_dequantize_rows_mxfp4(const uint8_t* q, const uint8_t* scales, int64_t rows, int64_t cols,
                                         int32_t tiled_scales, void* y, int32_t dtype, void* stream) {
    if (int rc = check_rows(rows, cols)) return rc;
    if (!dtype_ok(dtype)) return fail(MOE_ERR_INVALID, "bad dtype");
    if (rows == 0) return MOE_OK;
    if (!y || !q || !scales) return fail(MOE_ERR_INVALID, "null pointer");
    if (!aligned(y, 16) || !aligned(q, 4)) return fail(MOE_ERR_INVALID, "y must be 16-byte, the codes 4-byte aligned");
    int dev = 0, sms = 0;
    CUDA_TRY(cudaGetDevice(&dev));
    if (int rc = sm_count(dev, &sms)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool tiled = tiled_scales != 0;
    return dtype == MOE_F32    ? dequantize_launch<MOE_F32>(q, scales, rows, cols, y, tiled, sms, st)
           : dtype == MOE_BF16 ? dequantize_launch<MOE_BF16>(q, scales, rows, cols, y, tiled, sms, st)
                               : dequantize_launch<MOE_F16>(q, scales, rows, cols, y, tiled, sms, st);
}

extern "C" int moe_mxfp4_tile_scales(const uint8_t* scales, int64_t rows, int64_t cols, uint8_t* tiles, void* stream) {
    if (int rc = check_rows(rows, cols)) return rc;
    if (rows == 0) return MOE_OK;
    if (!scales || !tiles) return fail(MOE_ERR_INVALID, "null pointer");
    if (!aligned(tiles, 16)) return fail(MOE_ERR_INVALID, "tiled scales must be 16-byte aligned");
    const int64_t n = ceil_div(rows, 128) * 128 * ceil_div(cols, 128);
    mx::tile_scales_kernel<<<(unsigned)std::min<int64_t>(ceil_div(n, 256), 4096), 256, 0, static_cast<cudaStream_t>(stream)>>>(
        scales, rows, (int)(cols / 32), tiles);
    CUDA_TRY(cudaGetLastError());
    return MOE_OK;
}

extern "C" int moe_mxfp4_matmul(const uint8_t* a, const uint8_t* a_scales, const uint8_t* b, const uint8_t* b_scales,
                                int64_t M, int64_t N, int64_t K, void* y, int32_t out_dtype, void* stream) {
    if (M < 0 || N <= 0 || K <= 0 || K % 32 != 0) return fail(MOE_ERR_INVALID, "K must be a positive multiple of 32, N positive");
    if (M > (int64_t)1 << 30 || N > (int64_t)1 << 30 || K > (int64_t)1 << 30) return fail(MOE_ERR_INVALID, "M, N or K too large");
    if (!dtype_ok(out_dtype)) return fail(MOE_ERR_INVALID, "bad output dtype");
    if (M == 0) return MOE_OK;
    if (!a || !a_scales || !b || !b_scales || !y) return fail(MOE_ERR_INVALID, "null pointer");
    if (!aligned(a, 16) || !aligned(b, 16) || !aligned(a_scales, 16) || !aligned(b_scales, 16) || !aligned(y, 16))
        return fail(MOE_ERR_INVALID, "operands, scales and the output must be 16-byte aligned");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int dev = 0, sms = 0;
    CUDA_TRY(cudaGetDevice(&dev));
    if (int rc = sm_count(dev, &sms)) return rc;
    mx::GemmParams p{};
    if (int rc = product_error_word(dev, &p.err)) return rc;
    if (*reinterpret_cast<volatile int32_t*>(p.err) != 0) {
        *reinterpret_cast<volatile int32_t*>(p.err) = 0;
        return fail(MOE_ERR_DEVICE, "an earlier MXFP4 product failed on the device (a bounded wait expired); its output is invalid");
    }
    CUtensorMap ta, tb;
    if (int rc = encode(&ta, a, K / 2, M, 128)) return rc;
    // narrow tiles while all of them run at once
    const bool wide = ceil_div(M, 128) * ceil_div(N, Narrow::NT) > (int64_t)sms * Narrow::kCtas;
    p.mt_count = (int)ceil_div(M, wide ? Pair::kTileRows : Narrow::kTileRows);
    if (int rc = encode(&tb, b, K / 2, N, wide ? Pair::NT / 2 : Narrow::NT)) return rc;
    p.M = (int)M; p.N = (int)N; p.K = (int)K;
    p.kb = (int)ceil_div(K, 128);
    p.sfa = a_scales;
    p.sfb = b_scales;
    p.out = y;
    p.out_dtype = out_dtype;
    CUtensorMap to = ta;  // unused unless tma_out
    const int64_t esz = out_dtype == MOE_F32 ? 4 : 2;
    p.tma_out = wide && N * esz % 16 == 0;
    if (p.tma_out)
        if (int rc = encode_out(&to, y, esz, N, M)) return rc;
    if (!wide) return launch_gemm<mx::kDense, Narrow>(ta, tb, ta, to, ta, ta, p, p.mt_count, sms, false, st);
    CUtensorMap tfa, tfb;
    if (int rc = encode_scales(&tfa, a_scales, p.kb * 128, ceil_div(M, 128), 1)) return rc;
    if (int rc = encode_scales(&tfb, b_scales, p.kb * 128, ceil_div(N, 128), 2)) return rc;
    return launch_gemm<mx::kDense, Pair>(ta, tb, ta, to, tfa, tfb, p, p.mt_count, sms, false, st);
}

// ------------------------------------------------------------------ expert layer
namespace moe {

struct MxLayer {
    moe_config cfg{};
    int sms = 0;
    int64_t all_experts = 0;   // of the whole layer
    int64_t kb1 = 0, kb2 = 0;  // scale tiles along K of gate_up (1) and down (2)
    int64_t st1 = 0, st2 = 0, pn1 = 0, pn2 = 0;  // panels along K and N
    // panels of codes and their scales; maps of 128 and of 256 rows
    uint8_t *q1 = nullptr, *s1 = nullptr, *q2 = nullptr, *s2 = nullptr;
    CUtensorMap t1[2]{}, t2[2]{};
    uint8_t* ws = nullptr;
    size_t ws_bytes = 0;
    uint8_t* retired[64] = {};  // earlier workspaces: captured graphs may still hold them
    int n_retired = 0;
    size_t q1_expert() const { return (size_t)pn1 * st1 * mx::kPanel; }
    size_t q2_expert() const { return (size_t)pn2 * st2 * mx::kPanel; }
    size_t s1_expert() const { return (size_t)pn1 * st1 * mx::kPanelScales; }
    size_t s2_expert() const { return (size_t)pn2 * st2 * mx::kPanelScales; }
};

namespace layer {

// Row of the input contract for row r of the layer: gate_up (map) rows lie in groups of 32 gate rows
// and the 32 up rows of the same units.
MOE_DEV int64_t source_row(int64_t r, int map, int64_t I) { return map ? ((r >> 5) & 1) * I + (r >> 6) * 32 + (r & 31) : r; }

// Codes of a matrix [rows][bytes] between the input contract and the layer's panels, 16 bytes a thread.
__global__ void mx_panel_codes_kernel(uint8_t* panels, uint8_t* codes, int64_t rows, int64_t bytes, int64_t stages, int64_t expert,
                                      int map, int64_t I, int to_panels) {
    const int64_t n16 = bytes / 16, n = rows * n16, e = blockIdx.y;
    panels += e * expert;
    codes += e * rows * bytes;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t r = i / n16, c = i - r * n16;
        uint4* a = reinterpret_cast<uint4*>(panels + mx::panel_code_at(r, c * 16, stages));
        uint4* b = reinterpret_cast<uint4*>(codes) + source_row(r, map, I) * n16 + c;
        if (to_panels) *a = *b;
        else *b = *a;
    }
}

// Scales [rows][nb] between the input contract and the panels'.
__global__ void mx_panel_scales_kernel(uint8_t* scales, uint8_t* s, int64_t rows, int nb, int64_t stages, int64_t expert, int map,
                                       int64_t I, int to_panels) {
    const int64_t n = rows * nb, e = blockIdx.y;
    scales += e * expert;
    s += e * n;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t r = i / nb, b = i - r * nb;
        uint8_t* p = scales + mx::panel_scale_at(r, b, stages);
        uint8_t* v = s + source_row(r, map, I) * nb + b;
        if (to_panels) *p = *v;
        else *v = *p;
    }
}

// Online quantisation of rows [n][cols] to layer rows: row j goes to layer row
// (j / 32) * 64 + 32 * half + j % 32 (gate_up, half 0 gate, 1 up) or j (down, half -1).
template <int DT>
__global__ void mx_store_rows_kernel(const void* w, int64_t n, int cols, int half, uint8_t* panels, uint8_t* scales) {
    const int64_t per = cols >> 3, total = n * per, stages = (cols + 255) >> 8;
    for (int64_t i0 = (int64_t)blockIdx.x * blockDim.x; i0 < total; i0 += (int64_t)gridDim.x * blockDim.x) {
        const int64_t i = i0 + threadIdx.x;
        float v[8] = {};
        if (i < total) mx::load8<DT>(w, i * 8, v);
        uint32_t sc;
        const uint32_t c = mx::quant8(v, sc);
        if (i >= total) continue;
        const int64_t j = i / per, k = i - j * per;
        const int64_t r = half < 0 ? j : (j >> 5) * 64 + 32 * half + (j & 31);
        *reinterpret_cast<uint32_t*>(panels + mx::panel_code_at(r, k * 4, stages)) = c;
        if ((i & 3) == 0) scales[mx::panel_scale_at(r, k >> 2, stages)] = (uint8_t)sc;
    }
}

struct Workspace {
    int2* mt_list;
    int32_t *ppos, *counts;
    uint8_t *xq, *xs, *hq, *hs;
    float* part;  // [rows][H]
    int64_t mt;
    int tile;
};

LayerShape shape_of(const MxLayer* l, bool dense) {
    return {l->cfg.num_experts, l->cfg.hidden_size, l->cfg.intermediate_size, dense ? 0 : l->all_experts};
}

// The parts of the workspace for a call that runs in one pass.
int carve(const MxLayer* l, const MxForward& f, int64_t T, Workspace& w) {
    const Layout o = layout_of(shape_of(l, f.dense), T, f.K);
    if (o.bytes > l->ws_bytes) return fail(MOE_ERR_STATE, "the workspace is too small for this call");
    w.mt_list = reinterpret_cast<int2*>(l->ws + o.mt_list);
    w.ppos = reinterpret_cast<int32_t*>(l->ws + o.ppos);
    w.counts = reinterpret_cast<int32_t*>(l->ws + o.counts);
    w.xq = l->ws + o.xq;
    w.xs = l->ws + o.xs;
    w.hq = l->ws + o.hq;
    w.hs = l->ws + o.hs;
    w.part = reinterpret_cast<float*>(l->ws + o.part);
    w.mt = o.mt;
    w.tile = o.tile;
    return MOE_OK;
}

// A workspace of at least `bytes`.  An outgrown one is kept until the engine goes, since captured
// graphs refer to it; sizes double, so that all of them hold at most twice the last.
int grow(MxLayer* l, size_t bytes) {
    if (bytes <= l->ws_bytes) return MOE_OK;
    if (l->n_retired == 64) return fail(MOE_ERR_STATE, "the workspace has grown too often");
    const size_t want = std::max(bytes, 2 * l->ws_bytes);
    uint8_t* p = nullptr;
    cudaError_t e = cudaMalloc(&p, want);
    size_t got = want;
    if (e != cudaSuccess && want > bytes) {
        cudaGetLastError();
        e = cudaMalloc(&p, bytes);
        got = bytes;
    }
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(MOE_ERR_CUDA, std::string("workspace of ") + std::to_string(bytes) + " bytes: " + cudaGetErrorString(e));
    }
    if (l->ws) l->retired[l->n_retired++] = l->ws;
    l->ws = p;
    l->ws_bytes = got;
    return MOE_OK;
}

template <int DT>
int combine_launch(const MxLayer* l, const MxForward& f, const float* tw, void* y, const Workspace& w, int64_t T, cudaStream_t st) {
    const int H = (int)l->cfg.hidden_size;
    return launch(mx::mx_combine_kernel<DT>, (unsigned)std::min<int64_t>(ceil_div(T * ceil_div(H, 256), 8), l->sms * 16), 256, 0,
                  f.pdl, st, (const float*)w.part, (const int32_t*)w.ppos, tw, (int)T, (int)f.K, H, y);
}

// Two kernels: gate_up (routing, token rows quantised as they are needed), down with the weighted sum.
int forward_fused(MxLayer* l, const MxForward& f, const void* x, void* y, const int32_t* ids, const float* tw, int64_t T,
                  cudaStream_t st) {
    const int64_t H = l->cfg.hidden_size, I = l->cfg.intermediate_size;
    Workspace w;
    if (int rc = carve(l, f, T, w)) return rc;
    CUtensorMap th;
    if (int rc = encode(&th, w.hq, I / 2, w.mt * w.tile, w.tile)) return rc;
    mx::GemmParams p{};
    p.err = f.err;
    p.x = x; p.ids = ids; p.tw = tw;
    p.T = (int)T; p.topk = (int)f.K; p.E = (int)l->cfg.num_experts; p.e_off = l->cfg.expert_offset;
    p.emap = f.emap; p.emap_n = f.emap_n; p.act_bf16 = f.act_dtype == MOE_BF16;
    p.I = (int)I;
    mx::GemmParams g1 = p;
    g1.N = (int)(2 * I); g1.K = (int)H; g1.kb = (int)l->kb1;
    g1.sfb = l->s1; g1.hq = w.hq; g1.hs = w.hs; g1.hkb = (int)l->kb2;
    if (int rc = launch_gemm<mx::kGateUp, FusedUp>(th, l->t1[0], th, th, th, th, g1, w.mt, l->sms, f.pdl, st)) return rc;
    mx::GemmParams g2 = p;
    g2.N = (int)H; g2.K = (int)I; g2.kb = (int)l->kb2;
    g2.sfa = w.hs; g2.sfb = l->s2; g2.out = w.part; g2.out_dtype = MOE_F32;
    g2.y = y; g2.y_dtype = f.out_dtype; g2.cnt = f.cnt;
    return launch_gemm<mx::kDown, FusedDown>(th, l->t2[0], th, th, th, th, g2, w.mt, l->sms, f.pdl, st);
}

int forward_slice(MxLayer* l, const MxForward& f, const void* x, void* y, const int32_t* ids, const float* tw, int64_t T,
                  cudaStream_t st) {
    const int64_t E = l->cfg.num_experts, H = l->cfg.hidden_size, I = l->cfg.intermediate_size;
    const Plan plan = plan_of(shape_of(l, f.dense), T, f.K);
    if (plan == kPlanFused) return forward_fused(l, f, x, y, ids, tw, T, st);
    const bool wide = plan == kPlanWide;
    Workspace w;
    if (int rc = carve(l, f, T, w)) return rc;
    mx::PrepParams r{};
    r.x = x; r.ids = ids;
    r.T = (int)T; r.K = (int)f.K; r.H = (int)H; r.E = (int)E; r.e_off = l->cfg.expert_offset;
    r.emap = f.emap; r.emap_n = f.emap_n;
    r.tokens = (int)prep_tokens(T, f.K, l->sms);
    r.tile_log2 = wide ? 7 : 5;
    r.mt_list = w.mt_list; r.mt_bound = (int)w.mt; r.ppos = w.ppos;
    r.xq = w.xq; r.xs = w.xs; r.kb = (int)l->kb1;
    const unsigned runs = (unsigned)ceil_div(T, r.tokens);
    const bool self = T * f.K <= mx::kPrepSelf;
    if (!self) {
        r.counts = w.counts;
        if (int rc = launch(mx::mx_count_kernel, runs, mx::kPrepThreads, (size_t)E * 4, f.pdl, st, r, w.counts)) return rc;
    }
    const size_t psmem = ((size_t)(mx::kPrepWarps + 1) * E + (self ? T * f.K : r.tokens * f.K + 2 * E)) * 4;
    auto prep = f.act_dtype == MOE_BF16 ? mx::mx_prep_kernel<MOE_BF16> : mx::mx_prep_kernel<MOE_F16>;
    static std::atomic<uint64_t> prep_devices[2] = {};
    if (int rc = allow_smem(reinterpret_cast<const void*>(prep), 128 * 1024, prep_devices[f.act_dtype == MOE_BF16])) return rc;
    if (int rc = launch(prep, runs, mx::kPrepThreads, psmem, f.pdl, st, r)) return rc;
    CUtensorMap tx, th, tx32, th32;  // boxes of a whole tile, and of 32 rows for tiles that are not full
    if (int rc = encode(&tx, w.xq, H / 2, w.mt * w.tile, w.tile)) return rc;
    if (int rc = encode(&th, w.hq, I / 2, w.mt * w.tile, w.tile)) return rc;
    tx32 = tx, th32 = th;
    if (wide) {
        if (int rc = encode(&tx32, w.xq, H / 2, w.mt * w.tile, 32)) return rc;
        if (int rc = encode(&th32, w.hq, I / 2, w.mt * w.tile, 32)) return rc;
    }
    mx::GemmParams p{};
    p.mt_list = w.mt_list; p.mt_count = (int)w.mt;
    p.err = f.err;
    p.I = (int)I;
    mx::GemmParams g1 = p;
    g1.N = (int)(2 * I); g1.K = (int)H; g1.kb = (int)l->kb1;
    g1.sfa = w.xs; g1.sfb = l->s1; g1.hq = w.hq; g1.hs = w.hs; g1.hkb = (int)l->kb2;
    if (self && !wide && f.pdl) {  // gate_up starts beside the token kernel, and finds its first weights by the ids
        g1.ids = ids;
        g1.T = (int)T; g1.topk = (int)f.K; g1.E = (int)E; g1.e_off = l->cfg.expert_offset;
        g1.emap = f.emap; g1.emap_n = f.emap_n;
    }
    if (int rc = wide ? launch_gemm<mx::kGateUp, Wide>(tx, l->t1[1], tx32, tx, tx, tx, g1, w.mt, l->sms, f.pdl, st)
                      : launch_gemm<mx::kGateUp, Slim>(tx, l->t1[0], tx, tx, tx, tx, g1, w.mt, l->sms, f.pdl, st))
        return rc;
    mx::GemmParams g2 = p;
    g2.N = (int)H; g2.K = (int)I; g2.kb = (int)l->kb2;
    g2.sfa = w.hs; g2.sfb = l->s2; g2.out = w.part; g2.out_dtype = MOE_F32;
    CUtensorMap tp = th;  // used by wide tiles
    if (wide)
        if (int rc = encode_out(&tp, w.part, 4, H, w.mt * w.tile)) return rc;
    if (int rc = wide ? launch_gemm<mx::kDown, WideDown>(th, l->t2[1], th32, tp, th, th, g2, w.mt, l->sms, f.pdl, st)
                      : launch_gemm<mx::kDown, Slim>(th, l->t2[0], th, tp, th, th, g2, w.mt, l->sms, f.pdl, st))
        return rc;
    return f.out_dtype == MOE_F32    ? combine_launch<MOE_F32>(l, f, tw, y, w, T, st)
           : f.out_dtype == MOE_BF16 ? combine_launch<MOE_BF16>(l, f, tw, y, w, T, st)
                                     : combine_launch<MOE_F16>(l, f, tw, y, w, T, st);
}

}  // namespace layer
using namespace layer;

int mx_create(const moe_config& cfg, int num_sms, MxLayer** out) {
    *out = nullptr;
    if (cfg.num_experts > 1024) return fail(MOE_ERR_INVALID, "MXFP4 engines hold at most 1024 experts");
    if (cfg.hidden_size > 1 << 20 || cfg.intermediate_size > 1 << 20) return fail(MOE_ERR_INVALID, "hidden or intermediate size too large");
    auto* l = new (std::nothrow) MxLayer();
    if (!l) return fail(MOE_ERR_STATE, "out of host memory");
    l->cfg = cfg;
    l->sms = num_sms;
    const int64_t H = cfg.hidden_size, I = cfg.intermediate_size;
    l->kb1 = ceil_div(H, 128);
    l->kb2 = ceil_div(I, 128);
    l->st1 = ceil_div(H, 256);
    l->st2 = ceil_div(I, 256);
    l->pn1 = ceil_div(2 * I, mx::kPanelRows);
    l->pn2 = ceil_div(H, mx::kPanelRows);
    // the maps' row coordinates are 32-bit integers
    if (cfg.num_experts * std::max(l->pn1 * l->st1, l->pn2 * l->st2) * mx::kPanelRows > (int64_t)1 << 31) {
        mx_destroy(l);
        return fail(MOE_ERR_INVALID, "MXFP4 weights too large for one engine");
    }
    MxBuffer b[kMxBuffers];
    mx_buffers(l, b);
    for (auto& x : b) {
        cudaError_t e = cudaMalloc(x.ptr, x.bytes);
        if (e == cudaSuccess) e = cudaMemset(*x.ptr, 0, x.bytes);
        if (e != cudaSuccess) {
            cudaGetLastError();
            mx_destroy(l);
            return fail(MOE_ERR_CUDA, std::string("MXFP4 weights: ") + cudaGetErrorString(e));
        }
    }
    int rc = MOE_OK;
    for (int w = 0; w < 2 && rc == MOE_OK; ++w) {
        const int box = w ? Wide::NT : Slim::NT;
        rc = encode(&l->t1[w], l->q1, 128, cfg.num_experts * l->pn1 * l->st1 * mx::kPanelRows, box);
        if (rc == MOE_OK) rc = encode(&l->t2[w], l->q2, 128, cfg.num_experts * l->pn2 * l->st2 * mx::kPanelRows, box);
    }
    if (rc != MOE_OK) {
        mx_destroy(l);
        return rc;
    }
    *out = l;
    return MOE_OK;
}

void mx_destroy(MxLayer* l) {
    if (!l) return;
    for (uint8_t* p : {l->q1, l->s1, l->q2, l->s2, l->ws}) cudaFree(p);
    for (uint8_t* p : l->retired) cudaFree(p);  // null where none is
    delete l;
}

void mx_buffers(MxLayer* l, MxBuffer (&b)[kMxBuffers]) {
    const size_t E = l->cfg.num_experts;
    b[0] = {&l->q1, E * l->q1_expert()};
    b[1] = {&l->s1, E * l->s1_expert()};
    b[2] = {&l->q2, E * l->q2_expert()};
    b[3] = {&l->s2, E * l->s2_expert()};
}

int mx_load(MxLayer* l, const uint8_t* w13_q, const uint8_t* w13_s, const uint8_t* w2_q, const uint8_t* w2_s, cudaStream_t st) {
    const int64_t E = l->cfg.num_experts, H = l->cfg.hidden_size, I = l->cfg.intermediate_size;
    if (!aligned(w13_q, 16) || !aligned(w2_q, 16)) return fail(MOE_ERR_INVALID, "weight codes must be 16-byte aligned");
    const dim3 g(128, (unsigned)E);
    mx_panel_codes_kernel<<<g, 256, 0, st>>>(l->q1, const_cast<uint8_t*>(w13_q), 2 * I, H / 2, l->st1, l->q1_expert(), 1, I, 1);
    mx_panel_codes_kernel<<<g, 256, 0, st>>>(l->q2, const_cast<uint8_t*>(w2_q), H, I / 2, l->st2, l->q2_expert(), 0, I, 1);
    mx_panel_scales_kernel<<<g, 256, 0, st>>>(l->s1, const_cast<uint8_t*>(w13_s), 2 * I, (int)(H / 32), l->st1, l->s1_expert(), 1, I, 1);
    mx_panel_scales_kernel<<<g, 256, 0, st>>>(l->s2, const_cast<uint8_t*>(w2_s), H, (int)(I / 32), l->st2, l->s2_expert(), 0, I, 1);
    CUDA_TRY(cudaGetLastError());
    return MOE_OK;
}

int mx_quantize_store(MxLayer* l, int64_t expert, int32_t proj, const void* w, int32_t dtype, cudaStream_t st) {
    const int64_t H = l->cfg.hidden_size, I = l->cfg.intermediate_size;
    if (!aligned(w, 16)) return fail(MOE_ERR_INVALID, "weight must be 16-byte aligned");
    const int64_t n = proj == 2 ? H : I, cols = proj == 2 ? I : H;
    uint8_t* q = proj == 2 ? l->q2 + expert * l->q2_expert() : l->q1 + expert * l->q1_expert();
    uint8_t* s = proj == 2 ? l->s2 + expert * l->s2_expert() : l->s1 + expert * l->s1_expert();
    const int half = proj == 2 ? -1 : proj;
    const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(n * (cols / 8), 256), (int64_t)l->sms * 16);
    if (dtype == MOE_F32) mx_store_rows_kernel<MOE_F32><<<grid, 256, 0, st>>>(w, n, (int)cols, half, q, s);
    else if (dtype == MOE_BF16) mx_store_rows_kernel<MOE_BF16><<<grid, 256, 0, st>>>(w, n, (int)cols, half, q, s);
    else mx_store_rows_kernel<MOE_F16><<<grid, 256, 0, st>>>(w, n, (int)cols, half, q, s);
    CUDA_TRY(cudaGetLastError());
    return MOE_OK;
}

int mx_export(MxLayer* l, int64_t expert, int32_t which, void* q_out, void* s_out) {
    const int64_t H = l->cfg.hidden_size, I = l->cfg.intermediate_size;
    const int64_t rows = which == 0 ? 2 * I : H, cols = which == 0 ? H : I, nb = cols / 32;
    uint8_t* q = which == 0 ? l->q1 + expert * l->q1_expert() : l->q2 + expert * l->q2_expert();
    uint8_t* s = which == 0 ? l->s1 + expert * l->s1_expert() : l->s2 + expert * l->s2_expert();
    uint8_t* d = nullptr;
    CUDA_TRY(cudaMalloc(&d, rows * (cols / 2) + rows * nb));
    uint8_t* ds = d + rows * (cols / 2);
    const int64_t stages = which == 0 ? l->st1 : l->st2;
    mx_panel_codes_kernel<<<128, 256>>>(q, d, rows, cols / 2, stages, 0, which == 0, I, 0);
    mx_panel_scales_kernel<<<128, 256>>>(s, ds, rows, (int)nb, stages, 0, which == 0, I, 0);
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) e = cudaMemcpy(q_out, d, rows * (cols / 2), cudaMemcpyDeviceToHost);
    if (e == cudaSuccess) e = cudaMemcpy(s_out, ds, rows * nb, cudaMemcpyDeviceToHost);
    cudaFree(d);
    CUDA_TRY(e);
    return MOE_OK;
}

void mx_set_layer_experts(MxLayer* l, int64_t n) { l->all_experts = n; }

int mx_reserve(MxLayer* l, int64_t T, int64_t K) {
    if (T == 0) return MOE_OK;
    return grow(l, reserve_bytes(shape_of(l, false), T, K));
}

int mx_forward(MxLayer* l, const MxForward& f, cudaStream_t st) {
    if (!aligned(f.x, 16) || !aligned(f.y, 16)) return fail(MOE_ERR_INVALID, "hidden and output must be 16-byte aligned");
    const int64_t S = slice_tokens(f.T, f.K), H = l->cfg.hidden_size;
    const size_t need = call_bytes(shape_of(l, f.dense), f.T, f.K);
    if (need > l->ws_bytes) {
        cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
        CUDA_TRY(cudaStreamIsCapturing(st, &cap));
        if (cap != cudaStreamCaptureStatusNone)
            return fail(MOE_ERR_STATE, "the workspace is too small for this captured call: reserve(max_tokens, top_k) before capture");
        if (int rc = grow(l, need)) return rc;
    }
    const size_t ye = f.out_dtype == MOE_F32 ? 4 : 2;
    for (int64_t t0 = 0; t0 < f.T; t0 += S) {
        const int64_t n = std::min(S, f.T - t0);
        if (int rc = forward_slice(l, f, static_cast<const uint8_t*>(f.x) + (size_t)t0 * H * 2,
                                   static_cast<uint8_t*>(f.y) + (size_t)t0 * H * ye, f.ids + t0 * f.K, f.tw + t0 * f.K, n, st))
            return rc;
    }
    return MOE_OK;
}

}  // namespace moe
