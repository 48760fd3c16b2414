// Host side of the MXFP4 expert layer, used by the engine (engine.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/moe_b200.h"

namespace moe {

struct MxLayer;

// Device-resident weights of one engine: for gate_up, then for down, panels of codes and their scales.
constexpr int kMxBuffers = 4;
struct MxBuffer {
    uint8_t** ptr;
    size_t bytes;
};

struct MxForward {
    const void* x;
    void* y;
    const int32_t* ids;
    const float* tw;
    int64_t T, K;
    int32_t act_dtype, out_dtype;
    const int32_t* emap;
    int32_t emap_n;
    int32_t* err;
    unsigned int* cnt;  // counters [H / 64 or more], zero between calls
    bool pdl;
    bool dense;         // every pair is this engine's
};

int mx_create(const moe_config& cfg, int num_sms, MxLayer** out);
void mx_destroy(MxLayer* l);
int mx_load(MxLayer* l, const uint8_t* w13_q, const uint8_t* w13_s, const uint8_t* w2_q, const uint8_t* w2_s, cudaStream_t st);
int mx_quantize_store(MxLayer* l, int64_t expert, int32_t proj, const void* w, int32_t dtype, cudaStream_t st);
int mx_export(MxLayer* l, int64_t expert, int32_t which, void* q_out, void* s_out);
void mx_buffers(MxLayer* l, MxBuffer (&b)[kMxBuffers]);
void mx_set_layer_experts(MxLayer* l, int64_t n);
int mx_reserve(MxLayer* l, int64_t T, int64_t K);
int mx_forward(MxLayer* l, const MxForward& f, cudaStream_t st);

}  // namespace moe
