// Host-side interface of the mixture-of-experts kernels (arguments validated by
// the front end).
#pragma once

#include <hip/hip_runtime.h>

#include "bf_launch.h"

namespace bf {

struct RouteArgs {
    const void* logits;
    int f16;                   // logits are fp16, else fp32
    int64_t ldl;
    const float* bias;         // [E] or NULL
    int32_t* ids;              // [T][k]
    float* w;                  // [T][k]
    int T, E, k;
    int sigmoid, groups, top_groups, renorm;
    float factor;
};
hipError_t moe_route(const RouteArgs& a, hipStream_t st);

struct MoeArgs {
    int qtype;
    const uint8_t *gate, *gate_aux, *up, *up_aux, *down, *down_aux;   // expert e's rows behind expert e - 1's
    const uint16_t* A;
    int lda;
    const int32_t* ids;        // [T][k]
    const float* w;            // [T][k]
    void* C;
    int ldc, out_f16;
    int T, K, F, N, E, k;
};
// The matrix-core kernels serve these widths and alignments.
bool moe_fast(const MoeArgs& a);
size_t moe_scratch_bytes(const MoeArgs& a);
// ws: moe_scratch_bytes(a) bytes, 256-byte aligned
hipError_t moe_ffn(const MoeArgs& a, uint8_t* ws, hipStream_t st);

}  // namespace bf
