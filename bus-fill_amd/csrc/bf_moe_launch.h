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
bool moe_route_fits(int T);    // its grid fits a launch
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

// One of the two products over tiles of gathered rows (bf_moe_tile.hip).
constexpr int kMoeTileRows = 256;
struct MoeTileArgs {
    const uint8_t *W[2], *aux[2];  // gate and up, or down
    const uint16_t* A;         // rows of tokens, or of slots
    uint32_t a_bytes;          // from A on: below 4 GB
    int64_t lda;
    void* out;                 // h (fp16) or y (bf_moe_dev.h), by slot
    int R, K;                  // weight rows of an expert, their length
    int nt[2];                 // column tiles of a large and of a small tile's rows
    const int32_t* perm;       // slots by expert
    const int4* table;         // max_tiles large tiles, then the small ones: expert, first place in perm, rows
    const int* tiles;          // how many of either
    int max_tiles;             // of both together
    int run;                   // rows of a run: 64 (small tiles only) or kMoeTileRows
};

// y in 24 bits, else in 32 (bf_moe_dev.h).
constexpr int kMoeTileSlots = 24;                  // slots an expert, on average, from which tiles take the products
__host__ __device__ inline bool y_24(const MoeArgs& a) {
    return a.out_f16 && (int64_t)a.T * a.k >= kMoeTileSlots * (int64_t)a.E;
}
// Bytes of the plane of its upper 16 bits.
__host__ __device__ inline int64_t y_24_high(const MoeArgs& a) { return ((int64_t)a.T * a.k * a.N * 2 + 255) & ~(int64_t)255; }

hipError_t moe_tile(const MoeArgs& a, const MoeTileArgs& o, bool gu, hipStream_t st);

// The matrix-core kernels serve these widths and alignments.
bool moe_fast(const MoeArgs& a);
size_t moe_scratch_bytes(const MoeArgs& a);
// ws: moe_scratch_bytes(a) bytes, 256-byte aligned
hipError_t moe_ffn(const MoeArgs& a, uint8_t* ws, hipStream_t st);

}  // namespace bf
