// Host-side interface of the 4-bit cache's kernels (arguments validated by the
// front end).
#pragma once

#include <hip/hip_runtime.h>

#include "bf_kv4_plan.h"
#include "bf_launch.h"

namespace bf {

// The grid of T tokens' store or load fits a launch.
bool kv4_rows_fit(const Kv4Shape& c, int T);
hipError_t kv4_store(uint8_t* data, const Kv4Shape& c, const uint16_t* K, int64_t ldk, const uint16_t* V, int64_t ldv,
                     const int64_t* slots, int T, hipStream_t st);
hipError_t kv4_load(const uint8_t* data, const Kv4Shape& c, const int64_t* slots, uint16_t* K, int64_t ldk, uint16_t* V,
                    int64_t ldv, int T, hipStream_t st);

// Rotation by position of T tokens' queries and keys, and the keys' and values' store.
struct Kv4AppendArgs {
    uint8_t* data;
    Kv4Shape c;
    const uint16_t* Q;                             // NULL: no queries
    int64_t ldq;
    uint16_t* Qo;
    int64_t ldqo;
    const uint16_t* K;
    int64_t ldk;
    uint16_t* Ko;                                  // NULL: rotated keys go to the cache only
    int64_t ldko;
    const uint16_t* V;
    int64_t ldv;
    const int64_t* slots;
    const int64_t* positions;
    const float* freq;
    int q_heads, rot, pairs, T;
    float factor;
};
bool kv4_append_fits(int T);
hipError_t kv4_append(const Kv4AppendArgs& a, hipStream_t st);

// The grids fit a launch.
bool kv4_attention_fits(const Kv4Args& a);
size_t kv4_attention_scratch_bytes(const Kv4Args& a);
// ws: kv4_attention_scratch_bytes(a) bytes (NULL when 0)
hipError_t kv4_attention(const Kv4Args& a, float* ws, hipStream_t st);

// The prompt kernel (a plan with p.prompt set).
hipError_t kv4_prompt(const Kv4Args& a, const Kv4Plan& p, int cus, hipStream_t st);

}  // namespace bf
