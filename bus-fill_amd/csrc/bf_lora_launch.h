// Host-side interface of the low-rank adapters' kernels (arguments validated by
// the front end).
#pragma once

#include <hip/hip_runtime.h>

#include "bf_lora_plan.h"

namespace bf {

bool lora_fits(const LoraArgs& a);
size_t lora_scratch_bytes(const LoraArgs& a);
// ws: lora_scratch_bytes(a) bytes
hipError_t lora(const LoraArgs& a, float* ws, hipStream_t st);

}  // namespace bf
