// Device-side parts shared by the experts' kernels: the routing weight's two parts,
// and y, the down product of every slot, between the launch that makes it and the
// one that sums a row's slots.
//
// The weight: its power of two, from 1/8 to 1, goes into h before h is rounded to
// fp16, the rest multiplies y in the fp32 sum.  All of it in h makes h subnormal
// where weights are small (1e-4 over h of 0.05: up to 6e-3 of it lost); none of it makes h
// infinite from 65504 on, where eight weights of 1/8 reach 5e5.
//
// y is fp32; for fp16 outputs from kMoeTileSlots slots an expert on, where its bytes count
// (2000 rows of eight slots and 4096 outputs: 262 MB), the upper 24 bits of the fp32, to
// nearest: fp32's range, so terms that cancel may be of any size, and 2^-16 of a
// term's own size, 32 times finer than the output's rounding.  Two planes: the
// upper 16 bits, then the next eight.  (That block in us, y in fp16, in which a term
// above 65504 is infinite, 24 bits, fp32: 938, 963, 957; workspace for y 131, 197, 262 MB.)
#pragma once

#include "bf_device.h"
#include "bf_moe_launch.h"

namespace bf {
namespace {

__device__ __forceinline__ uint32_t weight_exponent(float w) {   // 124 (1/8) to 127 (1)
    return min(max((__builtin_bit_cast(uint32_t, w) >> 23) & 0xFFu, 124u), 127u);
}
__device__ __forceinline__ float weight_in_h(float w) { return __builtin_bit_cast(float, weight_exponent(w) << 23); }
__device__ __forceinline__ float weight_of_y(float w) { return w * __builtin_bit_cast(float, (254u - weight_exponent(w)) << 23); }   // (exact)

// The bits of v, its upper 24 to nearest (ties away from 0; to even, and NaNs apart,
// took 5 us more of the down products' 316).  Infinities stay, and so do NaNs: they
// come from fp16 operands and from sums, whose NaNs have clear low bits.
__device__ __forceinline__ uint32_t round24(float v) { return __builtin_bit_cast(uint32_t, v) + 0x80u; }

__device__ __forceinline__ void store_y(const MoeArgs& a, void* y, int64_t at, float v) {
    if (!y_24(a)) {
        ((float*)y)[at] = v;
        return;
    }
    const uint32_t r = round24(v);
    ((uint16_t*)y)[at] = (uint16_t)(r >> 16);
    ((uint8_t*)y + y_24_high(a))[at] = (uint8_t)(r >> 8);
}

// u[i] of lane 4 m + q and u[q] of lane 4 m + i change places.
__device__ __forceinline__ void transpose4(uint32_t u[4], int lane) {
    const bool odd = lane & 1, high = lane & 2;
#pragma unroll
    for (int p = 0; p < 4; p += 2) {
        const uint32_t got = (uint32_t)__builtin_amdgcn_mov_dpp((int)(odd ? u[p] : u[p + 1]), 0xB1, 0xF, 0xF, true);   // lane ^ 1
        if (odd) u[p] = got;
        else u[p + 1] = got;
    }
#pragma unroll
    for (int p = 0; p < 2; p++) {
        const uint32_t got = (uint32_t)__builtin_amdgcn_mov_dpp((int)(high ? u[p] : u[p + 2]), 0x4E, 0xF, 0xF, true);  // lane ^ 2
        if (high) u[p] = got;
        else u[p + 2] = got;
    }
}

// Four in a row, `at` and a.N multiples of 4: u are their bits (24 of them valid, for y in 24 bits).
__device__ __forceinline__ void store_y4(const MoeArgs& a, void* y, int64_t at, const uint32_t u[4]) {
    if (!y_24(a)) {
        *(u4*)((float*)y + at) = u4{u[0], u[1], u[2], u[3]};
        return;
    }
    *(uint2*)((uint16_t*)y + at) = uint2{perm_b32(u[1], u[0], 0x07060302u), perm_b32(u[3], u[2], 0x07060302u)};
    *(uint32_t*)((uint8_t*)y + y_24_high(a) + at) =
        perm_b32(perm_b32(u[3], u[2], 0x0C0C0501u), perm_b32(u[1], u[0], 0x0C0C0501u), 0x05040100u);
}

// Four in a row; whole: n % 4 == 0 and all four are there, else `left` of them (the others 0).
template <bool Y24>
__device__ __forceinline__ f4 load_y4(const MoeArgs& a, const void* y, int64_t at, bool whole, int left) {
    f4 v = f4{0.f, 0.f, 0.f, 0.f};
    if constexpr (!Y24) {
        const float* p = (const float*)y + at;
        if (whole) return *(const f4*)p;
        for (int i = 0; i < 4 && i < left; i++) v[i] = p[i];
    } else {
        const uint16_t* p = (const uint16_t*)y + at;
        const uint8_t* q = (const uint8_t*)y + y_24_high(a) + at;
        if (whole) {
            const uint2 h = *(const uint2*)p;
            const uint32_t l = *(const uint32_t*)q;
            return f4{__builtin_bit_cast(float, h.x << 16 | (l & 0xFFu) << 8), __builtin_bit_cast(float, (h.x & 0xFFFF0000u) | (l & 0xFF00u)),
                      __builtin_bit_cast(float, h.y << 16 | (l >> 8 & 0xFF00u)), __builtin_bit_cast(float, (h.y & 0xFFFF0000u) | (l >> 16 & 0xFF00u))};
        }
        for (int i = 0; i < 4 && i < left; i++) v[i] = __builtin_bit_cast(float, (uint32_t)p[i] << 16 | (uint32_t)q[i] << 8);
    }
    return v;
}

}  // namespace
}  // namespace bf
