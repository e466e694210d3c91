// Device-side parts shared by the attention kernels over the 4-bit cache: codes
// to fp16, the scaled probabilities, and which cached tokens a query sees.
#pragma once

#include "bf_device.h"
#include "bf_kv4_plan.h"

namespace bf {
namespace {

constexpr float kLow = -1e30f;                     // a maximum below every score

// Softmax over the tokens so far, kept so that fp16 holds probability times
// scale of a value: P = 2^(sc (s - base) + c), base the row's running maximum
// (raised only by a score that exceeds it by more than 3 / sc) and c = 26 - E,
// E the fp16 exponent field of the largest value scale so far of the tokens that
// some row of the wave (of the workgroup's 128 in the prompt kernel) sees.  A scale
// is below 2^(E - 14), so P d < 2^(3 + c + E - 14) = 2^15; and a product stays
// normal, hence rounded by 2^-11 of itself, down to 2^-25 of the largest
// probability's times the largest scale.  (With c = 0, values of 0.01 behind a
// token that takes most of the weight became subnormal or 0 from 12 powers of
// two on.)  The row's sum of P has the same factors.
// s - base is formed before the multiplication by sc: equal scores give equal P
// however large they are.  (Without all this, us: a prompt of 2000 tokens 92.8 and
// 93.4, 32 sequences of up to 8000 50.6 and 51.6, one of 131072 22.5 and 23.3, one of
// 519 8.05 and 8.4; heads of 96, a prompt of 2000 73 and 79.)
struct Range {
    float base = kLow;                             // (no score yet)
    float c = 26.f;                                // (c and top are the wave's)
    uint32_t top = 0x3FFu;                         // the largest scale of exponent field E
    __device__ __forceinline__ bool over(float s, float sc) const { return (s - base) * sc > 3.f; }
    __device__ __forceinline__ float p(float s, float sc) const {
        return __builtin_amdgcn_exp2f(__builtin_fmaf(s - base, sc, c));
    }
    // The row's largest score s of the tiles to come, the largest scale's field at the top: returns the factor of the
    // sums so far (0 where there are none).
    __device__ __forceinline__ float raise(float s, uint32_t to, float sc) {
        float f = 26.f - (float)(to >> 10) - c;
        c += f;
        top = to;
        if (s > base) {
            f = __builtin_fmaf(base - s, sc, f);
            base = s;
        }
        return __builtin_amdgcn_exp2f(f);
    }
    // log2 of what the row's sums are multiples of
    __device__ __forceinline__ float log2_unit(float sc) const { return base > kLow ? __builtin_fmaf(base, sc, -c) : kLow; }
};

// log2(e) |scale|: large enough that the first score exceeds kLow by 3 / sc, and a hidden token's -inf stays -inf
__device__ __forceinline__ float log2_scale(float scale) {
    return __builtin_fminf(__builtin_fmaxf(__builtin_fabsf(scale) * 1.44269504088896341f, 1e-29f), 3e38f);
}

// The larger magnitude of a word's two halves, as bits.
__device__ __forceinline__ uint32_t larger_half(uint32_t w) { return max(w & 0x7FFFu, (w >> 16) & 0x7FFFu); }
// Token t is in [lo, hi) or one of the first `sinks` below hi.
template <bool SINK> __device__ __forceinline__ bool sees(int t, int lo, int hi, int sinks) {
    return (t >= lo || (SINK && t < sinks)) && t < hi;
}
// ... of those that are finite and whose tokens t, t + 1 are seen
template <bool SINK>
__device__ __forceinline__ uint32_t larger_seen(uint32_t w, int t, int lo, int hi, int sinks) {
    const uint32_t a = w & 0x7FFFu, b = (w >> 16) & 0x7FFFu;
    return max(sees<SINK>(t, lo, hi, sinks) && a < 0x7C00u ? a : 0u, sees<SINK>(t + 1, lo, hi, sinks) && b < 0x7C00u ? b : 0u);
}
// top, or the largest value of the exponent field of the wave's largest d, if that is larger
__device__ __forceinline__ uint32_t top_of(uint32_t top, uint32_t d) {
    uint32_t e = 0;
#pragma unroll
    for (uint32_t b = 0x4000u; b >= 0x400u; b >>= 1)
        if (__any(d >= (e | b))) e |= b;
    return max(top, e | 0x3FFu);
}

__device__ __forceinline__ float half_of(const uint32_t* w, int i) { return half_bits_to_float((w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu); }

// Codes of two tokens or values per half: the nibbles at bits 0-3 / 4-7 of each half of x, minus 8.
__device__ __forceinline__ uint32_t low2(const Magic& mg, uint32_t x) {
    return as_u32(as_h2(and_or(x, mg.lo_mask, mg.lo_bits)) + h2{(_Float16)-1032.0f, (_Float16)-1032.0f});
}
__device__ __forceinline__ uint32_t high2(const Magic& mg, uint32_t x) {
    return as_u32(as_h2(and_or(x, mg.hi_mask, mg.hi_bits)) + h2{(_Float16)-72.0f, (_Float16)-72.0f});
}

// Eight K codes of one word, in order.
__device__ __forceinline__ h8 codes8(const Magic& mg, uint32_t x) {
    const uint32_t y = x >> 8;
    return __builtin_bit_cast(h8, u4{low2(mg, x), high2(mg, x), low2(mg, y), high2(mg, y)});
}

// {RN16(p d), RN16(q e)}: d and e the low or the high halves of two scale words.  (v_fma_mix forms
// the product in fp32 and rounds it once.)
__device__ __forceinline__ uint32_t scaled2(float p, float q, uint32_t d, uint32_t e, bool high) {
    uint32_t o;
    if (high) {
        asm("v_fma_mixlo_f16 %0, %1, %2, 0 op_sel:[0,1,0] op_sel_hi:[0,1,0]" : "=v"(o) : "v"(p), "v"(d));
        asm("v_fma_mixhi_f16 %0, %1, %2, 0 op_sel:[0,1,0] op_sel_hi:[0,1,0]" : "+v"(o) : "v"(q), "v"(e));
    } else {
        asm("v_fma_mixlo_f16 %0, %1, %2, 0 op_sel_hi:[0,1,0]" : "=v"(o) : "v"(p), "v"(d));
        asm("v_fma_mixhi_f16 %0, %1, %2, 0 op_sel_hi:[0,1,0]" : "+v"(o) : "v"(q), "v"(e));
    }
    return o;
}

// {RN16(p d), RN16(q e)}: d and e the low and the high half of one word.
__device__ __forceinline__ uint32_t scaled_pair(float p, float q, uint32_t de) {
    uint32_t o;
    asm("v_fma_mixlo_f16 %0, %1, %2, 0 op_sel_hi:[0,1,0]" : "=v"(o) : "v"(p), "v"(de));
    asm("v_fma_mixhi_f16 %0, %1, %2, 0 op_sel:[0,1,0] op_sel_hi:[0,1,0]" : "+v"(o) : "v"(q), "v"(de));
    return o;
}

struct Row {                                       // a row tile of a sequence
    int s, q0, nq, len, rows, row0;
    // Tiles of 32 cached tokens that it sees: t0 .. t1 - 1.  With first tokens in sight (sinks) whose tiles lie before
    // the window's: those below w0 stand for tiles 0 .. w0 - t0 - 1, the window's begin at w0.
    int t0, t1, w0;
    template <bool SINK> __device__ __forceinline__ int tile(int i) const { return SINK && i < w0 ? i - t0 : i; }
};

// Cached tokens [lo, hi) that query i of the sequence sees.
__device__ __forceinline__ int hi_of(const Kv4Args& a, const Row& o, int i) {
    return a.causal ? max(0, o.len - o.nq + i + 1) : o.len;
}
__device__ __forceinline__ int lo_of(const Kv4Args& a, const Row& o, int i) {
    return a.window > 0 ? max(0, max(0, o.len - o.nq + i + 1) - a.window) : 0;   // (positions down to -2^30, windows up to 2^31 - 1)
}

// Item i = s row_tiles + rt; false where it has no rows.
template <bool SINK>
__device__ __forceinline__ bool row_tile_of(const Kv4Args& a, const Kv4Plan& p, int i, Row& o) {
    int rt = 0;
    o.s = i;
    if (p.row_tiles > 1) {
        o.s = i / p.row_tiles;
        rt = i - o.s * p.row_tiles;
    }
    const int qa = a.q_start[o.s], qb = a.q_start[o.s + 1], len = a.kv_len[o.s];
    o.q0 = min(max(qa, 0), a.T);
    o.nq = min(min(max(qb, o.q0), a.T) - o.q0, a.max_q);
    o.len = min(max(len, 0), a.max_kv);
    o.row0 = rt * p.tile_rows;
    const int64_t left = (int64_t)o.nq * p.group - o.row0;
    o.rows = left < p.tile_rows ? (int)left : p.tile_rows;
    if (o.rows <= 0) return false;
    const int hi = hi_of(a, o, (o.row0 + o.rows - 1) / p.group);
    o.w0 = o.t0 = lo_of(a, o, o.row0 / p.group) / kKv4Tile;
    o.t1 = max(o.t0, (hi + kKv4Tile - 1) / kKv4Tile);
    if constexpr (SINK) {
        const int first = (min(a.sinks, hi) + kKv4Tile - 1) / kKv4Tile;    // tiles of the first tokens
        if (first < o.w0) o.t0 -= first;
        else o.w0 = o.t0 = 0;
    }
    return true;
}

__device__ __forceinline__ void store_out(const Kv4Args& a, int64_t at, float y) {
    if (a.out_f16) ((_Float16*)a.O)[at] = (_Float16)y;
    else ((float*)a.O)[at] = y;
}

}  // namespace
}  // namespace bf
