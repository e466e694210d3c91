// Rotation of queries and keys by their positions, and the store of keys and
// values into the 4-bit cache (layout: bf_kv4.h), in one launch.
//
// A pair (x, y) of a head, the i-th of rot / 2, turns by the angle t = position
// freq[i]:  (x cos t - y sin t, y cos t + x sin t) factor.  Far positions: the
// angle in turns, position (freq / 2 pi), is formed in 64 bits (24-bit freq times
// a position below 2^31: off by less than 2^-23 of a turn) and its fraction goes to fp32, where
// sine and cosine are good to an ulp or two; products and sums are fp32, rounded
// once to fp16.  Keys are quantized from those fp16 values with the rule of
// k_kv4_store (bf_kv4.hip), so rotating, rounding and storing in separate steps
// gives the same bits.
//
// Bound by memory (2 bytes in and 2 out per element of q; 2 in and 9/16 out per
// element of k and v).  A workgroup takes a token: its angles are formed once, in
// LDS, then every lane takes eight neighbouring elements of a head, whose angles
// it keeps for all heads.  Halves of a pair in other lanes come by shuffles, so
// rows may be rotated in place.
//
// Measured, 40 query heads over 8 of 128: 2000 tokens 13.8 to 15.4 us for 51 MB (3.5
// TB/s, where 51 MB at a copy's 4.87 TB/s are 10.5 us; vector instructions issue in 68 % of
// the cycles, and the values' codes, stored byte by byte because a word holds eight
// tokens', cost 10 MB of partial writes); 32 tokens 3.9 us, the chain of
// position, sine, rotation and store after the launch.  Loads four items ahead took
// 16.9 us where this took 15.2: registers, so fewer waves.
#include <algorithm>

#include "bf_device.h"
#include "bf_grid.h"
#include "bf_kv4_launch.h"

namespace bf {
namespace {

constexpr uint32_t kNan16 = 0x7E00u;
constexpr int kThreads = 256;

__device__ constexpr int knib(int e) { return (e >> 1) + 4 * (e & 1); }   // nibble of element e in a word of K codes

__device__ __forceinline__ uint32_t other(uint32_t x, int lane) { return (uint32_t)__shfl((int)x, lane); }

// Codes (one a nibble, element e at 4 e) of a lane's eight values, four neighbouring lanes a block of 32; the block's
// scale bits.  As quantize32 of bf_kv4.hip.
__device__ __forceinline__ uint32_t quantize8(const float x[8], int g, uint32_t& scale) {
    float hi = x[0], lo = x[0], bad = 0.f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        hi = __builtin_fmaxf(hi, x[e]);
        lo = __builtin_fminf(lo, x[e]);
        bad += x[e] * 0.f;                             // NaN from an infinity or NaN
    }
#pragma unroll
    for (int s = 1; s < 4; s <<= 1) {
        hi = __builtin_fmaxf(hi, __shfl_xor(hi, s));
        lo = __builtin_fminf(lo, __shfl_xor(lo, s));
        bad += __shfl_xor(bad, s);
    }
    float m = hi > -lo ? hi : lo;
    int first = 64;                                    // both magnitudes: the first of them
#pragma unroll
    for (int e = 7; e >= 0; e--)
        if (__builtin_fabsf(x[e]) == hi) first = 2 * (8 * g + e) + (x[e] < 0.f);
    first = min(first, __shfl_xor(first, 1));
    first = min(first, __shfl_xor(first, 2));
    if (hi == -lo) m = first & 1 ? lo : hi;
    const _Float16 d16 = (_Float16)(m * -0.125f);
    const float r = __builtin_amdgcn_rcpf((float)d16);
    uint32_t q = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float t = __builtin_floorf(__builtin_fmaf(x[e], r, 8.5f + 0x1p-14f));
        q |= (uint32_t)(int)__builtin_fminf(__builtin_fmaxf(t, 0.f), 15.f) << (4 * e);
    }
    scale = __builtin_bit_cast(uint16_t, d16);
    if (!(bad == 0.f) || d16 == (_Float16)0.f) {
        q = 0x88888888u;
        scale = bad == 0.f ? 0u : kNan16;
    }
    return q;
}

// Token `t` of a record at `rec`: a lane's eight codes of block b, part g.
__device__ __forceinline__ void put_key(uint8_t* rec, int D, int t, int b, int g, uint32_t q, uint32_t scale) {
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) w |= ((q >> (4 * e)) & 15u) << (4 * knib(e));
    *(uint32_t*)(rec + kv4_k_at(D, t, b, g)) = w;
    if (g == 0) *(uint16_t*)(rec + kv4_ks_at(D, t, b)) = (uint16_t)scale;
}
// ... of values: columns 8 (g % 2) + 4 (g / 2) .. + 3 of the block's 16, `far` the codes of lane g ^ 2
__device__ __forceinline__ void put_value(uint8_t* rec, int D, int t, int b, int g, uint32_t q, uint32_t far, uint32_t scale) {
    const uint32_t low = g < 2 ? q : far >> 16, high = g < 2 ? far : q >> 16;
    uint8_t* p = rec + kv4_v_at(D, t, b, 8 * (g & 1) + 4 * (g >> 1));
    const int step = kv4_v_at(D, t, b, 1) - kv4_v_at(D, t, b, 0);
#pragma unroll
    for (int e = 0; e < 4; e++) p[step * e] = (uint8_t)(((low >> (4 * e)) & 15u) | ((high >> (4 * e)) & 15u) << 4);
    if (g == 0) *(uint16_t*)(rec + kv4_vs_at(D, t, b)) = (uint16_t)scale;
}

// LN lanes a head (D / 8 of them at work).  Grid: tokens, parts of the heads.
template <int D, bool PAIRS>
__global__ __launch_bounds__(kThreads) void k_kv4_append(Kv4AppendArgs a) {
    constexpr int LN = D == 64 ? 8 : D == 256 ? 32 : 16, HW = 64 / LN;     // heads of a wave
    __shared__ float2 turn[D / 2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int64_t t = blockIdx.x;
    if ((int)threadIdx.x < a.rot / 2) {
        const double turns = (double)a.positions[t] * ((double)a.freq[threadIdx.x] * 0.15915494309189533577);
        float s, c;
        sincospif(2.f * (float)(turns - __builtin_rint(turns)), &s, &c);
        turn[threadIdx.x] = float2{c * a.factor, s * a.factor};
    }
    __syncthreads();
    const int p = lane % LN, el = 8 * p, half = a.rot / 2;
    const bool in = el < D, rotated = el < a.rot;
    // Angles of the lane's elements: of (el + e) mod half, or of el / 2 + e / 2
    float2 cs[8];
    if (rotated) {
#pragma unroll
        for (int e = 0; e < 8; e++) cs[e] = turn[PAIRS ? (el >> 1) + (e >> 1) : el < half ? el + e : el - half + e];
    }
    const int mate = PAIRS || !rotated ? lane : el < half ? lane + half / 8 : lane - half / 8;
    const int64_t slot = a.slots[t];
    int64_t page = slot / a.c.page_size;
    const bool stored = slot >= 0 && page < a.c.pages;
    const int at = (int)(slot - page * a.c.page_size);
    const int qi = a.Q ? (a.q_heads + HW - 1) / HW : 0, ki = (a.c.heads + HW - 1) / HW;
    for (int i = blockIdx.y * (kThreads / 64) + wave; i < qi + 2 * ki; i += gridDim.y * (kThreads / 64)) {
        const int kind = i < qi ? 0 : i < qi + ki ? 1 : 2;             // queries, keys, values: the same in a wave
        const int h = (i - (kind == 0 ? 0 : kind == 1 ? qi : qi + ki)) * HW + lane / LN;
        const bool live = in && h < (kind == 0 ? a.q_heads : a.c.heads);
        const int64_t from = (kind == 0 ? t * a.ldq : kind == 1 ? t * a.ldk : t * a.ldv) + h * D + el;
        u4 raw = u4{0, 0, 0, 0};
        if (live) raw = *(const u4*)((kind == 0 ? a.Q : kind == 1 ? a.K : a.V) + from);
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = half_bits_to_float((raw[e >> 1] >> (16 * (e & 1))) & 0xFFFFu);
        if (kind < 2) {
            u4 far;
#pragma unroll
            for (int w = 0; w < 4; w++) far[w] = PAIRS ? raw[w] : other(raw[w], mate);
            if (rotated) {
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float z = PAIRS ? x[e ^ 1] : half_bits_to_float((far[e >> 1] >> (16 * (e & 1))) & 0xFFFFu);
                    const bool first = PAIRS ? (e & 1) == 0 : el < half;
                    y[e] = x[e] * cs[e].x + (first ? -(z * cs[e].y) : z * cs[e].y);
                }
                raw = f32x8_to_f16(f4{y[0], y[1], y[2], y[3]}, f4{y[4], y[5], y[6], y[7]});
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = half_bits_to_float((raw[e >> 1] >> (16 * (e & 1))) & 0xFFFFu);
            }
            uint16_t* const to = kind == 0 ? a.Qo + t * a.ldqo : a.Ko ? a.Ko + t * a.ldko : nullptr;
            if (live && to) *(u4*)(to + h * D + el) = raw;
        }
        if (kind > 0) {
            const int b = p >> 2, g = p & 3;
            uint32_t scale;
            const uint32_t q = quantize8(x, g, scale), far = other(q, lane ^ 2);
            if (live && stored) {
                uint8_t* rec = a.data + kv4_record(page, h, at / kKv4Tile, a.c.heads, a.c.page_size / kKv4Tile) * kv4_record_bytes(D);
                if (kind == 1) put_key(rec, D, at % kKv4Tile, b, g, q, scale);
                else put_value(rec, D, at % kKv4Tile, b, g, q, far, scale);
            }
        }
    }
}

template <int D> void go(const Kv4AppendArgs& a, hipStream_t st) {
    constexpr int HW = 64 / (D == 64 ? 8 : D == 256 ? 32 : 16);
    const int items = (a.Q ? (a.q_heads + HW - 1) / HW : 0) + 2 * ((a.c.heads + HW - 1) / HW);
    // few tokens: the heads over several workgroups, a turn each
    const int turns = (items + kThreads / 64 - 1) / (kThreads / 64), most = std::max(1, 512 / a.T);
    const dim3 grid((unsigned)a.T, (unsigned)std::min(turns, most));
    if (a.pairs) hipLaunchKernelGGL((k_kv4_append<D, true>), grid, dim3(kThreads), 0, st, a);
    else hipLaunchKernelGGL((k_kv4_append<D, false>), grid, dim3(kThreads), 0, st, a);
}

}  // namespace

bool kv4_append_fits(int T) { return launch_fits(T, kThreads); }

hipError_t kv4_append(const Kv4AppendArgs& a, hipStream_t st) {
    switch (a.c.dim) {
        case 64: go<64>(a, st); break;
        case 96: go<96>(a, st); break;
        case 128: go<128>(a, st); break;
        default: go<256>(a, st); break;
    }
    return hipGetLastError();
}

}  // namespace bf
