// Store and read-back of the 4-bit key/value cache (layout: bf_kv4.h).
//
// Store, per 32 values x of a head: m = the value of largest magnitude (the
// first of equals), d = RN16(m / -8), q = clamp(floor(x / d + 8.5), 0, 15), so
// m itself is code 0 and x is at most d / 2 from (q - 8) d inside the range (d
// on the far side, where +m would be code 16).  x and d are fp16, 11-bit
// integers times powers of two, so x / d is either exactly half way between two
// integers or at least 2^-13 from it: floor(x rcp(d) + 8.5 + 2^-14), off by less
// than 2^-18 in fp32, gives the codes of the exact formula without a division.
// d = 0: all codes 8.  A block with an infinity or a NaN gets d = NaN, codes 8: it
// reads as NaN, not as a finite guess.
//
// Bytes: 2 read and 9/16 written per value (the read-back the other way).  2000
// tokens of 8 heads of 128: 5.7 us to store and 6.0 to load 10.5 MB (a copy's rate
// would be 2.2), 131072 tokens of 4 heads 88 us, 3.9 TB/s; 32 tokens 4.1 and 3.7 us,
// a launch and its first loads.  A block per thread, so that its scale needs no
// other lane; the price is values' codes stored byte by byte, 32 tokens apart.
#include "bf_device.h"
#include "bf_grid.h"
#include "bf_kv4_launch.h"

namespace bf {
namespace {

constexpr uint32_t kNan16 = 0x7E00u;

// Nibble of element e (0..7) in a word of K codes.
__device__ constexpr int knib(int e) { return (e >> 1) + 4 * (e & 1); }

__device__ __forceinline__ float half_at(const u4 x[4], int e) {
    return half_bits_to_float((x[e >> 3][(e >> 1) & 3] >> (16 * (e & 1))) & 0xFFFFu);
}

// One block's scale bits and codes.
__device__ __forceinline__ uint32_t quantize32(const u4 x[4], uint8_t q[32]) {
    float hi = half_at(x, 0), lo = hi, bad = 0.f;
    const h2 none = {(_Float16)0.f, (_Float16)0.f};
#pragma unroll
    for (int e = 0; e < 32; e++) {
        hi = __builtin_fmaxf(hi, half_at(x, e));
        lo = __builtin_fminf(lo, half_at(x, e));
        if ((e & 1) == 0) bad = __builtin_amdgcn_fdot2(as_h2(x[e >> 3][(e >> 1) & 3]), none, bad, false);   // NaN from an infinity or NaN
    }
    float m = hi > -lo ? hi : lo;
    if (hi == -lo)                                     // both magnitudes: the first of them
#pragma unroll
        for (int e = 31; e >= 0; e--)
            if (__builtin_fabsf(half_at(x, e)) == hi) m = half_at(x, e);
    const _Float16 d16 = (_Float16)(m * -0.125f);
    const float r = __builtin_amdgcn_rcpf((float)d16);
#pragma unroll
    for (int e = 0; e < 32; e++) {
        const float t = __builtin_floorf(__builtin_fmaf(half_at(x, e), r, 8.5f + 0x1p-14f));
        q[e] = (uint8_t)(int)__builtin_fminf(__builtin_fmaxf(t, 0.f), 15.f);
    }
    if (bad == 0.f && d16 != (_Float16)0.f) return __builtin_bit_cast(uint16_t, d16);
#pragma unroll
    for (int e = 0; e < 32; e++) q[e] = 8;
    return bad == 0.f ? 0u : kNan16;
}

// The record and token of a slot; false for a slot outside the cache.
__device__ __forceinline__ bool slot_at(const Kv4Shape& c, int64_t slot, int head, int64_t& rec, int& t) {
    if (slot < 0) return false;
    const int64_t page = slot / c.page_size;
    if (page >= c.pages) return false;
    const int in = (int)(slot - page * c.page_size);
    rec = kv4_record(page, head, in / kKv4Tile, c.heads, c.page_size / kKv4Tile);
    t = in % kKv4Tile;
    return true;
}

// One block (32 values) per thread: token, block; heads along grid y, keys and
// values along z (a wave of both would take both ways through the codes' places).
__global__ __launch_bounds__(256) void k_kv4_store(uint8_t* __restrict__ data, Kv4Shape c, const uint16_t* __restrict__ K,
                                                   int64_t ldk, const uint16_t* __restrict__ V, int64_t ldv,
                                                   const int64_t* __restrict__ slots, int T) {
    const int nb = c.dim / 32, head = blockIdx.y;
    const int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x;
    const int64_t t = i / nb;
    if (t >= T) return;
    const int b = (int)(i - t * nb);
    const bool isv = blockIdx.z;
    const uint16_t* src = (isv ? V + t * ldv : K + t * ldk) + head * c.dim + 32 * b;
    u4 x[4];
#pragma unroll
    for (int w = 0; w < 4; w++) x[w] = *(const u4*)(src + 8 * w);
    int64_t rec;
    int tok;
    if (!slot_at(c, slots[t], head, rec, tok)) return;
    uint8_t q[32];
    const uint32_t d = quantize32(x, q);
    uint8_t* r = data + rec * kv4_record_bytes(c.dim);
    if (isv) {
        uint8_t* p = r + kv4_v_at(c.dim, tok, b, 0);
        const int step = kv4_v_at(c.dim, tok, b, 1) - kv4_v_at(c.dim, tok, b, 0);
#pragma unroll
        for (int e = 0; e < 16; e++) p[step * e] = (uint8_t)(q[e] | q[16 + e] << 4);
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            uint32_t w = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) w |= (uint32_t)q[8 * k + e] << (4 * knib(e));
            *(uint32_t*)(r + kv4_k_at(c.dim, tok, b, k)) = w;
        }
    }
    *(uint16_t*)(r + (isv ? kv4_vs_at(c.dim, tok, b) : kv4_ks_at(c.dim, tok, b))) = (uint16_t)d;
}

// The same units back to fp16: RN16((q - 8) d), the product exact in fp32.
__global__ __launch_bounds__(256) void k_kv4_load(const uint8_t* __restrict__ data, Kv4Shape c,
                                                  const int64_t* __restrict__ slots, uint16_t* __restrict__ K,
                                                  int64_t ldk, uint16_t* __restrict__ V, int64_t ldv, int T) {
    const int nb = c.dim / 32, head = blockIdx.y;
    const int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x;
    const int64_t t = i / nb;
    if (t >= T) return;
    const int b = (int)(i - t * nb);
    const bool isv = blockIdx.z;
    u4 out[4] = {};
    int64_t rec;
    int tok;
    if (slot_at(c, slots[t], head, rec, tok)) {
        const uint8_t* r = data + rec * kv4_record_bytes(c.dim);
        const float d = half_bits_to_float(*(const uint16_t*)(r + (isv ? kv4_vs_at(c.dim, tok, b) : kv4_ks_at(c.dim, tok, b))));
        uint8_t q[32];
        if (isv) {
            const uint8_t* p = r + kv4_v_at(c.dim, tok, b, 0);
            const int step = kv4_v_at(c.dim, tok, b, 1) - kv4_v_at(c.dim, tok, b, 0);
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const uint32_t v = p[step * e];
                q[e] = v & 15;
                q[16 + e] = v >> 4;
            }
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const uint32_t w = *(const uint32_t*)(r + kv4_k_at(c.dim, tok, b, k));
#pragma unroll
                for (int e = 0; e < 8; e++) q[8 * k + e] = (w >> (4 * knib(e))) & 15;
            }
        }
#pragma unroll
        for (int e = 0; e < 32; e++)
            out[e >> 3][(e >> 1) & 3] |=
                (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)((float)((int)q[e] - 8) * d)) << (16 * (e & 1));
    }
    uint16_t* dst = (isv ? V + t * ldv : K + t * ldk) + head * c.dim + 32 * b;
#pragma unroll
    for (int w = 0; w < 4; w++) *(u4*)(dst + 8 * w) = out[w];
}

int64_t units_groups(const Kv4Shape& c, int T) { return ((int64_t)T * (c.dim / 32) + 255) / 256; }
dim3 units_grid(const Kv4Shape& c, int T) { return dim3((unsigned)units_groups(c, T), (unsigned)c.heads, 2); }

}  // namespace

bool kv4_rows_fit(const Kv4Shape& c, int T) { return launch_fits(units_groups(c, T), 256); }

hipError_t kv4_store(uint8_t* data, const Kv4Shape& c, const uint16_t* K, int64_t ldk, const uint16_t* V, int64_t ldv,
                     const int64_t* slots, int T, hipStream_t st) {
    hipLaunchKernelGGL(k_kv4_store, units_grid(c, T), dim3(256), 0, st, data, c, K, ldk, V, ldv, slots, T);
    return hipGetLastError();
}

hipError_t kv4_load(const uint8_t* data, const Kv4Shape& c, const int64_t* slots, uint16_t* K, int64_t ldk, uint16_t* V,
                    int64_t ldv, int T, hipStream_t st) {
    hipLaunchKernelGGL(k_kv4_load, units_grid(c, T), dim3(256), 0, st, data, c, slots, K, ldk, V, ldv, T);
    return hipGetLastError();
}

}  // namespace bf
