// Low-rank adapters of many requests beside a shared projection:
//   Y[t] = C[t] + scale_e B_e (A_e x[t]),  e = ids[t]  (no adapter: Y[t] = C[t]),
// for up to four parts (a fused projection's slices), each with its A and B.
//
// Two launches: s = A x in fp32 (k_lora_down), then C + scale B s (k_lora_up).
// Rows are taken 16 at a time, as one operand of 16x16x32 MFMAs; a tile's rows
// may be of 16 different adapters, and each adapter of a tile is multiplied with
// all 16 rows, of which its own are kept.  So nothing is sorted and no row moves:
// single tokens of many requests are bound by the adapters' bytes whatever the
// products do, and in prompts neighbouring rows are of one adapter.
//
// Down: operands go from memory to registers; x and A are fp16, their products
// exact, sums fp32.  K is cut into pieces (partial sums in the workspace, added
// by the up products in their order), so that a few rows fill the chip.
// Up: s, times a power of two that brings the row's largest to 2^14..2^15, is
// taken as two fp16 numbers (rounded, and the rest rounded: 2^-22 of s), so the
// products lose nothing that fp32 would keep; sums fp32, one rounding of Y.
#include "bf_device.h"
#include "bf_grid.h"
#include "bf_launch.h"
#include "bf_lora_launch.h"

namespace bf {
namespace {

constexpr int kWaves = 4;

// A tile's adapters: lane l holds row l % 16's (-1: none; -2: past the last row).
struct Tile {
    int t0, id;
    uint32_t firsts;                               // rows that are the first of their adapter
};

__device__ __forceinline__ Tile tile_at(const LoraArgs& a, int tile, int lane) {
    Tile o;
    o.t0 = tile * kLoraRows;
    const int t = o.t0 + (lane & 15);
    o.id = -2;
    if (t < a.T) {
        o.id = a.ids[t];
        if (o.id < 0 || o.id >= a.adapters) o.id = -1;
    }
    bool first = lane < 16 && o.id != -2;
#pragma unroll
    for (int r = 0; r < 15; r++) {
        const int e = __builtin_amdgcn_readlane(o.id, r);
        if (lane > r && o.id == e) first = false;
    }
    o.firsts = (uint32_t)__ballot(first);
    return o;
}

__device__ __forceinline__ int rank_of(const LoraArgs& a, int e) {
    return a.ranks ? min(max(a.ranks[e], 0), a.rank) : a.rank;
}

__device__ __forceinline__ h8 zero8() {
    const h8 z = {};
    return z;
}

// Unit: part, ranks, piece of K, tile, sharer (the fastest).
__global__ __launch_bounds__(64 * kWaves) void k_lora_down(LoraArgs a, LoraPlan p, float* __restrict__ ws) {
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    int64_t u = (int64_t)blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    if (u >= p.down_units) return;
    const int share = (int)(u % p.down_sharers);
    u /= p.down_sharers;
    const int tile = (int)(u % p.tiles);
    u /= p.tiles;
    const int piece = (int)(u % p.pieces);
    u /= p.pieces;
    const int r0 = (int)(u % p.rank_parts) * kLoraRanks, part = (int)(u / p.rank_parts);
    const Tile o = tile_at(a, tile, lane);
    const int k0 = piece * p.piece * kLoraStep, k1 = min(a.K, k0 + p.piece * kLoraStep);
    const uint16_t* const x = a.X + (int64_t)min(o.t0 + r, a.T - 1) * a.ldx;
    float* const out = ws + ((int64_t)part * p.pieces + piece) * a.T * a.rank;
    int nth = 0;
    for (uint32_t left = o.firsts; left; left &= left - 1) {
        const int e = __builtin_amdgcn_readlane(o.id, __builtin_ctz(left));
        if (e < 0 || nth++ % p.down_sharers != share) continue;
        const int ranks = rank_of(a, e);
        if (r0 >= ranks) continue;
        const uint16_t* const A = a.part[part].A + (int64_t)e * a.rank * a.K;
        const uint16_t* w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = A + (int64_t)min(r0 + 16 * i + r, ranks - 1) * a.K;   // (rows past the rank: not kept)
        const int tiles = min(4, (ranks - r0 + 15) / 16);
        f4 acc[4];
#pragma unroll
        for (int i = 0; i < 4; i++) acc[i] = f4{0.f, 0.f, 0.f, 0.f};
        for (int k = k0; k < k1; k += kLoraStep) {
            const int kk = k + 8 * g;
            const bool in = kk < k1;               // (K % 8 == 0)
            const h8 xv = in ? *(const h8*)(x + kk) : zero8();
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (i < tiles) acc[i] = mfma16x16x32(in ? *(const h8*)(w[i] + kk) : zero8(), xv, acc[i]);
        }
        // lane: row r of the tile, ranks r0 + 16 i + 4 g ..
        if (o.id == e) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int at = r0 + 16 * i + 4 * g;
                if (i < tiles && at < a.rank) *(f4*)(out + (int64_t)(o.t0 + r) * a.rank + at) = acc[i];   // (rank % 8 == 0)
            }
        }
    }
}

__device__ __forceinline__ float load_c(const LoraArgs& a, int64_t i) {
    return a.out_f16 ? (float)((const _Float16*)a.C)[i] : ((const float*)a.C)[i];
}
__device__ __forceinline__ void store_y(const LoraArgs& a, int64_t i, float y) {
    if (a.out_f16) ((_Float16*)a.Y)[i] = (_Float16)y;
    else ((float*)a.Y)[i] = y;
}

// Sixteen neighbouring columns of a row, n of them inside: Y = C + f d.
__device__ __forceinline__ void add16(const LoraArgs& a, int64_t ci, int64_t yi, const float* d, float f, int n) {
    if (a.wide && n >= 16) {
        if (a.out_f16) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const h8 c = *(const h8*)((const _Float16*)a.C + ci + 8 * i);
                f4 lo, hi;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    lo[e] = __builtin_fmaf(f, d[8 * i + e], (float)c[e]);
                    hi[e] = __builtin_fmaf(f, d[8 * i + 4 + e], (float)c[4 + e]);
                }
                *(u4*)((_Float16*)a.Y + yi + 8 * i) = f32x8_to_f16(lo, hi);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                f4 c = *(const f4*)((const float*)a.C + ci + 4 * i);
#pragma unroll
                for (int e = 0; e < 4; e++) c[e] = __builtin_fmaf(f, d[4 * i + e], c[e]);
                *(f4*)((float*)a.Y + yi + 4 * i) = c;
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 16; e++)
            if (e < n) store_y(a, yi + e, __builtin_fmaf(f, d[e], load_c(a, ci + e)));
    }
}

// Unit: tile, steps of columns of the parts, sharer (the fastest).
__global__ __launch_bounds__(64 * kWaves) void k_lora_up(LoraArgs a, LoraPlan p, const float* __restrict__ ws) {
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    int64_t u = (int64_t)blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    if (u >= p.up_units) return;
    const int share = (int)(u % p.up_sharers);
    u /= p.up_sharers;
    const int64_t all = p.up_units / p.up_sharers / p.tiles;
    const int tile = (int)(u / all);
    int at = (int)(u % all), part = 0;
    for (; part < a.parts - 1; part++) {
        const int n = ((a.part[part].N + kLoraCols - 1) / kLoraCols + p.up_steps - 1) / p.up_steps;
        if (at < n) break;
        at -= n;
    }
    const LoraPart& w = a.part[part];
    const int n0 = at * p.up_steps * kLoraCols, n1 = min(w.N, n0 + p.up_steps * kLoraCols);
    const Tile o = tile_at(a, tile, lane);
    const int row = o.t0 + r;
    const float* const s0 = ws + (int64_t)part * p.pieces * a.T * a.rank + (int64_t)min(row, a.T - 1) * a.rank;
    int nth = 0;
    for (uint32_t left = o.firsts; left; left &= left - 1) {
        const int e = __builtin_amdgcn_readlane(o.id, __builtin_ctz(left));
        if (nth++ % p.up_sharers != share) continue;
        const bool mine = o.id == e;
        const int64_t ci = (int64_t)row * a.ldc + w.at, yi = (int64_t)row * a.ldy + w.at;
        const int ranks = e < 0 ? 0 : rank_of(a, e);
        if (ranks == 0) {                          // no adapter: a copy
            if (mine && a.Y != a.C)
                for (int n = n0 + 16 * g; n < n1; n += kLoraCols) {
                    const float none[16] = {};
                    add16(a, ci + n, yi + n, none, 0.f, n1 - n);
                }
            continue;
        }
        // s of the lane's row, eight ranks of every 32: hi + lo, times 2^shift
        float top = 0.f;
        for (int k = 8 * g; k < ranks; k += 32) {
            float s[8] = {};
            for (int i = 0; i < p.pieces; i++)
#pragma unroll
                for (int j = 0; j < 8; j++) s[j] += mine ? s0[(int64_t)i * a.T * a.rank + k + j] : 0.f;
#pragma unroll
            for (int j = 0; j < 8; j++) top = k + j < ranks ? __builtin_fmaxf(top, __builtin_fabsf(s[j])) : top;
        }
        top = __builtin_fmaxf(top, __shfl_xor(top, 16));
        top = __builtin_fmaxf(top, __shfl_xor(top, 32));
        // (s is a sum of products of fp16 numbers, a multiple of 2^-48: the shift is at most 63)
        const int shift = top > 0.f && top < __builtin_inff() ? 15 - __builtin_amdgcn_frexp_expf(top) : 0;
        const float up = __builtin_ldexpf(1.f, shift), f = __builtin_ldexpf(a.scales ? a.scales[e] : 1.f, -shift);
        const uint16_t* const B = w.B + (int64_t)e * w.N * a.rank;
        for (int n = n0; n < n1; n += kLoraCols) {
            f4 acc[4];
#pragma unroll
            for (int i = 0; i < 4; i++) acc[i] = f4{0.f, 0.f, 0.f, 0.f};
            for (int k0 = 0; k0 < ranks; k0 += 32) {
                const int k = k0 + 8 * g;
                h8 hi = zero8(), lo = zero8();
                float s[8] = {};
                if (mine && k < ranks)
                    for (int i = 0; i < p.pieces; i++)
#pragma unroll
                        for (int j = 0; j < 8; j++) s[j] += s0[(int64_t)i * a.T * a.rank + k + j];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float v = k + j < ranks ? s[j] * up : 0.f;
                    hi[j] = (_Float16)v;
                    lo[j] = (_Float16)(v - (float)hi[j]);
                }
                // column n + 16 (i / 4) + 4 j + i % 4 is row i of operand j: a lane's sums are of 16 neighbouring columns
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int col = min(n + 16 * (r >> 2) + 4 * j + (r & 3), w.N - 1);
                    h8 b = k < ranks ? *(const h8*)(B + (int64_t)col * a.rank + k) : zero8();
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        if (k + i >= ranks) b[i] = (_Float16)0.f;
                    acc[j] = mfma16x16x32(b, hi, acc[j]);
                    acc[j] = mfma16x16x32(b, lo, acc[j]);
                }
            }
            if (mine) {
                float d[16];
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int i = 0; i < 4; i++) d[4 * j + i] = acc[j][i];
                if (n + 16 * g < n1) add16(a, ci + n + 16 * g, yi + n + 16 * g, d, f, n1 - n - 16 * g);
            }
        }
    }
}

LoraPlan plan_of(const LoraArgs& a) { return plan_lora(a, device_cus() > 0 ? device_cus() : 256); }
int64_t groups_of(int64_t units) { return (units + kWaves - 1) / kWaves; }

}  // namespace

bool lora_fits(const LoraArgs& a) {
    const LoraPlan p = plan_of(a);
    return launch_fits(groups_of(p.down_units), 64 * kWaves) && launch_fits(groups_of(p.up_units), 64 * kWaves);
}

size_t lora_scratch_bytes(const LoraArgs& a) { return plan_of(a).bytes; }

hipError_t lora(const LoraArgs& a, float* ws, hipStream_t st) {
    const LoraPlan p = plan_of(a);
    hipLaunchKernelGGL(k_lora_down, dim3((unsigned)groups_of(p.down_units)), dim3(64 * kWaves), 0, st, a, p, ws);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(k_lora_up, dim3((unsigned)groups_of(p.up_units)), dim3(64 * kWaves), 0, st, a, p, ws);
    return hipGetLastError();
}

}  // namespace bf
