// Low-rank adapters of many requests beside a shared projection:
//   Y[t] = C[t] + scale_e B_e (A_e x[t]),  e = ids[t]  (no adapter: Y[t] = C[t]),
// for up to four parts (a fused projection's slices), each with its A and B.
//
// Two launches: s = A x in fp32 (k_lora_down), then C + scale B s (k_lora_up).
// Rows are taken in tiles of 16 (few rows) or 64, operands of 16x16x32 MFMAs; a
// tile's rows may be of as many adapters, and each adapter of a tile is multiplied
// with the operands that hold rows of it, of which its own are kept.  So nothing
// is sorted and no row moves: single tokens of many requests are bound by the
// adapters' bytes whatever the products do, and in prompts neighbouring rows are
// of one adapter.
//
// Down: operands go from memory to registers; x and A are fp16, their products
// exact, sums fp32.  K is cut between a workgroup's waves, whose sums meet in LDS,
// and into pieces (partial sums in the workspace, added by the up products in
// their order), so that a few rows fill the chip.
// Up: s, times a power of two that brings the row's largest to 2^14..2^15, is
// taken as two fp16 numbers (rounded, and the rest rounded: 2^-22 of the largest), so
// the products lose nothing that fp32 would keep; sums fp32, one rounding of Y.
#include <atomic>

#include "bf_device.h"
#include "bf_grid.h"
#include "bf_launch.h"
#include "bf_lora_launch.h"

namespace bf {
namespace {

// Lane l holds the adapter of the tile's row l (-1: none; -2: past the last row).
__device__ __forceinline__ int adapter_of(const LoraArgs& a, int64_t t0, int rows, int lane) {
    if (lane >= rows || t0 + lane >= a.T) return -2;
    const int id = a.ids[t0 + lane];
    return id < 0 || id >= a.adapters ? -1 : id;
}

__device__ __forceinline__ int rank_of(const LoraArgs& a, int e) {
    return a.ranks ? min(max(a.ranks[e], 0), a.rank) : a.rank;
}

__device__ __forceinline__ h8 masked(h8 v, bool in) {
    const h8 zero = {};
    return in ? v : zero;
}

// Steps [s0, s1) of K: acc[sub][i] += ranks' operand i times rows' operand sub.
template <int SUBS, int NT, int U>
__device__ __forceinline__ void dot(f4 (&acc)[SUBS][4], const uint16_t* const (&x)[SUBS], const uint16_t* const (&w)[4], int s0,
                                    int s1, int K, int g) {
    for (int s = s0; s < s1; s += U) {
        h8 xv[U][SUBS], wv[U][NT];
#pragma unroll
        for (int j = 0; j < U; j++) {              // (past the last step: the last one again, not used)
            const int k = min(kLoraStep * min(s + j, s1 - 1) + 8 * g, K - 8);
#pragma unroll
            for (int i = 0; i < SUBS; i++) xv[j][i] = *(const h8*)(x[i] + k);
#pragma unroll
            for (int i = 0; i < NT; i++) wv[j][i] = *(const h8*)(w[i] + k);
        }
#pragma unroll
        for (int j = 0; j < U; j++) {
            if (s + j >= s1) break;
            if (kLoraStep * (s + j + 1) > K) {     // the last step of a K off 32
                const bool in = kLoraStep * (s + j) + 8 * g < K;
#pragma unroll
                for (int i = 0; i < SUBS; i++) xv[j][i] = masked(xv[j][i], in);
#pragma unroll
                for (int i = 0; i < NT; i++) wv[j][i] = masked(wv[j][i], in);
            }
#pragma unroll
            for (int i = 0; i < NT; i++)
#pragma unroll
                for (int b = 0; b < SUBS; b++) acc[b][i] = mfma16x16x32(wv[j][i], xv[j][b], acc[b][i]);
        }
    }
}

// Grid x: tile and sharer (the fastest), y: piece of K, z: part and ranks.
template <int SUBS, int NT, int WV>
__global__ __launch_bounds__(64 * WV) void k_lora_down(LoraArgs a, LoraPlan p, float* __restrict__ ws) {
    constexpr int ROWS = kLoraSub * SUBS, U = SUBS == 1 ? 4 : 2;
    __shared__ f4 meet[WV - 1][SUBS * NT][64];
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int tile = blockIdx.x / p.sharers, share = blockIdx.x - tile * p.sharers, piece = blockIdx.y;
    const int part = blockIdx.z / p.rank_parts, r0 = (blockIdx.z - part * p.rank_parts) * kLoraRanks;
    const int64_t t0 = (int64_t)tile * ROWS;
    const int id = adapter_of(a, t0, ROWS, lane);
    const int64_t steps = (a.K + kLoraStep - 1) / kLoraStep, shares = (int64_t)p.pieces * WV, mine = (int64_t)piece * WV + wave;
    const int s0 = (int)(steps * mine / shares), s1 = (int)(steps * (mine + 1) / shares);
    const uint16_t* x[SUBS];
#pragma unroll
    for (int b = 0; b < SUBS; b++) x[b] = a.X + min(t0 + 16 * b + r, (int64_t)a.T - 1) * a.ldx;
    float* const out = ws + ((int64_t)part * p.pieces + piece) * a.T * a.rank;
    int nth = 0;
    for (uint64_t left = __ballot(id >= 0); left;) {
        const int e = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
        const uint64_t rows = __ballot(id == e);
        left &= ~rows;
        if (p.sharers > 1 && nth++ != share) continue;
        const int ranks = rank_of(a, e);
        if (r0 >= ranks) continue;
        const uint16_t* const A = a.part[part].A + (int64_t)e * a.rank * a.K;
        const uint16_t* w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = A + (int64_t)min(r0 + 16 * i + r, ranks - 1) * a.K;   // (rows past the rank: not kept)
        const int tiles = min(NT, (ranks - r0 + 15) / 16);
        f4 acc[SUBS][4];
#pragma unroll
        for (int b = 0; b < SUBS; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) acc[b][i] = f4{0.f, 0.f, 0.f, 0.f};
        if (NT == 1 || tiles == 1) dot<SUBS, 1, U>(acc, x, w, s0, s1, a.K, g);
        else if (NT == 2 || tiles == 2) dot<SUBS, 2, U>(acc, x, w, s0, s1, a.K, g);
        else dot<SUBS, 4, U>(acc, x, w, s0, s1, a.K, g);
        // the waves' sums, added in their order: register set m of all by wave m % WV
        __syncthreads();                           // the last adapter's are read
        if (wave > 0)
#pragma unroll
            for (int b = 0; b < SUBS; b++)
#pragma unroll
                for (int i = 0; i < NT; i++)
                    if (i < tiles) meet[wave - 1][b * NT + i][lane] = acc[b][i];
        __syncthreads();
        if (wave > 0) continue;
        // lane: row 16 b + r of the tile, ranks r0 + 16 i + 4 g ..
#pragma unroll
        for (int b = 0; b < SUBS; b++) {
            if (!((rows >> (16 * b + r)) & 1)) continue;
#pragma unroll
            for (int i = 0; i < NT; i++) {
                const int at = r0 + 16 * i + 4 * g;
                if (i >= tiles || at >= a.rank) continue;                  // (rank % 8 == 0)
                f4 s = acc[b][i];
                for (int v = 0; v < WV - 1; v++) s += meet[v][b * NT + i][lane];
                *(f4*)(out + (t0 + 16 * b + r) * a.rank + at) = s;
            }
        }
    }
}

// Sixteen neighbouring columns of a row, n of them inside: Y = C + f d.
__device__ __forceinline__ void add16(const LoraArgs& a, int64_t ci, int64_t yi, const f4 (&d)[4], float f, int n) {
    if (a.wide && n >= 16) {
        if (a.out_f16) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const h8 c = *(const h8*)((const _Float16*)a.C + ci + 8 * i);
                f4 lo, hi;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    lo[e] = __builtin_fmaf(f, d[2 * i][e], (float)c[e]);
                    hi[e] = __builtin_fmaf(f, d[2 * i + 1][e], (float)c[4 + e]);
                }
                *(u4*)((_Float16*)a.Y + yi + 8 * i) = f32x8_to_f16(lo, hi);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                f4 c = *(const f4*)((const float*)a.C + ci + 4 * i);
#pragma unroll
                for (int e = 0; e < 4; e++) c[e] = __builtin_fmaf(f, d[i][e], c[e]);
                *(f4*)((float*)a.Y + yi + 4 * i) = c;
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 16; e++) {
            if (e >= n) break;
            const float v = f * d[e >> 2][e & 3];
            if (a.out_f16) ((_Float16*)a.Y)[yi + e] = (_Float16)((float)((const _Float16*)a.C)[ci + e] + v);
            else ((float*)a.Y)[yi + e] = ((const float*)a.C)[ci + e] + v;
        }
    }
}

__device__ __forceinline__ void copy16(const LoraArgs& a, int64_t ci, int64_t yi, int n) {
    if (a.wide && n >= 16) {
        const int size = a.out_f16 ? 2 : 4;
        for (int i = 0; i < size; i++) ((u4*)((char*)a.Y + yi * size))[i] = ((const u4*)((const char*)a.C + ci * size))[i];
    } else {
        for (int e = 0; e < min(n, 16); e++) {
            if (a.out_f16) ((uint16_t*)a.Y)[yi + e] = ((const uint16_t*)a.C)[ci + e];
            else ((uint32_t*)a.Y)[yi + e] = ((const uint32_t*)a.C)[ci + e];
        }
    }
}

// Grid: tile (the fastest), steps of columns of the parts.
template <int SUBS>
__global__ __launch_bounds__(64 * kLoraUpWaves) void k_lora_up(LoraArgs a, LoraPlan p, const float* __restrict__ ws) {
    constexpr int ROWS = kLoraSub * SUBS, NTH = 64 * kLoraUpWaves, PER = NTH / ROWS;   // threads a row of sums
    constexpr int HELD = 2;                        // fours of sums that a thread keeps
    extern __shared__ __attribute__((aligned(16))) _Float16 sums[];        // [hi, lo][ROWS][ld]
    __shared__ float factor[ROWS];
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int tile = blockIdx.x % p.tiles;
    int at = blockIdx.x / p.tiles, part = 0;
    for (; part < a.parts - 1; part++) {
        const int n = ((a.part[part].N + kLoraCols - 1) / kLoraCols + p.up_steps - 1) / p.up_steps;
        if (at < n) break;
        at -= n;
    }
    const LoraPart& w = a.part[part];
    const int n0 = at * p.up_steps * kLoraCols, n1 = min(w.N, n0 + p.up_steps * kLoraCols);
    const int64_t t0 = (int64_t)tile * ROWS;
    const int id = adapter_of(a, t0, ROWS, lane);
    const int ld = lora_lds_ranks(a.rank), ranks32 = ld - 8;

    // s of row tid / PER, fours of ranks in turn: the pieces' sums, as two fp16 numbers times 2^shift
    {
        const int row = tid / PER, e = row < 64 ? __shfl(id, row) : -2;
        const int ranks = e >= 0 ? rank_of(a, e) : 0;
        const float* const s0 = ws + ((int64_t)part * p.pieces * a.T + t0 + row) * a.rank;
        auto sum = [&](int k) {
            f4 s = f4{0.f, 0.f, 0.f, 0.f};
            if (k < ranks) {
                for (int i = 0; i < p.pieces; i++) s += *(const f4*)(s0 + (int64_t)i * a.T * a.rank + k);
#pragma unroll
                for (int j = 1; j < 4; j++)
                    if (k + j >= ranks) s[j] = 0.f;
            }
            return s;
        };
        f4 held[HELD];
        float top = 0.f;
        for (int i = 0, k = 4 * (tid % PER); k < ranks32; k += 4 * PER, i++) {
            const f4 s = sum(k);
            if (i == 0) held[0] = s;
            if (i == 1) held[1] = s;
#pragma unroll
            for (int j = 0; j < 4; j++) top = __builtin_fmaxf(top, __builtin_fabsf(s[j]));
        }
#pragma unroll
        for (int x = 1; x < PER; x <<= 1) top = __builtin_fmaxf(top, __shfl_xor(top, x));
        // (s is a sum of products of fp16 numbers, a multiple of 2^-48: the shift is at most 63)
        const int shift = top > 0.f && top < __builtin_inff() ? 15 - __builtin_amdgcn_frexp_expf(top) : 0;
        const float up = __builtin_ldexpf(1.f, shift);
        if (tid % PER == 0) factor[row] = ranks > 0 ? __builtin_ldexpf(a.scales ? a.scales[e] : 1.f, -shift) : 0.f;
        for (int i = 0, k = 4 * (tid % PER); k < ranks32; k += 4 * PER, i++) {
            const f4 s = i == 0 ? held[0] : i == 1 ? held[1] : sum(k);
            _Float16 hi[4], lo[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float v = s[j] * up;
                hi[j] = (_Float16)v;
                lo[j] = (_Float16)(v - (float)hi[j]);
            }
            _Float16* const to = sums + row * ld + k;
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
                *(h2*)(to + j) = h2{hi[j], hi[j + 1]};
                *(h2*)(to + ROWS * ld + j) = h2{lo[j], lo[j + 1]};
            }
        }
    }
    __syncthreads();

    int nth = 0;                                   // pairs of adapter and step
    for (uint64_t left = __ballot(id != -2); left;) {
        const int e = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
        const uint64_t rows = __ballot(id == e);
        left &= ~rows;
        const int ranks = e < 0 ? 0 : rank_of(a, e);
        const uint16_t* const B = ranks > 0 ? w.B + (int64_t)e * w.N * a.rank : nullptr;
        for (int n = n0; n < n1; n += kLoraCols, nth++) {
            if (nth % kLoraUpWaves != wave) continue;
            const int first = n + 16 * g, inside = n1 - first;             // the lane's columns
            f4 acc[SUBS][4];
#pragma unroll
            for (int b = 0; b < SUBS; b++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[b][j] = f4{0.f, 0.f, 0.f, 0.f};
            for (int k0 = 0; k0 < ranks; k0 += kLoraStep) {
                const int k = k0 + 8 * g;
                h8 bv[4];
                // column n + 16 (i / 4) + 4 j + i % 4 is row i of operand j: a lane's sums are of 16 neighbouring columns
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int col = min(n + 16 * (r >> 2) + 4 * j + (r & 3), w.N - 1);
                    bv[j] = *(const h8*)(B + (int64_t)col * a.rank + min(k, a.rank - 8));
                }
                if (k0 + kLoraStep > ranks) {      // what lies past the rank may be anything
#pragma unroll
                    for (int j = 0; j < 4; j++)
#pragma unroll
                        for (int i = 0; i < 8; i++) bv[j][i] = k + i < ranks ? bv[j][i] : (_Float16)0.f;
                }
#pragma unroll
                for (int b = 0; b < SUBS; b++) {
                    if (!((rows >> (16 * b)) & 0xFFFFu)) continue;
                    const _Float16* const s = sums + (16 * b + r) * ld + k;
                    const h8 hi = *(const h8*)s, lo = *(const h8*)(s + ROWS * ld);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        acc[b][j] = mfma16x16x32(bv[j], hi, acc[b][j]);
                        acc[b][j] = mfma16x16x32(bv[j], lo, acc[b][j]);
                    }
                }
            }
            if (inside <= 0) continue;
#pragma unroll
            for (int b = 0; b < SUBS; b++) {
                if (!((rows >> (16 * b + r)) & 1)) continue;
                const int64_t row = t0 + 16 * b + r, ci = row * a.ldc + w.at + first, yi = row * a.ldy + w.at + first;
                if (ranks > 0) add16(a, ci, yi, acc[b], factor[16 * b + r], inside);
                else if (a.Y != a.C) copy16(a, ci, yi, inside);
            }
        }
    }
}

template <int SUBS, int NT> void down(const LoraArgs& a, const LoraPlan& p, float* ws, hipStream_t st) {
    constexpr int WV = SUBS == 1 ? 8 : 4;
    const dim3 grid((unsigned)(p.tiles * (int64_t)p.sharers), (unsigned)p.pieces, (unsigned)(a.parts * p.rank_parts));
    hipLaunchKernelGGL((k_lora_down<SUBS, NT, WV>), grid, dim3(64 * WV), 0, st, a, p, ws);
}

template <int SUBS> hipError_t go(const LoraArgs& a, const LoraPlan& p, float* ws, hipStream_t st) {
    auto k = k_lora_up<SUBS>;
    const size_t lds = (size_t)4 * kLoraSub * SUBS * lora_lds_ranks(a.rank);
    static std::atomic<uint64_t> attr_set{0};      // one bit per device: LDS limit raised
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (!(attr_set.load(std::memory_order_acquire) & bit)) {
        e = hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize,
                                4 * kLoraSub * SUBS * lora_lds_ranks(SUBS == 1 ? kLoraMaxRank : 256));
        if (e != hipSuccess) return e;
        attr_set.fetch_or(bit, std::memory_order_acq_rel);
    }
    if (p.rank_tiles == 1) down<SUBS, 1>(a, p, ws, st);
    else if (p.rank_tiles == 2) down<SUBS, 2>(a, p, ws, st);
    else down<SUBS, 4>(a, p, ws, st);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(k, dim3((unsigned)p.up_groups), dim3(64 * kLoraUpWaves), lds, st, a, p, ws);
    return hipGetLastError();
}

LoraPlan plan_of(const LoraArgs& a) { return plan_lora(a, device_cus() > 0 ? device_cus() : 256); }

}  // namespace

bool lora_fits(const LoraArgs& a) {
    const LoraPlan p = plan_of(a);
    return launch_fits(p.tiles * (int64_t)p.sharers, 64 * p.down_waves) && launch_fits(p.up_groups, 64 * kLoraUpWaves);
}

size_t lora_scratch_bytes(const LoraArgs& a) { return plan_of(a).bytes; }

hipError_t lora(const LoraArgs& a, float* ws, hipStream_t st) {
    const LoraPlan p = plan_of(a);
    return p.subs == 1 ? go<1>(a, p, ws, st) : go<4>(a, p, ws, st);
}

}  // namespace bf
