// The experts' feed-forward block of a mixture-of-experts layer:
//
//   c[t] = sum_j w[t][j] Wd_e . (SiLU(Wg_e . a_t) * (Wu_e . a_t)),   e = ids[t][j]
//
// over 4-bit weights in place.  A slot is one (t, j).  Three launches: h of
// every slot (gate and up of the same 16 rows in one workgroup, SiLU(g) u w
// rounded once to fp16), y = Wd h of every slot (fp32), and the sum of a row's
// slots in their order.  The row's weight goes into h before its rounding.
//
// Bound by the weights of the experts in use, each read once.
#include <algorithm>
#include <climits>

#include "bf_formats.h"
#include "bf_grid.h"
#include "bf_moe_launch.h"

namespace bf {
namespace {

constexpr int kMoeWaves = 4;
constexpr int kScanSlots = 1024;                   // up to so many slots a workgroup finds its expert's by itself

// Slots of one expert: in LDS (found by the workgroup), or in the plan's list.
struct Lists {
    const int32_t* perm;                           // slots, by expert, in order
    const int32_t* offs;                           // [E + 1]
};

template <int QT, int NM> struct MoeW {
    const uint8_t* W[NM];
    const uint8_t* aux[NM];
};

// Sums of a lane's two 32-value sub-blocks as the operand that meets the mins:
// {S / 32, S' / 32, 64 (S - hi), 64 (S' - hi')}, zero above.
__device__ __forceinline__ h8 block_sums(const h8 a[8]) {
    const h2 one = {(_Float16)1.0f, (_Float16)1.0f};
    h8 o;
#pragma unroll
    for (int e = 0; e < 8; e++) o[e] = (_Float16)0.f;
#pragma unroll
    for (int b = 0; b < 2; b++) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int e = 0; e < 8; e += 2) s = __builtin_amdgcn_fdot2(h2{a[4 * b + i][e], a[4 * b + i][e + 1]}, one, s, false);
        const _Float16 hi = (_Float16)(s * 0.03125f);
        o[b] = hi;
        o[2 + b] = (_Float16)((s - 32.f * (float)hi) * 64.f);
    }
    return o;
}

// One super-group: acc += a . w for NM matrices' 16 rows.  Q4_K weights enter as
// the integers sc q, exact, and d and dmin multiply the super-group's sums; the
// Q4_0 formats' as their fp16 dequant.
template <int QT, int NM, int MT>
__device__ __forceinline__ void multiply(const Magic& mg, const Raw<QT> raw[NM], const h8 a[MT][8], int kg, f4 acc[NM][MT]) {
    if constexpr (QT == QT_Q4_K) {
        h8 as[MT];
#pragma unroll
        for (int t = 0; t < MT; t++) as[t] = block_sums(a[t]);
#pragma unroll
        for (int m = 0; m < NM; m++) {
            const SclK sc = scales_int(raw[m], kg);
            f4 s[MT], z[MT];
#pragma unroll
            for (int t = 0; t < MT; t++) s[t] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const h8 w = weights_int(mg, raw[m], sc, i);
#pragma unroll
                for (int t = 0; t < MT; t++) s[t] = mfma16x16x32(a[t][i], w, s[t]);
            }
            const h8 mn = __builtin_bit_cast(h8, u4{sc.min_hi, sc.min_lo, 0u, 0u});
#pragma unroll
            for (int t = 0; t < MT; t++) {
                z[t] = mfma16x16x32(as[t], mn, f4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                for (int e = 0; e < 4; e++)
                    acc[m][t][e] = __builtin_fmaf(sc.d, s[t][e], __builtin_fmaf(-sc.dmin, z[t][e], acc[m][t][e]));
            }
        }
    } else {
#pragma unroll
        for (int m = 0; m < NM; m++) {
            const Scl<QT> sc = scales(raw[m], kg);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const h8 w = weights(mg, raw[m], sc, i);
#pragma unroll
                for (int t = 0; t < MT; t++) acc[m][t] = mfma16x16x32(a[t][i], w, acc[m][t]);
            }
        }
    }
}

// Up to 16 MT slots of one expert against 16 weight rows of NM matrices: the
// waves take super-groups in turn and meet in LDS.  GU: h of the slots; else y.
template <int QT, int MT, bool GU>
__device__ __forceinline__ void rows_of(const MoeArgs& a, const MoeW<QT, GU ? 2 : 1>& w, const uint16_t* A, int64_t lda,
                                        void* out, int R, int K, int64_t n0, int f0, const int32_t* list, int cnt,
                                        float* red) {
    constexpr int NM = GU ? 2 : 1, RS = 20;        // LDS row stride: the four row groups of a wave on distinct banks
    const int lane = threadIdx.x & 63, r = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nsg = K >> 8;
    const int64_t n = n0 + min(f0 + r, R - 1);
    const uint16_t* ap[MT];
#pragma unroll
    for (int t = 0; t < MT; t++) {
        const int i = 16 * t + r;
        ap[t] = i < cnt ? A + (int64_t)(GU ? list[i] / a.k : list[i]) * lda + 64 * kg : nullptr;
    }
    const Magic mg = make_magic();
    f4 acc[NM][MT];
#pragma unroll
    for (int m = 0; m < NM; m++)
#pragma unroll
        for (int t = 0; t < MT; t++) acc[m][t] = f4{0.f, 0.f, 0.f, 0.f};
    Raw<QT> raw[NM], nxt[NM];
    if (wave < nsg) {
#pragma unroll
        for (int m = 0; m < NM; m++) load_raw<QT>(raw[m], w.W[m], w.aux[m], n, wave, kg, K);
    }
    for (int s = wave; s < nsg; s += kMoeWaves) {
        h8 x[MT][8];
#pragma unroll
        for (int t = 0; t < MT; t++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[t][i] = h8{};
                if (ap[t]) x[t][i] = ld_act(ap[t] + 256 * s + 8 * i);
            }
        if (s + kMoeWaves < nsg) {
#pragma unroll
            for (int m = 0; m < NM; m++) load_raw<QT>(nxt[m], w.W[m], w.aux[m], n, s + kMoeWaves, kg, K);
        }
        multiply<QT, NM, MT>(mg, raw, x, kg, acc);
#pragma unroll
        for (int m = 0; m < NM; m++) raw[m] = nxt[m];
    }
    __syncthreads();                               // the last use of red and of the list is over
#pragma unroll
    for (int m = 0; m < NM; m++)
#pragma unroll
        for (int t = 0; t < MT; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) red[((wave * NM + m) * MT + t) * (16 * RS) + (4 * kg + e) * RS + r] = acc[m][t][e];
    __syncthreads();
    const int row = threadIdx.x >> 4, col = threadIdx.x & 15;
#pragma unroll
    for (int t = 0; t < MT; t++) {
        const int i = 16 * t + row;
        if (i >= cnt || f0 + col >= R) continue;
        float v[NM];
#pragma unroll
        for (int m = 0; m < NM; m++) {
            v[m] = 0.f;
#pragma unroll
            for (int q = 0; q < kMoeWaves; q++) v[m] += red[((q * NM + m) * MT + t) * (16 * RS) + row * RS + col];
        }
        const int slot = list[i];
        if constexpr (GU) {
            const float e = __builtin_amdgcn_exp2f(v[0] * -1.44269504088896341f);
            ((_Float16*)out)[(int64_t)slot * R + f0 + col] = (_Float16)(v[0] * __builtin_amdgcn_rcpf(1.0f + e) * v[NM - 1] * a.w[slot]);
        } else {
            ((float*)out)[(int64_t)slot * R + f0 + col] = v[0];
        }
    }
}

// grid x: tiles of 16 weight rows; y: experts, or slots where there are fewer
// of them (the first slot of an expert stands for it).
template <int QT, int MT, bool GU>
__global__ __launch_bounds__(64 * kMoeWaves) void k_moe_rows(MoeArgs a, MoeW<QT, GU ? 2 : 1> w, const uint16_t* A, int64_t lda,
                                                             void* out, int R, int K, int by_slot, Lists l) {
    constexpr int NM = GU ? 2 : 1;
    __shared__ float red[kMoeWaves * NM * MT * 16 * 20];
    __shared__ int32_t found[kScanSlots];
    __shared__ int wave_cnt[kMoeWaves];
    const int slots = a.T * a.k;
    const int e = by_slot ? a.ids[blockIdx.y] : (int)blockIdx.y;
    if (e < 0 || e >= a.E) return;
    const int f0 = 16 * blockIdx.x;
    const int32_t* list = found;
    int cnt = 0;
    if (l.perm) {
        list = l.perm + l.offs[e];
        cnt = l.offs[e + 1] - l.offs[e];
    } else {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        bool first = true;                         // no earlier slot has this expert
        for (int s0 = 0; s0 < slots; s0 += 64 * kMoeWaves) {
            const int s = s0 + (int)threadIdx.x;
            const bool hit = s < slots && a.ids[s] == e;
            const uint64_t b = __ballot(hit);
            if (s0) __syncthreads();
            if (lane == 0) wave_cnt[wave] = __builtin_popcountll(b);
            __syncthreads();
            int at = cnt;
#pragma unroll
            for (int q = 0; q < kMoeWaves; q++) {
                if (q < wave) at += wave_cnt[q];
                cnt += wave_cnt[q];
            }
            if (hit) found[at + __builtin_popcountll(b & ((1ull << lane) - 1))] = s;
        }
        __syncthreads();
        if (by_slot) first = found[0] == (int)blockIdx.y;
        if (!first) return;
    }
    const int64_t n0 = (int64_t)e * R;
    for (int c = 0; c < cnt; c += 16 * MT) {
        const int left = cnt - c;
        if (MT > 2 && left > 32) rows_of<QT, MT, GU>(a, w, A, lda, out, R, K, n0, f0, list + c, left < 16 * MT ? left : 16 * MT, red);
        else if (MT > 1 && left > 16) rows_of<QT, MT < 2 ? MT : 2, GU>(a, w, A, lda, out, R, K, n0, f0, list + c, left < 32 ? left : 32, red);
        else rows_of<QT, 1, GU>(a, w, A, lda, out, R, K, n0, f0, list + c, left < 16 ? left : 16, red);
    }
}

// Element k of weight row n, for widths off the super-group grid (Q4_0 formats).
template <int QT>
__device__ __forceinline__ float elem(const uint8_t* W, const uint8_t* aux, int64_t n, int k, int K) {
    if constexpr (QT == QT_PLANES) {
        const uint32_t b = W[n * (int64_t)(K >> 1) + (k >> 1)];
        return (float)((int)((k & 1) ? b >> 4 : b & 15) - 8) * half_bits_to_float(((const uint16_t*)aux)[n * (int64_t)(K >> 5) + (k >> 5)]);
    } else {
        const uint8_t* p = W + (n * (int64_t)(K >> 5) + (k >> 5)) * 18;
        const uint32_t b = p[2 + (k & 15)];
        return (float)((int)((k & 16) ? b >> 4 : b & 15) - 8) * half_bits_to_float(*(const uint16_t*)p);
    }
}

// The same two products, one thread an output: widths that are not whole
// super-groups, unaligned operands (Q4_0 formats).
template <int QT, bool GU>
__global__ __launch_bounds__(256) void k_moe_simple(MoeArgs a, MoeW<QT, GU ? 2 : 1> w, const uint16_t* A, int64_t lda,
                                                    void* out, int R, int K) {
    const int64_t slots = (int64_t)a.T * a.k;
    for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < slots * R; i += (int64_t)gridDim.x * 256) {
        const int64_t slot = i / R;
        const int f = (int)(i - slot * R), e = a.ids[slot];
        if (e < 0 || e >= a.E) continue;
        const uint16_t* x = A + (GU ? slot / a.k : slot) * lda;
        float v[2] = {0.f, 0.f};
        for (int k = 0; k < K; k++) {
            const float xv = half_bits_to_float(x[k]);
#pragma unroll
            for (int m = 0; m < (GU ? 2 : 1); m++) v[m] = __builtin_fmaf(xv, elem<QT>(w.W[m], w.aux[m], (int64_t)e * R + f, k, K), v[m]);
        }
        if constexpr (GU) {
            const float ex = __builtin_amdgcn_exp2f(v[0] * -1.44269504088896341f);
            ((_Float16*)out)[i] = (_Float16)(v[0] * __builtin_amdgcn_rcpf(1.0f + ex) * v[1] * a.w[slot]);
        } else {
            ((float*)out)[i] = v[0];
        }
    }
}

// Slots sorted by expert, in order within an expert, and the tiles they make:
// one workgroup an expert.  Each counts all experts' slots (in LDS; integer
// sums, so their order does not matter), then every wave writes its own run of
// slots.
constexpr int kPlanWaves = 16;
__global__ __launch_bounds__(64 * kPlanWaves) void k_moe_plan(const int32_t* __restrict__ ids, int slots, int E,
                                                              int32_t* __restrict__ perm, int32_t* __restrict__ offs,
                                                              int4* __restrict__ table, int* __restrict__ tiles) {
    extern __shared__ int hist[];
    __shared__ int same[kPlanWaves], sum[2][kPlanWaves];
    const int e = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < E; i += 64 * kPlanWaves) hist[i] = 0;
    __syncthreads();
    const int per = (slots + kPlanWaves - 1) / kPlanWaves, s0 = min(slots, wave * per), s1 = min(slots, s0 + per);
    int ns = 0;
    for (int s = s0 + lane; s < s1; s += 64) {
        const int id = ids[s];
        if (id >= 0 && id < E) atomicAdd(&hist[id], 1);
        ns += id == e;
    }
#pragma unroll
    for (int x = 32; x; x >>= 1) ns += __shfl_xor(ns, x);
    if (lane == 0) same[wave] = ns;
    __syncthreads();
    // slots and tiles of the experts before e
    int nl = 0, nt = 0;
    for (int i = threadIdx.x; i < e; i += 64 * kPlanWaves) {
        nl += hist[i];
        nt += (hist[i] + kMoeTileRows - 1) / kMoeTileRows;
    }
#pragma unroll
    for (int x = 32; x; x >>= 1) {
        nl += __shfl_xor(nl, x);
        nt += __shfl_xor(nt, x);
    }
    if (lane == 0) {
        sum[0][wave] = nl;
        sum[1][wave] = nt;
    }
    __syncthreads();
    int base = 0, tile = 0, at = 0;
#pragma unroll
    for (int q = 0; q < kPlanWaves; q++) {
        base += sum[0][q];
        tile += sum[1][q];
        if (q < wave) at += same[q];
    }
    const int total = hist[e], mine = (total + kMoeTileRows - 1) / kMoeTileRows;
    if (threadIdx.x == 0) {
        offs[e] = base;
        if (e == E - 1) {
            offs[E] = base + total;
            *tiles = tile + mine;
        }
    }
    for (int i = threadIdx.x; i < mine; i += 64 * kPlanWaves)
        table[tile + i] = int4{e, base + i * kMoeTileRows, min(kMoeTileRows, total - i * kMoeTileRows), 0};
    at += base;
    for (int s = s0; s < s1; s += 64) {
        const bool hit = s + lane < s1 && ids[s + lane] == e;
        const uint64_t b = __ballot(hit);
        if (hit) perm[at + __builtin_popcountll(b & ((1ull << lane) - 1))] = s + lane;
        at += __builtin_popcountll(b);
    }
}

// c[t] = the sum of its slots' y, in slot order; slots without an expert add nothing.
__global__ __launch_bounds__(256) void k_moe_sum(MoeArgs a, const float* __restrict__ y) {
    const int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x;
    if (i >= (int64_t)a.T * a.N) return;
    const int64_t t = i / a.N;
    const int n = (int)(i - t * a.N);
    float v = 0.f;
    for (int j = 0; j < a.k; j++) {
        const int e = a.ids[t * a.k + j];
        if (e >= 0 && e < a.E) v += y[(t * a.k + j) * a.N + n];
    }
    if (a.out_f16) ((_Float16*)a.C)[t * a.ldc + n] = (_Float16)v;
    else ((float*)a.C)[t * a.ldc + n] = v;
}

size_t up256(size_t b) { return (b + 255) & ~(size_t)255; }

// Workspace: h [slots][F] fp16, y [slots][N] fp32, the plan.
struct MoeWs {
    size_t y, perm, offs, table, tiles, end;
    int64_t max_tiles;
    explicit MoeWs(const MoeArgs& a) {
        const size_t slots = (size_t)a.T * a.k;
        y = up256(slots * a.F * 2);
        perm = y + up256(slots * a.N * 4);
        offs = perm + up256(slots * 4);
        table = offs + up256(((size_t)a.E + 1) * 4);
        max_tiles = (int64_t)std::min<size_t>(a.E, slots) + (int64_t)(slots / kMoeTileRows);
        tiles = table + up256((size_t)max_tiles * 16);
        end = tiles + 256;
    }
};

int64_t a_bytes(const MoeArgs& a) { return ((int64_t)(a.T - 1) * a.lda + a.K) * 2; }

// The tile kernel: rows addressed with 32 bits from the buffer's start, and a
// grid that fits a launch.
bool tiles_serve(const MoeArgs& a, const MoeWs& o) {
    const int64_t slots = (int64_t)a.T * a.k, nt = std::max<int64_t>(a.F / 64, (a.N + 127) / 128);
    return slots >= 16 * (int64_t)a.E && a_bytes(a) < (int64_t(1) << 32) && slots * a.F * 2 < (int64_t(1) << 32) &&
           launch_fits(o.max_tiles * nt, 512) && o.max_tiles * nt < INT32_MAX;
}

bool at16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <int QT, bool GU>
hipError_t launch_rows(const MoeArgs& a, const uint16_t* A, int64_t lda, void* out, const Lists& l, bool fast, hipStream_t st) {
    MoeW<QT, GU ? 2 : 1> w;
    w.W[0] = GU ? a.gate : a.down;
    w.aux[0] = GU ? a.gate_aux : a.down_aux;
    if constexpr (GU) {
        w.W[1] = a.up;
        w.aux[1] = a.up_aux;
    }
    const int R = GU ? a.F : a.N, K = GU ? a.K : a.F;
    const int64_t slots = (int64_t)a.T * a.k;
    if (!fast) {
        if constexpr (QT == QT_Q4_K) return hipErrorInvalidValue;   // the front end asks for aligned Q4_K operands
        else {
            const int64_t grid = std::min<int64_t>((slots * R + 255) / 256, 1 << 20);
            hipLaunchKernelGGL((k_moe_simple<QT, GU>), dim3((unsigned)grid), dim3(256), 0, st, a, w, A, lda, out, R, K);
            return hipGetLastError();
        }
    }
    const bool by_slot = !l.perm && slots < a.E;
    const dim3 grid((unsigned)((R + 15) / 16), (unsigned)(by_slot ? slots : a.E));
    auto k = a.T <= 16 ? k_moe_rows<QT, 1, GU> : a.T <= 32 ? k_moe_rows<QT, 2, GU> : k_moe_rows<QT, 4, GU>;
    hipLaunchKernelGGL(k, grid, dim3(64 * kMoeWaves), 0, st, a, w, A, lda, out, R, K, (int)by_slot, l);
    return hipGetLastError();
}

template <int QT>
hipError_t run(const MoeArgs& a, uint8_t* ws, hipStream_t st) {
    const MoeWs o(a);
    const int64_t slots = (int64_t)a.T * a.k;
    const bool fast = moe_fast(a);
    Lists l{nullptr, nullptr};
    if (fast && slots > kScanSlots) {
        l = Lists{(const int32_t*)(ws + o.perm), (const int32_t*)(ws + o.offs)};
        hipLaunchKernelGGL(k_moe_plan, dim3((unsigned)a.E), dim3(64 * kPlanWaves), a.E * 4, st, a.ids, (int)slots, a.E,
                           (int32_t*)(ws + o.perm), (int32_t*)(ws + o.offs), (int4*)(ws + o.table), (int*)(ws + o.tiles));
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    hipError_t e;
    if (l.perm && tiles_serve(a, o)) {
        MoeTileArgs t{};
        t.perm = l.perm;
        t.table = (const int4*)(ws + o.table);
        t.tiles = (const int*)(ws + o.tiles);
        t.W[0] = a.gate;
        t.W[1] = a.up;
        t.aux[0] = a.gate_aux;
        t.aux[1] = a.up_aux;
        t.A = a.A;
        t.lda = a.lda;
        t.a_bytes = (uint32_t)a_bytes(a);
        t.out = ws;
        t.R = a.F;
        t.K = a.K;
        t.nt = a.F / 64;
        e = moe_tile(a, t, true, o.max_tiles, st);
        if (e != hipSuccess) return e;
        t.W[0] = a.down;
        t.aux[0] = a.down_aux;
        t.A = (const uint16_t*)ws;
        t.lda = a.F;
        t.a_bytes = (uint32_t)(slots * a.F * 2);
        t.out = ws + o.y;
        t.R = a.N;
        t.K = a.F;
        t.nt = (a.N + 127) / 128;
        e = moe_tile(a, t, false, o.max_tiles, st);
    } else {
        e = launch_rows<QT, true>(a, a.A, a.lda, ws, l, fast, st);
        if (e != hipSuccess) return e;
        e = launch_rows<QT, false>(a, (const uint16_t*)ws, a.F, ws + o.y, l, fast, st);
    }
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(k_moe_sum, dim3((unsigned)(((int64_t)a.T * a.N + 255) / 256)), dim3(256), 0, st, a, (const float*)(ws + o.y));
    return hipGetLastError();
}

}  // namespace

bool moe_fast(const MoeArgs& a) {
    return at16(a.gate) && at16(a.up) && at16(a.down) && at16(a.A) && a.lda % 8 == 0 && a.K % 256 == 0 && a.F % 256 == 0 &&
           (((uintptr_t)a.gate_aux | (uintptr_t)a.up_aux | (uintptr_t)a.down_aux) & 3) == 0;
}

size_t moe_scratch_bytes(const MoeArgs& a) { return MoeWs(a).end; }

hipError_t moe_ffn(const MoeArgs& a, uint8_t* ws, hipStream_t st) {
    if (a.qtype == QT_PLANES) return run<QT_PLANES>(a, ws, st);
    if (a.qtype == QT_Q4_0) return run<QT_Q4_0>(a, ws, st);
    return run<QT_Q4_K>(a, ws, st);
}

}  // namespace bf
