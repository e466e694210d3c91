// The experts' feed-forward block of a mixture-of-experts layer:
//
//   c[t] = sum_j w[t][j] Wd_e . (SiLU(Wg_e . a_t) * (Wu_e . a_t)),   e = ids[t][j]
//
// over 4-bit weights in place.  A slot is one (t, j).  Three launches: h of
// every slot (gate and up of the same 16 rows in one workgroup, SiLU(g) u times
// the weight's first part rounded once to fp16), y = Wd h of every slot, and the
// fp32 sum of a row's slots in their order, times the second part (bf_moe_dev.h).
//
// Bound by the weights of the experts in use, each read once.  Up to 24
// slots an expert k_moe_rows takes the products (Q4_K, eight experts a row: one
// row of 2048 x 1024 14.2 us for 28 MB; 32 rows, 64 experts of 5120 x 1280, 161 us
// for 697 MB, 4.3 TB/s), above that k_moe_tile (2000 rows, 64 experts of 4096 x
// 1792, Q4_0: 942 to 966 us for 705 GFLOP).
#include <algorithm>
#include <atomic>
#include <climits>
#include <type_traits>

#include "bf_formats.h"
#include "bf_grid.h"
#include "bf_lds.h"
#include "bf_moe_dev.h"

namespace bf {
namespace {

constexpr int kMoeWaves = 8;
constexpr int kMoeStages = 2;                      // super-groups of a wave's weights in LDS
constexpr int kSumY = 32768;                       // rows of the sum along grid y
constexpr int kScanSlots = 1024;                   // up to so many slots a workgroup finds its expert's by itself

// Slots of one expert: in LDS (found by the workgroup), or in the plan's list.
struct Lists {
    const int32_t* perm;                           // slots, by expert, in order
    const int32_t* offs;                           // [E + 1]
};

struct MoeW {                                      // gate and up, or down
    const uint8_t *W[2], *aux[2];
};

// One super-group of 16 weight rows: acc += a . w.  Q4_K weights enter as the
// integers sc q and m, exact, and d and dmin multiply the super-group's sums: m
// is one number for all of a lane's 32 weights of a sub-block, so sum_k a_k m_k
// is a second product with that number as its operand (summing the activations
// per sub-block first takes 44 more vector instructions of 200, and the matrix
// unit has the time).  The Q4_0 formats' weights enter as their fp16 dequant, as in bf_gemm (one rounding
// of 2^-11 of a weight: their blocks' scales change within an instruction's k).
template <int QT, int MT>
__device__ __forceinline__ void multiply(const Magic& mg, const Raw<QT>& raw, const h8 a[MT][8], int kg, f4 acc[MT]) {
    if constexpr (QT == QT_Q4_K) {
        const SclK sc = scales_int(raw, kg);
        // {m, m'} of sub-blocks 2 kg, 2 kg + 1 (min_hi is 32 times them, exact)
        const h2 mm = as_h2(sc.min_hi) * h2{(_Float16)0.03125f, (_Float16)0.03125f};
        h8 mn[2];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            mn[0][e] = mm[0];
            mn[1][e] = mm[1];
        }
        f4 s[MT], z[MT];
#pragma unroll
        for (int t = 0; t < MT; t++) s[t] = z[t] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const h8 w = weights_int(mg, raw, sc, i);
#pragma unroll
            for (int t = 0; t < MT; t++) {
                s[t] = mfma16x16x32(a[t][i], w, s[t]);
                z[t] = mfma16x16x32(a[t][i], mn[i >> 2], z[t]);
            }
        }
#pragma unroll
        for (int t = 0; t < MT; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) acc[t][e] = __builtin_fmaf(sc.d, s[t][e], __builtin_fmaf(-sc.dmin, z[t][e], acc[t][e]));
    } else {
        const Scl<QT> sc = scales(raw, kg);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const h8 w = weights(mg, raw, sc, i);
#pragma unroll
            for (int t = 0; t < MT; t++) acc[t] = mfma16x16x32(a[t][i], w, acc[t]);
        }
    }
}

// What a launch of k_moe_rows computes: h (gate and up), y (down, by slot; or with
// all the activations of a pass in LDS), or the outputs of a single row (down over
// its slots' experts as one long sum).
enum : int { kMoeH = 0, kMoeY = 1, kMoeRow = 2, kMoeWhole = 3 };

// One super-group (144 bytes a row) of 16 weight rows into LDS, row after row:
// pieces of 16 bytes, nine to a row.  Neighbouring lanes fetch neighbouring
// pieces: as operand registers, where neighbouring lanes are different rows, the
// same bytes took 192 accesses to the L1 cache and the activations 128 more
// (86 % of its cycles; the whole block at 32 rows of 64 experts of 5120 x 1280,
// eight a row: 220 us so, 171 through LDS).
constexpr int kTileBytes = 16 * 144, kTileLoads = 3;
template <int QT> struct TileFetch {
    const uint8_t* src[kTileLoads];
    uint32_t step[kTileLoads];                     // bytes from one super-group to the next
    int64_t expert;                                // ... from one expert to the next (planes: of scales, eight times that of codes)
    __device__ __forceinline__ void init(const uint8_t* W, const uint8_t* aux, int64_t n0, int rows, int K, int lane) {
#pragma unroll
        for (int q = 0; q < kTileLoads; q++) {
            const int p = min(64 * q + lane, 143), row = p / 9, part = p - 9 * row;
            src[q] = w_piece<QT>(W, aux, n0 + min(row, rows - 1), 0, part, K);
            step[q] = QT != QT_PLANES ? 144 : part == 0 ? 16 : 128;
        }
    }
    __device__ __forceinline__ void get(int s, int e, uint32_t lds, int lane) const {
#pragma unroll
        for (int q = 0; q < kTileLoads; q++) {
            const int64_t at = expert * e * (QT == QT_PLANES && step[q] == 128 ? 8 : 1) + (uint64_t)step[q] * s;
            if (q < 2 || lane < 16) dma16(src[q] + at, lds + 1024 * q);
        }
    }
};

// The activations of a pass in LDS: slabs of CH super-groups of each row, two of
// them (one being multiplied, one on its way), rows 16 bytes apart in banks.
template <int CH> constexpr int kSlabRow = CH * 512 + 16;

// Waits until at most n + BASE of the wave's loads are on their way (n <= 8; else BASE).
template <int BASE>
__device__ __forceinline__ void wait_loads(int n) {
#define BF_WAIT(i) case i: asm volatile("s_waitcnt vmcnt(%0)" ::"n"(BASE + i) : "memory"); break;
    switch (n) {
        BF_WAIT(1) BF_WAIT(2) BF_WAIT(3) BF_WAIT(4) BF_WAIT(5) BF_WAIT(6) BF_WAIT(7) BF_WAIT(8)
        default: asm volatile("s_waitcnt vmcnt(%0)" ::"n"(BASE) : "memory");
    }
#undef BF_WAIT
}

// Up to 16 MT slots of one expert against the weight rows of a workgroup: eight
// waves, KS of them over the super-groups of one 16-row tile of one matrix (GU:
// gate, up), each through a ring of its own, the activations shared; the waves
// meet in LDS at the end.  GU: h of the slots; else y.
template <int QT, int MT, int MODE, int KS>
__device__ __forceinline__ void rows_of(const MoeArgs& a, const MoeW& w, const uint16_t* A, int64_t lda, void* out, int R,
                                        int K, int64_t e, int tile0, const int32_t* list, const float* rest, int cnt, int cap,
                                        uint8_t* lds) {
    constexpr bool GU = MODE == kMoeH, ONE = MODE == kMoeRow;
    constexpr int NM = GU ? 2 : 1, TW = kMoeWaves / (KS * NM), CH = KS < 2 ? 2 : KS, PER = CH / KS, ST = kMoeStages;
    constexpr int RS = 20, TS = 16 * RS;           // stride of the sums' rows: the four row groups of a wave on distinct banks
    const int lane = threadIdx.x & 63, r = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kp = wave % KS, mat = wave / KS % NM, tile = tile0 + wave / (KS * NM);
    // ONE: the row's slots one after the other, `list` their experts, `rest` what multiplies their products (K and
    // the activations run through them all)
    const int per = K >> 8, nsg = ONE ? a.k * per : per, slabs = (nsg + CH - 1) / CH, width = ONE ? a.k * K : K;
    float* const red = (float*)lds;                // [wave][MT][16][RS], over everything else at the end
    uint8_t* const ring = lds + wave * (ST * kTileBytes);
    const uint32_t ring0 = lds_addr(ring);
    uint8_t* const slab = lds + kMoeWaves * ST * kTileBytes;
    const int slab_bytes = cap * kSlabRow<CH>;
    const bool live = 16 * tile < R;
    TileFetch<QT> wf;
    wf.init(w.W[mat], w.aux[mat], e * R + (live ? 16 * tile : 0), live ? min(16, R - 16 * tile) : 1, K, lane);
    wf.expert = QT == QT_PLANES ? (int64_t)R * (K >> 4) : (int64_t)R * per * 144;
    auto weights_get = [&](int s, uint32_t to) {
        if constexpr (ONE) {
            const int j = s / per;
            wf.get(s - j * per, max(list[j], 0), to, lane);
        } else {
            wf.get(s, 0, to, lane);
        }
    };
    // slab t: rows wave, wave + 8, ...; CH / 2 loads of 1 KB a row (past the row's end: its start, not used)
    auto slab_get = [&](int t) {
        const uint32_t to = lds_addr(slab) + (t & 1) * slab_bytes;
        for (int i = wave; i < cnt; i += kMoeWaves) {
            const int slot = ONE ? 0 : list[i];
            const uint16_t* row = A + (int64_t)(GU ? slot / a.k : slot) * lda;
#pragma unroll
            for (int q = 0; q < CH / 2; q++) {
                const int c = 256 * CH * t + 512 * q + 8 * lane;
                dma16(row + (c < width ? c : 0), to + i * kSlabRow<CH> + 1024 * q);
            }
        }
    };
    // the wave's n-th super-group
    auto sg_at = [&](int n) { return n / PER * CH + kp + n % PER * KS; };
    const Magic mg = make_magic();
    f4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; t++) acc[t] = f4{0.f, 0.f, 0.f, 0.f};
    __syncthreads();                               // LDS is free
    slab_get(0);
    for (int n = 0; n < ST - 1; n++)
        if (sg_at(n) < nsg) weights_get(sg_at(n), ring0 + n * kTileBytes);
    int at = 0;                                    // ring stage of the wave's next super-group
    for (int t = 0; t < slabs; t++) {
        // slab t is there, for every wave: the loads issued after it are at most the ring's
        if (t == 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        barrier_lds();
        int newer = 0;                             // loads of the next slab
        if (t + 1 < slabs) {
            slab_get(t + 1);
            newer = cnt > wave ? (cnt - wave + kMoeWaves - 1) / kMoeWaves * (CH / 2) : 0;
        }
        bool more = true;
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int n = t * PER + j, s = sg_at(n), next = sg_at(n + ST - 1);
            if (s >= nsg) break;
            more = next < nsg;
            if (more) {
                const int to = at + ST - 1 < ST ? at + ST - 1 : at - 1;
                weights_get(next, ring0 + to * kTileBytes);
                // (the wave's first ST - 1 super-groups of a slab were fetched before the next slab's activations)
                wait_loads<(ST - 1) * kTileLoads>(j < ST - 1 ? newer : 0);
            } else {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            }
            Raw<QT> raw;
            lds_raw<QT>(raw, ring + at * kTileBytes + r * 144, kg);
            h8 x[MT][8];
#pragma unroll
            for (int m = 0; m < MT; m++) {
                const uint8_t* row = slab + (t & 1) * slab_bytes + min(16 * m + r, cnt - 1) * kSlabRow<CH> + (s - CH * t) * 512 + 128 * kg;
#pragma unroll
                for (int i = 0; i < 8; i++) x[m][i] = *(const h8*)(row + 16 * i);
            }
            if constexpr (ONE) {
                if (list[s / per] >= 0) {              // (a slot without an expert: h is not there)
                    f4 y[MT] = {f4{0.f, 0.f, 0.f, 0.f}};
                    multiply<QT, MT>(mg, raw, x, kg, y);
                    acc[0] += rest[s / per] * y[0];
                }
            } else {
                multiply<QT, MT>(mg, raw, x, kg, acc);
            }
            at = at + 1 < ST ? at + 1 : 0;
        }
        // the next slab's loads are older than the ring's last one
        if (t + 1 < slabs) {
            if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kTileLoads) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
    }
    __syncthreads();                               // everybody is done with ring and slabs
#pragma unroll
    for (int t = 0; t < MT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) red[(wave * MT + t) * TS + (4 * kg + i) * RS + r] = acc[t][i];
    __syncthreads();
    for (int u = threadIdx.x; u < TW * MT * 256; u += 64 * kMoeWaves) {
        const int tl = u / (MT * 256), t = u / 256 % MT, row = u / 16 % 16, col = u % 16;
        const int i = 16 * t + row, f = 16 * (tile0 + tl) + col;
        if (i >= cnt || f >= R) continue;
        float v[NM];
#pragma unroll
        for (int m = 0; m < NM; m++) {
            v[m] = 0.f;
#pragma unroll
            for (int q = 0; q < KS; q++) v[m] += red[(((tl * NM + m) * KS + q) * MT + t) * TS + row * RS + col];
        }
        if constexpr (ONE) {
            if (a.out_f16) ((_Float16*)a.C)[f] = (_Float16)v[0];
            else ((float*)a.C)[f] = v[0];
            continue;
        }
        const int slot = list[i];
        if constexpr (GU) {
            const float ex = __builtin_amdgcn_exp2f(v[0] * -1.44269504088896341f);
            ((_Float16*)out)[(int64_t)slot * R + f] = (_Float16)(v[0] * __builtin_amdgcn_rcpf(1.0f + ex) * v[NM - 1] * weight_in_h(a.w[slot]));
        } else {
            store_y(a, out, (int64_t)slot * R + f, v[0]);
        }
    }
}

// y of up to 16 slots of one expert against `many` tiles of 16 weight rows a
// wave, where all of the slots' activations fit in LDS: one barrier, then every
// wave streams its own tiles (32 rows, 64 experts, eight a row: 5120 x 1280 166.7
// us with rows_of, 160.9 so; 2048 x 1024 64.7 and 61.2; 100 rows, 128 experts of
// 4096 x 256, four a row: 74.2 and 60.1).
template <int QT>
__device__ __forceinline__ void rows_whole(const MoeArgs& a, const MoeW& w, const uint16_t* A, int64_t lda, void* out, int R,
                                           int K, int64_t e, int tile0, int many, const int32_t* list, int cnt, uint8_t* lds) {
    constexpr int ST = kMoeStages;
    const int lane = threadIdx.x & 63, r = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int per = K >> 8, tiles = R >> 4, first = tile0 + wave, mine = first < tiles ? min(many, (tiles - first + kMoeWaves - 1) / kMoeWaves) : 0;
    uint8_t* const ring = lds + wave * (ST * kTileBytes);
    const uint32_t ring0 = lds_addr(ring);
    uint8_t* const x0 = lds + kMoeWaves * ST * kTileBytes;
    const int stride = 2 * K + 16;
    TileFetch<QT> wf;
    wf.init(w.W[0], w.aux[0], e * R + (mine ? 16 * first : 0), 16, K, lane);
    wf.expert = 16 * kMoeWaves * (QT == QT_PLANES ? (int64_t)(K >> 4) : (int64_t)per * 144);   // (from one tile of the wave to the next)
    __syncthreads();                               // LDS is free
    int fs = 0, ft = 0;                            // the next super-group to fetch
    auto fetch = [&](int n) {
        wf.get(fs, ft, ring0 + (n % ST) * kTileBytes, lane);
        if (++fs == per) fs = 0, ft++;
    };
    const int total = mine * per;
    for (int i = wave; i < cnt; i += kMoeWaves) {
        const uint16_t* row = A + (int64_t)list[i] * lda;
        for (int c = 0; c < K; c += 512)
            if (c + 8 * lane < K) dma16(row + c + 8 * lane, lds_addr(x0) + i * stride + 2 * c);
    }
    if (total) fetch(0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    barrier_lds();
    const Magic mg = make_magic();
    const uint8_t* const row = x0 + min(r, cnt - 1) * stride + 128 * kg;
    int n = 0;
    for (int t = 0; t < mine; t++) {
        f4 acc[1] = {f4{0.f, 0.f, 0.f, 0.f}};
        for (int s = 0; s < per; s++, n++) {
            if (n + 1 < total) {
                fetch(n + 1);
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kTileLoads) : "memory");
            } else {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            }
            Raw<QT> raw;
            lds_raw<QT>(raw, ring + (n % ST) * kTileBytes + r * 144, kg);
            h8 x[1][8];
#pragma unroll
            for (int i = 0; i < 8; i++) x[0][i] = *(const h8*)(row + 512 * s + 16 * i);
            multiply<QT, 1>(mg, raw, x, kg, acc);
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (4 * kg + i < cnt) store_y(a, out, (int64_t)list[4 * kg + i] * R + 16 * (first + kMoeWaves * t) + r, acc[0][i]);
    }
}

// grid x: workgroups' weight rows; y: experts, or slots where there are fewer
// of them (the first slot of an expert stands for it).
template <int QT, int MT, int MODE, int KS>
__global__ __launch_bounds__(64 * kMoeWaves, MT == 1 ? 4 : 2)
void k_moe_rows(MoeArgs a, MoeW w, const uint16_t* A, int64_t lda, void* out, int R, int K, int by_slot, int cap, int many, Lists l) {
    constexpr int TW = kMoeWaves / (KS * (MODE == kMoeH ? 2 : 1));
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    __shared__ int32_t own[MODE == kMoeWhole ? 1 : kScanSlots];
    int32_t* const found = MODE == kMoeWhole ? (int32_t*)(lds + kMoeWaves * kMoeStages * kTileBytes + cap * (2 * K + 16)) : own;
    __shared__ int wave_cnt[kMoeWaves];
    const int slots = a.T * a.k;
    if constexpr (MODE == kMoeRow) {
        __shared__ float rest[kScanSlots];
        for (int j = threadIdx.x; j < a.k; j += 64 * kMoeWaves) {
            found[j] = a.ids[j] < a.E ? a.ids[j] : -1;
            rest[j] = weight_of_y(a.w[j]);
        }
        __syncthreads();
        rows_of<QT, 1, MODE, KS>(a, w, A, lda, out, R, K, 0, TW * (int)blockIdx.x, found, rest, 1, 1, lds);
        return;
    }
    const int e = by_slot ? a.ids[blockIdx.y] : (int)blockIdx.y;
    if (e < 0 || e >= a.E) return;
    const int32_t* list = found;
    int cnt = 0;
    if (l.perm) {
        list = l.perm + l.offs[e];
        cnt = l.offs[e + 1] - l.offs[e];
    } else {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
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
        if (by_slot && found[0] != (int)blockIdx.y) return;
    }
    const int tile0 = TW * (int)blockIdx.x;
    for (int c = 0; c < cnt; c += cap) {           // (cap <= 16 MT rows a pass)
        const int n = min(cnt - c, cap);
        if constexpr (MODE == kMoeWhole) {
            rows_whole<QT>(a, w, A, lda, out, R, K, e, TW * many * (int)blockIdx.x, many, list + c, n, lds);
            continue;
        }
        if (MT > 1 && n > 16) rows_of<QT, MT, MODE, KS>(a, w, A, lda, out, R, K, e, tile0, list + c, nullptr, n, cap, lds);
        else rows_of<QT, 1, MODE, KS>(a, w, A, lda, out, R, K, e, tile0, list + c, nullptr, n, cap, lds);
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
__global__ __launch_bounds__(256) void k_moe_simple(MoeArgs a, MoeW w, const uint16_t* A, int64_t lda,
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
            ((_Float16*)out)[i] = (_Float16)(v[0] * __builtin_amdgcn_rcpf(1.0f + ex) * v[1] * weight_in_h(a.w[slot]));
        } else {
            store_y(a, out, i, v[0]);
        }
    }
}

// Slots sorted by expert, in order within an expert, and the tiles they make:
// one workgroup an expert.  Each counts all experts' slots (in LDS; integer
// sums, so their order does not matter), then every wave writes its own run of
// slots.
constexpr int kPlanWaves = 16;
// Of n slots: runs of `run`.  Runs of 256 are large tiles, and so is a rest from
// `least` rows on (more than 256: no large tiles at all); all others small tiles.
__device__ __forceinline__ int large_tiles(int n, int least) {
    return least > kMoeTileRows ? 0 : n / kMoeTileRows + (n % kMoeTileRows >= least);
}
__device__ __forceinline__ int small_tiles(int n, int least, int run) { return (n + run - 1) / run - large_tiles(n, least); }
__global__ __launch_bounds__(64 * kPlanWaves) void k_moe_plan(const int32_t* __restrict__ ids, int slots, int E,
                                                              int32_t* __restrict__ perm, int32_t* __restrict__ offs,
                                                              int4* __restrict__ table, int* __restrict__ tiles, int max_tiles,
                                                              int least, int run) {
    extern __shared__ int hist[];
    __shared__ int same[kPlanWaves], sum[3][kPlanWaves];
    const int e = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < E; i += 64 * kPlanWaves) hist[i] = 0;
    __syncthreads();
    const int per = (slots + kPlanWaves - 1) / kPlanWaves, s0 = min(slots, wave * per), s1 = min(slots, s0 + per);
    int ns = 0;
    // (eight loads at a time: one by one the two passes over 16000 slots take 14 us)
    auto load8 = [&](int s, int id[8]) {
#pragma unroll
        for (int q = 0; q < 8; q++) id[q] = s + 64 * q + lane < s1 ? ids[s + 64 * q + lane] : -1;
    };
    for (int s = s0; s < s1; s += 512) {
        int id[8];
        load8(s, id);
#pragma unroll
        for (int q = 0; q < 8; q++) {
            if (id[q] >= 0 && id[q] < E) atomicAdd(&hist[id[q]], 1);
            ns += id[q] == e;
        }
    }
#pragma unroll
    for (int x = 32; x; x >>= 1) ns += __shfl_xor(ns, x);
    if (lane == 0) same[wave] = ns;
    __syncthreads();
    // slots and tiles (large, small) of the experts before e
    int n[3] = {0, 0, 0};
    for (int i = threadIdx.x; i < e; i += 64 * kPlanWaves) {
        n[0] += hist[i];
        n[1] += large_tiles(hist[i], least);
        n[2] += small_tiles(hist[i], least, run);
    }
#pragma unroll
    for (int c = 0; c < 3; c++) {
#pragma unroll
        for (int x = 32; x; x >>= 1) n[c] += __shfl_xor(n[c], x);
        if (lane == 0) sum[c][wave] = n[c];
    }
    __syncthreads();
    int before[3] = {0, 0, 0}, at = 0;
#pragma unroll
    for (int q = 0; q < kPlanWaves; q++) {
#pragma unroll
        for (int c = 0; c < 3; c++) before[c] += sum[c][q];
        if (q < wave) at += same[q];
    }
    const int base = before[0], total = hist[e], large = large_tiles(total, least), small = small_tiles(total, least, run);
    if (threadIdx.x == 0) {
        offs[e] = base;
        if (e == E - 1) {
            offs[E] = base + total;
            tiles[0] = before[1] + large;
            tiles[1] = before[2] + small;
        }
    }
    for (int i = threadIdx.x; i < large + small; i += 64 * kPlanWaves)
        table[i < large ? before[1] + i : max_tiles + before[2] + i - large] =
            int4{e, base + i * run, min(run, total - i * run), 0};
    at += base;
    for (int s = s0; s < s1; s += 512) {
        int id[8];
        load8(s, id);
#pragma unroll
        for (int q = 0; q < 8; q++) {
            const uint64_t b = __ballot(id[q] == e);
            if (id[q] == e) perm[at + __builtin_popcountll(b & ((1ull << lane) - 1))] = s + 64 * q + lane;
            at += __builtin_popcountll(b);
        }
    }
}

// c[t] = the sum of its slots' y, in slot order; slots without an expert add
// nothing.  Four outputs a thread, a row's slots read together.
template <bool Y24>
__global__ __launch_bounds__(256) void k_moe_sum(MoeArgs a, const void* __restrict__ y) {
    const int64_t t = (int64_t)blockIdx.z * kSumY + blockIdx.y;
    const int n = 4 * ((int)blockIdx.x * 256 + (int)threadIdx.x);
    if (t >= a.T || n >= a.N) return;
    const int32_t* ids = a.ids + t * a.k;
    const int64_t row = t * a.k * a.N + n;
    const bool whole = a.N % 4 == 0;
    f4 v = f4{0.f, 0.f, 0.f, 0.f};
    for (int j0 = 0; j0 < a.k; j0 += 8) {
        f4 x[8];
        float wt[8];
#pragma unroll
        for (int j = 0; j < 8; j++) wt[j] = a.w[t * a.k + min(j0 + j, a.k - 1)];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            x[j] = f4{0.f, 0.f, 0.f, 0.f};
            if (j0 + j >= a.k || ids[j0 + j] < 0 || ids[j0 + j] >= a.E) wt[j] = 0.f;
            else x[j] = load_y4<Y24>(a, y, row + (int64_t)(j0 + j) * a.N, whole, a.N - n);
        }
#pragma unroll
        for (int j = 0; j < 8; j++) v += weight_of_y(wt[j]) * x[j];
    }
    const int64_t at = t * a.ldc + n;
    if (a.out_f16 && whole && a.ldc % 4 == 0 && ((uintptr_t)a.C & 7) == 0) {
        typedef _Float16 h4 __attribute__((ext_vector_type(4)));
        *(h4*)((_Float16*)a.C + at) = h4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
        return;
    }
    for (int i = 0; i < 4 && n + i < a.N; i++) {
        if (a.out_f16) ((_Float16*)a.C)[at + i] = (_Float16)v[i];
        else ((float*)a.C)[at + i] = v[i];
    }
}

size_t up256(size_t b) { return (b + 255) & ~(size_t)255; }

// Slots of a run: 64, in a kernel of two workgroups a CU, up to 48 slots an expert
// on average, else 256 (64 and 256 in us, 64 experts, eight a row, of 4096 x 1792:
// 230 rows 360 and 393, 400 rows 416 and 422, 500 rows 516 and 469; of 2048 x 1024:
// 230 rows 116 and 136, 400 rows 127 and 148, 600 rows 191 and 195).
int run_rows(const MoeArgs& a) { return (int64_t)a.T * a.k < 48 * (int64_t)a.E ? 64 : kMoeTileRows; }

// Workspace: h [slots][F] fp16, y [slots][N] in 32 or 24 bits, the plan.
struct MoeWs {
    size_t y, perm, offs, table, tiles, end;
    int64_t max_tiles;
    explicit MoeWs(const MoeArgs& a) {
        const size_t slots = (size_t)a.T * a.k;
        y = up256(slots * a.F * 2);
        perm = y + (y_24(a) ? (size_t)y_24_high(a) + up256(slots * a.N) : up256(slots * a.N * 4));
        offs = perm + up256(slots * 4);
        table = offs + up256(((size_t)a.E + 1) * 4);
        max_tiles = (int64_t)std::min<size_t>(a.E, slots) + (int64_t)(slots / run_rows(a));
        tiles = table + up256((size_t)max_tiles * 32);
        end = tiles + 256;
    }
};

int64_t a_bytes(const MoeArgs& a) { return ((int64_t)(a.T - 1) * a.lda + a.K) * 2; }

// Rows from which a run of slots takes a large tile: 193 where whole runs alone
// make large tiles for 3/8 of the CUs, else none does (large and small only, us:
// 2000 rows of eight, 64 experts of 4096 x 1792, 868 tiles 934 and 1067; 500 rows of
// four, 8 experts, 98 tiles 181 and 203; 1000 rows of four, 16 experts of 2048 x
// 512, 60 tiles 102 and 83; 500 rows of two, 4 experts of 4096 x 1792, 42 tiles 163
// and 102).
int large_least(const MoeArgs& a) {
    const int64_t slots = (int64_t)a.T * a.k, cus = device_cus() > 0 ? device_cus() : 256;
    return run_rows(a) == kMoeTileRows && 8 * (slots / kMoeTileRows) * (std::min(2 * a.F, a.N) / 256) >= 3 * cus ? 193 : kMoeTileRows + 1;
}

// The tile kernels: from 24 slots an expert on average (rows and tiles in us, 64
// experts, eight a row, of 2048 x 1024: 160 rows 118 and 116, 200 rows 137 and 116; of
// 4096 x 1792: 200 rows 329 and 357, 225 rows 374 and 360), rows addressed with 32
// bits from the buffer's start, and a grid that fits a launch.
bool tiles_serve(const MoeArgs& a, const MoeWs& o) {
    const int64_t slots = (int64_t)a.T * a.k, nt = std::max<int64_t>(a.F / 64, (a.N + 127) / 128);
    return slots >= kMoeTileSlots * (int64_t)a.E && a_bytes(a) < (int64_t(1) << 32) && slots * a.F * 2 < (int64_t(1) << 32) &&
           launch_fits(o.max_tiles * nt, 512) && o.max_tiles * nt < INT32_MAX;
}

bool at16(const void* p) { return ((uintptr_t)p & 15) == 0; }

constexpr int kWholeMost = 81920 - 512;            // two workgroups a CU
// LDS of k_moe_rows in its kMoeWhole form: the waves' rings, the activations, the list of slots
int64_t whole_bytes(const MoeArgs& a, int K) {
    const int64_t slots = (int64_t)a.T * a.k;
    return kMoeWaves * kMoeStages * kTileBytes + std::min<int64_t>(16, slots) * (2 * (int64_t)K + 16) +
           4 * std::min<int64_t>(slots, kScanSlots);
}

template <int QT, int MODE, int MT, int KS>
hipError_t launch_split(int64_t experts, hipStream_t st, const MoeArgs& a, const MoeW& w, const uint16_t* A, int64_t lda, void* out,
                        int R, int K, int by_slot, const Lists& l) {
    constexpr int TW = kMoeWaves / (KS * (MODE == kMoeH ? 2 : 1)), CH = KS < 2 ? 2 : KS;
    constexpr int ring = kMoeWaves * kMoeStages * kTileBytes, meet = kMoeWaves * MT * 16 * 20 * 4;
    constexpr int rows = MODE == kMoeRow ? 1 : 16 * MT, most = std::max(ring + 2 * rows * kSlabRow<CH>, meet);
    const int cap = (int)std::min<int64_t>(rows, (int64_t)a.T * a.k);
    const int lds = std::max(ring + 2 * cap * kSlabRow<CH>, meet);
    const int tiles = (R + 15) / 16;
    auto k = k_moe_rows<QT, MT, MODE, KS>;
    static std::atomic<uint64_t> attr_set{0};      // one bit per device: LDS limit raised
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (!(attr_set.load(std::memory_order_acquire) & bit)) {
        e = hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, most);
        if (e != hipSuccess) return e;
        attr_set.fetch_or(bit, std::memory_order_acq_rel);
    }
    hipLaunchKernelGGL(k, dim3((unsigned)((tiles + TW - 1) / TW), (unsigned)experts), dim3(64 * kMoeWaves), lds, st, a, w, A, lda,
                       out, R, K, by_slot, cap, 1, l);
    return hipGetLastError();
}

template <int QT>
hipError_t launch_whole(int64_t experts, int many, hipStream_t st, const MoeArgs& a, const MoeW& w, const uint16_t* A, int64_t lda,
                        void* out, int R, int K, int by_slot, const Lists& l) {
    const int cap = (int)std::min<int64_t>(16, (int64_t)a.T * a.k);
    const int lds = (int)whole_bytes(a, K);
    auto k = k_moe_rows<QT, 1, kMoeWhole, 1>;
    static std::atomic<uint64_t> attr_set{0};      // one bit per device: LDS limit raised
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (!(attr_set.load(std::memory_order_acquire) & bit)) {
        e = hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, kWholeMost);
        if (e != hipSuccess) return e;
        attr_set.fetch_or(bit, std::memory_order_acq_rel);
    }
    const int per = kMoeWaves * many, tiles = R / 16;
    hipLaunchKernelGGL(k, dim3((unsigned)((tiles + per - 1) / per), (unsigned)experts), dim3(64 * kMoeWaves), lds, st, a, w, A, lda,
                       out, R, K, by_slot, cap, many, l);
    return hipGetLastError();
}

template <int QT, bool GU>
hipError_t launch_rows(const MoeArgs& a, const uint16_t* A, int64_t lda, void* out, const Lists& l, bool fast, hipStream_t st) {
    const MoeW w = GU ? MoeW{{a.gate, a.up}, {a.gate_aux, a.up_aux}} : MoeW{{a.down, nullptr}, {a.down_aux, nullptr}};
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
    const int64_t experts = by_slot ? slots : a.E;
    const int64_t waves = (int64_t)((R + 15) / 16) * (GU ? 2 : 1) * std::min<int64_t>(experts, slots);
    // One wave a tile, but where that leaves the chip empty (K = 2048, F = 1024,
    // gate and up / down in 4, 2, 1 parts: one row, 8 experts, 1024 waves 16.7,
    // 18.1, 22.4 us; eight rows, 32 slots, 4096 waves 52.8, 33.7, 29.8).
    const int ks = waves < 1536 ? 4 : waves < 3072 ? 2 : 1;
    if constexpr (!GU) {
        // As many tiles a wave as leave one round of two workgroups a CU (32 rows, 64
        // experts of 5120 x 1280: 5 tiles, 512 workgroups 160.9 us; 4 and 8 tiles 168.6
        // and 177.0; 2048 x 1024: 2 tiles 61.2, 1 and 3 tiles 63.8 and 65.7).
        const int64_t groups = (R / 16 + kMoeWaves - 1) / kMoeWaves, cus = device_cus() > 0 ? device_cus() : 256;
        const int many = (int)std::clamp<int64_t>((groups * std::min<int64_t>(experts, slots) + 2 * cus - 1) / (2 * cus), 1, 8);
        if (ks == 1 && slots <= 16 * (int64_t)a.E && R % 16 == 0 && whole_bytes(a, K) <= kWholeMost)
            return launch_whole<QT>(experts, many, st, a, w, A, lda, out, R, K, (int)by_slot, l);
    }
    const auto go = [&](auto mt) {
        constexpr int MT = decltype(mt)::value;
        constexpr int MODE = GU ? kMoeH : kMoeY;
        return ks == 1 ? launch_split<QT, MODE, MT, 1>(experts, st, a, w, A, lda, out, R, K, (int)by_slot, l)
               : ks == 2 || MT == 2 ? launch_split<QT, MODE, MT, 2>(experts, st, a, w, A, lda, out, R, K, (int)by_slot, l)
                                    : launch_split<QT, MODE, 1, 4>(experts, st, a, w, A, lda, out, R, K, (int)by_slot, l);
    };
    // Two row tiles a pass where most experts have more than one (one and two in us, 64
    // experts of 2048 x 1024, eight a row: 100 rows 89.5 and 93.1, 130 rows 107.8 and
    // 103.8; 8 experts of 4096 x 1792, two a row: 40 rows 35.3 and 43.9).
    return slots <= 16 * (int64_t)a.E ? go(std::integral_constant<int, 1>()) : go(std::integral_constant<int, 2>());
}

template <int QT>
hipError_t run(const MoeArgs& a, uint8_t* ws, hipStream_t st) {
    const MoeWs o(a);
    const int64_t slots = (int64_t)a.T * a.k;
    const bool fast = moe_fast(a);
    Lists l{nullptr, nullptr};
    if (fast && (slots > kScanSlots || tiles_serve(a, o))) {
        l = Lists{(const int32_t*)(ws + o.perm), (const int32_t*)(ws + o.offs)};
        hipLaunchKernelGGL(k_moe_plan, dim3((unsigned)a.E), dim3(64 * kPlanWaves), a.E * 4, st, a.ids, (int)slots, a.E,
                           (int32_t*)(ws + o.perm), (int32_t*)(ws + o.offs), (int4*)(ws + o.table), (int*)(ws + o.tiles), (int)o.max_tiles, large_least(a), run_rows(a));
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
        t.nt[0] = a.F / 128;
        t.nt[1] = a.F / 64;
        t.max_tiles = (int)o.max_tiles;
        t.run = run_rows(a);
        e = moe_tile(a, t, true, st);
        if (e != hipSuccess) return e;
        t.W[0] = a.down;
        t.aux[0] = a.down_aux;
        t.A = (const uint16_t*)ws;
        t.lda = a.F;
        t.a_bytes = (uint32_t)(slots * a.F * 2);
        t.out = ws + o.y;
        t.R = a.N;
        t.K = a.F;
        t.nt[0] = (a.N + 255) / 256;
        t.nt[1] = (a.N + 127) / 128;
        e = moe_tile(a, t, false, st);
    } else {
        e = launch_rows<QT, true>(a, a.A, a.lda, ws, l, fast, st);
        if (e != hipSuccess) return e;
        // One row: its slots' h lie one after the other, and the down products of
        // its experts are one sum (8 experts of 2048 x 1024: 16.7 us with y and its
        // sum, 14.2 without).
        if (fast && a.T == 1 && !l.perm && slots * a.F < (1 << 30))
            return launch_split<QT, kMoeRow, 1, 8>(1, st, a, MoeW{{a.down, nullptr}, {a.down_aux, nullptr}}, (const uint16_t*)ws, a.F,
                                                   nullptr, a.N, a.F, 0, l);
        e = launch_rows<QT, false>(a, (const uint16_t*)ws, a.F, ws + o.y, l, fast, st);
    }
    if (e != hipSuccess) return e;
    const dim3 grid((unsigned)((a.N + 1023) / 1024), (unsigned)std::min(a.T, kSumY), (unsigned)((a.T + kSumY - 1) / kSumY));
    if (y_24(a)) hipLaunchKernelGGL(k_moe_sum<true>, grid, dim3(256), 0, st, a, ws + o.y);
    else hipLaunchKernelGGL(k_moe_sum<false>, grid, dim3(256), 0, st, a, ws + o.y);
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
