// The tile of the prefill kernels: up to 256 activation rows x
// 128 or 256 weight rows, K in steps of 64, both operands of a step in LDS as
// fp16 (described in bf_gemm_tile.hip, which multiplies the rows of one matrix;
// bf_moe_tile.hip multiplies rows gathered by expert).
#pragma once

#include "bf_lds.h"
#include "bf_tile_plan.h"

namespace bf {
namespace {

struct __attribute__((packed, aligned(2))) U2a2 { uint32_t x, y; };
struct __attribute__((packed, aligned(2))) U4a2 { uint32_t x, y, z, w; };

// One thread's share of a super-group of its weight row: 4 / NB threads share
// a row (NB = 1: four, 8 code bytes of each 64-weight step; NB = 2: two, 16
// bytes), part j of each of the four steps, and the row's scales.  The code
// words of a step are reloaded for the next super-group as soon as they are
// decoded, so every load has four steps to arrive.
template <int NB> struct Codes { uint32_t w[2 * NB]; };
template <int QT, int NB> struct TileRaw;
template <int NB> struct TileRaw<QT_Q4_K, NB> { u4 hdr; Codes<NB> q[4]; };
template <int NB> struct TileRaw<QT_PLANES, NB> { u4 hdr; Codes<NB> q[4]; };
template <int NB> struct TileRaw<QT_Q4_0, NB> { uint32_t d[4]; Codes<NB> q[4]; };
template <int QT> constexpr int kStepLoads = QT == QT_Q4_0 ? 2 : 1;   // load instructions of a step's words
template <int QT> constexpr int kHdrLoads = QT == QT_Q4_0 ? 0 : 1;    // of the super-group's scales

template <int NB>
__device__ __forceinline__ void load_codes(Codes<NB>& c, const uint8_t* p) {
    if constexpr (NB == 1) {
        const U2a2 v = *(const U2a2*)p;
        c.w[0] = v.x; c.w[1] = v.y;
    } else {
        const U4a2 v = *(const U4a2*)p;
        c.w[0] = v.x; c.w[1] = v.y; c.w[2] = v.z; c.w[3] = v.w;
    }
}
// row: the row's first byte (planes: of the code plane; aux of the scale plane)
template <int QT, int NB>
__device__ __forceinline__ void load_step(TileRaw<QT, NB>& r, const uint8_t* row, int sg, int c, int j) {
    if constexpr (QT == QT_Q4_K) {
        load_codes<NB>(r.q[c], row + 144 * sg + 16 + 32 * c + 8 * NB * j);
    } else if constexpr (QT == QT_PLANES) {
        load_codes<NB>(r.q[c], row + 128 * sg + 32 * c + 8 * NB * j);
    } else {
        const uint8_t* p = row + 144 * sg + 36 * c + 18 * (NB == 1 ? j >> 1 : j);   // the block
        r.d[c] = *(const uint16_t*)p;
        load_codes<NB>(r.q[c], p + 2 + (NB == 1 ? 8 * (j & 1) : 0));
    }
}
template <int QT, int NB>
__device__ __forceinline__ void load_hdr(TileRaw<QT, NB>& r, const uint8_t* row, const uint8_t* aux, int sg) {
    if constexpr (QT == QT_Q4_K) r.hdr = *(const u4*)(row + 144 * sg);
    if constexpr (QT == QT_PLANES) r.hdr = ld16_a4(aux + 16 * sg);
}

// Scales of a super-group.  Q4_K: thread j of a row derives those of steps
// NB j .. NB j + NB - 1; step c takes them from its lane by DPP.
template <int QT, int NB> struct TileScl { u4 d; };
template <int NB> struct TileScl<QT_Q4_K, NB> { Scl<QT_Q4_K> s[NB]; };
template <int QT, int NB>
__device__ __forceinline__ void tile_scales(TileScl<QT, NB>& o, const TileRaw<QT, NB>& r, int j) {
    if constexpr (QT == QT_Q4_K) {
        Raw<QT_Q4_K> raw;
        raw.hdr = r.hdr;
#pragma unroll
        for (int i = 0; i < NB; i++) o.s[i] = scales(raw, NB * j + i);
    } else if constexpr (QT == QT_PLANES) {
        o.d = r.hdr;
    }
}
// lane C of the quad (NB = 1) or lane C of the lane pair (NB = 2)
template <int NB, int C>
__device__ __forceinline__ float row_lane(float v) {
    constexpr int ctrl = NB == 1 ? C * 0x55 : C | (C << 2) | ((2 + C) << 4) | ((2 + C) << 6);
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), ctrl, 0xF, 0xF, true));
}

// Piece I (0 .. 2 NB - 1) of a thread's 16 NB weights of step C: eight weights,
// k chunk tile_chunk(j, I) of the step.
template <int QT, int NB, int C, int I>
__device__ __forceinline__ h8 tile_decode(const Magic& mg, const TileRaw<QT, NB>& r, const TileScl<QT, NB>& s, int j) {
    if constexpr (QT == QT_PLANES) {
        return decode8_planes(mg, r.q[C].w[I], splat((s.d[C] >> (16 * (NB == 1 ? j >> 1 : j))) & 0xFFFFu));
    } else {
        constexpr bool HI = I >= NB;
        constexpr int w = 2 * (I % NB);
        if constexpr (QT == QT_Q4_0) {
            return decode8_q4_0<HI>(mg, r.q[C].w[w], r.q[C].w[w + 1], splat(r.d[C]));
        } else {
            const Scl<QT_Q4_K>& x = s.s[C % NB];
            constexpr int L = C / NB;
            return decode8_mix<HI>(r.q[C].w[w], r.q[C].w[w + 1], row_lane<NB, L>(HI ? x.sb : x.sa),
                                   row_lane<NB, L>(HI ? x.cb : x.ca));
        }
    }
}
template <int QT, int NB>
__host__ __device__ constexpr int tile_chunk(int j, int i) {
    if (QT == QT_PLANES) return 2 * NB * j + i;
    const int hi = i / NB, lo = i % NB;
    if (QT == QT_Q4_K) return NB * j + lo + 4 * hi;
    return NB == 1 ? 4 * (j >> 1) + (j & 1) + 2 * hi : 4 * j + lo + 2 * hi;
}

// Lane l copies 16 bytes from byte voff + soff of the buffer to LDS byte
// address m0 + 16 l.
__device__ __forceinline__ void dma16_buf(u4 rsrc, uint32_t voff, uint32_t soff, uint32_t m0) {
    asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds" :: "v"(voff), "s"(rsrc), "s"(soff), "{m0}"(m0)
                 : "memory");
}

template <int V>
__device__ __forceinline__ void wait_vm() {
    asm volatile("s_waitcnt vmcnt(%0)" :: "n"(V) : "memory");
}
// End of a phase: this wave's LDS traffic is done, and nothing moves across.
__device__ __forceinline__ void phase_end() {
    __builtin_amdgcn_sched_barrier(0);
    barrier_lds();
    __builtin_amdgcn_sched_barrier(0);
}

// Launch order -> unit: workgroup u runs on XCD u % 8, so each XCD gets a
// contiguous run of the n units (neighbouring units share operand panels, and
// each XCD has an L2 of its own).
__device__ __forceinline__ int xcd_unit(int u, int n) {
    const int x = u & 7, i = u >> 3, q = n >> 3, rem = n & 7;
    return x * q + min(x, rem) + i;
}

// x ^= D in place, where it is written (kept out of loop-invariant hoisting).
template <int D>
__device__ __forceinline__ void step_bits(uint32_t& x) {
    asm volatile("v_xor_b32 %0, %1, %0" : "+v"(x) : "n"(D));
}

// Tile index -> (m, n) tile: bands of kTlBand m-tiles, each n-tile by n-tile
// (the 32 tiles an XCD runs at once then share 4 + 8 operand panels; 1 % over
// m-tiles alone).
constexpr int kTlBand = 4;
__device__ __forceinline__ void tile_at(int tile, int mt, int nt, int& mi, int& ni) {
    const int b = tile / (kTlBand * nt), r = tile - b * kTlBand * nt, h = min(kTlBand, mt - b * kTlBand);
    ni = r / h;
    mi = b * kTlBand + r - ni * h;
}

// A tile of 64 TA batch rows x 128 NB weight rows.  NB = 2: 2 x 4 waves, each
// 32 TA x 64 outputs and the whole step.  NB = 1: 2 x 2 waves of the same size,
// twice (k groups 0 and 1: half of every step each, summed at the end).
template <int QT, int TA, int NB>
struct Tile {
    static constexpr int BM = 64 * TA, BN = 128 * NB, kAStage = BM * 128, kStage = kAStage + BN * 128;
    static constexpr int NS = NB == 1 ? 3 : 2;         // LDS stages
    static constexpr int KH = 2 * NB;                  // k16 slots of a step that a wave multiplies
    static constexpr int NP = 2 * NB;                  // decoded pieces of a thread and step
    static_assert(NS == 3 || kStage == 65536, "two stages differ in one address bit");

    u4 rsrc;
    uint32_t voff[TA];                   // activation DMA offsets
    uint32_t lds0;
    const uint8_t *row, *aux;
    int j, wave, last;
    // LDS bytes in a stage of this thread's first decoded piece and of the wave's
    // fragments of its first k16 slot; the other pieces and slots differ from
    // them in chunk bits only.  With two stages (64 KB apart) they walk through
    // pieces, slots and stages in place.
    uint32_t wst, fa, fw;
    Magic mg;
    TileRaw<QT, NB> raw;
    TileScl<QT, NB> scl;
    f16x acc[TA][2];
    h8 fa_[2][TA], fw_[2][2];

    __device__ __forceinline__ uint32_t piece(int i) const { return wst ^ (16u * tile_chunk<QT, NB>(0, i)); }
    // piece q of a step's activations
    __device__ __forceinline__ void dma(int q, int step, uint32_t stage) {
        dma16_buf(rsrc, voff[q], 128u * (uint32_t)step, lds0 + stage + 1024u * (uint32_t)(wave + 8 * q));
    }
    // Slot H of a step: its fragments are read from stage st while the previous
    // slot's multiply.
    template <int H>
    __device__ __forceinline__ void read(const uint8_t* lds, uint32_t st) {
        if constexpr (NS == 2) {
            step_bits<32 * (H ^ ((H + KH - 1) % KH)) | (H == 0 ? kStage : 0)>(fa);
            step_bits<32 * (H ^ ((H + KH - 1) % KH)) | (H == 0 ? kStage : 0)>(fw);
        }
        const uint32_t xa = NS == 2 ? fa : (fa ^ (32 * H)) + st, xw = NS == 2 ? fw : (fw ^ (32 * H)) + st;
#pragma unroll
        for (int b = 0; b < 2; b++) fw_[H & 1][b] = *(const h8*)(lds + xw + 4096 * b);
#pragma unroll
        for (int t = 0; t < TA; t++) fa_[H & 1][t] = *(const h8*)(lds + xa + 4096 * t);
    }
    template <int P>
    __device__ __forceinline__ void mma(int t0, int t1) {
#pragma unroll
        for (int t = t0; t < t1; t++)
#pragma unroll
            for (int b = 0; b < 2; b++) acc[t][b] = mfma32x32x16(fa_[P][t], fw_[P][b], acc[t][b]);
    }
    template <int H, int C, bool DEC, bool DMA, bool RELOAD>
    __device__ __forceinline__ void slot(uint8_t* lds, int sg, uint32_t st0, uint32_t st1, uint32_t std) {
        constexpr int TH = (TA + 1) / 2, D = (C + 1) & 3;
        const int ds = 4 * sg + C + NS - 1;
        h8 o;
        if constexpr (DMA && 2 * H < TA) dma(2 * H, ds, std);
        read<H>(lds, st0);
        mma<(H + 1) & 1>(0, TH);
        if constexpr (DEC) o = tile_decode<QT, NB, D, H>(mg, raw, scl, j);
        if constexpr (DMA && 2 * H + 1 < TA) dma(2 * H + 1, ds, std);
        if constexpr (RELOAD && H == KH - 1) {
            // the step's words are decoded: the next super-group's into their place
            load_step<QT, NB>(raw, row, C < 3 ? sg + 1 : min(sg + 2, last), D, j);
            if constexpr (C == 3) load_hdr<QT, NB>(raw, row, aux, min(sg + 2, last));
        }
        mma<(H + 1) & 1>(TH, TA);
        if constexpr (DEC) {
            if constexpr (NS == 2) {
                constexpr int P = (H + NP - 1) % NP;
                step_bits<16 * (tile_chunk<QT, NB>(0, H) ^ tile_chunk<QT, NB>(0, P)) | (H == 0 ? kStage : 0)>(wst);
                *(h8*)(lds + wst) = o;
            } else {
                *(h8*)(lds + piece(H) + st1) = o;
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    // Step C of super-group sg (LAST: the range's last one): multiplies stage
    // st0 (its last slot in the next step), decodes the next step's weights
    // into st1 and starts the activations NS - 1 steps ahead.
    template <int C, bool LAST>
    __device__ __forceinline__ void step(uint8_t* lds, int sg, uint32_t* st) {
        constexpr bool kDec = !(LAST && C == 3), kDma = !(LAST && C >= 5 - NS);
        constexpr int n0 = LAST ? 0 : kStepLoads<QT> + (C == 3 ? kHdrLoads<QT> : 0);     // this step's reloads
        constexpr int n1 = C == 0 ? kStepLoads<QT> + kHdrLoads<QT> : LAST ? 0 : kStepLoads<QT>;   // the previous step's
        // two stages alternate (a range starts on stage 0), three rotate
        const uint32_t x0 = NS == 2 ? (C & 1) * kStage : st[0], x1 = NS == 2 ? (1 - (C & 1)) * kStage : st[1];
        const uint32_t xd = NS == 2 ? x1 : st[NS - 1];
        if constexpr (!LAST && C == 3) tile_scales<QT, NB>(scl, raw, j);
        slot<0, C, kDec, kDma, !LAST>(lds, sg, x0, x1, xd);
        slot<1, C, kDec, kDma, !LAST>(lds, sg, x0, x1, xd);
        if constexpr (KH > 2) {
            slot<2, C, kDec, kDma, !LAST>(lds, sg, x0, x1, xd);
            slot<3, C, kDec, kDma, !LAST>(lds, sg, x0, x1, xd);
        }
        // the next step's activations have landed when at most the loads issued
        // after them are outstanding
        if constexpr (NS == 2) wait_vm<n0>();
        else wait_vm<kDma ? TA + n0 + n1 : 0>();
        phase_end();
        if constexpr (NS == 3) {
            const uint32_t t = st[0];
            st[0] = st[1];
            st[1] = st[2];
            st[2] = t;
        }
    }
    __device__ __forceinline__ void run(uint8_t* lds, int s0, int s1) {
        uint32_t st[NS];
#pragma unroll
        for (int i = 0; i < NS; i++) st[i] = i * kStage;
        last = s1 - 1;
        load_hdr<QT, NB>(raw, row, aux, s0);
#pragma unroll
        for (int c = 0; c < 4; c++) load_step<QT, NB>(raw, row, s0, c, j);
#pragma unroll
        for (int q = 0; q < TA; q++) dma(q, 4 * s0, st[0]);
        if constexpr (NS == 3) {
#pragma unroll
            for (int q = 0; q < TA; q++) dma(q, 4 * s0 + 1, st[1]);
        }
        tile_scales<QT, NB>(scl, raw, j);
        *(h8*)(lds + piece(0)) = tile_decode<QT, NB, 0, 0>(mg, raw, scl, j);
        *(h8*)(lds + piece(1)) = tile_decode<QT, NB, 0, 1>(mg, raw, scl, j);
        if constexpr (NP > 2) {
            *(h8*)(lds + piece(2)) = tile_decode<QT, NB, 0, 2 % NP>(mg, raw, scl, j);
            *(h8*)(lds + piece(3)) = tile_decode<QT, NB, 0, 3 % NP>(mg, raw, scl, j);
        }
        load_step<QT, NB>(raw, row, min(s0 + 1, last), 0, j);
        load_hdr<QT, NB>(raw, row, aux, min(s0 + 1, last));
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int e = 0; e < 8; e++) fw_[1][b][e] = 0;
#pragma unroll
        for (int t = 0; t < TA; t++)
#pragma unroll
            for (int e = 0; e < 8; e++) fa_[1][t][e] = 0;
        wait_vm<(NS - 2) * TA + kStepLoads<QT> + kHdrLoads<QT>>();
        phase_end();
        if constexpr (NS == 2) {                       // where the previous step would have left them
            fa ^= 32 * (KH - 1) | kStage;
            fw ^= 32 * (KH - 1) | kStage;
            wst = piece(NP - 1);
        }
        int sg = s0;
        for (; sg < last; sg++) {
            step<0, false>(lds, sg, st);
            step<1, false>(lds, sg, st);
            step<2, false>(lds, sg, st);
            step<3, false>(lds, sg, st);
        }
        step<0, true>(lds, sg, st);
        step<1, true>(lds, sg, st);
        step<2, true>(lds, sg, st);
        step<3, true>(lds, sg, st);
        mma<1>(0, TA);
    }
};

}  // namespace
}  // namespace bf
