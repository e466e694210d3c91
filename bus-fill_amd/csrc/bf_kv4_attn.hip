// Attention over the 4-bit key/value cache (layout: bf_kv4.h): k_kv4_attn.
//
//   o_i = sum_t p_it v_t / sum_t p_it,  p_it = exp(scale q_i . k_t - max),
//   over the tokens t that query i sees: t <= position (causal), t > position -
//   window or t < sinks, and t's page present.  No token seen: o = 0.
//
// Bound by the cache's bytes (4.5 bits a value) for single tokens.  One wave
// multiplies a record (32 tokens) at a time with 16 query rows (the heads of a
// group and the queries of a sequence), everything in registers:
//
// * Scores: A = key codes (16 tokens), B = query rows, one 16x16x32 MFMA per
//   block of 32 values, so that a key's scale multiplies the block's sum
//   afterwards, in fp32, and no code is scaled.  Codes become the fp16 integers
//   q - 8 with nine instructions for eight of them (masked in place onto the
//   exponent of 1024 or 64, minus 1032 or 72).  Codes left as fp16 subnormals
//   (five instructions, the zero point taken off the sums) were less exact:
//   the matrix unit aligns a subnormal as if it were 2^-14, which costs the sum
//   seven bits.
// * The scores' layout (lane: query l % 16, tokens 8 (l / 16) .. + 7 over the
//   two key operands) is the layout of the next product's A operand: no value
//   moves between lanes.
// * Values: P d_t in fp16 (one rounding; d differs from block to block, so
//   each block of 32 columns has its operand), times q - 8.  P is kept in the
//   range that the largest scale so far leaves (Range in bf_kv4_dev.h).
// * Running maximum and sum in fp32; the maximum is raised only when a score
//   exceeds it by a factor of more than 2^3, so the accumulators are rarely
//   rescaled.
// * A workgroup's four waves take a chunk's records in turn; they meet in LDS.
//   Sequences of several chunks are joined by a second launch.
// * A wave's records come to LDS by direct loads, the next one while one is
//   multiplied (from registers instead, 80 us where this took 54).
//
// Measured, one query a sequence, heads of 128: 32 sequences of 2000 to 8000 tokens,
// 40 heads over 8, 51 us for 184 MB (3.6 TB/s; the longest sequence's workgroup
// lasts until the end); one of 131072 tokens, 32 over 4, 23 us for 75 MB with the
// join's 4.5; one of 519 tokens 8.4 us, which are the chain of lengths, page ids, first
// record, three records a wave and the waves' meeting.  VALU 51 % busy, matrix units
// 9 %.
// With first tokens in sight (SINK; their tiles stand before the window's, Row in
// bf_kv4_dev.h, and a kernel without them is the one above, bit for bit): 32 sequences of up
// to 8000 tokens, window 2048 and 4, 19.3 us for 76 MB (3.9 TB/s); one of 131072, 32
// heads over 4, window 32768 and 100, 15.9 for 19 MB with the join's 4.6; one of 1200, window 1024 and 4, 11.5, five records a
// wave (sixteen waves instead of eight: 12.2).
#include <atomic>

#include "bf_grid.h"
#include "bf_kv4_dev.h"
#include "bf_kv4_launch.h"
#include "bf_lds.h"

namespace bf {
namespace {


// One record as a lane holds it.
template <int NB> struct Kv4Rec {
    uint32_t k[2][NB], v[2 * NB];
    uint32_t ks[4 * NB], vs[4 * NB];               // [block][8 tokens] halves
};

// Records of a wave in LDS: one being multiplied, the others on their way.
template <int NB> constexpr int kRecBytes = 1152 * NB;
template <int NB, int WV> constexpr int kStages = 2;
// Workgroups of four waves that a CU holds at once (registers and LDS).
template <int NB> constexpr int kPerCu = NB <= 4 ? 4 : 2;

// A record into LDS: 1 KB per load, the last one of the lanes that are left.
template <int NB>
__device__ __forceinline__ void fetch_rec(const uint8_t* rec, uint32_t lds, int lane) {
    constexpr int full = kRecBytes<NB> / 1024, rest = kRecBytes<NB> % 1024 / 16;
#pragma unroll
    for (int i = 0; i < full; i++) dma16(rec + 1024 * i + 16 * lane, lds + 1024 * i);
    if constexpr (rest > 0) {
        if (lane < rest) dma16(rec + 1024 * full + 16 * lane, lds + 1024 * full);
    }
}
template <int NB> constexpr int kRecLoads = (kRecBytes<NB> + 1023) / 1024;

// w words (a constant wherever this is unrolled) from an address aligned to w or four of them.
__device__ __forceinline__ void ld_words(uint32_t* dst, const uint8_t* p, int w) {
    if (w == 4) {
        const u4 v = *(const u4*)p;
        dst[0] = v.x; dst[1] = v.y; dst[2] = v.z; dst[3] = v.w;
    } else if (w == 2) {
        const uint2 v = *(const uint2*)p;
        dst[0] = v.x; dst[1] = v.y;
    } else {
        for (int i = 0; i < w; i++) dst[i] = ((const uint32_t*)p)[i];
    }
}

template <int NB>
__device__ __forceinline__ void read_rec(Kv4Rec<NB>& x, const uint8_t* rec, int lane) {
    const int g = lane >> 4;
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int b = 0; b < NB; b += 4)
            ld_words(x.k[i] + b, rec + 512 * b + (i * 64 + lane) * 4 * (NB - b < 4 ? NB - b : 4), NB - b < 4 ? NB - b : 4);
#pragma unroll
    for (int b = 0; b < NB; b += 2)
        ld_words(x.v + 2 * b, rec + 512 * NB + 512 * b + lane * 8 * (NB - b < 2 ? 1 : 2), NB - b < 2 ? 2 : 4);
#pragma unroll
    for (int b = 0; b < NB; b++) {
        ld_words(x.ks + 4 * b, rec + 1024 * NB + 16 * NB * g + 16 * b, 4);
        ld_words(x.vs + 4 * b, rec + 1088 * NB + 16 * NB * g + 16 * b, 4);
    }
}

// Tiles [c0, c1) of head h of a row tile: its rows of O where they are `all` of
// it, else a slot of the workspace.
template <int NB, int WV, bool SINK>
__device__ __forceinline__ void attend(const Kv4Args& a, const Kv4Plan& p, const Row& o, int h, int c0, int c1, bool all,
                                       int64_t slot, float* __restrict__ ws, uint8_t* lds, float (*xm)[kKv4Rows],
                                       float (*xl)[kKv4Rows]) {
    constexpr int D = 32 * NB, W = D < 128 ? D : 128, ST = kStages<NB, WV>;
    float (*const xo)[kKv4Rows][W + 4] = (float (*)[kKv4Rows][W + 4])lds;   // [WV], once the records are done with
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));                  // its multiples are formed here, not kept across units
    const int lane = tid & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ifirst = o.row0 / p.group, ilast = (o.row0 + o.rows - 1) / p.group;
    const int free0 = lo_of(a, o, ilast), free1 = hi_of(a, o, ifirst);   // tokens that every row sees

    // The lane's query row (rows past the last repeat it: computed, never stored)
    const int row = o.row0 + min(r, o.rows - 1), iq = row / p.group;
    const int lo = lo_of(a, o, iq), hi = hi_of(a, o, iq);
    const uint16_t* qp = a.Q + (int64_t)(o.q0 + iq) * a.ldq + (h * p.group + row - iq * p.group) * D + 8 * g;
    h8 q[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) {
        q[b] = *(const h8*)(qp + 32 * b);
        if (a.scale < 0.f) q[b] = -q[b];               // so that a larger sum is a larger score
    }
    const float sc = log2_scale(a.scale);
    const int seen0 = lo_of(a, o, ifirst), seen1 = hi_of(a, o, ilast);     // tokens that some row sees
    const Magic mg = make_magic();

    f4 olo[NB], ohi[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) olo[b] = ohi[b] = f4{0.f, 0.f, 0.f, 0.f};
    Range rg;
    float l = 0.f;

    const int per_page = a.c.page_size / kKv4Tile;
    const int32_t* const tab = a.table + (int64_t)o.s * a.ldt;
    // Lane n holds the record of the wave's n-th tile of the next 64 (-1: page absent)
    int recs = 0;
    auto look = [&](int n0) {
        const int at = c0 + wave + WV * (n0 + lane), tile = o.tile<SINK>(at);
        recs = -1;
        if (at < c1) {
            const int pg = tile / per_page, id = tab[pg];
            if (id >= 0 && id < a.c.pages) recs = (id * a.c.heads + h) * per_page + (tile - pg * per_page);
        }
    };
    const int mine = c1 - c0 > wave ? (c1 - c0 - wave + WV - 1) / WV : 0;
    const uint8_t* const ring = lds + wave * (ST * kRecBytes<NB>);
    const uint32_t ring0 = lds_addr(ring);
    // Record n into stage n % ST (where its page is absent: record 0, not used)
    uint32_t here = 0;                             // bit n % 32: record n's page is there
    auto fetch = [&](int n) {
        if ((n & 63) == 0) look(n);
        const int rec = __builtin_amdgcn_readlane(recs, n & 63);
        here = (here & ~(1u << (n & 31))) | ((rec >= 0 ? 1u : 0u) << (n & 31));
        fetch_rec<NB>(a.data + max(rec, 0) * kv4_record_bytes(D), ring0 + (n % ST) * kRecBytes<NB>, lane);
    };
    for (int n = 0; n < ST - 1 && n < mine; n++) fetch(n);
    for (int n = 0; n < mine; n++) {
        // the stage of record n - 1 is free: its values were in registers before they were used
        if (n + ST - 1 < mine) {
            fetch(n + ST - 1);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((ST - 1) * kRecLoads<NB>) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        if ((here >> (n & 31)) & 1) {
            Kv4Rec<NB> x;
            const uint8_t* const rec = ring + (n % ST) * kRecBytes<NB>;
            // the values' scales, a word (block b, tokens 8 g + 2 j, + 1: word 4 NB g + 4 b + j) a lane
            constexpr int SW = 16 * NB, SL = (SW + 63) / 64;
            uint32_t vw[SL], d = 0;
#pragma unroll
            for (int i = 0; i < SL; i++) {
                vw[i] = *(const uint32_t*)(rec + 1088 * NB + 4 * min(64 * i + lane, SW - 1));
                d = max(d, larger_half(vw[i]));
            }
            read_rec<NB>(x, rec, lane);
            const int tb = o.tile<SINK>(c0 + wave + WV * n) * kKv4Tile;
            const bool edge = (tb < free0 && !(SINK && tb + kKv4Tile <= a.sinks)) || tb + kKv4Tile > free1;
            float s[8];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                f4 t = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    const f4 d = mfma16x16x32(codes8(mg, x.k[i][b]), q[b], f4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                    for (int e = 0; e < 4; e++) t[e] = __builtin_fmaf(half_of(x.ks + 4 * b, 4 * i + e), d[e], t[e]);
                }
#pragma unroll
                for (int e = 0; e < 4; e++) s[4 * i + e] = t[e];
            }
            if (edge) {
                // hidden tokens: no score, and no scale either (a page's unwritten
                // tail may hold anything)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int t = tb + 8 * g + e;
                    const bool see = sees<SINK>(t, lo, hi, a.sinks);
                    s[e] = see ? s[e] : -__builtin_inff();
#pragma unroll
                    for (int b = 0; b < NB; b++)
                        if (!see) x.vs[4 * b + (e >> 1)] &= e & 1 ? 0x0000FFFFu : 0xFFFF0000u;
                }
            }
            float tm = s[0];
#pragma unroll
            for (int e = 1; e < 8; e++) tm = __builtin_fmaxf(tm, s[e]);
            if (__any(rg.over(tm, sc) || d > rg.top)) {
                tm = __builtin_fmaxf(tm, __shfl_xor(tm, 16));
                tm = __builtin_fmaxf(tm, __shfl_xor(tm, 32));
                d = 0;
#pragma unroll
                for (int i = 0; i < SL; i++) {
                    const int w = min(64 * i + lane, SW - 1);
                    d = max(d, larger_seen<SINK>(vw[i], tb + 8 * (w / (4 * NB)) + 2 * (w % 4), seen0, seen1, a.sinks));
                }
                const float al = rg.raise(tm, top_of(rg.top, d), sc);
                l *= al;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float f = __shfl(al, 4 * g + e);
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        olo[b][e] *= f;
                        ohi[b][e] *= f;
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < 8; e++) {
                s[e] = rg.p(s[e], sc);
                l += s[e];
            }
#pragma unroll
            for (int b = 0; b < NB; b++) {
                uint32_t pd4[4];                       // tokens 0 2, 1 3, 4 6, 5 7, as the masked bytes come
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int t = (i & 2) * 2 + (i & 1);
                    pd4[i] = scaled2(s[t], s[t + 2], x.vs[4 * b + (t >> 1)], x.vs[4 * b + (t >> 1) + 1], i & 1);
                }
                const h8 pd = __builtin_bit_cast(h8, u4{pd4[0], pd4[1], pd4[2], pd4[3]});
                const uint32_t v0 = x.v[2 * b], v1 = x.v[2 * b + 1], w0 = v0 >> 8, w1 = v1 >> 8;
                const h8 vl = __builtin_bit_cast(h8, u4{low2(mg, v0), low2(mg, w0), low2(mg, v1), low2(mg, w1)});
                const h8 vh = __builtin_bit_cast(h8, u4{high2(mg, v0), high2(mg, w0), high2(mg, v1), high2(mg, w1)});
                olo[b] = mfma16x16x32(pd, vl, olo[b]);
                ohi[b] = mfma16x16x32(pd, vh, ohi[b]);
            }
        }
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);

    // The waves' results meet, 128 columns at a time.
    if (g == 0) {
        xm[wave][r] = rg.log2_unit(sc);
        xl[wave][r] = l;
    }
    __syncthreads();                               // every wave is done with its records
#pragma unroll
    for (int cc = 0; cc < D; cc += W) {
        if (cc) __syncthreads();
#pragma unroll
        for (int b = cc / 32; b < (cc + W) / 32 && b < NB; b++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                xo[wave][4 * g + e][32 * b - cc + r] = olo[b][e];
                xo[wave][4 * g + e][32 * b - cc + 16 + r] = ohi[b][e];
            }
        __syncthreads();
        constexpr int TPR = 64 * WV / kKv4Rows;
        const int orow = tid / TPR, oc = tid % TPR;
        if (orow >= o.rows) continue;
        const int arow = o.row0 + orow, ai = arow / p.group, ah = h * p.group + arow - ai * p.group;
        float M = xm[0][orow], L = 0.f, f[WV];
#pragma unroll
        for (int w = 1; w < WV; w++) M = __builtin_fmaxf(M, xm[w][orow]);
#pragma unroll
        for (int w = 0; w < WV; w++) {
            f[w] = __builtin_amdgcn_exp2f(xm[w][orow] - M);
            L += xl[w][orow] * f[w];
        }
        const float inv = L == 0.f ? 0.f : 1.f / L;
        for (int c = oc; c < W && cc + c < D; c += TPR) {
            float y = 0.f;
#pragma unroll
            for (int w = 0; w < WV; w++) y += xo[w][orow][c] * f[w];
            if (!all) ws[slot * (kKv4Rows * D) + orow * D + cc + c] = y;
            else store_out(a, (int64_t)(o.q0 + ai) * a.ldo + ah * D + cc + c, y * inv);
        }
        if (cc == 0 && oc == 0) {
            if (!all) {
                float* ml = ws + p.slots * (kKv4Rows * D) + slot * (2 * kKv4Rows) + 2 * orow;
                ml[0] = M;
                ml[1] = L;
            } else if (a.lse) {
                a.lse[(int64_t)(o.q0 + ai) * a.q_heads + ah] =
                    L == 0.f ? -__builtin_inff() : (M + __builtin_log2f(L)) * 0.693147180559945309f;
            }
        }
    }
}

// Item of a workgroup: grid y, and z in steps of kGridY.
constexpr int kGridY = 32768;
__device__ __forceinline__ int64_t grid_item() { return (int64_t)blockIdx.z * kGridY + blockIdx.y; }

template <int NB, int WV, bool SINK>
__global__ __launch_bounds__(64 * WV, kPerCu<NB>) void k_kv4_attn(Kv4Args a, Kv4Plan p, float* __restrict__ ws) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    __shared__ float xm[WV][kKv4Rows], xl[WV][kKv4Rows];
    const int64_t item = grid_item();
    if (item >= p.items) return;
    int sp = 0, h = blockIdx.x;
    if (p.splits > 1) {
        sp = blockIdx.x / a.c.heads;
        h = blockIdx.x - sp * a.c.heads;
    }
    Row o;
    if (!row_tile_of<SINK>(a, p, (int)item, o)) return;
    const int c0 = o.t0 + sp * p.chunk;
    if (sp > 0 && c0 >= o.t1) return;
    attend<NB, WV, SINK>(a, p, o, h, c0, min(o.t1, c0 + p.chunk), o.t1 - o.t0 <= p.chunk, (item * a.c.heads + h) * p.splits + sp,
                   ws, lds, xm, xl);
}

// The chunks of a row, joined: one workgroup a row, its waves taking chunks in turn.
template <int NB, int WV, bool SINK>
__global__ __launch_bounds__(64 * WV) void k_kv4_join(Kv4Args a, Kv4Plan p, int most, const float* __restrict__ ws) {
    constexpr int D = 32 * NB, C = (D + 63) / 64;
    __shared__ float xo[WV][D];
    __shared__ float xl[WV];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t item = grid_item();
    if (item >= p.items) return;
    const int h = blockIdx.x / most, row = blockIdx.x - h * most;
    Row o;
    if (!row_tile_of<SINK>(a, p, (int)item, o) || row >= o.rows) return;
    const int parts = (o.t1 - o.t0 + p.chunk - 1) / p.chunk;
    if (parts <= 1) return;
    const int64_t slot = (item * a.c.heads + h) * p.splits;
    const float* const mls = ws + p.slots * (kKv4Rows * D) + 2 * row;
    float M = kLow;
    for (int i = lane; i < parts; i += 64) M = __builtin_fmaxf(M, mls[(slot + i) * (2 * kKv4Rows)]);
#pragma unroll
    for (int x = 32; x; x >>= 1) M = __builtin_fmaxf(M, __shfl_xor(M, x));
    float y[C] = {}, L = 0.f;
#pragma unroll 4
    for (int i = wave; i < parts; i += WV) {
        const int64_t s = slot + i;
        const float f = __builtin_amdgcn_exp2f(mls[s * (2 * kKv4Rows)] - M);
        L += f * mls[s * (2 * kKv4Rows) + 1];
        const float* src = ws + s * (kKv4Rows * D) + row * D;
#pragma unroll
        for (int c = 0; c < C; c++)
            if (lane + 64 * c < D) y[c] += f * src[lane + 64 * c];
    }
#pragma unroll
    for (int c = 0; c < C; c++)
        if (lane + 64 * c < D) xo[wave][lane + 64 * c] = y[c];
    if (lane == 0) xl[wave] = L;
    __syncthreads();
    const int arow = o.row0 + row, ai = arow / p.group, ah = h * p.group + arow - ai * p.group;
    L = 0.f;
#pragma unroll
    for (int w = 0; w < WV; w++) L += xl[w];
    const float inv = L == 0.f ? 0.f : 1.f / L;
    for (int c = threadIdx.x; c < D; c += 64 * WV) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < WV; w++) v += xo[w][c];
        store_out(a, (int64_t)(o.q0 + ai) * a.ldo + ah * D + c, v * inv);
    }
    if (a.lse && threadIdx.x == 0)
        a.lse[(int64_t)(o.q0 + ai) * a.q_heads + ah] =
            L == 0.f ? -__builtin_inff() : (M + __builtin_log2f(L)) * 0.693147180559945309f;
}

int join_rows(const Kv4Args& a, const Kv4Plan& p) { return (int)std::min<int64_t>(kKv4Rows, (int64_t)a.max_q * p.group); }

dim3 grid_of(const Kv4Plan& p, int64_t x) {
    return dim3((unsigned)x, (unsigned)std::min<int64_t>(p.items, kGridY), (unsigned)((p.items + kGridY - 1) / kGridY));
}

template <int NB, int WV, bool SINK>
hipError_t launch(const Kv4Args& a, const Kv4Plan& p, float* ws, hipStream_t st) {
    constexpr int W = NB < 4 ? 32 * NB : 128, ring = WV * kStages<NB, WV> * kRecBytes<NB>, meet = WV * kKv4Rows * (W + 4) * 4;
    constexpr int lds = ring > meet ? ring : meet;
    auto k = k_kv4_attn<NB, WV, SINK>;
    static std::atomic<uint64_t> attr_set{0};      // one bit per device: LDS limit raised
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (!(attr_set.load(std::memory_order_acquire) & bit)) {
        e = hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return e;
        attr_set.fetch_or(bit, std::memory_order_acq_rel);
    }
    hipLaunchKernelGGL(k, grid_of(p, (int64_t)p.splits * a.c.heads), dim3(64 * WV), lds, st, a, p, ws);
    e = hipGetLastError();
    if (e != hipSuccess || p.slots == 0) return e;
    const int most = join_rows(a, p);
    const dim3 grid = grid_of(p, (int64_t)a.c.heads * most);
    // many chunks a row: more waves on each
    if (p.splits > 32) hipLaunchKernelGGL((k_kv4_join<NB, 16, SINK>), grid, dim3(1024), 0, st, a, p, most, ws);
    else hipLaunchKernelGGL((k_kv4_join<NB, 4, SINK>), grid, dim3(256), 0, st, a, p, most, ws);
    return hipGetLastError();
}

template <int NB>
hipError_t launch(const Kv4Args& a, const Kv4Plan& p, float* ws, hipStream_t st) {
    if (a.sinks > 0) return p.waves == 8 ? launch<NB, 8, true>(a, p, ws, st) : launch<NB, 4, true>(a, p, ws, st);
    return p.waves == 8 ? launch<NB, 8, false>(a, p, ws, st) : launch<NB, 4, false>(a, p, ws, st);
}

Kv4Plan plan_of(const Kv4Args& a) { return plan_kv4(a, device_cus() > 0 ? device_cus() : 256); }

}  // namespace

bool kv4_attention_fits(const Kv4Args& a) {
    const Kv4Plan p = plan_of(a);
    if (p.prompt) return launch_fits(p.items * a.c.heads, 256);
    return launch_fits((int64_t)p.splits * a.c.heads, 64 * p.waves) && launch_fits((int64_t)a.c.heads * kKv4Rows, 1024) &&
           p.items <= (int64_t)kGridY * 65535 && p.items * a.c.heads * p.splits * (64 * p.waves) < (int64_t(1) << 40);
}

size_t kv4_attention_scratch_bytes(const Kv4Args& a) { return plan_of(a).bytes; }

hipError_t kv4_attention(const Kv4Args& a, float* ws, hipStream_t st) {
    const Kv4Plan p = plan_of(a);
    if (p.prompt) return kv4_prompt(a, p, device_cus() > 0 ? device_cus() : 256, st);
    switch (a.c.dim) {
        case 64: return launch<2>(a, p, ws, st);
        case 96: return launch<3>(a, p, ws, st);
        case 128: return launch<4>(a, p, ws, st);
        default: return launch<8>(a, p, ws, st);
    }
}

}  // namespace bf
