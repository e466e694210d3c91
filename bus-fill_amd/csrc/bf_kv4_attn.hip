// Attention over the 4-bit key/value cache (layout: bf_kv4.h): k_kv4_attn.
//
//   o_i = sum_t p_it v_t / sum_t p_it,  p_it = exp(scale q_i . k_t - max),
//   over the tokens t that query i sees: t <= position (causal), t > position -
//   window, and t's page present.  No token seen: o = 0.
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
//   each block of 32 columns has its operand), times q - 8.
// * Running maximum and sum in fp32; the maximum is raised only when a score
//   exceeds it by more than 2^3, so P <= 8 and P d_t <= 65504 always holds, and
//   the accumulators are rarely rescaled.
// * A workgroup's four waves take a chunk's records in turn; they meet in LDS.
//   Sequences of several chunks are joined by a second launch.
#include "bf_device.h"
#include "bf_grid.h"
#include "bf_kv4_launch.h"

namespace bf {
namespace {

constexpr int kAtWaves = 4;
constexpr float kLow = -1e30f;                     // a maximum below every score

template <int BYTES, int ALIGN>
__device__ __forceinline__ void ld_words(uint32_t* dst, const uint8_t* p) {
    __builtin_memcpy(dst, __builtin_assume_aligned(p, ALIGN), BYTES);
}

// One record as a lane holds it.
template <int NB> struct Kv4Rec {
    uint32_t k[2][NB], v[2 * NB];
    uint32_t ks[4 * NB], vs[4 * NB];               // [block][8 tokens] halves
};

constexpr int align_of(int bytes) { return bytes % 16 == 0 ? 16 : bytes % 8 == 0 ? 8 : 4; }

template <int NB>
__device__ __forceinline__ void load_rec(Kv4Rec<NB>& x, const uint8_t* rec, int r, int g) {
    const uint8_t* kp = rec + 16 * NB * (8 * (r >> 2) + (r & 3)) + 4 * NB * g;
    ld_words<4 * NB, align_of(4 * NB)>(x.k[0], kp);
    ld_words<4 * NB, align_of(4 * NB)>(x.k[1], kp + 64 * NB);
    ld_words<8 * NB, align_of(8 * NB)>(x.v, rec + kv4_v_at(32 * NB) + 128 * NB * g + 8 * NB * r);
    ld_words<16 * NB, 16>(x.ks, rec + kv4_ks_at(32 * NB) + 16 * NB * g);
    ld_words<16 * NB, 16>(x.vs, rec + kv4_vs_at(32 * NB) + 16 * NB * g);
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

struct Row {                                       // of a row tile
    int q0, nq, len, rows, row0, h, s;
};

// The row tile of unit u: ((s heads + h) row_tiles + rt); false where it has no rows.
__device__ __forceinline__ bool row_tile_of(const Kv4Args& a, const Kv4Plan& p, int u, Row& o) {
    const int rt = u % p.row_tiles;
    u /= p.row_tiles;
    o.h = u % a.c.heads;
    o.s = u / a.c.heads;
    o.q0 = min(max(a.q_start[o.s], 0), a.T);
    const int q1 = min(max(a.q_start[o.s + 1], o.q0), a.T);
    o.nq = min(q1 - o.q0, a.max_q);
    o.len = min(max(a.kv_len[o.s], 0), a.max_kv);
    o.row0 = rt * kKv4Rows;
    const int64_t left = (int64_t)o.nq * p.group - o.row0;
    o.rows = left < kKv4Rows ? (int)left : kKv4Rows;
    return o.rows > 0;
}

// Cached tokens [lo, hi) that query i of the sequence sees.
__device__ __forceinline__ int hi_of(const Kv4Args& a, const Row& o, int i) {
    return a.causal ? max(0, o.len - o.nq + i + 1) : o.len;
}
__device__ __forceinline__ int lo_of(const Kv4Args& a, const Row& o, int i) {
    return a.window > 0 ? max(0, o.len - o.nq + i - a.window + 1) : 0;
}
// Tiles [t0, t1) that the row tile sees, and the chunks they make (at least one, perhaps empty).
__device__ __forceinline__ int chunks_of(const Kv4Args& a, const Kv4Plan& p, const Row& o, int& t0, int& t1) {
    t0 = lo_of(a, o, o.row0 / p.group) / kKv4Tile;
    t1 = (hi_of(a, o, (o.row0 + o.rows - 1) / p.group) + kKv4Tile - 1) / kKv4Tile;
    const int n = t1 - t0;
    return n > p.chunk ? (n + p.chunk - 1) / p.chunk : 1;
}

__device__ __forceinline__ void store_out(const Kv4Args& a, int64_t at, float y) {
    if (a.out_f16) ((_Float16*)a.O)[at] = (_Float16)y;
    else ((float*)a.O)[at] = y;
}

template <int NB>
__global__ __launch_bounds__(64 * kAtWaves) void k_kv4_attn(Kv4Args a, Kv4Plan p, float* __restrict__ ws) {
    constexpr int D = 32 * NB, W = D < 128 ? D : 128;
    __shared__ float xo[kAtWaves][kKv4Rows][W + 4];
    __shared__ float xm[kAtWaves][kKv4Rows], xl[kAtWaves][kKv4Rows];
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int sp = blockIdx.x % p.splits, unit = blockIdx.x / p.splits;
    Row o;
    if (!row_tile_of(a, p, unit, o)) return;
    int t0, t1;
    const int chunks = chunks_of(a, p, o, t0, t1);
    if (sp >= chunks) return;
    const int c0 = t0 + sp * p.chunk, c1 = min(t1, c0 + p.chunk);
    const int ifirst = o.row0 / p.group, ilast = (o.row0 + o.rows - 1) / p.group;
    const int free0 = lo_of(a, o, ilast), free1 = hi_of(a, o, ifirst);   // tokens that every row sees

    // The lane's query row (rows past the last repeat it: computed, never stored)
    const int row = o.row0 + min(r, o.rows - 1), iq = row / p.group;
    const int lo = lo_of(a, o, iq), hi = hi_of(a, o, iq);
    const uint16_t* qp = a.Q + (int64_t)(o.q0 + iq) * a.ldq + (o.h * p.group + row - iq * p.group) * D + 8 * g;
    h8 q[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) q[b] = *(const h8*)(qp + 32 * b);
    const float sc = a.scale * 1.44269504088896341f;
    const Magic mg = make_magic();

    f4 olo[NB], ohi[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) olo[b] = ohi[b] = f4{0.f, 0.f, 0.f, 0.f};
    float m = kLow, l = 0.f;

    const int per_page = a.c.page_size / kKv4Tile;
    const int32_t* const tab = a.table + (int64_t)o.s * a.ldt;
    // Lane n holds the record of the wave's n-th tile of the next 64 (-1: page absent)
    int recs = 0;
    auto look = [&](int n0) {
        const int tile = c0 + wave + kAtWaves * (n0 + lane);
        recs = -1;
        if (tile < c1) {
            const int pg = tile / per_page, id = tab[pg];
            if (id >= 0 && id < a.c.pages) recs = (id * a.c.heads + o.h) * per_page + (tile - pg * per_page);
        }
    };
    const int mine = c1 - c0 > wave ? (c1 - c0 - wave + kAtWaves - 1) / kAtWaves : 0;
    Kv4Rec<NB> x, y;
    int rec = -1;
    if (mine > 0) {
        look(0);
        rec = __builtin_amdgcn_readlane(recs, 0);
        if (rec >= 0) load_rec<NB>(x, a.data + rec * kv4_record_bytes(D), r, g);
    }
    for (int n = 0; n < mine; n++) {
        int next = -1;
        if (n + 1 < mine) {
            if (((n + 1) & 63) == 0) look(n + 1);
            next = __builtin_amdgcn_readlane(recs, (n + 1) & 63);
            if (next >= 0) load_rec<NB>(y, a.data + next * kv4_record_bytes(D), r, g);
        }
        if (rec >= 0) {
            const int tb = (c0 + wave + kAtWaves * n) * kKv4Tile;
            const bool edge = tb < free0 || tb + kKv4Tile > free1;
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
                for (int e = 0; e < 4; e++) s[4 * i + e] = t[e] * sc;
            }
            if (edge) {
                // hidden tokens: no score, and no scale either (a page's unwritten
                // tail may hold anything)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int t = tb + 8 * g + e;
                    const bool see = t >= lo && t < hi;
                    s[e] = see ? s[e] : -__builtin_inff();
#pragma unroll
                    for (int b = 0; b < NB; b++)
                        if (!see) x.vs[4 * b + (e >> 1)] &= e & 1 ? 0x0000FFFFu : 0xFFFF0000u;
                }
            }
            float tm = s[0];
#pragma unroll
            for (int e = 1; e < 8; e++) tm = __builtin_fmaxf(tm, s[e]);
            if (__any(tm > m + 3.f)) {
                float mn = __builtin_fmaxf(m, tm);
                mn = __builtin_fmaxf(mn, __shfl_xor(mn, 16));
                mn = __builtin_fmaxf(mn, __shfl_xor(mn, 32));
                const float al = __builtin_amdgcn_exp2f(m - mn);
                m = mn;
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
                s[e] = __builtin_amdgcn_exp2f(s[e] - m);
                l += s[e];
            }
#pragma unroll
            for (int b = 0; b < NB; b++) {
                h8 pd;                                 // tokens 0 2 1 3 4 6 5 7, as the masked bytes come
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int t = (e & 4) | ((e & 1) << 1) | ((e >> 1) & 1);
                    pd[e] = (_Float16)(s[t] * half_of(x.vs + 4 * b, t));
                }
                const uint32_t v0 = x.v[2 * b], v1 = x.v[2 * b + 1], w0 = v0 >> 8, w1 = v1 >> 8;
                const h8 vl = __builtin_bit_cast(h8, u4{low2(mg, v0), low2(mg, w0), low2(mg, v1), low2(mg, w1)});
                const h8 vh = __builtin_bit_cast(h8, u4{high2(mg, v0), high2(mg, w0), high2(mg, v1), high2(mg, w1)});
                olo[b] = mfma16x16x32(pd, vl, olo[b]);
                ohi[b] = mfma16x16x32(pd, vh, ohi[b]);
            }
        }
        x = y;
        rec = next;
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);

    // The waves' results meet, 128 columns at a time.
    if (g == 0) {
        xm[wave][r] = m;
        xl[wave][r] = l;
    }
    float M = 0.f, L = 0.f, f[kAtWaves];
    const int orow = threadIdx.x >> 4, oc = threadIdx.x & 15;
    const int arow = o.row0 + orow, ai = arow / p.group, ah = o.h * p.group + arow - ai * p.group;
    const int64_t part = (int64_t)unit * p.splits + sp;
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
        if (cc == 0) {
            M = xm[0][orow];
#pragma unroll
            for (int w = 1; w < kAtWaves; w++) M = __builtin_fmaxf(M, xm[w][orow]);
#pragma unroll
            for (int w = 0; w < kAtWaves; w++) {
                f[w] = __builtin_amdgcn_exp2f(xm[w][orow] - M);
                L += xl[w][orow] * f[w];
            }
        }
        if (orow < o.rows) {
            const float inv = L == 0.f ? 0.f : 1.f / L;
            for (int c = oc; c < W && cc + c < D; c += 16) {
                float y = 0.f;
#pragma unroll
                for (int w = 0; w < kAtWaves; w++) y += xo[w][orow][c] * f[w];
                if (chunks > 1) ws[part * (kKv4Rows * D) + orow * D + cc + c] = y;
                else store_out(a, (int64_t)(o.q0 + ai) * a.ldo + ah * D + cc + c, y * inv);
            }
        }
    }
    if (orow < o.rows && oc == 0) {
        if (chunks > 1) {
            float* ml = ws + p.parts * (kKv4Rows * D) + part * (2 * kKv4Rows) + 2 * orow;
            ml[0] = M;
            ml[1] = L;
        } else if (a.lse) {
            a.lse[(int64_t)(o.q0 + ai) * a.q_heads + ah] =
                L == 0.f ? -__builtin_inff() : (M + __builtin_log2f(L)) * 0.693147180559945309f;
        }
    }
}

// The chunks of a row, joined: one workgroup a row, its waves taking chunks in turn.
template <int NB>
__global__ __launch_bounds__(256) void k_kv4_join(Kv4Args a, Kv4Plan p, const float* __restrict__ ws) {
    constexpr int D = 32 * NB, C = (D + 63) / 64;
    __shared__ float xo[4][D];
    __shared__ float xl[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int unit = blockIdx.x / kKv4Rows, row = blockIdx.x % kKv4Rows;
    Row o;
    if (!row_tile_of(a, p, unit, o) || row >= o.rows) return;
    int t0, t1;
    const int chunks = chunks_of(a, p, o, t0, t1);
    if (chunks == 1) return;
    const int64_t part = (int64_t)unit * p.splits;
    const float* ml = ws + p.parts * (kKv4Rows * D) + part * (2 * kKv4Rows) + 2 * row;
    float M = kLow;
    for (int s = lane; s < chunks; s += 64) M = __builtin_fmaxf(M, ml[s * (2 * kKv4Rows)]);
#pragma unroll
    for (int x = 32; x; x >>= 1) M = __builtin_fmaxf(M, __shfl_xor(M, x));
    float y[C] = {}, L = 0.f;
#pragma unroll 4
    for (int s = wave; s < chunks; s += 4) {
        const float f = __builtin_amdgcn_exp2f(ml[s * (2 * kKv4Rows)] - M);
        L += f * ml[s * (2 * kKv4Rows) + 1];
        const float* src = ws + (part + s) * (kKv4Rows * D) + row * D;
#pragma unroll
        for (int c = 0; c < C; c++)
            if (lane + 64 * c < D) y[c] += f * src[lane + 64 * c];
    }
#pragma unroll
    for (int c = 0; c < C; c++)
        if (lane + 64 * c < D) xo[wave][lane + 64 * c] = y[c];
    if (lane == 0) xl[wave] = L;
    __syncthreads();
    const int arow = o.row0 + row, ai = arow / p.group, ah = o.h * p.group + arow - ai * p.group;
    L = xl[0] + xl[1] + xl[2] + xl[3];
    const float inv = L == 0.f ? 0.f : 1.f / L;
    for (int c = threadIdx.x; c < D; c += 256)
        store_out(a, (int64_t)(o.q0 + ai) * a.ldo + ah * D + c, (xo[0][c] + xo[1][c] + xo[2][c] + xo[3][c]) * inv);
    if (a.lse && threadIdx.x == 0)
        a.lse[(int64_t)(o.q0 + ai) * a.q_heads + ah] =
            L == 0.f ? -__builtin_inff() : (M + __builtin_log2f(L)) * 0.693147180559945309f;
}

template <int NB>
hipError_t launch(const Kv4Args& a, const Kv4Plan& p, float* ws, hipStream_t st) {
    const int64_t units = (int64_t)a.S * a.c.heads * p.row_tiles;
    hipLaunchKernelGGL(k_kv4_attn<NB>, dim3((unsigned)(units * p.splits)), dim3(64 * kAtWaves), 0, st, a, p, ws);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits == 1) return e;
    hipLaunchKernelGGL(k_kv4_join<NB>, dim3((unsigned)(units * kKv4Rows)), dim3(256), 0, st, a, p, ws);
    return hipGetLastError();
}

Kv4Plan plan_of(const Kv4Args& a) { return plan_kv4(a, device_cus() > 0 ? device_cus() : 256); }

}  // namespace

bool kv4_attention_fits(const Kv4Args& a) {
    const Kv4Plan p = plan_of(a);
    const int64_t units = (int64_t)a.S * a.c.heads * p.row_tiles;
    return launch_fits(units * p.splits, 64 * kAtWaves) && launch_fits(units * kKv4Rows, 256);
}

size_t kv4_attention_scratch_bytes(const Kv4Args& a) { return plan_of(a).bytes; }

hipError_t kv4_attention(const Kv4Args& a, float* ws, hipStream_t st) {
    const Kv4Plan p = plan_of(a);
    switch (a.c.dim) {
        case 64: return launch<2>(a, p, ws, st);
        case 96: return launch<3>(a, p, ws, st);
        case 128: return launch<4>(a, p, ws, st);
        default: return launch<8>(a, p, ws, st);
    }
}

}  // namespace bf
