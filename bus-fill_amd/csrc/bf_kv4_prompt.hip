// Attention of many queries a sequence over the 4-bit cache: k_kv4_prompt (the
// formula: bf_kv4_attn.hip, whose kernel keeps 16 rows a wave in registers and
// decodes every record for each of them).
//
// A workgroup of four waves takes 128 rows (queries x heads of a group) of one
// key/value head and walks over the records that they see.  A record is decoded
// once for all of them: its codes as the fp16 integers q - 8 and its scales go
// to LDS, keys by token, values by column, two records by turns.  Each wave
// multiplies with its 32 rows:
//
// * S^T = K Q^T, a 32 x 32 tile of v_mfma_f32_32x32x16_f16 per block of 32
//   values, whose sums the keys' scales multiply in fp32.  A lane then holds 16
//   of the 32 tokens of its query; as the A operand of P V it needs eight tokens
//   per instruction in the same lane, so the values' columns are stored with
//   their tokens in that order and nothing moves between lanes.
// * P d in fp16 for each block of 32 columns (one rounding; P in the range that
//   the scales leave, Range in bf_kv4_dev.h: the waves that decode a record leave the
//   largest scale so far beside it), times q - 8.  Scores and probabilities are as exact as the single-token kernel's.  (Keys
//   and values as exact fp16 pairs in LDS instead, hi and lo of (q - 8) d, need
//   no scales here and twice the matrix products: 114 us where this took 95.)
// * 2000 causal tokens, 40 heads over 8 of 128: 94 us, 436 TFLOP/s of the visible
//   pairs; vector instructions issue in 67 % of the SIMDs' cycles, matrix products
//   in 21 %.  A record takes 1.2 us of a CU that holds two workgroups or more, 1.4
//   where one is alone; decoding is 19 us of the 93 (timed without it).  A window of 512
//   with 4 first tokens in sight: 64.5 us, a record more a unit for those; 632 units of 16
//   to 21 records over 512 places, vector instructions in 59 %.
//
// Causal rows see ever more tokens: units go out longest first, every other
// round of one per CU in reverse, so that the units that meet on a CU add up to
// about the same.
#include <atomic>

#include "bf_grid.h"
#include "bf_kv4_dev.h"
#include "bf_kv4_launch.h"

namespace bf {
namespace {

constexpr int kPrWaves = 4, kPrThreads = 64 * kPrWaves;
static_assert(kKv4PromptRows == 32 * kPrWaves);

// LDS rows: 16 bytes past a multiple of 128 (keys, by token) or at 80 bytes
// (values, by column): the eight rows of a 16-byte read on distinct banks.
template <int NB> struct PrLds {
    static constexpr int D = 32 * NB, KRow = 2 * D + 16, VRow = 80;
    static constexpr int V = kKv4Tile * KRow, S = V + D * VRow, Top = S + 128 * NB, Bytes = Top + 16;
};

// A thread's share of a record on its way to LDS.
template <int NB> struct PrRaw {
    static constexpr int KW = (128 * NB + kPrThreads - 1) / kPrThreads, VW = (64 * NB + kPrThreads - 1) / kPrThreads;
    uint32_t k[KW];
    uint2 v[VW];
    uint32_t ks, vs;
};

template <int NB>
__device__ __forceinline__ void load(PrRaw<NB>& x, const uint8_t* rec, int tid) {
#pragma unroll
    for (int i = 0; i < PrRaw<NB>::KW; i++) x.k[i] = *(const uint32_t*)(rec + 4 * min(tid + kPrThreads * i, 128 * NB - 1));
#pragma unroll
    for (int i = 0; i < PrRaw<NB>::VW; i++) x.v[i] = *(const uint2*)(rec + 512 * NB + 8 * min(tid + kPrThreads * i, 64 * NB - 1));
    x.ks = *(const uint32_t*)(rec + 1024 * NB + 4 * min(tid, 16 * NB - 1));
    x.vs = *(const uint32_t*)(rec + 1088 * NB + 4 * min(tid, 16 * NB - 1));
}

// Values of column d, tokens 8 g + 4 h + c, at place 16 (g / 2) + 8 h + 4 (g % 2) + c
// of the column; scales of block b at 32 b + 16 h + 4 g + c (keys', then values').
// top: the range of the values' scales so far (Range), of tokens tb ... in
// [lo, hi) (and first ones); each wave that holds scales leaves its own beside the record.
template <int NB, bool SINK>
__device__ __forceinline__ void decode(const Magic& mg, const PrRaw<NB>& x, uint8_t* lds, int tid, uint32_t& top, int tb, int lo,
                                       int hi, int sinks) {
    using L = PrLds<NB>;
#pragma unroll
    for (int i = 0; i < PrRaw<NB>::KW; i++) {
        const int u = tid + kPrThreads * i;
        if (128 * NB % kPrThreads && u >= 128 * NB) break;
        const int p = u / 512, w = NB - 4 * p < 4 ? NB - 4 * p : 4, at = u - 512 * p, idx = at / w, b = 4 * p + at - idx * w;
        const int r = idx & 15, t = 8 * (r >> 2) + 4 * (idx >> 6) + (r & 3), g = (idx >> 4) & 3;
        *(h8*)(lds + t * L::KRow + 64 * b + 16 * g) = codes8(mg, x.k[i]);
    }
#pragma unroll
    for (int i = 0; i < PrRaw<NB>::VW; i++) {
        const int u = tid + kPrThreads * i;
        if (64 * NB % kPrThreads && u >= 64 * NB) break;
        const int p = u / 128, w = NB - 2 * p < 2 ? 1 : 2, at = u - 128 * p, idx = at / w, b = 2 * p + at - idx * w;
        const int g = idx >> 4, c = idx & 15;
        uint8_t* col = lds + L::V + (32 * b + c) * L::VRow + 32 * (g >> 1) + 8 * (g & 1);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            // tokens 0 2 and 1 3 of four, as masks leave them, into 0 1 and 2 3
            const uint32_t v = h ? x.v[i].y : x.v[i].x, w8 = v >> 8;
            const uint32_t a0 = low2(mg, v), a1 = low2(mg, w8), b0 = high2(mg, v), b1 = high2(mg, w8);
            *(uint2*)(col + 16 * h) = uint2{perm_b32(a1, a0, 0x05040100u), perm_b32(a1, a0, 0x07060302u)};
            *(uint2*)(col + 16 * L::VRow + 16 * h) = uint2{perm_b32(b1, b0, 0x05040100u), perm_b32(b1, b0, 0x07060302u)};
        }
    }
    if (tid < 16 * NB) {
        // A values' scale that is no number becomes 0, and the keys' scale of that
        // token and block NaN instead: rows that do not see the token multiply its
        // values by 0, which must give 0 whatever an unwritten page holds.
        uint32_t bad = 0;
        if ((x.vs & 0x7C00u) == 0x7C00u) bad |= 0x0000FFFFu;
        if ((x.vs & 0x7C000000u) == 0x7C000000u) bad |= 0xFFFF0000u;
        const int g = tid / (4 * NB), b = tid / 4 % NB, e = tid % 4;
        uint8_t* to = lds + L::S + 2 * (32 * b + 16 * (e >> 1) + 4 * g + 2 * (e & 1));
        *(uint32_t*)to = x.ks | bad;
        *(uint32_t*)(to + 64 * NB) = x.vs & ~bad;
        if (__any(larger_half(x.vs & ~bad) > top)) top = top_of(top, larger_seen<SINK>(x.vs, tb + 8 * g + 2 * e, lo, hi, sinks));
        if ((tid & 63) == 0) *(uint32_t*)(lds + L::Top + (tid >> 4)) = top;
    }
}

template <int NB, bool SINK>
__global__ __launch_bounds__(kPrThreads, NB == 8 ? 1 : 2) void k_kv4_prompt(Kv4Args a, Kv4Plan p, int cus) {
    using L = PrLds<NB>;
    constexpr int D = 32 * NB;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, h2 = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // longest units first, every other round of `cus` in reverse
    const int units = (int)(p.items * a.c.heads), round = blockIdx.x / cus, in = blockIdx.x - round * cus;
    const int rank = round & 1 ? min((round + 1) * cus, units) - 1 - in : (int)blockIdx.x;
    const int h = rank % a.c.heads, rest = rank / a.c.heads, s = rest % a.S, rt = p.row_tiles - 1 - rest / a.S;
    Row o;
    if (!row_tile_of<SINK>(a, p, s * p.row_tiles + rt, o)) return;

    // the lane's query row; rows past the last repeat it
    const int row = o.row0 + min(32 * wave + col, o.rows - 1), iq = row / p.group;
    const int lo = lo_of(a, o, iq), hi = hi_of(a, o, iq);
    const int w0 = o.row0 + min(32 * wave, o.rows - 1), w1 = o.row0 + min(32 * wave + 31, o.rows - 1);
    const int wlo = lo_of(a, o, w0 / p.group), whi = hi_of(a, o, w1 / p.group);     // tokens that some row of the wave sees
    const int free0 = lo_of(a, o, w1 / p.group), free1 = hi_of(a, o, w0 / p.group); // ... that all do
    const int head = h * p.group + row - iq * p.group;
    const uint16_t* qp = a.Q + (int64_t)(o.q0 + iq) * a.ldq + head * D + 8 * h2;
    h8 q[2 * NB];
#pragma unroll
    for (int c = 0; c < 2 * NB; c++) {
        q[c] = *(const h8*)(qp + 16 * c);
        if (a.scale < 0.f) q[c] = -q[c];               // so that a larger sum is a larger score
    }
    const float sc = log2_scale(a.scale);
    const Magic mg = make_magic();
    f16x acc[NB];
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[b][e] = 0.f;
    Range rg;
    float l = 0.f;

    const int per_page = a.c.page_size / kKv4Tile;
    const int32_t* const tab = a.table + (int64_t)o.s * a.ldt;
    // Lane n holds the record of the n-th tile of the next 64 (-1: page absent, or no such tile)
    int recs = -1;
    auto look = [&](int n0) {
        const int at = o.t0 + n0 + lane, tile = o.tile<SINK>(at);
        recs = -1;
        if (at < o.t1) {
            const int pg = tile / per_page, id = tab[pg];
            if (id >= 0 && id < a.c.pages) recs = (id * a.c.heads + h) * per_page + (tile - pg * per_page);
        }
    };
    // One record, of tokens tb ...
    auto tile_of = [&](const uint8_t* buf, int tb) {
        // LDS reads run a phase ahead: the keys of up to four blocks before their
        // products, the values before the exponentials (left to the compiler each
        // stood right before its use, 27 waits a record).
        constexpr int HB = NB < 4 ? NB : 4;
        float x[16];
        uint32_t top = *(const uint32_t*)(buf + L::Top);
        if constexpr (NB > 4) top = max(top, *(const uint32_t*)(buf + L::Top + 4));
#pragma unroll
        for (int b0 = 0; b0 < NB; b0 += HB) {
            h8 kf[HB][2], ks[HB][2];
#pragma unroll
            for (int b = 0; b < HB; b++)
#pragma unroll
                for (int i = 0; i < 2; i++) kf[b][i] = *(const h8*)(buf + col * L::KRow + 64 * (b0 + b) + 16 * h2 + 32 * i);
#pragma unroll
            for (int b = 0; b < HB; b++)
#pragma unroll
                for (int i = 0; i < 2; i++) ks[b][i] = *(const h8*)(buf + L::S + 64 * (b0 + b) + 32 * h2 + 16 * i);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int b = 0; b < HB; b++) {
                const f16x zero = {};
                const f16x d = mfma32x32x16(kf[b][1], q[2 * (b0 + b) + 1], mfma32x32x16(kf[b][0], q[2 * (b0 + b)], zero));
#pragma unroll
                for (int e = 0; e < 16; e++)
                    x[e] = __builtin_fmaf((float)ks[b][e >> 3][e & 7], d[e], b0 + b ? x[e] : 0.f);   // (one v_fma_mix_f32 each)
            }
        }
        h8 vf[HB][2];
        u4 vs[HB][2];
        auto values = [&](int b0) {
#pragma unroll
            for (int b = 0; b < HB; b++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    vs[b][i] = *(const u4*)(buf + L::S + 64 * NB + 64 * (b0 + b) + 32 * h2 + 16 * i);
                    vf[b][i] = *(const h8*)(buf + L::V + (32 * (b0 + b) + col) * L::VRow + 16 * h2 + 32 * i);
                }
        };
        __builtin_amdgcn_sched_barrier(0);
        values(0);
        __builtin_amdgcn_sched_barrier(0);
        // the lane's tokens: register 4 a + c is token 8 a + 4 h2 + c
        if ((tb < free0 && !(SINK && tb + kKv4Tile <= a.sinks)) || tb + kKv4Tile > free1) {   // hidden from some row of the wave
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int t = tb + 8 * (e >> 2) + 4 * h2 + (e & 3);
                x[e] = sees<SINK>(t, lo, hi, a.sinks) ? x[e] : -__builtin_inff();
            }
        }
        float tm = x[0];
#pragma unroll
        for (int e = 1; e < 16; e++) tm = __builtin_fmaxf(tm, x[e]);
        if (__any(rg.over(tm, sc) || top > rg.top)) {
            tm = __builtin_fmaxf(tm, __shfl_xor(tm, 32));
            const float al = rg.raise(tm, max(rg.top, (uint32_t)__builtin_amdgcn_readfirstlane((int)top)), sc);
            l *= al;
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const float f = __shfl(al, 8 * (e >> 2) + 4 * h2 + (e & 3));
#pragma unroll
                for (int b = 0; b < NB; b++) acc[b][e] *= f;
            }
        }
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 16; e++) {
            x[e] = rg.p(x[e], sc);
            part[e & 3] += x[e];
        }
        l += (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
        for (int b0 = 0; b0 < NB; b0 += HB) {
            if (b0) values(b0);
#pragma unroll
            for (int b = 0; b < HB; b++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    u4 pd;
#pragma unroll
                    for (int e = 0; e < 4; e++) pd[e] = scaled_pair(x[8 * i + 2 * e], x[8 * i + 2 * e + 1], vs[b][i][e]);
                    acc[b0 + b] = mfma32x32x16(__builtin_bit_cast(h8, pd), vf[b][i], acc[b0 + b]);
                }
        }
    };
    // Tile t0 + n's record (-1: record 0 is read and not used).
    PrRaw<NB> raw;
    auto fetch = [&](int n) {
        if ((n & 63) == 0) look(n);
        const int rec = __builtin_amdgcn_readlane(recs, n & 63);
        load<NB>(raw, a.data + max(rec, 0) * kv4_record_bytes(D), tid);
        return rec;
    };
    const int walk = o.t1 - o.t0;
    const int seen0 = lo_of(a, o, o.row0 / p.group), seen1 = hi_of(a, o, (o.row0 + o.rows - 1) / p.group);   // by some row
    uint32_t seen_top = rg.top;
    int rec = -1, next = -1;
    if (walk > 0) {
        rec = fetch(0);
        decode<NB, SINK>(mg, raw, lds, tid, seen_top, o.tile<SINK>(o.t0) * kKv4Tile, seen0, rec >= 0 ? seen1 : 0, a.sinks);
        next = fetch(1);
        __syncthreads();
    }
    for (int n = 0; n < walk; n++) {
        if (n + 1 < walk)
            decode<NB, SINK>(mg, raw, lds + ((n + 1) & 1) * L::Bytes, tid, seen_top, o.tile<SINK>(o.t0 + n + 1) * kKv4Tile, seen0,
                             next >= 0 ? seen1 : 0, a.sinks);
        const int after = n + 2 < walk ? fetch(n + 2) : -1;
        const int tb = o.tile<SINK>(o.t0 + n) * kKv4Tile;
        if (rec >= 0 && tb < whi && (tb + kKv4Tile > wlo || (SINK && tb < a.sinks))) tile_of(lds + (n & 1) * L::Bytes, tb);
        rec = next;
        next = after;
        __syncthreads();
    }
    l += __shfl_xor(l, 32);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int64_t at = (int64_t)(o.q0 + iq) * a.ldo + head * D;
#pragma unroll
    for (int e = 0; e < 16; e++) {
        const int r = 8 * (e >> 2) + 4 * h2 + (e & 3);             // the row of the lane's sums, held by lane r as a query
        const float g0 = __shfl(inv, r);
        const int64_t to = (int64_t)__shfl((long long)at, r);
        if (32 * wave + r >= o.rows) continue;
#pragma unroll
        for (int b = 0; b < NB; b++) store_out(a, to + 32 * b + col, acc[b][e] * g0);
    }
    if (a.lse && h2 == 0 && 32 * wave + col < o.rows)
        a.lse[(int64_t)(o.q0 + iq) * a.q_heads + head] =
            l == 0.f ? -__builtin_inff() : (rg.log2_unit(sc) + __builtin_log2f(l)) * 0.693147180559945309f;
}

template <int NB, bool SINK>
hipError_t launch(const Kv4Args& a, const Kv4Plan& p, int cus, hipStream_t st) {
    auto k = k_kv4_prompt<NB, SINK>;
    constexpr int lds = 2 * PrLds<NB>::Bytes;

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
    hipLaunchKernelGGL(k, dim3((unsigned)(p.items * a.c.heads)), dim3(kPrThreads), lds, st, a, p, cus);
    return hipGetLastError();
}

template <int NB>
hipError_t launch(const Kv4Args& a, const Kv4Plan& p, int cus, hipStream_t st) {
    return a.sinks > 0 ? launch<NB, true>(a, p, cus, st) : launch<NB, false>(a, p, cus, st);
}

}  // namespace

hipError_t kv4_prompt(const Kv4Args& a, const Kv4Plan& p, int cus, hipStream_t st) {
    switch (a.c.dim) {
        case 64: return launch<2>(a, p, cus, st);
        case 96: return launch<3>(a, p, cus, st);
        case 128: return launch<4>(a, p, cus, st);
        default: return launch<8>(a, p, cus, st);
    }
}

}  // namespace bf
