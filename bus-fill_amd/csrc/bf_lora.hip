// Low-rank adapters of many requests beside a shared projection:
//   Y[t] = C[t] + scale_e B_e (A_e x[t]),  e = ids[t]  (no adapter: Y[t] = C[t]),
// for up to four parts (a fused projection's slices), each with its A and B.
//
// Up to 128 rows (256 of fewer than eight adapters), two launches: s = A x in fp32 (k_lora_down), then C + scale B s
// (k_lora_up).  Rows are taken as they come, in tiles of 16, which may be of as many
// adapters; each adapter of a tile is multiplied with the whole tile (an operand of
// 16x16x32 MFMAs), of which its own rows are kept.  Single tokens of many requests are
// bound by the adapters' bytes whatever the products do.
// More rows are sorted by adapter first (k_lora_order), then taken in tiles of up to 64
// of one adapter (k_lora_down_many, k_lora_up_many, with k_lora_join between them where
// an adapter has more than 64 ranks).  Without the order, tiles of 64 rows as they
// come: 2000 rows of 64 adapters in no order, rank 16, 322 us instead of 34, of 8
// adapters, rank 64, 104 instead of 37; in runs of an adapter it saved nothing (36).
// Every adapter of the pool may have a tile of its own, so that more workgroups are
// launched than have work: 0.5 us for 64 adapters, 12 for 1000.  Above 2047 adapters, or with
// fewer than two rows an adapter, rows are taken as they come (2000 rows, rank 16: 207 to
// 243 us with as many adapters as rows, 37 with one).
//
// Matrices come to LDS by direct loads, eight neighbouring lanes 128 bytes of a row,
// the row's 16-byte pieces in an order that spreads an operand's reads over the banks.
// (Operands straight from memory, a lane's 16 bytes in another row than its
// neighbours', take the load path a cycle a lane: 23 us for the down products of 32
// rows below, 10 through LDS.)
//
// Down: x and A are fp16, their products exact, sums fp32.  K is cut between a
// workgroup's waves, whose sums meet in LDS, and into pieces (partial sums in the
// workspace, added in their order by the next kernel), so that a few rows fill the
// chip.
// Up: s, times a power of two that brings the row's largest to 2^14..2^15, is
// taken as two fp16 numbers of its sign (cut, and the rest rounded: 2^-22 of the
// largest), neither 0 unless s is: times an infinity of B both give the infinity
// that s gives, where a rest of 0 or of the other sign would give NaN.  Sums fp32,
// one rounding of Y.  The matrix unit aligns a product of a subnormal B (below 2^-14) as
// if B were 2^-14, so a column of nothing else loses bits of lo: 2^-17 of |B| |s| at
// 2^-22, where columns from 2^-14 up are within 2^-23.  (B is not scaled: its largest is
// not known before all of it has been read.)
//
// Measured, K = 5120, fp16 C and Y.  One row, rank 16, parts of 5120, 1024 and 1024
// columns: 10.2 us, 4.1 down and 6 up; a launch that does nothing is 2.5, the rest
// is the chain of ids, operands, sums and outputs.  32 rows of 32 adapters of ranks
// 16 to 64, the same parts: 20.6 to 21.9 us, 9.5 and 11.5, for 33 MB of adapters (1.6 TB/s; 2.8
// TB/s of down products with all ranks 64).  2000 rows of six adapters of rank 64, one
// part of 5120 columns: 34 to 37 us, 4 to 5 the order, 12 down and 21 up, for 69 MB.  (Sums
// taken to two numbers of one sign rather than one number and its rest: 0.6 us of that.)
#include <atomic>

#include "bf_device.h"
#include "bf_grid.h"
#include "bf_launch.h"
#include "bf_lds.h"
#include "bf_lora_launch.h"

namespace bf {
namespace {

// Lane l holds the adapter of the tile's row l (-1: none; -2: past the last row).
__device__ __forceinline__ int adapter_of(const LoraArgs& a, int64_t t0, int rows, int lane) {
    if (lane >= rows || t0 + lane >= a.T) return -2;
    const int id = a.ids[t0 + lane];
    return id < 0 || id >= a.adapters ? -1 : id;
}

// ... and how many ranks of it count (0: none).
__device__ __forceinline__ int ranks_of(const LoraArgs& a, int id) {
    if (id < 0) return 0;
    return a.ranks ? min(max(a.ranks[id], 0), a.rank) : a.rank;
}

__device__ __forceinline__ h8 masked(h8 v, bool in) {
    const h8 zero = {};
    return in ? v : zero;
}

// A unit in LDS: operands of 16 rows of 128 bytes, those of A first, piece c of row r at place c ^ (r % 8).
template <int NT> constexpr int kUnitBytes = 2048 * (1 + NT);
__device__ __forceinline__ h8 piece_of(const uint8_t* unit, int operand, int r, int c) {
    return *(const h8*)(unit + 2048 * operand + 128 * r + 16 * (c ^ (r & 7)));
}

// Units [u0, u1) of K: acc[i] += ranks' operand i times the rows.
template <int NT>
__device__ __forceinline__ void dot(f4 (&acc)[4], const uint16_t* x, int64_t ldx, int64_t rows_left, const uint16_t* A, int ranks,
                                    int K, int u0, int u1, const uint8_t* ring, int lane) {
    constexpr int LOADS = 2 * (1 + NT), BYTES = kUnitBytes<NT>;
    const int r = lane & 15, g = lane >> 4, row = lane >> 3, piece = (lane & 7) ^ row;   // (as lanes load: eight rows at once)
    const uint16_t *wp[2 * NT], *xp[2];
#pragma unroll
    for (int i = 0; i < 2 * NT; i++) wp[i] = A + (int64_t)min(8 * i + row, ranks - 1) * K;   // (rows past the rank: not kept)
#pragma unroll
    for (int i = 0; i < 2; i++) xp[i] = x + min((int64_t)(8 * i + row), rows_left - 1) * ldx;
    const uint32_t ring0 = lds_addr(ring);
    auto fetch = [&](int u) {
        const uint32_t to = ring0 + (u & 1) * BYTES;
        const int k = min(kLoraUnit * u + 8 * piece, K - 8);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                  // what was read there has been read
#pragma unroll
        for (int i = 0; i < 2 * NT; i++) dma16(wp[i] + k, to + 1024 * i);
#pragma unroll
        for (int i = 0; i < 2; i++) dma16(xp[i] + k, to + 2048 * NT + 1024 * i);
    };
    if (u0 < u1) fetch(u0);
    for (int u = u0; u < u1; u++) {
        if (u + 1 < u1) {
            fetch(u + 1);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LOADS) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        const uint8_t* const unit = ring + (u & 1) * BYTES;
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const bool in = kLoraUnit * u + 32 * s + 8 * g < K, off = kLoraUnit * (u + 1) > K;   // (the last unit of a K off 64)
            h8 v = piece_of(unit, NT, r, 4 * s + g);
            if (off) v = masked(v, in);
#pragma unroll
            for (int i = 0; i < NT; i++) {
                h8 w = piece_of(unit, i, r, 4 * s + g);
                if (off) w = masked(w, in);
                acc[i] = mfma16x16x32(w, v, acc[i]);
            }
        }
    }
}

// What a workgroup takes of its tile: piece of K (the fastest), ranks, part, sharer.
struct Share {
    int piece, r0, part, share;
};
__device__ __forceinline__ Share share_of(const LoraArgs& a, const LoraPlan& p, int in) {
    Share s;
    s.piece = in % p.pieces;
    in /= p.pieces;
    s.r0 = in % p.rank_parts * kLoraRanks;
    in /= p.rank_parts;
    s.part = in % a.parts;
    s.share = in / a.parts;
    return s;
}

template <int NT>
__global__ __launch_bounds__(64 * kLoraDownWaves) void k_lora_down(LoraArgs a, LoraPlan p, float* __restrict__ ws) {
    constexpr int WV = kLoraDownWaves;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];        // a ring of two units a wave, then the waves' sums
    f4 (*const meet)[NT][64] = (f4 (*)[NT][64])lds;
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    int tile, in;
    if (!lora_place(p.down, blockIdx.x, tile, in)) return;
    const Share q = share_of(a, p, in);
    const int64_t t0 = (int64_t)tile * kLoraSub;
    const int id = adapter_of(a, t0, kLoraSub, lane), rk = ranks_of(a, id);
    const int64_t units = (a.K + kLoraUnit - 1) / kLoraUnit, shares = (int64_t)p.pieces * WV, mine = (int64_t)q.piece * WV + wave;
    const int u0 = (int)(units * mine / shares), u1 = (int)(units * (mine + 1) / shares);
    float* const out = ws + ((int64_t)q.part * p.pieces + q.piece) * a.T * a.rank;
    const uint8_t* const ring = lds + wave * 2 * kUnitBytes<NT>;
    int nth = 0;
    for (uint64_t left = __ballot(id >= 0); left; nth++) {
        const int first = __builtin_ctzll(left), e = __builtin_amdgcn_readlane(id, first), ranks = __builtin_amdgcn_readlane(rk, first);
        const uint64_t rows = __ballot(id == e);
        left &= ~rows;
        if (nth != q.share) continue;              // (as many sharers as a tile can have adapters)
        if (q.r0 >= ranks) return;
        const uint16_t* const A = a.part[q.part].A + ((int64_t)e * a.rank + q.r0) * a.K;
        const uint16_t* const x = a.X + t0 * a.ldx;
        const int tiles = min(NT, (ranks - q.r0 + 15) / 16);
        f4 acc[4];
#pragma unroll
        for (int i = 0; i < 4; i++) acc[i] = f4{0.f, 0.f, 0.f, 0.f};
        if (NT == 1 || tiles == 1) dot<1>(acc, x, a.ldx, a.T - t0, A, ranks - q.r0, a.K, u0, u1, ring, lane);
        else if (NT == 2 || tiles == 2) dot<2>(acc, x, a.ldx, a.T - t0, A, ranks - q.r0, a.K, u0, u1, ring, lane);
        else dot<NT>(acc, x, a.ldx, a.T - t0, A, ranks - q.r0, a.K, u0, u1, ring, lane);
        // the waves' sums, added in their order
        __syncthreads();                           // every wave is done with its ring
#pragma unroll
        for (int i = 0; i < NT; i++) meet[wave][i][lane] = acc[i];
        __syncthreads();
        // wave i: lane's row r of the tile, ranks r0 + 16 i + 4 g ..
        const int at = q.r0 + 16 * wave + 4 * g;
        if (wave < tiles && ((rows >> r) & 1) && at < a.rank) {            // (rank % 8 == 0)
            f4 s = meet[0][wave][lane];
#pragma unroll
            for (int v = 1; v < WV; v++) s += meet[v][wave][lane];
            *(f4*)(out + (t0 + r) * a.rank + at) = s;
        }
        return;
    }
}

// Many rows' order by adapter and its tiles of up to 64, by one workgroup: rows are
// counted, adapters' tiles summed up, rows placed (in which order within an adapter
// changes no result: a row's sums depend on no other row).  2000 rows: 4.2 us, of which
// a launch that does nothing is 2.  (Every workgroup of the down products for itself, up
// to 4096 rows: 5.7 us more there.)
constexpr int kOrderThreads = 1024, kOrderRows = 4;                        // rows a thread and turn
// Increments bins[id] for the lanes with live; the value before (of lane after lane where a wave's lanes are of one adapter).
__device__ __forceinline__ int claim(int* bins, int id, bool live, int lane) {
    const int first = __builtin_amdgcn_readfirstlane(id);
    const uint64_t all = __ballot(live);
    if (__ballot(live && id == first) != all) return live ? atomicAdd(&bins[id], 1) : 0;
    int at = 0;
    if (lane == 0 && all) at = atomicAdd(&bins[first], __builtin_popcountll(all));
    return __builtin_amdgcn_readfirstlane(at) + lane;                      // (live lanes come first)
}
__global__ __launch_bounds__(kOrderThreads) void k_lora_order(LoraArgs a, LoraPlan p, float* __restrict__ ws) {
    __shared__ int bins[kLoraBins];                // a counter an adapter, and one for rows without
    __shared__ int part[kOrderThreads / 64];
    LoraTile* const tiles = (LoraTile*)(ws + p.tiles);
    int* const rows = (int*)(ws + p.rows);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = a.adapters + 1;
    int ids[kOrderRows];
    auto load = [&](int64_t t0) {
#pragma unroll
        for (int i = 0; i < kOrderRows; i++) {
            const int id = a.ids[min(t0 + kOrderThreads * i + tid, (int64_t)a.T - 1)];
            ids[i] = id < 0 || id >= a.adapters ? a.adapters : id;
        }
    };
    // (waits for LDS only, not for stores)
    auto meet = [] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    const int64_t turn = kOrderThreads * kOrderRows;
    load(0);
    // a thread's adapters: b0 .. b1 - 1
    const int per = (n + kOrderThreads - 1) / kOrderThreads, b0 = min(tid * per, n), b1 = min(b0 + per, n);
    const int rk0 = b0 < a.adapters ? ranks_of(a, b0) : 0;
    for (int i = tid; i < n; i += kOrderThreads) bins[i] = 0;
    meet();
    for (int64_t t0 = 0; t0 < a.T; t0 += turn) {
        if (t0) load(t0);
#pragma unroll
        for (int i = 0; i < kOrderRows; i++)
            if (t0 + kOrderThreads * i < a.T) claim(bins, ids[i], t0 + kOrderThreads * i + tid < a.T, lane);
    }
    meet();
    // the tiles before them; from here on a counter holds the place, 64 a tile, of its adapter's next row
    int count = 0;
    for (int b = b0; b < b1; b++) count += (bins[b] + 63) / 64;
    int before = count;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) {
        const int c = __shfl_up(before, x);
        if (lane >= x) before += c;
    }
    if (lane == 63) part[wave] = before;
    before -= count;
    meet();
    int total = 0;
#pragma unroll
    for (int w = 0; w < kOrderThreads / 64; w++) {
        before += w < wave ? part[w] : 0;
        total += part[w];
    }
    for (int b = b0; b < b1; b++) {
        const int here = bins[b];
        bins[b] = 64 * before;
        const int e = b < a.adapters ? b : -1, rk = !here || e < 0 ? 0 : b == b0 ? rk0 : ranks_of(a, e);
        for (int i = 0; i < here; i += 64) tiles[before++] = LoraTile{e, min(64, here - i), rk, 0};
    }
    if (tid == 0) tiles[p.most].adapter = total;
    meet();
    for (int64_t t0 = 0; t0 < a.T; t0 += turn) {
        if (a.T > turn) load(t0);
#pragma unroll
        for (int i = 0; i < kOrderRows; i++) {
            if (t0 + kOrderThreads * i >= a.T) break;
            const int64_t t = t0 + kOrderThreads * i + tid;
            const int at = claim(bins, ids[i], t < a.T, lane);
            if (t < a.T) rows[at] = (int)t;
        }
    }
}

// Workgroup's tile of many rows, its rows, and which of the tile's workgroups it is.
__device__ __forceinline__ bool tile_of(const LoraPlan& p, const LoraGrid& g, const float* ws, LoraTile& o, const int*& rows, int& in) {
    const LoraTile* const tiles = (const LoraTile*)(ws + p.tiles);
    int tile;
    if (!lora_place(lora_grid(tiles[p.most].adapter, g.inner), blockIdx.x, tile, in)) return false;
    o = tiles[tile];
    rows = (const int*)(ws + p.rows) + 64 * (int64_t)tile;
    return true;
}

// Many rows: a wave takes 16 of 64 rows and half of each slab of K; x comes to its
// registers, A's rows, two slabs by turns, to LDS for all eight.  (Four waves with whole
// slabs: 11.1 us for 2000 rows of one adapter, K = 5120, 64 ranks, where this took 9.9; LDS
// gives eight waves 1.7 times what it gives four.)
template <int NT>
__global__ __launch_bounds__(64 * kLoraManyWaves) void k_lora_down_many(LoraArgs a, LoraPlan p, float* __restrict__ ws) {
    constexpr int WV = kLoraManyWaves, STEPS = kLoraSlab / kLoraStep / 2, UNITS = kLoraSlab / kLoraUnit, BYTES = UNITS * NT * 2048;
    constexpr int LOADS = UNITS * NT * 2;          // direct loads of a slab, eight rows of 128 bytes each: wave w does every WV-th
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];        // two slabs, [unit][operand][16 rows of 128 bytes]
    f4 (*const meet)[NT][64] = (f4 (*)[NT][64])lds;                        // at the end: [4], sums of the waves with the second halves
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4, row = lane >> 3, piece = (lane & 7) ^ row;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), sub = wave & 3, half = wave >> 2;
    LoraTile o;
    const int* rows;
    int in;
    if (!tile_of(p, p.down, ws, o, rows, in)) return;
    const Share q = share_of(a, p, in);
    const int ranks = o.ranks - q.r0;
    if (ranks <= 0) return;
    const int64_t mine = rows[min(16 * sub + r, o.rows - 1)];
    const bool busy = 16 * sub < o.rows;           // the wave has rows
    const int64_t units = (a.K + kLoraUnit - 1) / kLoraUnit;
    const int k0 = kLoraUnit * (int)(units * q.piece / p.pieces), k1 = min(a.K, kLoraUnit * (int)(units * (q.piece + 1) / p.pieces));
    const uint16_t* const x = a.X + mine * a.ldx;
    const uint16_t* const A = a.part[q.part].A + ((int64_t)o.adapter * a.rank + q.r0) * a.K;

    h8 xv[2][STEPS];
    // (the buffer's readers have passed a barrier)
    auto fetch = [&](int k, int buf, h8 (&v)[STEPS]) {
#pragma unroll
        for (int i = 0; i < (LOADS + WV - 1) / WV; i++) {
            const int n = WV * i + wave;           // unit, eight rows
            if (n >= LOADS) break;
            const int u = n / (2 * NT), m = n % (2 * NT), at = min(k + kLoraUnit * u + 8 * piece, a.K - 8);
            dma16(A + (int64_t)min(8 * m + row, ranks - 1) * a.K + at, lds_addr(lds) + buf * BYTES + 1024 * n);
        }
        if (busy)
#pragma unroll
            for (int i = 0; i < STEPS; i++) v[i] = *(const h8*)(x + min(k + kLoraStep * (STEPS * half + i) + 8 * g, a.K - 8));
    };
    f4 acc[NT];
#pragma unroll
    for (int i = 0; i < NT; i++) acc[i] = f4{0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](int k, int buf, const h8 (&v)[STEPS]) {
        // A's operands are read a step ahead of their products
        h8 w[2][NT];
        auto read = [&](int i) {
            const int n = STEPS * half + i;
#pragma unroll
            for (int m = 0; m < NT; m++)
                w[i & 1][m] = piece_of(lds + buf * BYTES + (n >> 1) * (2048 * NT), m, r, 4 * (n & 1) + g);
        };
        read(0);
#pragma unroll
        for (int i = 0; i < STEPS; i++) {
            const int at = k + kLoraStep * (STEPS * half + i);
            if (at >= k1) break;
            if (i + 1 < STEPS) read(i + 1);
            __builtin_amdgcn_sched_barrier(0);
            const bool off = at + kLoraStep > k1, ok = at + 8 * g < k1;
            const h8 b = off ? masked(v[i], ok) : v[i];
#pragma unroll
            for (int m = 0; m < NT; m++) acc[m] = mfma16x16x32(off ? masked(w[i & 1][m], ok) : w[i & 1][m], b, acc[m]);
        }
    };
    // one slab; false after the last
    auto turn = [&](int k, int buf, const h8 (&v)[STEPS], h8 (&w)[STEPS]) -> bool {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();                           // this slab is here, the other one has been read
        const bool more = k + kLoraSlab < k1;
        if (more) fetch(k + kLoraSlab, 1 - buf, w);
        if (busy) multiply(k, buf, v);
        return more;
    };
    fetch(k0, 0, xv[0]);
    for (int k = k0; turn(k, 0, xv[0], xv[1]) && turn(k + kLoraSlab, 1, xv[1], xv[0]); k += 2 * kLoraSlab) {
    }
    __syncthreads();
    if (half && busy)
#pragma unroll
        for (int m = 0; m < NT; m++) meet[sub][m][lane] = acc[m];
    __syncthreads();
    if (half || 16 * sub + r >= o.rows) return;
    float* const out = ws + (((int64_t)q.part * p.pieces + q.piece) * a.T + mine) * a.rank;
#pragma unroll
    for (int m = 0; m < NT; m++) {
        const int at = q.r0 + 16 * m + 4 * g;
        if (at < a.rank) *(f4*)(out + at) = acc[m] + meet[sub][m][lane];
    }
}

// Of a row with `ranks` ranks, at s0 the pieces' sums (`step` apart): the sum of ranks k .. k + 3, pieces in their order.
__device__ __forceinline__ f4 sum4(const float* s0, int64_t step, int pieces, int k, int ranks) {
    f4 s = f4{0.f, 0.f, 0.f, 0.f};
    if (k < ranks) {
        f4 v[kLoraPieces];                         // (loads of all pieces at once)
#pragma unroll
        for (int i = 0; i < kLoraPieces; i++) v[i] = *(const f4*)(s0 + min(i, pieces - 1) * step + k);
        s = v[0];
#pragma unroll
        for (int i = 1; i < kLoraPieces; i++)
            if (i < pieces) s += v[i];
#pragma unroll
        for (int j = 1; j < 4; j++)
            if (k + j >= ranks) s[j] = 0.f;
    }
    return s;
}

// A pair of numbers to two fp16 numbers each: hi the largest below it in magnitude, lo the rest rounded, both of at least
// 2^-24 and of its sign (0 of 0).  NaN: hi NaN; infinite: hi infinite.  Magnitudes 0, or 2^-100 and up, to below 2^15.
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
    const float v[2] = {__builtin_fabsf(a), __builtin_fabsf(b)};
    float least[2], low[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        least[i] = __builtin_fminf(v[i] * 0x1p100f, 0x1p-24f);
        const float cut = v[i] * (1.f - 0x1p-24f);                         // (the fp32 number below)
        low[i] = cut < least[i] ? least[i] : cut;
    }
    const h2 h = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(low[0], low[1]));
#pragma unroll
    for (int i = 0; i < 2; i++) low[i] = __builtin_fmaxf(v[i] - (float)h[i], least[i]);   // (an infinity's rest: the least)
    const uint32_t sign = (__builtin_bit_cast(uint32_t, a) >> 16 & 0x8000u) | (__builtin_bit_cast(uint32_t, b) & 0x80000000u);
    hi = as_u32(h) | sign;
    lo = as_u32(h2{(_Float16)low[0], (_Float16)low[1]}) | sign;
}

// A row's sums, fours of ranks by PER neighbouring lanes in turn (this one `me`), to
// two fp16 numbers each, times 2^shift: put(k, hi, lo) of ranks k .. k + 3, k below
// `padded`.  Returns the shift.
template <int PER, class P>
__device__ __forceinline__ int split_row(const float* s0, int64_t step, int pieces, int ranks, int me, int padded, P put) {
    f4 held[2];
    float top = 0.f;
    for (int i = 0, k = 4 * me; k < padded; k += 4 * PER, i++) {
        const f4 s = sum4(s0, step, pieces, k, ranks);
        if (i == 0) held[0] = s;
        if (i == 1) held[1] = s;
#pragma unroll
        for (int j = 0; j < 4; j++) top = __builtin_fmaxf(top, __builtin_fabsf(s[j]));
    }
#pragma unroll
    for (int x = 1; x < PER; x <<= 1) top = __builtin_fmaxf(top, __shfl_xor(top, x));
    // (s is a sum of products of fp16 numbers, a multiple of 2^-48 and below 2^57 where x is finite: the shift is -42 to 63;
    // beside an infinity no number's value matters, but all stay finite)
    const int shift = !(top > 0.f) ? 0 : top < __builtin_inff() ? 15 - __builtin_amdgcn_frexp_expf(top) : -48;
    const float up = __builtin_ldexpf(1.f, shift);
    for (int i = 0, k = 4 * me; k < padded; k += 4 * PER, i++) {
        const f4 s = i == 0 ? held[0] : i == 1 ? held[1] : sum4(s0, step, pieces, k, ranks);
        uint2 hi, lo;
        split2(s[0] * up, s[1] * up, hi.x, lo.x);
        split2(s[2] * up, s[3] * up, hi.y, lo.y);
        put(k, hi, lo);
    }
    return shift;
}

// The joined sums of many rows in the workspace.
struct Joined {
    _Float16 *hi, *lo;                             // [part][T][padded]
    float* factor;                                 // [part][T]: scale 2^-shift (0: no adapter)
};
__device__ __forceinline__ Joined joined_of(const LoraArgs& a, const LoraPlan& p, float* ws) {
    Joined j;
    const int64_t n = (int64_t)a.parts * a.T * p.padded;
    j.hi = (_Float16*)(ws + p.joined);
    j.lo = j.hi + n;
    j.factor = (float*)(j.lo + n);
    return j;
}

// Sixteen lanes a row; grid y: part.
constexpr int kJoinRows = 16;
__global__ __launch_bounds__(16 * kJoinRows) void k_lora_join(LoraArgs a, LoraPlan p, float* __restrict__ ws) {
    const int64_t t = (int64_t)blockIdx.x * kJoinRows + threadIdx.x / 16;
    if (t >= a.T) return;
    const int part = blockIdx.y, me = threadIdx.x % 16;
    int id = a.ids[t];
    if (id < 0 || id >= a.adapters) id = -1;
    const int ranks = ranks_of(a, id);
    const Joined j = joined_of(a, p, ws);
    const int64_t row = (int64_t)part * a.T + t;
    const int shift = split_row<16>(ws + ((int64_t)part * p.pieces * a.T + t) * a.rank, (int64_t)a.T * a.rank, p.pieces, ranks, me,
                                    p.padded, [&](int k, uint2 hi, uint2 lo) {
                                        *(uint2*)(j.hi + row * p.padded + k) = hi;
                                        *(uint2*)(j.lo + row * p.padded + k) = lo;
                                    });
    if (me == 0) j.factor[row] = id < 0 ? 0.f : __builtin_ldexpf(a.scales ? a.scales[id] : 1.f, -shift);
}

// Four neighbouring columns of a row, n of them inside, as they are held.
template <bool F16> struct Held {
    typedef f4 type;
};
template <> struct Held<true> {
    typedef uint2 type;
};
template <bool F16> __device__ __forceinline__ typename Held<F16>::type load_c(const LoraArgs& a, int64_t i, int n) {
    typename Held<F16>::type c = {};
    if constexpr (F16) {
        const uint16_t* const p = (const uint16_t*)a.C + i;
        if (a.wide && n >= 4) c = *(const uint2*)p;
        else {
            if (n > 0) c.x = p[0];
            if (n > 1) c.x |= (uint32_t)p[1] << 16;
            if (n > 2) c.y = p[2];
            if (n > 3) c.y |= (uint32_t)p[3] << 16;
        }
    } else {
        const float* const p = (const float*)a.C + i;
        if (a.wide && n >= 4) c = *(const f4*)p;
        else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (e < n) c[e] = p[e];
        }
    }
    return c;
}
template <bool F16> __device__ __forceinline__ void store_y(const LoraArgs& a, int64_t i, typename Held<F16>::type y, int n) {
    if constexpr (F16) {
        uint16_t* const p = (uint16_t*)a.Y + i;
        if (a.wide && n >= 4) *(uint2*)p = y;
        else {
            if (n > 0) p[0] = (uint16_t)y.x;
            if (n > 1) p[1] = (uint16_t)(y.x >> 16);
            if (n > 2) p[2] = (uint16_t)y.y;
            if (n > 3) p[3] = (uint16_t)(y.y >> 16);
        }
    } else {
        float* const p = (float*)a.Y + i;
        if (a.wide && n >= 4) *(f4*)p = y;
        else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (e < n) p[e] = y[e];
        }
    }
}
// c + f d
__device__ __forceinline__ f4 add(f4 c, float f, f4 d) {
#pragma unroll
    for (int e = 0; e < 4; e++) c[e] = __builtin_fmaf(f, d[e], c[e]);
    return c;
}
__device__ __forceinline__ uint2 add(uint2 c, float f, f4 d) {
    const h2 lo = as_h2(c.x), hi = as_h2(c.y);
    const f4 y = add(f4{(float)lo[0], (float)lo[1], (float)hi[0], (float)hi[1]}, f, d);
    return uint2{as_u32(h2{(_Float16)y[0], (_Float16)y[1]}), as_u32(h2{(_Float16)y[2], (_Float16)y[3]})};
}

// 16 neighbouring bytes of a row, n of their elements inside.
template <bool F16> struct Run {
    typedef f4 type;
};
template <> struct Run<true> {
    typedef u4 type;
};
template <bool F16> __device__ __forceinline__ typename Run<F16>::type load_run(const LoraArgs& a, int64_t i, int n) {
    typename Run<F16>::type c = {};
    if constexpr (F16) {
        const uint16_t* const p = (const uint16_t*)a.C + i;
        if (a.wide && n >= 8) c = *(const u4*)p;
        else {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (e < n) c[e >> 1] |= (uint32_t)p[e] << (16 * (e & 1));
        }
        return c;
    } else {
        return load_c<false>(a, i, n);
    }
}
template <bool F16> __device__ __forceinline__ void store_run(const LoraArgs& a, int64_t i, typename Run<F16>::type y, int n) {
    if constexpr (F16) {
        uint16_t* const p = (uint16_t*)a.Y + i;
        if (a.wide && n >= 8) *(u4*)p = y;
        else {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (e < n) p[e] = (uint16_t)(y[e >> 1] >> (16 * (e & 1)));
        }
    } else {
        store_y<false>(a, i, y, n);
    }
}
__device__ __forceinline__ f4 add_run(f4 c, float f, const float (&d)[4]) { return add(c, f, f4{d[0], d[1], d[2], d[3]}); }
__device__ __forceinline__ u4 add_run(u4 c, float f, const float (&d)[8]) {
    const uint2 lo = add(uint2{c.x, c.y}, f, f4{d[0], d[1], d[2], d[3]}), hi = add(uint2{c.z, c.w}, f, f4{d[4], d[5], d[6], d[7]});
    return u4{lo.x, lo.y, hi.x, hi.y};
}

// Step `at` of the parts' columns, `steps` operands' blocks of 64 each.
__device__ __forceinline__ int part_of(const LoraArgs& a, int steps, int& at) {
    int part = 0;
    for (; part < a.parts - 1; part++) {
        const int n = ((a.part[part].N + kLoraCols - 1) / kLoraCols + steps - 1) / steps;
        if (at < n) break;
        at -= n;
    }
    return part;
}

// A block of B in LDS, columns of RC ranks: the place of a column's piece of eight ranks, such that neighbouring lanes, which
// read columns 2^SH apart, meet different banks.
template <int RC, int SH> __device__ __forceinline__ int place(int col, int piece) { return piece ^ ((col >> SH) & (RC / 8 - 1)); }
// Column c's ranks k0 + k .. of a block that holds k0 .., of which `ranks` count (what lies past them may be anything).
template <int RC, int SH> __device__ __forceinline__ h8 block_at(const uint8_t* block, int c, int k0, int k, int ranks) {
    h8 b = *(const h8*)(block + 2 * RC * c + 16 * place<RC, SH>(c, (k / 8) & (RC / 8 - 1)));
    if (k0 + (k & ~31) + 32 > ranks || RC < 32)
#pragma unroll
        for (int i = 0; i < 8; i++) b[i] = k < RC && k0 + k + i < ranks ? b[i] : (_Float16)0.f;
    return b;
}

// Few rows.  RC: ranks of B that come to LDS at once.
template <int RC, bool F16>
__global__ __launch_bounds__(64 * kLoraUpWaves) void k_lora_up(LoraArgs a, LoraPlan p, const float* __restrict__ ws) {
    constexpr int ROWS = kLoraSub, WV = kLoraUpWaves, PER = 64 * WV / ROWS;   // lanes a row of sums
    constexpr int PIECES = RC / 8, KS = (RC + 31) / 32, BYTES = 2 * kLoraCols * RC;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];        // a block of B a wave, then the sums: fp16 [hi, lo][ROWS][ld]
    __shared__ f4 factor4[ROWS / 4];
    float* const factor = (float*)factor4;
    _Float16* const sums = (_Float16*)(lds + WV * BYTES);
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int tile, at;
    if (!lora_place(p.up, blockIdx.x, tile, at)) return;
    const int part = part_of(a, p.up_steps, at);
    const LoraPart& w = a.part[part];
    const int n0 = at * p.up_steps * kLoraCols, n1 = min(w.N, n0 + p.up_steps * kLoraCols);
    const int64_t t0 = (int64_t)tile * ROWS;
    const int id = adapter_of(a, t0, ROWS, lane), rk = ranks_of(a, id);
    const float sc = id < 0 ? 0.f : a.scales ? a.scales[id] : 1.f;
    const int ld = lora_lds_ranks(a.rank), padded = ld - 8;

    // The wave's pairs of adapter and step, in turn
    uint64_t left = __ballot(id != -2), rows = 0;
    int nth = -1, n = n1, e = -1, ranks = 0;
    auto next = [&]() -> bool {
        for (;;) {
            n += kLoraCols;
            if (n >= n1) {
                if (!left) return false;
                const int first = __builtin_ctzll(left);
                e = __builtin_amdgcn_readlane(id, first);
                ranks = __builtin_amdgcn_readlane(rk, first);
                rows = __ballot(id == e);
                left &= ~rows;
                n = n0;
            }
            if (++nth % WV == wave) return true;
        }
    };
    // Columns n .. n + 63, ranks k0 .. k0 + RC - 1 of B
    const uint8_t* const block = lds + wave * BYTES;
    auto fetch = [&](int k0) {
        const uint16_t* const B = w.B + (int64_t)e * w.N * a.rank;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                 // what was read there has been read
#pragma unroll
        for (int i = 0; i < PIECES; i++) {
            const int q = 64 * i + lane, col = q / PIECES, k = k0 + 8 * place<RC, 2>(col, q % PIECES);
            if (k < ranks) dma16(B + (int64_t)min(n + col, w.N - 1) * a.rank + k, lds_addr(block) + 1024 * i);
        }
    };
    // ... and what it adds to: columns n + 4 r .. of rows 4 g + i
    typename Held<F16>::type cnext[4];
    auto start = [&]() -> bool {
        if (!next()) return false;
        const int col = n + 4 * r;
#pragma unroll
        for (int i = 0; i < 4; i++)
            cnext[i] = load_c<F16>(a, (t0 + 4 * g + i) * a.ldc + w.at + col, (rows >> (4 * g + i)) & 1 ? n1 - col : 0);
        if (ranks > 0) fetch(0);
        return true;
    };
    bool more = start();

    {
        const int row = tid / PER, mr = __shfl(rk, row);
        const float scale = __shfl(sc, row);
        const int shift = split_row<PER>(ws + ((int64_t)part * p.pieces * a.T + t0 + row) * a.rank, (int64_t)a.T * a.rank, p.pieces, mr,
                                         tid % PER, padded, [&](int k, uint2 hi, uint2 lo) {
                                             *(uint2*)(sums + row * ld + k) = hi;
                                             *(uint2*)(sums + (ROWS + row) * ld + k) = lo;
                                         });
        if (tid % PER == 0) factor[row] = __builtin_ldexpf(scale, -shift);
    }
    __syncthreads();

    while (more) {
        // this pair; the next one's block comes while this one's products run
        const int cn = n, cr = ranks;
        const uint64_t crows = rows;
        const int col = cn + 4 * r, inside = n1 - col;                     // the lane's four columns, of rows 4 g + i
        typename Held<F16>::type c[4];
#pragma unroll
        for (int i = 0; i < 4; i++) c[i] = cnext[i];
        f4 acc[4];
#pragma unroll
        for (int j = 0; j < 4; j++) acc[j] = f4{0.f, 0.f, 0.f, 0.f};
        for (int k0 = 0; k0 < cr; k0 += RC) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
            for (int s = 0; s < KS; s++) {
                if (k0 + 32 * s >= cr) break;
                const _Float16* const v = sums + r * ld + k0 + 32 * s + 8 * g;
                const h8 hi = *(const h8*)v, lo = *(const h8*)(v + ROWS * ld);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const h8 b = block_at<RC, 2>(block, 4 * r + j, k0, 32 * s + 8 * g, cr);   // operand j: columns 4 i + j
                    acc[j] = mfma16x16x32(hi, b, acc[j]);
                    acc[j] = mfma16x16x32(lo, b, acc[j]);
                }
            }
            if (k0 + RC < cr) fetch(k0 + RC);
            else more = start();
        }
        if (cr == 0) more = start();
        if (cr == 0 && a.Y == a.C) continue;       // (no adapter, in place)
        const f4 f = factor4[g];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (cr > 0) c[i] = add(c[i], f[i], f4{acc[0][i], acc[1][i], acc[2][i], acc[3][i]});   // (no adapter: a copy, through no arithmetic)
            store_y<F16>(a, (t0 + 4 * g + i) * a.ldy + w.at + col, c[i], (crows >> (4 * g + i)) & 1 ? inside : 0);
        }
    }
}

// Many rows: a workgroup takes a tile of 64 rows of one adapter by 256 columns, wave w
// rows 16 (w % 4) .. and columns 128 (w / 4) .. of those.  Operand j of its eight holds
// the columns that leave a lane 16 neighbouring bytes of a row of C (8 i + j in fp16, 64
// (j / 4) + 4 i + j % 4 in fp32), so that a wave reads and writes runs of 256 bytes
// (128-byte runs of 8-byte pieces: 25 us where this took 15).  JOIN: the pieces' sums are
// joined here, for ranks that are one block; else k_lora_join did it.  Three workgroups a
// CU where registers allow it without going to memory (2000 rows, rank 16: 25.5 us for all,
// with two 27.0; rank 64, whose sums need more: 44 with three, 38 with two).
template <int RC, bool F16, bool JOIN>
__global__ __launch_bounds__(64 * kLoraUpWaves, RC < 64 && F16 ? 6 : 4) void k_lora_up_many(LoraArgs a, LoraPlan p, float* __restrict__ ws) {
    constexpr int WV = kLoraUpWaves, ROWS = 64, COLS = 128, PIECES = RC / 8, KS = (RC + 31) / 32, BYTES = 2 * COLS * RC;
    constexpr int SH = F16 ? 3 : 2, PER = F16 ? 1 : 2, W = F16 ? 8 : 4;    // runs of a lane in a row, their columns
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * BYTES + 2 * 2 * ROWS * RC];   // two blocks of B, the sums' hi and lo
    __shared__ float factor[ROWS];
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), sub = wave & 3;
    LoraTile o;
    const int* rows;
    int at;
    if (!tile_of(p, p.up, ws, o, rows, at)) return;
    const int ranks = o.ranks;
    if (ranks == 0 && a.Y == a.C) return;          // (no adapter, in place)
    const int part = part_of(a, p.up_steps, at);
    const LoraPart& w = a.part[part];
    const int n = at * p.up_steps * kLoraCols + COLS * (wave >> 2), col = n + W * r;         // (the lane's second run: col + 64)
    const int t = rows[min(lane, o.rows - 1)];                // lane l: the tile's row l
    const Joined sums = joined_of(a, p, ws);
    uint8_t* const block = lds + (wave >> 2) * BYTES;
    uint8_t* const rows_lds = lds + 2 * BYTES;                             // [hi, lo][64 rows][RC]

    // the wave's quarter of its block: ranks k0 .., as far as they count; and its share of the sums
    auto fetch = [&](int k0) {
        const uint16_t* const B = w.B + (int64_t)o.adapter * w.N * a.rank;
#pragma unroll
        for (int i = 0; i < PIECES / 2; i++) {
            const int m = 4 * i + sub, q = 64 * m + lane, c = q / PIECES, k = k0 + 8 * place<RC, SH>(c, q % PIECES);
            if (k < ranks) dma16(B + (int64_t)min(n + c, w.N - 1) * a.rank + k, lds_addr(block) + 1024 * m);
        }
        if (JOIN) return;
#pragma unroll
        for (int i = 0; i < (2 * PIECES + WV - 1) / WV; i++) {             // (of both planes)
            const int m = WV * i + wave;
            if (m >= 2 * PIECES) break;
            const int q = 64 * (m % PIECES) + lane, row = q / PIECES, k = k0 + 8 * place<RC, 0>(row, q % PIECES);
            const _Float16* const s = (m < PIECES ? sums.hi : sums.lo) + ((int64_t)part * a.T + __shfl(t, row)) * p.padded;
            if (k < p.padded) dma16(s + k, lds_addr(rows_lds) + 1024 * m);
        }
    };
    if (ranks > 0) fetch(0);
    f4 acc[8];
#pragma unroll
    for (int j = 0; j < 8; j++) acc[j] = f4{0.f, 0.f, 0.f, 0.f};
    if (ranks > 0) {
        if (JOIN) {
            const int row = tid / 8, mr = row < o.rows ? ranks : 0;
            const int shift = split_row<8>(ws + ((int64_t)part * p.pieces * a.T + __shfl(t, row)) * a.rank, (int64_t)a.T * a.rank,
                                           p.pieces, mr, tid % 8, RC, [&](int k, uint2 hi, uint2 lo) {
                                               uint8_t* const to = rows_lds + row * (2 * RC) + 16 * place<RC, 0>(row, k / 8) + 2 * (k & 7);
                                               *(uint2*)to = hi;
                                               *(uint2*)(to + 2 * ROWS * RC) = lo;
                                           });
            if (tid % 8 == 0) factor[row] = __builtin_ldexpf(a.scales ? a.scales[o.adapter] : 1.f, -shift);
        } else if (tid < ROWS) {
            factor[tid] = sums.factor[(int64_t)part * a.T + t];
        }
        for (int k0 = 0; k0 < ranks; k0 += RC) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            if (16 * sub < o.rows) {
                const int row = 16 * sub + r;
#pragma unroll
                for (int s = 0; s < KS; s++) {
                    if (k0 + 32 * s >= ranks) break;
                    const int k = 32 * s + 8 * g;
                    h8 v[2];
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        v[h] = *(const h8*)(rows_lds + (h * ROWS + row) * (2 * RC) + 16 * place<RC, 0>(row, (k / 8) & (PIECES - 1)));
                        if (RC < 32) v[h] = masked(v[h], k < RC);
                    }
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const h8 b = block_at<RC, SH>(block, F16 ? 8 * r + j : 64 * (j >> 2) + 4 * r + (j & 3), k0, k, ranks);
                        acc[j] = mfma16x16x32(v[0], b, acc[j]);
                        acc[j] = mfma16x16x32(v[1], b, acc[j]);
                    }
                }
            }
            if (k0 + RC < ranks) {
                __syncthreads();                   // the blocks have been read
                fetch(k0 + RC);
            }
        }
    }
    typename Run<F16>::type c[4][PER];             // what is added to, of rows 16 sub + 4 g + i
    int64_t tr[4];
    bool in[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        tr[i] = __shfl(t, 16 * sub + 4 * g + i);
        in[i] = 16 * sub + 4 * g + i < o.rows;
#pragma unroll
        for (int h = 0; h < PER; h++)
            c[i][h] = load_run<F16>(a, tr[i] * a.ldc + w.at + col + 64 * h, in[i] ? w.N - col - 64 * h : 0);
    }
    f4 f = f4{0.f, 0.f, 0.f, 0.f};
    if (ranks > 0) f = *(const f4*)(factor + 16 * sub + 4 * g);
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int h = 0; h < PER; h++) {
            typename Run<F16>::type y = c[i][h];
            if (ranks > 0) {                       // (no adapter: a copy, through no arithmetic)
                float d[W];
#pragma unroll
                for (int j = 0; j < W; j++) d[j] = acc[4 * h + j][i];
                y = add_run(y, f[i], d);
            }
            store_run<F16>(a, tr[i] * a.ldy + w.at + col + 64 * h, y, in[i] ? w.N - col - 64 * h : 0);
        }
}

template <class K> hipError_t raise_lds(K k, std::atomic<uint64_t>& set, int bytes) {
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (set.load(std::memory_order_acquire) & bit) return hipSuccess;
    e = hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == hipSuccess) set.fetch_or(bit, std::memory_order_acq_rel);
    return e;
}

template <int NT> hipError_t down(const LoraArgs& a, const LoraPlan& p, float* ws, hipStream_t st) {
    constexpr int few = kLoraDownWaves * 2 * kUnitBytes<NT>, many = 2 * kLoraSlab / kLoraUnit * NT * 2048;
    static std::atomic<uint64_t> set{0}, set_many{0};                      // one bit per device: LDS limit raised
    auto k = p.many ? k_lora_down_many<NT> : k_lora_down<NT>;
    const int lds = p.many ? many : few;
    const hipError_t e = raise_lds(k, p.many ? set_many : set, lds);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(k, dim3((unsigned)p.down.groups), dim3(64 * (p.many ? kLoraManyWaves : kLoraDownWaves)), lds, st, a, p, ws);
    return hipGetLastError();
}

template <int RC, bool F16> hipError_t up_few(const LoraArgs& a, const LoraPlan& p, const float* ws, hipStream_t st) {
    constexpr int WV = kLoraUpWaves, blocks = WV * 2 * kLoraCols * RC;
    const auto sums = [](int rank) { return 4 * kLoraSub * lora_lds_ranks(rank); };
    static std::atomic<uint64_t> set{0};
    auto k = k_lora_up<RC, F16>;
    const hipError_t e = raise_lds(k, set, blocks + sums(RC < 64 ? RC : kLoraMaxRank));
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(k, dim3((unsigned)p.up.groups), dim3(64 * WV), (size_t)(blocks + sums(a.rank)), st, a, p, ws);
    return hipGetLastError();
}

template <int RC, bool F16, bool JOIN> hipError_t up_many(const LoraArgs& a, const LoraPlan& p, float* ws, hipStream_t st) {
    if (!JOIN) {
        hipLaunchKernelGGL(k_lora_join, dim3((unsigned)((a.T + kJoinRows - 1) / kJoinRows), (unsigned)a.parts), dim3(16 * kJoinRows), 0, st,
                           a, p, ws);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((k_lora_up_many<RC, F16, JOIN>), dim3((unsigned)p.up.groups), dim3(64 * kLoraUpWaves), 0, st, a, p, ws);
    return hipGetLastError();
}

template <int RC, bool F16> hipError_t up(const LoraArgs& a, const LoraPlan& p, float* ws, hipStream_t st) {
    if (!p.many) return up_few<RC, F16>(a, p, ws, st);
    if constexpr (RC == 64) {
        if (a.rank > RC) return up_many<RC, F16, false>(a, p, ws, st);
    }
    return up_many<RC, F16, true>(a, p, ws, st);
}

hipError_t order(const LoraArgs& a, const LoraPlan& p, float* ws, hipStream_t st) {
    hipLaunchKernelGGL(k_lora_order, dim3(1), dim3(kOrderThreads), 0, st, a, p, ws);
    return hipGetLastError();
}

template <int RC> hipError_t both(const LoraArgs& a, const LoraPlan& p, float* ws, hipStream_t st) {
    hipError_t e = p.many ? order(a, p, ws, st) : hipSuccess;
    if (e == hipSuccess) e = down<RC / 16>(a, p, ws, st);
    if (e != hipSuccess) return e;
    return a.out_f16 ? up<RC, true>(a, p, ws, st) : up<RC, false>(a, p, ws, st);
}

int cus() { return device_cus() > 0 ? device_cus() : 256; }
LoraPlan plan_of(const LoraArgs& a) { return plan_lora(a, cus()); }

}  // namespace

bool lora_fits(const LoraArgs& a) {
    const LoraPlan p = plan_of(a);
    return launch_fits(p.down.groups, 64 * kLoraManyWaves) && launch_fits(p.up.groups, 64 * kLoraUpWaves) && launch_fits(a.T, 16);
}

size_t lora_scratch_bytes(const LoraArgs& a) { return lora_reserve(a, plan_of(a), cus()); }

hipError_t lora(const LoraArgs& a, float* ws, hipStream_t st) {
    const LoraPlan p = plan_of(a);
    switch (lora_block(a.rank)) {
        case 16: return both<16>(a, p, ws, st);
        case 32: return both<32>(a, p, ws, st);
        default: return both<64>(a, p, ws, st);
    }
}

}  // namespace bf
