// The experts' products for prompts: k_moe_tile, the tile of the prefill GEMM
// (bf_tile.h) over rows gathered by expert.
//
// An expert's slots are cut into runs of 256 (of 64 where experts have few: the
// caller's rule, k_moe_tile64).  Whole runs, and a rest of more
// than 192, take a large tile, 256 rows x 256 weight rows (NB = 2 of bf_tile.h);
// a shorter rest a small one, 64, 128 or 192 rows x 128 weight rows.  Activation
// rows are fetched through the slot list, row by row, by the direct-to-LDS
// loads' own per-lane addresses, so nothing is gathered beforehand.
//
// Gate and up: a tile's weight rows are 32 gate rows, the same 32 up rows, and
// the next 32 of both, which puts g and u of one output into the two column
// tiles of one wave: h = SiLU(g) u leaves the registers as the one fp16 row
// that the down product reads.  (Small tiles: two k groups of waves hold half of
// each sum; each hands the other half of the rows over and finishes the rest.)
//
// 2000 rows of eight, 64 experts of 4096 x 1792 (Q4_0): gate and up 575 us, 820
// TFLOP/s, down 312, 750; the prefill GEMM with whole tiles only reaches 950.  A third
// of the experts have a few rows more than 256, whose small tiles decode as many
// weights as a full one, and the last round of large tiles is half empty.  Matrix
// units 42 to 47 % busy, vector instructions 27 %.
#include <algorithm>
#include <atomic>

#include "bf_moe_dev.h"
#include "bf_tile.h"

namespace bf {
namespace {

// One output pair of a lane: columns c (tile 0) and c + 32 (tile 1) of the wave's 64.
template <bool GU>
__device__ __forceinline__ void put(const MoeArgs& a, const MoeTileArgs& o, int slot, int c64, int lane, float y0, float y1) {
    if constexpr (GU) {
        const float ex = __builtin_amdgcn_exp2f(y0 * -1.44269504088896341f);
        ((_Float16*)o.out)[(int64_t)slot * o.R + c64 / 2 + (lane & 31)] =
            (_Float16)(y0 * __builtin_amdgcn_rcpf(1.0f + ex) * y1 * weight_in_h(a.w[slot]));
    } else {
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const int n = c64 + 32 * b + (lane & 31);
            const int64_t at = (int64_t)slot * o.R + n;
            if (n >= o.R) continue;
            store_y(a, o.out, at, b ? y1 : y0);
        }
    }
}

// Output pairs of a lane in rows r .. r + 3 of the tile.  y: lane q of four takes
// row r + q and the four's columns (a lane storing its own column, a row at a
// time, takes four times the stores: 1015 us the whole block where this takes 963, 2000
// rows of eight, 64 experts of 4096 x 1792).
template <bool GU>
__device__ __forceinline__ void put4(const MoeArgs& a, const MoeTileArgs& o, const int32_t* list, int r, int rows, int c64, int lane,
                                     const float (&y)[2][4]) {
    if (GU || o.R % 4) {
#pragma unroll
        for (int c = 0; c < 4; c++)
            if (r + c < rows) put<GU>(a, o, list[r + c], c64, lane, y[0][c], y[1][c]);
        return;
    }
    const int row = r + (lane & 3);
    const int64_t slot = list[min(row, rows - 1)];
#pragma unroll
    for (int b = 0; b < 2; b++) {
        uint32_t u[4];
#pragma unroll
        for (int c = 0; c < 4; c++) u[c] = y_24(a) ? round24(y[b][c]) : __builtin_bit_cast(uint32_t, y[b][c]);
        transpose4(u, lane);
        const int n = c64 + 32 * b + (lane & 28);
        if (row < rows && n < o.R) store_y4(a, o.out, slot * o.R + n, u);
    }
}

// The outputs of a tile: run() of bf_tile.h, then the epilogue above.
template <int QT, int TA, int NB, bool GU>
__device__ __forceinline__ void moe_tile(uint8_t* lds, const MoeArgs& a, const MoeTileArgs& o, const int32_t* list, int rows,
                                         int64_t e, int ni) {
    using T = Tile<QT, TA, NB>;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    T t;
    t.rsrc = u4{(uint32_t)(uintptr_t)o.A, (uint32_t)((uintptr_t)o.A >> 32) & 0xFFFFu, o.a_bytes, 0x00020000u};
#pragma unroll
    for (int q = 0; q < TA; q++) {
        const int slot = list[min(8 * (wave + 8 * q) + (lane >> 3), rows - 1)];
        t.voff[q] = (uint32_t)(GU ? slot / a.k : slot) * (uint32_t)o.lda * 2u +
                    16u * (((uint32_t)lane & 7u) ^ (4u * (wave & 1) + (lane >> 4)));
    }
    t.lds0 = lds_addr(lds);
    t.wave = wave;
    constexpr int TPR = 4 / NB;                    // threads of a weight row
    t.j = threadIdx.x % TPR;
    const int wr = threadIdx.x / TPR;
    // tile column -> weight row: GU 64 outputs of gate and up, 32 and 32 in turn
    const int f = GU ? T::BN / 2 * ni + 32 * (wr >> 6) + (wr & 31) : T::BN * ni + wr;
    const bool up = GU && (wr & 32);
    const int64_t n = e * o.R + min(f, o.R - 1);
    t.row = (up ? o.W[1] : o.W[0]) + n * row_bytes(QT, o.K);
    t.aux = QT == QT_PLANES ? (up ? o.aux[1] : o.aux[0]) + n * (o.K >> 4) : nullptr;
    t.wst = T::kAStage + wr * 128 + 16 * (tile_chunk<QT, NB>(t.j, 0) ^ ((wr >> 1) & 7));
    const int kg = NB == 1 ? wave >> 2 : 0, wm = NB == 1 ? (wave >> 1) & 1 : wave >> 2, wn = wave & (2 * NB - 1);
    const uint32_t fr = (lane & 31) * 128 + 16 * ((4 * kg + (lane >> 5)) ^ ((lane >> 1) & 7));
    t.fa = wm * (32 * TA * 128) + fr;
    t.fw = T::kAStage + wn * (64 * 128) + fr;
    t.mg = make_magic();
#pragma unroll
    for (int i = 0; i < TA; i++)
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int x = 0; x < 16; x++) t.acc[i][b][x] = 0.f;
    t.run(lds, 0, o.K >> 8);

    const int c64 = T::BN * ni + 64 * wn;
    if constexpr (NB == 2) {
#pragma unroll
        for (int i = 0; i < TA; i++)
#pragma unroll
            for (int x = 0; x < 16; x += 4) {
                const f16x &v = t.acc[i][0], &w = t.acc[i][1];
                put4<GU>(a, o, list, 32 * TA * wm + 32 * i + 2 * x + 4 * (lane >> 5), rows, c64, lane,
                         {{v[x], v[x + 1], v[x + 2], v[x + 3]}, {w[x], w[x + 1], w[x + 2], w[x + 3]}});
            }
        return;
    }

    // Group kg finishes accumulator registers 8 kg .. 8 kg + 7 of every tile.
    uint8_t* const xch = lds + (threadIdx.x & 255) * 16;
    constexpr int XB = TA * 4 * 4096;
#pragma unroll
    for (int i = 0; i < TA; i++)
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int x = 0; x < 8; x += 4) {
                const f16x& v = t.acc[i][b];
                *(f4*)(xch + kg * XB + ((i * 2 + b) * 2 + x / 4) * 4096) =
                    kg ? f4{v[x], v[x + 1], v[x + 2], v[x + 3]} : f4{v[8 + x], v[9 + x], v[10 + x], v[11 + x]};
            }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TA; i++)
#pragma unroll
        for (int x = 0; x < 8; x += 4) {
            float y[2][4];
#pragma unroll
            for (int b = 0; b < 2; b++) {
                const f4 p = *(const f4*)(xch + (1 - kg) * XB + ((i * 2 + b) * 2 + x / 4) * 4096);
                const f16x& v = t.acc[i][b];
#pragma unroll
                for (int c = 0; c < 4; c++) y[b][c] = kg ? p[c] + v[8 + x + c] : v[x + c] + p[c];
            }
            put4<GU>(a, o, list, 32 * TA * wm + 32 * i + 16 * kg + 2 * x + 4 * (lane >> 5), rows, c64, lane, y);
        }
}

template <int QT, bool GU>
__global__ __launch_bounds__(kTlThreads) __attribute__((amdgpu_waves_per_eu(2, 2)))
void k_moe_tile(MoeArgs a, MoeTileArgs o) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    // large tiles first, so that the small ones fill the last round
    const int large = o.tiles[0] * o.nt[0], units = large + o.tiles[1] * o.nt[1];
    if ((int)blockIdx.x >= units) return;
    const bool big = (int)blockIdx.x < large;
    const int v = big ? xcd_unit((int)blockIdx.x, large) : xcd_unit((int)blockIdx.x - large, units - large);
    const int nt = big ? o.nt[0] : o.nt[1], i = v / nt, ni = v - i * nt;
    const int4 d = o.table[(big ? 0 : o.max_tiles) + i];
    const int e = __builtin_amdgcn_readfirstlane(d.x), rows = __builtin_amdgcn_readfirstlane(d.z);
    const int32_t* list = o.perm + __builtin_amdgcn_readfirstlane(d.y);
    if (big) moe_tile<QT, 4, 2, GU>(lds, a, o, list, rows, e, ni);
    else if (rows > 192) moe_tile<QT, 4, 1, GU>(lds, a, o, list, rows, e, ni);
    else if (rows > 128) moe_tile<QT, 3, 1, GU>(lds, a, o, list, rows, e, ni);
    else if (rows > 64) moe_tile<QT, 2, 1, GU>(lds, a, o, list, rows, e, ni);
    else moe_tile<QT, 1, 1, GU>(lds, a, o, list, rows, e, ni);
}

// Runs of 64 rows only, with the registers and LDS of two workgroups a CU: their
// weights are decoded once a run as well, which a CU alone with eight waves waits for.
template <int QT, bool GU>
__global__ __launch_bounds__(kTlThreads) __attribute__((amdgpu_waves_per_eu(4, 4)))
void k_moe_tile64(MoeArgs a, MoeTileArgs o) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int units = o.tiles[1] * o.nt[1];
    if ((int)blockIdx.x >= units) return;
    const int v = xcd_unit((int)blockIdx.x, units), i = v / o.nt[1];
    const int4 d = o.table[o.max_tiles + i];
    moe_tile<QT, 1, 1, GU>(lds, a, o, o.perm + __builtin_amdgcn_readfirstlane(d.y), __builtin_amdgcn_readfirstlane(d.z),
                           __builtin_amdgcn_readfirstlane(d.x), v - i * o.nt[1]);
}

template <int QT, bool GU, bool SMALL>
hipError_t launch(const MoeArgs& a, const MoeTileArgs& o, hipStream_t st) {
    using T1 = Tile<QT, 1, 1>;
    auto k = SMALL ? k_moe_tile64<QT, GU> : k_moe_tile<QT, GU>;
    constexpr int lds = SMALL ? T1::NS * T1::kStage
                              : std::max(Tile<QT, 4, 1>::NS * Tile<QT, 4, 1>::kStage, Tile<QT, 4, 2>::NS * Tile<QT, 4, 2>::kStage);
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
    hipLaunchKernelGGL(k, dim3((unsigned)((int64_t)o.max_tiles * o.nt[1])), dim3(kTlThreads), lds, st, a, o);
    return hipGetLastError();
}

template <int QT>
hipError_t dispatch(const MoeArgs& a, const MoeTileArgs& o, bool gu, hipStream_t st) {
    if (o.run != kMoeTileRows) return gu ? launch<QT, true, true>(a, o, st) : launch<QT, false, true>(a, o, st);
    return gu ? launch<QT, true, false>(a, o, st) : launch<QT, false, false>(a, o, st);
}

}  // namespace

hipError_t moe_tile(const MoeArgs& a, const MoeTileArgs& o, bool gu, hipStream_t st) {
    if (a.qtype == QT_PLANES) return dispatch<QT_PLANES>(a, o, gu, st);
    if (a.qtype == QT_Q4_0) return dispatch<QT_Q4_0>(a, o, gu, st);
    return dispatch<QT_Q4_K>(a, o, gu, st);
}

}  // namespace bf
