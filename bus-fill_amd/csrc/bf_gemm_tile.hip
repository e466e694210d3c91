// Tiled MFMA GEMM for prefill batches (more than 128 rows): k_gemm_tile.
//
//   C[m][n] = sum_k A[m][k] * dequant(W)[n][k]      (fp32 accumulation)
//
// Above 128 rows the dense kernel runs one launch per 128 rows, and each of
// them streams and decodes every weight again (17408 x 5120 at 2000 rows:
// 16 launches, 609-648 us, 545-585 TFLOP/s).  Here a workgroup computes a tile
// of up to 256 batch rows x 256 weight rows, K in steps of 64: both operands
// of a step sit in LDS as fp16, so a weight is decoded once per 256 rows and
// read from LDS by the waves of every column of the tile.
//
// * Eight waves, two per SIMD, 32 TA x 64 outputs each (TA x 2 tiles of
//   v_mfma_f32_32x32x16_f16: TA + 2 LDS reads feed 2 TA MFMAs).  NB = 2: 2 x 4
//   waves over a 256 x 256 tile.  NB = 1: 2 x 2 waves over a 64 TA x 128 tile,
//   twice, each set multiplying half of every step (their sums meet in LDS at
//   the end): the same reads per MFMA where 256 x 256 tiles leave CUs idle.
// * Activations: direct-to-LDS loads, one or two steps ahead (NS stages).
//   Weights: the quantized words in registers, loaded one super-group (four
//   steps) ahead, decoded to fp16 and written to the next step's stage.
// * One barrier per step.  A slot's fragments (16 k) are read from LDS while
//   the previous slot's multiply, across the barrier too, so the MFMAs never
//   wait for the LDS reads they use; the DMA instructions and the decode are
//   spread between the MFMAs, for one wave's issue stalls beside the other's
//   MFMAs (all of a step's DMA at its start: 388 us where spread takes 356,
//   2048 x 16384 x 5120).
// * LDS rows are 128 bytes (64 k); their 16-byte chunk c sits at c ^ ((row / 2)
//   % 8), so the 32 rows of a fragment read fall on distinct banks.
// * Bound by neither the matrix cores' rate nor the clock alone: MFMAs take
//   57-61 % of the SIMD cycles at 1.6-1.7 GHz with NB = 2 (2048 x 16384 x 5120:
//   328-336 us, 1020-1050 TFLOP/s) and 43-47 % at 1.9-2.0 GHz with NB = 1 (512 x
//   16384 x 5120: 93-97 us); an 8192^3 bf16 library product reached 1211 TFLOP/s on
//   such a chip, a library fp16 product of the first size takes 386-395 us on
//   decoded weights.  The compiler's own waits for the weight words count the DMAs
//   too (vmcnt(3) to vmcnt(6) once per step; planes, whose scales are copied while
//   fresh, vmcnt(0) once per super-group): stricter than the data needs, and not
//   yet taken out.  NB = 2 halves the operand traffic per flop of NB = 1 (2048
//   rows: 356 -> 327-340 us).
// * Measured (Q4_K, us per GEMM, before -> after): 17408 x 5120 at 512 / 2000
//   rows 150-165 / 609-648 -> 108 / 355-369; 5120 x 17408 at 2000 rows
//   572-606 -> 348-359; 5120 x 5120 at 300 / 512 rows 52-58 / 76-80 -> 35 / 43.
#include <atomic>

#include "bf_launch.h"
#include "bf_tile.h"

namespace bf {
namespace {

// Workgroups [0, F): whole tiles, straight to C.  Workgroups F ..: the R =
// tiles - F remaining ones, each cut in S ranges of super-groups whose sums go
// to the workspace ([split][tile][row][128 NB] fp32; S > 1) for k_tile_sum.
template <int QT, int TA, int NB>
__global__ __launch_bounds__(kTlThreads) __attribute__((amdgpu_waves_per_eu(2, 2)))
void k_gemm_tile(const uint8_t* W, const uint8_t* Waux, const uint16_t* A, int lda, void* C, int ldc, int out_f16,
                 int M, int N, int K, int mt, int F, int R, int S, float* ws) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    using T = Tile<QT, TA, NB>;
    constexpr int BM = T::BM, BN = T::BN;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nsg = K >> 8;
    int tile, sp = 0, s0 = 0, s1 = nsg;
    if ((int)blockIdx.x < F) {
        tile = xcd_unit((int)blockIdx.x, F);
    } else {
        const int v = xcd_unit((int)blockIdx.x - F, R * S);
        sp = v / R;
        tile = F + v - sp * R;
        s0 = sp * nsg / S;
        s1 = (sp + 1) * nsg / S;
    }
    int mi, ni;
    tile_at(tile, mt, (N + BN - 1) / BN, mi, ni);
    const int m0 = mi * BM, n0 = ni * BN;
    const int rows = min(BM, M - m0);

    T t;
    const uint16_t* const a0 = A + (int64_t)m0 * lda;
    t.rsrc = u4{(uint32_t)(uintptr_t)a0, (uint32_t)((uintptr_t)a0 >> 32) & 0xFFFFu,
                (uint32_t)(((int64_t)(rows - 1) * lda + K) * 2), 0x00020000u};
#pragma unroll
    for (int q = 0; q < TA; q++) {
        const int r = min(8 * (wave + 8 * q) + (lane >> 3), rows - 1);
        t.voff[q] = (uint32_t)r * (uint32_t)lda * 2u + 16u * (((uint32_t)lane & 7u) ^ (4u * (wave & 1) + (lane >> 4)));
    }
    t.lds0 = lds_addr(lds);
    t.wave = wave;
    constexpr int TPR = 4 / NB;                        // threads of a weight row
    t.j = threadIdx.x % TPR;
    const int wr = threadIdx.x / TPR;
    const int64_t n = min(n0 + wr, N - 1);
    t.row = W + n * row_bytes(QT, K);
    t.aux = QT == QT_PLANES ? Waux + n * (K >> 4) : nullptr;
    t.wst = T::kAStage + wr * 128 + 16 * (tile_chunk<QT, NB>(t.j, 0) ^ ((wr >> 1) & 7));
    const int kg = NB == 1 ? wave >> 2 : 0, wm = NB == 1 ? (wave >> 1) & 1 : wave >> 2, wn = wave & (2 * NB - 1);
    const uint32_t f = (lane & 31) * 128 + 16 * ((4 * kg + (lane >> 5)) ^ ((lane >> 1) & 7));
    t.fa = wm * (32 * TA * 128) + f;
    t.fw = T::kAStage + wn * (64 * 128) + f;
    t.mg = make_magic();
#pragma unroll
    for (int a = 0; a < TA; a++)
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int e = 0; e < 16; e++) t.acc[a][b][e] = 0.f;
    t.run(lds, s0, s1);

    // Outputs of the wave: rows mr + (8 (e / 4) + e % 4) of every 32-row tile,
    // column nn (+ 32 b).
    const int nc = n0 + 64 * wn + (lane & 31), mr = 32 * TA * wm + 4 * (lane >> 5);
    const bool part = (int)blockIdx.x >= F && S > 1;
    float* const pw = ws + (size_t)(sp * R + tile - F) * (BM * BN) + (size_t)mr * BN + (nc - n0);
    auto store = [&](int dm, int b, float y) {
        const int m = m0 + mr + dm, nn = nc + 32 * b;
        if (m >= M) return;
        if (part) {
            pw[(size_t)dm * BN + 32 * b] = y;
        } else if (nn < N) {
            const int64_t o = (int64_t)m * ldc + nn;
            if (out_f16) ((_Float16*)C)[o] = (_Float16)y;
            else ((float*)C)[o] = y;
        }
    };
    if constexpr (NB == 2) {
#pragma unroll
        for (int a = 0; a < TA; a++)
#pragma unroll
            for (int e = 0; e < 16; e++)
#pragma unroll
                for (int b = 0; b < 2; b++) store(32 * a + 8 * (e / 4) + e % 4, b, t.acc[a][b][e]);
    } else {
        // The two k groups' sums: wave (kg, wm, wn) hands the column tile 1 - kg
        // to its partner and finishes column tile kg.
        uint8_t* const xch = lds + (threadIdx.x & 255) * 16;
        constexpr int XB = TA * 4 * 4096;              // bytes handed over by one k group
#pragma unroll
        for (int a = 0; a < TA; a++)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const f16x& v = kg ? t.acc[a][0] : t.acc[a][1];
                *(f4*)(xch + kg * XB + (a * 4 + e / 4) * 4096) = f4{v[e], v[e + 1], v[e + 2], v[e + 3]};
            }
        __syncthreads();
#pragma unroll
        for (int a = 0; a < TA; a++)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const f4 x = *(const f4*)(xch + (1 - kg) * XB + (a * 4 + e / 4) * 4096);
                const f16x& v = kg ? t.acc[a][1] : t.acc[a][0];
#pragma unroll
                for (int i = 0; i < 4; i++) store(32 * a + 2 * e + i, kg, kg ? x[i] + v[e + i] : v[e + i] + x[i]);
            }
    }
}

// C of the cut tiles: their S partial sums in split order.  Block (r, y):
// 1024 / BN rows of the r-th cut tile, four columns per thread.
template <int BM, int BN>
__global__ __launch_bounds__(256) void k_tile_sum(const float* __restrict__ ws, void* __restrict__ C, int ldc,
                                                  int out_f16, int M, int N, int mt, int F, int R, int S) {
    constexpr int Q = BN / 4;                          // column quads of a row
    const int r = (int)blockIdx.x, tile = F + r;
    int mi, ni;
    tile_at(tile, mt, (N + BN - 1) / BN, mi, ni);
    const int dm = 256 / Q * (int)blockIdx.y + (int)threadIdx.x / Q, m = mi * BM + dm, nl = 4 * ((int)threadIdx.x % Q);
    if (m >= M) return;
    const float* p = ws + (size_t)r * (BM * BN) + (size_t)dm * BN + nl;
    const size_t ps = (size_t)R * (BM * BN);
    f4 s = f4{0.f, 0.f, 0.f, 0.f};
    for (int q0 = 0; q0 < S; q0 += 8) {
        f4 x[8];
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = q0 + k < S ? *(const f4*)(p + (q0 + k) * ps) : f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (q0 + k < S) s += x[k];
    }
    const int64_t n0 = (int64_t)ni * BN + nl, o = (int64_t)m * ldc + n0;
    if (((uintptr_t)C & 15) == 0 && (ldc & 3) == 0 && n0 + 3 < N) {
        if (out_f16) {
            typedef _Float16 h4 __attribute__((ext_vector_type(4)));
            *(h4*)((_Float16*)C + o) = h4{(_Float16)s[0], (_Float16)s[1], (_Float16)s[2], (_Float16)s[3]};
        } else {
            *(f4*)((float*)C + o) = s;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (n0 + i >= N) break;
            if (out_f16) ((_Float16*)C)[o + i] = (_Float16)s[i];
            else ((float*)C)[o + i] = s[i];
        }
    }
}

bool plan_of(const GemmArgs& g, TilePlan& p) {
    if ((int64_t)g.lda >= (1 << 22)) return false;     // activation offsets of a tile in 32 bits
    // a caller's workspace of the size that 128-row launches of the dense kernel
    // take on this matrix serves here too
    GemmArgs slice = g;
    slice.M = 128;
    const size_t scratch = dense_supports(slice) ? dense_scratch_bytes(slice) : 0;
    return plan_tile(g.M, g.N, g.K, device_cus() > 0 ? device_cus() : 256, scratch, p);
}

template <int QT, int TA, int NB>
hipError_t launch_tile(const GemmArgs& g, const TilePlan& p, const Scratch* scratch, hipStream_t st) {
    using T = Tile<QT, TA, NB>;
    auto k = k_gemm_tile<QT, TA, NB>;
    constexpr int lds = T::NS * T::kStage;
    static std::atomic<uint64_t> attr_set{0};          // one bit per device: LDS limit raised
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (!(attr_set.load(std::memory_order_acquire) & bit)) {
        e = hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return e;
        attr_set.fetch_or(bit, std::memory_order_acq_rel);
    }
    unsigned* counters = nullptr;
    float* parts = nullptr;
    if (p.part) {
        e = split_workspace(scratch, st, 0, p.part, &counters, &parts);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(k, dim3(p.F + p.R * p.S), dim3(kTlThreads), lds, st, g.W, g.Waux, g.A, g.lda, g.C, g.ldc,
                       g.out_f16, g.M, g.N, g.K, p.mt, p.F, p.R, p.S, parts);
    e = hipGetLastError();
    if (e != hipSuccess || !p.part) return e;
    hipLaunchKernelGGL((k_tile_sum<T::BM, T::BN>), dim3(p.R, T::BM * T::BN / 1024), dim3(256), 0, st, (const float*)parts,
                       g.C, g.ldc, g.out_f16, g.M, g.N, p.mt, p.F, p.R, p.S);
    return hipGetLastError();
}

template <int QT>
hipError_t dispatch_tile(const GemmArgs& g, const TilePlan& p, const Scratch* scratch, hipStream_t st) {
    if (p.NB == 2) return launch_tile<QT, 4, 2>(g, p, scratch, st);
    if (p.TA == 2) return launch_tile<QT, 2, 1>(g, p, scratch, st);
    if (p.TA == 3) return launch_tile<QT, 3, 1>(g, p, scratch, st);
    return launch_tile<QT, 4, 1>(g, p, scratch, st);
}

}  // namespace

bool tile_supports(const GemmArgs& g) {
    TilePlan p;
    if (!plan_of(g, p)) return false;
    GemmArgs slice = g;
    slice.M = 128;
    return !(dense_supports(slice) &&
             slices_faster(g.M, g.N, g.K, device_cus() > 0 ? device_cus() : 256,
                           g.qtype == QT_PLANES ? 1.12 : g.qtype == QT_Q4_0 ? 1.08 : 1.04, p));
}

size_t tile_scratch_bytes(const GemmArgs& g) {
    TilePlan p;
    return plan_of(g, p) ? p.part : 0;
}

WsNeed tile_ws_need(const GemmArgs& g) {
    WsNeed w;
    w.p = tile_scratch_bytes(g);
    return w;
}

hipError_t gemm_tile(const GemmArgs& g, const Scratch* scratch, hipStream_t st) {
    TilePlan p;
    if (!plan_of(g, p)) return hipErrorInvalidValue;
    if (g.qtype == QT_PLANES) return dispatch_tile<QT_PLANES>(g, p, scratch, st);
    if (g.qtype == QT_Q4_0) return dispatch_tile<QT_Q4_0>(g, p, scratch, st);
    return dispatch_tile<QT_Q4_K>(g, p, scratch, st);
}

}  // namespace bf
