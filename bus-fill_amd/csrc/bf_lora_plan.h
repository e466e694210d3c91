// Arguments and launch plan of the low-rank adapters.  Plain C++ without HIP:
// the kernel file includes it, and so does the CPU check of the plans.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

namespace bf {

constexpr int kLoraParts = 4;
constexpr int kLoraRows = 16;                      // rows of a tile (one matrix operand)
constexpr int kLoraRanks = 64;                     // ranks of a unit of the down products (four operands)
constexpr int kLoraCols = 64;                      // columns of a step of the up products
constexpr int kLoraStep = 32;                      // k of a matrix instruction

struct LoraPart {
    const uint16_t* A;                             // [adapters][rank][K]
    const uint16_t* B;                             // [adapters][N][rank]
    int N, at;
};

struct LoraArgs {
    const uint16_t* X;
    int64_t ldx;
    const int32_t* ids;
    const float* scales;                           // NULL: 1
    const int32_t* ranks;                          // NULL: rank
    int adapters, rank, parts;
    LoraPart part[kLoraParts];
    const void* C;
    int64_t ldc;
    void* Y;
    int64_t ldy;
    int out_f16, wide;                             // wide: C and Y rows in whole 16-byte pieces
    int T, K;
};

// Down products: a wave (unit) takes a tile of 16 rows, a piece of K and up to 64
// ranks, and every `sharers`-th of the tile's adapters; its sums are a partial
// result.  Up products: a wave takes a tile of rows, `steps` steps of 64 columns
// and every `sharers`-th adapter, and adds the pieces' sums first.
struct LoraPlan {
    int tiles, rank_parts, pieces, piece;          // piece: steps of K
    int down_sharers, up_sharers, up_steps;
    int64_t down_units, up_units;                  // waves
    size_t bytes;                                  // partial results
};

inline LoraPlan plan_lora(const LoraArgs& a, int cus) {
    LoraPlan p;
    p.tiles = a.T / kLoraRows + (a.T % kLoraRows ? 1 : 0);
    p.rank_parts = (a.rank + kLoraRanks - 1) / kLoraRanks;
    const int per_tile = std::min(std::min(a.T, kLoraRows), a.adapters);   // adapters that a tile can have
    const int64_t want = 4 * (int64_t)cus;
    // few tiles: their adapters over several waves (with many, neighbouring rows are mostly of one adapter)
    p.down_sharers = p.tiles <= 8 ? per_tile : 1;
    const int64_t base = (int64_t)p.tiles * p.rank_parts * a.parts * p.down_sharers;   // (a grid that fits: T < 2^30)
    const int steps = (a.K + kLoraStep - 1) / kLoraStep;
    const int most = std::max(1, steps / 8);       // pieces of at least eight steps
    p.pieces = (int)std::min<int64_t>(most, std::max<int64_t>(1, (want + base - 1) / base));
    p.piece = (steps + p.pieces - 1) / p.pieces;
    p.pieces = (steps + p.piece - 1) / p.piece;
    p.down_units = base * p.pieces;
    int64_t cols = 0;                              // steps of columns of all parts
    for (int i = 0; i < a.parts; i++) cols += (a.part[i].N + kLoraCols - 1) / kLoraCols;
    p.up_sharers = p.tiles <= 8 ? std::min(per_tile, 4) : 1;
    p.up_steps = (int)std::min<int64_t>(8, std::max<int64_t>(1, p.tiles * cols * p.up_sharers / (2 * want)));
    p.up_units = 0;
    for (int i = 0; i < a.parts; i++) {
        const int64_t n = (a.part[i].N + kLoraCols - 1) / kLoraCols;
        p.up_units += (n + p.up_steps - 1) / p.up_steps;
    }
    p.up_units *= (int64_t)p.tiles * p.up_sharers;
    p.bytes = (size_t)a.parts * p.pieces * a.T * a.rank * sizeof(float);
    return p;
}

}  // namespace bf
