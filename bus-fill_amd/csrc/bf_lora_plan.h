// Arguments and launch plan of the low-rank adapters.  Plain C++ without HIP:
// the kernel file includes it, and so does the CPU check of the plans.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

namespace bf {

constexpr int kLoraParts = 4;
constexpr int kLoraMaxRank = 1024;
constexpr int kLoraSub = 16;                       // rows of a matrix operand
constexpr int kLoraRanks = 64;                     // ranks of a workgroup of the down products (four operands)
constexpr int kLoraCols = 64;                      // columns of a step of the up products
constexpr int kLoraStep = 32;                      // k of a matrix instruction
constexpr int kLoraUpWaves = 8;

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

// A tile is `subs` operands of rows (16 rows, or 64).  Down products: a workgroup
// takes a tile, a part, up to 64 ranks, a piece of K (its waves shares of that) and
// every `sharers`-th of the tile's adapters.  Up products: a workgroup takes a
// tile, `up_steps` steps of 64 columns of a part and all of the tile's adapters,
// its waves the pairs of adapter and step in turn.
struct LoraPlan {
    int subs, tiles, rank_parts, rank_tiles;       // rank_tiles: operands of ranks of a down workgroup (1, 2 or 4)
    int pieces, down_waves, sharers;
    int up_steps;
    int64_t down_groups, up_groups;
    size_t bytes;                                  // partial sums: [part][piece][T][rank]
};

inline LoraPlan plan_lora(const LoraArgs& a, int cus) {
    LoraPlan p;
    p.subs = a.T > 16 * kLoraSub && a.rank <= 256 ? 4 : 1;
    const int rows = kLoraSub * p.subs;
    p.tiles = a.T / rows + (a.T % rows ? 1 : 0);
    p.rank_parts = (a.rank + kLoraRanks - 1) / kLoraRanks;
    p.rank_tiles = a.rank <= 16 ? 1 : a.rank <= 32 ? 2 : 4;
    const int per_tile = std::min(std::min(a.T, rows), a.adapters);        // adapters that a tile can have
    // few rows: a tile's adapters over several workgroups (of many rows, neighbours are mostly of one adapter)
    p.sharers = p.subs == 1 ? per_tile : 1;
    p.down_waves = p.subs == 1 ? 8 : 4;
    const int64_t base = (int64_t)p.tiles * p.rank_parts * a.parts * p.sharers;
    const int64_t steps = (a.K + kLoraStep - 1) / kLoraStep;
    const int64_t most = std::max<int64_t>(1, steps / (4 * p.down_waves));   // at least four steps a wave
    p.pieces = (int)std::min<int64_t>(std::min<int64_t>(most, 4), std::max<int64_t>(1, 2 * cus / base));
    p.down_groups = base * p.pieces;
    int64_t cols = 0;                              // steps of columns of all parts
    for (int i = 0; i < a.parts; i++) cols += (a.part[i].N + kLoraCols - 1) / kLoraCols;
    // as many steps a workgroup as leave two workgroups a CU, eight at most
    p.up_steps = (int)std::min<int64_t>(kLoraUpWaves, std::max<int64_t>(1, p.tiles * cols / (2 * cus)));
    p.up_groups = 0;
    for (int i = 0; i < a.parts; i++) {
        const int64_t n = (a.part[i].N + kLoraCols - 1) / kLoraCols;
        p.up_groups += (n + p.up_steps - 1) / p.up_steps;
    }
    p.up_groups *= p.tiles;
    p.bytes = (size_t)a.parts * p.pieces * a.T * a.rank * sizeof(float);
    return p;
}

// LDS rows of the inner sums (two planes of fp16): whole steps of 32, 16 bytes past a multiple of 64.
constexpr int lora_lds_ranks(int rank) { return (rank + kLoraStep - 1) / kLoraStep * kLoraStep + 8; }

}  // namespace bf
