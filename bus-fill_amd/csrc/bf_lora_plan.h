// Arguments and launch plan of the low-rank adapters.  Plain C++ without HIP:
// the kernel file includes it, and so does the CPU check of the plans.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

namespace bf {

constexpr int kLoraParts = 4;
constexpr int kLoraMaxRank = 1024;
constexpr int kLoraSub = 16;                       // rows of a matrix operand, and of a tile of few rows
constexpr int kLoraMany = 256;                     // rows from which on tiles are of 64
constexpr int kLoraRanks = 64;                     // ranks of a workgroup of the down products (four operands)
constexpr int kLoraCols = 64;                      // columns of a wave of the up products
constexpr int kLoraStep = 32;                      // k of a matrix instruction
constexpr int kLoraUnit = 64;                      // few rows: k of a row that comes to LDS at once (128 bytes)
constexpr int kLoraSlab = 320;                     // many rows: ... of A's rows
constexpr int kLoraPieces = 8;                     // pieces of K at most
constexpr int kLoraXcds = 8;                       // (a launch's workgroups go round them)
constexpr int kLoraDownWaves = 4;                  // of a workgroup of the down products of few rows
constexpr int kLoraManyWaves = 8;                  // ... of many
constexpr int kLoraUpWaves = 8;                    // ... of the up products (many rows: of 64 rows and four steps of columns)

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

// Workgroups of a launch: `inner` for each of `tiles` tiles of rows.  Where there
// are many tiles, each XCD takes a run of them, whose adapters and sums its L2
// then holds; few are spread over all.
struct LoraGrid {
    int tiles, inner, per_xcd;                     // per_xcd: tiles of an XCD (0: spread)
    int64_t groups;
};
inline LoraGrid lora_grid(int tiles, int64_t inner) {
    LoraGrid g;
    g.tiles = tiles;
    g.inner = (int)inner;
    g.per_xcd = tiles >= 4 * kLoraXcds ? tiles / kLoraXcds + (tiles % kLoraXcds ? 1 : 0) : 0;
    g.groups = (g.per_xcd ? (int64_t)g.per_xcd * kLoraXcds : tiles) * inner;
    return g;
}

// Workgroup b's tile and which of the tile's it is; false where there is none.
#ifdef __HIPCC__
__host__ __device__
#endif
inline bool lora_place(const LoraGrid& g, int b, int& tile, int& in) {
    if (g.per_xcd) {
        const int turn = b / kLoraXcds;
        tile = b % kLoraXcds * g.per_xcd + turn / g.inner;
        in = turn % g.inner;
    } else {
        tile = b % g.tiles;
        in = b / g.tiles;
    }
    return tile < g.tiles;
}

// Few rows (tiles of 16): down, a workgroup takes a tile, a part, up to 64 ranks, a
// piece of K (its waves shares of that) and every `sharers`-th of the tile's
// adapters; up, a workgroup takes a tile, up_steps steps of 64 columns of a part and
// all of the tile's adapters, its waves the pairs of adapter and step in turn, and adds the pieces' sums first.  Many rows (tiles of 64): down, a tile, a
// part, up to 64 ranks, and a piece of K; a join of the pieces; up, a tile and four
// steps of columns.
struct LoraPlan {
    int many;
    int rank_parts, rank_tiles;                    // rank_tiles: operands of ranks of a down workgroup (1, 2 or 4)
    int padded;                                    // many: ranks of the joined sums, in whole blocks
    int pieces, sharers;
    int up_steps;
    LoraGrid down, up;
    int64_t joined;                                // many: fp32 words of the partial sums, behind which the joined ones lie
    size_t bytes;                                  // [part][piece][T][rank] fp32; many: hi and lo [part][T][padded] fp16, [part][T] factors
};

// Ranks of B that come to LDS at once.
constexpr int lora_block(int rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : 64; }

inline LoraPlan plan_lora(const LoraArgs& a, int cus) {
    LoraPlan p;
    const auto tiles = [&](int rows) { return a.T / rows + (a.T % rows ? 1 : 0); };
    const int rc = lora_block(a.rank);
    p.many = a.T > kLoraMany;
    const int t = tiles(p.many ? 4 * kLoraSub : kLoraSub), per_tile = std::min(std::min(a.T, kLoraSub), a.adapters);
    p.rank_parts = (a.rank + kLoraRanks - 1) / kLoraRanks;
    p.rank_tiles = rc / 16;
    p.padded = (a.rank + rc - 1) / rc * rc;
    p.sharers = p.many ? 1 : per_tile;             // (of many rows, neighbours are mostly of one adapter)
    const int64_t base = (int64_t)t * p.rank_parts * a.parts * p.sharers;
    // at least two units a wave, or a slab
    const int64_t least = p.many ? kLoraSlab : 2 * kLoraDownWaves * kLoraUnit, most = std::min<int64_t>(kLoraPieces, a.K / least);
    p.pieces = (int)std::min(std::max<int64_t>(1, most), std::max<int64_t>(1, 2 * cus / base));
    p.down = lora_grid(t, (int64_t)p.rank_parts * a.parts * p.sharers * p.pieces);
    int64_t cols = 0;                              // steps of columns of all parts
    for (int i = 0; i < a.parts; i++) cols += (a.part[i].N + kLoraCols - 1) / kLoraCols;
    // few: as many steps a workgroup as leave two workgroups a CU
    p.up_steps = p.many ? 4 : (int)std::min<int64_t>(16, std::max<int64_t>(1, (t * cols + 2 * cus - 1) / (2 * cus)));
    int64_t groups = 0;
    for (int i = 0; i < a.parts; i++) {
        const int64_t n = (a.part[i].N + kLoraCols - 1) / kLoraCols;
        groups += (n + p.up_steps - 1) / p.up_steps;
    }
    p.up = lora_grid(t, groups);
    p.joined = (int64_t)a.parts * p.pieces * a.T * a.rank;
    p.bytes = (size_t)p.joined * sizeof(float);
    if (p.many && a.rank > rc) p.bytes += (size_t)a.parts * a.T * (4 * (size_t)p.padded + 4);
    return p;
}

// LDS rows of the inner sums (two planes of fp16): whole steps of 32, 16 bytes past a multiple of 64.
constexpr int lora_lds_ranks(int rank) { return (rank + kLoraStep - 1) / kLoraStep * kLoraStep + 8; }

}  // namespace bf
