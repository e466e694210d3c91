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
constexpr int kLoraMany = 128;                     // more rows, two an adapter or more: sorted by adapter, tiles of 64
constexpr int kLoraManyFew = 256;                  // ... with fewer than eight adapters
constexpr int kLoraBins = 2048;                    // ... with fewer adapters than that
constexpr int kLoraRanks = 64;                     // ranks of a workgroup of the down products (four operands)
constexpr int kLoraCols = 64;                      // columns of a wave of the up products
constexpr int kLoraStep = 32;                      // k of a matrix instruction
constexpr int kLoraUnit = 64;                      // few rows: k of a row that comes to LDS at once (128 bytes)
constexpr int kLoraSlab = 320;                     // many rows: ... of A's rows (two of 64 ranks take 80 KB: two workgroups a CU)
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

#ifdef __HIPCC__
#define BF_BOTH __host__ __device__
#else
#define BF_BOTH
#endif
// Workgroups of a launch: `inner` for each of `tiles` tiles of rows.  Where there
// are many tiles, each XCD takes a run of them, whose adapters and sums its L2
// then holds; few are spread over all.
struct LoraGrid {
    int tiles, inner, per_xcd;                     // per_xcd: tiles of an XCD (0: spread)
    int64_t groups;
};
BF_BOTH inline LoraGrid lora_grid(int tiles, int64_t inner) {
    LoraGrid g;
    g.tiles = tiles;
    g.inner = (int)inner;
    g.per_xcd = tiles >= 4 * kLoraXcds ? tiles / kLoraXcds + (tiles % kLoraXcds ? 1 : 0) : 0;
    g.groups = (g.per_xcd ? (int64_t)g.per_xcd * kLoraXcds : tiles) * inner;
    return g;
}

// Workgroup b's tile and which of the tile's it is; false where there is none (b may be past the grid: one made for more tiles).
BF_BOTH inline bool lora_place(const LoraGrid& g, int b, int& tile, int& in) {
    if (g.tiles < 1) return false;
    if (g.per_xcd) {
        const int turn = b / kLoraXcds, nth = turn / g.inner;
        tile = b % kLoraXcds * g.per_xcd + nth;
        in = turn % g.inner;
        return nth < g.per_xcd && tile < g.tiles;
    }
    tile = b % g.tiles;
    in = b / g.tiles;
    return in < g.inner;
}
#undef BF_BOTH

// Many rows: `rows` rows of an adapter (-1: rows without one) and the ranks that count.
struct LoraTile {
    int adapter, rows, ranks, unused;
};

// Few rows (tiles of 16): down, a workgroup takes a tile, a part, up to 64 ranks, a
// piece of K (its waves shares of that) and every `sharers`-th of the tile's
// adapters; up, a workgroup takes a tile, up_steps steps of 64 columns of a part and
// all of the tile's adapters, its waves the pairs of adapter and step in turn, and
// adds the pieces' sums first.  Many rows: an order of the rows by adapter, then
// down, a workgroup takes a tile of 64 rows of one adapter, a part, up to 64 ranks and a piece
// of K; up, a tile and four steps of columns, with the pieces' sums (of more than 64
// ranks: joined in a launch of its own).
struct LoraPlan {
    int many;
    int rank_parts, rank_tiles;                    // rank_tiles: operands of ranks of a down workgroup (1, 2 or 4)
    int padded;                                    // many: ranks of the joined sums, in whole blocks
    int pieces, sharers;
    int up_steps;
    int most;                                      // many: as many tiles as there can be (how many there are is found on the device)
    LoraGrid down, up;                             // many: of `most` tiles
    int64_t tiles, rows, joined;                   // many: where [most + 1] tiles (the last: their number), their rows [most][64] and the joined sums lie, in words
    size_t bytes;                                  // [part][piece][T][rank] fp32; many: also the above, joined: hi and lo [part][T][padded] fp16, [part][T] factors
};

// Ranks of B that come to LDS at once.
constexpr int lora_block(int rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : 64; }

inline LoraPlan plan_lora(const LoraArgs& a, int cus) {
    LoraPlan p;
    const auto tiles = [&](int rows) { return a.T / rows + (a.T % rows ? 1 : 0); };
    const int rc = lora_block(a.rank);
    // (192 rows in no order, as they come and sorted: 8 adapters of rank 64 26 and 19 us, 64 of rank 16 29 and 24, 4 of rank 16
    // 14 and 18; in runs 14 and 19, 18 and 24, 11 and 18.  At 100 rows the first two meet.)
    p.many = a.T > (a.adapters < 8 ? kLoraManyFew : kLoraMany) && a.adapters <= a.T / 2 && a.adapters < kLoraBins;
    const int t = tiles(p.many ? 4 * kLoraSub : kLoraSub), per_tile = std::min(std::min(a.T, kLoraSub), a.adapters);
    p.most = p.many ? a.T / (4 * kLoraSub) + std::min(a.adapters + 1, a.T) : t;    // (each adapter's last tile may hold fewer rows)
    p.rank_parts = (a.rank + kLoraRanks - 1) / kLoraRanks;
    p.rank_tiles = rc / 16;
    p.padded = (a.rank + rc - 1) / rc * rc;
    p.sharers = p.many ? 1 : per_tile;
    const int64_t base = (int64_t)t * p.rank_parts * a.parts * p.sharers;
    // at least two units a wave, or a slab
    const int64_t least = p.many ? kLoraSlab : 2 * kLoraDownWaves * kLoraUnit, most = std::min<int64_t>(kLoraPieces, a.K / least);
    // few: two workgroups a CU; many: one, with as many short tiles as a handful of adapters make (how many there are the host does
    // not know), or two where that leaves one piece (2000 rows of six adapters, rank 64: 6 pieces 34.3 us, 8, which are more workgroups
    // than CUs, 38.5; 4000: 3 pieces 47, 8 54.  64 adapters in no order make up to 96 tiles of those 2000 rows, with 6 pieces
    // each still: not measured otherwise)
    const int64_t one = p.many ? cus / (base + 8) : 0;
    p.pieces = (int)std::min(std::max<int64_t>(1, most), one >= 2 ? one : std::max<int64_t>(1, 2 * cus / base));
    p.down = lora_grid(p.most, (int64_t)p.rank_parts * a.parts * p.sharers * p.pieces);
    int64_t cols = 0;                              // steps of columns of all parts
    for (int i = 0; i < a.parts; i++) cols += (a.part[i].N + kLoraCols - 1) / kLoraCols;
    // few: as many steps a workgroup as leave two workgroups a CU
    p.up_steps = p.many ? 4 : (int)std::min<int64_t>(16, std::max<int64_t>(1, (t * cols + 2 * cus - 1) / (2 * cus)));
    int64_t groups = 0;
    for (int i = 0; i < a.parts; i++) {
        const int64_t n = (a.part[i].N + kLoraCols - 1) / kLoraCols;
        groups += (n + p.up_steps - 1) / p.up_steps;
    }
    p.up = lora_grid(p.most, groups);
    p.tiles = (int64_t)a.parts * p.pieces * a.T * a.rank;
    p.rows = p.tiles + (p.many ? 4 * ((int64_t)p.most + 1) : 0);
    p.joined = p.rows + (p.many ? 64 * (int64_t)p.most : 0);
    p.bytes = (size_t)p.joined * sizeof(float);
    if (p.many && a.rank > rc) p.bytes += (size_t)a.parts * a.T * (4 * (size_t)p.padded + 4);
    return p;
}

// Bytes of workspace that a call takes hold of: never fewer than one of fewer rows with the same adapters, ranks, parts and K
// needs, so that the largest call's workspace serves all.  (More rows have fewer pieces of K, and so may need less themselves.)
// Of few rows, pieces rows <= rows or <= 2 cus rows / (tiles rank_parts parts sharers), where rows / (tiles sharers) is at most
// 16 / min(16, adapters); of many, rows or 2 cus rows / (tiles rank_parts parts), rows / tiles at most 64.
inline size_t lora_reserve(const LoraArgs& a, const LoraPlan& p, int cus) {
    const auto most = [&](int least, int64_t shared) {
        return std::max<int64_t>(a.T, std::min(std::max<int64_t>(1, std::min(kLoraPieces, a.K / least)) * a.T, shared));
    };
    const int64_t each = (int64_t)p.rank_parts * a.parts;
    int64_t rows = most(2 * kLoraDownWaves * kLoraUnit, 2 * cus * kLoraSub / (each * std::min(kLoraSub, a.adapters)));
    if (p.many) rows = std::max(rows, most(kLoraSlab, 2 * cus * 4 * kLoraSub / each));
    return p.bytes + (size_t)a.parts * a.rank * (rows - (int64_t)p.pieces * a.T) * sizeof(float);
}

// LDS rows of the inner sums (two planes of fp16): whole steps of 32, 16 bytes past a multiple of 64.
constexpr int lora_lds_ranks(int rank) { return (rank + kLoraStep - 1) / kLoraStep * kLoraStep + 8; }

}  // namespace bf
