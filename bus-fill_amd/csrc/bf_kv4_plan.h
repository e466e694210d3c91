// Launch plan of the attention over the 4-bit cache.  Plain C++ without HIP:
// the kernel file includes it, and so does the CPU check of the plans.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

#include "bf_kv4.h"

namespace bf {

struct Kv4Args {
    uint8_t* data;
    Kv4Shape c;
    const uint16_t* Q;
    int64_t ldq;
    void* O;
    int64_t ldo;
    int out_f16;
    float* lse;
    const int32_t* q_start;
    const int32_t* kv_len;
    const int32_t* table;
    int ldt;
    int S, T, q_heads, max_q, max_kv;
    float scale;
    int causal, window;
};

constexpr int kKv4Rows = 16;                       // query rows of a row tile (one matrix operand)
constexpr int kKv4MaxSplits = 128;

// Rows of one key/value head: query i and head j of the group, row i G + j.
// Row tiles of 16; the tiles of 32 cached tokens that a row tile sees are cut
// into chunks, one workgroup each.  A sequence's chunks are counted by the
// kernel from its own length; `splits` is the most any of them can have.
struct Kv4Plan {
    int group, row_tiles, chunk, splits;
    int64_t parts;                                 // partial results (0 where no sequence can have two chunks)
    size_t bytes;                                  // their workspace
};

inline Kv4Plan plan_kv4(const Kv4Args& a, int cus) {
    Kv4Plan p;
    p.group = a.q_heads / a.c.heads;
    p.row_tiles = (int)(((int64_t)a.max_q * p.group + kKv4Rows - 1) / kKv4Rows);
    int64_t seen = a.max_kv;                       // cached tokens a row tile can see
    if (a.window > 0) {
        const int64_t span = std::min<int64_t>(a.max_q, (kKv4Rows + p.group - 2) / p.group + 1);
        seen = std::min<int64_t>(seen, (int64_t)a.window + span - 1);
    }
    const int64_t most = (seen + 2 * kKv4Tile - 2) / kKv4Tile;   // the range may start inside a tile
    const int64_t units = (int64_t)a.S * a.c.heads * p.row_tiles;
    // About three workgroups of four waves per CU, at least a tile for each wave
    const int64_t want = (units * most + 3 * cus - 1) / (3 * cus);
    const int64_t least = (most + kKv4MaxSplits - 1) / kKv4MaxSplits;
    p.chunk = (int)std::min(most, std::max({want, least, (int64_t)4}));
    p.splits = (int)((most + p.chunk - 1) / p.chunk);
    p.parts = p.splits > 1 ? units * p.splits : 0;
    p.bytes = (size_t)p.parts * kKv4Rows * (a.c.dim + 2) * sizeof(float);
    return p;
}

}  // namespace bf
