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
constexpr int kKv4PromptRows = 128;                // ... of the prompt kernel's (four waves of 32)

// Rows of one key/value head: query i and head j of the group, row i G + j, in
// row tiles of 16.  An item is a row tile of a sequence; with a head it is a
// unit.  The tiles of 32 cached tokens that a unit sees are cut into chunks, a
// workgroup each; how many chunks a unit has the kernel finds from the lengths,
// which live in device memory (`splits`: the most that any can have).  Units of
// several chunks leave partial results, which a second launch joins.
struct Kv4Plan {
    int group, tile_rows, row_tiles, waves, chunk, splits;
    int prompt;                                    // the prompt kernel: no chunks
    int64_t items;                                 // sequences x row tiles
    int64_t slots;                                 // partial results (0: no unit can have two chunks)
    size_t bytes;                                  // their workspace
};

constexpr int kKv4Alone = 40;                      // tiles that one workgroup takes rather than share them
constexpr int kKv4LeastChunk = 20;
constexpr int kKv4PerCu = 4;                       // workgroups of four waves that a CU holds

// Chunks: three times as many as the chip has places where that leaves each
// kKv4LeastChunk tiles, so that sequences of different lengths even out
// (measured at 32 sequences of 2000 to 8000 tokens, 8 heads of 128: chunks of
// 12 / 20 / 40 / 64 tiles 60.6 / 58.6 / 58.7 / 64.0 us; one sequence of 131072,
// 4 heads: 16 / 24 / 40 / 64 tiles 29.1 / 27.6 / 27.6 / 33.8 us).  Short
// sequences are not cut (16 queries' heads over 1024 tokens of 64 values: 8.0
// us alone, 11.3 us in chunks of 12).
inline Kv4Plan plan_kv4(const Kv4Args& a, int cus) {
    Kv4Plan p;
    p.group = a.q_heads / a.c.heads;
    // The prompt kernel from 64 rows a sequence and head on, where its row tiles
    // fill half the chip.
    const int64_t rows = (int64_t)a.max_q * p.group, blocks = (rows + kKv4PromptRows - 1) / kKv4PromptRows;
    p.prompt = rows >= 64 && (int64_t)a.S * a.c.heads * blocks >= cus / 2;
    p.tile_rows = p.prompt ? kKv4PromptRows : kKv4Rows;
    p.row_tiles = (int)((rows + p.tile_rows - 1) / p.tile_rows);
    int64_t seen = a.max_kv;                       // cached tokens a row tile can see
    if (a.window > 0) {
        const int64_t span = std::min<int64_t>(a.max_q, (p.tile_rows + p.group - 2) / p.group + 1);
        seen = std::min<int64_t>(seen, (int64_t)a.window + span - 1);
    }
    const int64_t most = std::max<int64_t>(1, (seen + 2 * kKv4Tile - 2) / kKv4Tile);   // the range may start inside a tile
    p.items = (int64_t)a.S * p.row_tiles;
    const int64_t units = p.items * a.c.heads, places = (int64_t)cus * (a.c.dim == 256 ? 2 : kKv4PerCu);
    p.chunk = (int)(p.prompt || most <= kKv4Alone ? most : std::min(most, std::max<int64_t>(kKv4LeastChunk, (units * most + 3 * places - 1) / (3 * places))));
    p.splits = (int)((most + p.chunk - 1) / p.chunk);
    p.waves = units * p.splits < cus ? 8 : 4;      // few workgroups: twice the waves on each
    p.slots = p.splits > 1 ? units * p.splits : 0;
    p.bytes = (size_t)p.slots * kKv4Rows * (a.c.dim + 2) * sizeof(float);
    return p;
}

}  // namespace bf
