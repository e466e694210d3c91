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
    int sinks;                                     // first tokens that a window leaves visible (0 without one)
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

// The prompt kernel takes 128 rows through a record in 1.2 to 1.4 us (heads of 128),
// and as long where a workgroup has a CU to itself; k_kv4_attn takes 16 rows
// through one in 0.19 us of a CU.  So the first where there is work for several
// rounds of the CUs (row tiles of 16, times the share of the longest row's tokens
// that the average one sees, at least seven a CU) and its blocks of 128 rows are
// at least 3/4 full.  Prompt kernel and k_kv4_attn in us, 40 heads over 8 of 128:
// prompts of 1000 tokens 52 and 41, 1500 73 and 87, 2000 93 and 134, 16 of 256 45 and
// 72; 512 queries over 2000 91 and 56; 32 times 20 queries over 2000 93 and 81, 48
// queries 132 and 169.  16 heads over 8 of 64: 2000 tokens 59 and 38, 4000 113 and
// 112, 8 prompts of 1000 49 and 67; 16 over 4 of 256: 3000 tokens 280 and 267.
inline bool prompt_serves(const Kv4Args& a, int group, int cus) {
    const int64_t rows = (int64_t)a.max_q * group, tiles = (rows + kKv4Rows - 1) / kKv4Rows;
    if (tiles < 6 * ((rows + kKv4PromptRows - 1) / kKv4PromptRows)) return false;
    const int64_t all = std::min(a.S * tiles, (int64_t)a.T * group / kKv4Rows + a.S) * a.c.heads;
    double share = 1.0;                            // causal rows: the first ones see less
    if (a.causal && a.max_kv > 0) {
        const double reach = a.window > 0 ? std::min<int64_t>((int64_t)a.window + a.sinks, a.max_kv) : a.max_kv;
        const double ramp = std::min<double>(a.max_q, std::max(0.0, reach - (a.max_kv - std::min(a.max_q, a.max_kv))));
        share -= ramp * ramp / (2.0 * a.max_q * reach);
    }
    return (double)all * share >= 7.0 * cus;
}

constexpr int kKv4PerCu = 4;                       // workgroups of four waves that a CU holds
constexpr int kKv4Alone = 40;                      // tiles that one workgroup takes rather than share them
constexpr int kKv4AloneMany = 256;                 // ... where there are workgroups enough without
constexpr int kKv4LeastFill = 8;                   // tiles of a chunk (a wave each)
constexpr int kKv4LeastChunk = 20;                 // ... where sequences differ in length

// Chunks.  A joining launch costs 4 to 6 us and an unevenly filled last round of
// workgroups as much, lengths are in device memory (max_kv is all the host
// knows), and a chip of 256 CUs reads at full rate with eight waves on each.
// Measured in us, 8 key/value heads of 128 unless said, one query a sequence:
// * Up to 40 tiles, alone (1030 tokens: 10.8, in chunks of 8 tiles 10.5; 16
//   sequences of up to 1100: 11.6 and 14.0).
// * From 3/4 as many units as CUs and up to 256 tiles, alone, eight waves (64
//   sequences of up to 2048: 25.3, chunks of 20 tiles and four waves 38.7; 24 of
//   up to 3000: 21.8 and 23.9; 32 of up to 8000: 49.7 and 53.3).  Past that a
//   sequence much longer than the others would keep one workgroup too long.
// * One sequence, or chunks of up to 32 tiles: as many chunks as fill the CUs
//   once, eight waves (131072 tokens, 4 heads: 65 tiles 22.7, 33 tiles 25.4, 20
//   tiles and four waves 30.0; 32768: 17.0 and 19.2; 2048: 10.7 and 12.5).
// * Else three times as many as the chip has places of four waves, so that
//   sequences of different lengths even out (20 of up to 8000: 37.8, filling
//   once 42.8 to 47).
inline Kv4Plan plan_kv4(const Kv4Args& a, int cus) {
    Kv4Plan p;
    p.group = a.q_heads / a.c.heads;
    const int64_t rows = (int64_t)a.max_q * p.group;
    p.prompt = prompt_serves(a, p.group, cus);
    p.tile_rows = p.prompt ? kKv4PromptRows : kKv4Rows;
    p.row_tiles = (int)((rows + p.tile_rows - 1) / p.tile_rows);
    int64_t seen = a.max_kv;                       // cached tokens a row tile can see
    if (a.window > 0) {
        const int64_t span = std::min<int64_t>(a.max_q, (p.tile_rows + p.group - 2) / p.group + 1);
        seen = std::min<int64_t>(seen, (int64_t)a.window + span - 1);
    }
    int64_t most = std::max<int64_t>(1, (seen + (a.window > 0 ? 2 : 1) * (kKv4Tile - 1)) / kKv4Tile);   // (a window may start inside a tile)
    // first tokens' tiles, but no more in all than there are
    if (a.sinks > 0)
        most = std::max(most, std::min(most + (std::min<int64_t>(a.sinks, a.max_kv) + kKv4Tile - 1) / kKv4Tile,
                                       ((int64_t)a.max_kv + kKv4Tile - 1) / kKv4Tile));
    p.items = (int64_t)a.S * p.row_tiles;
    const int64_t units = p.items * a.c.heads, places = (int64_t)cus * (a.c.dim == 256 ? 2 : kKv4PerCu);
    const int64_t share = std::max<int64_t>(1, cus / units), fill = (most + share - 1) / share;
    if (p.prompt || most <= kKv4Alone || (4 * units >= 3 * (int64_t)cus && most <= kKv4AloneMany)) p.chunk = (int)most;
    else if (share > 1 && (a.S == 1 || fill <= 32)) p.chunk = (int)std::max<int64_t>(kKv4LeastFill, fill);
    else p.chunk = (int)std::min(most, std::max<int64_t>(kKv4LeastChunk, (units * most + 3 * places - 1) / (3 * places)));
    p.splits = (int)((most + p.chunk - 1) / p.chunk);
    // Eight waves where there are no more workgroups than CUs, or long walks of whole sequences (64 of up to 500
    // tokens: 12.1 with eight, 11.8 with four; 24 of up to 3000: 21.6 and 26.0)
    p.waves = units * p.splits <= cus || (p.splits == 1 && most > kKv4Alone) ? 8 : 4;
    p.slots = p.splits > 1 ? units * p.splits : 0;
    p.bytes = (size_t)p.slots * kKv4Rows * (a.c.dim + 2) * sizeof(float);
    return p;
}

}  // namespace bf
