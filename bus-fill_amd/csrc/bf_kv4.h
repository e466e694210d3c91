// Layout of the 4-bit key/value cache, shared by its store, its read-back and
// the attention kernels.  Plain C++: the CPU tests of the launch plans include
// it too.
//
// A cached row (one token of one head, D values) is quantized like a row of
// Q4_0 weights: per 32 values a scale d (fp16) and codes q with value
// (q - 8) d.  The cache is pages of `page_size` tokens (a multiple of 32); page
// p holds, head by head, page_size / 32 records of 32 tokens:
//
//   record = K codes (16 D) | V codes (16 D) | K scales (2 D) | V scales (2 D)   bytes
//
// so a head's tokens of a page are one run of memory, and a record is what a
// wave multiplies at once: 32 keys, then 32 values.  The order of the codes in
// a record is the order in which matrix instructions take them, so that the
// attention kernels mask nibbles in place and move nothing between lanes:
//
//   K: token t at byte D/2 t.  Its D/8-byte part g = 0..3 holds for block b the
//      word b with values 32 b + 8 g + e: e = 0..7 in nibbles 0 4 1 5 2 6 3 7
//      (word & 0x000F000F, word & 0x00F000F0, and the same of word >> 8, are
//      then the pairs 01, 23, 45, 67).
//   V: tokens 8 g .. 8 g + 7 at byte 4 D g.  Column c = 0..15 at byte D/4 c of
//      that: for block b eight bytes, one per token, low nibble value 32 b + c,
//      high nibble value 32 b + 16 + c.
//   scales: tokens 8 g .. 8 g + 7 at byte D/2 g: for block b eight halves, one
//      per token.
#pragma once

#include <cstdint>

namespace bf {

constexpr int kKv4Tile = 32;                       // tokens of a record

struct Kv4Shape {
    int pages, page_size, heads, dim;
};

#ifdef __HIPCC__
#define BF_HD __host__ __device__
#else
#define BF_HD
#endif

BF_HD constexpr int64_t kv4_record_bytes(int D) { return 36 * (int64_t)D; }
BF_HD constexpr int kv4_v_at(int D) { return 16 * D; }
BF_HD constexpr int kv4_ks_at(int D) { return 32 * D; }
BF_HD constexpr int kv4_vs_at(int D) { return 34 * D; }

// record of tile `tile` of a page
BF_HD inline int64_t kv4_record(int64_t page, int head, int tile, int heads, int tiles_per_page) {
    return (page * heads + head) * tiles_per_page + tile;
}

#undef BF_HD

}  // namespace bf
