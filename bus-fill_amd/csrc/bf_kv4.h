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
// wave multiplies at once: 32 keys, then 32 values.  Codes lie in the order in
// which the lanes of a wave take them as matrix operands: lane l = 16 g + r
// reads its 16 bytes of a plane at 16 l, masks nibbles in place and gets
// nothing from another lane.
//
//   K: planes of four blocks of 32 values (the last of NB % 4, if any).  Token
//      8 a + 4 i + j (a, j = 0..3, i = 0, 1) is row r = 4 a + j of operand i;
//      lane 16 g + r of operand i holds for block b the word with values 32 b +
//      8 g + e: e = 0..7 in nibbles 0 4 1 5 2 6 3 7 (word & 0x000F000F, word &
//      0x00F000F0, and the same of word >> 8, are then the pairs 01, 23, 45, 67).
//   V: planes of two blocks (the last of NB % 2).  Lane 16 g + c holds tokens
//      8 g .. 8 g + 7 of columns c: for block b eight bytes, one per token, low
//      nibble value 32 b + c, high nibble value 32 b + 16 + c.
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
// Byte offsets in a record: the K word of token t, block b, part g; the V byte
// of token t, block b, column c; the scale of token t, block b.
BF_HD constexpr int kv4_k_at(int D, int t, int b, int g) {
    const int p = b / 4, w = D / 32 - 4 * p < 4 ? D / 32 - 4 * p : 4;
    return p * 2048 + ((t >> 2 & 1) * 64 + g * 16 + (t >> 3) * 4 + (t & 3)) * 4 * w + 4 * (b - 4 * p);
}
BF_HD constexpr int kv4_v_at(int D, int t, int b, int c) {
    const int p = b / 2, w = D / 32 - 2 * p < 2 ? D / 32 - 2 * p : 2;
    return 16 * D + p * 1024 + ((t >> 3) * 16 + c) * 8 * w + 8 * (b - 2 * p) + (t & 7);
}
BF_HD constexpr int kv4_ks_at(int D, int t, int b) { return 32 * D + (t >> 3) * (D / 2) + 16 * b + 2 * (t & 7); }
BF_HD constexpr int kv4_vs_at(int D, int t, int b) { return 2 * D + kv4_ks_at(D, t, b); }

// record of tile `tile` of a page
BF_HD inline int64_t kv4_record(int64_t page, int head, int tile, int heads, int tiles_per_page) {
    return (page * heads + head) * tiles_per_page + tile;
}

#undef BF_HD

}  // namespace bf
