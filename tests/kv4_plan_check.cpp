// CPU check of the 4-bit cache's layout and of the attention's launch plans
// (bus-fill_amd/csrc/bf_kv4.h, bf_kv4_plan.h).  Prints what it expected on
// failure; exit status 0 when all holds.  `kv4_plan_check plan S T heads group
// max_q max_kv causal window` prints a plan on 256 CUs, heads of 128 (prompt kernel, chunk, splits, waves).
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>

#include "bf_kv4_plan.h"

using namespace bf;

namespace {

int failures = 0;

void expect(bool ok, const char* what, int64_t a = 0, int64_t b = 0, int64_t c = 0) {
    if (ok) return;
    failures++;
    std::printf("FAIL %s (%lld, %lld, %lld)\n", what, (long long)a, (long long)b, (long long)c);
}

// Every byte of a record belongs to exactly one word of keys, byte of values or
// scale, words and halves at multiples of their size.
void check_layout() {
    for (int D : {64, 96, 128, 256}) {
        std::vector<int> used((size_t)kv4_record_bytes(D), 0);
        const auto take = [&](int at, int n, const char* what) {
            expect(at >= 0 && at + n <= (int)used.size() && at % n == 0, what, D, at);
            for (int i = at; i < at + n && i >= 0 && i < (int)used.size(); i++) used[i]++;
        };
        for (int t = 0; t < kKv4Tile; t++)
            for (int b = 0; b < D / 32; b++) {
                for (int g = 0; g < 4; g++) take(kv4_k_at(D, t, b, g), 4, "word of keys");
                for (int c = 0; c < 16; c++) take(kv4_v_at(D, t, b, c), 1, "byte of values");
                take(kv4_ks_at(D, t, b), 2, "keys' scale");
                take(kv4_vs_at(D, t, b), 2, "values' scale");
            }
        for (size_t i = 0; i < used.size(); i++) expect(used[i] == 1, "bytes used once", D, (int64_t)i, used[i]);
    }
    // records of neighbouring tiles, heads and pages follow each other, past 32 bits of bytes too
    expect(kv4_record(0, 0, 1, 8, 4) == 1 && kv4_record(0, 1, 0, 8, 4) == 4 && kv4_record(1, 0, 0, 8, 4) == 32, "records");
    expect(kv4_record(1 << 20, 7, 3, 8, 4) * kv4_record_bytes(256) == (((int64_t)1 << 25) + 31) * 9216, "far records");
}

// Tokens that the rows of a row tile can see are inside splits x chunk tiles,
// wherever the range starts; workspace only where a unit may have two chunks.
void check_plans() {
    for (int cus : {64, 256, 304})
        for (int dim : {64, 96, 128, 256})
            for (int heads : {1, 2, 8})
                for (int group : {1, 4, 5, 16})
                    for (int S : {1, 3, 32, 500})
                        for (int nq : {1, 2, 7, 16, 17, 100, 2000})
                            for (int kv : {0, 1, 31, 32, 519, 1280, 1281, 8000, 131072, 2000000})
                                for (int window : {0, 1, 100, 1024, 5000}) {
                                    Kv4Args a;
                                    std::memset(&a, 0, sizeof a);
                                    a.c = Kv4Shape{1, 64, heads, dim};
                                    a.q_heads = heads * group;
                                    a.S = S;
                                    a.T = S * nq;
                                    a.max_q = nq;
                                    a.max_kv = kv;
                                    a.causal = 1;
                                    a.window = window;
                                    const Kv4Plan p = plan_kv4(a, cus);
                                    const int64_t rows = (int64_t)nq * group;
                                    expect(p.group == group && (int64_t)p.row_tiles * p.tile_rows >= rows &&
                                               (int64_t)(p.row_tiles - 1) * p.tile_rows < rows, "row tiles", nq, group, p.row_tiles);
                                    expect(p.items == (int64_t)S * p.row_tiles, "items", S, p.row_tiles, p.items);
                                    int64_t seen = kv;
                                    if (window) {      // queries that share a row tile, each seeing `window` tokens
                                        int64_t span = 0;
                                        for (int64_t r = 0; r < rows; r += p.tile_rows) {
                                            const int64_t last = r + p.tile_rows < rows ? r + p.tile_rows - 1 : rows - 1;
                                            if (last / group - r / group + 1 > span) span = last / group - r / group + 1;
                                        }
                                        if (window + span - 1 < seen) seen = window + span - 1;
                                    }
                                    // a window's range may start at any token of a tile, others start at token 0
                                    const int64_t off = window ? kKv4Tile - 1 : 0, tiles = seen == 0 ? 0 : (off + seen + kKv4Tile - 1) / kKv4Tile;
                                    expect((int64_t)p.chunk * p.splits >= tiles, "chunks cover the tiles", tiles, p.chunk, p.splits);
                                    expect(p.splits == 1 || (p.chunk >= kKv4LeastFill && !p.prompt), "chunks of a size", p.chunk, p.splits, p.prompt);
                                    expect(p.slots == (p.splits > 1 ? p.items * heads * p.splits : 0), "slots", p.slots);
                                    expect(p.bytes == (size_t)p.slots * 16 * (dim + 2) * 4, "bytes", p.slots, (int64_t)p.bytes);
                                    expect(p.waves == 4 || p.waves == 8, "waves", p.waves);
                                    expect(p.bytes < (size_t)1 << 30, "partial results of a call", S, kv, (int64_t)p.bytes);
                                }
}

}  // namespace

int main(int argc, char** argv) {
    if (argc == 10 && !std::strcmp(argv[1], "plan")) {
        Kv4Args a;
        std::memset(&a, 0, sizeof a);
        int v[8];
        for (int i = 0; i < 8; i++) v[i] = std::atoi(argv[2 + i]);
        a.c = Kv4Shape{1, 64, v[2], 128};
        a.S = v[0];
        a.T = v[1];
        a.q_heads = v[2] * v[3];
        a.max_q = v[4];
        a.max_kv = v[5];
        a.causal = v[6];
        a.window = v[7];
        const Kv4Plan p = plan_kv4(a, 256);
        std::printf("%d %d %d %d\n", p.prompt, p.chunk, p.splits, p.waves);
        return 0;
    }
    if (argc < 2 || !std::strcmp(argv[1], "layout")) check_layout();
    if (argc < 2 || !std::strcmp(argv[1], "plans")) check_plans();
    std::printf("%d failures\n", failures);
    return failures ? 1 : 0;
}
