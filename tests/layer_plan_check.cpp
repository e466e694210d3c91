// CPU check of the low-rank adapters' launch plans (bus-fill_amd/csrc/bf_lora_plan.h)
// and of those of the attention with first tokens in sight (bf_kv4_plan.h).  Prints
// what it expected on failure; exit status 0 when all holds.
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <vector>

#include "bf_kv4_plan.h"
#include "bf_lora_plan.h"

using namespace bf;

namespace {

int failures = 0;

void expect(bool ok, const char* what, int64_t a = 0, int64_t b = 0, int64_t c = 0) {
    if (ok) return;
    failures++;
    std::printf("FAIL %s (%lld, %lld, %lld)\n", what, (long long)a, (long long)b, (long long)c);
}

// Every (tile, share) of `tiles` tiles has one of the grid's workgroups (a grid may be made for more tiles than there are).
void check_grid(const LoraGrid& made, int tiles, int64_t inner) {
    std::vector<int> seen((size_t)(tiles * inner), 0);
    const LoraGrid g = lora_grid(tiles, inner);
    for (int64_t b = 0; b < made.groups; b++) {
        int tile = -1, in = -1;
        if (!lora_place(g, (int)b, tile, in)) continue;
        expect(tile >= 0 && tile < tiles && in >= 0 && in < inner, "workgroup in its tile", b, tile, in);
        if (tile >= 0 && tile < tiles && in >= 0 && in < inner) seen[(size_t)(tile * inner + in)]++;
    }
    for (size_t i = 0; i < seen.size(); i++) expect(seen[i] == 1, "one workgroup each", (int64_t)i, seen[i], tiles);
}

void check_lora() {
    for (int cus : {64, 256, 304})
        for (int T : {1, 5, 16, 17, 100, 128, 129, 256, 257, 600, 2000, 5000})
            for (int K : {8, 64, 1000, 5120, 17408})
                for (int rank : {8, 16, 24, 64, 72, 256, 1024})
                    for (int E : {1, 3, 64, 700, 5000})
                        for (int N : {1, 64, 300, 5120}) {
                            LoraArgs a;
                            std::memset(&a, 0, sizeof a);
                            a.T = T;
                            a.K = K;
                            a.rank = rank;
                            a.adapters = E;
                            a.parts = N == 300 ? 3 : 1;
                            for (int i = 0; i < a.parts; i++) a.part[i].N = N + 70 * i;
                            const LoraPlan p = plan_lora(a, cus);
                            const int rows = p.many ? 64 : kLoraSub, tiles = (T + rows - 1) / rows;
                            expect(p.pieces >= 1 && p.pieces <= kLoraPieces, "pieces", p.pieces);
                            expect((int64_t)p.rank_parts * kLoraRanks >= rank && (int64_t)(p.rank_parts - 1) * kLoraRanks < rank, "ranks", rank);
                            expect(p.padded >= rank && p.padded % lora_block(rank) == 0, "padded ranks", rank, p.padded);
                            const int most = E < rows ? E : rows;          // adapters that a tile of few rows can have
                            expect(p.many == ((T > 256 || (T > 128 && E >= 8)) && E <= T / 2 && E < 2048), "many", T, p.many);
                            expect(p.most >= tiles && (!p.many || p.most >= tiles + (E + 1 < T ? E : T - tiles)), "tiles", T, E, p.most);
                            expect(p.many ? p.sharers == 1 : p.sharers >= (most < T ? most : T), "sharers", T, E, p.sharers);
                            // pieces of K: units of 64, none empty of all waves' shares
                            const int64_t units = (K + kLoraUnit - 1) / kLoraUnit;
                            for (int i = 0; i < p.pieces; i++)
                                expect(units * (i + 1) / p.pieces > units * i / p.pieces, "piece of K", K, i, p.pieces);
                            int64_t groups = 0;
                            for (int i = 0; i < a.parts; i++)
                                groups += ((a.part[i].N + kLoraCols - 1) / kLoraCols + p.up_steps - 1) / p.up_steps;
                            if (cus == 256 && K == 5120) {
                                for (int n : {tiles, p.most, (tiles + p.most) / 2, 31, 32, 33}) {
                                    if (n < tiles || n > p.most) continue;
                                    check_grid(p.down, n, (int64_t)p.rank_parts * a.parts * p.sharers * p.pieces);
                                    check_grid(p.up, n, groups);
                                }
                            }
                            const int64_t sums = (int64_t)a.parts * p.pieces * T * rank;
                            expect(p.tiles == sums && p.tiles % 4 == 0, "partial sums", p.tiles, sums);
                            expect(p.rows - p.tiles == (p.many ? 4 * (p.most + 1) : 0), "tiles' place", p.rows, p.tiles, p.most);
                            expect(p.joined - p.rows == (p.many ? 64 * (int64_t)p.most : 0) && p.joined % 4 == 0, "rows' place", p.joined, p.rows, T);
                            const int64_t joined = p.many && rank > 64 ? (int64_t)a.parts * T * (4 * p.padded + 4) : 0;
                            expect((int64_t)p.bytes == 4 * p.joined + joined, "bytes", (int64_t)p.bytes, 4 * p.joined + joined);
                            expect(p.many || 8 * 2 * kLoraCols * lora_block(rank) + 64 * lora_lds_ranks(rank) <= 159 * 1024, "LDS", rank);
                        }
}

// Tiles that a row tile walks over, with first tokens in sight, fit its chunks.
void check_sinks() {
    for (int heads : {1, 8})
        for (int group : {1, 5, 16})
            for (int S : {1, 32})
                for (int nq : {1, 7, 100, 2000})
                    for (int kv : {0, 1, 33, 1200, 8000, 131072})
                        for (int window : {1, 31, 1000, 5000, 2147483647})
                            for (int sinks : {1, 4, 32, 33, 5000, 2147483647}) {
                                Kv4Args a;
                                std::memset(&a, 0, sizeof a);
                                a.c = Kv4Shape{1, 64, heads, 128};
                                a.q_heads = heads * group;
                                a.S = S;
                                a.T = S * nq;
                                a.max_q = nq;
                                a.max_kv = kv;
                                a.causal = 1;
                                a.window = window;
                                const Kv4Plan without = plan_kv4(a, 256);
                                a.sinks = sinks;
                                const Kv4Plan p = plan_kv4(a, 256);
                                expect(p.bytes == (size_t)p.slots * 16 * (128 + 2) * 4, "bytes", p.slots, (int64_t)p.bytes);
                                expect((int64_t)p.chunk * p.splits >= (int64_t)without.chunk * without.splits || p.prompt != without.prompt ||
                                           without.splits > 1, "chunks", p.chunk, p.splits);
                                for (int len : {0, 1, 31, 32, 33, 100, kv / 2, kv}) {
                                    if (len > kv) continue;
                                    for (int64_t row0 = 0; row0 < (int64_t)nq * group; row0 += p.tile_rows) {
                                        const int64_t last = row0 + p.tile_rows < (int64_t)nq * group ? row0 + p.tile_rows - 1 : (int64_t)nq * group - 1;
                                        const int64_t first_end = len - nq + row0 / group + 1, end = len - nq + last / group + 1;
                                        const int64_t hi = end > 0 ? end : 0, fe = first_end > 0 ? first_end : 0, lo = fe > window ? fe - window : 0;
                                        const int64_t w0 = lo / 32, ahead = ((sinks < hi ? sinks : hi) + 31) / 32, t1 = (hi + 31) / 32 > w0 ? (hi + 31) / 32 : w0;
                                        const int64_t walk = ahead < w0 ? ahead + t1 - w0 : t1;
                                        expect(walk <= (int64_t)p.chunk * p.splits, "walk fits its chunks", walk, p.chunk, p.splits);
                                    }
                                }
                            }
}

}  // namespace

int main(int argc, char** argv) {
    if (argc < 2 || !std::strcmp(argv[1], "lora")) check_lora();
    if (argc < 2 || !std::strcmp(argv[1], "sinks")) check_sinks();
    std::printf("%d failures\n", failures);
    return failures ? 1 : 0;
}
