// CPU check of the launch plans of the attention with first tokens in sight
// (bus-fill_amd/csrc/bf_kv4_plan.h): a plan reckons with no more tiles than the cache can
// have.  Prints what it expected on failure; exit status 0 when all holds.
#include <cstdio>
#include <cstring>

#include "bf_kv4_plan.h"

using namespace bf;

int main() {
    int failures = 0;
    for (int cus : {64, 256})
        for (int heads : {1, 8})
            for (int group : {1, 5})
                for (int S : {1, 8, 16, 64})
                    for (int nq : {1, 7, 300})
                        for (int kv : {1, 33, 600, 1200, 8000, 131072, 2147483583})
                            for (int window : {1, 1000, 8000, 2147483647})
                                for (int sinks : {1, 4, 100, 4000, 1 << 30, 2147483647}) {
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
                                    const Kv4Plan own = plan_kv4(a, cus);
                                    a.sinks = sinks;
                                    const Kv4Plan p = plan_kv4(a, cus);
                                    const int64_t all = ((int64_t)kv + 31) / 32, walk = (int64_t)p.chunk * (p.splits - 1);
                                    // the last chunk has a tile, or the plan is the one without first tokens
                                    const bool same = p.chunk == own.chunk && p.splits == own.splits && p.waves == own.waves && p.bytes == own.bytes;
                                    const bool ok = (p.splits == 1 || walk < all || same) && (window < kv || p.prompt != own.prompt || same);
                                    if (ok) continue;
                                    failures++;
                                    std::printf("FAIL cus %d heads %d group %d S %d nq %d kv %d window %d sinks %d: chunks %d of %d, without %d of %d\n",
                                                cus, heads, group, S, nq, kv, window, sinks, p.splits, p.chunk, own.splits, own.chunk);
                                }
    std::printf("%d failures\n", failures);
    return failures ? 1 : 0;
}
