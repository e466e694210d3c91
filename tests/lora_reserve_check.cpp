// CPU check of the low-rank adapters' workspace (bus-fill_amd/csrc/bf_lora_plan.h): what a
// call takes hold of holds what it needs, and never falls as the number of rows grows.
// Prints what it expected on failure; exit status 0 when all holds.
#include <cstdio>
#include <cstring>

#include "bf_lora_plan.h"

using namespace bf;

int main() {
    int failures = 0;
    for (int cus : {64, 256, 304})
        for (int K : {8, 600, 1000, 5000, 5120, 17408})
            for (int rank : {8, 64, 72, 256, 1024})
                for (int E : {1, 3, 7, 8, 32, 700, 2047, 2048})
                    for (int parts : {1, 3, 4}) {
                        LoraArgs a;
                        std::memset(&a, 0, sizeof a);
                        a.K = K;
                        a.rank = rank;
                        a.adapters = E;
                        a.parts = parts;
                        for (int i = 0; i < parts; i++) a.part[i].N = 1000;
                        size_t before = 0;
                        for (int T = 1; T < 9000; T += T < 700 ? 1 : 37) {
                            a.T = T;
                            const LoraPlan p = plan_lora(a, cus);
                            const size_t n = lora_reserve(a, p, cus);
                            if (n < p.bytes || n < before || n % 4) {
                                failures++;
                                std::printf("FAIL cus %d K %d rank %d adapters %d parts %d T %d: %zu bytes, needs %zu, fewer rows %zu\n",
                                            cus, K, rank, E, parts, T, n, p.bytes, before);
                            }
                            before = n;
                        }
                    }
    std::printf("%d failures\n", failures);
    return failures ? 1 : 0;
}
