// Host-only check of lt_rounds (crabml_b200/csrc/latent_ring.cuh): four warps that meet at a barrier twice a round, where waits run out in some of them from some round on.  Prints how often the
// warps passed the barrier a different number of times ("rounds": by lt_rounds; "leave": a warp leaves its loop, which is wrong), how often one worked after its wait had run out, and how often one
// waited again.  No CUDA call is made.
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <random>

#include "../../crabml_b200/csrc/latent_ring.cuh"

int main(int argc, char** argv) {
    const bool rounds = !std::strcmp(argv[1], "rounds");
    long apart = 0, worked = 0, again = 0;
    for (int seed = 0; seed < 1000; seed++) {
        std::mt19937 rng(seed);
        const int lo = (int)(rng() % 3), hi = lo + (int)(rng() % 20);
        int passed[4] = {};
        for (int w = 0; w < 4; w++) {
            const int out = lo + (int)(rng() % 24);      // the round from which on this warp's wait runs out
            int waits_out = 0;
            auto wait = [&](int i) { again += waits_out; waits_out += i >= out; return i < out; };
            auto body = [&](int i, bool ok) { passed[w] += 2; worked += ok && i >= out; };
            if (rounds) lt_rounds(lo, hi, wait, body);
            else
                for (int i = lo; i < hi; i++) {
                    if (!wait(i)) break;
                    body(i, true);
                }
        }
        apart += passed[0] != passed[1] || passed[1] != passed[2] || passed[2] != passed[3];
    }
    std::printf("%ld %ld %ld\n", apart, worked, again);
}
