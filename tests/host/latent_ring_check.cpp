// Host-only model of the ring of latent_rows_kernel (crabml_b200/csrc/latent_ring.cuh): two groups of warps, copies that land after a while, barriers that only know their phase's parity.
// Arguments: slots, seeds, "step" (places by lr_place) or "slot" (a barrier a slot, which is wrong).  Prints how many steps were read before their rows lay there, whether a step was lost, and how
// many runs of steps did not end.  No CUDA call is made.
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <random>
#include <vector>

#include "../../crabml_b200/csrc/latent_ring.cuh"

struct Bar { int phase = 0; };                    // phases that are complete
struct Copy { int step; double lands; };

int main(int argc, char** argv) {
    const int slots = std::atoi(argv[1]), seeds = std::atoi(argv[2]);
    const bool by_step = !std::strcmp(argv[3], "step");
    auto place = [&](int step) { return by_step ? lr_place(step, slots) : LrPlace{step % slots, step % slots, (unsigned)(step / slots) & 1u}; };
    long early = 0, lost = 0, stuck = 0;
    for (int seed = 0; seed < seeds; seed++) {
        std::mt19937 rng(seed);
        auto uni = [&](double lo, double hi) { return std::uniform_real_distribution<double>(lo, hi)(rng); };
        // a run of segments; the groups meet between two of them
        std::vector<int> ends;
        int n = 0;
        for (int i = 0, many = 1 + (int)(rng() % 5); i < many; i++) { n += (int)(rng() % (3 * slots + 2)); ends.push_back(n); }
        std::vector<Bar> bars(LR_GROUPS * LR_SLOTS);
        std::vector<int> holds(slots, -1);        // what lies in a slot: the step, -1 while rows are on their way
        std::vector<Copy> under_way;
        // times in a step's work: copies land after a fraction of one or, rarely, several
        auto ask = [&](int step, double now) {
            if (step >= n) return;
            holds[place(step).slot] = -1;
            under_way.push_back({step, now + (rng() % 6 ? uni(0.1, 1.0) : uni(1.0, 12.0))});
        };
        double now = 0.0;
        for (int s = 0; s < slots; s++) ask(s, now);
        // each group: the step that it waits for or works on, when it is through with it, the last step whose slot it has not asked for again
        struct Group { int step; double until; int last; bool works; } g[LR_GROUPS];
        for (int i = 0; i < LR_GROUPS; i++) g[i] = {i, 0.0, -1, false};
        size_t seg = 0;
        for (int turns = 0; ; turns++) {
            if (turns > 100000) { stuck++; break; }
            // what has landed, in its order
            for (;;) {
                int first = -1;
                for (size_t i = 0; i < under_way.size(); i++)
                    if (under_way[i].lands <= now && (first < 0 || under_way[i].lands < under_way[first].lands)) first = (int)i;
                if (first < 0) break;
                const LrPlace p = place(under_way[first].step);
                holds[p.slot] = under_way[first].step;
                bars[p.bar].phase++;
                under_way.erase(under_way.begin() + first);
            }
            // a segment ends when both groups are through with theirs of it; they ask for what is free
            while (seg < ends.size()) {
                bool all = true;
                for (auto& x : g) all &= !x.works && x.step >= ends[seg];
                if (!all) break;
                for (auto& x : g) if (x.last >= 0) { ask(x.last + slots, now); x.last = -1; }
                seg++;
            }
            if (seg >= ends.size()) break;
            for (auto& x : g) {
                if (x.works && x.until <= now) { x.works = false; x.last = x.step; x.step += LR_GROUPS; }
                if (x.works || x.step >= ends[seg]) continue;
                const LrPlace p = place(x.step);
                if (((bars[p.bar].phase + 1) & 1) != (int)p.parity) continue;      // the phase of that parity is not the one that is complete
                if (holds[p.slot] != x.step) early++;
                // all of the group are through with the step before: its slot is asked for
                if (x.last >= 0) { ask(x.last + slots, now); x.last = -1; }
                x.works = true; x.until = now + uni(0.8, 1.2);
            }
            now += 0.05;
        }
        for (const Copy& c : under_way) lost += c.step < n;
    }
    std::printf("%ld %ld %ld\n", early, lost, stuck);
}
