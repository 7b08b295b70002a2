// Host-only check of the plan of a step over several sequences (crabml_b200/csrc/paged_plan.hpp).  Reads plans from standard input, each
//   n_seqs page_size table_cols n_pages n_slots has_slots, then pos0, counts, the table's rows and, where has_slots, the slots;
// prints "wrong <text>", or "plan <items> <tokens>" and a line for each segment.  No CUDA call is made.
#include <cstdio>
#include <iostream>

#include "../../crabml_b200/csrc/paged_plan.hpp"

int main() {
    long long n, page, cols, pages, slots, has;
    while (std::cin >> n >> page >> cols >> pages >> slots >> has) {
        std::vector<int64_t> pos0(n > 0 ? n : 0);
        std::vector<int32_t> counts(pos0.size()), table(pos0.size() * (cols > 0 ? cols : 0)), which(pos0.size());
        for (auto& x : pos0) std::cin >> x;
        for (auto& x : counts) std::cin >> x;
        for (auto& x : table) std::cin >> x;
        if (has) for (auto& x : which) std::cin >> x;
        cc_page_plan_desc d{(int32_t)n, (int32_t)page, (int32_t)cols, pages, slots, pos0.data(), counts.data(), table.data(), has ? which.data() : nullptr};
        PgParts parts;
        const std::string wrong = pg_build(d, parts);
        if (!wrong.empty()) { std::printf("wrong %s\n", wrong.c_str()); continue; }
        std::printf("plan %d %lld %zu\n", parts.n_items, (long long)parts.tokens, parts.segments.size());
        for (auto& g : parts.segments)
            std::printf("%d %d %d %d %d %d %d %d %d %d\n", g.seq, g.block, g.page, g.token0, g.row0, g.rows, g.half, g.flags, g.next, g.pos0);
    }
}
