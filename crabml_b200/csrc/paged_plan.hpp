// paged_plan.hpp -- the plan of a step over several sequences (include/crabml_paged.h) on the host: every check, and the segments that an append works on.  No CUDA in
// here, so that it is tested without a GPU.
#pragma once
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>
#include <string>
#include <utility>
#include <vector>

#include "../../include/crabml_paged.h"

struct PgSeq { int first, count, pos0, slot; };          // first: its first new token among the call's rows
// new tokens of one sequence that fall into one block: rows row0 .. row0 + rows of the block
struct PgSegment {
    int seq, block, page, token0, row0, rows;
    int half;                                            // where the block lies while it is open: 2 * slot + block % 2
    int flags;                                           // PG_FULL ..
    int next;                                            // the segment that the same CTA takes after this one (-1: none)
    int pos0;                                            // position of the first of its tokens
    int pad[2];
};
#define PG_FULL 1                                        // the block is complete with this call
#define PG_KEPT 2                                        // .. and open, or the one before the open one: its rows stay as 16-bit numbers

struct PgParts {
    std::vector<PgSeq> seqs;
    std::vector<PgSegment> segments;                     // the first n_items are a CTA's first ones
    std::vector<int> table;                              // [n_seqs, table_cols], 0 where no token needs a page
    int n_items = 0;
    int64_t tokens = 0;
};

// "" or what is wrong
inline std::string pg_build(const cc_page_plan_desc& d, PgParts& out) {
    char text[256];
#define PG_NEED(cond, ...)                               \
    do {                                                 \
        if (!(cond)) {                                   \
            snprintf(text, sizeof(text), __VA_ARGS__);   \
            return text;                                 \
        }                                                \
    } while (0)
    typedef long long ll;
    const int P = d.page_size;
    PG_NEED(P == 16 || P == 32 || P == 64 || P == 128, "pages of %d tokens (16, 32, 64 or 128)", P);
    PG_NEED(d.n_seqs >= 0 && d.n_seqs <= (1 << 20) && d.table_cols >= 0 && (int64_t)d.n_seqs * d.table_cols < ((int64_t)1 << 28), "%d sequences of %d pages", d.n_seqs, d.table_cols);
    PG_NEED(d.n_pages >= 0 && d.n_pages < ((int64_t)1 << 31) && d.n_slots >= 0 && d.n_slots < ((int64_t)1 << 30), "%lld pages, %lld slots", (ll)d.n_pages, (ll)d.n_slots);
    auto blocks = [&](int64_t tokens) { return (tokens + P - 1) / P; };
    auto page_of = [&](int i, int64_t b) { return d.table[(int64_t)i * d.table_cols + b]; };
    std::vector<PgSegment> heads, rest;
    std::vector<int64_t> taken;                          // slots
    for (int i = 0; i < d.n_seqs; i++) {
        const int64_t pos0 = d.pos0[i], n = d.counts[i], slot = d.slots ? d.slots[i] : i, most = ((int64_t)1 << 31) - 256;
        PG_NEED(pos0 >= 0 && n >= 0 && pos0 < most && pos0 + n < most, "sequence %d has %lld tokens and %lld new ones", i, (ll)pos0, (ll)n);
        const int64_t end = pos0 + n;
        PG_NEED(blocks(end) <= d.table_cols, "sequence %d of %lld tokens needs more than %d pages", i, (ll)end, d.table_cols);
        PG_NEED(out.tokens + n < ((int64_t)1 << 24), "more than 16 million tokens");
        for (int64_t b = 0; b < blocks(end); b++) PG_NEED(page_of(i, b) >= 0 && page_of(i, b) < d.n_pages, "page %d of sequence %d is not one of %lld", page_of(i, b), i, (ll)d.n_pages);
        if (d.n_slots > 0) {
            PG_NEED(slot >= 0 && slot < d.n_slots, "slot %lld of sequence %d is not one of %lld", (ll)slot, i, (ll)d.n_slots);
            taken.push_back(slot);
        }
        PgSeq s;
        s.first = (int)out.tokens; s.count = (int)n; s.pos0 = (int)pos0; s.slot = d.n_slots > 0 ? (int)slot : 0;
        out.seqs.push_back(s);
        size_t first = 0;                                // the sequence's first segment
        for (int64_t b = pos0 / P; n > 0 && b <= (end - 1) / P; b++) {
            const int64_t lo = std::max(pos0, b * P), hi = std::min(end, (b + 1) * P);
            PgSegment g{};
            g.seq = i; g.block = (int)b; g.page = page_of(i, b);
            g.token0 = s.first + (int)(lo - pos0); g.row0 = (int)(lo - b * P); g.rows = (int)(hi - lo); g.pos0 = (int)lo;
            g.half = 2 * s.slot + (int)(b & 1);
            g.flags = (hi == (b + 1) * P ? PG_FULL : 0) | (b >= end / P - 1 ? PG_KEPT : 0);
            g.next = -1;
            if (b == pos0 / P) first = heads.size();
            const PgSegment* f = b == pos0 / P ? nullptr : &heads[first];
            // a block that is kept overwrites the open rows that the sequence's first block began with, where both lie in one half: the same CTA takes it behind that one (there is
            // one such block at most: of the two that are kept every second lies there)
            if (f && (g.flags & PG_KEPT) && (f->flags & PG_FULL) && f->row0 > 0 && f->half == g.half) {
                heads[first].next = (int)rest.size();
                rest.push_back(g);
            } else heads.push_back(g);
        }
        out.tokens += n;
    }
    std::sort(taken.begin(), taken.end());
    const auto twice = std::adjacent_find(taken.begin(), taken.end());
    PG_NEED(twice == taken.end(), "two sequences with slot %lld", (ll)*twice);
    // pages that take new tokens, with 1 + their sequence: as many places as it needs, not as the pool has (64 sequences of 4000 tokens took 258 us of a pool of a million pages)
    int bits = 10;
    while (((size_t)1 << bits) < 8 * (heads.size() + rest.size())) bits++;
    const size_t places = (size_t)1 << bits;
    std::vector<std::pair<int, int>> owners(places, {0, 0});
    auto owner = [&](int page) -> std::pair<int, int>& {
        size_t at = (uint32_t)page * 2654435769u >> (32 - bits);
        while (owners[at].second && owners[at].first != page) at = (at + 1) & (places - 1);
        return owners[at];
    };
    for (auto* v : {&heads, &rest})
        for (auto& g : *v) {
            auto& o = owner(g.page);
            PG_NEED(!o.second, "page %d takes tokens of two blocks", g.page);
            o = {g.page, 1 + g.seq};
        }
    // no page that takes new tokens may be read by another sequence, nor stand twice in its own row
    for (int i = 0; i < d.n_seqs; i++) {
        const int64_t end = d.pos0[i] + d.counts[i], first_new = d.counts[i] > 0 ? d.pos0[i] / P : blocks(end);
        for (int64_t b = 0; b < blocks(end); b++) {
            const int own = owner(page_of(i, b)).second;
            PG_NEED(own == 0 || (own == 1 + i && b >= first_new), "page %d takes new tokens and is block %lld of sequence %d too", page_of(i, b), (ll)b, i);
        }
    }
#undef PG_NEED
    out.n_items = (int)heads.size();
    for (auto* v : {&heads, &rest})
        for (auto& g : *v)
            if (g.next >= 0) g.next += out.n_items;
    out.segments = heads;
    out.segments.insert(out.segments.end(), rest.begin(), rest.end());
    out.table.assign((size_t)d.n_seqs * d.table_cols, 0);
    for (int i = 0; i < d.n_seqs; i++)
        for (int64_t b = 0; b < blocks(d.pos0[i] + d.counts[i]); b++) out.table[(size_t)((int64_t)i * d.table_cols + b)] = page_of(i, b);
    return "";
}
