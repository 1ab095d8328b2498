// CPU test of the batched token mixers' index arithmetic (csrc/q38_paged.hpp): rows of ragged
// batches, pages, and the split of attention's steps into shares. No GPU call is made.
#include "q38_paged.hpp"

#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <set>
#include <vector>

using namespace q38;

static int g_checks = 0;
#define CHECK(x)                                                        \
    do {                                                                \
        ++g_checks;                                                     \
        if (!(x)) {                                                     \
            std::printf("FAILED %s:%d: %s\n", __FILE__, __LINE__, #x);  \
            std::exit(1);                                               \
        }                                                               \
    } while (0)

static void rows_and_pages() {
    const std::vector<int32_t> off = {2, 2, 5, 5, 9};
    CHECK(row_sequence(off.data(), 4, 0) == -1 && row_sequence(off.data(), 4, 1) == -1);
    CHECK(row_sequence(off.data(), 4, 2) == 1 && row_sequence(off.data(), 4, 4) == 1);
    CHECK(row_sequence(off.data(), 4, 5) == 3 && row_sequence(off.data(), 4, 8) == 3);
    CHECK(row_sequence(off.data(), 4, 9) == -1 && row_sequence(off.data(), 0, 0) == -1);
    CHECK(row_span(off.data(), 3, 7).begin == 5 && row_span(off.data(), 3, 7).end == 7);
    const std::vector<int32_t> wild = {-5, 1000, -7, 3};
    for (int i = 0; i < 3; ++i) {
        const RowSpan s = row_span(wild.data(), i, 10);
        CHECK(s.begin >= 0 && s.end >= s.begin && (s.end <= 10 || s.begin == s.end));
    }
    for (int r = 0; r < 12; ++r) {
        const int s = row_sequence(wild.data(), 3, r);
        CHECK(s >= -1 && s < 3);
    }
    // bad pages are never followed; places beyond 2^31 keep their bits
    CHECK(cache_row(-1, 8, 2, 0, 4, 3) == -1 && cache_row(8, 8, 2, 0, 4, 3) == -1 && cache_row(1 << 30, 8, 2, 0, 4, 3) == -1);
    CHECK(cache_row(7, 8, 2, 1, 4, 35) == (7 * 2 + 1) * 16 + 3);
    CHECK(cache_row(3000000, 3000001, 64, 63, 10, 1023) == ((int64_t{3000000} * 64 + 63) << 10) + 1023);
}

static void sums(std::mt19937& rng) {
    for (int n = 0; n < 3000; ++n) {
        const uint32_t m = 1 + rng() % 300, a = rng() % 300, b = rng() % 5000, k = rng() % 200;
        int64_t want = 0;
        for (uint32_t i = 0; i < k; ++i) want += (a * i + b) / m;
        CHECK(floor_sum(k, m, a, b) == want);
    }
    CHECK(floor_sum(1u << 19, 128, 1, (1u << 30)) > 0);
}

// Every step of every item is in exactly one share's piece, in order; pieces that are not whole
// items have a slot of their own; and the joining side finds the same pieces from the cuts.
static void split(std::mt19937& rng, int seqs, int max_rows, int max_tokens, const AttnSplit& S, int W, bool wild) {
    auto pick = [&](int lo, int hi) { return static_cast<int>(rng() % static_cast<unsigned>(hi - lo + 1)) + lo; };
    const int shift = 4, width = max_tokens / 16 + 1;
    std::vector<int32_t> off{pick(0, 2)}, tokens;
    for (int i = 0; i < seqs; ++i) {
        const int n = pick(0, 3) ? pick(0, max_rows) : 0;
        off.push_back(off.back() + n);
        tokens.push_back(pick(0, 4) ? pick(n, std::max(n, max_tokens)) : pick(0, n));
        if (wild && pick(0, 5) == 0) tokens.back() = pick(0, 1) ? -3 : width * 16 + 1;
    }
    const int rows = off.back() + pick(0, 2);
    if (wild) off[static_cast<size_t>(pick(0, seqs))] = pick(-9, rows + 20);
    const PagedBatchDev B{off.data(), tokens.data(), nullptr, seqs, rows, width};
    std::vector<int64_t> start{0};
    for (int i = 0; i < seqs; ++i) {
        AttnItem it;
        attn_sequence(B, shift, i, &it);
        int64_t sum = 0;
        for (int j = 0; j < attn_tiles(S, it.rows); ++j) {
            CHECK(attn_before(S, it, j) == sum);
            attn_tile(S, j, &it);
            sum += it.steps;
        }
        CHECK(attn_weight(S, it) == sum);
        start.push_back(start.back() + sum);
    }
    auto sequence_at = [&](int64_t pos) {
        int seq = 0;
        while (seq < seqs && start[static_cast<size_t>(seq) + 1] <= pos) ++seq;
        return seq;
    };
    auto seek = [&](int seq, int64_t pos) {
        AttnItem it;
        attn_sequence(B, shift, seq, &it);
        return attn_seek(S, it, start[static_cast<size_t>(seq)], pos);
    };
    const int64_t total = start.back(), share = (total + W - 1) / W;
    std::map<std::pair<int, int>, int> seen;  // item -> steps so far
    std::map<std::pair<int, int>, std::set<std::pair<int64_t, int>>> parts;
    for (int64_t w = 0; w < W && w * share < total; ++w) {
        const int64_t end = std::min(total, (w + 1) * share);
        int64_t pos = w * share, before = pos;
        const int seq = sequence_at(pos);
        AttnCursor at = seek(seq, pos);
        std::set<int> slots;
        AttnPiece p;
        while (attn_next(S, B, shift, end, &at, &pos, &p)) {
            CHECK(p.from >= 0 && p.from < p.to && p.to <= p.it.steps && pos - before == p.to - p.from);
            before = pos;
            CHECK(p.it.seq >= 0 && p.it.seq < seqs && p.it.rows > 0 && p.it.tile * S.rows() < p.it.rows);
            CHECK(p.it.first >= 0 && p.it.first + p.it.rows <= rows);
            CHECK(static_cast<int64_t>(p.it.see) <= static_cast<int64_t>(width) * 16);
            CHECK(static_cast<int64_t>(p.it.steps) * S.T >= p.it.see && (p.it.steps - 1) * S.T < std::max(1, p.it.see));
            int& got = seen[{p.it.seq, p.it.tile}];
            CHECK(got == p.from);
            got = p.to;
            if (p.to - p.from < p.it.steps) {
                CHECK(slots.insert(attn_slot(p.start, share, w)).second);
                parts[{p.it.seq, p.it.tile}].insert({w, attn_slot(p.start, share, w)});
            }
        }
        CHECK(pos == end);
    }
    for (int i = 0; i < seqs; ++i) {
        AttnItem it;
        attn_sequence(B, shift, i, &it);
        for (int j = 0; j < attn_tiles(S, it.rows); ++j) {
            attn_tile(S, j, &it);
            CHECK((seen[{i, j}] == it.steps));
        }
    }
    // the joining side: an item is joined once, at the first cut inside it
    std::map<std::pair<int, int>, std::set<std::pair<int64_t, int>>> joined;
    for (int64_t w = 1; w < W && w * share < total; ++w) {
        const int seq = sequence_at(w * share);
        const AttnCursor at = seek(seq, w * share);
        if (at.start == w * share || at.start / share + 1 != w) continue;
        AttnItem it;
        attn_sequence(B, shift, at.seq, &it);
        attn_tile(S, at.tile, &it);
        auto& found = joined[{at.seq, at.tile}];
        CHECK(found.empty());
        for (int64_t v = at.start / share; v <= (at.start + it.steps - 1) / share; ++v) found.insert({v, v < w ? 1 : 0});
    }
    CHECK(joined == parts);
}

int main() {
    rows_and_pages();
    std::mt19937 rng(7);
    sums(rng);
    for (int n = 0; n < 4000; ++n) {
        const int M = 16 << (rng() % 4), G = 1 + static_cast<int>(rng() % (M < 20 ? M : 20));
        const AttnSplit S{G, M, 32 << (rng() % 3)};
        split(rng, 1 + static_cast<int>(rng() % 40), 1 + static_cast<int>(rng() % 50), 1 + static_cast<int>(rng() % 3000), S,
              1 + static_cast<int>(rng() % 300), n & 1);
    }
    std::printf("paged_test: %d checks passed\n", g_checks);
    return 0;
}
