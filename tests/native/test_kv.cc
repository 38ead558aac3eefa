// Host tests of the paged cache's index arithmetic and of paged attention's
// plan: every block of every tile is done by exactly one CTA, every key that
// a row sees lies in its tile's blocks, and tables with anything in them give
// nothing outside the rows and pages there are.
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <set>
#include <tuple>
#include <vector>

#include "kernels/attention_plan.h"
#include "kernels/kv_overlap.h"

using namespace mpcomm::kern;

static long g_checks = 0;
#define CHECK(cond)                                                          \
    do {                                                                     \
        ++g_checks;                                                          \
        if (!(cond)) {                                                       \
            std::printf("FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond);    \
            std::exit(1);                                                    \
        }                                                                    \
    } while (0)

static void test_places() {
    std::vector<int32_t> starts{0, 3, 3, 10};
    std::vector<int64_t> table{4, 99, -1, 7, 0, 2};
    KvBatch k;
    k.starts.ptr = starts.data();
    k.table.ptr = table.data();
    k.table.is64 = 1;
    k.table_stride = 2;
    k.table_width = 2;
    k.pages = 8;
    k.seqs = 3;
    k.page_tokens = 5;
    const int want[] = {0, 0, 0, 2, 2, 2, 2, 2, 2, 2, -1, -1};
    for (int r = 0; r < 12; ++r) CHECK(sequence_of(k, r) == want[r]);
    CHECK(page_of(k, 0, 0) == 4 && page_of(k, 0, 4) == 4 && page_of(k, 0, 5) == -1);  // 99 is no page
    CHECK(page_of(k, 1, 0) == -1 && page_of(k, 1, 9) == 7 && page_of(k, 1, 10) == -1 && page_of(k, 2, -1) == -1);
    CHECK(page_of(k, 2, int64_t{1} << 40) == -1);
    k.seqs = 0;
    CHECK(sequence_of(k, 0) == -1);
    // tables that are not ascending still give a sequence there is, or none
    std::mt19937 rng(1);
    for (int t = 0; t < 200; ++t) {
        for (auto &s : starts) s = static_cast<int32_t>(rng());
        k.seqs = 3;
        for (int r = 0; r < 20; ++r) {
            const int b = sequence_of(k, r);
            CHECK(b >= -1 && b < 3);
        }
    }
}

static void test_div() {
    const int64_t v[] = {0, 1, 2, 7, 255, 0x7fffffff, 0xffffffffll, 0x100000000ll, 0x123456789abll, INT64_MAX};
    for (int64_t a : v)
        for (int64_t b : v)
            if (b) CHECK(plan_div(a, b) == a / b);
    std::mt19937 rng(3);
    for (uint32_t d = 1; d < 70000; d += d < 300 ? 1 : 1 + rng() % 97) {
        const FastDiv f(d);
        for (uint32_t n : {0u, 1u, d - 1, d, d + 1, 0x7fffffffu, 0x7fffffffu / d * d, 0x7fffffffu / d * d - 1, static_cast<uint32_t>(rng() >> 1)})
            CHECK(n > 0x7fffffffu || f.div(static_cast<int>(n)) == static_cast<int>(n / d));
    }
    for (uint32_t d : {0x40000000u, 0x7fffffffu, 0x10000001u})
        CHECK(FastDiv(d).div(0x7fffffff) == static_cast<int>(0x7fffffffu / d) && FastDiv(d).div(static_cast<int>(d) - 1) == 0);
}

static void check_plan(const PlanShape &s, const std::vector<int64_t> &starts, const std::vector<int64_t> &lens, int ctas) {
    const int seqs = static_cast<int>(lens.size());
    std::vector<PlanSeq> q;
    int64_t units = 0;
    for (int b = 0; b < seqs; ++b) {
        q.push_back(plan_seq(s, starts[b], starts[b + 1], lens[b]));
        CHECK(q[b].q0 >= 0 && q[b].new_tokens >= 0 && q[b].q0 + q[b].new_tokens <= s.rows);
        CHECK(q[b].end >= 0 && q[b].end <= s.tokens);
        units += s.parts * plan_part_units(s, q[b]);
        int tokens = 0;
        for (int m = 0; m < q[b].tiles; ++m) {
            const PlanTile t = plan_tile(s, q[b], m);
            CHECK(t.tokens > 0 && t.tokens <= 2 * s.tokens_stream && t.blocks > 0 && t.block0 >= 0);
            CHECK(t.lo >= 0 && t.hi <= q[b].end && t.lo <= t.hi);
            CHECK(t.block0 * kBlockKeys <= t.lo && (t.block0 + t.blocks) * kBlockKeys >= t.hi);
            tokens += t.tokens;
            int lo = 1 << 30, hi = 0;
            for (int r = 0; r < t.tokens; ++r) {
                const int at = q[b].first + m * 2 * s.tokens_stream + r;
                int to = q[b].end, from = 0;
                if (s.causal && at + 1 < to) to = at + 1;
                if (s.window && at + 1 - s.window > 0) from = at + 1 - s.window;
                if (from < to) {
                    lo = from < lo ? from : lo;
                    hi = to > hi ? to : hi;
                }
            }
            if (hi) CHECK(t.lo <= lo && t.hi >= hi);
        }
        CHECK(tokens == q[b].new_tokens);
        CHECK(plan_part_units(s, q[b]) == plan_part_units(s, q[b], 0, 3) + plan_part_units(s, q[b], 1, 3) + plan_part_units(s, q[b], 2, 3));
    }
    const int64_t share = plan_share(units, ctas);
    CHECK(share * ctas >= units);
    std::map<std::tuple<int, int, int, int>, int> done;
    for (int c = 0; c < ctas; ++c) {
        int64_t begin = c * share, left = units - begin < share ? units - begin : share;
        if (left <= 0) continue;
        int b = 0;
        int64_t head = 0;
        for (;; ++b) {
            head = plan_part_units(s, q[b]);
            if (begin < s.parts * head) break;
            begin -= s.parts * head;
        }
        PlanCursor cur;
        cur.part = static_cast<int>(plan_div(begin, head));
        begin -= cur.part * head;
        for (; begin >= plan_tile(s, q[b], cur.m).blocks; ++cur.m) begin -= plan_tile(s, q[b], cur.m).blocks;
        cur.block = static_cast<int>(begin);
        while (left > 0) {
            PlanRun run;
            if (!cur.next(s, q[b], left, &run)) {
                ++b;
                CHECK(b < seqs);
                cur = PlanCursor();
                continue;
            }
            CHECK(run.from < run.to && run.to <= run.tile.blocks);
            for (int i = run.from; i < run.to; ++i) ++done[{b, run.part, run.m, i}];
            left -= run.to - run.from;
        }
    }
    CHECK(static_cast<int64_t>(done.size()) == units);
    for (const auto &d : done) CHECK(d.second == 1);
}

static void test_plan() {
    std::mt19937 rng(7);
    auto pick = [&](int lo, int hi) { return lo + static_cast<int>(rng() % (hi - lo + 1)); };
    for (int t = 0; t < 400; ++t) {
        PlanShape s;
        const int group = pick(1, t % 5 ? 9 : 300), kv_heads = pick(1, 4);
        plan_parts(&s, kv_heads, group);
        CHECK(s.parts % kv_heads == 0 && s.heads * s.tokens_stream <= kStreamRows && s.tokens_stream > 0);
        const int each = s.parts / kv_heads;  // every query head is in one part of its key head
        CHECK(s.heads * each >= group && s.heads * (each - 1) < group);
        s.causal = t % 4 != 0;
        s.window = s.causal && t % 3 == 0 ? pick(1, 700) : 0;
        s.tokens = pick(0, 2000);
        const int seqs = pick(1, 12);
        std::vector<int64_t> starts{0}, lens;
        for (int b = 0; b < seqs; ++b) {
            const int n = t % 2 ? pick(0, 2) : pick(0, 300);
            starts.push_back(starts.back() + n);
            lens.push_back(pick(0, 2) ? n + pick(0, 1500) : pick(0, 50));
        }
        s.rows = static_cast<int>(starts.back()) + pick(0, 3);
        if (t % 10 == 9) {  // anything in the tables
            for (auto &v : starts) v = static_cast<int64_t>(rng() % 4000) - 2000;
            for (auto &v : lens) v = static_cast<int64_t>(rng()) << pick(0, 31);
            lens[0] = -lens[0];
        }
        check_plan(s, starts, lens, t % 7 ? 148 : pick(1, 20));
    }
}

// A sequence whose keys go past the columns of the page table, or past a length that positions can have, is marked
// where it has new tokens, and is as long as the table has room for.
static void test_cut() {
    PlanShape s;
    s.rows = 10;
    for (int tokens : {0, 64, kMostTokens})
        for (int64_t len : {int64_t{0}, int64_t{1}, int64_t{64}, int64_t{65}, int64_t{kMostTokens}, int64_t{kMostTokens} + 1, INT64_MAX, int64_t{-5}})
            for (int64_t news : {0, 1, 3})
                for (int causal : {0, 1}) {
                    s.tokens = tokens;
                    s.causal = causal;
                    const PlanSeq q = plan_seq(s, 2, 2 + news, len);
                    CHECK(q.cut == (news > 0 && len > tokens));
                    CHECK(q.end <= tokens && (q.cut || len < 0 || q.end == len || news == 0));
                }
    s.tokens = 64;
    CHECK(!plan_seq(s, 10, 12, 100).cut && !plan_seq(s, 5, 3, 100).cut);  // rows that there are not
}

// Against every byte of both sets.
static void test_overlap() {
    std::mt19937 rng(11);
    auto pick = [&](int lo, int hi) { return lo + static_cast<int>(rng() % (hi - lo + 1)); };
    auto make = [&](bool nested) {
        int64_t e[4], s[4], step = 1;
        for (int k = 3; k >= 0; --k) {
            e[k] = pick(nested ? 1 : 0, 4);
            s[k] = pick(0, 9) ? step : 0;
            step *= e[k] > 0 ? e[k] + pick(0, 2) : 1;
            if (!nested) s[k] = pick(-3, 12);
        }
        return StridedSet(reinterpret_cast<void *>(uintptr_t{1 << 20} + pick(0, 300)),
                          {{s[0], e[0]}, {s[1], e[1]}, {s[2], e[2]}, {s[3], e[3]}});
    };
    auto bytes = [](const StridedSet &a, int size) {
        std::vector<int64_t> at{static_cast<int64_t>(a.base)};
        for (int k = 0; k < a.axes; ++k) {
            const size_t n = at.size();
            for (int64_t i = 1; i < a.extent[k]; ++i)
                for (size_t j = 0; j < n; ++j) at.push_back(at[j] + i * a.stride[k] * size);
        }
        std::set<int64_t> all;
        if (!a.empty)
            for (int64_t p : at)
                for (int b = 0; b < size; ++b) all.insert(p + b);
        return all;
    };
    int met = 0;
    for (int t = 0; t < 20000; ++t) {
        const StridedSet a = make(t % 3), b = make(t % 2);
        const int size = t % 5 ? 2 : 4;
        const auto in_a = bytes(a, size), in_b = bytes(b, size);
        bool meet = false;
        for (int64_t p : in_a) meet = meet || in_b.count(p);
        CHECK(sets_overlap(a, b, size) == meet);
        met += meet;
    }
    CHECK(met > 2000 && met < 18000);
    // large sets are decided by their strides: heads of one projection of 2^20 rows, side by side and one too far
    const int64_t rows = 1 << 20, heads = 8, dim = 128;
    auto part = [&](int64_t first) {
        return StridedSet(reinterpret_cast<void *>((uintptr_t{1} << 40) + first * dim * 2), {{3 * heads * dim, rows}, {dim, heads}, {1, dim}});
    };
    CHECK(!sets_overlap(part(0), part(heads), 2) && !sets_overlap(part(2 * heads), part(0), 2) && sets_overlap(part(0), part(heads - 1), 2));
    CHECK(part(1) == part(1) && !(part(1) == part(2)));
}

int main() {
    test_places();
    test_div();
    test_plan();
    test_cut();
    test_overlap();
    std::printf("ok: %ld checks\n", g_checks);
    return 0;
}
