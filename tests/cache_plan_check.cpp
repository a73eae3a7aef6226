// Checks the work shares of the attention over a bounded paged cache
// (csrc/cache_plan.hpp) against a brute-force walk; run by test_cache.py.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <set>
#include <utility>
#include <vector>

#include "../inference_b200/csrc/cache_plan.hpp"

using namespace q3;

#define REQUIRE(x)                                             \
    do {                                                       \
        if (!(x)) {                                            \
            std::printf("line %d: %s\n", __LINE__, #x);        \
            std::exit(1);                                      \
        }                                                      \
    } while (0)

static void check_totals(int total, int workers) {
    const Plan p = plan_make(total, workers, plan_inverse(workers));
    REQUIRE(p.region.base == total / workers && p.region.extra == total % workers);
    REQUIRE(p.tiers >= 1 && p.tiers <= 31 && p.chunks <= p.tiers * workers);
    REQUIRE(plan_make(total + 5, workers, plan_inverse(workers)).tiers >= p.tiers);  // the workspace's bound
    std::vector<std::pair<int, int>> at(static_cast<size_t>(p.tiers) * workers, {-1, -1});
    for (int id = 0; id < p.chunks; ++id) {
        int first = 0, end = 0, place = 0;
        plan_chunk(p, id, first, end, place);
        REQUIRE(first < end && end <= total && place >= 0 && place < p.tiers * workers);
        REQUIRE(at[place].first < 0);
        at[place] = {first, end};
        REQUIRE(plan_place_of(p, first) == place && plan_place_of(p, end - 1) == place);
        REQUIRE(p.region.base < kPlanTiered || end - first >= kPlanSmall);
    }
    int next = 0;
    for (const auto& c : at)
        if (c.first >= 0) {
            REQUIRE(c.first == next);
            next = c.second;
        }
    REQUIRE(next == total);
    for (const int parts : {1, 7, workers, 4 * workers}) {
        const Equal e = equal_make(total, parts);
        REQUIRE(equal_first(e, 0) == 0 && equal_first(e, parts) == total);
        for (int i = 0; i < parts; ++i) {
            const int a = equal_first(e, i), b = equal_first(e, i + 1);
            REQUIRE(a <= b);
            if (a < b) REQUIRE(equal_share_of(e, a) == i && equal_share_of(e, b - 1) == i);
        }
    }
}

static void check(const std::vector<int32_t>& lens, int kvh, int max_len, int workers, int groups) {
    const int rows = static_cast<int>(lens.size());
    struct T {
        int row, head, tile, tiles, run0;
    };
    std::vector<T> all;
    for (int r = 0; r < rows; ++r) {
        const int n = lens[r] > 0 && lens[r] <= max_len ? (lens[r] + 63) / 64 : 0;
        REQUIRE(plan_tiles(lens[r], max_len) == n);
        for (int h = 0; h < kvh; ++h) {
            const int run0 = static_cast<int>(all.size());
            for (int i = 0; i < n; ++i) all.push_back({r, h, i, n, run0});
        }
    }
    const int total = static_cast<int>(all.size());
    check_totals(total, workers);
    const Plan plan = plan_make(total, workers, plan_inverse(workers));
    std::vector<int> before(groups + 1, 0);
    const int per = plan_group_rows(rows, groups);
    for (int i = 0; i < groups; ++i) {
        before[i + 1] = before[i];
        for (int r = i * per; r < rows && r < (i + 1) * per; ++r) before[i + 1] += plan_tiles(lens[r], max_len);
    }
    REQUIRE(before[groups] * kvh == total);
    // every tile in exactly one chunk, found within reach of the unmoved chunk; a run's tiles in the chunks at
    // its places, each with a tile of it at least; a short run in one chunk
    std::vector<int> owner(total, -1);
    std::set<std::pair<int, int>> used;
    int next = 0;  // chunks in order of their places hold the tiles in order
    std::vector<std::pair<int, int>> order;
    for (int c = 0; c < plan.chunks; ++c) {
        int t0 = 0, t1 = 0, place = 0;
        plan_chunk(plan, c, t0, t1, place);
        order.push_back({place, c});
    }
    std::sort(order.begin(), order.end());
    for (const auto& o : order) {
        int t0 = 0, t1 = 0, place = 0;
        plan_chunk(plan, o.second, t0, t1, place);
        for (int t = t0 - kPlanReach < 0 ? 0 : t0 - kPlanReach; t < total && t < t1 + kPlanReach; ++t) {
            const PlanPlace p = plan_locate(t, lens.data(), rows, max_len, kvh, before.data(), groups, per);
            const T& w = all[t];
            REQUIRE(p.row == w.row && p.head == w.head && p.tile == w.tile && p.tiles == w.tiles &&
                    p.len == lens[w.row]);
            const bool here = plan_behind(plan, w.run0, w.tiles, w.tile, t0) && (t1 == total || !plan_behind(plan, w.run0, w.tiles, w.tile, t1));
            if (!here) continue;
            REQUIRE(owner[t] < 0 && t == next);
            owner[t] = place;
            ++next;
            int c0 = 0, c1 = 0;
            plan_run(plan, w.run0, w.tiles, c0, c1);
            REQUIRE(c0 <= place && place <= c1);
            if (w.tile == 0) REQUIRE(place == c0);
            if (w.tile == w.tiles - 1) REQUIRE(place == c1);
            if (w.tiles <= plan.snap) REQUIRE(c0 == c1);
            if (c0 != c1 && (w.tile == 0 || owner[t - 1] != place)) {  // a part: its slot is its own
                REQUIRE(place == c0 || owner[t - 1] == place - 1);
                REQUIRE(used.insert({place, place == c0 ? 1 : 0}).second);
            }
        }
    }
    REQUIRE(next == total);
}

int main() {
    std::mt19937 rng(1);
    auto pick = [&](int lo, int hi) { return lo + static_cast<int>(rng() % (hi - lo + 1)); };
    for (int i = 0; i < 400; ++i) {
        const int rows = pick(1, i % 5 ? 40 : 700), max_len = pick(1, 3000);
        std::vector<int32_t> lens(rows);
        for (auto& n : lens) {
            const int kind = pick(0, 9);
            n = kind == 0 ? 0 : kind == 1 ? -pick(1, 100) : kind == 2 ? max_len + pick(1, 9) : pick(0, max_len);
        }
        check(lens, pick(1, 9), max_len, pick(1, 300), std::vector<int>{32, 128, 160}[pick(0, 2)]);
    }
    check({20000, 3, 500, 9000, 512, 513, 20000}, 3, 20000, 20, 160);
    check(std::vector<int32_t>(4096, 1), 1, 1, 296, 160);
    check(std::vector<int32_t>(4096, 65), 2, 130, 296, 128);
    check({1000000}, 3, 1 << 20, 296, 160);
    check({0, -1, 500}, 3, 100, 296, 160);
    for (int t = 0; t < 3000; ++t) check_totals(t, pick(1, 400));
    for (const int workers : {1, 2, 147, 296, 1000})
        for (const int t : {7 * workers, 8 * workers - 1, 8 * workers, 8 * workers + 1, 1000 * workers + 5, 1 << 24, 1 << 30})
            check_totals(t, workers);
    std::puts("ok");
}
