// Checks the work shares of the attention over a bounded paged cache
// (csrc/cache_plan.hpp) against a brute-force walk; run by test_cache.py.
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

static void check(const std::vector<int32_t>& lens, int kvh, int max_len, int most, int chunks) {
    const int rows = static_cast<int>(lens.size());
    struct T {
        int row, head, tile, tiles;
        long long run0;
    };
    std::vector<T> all;
    for (int r = 0; r < rows; ++r) {
        const int n = lens[r] > 0 && lens[r] <= max_len ? (lens[r] + 63) / 64 : 0;
        REQUIRE(plan_tiles(lens[r], max_len) == n);
        for (int h = 0; h < kvh; ++h) {
            const long long run0 = static_cast<long long>(all.size());
            for (int i = 0; i < n; ++i) all.push_back({r, h, i, n, run0});
        }
    }
    const long long total = static_cast<long long>(all.size());
    if (total == 0) return;
    std::vector<int> chunk(chunks + 1, 0);
    const int per = plan_chunk_rows(rows, chunks);
    for (int i = 0; i < chunks; ++i) {
        chunk[i + 1] = chunk[i];
        for (int r = i * per; r < rows && r < (i + 1) * per; ++r) chunk[i + 1] += plan_tiles(lens[r], max_len);
    }
    REQUIRE(static_cast<long long>(chunk[chunks]) * kvh == total);
    const int shares = plan_shares(total, most);
    REQUIRE(shares >= 1 && shares <= most);
    REQUIRE(plan_first(total, shares, 0) == 0 && plan_first(total, shares, shares) == total);
    std::set<std::pair<int, int>> used;
    for (int b = 0; b < shares; ++b) {
        const long long t0 = plan_first(total, shares, b), t1 = plan_first(total, shares, b + 1);
        REQUIRE(t1 > t0 && t1 - t0 >= total / shares && t1 - t0 <= total / shares + 1);
        for (long long t = t0; t < t1; ++t) {
            REQUIRE(plan_share(total, shares, t) == b);
            const PlanPlace p = plan_locate(t, lens.data(), rows, max_len, kvh, chunk.data(), chunks);
            const T& w = all[t];
            REQUIRE(p.row == w.row && p.head == w.head && p.tile == w.tile && p.tiles == w.tiles &&
                    p.len == lens[w.row]);
            const bool first = t == t0 || w.tile == 0;
            const bool whole = w.run0 >= t0 && w.run0 + w.tiles <= t1;
            if (first && !whole) {  // a part: its slot is its own
                const int slot = plan_slot(total, shares, b, w.run0);
                REQUIRE(slot == (w.run0 >= t0 ? 1 : 0));
                REQUIRE(used.insert({b, slot}).second);
                // found again from the run alone: the first share in its slot, the others in slot 0
                const int c0 = plan_share(total, shares, w.run0);
                REQUIRE(c0 <= b && b <= plan_share(total, shares, w.run0 + w.tiles - 1));
                REQUIRE(b == c0 ? slot == 1 : slot == 0);
            }
        }
    }
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
        check(lens, pick(1, 9), max_len, pick(1, 300), pick(0, 1) ? 160 : 512);
    }
    check(std::vector<int32_t>(4096, 1), 1, 1, 296, 160);
    check(std::vector<int32_t>(4096, 65), 2, 130, 296, 512);
    check({1000000}, 3, 1 << 20, 296, 160);
    // the largest total stays inside 64 bits
    const long long most = 4096ll * 1024 * 16384;
    REQUIRE(plan_share(most, 296, most - 1) == 295 && plan_first(most, 296, 296) == most);
    std::puts("ok");
}
