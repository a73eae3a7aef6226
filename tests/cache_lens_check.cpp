// Checks that the look-up of a tile (csrc/cache_plan.hpp) reads lengths through its
// caller's reader alone, as the joining kernel's read behind the first-level cache needs,
// and reads none outside of the rows; run by test_cache.py.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../inference_b200/csrc/cache_plan.hpp"

using namespace q3;

struct Reader {
    const std::vector<int32_t>* lens;
    mutable int reads = 0;
    int operator[](int r) const {
        ++reads;
        return lens->at(r);
    }
};

int main() {
    const std::vector<int32_t> lens = {0, 130, -3, 64, 1, 500, 0, 65};
    const int rows = static_cast<int>(lens.size()), kvh = 3, max_len = 400;  // 500 is out of range
    for (const int groups : {32, 128}) {
        const int per = plan_group_rows(rows, groups);
        std::vector<int> before(groups + 1, 0);
        for (int i = 0; i < groups; ++i) {
            before[i + 1] = before[i];
            for (int r = i * per; r < rows && r < (i + 1) * per; ++r) before[i + 1] += plan_tiles(lens[r], max_len);
        }
        for (int t = 0; t < before[groups] * kvh; ++t) {
            Reader reader{&lens};
            const PlanPlace a = plan_locate(t, reader, rows, max_len, kvh, before.data(), groups, per);
            const PlanPlace b = plan_locate(t, lens.data(), rows, max_len, kvh, before.data(), groups, per);
            if (reader.reads == 0 || a.row != b.row || a.head != b.head || a.tile != b.tile || a.tiles != b.tiles ||
                a.len != b.len || a.len != lens[a.row]) {
                std::printf("tile %d\n", t);
                return 1;
            }
        }
    }
    std::puts("ok");
}
