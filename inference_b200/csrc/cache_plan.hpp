// cache_plan.hpp -- how the attention over a bounded paged cache is cut into
// pieces of work, host and device.
//
// Every (sequence, kv head) with slots is a run of 64-slot tiles.  All runs laid
// end to end -- sequences in order, within one its heads, within one its tiles --
// are cut into contiguous chunks.  A run that lies in one chunk is finished there;
// one cut between chunks leaves a part in each, in one of the chunk's two part
// slots: slot 1 if the run begins in the chunk, else slot 0 (a chunk has at most
// one of either kind).  The cuts follow from the lengths alone, so results do not
// depend on which CTA takes a chunk.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define Q3_HD __host__ __device__ __forceinline__
#else
#define Q3_HD inline
#endif

namespace q3 {

constexpr int kPlanTile = 64;
constexpr int kPlanTiers = 34;   // halvings of a 31-bit number, and the ends
constexpr int kPlanSmall = 3;    // tiles of the last tier's chunks

Q3_HD int plan_tiles(int len, int max_len) {
    return len > 0 && len <= max_len ? (len + kPlanTile - 1) / kPlanTile : 0;
}

// Tiers of equal chunks.  With fewer than 8 tiles a worker: one chunk each, sizes
// differing by one tile.  Otherwise 5/8 of the tiles as one chunk each, which the
// workers begin with; the rest is taken as workers become free, every further tier
// half of what is left, down to chunks of 3 tiles: SMs differ in the bandwidth they
// get (on a B200, equal shares of 125 tiles took 157 to 204 us), and what a worker
// finishes late is then at most a small chunk.
struct Plan {
    int total, tiers, chunks;
    int tile0[kPlanTiers + 1], chunk0[kPlanTiers + 1], size[kPlanTiers];
};
Q3_HD void plan_add(Plan& p, int size, int count) {
    if (size <= 0 || count <= 0) return;
    p.size[p.tiers] = size;
    ++p.tiers;
    const long long end = static_cast<long long>(size) * count + p.tile0[p.tiers - 1];
    p.tile0[p.tiers] = end < p.total ? static_cast<int>(end) : p.total;
    p.chunks += count;
    p.chunk0[p.tiers] = p.chunks;
}
Q3_HD void plan_make(Plan& p, int total, int workers) {
    p.total = total;
    p.tiers = p.chunks = 0;
    p.tile0[0] = p.chunk0[0] = 0;
    const int base = total / workers;
    if (base < 8) {
        plan_add(p, base + 1, total - base * workers);
        plan_add(p, base, workers - (total - base * workers));
        return;
    }
    int left = total;
    int size = static_cast<int>(static_cast<long long>(base) * 5 / 8);
    while (size >= kPlanSmall) {
        plan_add(p, size, workers);
        left -= size * workers;
        size = left / (2 * workers);
    }
    plan_add(p, kPlanSmall, (left + kPlanSmall - 1) / kPlanSmall);
}
// No plan of at most `total` tiles has more chunks than this.
Q3_HD int plan_most_chunks(int total, int workers) {
    if (total < workers) return total < 1 ? 1 : total;
    int tiers = 3;  // the first, and less than 2 chunks of 3 tiles a worker left for the last, and one
    for (int base = total / workers; base >= 8; base /= 2) ++tiers;
    return tiers * workers;
}
// Tiles [first, end) of chunk c.
Q3_HD void plan_chunk(const Plan& p, int c, int& first, int& end) {
    int k = 0;
    while (k + 1 < p.tiers && p.chunk0[k + 1] <= c) ++k;
    first = p.tile0[k] + (c - p.chunk0[k]) * p.size[k];
    end = p.tile0[k + 1] - first > p.size[k] ? first + p.size[k] : p.tile0[k + 1];
}
// The chunk that holds tile t.
Q3_HD int plan_chunk_of(const Plan& p, int t) {
    int k = 0;
    while (k + 1 < p.tiers && p.tile0[k + 1] <= t) ++k;
    return p.chunk0[k] + (t - p.tile0[k]) / p.size[k];
}

// `total` tiles in `parts` equal shares (sizes differ by one): the first tile of share
// i, and the share that holds tile t.
Q3_HD int equal_first(int total, int parts, int i) {
    const int base = total / parts, extra = total - base * parts;
    return i * base + (i < extra ? i : extra);
}
Q3_HD int equal_share_of(int total, int parts, int t) {
    const int base = total / parts, extra = total - base * parts, big = extra * (base + 1);
    return t < big ? t / (base + 1) : extra + (t - big) / base;
}

// Rows are scanned in `groups` groups of consecutive rows; before[i] = tiles of one
// head before group i, before[groups] = all.
Q3_HD int plan_group_rows(int rows, int groups) { return (rows + groups - 1) / groups; }

// Tile t: its row, kv head, index in the run, the run's tiles and the row's length.
struct PlanPlace {
    int row, head, tile, tiles, len;
};
Q3_HD PlanPlace plan_locate(int t, const int32_t* lens, int rows, int max_len, int kv_heads, const int* before,
                            int groups) {
    const int u = t / kv_heads;  // lies in the row that holds tile u of one head
    int lo = 0, hi = groups;     // before[lo] <= u < before[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (before[mid] <= u)
            lo = mid;
        else
            hi = mid;
    }
    PlanPlace p;
    p.row = lo * plan_group_rows(rows, groups);
    int first = before[lo];
    for (;;) {
        p.len = lens[p.row];
        p.tiles = plan_tiles(p.len, max_len);
        if (u < first + p.tiles || p.row + 1 >= rows) break;
        first += p.tiles;
        ++p.row;
    }
    const int rem = t - first * kv_heads;
    p.head = rem / p.tiles;
    p.tile = rem - p.head * p.tiles;
    return p;
}

}  // namespace q3
