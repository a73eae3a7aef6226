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
constexpr int kPlanTiered = 32;  // tiles a worker from which on work is taken dynamically
constexpr int kPlanSmall = 3;    // the least tiles of a tier
constexpr int kPlanWhole = 2;    // tiles a worker from which on short runs are spared
constexpr int kPlanSnap = 6;     // runs up to so many tiles are not cut
constexpr int kPlanReach = 3;    // how far a cut moves to spare a run

// n / d for 0 <= n < 2^24, d > 0.
Q3_HD int plan_quotient(int n, int d) {
#ifdef __CUDA_ARCH__
    // the float quotient is off by less than one
    int q = static_cast<int>(__fdividef(static_cast<float>(n), static_cast<float>(d)));
    const int r = n - q * d;
    return q + (r >= d) - (r < 0);
#else
    return n / d;
#endif
}

Q3_HD int plan_tiles(int len, int max_len) {
    return len > 0 && len <= max_len ? (len + kPlanTile - 1) / kPlanTile : 0;
}

// n / d for 0 <= n <= 2^30 from 2^32 / d, rounded up: the product is above the quotient by less than 1 / 4.
inline uint32_t plan_inverse(int d) { return d > 1 ? static_cast<uint32_t>((1ull << 32) / d + 1) : 0; }
Q3_HD int plan_over(int n, int d, uint32_t inverse) {
    if (d == 1) return n;
    const int q = static_cast<int>((static_cast<uint64_t>(n) * inverse) >> 32);
    return q - (q * d > n);
}

// `total` tiles in `parts` equal shares (sizes differ by one): the first tile of share
// i, and the share that holds tile t.
struct Equal {
    int base, extra;
};
Q3_HD Equal equal_make(int total, int parts) {
    Equal e;
    e.base = total / parts;
    e.extra = total - e.base * parts;
    return e;
}
Q3_HD int equal_first(const Equal& e, int i) { return i * e.base + (i < e.extra ? i : e.extra); }
Q3_HD int equal_share_of(const Equal& e, int t) {
    const int big = e.extra * (e.base + 1);
    return t < big ? t / (e.base + 1) : e.extra + (t - big) / e.base;
}

// Every worker (CTA) has an equal region of the tiles.  Its first 5/8 are one chunk,
// which it begins with; the rest is cut into chunks that halve down to 3 tiles and
// are taken by whichever worker is free, the larger ones of all regions first: SMs
// differ in the bandwidth they get (on a B200, whole regions of 128 tiles took 157 to
// 204 us), and what a worker finishes late is at most a small chunk.  Regions below
// 32 tiles stay whole: more cuts cost what they gain.  With tiers and without, 64 sequences
// of up to 8192 slots with 8 kv heads (128 tiles a worker) take 205 and 217 us, one of
// 100001 (42 tiles) 75 and 73; 16 of up to 4096 (16 tiles) take 34.7 us either way.  Halving
// down to 5 tiles instead of 3, the one of 100001 takes 72.8 us for 74.3 and 73 of up to
// 2713 (49 tiles) 80.6 for 79.2.
// Chunk id = tier * workers + region gives the order of taking; the order along the tiles
// is region * tiers + tier.
//
// A cut inside a run costs a part to write and to join, so from two tiles a worker on
// cuts move to a run's nearer end where the run has at most 6 tiles, or the end is at
// most 2 tiles away (plan_down, plan_up).  A chunk may be empty then; those of one run
// are consecutive.  With less work a run's tiles side by side are worth their parts: 5
// tiles in each of 8 runs take 8.7 us apart and 10.3 us together, 64 in each of 8 12.5
// and 14.0 us; from four tiles a worker on instead of two, 200 sequences of 64 .. 500
// slots with one kv head take 19.5 us for 18.6.  Sparing runs of up to 4, 6 and 8 tiles,
// those take 18.4, 17.9 and 18.1 us, and 20 of up to 638 with 8 heads 16.1, 16.0 and 16.5.
Q3_HD int plan_rest(int base) { return base / 8 * 3 + base % 8 * 3 / 8; }
struct Plan {
    Equal region;
    int workers, tiers, chunks;
    int snap, slack;  // runs up to `snap` tiles are not cut; in longer ones cuts move by up to `slack`
};
Q3_HD Plan plan_make(int total, int workers, uint32_t inverse) {
    Plan p;
    p.region.base = plan_over(total, workers, inverse);
    p.region.extra = total - p.region.base * workers;
    p.workers = workers;
    p.tiers = 1;
    p.snap = p.region.base < kPlanWhole ? 0 : kPlanSnap;
    p.slack = p.region.base < kPlanWhole ? 0 : 2;
    if (p.region.base >= kPlanTiered)
        for (int left = plan_rest(p.region.base); left >= kPlanSmall; left /= 2) ++p.tiers;
    p.chunks = p.region.base > 0 ? p.tiers * workers : p.region.extra;
    return p;
}
// The first tile of a tier in its region.
Q3_HD int plan_tier(const Plan& p, int tier) {
    if (tier == 0) return 0;
    return p.region.base - (plan_rest(p.region.base) >> (tier - 1));
}
// Tiles [first, end) of chunk `id`, and its place along the tiles.
Q3_HD void plan_chunk(const Plan& p, int id, int& first, int& end, int& place) {
    int tier = 0, region = id;
    while (region >= p.workers) region -= p.workers, ++tier;
    const int begin = equal_first(p.region, region);
    first = begin + plan_tier(p, tier);
    end = tier + 1 < p.tiers ? begin + plan_tier(p, tier + 1) : equal_first(p.region, region + 1);
    place = region * p.tiers + tier;
}
// The place of the chunk that would hold tile t if no cut moved.
Q3_HD int plan_place_of(const Plan& p, int t) {
    const int region = equal_share_of(p.region, t), at = t - equal_first(p.region, region);
    int tier = 0;
    while (tier + 1 < p.tiers && plan_tier(p, tier + 1) <= at) ++tier;
    return region * p.tiers + tier;
}
// Cuts at most this many tiles behind a run's begin move to it, and cuts at most this
// many tiles before its end to the end.
Q3_HD int plan_down(const Plan& p, int tiles) { return tiles <= p.snap ? (tiles - 1) / 2 : p.slack; }
Q3_HD int plan_up(const Plan& p, int tiles) { return tiles <= p.snap ? tiles / 2 : p.slack; }
// Whether tile run0 + tile of the run [run0, run0 + tiles) lies at or behind a cut that
// the plan has at tile `cut`, wherever that moved.
Q3_HD bool plan_behind(const Plan& p, int run0, int tiles, int tile, int cut) {
    return (cut <= run0 + plan_down(p, tiles)) | ((cut < run0 + tiles - plan_up(p, tiles)) & (run0 + tile >= cut));
}
// The places of the chunks that hold a run's first and last tile: the run's parts are
// in the chunks at these places and between.
Q3_HD void plan_run(const Plan& p, int run0, int tiles, int& first, int& last) {
    first = plan_place_of(p, run0 + plan_down(p, tiles));
    last = plan_place_of(p, run0 + tiles - plan_up(p, tiles) - 1);
}

Q3_HD int plan_log2(int n) {
#ifdef __CUDA_ARCH__
    return 31 - __clz(n);
#else
    return 31 - __builtin_clz(n);
#endif
}
// Rows are scanned in `groups` (at most 256) groups of `per` consecutive rows; before[i] = tiles of
// one head before group i, before[groups] = all.
Q3_HD int plan_group_rows(int rows, int groups) { return (rows + groups - 1) / groups; }

// Tile t: its row, kv head, index in the run, the run's tiles and the row's length.
// lens[r] is how the lengths are read: an array, or what reads it in a way of its own.
struct PlanPlace {
    int row, head, tile, tiles, len;
};
template <class Lens>
Q3_HD PlanPlace plan_locate(int t, const Lens& lens, int rows, int max_len, int kv_heads, const int* before, int groups,
                            int per) {
    // lies in the row that holds tile u of one head
    const int u = (kv_heads & (kv_heads - 1)) == 0 ? t >> plan_log2(kv_heads) : t / kv_heads;
    // the last group that begins at or before u, by steps of 32, 4 and 1 groups whose loads do not wait for
    // one another
    int lo = 0;
    for (int step = groups > 32 ? 32 : 4; step >= 1; step = step == 32 ? 4 : step == 4 ? 1 : 0) {
        int n = 0;
#ifdef __CUDA_ARCH__
#pragma unroll
#endif
        for (int j = 1; j < 8; ++j)
            if (lo + j * step < groups) n += before[lo + j * step] <= u;
        lo += n * step;
    }
    PlanPlace p;
    p.row = lo * per;
    int first = before[lo];
    for (;;) {
        p.len = lens[p.row];
        p.tiles = plan_tiles(p.len, max_len);
        if (u < first + p.tiles || p.row + 1 >= rows) break;
        first += p.tiles;
        ++p.row;
    }
    const int rem = t - first * kv_heads;
    p.head = plan_quotient(rem, p.tiles);
    p.tile = rem - p.head * p.tiles;
    return p;
}

}  // namespace q3
