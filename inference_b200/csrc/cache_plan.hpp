// cache_plan.hpp -- how the attention over a bounded paged cache is cut into
// equal shares, host and device.
//
// Every (sequence, kv head) with slots is a run of 64-slot tiles.  All runs laid
// end to end -- sequences in order, within one its heads, within one its tiles --
// are cut into `shares` contiguous shares whose sizes differ by one tile at
// most.  A run that lies in one share is finished there; one cut between shares
// leaves a part in each, in one of the share's two part slots: slot 1 if the run
// begins in the share, else slot 0 (a share has at most one of either kind).
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define Q3_HD __host__ __device__ __forceinline__
#else
#define Q3_HD inline
#endif

namespace q3 {

constexpr int kPlanTile = 64;

Q3_HD int plan_tiles(int len, int max_len) {
    return len > 0 && len <= max_len ? (len + kPlanTile - 1) / kPlanTile : 0;
}
// No share of a total above 0 is empty: a run's shares are consecutive.
Q3_HD int plan_shares(long long total, int most) {
    return total < 1 ? 1 : total < most ? static_cast<int>(total) : most;
}
// Tiles [first, next first) of share b of `total` tiles.
Q3_HD long long plan_first(long long total, int shares, int b) { return total * b / shares; }
// The share that holds tile t.
Q3_HD int plan_share(long long total, int shares, long long t) {
    return static_cast<int>(((t + 1) * shares - 1) / total);
}
// The part slot of a run beginning at tile run0 in share b.
Q3_HD int plan_slot(long long total, int shares, int b, long long run0) {
    return run0 >= plan_first(total, shares, b) ? 1 : 0;
}


// Rows are scanned in `chunks` chunks of consecutive rows; chunk[i] = tiles of one
// head before chunk i, chunk[chunks] = all.
Q3_HD int plan_chunk_rows(int rows, int chunks) { return (rows + chunks - 1) / chunks; }

// Tile t: its row, kv head, index in the run, the run's tiles and the row's length.
struct PlanPlace {
    int row, head, tile, tiles, len;
};
Q3_HD PlanPlace plan_locate(long long t, const int32_t* lens, int rows, int max_len, int kv_heads, const int* chunk,
                            int chunks) {
    const int u = static_cast<int>(t / kv_heads);  // lies in the row that holds tile u of one head
    int lo = 0, hi = chunks;                       // chunk[lo] <= u < chunk[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (chunk[mid] <= u)
            lo = mid;
        else
            hi = mid;
    }
    PlanPlace p;
    p.row = lo * plan_chunk_rows(rows, chunks);
    int before = chunk[lo];
    for (;;) {
        p.len = lens[p.row];
        p.tiles = plan_tiles(p.len, max_len);
        if (u < before + p.tiles || p.row + 1 >= rows) break;
        before += p.tiles;
        ++p.row;
    }
    const int rem = static_cast<int>(t - static_cast<long long>(before) * kv_heads);
    p.head = rem / p.tiles;
    p.tile = rem - p.head * p.tiles;
    return p;
}

}  // namespace q3
