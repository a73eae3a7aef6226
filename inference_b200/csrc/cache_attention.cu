// cache_attention.cu -- attention of one query token per sequence over a bounded
// paged cache, with the attention every slot receives accumulated.
//
//   s_gj = q_g . k_j / sqrt(128);  p_gj = 2^(s_gj log2 e - m_g) / l_g
//   out_g = sum_j p_gj v_j;  weight_j += sum_g p_gj   (g: the kv head's query heads)
//
// Bound: HBM.  K and V of every slot cross it once (512 bytes a slot and kv head)
// for 512 G flops; everything else is two orders smaller.  So:
//   * all sequences' 64-slot tiles are cut into chunks (cache_plan.hpp) from the
//     lengths in device memory, so one launch shape serves any mix of lengths; two
//     CTAs an SM take chunks as they become free;
//   * in a CTA one warp streams K and V tiles through a ring of 32 KB stages by
//     swizzled 2-D TMA (a last, partial tile by boxes of 16 slots), reading page
//     table entries for 32 tiles at a time; four warps take 16 slots of a tile
//     each: S^T = K Q^T and O^T += V^T P^T on the tensor cores with the slots as
//     M and the group's query heads as N, online softmax in fp32, P as the sum of
//     three BF16 parts, which is exact (with two parts, off by up to 2^-17 of P, 0.2 %
//     of the outputs are not the nearest BF16 value, with three 0.02 to 0.15 %; the
//     third costs 200 x <= 500 slots 0.25 us, the other cases 0 to 0.2 us);
//   * a run (sequence, kv head) within one chunk is finished there; parts of a cut
//     run (maximum, sum, unnormalised output in fp32) are joined by the second
//     kernel in chunk order, so results do not depend on timing;
//   * probabilities need the run's final maximum and sum: the first kernel leaves
//     the raw scores (fp32, 4 G bytes a slot, written once and mostly read back
//     from L2), the second turns them into weights.
//
// mma.sync, not tcgen05: with G of 1 .. 16 query heads a 64-slot tile's two products
// are 2 x 64 x 128 x 8 .. 16 multiply-adds against 32 KB to load, and S, P and O stay in
// registers from one product to the next; ncu has the tensor pipe far from busy.
//
// Measured (B200, captured into a graph, weights accumulated but for the long one; the
// share is that of the bytes above at the measured copy rate of 6.55 TB/s):
//   64 sequences of 1118 .. 8192, 32 / 8 heads  204 us, 94 % (without weights 182 us; K and
//                                             V are 1.24 GB, and the first kernel reads no
//                                             more)
//   one of 100001 slots, 64 / 8 heads          74 us, 84 %
//   16 of 635 .. 4096, 32 / 8 heads            35 us, 68 %  (join 7 us)
//   200 of 64 .. 500, 8 / 1 heads              18.1 us, 25 % (a worker's longest uncut run
//                                             at 1 us a tile, start, join)
//   one of 4095, 32 / 8 heads                  11.1 us      start, look-ups, one tile's
//   one of 300, 16 / 8 heads                   7.8 us       latency, join
// One kernel with a grid barrier in place of the second launch cost 2.3 us where the
// programmatic launch costs 0.7; letting the last part of a run find its maximum and sum
// (a fence and an atomic a part) took 50 us instead of 43 at 16 x 4096.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "cache.cuh"
#include "cache_plan.hpp"
#include "mma.cuh"

namespace q3 {
namespace {

constexpr int kWarps = 4;                      // consumer warps, 16 slots of a tile each
constexpr int kConsumers = kWarps * 32;
constexpr int kThreads = kConsumers + 32;      // + producer warp
constexpr int kTileBytes = kCachePage * kCacheHd * 2;
constexpr int kAccPitch = kCacheHd + 4;         // floats of a head in the merge buffer: conflict-free
constexpr float kScoreScale = 0.08838834764831845f * 1.4426950408889634f;  // log2(e) / sqrt(128)

// What the producer tells the consumers about a stage's tile.
enum : int {
    TILE_FIRST = 1,  // first tile of its run in this chunk
    TILE_LAST = 2,   // last tile of its run in this chunk
    TILE_WHOLE = 4,  // the run lies in this chunk
    TILE_BEGIN = 8,  // the run begins in this chunk
    TILE_BAD = 16,   // its page lies outside the pool: nothing was loaded
    TILE_END = 32,   // no tile: the CTA is done
};

// NT: 8-head column tiles (1: up to 8 query heads per kv head, 2: up to 16).
template <int NT>
struct Cfg {
    static constexpr int kHeads = 8 * NT;
    static constexpr int kStages = NT == 1 ? 3 : 2;
    static constexpr int kStageBytes = 2 * kTileBytes + kHeads * kCacheHd * 2;
};

template <int NT>
struct Smem {
    // K tile, V tile, the run's queries (first tile only); after a run's last tile the
    // stage is where the warps' outputs meet ([warp][head][kAccPitch] floats)
    uint8_t ring[Cfg<NT>::kStages][Cfg<NT>::kStageBytes];
    float m[kWarps][Cfg<NT>::kHeads], l[kWarps][Cfg<NT>::kHeads];
    int4 tile[Cfg<NT>::kStages];        // row, head, tile, flags | live slots << 8 | chunk's place << 16
    uint64_t full[Cfg<NT>::kStages], empty[Cfg<NT>::kStages];
    int before[kThreads + 1];           // tiles before each group of rows
    int scan[kThreads / 32];
};
static_assert(kWarps * Cfg<1>::kHeads * kAccPitch * 4 <= Cfg<1>::kStageBytes, "merge buffer");
static_assert(kWarps * Cfg<2>::kHeads * kAccPitch * 4 <= Cfg<2>::kStageBytes, "merge buffer");

struct Parts {
    float2* ml;    // [rows][q_heads]: maximum (log2) and 1 / sum of runs within one chunk (0: a bad page)
    float2* pml;   // [chunk's place][2][G]: maximum and sum of parts
    float* po;     // [chunk's place][2][G][128]: unnormalised outputs of parts
    float* score;  // [tile][64][G]: raw scores in log2 units
    int workers;
    uint32_t inverse;  // of workers
};

// 2^x by the exponential unit: off by 2 units of 2^-23 at most, results below 2^-126 are 0.
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two BF16 values, infinities and NaN replaced by the largest finite value (with the sign
// that they have).
__device__ __forceinline__ uint32_t clamp_bf2(uint32_t x) {
    uint32_t y;
    asm("min.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(0x7F7F7F7Fu));
    return y;
}

// Groups of consecutive rows, one per thread: before[t] = tiles (of one kv head)
// before thread t's rows, before[threads] = all.
template <int THREADS, class Lens>
__device__ __forceinline__ void scan_rows(const Lens& lens, const CacheView& c, int* before, int* scan) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int per = plan_group_rows(c.rows, THREADS);
    int sum = 0;
    for (int r = tid * per; r < min(c.rows, tid * per + per); ++r) sum += plan_tiles(lens[r], c.max_len);
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
    }
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    for (int i = 0; i < warp; ++i) incl += scan[i];
    before[tid + 1] = incl;
    if (tid == 0) before[0] = 0;
    __syncthreads();
}

// The same by one warp, in 32 groups: `per` rows a lane.
__device__ __forceinline__ void scan_rows_warp(const int32_t* lens, const CacheView& c, int per, int* before) {
    const int lane = threadIdx.x & 31;
    int incl = 0;
#pragma unroll 4
    for (int r = lane * per; r < min(c.rows, lane * per + per); ++r) incl += plan_tiles(lens[r], c.max_len);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
    }
    before[lane + 1] = incl;
    if (lane == 0) before[0] = 0;
    __syncwarp();
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

__device__ __forceinline__ void tma_tile(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
        " [%0], [%1, {%2, %3}], [%4], %5;" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar)), "l"(policy)
        : "memory");
}

template <int NT>
__global__ void __maxnreg__(NT == 1 ? 128 : 168)
    cache_attention_kernel(const __grid_constant__ CacheAttnArgs a, const __grid_constant__ CacheMaps maps,
                           const __grid_constant__ Parts parts) {
    using C = Cfg<NT>;
    constexpr int S = C::kStages;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    Smem<NT>& sm = *reinterpret_cast<Smem<NT>*>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
    const CacheView& c = a.c;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = a.q_heads / c.kv_heads;
    if (tid == kConsumers) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&sm.full[s], 1);
            mbar_init(&sm.empty[s], kWarps);
        }
        fence_barrier_init();
        prefetch_map(&maps.k64);
        prefetch_map(&maps.v64);
        prefetch_map(&maps.k16);
        prefetch_map(&maps.v16);
    }
    __syncthreads();  // the barriers are set up
    pdl_wait();     // what ran before may have written the lengths, queries and pages
    pdl_trigger();  // the joining kernel may set itself up; it waits for this one's end
    // only the producer looks tiles up: few rows it scans by itself
    const bool few = c.rows <= 256;
    if (!few) scan_rows<kThreads>(a.lens, c, sm.before, sm.scan);

    if (warp == kWarps) {
        // ------------------------------------------------------------ producer
        const int groups = few ? 32 : kThreads;
        const int per = few ? (c.rows + 31) / 32 : plan_group_rows(c.rows, kThreads);
        if (few) scan_rows_warp(a.lens, c, per, sm.before);
        const int total = sm.before[groups] * c.kv_heads;
        const Plan plan = plan_make(total, parts.workers, parts.inverse);
        const uint64_t pol = policy_evict_first();
        int k = 0, s = 0, round = 0;  // tiles sent for; the stage for the next, used `round` times before
        bool ok = true;
        auto stage_free = [&]() {
            return round == 0 || mbar_wait(&sm.empty[s], (round - 1) & 1, c.err, DEV_TMA_WAIT_TIMEOUT);
        };
        int chunk = blockIdx.x;
        while (ok && chunk < plan.chunks) {
            int t0, t1, place;
            plan_chunk(plan, chunk, t0, t1, place);
            // the chunk's cuts may have moved by up to kPlanReach tiles
            const int stop = min(total, t1 + kPlanReach);
            for (int i0 = max(0, t0 - kPlanReach); i0 < stop && ok; i0 += 32) {
                // lane i: tile i0 + i
                int4 d = make_int4(0, 0, 0, 0);
                int y = 0;
                bool here = false;
                if (i0 + lane < stop) {
                    const int t = i0 + lane;
                    const PlanPlace p = plan_locate(t, a.lens, c.rows, c.max_len, c.kv_heads, sm.before, groups, per);
                    const int run0 = t - p.tile;
                    auto behind = [&](int tile, int cut) { return plan_behind(plan, run0, p.tiles, tile, cut); };
                    here = behind(p.tile, t0) && (t1 == total || !behind(p.tile, t1));
                    const bool begins = behind(0, t0), ends = t1 == total || !behind(p.tiles - 1, t1);
                    int flags = 0;
                    if (p.tile == 0 || !behind(p.tile - 1, t0)) flags |= TILE_FIRST;
                    if (p.tile == p.tiles - 1 || (t1 < total && behind(p.tile + 1, t1))) flags |= TILE_LAST;
                    if (begins && ends) flags |= TILE_WHOLE;
                    if (begins) flags |= TILE_BEGIN;
                    const int page = here ? c.tables[p.row * c.table_stride + p.tile] : 0;
                    if (page < 0 || page >= c.num_pages) {
                        flags |= TILE_BAD;
                        record_error(c.err, DEV_BAD_PAGE);
                    } else {
                        y = (page * c.kv_heads + p.head) * kCachePage;
                    }
                    d = make_int4(p.row, p.head, t, flags | min(kCachePage, p.len - p.tile * kCachePage) << 8 | place << 16);
                }
                // each lane sends for its own tile in turn
                for (unsigned left = __ballot_sync(0xffffffffu, here); left && ok; left &= left - 1) {
                    const int i = __ffs(left) - 1;
                    if (lane == i) {
                        ok = stage_free();
                        if (ok) {
                            sm.tile[s] = d;
                            if (d.w & TILE_BAD) {
                                mbar_arrive(&sm.full[s]);
                            } else {
                                uint8_t* st = sm.ring[s];
                                const int boxes = (((d.w >> 8) & 127) + 15) / 16;  // of 16 slots
                                const uint32_t q_bytes = (d.w & TILE_FIRST) ? G * kCacheHd * 2 : 0;
                                mbar_arrive_expect_tx(&sm.full[s], boxes * (2 * 16 * kCacheHd * 2) + q_bytes);
                                if (boxes == 4) {
                                    for (int h = 0; h < 2; ++h) {
                                        tma_tile(st + h * 8192, &maps.k64, h * 64, y, &sm.full[s], pol);
                                        tma_tile(st + kTileBytes + h * 8192, &maps.v64, h * 64, y, &sm.full[s], pol);
                                    }
                                } else {
                                    for (int x = 0; x < boxes; ++x)
                                        for (int h = 0; h < 2; ++h) {
                                            uint8_t* to = st + h * 8192 + x * 2048;
                                            tma_tile(to, &maps.k16, h * 64, y + 16 * x, &sm.full[s], pol);
                                            tma_tile(to + kTileBytes, &maps.v16, h * 64, y + 16 * x, &sm.full[s], pol);
                                        }
                                }
                                if (q_bytes)
                                    bulk_g2s(st + 2 * kTileBytes,
                                             a.q + d.x * a.q_stride + static_cast<size_t>(d.y) * G * kCacheHd, q_bytes,
                                             &sm.full[s], pol);
                            }
                        }
                    }
                    ok = __shfl_sync(0xffffffffu, ok, i);
                    if (ok) {
                        ++k;
                        if (++s == S) s = 0, ++round;
                    }
                }
            }
            // the next chunk, when this one's last copies are on their way: whoever is free first takes it
            int next = plan.chunks;
            if (lane == 0 && plan.chunks > gridDim.x) next = gridDim.x + static_cast<int>(atomicAdd(c.next_chunk, 1u));
            chunk = __shfl_sync(0xffffffffu, next, 0);
        }
        if (lane == 0) {
            ok = ok && stage_free();
            if (ok) {
                sm.tile[s].w = TILE_END;
                mbar_arrive(&sm.full[s]);
            } else {
                // a wait ran out: leave no copy in flight behind
                for (int i = max(0, k - S); i < k; ++i) mbar_wait(&sm.full[i % S], (i / S) & 1, nullptr, 0);
            }
        }
        return;
    }

    // sequences without a tile: length 0 gives zeros, a length out of range NaN
    for (int r = blockIdx.x; r < c.rows; r += gridDim.x) {
        const int len = a.lens[r];
        if (len > 0 && len <= c.max_len) continue;
        if (len != 0 && tid == 0) record_error(c.err, DEV_BAD_LENGTH);
        const uint32_t v = len == 0 ? 0u : 0x7FC07FC0u;
        uint4* o = reinterpret_cast<uint4*>(a.out + r * a.out_stride);
        for (int i = tid; i < a.q_heads * kCacheHd / 8; i += kConsumers) o[i] = make_uint4(v, v, v, v);
    }

    // ---------------------------------------------------------------- consumers
    const int g = lane >> 2, t4 = lane & 3;  // fragment row and column pair
    uint32_t qf[NT][8][2];                   // Q^T as the B operand: dims 16 kk + 2 t4 (+ 8), head 8 nt + g
    float o[NT][8][4];                       // O^T: dims 16 dt + g (+ 8), heads 8 nt + 2 t4 (+ 1)
    float m_run[NT][2], l_run[NT][2];        // of those heads: maximum (log2), this lane's share of the sum
    bool poisoned = false;
    // this lane's place in a tile's scores; whether it has a second head, and pairs are 8-byte aligned
    float* const score_lane = parts.score + static_cast<size_t>(warp * 16 + g) * G + 2 * t4;
    const size_t score_tile = static_cast<size_t>(kCachePage) * G;
    const bool pairs = G % 2 == 0;
    for (int s = 0, round = 0;; ++s == S ? (s = 0, ++round) : 0) {
        // All four warps go on or none: a wait that ran out in one of them ends them all, as the last tile does.
        if (!mbar_wait(&sm.full[s], round & 1, c.err, DEV_TMA_WAIT_TIMEOUT)) sm.tile[s].w = TILE_END;
        named_bar(1, kConsumers);
        const int4 d = sm.tile[s];
        if (d.w & TILE_END) return;
        uint8_t* kt = sm.ring[s];
        uint8_t* vt = kt + kTileBytes;
        if (d.w & TILE_FIRST) {
            poisoned = false;
            const uint32_t* q = reinterpret_cast<const uint32_t*>(kt + 2 * kTileBytes);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const bool in = nt * 8 + g < G;
#pragma unroll
                for (int kk = 0; kk < 8; ++kk) {
                    qf[nt][kk][0] = in ? q[(nt * 8 + g) * 64 + kk * 8 + t4] : 0u;
                    qf[nt][kk][1] = in ? q[(nt * 8 + g) * 64 + kk * 8 + 4 + t4] : 0u;
                }
#pragma unroll
                for (int dt = 0; dt < 8; ++dt) o[nt][dt][0] = o[nt][dt][1] = o[nt][dt][2] = o[nt][dt][3] = 0.f;
                m_run[nt][0] = m_run[nt][1] = -INFINITY;
                l_run[nt][0] = l_run[nt][1] = 0.f;
            }
        }
        if (d.w & TILE_BAD) poisoned = true;
        const int valid = (d.w >> 8) & 127;
        bool wrote = false;
        if (warp * 16 < valid && !(d.w & TILE_BAD)) {
            if (valid < warp * 16 + 16) {
                // slots behind the length become zeros in V (their P is 0, they may hold NaN)
                for (int r = valid; r < warp * 16 + 16; ++r)
                    reinterpret_cast<uint2*>(vt + (lane >> 4) * 8192 + r * 128)[lane & 15] = make_uint2(0u, 0u);
                __syncwarp();
                wrote = true;
            }
            // ---- S^T = K Q^T, even and odd k-steps apart
            float sa[NT][4], sb[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) sa[nt][e] = sb[nt][e] = 0.f;
            {
                const int q = lane >> 3, row = warp * 16 + (q & 1) * 8 + (lane & 7);
#pragma unroll
                for (int kk = 0; kk < 8; ++kk) {
                    uint32_t a0, a1, a2, a3;
                    ldmatrix_x4(kt + tile_off(row, kk * 2 + (q >> 1)), a0, a1, a2, a3);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        mma_bf16_16816((kk & 1) ? sb[nt] : sa[nt], a0, a1, a2, a3, qf[nt][kk][0], qf[nt][kk][1]);
                }
            }
            uint32_t pf[NT][3][2];
            float score[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                // slots g (elements 0, 1) and g + 8 (2, 3), heads 2 t4 (0, 2) and 2 t4 + 1 (1, 3)
                const int tok = warp * 16 + g;
                float sc[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    sc[e] = tok + (e >> 1) * 8 < valid ? (sa[nt][e] + sb[nt][e]) * kScoreScale : -INFINITY;
                float mx[2] = {fmaxf(sc[0], sc[2]), fmaxf(sc[1], sc[3])};
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) {
                    mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], off));
                    mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], off));
                }
                float p[4], corr[2];
#pragma unroll
                for (int e = 0; e < 4; ++e) score[nt][e] = sc[e];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float mn = fmaxf(m_run[nt][j], mx[j]);
                    // nothing above -infinity yet: the exponentials' base is 0, not -infinity
                    const float base = mn == -INFINITY ? 0.f : mn;
                    corr[j] = ex2(m_run[nt][j] - base);
                    p[j] = ex2(sc[j] - base);
                    p[j + 2] = ex2(sc[j + 2] - base);
                    m_run[nt][j] = mn;
                    l_run[nt][j] = l_run[nt][j] * corr[j] + p[j] + p[j + 2];
                }
                // a new maximum (seldom after a run's first tiles) rescales what there is
                if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
                    for (int dt = 0; dt < 8; ++dt) {
                        o[nt][dt][0] *= corr[0];
                        o[nt][dt][1] *= corr[1];
                        o[nt][dt][2] *= corr[0];
                        o[nt][dt][3] *= corr[1];
                    }
                }
                // P as the sum of three BF16 parts, 8 of its 24 bits each: nothing is rounded
                uint32_t part[3][4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float left = p[e];
#pragma unroll
                    for (int i = 0; i < 3; ++i) {
                        part[i][e] = __float_as_uint(left);
                        left -= __uint_as_float(part[i][e] & 0xFFFF0000u);
                    }
                }
#pragma unroll
                for (int i = 0; i < 3; ++i) {
                    pf[nt][i][0] = movmatrix_trans(__byte_perm(part[i][0], part[i][1], 0x7632));
                    pf[nt][i][1] = movmatrix_trans(__byte_perm(part[i][2], part[i][3], 0x7632));
                }
            }
            // ---- O^T += V^T P^T.  P's first part is positive where P is, so an infinite value and
            // NaN come through its product as the formula has them; the other parts may be 0, which
            // would make NaN of infinity: their products take finite values alone.
            {
                const int q = lane >> 3, row = warp * 16 + (q >> 1) * 8 + (lane & 7);
#pragma unroll
                for (int dt = 0; dt < 8; ++dt) {
                    uint32_t a0, a1, a2, a3;
                    ldmatrix_x4_trans(vt + tile_off(row, 2 * dt + (q & 1)), a0, a1, a2, a3);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma_bf16_16816(o[nt][dt], a0, a1, a2, a3, pf[nt][0][0], pf[nt][0][1]);
                    a0 = clamp_bf2(a0), a1 = clamp_bf2(a1), a2 = clamp_bf2(a2), a3 = clamp_bf2(a3);
#pragma unroll
                    for (int i = 1; i < 3; ++i)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
                            mma_bf16_16816(o[nt][dt], a0, a1, a2, a3, pf[nt][i][0], pf[nt][i][1]);
                }
            }
            if (a.accumulate) {
                float* const to = score_lane + static_cast<size_t>(d.z) * score_tile;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const bool h0 = nt * 8 + 2 * t4 < G, h1 = nt * 8 + 2 * t4 + 1 < G;
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        float* const at = to + 8 * r * G + nt * 8;
                        const bool in = warp * 16 + g + 8 * r < valid;
                        if (pairs) {
                            if (in && h0)
                                *reinterpret_cast<float2*>(at) = make_float2(score[nt][2 * r], score[nt][2 * r + 1]);
                        } else {
                            if (in && h0) at[0] = score[nt][2 * r];
                            if (in && h1) at[1] = score[nt][2 * r + 1];
                        }
                    }
                }
            }
        }
        if (d.w & TILE_LAST) {
            // ---- merge the warps' states in warp order; finish the run or leave its part
            named_bar(1, kConsumers);  // the stage has been read by all
            float* acc = reinterpret_cast<float*>(kt);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float l = l_run[nt][j];
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
                    if (g == 0) {
                        sm.m[warp][nt * 8 + 2 * t4 + j] = m_run[nt][j];
                        sm.l[warp][nt * 8 + 2 * t4 + j] = l;
                    }
                }
#pragma unroll
                for (int dt = 0; dt < 8; ++dt)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        acc[(warp * C::kHeads + nt * 8 + 2 * t4 + (e & 1)) * kAccPitch + dt * 16 + g + (e >> 1) * 8] =
                            o[nt][dt][e];
            }
            wrote = true;
            named_bar(1, kConsumers);
            const bool whole = (d.w & TILE_WHOLE) != 0;
            const int part = (d.w >> 16) * 2 + ((d.w & TILE_BEGIN) ? 1 : 0);
            // side by side: `across` threads a head, four dims each, all heads at once (16 heads: in four turns)
            const int across_log = G <= 4 ? 5 : G <= 8 ? 4 : 3, across = 1 << across_log, h = tid >> across_log;
            if (h < G) {
                float m[kWarps], f[kWarps], L = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) m[w] = sm.m[w][h];
                const float M = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
                const float base = M == -INFINITY ? 0.f : M;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    f[w] = ex2(m[w] - base);
                    L += sm.l[w][h] * f[w];
                }
                const float inv = poisoned ? 0.f : 1.f / L;
                const size_t at = static_cast<size_t>(part) * G + h;
                if ((tid & (across - 1)) == 0) {
                    if (whole)
                        parts.ml[static_cast<size_t>(d.x) * a.q_heads + d.y * G + h] = make_float2(base, inv);
                    else
                        // no other part has a poisoned one's pair: the sum to an infinite maximum is NaN
                        parts.pml[at] = poisoned ? make_float2(INFINITY, 0.f) : make_float2(M, L);
                }
                for (int dd = (tid & (across - 1)) * 4; dd < kCacheHd; dd += across * 4) {
                    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) {
                        const float4 v = *reinterpret_cast<const float4*>(&acc[(w * C::kHeads + h) * kAccPitch + dd]);
                        x.x += v.x * f[w], x.y += v.y * f[w], x.z += v.z * f[w], x.w += v.w * f[w];
                    }
                    if (whole) {
                        const float nan = __int_as_float(0x7FC00000);
                        uint2 u;
                        u.x = poisoned ? pack_bf2(f2bf(nan), f2bf(nan)) : pack_bf2(f2bf(x.x * inv), f2bf(x.y * inv));
                        u.y = poisoned ? u.x : pack_bf2(f2bf(x.z * inv), f2bf(x.w * inv));
                        *reinterpret_cast<uint2*>(a.out + d.x * a.out_stride +
                                                  (static_cast<size_t>(d.y) * G + h) * kCacheHd + dd) = u;
                    } else {
                        *reinterpret_cast<float4*>(parts.po + at * kCacheHd + dd) = x;
                    }
                }
            }
        }
        // the async proxy refills the stage after this warp's own writes to it
        if (wrote) fence_proxy_async_cta();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.empty[s]);
    }
}

// The second kernel: joins the parts of cut runs and turns scores into weights.  Each
// CTA takes an equal contiguous share of the tiles: for every run that it meets it finds
// the maximum and sum from the run's parts, joins a slice of the run's outputs (as many
// slices as CTAs that meet the run) and writes the weights of its own slots.  Two CTAs an
// SM, small enough to be resident beside two of the first kernel: what depends on the
// lengths alone (the share's runs) is done while that one runs.  The lengths are there
// before the wait: the first kernel lets this one start only behind its own wait for what
// wrote them.  An SM's first-level cache may still hold older ones, so they are read from
// L2, where all SMs' writes meet.
struct LensBehindL1 {
    const int32_t* at;
    __device__ __forceinline__ int operator[](int r) const { return __ldcg(at + r); }
};
constexpr int kJoinThreads = 128;
constexpr int kJoinWarps = kJoinThreads / 32;
constexpr int kJoinTiles = 64;  // tiles whose runs are looked up at a time, a thread each
constexpr int kJoinRuns = 8;    // runs joined between two barriers
struct JoinSmem {
    int4 where[kJoinTiles];                      // of a run met: row, head, first tile here, slots here
    int4 span[kJoinTiles];                       // its first tile of all, first and last chunk's place; slice: turns << 24 | first unit << 12 | last
    float2 part[kJoinRuns][kJoinWarps][16];      // each warp's maximum and sum
    float2 ml[kJoinRuns][16];                    // maximum, 1 / sum (0: a bad page, no weights)
    int before[kJoinThreads + 1];
    int scan[kJoinWarps];
    unsigned starts[kJoinTiles / 32];
};

// Weights of n slots from their scores: w[j] += sum_h 2^(s[j][h] - m_h) / l_h.  GV: the
// heads (0: any number, in `heads`); U slots a thread in flight.
template <int GV, int U>
__device__ __forceinline__ void add_weights(float* w, const float* s, const float2* ml, int n, int heads, int me, int threads) {
    const int G = GV ? GV : heads;
    for (int j0 = 0; j0 < n; j0 += threads * U) {
        float x[U], sc[U][GV ? GV : 1];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + u * threads + me;
            x[u] = j < n ? w[j] : 0.f;
            if constexpr (GV > 0) {
#pragma unroll
                for (int h = 0; h < GV; h += 4) {
                    if constexpr (GV >= 4) {
                        const float4 v = j < n ? *reinterpret_cast<const float4*>(s + static_cast<size_t>(j) * GV + h)
                                               : make_float4(0.f, 0.f, 0.f, 0.f);
                        sc[u][h] = v.x, sc[u][h + 1] = v.y, sc[u][h + 2] = v.z, sc[u][h + 3] = v.w;
                    } else if constexpr (GV == 2) {
                        const float2 v = j < n ? *reinterpret_cast<const float2*>(s + static_cast<size_t>(j) * 2)
                                               : make_float2(0.f, 0.f);
                        sc[u][0] = v.x, sc[u][1] = v.y;
                    } else {
                        sc[u][0] = j < n ? s[j] : 0.f;
                    }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + u * threads + me;
            float p = 0.f;
            if constexpr (GV > 0) {
#pragma unroll
                for (int h = 0; h < GV; ++h) p += ex2(sc[u][h] - ml[h].x) * ml[h].y;
            } else if (j < n) {
                for (int h = 0; h < G; ++h) p += ex2(s[static_cast<size_t>(j) * G + h] - ml[h].x) * ml[h].y;
            }
            if (j < n) w[j] = x[u] + p;
        }
    }
}

__global__ void __maxnreg__(64)
    cache_join_kernel(const __grid_constant__ CacheAttnArgs a, const __grid_constant__ Parts parts) {
    __shared__ JoinSmem sm;
    const CacheView& c = a.c;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, me = blockIdx.x;
    const int G = a.q_heads / c.kv_heads;
    const LensBehindL1 lens{a.lens};
    scan_rows<kJoinThreads>(lens, c, sm.before, sm.scan);
    const int total = sm.before[kJoinThreads] * c.kv_heads;
    const Plan plan = plan_make(total, parts.workers, parts.inverse);
    const Equal mine = equal_make(total, gridDim.x);
    const int t0 = equal_first(mine, me), t1 = equal_first(mine, me + 1);
    // the runs met by tiles [t, t + 64) of the share
    int runs = 0;
    auto look_up = [&](int t) {
        const int n = min(kJoinTiles, t1 - t);
        PlanPlace p;
        bool starts = false;
        if (tid < kJoinTiles) {
            if (tid < n) {
                p = plan_locate(t + tid, lens, c.rows, c.max_len, c.kv_heads, sm.before, kJoinThreads,
                                plan_group_rows(c.rows, kJoinThreads));
                starts = tid == 0 || p.tile == 0;
            }
            const unsigned who = __ballot_sync(0xffffffffu, starts);
            if (lane == 0) sm.starts[warp] = who;
        }
        __syncthreads();
        runs = __popc(sm.starts[0]) + __popc(sm.starts[1]);
        if (starts) {
            const int at = __popc(sm.starts[warp] & ((1u << lane) - 1)) + (warp ? __popc(sm.starts[0]) : 0);
            const int run0 = t + tid - p.tile, here = min(n - tid, p.tiles - p.tile);
            sm.where[at] = make_int4(p.row, p.head, p.tile, min(here * kCachePage, p.len - p.tile * kCachePage));
            int c0, c1;
            plan_run(plan, run0, p.tiles, c0, c1);
            int slice = 0;  // of the run's outputs, in units of 4 dims
            if (c0 != c1 && max(run0, t0) == t + tid) {  // cut, and not met before in this share
                const int first = equal_share_of(mine, run0);
                const Equal part = equal_make(G * kCacheHd / 4, equal_share_of(mine, run0 + p.tiles - 1) - first + 1);
                const int u0 = equal_first(part, me - first), u1 = equal_first(part, me - first + 1), P = c1 - c0 + 1;
                // lanes that share a unit: as few as take up to four parts each
                int turns = 0;
                while (turns < 5 && 4 << turns < P) ++turns;
                slice = turns << 24 | u0 << 12 | u1;
            }
            sm.span[at] = make_int4(run0, c0, c1, slice);
        }
        __syncthreads();
    };
    if (t0 < t1) look_up(t0);
    pdl_wait();
    pdl_trigger();
    if (me == 0 && tid == 0) *c.next_chunk = 0;  // for the cache's next attention

    // heads side by side in a warp: the power of two that holds G (powers of two as shifts throughout: an integer
    // division is some 150 cycles of the chain between the two kernels)
    const int wide_log = G <= 1 ? 0 : G <= 2 ? 1 : G <= 4 ? 2 : G <= 8 ? 3 : 4, wide = 1 << wide_log;
    for (int t = t0; t < t1; t += kJoinTiles) {
        if (t > t0) look_up(t);
        for (int r0 = 0; r0 < runs; r0 += kJoinRuns) {
            const int nr = min(kJoinRuns, runs - r0);
            // ---- maximum and sum; thread: head tid % wide of every (threads / wide)-th part
            for (int r = 0; r < nr; ++r) {
                const int c0 = sm.span[r0 + r].y, c1 = sm.span[r0 + r].z;
                if (c0 == c1) continue;
                // (heads that there are not: the last one's, and nobody's)
                const int h = min(tid & (wide - 1), G - 1), deal = kJoinThreads >> wide_log;
                float m = -INFINITY, l = 0.f;
                bool bad = false;
                for (int s0 = c0 + (tid >> wide_log); s0 <= c1; s0 += 8 * deal) {
                    float2 x[8];
#pragma unroll
                    for (int u = 0; u < 8; ++u) {
                        const int s = min(s0 + u * deal, c1);
                        // the run begins in chunk c0: its part there is in slot 1, the others' in slot 0
                        x[u] = parts.pml[static_cast<size_t>(s * 2 + (s == c0)) * G + h];
                    }
                    const float before = m;
#pragma unroll
                    for (int u = 0; u < 8; ++u) {
                        if (s0 + u * deal > c1) x[u].y = 0.f, x[u].x = -INFINITY;
                        bad |= (x[u].x == INFINITY) & (x[u].y == 0.f);  // a bad page: see the parts
                        m = fmaxf(m, x[u].x);
                    }
                    const float base = m == -INFINITY ? 0.f : m;
                    l *= ex2(before - base);
#pragma unroll
                    for (int u = 0; u < 8; ++u) l += x[u].y * ex2(x[u].x - base);
                }
                float M = m;
                for (int off = wide; off < 32; off <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
                l *= ex2(m - (M == -INFINITY ? 0.f : M));
                for (int off = wide; off < 32; off <<= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
                bad = __any_sync(0xffffffffu, bad);
                if (lane < wide) sm.part[r][warp][lane] = make_float2(bad ? INFINITY : M, bad ? 0.f : l);
            }
            __syncthreads();
            {
                const int r = tid >> 4, h = tid & 15;
                if (r < nr && h < G) {
                    const int4 w = sm.where[r0 + r], sp = sm.span[r0 + r];
                    if (sp.y == sp.z) {
                        if (a.accumulate)
                            sm.ml[r][h] = parts.ml[static_cast<size_t>(w.x) * a.q_heads + w.y * G + h];
                    } else {
                        float2 x[kJoinWarps];
                        float M = -INFINITY, L = 0.f;
                        bool bad = false;
#pragma unroll
                        for (int i = 0; i < kJoinWarps; ++i) {
                            x[i] = sm.part[r][i][h];
                            bad |= (x[i].x == INFINITY) & (x[i].y == 0.f);
                            M = fmaxf(M, x[i].x);
                        }
                        const float base = M == -INFINITY ? 0.f : M;
#pragma unroll
                        for (int i = 0; i < kJoinWarps; ++i) L += x[i].y * ex2(x[i].x - base);
                        sm.ml[r][h] = make_float2(base, bad ? 0.f : __fdividef(1.f, L));
                    }
                }
            }
            __syncthreads();
            // With few slots to write, two warps join outputs while the other two write weights; else all do both.
            int slots = 0;
            bool cut = false;
            for (int r = 0; r < nr; ++r) slots += sm.where[r0 + r].w, cut = cut || sm.span[r0 + r].w != 0;
            const bool apart = a.accumulate && cut && slots <= 4 * kJoinThreads;
            const int o_warps = apart ? kJoinWarps / 2 : kJoinWarps;
            // ---- outputs of cut runs, in units of 4 dims: a warp takes units, its lanes their parts
            for (int r = 0; r < nr && warp < o_warps; ++r) {
                const int4 w = sm.where[r0 + r], sp = sm.span[r0 + r];
                const int u0 = sp.w >> 12 & 0xFFF, u1 = sp.w & 0xFFF, c0 = sp.y, c1 = sp.z;
                const int turns_log = sp.w >> 24, turns = 1 << turns_log, width = 32 >> turns_log;
                const int turn = lane >> (5 - turns_log), column = lane & (width - 1);
                for (int u = u0 + warp * width; u < u1; u += o_warps * width) {
                    const int unit = u + column, h = min(unit, u1 - 1) / (kCacheHd / 4);
                    const float2 ml = sm.ml[r][h];
                    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                    // four parts' loads under way together; behind the last one: that one again, for nothing
                    for (int s0 = c0 + turn; s0 <= c1; s0 += 4 * turns) {
                        float m[4];
                        float4 v[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int s = min(s0 + i * turns, c1);
                            const size_t at = static_cast<size_t>(s * 2 + (s == c0)) * G + h;
                            m[i] = parts.pml[at].x;
                            v[i] = reinterpret_cast<const float4*>(parts.po + at * kCacheHd)[unit % (kCacheHd / 4)];
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if (s0 + i * turns > c1) v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                            const float f = ex2(m[i] - ml.x);
                            x.x += v[i].x * f, x.y += v[i].y * f, x.z += v[i].z * f, x.w += v[i].w * f;
                        }
                    }
                    for (int off = width; off < 32; off <<= 1) {
                        x.x += __shfl_xor_sync(0xffffffffu, x.x, off);
                        x.y += __shfl_xor_sync(0xffffffffu, x.y, off);
                        x.z += __shfl_xor_sync(0xffffffffu, x.z, off);
                        x.w += __shfl_xor_sync(0xffffffffu, x.w, off);
                    }
                    if (turn == 0 && unit < u1) {
                        if (ml.y == 0.f) x = make_float4(NAN, NAN, NAN, NAN);
                        const float k = ml.y == 0.f ? 1.f : ml.y;
                        uint2 o;
                        o.x = pack_bf2(f2bf(x.x * k), f2bf(x.y * k));
                        o.y = pack_bf2(f2bf(x.z * k), f2bf(x.w * k));
                        reinterpret_cast<uint2*>(a.out + w.x * a.out_stride + static_cast<size_t>(w.y) * G * kCacheHd)[unit] = o;
                    }
                }
            }
            // ---- weights
            // several short runs side by side: one after the other each waits for its own loads (131 x 98 slots, 8
            // heads: 21.6 us for 19.4)
            const int w_first = apart ? kJoinThreads / 2 : 0;
            const int side_log = nr < 2 || slots > 8 * kJoinThreads ? 0 : nr >= 4 && !apart ? 2 : 1;
            const int w_threads = (kJoinThreads - w_first) >> side_log, w_me = tid & (w_threads - 1);
            if (a.accumulate && tid >= w_first)
                for (int r = (tid - w_first) >> (apart ? 6 - side_log : 7 - side_log); r < nr; r += 1 << side_log) {
                    const int4 w = sm.where[r0 + r];
                    const float2* ml = sm.ml[r];
                    if (ml[0].y == 0.f) continue;  // a bad page: all heads' then
                    float* to = c.weights + cache_slot_index(c, w.x, w.y) + w.z * kCachePage;
                    const float* s = parts.score + static_cast<size_t>(sm.span[r0 + r].x + w.z) * kCachePage * G;
                    switch (G) {
                        case 1: add_weights<1, 8>(to, s, ml, w.w, G, w_me, w_threads); break;
                        case 2: add_weights<2, 6>(to, s, ml, w.w, G, w_me, w_threads); break;
                        case 4: add_weights<4, 4>(to, s, ml, w.w, G, w_me, w_threads); break;
                        case 8: add_weights<8, 2>(to, s, ml, w.w, G, w_me, w_threads); break;
                        case 16: add_weights<16, 1>(to, s, ml, w.w, G, w_me, w_threads); break;
                        default: add_weights<0, 2>(to, s, ml, w.w, G, w_me, w_threads);
                    }
                }
            __syncthreads();  // sm.ml and sm.part are the next runs'
        }
    }
}

bool make_map(CUtensorMap* map, const bf16* base, long long rows, int box_rows) {
    auto fn = tensor_map_encoder();
    if (!fn) return false;
    const cuuint64_t dims[2] = {kCacheHd, static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {kCacheHd * 2};
    const cuuint32_t box[2] = {64, static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t estr[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<bf16*>(base), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

size_t pad256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

size_t max_tiles(const CacheView& c) {
    return static_cast<size_t>(c.rows) * c.kv_heads * ((c.max_len + kCachePage - 1) / kCachePage);
}

// Two resident CTAs an SM, no more than there can be tiles, nor than 15 bits number the
// chunks of (a region has at most 20: there are at most 2^30 tiles).
int workers_of(const CacheView& c, int sms) {
    return static_cast<int>(std::min(static_cast<size_t>(std::min(2 * sms, 1024)), max_tiles(c)));
}

// The workspace's arrays from its start; returns its size.
size_t layout(const CacheView& c, int q_heads, int accumulate, int sms, uint8_t* ws, Parts* p) {
    const int G = q_heads / c.kv_heads, workers = workers_of(c, sms);
    const size_t parts = 2 * static_cast<size_t>(workers) * plan_make(static_cast<int>(max_tiles(c)), workers, plan_inverse(workers)).tiers;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        uint8_t* to = ws + at;
        at += pad256(bytes);
        return to;
    };
    p->workers = workers;
    p->inverse = plan_inverse(workers);
    p->ml = reinterpret_cast<float2*>(take(static_cast<size_t>(c.rows) * q_heads * 8));
    p->pml = reinterpret_cast<float2*>(take(parts * G * 8));
    p->po = reinterpret_cast<float*>(take(parts * G * kCacheHd * 4));
    p->score = reinterpret_cast<float*>(take(accumulate ? max_tiles(c) * kCachePage * G * 4 : 0));
    return at;
}

static_assert(2 * (sizeof(Smem<1>) + 1024 + 1024) <= 228 * 1024, "two CTAs must share an SM");
static_assert(2 * (sizeof(Smem<2>) + 1024 + 1024) <= 228 * 1024, "two CTAs must share an SM");

template <int NT>
cudaError_t launch_nt(const CacheAttnArgs& a, const CacheMaps& maps, const Parts& parts, cudaStream_t s) {
    // the shared-memory opt-in once per device (not per launch: launches may be captured)
    static std::atomic<uint64_t> configured{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (!(configured.load() & bit)) {
        e = cudaFuncSetAttribute(cache_attention_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 static_cast<int>(sizeof(Smem<NT>) + 1024));
        if (e != cudaSuccess) return e;
        configured.fetch_or(bit);
    }
    return launch_after(cache_attention_kernel<NT>, dim3(parts.workers), kThreads, sizeof(Smem<NT>) + 1024, s, a, maps, parts);
}

}  // namespace

size_t cache_attention_ws_bytes(const CacheView& c, int q_heads, int accumulate, int sms) {
    Parts p;
    return layout(c, q_heads, accumulate, sms, nullptr, &p);
}

bool cache_maps(const CacheView& c, CacheMaps* maps) {
    const long long rows = static_cast<long long>(c.num_pages) * c.kv_heads * kCachePage;
    return make_map(&maps->k64, c.k, rows, 64) && make_map(&maps->v64, c.v, rows, 64) &&
           make_map(&maps->k16, c.k, rows, 16) && make_map(&maps->v16, c.v, rows, 16);
}

cudaError_t launch_cache_attention(const CacheAttnArgs& a, const CacheMaps& maps, int sms, cudaStream_t s) {
    const CacheView& c = a.c;
    Parts parts;
    layout(c, a.q_heads, a.accumulate, sms, static_cast<uint8_t*>(a.ws), &parts);
    cudaError_t e = a.q_heads / c.kv_heads <= 8 ? launch_nt<1>(a, maps, parts, s) : launch_nt<2>(a, maps, parts, s);
    if (e != cudaSuccess) return e;
    // two CTAs an SM are resident beside the first kernel's; with 8 tiles a worker or more the work is worth
    // eight, though the others start (and look up their runs) only when that one ends: 64 x 8192 takes 220,
    // 209, 206, 204 and 210 us with 1, 2, 3, 4 and 6 times the workers, 16 x 4096 37.1, 36.7, 36.4, 36.1 and 40.4
    // (sequences of up to so many slots, 32 / 8 heads)
    const int join_ctas = max_tiles(c) >= 8 * static_cast<size_t>(parts.workers) ? 4 * parts.workers : parts.workers;
    return launch_after(cache_join_kernel, dim3(join_ctas), kJoinThreads, 0, s, a, parts);
}

}  // namespace q3
