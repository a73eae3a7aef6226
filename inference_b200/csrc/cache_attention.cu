// cache_attention.cu -- attention of one query token per sequence over a bounded
// paged cache, with the attention every slot receives accumulated.
//
//   s_gj = q_g . k_j / sqrt(128);  p_gj = 2^(s_gj log2 e - m_g) / l_g
//   out_g = sum_j p_gj v_j;  weight_j += sum_g p_gj   (g: the kv head's query heads)
//
// Bound: HBM.  K and V of every slot cross it once (512 bytes a slot and kv head)
// for 512 G flops; everything else is two orders smaller.  So:
//   * all sequences' 64-slot tiles are cut into equal shares (cache_plan.hpp), one
//     per resident CTA (two an SM), from the lengths in device memory: one launch
//     shape serves any mix of lengths, and no SM waits for the longest sequence;
//   * in a CTA one warp streams K and V tiles through a ring of 32 KB stages by
//     swizzled 2-D TMA (a last, partial tile by boxes of 16 slots), reading page
//     table entries for 32 tiles at a time; four warps take 16 slots of a tile
//     each: S^T = K Q^T and O^T += V^T P^T on the tensor cores with the slots as
//     M and the group's query heads as N, online softmax in fp32, P as the sum of
//     two BF16 parts (2^-16 of its size);
//   * a run (sequence, kv head) within one share is finished by it; parts of a cut
//     run (maximum, sum, unnormalised output in fp32) are joined by the second
//     kernel in share order, so results do not depend on timing;
//   * probabilities need the run's final maximum and sum: the first kernel leaves
//     the raw scores (fp32, 4 G bytes a slot, written once and mostly read back
//     from L2), the second turns them into weights, share by share.
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
constexpr int kJoinThreads = 512;
constexpr int kAccPitch = 68;                  // floats of a head's 64 dims in the merge buffer: conflict-free
constexpr float kScoreScale = 0.08838834764831845f * 1.4426950408889634f;  // log2(e) / sqrt(128)

// What the producer tells the consumers about a stage's tile.
enum : int {
    TILE_FIRST = 1,  // first tile of its run in this share
    TILE_LAST = 2,   // last tile of its run in this share
    TILE_WHOLE = 4,  // the run lies in this share
    TILE_BEGIN = 8,  // the run begins in this share
    TILE_BAD = 16,   // its page lies outside the pool: nothing was loaded
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
    uint8_t ring[Cfg<NT>::kStages][Cfg<NT>::kStageBytes];  // K tile, V tile, the run's queries (first tile only)
    float acc[kWarps][Cfg<NT>::kHeads][kAccPitch];         // 64 dims of every warp's output, merging
    float m[kWarps][Cfg<NT>::kHeads], l[kWarps][Cfg<NT>::kHeads];
    float f[kWarps][Cfg<NT>::kHeads];                      // a warp's weight in the merge
    float cm[Cfg<NT>::kHeads], cl[Cfg<NT>::kHeads];
    int4 tile[Cfg<NT>::kStages];                           // row, head, live slots, flags
    uint64_t full[Cfg<NT>::kStages], empty[Cfg<NT>::kStages];
    uint64_t meet;                                         // the consumer warps' barrier in a merge
    int chunk[kThreads + 1];                               // tiles before each chunk of rows
    int scan[kThreads / 32];
};

struct Parts {
    float2* ml;    // [rows][q_heads]: maximum (log2) and sum of runs within one share
    float2* pml;   // [shares][2][heads]: of parts
    float* po;     // [shares][2][heads][128]: unnormalised outputs of parts
    float* score;  // [tile][64][G]: raw scores in log2 units
    int shares, heads;
};

// Chunks of consecutive rows, one per thread: chunk[t] = tiles (of one kv head)
// before thread t's rows, chunk[threads] = all.
template <int THREADS>
__device__ __forceinline__ void scan_rows(const int32_t* lens, const CacheView& c, int* chunk, int* scan) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int per = plan_chunk_rows(c.rows, THREADS);
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
    int before = 0;
    for (int i = 0; i < warp; ++i) before += scan[i];
    chunk[tid + 1] = before + incl;
    if (tid == 0) chunk[0] = 0;
    __syncthreads();
}

template <int THREADS>
__device__ __forceinline__ PlanPlace locate(long long t, const int32_t* lens, const CacheView& c, const int* chunk) {
    return plan_locate(t, lens, c.rows, c.max_len, c.kv_heads, chunk, THREADS);
}

__device__ __forceinline__ void tma_tile(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
        " [%0], [%1, {%2, %3}], [%4], %5;" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar)), "l"(policy)
        : "memory");
}

// Tensor maps of the K and V pools as [num_pages x kv_heads x 64, 128] matrices:
// boxes of 64 columns by 64 rows (a full tile's half) and by 16.
struct Maps {
    CUtensorMap k64, v64, k16, v16;
};

template <int NT>
__global__ void __launch_bounds__(kThreads, 2)
    cache_attention_kernel(const __grid_constant__ CacheAttnArgs a, const __grid_constant__ Maps maps, const Parts parts) {
    using C = Cfg<NT>;
    constexpr int S = C::kStages;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    Smem<NT>& sm = *reinterpret_cast<Smem<NT>*>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
    const CacheView& c = a.c;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, b = blockIdx.x;
    const int G = a.q_heads / c.kv_heads;
    if (tid == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&sm.full[s], 1);
            mbar_init(&sm.empty[s], kWarps);
        }
        mbar_init(&sm.meet, kWarps);
        fence_barrier_init();
    }
    scan_rows<kThreads>(a.lens, c, sm.chunk, sm.scan);
    pdl_trigger();  // the joining kernel may set itself up; it waits for this one's end
    const long long total = static_cast<long long>(sm.chunk[kThreads]) * c.kv_heads;
    const int shares = plan_shares(total, parts.shares);
    const long long t0 = plan_first(total, shares, b);
    const int n = b < shares ? static_cast<int>(plan_first(total, shares, b + 1) - t0) : 0;

    // sequences without a tile: length 0 gives zeros, a length out of range NaN
    for (int r = b; r < c.rows; r += gridDim.x) {
        const int len = a.lens[r];
        if (len > 0 && len <= c.max_len) continue;
        if (len != 0 && tid == 0) record_error(c.err, DEV_BAD_LENGTH);
        const uint32_t v = len == 0 ? 0u : 0x7FC07FC0u;
        uint4* o = reinterpret_cast<uint4*>(a.out + r * a.out_stride);
        for (int i = tid; i < a.q_heads * kCacheHd / 8; i += kThreads) o[i] = make_uint4(v, v, v, v);
    }
    if (n == 0) return;

    if (warp == kWarps) {
        // ------------------------------------------------------------ producer
        const uint64_t pol = policy_evict_first();
        int issued = 0;
        bool stop = false;
        for (int i0 = 0; i0 < n && !stop; i0 += 32) {
            // lane i: tile i0 + i
            int4 d = make_int4(0, 0, 0, 0);
            int y = 0;
            if (i0 + lane < n) {
                const long long t = t0 + i0 + lane;
                const PlanPlace p = locate<kThreads>(t, a.lens, c, sm.chunk);
                const long long run0 = t - p.tile;
                const bool begins = run0 >= t0, ends = run0 + p.tiles <= t0 + n;
                const int page = c.tables[p.row * c.table_stride + p.tile];
                int flags = 0;
                if (p.tile == 0 || i0 + lane == 0) flags |= TILE_FIRST;
                if (p.tile == p.tiles - 1 || i0 + lane == n - 1) flags |= TILE_LAST;
                if (begins && ends) flags |= TILE_WHOLE;
                if (begins) flags |= TILE_BEGIN;
                if (page < 0 || page >= c.num_pages) {
                    flags |= TILE_BAD;
                    record_error(c.err, DEV_BAD_PAGE);
                } else {
                    y = (page * c.kv_heads + p.head) * kCachePage;
                }
                d = make_int4(p.row, p.head, min(kCachePage, p.len - p.tile * kCachePage), flags);
            }
            for (int i = 0; i < 32 && i0 + i < n; ++i) {
                const int4 t = make_int4(__shfl_sync(0xffffffffu, d.x, i), __shfl_sync(0xffffffffu, d.y, i),
                                         __shfl_sync(0xffffffffu, d.z, i), __shfl_sync(0xffffffffu, d.w, i));
                const int row0 = __shfl_sync(0xffffffffu, y, i);
                const int k = i0 + i, s = k % S;
                int ok = 1;
                if (lane == 0) {
                    if (k >= S) ok = mbar_wait(&sm.empty[s], ((k / S) - 1) & 1, c.err, DEV_TMA_WAIT_TIMEOUT);
                    if (ok) {
                        sm.tile[s] = t;
                        uint8_t* st = sm.ring[s];
                        if (t.w & TILE_BAD) {
                            mbar_arrive(&sm.full[s]);
                        } else {
                            const int boxes = (t.z + 15) / 16;  // of 16 slots
                            const uint32_t q_bytes = (t.w & TILE_FIRST) ? G * kCacheHd * 2 : 0;
                            mbar_arrive_expect_tx(&sm.full[s], boxes * (2 * 16 * kCacheHd * 2) + q_bytes);
                            if (q_bytes)
                                bulk_g2s(st + 2 * kTileBytes,
                                         a.q + t.x * a.q_stride + static_cast<size_t>(t.y) * G * kCacheHd, q_bytes,
                                         &sm.full[s], pol);
                            if (boxes == 4) {
                                for (int h = 0; h < 2; ++h) {
                                    tma_tile(st + h * 8192, &maps.k64, h * 64, row0, &sm.full[s], pol);
                                    tma_tile(st + kTileBytes + h * 8192, &maps.v64, h * 64, row0, &sm.full[s], pol);
                                }
                            } else {
                                for (int x = 0; x < boxes; ++x)
                                    for (int h = 0; h < 2; ++h) {
                                        uint8_t* to = st + h * 8192 + x * 2048;
                                        tma_tile(to, &maps.k16, h * 64, row0 + 16 * x, &sm.full[s], pol);
                                        tma_tile(to + kTileBytes, &maps.v16, h * 64, row0 + 16 * x, &sm.full[s], pol);
                                    }
                            }
                        }
                    }
                }
                ok = __shfl_sync(0xffffffffu, ok, 0);
                if (!ok) {
                    stop = true;
                    break;
                }
                issued = k + 1;
            }
        }
        // leave no copy in flight behind a wait that ran out
        if (stop && lane == 0)
            for (int k = max(0, issued - S); k < issued; ++k) mbar_wait(&sm.full[k % S], (k / S) & 1, nullptr, 0);
        return;
    }

    // ---------------------------------------------------------------- consumers
    const int g = lane >> 2, t4 = lane & 3;  // fragment row and column pair
    uint32_t qf[NT][8][2];                   // Q^T as the B operand: dims 16 kk + 2 t4 (+ 8), head 8 nt + g
    float o[NT][8][4];                       // O^T: dims 16 dt + g (+ 8), heads 8 nt + 2 t4 (+ 1)
    float m_run[NT][2], l_run[NT][2];        // of those heads: maximum (log2), this lane's share of the sum
    bool poisoned = false;
    // All four warps meet here in a merge.  An mbarrier, so that no wait is unbounded: a
    // warp whose wait ran out returns, and the others' waits run out in turn.
    uint32_t meet_phase = 0;
    auto meet = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.meet);
        const bool ok = mbar_wait(&sm.meet, meet_phase, c.err, DEV_TMA_WAIT_TIMEOUT);
        meet_phase ^= 1;
        return ok;
    };
    for (int k = 0; k < n; ++k) {
        const int s = k % S;
        if (!mbar_wait(&sm.full[s], (k / S) & 1, c.err, DEV_TMA_WAIT_TIMEOUT)) return;
        const int4 d = sm.tile[s];
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
        const int valid = d.z;
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
            uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                // slots g (elements 0, 1) and g + 8 (2, 3), heads 2 t4 (0, 2) and 2 t4 + 1 (1, 3)
                const int tok = warp * 16 + g, h0 = nt * 8 + 2 * t4;
                float sc[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    sc[e] = tok + (e >> 1) * 8 < valid ? (sa[nt][e] + sb[nt][e]) * kScoreScale : -INFINITY;
                if (a.accumulate) {
                    float* to = parts.score + ((t0 + k) * kCachePage + tok) * G + h0;
#pragma unroll
                    for (int r = 0; r < 2; ++r)
                        if (tok + 8 * r < valid) {
                            if (h0 < G) to[8 * r * G] = sc[2 * r];
                            if (h0 + 1 < G) to[8 * r * G + 1] = sc[2 * r + 1];
                        }
                }
                float mx[2] = {fmaxf(sc[0], sc[2]), fmaxf(sc[1], sc[3])};
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) {
                    mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], off));
                    mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], off));
                }
                float p[4], corr[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float mn = fmaxf(m_run[nt][j], mx[j]);
                    // nothing above -infinity yet: the exponentials' base is 0, not -infinity
                    const float base = mn == -INFINITY ? 0.f : mn;
                    corr[j] = exp2f(m_run[nt][j] - base);
                    p[j] = exp2f(sc[j] - base);
                    p[j + 2] = exp2f(sc[j + 2] - base);
                    m_run[nt][j] = mn;
                    l_run[nt][j] = l_run[nt][j] * corr[j] + p[j] + p[j + 2];
                }
#pragma unroll
                for (int dt = 0; dt < 8; ++dt) {
                    o[nt][dt][0] *= corr[0];
                    o[nt][dt][1] *= corr[1];
                    o[nt][dt][2] *= corr[0];
                    o[nt][dt][3] *= corr[1];
                }
                // P as two BF16 parts: the second holds what the first's rounding left
                bf16 hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    hi[e] = f2bf(p[e]);
                    lo[e] = f2bf(p[e] - bf2f(hi[e]));
                }
                ph[nt][0] = movmatrix_trans(pack_bf2(hi[0], hi[1]));
                ph[nt][1] = movmatrix_trans(pack_bf2(hi[2], hi[3]));
                pl[nt][0] = movmatrix_trans(pack_bf2(lo[0], lo[1]));
                pl[nt][1] = movmatrix_trans(pack_bf2(lo[2], lo[3]));
            }
            // ---- O^T += V^T P^T
            {
                const int q = lane >> 3, row = warp * 16 + (q >> 1) * 8 + (lane & 7);
#pragma unroll
                for (int dt = 0; dt < 8; ++dt) {
                    uint32_t a0, a1, a2, a3;
                    ldmatrix_x4_trans(vt + tile_off(row, 2 * dt + (q & 1)), a0, a1, a2, a3);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma_bf16_16816(o[nt][dt], a0, a1, a2, a3, ph[nt][0], ph[nt][1]);
                        mma_bf16_16816(o[nt][dt], a0, a1, a2, a3, pl[nt][0], pl[nt][1]);
                    }
                }
            }
        }
        // the async proxy refills the stage after this warp's own writes to it
        if (wrote) fence_proxy_async_cta();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.empty[s]);

        if (d.w & TILE_LAST) {
            // ---- merge the warps' states in warp order; finish the run or leave its part
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
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
            if (!meet()) return;
            const bool whole = (d.w & TILE_WHOLE) != 0;
            const int part = b * 2 + ((d.w & TILE_BEGIN) ? 1 : 0);
            if (tid < C::kHeads) {
                float M = -INFINITY, L = 0.f;
                for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm.m[w][tid]);
                const float base = M == -INFINITY ? 0.f : M;
                for (int w = 0; w < kWarps; ++w) {
                    sm.f[w][tid] = exp2f(sm.m[w][tid] - base);
                    L += sm.l[w][tid] * sm.f[w][tid];
                }
                if (poisoned) M = INFINITY, L = 0.f;  // no sum has this pair: an infinite score's sum is NaN
                sm.cm[tid] = M;
                sm.cl[tid] = L;
                if (tid < G) {
                    if (!whole)
                        parts.pml[static_cast<size_t>(part) * parts.heads + tid] = make_float2(M, L);
                    else if (a.accumulate)
                        parts.ml[static_cast<size_t>(d.x) * a.q_heads + d.y * G + tid] = make_float2(M, L);
                }
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            sm.acc[warp][nt * 8 + 2 * t4 + (e & 1)][dt * 16 + g + (e >> 1) * 8] = o[nt][half * 4 + dt][e];
                if (!meet()) return;
                for (int i = tid; i < G * 32; i += kConsumers) {
                    const int h = i >> 5, dd = (i & 31) * 2;
                    float x = 0.f, y = 0.f;
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) {
                        const float2 v = *reinterpret_cast<const float2*>(&sm.acc[w][h][dd]);
                        x += v.x * sm.f[w][h];
                        y += v.y * sm.f[w][h];
                    }
                    if (whole) {
                        const float L = sm.cl[h];
                        const bool nan = sm.cm[h] == INFINITY && L == 0.f;
                        const bf16 u = f2bf(nan ? __int_as_float(0x7FC00000) : x / L);
                        const bf16 v = f2bf(nan ? __int_as_float(0x7FC00000) : y / L);
                        *reinterpret_cast<uint32_t*>(a.out + d.x * a.out_stride +
                                                     (static_cast<size_t>(d.y) * G + h) * kCacheHd + half * 64 + dd) =
                            pack_bf2(u, v);
                    } else {
                        *reinterpret_cast<float2*>(parts.po + (static_cast<size_t>(part) * parts.heads + h) * kCacheHd +
                                                   half * 64 + dd) = make_float2(x, y);
                    }
                }
                if (!meet()) return;
            }
        }
    }
}

// The second kernel, one CTA per share: joins the parts of cut runs (each of a run's
// shares takes an equal slice of its outputs) and turns the share's scores into
// weights (a warp per tile).
struct JoinSmem {
    float2 ml[2][16];  // of the share's parts, by slot: maximum, 1 / sum; 1 / sum = 0: a bad page, no weights
    int chunk[kJoinThreads + 1];
    int scan[kJoinThreads / 32];
};

__global__ void __launch_bounds__(kJoinThreads) cache_join_kernel(const __grid_constant__ CacheAttnArgs a, const Parts parts) {
    __shared__ JoinSmem sm;
    const CacheView& c = a.c;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, b = blockIdx.x;
    const int G = a.q_heads / c.kv_heads;
    scan_rows<kJoinThreads>(a.lens, c, sm.chunk, sm.scan);
    const long long total = static_cast<long long>(sm.chunk[kJoinThreads]) * c.kv_heads;
    const int shares = plan_shares(total, parts.shares);
    const long long t0 = plan_first(total, shares, b);
    const int n = b < shares ? static_cast<int>(plan_first(total, shares, b + 1) - t0) : 0;
    pdl_wait();
    if (n == 0) return;
    // ---- the share's first and last run, where they are cut
    for (int e = 0; e < 2; ++e) {
        const long long t = e == 0 ? t0 : t0 + n - 1;
        const PlanPlace p = locate<kJoinThreads>(t, a.lens, c, sm.chunk);
        const long long run0 = t - p.tile;
        const int c0 = plan_share(total, shares, run0);
        const int c1 = plan_share(total, shares, run0 + p.tiles - 1);
        if (c0 == c1 || (e == 1 && run0 <= t0)) continue;  // whole, or the first run again
        const int slot = plan_slot(total, shares, b, run0);
        // the run begins in share c0: its part there is in slot 1, the others' in slot 0
        auto part_of = [&](int share) { return static_cast<size_t>(share * 2 + (share == c0 ? 1 : 0)); };
        for (int h = warp; h < G; h += kJoinThreads / 32) {
            float M = -INFINITY;
            bool bad = false;
            for (int s = c0 + lane; s <= c1; s += 32) {
                const float2 v = parts.pml[part_of(s) * parts.heads + h];
                bad = bad || (v.x == INFINITY && v.y == 0.f);
                M = fmaxf(M, v.x);
            }
            M = warp_max(M);
            const float base = M == -INFINITY ? 0.f : M;
            float L = 0.f;
            for (int s = c0 + lane; s <= c1; s += 32) {
                const float2 v = parts.pml[part_of(s) * parts.heads + h];
                L += v.y * exp2f(v.x - base);
            }
            L = warp_sum(L);
            bad = __any_sync(0xffffffffu, bad);
            if (lane == 0) sm.ml[slot][h] = make_float2(base, bad ? 0.f : 1.f / L);
        }
        __syncthreads();
        const int P = c1 - c0 + 1, outputs = G * kCacheHd;
        const int o0 = static_cast<int>(static_cast<long long>(outputs) * (b - c0) / P);
        const int o1 = static_cast<int>(static_cast<long long>(outputs) * (b - c0 + 1) / P);
        for (int i = o0 + tid; i < o1; i += kJoinThreads) {
            const int h = i / kCacheHd;
            const float2 ml = sm.ml[slot][h];
            float x = 0.f;
            for (int s = c0; s <= c1; ++s) {
                const size_t at = part_of(s) * parts.heads + h;
                x += parts.po[at * kCacheHd + i % kCacheHd] * exp2f(parts.pml[at].x - ml.x);
            }
            a.out[p.row * a.out_stride + static_cast<size_t>(p.head) * outputs + i] =
                f2bf(ml.y == 0.f ? __int_as_float(0x7FC00000) : x * ml.y);
        }
    }
    if (!a.accumulate) return;
    // ---- weights
    for (int k = warp; k < n; k += kJoinThreads / 32) {
        const long long t = t0 + k;
        const PlanPlace p = locate<kJoinThreads>(t, a.lens, c, sm.chunk);
        const long long run0 = t - p.tile;
        const bool whole = run0 >= t0 && run0 + p.tiles <= t0 + n;
        const int slot = run0 >= t0 ? 1 : 0;
        const int valid = min(kCachePage, p.len - p.tile * kCachePage);
        float* w = c.weights + cache_slot_index(c, p.row, p.head) + p.tile * kCachePage;
        const float2* whole_ml = parts.ml + static_cast<size_t>(p.row) * a.q_heads + p.head * G;
        for (int j = lane; j < valid; j += 32) {
            const float* s = parts.score + (t * kCachePage + j) * G;
            float sum = 0.f;
            bool bad = false;
            for (int h = 0; h < G; ++h) {
                float2 ml;
                if (whole) {
                    ml = whole_ml[h];
                    bad = bad || (ml.x == INFINITY && ml.y == 0.f);
                    ml = make_float2(ml.x == -INFINITY ? 0.f : ml.x, 1.f / ml.y);
                } else {
                    ml = sm.ml[slot][h];
                    bad = bad || ml.y == 0.f;
                }
                sum += exp2f(s[h] - ml.x) * ml.y;
            }
            if (!bad) w[j] += sum;
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

// Two resident CTAs an SM, no more than there can be tiles.
int shares_of(const CacheView& c, int sms) {
    return static_cast<int>(std::min(static_cast<size_t>(2 * sms), max_tiles(c)));
}

// The workspace's arrays from its start; returns its size.
size_t layout(const CacheView& c, int q_heads, int accumulate, int sms, uint8_t* ws, Parts* p) {
    const int G = q_heads / c.kv_heads, shares = shares_of(c, sms);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        uint8_t* to = ws + at;
        at += pad256(bytes);
        return to;
    };
    p->shares = shares;
    p->heads = G;
    p->ml = reinterpret_cast<float2*>(take(static_cast<size_t>(c.rows) * q_heads * 8));
    p->pml = reinterpret_cast<float2*>(take(static_cast<size_t>(shares) * 2 * G * 8));
    p->po = reinterpret_cast<float*>(take(static_cast<size_t>(shares) * 2 * G * kCacheHd * 4));
    p->score = reinterpret_cast<float*>(take(accumulate ? max_tiles(c) * kCachePage * G * 4 : 0));
    return at;
}

static_assert(2 * (sizeof(Smem<1>) + 1024 + 1024) <= 228 * 1024, "two CTAs must share an SM");
static_assert(2 * (sizeof(Smem<2>) + 1024 + 1024) <= 228 * 1024, "two CTAs must share an SM");

template <int NT>
cudaError_t launch_nt(const CacheAttnArgs& a, const Maps& maps, const Parts& parts, cudaStream_t s) {
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
    cache_attention_kernel<NT><<<parts.shares, kThreads, sizeof(Smem<NT>) + 1024, s>>>(a, maps, parts);
    return cudaGetLastError();
}

}  // namespace

size_t cache_attention_ws_bytes(const CacheView& c, int q_heads, int accumulate, int sms) {
    Parts p;
    return layout(c, q_heads, accumulate, sms, nullptr, &p);
}

cudaError_t launch_cache_attention(const CacheAttnArgs& a, int sms, cudaStream_t s) {
    const CacheView& c = a.c;
    Maps maps;
    const long long rows = static_cast<long long>(c.num_pages) * c.kv_heads * kCachePage;
    if (!make_map(&maps.k64, c.k, rows, 64) || !make_map(&maps.v64, c.v, rows, 64) ||
        !make_map(&maps.k16, c.k, rows, 16) || !make_map(&maps.v16, c.v, rows, 16))
        return cudaErrorInvalidValue;
    Parts parts;
    layout(c, a.q_heads, a.accumulate, sms, static_cast<uint8_t*>(a.ws), &parts);
    cudaError_t e = a.q_heads / c.kv_heads <= 8 ? launch_nt<1>(a, maps, parts, s) : launch_nt<2>(a, maps, parts, s);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(parts.shares);
    cfg.blockDim = dim3(kJoinThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, cache_join_kernel, a, parts);
}

}  // namespace q3
