// cache_evict.cu -- eviction from a bounded paged KV cache by accumulated
// attention weight.
//
// Per (sequence, kv head) longer than `keep`: the kept set is the `keep` largest
// slots by (recent, weight, lower slot).  The slots behind `keep` that are kept
// (movers) fill the slots before it that are not (holes), both in ascending
// order: there are as many of one as of the other, sources and targets do not
// overlap, and no other slot moves -- the fewest bytes that leave the kept slots
// in front.
//
// One thread-block cluster per (sequence, kv head), each CTA a contiguous piece of
// its slots.  The `keep`-th largest key is found by a radix
// select over 52 bits, weight above (inverted) slot, so that no two keys are
// equal: 2048-bin histograms of 11 bits a pass, summed over the cluster through
// distributed shared memory, until at most 256 candidates are left, which are
// ranked by counting (one or two passes for weights of a usual spread).  Then a
// bitmap of the kept slots, the ordered lists of holes and movers from its
// population counts, and the moves, 16 lanes a slot and tensor: by the same CTAs
// where at most 64 slots a head can move, else by a second launch over all SMs.
// Bound: latency (a dozen dependent steps of 0.3 to 0.5 us) for a few evicted
// slots, HBM for many: 8 bytes a slot read, 1 KB a moved slot.
#include <algorithm>
#include <atomic>
#include <climits>

#include "cache.cuh"

namespace q3 {
namespace {

constexpr int kThreads = 512;               // two CTAs an SM
constexpr int kWarps = kThreads / 32;
constexpr int kHeld = 8;                    // slots a thread holds in registers (more are read again in every pass)
constexpr int kDigit = 11;                  // bits a pass
constexpr int kBins = 1 << kDigit;
constexpr int kSlotBits = 20;               // max_len <= 2^20
constexpr int kTopShift = 32 + kSlotBits - kDigit;
constexpr int kCandidates = 256;
constexpr int kMaxCluster = 8;
constexpr int kMovesHere = 64;  // at most so many moves a head: by the selecting CTAs
constexpr int kMoveThreads = 256;
constexpr int kMoveChunk = 64;
static_assert(kBins == 4 * kThreads && kCandidates * 2 == kThreads, "bins and candidates are dealt to the threads");

// Larger key = kept earlier.  Slots of the recent window come before every
// number, NaN after every number, and -0 equals +0; among equals the lower slot.
__device__ __forceinline__ uint64_t evict_key(float w, bool recent, int slot) {
    uint32_t k = 0u;
    if (recent) {
        k = 0xFFFFFFFFu;
    } else if (!isnan(w)) {
        const uint32_t b = __float_as_uint(w + 0.0f);
        k = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    }
    return (static_cast<uint64_t>(k) << kSlotBits) | static_cast<uint32_t>((1 << kSlotBits) - 1 - slot);
}

// A slot and the row of the K and V pools that holds it: (page * kv_heads + head) * 64 + slot % 64.
struct Lists {
    int32_t* bad;     // [rows]: the sequence has a bad length or page and stays as it is
    int32_t* count;   // [rows * kv_heads]: moves
    int2 *dst, *src;  // [rows * kv_heads][cap]: holes and movers
    int cap;
};

struct Smem {
    int hist[2][kBins];  // alternately: one is cleared while peers may still read the other
    uint64_t mine[kCandidates], all[kCandidates];
    int2 dst[kMovesHere], src[kMovesHere];
    int n_mine;
    int warp_sum[kWarps];
    int warp_holes[kWarps], warp_movers[kWarps];
    int holes, movers;       // of this CTA's piece
    int digit, need, count;  // the bin that holds the threshold
    uint64_t threshold;
    uint32_t kept[];  // bitmap of the piece
};

// Moves i = first, first + step, ... below n, each by the 16 lanes that share `first`:
// 16 bytes of K and of V a lane, four moves in flight.
__device__ __forceinline__ void move_slots(const CacheEvictArgs& a, const int2* dst, const int2* src, size_t at, int first,
                                           int step, int n) {
    const CacheView& c = a.c;
    float* wo = a.weights_out ? a.weights_out : c.weights;
    int32_t* po = a.positions_out ? a.positions_out : c.positions;
    const int sub = threadIdx.x & 15;
    const uint4 *kp = reinterpret_cast<const uint4*>(c.k) + sub, *vp = reinterpret_cast<const uint4*>(c.v) + sub;
    constexpr int U = 4;
    for (int i = first; i < n; i += U * step) {
        int2 d[U], s[U];
        uint4 k[U], v[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + u * step < n) d[u] = dst[i + u * step], s[u] = src[i + u * step];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + u * step < n) k[u] = kp[static_cast<size_t>(s[u].y) * 16], v[u] = vp[static_cast<size_t>(s[u].y) * 16];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + u * step < n) {
                const_cast<uint4*>(kp)[static_cast<size_t>(d[u].y) * 16] = k[u];
                const_cast<uint4*>(vp)[static_cast<size_t>(d[u].y) * 16] = v[u];
                // one lane a move takes its weight, another its position
                if (sub == 0) wo[at + d[u].x] = c.weights[at + s[u].x];
                if (sub == 1) po[at + d[u].x] = c.positions[at + s[u].x];
            }
    }
}

// `p` of this CTA's shared memory in cluster CTA `rank`.
template <class T>
__device__ __forceinline__ const T* peer(const T* p, int rank) {
    return static_cast<const T*>(map_cluster_rank(const_cast<T*>(p), static_cast<uint32_t>(rank)));
}

// A barrier over the cluster that orders shared and global memory.
template <int C>
__device__ __forceinline__ void cluster_sync() {
    if constexpr (C == 1) {
        __syncthreads();
    } else {
        __syncwarp();  // the cluster's barrier instructions are warp-aligned
        cluster_arrive_release();
        cluster_wait();
    }
}

template <int C>
__global__ void __launch_bounds__(kThreads, 2) cache_evict_kernel(const CacheEvictArgs a, const Lists m, int moves_here) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
    const CacheView& c = a.c;
    const int rh = blockIdx.x / C, rank = blockIdx.x % C, row = rh / c.kv_heads, head = rh % c.kv_heads;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int len = a.lens[row];
    const int first_recent =
        static_cast<int>(max(static_cast<long long>(a.next_pos[row]) - a.recent, static_cast<long long>(INT_MIN)));
    const int32_t* table = c.tables + row * c.table_stride;
    const size_t at = cache_slot_index(c, row, head);
    const float* w = c.weights + at;
    const int32_t* pos = c.positions + at;
    if (!moves_here) pdl_trigger();
    for (int i = tid; i < kBins; i += kThreads) sm.hist[0][i] = 0;
    if (tid == 0) sm.n_mine = 0;

    // the piece: words of 32 slots, a warp a contiguous run of them
    const bool length_ok = len >= 0 && len <= c.max_len, shrinks = length_ok && len > a.keep;
    const int words = length_ok ? (len + 31) / 32 : 0;
    const int word0 = static_cast<int>(static_cast<long long>(words) * rank / C);
    const int nw = static_cast<int>(static_cast<long long>(words) * (rank + 1) / C) - word0;
    const int wa = nw * warp / kWarps, wb = nw * (warp + 1) / kWarps;
    float hx[kHeld];
    int32_t hp[kHeld];
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
        const int s = (word0 + wa + u) * 32 + lane;
        const bool in = wa + u < wb && s < len;
        hx[u] = in ? w[s] : 0.f;
        hp[u] = in ? pos[s] : 0;
    }
    // f(word of the piece, slot, weight, position) for the warp's words, by the whole warp
    auto each_word = [&](auto&& f) {
#pragma unroll
        for (int u = 0; u < kHeld; ++u)
            if (wa + u < wb) f(wa + u, (word0 + wa + u) * 32 + lane, hx[u], hp[u]);
        for (int i = wa + kHeld; i < wb; i += 4) {
            float x[4];
            int32_t p[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int s = (word0 + i + u) * 32 + lane;
                const bool in = i + u < wb && s < len;
                x[u] = in ? w[s] : 0.f;
                p[u] = in ? pos[s] : 0;
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (i + u < wb) f(i + u, (word0 + i + u) * 32 + lane, x[u], p[u]);
        }
    };
    uint32_t bad = length_ok ? DEV_OK : DEV_BAD_LENGTH;
    if (shrinks)
        for (int p = tid; p < (len + kCachePage - 1) / kCachePage; p += kThreads)
            if (table[p] < 0 || table[p] >= c.num_pages) bad = DEV_BAD_PAGE;
    const bool stays = __syncthreads_or(bad) != 0;
    if (bad && rank == 0) record_error(c.err, bad);

    // Lengths are read by every CTA of a sequence, and lens_out may be the same array: the
    // last CTA of the grid to come here, when all have read theirs, writes it (at its end).
    bool last = false;
    if (tid == kThreads - 1) {
        if (head == 0 && rank == 0) m.bad[row] = stays;
        __threadfence();
        last = atomicAdd(c.arrived, 1u) == gridDim.x - 1;
        if (last) {
            __threadfence();
            *c.arrived = 0;
        }
    }
    auto finish = [&]() {
        if (!__syncthreads_or(last)) return;
        for (int r = tid; r < c.rows; r += kThreads) {
            const int n = a.lens[r];
            a.lens_out[r] = __ldcg(m.bad + r) ? n : min(n, a.keep);
        }
    };
    if (stays || !shrinks) {
        if (tid == 0 && rank == 0) m.count[rh] = 0;
        if (!stays && a.weights_out)
            each_word([&](int, int s, float x, int32_t p) {
                if (s < len) a.weights_out[at + s] = x, a.positions_out[at + s] = p;
            });
        finish();
        return;
    }

    // ---- the threshold: the keep-th largest key
    uint64_t prefix = 0;
    int need = a.keep;
    // at the last shift, 8, at most 256 slots share a prefix: the loop ends by a break
    for (int pass = 0, shift = kTopShift; shift >= 0; ++pass, shift -= kDigit) {
        int* hist = sm.hist[pass & 1];
        if (pass > 0) {
            for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
            __syncthreads();
        }
        each_word([&](int, int s, float x, int32_t p) {
            const uint64_t k = evict_key(x, p >= first_recent, s);
            const bool in = s < len && (k >> (shift + kDigit)) == prefix;
            const unsigned here = __ballot_sync(0xffffffffu, in);
            if (!here) return;
            const int d = static_cast<int>(k >> shift) & (kBins - 1);
            // lanes with one digit between them (equal weights) count as one
            const int first = __ffs(here) - 1;
            const int theirs = __shfl_sync(0xffffffffu, d, first);
            const bool same = __all_sync(0xffffffffu, !in || d == theirs) != 0;
            if (!same) {
                if (in) atomicAdd(&hist[d], 1);
            } else if (lane == first) {
                atomicAdd(&hist[d], __popc(here));
            }
        });
        cluster_sync<C>();
        // thread t has the bins 2047 - 4 t - i, i = 0 .. 3, from the top
        int4 part[C];
#pragma unroll
        for (int r = 0; r < C; ++r)
            part[r] = reinterpret_cast<const int4*>(C == 1 ? hist : peer(hist, r))[kBins / 4 - 1 - tid];
        int four[4] = {0, 0, 0, 0};
#pragma unroll
        for (int r = 0; r < C; ++r) four[0] += part[r].w, four[1] += part[r].z, four[2] += part[r].y, four[3] += part[r].x;
        const int all = four[0] + four[1] + four[2] + four[3];
        int incl = all;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
        }
        if (lane == 31) sm.warp_sum[warp] = incl;
        __syncthreads();
        // larger than this thread's bins: the warps and lanes before
        int above = __reduce_add_sync(0xffffffffu, lane < warp ? sm.warp_sum[lane & (kWarps - 1)] : 0) + incl - all;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (above < need && need <= above + four[i])
                sm.digit = kBins - 1 - 4 * tid - i, sm.need = need - above, sm.count = four[i];
            above += four[i];
        }
        __syncthreads();
        prefix = (prefix << kDigit) | static_cast<uint64_t>(sm.digit);
        need = sm.need;
        const int count = sm.count;
        if (count == need) {  // the whole bin is kept
            if (tid == 0) sm.threshold = prefix << shift;
            break;
        }
        if (count <= kCandidates) {
            // few candidates: the one with need - 1 larger ones is the threshold
            each_word([&](int, int s, float x, int32_t p) {
                const uint64_t k = evict_key(x, p >= first_recent, s);
                if (s < len && (k >> shift) == prefix) sm.mine[atomicAdd(&sm.n_mine, 1)] = k;
            });
            cluster_sync<C>();
            const uint64_t* from = sm.mine;
            if constexpr (C > 1) {
                int nr[C], n = 0;
#pragma unroll
                for (int r = 0; r < C; ++r) nr[r] = *peer(&sm.n_mine, r);
#pragma unroll
                for (int r = 0; r < C; ++r) {
                    if (tid < nr[r]) sm.all[n + tid] = peer(sm.mine, r)[tid];
                    n += nr[r];
                }
                from = sm.all;
                __syncthreads();
            }
            // two threads a candidate
            const int i = tid >> 1;
            if (i < count) {
                const uint64_t k = from[i];
                int larger = 0;
#pragma unroll 8
                for (int j = tid & 1; j < count; j += 2) larger += from[j] > k;
                larger += __shfl_xor_sync(0x3u << (lane & ~1), larger, 1);
                if (larger == need - 1 && (tid & 1) == 0) sm.threshold = k;
            }
            break;
        }
    }
    __syncthreads();
    const uint64_t threshold = sm.threshold;

    // ---- the kept slots' bitmap
    // bit i of the mask: slot 32 * word + i is below keep
    auto below = [&](int word) {
        const int n = a.keep - word * 32;
        return n >= 32 ? 0xFFFFFFFFu : n <= 0 ? 0u : (1u << n) - 1;
    };
    int holes = 0, movers = 0;
    each_word([&](int i, int s, float x, int32_t p) {
        const bool keep = s < len && evict_key(x, p >= first_recent, s) >= threshold;
        const uint32_t mask = __ballot_sync(0xffffffffu, keep), low = below(word0 + i);
        if (lane == 0) sm.kept[i] = mask;
        holes += __popc(~mask & low);
        movers += __popc(mask & ~low);
        if (a.weights_out && keep && s < a.keep) a.weights_out[at + s] = x, a.positions_out[at + s] = p;
    });
    if (lane == 0) sm.warp_holes[warp] = holes, sm.warp_movers[warp] = movers;
    __syncthreads();
    // lists in order: the pieces before this one, the warps before this one
    const int my_holes = lane < kWarps ? sm.warp_holes[lane] : 0, my_movers = lane < kWarps ? sm.warp_movers[lane] : 0;
    int hole = __reduce_add_sync(0xffffffffu, lane < warp ? my_holes : 0);
    int mover = __reduce_add_sync(0xffffffffu, lane < warp ? my_movers : 0);
    int n = __reduce_add_sync(0xffffffffu, my_movers);
    if constexpr (C > 1) {
        const int piece_holes = __reduce_add_sync(0xffffffffu, my_holes);
        if (tid == 0) sm.holes = piece_holes, sm.movers = n;
        cluster_sync<C>();
        int h[C], v[C];
#pragma unroll
        for (int r = 0; r < C; ++r) h[r] = *peer(&sm.holes, r), v[r] = *peer(&sm.movers, r);
        n = 0;
#pragma unroll
        for (int r = 0; r < C; ++r) {
            if (r < rank) hole += h[r], mover += v[r];
            n += v[r];
        }
    }
    // one CTA's few moves stay in its shared memory
    const bool local = C == 1 && moves_here;
    int2* dst = local ? sm.dst : m.dst + static_cast<size_t>(rh) * m.cap;
    int2* src = local ? sm.src : m.src + static_cast<size_t>(rh) * m.cap;
    const unsigned lower = (1u << lane) - 1;
    auto place_of = [&](int s) { return make_int2(s, (table[s / kCachePage] * c.kv_heads + head) * kCachePage + s % kCachePage); };
    for (int i = wa; i < wb; ++i) {
        const uint32_t mask = sm.kept[i], low = below(word0 + i), h = ~mask & low, v = mask & ~low;
        const int s = (word0 + i) * 32 + lane;
        if (h >> lane & 1) dst[hole + __popc(h & lower)] = place_of(s);
        if (v >> lane & 1) src[mover + __popc(v & lower)] = place_of(s);
        hole += __popc(h);
        mover += __popc(v);
    }
    if (moves_here) {
        cluster_sync<C>();
        move_slots(a, dst, src, at, rank * (kThreads / 16) + (tid >> 4), C * (kThreads / 16), n);
    } else {
        if (tid == 0 && rank == 0) m.count[rh] = n;
        if (C > 1) cluster_sync<C>();  // peers may still read this CTA's shared memory
    }
    finish();
}

// 64 moves a CTA.
__global__ void __launch_bounds__(kMoveThreads, 4) cache_evict_move_kernel(const CacheEvictArgs a, const Lists m, int chunks) {
    const int rh = blockIdx.x / chunks, first = blockIdx.x % chunks * kMoveChunk;
    pdl_wait();
    const int n = min(m.count[rh], first + kMoveChunk);
    const size_t list = static_cast<size_t>(rh) * m.cap;
    move_slots(a, m.dst + list, m.src + list, static_cast<size_t>(rh) * a.c.slot_stride, first + (threadIdx.x >> 4),
               kMoveThreads / 16, n);
}

size_t pad16(size_t n) { return (n + 15) & ~static_cast<size_t>(15); }

int max_moves(const CacheView& c, int keep) { return std::max(0, std::min(keep, c.max_len - keep)); }

// CTAs a (sequence, kv head): as many as leave no more than one CTA an SM (so that
// few long sequences use the whole GPU), each with at least 1024 slots.
int cluster_of(const CacheView& c, int sms) {
    const long long rh = static_cast<long long>(c.rows) * c.kv_heads;
    int C = 1;
    while (C < kMaxCluster && rh * C * 2 <= sms && c.max_len / (C * 2) >= 1024) C *= 2;
    return C;
}

template <int C>
cudaError_t launch_select(const CacheEvictArgs& a, const Lists& m, int moves_here, cudaStream_t s) {
    const CacheView& c = a.c;
    static std::atomic<uint64_t> configured{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (!(configured.load() & bit)) {
        e = cudaFuncSetAttribute(cache_evict_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 static_cast<int>(sizeof(Smem) + ((1 << kSlotBits) / 32 + 2) * 4));
        if (e != cudaSuccess) return e;
        configured.fetch_or(bit);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(c.rows) * c.kv_heads * C);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = sizeof(Smem) + (static_cast<size_t>(c.max_len) / 32 / C + 2) * 4;  // the largest piece's bitmap
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, cache_evict_kernel<C>, a, m, moves_here);
}

}  // namespace

size_t cache_evict_ws_bytes(const CacheView& c, int keep) {
    const size_t rh = static_cast<size_t>(c.rows) * c.kv_heads;
    return pad16(static_cast<size_t>(c.rows) * 4) + pad16(rh * 4) + 2 * rh * max_moves(c, keep) * 8 + 16;
}

cudaError_t launch_cache_evict(const CacheEvictArgs& a, int sms, cudaStream_t s) {
    const CacheView& c = a.c;
    const size_t rh = static_cast<size_t>(c.rows) * c.kv_heads;
    Lists m;
    m.cap = max_moves(c, a.keep);
    uint8_t* ws = static_cast<uint8_t*>(a.ws);
    m.bad = reinterpret_cast<int32_t*>(ws);
    m.count = reinterpret_cast<int32_t*>(ws += pad16(static_cast<size_t>(c.rows) * 4));
    m.dst = reinterpret_cast<int2*>(ws + pad16(rh * 4));
    m.src = m.dst + rh * m.cap;
    const int moves_here = m.cap <= kMovesHere;
    cudaError_t e = cudaSuccess;
    switch (cluster_of(c, sms)) {
        case 1: e = launch_select<1>(a, m, moves_here, s); break;
        case 2: e = launch_select<2>(a, m, moves_here, s); break;
        case 4: e = launch_select<4>(a, m, moves_here, s); break;
        default: e = launch_select<8>(a, m, moves_here, s);
    }
    if (e != cudaSuccess || moves_here) return e;
    const int chunks = (m.cap + kMoveChunk - 1) / kMoveChunk;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(rh) * chunks);
    cfg.blockDim = dim3(kMoveThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, cache_evict_move_kernel, a, m, chunks);
}

}  // namespace q3
