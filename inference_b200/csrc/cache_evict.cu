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
// One launch, one thread-block cluster per (sequence, kv head), each CTA a
// contiguous piece of its slots.  The `keep`-th largest key is found by a radix
// select over 52 bits, weight above (inverted) slot, so that no two keys are
// equal: 2048-bin histograms of 11 bits a pass, summed over the cluster through
// distributed shared memory, until at most 256 candidates are left, which are
// ranked by counting (one or two passes for weights of a usual spread).  Then a
// bitmap of the kept slots, the ordered lists of holes and movers from its
// population counts, and the moves, 16 lanes a slot and tensor.  Bound: latency
// (a dozen dependent steps of 0.3 to 0.5 us) for a few evicted slots, HBM for
// many: 8 bytes a slot read, 1 KB a moved slot.
#include <algorithm>
#include <atomic>

#include "cache.cuh"

namespace q3 {
namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kDigit = 11;                  // bits a pass
constexpr int kBins = 1 << kDigit;
constexpr int kSlotBits = 20;               // max_len <= 2^20
constexpr int kTopShift = 32 + kSlotBits - kDigit;
constexpr int kCandidates = 256;
constexpr int kMaxCluster = 8;

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

struct Lists {
    int32_t* bad;        // [rows]: the sequence has a bad length or page and stays as it is
    int32_t *dst, *src;  // [rows * kv_heads][cap]: holes and movers
    int cap;
};

struct Smem {
    int hist[2][kBins];  // alternately: one is cleared while peers may still read the other
    uint64_t mine[kCandidates], all[kCandidates];
    int n_mine;
    int warp_sum[kWarps];
    int warp_holes[kWarps], warp_movers[kWarps];
    int holes, movers;       // of this CTA's piece
    int digit, need, count;  // the bin that holds the threshold
    uint64_t threshold;
    bool last;
    uint32_t kept[];  // bitmap of the piece
};

// The peer's view of a shared-memory object.
template <class T>
__device__ __forceinline__ const T* peer(const T* p, int rank) {
    return static_cast<const T*>(map_cluster_rank(const_cast<T*>(p), static_cast<uint32_t>(rank)));
}

// A barrier over the cluster that orders shared and global memory.
__device__ __forceinline__ void cluster_sync(int C) {
    if (C == 1) {
        __syncthreads();
    } else {
        cluster_arrive_release();
        cluster_wait();
    }
}

__global__ void __launch_bounds__(kThreads) cache_evict_kernel(const CacheEvictArgs a, const Lists m, int C) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
    const CacheView& c = a.c;
    const int rh = blockIdx.x / C, rank = blockIdx.x % C, row = rh / c.kv_heads, head = rh % c.kv_heads;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int len = a.lens[row];
    const long long first_recent = static_cast<long long>(a.next_pos[row]) - a.recent;
    const int32_t* table = c.tables + row * c.table_stride;
    const size_t at = cache_slot_index(c, row, head);
    const float* w = c.weights + at;
    const int32_t* pos = c.positions + at;
    // the piece: whole words of 32 slots
    const int words = (max(len, 0) + 31) / 32;
    const int word0 = static_cast<int>(static_cast<long long>(words) * rank / C);
    const int word1 = static_cast<int>(static_cast<long long>(words) * (rank + 1) / C);
    const int s0 = word0 * 32, s1 = min(len, word1 * 32);
    // f(key) for every slot of the piece, four slots' loads in flight a thread
    auto each_key = [&](auto&& f) {
        for (int s = s0 + tid; s < s1; s += 4 * kThreads) {
            float x[4];
            int32_t p[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (s + u * kThreads < s1) x[u] = w[s + u * kThreads], p[u] = pos[s + u * kThreads];
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (s + u * kThreads < s1) f(evict_key(x[u], p[u] >= first_recent, s + u * kThreads));
        }
    };

    uint32_t bad = len < 0 || len > c.max_len ? DEV_BAD_LENGTH : DEV_OK;
    if (!bad && len > a.keep)
        for (int p = tid; p < (len + kCachePage - 1) / kCachePage; p += kThreads)
            if (table[p] < 0 || table[p] >= c.num_pages) bad = DEV_BAD_PAGE;
    for (int i = tid; i < kBins; i += kThreads) sm.hist[0][i] = 0;
    if (tid == 0) sm.n_mine = 0;
    const bool stays = __syncthreads_or(bad) != 0;
    if (bad && rank == 0) record_error(c.err, bad);

    // Lengths are read by every CTA of a sequence, and lens_out may be the same array: the
    // last CTA of the grid to come here, when all have read theirs, writes it.
    if (tid == 0) {
        if (head == 0 && rank == 0) m.bad[row] = stays;
        __threadfence();
        sm.last = atomicAdd(c.arrived, 1u) == gridDim.x - 1;
        if (sm.last) __threadfence();
    }
    __syncthreads();
    if (sm.last) {
        if (tid == 0) *c.arrived = 0;
        for (int r = tid; r < c.rows; r += kThreads) {
            const int n = a.lens[r];
            a.lens_out[r] = __ldcg(m.bad + r) ? n : min(n, a.keep);
        }
    }
    if (stays) return;
    if (len <= a.keep) {
        if (a.weights_out)
            for (int s = s0 + tid; s < s1; s += kThreads) {
                a.weights_out[at + s] = w[s];
                a.positions_out[at + s] = pos[s];
            }
        return;
    }

    // ---- the threshold: the keep-th largest key
    uint64_t prefix = 0;
    int need = a.keep;
    for (int pass = 0, shift = kTopShift;; ++pass) {
        int* hist = sm.hist[pass & 1];
        if (pass > 0) {
            for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
            __syncthreads();
        }
        each_key([&](uint64_t k) {
            if ((k >> (shift + kDigit)) != prefix) return;
            const int d = static_cast<int>(k >> shift) & (kBins - 1);
            // lanes with one digit between them (equal weights) count as one
            const unsigned here = __activemask();
            int same = 0;
            __match_all_sync(here, d, &same);
            if (!same)
                atomicAdd(&hist[d], 1);
            else if (lane == __ffs(here) - 1)
                atomicAdd(&hist[d], __popc(here));
        });
        cluster_sync(C);
        // from the top: thread t has the bins 2047 - 2 t and 2046 - 2 t
        int hi = 0, lo = 0;
        for (int r = 0; r < C; ++r) {
            const int* h = C == 1 ? hist : peer(hist, r);
            hi += h[kBins - 1 - 2 * tid];
            lo += h[kBins - 2 - 2 * tid];
        }
        int incl = hi + lo;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
        }
        if (lane == 31) sm.warp_sum[warp] = incl;
        __syncthreads();
        {
            int before = lane < warp ? sm.warp_sum[lane] : 0;
            before = __reduce_add_sync(0xffffffffu, before);
            const int above = before + incl - hi - lo;  // larger than this thread's bins
            if (above < need && need <= above + hi) {
                sm.digit = kBins - 1 - 2 * tid, sm.need = need - above, sm.count = hi;
            } else if (above + hi < need && need <= above + hi + lo) {
                sm.digit = kBins - 2 - 2 * tid, sm.need = need - above - hi, sm.count = lo;
            }
        }
        __syncthreads();
        prefix = (prefix << kDigit) | static_cast<uint64_t>(sm.digit);
        need = sm.need;
        if (sm.count == need) {  // the whole bin is kept
            if (tid == 0) sm.threshold = prefix << shift;
            break;
        }
        if (sm.count <= kCandidates) {
            // few candidates: the one with need - 1 larger ones is the threshold
            each_key([&](uint64_t k) {
                if ((k >> shift) == prefix) sm.mine[atomicAdd(&sm.n_mine, 1)] = k;
            });
            cluster_sync(C);
            int n = 0;
            for (int r = 0; r < C; ++r) {
                const int nr = C == 1 ? sm.n_mine : *peer(&sm.n_mine, r);
                if (tid < nr) sm.all[n + tid] = C == 1 ? sm.mine[tid] : peer(sm.mine, r)[tid];
                n += nr;
            }
            __syncthreads();
            // four threads a candidate
            const int i = tid >> 2;
            if (i < n) {
                const uint64_t k = sm.all[i];
                int larger = 0;
                for (int j = tid & 3; j < n; j += 4) larger += sm.all[j] > k;
                const unsigned quad = 0xFu << (lane & ~3);
                larger += __shfl_xor_sync(quad, larger, 1);
                larger += __shfl_xor_sync(quad, larger, 2);
                if (larger == need - 1 && (tid & 3) == 0) sm.threshold = k;
            }
            break;
        }
        shift -= kDigit;  // at shift 8 at most 256 slots share a prefix
    }
    __syncthreads();
    const uint64_t threshold = sm.threshold;

    // ---- the kept slots' bitmap, a warp a contiguous run of words
    const int nw = word1 - word0;
    const int wa = static_cast<int>(static_cast<long long>(nw) * warp / kWarps);
    const int wb = static_cast<int>(static_cast<long long>(nw) * (warp + 1) / kWarps);
    // bit i of the mask: slot 32 * word + i is below keep
    auto below = [&](int word) {
        const int n = a.keep - word * 32;
        return n >= 32 ? 0xFFFFFFFFu : n <= 0 ? 0u : (1u << n) - 1;
    };
    int holes = 0, movers = 0;
#pragma unroll 4
    for (int i = wa; i < wb; ++i) {
        const int s = (word0 + i) * 32 + lane;
        const bool in = s < len;
        const float x = in ? w[s] : 0.f;
        const int32_t p = in ? pos[s] : 0;
        const bool keep = in && evict_key(x, p >= first_recent, s) >= threshold;
        const uint32_t mask = __ballot_sync(0xffffffffu, keep), low = below(word0 + i);
        if (lane == 0) sm.kept[i] = mask;
        holes += __popc(~mask & low);
        movers += __popc(mask & ~low);
        if (a.weights_out && keep && s < a.keep) {
            a.weights_out[at + s] = x;
            a.positions_out[at + s] = p;
        }
    }
    if (lane == 0) sm.warp_holes[warp] = holes, sm.warp_movers[warp] = movers;
    __syncthreads();
    // lists in order: the pieces before this one, the warps before this one
    const int my_holes = lane < kWarps ? sm.warp_holes[lane] : 0, my_movers = lane < kWarps ? sm.warp_movers[lane] : 0;
    int hole = __reduce_add_sync(0xffffffffu, lane < warp ? my_holes : 0);
    int mover = __reduce_add_sync(0xffffffffu, lane < warp ? my_movers : 0);
    const int piece_holes = __reduce_add_sync(0xffffffffu, my_holes);
    const int piece_movers = __reduce_add_sync(0xffffffffu, my_movers);
    int n = piece_movers;
    if (C > 1) {
        if (tid == 0) sm.holes = piece_holes, sm.movers = piece_movers;
        cluster_sync(C);
        n = 0;
        for (int r = 0; r < C; ++r) {
            const int h = *peer(&sm.holes, r), v = *peer(&sm.movers, r);
            if (r < rank) hole += h, mover += v;
            n += v;
        }
    }
    int32_t* dst = m.dst + static_cast<size_t>(rh) * m.cap;
    int32_t* src = m.src + static_cast<size_t>(rh) * m.cap;
    const unsigned lower = (1u << lane) - 1;
    for (int i = wa; i < wb; ++i) {
        const uint32_t mask = sm.kept[i], low = below(word0 + i), h = ~mask & low, v = mask & ~low;
        const int s = (word0 + i) * 32 + lane;
        if (h >> lane & 1) dst[hole + __popc(h & lower)] = s;
        if (v >> lane & 1) src[mover + __popc(v & lower)] = s;
        hole += __popc(h);
        mover += __popc(v);
    }
    cluster_sync(C);

    // ---- the moves, 16 lanes a slot, 16 bytes each of K and of V
    float* wo = a.weights_out ? a.weights_out : c.weights;
    int32_t* po = a.positions_out ? a.positions_out : c.positions;
    const int sub = tid & 15, step = C * (kThreads / 16);
#pragma unroll 2
    for (int i = rank * (kThreads / 16) + (tid >> 4); i < n; i += step) {
        const int d = __ldcg(dst + i), s = __ldcg(src + i);
        const size_t to = cache_kv_offset(c, table[d / kCachePage], head, d) + sub * 8;
        const size_t of = cache_kv_offset(c, table[s / kCachePage], head, s) + sub * 8;
        const uint4 k = *reinterpret_cast<const uint4*>(c.k + of), v = *reinterpret_cast<const uint4*>(c.v + of);
        *reinterpret_cast<uint4*>(c.k + to) = k;
        *reinterpret_cast<uint4*>(c.v + to) = v;
        if (sub == 0) {
            wo[at + d] = c.weights[at + s];
            po[at + d] = c.positions[at + s];
        }
    }
}

size_t pad16(size_t n) { return (n + 15) & ~static_cast<size_t>(15); }

int max_moves(const CacheView& c, int keep) { return std::max(0, std::min(keep, c.max_len - keep)); }

// CTAs a (sequence, kv head): as many as leave no more than one CTA an SM (so that
// few long sequences use the whole GPU), each with at least 2048 slots.
int cluster_of(const CacheView& c, int sms) {
    const long long rh = static_cast<long long>(c.rows) * c.kv_heads;
    int C = 1;
    while (C < kMaxCluster && rh * C * 2 <= sms && c.max_len / (C * 2) >= 2048) C *= 2;
    return C;
}

}  // namespace

size_t cache_evict_ws_bytes(const CacheView& c, int keep) {
    const size_t rh = static_cast<size_t>(c.rows) * c.kv_heads;
    return pad16(static_cast<size_t>(c.rows) * 4) + 2 * rh * max_moves(c, keep) * 4 + 16;
}

cudaError_t launch_cache_evict(const CacheEvictArgs& a, int sms, cudaStream_t s) {
    const CacheView& c = a.c;
    const int rh = c.rows * c.kv_heads, C = cluster_of(c, sms);
    Lists m;
    m.cap = max_moves(c, a.keep);
    m.bad = static_cast<int32_t*>(a.ws);
    m.dst = reinterpret_cast<int32_t*>(static_cast<uint8_t*>(a.ws) + pad16(static_cast<size_t>(c.rows) * 4));
    m.src = m.dst + static_cast<size_t>(rh) * m.cap;
    // the bitmap of the largest piece
    const size_t smem = sizeof(Smem) + (static_cast<size_t>(c.max_len) / 32 / C + 2) * 4;
    static std::atomic<uint64_t> configured{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (!(configured.load() & bit)) {
        e = cudaFuncSetAttribute(cache_evict_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 static_cast<int>(sizeof(Smem) + ((1 << kSlotBits) / 32 + 2) * 4));
        if (e != cudaSuccess) return e;
        configured.fetch_or(bit);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(rh) * C);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, cache_evict_kernel, a, m, C);
}

}  // namespace q3
