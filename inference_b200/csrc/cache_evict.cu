// cache_evict.cu -- eviction from a bounded paged KV cache by accumulated
// attention weight.
//
// Per (sequence, kv head) longer than `keep`: the kept set is the `keep` largest
// slots by (recent, weight, lower slot).  The slots behind `keep` that are kept
// (movers) fill the slots before it that are not (holes), both in ascending
// order: there are as many of one as of the other, sources and targets do not
// overlap, and no other slot moves.
#include <algorithm>

#include "cache.cuh"

namespace q3 {
namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kMoveThreads = 256;

// Larger key = kept earlier.  Slots of the recent window come before every
// number, NaN after every number, and -0 equals +0.
__device__ __forceinline__ uint32_t evict_key(float w, bool recent) {
    if (recent) return 0xFFFFFFFFu;
    if (isnan(w)) return 0u;
    const uint32_t b = __float_as_uint(w + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

struct MoveLists {
    int32_t* count;  // [rows * kv_heads]
    int32_t *dst, *src;  // [rows * kv_heads][cap]
    int cap;
};

// Exclusive rank of this thread among the block's set flags, in thread order, and
// their number.
__device__ __forceinline__ int block_rank(bool flag, int* warp_counts, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned b = __ballot_sync(0xffffffffu, flag);
    if (lane == 0) warp_counts[warp] = __popc(b);
    __syncthreads();
    int before = 0;
    total = 0;
    for (int i = 0; i < kWarps; ++i) {
        if (i < warp) before += warp_counts[i];
        total += warp_counts[i];
    }
    __syncthreads();
    return before + __popc(b & ((1u << lane) - 1));
}

// One CTA per (sequence, kv head): radix select of the key of rank `keep`, 8 bits a
// pass, then the ordered lists of holes and movers.
__global__ void __launch_bounds__(kThreads) cache_evict_select_kernel(const CacheEvictArgs a, const MoveLists m) {
    const CacheView& c = a.c;
    const int rh = blockIdx.x, row = rh / c.kv_heads, head = rh % c.kv_heads, tid = threadIdx.x;
    __shared__ int hist[256];
    __shared__ int counts[kWarps];
    __shared__ uint32_t s_prefix, s_need;
    __shared__ int bad;
    const int len = a.lens[row];
    const size_t at = cache_slot_index(c, row, head);
    const float* w = c.weights + at;
    const int32_t* pos = c.positions + at;
    if (tid == 0) bad = len < 0 || len > c.max_len ? DEV_BAD_LENGTH : 0;
    __syncthreads();
    if (!bad && len > a.keep)
        for (int p = tid; p < (len + kCachePage - 1) / kCachePage; p += kThreads) {
            const int page = c.tables[row * c.table_stride + p];
            if (page < 0 || page >= c.num_pages) bad = DEV_BAD_PAGE;
        }
    __syncthreads();
    if (bad || len <= a.keep) {
        if (tid == 0) {
            m.count[rh] = bad ? -1 : 0;
            if (bad) record_error(c.err, bad);
        }
        if (!bad && a.weights_out)
            for (int s = tid; s < len; s += kThreads) {
                a.weights_out[at + s] = w[s];
                a.positions_out[at + s] = pos[s];
            }
        return;
    }
    const long long first_recent = static_cast<long long>(a.next_pos[row]) - a.recent;
    uint32_t prefix = 0, need = a.keep;
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int s = tid; s < len; s += kThreads) {
            const uint32_t k = evict_key(w[s], pos[s] >= first_recent);
            if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1);
        }
        __syncthreads();
        if (tid == 0) {
            uint32_t left = need;
            int d = 255;
            while (d > 0 && static_cast<uint32_t>(hist[d]) < left) left -= hist[d--];
            s_prefix = prefix | (static_cast<uint32_t>(d) << shift);
            s_need = left;
        }
        __syncthreads();
        prefix = s_prefix;
        need = s_need;
    }
    // kept: key above the threshold, or equal to it and among the first `need` such slots
    int ties = 0, holes = 0, movers = 0;
    int32_t* dst = m.dst + static_cast<size_t>(rh) * m.cap;
    int32_t* src = m.src + static_cast<size_t>(rh) * m.cap;
    for (int s0 = 0; s0 < len; s0 += kThreads) {
        const int s = s0 + tid;
        const bool in = s < len;
        const uint32_t k = in ? evict_key(w[s], pos[s] >= first_recent) : 0u;
        const bool tie = in && k == prefix;
        int n;
        const int tr = block_rank(tie, counts, n) + ties;
        ties += n;
        const bool kept = in && (k > prefix || (tie && tr < static_cast<int>(need)));
        const bool hole = s < a.keep && !kept, mover = s >= a.keep && kept;
        const int hr = block_rank(hole, counts, n) + holes;
        holes += n;
        const int mr = block_rank(mover, counts, n) + movers;
        movers += n;
        if (hole) dst[hr] = s;
        if (mover) src[mr] = s;
        if (kept && s < a.keep && a.weights_out) {
            a.weights_out[at + s] = w[s];
            a.positions_out[at + s] = pos[s];
        }
    }
    if (tid == 0) m.count[rh] = movers;
}

// Moves the listed slots: 16 lanes a slot, 16 bytes each of K and of V.
__global__ void __launch_bounds__(kMoveThreads) cache_evict_move_kernel(const CacheEvictArgs a, const MoveLists m,
                                                                        int chunks) {
    const CacheView& c = a.c;
    const int rh = blockIdx.x / chunks, chunk = blockIdx.x % chunks, row = rh / c.kv_heads, head = rh % c.kv_heads;
    const int n = m.count[rh];
    if (head == 0 && chunk == 0 && threadIdx.x == 0) {
        const int len = a.lens[row];
        a.lens_out[row] = n < 0 ? len : min(len, a.keep);
    }
    const size_t at = cache_slot_index(c, row, head);
    float* wo = a.weights_out ? a.weights_out : c.weights;
    int32_t* po = a.positions_out ? a.positions_out : c.positions;
    const int32_t* table = c.tables + row * c.table_stride;
    const int sub = threadIdx.x & 15;
    for (int i = chunk * (kMoveThreads / 16) + (threadIdx.x >> 4); i < n; i += chunks * (kMoveThreads / 16)) {
        const int d = m.dst[static_cast<size_t>(rh) * m.cap + i], s = m.src[static_cast<size_t>(rh) * m.cap + i];
        const size_t to = cache_kv_offset(c, table[d / kCachePage], head, d);
        const size_t of = cache_kv_offset(c, table[s / kCachePage], head, s);
        reinterpret_cast<uint4*>(c.k + to)[sub] = reinterpret_cast<const uint4*>(c.k + of)[sub];
        reinterpret_cast<uint4*>(c.v + to)[sub] = reinterpret_cast<const uint4*>(c.v + of)[sub];
        if (sub == 0) {
            wo[at + d] = c.weights[at + s];
            po[at + d] = c.positions[at + s];
        }
    }
}

size_t pad16(size_t n) { return (n + 15) & ~static_cast<size_t>(15); }

int max_moves(const CacheView& c, int keep) { return std::max(0, std::min(keep, c.max_len - keep)); }

}  // namespace

size_t cache_evict_ws_bytes(const CacheView& c, int keep) {
    const size_t rh = static_cast<size_t>(c.rows) * c.kv_heads;
    return pad16(rh * 4) + 2 * rh * max_moves(c, keep) * 4 + 16;
}

cudaError_t launch_cache_evict(const CacheEvictArgs& a, cudaStream_t s) {
    const int rh = a.c.rows * a.c.kv_heads;
    MoveLists m;
    m.cap = max_moves(a.c, a.keep);
    m.count = static_cast<int32_t*>(a.ws);
    m.dst = reinterpret_cast<int32_t*>(static_cast<uint8_t*>(a.ws) + pad16(static_cast<size_t>(rh) * 4));
    m.src = m.dst + static_cast<size_t>(rh) * m.cap;
    cache_evict_select_kernel<<<rh, kThreads, 0, s>>>(a, m);
    const int per = kMoveThreads / 16;
    const int chunks = std::max(1, std::min(64, (m.cap + per - 1) / per));
    cache_evict_move_kernel<<<rh * chunks, kMoveThreads, 0, s>>>(a, m, chunks);
    return cudaGetLastError();
}

}  // namespace q3
