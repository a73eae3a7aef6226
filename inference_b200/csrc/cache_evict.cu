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
// its slots.  The weight of the `keep`-th slot is found by a radix select over the
// weights' 32-bit order-preserving keys: a histogram of the next 11 bits (8 in a
// cluster, whose CTAs read each other's through distributed shared memory) of the
// slots that share the bits so far -- at first of the bits that tell usual weights
// apart -- until at most 256 candidates are left, which are ranked by counting;
// usually one or two passes.  More candidates than that with all
// bits equal are a tie, cut by slot.  Then a bitmap of the kept slots, the ordered
// lists of holes and movers from its population counts, and the moves, 16 lanes a
// slot and tensor: by the same CTAs where at most 64 slots a head can move, else by
// a second launch over all SMs.  Bound: latency (a dozen dependent steps of 0.3 to
// 0.7 us) for a few evicted slots, HBM for many: 8 bytes a slot read, 1 KB a moved
// slot.
//
// Measured (B200, captured into a graph), 8 kv heads:
//   16 sequences, 2112 -> 2048 slots   9.0 us, all latency: launch, two passes of the
//                                      select, lists, moves by the same CTAs (a second
//                                      launch instead: 1.8 us more)
//   one, 32768 -> 4096                 22.2 us: select 13 (clusters of 8, exchanges of
//                                      histograms), moves 9
//   32, up to 8000 -> 2000             62 us: select 18, moves 41 at 5.75 TB/s, 88 % of
//                                      the measured copy rate
// Clusters of 16 CTAs and digits of 11 bits in clusters were slower.
#include <algorithm>
#include <atomic>
#include <climits>

#include "cache.cuh"

namespace q3 {
namespace {

constexpr int kThreads = 512;               // two CTAs an SM
constexpr int kWarps = kThreads / 32;
constexpr int kKeysHere = 20480;            // a piece's keys stay in shared memory up to so many slots (80 KB: two CTAs an
                                            // SM), else they are made again in every pass
constexpr int kCandidates = 256;
constexpr int kMaxCluster = 8;
constexpr int kMovesHere = 64;  // at most so many moves a head: by the selecting CTAs
constexpr int kMoveThreads = 256;
static_assert(kCandidates * 2 == kThreads, "two threads rank a candidate");

// Larger key = kept earlier.  Slots of the recent window come before every
// number, NaN after every number, and -0 equals +0.
__device__ __forceinline__ uint32_t evict_key(float w, bool recent) {
    const uint32_t b = __float_as_uint(w + 0.0f);
    const uint32_t k = b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
    return recent ? 0xFFFFFFFFu : isnan(w) ? 0u : k;
}

// A slot and the row of the K and V pools that holds it: (page * kv_heads + head) * 64 + slot % 64.
struct Lists {
    int32_t* bad;     // [rows]: the sequence has a bad length or page and stays as it is
    int32_t* count;   // [rows * kv_heads]: moves
    int2 *dst, *src;  // [rows * kv_heads][cap]: holes and movers
    int cap;
};

// Histogram digits: 11 bits for one CTA; 8 in a cluster, where every CTA reads every
// peer's histogram (at 11 bits that alone took 2 us a pass with 8 CTAs).
template <int C>
struct Digits {
    static constexpr int kBits = C == 1 ? 11 : 8;
    static constexpr int kBins = 1 << kBits;
    static constexpr int kPer = C == 1 ? 4 : 1;  // bins a thread
    // The first pass's bins: 32 (8) an octave for weights of 2^-44 .. 2^20 (2^-20 .. 2^12),
    // that is the keys' bits from kShift up, less kBase; the first and the last bin take what
    // lies outside.  (By the leading bits alone, a quarter of an octave or two octaves a bin,
    // more candidates were left to rank: 32 of up to 8000 slots took 64.3 us for 62.2.)
    static constexpr int kShift = C == 1 ? 18 : 20;
    static constexpr int kBase = C == 1 ? (256 + 127 - 44) << 5 : (256 + 127 - 20) << 3;
};

struct Smem {
    int hist[2][2048];  // alternately: one is cleared while peers may still read the other
    uint64_t mine[kCandidates], all[kCandidates];
    int2 dst[kMovesHere], src[kMovesHere];
    int n_mine;
    int warp_sum[kWarps];
    int warp_holes[kWarps], warp_movers[kWarps];
    int holes, movers, ties;  // of this CTA's piece
    int digit, need, count;   // the bin that holds the threshold
    uint32_t key;             // kept: a larger key, or this key and a slot up to
    int slot;                 // this one
    uint32_t words[];         // bitmap of the piece's kept slots, then their keys
};

// Moves of the lists' entries [first, first + 16) below n by 16 lanes: a lane looks up one
// entry (and moves its weight and position), all of them move its K and V, 16 bytes each
// a lane, four slots in flight.
__device__ __forceinline__ void move_slots(const CacheEvictArgs& a, const int2* dst, const int2* src, size_t at, int first,
                                           int n) {
    const CacheView& c = a.c;
    float* wo = a.weights_out ? a.weights_out : c.weights;
    int32_t* po = a.positions_out ? a.positions_out : c.positions;
    const int sub = threadIdx.x & 15;
    const unsigned lanes = 0xFFFFu << (threadIdx.x & 16);
    const uint4 *kp = reinterpret_cast<const uint4*>(c.k) + sub, *vp = reinterpret_cast<const uint4*>(c.v) + sub;
    const bool in = first + sub < n;
    const int2 d = in ? dst[first + sub] : make_int2(0, 0), s = in ? src[first + sub] : make_int2(0, 0);
    const float w = in ? c.weights[at + s.x] : 0.f;
    const int32_t p = in ? c.positions[at + s.x] : 0;
    constexpr int U = 4;
#pragma unroll
    for (int i = 0; i < 16; i += U) {
        if (first + i >= n) break;
        uint4 k[U], v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const size_t of = static_cast<size_t>(__shfl_sync(lanes, s.y, i + u, 16)) * 16;
            if (first + i + u < n) k[u] = kp[of], v[u] = vp[of];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const size_t to = static_cast<size_t>(__shfl_sync(lanes, d.y, i + u, 16)) * 16;
            if (first + i + u < n) const_cast<uint4*>(kp)[to] = k[u], const_cast<uint4*>(vp)[to] = v[u];
        }
    }
    if (in) {
        wo[at + d.x] = w;
        po[at + d.x] = p;
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
__global__ void __launch_bounds__(kThreads, 2) cache_evict_kernel(const CacheEvictArgs a, const Lists m, int moves_here,
                                                                  int key_words) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
    const CacheView& c = a.c;
    const int rh = blockIdx.x / C, rank = blockIdx.x % C, row = rh / c.kv_heads, head = rh % c.kv_heads;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_wait();
    pdl_trigger();
    const int len = a.lens[row];
    const int first_recent =
        static_cast<int>(max(static_cast<long long>(a.next_pos[row]) - a.recent, static_cast<long long>(INT_MIN)));
    const int32_t* table = c.tables + row * c.table_stride;
    const size_t at = cache_slot_index(c, row, head);
    const float* w = c.weights + at;
    const int32_t* pos = c.positions + at;
    using D = Digits<C>;
    for (int i = tid; i < D::kBins; i += kThreads) sm.hist[0][i] = 0;
    if (tid == 0) sm.n_mine = 0;

    // the piece: words of 32 slots, a warp a contiguous run of them
    const bool length_ok = len >= 0 && len <= c.max_len, shrinks = length_ok && len > a.keep;
    const int words = length_ok ? (len + 31) / 32 : 0;
    const int word0 = words / C * rank + words % C * rank / C;
    const int nw = words / C * (rank + 1) + words % C * (rank + 1) / C - word0;
    const int wa = nw * warp / kWarps, wb = nw * (warp + 1) / kWarps;
    uint32_t* kept = sm.words;
    uint32_t* keys = key_words ? sm.words + key_words : nullptr;
    auto slot_of = [&](int i) { return (word0 + i) * 32 + lane; };  // lane's slot of word i of the piece
    // f(word of the piece, slot, key) for the warp's words, by the whole warp
    auto each_word = [&](auto&& f) {
#pragma unroll 4
        for (int i = wa; i < wb; ++i) {
            const int s = slot_of(i);
            f(i, s, keys ? keys[i * 32 + lane] : s < len ? evict_key(w[s], pos[s] >= first_recent) : 0u);
        }
    };
    // four words' weights and positions, ahead of the page check
    constexpr int U = 4;
    float x[U];
    int32_t p[U];
    auto load_words = [&](int i) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = slot_of(i + u);
            const bool in = i + u < wb && s < len;
            x[u] = in ? w[s] : 0.f;
            p[u] = in ? pos[s] : 0;
        }
    };
    load_words(wa);
    uint32_t bad = length_ok ? DEV_OK : DEV_BAD_LENGTH;
    if (shrinks)
        for (int i = tid; i < (len + kCachePage - 1) / kCachePage; i += kThreads)
            if (table[i] < 0 || table[i] >= c.num_pages) bad = DEV_BAD_PAGE;
    const bool stays = __syncthreads_or(bad) != 0;
    if (bad && rank == 0) record_error(c.err, bad);

    // Lengths are read by every CTA of a sequence, and lens_out may be the same array: the
    // last CTA of the grid to count itself, when all have read theirs, writes it (at its
    // end).  Counted where no barrier waits for it (here it would be 750 cycles of the next
    // one), and the count looked at in the end.
    if (tid == kThreads - 1 && head == 0 && rank == 0) m.bad[row] = stays;
    uint32_t before_me = 0;
    auto arrive = [&]() {
        if (tid == kThreads - 1)
            asm volatile("atom.release.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before_me) : "l"(c.arrived) : "memory");
    };
    if (!moves_here) arrive();
    auto finish = [&]() {
        const bool last = tid == kThreads - 1 && before_me == gridDim.x - 1;
        if (last) {
            __threadfence();
            *c.arrived = 0;
        }
        if (!__syncthreads_or(last)) return;
        for (int r = tid; r < c.rows; r += kThreads) {
            const int n = a.lens[r];
            a.lens_out[r] = __ldcg(m.bad + r) ? n : min(n, a.keep);
        }
    };
    if (stays || !shrinks) {
        if (moves_here) arrive();
        if (tid == 0 && rank == 0) m.count[rh] = 0;
        if (!stays && a.weights_out)
            for (int i = wa; i < wb; i += U) {
                if (i > wa) load_words(i);
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (i + u < wb && slot_of(i + u) < len) {
                        a.weights_out[at + slot_of(i + u)] = x[u];
                        a.positions_out[at + slot_of(i + u)] = p[u];
                    }
            }
        finish();
        return;
    }

    // ---- the threshold: the keep-th largest key, and among equals the last slot kept
    uint32_t prefix = 0;  // the keys' bits above the shift
    int need = a.keep, count = len;
    bool found = false;
    for (int pass = 0, shift = D::kShift, bits = D::kBits; !found && bits > 0; ++pass) {
        int* hist = sm.hist[pass & 1];
        if (pass > 0) {
            for (int i = tid; i < D::kBins; i += kThreads) hist[i] = 0;
            __syncthreads();
        }
        auto first_bin = [](uint32_t k) {
            return min(max(static_cast<int>(k >> D::kShift) - D::kBase, 0), D::kBins - 1);
        };
        auto tally = [&](int s, uint32_t k) {
            const uint32_t top = k >> shift;
            if (pass == 0) {
                if (s < len) atomicAdd(&hist[first_bin(k)], 1);
            } else if (s < len && top >> bits == prefix) {
                atomicAdd(&hist[top & ((1u << bits) - 1)], 1);
            }
        };
        if (pass > 0) {
            each_word([&](int, int s, uint32_t k) { tally(s, k); });
        } else {
            // the first pass makes the keys, and copies the slots before keep where the kept ones go to
            // other arrays (the holes among them are filled by the moves)
            for (int i = wa; i < wb; i += U) {
                if (i > wa) load_words(i);
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (i + u < wb) {
                        const int s = slot_of(i + u);
                        const uint32_t k = evict_key(x[u], p[u] >= first_recent);
                        if (keys) keys[(i + u) * 32 + lane] = k;
                        tally(s, k);
                        if (a.weights_out && s < a.keep) a.weights_out[at + s] = x[u], a.positions_out[at + s] = p[u];
                    }
            }
        }
        cluster_sync<C>();
        // thread t has the kPer bins from kBins - 1 - kPer t downwards
        int four[4] = {0, 0, 0, 0};
        if (tid < D::kBins / D::kPer) {
            if constexpr (C == 1) {
                const int4 h = reinterpret_cast<const int4*>(hist)[D::kBins / 4 - 1 - tid];
                four[0] = h.w, four[1] = h.z, four[2] = h.y, four[3] = h.x;
            } else {
                int h[C];
#pragma unroll
                for (int r = 0; r < C; ++r) h[r] = peer(hist, r)[D::kBins - 1 - tid];
#pragma unroll
                for (int r = 0; r < C; ++r) four[0] += h[r];
            }
        }
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
        for (int i = 0; i < D::kPer; ++i) {
            if (above < need && need <= above + four[i])
                sm.digit = D::kBins - 1 - D::kPer * tid - i, sm.need = need - above, sm.count = four[i];
            above += four[i];
        }
        __syncthreads();
        const int digit = sm.digit;
        prefix = pass == 0 ? static_cast<uint32_t>(D::kBase + digit) : (prefix << bits) | static_cast<uint32_t>(digit);
        const int before = need;
        need = sm.need;
        count = sm.count;
        if (count == need) {  // the whole bin is kept
            if (tid == 0) sm.key = prefix << shift, sm.slot = INT_MAX;
            found = true;
        } else if (count <= kCandidates) {
            // few candidates: the one with need - 1 larger ones (the lower slot is the larger) is the last kept
            each_word([&](int, int s, uint32_t k) {
                if (s < len && (pass == 0 ? first_bin(k) == digit : k >> shift == prefix))
                    sm.mine[atomicAdd(&sm.n_mine, 1)] = (static_cast<uint64_t>(k) << 32) | static_cast<uint32_t>(~s);
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
            const int i = tid >> 1;  // two threads a candidate
            if (i < count) {
                const uint64_t k = from[i];
                int larger = 0;
#pragma unroll 8
                for (int j = tid & 1; j < count; j += 2) larger += from[j] > k;
                larger += __shfl_xor_sync(0x3u << (lane & ~1), larger, 1);
                if (larger == need - 1 && (tid & 1) == 0)
                    sm.key = static_cast<uint32_t>(k >> 32), sm.slot = static_cast<int>(~static_cast<uint32_t>(k));
            }
            found = true;
        } else if (pass == 0 && (digit == 0 || digit == D::kBins - 1)) {
            // many outside of the first pass's bins: all over by the leading bits
            prefix = 0;
            need = before;
            shift = 32;
        }
        // the next digit; none is left when the bin is one key
        bits = min(D::kBits, shift);
        shift -= bits;
    }
    if (!found) {
        // more than 256 slots of one key, of which the first `need` are kept: count them by warp
        int ties = 0;
        each_word([&](int, int s, uint32_t k) { ties += __popc(__ballot_sync(0xffffffffu, s < len && k == prefix)); });
        if (lane == 0) sm.warp_sum[warp] = ties;
        __syncthreads();
        const int theirs = lane < kWarps ? sm.warp_sum[lane] : 0;
        int before = __reduce_add_sync(0xffffffffu, lane < warp ? theirs : 0);
        if constexpr (C > 1) {
            const int piece = __reduce_add_sync(0xffffffffu, theirs);
            if (tid == 0) sm.ties = piece;
            cluster_sync<C>();
#pragma unroll
            for (int r = 0; r < C; ++r) {
                const int n = *peer(&sm.ties, r);
                if (r < rank) before += n;
            }
        }
        if (before < need && need <= before + ties) {
            // the need-th is in this warp
            each_word([&](int, int s, uint32_t k) {
                const bool tie = s < len && k == prefix;
                const uint32_t mask = __ballot_sync(0xffffffffu, tie);
                if (tie && before + __popc(mask & ((2u << lane) - 1)) == need)
                    for (int r = 0; r < C; ++r) {
                        Smem* to = C == 1 ? &sm : const_cast<Smem*>(peer(&sm, r));
                        to->key = prefix, to->slot = s;
                    }
                before += __popc(mask);
            });
        }
        if (C > 1) cluster_sync<C>();
    }
    __syncthreads();
    const uint32_t last_key = sm.key;
    const int last_slot = sm.slot;

    // ---- the kept slots' bitmap
    // bit i of the mask: slot 32 * word + i is below keep
    auto below = [&](int word) {
        const int n = a.keep - word * 32;
        return n >= 32 ? 0xFFFFFFFFu : n <= 0 ? 0u : (1u << n) - 1;
    };
    each_word([&](int i, int s, uint32_t k) {
        const bool keep = s < len && (k > last_key || (k == last_key && s <= last_slot));
        const uint32_t mask = __ballot_sync(0xffffffffu, keep);
        if (lane == 0) kept[i] = mask;
    });
    __syncwarp();
    int my_holes = 0, my_movers = 0;
    for (int i = wa + lane; i < wb; i += 32) {
        const uint32_t mask = kept[i], low = below(word0 + i);
        my_holes += __popc(~mask & low);
        my_movers += __popc(mask & ~low);
    }
    my_holes = __reduce_add_sync(0xffffffffu, my_holes);
    my_movers = __reduce_add_sync(0xffffffffu, my_movers);
    if (lane == 0) sm.warp_holes[warp] = my_holes, sm.warp_movers[warp] = my_movers;
    __syncthreads();
    // lists in order: the pieces before this one, the warps before this one
    my_holes = lane < kWarps ? sm.warp_holes[lane] : 0, my_movers = lane < kWarps ? sm.warp_movers[lane] : 0;
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
#pragma unroll 4
    for (int i = wa; i < wb; ++i) {
        const uint32_t mask = kept[i], low = below(word0 + i), h = ~mask & low, v = mask & ~low;
        const int s = slot_of(i);
        if (h >> lane & 1) dst[hole + __popc(h & lower)] = place_of(s);
        if (v >> lane & 1) src[mover + __popc(v & lower)] = place_of(s);
        hole += __popc(h);
        mover += __popc(v);
    }
    if (moves_here) {
        cluster_sync<C>();
        arrive();  // its warp has no moves, or the last ones
        // few: four moves at a time to every 16 lanes of the cluster
        for (int i = (rank * (kThreads / 16) + (tid >> 4)) * 4; i < n; i += C * kThreads / 4)
            move_slots(a, dst, src, at, i, min(n, i + 4));
    } else {
        if (tid == 0 && rank == 0) m.count[rh] = n;
        if (C > 1) cluster_sync<C>();  // peers may still read this CTA's shared memory
    }
    finish();
}

// `each` moves (4 or 16) to every 16 lanes.
__global__ void __launch_bounds__(kMoveThreads, 4)
    cache_evict_move_kernel(const CacheEvictArgs a, const Lists m, int chunks, int each) {
    const int rh = blockIdx.x / chunks, first = (blockIdx.x % chunks * (kMoveThreads / 16) + (threadIdx.x >> 4)) * each;
    pdl_wait();
    pdl_trigger();
    const int n = min(m.count[rh], first + each);
    const size_t list = static_cast<size_t>(rh) * m.cap;
    if (first < n) move_slots(a, m.dst + list, m.src + list, static_cast<size_t>(rh) * a.c.slot_stride, first, n);
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
    // the largest piece's bitmap, and its keys where they fit
    const int piece = c.max_len / 32 / C + 2, key_words = piece * 32 <= kKeysHere ? piece : 0;
    const size_t smem = sizeof(Smem) + static_cast<size_t>(key_words ? piece * 33 : piece) * 4;
    static std::atomic<uint64_t> configured{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (!(configured.load() & bit)) {
        e = cudaFuncSetAttribute(cache_evict_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 static_cast<int>(sizeof(Smem) + ((1 << 20) / 32 + 2) * 4));
        if (e != cudaSuccess) return e;
        configured.fetch_or(bit);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(c.rows) * c.kv_heads * C);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // as launch_after
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = C;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = C > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, cache_evict_kernel<C>, a, m, moves_here, key_words);
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
    // 16 moves to 16 lanes where that still gives every SM its threads, else 4
    const int each = rh * m.cap >= static_cast<size_t>(sms) * (2048 / 16) * 16 ? 16 : 4;
    const int chunk = kMoveThreads / 16 * each, chunks = (m.cap + chunk - 1) / chunk;
    return launch_after(cache_evict_move_kernel, dim3(static_cast<unsigned>(rh) * chunks), kMoveThreads, 0, s, a, m, chunks,
                        each);
}

}  // namespace q3
