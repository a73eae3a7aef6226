// cache.cu -- the bounded paged KV cache: its handle and C ABI, and the append
// of new tokens.
//
// The library's own decode path ties a token's cache slot to its position, so a
// sequence ends when its pages are full.  Here the two are separate: a token's
// query and key are rotated to its position, its K/V go to any slot, and the
// slots a sequence attends to can be cut to a budget (cache_evict.cu) by the
// attention they have received (cache_attention.cu).
#include <algorithm>
#include <atomic>
#include <climits>
#include <new>

#include "cache.cuh"
#include "host_util.hpp"

struct q3_cache {
    q3::CacheView view{};
    int device = 0;
    int sms = 148;
    q3::CacheMaps maps{};  // of the pools; mapped: they have been made
    bool mapped = false;
};

namespace q3 {
namespace {

constexpr int kAppendWarps = 16;    // most warps a row (few rows); consumer warps (many)
constexpr int kAppendStages = 16;   // most rows in flight a CTA
constexpr int kAppendRing = 200 * 1024;

// Two fp32 values in a 64-bit register, and the packed arithmetic on them (each
// element rounded as the scalar operation rounds it).
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pair(float lo, float hi) {
    f32x2 v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
__device__ __forceinline__ f32x2 pair(uint32_t bf) { return pair(bf_lo(bf), bf_hi(bf)); }  // of two BF16
__device__ __forceinline__ f32x2 mul2(f32x2 x, f32x2 y) {
    f32x2 v;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(x), "l"(y));
    return v;
}
__device__ __forceinline__ f32x2 fma2(f32x2 x, f32x2 y, f32x2 z) {
    f32x2 v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(x), "l"(y), "l"(z));
    return v;
}
__device__ __forceinline__ float2 unpair(f32x2 v) {
    float2 x;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x.x), "=f"(x.y) : "l"(v));
    return x;
}
__device__ __forceinline__ uint32_t to_bf2(f32x2 v) {
    const float2 x = unpair(v);
    const __nv_bfloat162 b = __floats2bfloat162_rn(x.x, x.y);
    return *reinterpret_cast<const uint32_t*>(&b);
}

// A unit is four heads of one kind (queries, keys or values), eight lanes each: lane j
// holds dims 8 j .. 8 j + 7 and 64 + 8 j .. of its head, so that both halves of a
// rotation sit in one lane.  RMSNorm and RoPE as qk_norm_rope
// (cuda/kernels/qk_norm_rope.cuh:14-90): fp32 throughout, one rounding; the norm's
// weights are multiplied into the rotation once for all of a row's heads, and the
// arithmetic runs on pairs.
struct Rotation {
    // (a, b), the halves of a pair of dims -> (a (w0 c) - b (w1 s), b (w1 c) + a (w0 s)), times the norm's scale
    f32x2 ac[4], as[4], bc[4], bs[4];
    __device__ __forceinline__ void make(uint4 n0, uint4 n1, const float* cos_row, const float* sin_row, int sub) {
        const uint32_t w0[4] = {n0.x, n0.y, n0.z, n0.w}, w1[4] = {n1.x, n1.y, n1.z, n1.w};
        float4 c[2], s[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            c[j] = reinterpret_cast<const float4*>(cos_row)[2 * sub + j];
            s[j] = reinterpret_cast<const float4*>(sin_row)[2 * sub + j];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const f32x2 c2 = j & 1 ? pair(c[j / 2].z, c[j / 2].w) : pair(c[j / 2].x, c[j / 2].y);
            const f32x2 s2 = j & 1 ? pair(s[j / 2].z, s[j / 2].w) : pair(s[j / 2].x, s[j / 2].y);
            ac[j] = mul2(pair(w0[j]), c2);
            as[j] = mul2(pair(w0[j]), s2);
            bc[j] = mul2(pair(w1[j]), c2);
            bs[j] = mul2(pair(w1[j]), mul2(s2, pair(-1.f, -1.f)));
        }
    }
    // one head by its eight lanes, four heads a warp
    __device__ __forceinline__ void apply(uint4& x, uint4& y, float eps) const {
        const uint32_t w0[4] = {x.x, x.y, x.z, x.w}, w1[4] = {y.x, y.y, y.z, y.w};
        f32x2 s2 = pair(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < 4; ++j) s2 = fma2(pair(w1[j]), pair(w1[j]), fma2(pair(w0[j]), pair(w0[j]), s2));
        float ss = unpair(s2).x + unpair(s2).y;
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float scale = 1.0f / sqrtf(ss / 128.0f + eps);
        const f32x2 scale2 = pair(scale, scale);
        uint32_t r0[4], r1[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const f32x2 a2 = pair(w0[j]), b2 = pair(w1[j]);
            r0[j] = to_bf2(mul2(fma2(b2, bs[j], mul2(a2, ac[j])), scale2));
            r1[j] = to_bf2(mul2(fma2(a2, as[j], mul2(b2, bc[j])), scale2));
        }
        x = make_uint4(r0[0], r0[1], r0[2], r0[3]);
        y = make_uint4(r1[0], r1[1], r1[2], r1[3]);
    }
};

// A new token's row, looked up: DEV_OK, or why it is left out.
__device__ __forceinline__ uint32_t append_check(const CacheAppendArgs& a, int slot, int pos, int seq) {
    if (slot < 0 || slot >= a.c.max_len) return DEV_BAD_SLOT;
    if (pos < 0 || pos >= a.max_pos) return DEV_BAD_POSITION;
    if (seq < 0 || seq >= a.c.rows) return DEV_BAD_SEQUENCE;
    return DEV_OK;
}
__device__ __forceinline__ bool append_page_bad(const CacheView& c, int page) { return page < 0 || page >= c.num_pages; }
__device__ __forceinline__ void append_state(const CacheView& c, int seq, int slot, int pos, int lane) {
    if (!c.weights) return;
    for (int h = lane; h < c.kv_heads; h += 32) {
        const size_t at = cache_slot_index(c, seq, h) + slot;
        c.weights[at] = 0.0f;
        c.positions[at] = pos;
    }
}

// Few rows: one CTA a row, its units dealt to the warps, in the order queries, keys,
// values.  Bound: latency (look-ups, then loads, then stores: 2.7 us for one row of
// 32 + 8 + 8 heads inside a graph, 3.5 us for 256).
__global__ void __launch_bounds__(kAppendWarps * 32) cache_append_kernel(const __grid_constant__ CacheAppendArgs a) {
    const CacheView& c = a.c;
    const int i = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane & 7;
    pdl_wait();
    pdl_trigger();
    const int slot = a.slots[i], pos = a.token_pos[i], seq = a.row_seq ? a.row_seq[i] : i;
    if (slot == -1) return;
    uint32_t bad = append_check(a, slot, pos, seq);
    const int page = bad ? 0 : c.tables[seq * c.table_stride + slot / kCachePage];
    if (!bad && append_page_bad(c, page)) bad = DEV_BAD_PAGE;
    if (bad) {
        if (threadIdx.x == 0) record_error(c.err, bad);
        return;
    }
    const int q_units = (a.q_heads + 3) / 4, kv_units = (c.kv_heads + 3) / 4;
    for (int u = warp; u < q_units + 2 * kv_units; u += blockDim.x / 32) {
        const bool is_q = u < q_units, is_k = !is_q && u < q_units + kv_units;
        const int h = 4 * (is_q ? u : is_k ? u - q_units : u - q_units - kv_units) + (lane >> 3);
        const bf16* src = is_q ? a.q + i * a.q_stride : is_k ? a.k + i * a.k_stride : a.v + i * a.v_stride;
        const bool live = h < (is_q ? a.q_heads : c.kv_heads);
        uint4 x = make_uint4(0u, 0u, 0u, 0u), y = x;
        if (live) {
            x = reinterpret_cast<const uint4*>(src + h * kCacheHd)[sub];
            y = reinterpret_cast<const uint4*>(src + h * kCacheHd)[sub + 8];
        }
        if (is_q || is_k) {
            const uint4* norm = reinterpret_cast<const uint4*>(is_q ? a.q_norm : a.k_norm);
            Rotation turn;
            turn.make(norm[sub], norm[sub + 8], a.rope_cos + static_cast<size_t>(pos) * 64,
                      a.rope_sin + static_cast<size_t>(pos) * 64, sub);
            turn.apply(x, y, a.eps);
        }
        if (live) {
            uint4* to = reinterpret_cast<uint4*>(is_q ? a.q_out + i * a.q_out_stride + h * kCacheHd
                                                      : (is_k ? c.k : c.v) + cache_kv_offset(c, page, h, slot));
            to[sub] = x;
            to[sub + 8] = y;
        }
    }
    if (warp == 0) append_state(c, seq, slot, pos, lane);
    // every thread has read slots[i] (lens_out may be the same array)
    __syncthreads();
    if (a.lens_out && threadIdx.x == 0) a.lens_out[i] = slot + 1;
}

// Many rows: a CTA an SM streams its rows (heads, and the position's cosines and sines)
// through a shared-memory ring by bulk copies, so that up to 200 KB an SM are in flight
// whatever the rows' look-ups wait for; 16 warps turn the heads and write them.  Bound:
// HBM: 4001 rows of 64 + 8 + 8 heads take 33.6 us, 75 % of the measured copy rate over
// the bytes in and out; one kernel for both row counts spilled or took 51 to 64 us.
struct AppendSmem {
    int4 row[kAppendStages];  // row (-1: the end), sequence, slot, position
    int page[kAppendStages];
    uint64_t full[kAppendStages], empty[kAppendStages];
};

__global__ void __launch_bounds__(kAppendWarps * 32 + 32, 1)
    cache_append_stream_kernel(const __grid_constant__ CacheAppendArgs a, int stages, int stage_bytes) {
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ AppendSmem sm;
    const CacheView& c = a.c;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane & 7;
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(&sm.full[s], 1);
            mbar_init(&sm.empty[s], kAppendWarps);
        }
        fence_barrier_init();
    }
    pdl_wait();
    pdl_trigger();
    __syncthreads();
    const int q_bytes = a.q_heads * kCacheHd * 2, kv_bytes = c.kv_heads * kCacheHd * 2;

    if (warp == kAppendWarps) {
        // ---- producer: lane j looks up the CTA's row j of every 32
        const uint64_t pol = policy_evict_first();
        int k = 0, s = 0;
        uint32_t round = 0;  // of the ring: stage s has been used `round` times
        bool ok = true;
        auto stage_free = [&]() {
            return round == 0 || mbar_wait(&sm.empty[s], (round - 1) & 1, c.err, DEV_TMA_WAIT_TIMEOUT);
        };
        auto advance = [&]() {
            ++k;
            if (++s == stages) s = 0, ++round;
        };
        const int step = gridDim.x;
        for (int i0 = blockIdx.x; i0 < a.n && ok; i0 += 32 * step) {
            const int i = i0 + lane * step;
            int4 row = make_int4(i, 0, -1, 0);
            int page = 0;
            if (i < a.n) {
                row.z = a.slots[i];
                row.w = a.token_pos[i];
                row.y = a.row_seq ? a.row_seq[i] : i;
                if (row.z != -1) {
                    uint32_t bad = append_check(a, row.z, row.w, row.y);
                    if (!bad) {
                        page = c.tables[row.y * c.table_stride + row.z / kCachePage];
                        if (append_page_bad(c, page)) bad = DEV_BAD_PAGE;
                    }
                    if (bad) {
                        record_error(c.err, bad);
                        row.z = -1;
                    }
                }
            }
            for (int j = 0; j < 32 && ok; ++j) {
                const int4 r = make_int4(__shfl_sync(0xffffffffu, row.x, j), __shfl_sync(0xffffffffu, row.y, j),
                                         __shfl_sync(0xffffffffu, row.z, j), __shfl_sync(0xffffffffu, row.w, j));
                const int pg = __shfl_sync(0xffffffffu, page, j);
                if (r.z < 0) continue;  // left out, or no such row
                if (lane == 0) {
                    ok = stage_free();
                    if (ok) {
                        uint8_t* st = ring + static_cast<size_t>(s) * stage_bytes;
                        sm.row[s] = r;
                        sm.page[s] = pg;
                        mbar_arrive_expect_tx(&sm.full[s], q_bytes + 2 * kv_bytes + 512);
                        bulk_g2s(st, a.q + r.x * a.q_stride, q_bytes, &sm.full[s], pol);
                        bulk_g2s(st + q_bytes, a.k + r.x * a.k_stride, kv_bytes, &sm.full[s], pol);
                        bulk_g2s(st + q_bytes + kv_bytes, a.v + r.x * a.v_stride, kv_bytes, &sm.full[s], pol);
                        st += q_bytes + 2 * kv_bytes;
                        bulk_g2s(st, a.rope_cos + static_cast<size_t>(r.w) * 64, 256, &sm.full[s], pol);
                        bulk_g2s(st + 256, a.rope_sin + static_cast<size_t>(r.w) * 64, 256, &sm.full[s], pol);
                    }
                }
                ok = __shfl_sync(0xffffffffu, ok, 0);
                if (ok) advance();
            }
        }
        if (lane == 0) {
            ok = ok && stage_free();
            if (ok) {
                sm.row[s].x = -1;
                mbar_arrive(&sm.full[s]);
            } else {
                // a wait ran out: leave no copy in flight behind
                for (int i = max(0, k - stages); i < k; ++i)
                    mbar_wait(&sm.full[i % stages], (i / stages) & 1, nullptr, 0);
            }
        }
        return;
    }

    const uint4 qn0 = reinterpret_cast<const uint4*>(a.q_norm)[sub], qn1 = reinterpret_cast<const uint4*>(a.q_norm)[sub + 8];
    const uint4 kn0 = reinterpret_cast<const uint4*>(a.k_norm)[sub], kn1 = reinterpret_cast<const uint4*>(a.k_norm)[sub + 8];
    const int q_units = (a.q_heads + 3) / 4, kv_units = (c.kv_heads + 3) / 4;
    // the rows' units one after the other, dealt to the warps: a warp's first unit of the row at hand
    const int units = q_units + 2 * kv_units, shift = units % kAppendWarps;
    int first = warp;
    for (int s = 0, round = 0;;) {
        if (!mbar_wait(&sm.full[s], round & 1, c.err, DEV_TMA_WAIT_TIMEOUT)) return;
        const int4 r = sm.row[s];
        if (r.x < 0) return;
        const int page = sm.page[s];
        const uint8_t* st = ring + static_cast<size_t>(s) * stage_bytes;
        const float* cos_row = reinterpret_cast<const float*>(st + q_bytes + 2 * kv_bytes);
        for (int u = first; u < units; u += kAppendWarps) {
            const bool is_q = u < q_units, is_k = !is_q && u < q_units + kv_units;
            const int h = 4 * (is_q ? u : is_k ? u - q_units : u - q_units - kv_units) + (lane >> 3);
            const bool live = h < (is_q ? a.q_heads : c.kv_heads);
            const uint4* src = reinterpret_cast<const uint4*>(st + (is_q ? 0 : is_k ? q_bytes : q_bytes + kv_bytes) + h * 256);
            uint4 x = make_uint4(0u, 0u, 0u, 0u), y = x;
            if (live) x = src[sub], y = src[sub + 8];
            if (is_q || is_k) {
                Rotation turn;
                turn.make(is_q ? qn0 : kn0, is_q ? qn1 : kn1, cos_row, cos_row + 64, sub);
                turn.apply(x, y, a.eps);
            }
            if (live) {
                uint4* to = reinterpret_cast<uint4*>(is_q ? a.q_out + r.x * a.q_out_stride + h * kCacheHd
                                                          : (is_k ? c.k : c.v) + cache_kv_offset(c, page, h, r.z));
                to[sub] = x;
                to[sub + 8] = y;
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.empty[s]);
        if (warp == kAppendWarps - 1) {
            append_state(c, r.y, r.z, r.w, lane);
            if (a.lens_out && lane == 0) a.lens_out[r.x] = r.z + 1;
        }
        if (++s == stages) s = 0, ++round;
        first = first < shift ? first + kAppendWarps - shift : first - shift;
    }
}

// The handle's device for the length of a call; the caller's afterwards.
struct DeviceScope {
    int before = -1;
    cudaError_t status;
    explicit DeviceScope(int device) {
        status = cudaGetDevice(&before);
        if (status == cudaSuccess && before != device)
            status = cudaSetDevice(device);
        else
            before = -1;
    }
    // a failure is reported by the call, not left for the next one's cudaGetLastError
    ~DeviceScope() {
        if (status != cudaSuccess) cudaGetLastError();
        if (before >= 0) cudaSetDevice(before);
    }
};

bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

const char* device_error_text(uint32_t code) {
    switch (code) {
        case DEV_TMA_WAIT_TIMEOUT: return "a TMA wait ran out";
        case DEV_BAD_POSITION: return "a token position lies outside the RoPE tables";
        case DEV_BAD_PAGE: return "a page table entry lies outside the pool";
        case DEV_BAD_LENGTH: return "a sequence length is negative or exceeds max_len";
        case DEV_BAD_SLOT: return "a slot is negative or not below max_len";
        case DEV_BAD_SEQUENCE: return "a row names a sequence outside the cache";
        default: return "unknown device error";
    }
}

int launched(cudaError_t e, const char* what) {
    if (e == cudaSuccess) return Q3_OK;
    return fail(Q3_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

}  // namespace

cudaError_t launch_cache_append(const CacheAppendArgs& a, int sms, cudaStream_t s) {
    const int q_units = (a.q_heads + 3) / 4, kv_units = (a.c.kv_heads + 3) / 4;
    const int stage = (a.q_heads + 2 * a.c.kv_heads) * kCacheHd * 2 + 512;
    // The ring takes 3 us more to start and per row about what a CTA a row spends on 24 heads, then runs at HBM's
    // pace.  Ring against CTA a row, us (148 SMs), where it loses: 4096 rows of 4 + 1 + 1 heads 17.9 / 7.6,
    // 1184 of 16 + 8 + 8 9.2 / 6.3, 592 of 32 + 8 + 8 7.2 / 5.9; even: 400 of 64 + 8 + 8 7.1 / 7.1; where it wins:
    // 4096 of 16 + 8 + 8 21.5 / 24.0, 1184 of 64 + 8 + 8 12.8 / 20.3, 4096 of those 34 / 61.
    const long long heads = a.q_heads + 2 * a.c.kv_heads;
    if (a.n * (heads - 24) >= 150ll * sms && 2 * stage <= kAppendRing) {
        const int stages = std::min(kAppendStages, kAppendRing / stage);
        static std::atomic<uint64_t> configured{0};
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        const uint64_t bit = 1ull << (dev & 63);
        if (!(configured.load() & bit)) {
            e = cudaFuncSetAttribute(cache_append_stream_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kAppendRing);
            if (e != cudaSuccess) return e;
            configured.fetch_or(bit);
        }
        return launch_after(cache_append_stream_kernel, dim3(sms), kAppendWarps * 32 + 32,
                            static_cast<size_t>(stages) * stage, s, a, stages, stage);
    }
    const int warps = std::min(q_units + 2 * kv_units, kAppendWarps);
    return launch_after(cache_append_kernel, dim3(a.n), warps * 32, 0, s, a);
}

}  // namespace q3

using namespace q3;

extern "C" {

int q3_cache_create(const q3_cache_desc* d, int device, q3_cache** out) {
    Q3_CHECK(d && out, "q3_cache_create: null argument");
    *out = nullptr;
    Q3_CHECK(d->k_pages_dev && d->v_pages_dev && d->page_tables_dev && d->state_dev, "q3_cache_create: null pointer");
    if (d->head_dim != kCacheHd) return fail(Q3_ERR_UNSUPPORTED, "q3_cache_create: head_dim must be 128");
    if (d->page_size != kCachePage) return fail(Q3_ERR_UNSUPPORTED, "q3_cache_create: page_size must be 64");
    Q3_CHECK(d->kv_heads >= 1 && d->kv_heads <= 1024, "q3_cache_create: kv_heads must be 1 .. 1024");
    Q3_CHECK(d->rows >= 1 && d->rows <= 4096, "q3_cache_create: rows must be 1 .. 4096");
    Q3_CHECK(d->max_len >= 1 && d->max_len <= (1u << 20), "q3_cache_create: max_len must be 1 .. 2^20");
    // tiles of 64 slots are numbered in 32 bits, all sequences' heads together
    Q3_CHECK(d->rows * d->kv_heads * ((d->max_len + kCachePage - 1) / kCachePage) <= (1u << 30),
             "q3_cache_create: rows * kv_heads * ceil(max_len / 64) must be at most 2^30");
    // rows of the pools are addressed by 32-bit tensor-map coordinates
    Q3_CHECK(d->num_pages >= 1 && d->num_pages <= INT_MAX / (kCachePage * d->kv_heads),
             "q3_cache_create: num_pages * kv_heads * 64 must be below 2^31");
    Q3_CHECK(d->table_stride >= (d->max_len + kCachePage - 1) / kCachePage && d->table_stride <= INT_MAX,
             "q3_cache_create: table_stride must cover ceil(max_len / 64) pages");
    Q3_CHECK((d->weights_dev == nullptr) == (d->positions_dev == nullptr),
             "q3_cache_create: weights and positions go together");
    Q3_CHECK(!d->weights_dev || (d->slot_stride >= d->max_len && d->slot_stride <= INT_MAX),
             "q3_cache_create: slot_stride must be at least max_len");
    Q3_CHECK(aligned(d->k_pages_dev, 16) && aligned(d->v_pages_dev, 16), "q3_cache_create: 16-byte aligned pages required");
    Q3_CHECK(aligned(d->page_tables_dev, 4) && aligned(d->weights_dev, 4) && aligned(d->positions_dev, 4) &&
                 aligned(d->state_dev, 4),
             "q3_cache_create: 4-byte aligned tables, weights, positions and state required");
    int devices = 0;
    if (cudaGetDeviceCount(&devices) != cudaSuccess) devices = 0;
    cudaGetLastError();  // without a GPU the descriptor can be checked all the same
    Q3_CHECK(device >= 0 && (devices == 0 || device < devices), "q3_cache_create: no such device");
    auto* c = new (std::nothrow) q3_cache();
    if (!c) return fail(Q3_ERR_OOM, "q3_cache_create: host allocation failed");
    c->device = device;
    c->sms = num_sms(device);
    if (devices == 0) cudaGetLastError();
    CacheView& v = c->view;
    v.k = reinterpret_cast<bf16*>(d->k_pages_dev);
    v.v = reinterpret_cast<bf16*>(d->v_pages_dev);
    v.num_pages = static_cast<int>(d->num_pages);
    v.tables = d->page_tables_dev;
    v.table_stride = static_cast<long long>(d->table_stride);
    v.weights = d->weights_dev;
    v.positions = d->positions_dev;
    v.slot_stride = static_cast<long long>(d->slot_stride);
    v.rows = static_cast<int>(d->rows);
    v.max_len = static_cast<int>(d->max_len);
    v.kv_heads = static_cast<int>(d->kv_heads);
    v.err = d->state_dev;
    v.next_chunk = d->state_dev + 1;
    v.arrived = d->state_dev + 2;
    c->mapped = cache_maps(v, &c->maps);
    *out = c;
    return Q3_OK;
}

int q3_cache_destroy(q3_cache* c) {
    delete c;
    return Q3_OK;
}

int q3_cache_sync(q3_cache* c, void* stream) {
    Q3_CHECK(c, "q3_cache_sync: null argument");
    DeviceScope scope(c->device);
    Q3_CUDA(scope.status);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    uint32_t code = 0;
    Q3_CUDA(cudaMemcpyAsync(&code, c->view.err, 4, cudaMemcpyDeviceToHost, s));
    Q3_CUDA(cudaStreamSynchronize(s));
    if (code == DEV_OK) return Q3_OK;
    // the work counters with it: a kernel that gave up may have left them anywhere
    Q3_CUDA(cudaMemsetAsync(c->view.err, 0, Q3_CACHE_STATE_WORDS * 4, s));
    Q3_CUDA(cudaStreamSynchronize(s));
    return fail(Q3_ERR_DEVICE, std::string("q3_cache: ") + device_error_text(code));
}

int q3_cache_append(q3_cache* c, const uint16_t* q, size_t q_stride, const uint16_t* k, size_t k_stride,
                    const uint16_t* v, size_t v_stride, const uint16_t* q_norm, const uint16_t* k_norm,
                    const float* cos_t, const float* sin_t, size_t max_pos, const int32_t* token_pos,
                    const int32_t* slots, const int32_t* row_seq, size_t n, size_t q_heads, uint16_t* q_out,
                    size_t q_out_stride, int32_t* lens_out, float eps, void* stream) {
    Q3_CHECK(c, "q3_cache_append: null cache");
    if (n == 0) return Q3_OK;
    Q3_CHECK(q && k && v && q_norm && k_norm && cos_t && sin_t && token_pos && slots && q_out,
             "q3_cache_append: null pointer");
    const CacheView& w = c->view;
    Q3_CHECK(n <= (1u << 24), "q3_cache_append: too many rows");
    Q3_CHECK(row_seq || n <= static_cast<size_t>(w.rows), "q3_cache_append: more rows than sequences");
    Q3_CHECK(q_heads >= 1 && q_heads <= 65536, "q3_cache_append: q_heads must be 1 .. 65536");
    Q3_CHECK(max_pos >= 1 && max_pos <= INT_MAX, "q3_cache_append: max_pos");
    const size_t qw = q_heads * kCacheHd, kw = static_cast<size_t>(w.kv_heads) * kCacheHd;
    Q3_CHECK(n == 1 || (q_stride >= qw && k_stride >= kw && v_stride >= kw && q_out_stride >= qw),
             "q3_cache_append: a row stride is shorter than the row");
    Q3_CHECK((q_stride | k_stride | v_stride | q_out_stride) % 8 == 0,
             "q3_cache_append: row strides must be multiples of 8");
    Q3_CHECK(q_stride <= INT_MAX && k_stride <= INT_MAX && v_stride <= INT_MAX && q_out_stride <= INT_MAX,
             "q3_cache_append: row stride too large");
    Q3_CHECK(aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(q_out, 16) && aligned(q_norm, 16) &&
                 aligned(k_norm, 16) && aligned(cos_t, 16) && aligned(sin_t, 16),
             "q3_cache_append: 16-byte alignment required");
    DeviceScope scope(c->device);
    Q3_CUDA(scope.status);
    CacheAppendArgs a{};
    a.c = w;
    a.q = reinterpret_cast<const bf16*>(q);
    a.k = reinterpret_cast<const bf16*>(k);
    a.v = reinterpret_cast<const bf16*>(v);
    a.q_stride = static_cast<long long>(q_stride);
    a.k_stride = static_cast<long long>(k_stride);
    a.v_stride = static_cast<long long>(v_stride);
    a.q_norm = reinterpret_cast<const bf16*>(q_norm);
    a.k_norm = reinterpret_cast<const bf16*>(k_norm);
    a.rope_cos = cos_t;
    a.rope_sin = sin_t;
    a.max_pos = static_cast<int>(max_pos);
    a.token_pos = token_pos;
    a.slots = slots;
    a.row_seq = row_seq;
    a.n = static_cast<int>(n);
    a.q_heads = static_cast<int>(q_heads);
    a.q_out = reinterpret_cast<bf16*>(q_out);
    a.q_out_stride = static_cast<long long>(q_out_stride);
    a.lens_out = lens_out;
    a.eps = eps;
    return launched(launch_cache_append(a, c->sms, static_cast<cudaStream_t>(stream)), "q3_cache_append");
}

size_t q3_cache_attention_workspace_bytes(const q3_cache* c, size_t q_heads, int accumulate) {
    if (!c || q_heads == 0 || q_heads % c->view.kv_heads || q_heads / c->view.kv_heads > 16) return 0;
    return cache_attention_ws_bytes(c->view, static_cast<int>(q_heads), accumulate, c->sms);
}

int q3_cache_attention(q3_cache* c, const uint16_t* q, size_t q_stride, const int32_t* lens, uint16_t* out,
                       size_t out_stride, size_t q_heads, int accumulate, void* ws, size_t ws_bytes, void* stream) {
    Q3_CHECK(c, "q3_cache_attention: null cache");
    Q3_CHECK(q && lens && out, "q3_cache_attention: null pointer");
    const CacheView& w = c->view;
    Q3_CHECK(q_heads >= 1 && q_heads % w.kv_heads == 0, "q3_cache_attention: q_heads must be a multiple of kv_heads");
    if (q_heads / w.kv_heads > 16)
        return fail(Q3_ERR_UNSUPPORTED, "q3_cache_attention: at most 16 query heads per kv head");
    const size_t qw = q_heads * kCacheHd;
    Q3_CHECK(w.rows == 1 || (q_stride >= qw && out_stride >= qw),
             "q3_cache_attention: a row stride is shorter than the row");
    Q3_CHECK(q_stride % 8 == 0 && out_stride % 8 == 0, "q3_cache_attention: row strides must be multiples of 8");
    Q3_CHECK(q_stride <= INT_MAX && out_stride <= INT_MAX, "q3_cache_attention: row stride too large");
    Q3_CHECK(aligned(q, 16) && aligned(out, 16), "q3_cache_attention: 16-byte alignment required");
    Q3_CHECK(!accumulate || w.weights, "q3_cache_attention: the cache has no weights to accumulate into");
    const size_t need = cache_attention_ws_bytes(w, static_cast<int>(q_heads), accumulate, c->sms);
    Q3_CHECK(ws && ws_bytes >= need && aligned(ws, 16),
             "q3_cache_attention: workspace missing, too small or not 16-byte aligned");
    DeviceScope scope(c->device);
    Q3_CUDA(scope.status);
    if (!c->mapped) return fail(Q3_ERR_CUDA, "q3_cache_attention: no tensor maps of the pages (no CUDA driver?)");
    CacheAttnArgs a{};
    a.c = w;
    a.q = reinterpret_cast<const bf16*>(q);
    a.q_stride = static_cast<long long>(q_stride);
    a.lens = lens;
    a.out = reinterpret_cast<bf16*>(out);
    a.out_stride = static_cast<long long>(out_stride);
    a.q_heads = static_cast<int>(q_heads);
    a.accumulate = accumulate != 0;
    a.ws = ws;
    return launched(launch_cache_attention(a, c->maps, c->sms, static_cast<cudaStream_t>(stream)), "q3_cache_attention");
}

size_t q3_cache_evict_workspace_bytes(const q3_cache* c, size_t keep) {
    if (!c || keep == 0) return 0;
    return cache_evict_ws_bytes(c->view, static_cast<int>(keep < (1u << 20) ? keep : (1u << 20)));
}

int q3_cache_evict(q3_cache* c, const int32_t* lens, const int32_t* next_pos, size_t keep, size_t recent,
                   float* weights_out, int32_t* positions_out, int32_t* lens_out, void* ws, size_t ws_bytes,
                   void* stream) {
    Q3_CHECK(c, "q3_cache_evict: null cache");
    Q3_CHECK(lens && next_pos && lens_out, "q3_cache_evict: null pointer");
    const CacheView& w = c->view;
    Q3_CHECK(w.weights, "q3_cache_evict: the cache has no accumulated weights");
    Q3_CHECK(keep >= 1, "q3_cache_evict: keep must be at least 1");
    if (weights_out == w.weights) weights_out = nullptr;
    if (positions_out == w.positions) positions_out = nullptr;
    Q3_CHECK((weights_out == nullptr) == (positions_out == nullptr),
             "q3_cache_evict: weights_out and positions_out go together");
    Q3_CHECK(recent <= INT_MAX, "q3_cache_evict: recent too large");
    Q3_CHECK(aligned(weights_out, 4) && aligned(positions_out, 4), "q3_cache_evict: 4-byte alignment required");
    const int kept = static_cast<int>(keep < (1u << 20) ? keep : (1u << 20));
    const size_t need = cache_evict_ws_bytes(w, kept);
    Q3_CHECK(ws && ws_bytes >= need && aligned(ws, 16),
             "q3_cache_evict: workspace missing, too small or not 16-byte aligned");
    DeviceScope scope(c->device);
    Q3_CUDA(scope.status);
    CacheEvictArgs a{};
    a.c = w;
    a.lens = lens;
    a.next_pos = next_pos;
    a.keep = kept;
    a.recent = static_cast<int>(recent);
    a.weights_out = weights_out;
    a.positions_out = positions_out;
    a.lens_out = lens_out;
    a.ws = ws;
    return launched(launch_cache_evict(a, c->sms, static_cast<cudaStream_t>(stream)), "q3_cache_evict");
}

}  // extern "C"
