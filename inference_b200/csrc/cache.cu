// cache.cu -- the bounded paged KV cache: its handle and C ABI, and the append
// of new tokens.
//
// The library's own decode path ties a token's cache slot to its position, so a
// sequence ends when its pages are full.  Here the two are separate: a token's
// query and key are rotated to its position, its K/V go to any slot, and the
// slots a sequence attends to can be cut to a budget (cache_evict.cu) by the
// attention they have received (cache_attention.cu).
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

constexpr int kAppendWarps = 8;

// One CTA per new token, one head per warp and turn.  A head is a 256-byte row:
// lane l holds dims l, l + 32, l + 64, l + 96, so that a rotation's two halves
// (i and i + 64) sit in one lane; RMSNorm and RoPE as qk_norm_rope
// (cuda/kernels/qk_norm_rope.cuh:14-90): fp32 throughout, one rounding.
__global__ void __launch_bounds__(kAppendWarps * 32) cache_append_kernel(const CacheAppendArgs a) {
    const CacheView& c = a.c;
    const int i = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    pdl_trigger();
    const int slot = a.slots[i];
    const int pos = a.token_pos[i];
    const int seq = a.row_seq ? a.row_seq[i] : i;
    if (slot == -1) return;
    uint32_t bad = 0;
    int page = 0;
    if (slot < 0 || slot >= c.max_len)
        bad = DEV_BAD_SLOT;
    else if (pos < 0 || pos >= a.max_pos)
        bad = DEV_BAD_POSITION;
    else if (seq < 0 || seq >= c.rows)
        bad = DEV_BAD_SEQUENCE;
    else {
        page = c.tables[seq * c.table_stride + slot / kCachePage];
        if (page < 0 || page >= c.num_pages) bad = DEV_BAD_PAGE;
    }
    if (bad) {
        if (threadIdx.x == 0) record_error(c.err, bad);
        return;
    }
    float cs[2], sn[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        cs[j] = a.rope_cos[static_cast<size_t>(pos) * 64 + lane + 32 * j];
        sn[j] = a.rope_sin[static_cast<size_t>(pos) * 64 + lane + 32 * j];
    }
    for (int h = warp; h < a.q_heads + c.kv_heads; h += kAppendWarps) {
        const bool is_q = h < a.q_heads;
        const int kh = h - a.q_heads;
        const bf16* src = is_q ? a.q + i * a.q_stride + h * kCacheHd : a.k + i * a.k_stride + kh * kCacheHd;
        const bf16* w = is_q ? a.q_norm : a.k_norm;
        float x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = bf2f(src[lane + 32 * j]);
        const float ss = warp_sum(x[0] * x[0] + x[1] * x[1] + x[2] * x[2] + x[3] * x[3]);
        const float scale = 1.0f / sqrtf(ss / 128.0f + a.eps);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = x[j] * bf2f(w[lane + 32 * j]) * scale;
        bf16* dst = is_q ? a.q_out + i * a.q_out_stride + h * kCacheHd : c.k + cache_kv_offset(c, page, kh, slot);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            dst[lane + 32 * j] = f2bf(x[j] * cs[j] - x[j + 2] * sn[j]);
            dst[lane + 32 * j + 64] = f2bf(x[j + 2] * cs[j] + x[j] * sn[j]);
        }
        if (!is_q) {
            const uint2* from = reinterpret_cast<const uint2*>(a.v + i * a.v_stride + kh * kCacheHd);
            reinterpret_cast<uint2*>(c.v + cache_kv_offset(c, page, kh, slot))[lane] = from[lane];
            if (c.weights && lane == 0) {
                const size_t at = cache_slot_index(c, seq, kh) + slot;
                c.weights[at] = 0.0f;
                c.positions[at] = pos;
            }
        }
    }
    // every warp has read slots[i] (lens_out may be the same array)
    __syncthreads();
    if (a.lens_out && threadIdx.x == 0) a.lens_out[i] = slot + 1;
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
    ~DeviceScope() {
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

cudaError_t launch_cache_append(const CacheAppendArgs& a, cudaStream_t s) {
    return launch_after(cache_append_kernel, dim3(a.n), kAppendWarps * 32, 0, s, a);
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
    Q3_CHECK(d->rows * d->kv_heads * ((d->max_len + kCachePage - 1) / kCachePage) <= INT_MAX,
             "q3_cache_create: rows * kv_heads * ceil(max_len / 64) must be below 2^31");
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
    Q3_CHECK(device >= 0, "q3_cache_create: bad device");
    auto* c = new (std::nothrow) q3_cache();
    if (!c) return fail(Q3_ERR_OOM, "q3_cache_create: host allocation failed");
    c->device = device;
    c->sms = num_sms(device);
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
    Q3_CHECK(q && k && v && q_norm && k_norm && cos_t && sin_t && token_pos && slots && q_out,
             "q3_cache_append: null pointer");
    if (n == 0) return Q3_OK;
    const CacheView& w = c->view;
    Q3_CHECK(n <= INT_MAX, "q3_cache_append: too many rows");
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
    Q3_CHECK(aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(q_out, 16),
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
    return launched(launch_cache_append(a, static_cast<cudaStream_t>(stream)), "q3_cache_append");
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
