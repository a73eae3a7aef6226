// cache.cuh -- the bounded paged KV cache: device view and launchers of its
// operators (append, attention with accumulated weights, eviction).
#pragma once

#include "kernels.cuh"

namespace q3 {

constexpr int kCachePage = 64;  // slots per page
constexpr int kCacheHd = 128;   // head dimension

// One layer's cache as the kernels see it (q3_cache_desc).  Slot s of sequence r,
// kv head h: K/V row ((page_table(r)[s / 64] * kv_heads + h) * 64 + s % 64) * 128,
// weights and positions at (r * kv_heads + h) * slot_stride + s.
struct CacheView {
    bf16 *k, *v;
    int num_pages;
    const int32_t* tables;
    long long table_stride;
    float* weights;
    int32_t* positions;
    long long slot_stride;
    int rows, max_len, kv_heads;
    // q3_cache_desc.state_dev: the error word; the attention's chunks taken; the eviction's CTAs arrived
    uint32_t *err, *next_chunk, *arrived;
};

__host__ __device__ inline size_t cache_slot_index(const CacheView& c, int row, int head) {
    return (static_cast<size_t>(row) * c.kv_heads + head) * c.slot_stride;
}
__device__ __forceinline__ size_t cache_kv_offset(const CacheView& c, int page, int head, int slot) {
    return ((static_cast<size_t>(page) * c.kv_heads + head) * kCachePage + slot % kCachePage) * kCacheHd;
}

// Launches behind the stream's previous kernel by programmatic dependent launch: the
// kernel's CTAs may become resident while that one ends, and wait for its end and its
// writes (pdl_wait) before they read or write any of the caller's memory.  Every kernel
// triggers its own dependents after that wait.
template <class Kernel, class... Args>
cudaError_t launch_after(Kernel kernel, dim3 grid, int threads, size_t smem, cudaStream_t s, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

struct CacheAppendArgs {
    CacheView c;
    const bf16 *q, *k, *v;
    long long q_stride, k_stride, v_stride;
    const bf16 *q_norm, *k_norm;
    const float *rope_cos, *rope_sin;
    int max_pos;
    const int32_t *token_pos, *slots, *row_seq;
    int n, q_heads;
    bf16* q_out;
    long long q_out_stride;
    int32_t* lens_out;
    float eps;
};
cudaError_t launch_cache_append(const CacheAppendArgs& a, int sms, cudaStream_t s);

struct CacheAttnArgs {
    CacheView c;
    const bf16* q;
    long long q_stride;
    const int32_t* lens;
    bf16* out;
    long long out_stride;
    int q_heads, accumulate;
    void* ws;
};
// Tensor maps of the K and V pools as [num_pages x kv_heads x 64, 128] matrices:
// boxes of 64 columns by 64 rows (a full tile's half) and by 16.
struct CacheMaps {
    CUtensorMap k64, v64, k16, v16;
};
bool cache_maps(const CacheView& c, CacheMaps* maps);  // false without a driver
size_t cache_attention_ws_bytes(const CacheView& c, int q_heads, int accumulate, int sms);
cudaError_t launch_cache_attention(const CacheAttnArgs& a, const CacheMaps& maps, int sms, cudaStream_t s);

struct CacheEvictArgs {
    CacheView c;
    const int32_t *lens, *next_pos;
    int keep, recent;
    float* weights_out;      // null: in place
    int32_t* positions_out;  // null: in place
    int32_t* lens_out;
    void* ws;
};
size_t cache_evict_ws_bytes(const CacheView& c, int keep);
cudaError_t launch_cache_evict(const CacheEvictArgs& a, int sms, cudaStream_t s);

}  // namespace q3
