// cache_attention.cu -- attention of one query token per sequence over a bounded
// paged cache, with the attention every slot receives accumulated.
#include "cache.cuh"

namespace q3 {
namespace {

constexpr int kThreads = 128;
constexpr float kLog2e = 1.4426950408889634f;

// One CTA per (sequence, kv head): scores of every slot to the workspace, their
// maximum and sum, then the probabilities' sums into the weights and the output.
__global__ void __launch_bounds__(kThreads) cache_attention_kernel(const CacheAttnArgs a, float* scores) {
    const CacheView& c = a.c;
    const int row = blockIdx.x / c.kv_heads, head = blockIdx.x % c.kv_heads;
    const int G = a.q_heads / c.kv_heads, tid = threadIdx.x;
    __shared__ float q[16][kCacheHd];
    __shared__ float red[kThreads];
    __shared__ float mx[16], sum[16];
    __shared__ int bad;
    const int32_t* table = c.tables + row * c.table_stride;
    bf16* out = a.out + row * a.out_stride + static_cast<size_t>(head) * G * kCacheHd;
    const int len = a.lens[row];
    if (tid == 0) bad = len < 0 || len > c.max_len ? DEV_BAD_LENGTH : 0;
    __syncthreads();
    if (!bad)
        for (int p = tid; p < (len + kCachePage - 1) / kCachePage; p += kThreads)
            if (table[p] < 0 || table[p] >= c.num_pages) bad = DEV_BAD_PAGE;
    for (int i = tid; i < G * kCacheHd; i += kThreads)
        q[i / kCacheHd][i % kCacheHd] = bf2f(a.q[row * a.q_stride + static_cast<size_t>(head) * G * kCacheHd + i]);
    __syncthreads();
    if (bad || len == 0) {
        if (bad && tid == 0) record_error(c.err, bad);
        for (int i = tid; i < G * kCacheHd; i += kThreads) out[i] = f2bf(bad ? __int_as_float(0x7fc00000) : 0.0f);
        return;
    }
    float* sc = scores + static_cast<size_t>(blockIdx.x) * c.max_len * G;
    for (int t = tid; t < len; t += kThreads) {
        const bf16* k = c.k + cache_kv_offset(c, table[t / kCachePage], head, t);
        for (int g = 0; g < G; ++g) {
            float s = 0.0f;
            for (int d = 0; d < kCacheHd; ++d) s = fmaf(q[g][d], bf2f(k[d]), s);
            sc[static_cast<size_t>(t) * G + g] = s * (0.08838834764831845f * kLog2e);
        }
    }
    __syncthreads();
    for (int g = 0; g < G; ++g) {
        float m = -INFINITY;
        for (int t = tid; t < len; t += kThreads) m = fmaxf(m, sc[static_cast<size_t>(t) * G + g]);
        red[tid] = m;
        __syncthreads();
        for (int i = 0; i < kThreads; ++i) m = fmaxf(m, red[i]);
        __syncthreads();
        float l = 0.0f;
        for (int t = tid; t < len; t += kThreads) l += exp2f(sc[static_cast<size_t>(t) * G + g] - m);
        red[tid] = l;
        __syncthreads();
        if (tid == 0) {
            l = 0.0f;
            for (int i = 0; i < kThreads; ++i) l += red[i];
            mx[g] = m;
            sum[g] = l;
        }
        __syncthreads();
    }
    float acc[16];
    for (int g = 0; g < 16; ++g) acc[g] = 0.0f;
    for (int t = 0; t < len; ++t) {
        const float v = bf2f(c.v[cache_kv_offset(c, table[t / kCachePage], head, t) + tid]);
#pragma unroll
        for (int g = 0; g < 16; ++g)
            if (g < G) acc[g] = fmaf(exp2f(sc[static_cast<size_t>(t) * G + g] - mx[g]) / sum[g], v, acc[g]);
    }
#pragma unroll
    for (int g = 0; g < 16; ++g)
        if (g < G) out[g * kCacheHd + tid] = f2bf(acc[g]);
    if (a.accumulate) {
        float* w = c.weights + cache_slot_index(c, row, head);
        for (int t = tid; t < len; t += kThreads) {
            float p = 0.0f;
            for (int g = 0; g < G; ++g) p += exp2f(sc[static_cast<size_t>(t) * G + g] - mx[g]) / sum[g];
            w[t] += p;
        }
    }
}

}  // namespace

size_t cache_attention_ws_bytes(const CacheView& c, int q_heads, int, int) {
    return static_cast<size_t>(c.rows) * q_heads * c.max_len * 4;
}

cudaError_t launch_cache_attention(const CacheAttnArgs& a, int, cudaStream_t s) {
    cache_attention_kernel<<<a.c.rows * a.c.kv_heads, kThreads, 0, s>>>(a, static_cast<float*>(a.ws));
    return cudaGetLastError();
}

}  // namespace q3
