// Attention of one new token over the paged cache: one warp a row and query head.
#include <cuda_runtime.h>

#include <cmath>

#include "attention.cuh"
#include "cache.hpp"
#include "ptx.cuh"
#include "quant.cuh"

namespace tb {

template <class T>
__device__ __forceinline__ float4 load4(const T* p, bool ok) {
    if (!ok) return make_float4(0.f, 0.f, 0.f, 0.f);
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const T* e = reinterpret_cast<const T*>(&u);
    return make_float4(static_cast<float>(e[0]), static_cast<float>(e[1]), static_cast<float>(e[2]),
                       static_cast<float>(e[3]));
}

// The warp's row over n keys; key(j) / value(j) give the rows. Each lane holds four dimensions.
template <class T, class Key, class Value>
__device__ __forceinline__ void attend_row(const T* q, T* out, float* lse, int d, float scale_log2, long long n,
                                           Key key, Value value) {
    const int lane = threadIdx.x & 31;
    const bool ok = lane * 4 < d;
    const float4 x = load4(q + lane * 4, ok);
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (long long j = 0; j < n; ++j) {
        const float4 y = load4(key(j) + lane * 4, ok);
        float s = x.x * y.x + x.y * y.y + x.z * y.z + x.w * y.w;
#pragma unroll
        for (int i = 16; i > 0; i >>= 1) s += __shfl_xor_sync(0xffffffffu, s, i);
        s *= scale_log2;
        const float m1 = fmaxf(m, s);
        const float base = m1 == -INFINITY ? 0.f : m1;
        const float f = exp2f(m - base), p = exp2f(s - base);
        m = m1;
        const float4 z = load4(value(j) + lane * 4, ok);
        l = l * f + p;
        o.x = o.x * f + p * z.x;
        o.y = o.y * f + p * z.y;
        o.z = o.z * f + p * z.z;
        o.w = o.w * f + p * z.w;
    }
    const float r = n > 0 ? 1.f / l : 0.f;
    if (ok) {
        T* t = out + lane * 4;
        t[0] = static_cast<T>(o.x * r);
        t[1] = static_cast<T>(o.y * r);
        t[2] = static_cast<T>(o.z * r);
        t[3] = static_cast<T>(o.w * r);
    }
    if (lse != nullptr && lane == 0) *lse = n > 0 ? ((m == -INFINITY ? 0.f : m) + log2f(l)) * kLn2 : -INFINITY;
}

struct DecodeArgs {
    const void *q, *k, *v;  // k, v: the layer's pages
    void* out;
    float* lse;
    const int32_t *slots, *table, *lengths;
    long long q_seq, q_head, o_seq, o_head;
    int n, q_heads, kv_heads, head_dim, page_size, num_pages, max_seqs, max_pages;
    float scale_log2;
    uint32_t* err;
};

template <class T>
__global__ void __launch_bounds__(32) decode_rows_kernel(DecodeArgs a) {
    grid_dependency_wait();
    const int i = blockIdx.y, h = blockIdx.x;
    const int kh = h / (a.q_heads / a.kv_heads);
    const int slot = a.slots[i];
    int len = 0;
    bool bad = slot < 0 || slot >= a.max_seqs;
    if (!bad) {
        len = a.lengths[slot];
        bad = len < 0 || static_cast<long long>(len) > static_cast<long long>(a.max_pages) * a.page_size;
    }
    const int32_t* table = a.table + static_cast<long long>(bad ? 0 : slot) * a.max_pages;
    if (!bad)
        for (int j = threadIdx.x; j < (len + a.page_size - 1) / a.page_size; j += 32)
            if (table[j] < 0 || table[j] >= a.num_pages) bad = true;
    if (__any_sync(0xffffffffu, bad)) {
        if (threadIdx.x == 0) atomicOr(a.err, DEV_ERR_INDEX);
        return;
    }
    auto row = [&](long long j) {
        const long long p = table[j / a.page_size];
        return ((p * a.kv_heads + kh) * a.page_size + j % a.page_size) * a.head_dim;
    };
    attend_row<T>(static_cast<const T*>(a.q) + i * a.q_seq + h * a.q_head,
                  static_cast<T*>(a.out) + i * a.o_seq + h * a.o_head,
                  a.lse ? a.lse + static_cast<long long>(i) * a.q_heads + h : nullptr, a.head_dim, a.scale_log2, len,
                  [&](long long j) { return static_cast<const T*>(a.k) + row(j); },
                  [&](long long j) { return static_cast<const T*>(a.v) + row(j); });
}

}  // namespace tb

using namespace tb;

extern "C" {

TB_API tb_status tb_cache_attend(tb_cache* c, int32_t layer, const int32_t* slots, int32_t n, int32_t q_heads,
                                 float scale, const void* q, int64_t q_seq_stride, int64_t q_head_stride, void* out,
                                 int64_t out_seq_stride, int64_t out_head_stride, float* lse, void* stream) {
    if (!c) return fail(TB_ERR_INVALID_ARGUMENT, "cache attend: null cache");
    TB_TRY(attention_check("cache attend", c->d.dtype, q_heads, c->d.kv_heads, c->d.head_dim, scale));
    if (layer < 0 || layer >= c->d.layers)
        return fail(TB_ERR_SHAPE_MISMATCH, "cache attend: layer %d of %d", layer, c->d.layers);
    if (n < 0) return fail(TB_ERR_SHAPE_MISMATCH, "cache attend: negative count");
    if (n > 65535 || q_heads > 4096) return fail(TB_ERR_NOT_ACCELERATED, "cache attend: more than 65535 rows or 4096 heads");
    if (n == 0) return TB_OK;
    if (!slots || !q || !out) return fail(TB_ERR_INVALID_ARGUMENT, "cache attend: null pointer");
    if (q_seq_stride < 0 || q_head_stride < 0 || out_seq_stride < 0 || out_head_stride < 0)
        return fail(TB_ERR_SHAPE_MISMATCH, "cache attend: negative stride");
    if (!aligned16(q) || !aligned16(out) || ((q_seq_stride | q_head_stride | out_seq_stride | out_head_stride) & 7))
        return fail(TB_ERR_INVALID_ARGUMENT, "cache attend: tensors must be 16-byte aligned with strides that are multiples of 8");
    const long long layer_elems = static_cast<long long>(c->d.num_pages) * c->d.kv_heads * c->d.page_size * c->d.head_dim;
    const long long at = layer_elems * layer * 2;  // bytes
    DecodeArgs a{q, static_cast<const char*>(c->b.k_pages) + at, static_cast<const char*>(c->b.v_pages) + at, out, lse,
                 slots, c->b.page_table, c->b.lengths, q_seq_stride, q_head_stride, out_seq_stride, out_head_stride, n,
                 q_heads, c->d.kv_heads, c->d.head_dim, c->d.page_size, c->d.num_pages, c->d.max_seqs, c->d.max_pages,
                 scale * kLog2e, c->ctx->dev_err};
    const dim3 grid(q_heads, n);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (c->d.dtype == TB_DT_BF16) decode_rows_kernel<__nv_bfloat16><<<grid, 32, 0, st>>>(a);
    else decode_rows_kernel<__half><<<grid, 32, 0, st>>>(a);
    TB_LAUNCHED(c->ctx);
    return TB_OK;
}

}  // extern "C"
