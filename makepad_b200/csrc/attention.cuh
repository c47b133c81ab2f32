// Attention of the tokens of several requests over their own keys and values:
//
//   o[i] = sum_j p[i][j] v[j] / sum_j p[i][j],   p[i][j] = exp(scale * q[i].k[j] - max_j),   over the keys j <= lens - new + i
//
// of its request (lens keys, the last `new` of them the request's own new tokens).  Query head h reads head h / (q heads / kv heads) of
// the keys.  A row that sees no key is zero.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "norm.cuh"

namespace mpq {

// keys and values: pages of a cache, or rows beside the queries
struct AttnParams {
    const __nv_bfloat16 *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;   // elements between tokens (k, v: without a table)
    const int32_t *starts, *lens, *table;   // lens, table: null without a cache
    int64_t width;                          // entries of a table row
    int64_t pages;
    int page_shift;
    int64_t tokens;
    int n, q_heads, kv_heads;
    float scale;
    void* out;
    int out_f32;
};

// rows, first row and keys of request i, within the arrays whatever the lengths say
struct AttnRequest {
    int first, rows, keys;
};
__device__ __forceinline__ AttnRequest attn_request(const AttnParams& p, int i)
{
    const int64_t a = min(max((int64_t)p.starts[i], (int64_t)0), p.tokens), b = min(max((int64_t)p.starts[i + 1], a), p.tokens);
    AttnRequest r;
    r.first = (int)a;
    r.rows = (int)(b - a);
    r.keys = p.lens ? (int)min((int64_t)max(p.lens[i], 0), p.width << p.page_shift) : r.rows;
    return r;
}

// the simplest form: a warp per query row, its keys one after the other
template <int D>
__global__ void __launch_bounds__(128) attention_rows_kernel(const __grid_constant__ AttnParams p)
{
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    constexpr int PER = D / 32;
    const int lane = threadIdx.x & 31, h = blockIdx.y, kh = h / (p.q_heads / p.kv_heads);
    const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (t >= p.tokens) return;
    int i = 0;
    AttnRequest r = {};
    for (; i < p.n; ++i) {
        r = attn_request(p, i);
        if (t >= r.first && t < r.first + r.rows) break;
    }
    if (i == p.n) return;
    const int seen = max(0, min(r.keys, r.keys - r.rows + (int)(t - r.first) + 1));
    float q[PER], o[PER], m = -INFINITY, l = 0.f;
    for (int e = 0; e < PER; ++e) { q[e] = __bfloat162float(p.q[t * p.q_stride + (int64_t)h * D + lane * PER + e]); o[e] = 0.f; }
    for (int j = 0; j < seen; ++j) {
        const __nv_bfloat16 *k, *v;
        if (p.table) {
            const int page = p.table[i * p.width + (j >> p.page_shift)];
            const int64_t at = ((((int64_t)page * p.kv_heads + kh) << p.page_shift) + (j & ((1 << p.page_shift) - 1))) * D;
            k = v = nullptr;                                   // an entry outside the cache reads as zeros
            if (page >= 0 && page < p.pages) { k = p.k + at; v = p.v + at; }
        } else {
            k = p.k + (r.first + j) * p.k_stride + (int64_t)kh * D;
            v = p.v + (r.first + j) * p.v_stride + (int64_t)kh * D;
        }
        float s = 0.f;
        for (int e = 0; e < PER; ++e) s = fmaf(q[e], k ? __bfloat162float(k[lane * PER + e]) : 0.f, s);
        for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(~0u, s, x);
        s *= p.scale;
        const float m2 = fmaxf(m, s), a = m == -INFINITY ? 0.f : __expf(m - m2), w = __expf(s - m2);
        l = l * a + w;
        for (int e = 0; e < PER; ++e) o[e] = o[e] * a + w * (v ? __bfloat162float(v[lane * PER + e]) : 0.f);
        m = m2;
    }
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    for (int e = 0; e < PER; ++e) {
        const int64_t at = (t * p.q_heads + h) * D + lane * PER + e;
        if (p.out_f32) static_cast<float*>(p.out)[at] = o[e] * inv;
        else static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(o[e] * inv);
    }
}

}  // namespace mpq
