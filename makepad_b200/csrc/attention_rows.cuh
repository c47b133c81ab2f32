// the simplest form: a warp per query row, its keys one after the other
#pragma once
#include "attention.cuh"

namespace mpq {

template <int D>
__global__ void __launch_bounds__(128) attention_rows_kernel(const __nv_bfloat16* k_base, const __nv_bfloat16* v_base, int64_t k_stride, int64_t v_stride, const __grid_constant__ AttnParams p)
{
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    constexpr int PER = D / 32;
    const int lane = threadIdx.x & 31, h = blockIdx.y, kh = h / p.group;
    const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (t >= p.tokens) return;
    int i = 0;
    AttnRequest r = {};
    for (; i < p.n; ++i) {
        r = attn_request(p, i);
        if (t >= r.first && t < r.first + r.rows) break;
    }
    if (i == p.n) return;
    const int seen = attn_seen(r, t - r.first);
    float q[PER], o[PER], m = -INFINITY, l = 0.f;
    for (int e = 0; e < PER; ++e) { q[e] = __bfloat162float(p.q[t * p.q_stride + (int64_t)h * D + lane * PER + e]); o[e] = 0.f; }
    for (int j = 0; j < seen; ++j) {
        const __nv_bfloat16 *k = nullptr, *v = nullptr;
        if (p.table) {
            const int page = p.table[i * p.width + (j >> p.page_shift)];
            const int64_t at = ((((int64_t)page * p.kv_heads + kh) << p.page_shift) + (j & ((1 << p.page_shift) - 1))) * D;
            if (page >= 0 && page < p.pages) { k = k_base + at; v = v_base + at; }     // an entry outside the cache reads as zeros
        } else {
            k = k_base + (r.first + j) * k_stride + (int64_t)kh * D;
            v = v_base + (r.first + j) * v_stride + (int64_t)kh * D;
        }
        float s = 0.f;
        for (int e = 0; e < PER; ++e) s = fmaf(q[e], k ? __bfloat162float(k[lane * PER + e]) : 0.f, s);
        for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(~0u, s, x);
        s *= p.scale_log2;
        const float m2 = fmaxf(m, s), a = m == -INFINITY ? 0.f : exp2f(m - m2), w = exp2f(s - m2);
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
