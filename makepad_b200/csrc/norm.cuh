// The norms around a block and the residual sum between them, one pass over a row:
//
//   t  = x                                              (the block's output, M x H)
//   t  = t / sqrt(mean(t^2) + eps) * post_weight        if there is a norm behind the block
//   r' = r + alpha * gate * t                           gate: one value per column, or per element
//   y  = r' / sqrt(mean(r'^2) + eps) * weight           what the next block reads
//
// A CTA has a row, a thread NV groups of eight columns, which stay in registers (x as it came) from the load to the last store (above 16384 columns 1024 threads
// have 64 registers for four groups, and some 120 to 240 bytes of a thread go through local memory: 2048 bf16 rows of 32768 columns, both norms and a gate, 197 us, 4.1 TB/s; of
// 16384 columns 91 us, 4.4): x and r are read once, r' and y written once.  Sums of squares are fp32, in a fixed order.  Bound: HBM, (x + 4 + 4 + y) bytes per element: 8192 bf16 rows of 8192 columns, both norms,
// a gate 139 us (in place, 5.8 TB/s; 153 with other rows to write to); without the norm behind the block 119, 6.8 TB/s.  What is between is the first sum, during which a row has no traffic: rows on an SM count.  (CTAs that stay, the
// next row's loads in registers and the weights in shared memory: 151; in a ring of bulk copies 174, of cp.async 197.)
// The weights and a gate of one row are read by every CTA and come from L1 / L2.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "pdl.cuh"

namespace mpq {

struct NormParams {
    const void* x;
    const float* residual;      // or null: zeros
    float* residual_out;        // or null; may be residual
    const float* post_weight;   // or null: no norm behind the block
    const float* gate;          // or null: ones
    const float* weight;        // or null: ones
    void* y;                    // or null: no norm in front of the next block
    int64_t gate_stride;        // 0: one row for all
    int H;
    float alpha, eps;
};

constexpr int NORM_MOST_H = 32768;

struct Eight {
    float v[8];
};

// bf16 -> fp32 is a shift
__device__ __forceinline__ Eight eight_of_bf16(uint4 u)
{
    Eight e;
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        e.v[2 * i] = __uint_as_float(w[i] << 16);
        e.v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
    return e;
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint4 bf16_of_eight(const Eight& e)
{
    return make_uint4(pack_bf16(e.v[0], e.v[1]), pack_bf16(e.v[2], e.v[3]), pack_bf16(e.v[4], e.v[5]), pack_bf16(e.v[6], e.v[7]));
}
__device__ __forceinline__ Eight load_eight(const float* p)
{
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    return Eight{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
}
__device__ __forceinline__ Eight load_eight(const __nv_bfloat16* p) { return eight_of_bf16(*reinterpret_cast<const uint4*>(p)); }
__device__ __forceinline__ void store_eight(float* p, const Eight& e)
{
    *reinterpret_cast<float4*>(p) = make_float4(e.v[0], e.v[1], e.v[2], e.v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(e.v[4], e.v[5], e.v[6], e.v[7]);
}
__device__ __forceinline__ void store_eight(__nv_bfloat16* p, const Eight& e) { *reinterpret_cast<uint4*>(p) = bf16_of_eight(e); }

// the CTA's sum, the same bits in every thread; `sums` is used by one call only
__device__ __forceinline__ float norm_block_sum(float v, float* sums)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    const int warps = blockDim.x >> 5;
    if (warps == 1) return v;
    if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (int)(threadIdx.x & 31) < warps ? sums[threadIdx.x & 31] : 0.f;
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    return v;
}

// Eight columns as they lie in memory
template <class X>
struct RawEight;
template <>
struct RawEight<__nv_bfloat16> {
    uint4 a;
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { a = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ Eight eight() const { return eight_of_bf16(a); }
};
template <>
struct RawEight<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) { a = *reinterpret_cast<const float4*>(p); b = *reinterpret_cast<const float4*>(p + 4); }
    __device__ __forceinline__ Eight eight() const { return Eight{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}}; }
};

template <int THREADS, int CTAS, int NV, class X, class Y>
__global__ void __launch_bounds__(THREADS, CTAS) residual_norm_kernel(const __grid_constant__ NormParams p)
{
    __shared__ float s_sums[2][32];
    start_beside();
    const int64_t row = blockIdx.x, base = row * p.H;
    const int step = blockDim.x * 8, c0 = threadIdx.x * 8;
    const X* x = static_cast<const X*>(p.x) + base;
    RawEight<X> raw[NV];
    Eight r[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = c0 + i * step;
        raw[i] = RawEight<X>{};
        if (c < p.H) raw[i].load(x + c);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = c0 + i * step;
        if (p.residual && c < p.H) r[i] = load_eight(p.residual + base + c);
        else r[i] = Eight{};
    }
    float scale = 1.f;
    if (p.post_weight) {
        float sq = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const Eight t = raw[i].eight();
#pragma unroll
            for (int j = 0; j < 8; ++j) sq = fmaf(t.v[j], t.v[j], sq);
        }
        scale = 1.f / sqrtf(norm_block_sum(sq, s_sums[0]) / (float)p.H + p.eps);
    }
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = c0 + i * step;
        if (c < p.H) {
            Eight t = raw[i].eight();
            if (p.post_weight) {
                const Eight w = load_eight(p.post_weight + c);
#pragma unroll
                for (int j = 0; j < 8; ++j) t.v[j] = t.v[j] * scale * w.v[j];
            }
            if (p.gate) {
                const Eight g = load_eight(p.gate + row * p.gate_stride + c);
#pragma unroll
                for (int j = 0; j < 8; ++j) t.v[j] *= g.v[j];
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                r[i].v[j] = fmaf(p.alpha, t.v[j], r[i].v[j]);
                sq = fmaf(r[i].v[j], r[i].v[j], sq);
            }
            if (p.residual_out) store_eight(p.residual_out + base + c, r[i]);
        }
    }
    if (!p.y) return;
    scale = 1.f / sqrtf(norm_block_sum(sq, s_sums[1]) / (float)p.H + p.eps);
    Y* y = static_cast<Y*>(p.y) + base;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = c0 + i * step;
        if (c < p.H) {
            if (p.weight) {
                const Eight w = load_eight(p.weight + c);
#pragma unroll
                for (int j = 0; j < 8; ++j) r[i].v[j] = r[i].v[j] * scale * w.v[j];
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) r[i].v[j] *= scale;
            }
            store_eight(y + c, r[i]);
        }
    }
}

}  // namespace mpq
