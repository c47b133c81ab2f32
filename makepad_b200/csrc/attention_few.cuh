// Attention of few rows (one token, or a handful, per request and head of keys) over the pages of a cache: the cache is read once, at HBM's rate.
//
// A block is 16 rows, the M of mma.sync.m16n8k16; with one row a head the other fifteen are idle, and still the tensor work of 32 keys (64 MMAs) is
// under a fifth of the time that their 16 KB take to arrive at an SM's share of the memory bandwidth.  (tcgen05 wants 128 rows, or the keys as its M operand and
// the weights through shared memory, for nothing that is missing here.)
//
// A CTA has one producer warp and four warps that compute, 32 of a tile's 128 keys each.  The producer looks up the pages and keeps a ring of tiles full
// (TMA, 128-byte swizzle; it runs ahead into the next unit), each warp waits for its own keys only.  Scores stay in registers: the accumulators of q k^T are the
// A operand of the product with v.  At a unit's end the four warps' (maximum, sum, o) are joined through shared memory.
#pragma once
#include "attention.cuh"

namespace mpq {

constexpr int FEW_MOST_CTAS = 256, FEW_ROWS = 16, FEW_TILE = 128, FEW_WARPS = 4, FEW_KEYS = FEW_TILE / FEW_WARPS, FEW_THREADS = 32 * (FEW_WARPS + 1);
static_assert(FEW_THREADS >= ATTN_ENTRIES, "an entry per thread");

using FewCut = AttnCut<FEW_ROWS, FEW_TILE, 0, false>;

template <int D>
struct FewShape {
    static constexpr int WARP_BYTES = FEW_KEYS * D * 2;                      // keys (or values) of one warp
    static constexpr int STAGE_BYTES = 2 * FEW_WARPS * WARP_BYTES;           // [warp][k | v]
    static constexpr int STAGES = D == 128 ? 3 : 6;
    // the warps' parts of o; the factors of a cut unit's pieces and up to sixteen rows of sums
    static constexpr int JOIN_BYTES = 4 * (FEW_WARPS * FEW_ROWS * D > FEW_ROWS * FEW_MOST_CTAS + FEW_ROWS * D ? FEW_WARPS * FEW_ROWS * D : FEW_ROWS * FEW_MOST_CTAS + FEW_ROWS * D);
    static constexpr int SMEM = 1024 + STAGES * STAGE_BYTES + JOIN_BYTES;
    static constexpr int PIECE = FEW_ROWS * (D + 2);                         // floats of a piece in scratch: o, maxima, sums
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void few_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * FEW_WARPS) : "memory"); }

// BOX: keys per copy, 16 or 32 (a page of 16, or larger ones)
template <int D, int BOX>
__global__ void __launch_bounds__(FEW_THREADS, 1)
attention_few_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttnParams p)
{
    using S = FewShape<D>;
    extern __shared__ unsigned char smem_dyn[];
    __shared__ volatile int s_abort;
    __shared__ int s_last;
    __shared__ AttnShared s_shared;
    __shared__ float s_max[FEW_WARPS][FEW_ROWS], s_sum[FEW_WARPS][FEW_ROWS];
    __shared__ __align__(8) uint64_t s_bars[S::STAGES * (FEW_WARPS + 1)];
    const uint32_t smem0 = (s2u(smem_dyn) + 1023u) & ~1023u, bars = s2u(s_bars);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto full = [&](int s, int w) { return bars + 8 * (s * FEW_WARPS + w); };
    auto empty = [&](int s) { return bars + 8 * (S::STAGES * FEW_WARPS + s); };
    if (threadIdx.x == 0) {
        s_abort = 0;
        for (int s = 0; s < S::STAGES; ++s) {
            for (int w = 0; w < FEW_WARPS; ++w) bar_init(full(s, w), 1);
            bar_init(empty(s), FEW_WARPS);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const AttnTotals totals = attn_totals<FewCut>(p, s_shared);              // (its barriers publish the mbarriers)
    AttnWalk<FewCut> u;

    if (warp == FEW_WARPS) {
        // ---- producer: lane = (box of a tile, k or v); boxes behind the request's last key are not fetched
        constexpr int BOXES = FEW_TILE / BOX, PER_WARP = FEW_KEYS / BOX, BOX_BYTES = BOX * D * 2;
        const int box = lane % BOXES, what = lane / BOXES;                   // 0: k, 1: v
        int s = 0;
        uint32_t phase = 1;
        for (bool run = u.begin(p, totals, s_shared); run; run = u.next_run(p, totals, s_shared))
            for (; u.more(); u.step(p, totals)) {
                // (a tile's pages are looked up while the one before waits for its room)
                const int32_t* row = p.table + u.request * p.width;
                const int end = u.end(totals);
                auto page_of = [&](int t) {
                    const int key = t * FEW_TILE + box * BOX;
                    if (what > 1 || t >= end || key >= u.r.keys) return -1;
                    const int page = row[key >> p.page_shift];
                    return page < 0 || page >= p.pages ? (int)p.pages : page;                    // (beyond the cache: zeros)
                };
                int page = page_of(u.first());
                for (int t = u.first(); t < end; ++t) {
                    const int next = page_of(t + 1);
                    attn_wait(empty(s), phase, &s_abort, p.status, 41);
                    __syncwarp();
                    // what a warp of the tile gets: whole boxes up to the last key
                    if (lane < FEW_WARPS) {
                        const int left = (min(u.r.keys - t * FEW_TILE, FEW_TILE) - lane * FEW_KEYS + BOX - 1) / BOX;
                        bar_expect_tx(full(s, lane), 2 * BOX_BYTES * max(0, min(left, PER_WARP)));
                    }
                    __syncwarp();
                    if (page >= 0) {
                        const int key = t * FEW_TILE + box * BOX, w = box / PER_WARP;
                        const uint32_t dst = smem0 + s * S::STAGE_BYTES + w * 2 * S::WARP_BYTES + what * S::WARP_BYTES + (box % PER_WARP) * BOX_BYTES;
                        tma_load_4d(dst, what ? &map_v : &map_k, 0, key & ((1 << p.page_shift) - 1), 0, page * p.kv_heads + u.head, full(s, w));
                    }
                    page = next;
                    if (++s == S::STAGES) { s = 0; phase ^= 1u; }
                }
            }
    } else {
        const int g = lane >> 2, tq = lane & 3;
        float* join = reinterpret_cast<float*>(smem_dyn + (smem0 - s2u(smem_dyn)) + S::STAGES * S::STAGE_BYTES);
        // ldmatrix: lane -> row of the matrix that it points to
        const int km = lane >> 3, kr = lane & 7;
        int s = 0;
        uint32_t phase = 0;
        for (bool run = u.begin(p, totals, s_shared); run; run = u.next_run(p, totals, s_shared))
        for (; u.more(); u.step(p, totals)) {
            const int rows = attn_block_rows(u.r, p.group.d, u.block, FEW_ROWS);
            const int row0 = u.block * FEW_ROWS;
            // keys that rows g and g + 8 see
            const int seen0 = attn_seen(u.r, p.group.of(row0 + min(g, rows - 1))), seen1 = attn_seen(u.r, p.group.of(row0 + min(g + 8, rows - 1)));
            const int seen_all = attn_seen(u.r, p.group.of(row0));             // by every row of the block
            uint32_t qa[D / 16][4];
            {
                auto row_of = [&](int r) {
                    const int at = row0 + min(r, rows - 1), tok = p.group.of(at);
                    return p.q + (int64_t)(u.r.first + tok) * p.q_stride + ((u.head - tok) * (int)p.group.d + at) * D + 2 * tq;
                };
                const __nv_bfloat16 *q0 = row_of(g), *q1 = row_of(g + 8);
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    qa[k][0] = *reinterpret_cast<const uint32_t*>(q0 + 16 * k);
                    qa[k][1] = *reinterpret_cast<const uint32_t*>(q1 + 16 * k);
                    qa[k][2] = *reinterpret_cast<const uint32_t*>(q0 + 16 * k + 8);
                    qa[k][3] = *reinterpret_cast<const uint32_t*>(q1 + 16 * k + 8);
                }
            }
            float o[D / 8][4];
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
            float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
            const int end = u.end(totals);
            for (int t = u.first(); t < end; ++t) {
                attn_wait(full(s, warp), phase, &s_abort, p.status, 42);
                const uint32_t kb = smem0 + s * S::STAGE_BYTES + warp * 2 * S::WARP_BYTES, vb = kb + S::WARP_BYTES;
                const int key0 = t * FEW_TILE + warp * FEW_KEYS;
                // byte of 16-byte chunk c (of D/8) of key r (of 32): boxes of BOX keys, in them halves of 64 elements, rows of 128 bytes, swizzled
                auto place_of = [&](uint32_t base, int r, int c) {
                    return base + (r / BOX) * (BOX * D * 2) + (c >> 3) * (BOX * 128) + (r % BOX) * 128 + (((c & 7) ^ (r & 7)) << 4);
                };
                float sc[4][4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) sc[i][j] = 0.f;
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t b[4];
                        ldsm4(b, place_of(kb, 16 * h + (km >> 1) * 8 + kr, 2 * k + (km & 1)));
                        mma_bf16(sc[2 * h], qa[k], b[0], b[1]);
                        mma_bf16(sc[2 * h + 1], qa[k], b[2], b[3]);
                    }
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) sc[i][j] *= p.scale_log2;
                if (key0 + FEW_KEYS > seen_all) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (key0 + 8 * i + 2 * tq + (j & 1) >= (j < 2 ? seen0 : seen1)) sc[i][j] = -INFINITY;
                }
                float x0 = m0, x1 = m1;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x0 = fmaxf(x0, fmaxf(sc[i][0], sc[i][1]));
                    x1 = fmaxf(x1, fmaxf(sc[i][2], sc[i][3]));
                }
#pragma unroll
                for (int d = 1; d < 4; d <<= 1) {
                    x0 = fmaxf(x0, __shfl_xor_sync(~0u, x0, d));
                    x1 = fmaxf(x1, __shfl_xor_sync(~0u, x1, d));
                }
                if (__any_sync(~0u, x0 != m0 || x1 != m1)) {
                    const float a0 = x0 == -INFINITY ? 1.f : exp2f(m0 - x0), a1 = x1 == -INFINITY ? 1.f : exp2f(m1 - x1);
                    m0 = x0; m1 = x1;
                    l0 *= a0; l1 *= a1;
#pragma unroll
                    for (int i = 0; i < D / 8; ++i) { o[i][0] *= a0; o[i][1] *= a0; o[i][2] *= a1; o[i][3] *= a1; }
                }
                const float b0 = m0 == -INFINITY ? 0.f : m0, b1 = m1 == -INFINITY ? 0.f : m1;
                uint32_t pa[2][4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float e0 = exp2f(sc[i][0] - b0), e1 = exp2f(sc[i][1] - b0), e2 = exp2f(sc[i][2] - b1), e3 = exp2f(sc[i][3] - b1);
                    l0 += e0 + e1;
                    l1 += e2 + e3;
                    // bf16 is what the tensor cores take beside bf16 values; the sum keeps the weights as they were
                    pa[i >> 1][2 * (i & 1)] = pack_bf16(e0, e1);
                    pa[i >> 1][2 * (i & 1) + 1] = pack_bf16(e2, e3);
                }
                const int left = u.r.keys - key0;                            // keys of this warp that exist
#pragma unroll
                for (int c = 0; c < D / 16; ++c)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t b[4];
                        ldsm4_trans(b, place_of(vb, 16 * h + (km & 1) * 8 + kr, 2 * c + (km >> 1)));
                        if (left < FEW_KEYS) {                               // values behind the last key may be anything, and 0 * NaN is not 0
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const int key = 16 * h + (j & 1) * 8 + 2 * tq;
                                if (key >= left) b[j] = 0;
                                else if (key + 1 >= left) b[j] &= 0xFFFFu;
                            }
                        }
                        mma_bf16(o[2 * c], pa[h], b[0], b[1]);
                        mma_bf16(o[2 * c + 1], pa[h], b[2], b[3]);
                    }
                __syncwarp();
                if (lane == 0) bar_arrive(empty(s));
                if (++s == S::STAGES) { s = 0; phase ^= 1u; }
            }
            // ---- the four warps' parts: maxima, then everything at the common one
#pragma unroll
            for (int d = 1; d < 4; d <<= 1) {
                l0 += __shfl_xor_sync(~0u, l0, d);
                l1 += __shfl_xor_sync(~0u, l1, d);
            }
            if (tq == 0) {
                s_max[warp][g] = m0; s_max[warp][g + 8] = m1;
                s_sum[warp][g] = l0; s_sum[warp][g + 8] = l1;
            }
            few_sync();
            auto top_of = [&](int r) { return fmaxf(fmaxf(s_max[0][r], s_max[1][r]), fmaxf(s_max[2][r], s_max[3][r])); };
            auto factor = [&](float m, float top) { return m == -INFINITY ? 0.f : exp2f(m - top); };
            const float f0 = factor(m0, top_of(g)), f1 = factor(m1, top_of(g + 8));
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
                // columns of a row in eights, their order turned by the row: the eight rows of a store lie in different banks
                float* at = join + (warp * FEW_ROWS + g) * D + (((i ^ g) & 7) | (i & ~7)) * 8 + 2 * tq;
                *reinterpret_cast<float2*>(at) = make_float2(o[i][0] * f0, o[i][1] * f0);
                *reinterpret_cast<float2*>(at + 8 * D) = make_float2(o[i][2] * f1, o[i][3] * f1);
            }
            few_sync();
            const bool cut = u.cut(totals);
            const int opener = cut ? u.opener(totals) : 0, closer = cut ? u.closer(totals) : 0;
            // a row's columns and what stands beside them; `slot` of scratch: the unit that a run opened, or the one that it continues
            auto slot = [&](int r) { return p.partial + (int64_t)(2 * r + (r == opener ? 1 : 0)) * S::PIECE; };
            auto store = [&](int r, int c, float v) {
                const int at = row0 + r, tok = p.group.of(at);
                const int64_t to = ((int64_t)(u.r.first + tok) * p.q_heads + (u.head - tok) * (int)p.group.d + at) * D + c;
                if (p.out_f32) static_cast<float*>(p.out)[to] = v;
                else static_cast<__nv_bfloat16*>(p.out)[to] = __float2bfloat16_rn(v);
            };
            for (int e = threadIdx.x; e < rows * D; e += 32 * FEW_WARPS) {
                const int r = e / D, c = e % D, place = ((((c >> 3) ^ (r & 7)) & 7) | ((c >> 3) & ~7)) * 8 + (c & 7);
                float v = 0.f, l = 0.f;
                const float top = top_of(r);
#pragma unroll
                for (int w = 0; w < FEW_WARPS; ++w) {
                    v += join[(w * FEW_ROWS + r) * D + place];
                    l += s_sum[w][r] * factor(s_max[w][r], top);
                }
                if (!cut) store(r, c, l == 0.f ? 0.f : v / l);
                else {
                    float* mine = slot(u.run);
                    mine[r * D + c] = v;
                    if (c == 0) { mine[FEW_ROWS * D + r] = top; mine[FEW_ROWS * D + FEW_ROWS + r] = l; }
                }
            }
            if (cut) {
                few_sync();
                if (threadIdx.x == 0) {
                    const uint32_t before = attn_arrive(p.arrived + opener);
                    s_last = before == (uint32_t)(closer - opener);
                    if (s_last) p.arrived[opener] = 0;
                }
                few_sync();
                if (s_last) {
                    // Factors of the pieces' rows; then one, two or four groups of threads add their part of the pieces each, in order, and the
                    // groups' sums are added in order.
                    const int pieces = closer - opener + 1;
                    float *fac = join, *acc = join + FEW_ROWS * FEW_MOST_CTAS;
                    for (int i = threadIdx.x; i < rows * pieces; i += 32 * FEW_WARPS) {
                        const int q = i / rows, r = i - q * rows;
                        fac[q * FEW_ROWS + r] = __ldcg(slot(opener + q) + FEW_ROWS * D + r);
                    }
                    few_sync();
                    if ((int)threadIdx.x < rows) {
                        const int r = threadIdx.x;
                        float top = -INFINITY, l = 0.f;
                        for (int q = 0; q < pieces; ++q) top = fmaxf(top, fac[q * FEW_ROWS + r]);
#pragma unroll 4
                        for (int q = 0; q < pieces; ++q) {
                            const float f = factor(fac[q * FEW_ROWS + r], top);
                            fac[q * FEW_ROWS + r] = f;
                            l = fmaf(f, __ldcg(slot(opener + q) + FEW_ROWS * D + FEW_ROWS + r), l);
                        }
                        s_sum[0][r] = l;
                    }
                    few_sync();
                    const int groups = rows <= 4 ? 4 : rows <= 8 ? 2 : 1, each = 32 * FEW_WARPS / groups, group = threadIdx.x / each;
                    const int q0 = pieces * group / groups, q1 = pieces * (group + 1) / groups;
                    for (int e = threadIdx.x - group * each; e < rows * D / 4; e += each) {
                        const int r = e / (D / 4);
                        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                        for (int q = q0; q < q1; q += 4) {
                            float4 a[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                if (q + k < q1) a[k] = __ldcg(reinterpret_cast<const float4*>(slot(opener + q + k)) + e);
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                if (q + k < q1) {
                                    const float f = fac[(q + k) * FEW_ROWS + r];
                                    v.x = fmaf(a[k].x, f, v.x); v.y = fmaf(a[k].y, f, v.y); v.z = fmaf(a[k].z, f, v.z); v.w = fmaf(a[k].w, f, v.w);
                                }
                        }
                        reinterpret_cast<float4*>(acc)[group * (rows * D / 4) + e] = v;
                    }
                    few_sync();
                    for (int e = threadIdx.x; e < rows * D; e += 32 * FEW_WARPS) {
                        float v = 0.f;
                        for (int w = 0; w < groups; ++w) v += acc[w * rows * D + e];
                        const float l = s_sum[0][e / D];
                        store(e / D, e % D, l == 0.f ? 0.f : v / l);
                    }
                }
            }
            few_sync();                                                      // the next unit writes what this one's threads read
        }
    }
    __syncthreads();
    settle_after_timeout(s_abort);
}

}  // namespace mpq
