// Attention of few rows (one token, or a handful, per request and head of keys) over the pages of a cache: the cache is read once, at HBM's rate.
//
// The KEYS are the M of mma.sync.m16n8k16 and up to 8 (or 16) rows its N: S^T = K Q^T, O^T += V^T P^T.  A tile of 128 keys is 256 MMAs (512 with 16 rows) for the
// 64 KB (D = 128) that take an SM 2700 cycles of its share of the memory bandwidth.  With the rows as M, most of them idle, twice
// the MMAs took 2150 cycles a tile, and no stall of the memory was ever caught up.  (tcgen05 wants 128 rows, or the weights
// through shared memory, for nothing that is missing here.)
// 64 requests of 1000 to 8000 tokens, 64 heads on 8 heads of keys of 128: 1.24 GB in 195 us, 6.35 TB/s.  One request of 4001 tokens, 32 heads of keys: 66 MB in 20 us, of
// which about 9 are the first look at lengths and pages, the first bytes' latency, and the joining of each head's pieces.
//
// A CTA has one producer warp and four warps that compute, 32 of a tile's 128 keys each.  The producer looks up the pages and keeps a ring of tiles full
// (TMA, 128-byte swizzle; it runs ahead into the next unit), each warp waits for its own keys only.  Weights stay in registers: transposed 8 x 8 at a
// time (movmatrix), the accumulators of K Q^T are the B operand of the product with V^T.  At a unit's end the four warps' (maximum, sum, o) are
// joined through shared memory.
#pragma once
#include "attention.cuh"

namespace mpq {

constexpr int FEW_MOST_CTAS = 256, FEW_TILE = 128, FEW_WARPS = 4, FEW_KEYS = FEW_TILE / FEW_WARPS, FEW_THREADS = 32 * (FEW_WARPS + 1);
// a unit's end (sums joined, pieces stored and counted) takes a CTA about as long as two tiles
template <int NT>
using FewCut = AttnCut<8 * NT, FEW_TILE, 2, 2, false, 0>;
static_assert(FEW_THREADS >= ATTN_ENTRIES, "an entry per thread");

template <int D, int NT>
struct FewShape {
    static constexpr int ROWS = 8 * NT;
    static constexpr int WARP_BYTES = FEW_KEYS * D * 2;                      // keys (or values) of one warp
    static constexpr int STAGE_BYTES = 2 * FEW_WARPS * WARP_BYTES;           // [warp][k | v]
    static constexpr int STAGES = D == 128 ? 3 : 6;
    static constexpr int SMEM = 1024 + STAGES * STAGE_BYTES + FEW_WARPS * ROWS * D * 4;      // ... and the warps' parts of o
    static constexpr int PIECE = ROWS * (D + 2);                             // floats of a piece in scratch: o, maxima, sums
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transposed(uint32_t v)
{
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void few_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * FEW_WARPS) : "memory"); }

// NT: rows in eights.  BOX: keys per copy, 16 or 32 (a page of 16, or larger ones)
template <int D, int BOX, int NT>
__global__ void __launch_bounds__(FEW_THREADS, 1)
attention_few_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttnParams p)
{
    using S = FewShape<D, NT>;
    constexpr int ROWS = S::ROWS;
    extern __shared__ unsigned char smem_dyn[];
    __shared__ volatile int s_abort;
    __shared__ int s_last;
    __shared__ AttnShared s_shared;
    __shared__ float s_max[FEW_WARPS][ROWS], s_sum[FEW_WARPS][ROWS];
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
    start_beside();
    const AttnTotals totals = attn_totals<FewCut<NT>>(p, s_shared);          // (its barriers publish the mbarriers)
    AttnWalk<FewCut<NT>> u;

    if (warp == FEW_WARPS) {
        // ---- producer: lane = (box of a tile, k or v); boxes behind the request's last key are not fetched
        constexpr int BOXES = FEW_TILE / BOX, PER_WARP = FEW_KEYS / BOX, BOX_BYTES = BOX * D * 2;
        const int box = lane % BOXES, what = lane / BOXES;                   // 0: k, 1: v
        int s = 0;
        uint32_t phase = 1;
        for (bool run = u.begin(p, totals, s_shared); run; run = u.next_run(p, totals, s_shared))
            for (; u.more(totals); u.step(p, totals)) {
                // (a tile's pages are looked up while the one before waits for its room)
                const int32_t* row = p.table + u.request * p.width;
                const int end = u.end(totals);
                auto page_of = [&](int t) {
                    const int key = t * FEW_TILE + box * BOX;
                    if (what > 1 || t >= end || key >= u.r.keys) return -1;
                    const int page = row[key >> p.page_shift];
                    return page < 0 || page >= p.pages ? (int)p.pages : page;                    // (beyond the cache: zeros)
                };
                int page = page_of(u.first(totals));
                for (int t = u.first(totals); t < end; ++t) {
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
        const int g = lane >> 2, tq = lane & 3;              // an accumulator's lane: key (or column of o) g and g + 8, rows 2 tq and 2 tq + 1
        const int km = lane >> 3, kr = lane & 7;             // ldmatrix: matrix and row that the lane points to
        float* join = reinterpret_cast<float*>(smem_dyn + (smem0 - s2u(smem_dyn)) + S::STAGES * S::STAGE_BYTES);
        int s = 0;
        uint32_t phase = 0;
        for (bool run = u.begin(p, totals, s_shared); run; run = u.next_run(p, totals, s_shared))
        for (; u.more(totals); u.step(p, totals)) {
            const int rows = attn_block_rows(u.r, p.group.d, u.block, ROWS);
            const int row0 = u.block * ROWS;
            // keys that the rows see: this lane's, and every row of the block
            int seen[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) seen[n][i] = attn_seen(u.r, p.group.of(row0 + min(8 * n + 2 * tq + i, rows - 1)));
            const int seen_all = attn_seen(u.r, p.group.of(row0));
            uint32_t q[NT][D / 16][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int at = row0 + min(8 * n + g, rows - 1), tok = p.group.of(at);
                const __nv_bfloat16* from = p.q + (int64_t)(u.r.first + tok) * p.q_stride + ((u.head - tok) * (int)p.group.d + at) * D + 2 * tq;
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    q[n][k][0] = *reinterpret_cast<const uint32_t*>(from + 16 * k);
                    q[n][k][1] = *reinterpret_cast<const uint32_t*>(from + 16 * k + 8);
                }
            }
            float o[D / 16][NT][4], m[NT][2], l[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int c = 0; c < D / 16; ++c)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[c][n][j] = 0.f;
                m[n][0] = m[n][1] = -INFINITY;
                l[n][0] = l[n][1] = 0.f;
            }
            const int end = u.end(totals);
            for (int t = u.first(totals); t < end; ++t) {
                attn_wait(full(s, warp), phase, &s_abort, p.status, 42);
                const uint32_t kb = smem0 + s * S::STAGE_BYTES + warp * 2 * S::WARP_BYTES, vb = kb + S::WARP_BYTES;
                const int key0 = t * FEW_TILE + warp * FEW_KEYS;
                // byte of 16-byte chunk c (of D/8) of key r (of 32): boxes of BOX keys, in them halves of 64 elements, rows of 128 bytes, swizzled
                auto place_of = [&](uint32_t base, int r, int c) {
                    return base + (r / BOX) * (BOX * D * 2) + (c >> 3) * (BOX * 128) + (r % BOX) * 128 + (((c & 7) ^ (r & 7)) << 4);
                };
                float sc[2][NT][4];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int j = 0; j < 4; ++j) sc[h][n][j] = 0.f;
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t a[4];
                        ldsm4(a, place_of(kb, 16 * h + (km & 1) * 8 + kr, 2 * k + (km >> 1)));
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma_bf16(sc[h][n], a, q[n][k][0], q[n][k][1]);
                    }
                const bool ragged = key0 + FEW_KEYS > seen_all;
                float x[NT][2];
                bool moved = false;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            sc[h][n][j] *= p.scale_log2;
                            if (ragged && key0 + 16 * h + g + 8 * (j >> 1) >= seen[n][j & 1]) sc[h][n][j] = -INFINITY;
                        }
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        x[n][i] = fmaxf(m[n][i], fmaxf(fmaxf(sc[0][n][i], sc[0][n][i + 2]), fmaxf(sc[1][n][i], sc[1][n][i + 2])));
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) x[n][i] = fmaxf(x[n][i], __shfl_xor_sync(~0u, x[n][i], d));
                        moved |= x[n][i] != m[n][i];
                    }
                }
                if (__any_sync(~0u, moved)) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const float f = x[n][i] == -INFINITY ? 1.f : exp2f(m[n][i] - x[n][i]);
                            m[n][i] = x[n][i];
                            l[n][i] *= f;
#pragma unroll
                            for (int c = 0; c < D / 16; ++c) { o[c][n][i] *= f; o[c][n][i + 2] *= f; }
                        }
                }
                uint32_t pb[2][NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float b0 = m[n][0] == -INFINITY ? 0.f : m[n][0], b1 = m[n][1] == -INFINITY ? 0.f : m[n][1];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float e0 = exp2f(sc[h][n][0] - b0), e1 = exp2f(sc[h][n][1] - b1), e2 = exp2f(sc[h][n][2] - b0), e3 = exp2f(sc[h][n][3] - b1);
                        l[n][0] += e0 + e2;
                        l[n][1] += e1 + e3;
                        // bf16 is what the tensor cores take beside bf16 values; the sum keeps the weights as they were
                        pb[h][n][0] = transposed(pack_bf16(e0, e1));
                        pb[h][n][1] = transposed(pack_bf16(e2, e3));
                    }
                }
                const int left = u.r.keys - key0;                            // keys of this warp that exist
#pragma unroll
                for (int c = 0; c < D / 16; ++c)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t a[4];
                        ldsm4_trans(a, place_of(vb, 16 * h + (km >> 1) * 8 + kr, 2 * c + (km & 1)));
                        if (left < FEW_KEYS) {                               // values behind the last key may be anything, and 0 * NaN is not 0
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const int key = 16 * h + (j >> 1) * 8 + 2 * tq;
                                if (key >= left) a[j] = 0;
                                else if (key + 1 >= left) a[j] &= 0xFFFFu;
                            }
                        }
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma_bf16(o[c][n], a, pb[h][n][0], pb[h][n][1]);
                    }
                __syncwarp();
                if (lane == 0) bar_arrive(empty(s));
                if (++s == S::STAGES) { s = 0; phase ^= 1u; }
            }
            // ---- the four warps' parts: maxima, then everything at the common one
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) l[n][i] += __shfl_xor_sync(~0u, l[n][i], d);
                    if (g == 0) { s_max[warp][8 * n + 2 * tq + i] = m[n][i]; s_sum[warp][8 * n + 2 * tq + i] = l[n][i]; }
                }
            few_sync();
            auto top_of = [&](int r) { return fmaxf(fmaxf(s_max[0][r], s_max[1][r]), fmaxf(s_max[2][r], s_max[3][r])); };
            auto factor = [&](float m, float top) { return m == -INFINITY ? 0.f : exp2f(m - top); };
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int r = 8 * n + 2 * tq + i;
                    const float f = factor(m[n][i], top_of(r));
                    // (columns of a row in eights, turned by the row: the lanes of a store lie in different banks)
                    float* at = join + (warp * ROWS + r) * D;
                    if (r < rows)
#pragma unroll
                        for (int c = 0; c < D / 16; ++c) {
                            at[(16 * c + g) ^ (8 * tq)] = o[c][n][i] * f;
                            at[(16 * c + 8 + g) ^ (8 * tq)] = o[c][n][i + 2] * f;
                        }
                }
            few_sync();
            const bool cut = u.cut(totals);
            const int opener = cut ? u.opener(totals) : 0, closer = cut ? u.closer(totals) : 0;
            // a row's columns; `slot` of scratch: the unit that a run opened, or the one that it continues
            auto slot = [&](int r) { return p.partial + (int64_t)(2 * r + (r == opener ? 1 : 0)) * S::PIECE; };
            auto store = [&](int r, int c, float4 v) {
                const int at = row0 + r, tok = p.group.of(at);
                const int64_t to = ((int64_t)(u.r.first + tok) * p.q_heads + (u.head - tok) * (int)p.group.d + at) * D + c;
                if (p.out_f32) *reinterpret_cast<float4*>(static_cast<float*>(p.out) + to) = v;
                else *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + to) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
            };
            for (int e = threadIdx.x; e < rows * (D / 4); e += 32 * FEW_WARPS) {
                const int r = e / (D / 4), c = e % (D / 4) * 4;
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                float l = 0.f;
                const float top = top_of(r);
#pragma unroll
                for (int w = 0; w < FEW_WARPS; ++w) {
                    const float4 a = *reinterpret_cast<const float4*>(join + (w * ROWS + r) * D + (c ^ (8 * ((r >> 1) & 3))));
                    v.x += a.x; v.y += a.y; v.z += a.z; v.w += a.w;
                    l += s_sum[w][r] * factor(s_max[w][r], top);
                }
                if (!cut) {
                    const float f = l == 0.f ? 0.f : 1.f / l;
                    store(r, c, make_float4(v.x * f, v.y * f, v.z * f, v.w * f));
                } else {
                    float* mine = slot(u.run);
                    *reinterpret_cast<float4*>(mine + r * D + c) = v;
                    if (c == 0) { mine[ROWS * D + r] = top; mine[ROWS * D + ROWS + r] = l; }
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
                if (s_last)
                    // the pieces in order, eight at a time (all their loads in one latency), rescaled when a larger maximum comes
                    for (int e = threadIdx.x; e < rows * (D / 4); e += 32 * FEW_WARPS) {
                        const int r = e / (D / 4), c = e % (D / 4) * 4;
                        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                        float top = -INFINITY, l = 0.f;
                        for (int r0 = opener; r0 <= closer; r0 += 8) {
                            float4 a[8];
                            float pm[8], pl[8], both = top;
#pragma unroll
                            for (int k = 0; k < 8; ++k) {
                                pm[k] = -INFINITY;
                                if (r0 + k <= closer) {
                                    const float* from = slot(r0 + k);
                                    pm[k] = load_l2(from + ROWS * D + r);
                                    pl[k] = load_l2(from + ROWS * D + ROWS + r);
                                    a[k] = load_l2(reinterpret_cast<const float4*>(from + r * D + c));
                                }
                            }
#pragma unroll
                            for (int k = 0; k < 8; ++k) both = fmaxf(both, pm[k]);
                            const float f = factor(top, both);
                            top = both;
                            l *= f; v.x *= f; v.y *= f; v.z *= f; v.w *= f;
#pragma unroll
                            for (int k = 0; k < 8; ++k)
                                if (r0 + k <= closer) {
                                    const float h = factor(pm[k], top);
                                    l = fmaf(pl[k], h, l);
                                    v.x = fmaf(a[k].x, h, v.x); v.y = fmaf(a[k].y, h, v.y); v.z = fmaf(a[k].z, h, v.z); v.w = fmaf(a[k].w, h, v.w);
                                }
                        }
                        const float f = l == 0.f ? 0.f : 1.f / l;
                        store(r, c, make_float4(v.x * f, v.y * f, v.z * f, v.w * f));
                    }
            }
            few_sync();                                                      // the next unit writes what this one's threads read
        }
    }
    __syncthreads();
    settle_after_timeout(s_abort);
}

}  // namespace mpq
