// Attention of many rows (prompts, chunks of prompts) on the fifth-generation tensor cores.
//
// A unit is 256 rows (two tiles of 128) and a head of keys; its keys come 128 at a time.  Per tile and 128 keys:
//   S = Q K^T      tcgen05.mma kind::f16, Q and K from shared memory, S in tensor memory
//   P = 2^(S - m)  a thread per row: S to registers, running maximum m and sum, P back over S as bf16
//   O += P V       P from tensor memory, V from shared memory (as it lies: keys are its rows, the MMA's K), O in tensor memory
// While the threads of one tile work on their S, the tensor core does the other tile's products: 4 x 128 x 128 x D x 2 flop per 128 keys
// in two bursts of 1024 cycles, which is also what 2 x 128 x 128 exponentials take.
//
// The maximum that the weights stand against follows late: only when a row's own maximum is 2^8 above it is O scaled (read, multiplied, written
// back); until then the weights just grow, which costs neither bf16 nor fp32 any of their bits.
//
// ROLES, 12 warps: two teams of four (a tile each): softmax, epilogue.  Warp 8 issues the MMAs, warp 9 fetches keys and values (TMA, by pages or
// by rows), warps 10 and 11 the rows of Q (any number of heads shares a head of keys, so a tile's rows are no box), a unit ahead.
// Tensor memory: S0, S1, O0, O1 of 128 columns each, all of it.
#pragma once
#include "attention.cuh"

namespace mpq {

constexpr int MANY_ROWS = 256, MANY_TILE = 128, MANY_THREADS = 384;
constexpr int MANY_REGS_WORK = 200, MANY_REGS_REST = 104;        // 2 x 200 + 104 = 3 x 168, what a thread is launched with
using ManyCut = AttnCut<MANY_ROWS, MANY_TILE, 1, MANY_THREADS / 32>;
constexpr float MANY_LATE = 8.f;                                  // log2 of how far a row's maximum runs ahead of the one in use

template <int D>
struct ManyShape {
    static constexpr int HALVES = D / 64, HALF_BYTES = 128 * 128;            // 128 keys (or rows) of 64 elements, 128-byte swizzle
    static constexpr int TILE_BYTES = HALVES * HALF_BYTES;
    static constexpr int STAGES = D == 128 ? 5 : 8;                          // K and V tiles in turn
    static constexpr int SMEM = 1024 + (2 + STAGES) * TILE_BYTES;
    static constexpr int PIECE = MANY_ROWS * (D + 2);                        // floats of a piece in scratch: o, maxima, sums
};

// both operands from shared memory
__device__ __forceinline__ void tc_mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// A from tensor memory
__device__ __forceinline__ void tc_mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// Operand whose rows (64 elements, 128 bytes, swizzled, eight of them 1024 bytes apart) run along the MMA's K: the next 64 of N or M lie
// HALF_BYTES on
__device__ __forceinline__ uint64_t smem_desc_sw128_mn(uint32_t addr)
{
    uint64_t d = 0;
    d |= (uint64_t)((addr >> 4) & 0x3FFF);
    d |= (uint64_t)((128 * 128) >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <int N>
__device__ __forceinline__ void team_sync(int team) { asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(N) : "memory"); }

struct ManyBars {
    uint32_t q_full, q_empty, s_full, p_full, o_full, o_empty, kv_full, kv_empty;
};

// PAGED: boxes of a page's keys; else boxes of 128 rows beside the queries
template <int D, bool PAGED>
__global__ void __launch_bounds__(MANY_THREADS, 1)
attention_many_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttnParams p)
{
    using S = ManyShape<D>;
    using Walk = AttnWalk<ManyCut>;
    extern __shared__ unsigned char smem_dyn[];
    __shared__ uint32_t s_tmem_base;
    __shared__ volatile int s_abort;
    __shared__ int s_last[2];
    __shared__ __align__(8) uint64_t s_bars[10 + 2 * S::STAGES];
    const uint32_t smem0 = (s2u(smem_dyn) + 1023u) & ~1023u, smem_kv = smem0 + 2 * S::TILE_BYTES, b0 = s2u(s_bars);
    const ManyBars bar = {b0, b0 + 8, b0 + 16, b0 + 32, b0 + 48, b0 + 64, b0 + 80, b0 + 80 + 8 * S::STAGES};
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        s_abort = 0;
        bar_init(bar.q_full, 64);
        bar_init(bar.q_empty, 1);
        for (int t = 0; t < 2; ++t) {
            bar_init(bar.s_full + 8 * t, 1);
            bar_init(bar.p_full + 8 * t, 128);
            bar_init(bar.o_full + 8 * t, 1);
            bar_init(bar.o_empty + 8 * t, 128);
        }
        for (int s = 0; s < S::STAGES; ++s) {
            bar_init(bar.kv_full + 8 * s, 1);
            bar_init(bar.kv_empty + 8 * s, 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s2u(&s_tmem_base)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem_base;
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const bool whole = !p.partial;
    const AttnPlace place = attn_locate<ManyCut>(p, whole, reinterpret_cast<uint32_t*>(smem_dyn));
    Walk u;
    u.begin(p, place, whole);
    // tiles of keys of row tile t of the unit: up to this one (none where it has no rows)
    auto tiles_of = [&](int t) {
        const int rows = attn_block_rows(u.r, p.group.d, u.block, MANY_ROWS) - 128 * t;
        if (rows <= 0) return 0;
        return attn_tiles(attn_seen(u.r, p.group.of(u.block * MANY_ROWS + 128 * t + min(rows, 128) - 1)), MANY_TILE);
    };

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(MANY_REGS_REST));
        if (warp == 8) {
            // ---- MMA issue
            const uint32_t idesc_s = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 3) << 17) | ((128u >> 4) << 24);                 // bf16 x bf16 -> f32, both K-major
            const uint32_t idesc_o = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((128u >> 4) << 24);      // V: rows along K
            int s = 0;
            uint32_t kv_phase = 0, q_phase = 0, p_phase[2] = {0, 0}, oe_phase[2] = {1, 1};
            auto advance = [&] { if (++s == S::STAGES) { s = 0; kv_phase ^= 1u; } };
            auto issue_s = [&](int t, int stage) {
                if (lane == 0) {
                    const uint64_t a = smem_desc_sw128(smem0 + t * S::TILE_BYTES), b = smem_desc_sw128(smem_kv + stage * S::TILE_BYTES);
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        const uint64_t off = (uint64_t)(((k >> 2) * S::HALF_BYTES + (k & 3) * 32) >> 4);
                        tc_mma_f16_ss(tmem + 128 * t, a + off, b + off, idesc_s, k ? 1u : 0u);
                    }
                    tc_commit(bar.s_full + 8 * t);
                }
            };
            for (; u.more(); u.step(p)) {
                const int first = u.first(), end = u.end(), e[2] = {min(end, tiles_of(0)), min(end, tiles_of(1))};
                attn_wait(bar.q_full, q_phase, &s_abort, p.status, 51);
                q_phase ^= 1u;
                attn_wait(bar.kv_full + 8 * s, kv_phase, &s_abort, p.status, 52);
                tc_fence_after();
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    if (first < e[t]) issue_s(t, s);
                if (lane == 0) {
                    tc_commit(bar.kv_empty + 8 * s);
                    if (first + 1 >= end) tc_commit(bar.q_empty);
                }
                advance();
                for (int j = first; j < end; ++j) {
                    const int v = s;
                    attn_wait(bar.kv_full + 8 * v, kv_phase, &s_abort, p.status, 53);
                    advance();
                    const int left = u.r.keys - j * MANY_TILE;
                    if (left < MANY_TILE) {
                        // values behind the last key may be anything, and 0 * NaN is not 0
                        const int rows = MANY_TILE - max(left, 0), from = max(left, 0);
                        for (int i = lane; i < rows * 8 * S::HALVES; i += 32) {
                            const int h = i / (rows * 8), at = i - h * rows * 8;
                            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(smem_kv + v * S::TILE_BYTES + h * S::HALF_BYTES + from * 128 + at * 16), "r"(0) : "memory");
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                    }
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                        if (j < e[t]) {
                            if (j == first) {
                                attn_wait(bar.o_empty + 8 * t, oe_phase[t], &s_abort, p.status, 54);
                                oe_phase[t] ^= 1u;
                            }
                            attn_wait(bar.p_full + 8 * t, p_phase[t], &s_abort, p.status, 55);
                            p_phase[t] ^= 1u;
                            tc_fence_after();
                            if (lane == 0) {
                                const uint64_t b = smem_desc_sw128_mn(smem_kv + v * S::TILE_BYTES);
#pragma unroll
                                for (int k = 0; k < MANY_TILE / 16; ++k)
                                    tc_mma_f16_ts(tmem + 256 + 128 * t, tmem + 128 * t + 8 * k, b + (uint64_t)((k * 16 * 128) >> 4), idesc_o, j > first || k ? 1u : 0u);
                                if (j + 1 == e[t]) tc_commit(bar.o_full + 8 * t);
                            }
                            if (j + 1 < e[t]) {
                                attn_wait(bar.kv_full + 8 * s, kv_phase, &s_abort, p.status, 56);
                                tc_fence_after();
                                issue_s(t, s);
                            }
                        }
                    if (lane == 0) {
                        tc_commit(bar.kv_empty + 8 * v);
                        if (j + 1 < end) {
                            tc_commit(bar.kv_empty + 8 * s);
                            if (j + 2 >= end) tc_commit(bar.q_empty);
                        }
                    }
                    if (j + 1 < end) advance();
                }
            }
        } else if (warp == 9) {
            // ---- keys and values: a lane per box and half
            int s = 0;
            uint32_t phase = 1;
            const int shift = PAGED ? min(p.page_shift, 7) : 7, boxes = MANY_TILE >> shift;
            const int h = lane % S::HALVES, box = lane / S::HALVES;
            const uint32_t box_bytes = 128u << shift;                          // of one half
            for (; u.more(); u.step(p)) {
                const int32_t* row = PAGED ? p.table + u.request * p.width : nullptr;
                const int end = u.end();
                for (int j = u.first(); j < end; ++j) {
                    const int key = j * MANY_TILE + (box << shift);
                    const bool mine = box < boxes && key < u.r.keys;
                    // at least one box is asked for, so that the barrier has something to count: of a unit without keys the first
                    const int there = (max(min(u.r.keys, (j + 1) * MANY_TILE) - j * MANY_TILE, 0) + (1 << shift) - 1) >> shift;
                    int page = 0;
                    if (PAGED && mine) {
                        page = row[key >> p.page_shift];
                        if (page < 0 || page >= p.pages) page = (int)p.pages;  // (beyond the cache: zeros)
                    }
#pragma unroll
                    for (int what = 0; what < 2; ++what) {
                        attn_wait(bar.kv_empty + 8 * s, phase, &s_abort, p.status, 57);
                        if (lane == 0) bar_expect_tx(bar.kv_full + 8 * s, there * S::HALVES * box_bytes);
                        __syncwarp();
                        if (mine) {
                            const uint32_t dst = smem_kv + s * S::TILE_BYTES + h * S::HALF_BYTES + box * box_bytes;
                            const CUtensorMap* map = what ? &map_v : &map_k;
                            if (PAGED) tma_load_4d(dst, map, 0, key & ((1 << p.page_shift) - 1), h, page * p.kv_heads + u.head, bar.kv_full + 8 * s);
                            else tma_load_4d(dst, map, 0, u.r.first + key, h, u.head, bar.kv_full + 8 * s);
                        }
                        if (++s == S::STAGES) { s = 0; phase ^= 1u; }
                    }
                }
            }
        } else if (warp >= 10) {
            // ---- rows of Q: 16 bytes at a time into the swizzled tiles
            uint32_t phase = 1;
            const int tid = threadIdx.x - 320;
            constexpr int CH = D / 8, STEP = 64 / CH;
            const int c = tid % CH, r0 = tid / CH;
            for (; u.more(); u.step(p)) {
                attn_wait(bar.q_empty, phase, &s_abort, p.status, 58);
                phase ^= 1u;
                const int rows = attn_block_rows(u.r, p.group.d, u.block, MANY_ROWS);
                // thread: chunk c of every fourth (or eighth) row; token and head of the row go on with it
                const int all = rows <= 128 ? 128 : 256, group = p.group.d;
                const int tok_step = p.group.of(STEP), head_step = STEP - tok_step * group;
                int tok = p.group.of(u.block * MANY_ROWS + r0), head = u.block * MANY_ROWS + r0 - tok * group;
#pragma unroll 4
                for (int r = r0; r < all; r += STEP) {
                    const __nv_bfloat16* src = p.q + (int64_t)(u.r.first + (r < rows ? tok : 0)) * p.q_stride + (u.head * group + head) * D + c * 8;
                    const uint32_t dst = smem0 + (r >> 7) * S::TILE_BYTES + (c >> 3) * S::HALF_BYTES + (r & 127) * 128 + (((c & 7) ^ (r & 7)) << 4);
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(r < rows ? 16 : 0) : "memory");
                    tok += tok_step;
                    head += head_step;
                    if (head >= group) { head -= group; ++tok; }
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                bar_arrive(bar.q_full);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(MANY_REGS_WORK));
        // ---- a thread per row
        const int t = warp >> 2, row = threadIdx.x & 127;                      // (a warp of a team reaches the lanes 32 (warp % 4) ..)
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lanes + 128 * t, to = tmem + lanes + 256 + 128 * t;
        uint32_t s_phase = 0, o_phase = 0;
            for (; u.more(); u.step(p)) {
                const int rows = attn_block_rows(u.r, p.group.d, u.block, MANY_ROWS) - 128 * t;
                if (rows <= 0) continue;
                const int at = u.block * MANY_ROWS + 128 * t + min(row, rows - 1), tok = p.group.of(at);
                const int seen = attn_seen(u.r, tok), seen_all = attn_seen(u.r, p.group.of(u.block * MANY_ROWS + 128 * t));
                const int first = u.first(), end = min(u.end(), tiles_of(t));
                float m = -INFINITY, l = 0.f;                                  // m in units of the scores as they come
                for (int j = first; j < end; ++j) {
                    attn_wait(bar.s_full + 8 * t, s_phase, &s_abort, p.status, 59);
                    s_phase ^= 1u;
                    tc_fence_after();
                    // S is read twice, for the maximum and for the weights: 128 registers less, for 128 cycles of tensor memory
                    const bool ragged = (j + 1) * MANY_TILE > seen_all;
                    const int left = seen - j * MANY_TILE;
                    auto hide = [&](uint32_t (&x)[32], int c) {
                        if (ragged) {
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (32 * c + i >= left) x[i] = 0xFF800000u;
                        }
                    };
                    float y[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int c = 0; c < 4; c += 2) {
                        uint32_t x[2][32];
                        tc_ld32(ts + 32 * c, x[0]);
                        tc_ld32(ts + 32 * c + 32, x[1]);
                        tc_ld_wait();
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            hide(x[h], c + h);
#pragma unroll
                            for (int i = 0; i < 32; ++i) y[i & 3] = fmaxf(y[i & 3], __uint_as_float(x[h][i]));
                        }
                    }
                    const float top = fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]));
                    if (j == first) m = top;
                    else if (__any_sync(~0u, (top - m) * p.scale_log2 > MANY_LATE)) {
                        // (this S came behind the last product into O)
                        const float m2 = fmaxf(m, top), f = m2 == -INFINITY ? 1.f : ex2((m - m2) * p.scale_log2);
                        m = m2;
                        l *= f;
#pragma unroll 1
                        for (int c = 0; c < D / 32; ++c) {
                            uint32_t o[32];
                            tc_ld32(to + 32 * c, o);
                            tc_ld_wait();
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                            tc_st16(to + 32 * c, o);
                            tc_st16(to + 32 * c + 16, o + 16);
                        }
                    }
                    const float base = m == -INFINITY ? 0.f : m * p.scale_log2;
                    float sum[2] = {0.f, 0.f};
                    // (the weights of 32 keys take the place of 16 scores that have been read: the next 32 are, before they are overwritten)
                    uint32_t x[2][32];
                    tc_ld32(ts, x[0]);
                    tc_ld_wait();
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        if (c < 3) tc_ld32(ts + 32 * (c + 1), x[(c + 1) & 1]);
                        hide(x[c & 1], c);
                        uint32_t w[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float e0 = ex2(fmaf(__uint_as_float(x[c & 1][2 * i]), p.scale_log2, -base)), e1 = ex2(fmaf(__uint_as_float(x[c & 1][2 * i + 1]), p.scale_log2, -base));
                            sum[0] += e0;
                            sum[1] += e1;
                            // bf16 is what the tensor cores take beside bf16 values; the sum keeps the weights as they were
                            w[i] = pack_bf16(e0, e1);
                        }
                        if (c < 3) tc_ld_wait();
                        tc_st16(ts + 16 * c, w);
                    }
                    l += sum[0] + sum[1];
                    tc_st_wait();
                    tc_fence_before();
                    bar_arrive(bar.p_full + 8 * t);
                }
                // ---- the unit's end: O, unscaled
                const bool some = first < end;
                if (some) {
                    attn_wait(bar.o_full + 8 * t, o_phase, &s_abort, p.status, 60);
                    o_phase ^= 1u;
                    tc_fence_after();
                }
                const bool cut = u.cut();
                const int opener = cut ? u.opener() : 0, closer = cut ? u.closer() : 0;
                const int64_t to_row = ((int64_t)(u.r.first + tok) * p.q_heads + (u.head - tok) * (int)p.group.d + at) * D;
                auto store16 = [&](int c, const float* v) {                    // 16 columns from c on
                    if (row >= rows) return;
                    if (p.out_f32) {
                        float* out = static_cast<float*>(p.out) + to_row + c;
#pragma unroll
                        for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(out + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                    } else {
                        uint32_t* out = reinterpret_cast<uint32_t*>(static_cast<__nv_bfloat16*>(p.out) + to_row + c);
                        uint32_t w[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
                        *reinterpret_cast<uint4*>(out) = make_uint4(w[0], w[1], w[2], w[3]);
                        *reinterpret_cast<uint4*>(out + 4) = make_uint4(w[4], w[5], w[6], w[7]);
                    }
                };
                // a piece: [column / 4][row][4], so that a warp's threads lie beside each other; then maxima, sums
                auto slot = [&](int cta) { return p.partial + (int64_t)(2 * cta + (cta == opener ? 1 : 0)) * S::PIECE; };
                const int mine = 128 * t + row;
                const float inv = l == 0.f ? 0.f : 1.f / l;
                if (some) {
#pragma unroll
                    for (int c = 0; c < D; c += 16) {
                        uint32_t o[16];
                        tc_ld16(to + c, o);
                        tc_ld_wait();
                        float v[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(o[i]) * (cut ? 1.f : inv);
                        if (!cut) store16(c, v);
                        else {
                            float4* to4 = reinterpret_cast<float4*>(slot(blockIdx.x)) + (c >> 2) * MANY_ROWS + mine;
#pragma unroll
                            for (int i = 0; i < 4; ++i) to4[i * MANY_ROWS] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                        }
                    }
                    tc_fence_before();
                    bar_arrive(bar.o_empty + 8 * t);
                }
                if (cut) {
                    float* head = slot(blockIdx.x) + MANY_ROWS * D;
                    head[mine] = m == -INFINITY ? m : m * p.scale_log2;
                    head[MANY_ROWS + mine] = l;
                    __threadfence();
                    team_sync<128>(t);
                    if (row == 0) {
                        const uint32_t before = atomicAdd(p.arrived + 2 * opener + t, 1u);
                        s_last[t] = before == (uint32_t)(closer - opener);
                        if (s_last[t]) p.arrived[2 * opener + t] = 0;
                        __threadfence();
                    }
                    team_sync<128>(t);
                    if (s_last[t]) {
                        float top = -INFINITY, sum = 0.f;
                        for (int cta = opener; cta <= closer; ++cta) top = fmaxf(top, __ldcg(slot(cta) + MANY_ROWS * D + mine));
                        for (int cta = opener; cta <= closer; ++cta) {
                            const float mm = __ldcg(slot(cta) + MANY_ROWS * D + mine);
                            if (mm != -INFINITY) sum = fmaf(exp2f(mm - top), __ldcg(slot(cta) + MANY_ROWS * D + MANY_ROWS + mine), sum);
                        }
                        const float scale = sum == 0.f ? 0.f : 1.f / sum;
                        for (int c = 0; c < D; c += 16) {
                            float v[16];
#pragma unroll
                            for (int i = 0; i < 16; ++i) v[i] = 0.f;
                            for (int cta = opener; cta <= closer; ++cta) {
                                const float mm = __ldcg(slot(cta) + MANY_ROWS * D + mine);
                                if (mm == -INFINITY) continue;                 // (nothing of this piece is seen: its o was not written)
                                const float f = exp2f(mm - top) * scale;
                                const float4* from = reinterpret_cast<const float4*>(slot(cta)) + (c >> 2) * MANY_ROWS + mine;
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    const float4 a = __ldcg(from + i * MANY_ROWS);
                                    v[4 * i] = fmaf(a.x, f, v[4 * i]); v[4 * i + 1] = fmaf(a.y, f, v[4 * i + 1]);
                                    v[4 * i + 2] = fmaf(a.z, f, v[4 * i + 2]); v[4 * i + 3] = fmaf(a.w, f, v[4 * i + 3]);
                                }
                            }
                            store16(c, v);
                        }
                    }
                    team_sync<128>(t);                                         // (s_last is the next unit's then)
                }
            }
    }
    tc_fence_before();
    __syncthreads();
    settle_after_timeout(s_abort);
    if (warp == 8) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

}  // namespace mpq
