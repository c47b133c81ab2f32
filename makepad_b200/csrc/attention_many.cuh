// Attention of many rows (prompts, chunks of prompts) on the fifth-generation tensor cores.
//
// A unit is 256 rows (two tiles of 128) and a head of keys; its keys come 128 at a time.  Per tile and 128 keys:
//   S = Q K^T      tcgen05.mma kind::f16, Q and K from shared memory, S in tensor memory
//   P = 2^(S - m)  S to registers, running maximum m and sum, P back over S as bf16
//   O += P V       P from tensor memory, V from shared memory (as it lies: keys are its rows, the MMA's K), O in tensor memory
// P lies over S, so the chain of a tile is S, softmax, P V, next S; while one tile's softmax runs the tensor core does the other tile's products
// (1024 cycles at D = 128).  The softmax is therefore made short: two teams of four warps per tile, a thread per row and half of the
// keys; a quarter of the exponentials by polynomial (power2); the product begins with the first half of each team's keys.
// Cycles per 128 keys of both tiles: one team per tile 3960; as it is 3250, of them 2048 of tensor pipe at D = 128, 1536 of special-function units, 65 % of all issue
// slots used.  (Sixteen warps for one tile and then the other: 4500, they all wait for the same exchange of maxima.  Half, a third, an eighth or none of the
// exponentials by polynomial: 0 to 10 % slower.)
// A prompt of 8192 tokens, 32 heads on 8 of 128: 551 GFLOP in 0.48 ms (1.14 PFLOP/s; 0.55 ms when it runs for seconds and the power is capped).  A unit's end takes
// about 4000 cycles, a piece of a cut one 8000 more.
//
// The running maximum and sum are the published one-pass softmax (Milakov and Gimelshein 2018); that the maximum may follow late, and that some of the exponentials are
// better made by fused multiply-adds (rounding to a whole exponent and a polynomial for the rest, after Cody and Waite), is known of attention on this chip, too: neither is this library's
// idea.  The maximum that the weights stand against follows late: only when a row's own maximum is 2^8 above it is O scaled (read, multiplied, written
// back); until then the weights just grow, which costs neither bf16 nor fp32 any of their bits.
//
// ROLES, 20 warps: 0..15 softmax and epilogue (tile, half, quarter of the rows).  16 and 17 issue the MMAs, a tile each: one warp for both had its
// own bookkeeping between the tiles' products.  18 fetches keys and values (TMA, by pages or by rows), 19 walks the units and says to the others what
// each is, ahead of them.  A tile's rows of Q (any number of heads shares a head of keys, so they are no box) are copied by its softmax teams behind
// their last weights, while the last product runs (as boxes, where they are some, they came no sooner).  Tensor memory: S0, S1, O0, O1 of 128 columns each, all of it.
#pragma once
#include <type_traits>

#include "attention.cuh"

namespace mpq {

constexpr int MANY_ROWS = 256, MANY_TILE = 128, MANY_THREADS = 640;
constexpr int MANY_REGS_WORK = 104, MANY_REGS_REST = 64;         // 4 x 104 + 64 = 5 x 96, what a thread is launched with
using ManyCut = AttnCut<MANY_ROWS, MANY_TILE, 1, 4, true, 6>;
constexpr int MANY_POWERS = 4;                                    // every so many pairs of weights by a polynomial: see power2
constexpr float MANY_LATE = 8.f;                                  // log2 of how far a row's maximum runs ahead of the one in use

constexpr int MANY_UNITS = 4;                                     // units that are known at a time
struct ManyUnit {
    int there;                               // 0: no more units
    int first, end, ends[2];                 // tiles of keys of this CTA: all, and up to where the row tiles want them
    int keys, new_rows, first_row;           // of the request
    int row0, rows, head, request;           // first packed row of the block, rows of it
    int cut, opener, closer, run;            // whether other runs have tiles of the unit, and which; this one
};
struct ManyShared {
    uint64_t q_full[2], s_full[2], p_half[2], p_full[2], o_full[2], o_empty[2], kv_full[8], kv_empty[8], unit_full[MANY_UNITS], unit_empty[MANY_UNITS], told[16], turn[2], pair[8], team[2];
    ManyUnit units[MANY_UNITS];
    AttnShared totals;
    uint32_t tmem;
    int last[2];
    volatile int abort;
};

template <int D>
struct ManyShape {
    static constexpr int HALVES = D / 64, HALF_BYTES = 128 * 128;            // 128 keys (or rows) of 64 elements, 128-byte swizzle
    static constexpr int TILE_BYTES = HALVES * HALF_BYTES;
    static constexpr int STAGES = D == 128 ? 4 : 8;                          // K and V tiles in turn
    static constexpr int STORE_BYTES = 16 * 2048;                            // per softmax warp: 64 bytes of 32 rows on their way out
    static constexpr int SMEM = (2 + STAGES) * TILE_BYTES + STORE_BYTES + sizeof(ManyShared);
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
// one lane of a converged warp
__device__ __forceinline__ bool elect_one()
{
    uint32_t pred;
    asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xffffffff;\n\tselp.u32 %0, 1, 0, P;\n\t}" : "=r"(pred));
    return pred != 0;
}
// a value that is the same in all lanes, where the compiler cannot see it: operands of an MMA that it does not know to be uniform go from a register to a
// uniform one in front of every instruction (16 MMAs took 1760 cycles to issue; their pipe time is 1024)
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(~0u, x, 0); }
__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// NaN wins
__device__ __forceinline__ float max_nan(float a, float b, float c)
{
    float y;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
// two fp32 in a register pair
__device__ __forceinline__ uint64_t pair_of(uint32_t a, uint32_t b)
{
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(a), "r"(b));
    return v;
}
__device__ __forceinline__ uint64_t pair_of(float a, float b) { return pair_of(__float_as_uint(a), __float_as_uint(b)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b)
{
    uint64_t v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
// 2^t of both by multiplications and additions, for t <= 8 (below -126: 2^-126): t = n + f with |f| <= 1/2, by adding and taking away 1.5 * 2^23,
// whose low bits are then n; 2^f by the polynomial of degree 3 with the least relative error there, 7.5e-5 (a linear programme over 4001
// points), a twentieth of what bf16 rounds off; n goes into the exponent.
__device__ __forceinline__ uint64_t power2(uint64_t t)
{
    const float lo = fmaxf(__uint_as_float((uint32_t)t), -126.f), hi = fmaxf(__uint_as_float((uint32_t)(t >> 32)), -126.f);
    const uint64_t x = pair_of(lo, hi), big = pair_of(12582912.f, 12582912.f), n = add2(x, big);
    const uint64_t f = add2(x, fma2(n, pair_of(-1.f, -1.f), big));
    uint64_t y = fma2(f, pair_of(0.0551716685295105f, 0.0551716685295105f), pair_of(0.2426111251115799f, 0.2426111251115799f));
    y = fma2(y, f, pair_of(0.6932609677314758f, 0.6932609677314758f));
    y = fma2(y, f, pair_of(0.9999280571937561f, 0.9999280571937561f));
    return pair_of((uint32_t)y + ((uint32_t)n << 23), (uint32_t)(y >> 32) + ((uint32_t)(n >> 32) << 23));
}
// registers of a load from tensor memory that is waited for here: nothing that reads them moves in front of it
template <int N>
__device__ __forceinline__ void tc_ld_wait_for(uint32_t (&r)[N])
{
    tc_ld_wait();
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}
// PAGED: boxes of a page's keys; else boxes of 128 rows beside the queries
template <int D, bool PAGED>
__global__ void __launch_bounds__(MANY_THREADS, 1)
attention_many_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttnParams p)
{
    using S = ManyShape<D>;
    using Walk = AttnWalk<ManyCut>;
    extern __shared__ __align__(1024) unsigned char smem_many[];              // (no other shared memory: 227 KB are just enough)
    ManyShared& sh = *reinterpret_cast<ManyShared*>(smem_many + (2 + S::STAGES) * S::TILE_BYTES + S::STORE_BYTES);
    const uint32_t smem0 = s2u(smem_many), smem_kv = smem0 + 2 * S::TILE_BYTES;
    const uint32_t q_full = s2u(sh.q_full), s_full = s2u(sh.s_full), p_half = s2u(sh.p_half), p_full = s2u(sh.p_full), o_full = s2u(sh.o_full),
                   o_empty = s2u(sh.o_empty), kv_full = s2u(sh.kv_full), kv_empty = s2u(sh.kv_empty), unit_full = s2u(sh.unit_full), unit_empty = s2u(sh.unit_empty);
    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (smem0 & 1023u) {                                                       // (the swizzle counts on it; so does every tile's address)
        if (threadIdx.x == 0) atomicExch(p.status, 50);
        return;
    }
    if (threadIdx.x == 0) {
        sh.abort = 0;
        for (int t = 0; t < 2; ++t) {
            bar_init(s2u(&sh.turn[t]), 1);
            bar_init(q_full + 8 * t, 256);
            bar_init(s_full + 8 * t, 1);
            bar_init(p_half + 8 * t, 256);
            bar_init(p_full + 8 * t, 256);
            bar_init(o_full + 8 * t, 1);
            bar_init(o_empty + 8 * t, 256);
        }
        for (int s = 0; s < S::STAGES; ++s) {
            bar_init(kv_full + 8 * s, 1);
            bar_init(kv_empty + 8 * s, 2);
        }
        for (int i = 0; i < 16; ++i) bar_init(s2u(&sh.told[i]), 1);
        for (int i = 0; i < 8; ++i) bar_init(s2u(&sh.pair[i]), 2);
        for (int i = 0; i < 2; ++i) bar_init(s2u(&sh.team[i]), 8);
        for (int i = 0; i < MANY_UNITS; ++i) {
            bar_init(unit_full + 8 * i, 1);
            bar_init(unit_empty + 8 * i, 19);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s2u(&sh.tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = (uint32_t)uniform((int)sh.tmem);
    start_beside();
    const AttnTotals totals = attn_totals<ManyCut>(p, sh.totals);
    // the units, for the warps that are told of them: the next one, or false behind the last
    int unit_at = 0;
    uint32_t unit_phase = 0;
    auto next_unit = [&](ManyUnit& u) {
        attn_spin(unit_full + 8 * unit_at, unit_phase, &sh.abort, p.status, 62);
        if (sh.abort) return false;
        u = sh.units[unit_at];
        __syncwarp();
        if (lane == 0) bar_arrive(unit_empty + 8 * unit_at);
        if (++unit_at == MANY_UNITS) { unit_at = 0; unit_phase ^= 1u; }
        return u.there != 0;
    };
    ManyUnit u;

    if (warp >= 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(MANY_REGS_REST));
        if (warp < 18) {
            // ---- MMA issue of tile t
            const int t = warp - 16;
            constexpr uint32_t idesc_s = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 3) << 17) | ((128u >> 4) << 24);             // bf16 x bf16 -> f32, both K-major
            constexpr uint32_t idesc_o = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((128u >> 4) << 24);      // V: rows along K
            const uint32_t ts = tmem + 128 * t, to = tmem + 256 + 128 * t, mine = 8 * t;
            const uint64_t a = smem_desc_sw128(smem0 + t * S::TILE_BYTES);
            int s = 0;
            uint32_t kv_phase = 0, q_phase = 0, p_phase = 0, oe_phase = 1, turn_phase = 1 - t;
            // The tiles take turns at the end of a product and the next scores: else their softmaxes fall into step, contend for the exponentials at one
            // time and for the tensor core at the other (4200 cycles per 128 keys)
            const uint32_t my_turn = s2u(&sh.turn[t ^ 1]), turn_over = s2u(&sh.turn[t]);
            auto advance = [&] { if (++s == S::STAGES) { s = 0; kv_phase ^= 1u; } };
            while (next_unit(u)) {
                const int first = u.first, end = u.end, e = t ? u.ends[1] : u.ends[0], keys = u.keys;
                if (first < e) {
                    attn_spin(q_full + mine, q_phase, &sh.abort, p.status, 51);
                    q_phase ^= 1u;
                }
                // j: the keys whose scores are made; in front of them the product with the values of those before
                for (int j = first; j <= end; ++j) {
                    int v = 0, k0 = 0;
                    if (j > first) {
                        v = uniform(s);
                        attn_spin(kv_full + 8 * v, kv_phase, &sh.abort, p.status, 53);
                        advance();
                        const int from = max(keys - (j - 1) * MANY_TILE, 0);
                        if (from < MANY_TILE) {
                            // values behind the last key may be anything, and 0 * NaN is not 0 (both tiles' warps write the same zeros)
                            const int rows = MANY_TILE - from;
                            for (int i = lane; i < rows * 8 * S::HALVES; i += 32) {
                                const int h = i >= rows * 8 ? 1 : 0, at = i - h * rows * 8;
                                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(smem_kv + v * S::TILE_BYTES + h * S::HALF_BYTES + from * 128 + at * 16), "r"(0) : "memory");
                            }
                            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                            __syncwarp();
                        }
                    }
                    // (the next keys are waited for here, and not between the product and the scores)
                    if (j < end) {
                        k0 = uniform(s);
                        attn_spin(kv_full + 8 * k0, kv_phase, &sh.abort, p.status, 56);
                        advance();
                    }
                    const uint64_t bv = smem_desc_sw128_mn(smem_kv + v * S::TILE_BYTES), bk = smem_desc_sw128(smem_kv + k0 * S::TILE_BYTES);
                    const bool multiply = j > first && j <= e;
                    // (the first 32 keys of each team, then the others)
                    auto product = [&](int part) {
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const int k = (q >> 1) * 4 + 2 * part + (q & 1);
                            tc_mma_f16_ts(to, ts + 8 * k, bv + (uint64_t)((k * 16 * 128) >> 4), idesc_o, part || q || j > first + 1 ? 1u : 0u);
                        }
                    };
                    if (multiply) {
                        if (j == first + 1) {
                            attn_spin(o_empty + mine, oe_phase, &sh.abort, p.status, 54);
                            oe_phase ^= 1u;
                        }
                        attn_spin(p_half + mine, p_phase, &sh.abort, p.status, 61);
                        tc_fence_after();
                        if (elect_one()) product(0);
                        __syncwarp();
                        attn_spin(p_full + mine, p_phase, &sh.abort, p.status, 55);
                        p_phase ^= 1u;
                    }
                    attn_spin(my_turn, turn_phase, &sh.abort, p.status, 66);
                    turn_phase ^= 1u;
                    tc_fence_after();
                    if (elect_one()) {
                        if (multiply) {
                            product(1);
                            if (j == e) tc_commit(o_full + mine);
                        }
                        if (j < e) {
#pragma unroll
                            for (int k = 0; k < D / 16; ++k) {
                                const uint64_t off = (uint64_t)(((k >> 2) * S::HALF_BYTES + (k & 3) * 32) >> 4);
                                tc_mma_f16_ss(ts, a + off, bk + off, idesc_s, k ? 1u : 0u);
                            }
                            tc_commit(s_full + mine);
                        }
                        bar_arrive(turn_over);
                        if (j > first) tc_commit(kv_empty + 8 * v);
                        if (j < end) tc_commit(kv_empty + 8 * k0);
                    }
                    __syncwarp();
                }
            }
        } else if (warp == 18) {
            // ---- keys and values: a lane per box and half
            int s = 0;
            uint32_t phase = 1;
            const int shift = PAGED ? min(p.page_shift, 7) : 7, boxes = MANY_TILE >> shift;
            const int h = lane % S::HALVES, box = lane / S::HALVES;
            const uint32_t box_bytes = 128u << shift;                          // of one half
            while (next_unit(u)) {
                // (a tile's pages are looked up while the one before waits for its room)
                const int32_t* row = PAGED ? p.table + u.request * p.width : nullptr;
                auto page_of = [&](int j) {
                    const int key = j * MANY_TILE + (box << shift);
                    if (box >= boxes || j >= u.end || key >= u.keys) return -1;
                    if (!PAGED) return 0;
                    const int page = row[key >> p.page_shift];
                    return page < 0 || page >= p.pages ? (int)p.pages : page;  // (beyond the cache: zeros)
                };
                int page = page_of(u.first);
                for (int j = u.first; j < u.end; ++j) {
                    const int key = j * MANY_TILE + (box << shift), next = page_of(j + 1);
                    const int there = (max(min(u.keys - j * MANY_TILE, MANY_TILE), 0) + (1 << shift) - 1) >> shift;
#pragma unroll
                    for (int what = 0; what < 2; ++what) {
                        attn_wait(kv_empty + 8 * s, phase, &sh.abort, p.status, 57);
                        if (lane == 0) bar_expect_tx(kv_full + 8 * s, there * S::HALVES * box_bytes);
                        __syncwarp();
                        if (page >= 0) {
                            const uint32_t dst = smem_kv + s * S::TILE_BYTES + h * S::HALF_BYTES + box * box_bytes;
                            const CUtensorMap* map = what ? &map_v : &map_k;
                            if (PAGED) tma_load_4d(dst, map, 0, key & ((1 << p.page_shift) - 1), h, page * p.kv_heads + u.head, kv_full + 8 * s);
                            else tma_load_4d(dst, map, 0, u.first_row + key, h, u.head, kv_full + 8 * s);
                        }
                        __syncwarp();
                        if (++s == S::STAGES) { s = 0; phase ^= 1u; }
                    }
                    page = next;
                }
            }
        } else {
            // ---- the units
            Walk w;
            uint32_t phase = 1;
            int at = 0;
            bool there = w.begin(p, totals, sh.totals);
            do {
                while (there && !w.more(totals)) there = w.next_run(p, totals, sh.totals);
                attn_wait(unit_empty + 8 * at, phase, &sh.abort, p.status, 63);
                if (lane == 0) {
                    ManyUnit n = {};
                    n.there = there;
                    if (there) {
                        n.first = w.first(totals); n.end = w.end(totals);
                        n.keys = w.r.keys; n.new_rows = w.r.rows; n.first_row = w.r.first;
                        n.row0 = w.block * MANY_ROWS; n.rows = attn_block_rows(w.r, p.group.d, w.block, MANY_ROWS);
                        n.head = w.head; n.request = w.request;
                        n.cut = w.cut(totals); n.run = w.run;
                        if (n.cut) { n.opener = w.opener(totals); n.closer = w.closer(totals); }
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            const int rows = min(n.rows - 128 * t, 128);
                            n.ends[t] = rows <= 0 ? 0 : min(n.end, attn_tiles(attn_seen(w.r, p.group.of(n.row0 + 128 * t + rows - 1)), MANY_TILE));
                        }
                    }
                    sh.units[at] = n;
                    bar_arrive(unit_full + 8 * at);
                }
                __syncwarp();
                if (++at == MANY_UNITS) { at = 0; phase ^= 1u; }
                if (there) w.step(p, totals);
                else break;
            } while (!sh.abort);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(MANY_REGS_WORK));
        // ---- a thread per row and half of a tile's keys (and, at the end, half of the columns of O); a warp reaches the lanes 32 (warp % 4) ..
        const int t = warp >> 3, half = (warp >> 2) & 1, quarter = warp & 3, row = quarter * 32 + lane;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        const uint32_t ts = tmem + lanes + 128 * t, to = tmem + lanes + 256 + 128 * t + half * (D / 2);
        uint32_t phases = 0;                                                   // of s_full, o_full, told, team and pair: a bit each (every register counts here)
        // This warp's 2 KB, and those of the warp with the other half: a row's maximum or sum there (a float per lane) while a unit is worked on, at its
        // end rows on their way out.
        unsigned char* room = smem_many + (2 + S::STAGES) * S::TILE_BYTES + warp * 2048;
        float *tell = reinterpret_cast<float*>(room) + lane, *told = reinterpret_cast<float*>(room + (half ? -4 : 4) * 2048) + lane;
        // the larger of this thread's and the other half's
        auto say = [&](float v) {
            *tell = v;
            __syncwarp();
            if (lane == 0) bar_arrive(s2u(&sh.told[warp]));
        };
        auto hear = [&] {
            attn_spin(s2u(&sh.told[warp ^ 4]), phases >> 2 & 1u, &sh.abort, p.status, 65);
            phases ^= 4u;
            return *told;
        };
        // Warps meet (the two with these rows; the tile's eight) at barriers that give up, and not at bar.sync: a warp that has given up goes to its end.
        auto meet = [&](uint64_t* bar, uint32_t bit, int code) {
            __syncwarp();
            if (lane == 0) bar_arrive(s2u(bar));
            attn_spin(s2u(bar), phases >> bit & 1u, &sh.abort, p.status, code);
            phases ^= 1u << bit;
        };
        auto hide = [](uint32_t (&x)[32], int from) {                          // scores of keys that the row does not see
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (i >= from) x[i] = 0xFF800000u;
        };
        // The next unit's rows of Q into the swizzled tile, 16 bytes at a time: chunk c of every sixteenth (or thirty-second) row; token and head of the
        // row go on with it.  The tile is free: this thread has seen the last S that was made of it.  True where q_there has to follow.
        auto fetch_q = [&] {
            attn_spin(unit_full + 8 * unit_at, unit_phase, &sh.abort, p.status, 64);
            if (sh.abort) return false;
            const ManyUnit& n = sh.units[unit_at];
            if (!n.there || n.first >= n.ends[t]) return false;
            const int rows = n.rows - 128 * t, group = p.group.d;
            constexpr int CH = D / 8, STEP = 256 / CH;
            const int c = threadIdx.x % CH, r0 = (threadIdx.x & 255) / CH;
            const int tok_step = p.group.of(STEP), head_step = STEP - tok_step * group;
            int tok = p.group.of(n.row0 + 128 * t + r0), head = n.row0 + 128 * t + r0 - tok * group;
            const __nv_bfloat16* base = p.q + (int64_t)n.first_row * p.q_stride + (int64_t)n.head * group * D + c * 8;
#pragma unroll
            for (int r = r0; r < 128; r += STEP) {
                const __nv_bfloat16* src = base + (r < rows ? tok * p.q_stride + head * D : 0);
                const uint32_t dst = smem0 + t * S::TILE_BYTES + (c >> 3) * S::HALF_BYTES + r * 128 + (((c & 7) ^ (r & 7)) << 4);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(r < rows ? 16 : 0) : "memory");
                tok += tok_step;
                head += head_step;
                if (head >= group) { head -= group; ++tok; }
            }
            return true;
        };
        auto q_there = [&] {
            asm volatile("cp.async.wait_all;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            bar_arrive(q_full + 8 * t);
        };
        if (fetch_q()) q_there();
        while (next_unit(u)) {
            const int rows = u.rows - 128 * t;
            if (rows <= 0) {
                if (fetch_q()) q_there();
                continue;
            }
            const int at = u.row0 + 128 * t + min(row, rows - 1), tok = p.group.of(at);
            const int first = u.first, end = t ? u.ends[1] : u.ends[0];
            // key from which on the row sees none, and the first row's: counted from this thread's keys of the tile
            const int origin = u.keys - u.new_rows + 1 - first * MANY_TILE - 64 * half;
            int left = origin + tok, left_all = origin + p.group.of(u.row0 + 128 * t);
            float m = -INFINITY, l = 0.f;                                      // m in units of the scores as they come; l of this half
            for (int j = first; j < end; ++j, left -= MANY_TILE, left_all -= MANY_TILE) {
                attn_spin(s_full + 8 * t, phases & 1u, &sh.abort, p.status, 59);
                phases ^= 1u;
                tc_fence_after();
                uint32_t x[2][32];
#pragma unroll
                for (int c = 0; c < 2; ++c) tc_ld32(ts + 64 * half + 32 * c, x[c]);
#pragma unroll
                for (int c = 0; c < 2; ++c) tc_ld_wait_for(x[c]);
                const bool ragged = left_all < 64;
                if (ragged) {
                    hide(x[0], left);
                    hide(x[1], left - 32);
                }
                // this thread's maximum
                auto top_of = [&] {
                    float y[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const uint32_t* z = &x[c >> 1][16 * (c & 1)];
                        y[c] = max_nan(__uint_as_float(z[0]), __uint_as_float(z[1]), __uint_as_float(z[2]));
#pragma unroll
                        for (int i = 3; i < 15; i += 2) y[c] = max_nan(y[c], __uint_as_float(z[i]), __uint_as_float(z[i + 1]));
                    }
                    return max_nan(max_nan(y[0], y[1], __uint_as_float(x[0][15])), max_nan(y[2], y[3], __uint_as_float(x[0][31])), max_nan(__uint_as_float(x[1][15]), __uint_as_float(x[1][31]), -INFINITY));
                };
                // The weights stand against the maximum in use; this tile's is found and exchanged beside them, and only then is it looked at whether they are
                // right (the first tile of a unit has none to begin with).  (The other team's reading of the last one is behind its arrival at p_full, which this
                // S waited for.)
                if (j == first) {
                    const float top = top_of();
                    say(top);
                    m = max_nan(top, hear(), -INFINITY);
                    if (m == INFINITY) m = NAN;                                // (what inf - inf would make of the row)
                }
                float sum[2];
                // group g: sixteen of a block's 32 keys
                auto weights = [&](const uint32_t (&x)[32], uint32_t (&w)[16], int g, auto with_powers) {
                    constexpr bool POWERS = decltype(with_powers)::value;
                    const float base = m == -INFINITY ? 0.f : m * p.scale_log2;
                    const uint64_t scale2 = pair_of(p.scale_log2, p.scale_log2), base2 = pair_of(-base, -base);
#pragma unroll
                    for (int i = 8 * g; i < 8 * g + 8; ++i) {
                        const uint64_t a = fma2(pair_of(x[2 * i], x[2 * i + 1]), scale2, base2);
                        float e0, e1;
                        if (POWERS && i % MANY_POWERS == MANY_POWERS - 1) {
                            const uint64_t e = power2(a);
                            e0 = __uint_as_float((uint32_t)e);
                            e1 = __uint_as_float((uint32_t)(e >> 32));
                        } else {
                            e0 = ex2(__uint_as_float((uint32_t)a));
                            e1 = ex2(__uint_as_float((uint32_t)(a >> 32)));
                        }
                        // bf16 is what the tensor cores take beside bf16 values; the sums keep the weights as they were
                        sum[0] += e0;
                        sum[1] += e1;
                        w[i] = pack_bf16(e0, e1);
                    }
                };
                auto hand_over = [&](uint32_t bar) {
                    tc_st_wait();
                    tc_fence_before();
                    bar_arrive(bar + 8 * t);
                };
                // What is waited for (the other team's maximum, stores into tensor memory) has a group of weights in front of it
                auto all_weights = [&](auto with_powers) {
                    uint32_t w[16];
                    sum[0] = sum[1] = 0.f;
                    weights(x[0], w, 0, with_powers);
                    float top = 0.f;
                    if (j > first) {
                        top = top_of();
                        say(top);
                    }
                    weights(x[0], w, 1, with_powers);
                    if (j > first) {
                        top = max_nan(top, hear(), -INFINITY);
                        if (top == INFINITY) top = NAN;
                        if (__any_sync(~0u, !((top - m) * p.scale_log2 <= MANY_LATE))) {
                            // the maximum moves (this S came behind the last product into O), and the weights are made once more: the scores are still there
                            const float m2 = max_nan(m, top, top), f = m2 == -INFINITY ? 1.f : ex2((m - m2) * p.scale_log2);
                            m = m2;
                            l *= f;
#pragma unroll 1
                            for (int c = 0; c < D / 2; c += 16) {
                                uint32_t o[16];
                                tc_ld16(to + c, o);
                                tc_ld_wait_for(o);
#pragma unroll
                                for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                                tc_st16(to + c, o);
                            }
                            tc_ld32(ts + 64 * half, x[0]);
                            tc_ld_wait_for(x[0]);
                            if (ragged) hide(x[0], left);
                            sum[0] = sum[1] = 0.f;
                            weights(x[0], w, 0, std::false_type{});
                            weights(x[0], w, 1, std::false_type{});
                        }
                    }
                    tc_st16(ts + 32 * half, w);
                    weights(x[1], w, 0, with_powers);
                    hand_over(p_half);
                    weights(x[1], w, 1, with_powers);
                    tc_st16(ts + 32 * half + 16, w);
                    hand_over(p_full);
                };
                if (ragged) all_weights(std::false_type{});
                else all_weights(std::true_type{});
                l += sum[0] + sum[1];
            }
            // ---- the unit's end: O, unscaled, and the sums of both halves
            const bool some = first < end, fetched = fetch_q();
            // Rows leave through shared memory, 64 bytes of each of the warp's rows at a time (16-byte chunks, their order turned so that neither side meets a bank
            // twice): four lanes store 64 bytes of a row.  Where they go is found while the last product runs.
            const int size = p.out_f32 ? 4 : 2;
            char* to_row[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int q = quarter * 32 + 8 * i + (lane >> 2), to = u.row0 + 128 * t + min(q, rows - 1), token = p.group.of(to);
                const int64_t place = (int64_t)(u.first_row + token) * p.q_heads + (u.head - token) * (int)p.group.d + to;
                to_row[i] = q < rows ? static_cast<char*>(p.out) + (place * D + half * (D / 2)) * size + (lane & 3) * 16 : nullptr;
            }
            auto send = [&](int c, const uint32_t (&w)[16]) {                  // from column c of this thread's half on
                const uint32_t mine = s2u(room) + lane * 64, theirs = s2u(room) + (lane >> 2) * 64;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(mine + ((i ^ ((lane >> 1) & 3)) << 4)), "r"(w[4 * i]), "r"(w[4 * i + 1]), "r"(w[4 * i + 2]), "r"(w[4 * i + 3]) : "memory");
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint4 v;
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(theirs + i * 512 + (((lane & 3) ^ ((lane >> 3) & 3)) << 4)) : "memory");
                    if (to_row[i]) *reinterpret_cast<uint4*>(to_row[i] + c * size) = v;
                }
                __syncwarp();
            };
            auto send32 = [&](int c, const uint32_t (&o)[32], float f) {       // 32 columns, times f
                uint32_t w[16];
                if (p.out_f32) {
#pragma unroll
                    for (int h = 0; h < 32; h += 16) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(__uint_as_float(o[h + i]) * f);
                        send(c + h, w);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) w[i] = pack_bf16(__uint_as_float(o[2 * i]) * f, __uint_as_float(o[2 * i + 1]) * f);
                    send(c, w);
                }
            };
            if (some) {
                attn_spin(o_full + 8 * t, phases >> 1 & 1u, &sh.abort, p.status, 60);
                phases ^= 2u;
                tc_fence_after();
            }
            if (fetched) q_there();
            say(l);                                                            // (behind o_full, so behind the other team's last reading, too)
            l += hear();
            meet(&sh.pair[4 * t + quarter], 4, 67);                             // (both have read: rows go there now)
            const bool cut = u.cut;
            const int opener = u.opener, closer = u.closer;
            // a piece: [column / 4][row][4], so that a warp's threads lie beside each other; then maxima, sums
            const int mine = 128 * t + row, col4 = half * (D / 8);
            auto slot = [&](int r) { return p.partial + (int64_t)(2 * r + (r == opener ? 1 : 0)) * S::PIECE; };
            if (some) {
                const float scale = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
                for (int c = 0; c < D / 2; c += 32) {
                    uint32_t o[32];
                    tc_ld32(to + c, o);
                    tc_ld_wait_for(o);
                    if (!cut) send32(c, o, scale);
                    else {
                        uint4* to4 = reinterpret_cast<uint4*>(slot(u.run)) + (col4 + (c >> 2)) * MANY_ROWS + mine;
#pragma unroll
                        for (int i = 0; i < 8; ++i) to4[i * MANY_ROWS] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                    }
                }
                tc_fence_before();
                bar_arrive(o_empty + 8 * t);
            }
            if (cut) {
                if (half == 0) {
                    float* head = slot(u.run) + MANY_ROWS * D;
                    head[mine] = m == -INFINITY ? m : m * p.scale_log2;
                    head[MANY_ROWS + mine] = l;
                }
                meet(&sh.team[t], 3, 68);
                if ((threadIdx.x & 255) == 0) {
                    const uint32_t before = attn_arrive(p.arrived + 2 * opener + t);
                    sh.last[t] = before == (uint32_t)(closer - opener);
                    if (sh.last[t]) p.arrived[2 * opener + t] = 0;
                }
                meet(&sh.team[t], 3, 69);
                if (sh.last[t]) {
                    // the pieces in order, rescaled when a larger maximum comes; 32 columns at a time
                    float sum = 0.f;
#pragma unroll 1
                    for (int c = 0; c < D / 2; c += 32) {
                        float v[32], top = -INFINITY;
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = 0.f;
                        sum = 0.f;
                        for (int r = opener; r <= closer; ++r) {
                            const float* head = slot(r) + MANY_ROWS * D + mine;
                            const float4* from = reinterpret_cast<const float4*>(slot(r)) + (col4 + (c >> 2)) * MANY_ROWS + mine;
                            float4 a[8];
                            const float mm = load_l2(head), ll = load_l2(head + MANY_ROWS);
#pragma unroll
                            for (int i = 0; i < 8; ++i) a[i] = load_l2(from + i * MANY_ROWS);
                            if (mm == -INFINITY) continue;                     // (nothing of this piece is seen: its o need not be there)
                            const float both = max_nan(top, mm, mm), f = top == -INFINITY ? 0.f : ex2(top - both), g = ex2(mm - both);
                            top = both;
                            sum = fmaf(sum, f, ll * g);
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                float* w = &v[4 * i];
                                w[0] = fmaf(a[i].x, g, w[0] * f); w[1] = fmaf(a[i].y, g, w[1] * f); w[2] = fmaf(a[i].z, g, w[2] * f); w[3] = fmaf(a[i].w, g, w[3] * f);
                            }
                        }
                        uint32_t o[32];
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(v[i]);
                        send32(c, o, sum == 0.f ? 0.f : 1.f / sum);
                    }
                }
                meet(&sh.team[t], 3, 70);                                         // (sh.last is the next unit's then)
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    settle_after_timeout(sh.abort);
    if (warp == 16) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

}  // namespace mpq
