// Attention of the tokens of several requests over their own keys and values:
//
//   o[i] = sum_j p[i][j] v[j] / sum_j p[i][j],   p[i][j] = exp(scale * q[i].k[j] - max_j),   over the keys j <= lens - new + i
//
// of its request (lens keys, the last `new` of them the request's own new tokens).  Query head h reads head h / (q heads / kv heads) of
// the keys.  A row that sees no key is zero.
//
// One pass over the keys with the running maximum and sum of each row; a unit whose keys are shared by several CTAs (attention_plan.h)
// leaves (maximum, sum, unscaled o) of each piece in scratch, and the CTA that is last to arrive adds them in the order of the keys: no waiting, and the
// same bits whoever is last.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "attention_plan.h"
#include "norm.cuh"
#include "nvfp4_ptx.cuh"
#include "settle.cuh"

namespace mpq {

// keys and values: pages of a cache, or rows beside the queries
struct AttnParams {
    const __nv_bfloat16* q;
    int64_t q_stride;                       // elements between tokens
    const int32_t *starts, *lens, *table;   // lens, table: null without a cache
    int64_t width;                          // entries of a table row
    int64_t pages;
    int page_shift;
    int64_t tokens;
    int n, q_heads, kv_heads;
    AttnDivisor group;
    float scale_log2;                       // scale / ln 2: the weights are powers of two
    void* out;
    int out_f32;
    float* partial;                         // pieces of cut units; null: units stay whole
    uint32_t* arrived;                      // per CTA: pieces of the unit that it opened
    int* status;
};

constexpr uint32_t ATTN_TRIES = 1u << 17;   // of a suspended wait (up to 4 us each)

__device__ __forceinline__ AttnRequest attn_request(const AttnParams& p, int i)
{
    return attn_request(p.starts[i], p.starts[i + 1], p.tokens, p.lens != nullptr, p.lens ? p.lens[i] : 0, p.width << p.page_shift);
}

// a CTA's place in the order of all tiles
struct AttnPlace {
    int64_t total, unit;                    // all tiles; first tile of the unit
    int block, request, head;
};

// How a kernel cuts its work: rows of a block, keys of a tile, what a unit costs beside its tiles, and whether a warp (of WARPS) adds up
// a request's blocks (many of them), while there are few requests
template <int ROWS_, int TILE_, int EXTRA_, int WARPS_>
struct AttnCut {
    static constexpr int ROWS = ROWS_, TILE = TILE_, EXTRA = EXTRA_, WARPS = WARPS_;
};
template <class Cut>
__device__ __forceinline__ int attn_unit_cost(const AttnParams& p, const AttnRequest& r, int b, bool whole)
{
    return whole ? 1 : attn_block_tiles(r, p.group, b, Cut::ROWS, Cut::TILE) + Cut::EXTRA;
}

struct AttnShared {
    long long sums[32], total, before;
    AttnPlace place;
    int request;
};
// Where the CTA's run begins: every CTA adds up all requests.  By all threads, with barriers in it; `room` is shared memory of 4 bytes per thread.
template <class Cut>
__device__ __forceinline__ AttnPlace attn_locate(const AttnParams& p, bool whole, AttnShared& sh, uint32_t* room)
{
    const int threads = blockDim.x, warps = threads >> 5, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool by_warps = Cut::WARPS && p.n <= threads;
    const int per = (p.n + threads - 1) / threads, i0 = min(p.n, (int)threadIdx.x * per), i1 = min(p.n, i0 + per);
    long long mine = 0;
    if (by_warps) {
        // the warp's requests, a lane each, then one after the other with a lane per block
        AttnRequest all = {};
        if (warp + warps * lane < p.n) all = attn_request(p, warp + warps * lane);
        for (int k = 0; warp + warps * k < p.n; ++k) {
            AttnRequest r;
            r.first = __shfl_sync(~0u, all.first, k); r.rows = __shfl_sync(~0u, all.rows, k); r.keys = __shfl_sync(~0u, all.keys, k);
            const int blocks = attn_blocks(r, p.group.d, Cut::ROWS);
            uint32_t sum = 0;
            for (int b = lane; b < blocks; b += 32) sum += attn_unit_cost<Cut>(p, r, b, whole);
            sum = __reduce_add_sync(~0u, sum);
            if (lane == 0) room[warp + warps * k] = sum;
        }
        __syncthreads();
        if ((int)threadIdx.x < p.n) mine = room[threadIdx.x];
    } else {
        for (int i = i0; i < i1; ++i) {
            const AttnRequest r = attn_request(p, i);
            const int blocks = attn_blocks(r, p.group.d, Cut::ROWS);
            for (int b = 0; b < blocks; ++b) mine += attn_unit_cost<Cut>(p, r, b, whole);
        }
    }
    mine *= p.kv_heads;
    long long run = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(~0u, run, o);
        if (lane >= o) run += up;
    }
    if (lane == 31) sh.sums[warp] = run;
    if (threadIdx.x == 0) sh.request = -1;
    __syncthreads();
    long long before = run - mine, total = 0;
    for (int w = 0; w < warps; ++w) {
        if (w < warp) before += sh.sums[w];
        total += sh.sums[w];
    }
    if (threadIdx.x == 0) sh.total = total;
    const int64_t ctas = min((int64_t)gridDim.x, (int64_t)total), lo = blockIdx.x < ctas ? attn_run(blockIdx.x, total, ctas) : total;
    if (mine && before <= lo && lo < before + mine) {
        if (by_warps) {
            sh.request = threadIdx.x;
            sh.before = before;
        } else {
            int64_t at = before;
            for (int i = i0; i < i1; ++i) {
                const AttnRequest r = attn_request(p, i);
                const int blocks = attn_blocks(r, p.group.d, Cut::ROWS);
                for (int b = 0; b < blocks; ++b) {
                    const int cost = attn_unit_cost<Cut>(p, r, b, whole);
                    const int64_t all = (int64_t)cost * p.kv_heads;
                    if (lo < at + all) {
                        const int head = (int)(lo - at) / cost;
                        sh.place = AttnPlace{0, at + (int64_t)head * cost, b, i, head};
                        b = blocks;
                        i = i1;
                    }
                    at += all;
                }
            }
        }
    }
    __syncthreads();
    if (by_warps && sh.request >= 0 && warp == 0) {
        const AttnRequest r = attn_request(p, sh.request);
        const int blocks = attn_blocks(r, p.group.d, Cut::ROWS);
        long long at = sh.before;
        for (int b0 = 0; b0 < blocks; b0 += 32) {
            const int cost = b0 + lane < blocks ? attn_unit_cost<Cut>(p, r, b0 + lane, whole) : 0;
            long long sum = (long long)cost * p.kv_heads;
            const long long own = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long up = __shfl_up_sync(~0u, sum, o);
                if (lane >= o) sum += up;
            }
            const long long from = at + sum - own;
            if (own && from <= lo && lo < from + own) {
                const int head = (int)(lo - from) / cost;
                sh.place = AttnPlace{0, from + (long long)head * cost, b0 + lane, sh.request, head};
            }
            at += __shfl_sync(~0u, sum, 31);
            if (at > lo) break;
        }
    }
    __syncthreads();
    AttnPlace place = sh.place;
    place.total = sh.total;
    return place;
}

// The units of a CTA's run, one after the other.  The next request's lengths are fetched when this one's are first used.
template <class Cut>
struct AttnWalk {
    AttnRequest r, next;
    int64_t lo, hi, unit, total;
    int block, blocks, request, head, tiles, ctas;
    bool whole;

    __device__ __forceinline__ void fetch(const AttnParams& p, int i)
    {
        if (i < p.n) next = attn_request(p, i);
    }
    __device__ __forceinline__ void enter(const AttnParams& p)
    {
        r = next;
        blocks = attn_blocks(r, p.group.d, Cut::ROWS);
        fetch(p, request + 1);
    }
    __device__ __forceinline__ void size(const AttnParams& p) { tiles = attn_block_tiles(r, p.group, block, Cut::ROWS, Cut::TILE); }

    __device__ __forceinline__ void begin(const AttnParams& p, const AttnPlace& at, bool whole_units)
    {
        whole = whole_units;
        total = at.total;
        ctas = (int)min((int64_t)gridDim.x, total);
        lo = (int)blockIdx.x < ctas ? attn_run(blockIdx.x, total, ctas) : total;
        hi = (int)blockIdx.x < ctas ? attn_run(blockIdx.x + 1, total, ctas) : total;
        unit = hi;
        if (lo >= hi) return;
        unit = at.unit; block = at.block; request = at.request; head = at.head;
        fetch(p, request);
        enter(p);
        size(p);
        if (!whole && lo >= unit + tiles) step(p);             // (what is left of the unit is what it costs beside its tiles)
    }
    __device__ __forceinline__ bool more() const { return unit < hi; }
    __device__ __forceinline__ int cost() const { return whole ? 1 : tiles + Cut::EXTRA; }
    // tiles of the unit that are this CTA's: [first, end)
    __device__ __forceinline__ int first() const { return whole || lo <= unit ? 0 : (int)(lo - unit); }
    __device__ __forceinline__ int end() const { return whole || unit + tiles <= hi ? tiles : (int)(hi - unit); }
    __device__ __forceinline__ void step(const AttnParams& p)
    {
        unit += cost();
        if (++head < p.kv_heads || unit >= hi) return;
        head = 0;
        if (++block >= blocks) {
            block = 0;
            do {
                ++request;
                enter(p);
            } while (!blocks);                                 // (there is one: unit < hi)
        }
        size(p);
    }
    // whether other CTAs have tiles of the unit, and the CTAs that have some
    __device__ __forceinline__ bool cut() const { return !whole && (unit < lo || unit + tiles > hi); }
    __device__ __forceinline__ int opener() const { return attn_owner(unit, total, ctas); }
    __device__ __forceinline__ int closer() const { return attn_owner(unit + tiles - 1, total, ctas); }
};

// Waits that give up: after that nothing is waited for any more, and the kernel runs to its end.  The first one is suspended, the second looks at the
// barrier all the time: what stands around a suspended wait costs 200 cycles also where the barrier has been reached, which is where most
// hand-offs of the tensor cores are.
constexpr uint32_t ATTN_LOOKS = 1u << 25;
__device__ __forceinline__ void attn_wait(uint32_t bar, uint32_t parity, volatile int* abort, int* status, int code)
{
    if (*abort) return;
    if (!bar_wait(bar, parity, ATTN_TRIES)) {
        *abort = 1;
        atomicExch(status, code);
    }
}
__device__ __forceinline__ void attn_spin(uint32_t bar, uint32_t parity, volatile int* abort, int* status, int code)
{
    for (uint32_t n = 0; !bar_test(bar, parity); ++n) {
        if ((n & 1023u) == 1023u && *abort) return;
        if (n > ATTN_LOOKS) {
            *abort = 1;
            atomicExch(status, code);
            return;
        }
    }
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int a, int b, int c, int d, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(map), "r"(a), "r"(b), "r"(c), "r"(d), "r"(bar) : "memory");
}

}  // namespace mpq
