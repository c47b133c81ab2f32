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
#include "context.h"
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
    float* partial;                         // pieces of cut units, two per run; null: units stay whole
    uint32_t* arrived;                      // per run: pieces of the unit that it opened
    int most_parts;                         // of attn_parts, for which there is room
    int64_t kv_bytes;                       // of a key and its value in all heads
    int* status;
};

constexpr uint32_t ATTN_TRIES = 1u << 17;   // of a suspended wait (up to 4 us each)

__device__ __forceinline__ AttnRequest attn_request(const AttnParams& p, int i)
{
    return attn_request(p.starts[i], p.starts[i + 1], p.tokens, p.lens != nullptr, p.lens ? p.lens[i] : 0, p.width << p.page_shift);
}

// How a kernel cuts its work: rows of a block, keys of a tile, what a unit costs beside its tiles, tiles that a piece has at least, whether a
// request may have many blocks, and what the pieces of a run cost
template <int ROWS_, int TILE_, int EXTRA_, int LEAST_, bool MANY_, int PIECES_>
struct AttnCut {
    static constexpr int ROWS = ROWS_, TILE = TILE_, EXTRA = EXTRA_, LEAST = LEAST_;
    static constexpr bool MANY = MANY_;
    static constexpr int PIECES = PIECES_;
};
template <class Cut>
__device__ __forceinline__ int attn_unit_cost(const AttnParams& p, const AttnRequest& r, int b, bool whole)
{
    return whole ? 1 : attn_block_tiles(r, p.group, b, Cut::ROWS, Cut::TILE) + Cut::EXTRA;
}
// What is too much stays too much: a sum of costs (each below 2^24) that is above 2^31, of lanes' shares above 2^26, goes no further, and any such call is above ATTN_MOST_TILES
__device__ __forceinline__ uint32_t attn_sum(uint32_t sum, int more, uint32_t most) { return min(sum + (uint32_t)more, most); }
// tiles of a request in one head, by a warp
template <class Cut>
__device__ __forceinline__ uint32_t attn_request_cost(const AttnParams& p, const AttnRequest& r, bool whole)
{
    const int blocks = attn_blocks(r, p.group.d, Cut::ROWS);
    uint32_t sum = 0;
    for (int b = threadIdx.x & 31; b < blocks; b += 32) sum = attn_sum(sum, attn_unit_cost<Cut>(p, r, b, whole), 1u << 26);
    return __reduce_add_sync(~0u, sum);
}

struct AttnShared {
    uint32_t cost[ATTN_ENTRIES];            // tiles of a head, of `per` requests each
    long long total[5], keys[5], units[5];  // of 32 entries each
    int most[5];                            // tiles of a unit
};
struct AttnTotals {
    int total;                              // tiles, of all heads
    int per, runs;                          // requests of an entry; runs of all CTAs
    bool whole;
};
// What there is to do: every CTA adds up all requests.  By all threads (at least ATTN_ENTRIES), with barriers in it.
template <class Cut>
__device__ __forceinline__ AttnTotals attn_totals(const AttnParams& p, AttnShared& sh)
{
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    AttnTotals t;
    t.whole = !p.partial;
    t.per = attn_per(p.n);
    long long keys = 0, units = 0;
    int most = 0;
    uint32_t cost = 0;
    const bool by_warps = Cut::MANY && t.per == 1;
    if ((int)threadIdx.x < ATTN_ENTRIES) {
        const int i0 = min(p.n, (int)threadIdx.x * t.per), i1 = min(p.n, i0 + t.per);
        for (int i = i0; i < i1; ++i) {
            const AttnRequest r = attn_request(p, i);
            keys += r.keys;
            const int blocks = attn_blocks(r, p.group.d, Cut::ROWS);
            units += blocks;
            if (Cut::MANY && blocks) most = max(most, attn_block_tiles(r, p.group, blocks - 1, Cut::ROWS, Cut::TILE));       // (its last block sees the most)
            for (int b = 0; b < blocks && !by_warps; ++b) cost = attn_sum(cost, attn_unit_cost<Cut>(p, r, b, t.whole), 1u << 31);
        }
        if (!by_warps) sh.cost[threadIdx.x] = cost;
    }
    if (by_warps) {
        // the warp's requests, a lane each, then one after the other with a lane per block
        AttnRequest all = {};
        if (warp + warps * lane < p.n) all = attn_request(p, warp + warps * lane);
        for (int k = 0; warp + warps * k < ATTN_ENTRIES; ++k) {
            AttnRequest r;
            r.first = __shfl_sync(~0u, all.first, k); r.rows = __shfl_sync(~0u, all.rows, k); r.keys = __shfl_sync(~0u, all.keys, k);
            const uint32_t sum = attn_request_cost<Cut>(p, r, t.whole);
            if (lane == 0) sh.cost[warp + warps * k] = sum;
        }
    }
    __syncthreads();
    if (warp < ATTN_ENTRIES / 32) {
        const uint32_t own = sh.cost[threadIdx.x];
        const uint32_t low = __reduce_add_sync(~0u, own & 0xFFFFu), high = __reduce_add_sync(~0u, own >> 16);
        if (p.most_parts > 1)
#pragma unroll
            for (int o = 16; o; o >>= 1) keys += __shfl_xor_sync(~0u, keys, o);
        if (Cut::MANY) {
            const uint32_t all = __reduce_add_sync(~0u, (uint32_t)min(units, 1ll << 24));          // (more than that are not whole anyway)
            const int top = __reduce_max_sync(~0u, most);
            if (lane == 0) { sh.units[warp] = all; sh.most[warp] = top; }
        }
        if (lane == 0) { sh.total[warp] = ((long long)high << 16) + low; sh.keys[warp] = keys; }
    }
    __syncthreads();
    const int ctas = gridDim.x;
    long long total = keys = 0;
#pragma unroll
    for (int w = 0; w < ATTN_ENTRIES / 32; ++w) { total += sh.total[w]; keys += sh.keys[w]; }
    total *= p.kv_heads;
    if (Cut::MANY && !t.whole) {
        // A CTA for each unit, and none is cut, where the longest one takes no longer than an equal run and its pieces (16 requests, 32 new tokens each over 1500, 32 heads on
        // 8: 29.8 us, cut 37.7; 1000 over 2000, 32 heads: 40.4, cut 46.6; a prompt of 4096 on 8 heads: 69, cut 54)
        long long all = 0;
        int top = 0;
#pragma unroll
        for (int w = 0; w < ATTN_ENTRIES / 32; ++w) { all += sh.units[w]; top = max(top, sh.most[w]); }
        all *= p.kv_heads;
        if (all <= ctas && top + Cut::EXTRA <= total / ctas + Cut::PIECES) {
            t.whole = true;
            total = all;
            if ((int)threadIdx.x < ATTN_ENTRIES) sh.cost[threadIdx.x] = (uint32_t)units;
            __syncthreads();
        }
    }
    if (total > ATTN_MOST_TILES) {
        if (threadIdx.x == 0) atomicExch(p.status, ATTN_TOO_MUCH);
        total = 0;
    }
    t.total = (int)total;
    t.runs = min(t.whole || p.most_parts == 1 ? ctas : ctas * attn_parts(t.total, ctas, keys * p.kv_bytes, p.most_parts), t.total);
    return t;
}

// The units of a run, one after the other, for a whole warp.  The next request's lengths are fetched when this one's are first used.
template <class Cut>
struct AttnWalk {
    AttnRequest r, next;
    int lo, hi, unit;
    int run, block, blocks, request, head, tiles;

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
    // to the next request with rows (there is one: the run goes on), a lane for each of 32
    __device__ __forceinline__ void skip(const AttnParams& p)
    {
        for (uint32_t some = 0; !some && ++request < p.n;) {
            const int i = request + (threadIdx.x & 31);
            some = __ballot_sync(~0u, i < p.n && attn_request(p, i).rows > 0);
            request += some ? __ffs(some) - 1 : 31;
        }
        fetch(p, request);
        enter(p);
    }
    __device__ __forceinline__ void size(const AttnParams& p) { tiles = attn_block_tiles(r, p.group, block, Cut::ROWS, Cut::TILE); }

    // a lane's `own` tiles behind all lanes in front of it and `at`: the lane with tile lo, and everything in front of it passed
    __device__ __forceinline__ bool pass(int own, int& at, int& which, int base) const
    {
        const int lane = threadIdx.x & 31;
        int sum = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(~0u, sum, o);
            if (lane >= o) sum += up;
        }
        const uint32_t behind = __ballot_sync(~0u, at + sum > lo);
        if (behind) {
            const int l = __ffs(behind) - 1;
            which = base + l;
            at += __shfl_sync(~0u, sum - own, l);
            return true;
        }
        at += __shfl_sync(~0u, sum, 31);
        return false;
    }
    // the CTA's first run, or its next: false behind the last
    __device__ __forceinline__ bool begin(const AttnParams& p, const AttnTotals& t, const AttnShared& sh) { return seek(p, t, sh, blockIdx.x); }
    __device__ __forceinline__ bool next_run(const AttnParams& p, const AttnTotals& t, const AttnShared& sh) { return seek(p, t, sh, run + gridDim.x); }
    __device__ __forceinline__ bool seek(const AttnParams& p, const AttnTotals& t, const AttnShared& sh, int which)
    {
        run = which;
        if (run >= t.runs) return false;
        lo = attn_run(run, t.total, t.runs);
        hi = attn_run(run + 1, t.total, t.runs);
        const int lane = threadIdx.x & 31;
        // the entry with tile lo, then its request, head and block; everything in front of `at` has been passed
        int at = 0, entry = 0;
        for (int e0 = 0; e0 < ATTN_ENTRIES; e0 += 32) {
            const int own = (int)sh.cost[e0 + lane] * p.kv_heads;
            if (pass(own, at, entry, e0)) break;
        }
        int cost = 0;                                            // of the request in one head
        for (request = entry * t.per;; ++request) {
            r = attn_request(p, request);
            cost = t.per == 1 ? (int)sh.cost[request] : (int)attn_request_cost<Cut>(p, r, t.whole);
            if (at + cost * p.kv_heads > lo || request + 1 >= p.n) break;
            at += cost * p.kv_heads;
        }
        fetch(p, request + 1);
        blocks = attn_blocks(r, p.group.d, Cut::ROWS);
        head = (lo - at) / cost;
        at += head * cost;
        block = 0;
        if (blocks > 1)
            for (int b0 = 0; b0 < blocks; b0 += 32) {
                const int own = b0 + lane < blocks ? attn_unit_cost<Cut>(p, r, b0 + lane, t.whole) : 0;
                if (pass(own, at, block, b0)) break;
            }
        unit = at;
        size(p);
        if (!t.whole && attn_first(lo, unit, tiles, Cut::LEAST) == tiles) step(p, t);      // (what the run has of the unit is not worth a piece, or beside its tiles)
        return true;
    }
    __device__ __forceinline__ bool more(const AttnTotals& t) const { return unit < hi && (t.whole || !attn_behind(hi, unit, tiles, Cut::LEAST)); }
    // tiles of the unit that are this run's: [first, end)
    __device__ __forceinline__ int first(const AttnTotals& t) const { return t.whole || lo <= unit ? 0 : attn_first(lo, unit, tiles, Cut::LEAST); }
    __device__ __forceinline__ int end(const AttnTotals& t) const { return t.whole ? tiles : attn_end(hi, unit, tiles, Cut::LEAST); }
    __device__ __forceinline__ void step(const AttnParams& p, const AttnTotals& t)
    {
        unit += t.whole ? 1 : tiles + Cut::EXTRA;
        if (unit >= hi) return;
        if (++block >= blocks) {
            block = 0;
            if (++head >= p.kv_heads) {
                head = 0;
                ++request;
                enter(p);
                if (!blocks) skip(p);
            }
        }
        size(p);
    }
    // whether other runs have tiles of the unit, and the runs that have some
    __device__ __forceinline__ bool cut(const AttnTotals& t) const { return first(t) > 0 || end(t) < tiles; }
    __device__ __forceinline__ int opener(const AttnTotals& t) const { return attn_opener(unit, tiles, Cut::LEAST, t.total, t.runs); }
    __device__ __forceinline__ int closer(const AttnTotals& t) const { return attn_closer(unit, tiles, Cut::LEAST, t.total, t.runs); }
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

// One more of `counter`, behind everything that the threads of this barrier's sides have stored, and in front of what they read of the others' (the thread
// that says it releases and acquires for all of them)
__device__ __forceinline__ uint32_t attn_arrive(uint32_t* counter)
{
    uint32_t before;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
    return before;
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int a, int b, int c, int d, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(map), "r"(a), "r"(b), "r"(c), "r"(d), "r"(bar) : "memory");
}

}  // namespace mpq
