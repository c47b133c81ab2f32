// The paged cache of keys and values: who has which pages, and the rows that go there.
//
// A cache is two bf16 arrays [pages][kv heads][page size][head dim]: the rows of one head in a page are contiguous, which is what
// an attention kernel copies.  Slot = page * page size + place in the page.  Pages that nobody has are a stack.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "norm.cuh"

namespace mpq {

// ---------------------------------------------------------------------------------------------------------------------------
// the plan of a step
// ---------------------------------------------------------------------------------------------------------------------------
// Request i had old_i tokens in its pages; new_i >= 0 follow, or it has ended (new_i < 0).  Three running sums over the requests
// say everything: pages given back, pages wanted, tokens.  The page of rank q among the wanted ones is the stack's entry
// count + given - 1 - q; where that entry is one of this step's own returns, it is read from the row of the table that returns it, so
// that no thread waits for another's store.
//
// One cluster, every CTA of which makes the sums for itself (a thread has up to PLAN_PER requests), then takes its share of
// pages and, behind a barrier, of tokens.  The lengths and the count are read before the first barrier and written behind it: they may be
// updated in place.  Bound: latency.  64 requests of a token each 4.4 us (one CTA; of it 2.3 launch and sums), 1000 requests with 29 000 tokens and
// 28 000 pages given back 14.0 (a search per token and page, and 64-bit ones: 17.2; clusters of sixteen: 14.1).
struct PlanParams {
    const int32_t *new_lens, *lens;
    int32_t *lens_out, *table, *free;
    const int32_t* count;
    int32_t *count_out, *starts, *positions;
    int64_t* slots;
    int32_t* missing;
    int n, page_shift, pages, width;
    int64_t tokens;
};

constexpr int PLAN_THREADS = 1024, PLAN_PER = 8, PLAN_MOST_N = PLAN_THREADS * PLAN_PER, PLAN_CLUSTER = 8;
constexpr int PLAN_MISSING_LONG = -1, PLAN_MISSING_TOKENS = -2;

struct PlanSums {
    long long given, need, grow;
    __device__ void add(const PlanSums& o) { given += o.given; need += o.need; grow += o.grow; }
};

struct PlanRequest {
    int old, before, grow, had, kept;
    long long need;
};

__device__ __forceinline__ PlanRequest plan_request(const PlanParams& p, int i)
{
    const int fresh = p.new_lens[i], old = max(0, min(p.lens[i], p.width << p.page_shift)), up = (1 << p.page_shift) - 1;
    PlanRequest r;
    r.old = old;
    r.had = (old + up) >> p.page_shift;
    const bool ended = fresh < 0;
    r.before = ended ? 0 : old;
    r.grow = ended ? 0 : fresh;
    r.kept = ended ? 0 : r.had;
    r.need = (((long long)r.before + r.grow + up) >> p.page_shift) - r.kept;
    return r;
}

// last index with at[index] <= v among n ascending numbers, at[0] = 0
__device__ __forceinline__ int plan_find(const int* at, int n, int v)
{
    int lo = 0;
    for (int step = 1 << (31 - __clz(n)); step; step >>= 1)
        if (lo + step < n && at[lo + step] <= v) lo += step;
    return lo;
}

__global__ void __launch_bounds__(PLAN_THREADS) kv_plan_kernel(const __grid_constant__ PlanParams p)
{
    extern __shared__ int s_req[];            // [5][n]: pages given in front, pages wanted in front, tokens in front, pages kept, tokens before the step
    __shared__ PlanSums s_warp[33];
    __shared__ int s_long;
    int *s_given = s_req, *s_need = s_req + p.n, *s_start = s_req + 2 * p.n, *s_kept = s_req + 3 * p.n, *s_before = s_req + 4 * p.n;
    start_beside();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = blockIdx.x, ranks = gridDim.x;
    if (tid == 0) s_long = 0;
    __syncthreads();
    const int per = (p.n + PLAN_THREADS - 1) / PLAN_THREADS, i0 = min(p.n, tid * per), i1 = min(p.n, i0 + per);
    const long long count = max(0, min(*p.count, p.pages));
    PlanSums mine = {0, 0, 0};
    for (int i = i0; i < i1; ++i) {
        const PlanRequest r = plan_request(p, i);
        if ((long long)r.before + r.grow > (long long)p.width << p.page_shift) s_long = 1;
        mine.add(PlanSums{r.before == 0 && p.new_lens[i] < 0 ? r.had : 0, r.need, r.grow});
    }
    PlanSums run = mine;                       // inclusive over the warp, then over the CTA
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const PlanSums up = {__shfl_up_sync(~0u, run.given, o), __shfl_up_sync(~0u, run.need, o), __shfl_up_sync(~0u, run.grow, o)};
        if (lane >= o) run.add(up);
    }
    if (lane == 31) s_warp[warp] = run;
    __syncthreads();
    if (warp == 0) {
        PlanSums w = s_warp[lane];
        const PlanSums own = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const PlanSums up = {__shfl_up_sync(~0u, w.given, o), __shfl_up_sync(~0u, w.need, o), __shfl_up_sync(~0u, w.grow, o)};
            if (lane >= o) w.add(up);
        }
        if (lane == 31) s_warp[32] = w;
        s_warp[lane] = PlanSums{w.given - own.given, w.need - own.need, w.grow - own.grow};
    }
    __syncthreads();
    const PlanSums total = s_warp[32];
    const long long held = min(count + total.given, (long long)p.pages);      // (a table that names pages twice could give back more than there are)
    int missing = (int)min(max(total.need - held, 0ll), 0x7FFFFFFFll);
    if (total.grow > p.tokens) missing = PLAN_MISSING_TOKENS;
    if (s_long) missing = PLAN_MISSING_LONG;
    const bool fits = missing == 0;
    PlanSums at = s_warp[warp];
    at.add(PlanSums{run.given - mine.given, run.need - mine.need, run.grow - mine.grow});
    for (int i = i0; i < i1; ++i) {
        const PlanRequest r = plan_request(p, i);
        const bool ended = p.new_lens[i] < 0;
        s_given[i] = (int)min(at.given, 0x7FFFFFFFll);
        s_need[i] = fits ? (int)at.need : 0;
        s_start[i] = fits ? (int)at.grow : 0;
        s_kept[i] = r.kept;
        s_before[i] = r.before;
        at.add(PlanSums{ended ? r.had : 0, r.need, r.grow});
    }
    // everything that may be updated in place has been read, by every CTA
    asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    const long long wants = fits ? total.need : 0;
    if (rank == 0) {
        long long grown = 0;
        for (int i = i0; i < i1; ++i) {
            grown = (i + 1 < p.n ? s_start[i + 1] : fits ? total.grow : 0) - s_start[i];
            p.lens_out[i] = s_before[i] + (int)grown;
            p.starts[i] = s_start[i];
        }
        if (tid == 0) {
            p.starts[p.n] = (int)(fits ? total.grow : 0);
            *p.count_out = (int)(held - wants);
            *p.missing = missing;
        }
    }
    // Numbers 0 .. end - 1 that requests have in a row from at[i] on: a thread takes one, or, with one search and a walk, four that lie a warp apart (so that a
    // warp's stores are beside each other); it looks all of them up before it stores any.
    auto each = [&](int end, const int* at, auto look, auto store) {
        const int take = end > ranks * PLAN_THREADS ? 4 : 1;
        for (long long w0 = (long long)(rank * (PLAN_THREADS / 32) + warp) * 32 * take; w0 < end; w0 += ranks * PLAN_THREADS * take) {
            int who[4], v[4];
            who[0] = plan_find(at, p.n, (int)min(w0 + lane, (long long)end - 1));
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const long long g = w0 + 32 * k + lane;
                if (k < take && g < end) {
                    if (k) who[k] = who[k - 1];
                    while (who[k] + 1 < p.n && at[who[k] + 1] <= (int)g) ++who[k];
                    v[k] = look((int)g, who[k], (int)g - at[who[k]]);
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const long long g = w0 + 32 * k + lane;
                if (k < take && g < end) store((int)g, who[k], (int)g - at[who[k]], v[k]);
            }
        }
    };
    // pages given back
    each((int)(held - count), s_given, [&](int, int i, int k) { return p.table[(int64_t)i * p.width + k]; }, [&](int g, int, int, int page) { p.free[count + g] = page; });
    // pages taken: the one of rank q among them
    each((int)wants, s_need,
         [&](int q, int, int) {
             const int e = (int)held - 1 - q, back = e - (int)count;
             if (back < 0) return p.free[e];
             const int i = plan_find(s_given, p.n, back);
             return p.table[(int64_t)i * p.width + (back - s_given[i])];
         },
         [&](int, int i, int k, int page) { p.table[(int64_t)i * p.width + s_kept[i] + k] = page; });
    // the tokens' slots, from the table as it is now
    asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    const long long live = fits ? total.grow : 0;
    each((int)live, s_start, [&](int, int i, int k) { return p.table[(int64_t)i * p.width + ((s_before[i] + k) >> p.page_shift)]; },
         [&](int t, int i, int k, int page) {
             const int pos = s_before[i] + k;
             p.positions[t] = pos;
             p.slots[t] = ((long long)page << p.page_shift) + (pos & ((1 << p.page_shift) - 1));
         });
    for (long long t = live + (long long)rank * PLAN_THREADS + tid; t < p.tokens; t += (long long)ranks * PLAN_THREADS) {
        p.positions[t] = 0;
        p.slots[t] = -1;
    }
}

// ---------------------------------------------------------------------------------------------------------------------------
// rows of the QKV projection: rotary positions, q out, k and v into the cache
// ---------------------------------------------------------------------------------------------------------------------------
// A pair (a, b) of a head becomes (a cos - b sin, b cos + a sin) with the angle position * frequency.  The angle is a product in 64
// bits, reduced there to [-pi, pi] (in 32 bits position 100000 would be off by 0.004), sine and cosine are fp32.  One rounding, to bf16.
//
// A CTA has a token: 64 threads make its sines and cosines, and behind a barrier all of them load and turn its rows (the other CTAs on the SM have theirs on the way meanwhile).
// An item is 16 elements of a head that turn together: (8 + 8 a half apart, or 16 in a row).  Bound: HBM, (size of x + 2) bytes per element: 8000 bf16 rows of 80 heads of 128 55 us, 5.9 TB/s (the
// sines are a CTA's latency: with 8 warps instead of 4, and half as many tokens on an SM, 61; with 2 56; rows of 36 heads of 64 19.3, 24.1 and 17.7).
struct AppendParams {
    const void* x;
    int64_t x_stride;
    const int32_t* positions;
    const double* freq;
    const int64_t* slots;
    __nv_bfloat16 *q_out, *k_out, *v_out, *k_cache, *v_cache;
    int64_t slot_end;           // pages * page size
    int page_shift;
    int q_heads, kv_heads, head_dim, rot;
};

constexpr int APPEND_THREADS = 128, APPEND_MOST_D = 256;

template <class X, bool INTERLEAVED>
__global__ void __launch_bounds__(APPEND_THREADS) kv_append_kernel(const __grid_constant__ AppendParams p)
{
    __shared__ float s_cos[APPEND_MOST_D / 2], s_sin[APPEND_MOST_D / 2];
    start_beside();
    const int64_t t = blockIdx.x;
    const int64_t slot = p.slots ? p.slots[t] : 0;
    if (slot < 0) return;                                       // a row behind the last token of the step
    const X* x = static_cast<const X*>(p.x) + t * p.x_stride;
    const int d = p.head_dim, half = p.rot / 2, per_head = d / 16, heads = p.q_heads + 2 * p.kv_heads, items = heads * per_head;
    for (int i = threadIdx.x; i < half; i += APPEND_THREADS) {
        const double angle = (double)p.positions[t] * p.freq[i];
        const double turns = rint(angle * 0.15915494309189533577);
        const float a = (float)fma(turns, -6.283185307179586477, angle);
        float s, c;
        sincosf(a, &s, &c);
        s_cos[i] = c;
        s_sin[i] = s;
    }
    __syncthreads();
    const bool cached = p.slots && slot < p.slot_end;
    const int64_t page = slot >> p.page_shift, place = slot & ((1ll << p.page_shift) - 1);
    for (int it = threadIdx.x; it < items; it += APPEND_THREADS) {
        const int h = it / per_head, j = it - h * per_head;
        const bool turns = h < p.q_heads + p.kv_heads && 16 * j < p.rot;
        const int c0 = !INTERLEAVED && turns ? 8 * j : 16 * j, c1 = !INTERLEAVED && turns ? half + 8 * j : 16 * j + 8;
        Eight a = load_eight(x + h * d + c0), b = load_eight(x + h * d + c1);
        if (turns) {
            if (INTERLEAVED) {
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float ca = s_cos[8 * j + e / 2], sa = s_sin[8 * j + e / 2], cb = s_cos[8 * j + 4 + e / 2], sb = s_sin[8 * j + 4 + e / 2];
                    const float a0 = a.v[e], a1 = a.v[e + 1], b0 = b.v[e], b1 = b.v[e + 1];
                    a.v[e] = a0 * ca - a1 * sa; a.v[e + 1] = a1 * ca + a0 * sa;
                    b.v[e] = b0 * cb - b1 * sb; b.v[e + 1] = b1 * cb + b0 * sb;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float c = s_cos[8 * j + e], s = s_sin[8 * j + e], a0 = a.v[e], b0 = b.v[e];
                    a.v[e] = a0 * c - b0 * s;
                    b.v[e] = b0 * c + a0 * s;
                }
            }
        }
        const uint4 ua = bf16_of_eight(a), ub = bf16_of_eight(b);
        auto put = [&](__nv_bfloat16* row) {
            *reinterpret_cast<uint4*>(row + c0) = ua;
            *reinterpret_cast<uint4*>(row + c1) = ub;
        };
        if (h < p.q_heads) {
            put(p.q_out + (t * p.q_heads + h) * d);
        } else {
            const bool key = h < p.q_heads + p.kv_heads;
            const int kh = h - p.q_heads - (key ? 0 : p.kv_heads);
            __nv_bfloat16 *rows = key ? p.k_out : p.v_out, *cache = key ? p.k_cache : p.v_cache;
            if (rows) put(rows + (t * p.kv_heads + kh) * d);
            if (cached) put(cache + (((page * p.kv_heads + kh) << p.page_shift) + place) * d);
        }
    }
}

}  // namespace mpq
