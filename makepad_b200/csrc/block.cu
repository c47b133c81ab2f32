// The entry points between a decoder layer's projections: norms, the paged cache, attention.
#include <algorithm>

#include "attention.cuh"
#include "attention_few.cuh"
#include "attention_many.cuh"
#include "context.h"
#include "kv_cache.cuh"
#include "launch.h"
#include "norm.cuh"
#include "overlap.h"
#include "per_device.h"

using namespace mpq;

namespace {

// A launch that may start beside the kernel in front of it; every kernel here waits for that one before it reads.
template <class... P, class... A>
cudaError_t launch_beside(const mpq_context* ctx, void (*kernel)(P...), dim3 grid, unsigned block, size_t smem, unsigned cluster, cudaStream_t s, A... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    if (ctx->pdl) {
        at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        at[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        at[cfg.numAttrs].val.clusterDim.x = cluster;
        at[cfg.numAttrs].val.clusterDim.y = at[cfg.numAttrs].val.clusterDim.z = 1;
        ++cfg.numAttrs;
    }
    cfg.attrs = at;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

bool power_of_two(int64_t v) { return v > 0 && !(v & (v - 1)); }
int log2_of(int64_t v) { int s = 0; while ((1ll << s) < v) ++s; return s; }
bool page_ok(int64_t page_size) { return power_of_two(page_size) && page_size >= 16 && page_size <= 256; }

constexpr int64_t MOST = 0x7FFFFFFF;
constexpr int64_t MOST_KEYS = 1ll << 30;      // of a request, and rows of a call: what is added to one stays an int

}  // namespace

// ---------------------------------------------------------------------------
// norms around a block
// ---------------------------------------------------------------------------
template <class X, class Y>
static cudaError_t norm_launch(const mpq_context* ctx, const NormParams& p, int64_t M, cudaStream_t s)
{
    // Groups of eight columns per thread, and CTAs on an SM.  Two groups: 8192 bf16 rows of 4096 columns, both norms and a gate, 72 us (one group, twice the warps at their
    // barriers, 76; four 71), 500 rows 6.4 (6.8; 7.8), fp32 rows of 8192 columns 199 (203; 214).  A row of more than 4096 bf16 columns with a norm behind the block has nothing on its
    // way while its first sum is made: four groups put a third row on an SM where two groups put two, above 5120 columns, once each SM has two.  Two groups and four, us:
    // 8192 rows of 8192 columns 151 / 138, 300 rows 9.0 / 7.9, 150 rows 6.0 / 7.4; of 5632 columns 116 / 96, 8.0 / 7.0, 4.7 / 6.4.  Up to 5120 columns three rows of two groups fit as
    // well, and four groups pay only for many rows: 8192 rows of 5120 columns 93 / 89, 2000 rows 26.7 / 26.7, 700 rows 10.6 / 12.3, 300 rows 5.8 / 6.8.
    const int groups = p.H / 8, sms = ctx->prop.multiProcessorCount;
    const bool three = sizeof(X) == 2 && p.post_weight && groups > 512 && groups <= 1024 && M > (groups > 640 ? 2 : 16) * (int64_t)sms;
    const int nv = three || groups > 2048 ? 4 : 2;
    const unsigned threads = (unsigned)((groups + nv - 1) / nv + 31) / 32 * 32;
    auto kernel = groups <= 1024 ? residual_norm_kernel<512, 2, 2, X, Y> : groups <= 2048 ? residual_norm_kernel<1024, 1, 2, X, Y> : residual_norm_kernel<1024, 1, 4, X, Y>;
    if constexpr (sizeof(X) == 2)
        if (three) kernel = residual_norm_kernel<256, 3, 4, X, Y>;
    return launch_beside(ctx, kernel, dim3((unsigned)M), threads, 0, 1, s, p);
}

extern "C" int32_t mpq_residual_norm(mpq_context* ctx, const void* x_dev, int32_t x_is_bf16, int64_t M, int64_t H, const float* residual_dev,
                                     float* residual_out_dev, const float* post_weight_dev, const float* gate_dev, int64_t gate_stride, float alpha,
                                     const float* weight_dev, float eps, void* y_dev, int32_t y_is_bf16, void* stream)
{
    if (!ctx_ok(ctx)) return MPQ_ERR_INVALID_ARG;
    if (!x_dev || (!residual_out_dev && !y_dev)) return fail(ctx, MPQ_ERR_INVALID_ARG, "null pointer: x, or both outputs");
    if (M <= 0 || M > MOST || H <= 0 || H % 8) return fail(ctx, MPQ_ERR_SHAPE, "the norm needs 0 < M < 2^31 and H a positive multiple of 8 (M=%lld H=%lld)", (long long)M, (long long)H);
    if (H > NORM_MOST_H) return fail(ctx, MPQ_ERR_UNSUPPORTED, "rows of more than %d columns", NORM_MOST_H);
    if (gate_stride && (gate_stride < H || gate_stride % 4)) return fail(ctx, MPQ_ERR_SHAPE, "gate_stride is 0 or at least H, a multiple of 4");
    if (!(eps >= 0.f)) return fail(ctx, MPQ_ERR_INVALID_ARG, "eps must not be negative");
    for (const void* ptr : {x_dev, (const void*)residual_dev, (const void*)residual_out_dev, (const void*)post_weight_dev, (const void*)gate_dev, (const void*)weight_dev, (const void*)y_dev})
        if (!aligned16(ptr)) return fail(ctx, MPQ_ERR_ALIGN, "pointers must be 16-byte aligned");
    // (a row of an output may lie over other rows' input, or over columns that other threads still read)
    const int64_t row = 4 * H, all = M * row, x_bytes = M * H * (x_is_bf16 ? 2 : 4), y_bytes = M * H * (y_is_bf16 ? 2 : 4);
    auto over = [&](const void* out, int64_t bytes) {
        return overlaps(out, bytes, post_weight_dev, row) || overlaps(out, bytes, weight_dev, row) || overlaps(out, bytes, gate_dev, gate_stride ? M : 1, row, gate_stride ? (__int128)gate_stride * 4 : row);
    };
    const bool same_x = !x_is_bf16 && (const void*)residual_out_dev == x_dev;             // a thread reads its columns of x and of the residual in front of its stores
    if (over(y_dev, y_bytes) || overlaps(y_dev, y_bytes, x_dev, x_bytes) || overlaps(y_dev, y_bytes, residual_dev, all) || overlaps(y_dev, y_bytes, residual_out_dev, all) ||
        over(residual_out_dev, all) || (!same_x && overlaps(residual_out_dev, all, x_dev, x_bytes)) || (residual_out_dev != residual_dev && overlaps(residual_out_dev, all, residual_dev, all)))
        return fail(ctx, MPQ_ERR_INVALID_ARG, "outputs must not overlap, nor lie over an input (residual_out may be residual, or x)");
    const OnDevice on(ctx->device);
    CU_TRY(ctx, on.error);
    const NormParams p = {x_dev, residual_dev, residual_out_dev, post_weight_dev, gate_dev, weight_dev, y_dev, gate_stride, (int)H, alpha, eps};
    cudaStream_t s = (cudaStream_t)stream;
    ctx->launches += 1;
    if (x_is_bf16) CU_TRY(ctx, y_is_bf16 ? (norm_launch<__nv_bfloat16, __nv_bfloat16>(ctx, p, M, s)) : (norm_launch<__nv_bfloat16, float>(ctx, p, M, s)));
    else CU_TRY(ctx, y_is_bf16 ? (norm_launch<float, __nv_bfloat16>(ctx, p, M, s)) : (norm_launch<float, float>(ctx, p, M, s)));
    return MPQ_OK;
}

// ---------------------------------------------------------------------------
// the paged cache
// ---------------------------------------------------------------------------
extern "C" int32_t mpq_kv_plan(mpq_context* ctx, int64_t n, const int32_t* new_lens_dev, const int32_t* lens_dev, int32_t* lens_out_dev, int32_t* block_table_dev,
                               int64_t max_blocks, int32_t* free_dev, int64_t pages, const int32_t* free_count_dev, int32_t* free_count_out_dev, int32_t page_size,
                               int64_t tokens, int32_t* starts_dev, int32_t* positions_dev, int64_t* slots_dev, int32_t* missing_dev, void* stream)
{
    if (!ctx_ok(ctx)) return MPQ_ERR_INVALID_ARG;
    if (!new_lens_dev || !lens_dev || !lens_out_dev || !block_table_dev || !free_dev || !free_count_dev || !free_count_out_dev || !starts_dev || !missing_dev ||
        (tokens > 0 && (!positions_dev || !slots_dev)))
        return fail(ctx, MPQ_ERR_INVALID_ARG, "null pointer");
    if (n <= 0 || max_blocks <= 0 || pages <= 0 || tokens < 0 || tokens > MOST || pages > MOST) return fail(ctx, MPQ_ERR_SHAPE, "n, max_blocks and pages must be positive, tokens not negative, all below 2^31");
    if (!page_ok(page_size)) return fail(ctx, MPQ_ERR_SHAPE, "page_size must be a power of two from 16 to 256 (%d)", page_size);
    if (max_blocks > MOST_KEYS / page_size) return fail(ctx, MPQ_ERR_SHAPE, "max_blocks * page_size must be at most 2^30");
    if (n > PLAN_MOST_N) return fail(ctx, MPQ_ERR_UNSUPPORTED, "more than %d requests", PLAN_MOST_N);
    const OnDevice on(ctx->device);
    CU_TRY(ctx, on.error);
    static PerDeviceOnce raised;
    const size_t smem = 5 * sizeof(int) * (size_t)n;
    if (raised.needs(ctx->device)) {
        CU_TRY(ctx, cudaFuncSetAttribute(kv_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 5 * (int)sizeof(int) * PLAN_MOST_N));
        raised.mark(ctx->device);
    }
    const PlanParams p = {new_lens_dev, lens_dev, lens_out_dev, block_table_dev, free_dev, free_count_dev, free_count_out_dev, starts_dev, positions_dev, slots_dev, missing_dev,
                          (int)n, log2_of(page_size), (int)pages, (int)max_blocks, tokens};
    // one CTA while it has about one token and one request per thread
    const unsigned ctas = n <= PLAN_THREADS / 2 && tokens <= PLAN_THREADS ? 1 : PLAN_CLUSTER;
    ctx->launches += 1;
    CU_TRY(ctx, launch_beside(ctx, kv_plan_kernel, dim3(ctas), PLAN_THREADS, smem, ctas, (cudaStream_t)stream, p));
    return MPQ_OK;
}

extern "C" int32_t mpq_kv_append(mpq_context* ctx, const void* qkv_dev, int32_t x_is_bf16, int64_t row_stride, int64_t tokens, int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                                 const int32_t* positions_dev, const double* frequencies_dev, int32_t rot_dim, int32_t interleaved, uint16_t* q_dev, uint16_t* k_dev, uint16_t* v_dev,
                                 const int64_t* slots_dev, uint16_t* k_cache_dev, uint16_t* v_cache_dev, int64_t pages, int32_t page_size, void* stream)
{
    if (!ctx_ok(ctx)) return MPQ_ERR_INVALID_ARG;
    if (!qkv_dev || !q_dev || (rot_dim > 0 && (!positions_dev || !frequencies_dev)) || (slots_dev && (!k_cache_dev || !v_cache_dev))) return fail(ctx, MPQ_ERR_INVALID_ARG, "null pointer");
    if (tokens <= 0 || tokens > MOST || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || q_heads > 4096)
        return fail(ctx, MPQ_ERR_SHAPE, "tokens must be positive, q_heads a multiple of kv_heads, at most 4096 (tokens=%lld, %d and %d heads)", (long long)tokens, q_heads, kv_heads);
    if (head_dim <= 0 || head_dim % 16 || head_dim > APPEND_MOST_D) return fail(ctx, MPQ_ERR_SHAPE, "head_dim must be a multiple of 16 up to %d (%d)", APPEND_MOST_D, head_dim);
    if (rot_dim < 0 || rot_dim % 16 || rot_dim > head_dim) return fail(ctx, MPQ_ERR_SHAPE, "rot_dim must be a multiple of 16 up to head_dim (%d)", rot_dim);
    if (row_stride < (int64_t)(q_heads + 2 * kv_heads) * head_dim || row_stride % 8) return fail(ctx, MPQ_ERR_SHAPE, "row_stride must be a multiple of 8 and hold the heads (%lld)", (long long)row_stride);
    if (slots_dev && (!page_ok(page_size) || pages <= 0 || pages > MOST)) return fail(ctx, MPQ_ERR_SHAPE, "pages must be positive, page_size a power of two from 16 to 256 (%lld pages of %d)", (long long)pages, page_size);
    for (const void* ptr : {qkv_dev, (const void*)q_dev, (const void*)k_dev, (const void*)v_dev, (const void*)k_cache_dev, (const void*)v_cache_dev})
        if (!aligned16(ptr)) return fail(ctx, MPQ_ERR_ALIGN, "rows and caches must be 16-byte aligned");
    // (CTAs have a token each, and go in no order)
    const int64_t kv_bytes = tokens * kv_heads * head_dim * 2, cache_bytes = slots_dev ? pages * kv_heads * page_size * head_dim * 2 : 0;
    const struct { const void* at; int64_t bytes; } outs[] = {{q_dev, tokens * q_heads * head_dim * 2}, {k_dev, kv_bytes}, {v_dev, kv_bytes}, {k_cache_dev, cache_bytes}, {v_cache_dev, cache_bytes}};
    const int size = x_is_bf16 ? 2 : 4;
    for (const auto& o : outs) {
        bool over = overlaps(o.at, o.bytes, qkv_dev, tokens, (int64_t)(q_heads + 2 * kv_heads) * head_dim * size, (__int128)row_stride * size) || overlaps(o.at, o.bytes, slots_dev, tokens * 8) ||
                    (rot_dim && (overlaps(o.at, o.bytes, positions_dev, tokens * 4) || overlaps(o.at, o.bytes, frequencies_dev, rot_dim * 4)));
        for (const auto* other = &o + 1; other != outs + 5; ++other) over |= overlaps(o.at, o.bytes, other->at, other->bytes);
        if (over) return fail(ctx, MPQ_ERR_INVALID_ARG, "outputs must not overlap, nor lie over an input");
    }
    const OnDevice on(ctx->device);
    CU_TRY(ctx, on.error);
    auto bf = [](uint16_t* ptr) { return reinterpret_cast<__nv_bfloat16*>(ptr); };
    const AppendParams p = {qkv_dev, row_stride, positions_dev, frequencies_dev, slots_dev, bf(q_dev), bf(k_dev), bf(v_dev), bf(k_cache_dev), bf(v_cache_dev),
                            slots_dev ? pages * page_size : 0, slots_dev ? log2_of(page_size) : 0, q_heads, kv_heads, head_dim, rot_dim};
    auto kernel = x_is_bf16 ? (interleaved ? kv_append_kernel<__nv_bfloat16, true> : kv_append_kernel<__nv_bfloat16, false>)
                            : (interleaved ? kv_append_kernel<float, true> : kv_append_kernel<float, false>);
    ctx->launches += 1;
    CU_TRY(ctx, launch_beside(ctx, kernel, dim3((unsigned)tokens), APPEND_THREADS, 0, 1, (cudaStream_t)stream, p));
    return MPQ_OK;
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------
namespace {

// keys and values of a call: the pages of a cache, or rows
struct AttnKeys {
    const uint16_t *k, *v;
    int64_t k_stride, v_stride;      // elements between rows (without pages)
    int64_t pages;
    int page_size;
    int64_t max_new;
};

}  // namespace

// what both forms want of their arguments
static int32_t attention_check(mpq_context* ctx, const AttnParams& p, const AttnKeys& kv, int64_t n, int64_t q_heads, int64_t kv_heads, int32_t head_dim, float scale)
{
    if (!p.q || !kv.k || !kv.v || !p.starts || !p.out) return fail(ctx, MPQ_ERR_INVALID_ARG, "null pointer");
    if (p.tokens <= 0 || p.tokens > MOST_KEYS || n <= 0) return fail(ctx, MPQ_ERR_SHAPE, "tokens and n must be positive, tokens at most 2^30");
    if (n > ATTN_MOST_REQUESTS) return fail(ctx, MPQ_ERR_UNSUPPORTED, "more than %lld requests", (long long)ATTN_MOST_REQUESTS);
    if (q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || q_heads > 4096)
        return fail(ctx, MPQ_ERR_SHAPE, "q_heads must be a multiple of kv_heads, at most 4096 (%lld and %lld)", (long long)q_heads, (long long)kv_heads);
    if (p.tokens * p.group.d > MOST) return fail(ctx, MPQ_ERR_UNSUPPORTED, "tokens * q_heads / kv_heads must be below 2^31");
    if (head_dim != 64 && head_dim != 128) return fail(ctx, MPQ_ERR_SHAPE, "head_dim must be 64 or 128 (%d)", head_dim);
    if (p.q_stride < q_heads * head_dim || p.q_stride % 8) return fail(ctx, MPQ_ERR_SHAPE, "a row stride must be a multiple of 8 and hold the heads");
    if (!(scale >= 0.f) || scale - scale != 0.f) return fail(ctx, MPQ_ERR_INVALID_ARG, "scale must be finite and not negative");
    if (!aligned16(p.q) || !aligned16(kv.k) || !aligned16(kv.v) || !aligned16(p.out)) return fail(ctx, MPQ_ERR_ALIGN, "q, k, v and out must be 16-byte aligned");
    // (other CTAs still read what one has written)
    const int64_t out_bytes = p.tokens * q_heads * head_dim * (p.out_f32 ? 4 : 2);
    if (overlaps(p.out, out_bytes, p.q, p.tokens, q_heads * head_dim * 2, (__int128)p.q_stride * 2) || overlaps(p.out, out_bytes, p.starts, 4 * (n + 1)))
        return fail(ctx, MPQ_ERR_INVALID_ARG, "out must not overlap an input");
    return MPQ_OK;
}

static void attention_params(AttnParams* p, const uint16_t* q, int64_t q_stride, int64_t tokens, int64_t n, const int32_t* starts, int32_t q_heads, int32_t kv_heads, float scale, void* out,
                             int32_t out_is_f32)
{
    *p = AttnParams{};
    p->q = reinterpret_cast<const __nv_bfloat16*>(q);
    p->q_stride = q_stride;
    p->starts = starts;
    p->tokens = tokens; p->n = (int)std::min(n, MOST);
    p->q_heads = q_heads; p->kv_heads = kv_heads; p->group = attn_divisor(kv_heads > 0 && q_heads >= kv_heads ? q_heads / kv_heads : 1);
    p->scale_log2 = std::max(scale * 1.44269504088896340736f, 1e-30f);     // (0 would make NaN of the -inf that stands for a key that is not seen)
    p->out = out; p->out_f32 = out_is_f32 != 0;
}

// Room for the pieces of cut units (two per run), by the first call outside a capture that wants so much: of `parts` runs per CTA, or of one where
// there is no more.  Without any units stay whole.
static void attention_scratch(mpq_context* ctx, AttnParams* p, int ctas, size_t piece, int parts, cudaStream_t s)
{
    const size_t each = 2 * (size_t)ctas * piece * sizeof(float);
    if (ctx->attn_partial.bytes() < each * parts && !stream_captures(s) && ctx->attn_partial.reserve(each * parts) != cudaSuccess && parts > 1) ctx->attn_partial.reserve(each);
    p->most_parts = (int)std::min<size_t>(parts, ctx->attn_partial.bytes() / each);
    p->partial = p->most_parts ? ctx->attn_partial.as<float>() : nullptr;
    p->arrived = ctx->attn_arrived;
    p->status = ctx->attn_status;
}

// a cache [pages][kv heads][page size][D] as boxes of `keys` keys of a page and head, `halves` times 64 elements
static bool cache_map(CUtensorMap* map, const void* base, const AttnKeys& kv, int kv_heads, int D, int keys, int halves)
{
    const uint64_t dims[4] = {64, (uint64_t)kv.page_size, (uint64_t)D / 64, (uint64_t)kv.pages * kv_heads};
    const uint64_t strides[3] = {2ull * D, 128, 2ull * D * kv.page_size};
    const uint32_t box[4] = {64, (uint32_t)keys, (uint32_t)halves, 1};
    return make_bf16_map(map, base, 4, dims, strides, box);
}

// rows [tokens][kv heads][D], `stride` elements apart, as boxes of `keys` rows of a head, 64 elements
static bool rows_map(CUtensorMap* map, const void* base, int64_t tokens, int64_t stride, int kv_heads, int D, int keys)
{
    const uint64_t dims[4] = {64, (uint64_t)tokens, (uint64_t)D / 64, (uint64_t)kv_heads};
    const uint64_t strides[3] = {2ull * stride, 128, 2ull * D};
    const uint32_t box[4] = {64, (uint32_t)keys, 1, 1};
    return make_bf16_map(map, base, 4, dims, strides, box);
}

template <int D, int BOX, int NT>
static int32_t attention_few(mpq_context* ctx, AttnParams p, const AttnKeys& kv, cudaStream_t s)
{
    const int ctas = std::min(ctx->prop.multiProcessorCount, FEW_MOST_CTAS);
    attention_scratch(ctx, &p, ctas, FewShape<D, NT>::PIECE, 1, s);
    static PerDeviceOnce raised;
    if (raised.needs(ctx->device)) {
        CU_TRY(ctx, cudaFuncSetAttribute(attention_few_kernel<D, BOX, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, FewShape<D, NT>::SMEM));
        raised.mark(ctx->device);
    }
    CUtensorMap map_k, map_v;
    if (!cache_map(&map_k, kv.k, kv, p.kv_heads, D, BOX, D / 64) || !cache_map(&map_v, kv.v, kv, p.kv_heads, D, BOX, D / 64)) return fail(ctx, MPQ_ERR_CUDA, "cuTensorMapEncodeTiled failed for the cache");
    ctx->launches += 1;
    CU_TRY(ctx, launch_beside(ctx, attention_few_kernel<D, BOX, NT>, dim3(ctas), FEW_THREADS, FewShape<D, NT>::SMEM, 1, s, map_k, map_v, p));
    return MPQ_OK;
}

template <int D, bool PAGED>
static int32_t attention_many(mpq_context* ctx, AttnParams p, const AttnKeys& kv, cudaStream_t s)
{
    constexpr int PARTS = 4;
    static_assert(2 * PARTS * FEW_MOST_CTAS <= ATTN_COUNTERS && PARTS * FEW_MOST_CTAS <= ATTN_MOST_RUNS, "a counter per run and row tile");
    const int ctas = std::min(ctx->prop.multiProcessorCount, FEW_MOST_CTAS);
    p.kv_bytes = 4ll * p.kv_heads * D;
    const int64_t keys = PAGED ? kv.pages * kv.page_size : p.tokens;
    attention_scratch(ctx, &p, ctas, ManyShape<D>::PIECE, attn_parts((int)MOST, ctas, keys * p.kv_bytes, PARTS), s);
    static PerDeviceOnce raised;
    if (raised.needs(ctx->device)) {
        CU_TRY(ctx, cudaFuncSetAttribute(attention_many_kernel<D, PAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize, ManyShape<D>::SMEM));
        raised.mark(ctx->device);
    }
    CUtensorMap maps[2];
    for (int i = 0; i < 2; ++i) {
        const void* base = i ? kv.v : kv.k;
        const bool made = PAGED ? cache_map(&maps[i], base, kv, p.kv_heads, D, std::min(kv.page_size, MANY_TILE), 1)
                                : rows_map(&maps[i], base, p.tokens, i ? kv.v_stride : kv.k_stride, p.kv_heads, D, MANY_TILE);
        if (!made) return fail(ctx, MPQ_ERR_CUDA, "cuTensorMapEncodeTiled failed for the keys or values");
    }
    ctx->launches += 1;
    CU_TRY(ctx, launch_beside(ctx, attention_many_kernel<D, PAGED>, dim3(ctas), MANY_THREADS, ManyShape<D>::SMEM, 1, s, maps[0], maps[1], p));
    return MPQ_OK;
}

static int32_t attention_launch(mpq_context* ctx, const AttnParams& p, const AttnKeys& kv, int32_t head_dim, cudaStream_t s)
{
    const OnDevice on(ctx->device);
    CU_TRY(ctx, on.error);
    const int64_t most_new = kv.max_new > 0 ? std::min(kv.max_new, p.tokens) : p.tokens;
    const int64_t rows = most_new * p.group.d;
    if (p.table && rows <= 16) {
        const bool wide = head_dim == 128, small = kv.page_size == 16;
        if (rows <= 8) return wide ? (small ? attention_few<128, 16, 1>(ctx, p, kv, s) : attention_few<128, 32, 1>(ctx, p, kv, s))
                                   : (small ? attention_few<64, 16, 1>(ctx, p, kv, s) : attention_few<64, 32, 1>(ctx, p, kv, s));
        return wide ? (small ? attention_few<128, 16, 2>(ctx, p, kv, s) : attention_few<128, 32, 2>(ctx, p, kv, s))
                    : (small ? attention_few<64, 16, 2>(ctx, p, kv, s) : attention_few<64, 32, 2>(ctx, p, kv, s));
    }
    if (p.table) return head_dim == 64 ? attention_many<64, true>(ctx, p, kv, s) : attention_many<128, true>(ctx, p, kv, s);
    return head_dim == 64 ? attention_many<64, false>(ctx, p, kv, s) : attention_many<128, false>(ctx, p, kv, s);
}

extern "C" int32_t mpq_paged_attention(mpq_context* ctx, const uint16_t* q_dev, int64_t q_row_stride, int64_t tokens, int32_t q_heads, const uint16_t* k_cache_dev,
                                       const uint16_t* v_cache_dev, int64_t pages, int32_t page_size, int32_t kv_heads, int32_t head_dim, int64_t n, const int32_t* starts_dev,
                                       const int32_t* lens_dev, const int32_t* block_table_dev, int64_t max_blocks, int64_t max_new, float scale, void* out_dev, int32_t out_is_f32,
                                       void* stream)
{
    if (!ctx_ok(ctx)) return MPQ_ERR_INVALID_ARG;
    AttnParams p;
    attention_params(&p, q_dev, q_row_stride, tokens, n, starts_dev, q_heads, kv_heads, scale, out_dev, out_is_f32);
    const AttnKeys kv = {k_cache_dev, v_cache_dev, 0, 0, pages, page_size, max_new};
    const int32_t st = attention_check(ctx, p, kv, n, q_heads, kv_heads, head_dim, scale);
    if (st) return st;
    if (!lens_dev || !block_table_dev) return fail(ctx, MPQ_ERR_INVALID_ARG, "null pointer");
    if (!page_ok(page_size) || pages <= 0 || pages > MOST) return fail(ctx, MPQ_ERR_SHAPE, "pages must be positive, page_size a power of two from 16 to 256 (%lld pages of %d)", (long long)pages, page_size);
    if (pages >= MOST / kv_heads) return fail(ctx, MPQ_ERR_UNSUPPORTED, "pages * kv_heads must be below 2^31");
    if (max_blocks <= 0 || max_blocks > MOST_KEYS / page_size) return fail(ctx, MPQ_ERR_SHAPE, "max_blocks * page_size must be positive and at most 2^30");
    if (max_new < 0) return fail(ctx, MPQ_ERR_SHAPE, "max_new must not be negative");
    const int64_t out_bytes = tokens * q_heads * head_dim * (out_is_f32 ? 4 : 2), cache_bytes = pages * kv_heads * page_size * head_dim * 2;
    if (overlaps(out_dev, out_bytes, k_cache_dev, cache_bytes) || overlaps(out_dev, out_bytes, v_cache_dev, cache_bytes) || overlaps(out_dev, out_bytes, lens_dev, 4 * n) ||
        overlaps(out_dev, out_bytes, block_table_dev, 4 * n * max_blocks))
        return fail(ctx, MPQ_ERR_INVALID_ARG, "out must not overlap an input");
    p.lens = lens_dev; p.table = block_table_dev;
    p.width = max_blocks; p.pages = pages; p.page_shift = log2_of(page_size);
    return attention_launch(ctx, p, kv, head_dim, (cudaStream_t)stream);
}

extern "C" int32_t mpq_prompt_attention(mpq_context* ctx, const uint16_t* q_dev, int64_t q_row_stride, const uint16_t* k_dev, int64_t k_row_stride, const uint16_t* v_dev,
                                        int64_t v_row_stride, int64_t tokens, int32_t q_heads, int32_t kv_heads, int32_t head_dim, int64_t n, const int32_t* starts_dev, float scale,
                                        void* out_dev, int32_t out_is_f32, void* stream)
{
    if (!ctx_ok(ctx)) return MPQ_ERR_INVALID_ARG;
    AttnParams p;
    attention_params(&p, q_dev, q_row_stride, tokens, n, starts_dev, q_heads, kv_heads, scale, out_dev, out_is_f32);
    const AttnKeys kv = {k_dev, v_dev, k_row_stride, v_row_stride, 0, 0, 0};
    const int32_t st = attention_check(ctx, p, kv, n, q_heads, kv_heads, head_dim, scale);
    if (st) return st;
    for (int64_t stride : {k_row_stride, v_row_stride})
        if (stride < (int64_t)kv_heads * head_dim || stride % 8) return fail(ctx, MPQ_ERR_SHAPE, "a row stride must be a multiple of 8 and hold the heads");
    const int64_t out_bytes = tokens * q_heads * head_dim * (out_is_f32 ? 4 : 2), row_bytes = 2ll * kv_heads * head_dim;
    if (overlaps(out_dev, out_bytes, k_dev, tokens, row_bytes, (__int128)k_row_stride * 2) || overlaps(out_dev, out_bytes, v_dev, tokens, row_bytes, (__int128)v_row_stride * 2))
        return fail(ctx, MPQ_ERR_INVALID_ARG, "out must not overlap an input");
    return attention_launch(ctx, p, kv, head_dim, (cudaStream_t)stream);
}
