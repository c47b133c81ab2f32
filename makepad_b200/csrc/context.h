// The context behind the C ABI, its error text and the checks that every entry point makes.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <cstdarg>
#include <cstdio>
#include <mutex>
#include <string>

#include "../../include/mpq.h"
#include "host_pages.h"
#include "nvfp4.cuh"
#include "on_device.h"
#include "scratch.h"
#include "upload.h"

struct mpq_context {
    uint32_t magic;
    int device;
    cudaDeviceProp prop;
    std::string err;
    int64_t launches;
    bool pdl;                 // programmatic dependent launch between consecutive linears
    int q4_variant;           // 0 = subnormal-fp16 weights (default), 1 = magic-number conversion
    // staging for the *_host convenience calls (grown on demand), one such call at a time
    std::mutex host_lock;
    float *hx, *hy;
    size_t hx_bytes, hy_bytes;
    mpq::HostPages host_x, host_y; // ... and the pages through which small rows travel
    // scratch of the streaming Q4 kernel: tagged partial tiles of row pair-tiles cut by a boundary
    // between two CTAs' runs (two slots per CTA; write-once / read-once per launch), one status word
    mpq::Scratch q4u_xs;       // staged activations of the tcgen05 kernels, then the row scales
    mpq::Scratch swiglu_buf;   // SwiGLU output for the Q4 kernels that do not fuse it
    int q4_umma_min;          // fewest activation rows routed to the tcgen05 kernel (0 = never)
    mpq::Scratch q4_partial;   // partial outputs: [K slices][M][N] of the rectangle kernel, the pieces of the tcgen05 kernels
    int q4_gemm_min;          // fewest activation rows routed to q4_gemm_kernel (0 = never: slabs of 64 through the tcgen05 kernel)
    bool q4_rect;             // use the rectangle kernel for 5..16 rows (else slabs of <= 4 rows through the streaming kernel)
    int q4_stream_max_m;      // most activation rows mpq_q4_linear_forward gives to the streaming kernel (1..4)
    int q4_rect_nks;          // experiment: at least so many K slices in the rectangle kernel (0 = the plan's choice)
    bool q4_rect_cluster;     // K slices of the rectangle kernel as clusters where they fit
    int q4_rect_depth;        // ring depth of the rectangle kernel: 0 = choose, else 1..8
    uint2* q4_partials;
    int q4_partials_ctas;
    int* q4_status;
    bool q4_stream;           // use the streaming kernel where the activation fits in shared memory
    bool q4_tile_mode;        // let CTAs own whole row pair-tiles when the matrix has enough of them
    int q4_group;             // chunks per bulk copy of the streaming kernel: 0 = choose, 1, 2 or 4
    int q4_depth;             // most ring stages per warp
    int q4_pre;               // stages copied before the dependency resolves (the rest right after the activation loads)
    bool q4_slab4;            // M > 4 as slabs of four rows through the streaming kernel
    // attention: pieces of units that CTAs share, then per CTA a counter of their arrivals, and a status word
    mpq::Scratch attn_partial;
    uint32_t* attn_arrived;
    int* attn_status;
    mpq::Nvfp4Scratch fp4;
    mpq::StagedUpload upload;  // pinned slots through which weights travel to the device
    cudaStream_t upload_stream;
};

namespace mpq {

constexpr int ATTN_COUNTERS = 4096;     // two for each run of an attention kernel, at most
constexpr int ATTN_TOO_MUCH = 40;       // in the attention kernels' status word: not a wait that ran out
constexpr uint32_t CTX_MAGIC = 0x4D505143u;

inline int32_t fail(mpq_context* ctx, int32_t code, const char* fmt, ...)
{
    if (code == MPQ_ERR_CUDA) cudaGetLastError();          // reported here: not left behind for a later call to find
    if (ctx) {
        char buf[512];
        va_list ap;
        va_start(ap, fmt);
        vsnprintf(buf, sizeof buf, fmt, ap);
        va_end(ap);
        ctx->err = buf;
    }
    return code;
}

#define CU_TRY(ctx, expr)                                                                         \
    do {                                                                                          \
        cudaError_t e__ = (expr);                                                                 \
        if (e__ != cudaSuccess)                                                                   \
            return fail(ctx, MPQ_ERR_CUDA, "%s failed: %s (%s:%d)", #expr, cudaGetErrorString(e__), __FILE__, __LINE__); \
    } while (0)

inline bool ctx_ok(const mpq_context* c) { return c && c->magic == CTX_MAGIC; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// true when the stream must not see an allocation now
inline bool stream_captures(cudaStream_t s)
{
    cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(s, &cs) != cudaSuccess) {
        cudaGetLastError();
        return true;
    }
    return cs != cudaStreamCaptureStatusNone;
}

}  // namespace mpq
