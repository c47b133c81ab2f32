// How the attention kernels cut their work.  Integer arithmetic for the device and, in tests, for the host.
//
// The new tokens of a request and the query heads that share a head of keys are its rows, packed token by token: row = token * group +
// head in the group.  A block is up to ROWS consecutive rows; a unit is a block and a head of keys; its tiles are the TILE keys at a time that
// its last row sees (one, empty, where it sees none: its rows of zeros are written all the same).  The tiles of all units in order
// (request, block, head) are cut into equal runs, one per CTA, wherever that falls: no shape leaves SMs idle.  A unit that a cut falls into has a piece
// in each CTA from the one with its first tile to the one with its last.  A CTA opens at most one such unit (its last) and continues at most one (its first).
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define MPQ_BOTH __host__ __device__ __forceinline__
#else
#define MPQ_BOTH inline
#endif

namespace mpq {

// rows and keys of a request, within the arrays whatever the lengths say
struct AttnRequest {
    int first, rows, keys;              // first row of q, new tokens, keys
};
MPQ_BOTH AttnRequest attn_request(int64_t start, int64_t next, int64_t tokens, bool paged, int64_t len, int64_t most_keys)
{
    start = start < 0 ? 0 : start > tokens ? tokens : start;
    next = next < start ? start : next > tokens ? tokens : next;
    AttnRequest r;
    r.first = (int)start;
    r.rows = (int)(next - start);
    r.keys = paged ? (int)(len < 0 ? 0 : len > most_keys ? most_keys : len) : r.rows;
    return r;
}

MPQ_BOTH int64_t attn_blocks(const AttnRequest& r, int group, int block_rows) { return ((int64_t)r.rows * group + block_rows - 1) / block_rows; }
// keys that new token j sees
MPQ_BOTH int attn_seen(const AttnRequest& r, int64_t j)
{
    const int64_t s = (int64_t)r.keys - r.rows + j + 1;
    return s < 0 ? 0 : s > r.keys ? r.keys : (int)s;
}
// rows of block b, and keys that the last one of its rows from `from` on (at most `count`) sees
MPQ_BOTH int attn_block_rows(const AttnRequest& r, int group, int64_t b, int block_rows)
{
    const int64_t left = (int64_t)r.rows * group - b * block_rows;
    return left < block_rows ? (int)left : block_rows;
}
MPQ_BOTH int attn_block_keys(const AttnRequest& r, int group, int64_t b, int block_rows)
{
    return attn_seen(r, (b * block_rows + attn_block_rows(r, group, b, block_rows) - 1) / group);
}
MPQ_BOTH int attn_block_tiles(const AttnRequest& r, int group, int64_t b, int block_rows, int tile)
{
    const int keys = attn_block_keys(r, group, b, block_rows);
    return keys <= tile ? 1 : (keys + tile - 1) / tile;
}

// run of CTA c of `ctas` (at most `total` of them have one), and the CTA that has tile t
MPQ_BOTH int64_t attn_run(int64_t c, int64_t total, int64_t ctas) { return c * total / ctas; }
MPQ_BOTH int attn_owner(int64_t t, int64_t total, int64_t ctas) { return (int)(((t + 1) * ctas - 1) / total); }

}  // namespace mpq
