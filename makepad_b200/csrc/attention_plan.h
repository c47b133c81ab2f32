// How the attention kernels cut their work.  Integer arithmetic for the device and, in tests, for the host.
//
// The new tokens of a request and the query heads that share a head of keys are its rows, packed token by token: row = token * group +
// head in the group.  A block is up to ROWS consecutive rows; a unit is a block and a head of keys; its tiles are the TILE keys at a time that
// its last row sees (one, empty, where it sees none: its rows of zeros are written all the same).  The tiles of all units in order
// (request, head, block) are cut into equal runs, one per CTA (or a few: attn_parts), wherever that falls: no shape leaves SMs idle.  What a unit
// costs beside its tiles (its queries, its end) counts as `extra` tiles behind them that nobody works on.  A unit that a cut falls into has a piece in each
// run from the one with its first tile to the one with its last.  A run opens at most one such unit (its last) and continues at most one (its first).  A piece costs the time of some tiles
// (its sums are stored and counted, and read again): a cut closer than that to a unit's end moves there.
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

// x / d for x < 2^31, without a division: (x + mulhi(x, mul)) >> shift
struct AttnDivisor {
    uint32_t d, mul, shift;
    MPQ_BOTH int of(int x) const
    {
#ifdef __CUDA_ARCH__
        return (int)((__umulhi((uint32_t)x, mul) + (uint32_t)x) >> shift);
#else
        return (int)(((uint32_t)(((uint64_t)(uint32_t)x * mul) >> 32) + (uint32_t)x) >> shift);
#endif
    }
};
inline AttnDivisor attn_divisor(uint32_t d)
{
    AttnDivisor a = {d, 0, 0};
    while ((1ull << a.shift) < d) ++a.shift;
    a.mul = (uint32_t)((((1ull << a.shift) - d) << 32) / d + 1);
    return a;
}

// (rows * group is below 2^31; block_rows and tile are powers of two)
MPQ_BOTH int attn_blocks(const AttnRequest& r, int group, int block_rows) { return (int)(((uint32_t)(r.rows * group) + block_rows - 1) / (uint32_t)block_rows); }
// keys that new token j sees
MPQ_BOTH int attn_seen(const AttnRequest& r, int j)
{
    const int s = r.keys - (r.rows - 1 - j);
    return s < 0 ? 0 : s;
}
// rows of block b, and the tiles of keys that the last of its rows sees
MPQ_BOTH int attn_block_rows(const AttnRequest& r, int group, int b, int block_rows)
{
    const int left = r.rows * group - b * block_rows;
    return left < block_rows ? left : block_rows;
}
MPQ_BOTH int attn_tiles(int keys, int tile) { return keys <= tile ? 1 : (int)(((uint32_t)keys + tile - 1) / (uint32_t)tile); }
MPQ_BOTH int attn_block_tiles(const AttnRequest& r, const AttnDivisor& group, int b, int block_rows, int tile)
{
    return attn_tiles(attn_seen(r, group.of(b * block_rows + attn_block_rows(r, (int)group.d, b, block_rows) - 1)), tile);
}

// First tile of run v of `runs` (at most `total`, and at most ATTN_MOST_RUNS), and the run that has tile t.
MPQ_BOTH int attn_run(int v, int total, int runs)
{
    const uint32_t q = (uint32_t)total / (uint32_t)runs, r = (uint32_t)total - q * runs;
    return (int)(v * q + (uint32_t)v * r / (uint32_t)runs);
}
MPQ_BOTH int attn_owner(int t, int total, int runs)
{
    if (total < (1 << 20)) return (int)(((uint32_t)(t + 1) * (uint32_t)runs - 1) / (uint32_t)total);
    return (int)((((uint64_t)t + 1) * runs - 1) / (uint32_t)total);
}
// Tiles that a piece has at least, of a unit of `tiles` (more than half of them: then there is no piece).
MPQ_BOTH int attn_least(int tiles, int least) { return least < tiles / 2 + 1 ? least : tiles / 2 + 1; }
// Of the run [lo, hi): whether the unit whose first tile is `unit` begins behind it; the unit's first tile in it (it is the run's first unit, or 0); its end there.
MPQ_BOTH bool attn_behind(int hi, int unit, int tiles, int least) { return hi - unit < attn_least(tiles, least); }
MPQ_BOTH int attn_first(int lo, int unit, int tiles, int least)
{
    const int d = lo - unit, n = attn_least(tiles, least);
    return d < n ? 0 : d > tiles - n ? tiles : d;              // (tiles: all of it is another run's)
}
MPQ_BOTH int attn_end(int hi, int unit, int tiles, int least) { return hi - unit > tiles - attn_least(tiles, least) ? tiles : hi - unit; }
// runs with the unit's first and last piece
MPQ_BOTH int attn_opener(int unit, int tiles, int least, int total, int runs) { return attn_owner(unit + attn_least(tiles, least) - 1, total, runs); }
MPQ_BOTH int attn_closer(int unit, int tiles, int least, int total, int runs) { return attn_owner(unit + tiles - attn_least(tiles, least), total, runs); }
constexpr int ATTN_MOST_RUNS = 2048;
// Requests of a call: every CTA adds them up in ATTN_ENTRIES entries and walks through those of one entry, and through the ones without rows, while others
// wait for it: 3 and 10 ms (many rows, few) for this many of which only the first and the last have rows.  The waits give up after a few hundred.
constexpr int64_t ATTN_MOST_REQUESTS = 1 << 20;
constexpr int ATTN_ENTRIES = 160;
MPQ_BOTH int attn_per(int n) { return (n + ATTN_ENTRIES - 1) / ATTN_ENTRIES; }
constexpr int64_t ATTN_MOST_TILES = 1ll << 30;         // of a call: what has more (hours of work) is not begun, and says so in the status word

// Into how many parts, one after the other, all tiles are cut before each part is cut into a run per CTA: so many that the keys and values of a part
// (in a part are the heads of few requests) stay in L2, but no runs of fewer than ATTN_LEAST_RUN tiles.
constexpr int64_t ATTN_PART_BYTES = 40 << 20;
constexpr int ATTN_LEAST_RUN = 48;
MPQ_BOTH int attn_parts(int total, int ctas, int64_t kv_bytes, int most)
{
    int parts = total / (ctas * ATTN_LEAST_RUN);
    if (parts > most) parts = most;
    for (; parts > 1 && (parts - 1) * ATTN_PART_BYTES >= kv_bytes;) --parts;
    return parts < 1 ? 1 : parts;
}

}  // namespace mpq
