"""How the attention kernels cut their work (attention_plan.h), compiled for the host: every tile of every unit belongs to one CTA, pieces are counted
by the CTAs that have them, and lengths that say nonsense stay inside the arrays."""
import os
import subprocess
import tempfile

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include "attention_plan.h"
#include <cstdio>
#include <random>
#include <vector>
using namespace mpq;
int main()
{
    std::mt19937 rng(1);
    auto pick = [&](int a, int b) { return a + (int)(rng() % (unsigned)(b - a + 1)); };
    long bad = 0;
    for (int trial = 0; trial < 4000; ++trial) {
        // owners of tiles agree with the runs, for fewer and for more tiles than CTAs
        const int total = trial % 5 == 0 ? pick(1, 1 << 30) : pick(1, trial % 2 ? 300 : 100000);
        const int ctas0 = pick(1, trial % 3 ? 160 : 1024), ctas = (int)(ctas0 < total ? ctas0 : total);
        if (attn_run(0, total, ctas) != 0 || attn_run(ctas, total, ctas) != total) ++bad;
        for (int c = 0; c < ctas; ++c) {
            const int lo = attn_run(c, total, ctas), hi = attn_run(c + 1, total, ctas);
            if (lo >= hi) ++bad;
            if (attn_owner(lo, total, ctas) != c || attn_owner(hi - 1, total, ctas) != c) ++bad;
        }
    }
    if (attn_owner((1 << 30) - 1, 1 << 30, ATTN_MOST_RUNS) != ATTN_MOST_RUNS - 1) ++bad;
    // units of unlike lengths in a row, cut into runs: every tile belongs to one run, pieces are counted by exactly the runs from opener to closer, and
    // none is shorter than it has to be
    for (int trial = 0; trial < 3000; ++trial) {
        const int units = pick(1, 60), extra = pick(0, 3), least = pick(1, 4), longest = trial % 3 ? 12 : 90;
        std::vector<int> at, tiles;
        int total = 0;
        for (int i = 0; i < units; ++i) { at.push_back(total); tiles.push_back(pick(1, longest)); total += tiles[i] + extra; }
        const int want = pick(1, 200), runs = want < total ? want : total;
        std::vector<std::vector<int>> had(units), by(units);
        for (int i = 0; i < units; ++i) had[i].assign(tiles[i], 0);
        for (int v = 0; v < runs; ++v) {
            const int lo = attn_run(v, total, runs), hi = attn_run(v + 1, total, runs);
            int i = 0;
            while (i + 1 < units && at[i + 1] <= lo) ++i;
            if (attn_first(lo, at[i], tiles[i], least) == tiles[i]) ++i;
            for (; i < units && at[i] < hi && !attn_behind(hi, at[i], tiles[i], least); ++i) {
                const int first = lo <= at[i] ? 0 : attn_first(lo, at[i], tiles[i], least), end = attn_end(hi, at[i], tiles[i], least);
                if (first >= end || end > tiles[i]) { ++bad; continue; }
                for (int t = first; t < end; ++t) ++had[i][t];
                if (first > 0 || end < tiles[i]) {
                    if (end - first < (least < tiles[i] / 2 + 1 ? 1 : 0)) ++bad;
                    if (first == 0 && attn_opener(at[i], tiles[i], least, total, runs) != v) ++bad;
                    if (end == tiles[i] && attn_closer(at[i], tiles[i], least, total, runs) != v) ++bad;
                    by[i].push_back(v);
                }
            }
        }
        for (int i = 0; i < units; ++i) {
            for (int n : had[i]) bad += n != 1;
            if (by[i].empty()) continue;
            const int o = attn_opener(at[i], tiles[i], least, total, runs), c = attn_closer(at[i], tiles[i], least, total, runs);
            if ((int)by[i].size() != c - o + 1 || by[i].front() != o || by[i].back() != c) ++bad;
            if (o >= runs || c >= runs) ++bad;
        }
    }
    // parts: one for little work or few keys, never runs of fewer tiles than ATTN_LEAST_RUN unless there is one part
    for (int trial = 0; trial < 2000; ++trial) {
        const int total = pick(1, 1 << 20);
        const int64_t bytes = (int64_t)pick(0, 1 << 20) << 10;
        const int ctas = pick(1, 256), parts = attn_parts(total, ctas, bytes, 4);
        if (parts < 1 || parts > 4 || (parts > 1 && (total / parts / ctas < ATTN_LEAST_RUN || (parts - 1) * ATTN_PART_BYTES >= bytes))) ++bad;
    }
    for (int d = 1; d <= 4096; ++d) {
        const AttnDivisor by = attn_divisor(d);
        for (int k = 0; k < 200; ++k) {
            const int x = k < 50 ? (int)(0x7FFFFFFF - k) : k < 100 ? k : (int)(rng() & 0x7FFFFFFF), y = x / d * d;
            for (int v : {x, y, y > 0 ? y - 1 : 0}) bad += by.of(v) != v / d;
        }
    }
    for (int trial = 0; trial < 3000; ++trial) {
        const int group = pick(1, 20), rows = trial % 2 ? 16 : 256, tile = 128;
        const int64_t tokens = pick(1, 900), start = pick(-5, 1000), next = pick(-5, 1000);
        const bool paged = trial % 3 != 0;
        const int64_t most = 16 * pick(1, 200), len = pick(-3, 4000);
        const AttnRequest r = attn_request(start, next, tokens, paged, len, most);
        if (r.first < 0 || r.rows < 0 || r.first + r.rows > tokens || r.keys < 0 || (paged && r.keys > most) || (!paged && r.keys != r.rows)) ++bad;
        const AttnDivisor by = attn_divisor(group);
        const int blocks = attn_blocks(r, group, rows);
        int64_t counted = 0;
        for (int b = 0; b < blocks; ++b) {
            const int mine = attn_block_rows(r, group, b, rows);
            if (mine < 1 || mine > rows) ++bad;
            counted += mine;
            // keys of the block: the most that any of its rows sees, by counting
            int seen = 0;
            for (int i = 0; i < mine; ++i) {
                const int j = (b * rows + i) / group;
                int n = 0;
                const int64_t last = (int64_t)r.keys - r.rows + j;
                if (last >= 0) n = (int)(last + 1 < r.keys ? last + 1 : r.keys);
                if (n != attn_seen(r, j)) ++bad;
                seen = n > seen ? n : seen;
            }
            const int tiles = attn_block_tiles(r, by, b, rows, tile);
            if (tiles < 1 || tiles * tile < seen || (tiles > 1 && (tiles - 1) * tile >= seen)) ++bad;
        }
        if (counted != (int64_t)r.rows * group) ++bad;
    }
    std::printf("%ld\n", bad);
    return bad != 0;
}
"""


def test_the_cut_of_the_work():
    with tempfile.TemporaryDirectory() as tmp:
        src, exe = os.path.join(tmp, "t.cpp"), os.path.join(tmp, "t")
        open(src, "w").write(PROGRAM)
        subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-I", os.path.join(ROOT, "makepad_b200", "csrc"), src, "-o", exe])
        out = subprocess.run([exe], capture_output=True, text=True)
        assert out.returncode == 0 and out.stdout.strip() == "0", out.stdout + out.stderr


def test_the_new_kernels_read_what_is_in_front_of_them_by_ordinary_loads():
    """Behind start_beside() there is no load through the read-only path, and no pointer that would let the compiler choose it."""
    csrc = os.path.join(ROOT, "makepad_b200", "csrc")
    kernels = 0
    for f in ("norm.cuh", "kv_cache.cuh", "attention.cuh", "attention_few.cuh", "attention_many.cuh"):
        text = open(os.path.join(csrc, f)).read()
        assert "__ldg" not in text and "__restrict__" not in text and "__ldc" not in text, f
        for kernel in text.split("__global__ ")[1:]:
            kernels += 1
            assert "start_beside();" in kernel[:kernel.index("\n}")], (f, kernel[:100])
    assert kernels == 5
