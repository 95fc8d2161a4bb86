"""The adapter pool's kernels trust no word of a plan: what they make of it
(pool_plan.hpp, compiled here for the host) stays inside the call's tensors
whatever the words are, also under a head that fits the call."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "foundry-trainer_amd", "csrc")

CHECK = r"""
#include "pool_plan.hpp"
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>
using namespace fa;

#define CHECK(x) do { if (!(x)) { printf("line %d: %s (T %d L %d)\n", __LINE__, #x, T, L); exit(1); } } while (0)

static std::mt19937_64 rng(7);
// words of every kind: any, small, next to a size, next to the ends of int
static int word(int T, int L) {
    const int near[] = {0, -1, 1, T, L, kPoolRows, kPoolChunk, INT32_MAX, INT32_MIN, T / kPoolRows, T / kPoolChunk};
    switch (rng() % 4) {
        case 0: return (int)rng();
        case 1: return (int)(rng() % 300) - 20;
        case 2: return (int)((unsigned)near[rng() % 11] + (unsigned)(rng() % 5) - 2u);
        default: return (int)(rng() % (unsigned)(T + 2)) - 1;
    }
}

// What the kernels do with a plan of these words, each index beside its buffer's size.
static long use(const std::vector<int> &words, int T, int L) {
    const PoolPlanView v = pool_plan_view(const_cast<int *>(words.data()), T, L);
    const int64_t most = pool_most_tiles(T, L, kPoolRows), most_chunks = pool_most_tiles(T, L, kPoolChunk);
    const int64_t entries = kPoolRows * most, slots = pool_grad_slots(T, L);
    CHECK((int64_t)words.size() == pool_plan_words(T, L));
    CHECK(v.token + entries == words.data() + words.size());
    long used = 0;
    auto row = [&](int64_t at) {
        CHECK(at >= 0 && at < entries);
        const int t = pool_row(v.token[at], T);
        CHECK(t >= 0 && t < T);
    };
    for (int chunk = 0; chunk < 2; ++chunk)
        for (int64_t i = 0; i < (chunk ? most_chunks : most); ++i) {
            if (!chunk)
                for (int x = 0; x < kPoolRows; ++x) row(i * kPoolRows + x);  // read beside the tile itself
            const PoolTile t = (chunk ? v.chunks : v.tiles)[i];
            if (!pool_tile_fits(v.head[chunk], v.head[2], v.head[3], t, i, chunk, T, L)) continue;
            CHECK(i < v.head[chunk] && t.adapter < L && t.rows > 0 && t.rows <= (chunk ? kPoolChunk : kPoolRows));
            for (int x = 0; x < t.rows; ++x) row((int64_t)t.tile * kPoolRows + x);
            ++used;
            if (!chunk || t.adapter < 0) continue;
            const int64_t slot = pool_grad_place(t.slot, v.slot0[t.adapter], slots);
            CHECK(slot == kPoolWhole || slot == kPoolNowhere || (slot >= 0 && slot < slots));
            CHECK((slot == kPoolWhole) == (t.slot < 0));
        }
    for (int a = 0; a < L; ++a) {
        const int64_t n = pool_partials(v.head[2], v.head[3], v.count[a], v.slot0[a], slots, T, L);
        CHECK(n == -1 || n == 0 || (n > 1 && v.slot0[a] >= 0 && v.slot0[a] + n <= slots));
        CHECK(n <= 0 || v.count[a] > kPoolChunk);
    }
    return used;
}

// The plan of an index, as the operator's definition has it.
static std::vector<int> plan_of(const std::vector<int> &index, int T, int L) {
    std::vector<int> words(pool_plan_words(T, L), 0);
    PoolPlanView v = pool_plan_view(words.data(), T, L);
    int tiles = 0, chunks = 0, slots = 0;
    for (int a = 0; a <= L; ++a) {
        std::vector<int> mine;
        for (int t = 0; t < T; ++t)
            if ((index[t] < 0 || index[t] >= L ? L : index[t]) == a) mine.push_back(t);
        const int n = (int)mine.size(), tile0 = tiles, nc = (n + kPoolChunk - 1) / kPoolChunk;
        for (int k = 0; k < n; ++k) v.token[tile0 * kPoolRows + k] = mine[k];
        for (int k = 0; k < n; k += kPoolRows)
            v.tiles[tiles++] = PoolTile{tile0 + k / kPoolRows, std::min(kPoolRows, n - k), a < L ? a : -1, 0};
        if (a == L) continue;
        v.count[a] = n;
        v.slot0[a] = nc > 1 ? slots : -1;
        for (int k = 0; k < nc; ++k)
            v.chunks[chunks++] = PoolTile{tile0 + k * (kPoolChunk / kPoolRows), std::min(kPoolChunk, n - k * kPoolChunk),
                                          a, nc > 1 ? k : -1};
        if (nc > 1) slots += nc;
    }
    v.head[0] = tiles, v.head[1] = chunks, v.head[2] = T, v.head[3] = L;
    CHECK(tiles <= pool_most_tiles(T, L, kPoolRows) && chunks <= pool_most_tiles(T, L, kPoolChunk));
    CHECK(slots <= pool_grad_slots(T, L));
    return words;
}

int main() {
    const int sizes[][2] = {{0, 1}, {1, 1}, {1, 7}, {5, 2048}, {63, 3}, {64, 1}, {65, 4}, {256, 1}, {257, 1}, {514, 2},
                            {700, 3}, {2000, 40}};
    long used = 0, whole = 0;
    for (auto &s : sizes) {
        const int T = s[0], L = s[1];
        for (int turn = 0; turn < 60; ++turn) {
            // a plan that is one is used whole
            std::vector<int> index(T);
            for (int &i : index) i = turn % 3 == 0 ? 0 : (int)(rng() % (L + 2)) - 1;
            std::vector<int> words = plan_of(index, T, L);
            const long all = use(words, T, L);
            CHECK(all == words[0] + words[1]);
            whole += all;
            // single words of it changed, then any words under a head that fits, then any head
            for (int n = 0; n < 8 && !words.empty(); ++n) words[rng() % words.size()] = word(T, L);
            used += use(words, T, L);
            for (int &w : words) w = word(T, L);
            words[0] = words[1] = INT32_MAX, words[2] = T, words[3] = L;
            used += use(words, T, L);
            words[rng() % 4] = word(T, L);
            used += use(words, T, L);
        }
    }
    // sizes at the ends of what a call may have: no sum leaves its type
    const int T = 1 << 28, L = 2048;
    for (int n = 0; n < 2000000; ++n) {
        const PoolTile t{word(T, L), word(T, L), word(T, L), word(T, L)};
        if (pool_tile_fits(INT32_MAX, T, L, t, rng() % 4000000, n & 1, T, L))
            CHECK((int64_t)t.tile * kPoolRows + t.rows <= kPoolRows * pool_most_tiles(T, L, kPoolRows));
        const int64_t slots = pool_grad_slots(T, L), at = pool_grad_place(t.slot, t.tile, slots);
        CHECK(at >= kPoolNowhere && at < slots);
        const int64_t c = pool_partials(T, L, t.rows, t.tile, slots, T, L);
        CHECK(c <= 0 || (t.tile >= 0 && t.tile + c <= slots));
    }
    CHECK(used > 1000 && whole > 1000);
    return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not available")
def test_no_word_leads_outside(tmp_path):
    src, exe = tmp_path / "check.cpp", tmp_path / "check"
    src.write_text(CHECK)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=undefined", "-D__host__=",
                    "-D__device__=", "-I", CSRC, "-o", str(exe), str(src)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout + run.stderr
