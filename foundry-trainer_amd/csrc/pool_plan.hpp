// The adapter pool's plan: where its words lie, and what a kernel makes of a word
// before it leads anywhere.  Plain arithmetic, the same on the host: whatever the
// memory holds, no index past the call's tensors comes out of it.
#pragma once

#include <algorithm>
#include <cstdint>

namespace fa {

constexpr int kPoolRows = 64;    // of a row tile
constexpr int kPoolChunk = 256;  // rows of a gradient chunk: whole tiles

// int32 words of a plan
struct PoolTile {
    int tile, rows, adapter, slot;  // rows token[64 * tile .. + rows); adapter -1: none
};
struct PoolPlanView {
    int *head;    // tiles, chunks, T, L
    int *count;   // [L] tokens of each adapter
    int *slot0;   // [L] its first partial gradient; -1: none (at most one chunk)
    PoolTile *tiles, *chunks;
    int *token;   // sorted by adapter, those without one last; each adapter begins a tile
};
__host__ __device__ inline int64_t pool_most_tiles(int64_t T, int64_t L, int rows) {
    return (T + rows - 1) / rows + (L + 1 < T ? L + 1 : T);
}
__host__ __device__ inline int64_t pool_round4(int64_t x) { return (x + 3) & ~int64_t(3); }
__host__ __device__ inline int64_t pool_plan_words(int64_t T, int64_t L) {
    return 4 + 2 * pool_round4(L) + (4 + kPoolRows) * pool_most_tiles(T, L, kPoolRows) +
           4 * pool_most_tiles(T, L, kPoolChunk);
}
__host__ __device__ inline PoolPlanView pool_plan_view(int *p, int64_t T, int64_t L) {
    PoolPlanView v;
    v.head = p;
    v.count = p + 4;
    v.slot0 = v.count + pool_round4(L);
    v.tiles = reinterpret_cast<PoolTile *>(v.slot0 + pool_round4(L));
    v.chunks = v.tiles + pool_most_tiles(T, L, kPoolRows);
    v.token = reinterpret_cast<int *>(v.chunks + pool_most_tiles(T, L, kPoolChunk));
    return v;
}

// Partial gradients: the chunks of adapters with more than one, all full but each
// adapter's last
__host__ __device__ inline int64_t pool_grad_slots(int T, int L) {
    return (int64_t)T / kPoolChunk + std::min<int64_t>(L, (int64_t)T / (kPoolChunk + 1));
}

// Whether `t`, read as tile (or chunk) i under a head of these words, is one of a
// call of T tokens and L adapters: its entries of `token` are in the plan, its
// adapter is below L (negative: none).
__host__ __device__ inline bool pool_tile_fits(int n, int head_t, int head_l, const PoolTile &t, int64_t i, bool chunk,
                                               int T, int L) {
    return head_t == T && head_l == L && i < n && t.tile >= 0 && t.rows > 0 && t.rows <= (chunk ? kPoolChunk : kPoolRows) &&
           (int64_t)t.tile + (t.rows + kPoolRows - 1) / kPoolRows <= pool_most_tiles(T, L, kPoolRows) && t.adapter < L;
}
// A word of `token` as a row of the call's tensors; 0 where it is none.
__host__ __device__ inline int pool_row(int word, int T) { return (unsigned)word < (unsigned)T ? word : 0; }
// Where the gradient of a chunk goes: a partial sum below `slots`, kPoolWhole for
// the result itself, kPoolNowhere for words that no plan has.  slot0: its adapter's.
constexpr int64_t kPoolWhole = -1, kPoolNowhere = -2;
__host__ __device__ inline int64_t pool_grad_place(int slot, int slot0, int64_t slots) {
    if (slot < 0) return kPoolWhole;
    const int64_t at = (int64_t)slot0 + slot;
    return at >= 0 && at < slots ? at : kPoolNowhere;
}
// Partial sums of an adapter of `count` tokens, from `first`: all of them below
// `slots`.  0: its gradient is zero; -1: there is nothing to add up for it.
__host__ __device__ inline int64_t pool_partials(int head_t, int head_l, int count, int first, int64_t slots, int T, int L) {
    if (head_t != T || head_l != L) return -1;
    const int64_t chunks = count > 0 ? ((int64_t)count + kPoolChunk - 1) / kPoolChunk : 0;
    if (chunks == 1) return -1;
    return chunks == 0 || (first >= 0 && first <= slots - chunks) ? chunks : -1;
}

}  // namespace fa
