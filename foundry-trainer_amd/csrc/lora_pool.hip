// A pool of LoRA adapters beside one shared projection.  Token t belongs to
// adapter i = index[t], or to none where index[t] is outside 0..L-1:
//   u[t]  = A_i x[t]             y[t]  += s_i B_i u[t]
//   v[t]  = B_i^T dy[t]          dx[t] += s_i A_i^T v[t]
//   dA_i  = s_i sum_t v[t] x[t]^T     dB_i = s_i sum_t dy[t] u[t]^T
// with A [L, r, K], B [L, M, r].
//
// The plan (pool_plan_kernel) sorts the tokens by adapter, stably, and cuts each
// adapter's tokens into row tiles of 64 and gradient chunks of 256; all other
// kernels run on a grid of the most tiles there can be and leave at once where
// there is none, so nothing of the index has to come back to the host.
//   pool_down   64 rows x a range of the wide axis: u or v, f32, over `splits`
//               ranges that the reader adds in order
//   pool_up     64 rows x 256 columns or twice that: y
//   pool_back   dx in the same way, and beside it dA and dB: a chunk x 256 (f32:
//               128) columns, straight to the result where the adapter has one
//               chunk, else a partial sum
//   pool_reduce the partial sums in order, and zeros for adapters without tokens
// u and v are f32 between the kernels.  bf16 products (v_mfma_f32_16x16x32) take
// them as the sum of three bf16 terms, high part first, which holds all 24 bits:
// with two (2^-17) y and dx round to another bf16 value than the f32 product's one
// time in a thousand.  f32 products are v_mfma_f32_16x16x4.  No atomics: the same
// bits every time.
#include <algorithm>
#include <type_traits>

#include "fa_device.hpp"
#include "fa_kernels.hpp"
#include "fa_lds.hpp"
#include "pool_plan.hpp"

namespace fa {
namespace {

typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));

constexpr int kRows = kPoolRows, kChunk = kPoolChunk;
constexpr int kPlanWaves = 16;
using Tile = PoolTile;
using PlanView = PoolPlanView;

// ---------------------------------------------------------------------------
// the plan
// ---------------------------------------------------------------------------
// Inclusive sum over the lanes before and at this one.
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);  // row_shr 1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row_bcast 15 into rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // row_bcast 31 into rows 2 and 3
    return x;
}

// One workgroup.  Wave w holds the w-th sixteenth of the tokens; hist[w][a]
// first counts its tokens of adapter a (a = L: none), then holds where in
// `token` they begin.  The lanes of a wave that hold the same adapter find each
// other by one ballot per bit of its number: 64 tokens of 48 adapters took 5 us
// by one ballot per adapter.  Latency-bound: the sums over adapters are one wave's,
// and up to kPlanKept tokens the index is read once, eight words a thread in flight
// together, and kept in LDS; of more tokens it is read twice, one step of 64 a wave
// ahead.  12 adapters, whole requests (token by token): 8192 tokens 7.5 us (9.5),
// 8193 9.4 (12.8), 13312 12, 65536 53.  3.7 us for 1 token (a launch that does
// nothing takes about 2), 4.4 for 64, 6.1 for 4096; it serves every projection of
// the step, and one workgroup needs no second launch.  More than 8192 would fit the
// LDS beside few adapters, at more registers for the words in flight: not tried.
constexpr int kPlanKept = 8192;
__host__ __device__ inline bool plan_keeps(int T, int L) { return T <= kPlanKept && L <= 1024; }
__host__ __device__ inline int plan_lds_words(int T, int L) {
    return kPlanWaves * (L + 1) + 3 * (L + 2) + (plan_keeps(T, L) ? T : 0);
}

__global__ __launch_bounds__(1024) void pool_plan_kernel(const int *index, int T, int L, int bits, int *plan) {
    extern __shared__ int hist[];  // [kPlanWaves][L + 1], [3][L + 2]: rows of a, tiles and chunks before it; the index
    __shared__ int total[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, A = L + 1;
    int *rows = hist + kPlanWaves * A, *tiles0 = rows + L + 2, *chunks0 = tiles0 + L + 2, *idx = chunks0 + L + 2;
    const PlanView v = pool_plan_view(plan, T, L);
    const int64_t share = (((int64_t)T + kPlanWaves - 1) / kPlanWaves + 63) / 64 * 64;
    const int64_t t0 = wave * share, t1 = std::min<int64_t>(T, t0 + share);
    const bool kept = plan_keeps(T, L);
    if (kept && T > 0) {
        int w[kPlanKept / 1024];  // all loads before the first wait
#pragma unroll
        for (int k = 0; k < kPlanKept / 1024; ++k) w[k] = index[std::min(k * 1024 + tid, T - 1)];
#pragma unroll
        for (int k = 0; k < kPlanKept / 1024; ++k)
            if (k * 1024 + tid < T) idx[k * 1024 + tid] = w[k];
    }
    for (int i = tid; i < kPlanWaves * A; i += 1024) hist[i] = 0;
    __syncthreads();
    auto adapter_of = [&](int64_t t) {
        if (t >= t1) return -1;
        const int a = kept ? idx[t] : index[t];
        return a < 0 || a >= L ? L : a;
    };
    // lanes that hold the same adapter as this one
    auto peers = [&](int a) {
        uint64_t same = __ballot(a >= 0);
        const int one = __builtin_amdgcn_readfirstlane(a);
        if (__ballot(a == one) == same) return same;  // a whole request's
#pragma unroll 1
        for (int b = 0; b < bits; ++b) {
            const uint64_t set = __ballot(a >> b & 1);
            same &= a >> b & 1 ? set : ~set;
        }
        return same;
    };
    const uint64_t below = (uint64_t(1) << lane) - 1;
    int ahead = adapter_of(t0 + lane);
#pragma unroll 1
    for (int64_t t = t0; t < t1; t += 64) {
        const int a = ahead;
        ahead = adapter_of(t + 64 + lane);
        const uint64_t same = peers(a);
        if (a < 0) continue;
        const int n = hist[wave * A + a];
        if (kept) idx[t + lane] = (n + __popcll(same & below)) << 12 | a;  // its place among the wave's of its adapter
        if (lane == __builtin_ctzll(same)) hist[wave * A + a] = n + __popcll(same);
    }
    __syncthreads();
    if (wave == 0) {
        int tiles = 0, chunks = 0, slots = 0;  // before these 64 adapters
#pragma unroll 1
        for (int a0 = 0; a0 < A; a0 += 64) {
            const int a = a0 + lane;
            int n = 0;
            if (a < A)
#pragma unroll
                for (int w = 0; w < kPlanWaves; ++w) n += hist[w * A + a];
            const int nt = (n + kRows - 1) / kRows, nc = a < L ? (n + kChunk - 1) / kChunk : 0, ns = nc > 1 ? nc : 0;
            const int st = wave_scan(nt), sc = wave_scan(nc), ss = wave_scan(ns);
            if (a < A) {
                const int tile0 = tiles + st - nt;
                rows[a] = n;
                tiles0[a] = tile0;
                chunks0[a] = chunks + sc - nc;
                int at = tile0 * kRows;
#pragma unroll
                for (int w = 0; w < kPlanWaves; ++w) {
                    const int c = hist[w * A + a];
                    hist[w * A + a] = at;
                    at += c;
                }
                if (a < L) {
                    v.count[a] = n;
                    v.slot0[a] = ns ? slots + ss - ns : -1;
                }
            }
            tiles += __builtin_amdgcn_readlane(st, 63);
            chunks += __builtin_amdgcn_readlane(sc, 63);
            slots += __builtin_amdgcn_readlane(ss, 63);
        }
        if (lane == 0) {
            total[0] = tiles;
            total[1] = chunks0[A] = chunks;
            *reinterpret_cast<u32x4 *>(v.head) = u32x4{(uint32_t)tiles, (uint32_t)chunks, (uint32_t)T, (uint32_t)L};
        }
    }
    __syncthreads();
    if (kept) {
        for (int64_t t = t0 + lane; t < t1; t += 64) {
            const int w = idx[t];
            v.token[hist[wave * A + (w & 4095)] + (w >> 12)] = (int)t;
        }
    } else {
        ahead = adapter_of(t0 + lane);
#pragma unroll 1
        for (int64_t t = t0; t < t1; t += 64) {
            const int a = ahead;
            ahead = adapter_of(t + 64 + lane);
            const uint64_t same = peers(a);
            if (a < 0) continue;
            const int n = hist[wave * A + a];
            v.token[n + __popcll(same & below)] = (int)t + lane;
            if (lane == __builtin_ctzll(same)) hist[wave * A + a] = n + __popcll(same);
        }
    }
    auto find = [&](const int *first, int i) {  // the last adapter a with first[a] <= i
        int lo = 0, hi = A - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (first[mid] <= i) lo = mid;
            else hi = mid - 1;
        }
        return lo;
    };
    for (int i = tid; i < total[0]; i += 1024) {
        const int a = find(tiles0, i), k = i - tiles0[a];
        v.tiles[i] = Tile{i, std::min(kRows, rows[a] - k * kRows), a < L ? a : -1, 0};
    }
    for (int i = tid; i < total[1]; i += 1024) {
        const int a = find(chunks0, i), k = i - chunks0[a];
        v.chunks[i] = Tile{tiles0[a] + k * (kChunk / kRows), std::min(kChunk, rows[a] - k * kChunk), a,
                           rows[a] > kChunk ? k : -1};
    }
}

// Workgroups run column by column of a tile, then the next tile: those at work at
// once hold whole rows.  (Tile by tile of a column block, a 512-byte piece of
// every row, 6000 x 8192 took the expand product 53 us.)
constexpr int kGridTiles = 32768;
dim3 tile_grid(int64_t columns, int64_t tiles) {
    return dim3((unsigned)columns, (unsigned)std::min<int64_t>(tiles, kGridTiles),
                (unsigned)((tiles + kGridTiles - 1) / kGridTiles));
}
__device__ __forceinline__ int64_t grid_tile() { return (int64_t)blockIdx.z * kGridTiles + blockIdx.y; }

// Tile or chunk i of the plan as the kernels trust it: nothing of it leads
// outside the call's tensors, whatever memory the plan was given.
__device__ __forceinline__ bool tile_of(const PoolParams &p, const PlanView &v, bool chunk, int64_t i, Tile &t) {
    // all loads at once: the tile's place holds some word, whether or not there is such a tile
    const u32x4 head = *reinterpret_cast<const u32x4 *>(v.head);
    const u32x4 w = *reinterpret_cast<const u32x4 *>((chunk ? v.chunks : v.tiles) + i);
    t = __builtin_bit_cast(Tile, w);
    return pool_tile_fits((int)(chunk ? head[1] : head[0]), (int)head[2], (int)head[3], t, i, chunk, p.T, p.L);
}
// The token in entry `at` of the plan's list; 0 where it holds no token.
__device__ __forceinline__ int token_at(const PoolParams &p, const PlanView &v, int64_t at) {
    return pool_row(v.token[at], p.T);
}
// Its tokens, for a lane that reads row 16 i + x of a row tile in its i-th load:
// rows past the end read the block's first (and are not written).
__device__ __forceinline__ void tile_tokens(const PoolParams &p, const PlanView &v, int64_t tile, int x, int (&token)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) token[i] = token_at(p, v, tile * kRows + 16 * i + x);
}
__device__ __forceinline__ void clamp_tokens(const Tile &t, int x, int (&token)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int first = __builtin_amdgcn_readfirstlane(token[i]);
        if (16 * i + x >= t.rows) token[i] = first;
    }
}

// ---------------------------------------------------------------------------
// loads and operands
// ---------------------------------------------------------------------------
// A wave's last step over a row of W elements begins where it ends with the row,
// so that all its loads lie in the row; `lo` is the first column that it has to
// do (the ones before it are another step's).  Only rows shorter than a step
// (FULL false) are loaded with a look at their end.
__device__ __forceinline__ int64_t step_base(int64_t lo, int step, int64_t W) {
    return W >= step ? std::min<int64_t>(lo, W - step) : lo;
}
// 16 bytes from column c of a row of n elements; past its end zero (FULL: none is)
template <bool FULL, typename T>
__device__ __forceinline__ u32x4 load16(const T *row, int64_t c, int64_t n) {
    constexpr int E = 16 / sizeof(T);
    if (FULL || c + E <= n) return *reinterpret_cast<const u32x4_any *>(row + c);
    T v[E] = {};
#pragma unroll
    for (int j = 0; j < E; ++j)
        if (c + j < n) v[j] = row[c + j];
    u32x4 r;
    __builtin_memcpy(&r, v, 16);
    return r;
}
// Columns lo .. n of 16 bytes at column c.
template <typename T>
__device__ __forceinline__ void store16(T *row, int64_t c, int64_t lo, int64_t n, u32x4 w) {
    constexpr int E = 16 / sizeof(T);
    if (c >= lo && c + E <= n) {
        *reinterpret_cast<u32x4_any *>(row + c) = w;
        return;
    }
    T v[E];
    __builtin_memcpy(v, &w, 16);
#pragma unroll
    for (int j = 0; j < E; ++j)
        if (c + j >= lo && c + j < n) row[c + j] = v[j];
}
// v with its first n elements zero
template <typename T>
__device__ __forceinline__ u32x4 zero_before(int n, u32x4 v) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if constexpr (sizeof(T) == 2)
            v[k] = n <= 2 * k ? v[k] : n == 2 * k + 1 ? v[k] & 0xffff0000u : 0u;
        else
            v[k] = n <= k ? v[k] : 0u;
    }
    return v;
}
__device__ __forceinline__ u32x4 zero_unless(bool keep, u32x4 v) {
    return u32x4{keep ? v[0] : 0u, keep ? v[1] : 0u, keep ? v[2] : 0u, keep ? v[3] : 0u};
}
// Ranks i .. of a row of r, zero past its end.  KIND 0: r fills its blocks of 16;
// 1: a multiple of 4; 2: any, with branches.
inline int rank_kind(int r) { return r % 16 == 0 ? 0 : r % 4 == 0 ? 1 : 2; }
template <int KIND>
__device__ __forceinline__ u32x4 load_ranks(const bf16 *row, int i, int r) {
    if constexpr (KIND == 1) {
        typedef u32x2 u32x2_any __attribute__((aligned(2)));
        const u32x2 lo = *reinterpret_cast<const u32x2_any *>(row + std::min(i, r - 4));
        const u32x2 hi = *reinterpret_cast<const u32x2_any *>(row + std::min(i + 4, r - 4));
        return u32x4{i < r ? lo[0] : 0u, i < r ? lo[1] : 0u, i + 4 < r ? hi[0] : 0u, i + 4 < r ? hi[1] : 0u};
    }
    return load16<KIND == 0>(row, i, r);
}
template <int KIND>
__device__ __forceinline__ u32x4 load_ranks(const float *row, int i, int r) {
    if constexpr (KIND == 1) return zero_unless(i < r, *reinterpret_cast<const u32x4_any *>(row + std::min(i, r - 4)));
    return load16<KIND == 0>(row, i, r);
}
__device__ __forceinline__ f32x4 load_f4(const float *base, int left) {
    if (left >= 4) return *reinterpret_cast<const f32x4_any *>(base);
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (j < left) v[j] = base[j];
    return v;
}
__device__ __forceinline__ void store_f4(float *base, int left, f32x4 v) {
    if (left >= 4) {
        *reinterpret_cast<f32x4_any *>(base) = v;
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (j < left) base[j] = v[j];
}

// acc += A B over the 16 bytes per lane of both: 8 bf16 (K = 32 with the four
// lane groups) or 4 f32 (K = 16)
template <typename T>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 acc) {
    if constexpr (sizeof(T) == 2) return mfma_16x16x32(as_bf16x8(a), as_bf16x8(b), acc);
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int j = 0; j < 4; ++j) acc = mfma_16x16x4_f32(x[j], y[j], acc);
    return acc;
}

// v as a sum of bf16 terms: term k rounds what the terms before it left.  A finite
// value past the largest bf16 is cut instead, one that is not finite has one term.
template <int TERMS>
__device__ __forceinline__ void split_terms(const float (&v)[8], u32x4 (&out)[TERMS]) {
    float rest[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) rest[j] = v[j];
#pragma unroll
    for (int k = 0; k < TERMS; ++k) {
        bf16x8 t;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            t[j] = f32_to_bf16(rest[j]);
            if (k == 0 && __builtin_isinf((float)t[j]) && __builtin_isfinite(rest[j]))
                t[j] = __builtin_bit_cast(bf16, (uint16_t)(__builtin_bit_cast(uint32_t, rest[j]) >> 16));
            rest[j] = __builtin_isfinite((float)t[j]) ? rest[j] - (float)t[j] : 0.f;
        }
        out[k] = as_u32x4(t);
    }
}
// A product's other operand, for the terms after the first: an infinity or NaN has
// met the whole value's in the first one already, and would make a NaN with a
// later term that is zero or of the other sign.
__device__ __forceinline__ u32x4 finite_only(u32x4 v) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t top = ((v[k] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;  // exponents of all ones
        v[k] &= ~((top >> 15) * 0xffffu);
    }
    return v;
}
// Whether some lane's values hold a NaN, or infinities of both signs.
template <int N>
__device__ __forceinline__ bool any_nan(const f32x4 (&v)[N]) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s += v[j][e];
    return __ballot(s != s) != 0;
}

// ---------------------------------------------------------------------------
// pool_down: u = A x (ROWMAJOR: the factor's rows run along the wide axis) or
// v = B^T dy (B [wide][r])
// ---------------------------------------------------------------------------
// D[rank][token]: the factor is the A operand, the tokens' rows the B operand.
// A wave takes every fourth 128-byte step of the range, two operands a lane; the
// four waves' sums are added through LDS.  64 rows a workgroup, so that the factor
// is read from L2 once per 64 rows.  Bound by x's bytes after some 5 us of
// latencies in a row: 10.6 to 12 us at 4096 x 4096 rank 16 (34 MB), 12 at
// 6000 x 2048 rank 32 (25 MB).  At ranks over 32 one wave a SIMD is left by the
// registers (f32 v over 48), and bf16 v spills 13 of them at ranks over 48:
// 4096 x 4096 rank 64 takes 18 us for u and 21 for v.
template <typename T, int RB, bool ROWMAJOR>
__global__ __launch_bounds__(256) void pool_down_kernel(PoolParams p) {
    constexpr int E = 16 / sizeof(T), STEP = 8 * E;
    __shared__ f32x4 sum[4][RB][4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, x = lane & 15, q = lane >> 4;
    const PlanView v = pool_plan_view(const_cast<int *>(p.plan), p.T, p.L);
    const int64_t at = grid_tile();
    if (at >= pool_most_tiles(p.T, p.L, kRows)) return;
    int token[4];
    tile_tokens(p, v, at, x, token);
    Tile t;
    if (!tile_of(p, v, false, at, t)) return;
    clamp_tokens(t, x, token);
    const int r = p.r, W = p.wide;
    const int64_t part = (int64_t)blockIdx.x * p.T;
    if (t.adapter < 0) {
        for (int i = threadIdx.x; i < t.rows * r; i += 256)
            p.low[(part + token_at(p, v, (int64_t)t.tile * kRows + i / r)) * r + i % r] = 0.f;
        return;
    }
    const int subs = (t.rows + 15) / 16;
    const int64_t steps = ((int64_t)W + STEP - 1) / STEP;
    const int64_t s0 = steps * blockIdx.x / gridDim.x, s1 = steps * (blockIdx.x + 1) / gridDim.x;
    const T *rows[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) rows[i] = static_cast<const T *>(p.x) + token[i] * p.ldx;
    const T *factor = static_cast<const T *>(p.factor) + (int64_t)t.adapter * r * W;
    f32x4 acc[RB][4];
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[b][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    u32x4 f[RB][2], d[4][2];
    // a factor row past the rank is the last one's again: its sums are not stored
    auto load_step = [&](auto full, int64_t lo) __attribute__((always_inline)) {
        constexpr bool FULL = decltype(full)::value;
        const int64_t base = step_base(lo, STEP, W);
        const int64_t c = base + E * q;  // its loads h: columns c + 4 E h, 64 contiguous bytes a row
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < subs) {
#pragma unroll
                for (int h = 0; h < 2; ++h) d[i][h] = load16<FULL>(rows[i], c + 4 * E * h, W);
            }
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            const int i = std::min(16 * b + x, r - 1);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if constexpr (ROWMAJOR) {
                    f[b][h] = load16<FULL>(factor + (int64_t)i * W, c + 4 * E * h, W);
                } else {
                    T w[E];
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const int64_t m = c + 4 * E * h + e;
                        w[e] = FULL || m < W ? factor[m * r + i] : (T)0.f;
                    }
                    __builtin_memcpy(&f[b][h], w, 16);
                }
            }
        }
    };
    auto load = [&](int64_t s) __attribute__((always_inline)) {
        if (W >= STEP) load_step(std::true_type{}, s * STEP);
        else load_step(std::false_type{}, s * STEP);
    };
    int64_t s = s0 + wave;
    if (s < s1) load(s);
    while (s < s1) {
        u32x4 fc[RB][2], dc[4][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int b = 0; b < RB; ++b) fc[b][h] = f[b][h];
#pragma unroll
            for (int i = 0; i < 4; ++i) dc[i][h] = d[i][h];
        }
        const int64_t lo = s * STEP, base = step_base(lo, STEP, W);
        s += 4;
        if (s < s1) load(s);
        if (base < lo)  // both operands: a product of what is not this step's must not be NaN
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int n = (int)(lo - base) - E * q - 4 * E * h;
#pragma unroll
                for (int i = 0; i < 4; ++i) dc[i][h] = zero_before<T>(n, dc[i][h]);
#pragma unroll
                for (int b = 0; b < RB; ++b) fc[b][h] = zero_before<T>(n, fc[b][h]);
            }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < subs) {
#pragma unroll
                for (int b = 0; b < RB; ++b)
#pragma unroll
                    for (int h = 0; h < 2; ++h) acc[b][i] = mfma16<T>(fc[b][h], dc[i][h], acc[b][i]);
            }
    }
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[wave][b][i][lane] = acc[b][i];
    __syncthreads();
    // wave i stores rows 16 i .. + 16: ranks 16 b + 4 q .. + 4 of token x
    if (16 * wave + x >= t.rows) return;
    const int mine = wave == 0 ? token[0] : wave == 1 ? token[1] : wave == 2 ? token[2] : token[3];
    float *out = p.low + (part + mine) * r;
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        f32x4 o = sum[0][b][wave][lane];
#pragma unroll
        for (int w = 1; w < 4; ++w) o += sum[w][b][wave][lane];
        store_f4(out + 16 * b + 4 * q, r - 16 * b - 4 * q, o);
    }
}

// ---------------------------------------------------------------------------
// pool_up: y += s B u (ROWMAJOR: the factor's rows run along the rank) or
// dx += s A^T v (A [r][wide])
// ---------------------------------------------------------------------------
// D[column][token]: a wave's step is 64 columns in four products; row 4 q + e of
// product j is column 32 (j / 2) + 8 q + 4 (j % 2) + e (f32: 16 j + 4 q + e), so
// that a lane ends with 16-byte runs of its token's row, the four lanes of a row
// with 64 bytes side by side.  Bound by y's bytes after some 5 us of latencies in a
// row (plan, low, factor, y): reading and writing y alone in this way took 43 us of
// the 48 that 6000 x 8192 rank 32 takes (196 MB of y, 4.1 TB/s; rank 64 66 us).  The
// tokens' operand stays in LDS and a step's loads follow the step before: with the
// operand in registers and the next step's loads ahead it took 54 us against 50 (low
// then in four parts).  Waves a SIMD: bf16 four up to rank 16, three up to 32, two
// above; f32 two.
constexpr int kUpStep = 64;                   // columns of a wave's step
constexpr int kUpPitch = kUpStep * 2 + 8;     // bytes of a staged bf16 factor row: 4 rows x 4 column groups hit distinct banks
constexpr int kUpPitchF = kUpStep * 4 + 16;   // the same, f32

template <typename T, int RB, bool ROWMAJOR>
struct UpLds {
    static constexpr int kPitch = sizeof(T) == 2 ? kUpPitch : kUpPitchF;
    // the tokens' operand of 16 ranks: bf16 its three terms and zeros, 32 bytes
    // each (the operands of two products); f32 as they are, 64 bytes
    static constexpr int kLow = sizeof(T) == 2 ? 128 : 64, kLowRow = RB * kLow + 16;
    __align__(16) char lowrow[kRows * kLowRow];
    __align__(16) char stage[ROWMAJOR ? 16 : 4 * RB * 16 * kPitch];
};

// Row tile `at`, the wave steps of block `block` of `blocks`.
template <typename T, int RB, bool ROWMAJOR, int KIND>
__device__ __forceinline__ void up_tile(const PoolParams &p, int64_t at, int block, int blocks,
                                        UpLds<T, RB, ROWMAJOR> &lds) {
    constexpr int E = 16 / sizeof(T), NY = 16 / E;  // elements of a load, loads of a lane's 16 columns
    constexpr int PITCH = UpLds<T, RB, ROWMAJOR>::kPitch, LOWROW = UpLds<T, RB, ROWMAJOR>::kLowRow;
    constexpr int LOW = UpLds<T, RB, ROWMAJOR>::kLow;
    char *const lowrow = lds.lowrow;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, x = lane & 15, q = lane >> 4;
    const PlanView v = pool_plan_view(const_cast<int *>(p.plan), p.T, p.L);
    if (at >= pool_most_tiles(p.T, p.L, kRows)) return;
    int token[4];
    tile_tokens(p, v, at, x, token);
    // four threads a row: its ranks 4 h .. of every 16, the parts in order
    const int h = threadIdx.x & 3, lrow = threadIdx.x >> 2;
    const int ltoken = token_at(p, v, at * kRows + lrow);
    Tile t;
    if (!tile_of(p, v, false, at, t)) return;
    clamp_tokens(t, x, token);
    const int r = p.r, W = p.wide, subs = (t.rows + 15) / 16;
    const bool live = t.adapter >= 0;
    if (!live && !(p.low_out && block == 0)) return;
    const float scale = live ? p.scale[t.adapter] : 0.f;
    const T *factor = static_cast<const T *>(p.factor) + (int64_t)(live ? t.adapter : 0) * r * W;
    T *out[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = static_cast<T *>(p.y) + token[i] * p.ldy;
    const int64_t step = (int64_t)blocks * 4 * kUpStep;
    int64_t c0 = ((int64_t)block * 4 + wave) * kUpStep;

    constexpr int RUN = 4 * E;  // columns of one load of the row's four lanes
    // column of row m of product j, and the first of the lane's load n
    auto column = [](int j, int m) { return sizeof(T) == 2 ? 32 * (j >> 1) + 8 * (m >> 2) + 4 * (j & 1) + (m & 3) : 16 * j + m; };
    u32x4 y[4][NY];
    u32x4 f[ROWMAJOR ? 4 : 1][RB];  // ROWMAJOR: the four products' operands
    u32x4 g[ROWMAJOR ? 1 : RB][ROWMAJOR ? 1 : 8 / E * 2];  // else rows as they lie, to be staged
    auto load_step = [&](auto full, int64_t col) __attribute__((always_inline)) {
        constexpr bool FULL = decltype(full)::value;
        col = step_base(col, kUpStep, W);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < subs) {
#pragma unroll
                for (int n = 0; n < NY; ++n) y[i][n] = load16<FULL>(out[i], col + RUN * n + E * q, W);
            }
        if constexpr (ROWMAJOR) {
            // of a row shorter than the step, a column past its end is the last one's again: not stored
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t c = col + column(j, x);
                const T *row = factor + (FULL ? c : std::min<int64_t>(c, W - 1)) * r;
#pragma unroll
                for (int b = 0; b < RB; ++b) {
                    const int k = sizeof(T) == 2 ? 16 * b + 8 * (q & 1) : 16 * b + 4 * q;
                    f[j][b] = load_ranks<KIND>(row, k, r);
                }
            }
        } else {
            constexpr int LANES = kUpStep / E;  // lanes of a row
#pragma unroll
            for (int b = 0; b < RB; ++b)
#pragma unroll
                for (int n = 0; n < 16 * LANES / 64; ++n) {
                    const int i = 16 * b + n * (64 / LANES) + lane / LANES;
                    const T *row = factor + (int64_t)std::min(i, r - 1) * W;
                    g[b][n] = zero_unless(i < r, load16<FULL>(row, col + E * (lane % LANES), W));
                }
        }
    };
    auto load = [&](int64_t col) __attribute__((always_inline)) {
        if (W >= kUpStep) load_step(std::true_type{}, col);
        else load_step(std::false_type{}, col);
    };
    if (live && c0 < W) load(c0);
    {
        f32x4 s[RB];
#pragma unroll
        for (int b = 0; b < RB; ++b) s[b] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (lrow < t.rows)
#pragma unroll 4
            for (int k = 0; k < p.splits; ++k)
#pragma unroll
                for (int b = 0; b < RB; ++b)
                    s[b] += __builtin_bit_cast(
                        f32x4, load_ranks<KIND>(p.low + ((int64_t)k * p.T + ltoken) * r, 16 * b + 4 * h, r));
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            if (p.low_out && block == 0 && lrow < t.rows)  // the parts' sum, for the backward
                store_f4(p.low_out + (int64_t)ltoken * r + 16 * b + 4 * h, r - 16 * b - 4 * h, s[b]);
            s[b] *= scale;
            char *d = lowrow + lrow * LOWROW + LOW * b;
            if constexpr (sizeof(T) == 2) {
                const float w[8] = {s[b][0], s[b][1], s[b][2], s[b][3], 0.f, 0.f, 0.f, 0.f};
                u32x4 terms[3];
                split_terms(w, terms);
#pragma unroll
                for (int k = 0; k < 3; ++k)
                    *reinterpret_cast<u32x2 *>(d + 32 * k + 8 * h) = u32x2{terms[k][0], terms[k][1]};
                *reinterpret_cast<u32x2 *>(d + 96 + 8 * h) = u32x2{0, 0};
            } else {
                *reinterpret_cast<f32x4 *>(d + 16 * h) = s[b];
            }
        }
    }
    if (!live) return;
    __syncthreads();
    char *mine = lds.stage + (ROWMAJOR ? 0 : wave * RB * 16 * PITCH);
    while (c0 < W) {
        u32x4 fc[4][RB];
        if constexpr (ROWMAJOR) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int b = 0; b < RB; ++b) fc[j][b] = f[j][b];
        } else {
            // through LDS of the wave's own: row i of the factor's 64 columns
            constexpr int LANES = kUpStep / E;
#pragma unroll
            for (int b = 0; b < RB; ++b)
#pragma unroll
                for (int n = 0; n < 16 * LANES / 64; ++n) {
                    char *d = mine + (16 * b + n * (64 / LANES) + lane / LANES) * PITCH + 16 * (lane % LANES);
                    *reinterpret_cast<u32x2 *>(d) = u32x2{g[b][n][0], g[b][n][1]};
                    *reinterpret_cast<u32x2 *>(d + 8) = u32x2{g[b][n][2], g[b][n][3]};
                }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int b = 0; b < RB; ++b) {
                    if constexpr (sizeof(T) == 2) {
                        // lane 4 e + k of 16 points at row e, the column of product row 4 k; lane m
                        // receives the column of product row m in the four rows
                        const uint32_t src = (16 * b + 8 * (q & 1) + (x >> 2)) * PITCH + column(j, 4 * (x & 3)) * 2;
                        fc[j][b] = as_u32x4(lds_read_col_frag(mine, src, src + 4 * PITCH));
                    } else {
                        const float *src = reinterpret_cast<const float *>(mine);
                        f32x4 w;
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            w[e] = src[(16 * b + 4 * q + e) * (PITCH / 4) + column(j, x)];
                        fc[j][b] = __builtin_bit_cast(u32x4, w);
                    }
                }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        const int64_t lo = c0, c = step_base(c0, kUpStep, W) + E * q;
        c0 += step;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i >= subs) continue;
            // bf16: lane groups 0 and 1 the first terms of 16 ranks, 2 and 3 the second, in
            // another product the third and zeros; f32: ranks 4 q ..
            constexpr int PARTS = LOW / 64;
            f32x4 acc[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < PARTS; ++k) {
                u32x4 low[RB];
#pragma unroll
                for (int b = 0; b < RB; ++b)
                    low[b] = *reinterpret_cast<const u32x4 *>(lowrow + (16 * i + x) * LOWROW + LOW * b + 64 * k + 16 * q);
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int b = 0; b < RB; ++b) acc[j] = mfma16<T>(fc[j][b], low[b], acc[j]);
            }
            if constexpr (sizeof(T) == 2)
                if (__builtin_expect(any_nan(acc), 0)) {  // perhaps of an infinity in the factor; the same sums, in the same order
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int k = 0; k < PARTS; ++k)
#pragma unroll
                        for (int b = 0; b < RB; ++b) {
                            const u32x4 low = *reinterpret_cast<const u32x4 *>(lowrow + (16 * i + x) * LOWROW + LOW * b +
                                                                               64 * k + 16 * q);
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                acc[j] = mfma16<T>(k == 0 && q < 2 ? fc[j][b] : finite_only(fc[j][b]), low, acc[j]);
                                __builtin_amdgcn_sched_barrier(0);  // one operand's registers at a time
                            }
                        }
                }
            if (16 * i + x >= t.rows) continue;
#pragma unroll
            for (int n = 0; n < NY; ++n) {
                if constexpr (sizeof(T) == 2) {
                    const bf16x8 old = as_bf16x8(y[i][n]);
                    bf16x8 o;
#pragma unroll
                    for (int e = 0; e < 8; ++e) o[e] = f32_to_bf16((float)old[e] + acc[2 * n + e / 4][e % 4]);
                    store16(out[i], c + RUN * n, lo, W, as_u32x4(o));
                } else {
                    store16(out[i], c + RUN * n, lo, W,
                            __builtin_bit_cast(u32x4, __builtin_bit_cast(f32x4, y[i][n]) + acc[n]));
                }
            }
        }
        if (c0 < W) load(c0);
    }
}

// Two waves a SIMD asked for, which all of its forms reach without spills: left to
// itself the compiler takes 258 to 271 registers for some at ranks over 48, one wave,
// 87 us against 63 at 6000 x 8192 rank 56.
template <typename T, int RB, int KIND>
__global__ __launch_bounds__(256, 2) void pool_up_kernel(PoolParams p) {
    __shared__ UpLds<T, RB, true> lds;
    up_tile<T, RB, true, KIND>(p, grid_tile(), blockIdx.x, gridDim.x, lds);
}

// ---------------------------------------------------------------------------
// gradients: sum over a chunk's rows of low[row][i] * wide[row][c], for pool_back
// ---------------------------------------------------------------------------
// D[rank][column]: the A operand is low (lane: rank), the B operand the wide
// rows (lane: column), both with the rows as k.  A lane loads 16 bytes of a row:
// bf16, 8 columns of 8 rows (32 rows per step), whose elements j make product
// j's operand: columns 8 x + j.  f32: 4 columns of one row, 4 rows a step.
//
// The chunk's tokens and its low, as the bf16 products take it (three terms,
// [rank block][term][32-row step][lane group][rank][8 rows]) or in f32 ([row][rank
// + 1 pad]), lie in LDS for all waves.  Two pairs of waves take every other step
// each; the second's sums are added through LDS.  A chunk is 256 rows: a partial
// sum of r x 256 f32 is then at most r / 128 of the bytes read for it.  Bound by the
// wide rows' bytes: 16 us alone at 4096 x 4096 rank 16, both gradients (67 MB).
constexpr int kGradRows = 32;  // of a step

template <typename T, int RB>
struct GradLds {
    int token[kChunk];
    union {
        u32x4 terms[sizeof(T) == 2 ? RB * 3 * kChunk * 2 : 1];  // 16 ranks x kChunk rows = 2 kChunk vectors of 8
        float low[sizeof(T) == 2 ? 1 : kChunk][RB * 16 + 1];
        f32x4 sum[2][RB][16 / sizeof(T)][64];
    };
};

template <typename T, int RB>
__device__ __forceinline__ void grad_chunk(const PoolGradParams &g, const PoolParams &p, const PlanView &v,
                                           const Tile &t, int block, GradLds<T, RB> &lds) {
    constexpr int E = 16 / sizeof(T), ROWS = 8;  // columns and rows of a lane's step
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, x = lane & 15, q = lane >> 4;
    const int pair = wave >> 1;
    const int r = p.r, W = p.wide;
    const int64_t lo = ((int64_t)block * 2 + (wave & 1)) * 16 * E, c = step_base(lo, 16 * E, W) + E * x;
    const int steps = (t.rows + kGradRows - 1) / kGradRows;
    {
        // rows past the end: the first one's token, negative (~token)
        const int i = threadIdx.x;
        const int token = token_at(p, v, (int64_t)t.tile * kRows + (i < t.rows ? i : 0));
        lds.token[i] = i < t.rows ? token : ~token;
    }
    __syncthreads();
    u32x4 d[ROWS];
    // bf16: rows 8 q + e of the step; f32: rows 4 e + q
    auto load_rows = [&](auto full, int s) __attribute__((always_inline)) {
        constexpr bool FULL = decltype(full)::value;
#pragma unroll
        for (int e = 0; e < ROWS; ++e) {
            const int token = lds.token[s * kGradRows + (sizeof(T) == 2 ? 8 * q + e : 4 * e + q)];
            const T *row = static_cast<const T *>(p.x) + (token < 0 ? ~token : token) * p.ldx;
            d[e] = zero_unless(token >= 0, load16<FULL>(row, c, W));
        }
    };
    auto load_wide = [&](int s) __attribute__((always_inline)) {
        if (W >= 16 * E) load_rows(std::true_type{}, s);
        else load_rows(std::false_type{}, s);
    };
    const bool any = lo < W;
    if (any && pair < steps) load_wide(pair);
    if constexpr (sizeof(T) == 2) {
        // thread: rank i % 16, rows 8 (i / 16) .. + 8
#pragma unroll
        for (int n = 0; n < 2 * kChunk / 256; ++n) {
            const int i = n * 256 + threadIdx.x;
            const int rank = i % 16, row = i / 16 * 8;
            float low[RB][8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int token = lds.token[row + e];
                const float *src = p.low + (int64_t)(token < 0 ? ~token : token) * r;
#pragma unroll
                for (int b = 0; b < RB; ++b) low[b][e] = src[std::min(16 * b + rank, r - 1)];
            }
            for (int k = 1; k < p.splits; ++k)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int token = lds.token[row + e];
                    const float *src = p.low + ((int64_t)k * p.T + (token < 0 ? ~token : token)) * r;
#pragma unroll
                    for (int b = 0; b < RB; ++b) low[b][e] += src[std::min(16 * b + rank, r - 1)];
                }
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int b = 0; b < RB; ++b)
                    low[b][e] = lds.token[row + e] >= 0 && 16 * b + rank < r ? low[b][e] : 0.f;
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                u32x4 terms[3];
                split_terms(low[b], terms);
#pragma unroll
                for (int k = 0; k < 3; ++k) lds.terms[(b * 3 + k) * 2 * kChunk + i] = terms[k];
            }
        }
    } else {
#pragma unroll 16
        for (int n = 0; n < RB * 16; ++n) {
            const int i = n * 256 + threadIdx.x, row = i / (RB * 16), rank = i % (RB * 16), token = lds.token[row];
            const float *src = p.low + (int64_t)(token < 0 ? ~token : token) * r + std::min(rank, r - 1);
            float w = src[0];
            for (int k = 1; k < p.splits; ++k) w += src[(int64_t)k * p.T * r];
            lds.low[row][rank] = token >= 0 && rank < r ? w : 0.f;
        }
    }
    __syncthreads();
    f32x4 acc[RB][E];
    // FINITE: the terms after the first take no infinities of the rows
    auto products = [&](auto finite) __attribute__((always_inline)) {
        constexpr bool FINITE = decltype(finite)::value;
#pragma unroll
        for (int b = 0; b < RB; ++b)
#pragma unroll
            for (int j = 0; j < E; ++j) acc[b][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int s = pair; s < steps; s += 2) {
            u32x4 w[ROWS];
#pragma unroll
            for (int e = 0; e < ROWS; ++e) w[e] = d[e];
            if (s + 2 < steps) load_wide(s + 2);
            if constexpr (sizeof(T) == 2) {
                bf16x8 low[RB][3];
#pragma unroll
                for (int b = 0; b < RB; ++b)
#pragma unroll
                    for (int k = 0; k < 3; ++k)
                        low[b][k] = as_bf16x8(lds.terms[(b * 3 + k) * 2 * kChunk + (s * 4 + q) * 16 + x]);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    bf16x8 col;
#pragma unroll
                    for (int e = 0; e < 8; ++e) col[e] = as_bf16x8(w[e])[j];
                    const bf16x8 rest = FINITE ? as_bf16x8(finite_only(as_u32x4(col))) : col;
#pragma unroll
                    for (int b = 0; b < RB; ++b)
#pragma unroll
                        for (int k = 0; k < 3; ++k) acc[b][j] = mfma_16x16x32(low[b][k], k ? rest : col, acc[b][j]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < ROWS; ++e) {
                    const f32x4 col = __builtin_bit_cast(f32x4, w[e]);
#pragma unroll
                    for (int b = 0; b < RB; ++b) {
                        const float low = lds.low[s * kGradRows + 4 * e + q][16 * b + x];
#pragma unroll
                        for (int j = 0; j < 4; ++j) acc[b][j] = mfma_16x16x4_f32(low, col[j], acc[b][j]);
                    }
                }
            }
        }
    };
    if (any) {
        products(std::false_type{});
        if constexpr (sizeof(T) == 2) {
            bool nan = false;
#pragma unroll
            for (int b = 0; b < RB; ++b) nan |= any_nan(acc[b]);
            if (__builtin_expect(nan, 0)) {
                if (pair < steps) load_wide(pair);
                products(std::true_type{});
            }
        }
    }
    __syncthreads();
    if (pair == 1)
#pragma unroll
        for (int b = 0; b < RB; ++b)
#pragma unroll
            for (int j = 0; j < E; ++j) lds.sum[wave & 1][b][j][lane] = acc[b][j];
    __syncthreads();
    if (pair == 1 || !any) return;
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int j = 0; j < E; ++j) acc[b][j] += lds.sum[wave][b][j][lane];
    const int64_t slot = pool_grad_place(t.slot, v.slot0[t.adapter], g.slots);
    if (slot == kPoolNowhere) return;  // not of a plan that this library made
    float *out = slot >= 0 ? g.part + slot * r * W : g.out + t.adapter * (int64_t)r * W;
    const float scale = slot >= 0 ? 1.f : p.scale[t.adapter];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        const int i = 16 * b + 4 * q;
        if (g.transpose) {  // [wide][r]
#pragma unroll
            for (int j = 0; j < E; ++j)
                if (c + j >= lo && c + j < W) store_f4(out + (c + j) * r + i, r - i, acc[b][j] * scale);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (i + e >= r) continue;
                float *row = out + (int64_t)(i + e) * W;
#pragma unroll
                for (int j = 0; j < E; j += 4)
                    store16(row, c + j, lo, W,
                            __builtin_bit_cast(u32x4, f32x4{acc[b][j][e], acc[b][j + 1][e], acc[b][j + 2][e],
                                                            acc[b][j + 3][e]} * scale));
            }
        }
    }
}

// dx, dA and dB in one launch: grid rows up to dx's row tiles, behind them the
// gradients' (chunk, column block) pairs one after another.  A launch after
// another costs some 5 us in which no memory is busy: 4096 x 4096 rank 16 took 17
// and 16 us in two launches, 30 in this one (x, dy, dx twice: 134 MB), 33 with the
// gradients first; 300 tokens 5 and 6.4, 7.3 in one.  Infinities kept, it takes 32
// (4.2 TB/s) and 7.9.  Both parts share the registers and the larger LDS, the
// gradients': three waves a SIMD in bf16 up to rank 16, two up to 32, one above (f32
// two up to rank 32, one above), also for dx.  4096 x 4096 bf16: rank 32 41 us, 48
// 65, 64 77; 2048 x 2048 f32: rank 16 29, 64 110.  Two launches were not measured
// at these ranks.
template <typename T, int RB, int KIND>
__global__ __launch_bounds__(256) void pool_back_kernel(PoolParams px, PoolParams pa, PoolGradParams ga, PoolParams pb,
                                                        PoolGradParams gb) {
    __shared__ union {
        GradLds<T, RB> grad;
        UpLds<T, RB, false> up;
    } lds;
    const int64_t tiles = px.y ? pool_most_tiles(px.T, px.L, kRows) : 0, at = grid_tile() - tiles;
    if (at < 0) {
        up_tile<T, RB, false, KIND>(px, at + tiles, blockIdx.x, gridDim.x, lds.up);
        return;
    }
    if (!ga.out) return;  // the grid's last rows, of a call for dx alone
    const PlanView v = pool_plan_view(const_cast<int *>(pa.plan), pa.T, pa.L);
    const int64_t i = at * gridDim.x + blockIdx.x, chunk = i / (ga.blocks + gb.blocks);
    const int block = (int)(i - chunk * (ga.blocks + gb.blocks));
    Tile t;
    if (chunk >= pool_most_tiles(pa.T, pa.L, kChunk) || !tile_of(pa, v, true, chunk, t) || t.adapter < 0) return;
    if (block < ga.blocks)
        grad_chunk<T, RB>(ga, pa, v, t, block, lds.grad);
    else
        grad_chunk<T, RB>(gb, pb, v, t, block - ga.blocks, lds.grad);
}

// Adapters of several chunks: the partial sums in order, times the scale;
// adapters without tokens: zeros.  grid (adapters, groups of 1024 elements, dA or dB).
// Latency-bound: 5.1 us for 20 chunks of 4 adapters at 4096 x 4096 rank 16 (10 MB).
__global__ __launch_bounds__(256) void pool_reduce_kernel(PoolParams p, PoolGradParams ga, PoolGradParams gb,
                                                          int64_t na, int64_t nb) {
    const int a = blockIdx.x;
    const PlanView v = pool_plan_view(const_cast<int *>(p.plan), p.T, p.L);
    const int first = v.slot0[a];
    const int64_t chunks = pool_partials(v.head[2], v.head[3], v.count[a], first, ga.slots, p.T, p.L);
    if (chunks < 0) return;
    const float scale = p.scale[a];
    const int64_t size = blockIdx.z ? nb : na;
    const float *part = (blockIdx.z ? gb.part : ga.part) + first * size;
    float *out = (blockIdx.z ? gb.out : ga.out) + a * size;
    for (int64_t e = ((int64_t)blockIdx.y * 256 + threadIdx.x) * 4; e < size; e += (int64_t)gridDim.y * 1024) {
        const int left = (int)std::min<int64_t>(4, size - e);
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int64_t k = 0; k < chunks; ++k) s += load_f4(part + k * size + e, left);
        store_f4(out + e, left, chunks ? s * scale : s);
    }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
// Ranges of the wide axis: about a workgroup a CU, a power of two so that the
// waves' steps divide evenly, none under 256 columns.  us of down + up, 6000 x 2048
// -> 8192 rank 32 (107 tiles): one range 63, two 59, four 63, eight 68; of both
// down, up and back, 4096 x 4096 rank 16 (69 tiles): one 103, two 82, four 74, eight 78.
int down_splits(int T, int L, int W) {
    const int64_t tiles = std::max<int64_t>(1, pool_most_tiles(T, L, kRows));
    const int64_t want = ((int64_t)device_cu_count() + tiles - 1) / tiles;
    int64_t splits = 1;
    while (2 * splits <= std::min<int64_t>(std::min<int64_t>(want, 64), W / 256)) splits *= 2;
    return (int)splits;
}
size_t align256(size_t x) { return (x + 255) & ~size_t(255); }
size_t low_bytes(int T, int r, int splits) { return align256((size_t)splits * T * r * sizeof(float)); }

template <typename T, bool ROWMAJOR>
hipError_t down_t(const PoolParams &p, hipStream_t s) {
    const dim3 grid = tile_grid(p.splits, pool_most_tiles(p.T, p.L, kRows)), block(256);
    switch ((p.r + 15) / 16) {
        case 1: hipLaunchKernelGGL((pool_down_kernel<T, 1, ROWMAJOR>), grid, block, 0, s, p); break;
        case 2: hipLaunchKernelGGL((pool_down_kernel<T, 2, ROWMAJOR>), grid, block, 0, s, p); break;
        case 3: hipLaunchKernelGGL((pool_down_kernel<T, 3, ROWMAJOR>), grid, block, 0, s, p); break;
        default: hipLaunchKernelGGL((pool_down_kernel<T, 4, ROWMAJOR>), grid, block, 0, s, p); break;
    }
    return hipGetLastError();
}
// Workgroups over a row of pool_up: two steps a wave where one each would not all
// fit the chip at once (three workgroups a CU)
int64_t up_blocks(int64_t tiles, int wide) {
    const int64_t blocks = ((int64_t)wide + 4 * kUpStep - 1) / (4 * kUpStep);
    return tiles * blocks > 3 * (int64_t)device_cu_count() ? (blocks + 1) / 2 : blocks;
}
template <typename T, int KIND>
hipError_t up_kind(const PoolParams &p, hipStream_t s) {
    const int64_t tiles = pool_most_tiles(p.T, p.L, kRows);
    const dim3 grid = tile_grid(up_blocks(tiles, p.wide), tiles), block(256);
    switch ((p.r + 15) / 16) {
        case 1: hipLaunchKernelGGL((pool_up_kernel<T, 1, KIND>), grid, block, 0, s, p); break;
        case 2: hipLaunchKernelGGL((pool_up_kernel<T, 2, KIND>), grid, block, 0, s, p); break;
        case 3: hipLaunchKernelGGL((pool_up_kernel<T, 3, KIND>), grid, block, 0, s, p); break;
        default: hipLaunchKernelGGL((pool_up_kernel<T, 4, KIND>), grid, block, 0, s, p); break;
    }
    return hipGetLastError();
}
template <typename T>
hipError_t up_t(const PoolParams &p, hipStream_t s) {
    switch (rank_kind(p.r)) {
        case 0: return up_kind<T, 0>(p, s);
        case 1: return up_kind<T, 1>(p, s);
        default: return up_kind<T, 2>(p, s);
    }
}
template <typename T, int KIND>
hipError_t back_kind(const PoolParams &px, const PoolParams &pa, const PoolGradParams &ga, const PoolParams &pb,
                     const PoolGradParams &gb, hipStream_t s) {
    const int64_t tiles = px.y ? pool_most_tiles(px.T, px.L, kRows) : 0;
    const int64_t pairs = ga.out ? pool_most_tiles(pa.T, pa.L, kChunk) * (ga.blocks + gb.blocks) : 0;
    const int64_t columns = tiles ? up_blocks(tiles, px.wide) : ga.blocks + gb.blocks;
    const dim3 grid = tile_grid(columns, tiles + (pairs + columns - 1) / columns), block(256);
    switch ((px.r + 15) / 16) {
        case 1: hipLaunchKernelGGL((pool_back_kernel<T, 1, KIND>), grid, block, 0, s, px, pa, ga, pb, gb); break;
        case 2: hipLaunchKernelGGL((pool_back_kernel<T, 2, KIND>), grid, block, 0, s, px, pa, ga, pb, gb); break;
        case 3: hipLaunchKernelGGL((pool_back_kernel<T, 3, KIND>), grid, block, 0, s, px, pa, ga, pb, gb); break;
        default: hipLaunchKernelGGL((pool_back_kernel<T, 4, KIND>), grid, block, 0, s, px, pa, ga, pb, gb); break;
    }
    return hipGetLastError();
}
template <typename T>
hipError_t back_t(const PoolParams &px, const PoolParams &pa, const PoolGradParams &ga, const PoolParams &pb,
                  const PoolGradParams &gb, hipStream_t s) {
    switch (rank_kind(px.r)) {
        case 0: return back_kind<T, 0>(px, pa, ga, pb, gb, s);
        case 1: return back_kind<T, 1>(px, pa, ga, pb, gb, s);
        default: return back_kind<T, 2>(px, pa, ga, pb, gb, s);
    }
}

}  // namespace

hipError_t prepare_pool_kernels() {
    return hipFuncSetAttribute(reinterpret_cast<const void *>(&pool_plan_kernel),
                               hipFuncAttributeMaxDynamicSharedMemorySize,
                               plan_lds_words(kPlanKept + 1, kPoolMaxAdapters) * (int)sizeof(int));
}

size_t pool_plan_bytes(int T, int L) { return (size_t)pool_plan_words(T, L) * sizeof(int); }

hipError_t launch_pool_plan(const int *index, int T, int L, int *plan, hipStream_t s) {
    const size_t lds = (size_t)plan_lds_words(T, L) * sizeof(int);
    hipLaunchKernelGGL(pool_plan_kernel, dim3(1), dim3(1024), lds, s, index, T, L, 32 - __builtin_clz(L), plan);
    return hipGetLastError();
}

size_t pool_fwd_workspace_bytes(const PoolCall &c) {
    const int splits = down_splits(c.T, c.L, c.K);
    return splits > 1 ? low_bytes(c.T, c.r, splits) : 0;
}

size_t pool_bwd_workspace_bytes(const PoolCall &c) {
    const int splits = down_splits(c.T, c.L, c.M);
    return low_bytes(c.T, c.r, splits) +
           align256((size_t)pool_grad_slots(c.T, c.L) * c.r * ((size_t)c.K + c.M) * sizeof(float));
}

static PoolParams pool_params(const PoolCall &c) {
    PoolParams p{};
    p.plan = c.plan;
    p.scale = c.scale;
    p.T = c.T;
    p.L = c.L;
    p.r = c.r;
    return p;
}

hipError_t launch_pool_fwd(const PoolCall &c, int dtype, hipStream_t s) {
    if (c.T == 0) return hipSuccess;
    PoolParams p = pool_params(c);
    p.splits = down_splits(c.T, c.L, c.K);
    p.x = c.x;
    p.ldx = c.ldx;
    p.factor = c.a;
    p.wide = c.K;
    p.low = p.splits > 1 ? static_cast<float *>(c.work) : c.u;
    hipError_t e = dtype == 0 ? down_t<bf16, true>(p, s) : down_t<float, true>(p, s);
    if (e != hipSuccess) return e;
    p.factor = c.b;
    p.wide = c.M;
    p.y = c.y;
    p.ldy = c.ldy;
    p.low_out = p.splits > 1 ? c.u : nullptr;
    return dtype == 0 ? up_t<bf16>(p, s) : up_t<float>(p, s);
}

hipError_t launch_pool_bwd(const PoolCall &c, int dtype, hipStream_t s) {
    const bool bf = dtype == 0;
    PoolParams pv = pool_params(c);  // v, from dy
    pv.splits = down_splits(c.T, c.L, c.M);
    pv.low = static_cast<float *>(c.work);
    hipError_t e = hipSuccess;
    PoolParams pa = pv, pb = pv;  // the gradients' products
    PoolGradParams ga{}, gb{};
    // workspace: v's parts, the partial gradients
    float *part = reinterpret_cast<float *>(static_cast<char *>(c.work) + low_bytes(c.T, c.r, pv.splits));
    const int64_t na = (int64_t)c.r * c.K, nb = (int64_t)c.r * c.M;
    const int cols = bf ? 256 : 128;
    ga.out = c.da;
    ga.slots = gb.slots = (int)pool_grad_slots(c.T, c.L);
    ga.part = part;
    ga.blocks = (c.K + cols - 1) / cols;
    gb.out = c.db;
    gb.part = part + ga.slots * na;
    gb.blocks = (c.M + cols - 1) / cols;
    gb.transpose = 1;
    if (c.T > 0) {
        pv.x = c.dy;
        pv.ldx = c.lddy;
        pv.factor = c.b;
        pv.wide = c.M;
        if ((e = bf ? down_t<bf16, false>(pv, s) : down_t<float, false>(pv, s)) != hipSuccess) return e;
        PoolParams px = pv;
        px.factor = c.a;
        px.wide = c.K;
        px.y = c.dx;
        px.ldy = c.lddx;
        pa.x = c.x;
        pa.ldx = c.ldx;
        pa.wide = c.K;
        pb.x = c.dy;
        pb.ldx = c.lddy;
        pb.wide = c.M;
        pb.low = c.u;
        pb.splits = 1;
        if ((c.dx || c.da) &&
            (e = bf ? back_t<bf16>(px, pa, ga, pb, gb, s) : back_t<float>(px, pa, ga, pb, gb, s)) != hipSuccess)
            return e;
    }
    if (!c.da) return hipSuccess;
    const int64_t per = (std::max(na, nb) + 1023) / 1024;
    hipLaunchKernelGGL(pool_reduce_kernel, dim3(c.L, (unsigned)std::min<int64_t>(per, 1024), 2), dim3(256), 0, s, pa,
                       ga, gb, na, nb);
    return hipGetLastError();
}

}  // namespace fa
