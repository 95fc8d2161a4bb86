// An optimiser step with an orthogonalised update, over many low-rank matrices
// (LoRA factors) at once.  For each matrix, r = min(rows, cols) <= 64 and n the
// long side:
//   m = beta * m + g;   u = nesterov ? g + beta * m : m
//   X_0 = u / (|u|_F + eps);   X_k+1 = a X_k + (b S + c S^2) X_k,  S = X_k X_k^T
//   p = p * (1 - lr * decay) - lr * scale * X_steps
// (the optimiser published as Muon, Jordan and others, 2024; the iteration is of
// Newton-Schulz type, its usual coefficients the caller's to pass).
// Every X_k is T_k X_0 with T_k a polynomial in G_0 = X_0 X_0^T, an r x r matrix:
//   Q_k = a I + b G_k + c G_k^2,   G_k+1 = Q_k G_k Q_k,   T_k+1 = Q_k T_k,
// so the long side is passed over twice, once for u u^T and once for T u, and
// the iteration stays on r x r.  All of its matrices are polynomials in G_0, so
// they are symmetric and commute.  G has the squares of X's singular values, and
// a step grows what rounding leaves in its small ones by up to a^2: the Gram
// sums and the r x r products are f64 (f32 would leave 1e-7 * a^(2 steps),
// several percent for singular values under 1e-3 of the largest).  T is rounded
// to f32 once, and T u is f32.
//
// Three launches: muon_gram_kernel (momentum, and u u^T over a chunk of the long
// side), muon_solve_kernel (a workgroup per matrix: chunks added in order, then
// the iteration), muon_apply_kernel.  No atomics: the same bits every time.
//
// f64 products are v_mfma_f64_16x16x4: A[m][k] in lane m + 16 k, B[k][n] in lane
// n + 16 k, D element i of lane l is D[4 i + l / 16][l % 16].  An operand read
// from a D tile's registers, element t for step t, holds rows 4 t + l / 16 of the
// tile in lane order l % 16: the B operand as it lies, and (the matrix being
// symmetric) the A operand of the mirrored tile.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "fa_device.hpp"
#include "fa_kernels.hpp"

namespace fa {
namespace {

typedef double f64x4 __attribute__((ext_vector_type(4)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));

__device__ __forceinline__ f64x4 mfma_f64(double a, double b, f64x4 c) {
    return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0);
}

constexpr int kTile = 256;  // elements of a 16 x 16 tile

// The matrix and chunk of block b: items' blocks are numbered one after another,
// per item matrix by matrix.
struct Place {
    int item, chunk;
    int64_t matrix;  // within the item
    int slot;        // over all items
};
__device__ __forceinline__ Place place_of(const MuonMany &p, int b) {
    int k = 0, end = p.items - 1;  // the last item that begins at or before b
    while (k < end) {
        const int mid = (k + end + 1) / 2;
        if (p.block0[mid] <= b) k = mid;
        else end = mid - 1;
    }
    const int local = b - p.block0[k];
    Place w;
    w.item = k;
    w.matrix = local / p.chunks[k];
    w.chunk = local - (int)w.matrix * p.chunks[k];
    w.slot = p.matrix0[k] + (int)w.matrix;
    return w;
}

// Four elements of the long side of row i, from column j, each at `step` from
// the last; zero outside r x n.
__device__ __forceinline__ f32x4 load4(const float *base, int64_t at, int64_t step, int left) {
    if (step == 1 && left >= 4) return *reinterpret_cast<const f32x4_any *>(base + at);
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < left) v[e] = base[at + e * step];
    return v;
}
__device__ __forceinline__ f32x4 load_full(const float *base, int64_t at, int64_t step) {
    if (step == 1) return *reinterpret_cast<const f32x4_any *>(base + at);
    return f32x4{base[at], base[at + step], base[at + 2 * step], base[at + 3 * step]};
}
__device__ __forceinline__ void store4(float *base, int64_t at, int64_t step, int left, f32x4 v) {
    if (step == 1 && left >= 4) {
        *reinterpret_cast<f32x4_any *>(base + at) = v;
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < left) base[at + e * step] = v[e];
}

// Momentum and the chunk's part of u u^T.  Wave w takes every fourth 16-column
// step of the chunk; lane l holds row 16 b + l % 16 of each of the RB row blocks
// and the step's columns 4 (l / 16) .. + 4.  Bound by HBM: 51.5 us for the
// f32 factors of 64 projections 2048 -> 8192 of rank 32, 21 M elements (read g and
// m, write m: 252 MB, 4.9 TB/s); at rank 64 by the f64 MFMA, 16 us for 8 matrices
// of 4096 columns.
template <int RB>
__global__ __launch_bounds__(256) void muon_gram_kernel(MuonMany p) {
    constexpr int NT = RB * (RB + 1) / 2;
    __shared__ double sum[4][NT * kTile];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Place at = place_of(p, blockIdx.x);
    const int k = at.item, r = p.r[k], n = p.n[k];
    const bool wide = p.wide[k];
    const int64_t off = at.matrix * (int64_t)r * n;
    const float *g = p.grad[k] + off;
    float *m = p.m[k] + off;
    const int64_t rs = wide ? n : 1, cs = wide ? 1 : r;  // strides of a row and of a column of the r x n matrix
    const int j0 = at.chunk * p.chunk[k], j1 = min(n, j0 + p.chunk[k]);
    const float beta = p.beta;
    f64x4 acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = f64x4{0, 0, 0, 0};
    // AT_ONCE steps at once: their loads go out side by side.  FULL: all of the
    // steps' columns and rows are there, and the loads need no branches.
    auto do_steps = [&](auto full, auto at_once, int j) __attribute__((always_inline)) {
        constexpr bool FULL = decltype(full)::value;
        constexpr int STEPS = decltype(at_once)::value;
        f32x4 gv[STEPS][RB], mv[STEPS][RB];
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                const int i = 16 * b + (lane & 15), jl = j + 64 * s + 4 * (lane >> 4);
                const int64_t e = i * rs + jl * cs;
                const int left = i < r ? j1 - jl : 0;
                gv[s][b] = FULL ? load_full(g, e, cs) : load4(g, e, cs, left);
                mv[s][b] = FULL ? load_full(m, e, cs) : load4(m, e, cs, left);
            }
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            f32x4 u[RB];
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                const int i = 16 * b + (lane & 15), jl = j + 64 * s + 4 * (lane >> 4);
                f32x4 mn;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    mn[q] = __builtin_fmaf(beta, mv[s][b][q], gv[s][b][q]);
                    u[b][q] = p.nesterov ? __builtin_fmaf(beta, mn[q], gv[s][b][q]) : mn[q];
                }
                store4(m, i * rs + jl * cs, cs, FULL ? 4 : i < r ? j1 - jl : 0, mn);
            }
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int b = 0, t = 0; b < RB; ++b)
#pragma unroll
                    for (int c = b; c < RB; ++c, ++t) acc[t] = mfma_f64((double)u[b][q], (double)u[c][q], acc[t]);
        }
    };
    constexpr int AT_ONCE = RB <= 2 ? 2 : 1;
    int j = j0 + wave * 16;
    if (r == 16 * RB)
        for (; j + 64 * (AT_ONCE - 1) + 16 <= j1; j += 64 * AT_ONCE)
            do_steps(std::true_type{}, std::integral_constant<int, AT_ONCE>{}, j);
    for (; j < j1; j += 64) do_steps(std::false_type{}, std::integral_constant<int, 1>{}, j);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[wave][t * kTile + i * 64 + lane] = acc[t][i];
    __syncthreads();
    double *out = p.gram + (p.gram0[k] + (at.matrix * p.chunks[k] + at.chunk) * (int64_t)(NT * kTile));
    for (int i = threadIdx.x; i < NT * kTile; i += 256) out[i] = sum[0][i] + sum[1][i] + sum[2][i] + sum[3][i];
}

// T of one matrix.  Element i of a tile in lane l is (row 4 i + l / 16, column
// l % 16).  Of up to 2 x 2 tiles each wave owns one (one alone stays in its
// wave's registers), of more a column of them.  Bound by the latency of the
// products one after another (four a step, three deep, an MFMA 64 cycles): 128
// matrices of rank 32 take 13.8 us, two of rank 16 6.9.  Only the tiles on and above the diagonal, mirrored
// in LDS, would be 10 of 16 products at rank 64, but measured 52 us against 47.
template <int RB>
__global__ __launch_bounds__(256) void muon_solve_kernel(MuonMany p) {
    constexpr int NT = RB * (RB + 1) / 2, ALL = RB * RB * kTile;
    constexpr int OWN = RB <= 2 ? 1 : RB, WAVES = RB * RB / OWN;  // tiles of a wave, waves that have some
    extern __shared__ double lds[];  // G, Q, T and H = G Q, each [RB][RB] tiles of [4][64]
    double *G = lds, *Q = lds + ALL, *T = lds + 2 * ALL, *H = lds + 3 * ALL;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int k = 0, end = p.items - 1;
    while (k < end) {
        const int mid = (k + end + 1) / 2;
        if (p.matrix0[mid] <= (int)blockIdx.x) k = mid;
        else end = mid - 1;
    }
    const int64_t matrix = blockIdx.x - p.matrix0[k];
    const int chunks = p.chunks[k];
    const double *part = p.gram + (p.gram0[k] + matrix * chunks * (int64_t)(NT * kTile));
    auto tile = [](double *M, int b, int c) { return M + (b * RB + c) * kTile; };
    double sum[NT] = {};  // element threadIdx.x of every tile; no branch between the loads
#pragma unroll 8
    for (int c = 0; c < chunks; ++c)
#pragma unroll
        for (int o = 0; o < NT; ++o) sum[o] += part[c * (int64_t)(NT * kTile) + o * kTile + threadIdx.x];
#pragma unroll
    for (int b = 0, o = 0; b < RB; ++b)
#pragma unroll
        for (int c = b; c < RB; ++c, ++o) {
            const int row = 4 * wave + lane / 16, col = lane % 16;
            tile(G, b, c)[threadIdx.x] = sum[o];
            if (c != b) tile(G, c, b)[(col / 4) * 64 + (col % 4) * 16 + row] = sum[o];
        }
    __syncthreads();
    // the trace, in every wave: lane d < 16 RB has diagonal element d
    double trace = 0;
    if (lane < 16 * RB) trace = tile(G, lane / 16, lane / 16)[(lane % 16 / 4) * 64 + (lane % 4) * 16 + lane % 16];
#pragma unroll
    for (int d = 32; d; d >>= 1) trace += __shfl_xor(trace, d, 64);
    const double norm = sqrt(trace) + p.eps, inv = 1.0 / norm;
    const bool mine = wave < WAVES;
    if (RB == 1 && !mine) return;  // no barrier follows
    const int b0 = OWN == 1 ? wave / RB : 0, c0 = mine ? wave % RB : 0;  // tiles (b0 + u, c0)
    f64x4 g[OWN], t[OWN];
    auto diagonal = [&](int u, int i) { return b0 + u == c0 && 4 * i + lane / 16 == lane % 16; };
#pragma unroll
    for (int u = 0; u < OWN; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            g[u][i] = mine ? tile(G, b0 + u, c0)[i * 64 + lane] * inv * inv : 0.0;  // inv * inv may be infinite
            t[u][i] = diagonal(u, i) ? 1.0 : 0.0;
        }
    const f64x4 zero = {0, 0, 0, 0};
    auto polynomial = [&](f64x4 (&q)[OWN]) {
#pragma unroll
        for (int u = 0; u < OWN; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) q[u][i] = p.c * q[u][i] + p.b * g[u][i] + (diagonal(u, i) ? p.a : 0.0);
    };
    if constexpr (RB == 1) {
        auto product = [&](f64x4 x, f64x4 y) {
            f64x4 z = zero;
#pragma unroll
            for (int i = 0; i < 4; ++i) z = mfma_f64(x[i], y[i], z);
            return z;
        };
        for (int step = 0; step < p.steps; ++step) {
            f64x4 q[1] = {product(g[0], g[0])};
            polynomial(q);
            t[0] = step ? product(t[0], q[0]) : q[0];
            g[0] = product(product(g[0], q[0]), q[0]);
        }
    } else {
        auto keep = [&](double *M, const f64x4 (&v)[OWN]) {
#pragma unroll
            for (int u = 0; u < OWN; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (mine) tile(M, b0 + u, c0)[i * 64 + lane] = v[u][i];
        };
        // the wave's tiles of X Y for symmetric, commuting X and Y; a single tile's in two chains
        auto product = [&](double *X, double *Y, f64x4 (&z)[OWN]) {
            if (!mine) return;
            constexpr int CHAINS = OWN == 1 ? 2 : 1;
            f64x4 w[OWN][CHAINS];
#pragma unroll
            for (int u = 0; u < OWN; ++u)
#pragma unroll
                for (int h = 0; h < CHAINS; ++h) w[u][h] = zero;
#pragma unroll
            for (int q = 0; q < RB; ++q)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const double y = tile(Y, q, c0)[i * 64 + lane];
#pragma unroll
                    for (int u = 0; u < OWN; ++u)
                        w[u][i % CHAINS] = mfma_f64(tile(X, q, b0 + u)[i * 64 + lane], y, w[u][i % CHAINS]);
                }
#pragma unroll
            for (int u = 0; u < OWN; ++u) z[u] = CHAINS == 2 ? w[u][0] + w[u][CHAINS - 1] : w[u][0];
        };
        __syncthreads();  // every wave has read its part of G unscaled
        keep(G, g);
        for (int step = 0; step < p.steps; ++step) {
            const bool last = step + 1 == p.steps;
            f64x4 v[OWN];
            __syncthreads();
            product(G, G, v);
            polynomial(v);
            keep(Q, v);
            __syncthreads();
            if (step) {
                product(T, Q, t);
            } else {
#pragma unroll
                for (int u = 0; u < OWN; ++u) t[u] = v[u];  // Q itself
            }
            if (last) break;
            product(G, Q, v);
            keep(H, v);
            __syncthreads();
            keep(T, t);
            product(H, Q, g);
            keep(G, g);
        }
    }
    if (!mine) return;
    // 1 / norm as a power of two, which u takes, and what is left, which T takes:
    // neither leaves f32's range, whatever the gradients' scale
    int expo;
    const double part_of_norm = frexp(norm, &expo);
#pragma unroll
    for (int u = 0; u < OWN; ++u) {
        float *out = p.turn + (int64_t)blockIdx.x * ALL + ((b0 + u) * RB + c0) * kTile;
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i * 64 + lane] = (float)(t[u][i] / part_of_norm);
    }
    if (threadIdx.x == 0) p.expo[blockIdx.x] = -expo;
}

__device__ __forceinline__ f32x4 load_param4(const float *base, int64_t at, int64_t step, int left) {
    return load4(base, at, step, left);
}
__device__ __forceinline__ f32x4 load_param4(const bf16 *base, int64_t at, int64_t step, int left) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (step == 1 && left >= 4) {
        const bf16x4 t = __builtin_bit_cast(bf16x4, *reinterpret_cast<const u32x2_any *>(base + at));
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (float)t[e];
        return v;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < left) v[e] = (float)base[at + e * step];
    return v;
}
__device__ __forceinline__ void store_param4(float *base, int64_t at, int64_t step, int left, f32x4 v) {
    store4(base, at, step, left, v);
}
__device__ __forceinline__ void store_param4(bf16 *base, int64_t at, int64_t step, int left, f32x4 v) {
    if (step == 1 && left >= 4) {
        *reinterpret_cast<u32x2_any *>(base + at) = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < left) base[at + e * step] = f32_to_bf16(v[e]);
}

// p = p * keep - lr * scale * T u.  The f32 16x16x4 product: A[m][k] in lane
// m + 16 k, B[k][n] in lane n + 16 k, D element i of lane l = D[4 (l / 16) + i][l % 16].
// Wide matrices (rows contiguous along n): a wave's step is 64 columns, product e
// those 4 x + e, so that a lane's loads and stores are 4 columns of a row.  Tall
// ones (contiguous along r): 16 columns, the step's k in the order a lane's 4
// elements of a column give it.  Bound by HBM: 63 us for those 21 M elements (read
// g, m, p, write p: 336 MB, 5.3 TB/s).  u is formed again from g and m: writing it
// in the first pass would move as many bytes more.
template <typename T, int RB, bool WIDE>
__device__ __forceinline__ void apply_matrix(const MuonMany &p, const Place &at, const float *turn) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, x = lane & 15, q = lane >> 4;
    const int k = at.item, r = p.r[k], n = p.n[k];
    const int64_t off = at.matrix * (int64_t)r * n;
    const float *g = p.grad[k] + off;
    const float *m = p.m[k] + off;
    T *param = static_cast<T *>(p.param[k]) + off;
    const int j0 = at.chunk * p.chunk[k], j1 = min(n, j0 + p.chunk[k]);
    const float hold = p.keep, rate = p.rate[k];
    // T[16 b + x][K] for the K of step s as `u` below holds it; T is symmetric
    // and lies in f64 tiles: element (row, col) of tile (c, b) at
    // [row / 4][(row % 4) * 16 + col]
    f32x4 t[RB][RB];  // [b][c]: elements e, K = 16 c + 4 e + q (wide) or 16 c + 4 q + e (tall)
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int c = 0; c < RB; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = WIDE ? 4 * e + q : 4 * q + e;
                t[b][c][e] = turn[(c * RB + b) * kTile + (row / 4) * 64 + (row % 4) * 16 + x];
            }
    const int expo = p.expo[at.slot];
    auto update = [&](f32x4 gv, f32x4 mv) {
        f32x4 u;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            u[e] = __builtin_ldexpf(p.nesterov ? __builtin_fmaf(p.beta, mv[e], gv[e]) : mv[e], expo);
        return u;
    };
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    if constexpr (WIDE) {
        for (int j = j0 + wave * 64; j < j1; j += 256) {
            const int jl = j + 4 * x;
            f32x4 u[RB][4];  // rows 16 c + 4 s + q, columns jl .. + 4
#pragma unroll
            for (int c = 0; c < RB; ++c)
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const int i = 16 * c + 4 * s + q;
                    const int left = i < r ? j1 - jl : 0;
                    const int64_t e = (int64_t)i * n + jl;
                    u[c][s] = update(p.nesterov ? load4(g, e, 1, left) : zero, load4(m, e, 1, left));
                }
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                f32x4 d[4] = {zero, zero, zero, zero};  // product e: rows 16 b + 4 q + i, column jl + e
#pragma unroll
                for (int c = 0; c < RB; ++c)
#pragma unroll
                    for (int s = 0; s < 4; ++s)
#pragma unroll
                        for (int e = 0; e < 4; ++e) d[e] = mfma_16x16x4_f32(t[b][c][s], u[c][s][e], d[e]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = 16 * b + 4 * q + i;
                    const int left = row < r ? j1 - jl : 0;
                    const int64_t e = (int64_t)row * n + jl;
                    f32x4 v = load_param4(param, e, 1, left);
#pragma unroll
                    for (int y = 0; y < 4; ++y) v[y] = __builtin_fmaf(-rate, d[y][i], v[y] * hold);
                    store_param4(param, e, 1, left, v);
                }
            }
        }
    } else {
        for (int j = j0 + wave * 16; j < j1; j += 64) {
            const int col = j + x;
            f32x4 u[RB];  // rows 16 c + 4 q .. + 4 of column col
#pragma unroll
            for (int c = 0; c < RB; ++c) {
                const int i = 16 * c + 4 * q;
                const int left = col < j1 ? r - i : 0;
                const int64_t e = (int64_t)col * r + i;
                u[c] = update(p.nesterov ? load4(g, e, 1, left) : zero, load4(m, e, 1, left));
            }
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                f32x4 d = zero;  // rows 16 b + 4 q + i, column col
#pragma unroll
                for (int c = 0; c < RB; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e) d = mfma_16x16x4_f32(t[b][c][e], u[c][e], d);
                const int i = 16 * b + 4 * q;
                const int left = col < j1 ? r - i : 0;
                const int64_t e = (int64_t)col * r + i;
                f32x4 v = load_param4(param, e, 1, left);
#pragma unroll
                for (int y = 0; y < 4; ++y) v[y] = __builtin_fmaf(-rate, d[y], v[y] * hold);
                store_param4(param, e, 1, left, v);
            }
        }
    }
}

template <typename T, int RB>
__global__ __launch_bounds__(256) void muon_apply_kernel(MuonMany p) {
    const Place at = place_of(p, blockIdx.x);
    const float *turn = p.turn + (int64_t)at.slot * (RB * RB * kTile);
    if (p.wide[at.item])
        apply_matrix<T, RB, true>(p, at, turn);
    else
        apply_matrix<T, RB, false>(p, at, turn);
}

// Row blocks of a launch: one kernel serves all its matrices.
int row_blocks(const MuonMany &p) {
    int r = 1;
    for (int k = 0; k < p.items; ++k) r = std::max(r, p.r[k]);
    return (r + 15) / 16;
}
size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

// Columns of a chunk of the long side: by the matrix alone, so that its bits
// do not depend on what else the call holds.  Short chunks fill the chip from one
// matrix, long ones halve the parts that the solve adds up.  us of the three launches,
// rank 32 f32, chunks of 256 and 512: one 4096 x 32 matrix and its pair 28 and 35, of
// 8192 30 and 36, of 65536 65 and 56, of 2^20 1075 and 773; 128 matrices of 2048 and
// 8192 126 and 133.  The two meet between 8192 and 65536 columns.
int chunk_columns(int n) { return n <= 4096 ? 256 : 512; }

// Where everything lies in the workspace; 0 if a launch would be too large.
size_t lay_out(MuonMany &p, int rb) {
    int64_t blocks = 0, matrices = 0;
    size_t gram = 0;
    for (int k = 0; k < p.items; ++k) {
        p.chunk[k] = chunk_columns(p.n[k]);
        p.chunks[k] = (p.n[k] + p.chunk[k] - 1) / p.chunk[k];
        p.block0[k] = (int)blocks;
        p.matrix0[k] = (int)matrices;
        p.gram0[k] = (int64_t)gram;
        blocks += p.count[k] * (int64_t)p.chunks[k];
        matrices += p.count[k];
        gram += (size_t)p.count[k] * p.chunks[k] * (rb * (rb + 1) / 2) * kTile;
        if (blocks * 256 > kMaxThreads || matrices * 256 > kMaxThreads) return 0;
    }
    p.block0[p.items] = (int)blocks;
    p.matrix0[p.items] = (int)matrices;
    p.turn_at = align256(gram * sizeof(double));
    p.expo_at = p.turn_at + align256((size_t)matrices * rb * rb * kTile * sizeof(float));
    return p.expo_at + align256((size_t)matrices * sizeof(int));
}

template <int RB>
hipError_t run_rb(const MuonMany &p, int dtype, hipStream_t s) {
    const dim3 blocks(p.block0[p.items]), matrices(p.matrix0[p.items]), t(256);
    const size_t lds = (RB == 1 ? 1 : 4) * RB * RB * kTile * sizeof(double);
    hipLaunchKernelGGL((muon_gram_kernel<RB>), blocks, t, 0, s, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((muon_solve_kernel<RB>), matrices, t, lds, s, p);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    if (dtype == 0)
        hipLaunchKernelGGL((muon_apply_kernel<bf16, RB>), blocks, t, 0, s, p);
    else
        hipLaunchKernelGGL((muon_apply_kernel<float, RB>), blocks, t, 0, s, p);
    return hipGetLastError();
}

}  // namespace

hipError_t prepare_muon_kernels() {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(&muon_solve_kernel<3>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, 4 * 9 * kTile * 8);
    if (e != hipSuccess) return e;
    return hipFuncSetAttribute(reinterpret_cast<const void *>(&muon_solve_kernel<4>),
                               hipFuncAttributeMaxDynamicSharedMemorySize, 4 * 16 * kTile * 8);
}

int muon_row_blocks(int rows, int cols) { return (std::min(rows, cols) + 15) / 16; }

size_t muon_workspace_bytes(MuonMany &p) { return lay_out(p, row_blocks(p)); }

hipError_t launch_muon_many(MuonMany &p, int dtype, void *work, hipStream_t s) {
    const int rb = row_blocks(p);
    if (!lay_out(p, rb)) return hipErrorInvalidValue;
    p.gram = static_cast<double *>(work);
    p.turn = reinterpret_cast<float *>(static_cast<char *>(work) + p.turn_at);
    p.expo = reinterpret_cast<int *>(static_cast<char *>(work) + p.expo_at);
    switch (rb) {
        case 1: return run_rb<1>(p, dtype, s);
        case 2: return run_rb<2>(p, dtype, s);
        case 3: return run_rb<3>(p, dtype, s);
        default: return run_rb<4>(p, dtype, s);
    }
}

}  // namespace fa
