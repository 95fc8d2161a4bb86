// Layer norm with a learned weight and bias over [N, C] rows, and its backward
// with the parameters' gradients:
//   n = (x - mean) * rstd,  rstd = 1 / sqrt(var + eps)  (biased variance)
//   y = n * w + b
//   dx = dres + rstd * (g - mean(g) - n * mean(g * n)),  g = dy * w
//   dw = sum over rows of dy * n,  db = sum over rows of dy
// HBM-bound: a row is read once (twice the variance's pass comes from
// registers).  Statistics, sums and gradients are f32, results are rounded once
// to the storage type.  Any C up to 32768, any strides: vectors of 8 elements
// move with 16-byte accesses aligned to the element only, the last few of a
// row one by one.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "fa_device.hpp"
#include "fa_kernels.hpp"

namespace fa {
namespace {

typedef u32x4 u32x4_any __attribute__((aligned(2)));  // 16 bytes at any element's address

// 8 consecutive elements as they lie in memory
struct ChunkBf16 {
    u32x4 w;
};
struct ChunkF32 {
    u32x4 w, w2;
};
template <typename T>
using Chunk = std::conditional_t<sizeof(T) == 2, ChunkBf16, ChunkF32>;

__device__ __forceinline__ float chunk_at(const ChunkBf16 &r, int j) { return (float)as_bf16x8(r.w)[j]; }
__device__ __forceinline__ float chunk_at(const ChunkF32 &r, int j) {
    return j < 4 ? __builtin_bit_cast(f32x4, r.w)[j] : __builtin_bit_cast(f32x4, r.w2)[j - 4];
}
__device__ __forceinline__ void chunk_zero(ChunkBf16 &r) { r.w = u32x4{0, 0, 0, 0}; }
__device__ __forceinline__ void chunk_zero(ChunkF32 &r) { r.w = r.w2 = u32x4{0, 0, 0, 0}; }
__device__ __forceinline__ void chunk_ld(const bf16 *p, ChunkBf16 &r) { r.w = *reinterpret_cast<const u32x4_any *>(p); }
__device__ __forceinline__ void chunk_ld(const float *p, ChunkF32 &r) {
    r.w = *reinterpret_cast<const u32x4_any *>(p);
    r.w2 = *reinterpret_cast<const u32x4_any *>(p + 4);
}

// Elements e .. e + 7 of a row of C; past its end they are zero.
template <typename T>
__device__ __forceinline__ void load_chunk(const T *row, int e, int C, Chunk<T> &r) {
    if (e + 8 <= C) {
        chunk_ld(row + e, r);
        return;
    }
    chunk_zero(r);
    if (e < C) {
        T t[8] = {};
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (e + j < C) t[j] = row[e + j];
        __builtin_memcpy(&r, t, sizeof(r));
    }
}

__device__ __forceinline__ void chunk_st(bf16 *p, const float v[8]) {
    bf16x8 a;
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = f32_to_bf16(v[j]);
    *reinterpret_cast<u32x4_any *>(p) = as_u32x4(a);
}
__device__ __forceinline__ void chunk_st(float *p, const float v[8]) {
    *reinterpret_cast<u32x4_any *>(p) = __builtin_bit_cast(u32x4, f32x4{v[0], v[1], v[2], v[3]});
    *reinterpret_cast<u32x4_any *>(p + 4) = __builtin_bit_cast(u32x4, f32x4{v[4], v[5], v[6], v[7]});
}
template <typename T>
__device__ __forceinline__ void store_chunk(T *row, int e, int C, const float v[8]) {
    if (e + 8 <= C) {
        chunk_st(row + e, v);
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (e + j < C) row[e + j] = (T)v[j];
}

template <int CTRL>
__device__ __forceinline__ float dpp_f32(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xF, 0xF, false));
}
// Sum over the wave, the same value in every lane.
__device__ __forceinline__ float wave_sum(float s) {
    s += dpp_f32<0xB1>(s);   // quad_perm [1,0,3,2]
    s += dpp_f32<0x4E>(s);   // quad_perm [2,3,0,1]
    s += dpp_f32<0x141>(s);  // row_half_mirror
    s += dpp_f32<0x140>(s);  // row_mirror
    s += __shfl_xor(s, 16, 64);
    return sum_xor32(s);
}

constexpr int kMaxWaves = 16;

// A row belongs to a group of G waves, P groups to a workgroup.  Wave w of the
// group holds elements (k * G + w) * 512 + 8 * lane .. + 8 for k < CH.  Bound by
// HBM: 15.6 us at 4096 x 4096 bf16 (67 MB, 4.3 TB/s), 26 to 30 at 32768 x 1024
// (134 MB, 4.5 to 5 TB/s), f32 4096 x 4096 31 (134 MB).  Under 512 columns lanes are
// idle: 100000 rows take 35 us at 64 columns and at 128 (26 and 51 MB).
template <typename T, typename WT, int CH>
__global__ __launch_bounds__(1024) void layer_norm_fwd_kernel(LayerNormParams p) {
    __shared__ float red[2][kMaxWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int G = p.G, P = (int)(blockDim.x >> 6) / G;
    const int group = wave / G, w0 = group * G, gw = wave - w0;
    const int C = p.C;
    const float inv_c = 1.f / (float)C;
    auto group_sum = [&](float s, float *buf) {
        s = wave_sum(s);
        if (G == 1) return s;
        if (lane == 0) buf[wave] = s;
        __syncthreads();
        s = 0.f;
        for (int i = 0; i < G; ++i) s += buf[w0 + i];
        return s;
    };
    for (int64_t base = (int64_t)blockIdx.x * P; base < p.N; base += (int64_t)gridDim.x * P) {
        const int64_t row = base + group;
        const bool live = row < p.N;
        const T *x = static_cast<const T *>(p.x) + row * p.ldx;
        Chunk<T> v[CH];
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < CH; ++k) {
            load_chunk(x, live ? (k * G + gw) * 512 + lane * 8 : C, C, v[k]);
#pragma unroll
            for (int j = 0; j < 8; ++j) s += chunk_at(v[k], j);
        }
        const float mean = group_sum(s, red[0]) * inv_c;
        float q = 0.f;
#pragma unroll
        for (int k = 0; k < CH; ++k) {
            const int e = (k * G + gw) * 512 + lane * 8;
            if (e + 8 <= C) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float d = chunk_at(v[k], j) - mean;
                    q = __builtin_fmaf(d, d, q);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float d = e + j < C ? chunk_at(v[k], j) - mean : 0.f;
                    q = __builtin_fmaf(d, d, q);
                }
            }
        }
        const float rstd = 1.f / sqrtf(group_sum(q, red[1]) * inv_c + p.eps);
        if (!live) continue;  // its group has met every barrier of this pass
        T *y = static_cast<T *>(p.y) + row * p.ldy;
#pragma unroll
        for (int k = 0; k < CH; ++k) {
            const int e = (k * G + gw) * 512 + lane * 8;
            if (e >= C) continue;
            Chunk<WT> w, b;
            load_chunk(static_cast<const WT *>(p.w), e, C, w);
            chunk_zero(b);
            if (p.b) load_chunk(static_cast<const WT *>(p.b), e, C, b);
            float o[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                o[j] = __builtin_fmaf((chunk_at(v[k], j) - mean) * rstd, chunk_at(w, j), chunk_at(b, j));
            store_chunk(y, e, C, o);
        }
        if (gw == 0 && lane == 0 && p.mean) {
            p.mean[row] = mean;
            p.rstd[row] = rstd;
        }
    }
}

// Backward: each group takes R rows at a time and keeps its columns' sums of
// dy * n and dy in registers; the workgroup adds its groups' in order and
// writes one row of partial sums [2][C], so that dw and db cost no second pass
// over x and dy.  Bound by HBM: 26 us at 4096 x 4096 bf16 (101 MB, 3.9 TB/s), 41 to
// 44 at 32768 x 1024 (201 MB, 4.6 to 4.9 TB/s), 59 at 2048 x 16384 (201 MB); without
// the next rows' loads ahead (AHEAD) more, as the two reductions of a row leave
// memory idle.  Not so at four chunks a lane, C > 16384: of the sums of 32 columns,
// the weights and the rows, 208 to 314 registers a lane lie in scratch memory, and
// 2048 x 16392 takes 274 us, 1024 x 32768 322 (201 MB both; f32 254).  Under 512
// columns lanes are idle: 100000 rows take 50 us at 64 columns and at 128.
template <typename T, typename WT, int CH, int R, bool AHEAD>
__global__ __launch_bounds__(1024) void layer_norm_bwd_kernel(LayerNormParams p) {
    __shared__ float red[2][kMaxWaves][2 * R];
    extern __shared__ float part[];  // [2][C], where P > 1
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int G = p.G, P = (int)(blockDim.x >> 6) / G;
    const int group = wave / G, w0 = group * G, gw = wave - w0;
    const int C = p.C;
    const float inv_c = 1.f / (float)C;
    Chunk<WT> w[CH];
    float dw[CH][8], db[CH][8];
#pragma unroll
    for (int k = 0; k < CH; ++k) {
        load_chunk(static_cast<const WT *>(p.w), (k * G + gw) * 512 + lane * 8, C, w[k]);
#pragma unroll
        for (int j = 0; j < 8; ++j) dw[k][j] = db[k][j] = 0.f;
    }
    Chunk<T> xn[R][CH], dyn[R][CH];  // the next rows
    float meann[R], rstdn[R];
    auto load_rows = [&](int64_t base) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int64_t row = base + group * R + i;
            const bool live = row < p.N;
            const T *xr = static_cast<const T *>(p.x) + row * p.ldx;
            const T *yr = static_cast<const T *>(p.dy) + row * p.lddy;
#pragma unroll
            for (int k = 0; k < CH; ++k) {
                const int e = live ? (k * G + gw) * 512 + lane * 8 : C;
                load_chunk(xr, e, C, xn[i][k]);
                load_chunk(yr, e, C, dyn[i][k]);
            }
            meann[i] = live ? p.mean[row] : 0.f;
            rstdn[i] = live ? p.rstd[row] : 0.f;
        }
    };
    const int64_t stride = (int64_t)gridDim.x * P * R;
    int turn = 0;
    if (AHEAD) load_rows((int64_t)blockIdx.x * P * R);
    for (int64_t base = (int64_t)blockIdx.x * P * R; base < p.N; base += stride, turn ^= 1) {
        Chunk<T> x[R][CH], dy[R][CH];
        float mean[R], rstd[R], sum[2 * R];
        if (!AHEAD) load_rows(base);
#pragma unroll
        for (int i = 0; i < R; ++i) {
#pragma unroll
            for (int k = 0; k < CH; ++k) {
                x[i][k] = xn[i][k];
                dy[i][k] = dyn[i][k];
            }
            mean[i] = meann[i];
            rstd[i] = rstdn[i];
        }
        if (AHEAD && base + stride < p.N) load_rows(base + stride);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            float a = 0.f, b = 0.f;
#pragma unroll
            for (int k = 0; k < CH; ++k)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float d = chunk_at(dy[i][k], j), n = (chunk_at(x[i][k], j) - mean[i]) * rstd[i];
                    const float g = d * chunk_at(w[k], j);
                    a += g;
                    b = __builtin_fmaf(g, n, b);
                    dw[k][j] = __builtin_fmaf(d, n, dw[k][j]);
                    db[k][j] += d;
                }
            sum[2 * i] = wave_sum(a);
            sum[2 * i + 1] = wave_sum(b);
        }
        if (G > 1) {
            if (lane == 0)
#pragma unroll
                for (int i = 0; i < 2 * R; ++i) red[turn][wave][i] = sum[i];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 2 * R; ++i) {
                sum[i] = 0.f;
                for (int v = 0; v < G; ++v) sum[i] += red[turn][w0 + v][i];
            }
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int64_t row = base + group * R + i;
            if (row >= p.N) break;
            const float ma = sum[2 * i] * inv_c, mb = sum[2 * i + 1] * inv_c;
            T *dx = static_cast<T *>(p.dx) + row * p.lddx;
#pragma unroll
            for (int k = 0; k < CH; ++k) {
                const int e = (k * G + gw) * 512 + lane * 8;
                if (e >= C) continue;
                Chunk<T> res;
                chunk_zero(res);
                if (p.dres) load_chunk(static_cast<const T *>(p.dres) + row * p.ldres, e, C, res);
                float o[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float n = (chunk_at(x[i][k], j) - mean[i]) * rstd[i];
                    const float g = chunk_at(dy[i][k], j) * chunk_at(w[k], j);
                    o[j] = __builtin_fmaf(rstd[i], __builtin_fmaf(-mb, n, g - ma), chunk_at(res, j));
                }
                store_chunk(dx, e, C, o);
            }
        }
    }
    if (!p.part) return;
    float *out = p.part + (int64_t)blockIdx.x * 2 * C;
    for (int i = 0; i < P; ++i) {
        if (group == i) {
#pragma unroll
            for (int k = 0; k < CH; ++k) {
                const int e = (k * G + gw) * 512 + lane * 8;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (e + j >= C) continue;
                    float a = dw[k][j], b = db[k][j];
                    if (i > 0) {
                        a += part[e + j];
                        b += part[C + e + j];
                    }
                    if (i + 1 < P) {
                        part[e + j] = a;
                        part[C + e + j] = b;
                    } else {
                        out[e + j] = a;
                        out[C + e + j] = b;
                    }
                }
            }
        }
        if (i + 1 < P) __syncthreads();
    }
}

// dw and db: the column sums of the partial rows [count][2][C], 64 columns and
// 16 interleaved row ranges per workgroup, added in order.  Latency-bound, 4 to
// 4.7 us: 256 partial rows at C = 4096 are 8 MB.
__global__ __launch_bounds__(1024) void layer_norm_reduce_kernel(const float *part, int count, int C, float *dw,
                                                                 float *db) {
    __shared__ float red[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t col = (int64_t)blockIdx.x * 64 + lane;
    float s = 0.f;
    if (col < 2 * (int64_t)C)
#pragma unroll 8
        for (int i = wave; i < count; i += 16) s += part[i * 2 * (int64_t)C + col];
    red[wave][lane] = s;
    __syncthreads();
    if (wave || col >= 2 * (int64_t)C) return;
    for (int i = 1; i < 16; ++i) s += red[i][lane];
    float *out = col < C ? dw : db;
    if (out) out[col < C ? col : col - C] = s;
}

// Waves per row of C elements with CH chunks of 512 per wave.
int group_waves(int C, int ch) { return (C + 512 * ch - 1) / (512 * ch); }

// Rows at a time of a group of waves, and whether the next are loaded ahead: what
// the 128 VGPRs of 1024 threads hold at one and two chunks a lane (four do not fit).
template <typename T, int CH>
constexpr int kBwdRows = sizeof(T) == 2 && CH == 1 ? 2 : 1;

struct BwdShape {
    int ch, G, P, blocks;
};
// 16 waves a workgroup, one workgroup a CU; fewer waves where the rows would not
// reach every CU otherwise.
BwdShape bwd_shape(int N, int C, int dtype) {
    BwdShape s{};
    // as few chunks a lane as 16 waves allow; us, bf16: 4096 x 8192 (one) 49, x 8200 (two)
    // 56; 2048 x 16384 (two) 59, x 16392 (four) 274
    s.ch = C <= 8192 ? 1 : C <= 16384 ? 2 : 4;
    s.G = group_waves(C, s.ch);
    const int64_t rows = dtype == 0 && s.ch == 1 ? 2 : 1, cus = device_cu_count();
    s.P = (int)std::max<int64_t>(1, std::min<int64_t>(kMaxWaves / s.G, N / (cus * rows)));
    s.blocks = (int)std::min<int64_t>(cus * std::max(1, 8 / (s.G * s.P)), (N + s.P * rows - 1) / (s.P * rows));
    return s;
}

template <typename T, typename WT>
hipError_t fwd_t(LayerNormParams p, hipStream_t s) {
    // us: 32768 x 1024 bf16 25.6 with two chunks a wave and 8 waves a workgroup, 27.4 with 4, 30.6 with
    // one chunk (2 waves a row); 4096 x 4096 15.6 with two chunks, 17.8 with one, 16.1 with four;
    // 4096 x 8192 (two) 32, x 8200 (four) 39
    const int ch = p.C <= 512 ? 1 : p.C <= 8192 ? 2 : 4;
    p.G = group_waves(p.C, ch);
    const int P = std::max(1, 8 / p.G);
    const int64_t want = ((int64_t)p.N + P - 1) / P;
    const dim3 grid((unsigned)std::min<int64_t>(want, 1 << 20)), block(64 * p.G * P);
    if (ch == 1)
        hipLaunchKernelGGL((layer_norm_fwd_kernel<T, WT, 1>), grid, block, 0, s, p);
    else if (ch == 2)
        hipLaunchKernelGGL((layer_norm_fwd_kernel<T, WT, 2>), grid, block, 0, s, p);
    else
        hipLaunchKernelGGL((layer_norm_fwd_kernel<T, WT, 4>), grid, block, 0, s, p);
    return hipGetLastError();
}

template <typename T, typename WT>
hipError_t bwd_t(LayerNormParams p, hipStream_t s) {
    const BwdShape sh = bwd_shape(p.N, p.C, sizeof(T) == 2 ? 0 : 1);
    p.G = sh.G;
    const dim3 grid(sh.blocks), block(64 * sh.G * sh.P);
    const size_t lds = p.part && sh.P > 1 ? (size_t)p.C * 8 : 0;
    if (sh.blocks > 0) {
        if (sh.ch == 1)
            hipLaunchKernelGGL((layer_norm_bwd_kernel<T, WT, 1, kBwdRows<T, 1>, true>), grid, block, lds, s, p);
        else if (sh.ch == 2)
            hipLaunchKernelGGL((layer_norm_bwd_kernel<T, WT, 2, kBwdRows<T, 2>, false>), grid, block, lds, s, p);
        else
            hipLaunchKernelGGL((layer_norm_bwd_kernel<T, WT, 4, kBwdRows<T, 4>, false>), grid, block, lds, s, p);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (p.part) {
        hipLaunchKernelGGL(layer_norm_reduce_kernel, dim3((unsigned)((2 * (int64_t)p.C + 63) / 64)), dim3(1024), 0, s,
                           p.part, sh.blocks, p.C, p.dw, p.db);
        return hipGetLastError();
    }
    return hipSuccess;
}

}  // namespace

size_t layer_norm_bwd_workspace_bytes(int N, int C, int dtype) {
    return (size_t)bwd_shape(N, C, dtype).blocks * 2 * C * sizeof(float);
}

hipError_t launch_layer_norm_fwd(const LayerNormParams &p, int dtype, int wdtype, hipStream_t s) {
    if (p.N == 0) return hipSuccess;
    if (dtype == 0) return wdtype == 0 ? fwd_t<bf16, bf16>(p, s) : fwd_t<bf16, float>(p, s);
    return wdtype == 0 ? fwd_t<float, bf16>(p, s) : fwd_t<float, float>(p, s);
}
hipError_t launch_layer_norm_bwd(const LayerNormParams &p, int dtype, int wdtype, hipStream_t s) {
    if (dtype == 0) return wdtype == 0 ? bwd_t<bf16, bf16>(p, s) : bwd_t<bf16, float>(p, s);
    return wdtype == 0 ? bwd_t<float, bf16>(p, s) : bwd_t<float, float>(p, s);
}

}  // namespace fa
