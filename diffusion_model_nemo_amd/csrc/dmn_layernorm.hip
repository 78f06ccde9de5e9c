// Layer norm over the last axis: forward, backward, and the reduction of the scale's and shift's gradients.
//
//   forward   m = mean(x), r = 1 / sqrt(mean((x - m)^2) + eps), xhat = (x - m) r, y = xhat w + b
//   backward  g = dy w, dx = r (g - mean(g) - xhat mean(g xhat)), dw = sum_rows dy xhat, db = sum_rows dy
//
// Bound by memory: x in, y out; x and dy in, dx out. A row is read once and stays in the registers of the threads that
// share it (TPR of them, NV vectors of 16 bytes each) for both the statistics and the result, so the variance is formed
// from the deviations themselves. All sums and statistics are float32. The threads keep their columns from row to row: w
// and b are read once, and the backward adds dw and db up in registers, one partial row per workgroup, which a second
// launch adds in a fixed order (the same bits on every run; no atomics). The next row is on its way while one is reduced.
// 16384 rows of 4096 bf16: forward 45 us (6.0 TB/s of x and y), backward 91 us (4.4 TB/s of x, dy and dx) and 4 us for the
// parameters; 65536 rows of 128 float32: 12 and 18 us. (A copy of 2 GB reaches 4.8 TB/s, a read 6.2.) 512 workgroups are
// best for the backward: 256 take 127 us, 768 and 1024 106 and 96.
#include "dmn_block.h"

namespace {

struct LnArgs {
    const void *x, *dy, *w, *b;
    void *y, *dx;
    float* stats;         // [rows][2] mean, 1 / deviation
    float* part;          // [2][blocks][width] partial sums of dw, db
    long long rows, ldx, lddy;
    int width, want_params;
    float eps;
};

// One number per row from TPR threads; NT > 64 threads per row meet through LDS. `turn` alternates the LDS slot from row to
// row, so that one barrier per sum is enough: a slot is written again only two barriers later.
template <int TPR> __device__ __forceinline__ float row_sum(float v, float* sh, int turn) {
    if constexpr (TPR <= 64) {
        return group_sum<TPR>(v);
    } else {
        constexpr int WAVES = TPR / 64;
        v = wave_sum(v);
        float* s = sh + turn * WAVES;
        if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
        __syncthreads();
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) t += s[i];
        return t;
    }
}
template <int TPR> __device__ __forceinline__ void row_sum2(float& a, float& b, float* sh, int turn) {
    if constexpr (TPR <= 64) {
        a = group_sum<TPR>(a);
        b = group_sum<TPR>(b);
    } else {
        constexpr int WAVES = TPR / 64;
        a = wave_sum(a);
        b = wave_sum(b);
        float* s = sh + turn * 2 * WAVES;
        if ((threadIdx.x & 63) == 0) {
            s[2 * (threadIdx.x >> 6)] = a;
            s[2 * (threadIdx.x >> 6) + 1] = b;
        }
        __syncthreads();
        a = b = 0.f;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {
            a += s[2 * i];
            b += s[2 * i + 1];
        }
    }
}

template <typename T, typename A, int TPR, int NV, int NT>
__global__ __launch_bounds__(NT) void ln_fwd_kernel(const LnArgs a) {
    constexpr int V = Pack<T>::N, RPB = NT / TPR;
    typedef typename Pack<T>::vec vec;
    __shared__ float sh[4 * (NT / 64)];
    const int t = threadIdx.x % TPR, slot = threadIdx.x / TPR, n = a.width;
    const T* x = (const T*)a.x;
    T* y = (T*)a.y;
    const float inv_n = 1.0f / (float)n;
    float w[NV][V], b[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
        for (int i = 0; i < V; ++i) w[k][i] = 1.f, b[k][i] = 0.f;
        const int at = (k * TPR + t) * V;
        if (a.w) load_params<T, A>((const A*)a.w, at, n, w[k]);
        if (a.b) load_params<T, A>((const A*)a.b, at, n, b[k]);
    }
    const long long step = (long long)gridDim.x * RPB;
    vec nx[NV];
    auto fetch = [&](long long row) {
        if (row >= a.rows) return;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int at = (k * TPR + t) * V;
            if (at < n) nx[k] = load16_tail(x + row * a.ldx, at, n);
        }
    };
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) nx[k][i] = (T)0.f;
    fetch((long long)blockIdx.x * RPB + slot);
    int turn = 0;
    for (long long base = (long long)blockIdx.x * RPB; base < a.rows; base += step) {
        const long long row = base + slot;
        float v[NV][V], s = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[k][i] = (float)nx[k][i];
                s += v[k][i];
            }
        fetch(row + step);   // the next row is on its way while this one is reduced
        const float mean = row_sum<TPR>(s, sh, turn) * inv_n;
        float q = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[k][i] -= mean;
                const bool in = (k * TPR + t) * V + i < n;
                q += in ? v[k][i] * v[k][i] : 0.f;
            }
        const float rstd = 1.0f / sqrtf(row_sum<TPR>(q, sh + 2 * (NT / 64), turn) * inv_n + a.eps);
        turn ^= 1;
        if (row < a.rows) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int at = (k * TPR + t) * V;
                if (at >= n) continue;
                vec o;
#pragma unroll
                for (int i = 0; i < V; ++i) o[i] = (T)(v[k][i] * rstd * w[k][i] + b[k][i]);
                store16_tail(y + row * n, at, n, o);
            }
            if (a.stats && t == 0) {
                a.stats[2 * row] = mean;
                a.stats[2 * row + 1] = rstd;
            }
        }
    }
}

// Rows wider than the registers of one workgroup hold: three passes over a row that its workgroup has just read.
template <typename T, typename A> __global__ __launch_bounds__(1024) void ln_fwd_wide_kernel(const LnArgs a) {
    __shared__ float sh[4 * 16];
    const int n = a.width;
    const float inv_n = 1.0f / (float)n;
    int turn = 0;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
        const T* x = (const T*)a.x + row * a.ldx;
        T* y = (T*)a.y + row * n;
        float s = 0.f, q = 0.f;
        for (int i = threadIdx.x; i < n; i += 1024) s += (float)x[i];
        const float mean = row_sum<1024>(s, sh, turn) * inv_n;
        for (int i = threadIdx.x; i < n; i += 1024) {
            const float d = (float)x[i] - mean;
            q += d * d;
        }
        const float rstd = 1.0f / sqrtf(row_sum<1024>(q, sh + 32, turn) * inv_n + a.eps);
        for (int i = threadIdx.x; i < n; i += 1024) {
            const float w = a.w ? (float)((const A*)a.w)[i] : 1.f, b = a.b ? (float)((const A*)a.b)[i] : 0.f;
            y[i] = (T)(((float)x[i] - mean) * rstd * w + b);
        }
        if (a.stats && threadIdx.x == 0) {
            a.stats[2 * row] = mean;
            a.stats[2 * row + 1] = rstd;
        }
    }
}

template <typename T, typename A, int TPR, int NV, int NT>
__global__ __launch_bounds__(NT) void ln_bwd_kernel(const LnArgs a) {
    constexpr int V = Pack<T>::N, RPB = NT / TPR, WAVES = NT / 64;
    constexpr int LANES = TPR < 64 ? TPR : 64;       // lanes of a wave with different columns
    typedef typename Pack<T>::vec vec;
    // the row sums' slots, and with several rows per workgroup one partial row of every wave
    __shared__ float sh[TPR > 64 ? 4 * WAVES : WAVES * NV * V * LANES];
    const int t = threadIdx.x % TPR, slot = threadIdx.x / TPR, n = a.width;
    const T *x = (const T*)a.x, *dy = (const T*)a.dy;
    T* dx = (T*)a.dx;
    const float inv_n = 1.0f / (float)n;
    float w[NV][V], dw[NV][V], db[NV][V];
    vec nx[NV], ny[NV];
    float nmean = 0.f, nrstd = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
        for (int i = 0; i < V; ++i) w[k][i] = 1.f, dw[k][i] = db[k][i] = 0.f;
        if (a.w) load_params<T, A>((const A*)a.w, (k * TPR + t) * V, n, w[k]);
    }
    const long long step = (long long)gridDim.x * RPB;
    auto fetch = [&](long long row) {
        const bool in = row < a.rows;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int at = (k * TPR + t) * V;
#pragma unroll
            for (int i = 0; i < V; ++i) nx[k][i] = ny[k][i] = (T)0.f;
            if (in && at < n) {
                nx[k] = load16_tail(x + row * a.ldx, at, n);
                ny[k] = load16_tail(dy + row * a.lddy, at, n);
            }
        }
        nmean = in ? a.stats[2 * row] : 0.f;
        nrstd = in ? a.stats[2 * row + 1] : 0.f;
    };
    fetch((long long)blockIdx.x * RPB + slot);
    int turn = 0;
    for (long long base = (long long)blockIdx.x * RPB; base < a.rows; base += step, turn ^= 1) {
        const long long row = base + slot;
        const float mean = nmean, rstd = nrstd;
        float xh[NV][V], g[NV][V], s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float d = (float)ny[k][i];
                const bool pad = (k * TPR + t) * V + i >= n;
                xh[k][i] = pad ? 0.f : ((float)nx[k][i] - mean) * rstd;
                dw[k][i] += d * xh[k][i];
                db[k][i] += d;
                g[k][i] = d * w[k][i];
                s1 += g[k][i];
                s2 += g[k][i] * xh[k][i];
            }
        fetch(row + step);
        row_sum2<TPR>(s1, s2, sh, turn);
        s1 *= inv_n;
        s2 *= inv_n;
        if (dx && row < a.rows) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int at = (k * TPR + t) * V;
                if (at >= n) continue;
                vec o;
#pragma unroll
                for (int i = 0; i < V; ++i) o[i] = (T)(rstd * (g[k][i] - s1 - xh[k][i] * s2));
                store16_tail(dx + row * n, at, n, o);
            }
        }
    }
    if (!a.want_params) return;
    float* part[2] = {a.part + (long long)blockIdx.x * n, a.part + ((long long)gridDim.x + blockIdx.x) * n};
    if constexpr (TPR > 64) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int at = (k * TPR + t) * V;
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (at + i < n) {
                    part[0][at + i] = dw[k][i];
                    part[1][at + i] = db[k][i];
                }
        }
    } else {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            __syncthreads();
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    float v = which ? db[k][i] : dw[k][i];
#pragma unroll
                    for (int o = TPR; o < 64; o <<= 1) v += __shfl_xor(v, o);
                    if (lane < LANES) sh[((wave * NV + k) * V + i) * LANES + lane] = v;
                }
            __syncthreads();
            for (int e = threadIdx.x; e < NV * V * LANES; e += NT) {
                const int col = ((e / (V * LANES)) * TPR + e % LANES) * V + e / LANES % V;
                float v = 0.f;
#pragma unroll
                for (int i = 0; i < WAVES; ++i) v += sh[i * NV * V * LANES + e];
                if (col < n) part[which][col] = v;
            }
        }
    }
}

template <typename T, typename A> __global__ __launch_bounds__(1024) void ln_bwd_wide_kernel(const LnArgs a) {
    __shared__ float sh[4 * 16];
    const int n = a.width;
    const float inv_n = 1.0f / (float)n;
    int turn = 0;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
        const T *x = (const T*)a.x + row * a.ldx, *dy = (const T*)a.dy + row * a.lddy;
        const float mean = a.stats[2 * row], rstd = a.stats[2 * row + 1];
        float s1 = 0.f, s2 = 0.f;
        for (int i = threadIdx.x; i < n; i += 1024) {
            const float g = (float)dy[i] * (a.w ? (float)((const A*)a.w)[i] : 1.f);
            s1 += g;
            s2 += g * (((float)x[i] - mean) * rstd);
        }
        row_sum2<1024>(s1, s2, sh, turn);
        s1 *= inv_n;
        s2 *= inv_n;
        T* dx = (T*)a.dx + row * n;
        for (int i = threadIdx.x; i < n; i += 1024) {
            const float g = (float)dy[i] * (a.w ? (float)((const A*)a.w)[i] : 1.f);
            dx[i] = (T)(rstd * (g - s1 - ((float)x[i] - mean) * rstd * s2));
        }
    }
}
// Column sums of wide rows: blockIdx.y takes every gridDim.y-th row.
template <typename T> __global__ __launch_bounds__(256) void ln_params_wide_kernel(const LnArgs a) {
    const int col = blockIdx.x * 256 + threadIdx.x, n = a.width;
    if (col >= n) return;
    float dw = 0.f, db = 0.f;
    for (long long row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float d = (float)((const T*)a.dy)[row * a.lddy + col];
        dw += d * (((float)((const T*)a.x)[row * a.ldx + col] - a.stats[2 * row]) * a.stats[2 * row + 1]);
        db += d;
    }
    a.part[(long long)blockIdx.y * n + col] = dw;
    a.part[((long long)gridDim.y + blockIdx.y) * n + col] = db;
}

// out[col] = sum over `parts` partial rows: 32 columns per workgroup, 32 threads per column, fixed order.
// blockIdx.y: 0 the scale's gradient, 1 the shift's.
template <typename A> __global__ __launch_bounds__(1024) void ln_params_kernel(const float* part, int parts, int n, A* dw, A* db) {
    __shared__ float sh[32][33];
    A* out = blockIdx.y ? db : dw;
    if (!out) return;
    const int c = threadIdx.x & 31, g = threadIdx.x >> 5, col = blockIdx.x * 32 + c;
    const float* p = part + (long long)blockIdx.y * parts * n;
    float s = 0.f;
    if (col < n) {
#pragma unroll 8
        for (int i = g; i < parts; i += 32) s += p[(long long)i * n + col];
    }
    sh[g][c] = s;
    __syncthreads();
    if (g == 0 && col < n) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) t += sh[i][c];
        out[col] = (A)t;
    }
}

// Threads per row, vectors per thread, threads per workgroup for rows of `vecs` 16-byte vectors of `per` elements. A thread
// holds at most 16 elements of a row: with 32 (64 threads for a row of 2048 bfloat16) the backward's registers leave one
// wave per SIMD, and 16384 rows took 64 us instead of 47; 16 float32 elements in four vectors are better than in one (81
// against 87 us for 32768 rows of 1024).
struct LnPlan {
    int tpr, nv, nt;
};
LnPlan ln_plan(long long vecs, int per) {
    if (vecs <= 8) return {8, 1, 256};
    if (vecs <= 16) return {16, 1, 256};
    if (vecs <= 32) return {32, 1, 256};
    if (vecs <= 64) return {64, 1, 256};
    if (vecs <= 128) return {64, 2, 256};
    if (vecs <= 256) return per == 4 ? LnPlan{64, 4, 256} : LnPlan{256, 1, 256};
    if (vecs <= 512) return {256, 2, 256};
    if (vecs <= 1024) return per == 4 ? LnPlan{256, 4, 256} : LnPlan{512, 2, 512};
    if (vecs <= 2048) return {1024, 2, 1024};
    return {0, 0, 0};
}
inline int elem_bytes(int dtype) { return dtype == DMN_DT_F32 ? 4 : 2; }
inline LnPlan ln_plan(int width, int dtype) { return ln_plan(((long long)width * elem_bytes(dtype) + 15) / 16, 16 / elem_bytes(dtype)); }

int ln_fwd_blocks(long long rows, const LnPlan& p) {
    const long long need = p.tpr ? (rows + p.nt / p.tpr - 1) / (p.nt / p.tpr) : rows;
    const long long cap = p.nt == 256 ? 2048 : 512;
    return (int)(need < cap ? need : cap);
}
int ln_bwd_blocks(long long rows, const LnPlan& p) {
    const long long need = p.tpr ? (rows + p.nt / p.tpr - 1) / (p.nt / p.tpr) : (rows + 15) / 16;
    const long long cap = p.nt == 1024 ? 256 : p.tpr >= 256 ? 512 : p.tpr ? 1024 : 64;
    return (int)(need < cap ? need : cap);
}

template <int A, int B, int C> struct LnShape { static constexpr int TPR = A, NV = B, NT = C; };
// Calls f with the shape of the plan (one that ln_plan gives for the type).
template <typename T, typename F> void ln_dispatch(const LnPlan& p, F f) {
    auto is = [&](auto shape) {
        if (p.tpr != shape.TPR || p.nv != shape.NV) return false;
        f(shape);
        return true;
    };
    if (is(LnShape<8, 1, 256>{}) || is(LnShape<16, 1, 256>{}) || is(LnShape<32, 1, 256>{}) || is(LnShape<64, 1, 256>{}) ||
        is(LnShape<64, 2, 256>{}) || is(LnShape<256, 2, 256>{}) || is(LnShape<1024, 2, 1024>{}))
        return;
    if constexpr (Pack<T>::N == 4) (void)(is(LnShape<64, 4, 256>{}) || is(LnShape<256, 4, 256>{}));
    else (void)(is(LnShape<256, 1, 256>{}) || is(LnShape<512, 2, 512>{}));
}

template <typename T, typename A> int ln_forward(const LnArgs& a, const LnPlan& p, hipStream_t s) {
    const int grid = ln_fwd_blocks(a.rows, p);
    if (p.tpr == 0) ln_fwd_wide_kernel<T, A><<<grid, 1024, 0, s>>>(a);
    else ln_dispatch<T>(p, [&](auto h) { ln_fwd_kernel<T, A, h.TPR, h.NV, h.NT><<<grid, h.NT, 0, s>>>(a); });
    DMN_BLOCK_LAUNCH_CHECK();
    return DMN_OK;
}

template <typename T, typename A> int ln_backward(const LnArgs& a, const LnPlan& p, void* dw, void* db, hipStream_t s) {
    const int grid = ln_bwd_blocks(a.rows, p);
    if (grid > 0 && p.tpr == 0) {
        if (a.dx) ln_bwd_wide_kernel<T, A><<<(int)(a.rows < 512 ? a.rows : 512), 1024, 0, s>>>(a);
        DMN_BLOCK_LAUNCH_CHECK();
        if (a.want_params) ln_params_wide_kernel<T><<<dim3((a.width + 255) / 256, grid), 256, 0, s>>>(a);
        DMN_BLOCK_LAUNCH_CHECK();
    } else if (grid > 0) {
        ln_dispatch<T>(p, [&](auto h) { ln_bwd_kernel<T, A, h.TPR, h.NV, h.NT><<<grid, h.NT, 0, s>>>(a); });
        DMN_BLOCK_LAUNCH_CHECK();
    }
    if (a.want_params) {
        ln_params_kernel<A><<<dim3((a.width + 31) / 32, 2), 1024, 0, s>>>(a.part, grid, a.width, (A*)dw, (A*)db);
        DMN_BLOCK_LAUNCH_CHECK();
    }
    return DMN_OK;
}

int ln_check(const char* who, int64_t rows, int width, int dtype, int affine_dtype, int64_t ld) {
    DMN_REQUIRE(dtype >= 0 && dtype <= 2 && (affine_dtype == dtype || affine_dtype == DMN_DT_F32), DMN_ERR_INVALID,
                "%s: dtype must be DMN_DT_F32, _BF16 or _F16 and affine_dtype the same or DMN_DT_F32", who);
    DMN_REQUIRE(rows >= 0 && width > 0, DMN_ERR_INVALID, "%s: rows must be >= 0 and width > 0", who);
    DMN_REQUIRE(width <= (1 << 30) && rows <= ((int64_t)1 << 40) / width, DMN_ERR_LIMIT, "%s: more than 2^40 elements", who);
    DMN_REQUIRE(rows <= 1 || ld >= width, DMN_ERR_INVALID, "%s: row stride %lld below the width %d", who, (long long)ld, width);
    return DMN_OK;
}

}  // namespace

extern "C" int dmn_layer_norm_forward(const void* x, int64_t ldx, const void* weight, const void* bias, void* y, float* stats,
                                      int64_t rows, int width, int dtype, int affine_dtype, float eps, void* stream) {
    int rc = ln_check("dmn_layer_norm_forward", rows, width, dtype, affine_dtype, ldx);
    if (rc || rows == 0) return rc;
    DMN_REQUIRE(x && y, DMN_ERR_INVALID, "dmn_layer_norm_forward: null argument");
    LnArgs a{};
    a.x = x;
    a.w = weight;
    a.b = bias;
    a.y = y;
    a.stats = stats;
    a.rows = rows;
    a.ldx = ldx;
    a.width = width;
    a.eps = eps;
    const LnPlan p = ln_plan(width, dtype);
    hipStream_t s = (hipStream_t)stream;
    if (dtype == DMN_DT_F32) return ln_forward<float, float>(a, p, s);
    if (dtype == DMN_DT_BF16) return affine_dtype == dtype ? ln_forward<__bf16, __bf16>(a, p, s) : ln_forward<__bf16, float>(a, p, s);
    return affine_dtype == dtype ? ln_forward<f16, f16>(a, p, s) : ln_forward<f16, float>(a, p, s);
}

extern "C" size_t dmn_layer_norm_workspace_bytes(int64_t rows, int width, int dtype) {
    if (rows < 0 || width <= 0 || dtype < 0 || dtype > 2) return 0;
    return (size_t)2 * ln_bwd_blocks(rows, ln_plan(width, dtype)) * width * sizeof(float) + 256;
}

extern "C" int dmn_layer_norm_backward(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* weight,
                                       const float* stats, void* dx, void* dweight, void* dbias, int64_t rows, int width, int dtype,
                                       int affine_dtype, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = ln_check("dmn_layer_norm_backward", rows, width, dtype, affine_dtype, ldx < lddy ? ldx : lddy);
    if (rc) return rc;
    DMN_REQUIRE(rows == 0 || (x && dy && stats), DMN_ERR_INVALID, "dmn_layer_norm_backward: null argument");
    LnArgs a{};
    a.x = x;
    a.dy = dy;
    a.w = weight;
    a.dx = dx;
    a.stats = (float*)stats;
    a.part = (float*)workspace;
    a.rows = rows;
    a.ldx = ldx;
    a.lddy = lddy;
    a.width = width;
    a.want_params = dweight || dbias;
    if (!dx && !a.want_params) return DMN_OK;
    DMN_REQUIRE(!a.want_params || (workspace && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= dmn_layer_norm_workspace_bytes(rows, width, dtype)),
                DMN_ERR_WORKSPACE, "dmn_layer_norm_backward: workspace of %zu bytes, %zu needed (16-byte aligned)", workspace_bytes,
                dmn_layer_norm_workspace_bytes(rows, width, dtype));
    const LnPlan p = ln_plan(width, dtype);
    hipStream_t s = (hipStream_t)stream;
    if (dtype == DMN_DT_F32) return ln_backward<float, float>(a, p, dweight, dbias, s);
    if (dtype == DMN_DT_BF16)
        return affine_dtype == dtype ? ln_backward<__bf16, __bf16>(a, p, dweight, dbias, s) : ln_backward<__bf16, float>(a, p, dweight, dbias, s);
    return affine_dtype == dtype ? ln_backward<f16, f16>(a, p, dweight, dbias, s) : ln_backward<f16, float>(a, p, dweight, dbias, s);
}
