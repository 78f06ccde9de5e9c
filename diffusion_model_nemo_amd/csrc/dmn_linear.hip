// Linear layer with its epilogue, and its backward pass:
//
//   forward   z = x W^T + b, y = act(z) + r
//   backward  dz = dy act'(z), dx = dz W, dW = dz^T x, db = sum_rows dz   (the residual's gradient is dy itself)
//
// All three products are C[m][n] = sum_k A(m, k) B(n, k) and differ in how their operands lie in memory: along k (rows of
// k, "K") or across it (rows of m or n, "X"): forward K K, dx K X, dW X X. One kernel serves all of them: tiles of both
// operands go through LDS as they lie in memory, and a fragment of an X tile is transposed on its way out of LDS
// (ds_read_b64_tr_b16; float32 reads single elements), so nothing is transposed in memory.
#include "dmn_block.h"

namespace {

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3 };

// ---- activations -------------------------------------------------------------------------------------------------------
// Lower tail of the normal distribution for z >= 0 over exp(-z^2 / 2): a polynomial in t = 1 / (1 + 0.265 z), fitted to
// erfcx(z / sqrt 2) / 2 for 0 <= z <= 14.5 with the smallest largest RELATIVE error: 4e-7 with float32 coefficients
// (float32 results), 1.1e-6 two degrees lower (results that are rounded to 16 bits). Built from the tail, z Phi(z) keeps
// its relative precision where 1 + erf cancels.
template <typename T> __device__ __forceinline__ float normal_tail_scaled(float az) {
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.265f, az, 1.0f));
    float q;
    if constexpr (sizeof(T) == 4) {
        q = 0.03062652051448822f;
        q = __builtin_fmaf(q, t, -0.14330996572971344f);
        q = __builtin_fmaf(q, t, 0.2159682959318161f);
        q = __builtin_fmaf(q, t, -0.11430533230304718f);
        q = __builtin_fmaf(q, t, 0.1365668922662735f);
        q = __builtin_fmaf(q, t, 0.060890380293130875f);
        q = __builtin_fmaf(q, t, 0.10255616903305054f);
        q = __builtin_fmaf(q, t, 0.10526663810014725f);
        q = __builtin_fmaf(q, t, 0.10574040561914444f);
    } else {
        q = -0.06783661246299744f;
        q = __builtin_fmaf(q, t, 0.19546012580394745f);
        q = __builtin_fmaf(q, t, -0.0666465237736702f);
        q = __builtin_fmaf(q, t, 0.14271365106105804f);
        q = __builtin_fmaf(q, t, 0.08285457640886307f);
        q = __builtin_fmaf(q, t, 0.10785627365112305f);
        q = __builtin_fmaf(q, t, 0.10559820383787155f);
    }
    return q * t;
}
template <typename T> __device__ __forceinline__ float normal_cdf(float z, float e) {   // e = exp(-z^2 / 2)
    const float tail = normal_tail_scaled<T>(fabsf(z)) * e;
    return z < 0.f ? tail : 1.0f - tail;
}
template <typename T> __device__ __forceinline__ float activate(float z, int act) {
    if (act == ACT_RELU) return z < 0.f ? 0.f : z;   // a NaN stays
    if (act == ACT_SILU) return z * __builtin_amdgcn_rcpf(1.0f + __expf(-z));
    if (act == ACT_GELU) return z * normal_cdf<T>(z, __expf(-0.5f * z * z));
    return z;
}
template <typename T> __device__ __forceinline__ float act_backward(float dy, float z, int act) {
    if (act == ACT_RELU) return z <= 0.f ? 0.f : dy;
    if (act == ACT_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.0f + __expf(-z));
        return dy * (s * __builtin_fmaf(z, 1.0f - s, 1.0f));
    }
    if (act == ACT_GELU) {
        const float e = __expf(-0.5f * z * z);
        return dy * __builtin_fmaf(z * 0.3989422804014327f, e, normal_cdf<T>(z, e));
    }
    return dy;
}

// ---- the product -----------------------------------------------------------------------------------------------------
struct GemmArgs {
    const void *a, *b;           // A(m, k): K: a[m * lda + k], X: a[k * lda + m]; B(n, k) alike
    long long lda, ldb;
    int M, N, K;
    int splits, tiles_per_split; // the k tiles are shared out over gridDim.y workgroups
    float* part;                 // splits > 1: [splits][M][N] partial products; else the epilogue below
    const void* bias;            // [N] or null
    const void* res;             // [M][ldr] or null, added behind the activation
    long long ldr;
    void* y;                     // [M][N]
    void* z;                     // [M][N] or null: receives the value in front of the activation
    int act;
};

// v_mfma on fragments of 16 bytes per lane: lane l holds row l & 15 of its operand; 16-bit types the eight k from 8 (l >> 4)
// of a step of 32, float32 the four k from 4 (l >> 4) of a step of 16 (four instructions, both operands in the same k
// order). The first operand's rows end up along a lane's four results, the second's across the lanes.
template <typename T> struct Frag;
template <> struct Frag<float> {
    typedef f32x4 type;
    static constexpr int KSTEP = 16;
    static __device__ __forceinline__ void mma(const type& p, const type& q, f32x4& c) {
#pragma unroll
        for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(p[s], q[s], c, 0, 0, 0);
    }
};
template <> struct Frag<__bf16> {
    typedef bf16x8 type;
    static constexpr int KSTEP = 32;
    static __device__ __forceinline__ void mma(const type& p, const type& q, f32x4& c) { c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(p, q, c, 0, 0, 0); }
};
template <> struct Frag<f16> {
    typedef f16x8 type;
    static constexpr int KSTEP = 32;
    static __device__ __forceinline__ void mma(const type& p, const type& q, f32x4& c) { c = __builtin_amdgcn_mfma_f32_16x16x32_f16(p, q, c, 0, 0, 0); }
};

// One operand's tile in LDS: R rows of m (or n) by 128 bytes of k, R * 8 chunks of 16 bytes.
//   K tile: chunk (row, c): 8 chunks per row, stored at row * 8 + (c ^ (row / 2 % 8)): the 16 rows a fragment read touches
//           at one k cover all 64 banks once.
//   X tile: chunk (k, c): R / E chunks per k row, stored at k * (R / E) + (c ^ swz(k)): the k rows that one read touches
//           lie in different banks.
template <typename T, bool X, int R> struct Tile {
    static constexpr int E = 16 / sizeof(T);               // elements per chunk
    static constexpr int BK = 128 / sizeof(T);
    static constexpr int CHUNKS = R * 8;
    static constexpr int CPR = X ? R / E : 8;              // chunks per stored row
    static constexpr int SWZ16 = CPR >= 16 ? 7 : CPR / 2 - 1;

    static __device__ __forceinline__ int swizzle(int row) {
        if constexpr (!X) return (row >> 1) & 7;
        else if constexpr (sizeof(T) == 4) return ((row >> 2) & 3) << 2;
        else return (((row & 3) | ((row >> 3) & 1) << 2) & SWZ16) << 1;
    }
    // chunk q of the tile as it is laid out: its k (K tile: first of E) and its m/n (X tile: first of E)
    static __device__ __forceinline__ void place(int q, int& k, int& r) {
        const int row = q / CPR, c = (q % CPR) ^ swizzle(row);
        k = X ? row : c * E;
        r = X ? c * E : row;
    }
    static __device__ __forceinline__ typename Frag<T>::type read(const char* lds, int r0, int step, int lane) {
        typedef typename Frag<T>::type frag;
        if constexpr (!X) {
            const int row = r0 + (lane & 15), c = step * 4 + (lane >> 4);
            return *(const frag*)(lds + row * 128 + ((c ^ swizzle(row)) << 4));
        } else if constexpr (sizeof(T) == 4) {
            frag f;
            const int r = r0 + (lane & 15);
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int k = step * 16 + (lane >> 4) * 4 + s;
                f[s] = *(const float*)(lds + k * (CPR * 16) + (((r >> 2) ^ swizzle(k)) << 4) + (r & 3) * 4);
            }
            return f;
        } else {
            // 16 lanes read four k rows of 16 elements and receive one column each: k = 8 (l >> 4) + 4 j + 0..3
            const int col = r0 + (lane & 3) * 4, k = step * 32 + (lane >> 4) * 8 + ((lane & 15) >> 2);
            s16x4 v[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int kk = k + 4 * j;
                const char* p = lds + kk * (CPR * 16) + (((col >> 3) ^ swizzle(kk)) << 4) + (col & 4) * 2;
                v[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
            }
            return __builtin_bit_cast(frag, __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
};

constexpr unsigned kOutOfRange = 0x80000000u;   // byte offset behind every buffer: such a load gives zero

// Staging of one operand: `rows` m/n rows from r0, k from k0 of K. Elements outside the matrix become zero.
// DIRECT: memory -> LDS without registers in 16-byte pieces through a buffer descriptor, whose range check supplies the
// zeros; base, row stride and the contiguous extent must be multiples of 16 bytes. Otherwise through registers, for any
// alignment.
template <typename T, bool X, int R, int NT, bool DIRECT> struct Stager {
    typedef Tile<T, X, R> Tl;
    static constexpr int PER = Tl::CHUNKS / NT;
    static_assert(Tl::CHUNKS % NT == 0, "whole chunks per thread");
    const T* base;
    long long ld;
    int extent, K;                // extent of m/n, of k
    unsigned off[DIRECT ? PER : 1];
    typename Pack<T>::vec reg[DIRECT ? 1 : PER];

    __device__ __forceinline__ void init(const void* p, long long ld_, int r0, int extent_, int K_) {
        ld = ld_;
        extent = extent_ - r0;
        K = K_;
        base = (const T*)p + (X ? (long long)r0 : (long long)r0 * ld_);
        if constexpr (DIRECT) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                int k, r;
                Tl::place(i * NT + threadIdx.x, k, r);
                off[i] = r < extent ? (unsigned)((X ? k * ld + r : r * ld + k) * sizeof(T)) : kOutOfRange;
            }
        }
    }
    __device__ __forceinline__ void fetch(int k0, char* lds) {
        if constexpr (DIRECT) {
            const T* p = base + (X ? (long long)k0 * ld : (long long)k0);
            __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, 0x7fffffff, 0x00020000);
            const int left = K - k0;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                unsigned o = off[i];
                if (left < Tl::BK) {
                    int k, r;
                    Tl::place(i * NT + threadIdx.x, k, r);
                    if (k >= left) o = kOutOfRange;
                }
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)(lds + (i * NT + (threadIdx.x & ~63)) * 16), 16, o, 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                int k, r;
                Tl::place(i * NT + threadIdx.x, k, r);
                typename Pack<T>::vec v;
#pragma unroll
                for (int j = 0; j < Pack<T>::N; ++j) v[j] = (T)0.f;
                if (k0 + k < K && r < extent) {
                    const long long kk = k0 + k;
                    v = X ? load16_tail(base + kk * ld, r, extent) : load16_tail(base + r * ld, (int)kk, K);
                }
                reg[i] = v;
            }
        }
    }
    __device__ __forceinline__ void commit(char* lds) {   // not DIRECT: registers -> LDS
        if constexpr (!DIRECT) {
#pragma unroll
            for (int i = 0; i < PER; ++i) *(typename Pack<T>::vec*)(lds + (i * NT + threadIdx.x) * 16) = reg[i];
        }
    }
};

// Four neighbouring results of row m from column n.
template <typename T> __device__ __forceinline__ void epilogue4(const GemmArgs& g, int m, int n, f32x4 v) {
    typedef T vec4 __attribute__((ext_vector_type(4)));
    const bool whole = n + 4 <= g.N;
    auto get = [&](const T* p, float* out) {
        if (whole) {
            vec4 t;
            __builtin_memcpy(&t, p, sizeof(t));
#pragma unroll
            for (int i = 0; i < 4; ++i) out[i] = (float)t[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) out[i] = n + i < g.N ? (float)p[i] : 0.f;
        }
    };
    auto put = [&](T* p, const float* in) {
        if (whole) {
            vec4 t;
#pragma unroll
            for (int i = 0; i < 4; ++i) t[i] = (T)in[i];
            __builtin_memcpy(p, &t, sizeof(t));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n + i < g.N) p[i] = (T)in[i];
        }
    };
    float z[4], o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = v[i];
    if (g.bias) {
        get((const T*)g.bias + n, o);
#pragma unroll
        for (int i = 0; i < 4; ++i) z[i] += o[i];
    }
    if (g.z) put((T*)g.z + (long long)m * g.N + n, z);
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = activate<T>(z[i], g.act);
    if (g.res) {
        get((const T*)g.res + (long long)m * g.ldr + n, o);
#pragma unroll
        for (int i = 0; i < 4; ++i) z[i] += o[i];
    }
    put((T*)g.y + (long long)m * g.N + n, z);
}

// Tile of workgroup `b`: workgroups go round the eight XCDs, each with an L2 of its own, so each XCD gets a run of
// neighbouring tiles, and a run walks down 8 tile rows before it moves to the next tile column.
__device__ __forceinline__ void tile_of(int b, int tm, int tn, int& im, int& in) {
    const int n = tm * tn, per = n / 8, rest = n % 8, x = b & 7;
    const int t = x * per + (x < rest ? x : rest) + (b >> 3);
    const int band = 8 * tn, i = t / band, rows = tm - i * 8 < 8 ? tm - i * 8 : 8;
    im = i * 8 + (t % band) % rows;
    in = (t % band) / rows;
}

template <typename T, bool XA, bool XB, int BM, int BN, int WM, int WN, bool DIRECT>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64) void gemm_kernel(const GemmArgs g) {
    constexpr int NT = (BM / WM) * (BN / WN) * 64;
    typedef Tile<T, XA, BM> TA;
    typedef Tile<T, XB, BN> TB;
    typedef typename Frag<T>::type frag;
    constexpr int BK = TA::BK, A_BYTES = BM * 128, B_BYTES = BN * 128, FM = WM / 16, FN = WN / 16;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = wave % (BM / WM) * WM, wn = wave / (BM / WM) * WN;
    int im, in;
    tile_of(blockIdx.x, (g.M + BM - 1) / BM, (g.N + BN - 1) / BN, im, in);
    const int m0 = im * BM, n0 = in * BN;
    const int k_tiles = (g.K + BK - 1) / BK, t0 = blockIdx.y * g.tiles_per_split;
    const int t1 = t0 + g.tiles_per_split < k_tiles ? t0 + g.tiles_per_split : k_tiles;
    Stager<T, XA, BM, NT, DIRECT> sa;
    Stager<T, XB, BN, NT, DIRECT> sb;
    sa.init(g.a, g.lda, m0, g.M, g.K);
    sb.init(g.b, g.ldb, n0, g.N, g.K);
    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (t0 < t1) {
        sa.fetch(t0 * BK, lds);
        sb.fetch(t0 * BK, lds + A_BYTES);
        sa.commit(lds);
        sb.commit(lds + A_BYTES);
    }
    for (int t = t0; t < t1; ++t) {
        __syncthreads();   // this tile has arrived, and nobody reads the other buffer any more
        char* cur = lds + ((t - t0) & 1) * (A_BYTES + B_BYTES);
        char* nxt = lds + ((t - t0 + 1) & 1) * (A_BYTES + B_BYTES);
        if (t + 1 < t1) {
            sa.fetch((t + 1) * BK, nxt);
            sb.fetch((t + 1) * BK, nxt + A_BYTES);
        }
#pragma unroll
        for (int s = 0; s < BK / Frag<T>::KSTEP; ++s) {
            frag fa[FM], fb[FN];
#pragma unroll
            for (int i = 0; i < FM; ++i) fa[i] = TA::read(cur, wm + i * 16, s, lane);
#pragma unroll
            for (int j = 0; j < FN; ++j) fb[j] = TB::read(cur + A_BYTES, wn + j * 16, s, lane);
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) Frag<T>::mma(fb[j], fa[i], acc[i][j]);
        }
        if (t + 1 < t1) {
            sa.commit(nxt);
            sb.commit(nxt + A_BYTES);
        }
    }
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const int m = m0 + wm + i * 16 + (lane & 15);
        if (m >= g.M) continue;
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            const int n = n0 + wn + j * 16 + (lane >> 4) * 4;
            if (n >= g.N) continue;
            if (g.part) {
                float* p = g.part + ((long long)blockIdx.y * g.M + m) * g.N + n;
                if (n + 4 <= g.N) __builtin_memcpy(p, &acc[i][j], 16);
                else
                    for (int e = 0; n + e < g.N; ++e) p[e] = acc[i][j][e];
            } else {
                epilogue4<T>(g, m, n, acc[i][j]);
            }
        }
    }
}

// Joins the partial products of the k ranges in their order and runs the epilogue. The results are taken four at a time
// along a row.
template <typename T> __global__ __launch_bounds__(256) void gemm_join_kernel(const GemmArgs g) {
    const int quads = (g.N + 3) / 4;
    const long long total = (long long)g.M * quads, stride = (long long)g.M * g.N;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const int m = (int)(i / quads), n = (int)(i % quads) * 4;
        const float* p = g.part + (long long)m * g.N + n;
        f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
        if (n + 4 <= g.N) {
            for (int s = 0; s < g.splits; ++s) {
                f32x4 w;
                __builtin_memcpy(&w, p + s * stride, 16);
                v += w;
            }
        } else {
            for (int s = 0; s < g.splits; ++s)
                for (int e = 0; n + e < g.N; ++e) v[e] += p[s * stride + e];
        }
        epilogue4<T>(g, m, n, v);
    }
}

// ---- what stands in front of the backward's products ------------------------------------------------------------------
// dz = dy act'(z), and partial column sums of dz: 16 threads of 16 bytes side by side, 16 rows at a time; workgroup
// (x, y) takes the y-th of gridDim.y runs of rows. dz is rounded to the operands' type: the matrix cores read it so.
struct DzArgs {
    const void *dy, *z;
    long long lddy;
    void* dz;             // null: only the column sums of dy
    float* part;          // [gridDim.y][N] or null
    int M, N, act;
};
template <typename T> __global__ __launch_bounds__(256) void dz_kernel(const DzArgs a) {
    constexpr int V = Pack<T>::N;
    __shared__ float sh[16][16 * V + 1];
    const int c = threadIdx.x & 15, r = threadIdx.x >> 4, n = (blockIdx.x * 16 + c) * V;
    const int per = (a.M + gridDim.y - 1) / gridDim.y, m0 = blockIdx.y * per, m1 = m0 + per < a.M ? m0 + per : a.M;
    float sum[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0.f;
    if (n < a.N) {
        for (int m = m0 + r; m < m1; m += 16) {
            auto v = load16_tail((const T*)a.dy + (long long)m * a.lddy, n, a.N);
            if (a.dz) {
                const auto z = load16_tail((const T*)a.z + (long long)m * a.N, n, a.N);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float d = act_backward<T>((float)v[i], (float)z[i], a.act);
                    sum[i] += d;
                    v[i] = (T)d;
                }
                store16_tail((T*)a.dz + (long long)m * a.N, n, a.N, v);
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) sum[i] += (float)v[i];
            }
        }
    }
    if (!a.part) return;
#pragma unroll
    for (int i = 0; i < V; ++i) sh[r][c * V + i] = sum[i];
    __syncthreads();
    if (threadIdx.x < 16 * V) {
        const int col = blockIdx.x * 16 * V + threadIdx.x;
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) t += sh[i][threadIdx.x];
        if (col < a.N) a.part[(long long)blockIdx.y * a.N + col] = t;
    }
}
// out[col] = sum over `parts` partial rows, in a fixed order: 32 columns per workgroup, 8 threads per column
template <typename T> __global__ __launch_bounds__(256) void column_join_kernel(const float* part, int parts, int n, T* out) {
    __shared__ float sh[8][33];
    const int c = threadIdx.x & 31, g = threadIdx.x >> 5, col = blockIdx.x * 32 + c;
    float s = 0.f;
    if (col < n) {
#pragma unroll 8
        for (int i = g; i < parts; i += 8) s += part[(long long)i * n + col];
    }
    sh[g][c] = s;
    __syncthreads();
    if (g == 0 && col < n) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) t += sh[i][c];
        out[col] = (T)t;
    }
}

template <typename T> __global__ __launch_bounds__(256) void zero_kernel(T* p, long long n) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) p[i] = (T)0.f;
}

// ---- host side ---------------------------------------------------------------------------------------------------------
inline int elem(int dtype) { return dtype == DMN_DT_F32 ? 4 : 2; }
inline long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// Tile and k split of a product, from its sizes and type alone.
struct GemmPlan {
    int bm, bn, splits, per;
};
GemmPlan gemm_plan(int M, int N, int K, int dtype) {
    GemmPlan p;
    const int bk = 128 / elem(dtype);
    const long long big = ceil_div(M, 128) * ceil_div(N, 128);
    p.bm = p.bn = big >= 200 ? 128 : 64;
    const long long tiles = ceil_div(M, p.bm) * ceil_div(N, p.bn), kt = ceil_div(K, bk);
    long long splits = 1;
    if (tiles < 256 && kt >= 8) {
        splits = 512 / tiles;
        if (splits > kt / 4) splits = kt / 4;
        if (splits > 64) splits = 64;
        if (splits < 1) splits = 1;
    }
    p.per = (int)ceil_div(kt, splits);
    p.splits = (int)ceil_div(kt, p.per);
    return p;
}
size_t gemm_workspace(int M, int N, int K, int dtype) {
    const GemmPlan p = gemm_plan(M, N, K, dtype);
    return p.splits > 1 ? block_align256((size_t)p.splits * M * N * sizeof(float)) : 0;
}

// 16-byte pieces of the operand can be addressed one by one
bool direct_ok(const void* p, long long ld, bool x, int rows, int K, int dtype) {
    const int e = elem(dtype);
    return (uintptr_t)p % 16 == 0 && ld * e % 16 == 0 && (long long)(x ? rows : K) * e % 16 == 0;
}

template <typename T, bool XA, bool XB, int B, int W, bool DIRECT> int gemm_launch(const GemmArgs& g, hipStream_t s) {
    constexpr int NT = (B / W) * (B / W) * 64, LDS = 2 * 2 * B * 128;
    const dim3 grid((unsigned)(ceil_div(g.M, B) * ceil_div(g.N, B)), g.splits);
    gemm_kernel<T, XA, XB, B, B, W, W, DIRECT><<<grid, NT, LDS, s>>>(g);
    DMN_BLOCK_LAUNCH_CHECK();
    return DMN_OK;
}
template <typename T, bool XA, bool XB> int gemm_run(GemmArgs& g, int dtype, void* ws, hipStream_t s) {
    const GemmPlan p = gemm_plan(g.M, g.N, g.K, dtype);
    g.splits = p.splits;
    g.tiles_per_split = p.per;
    g.part = p.splits > 1 ? (float*)ws : nullptr;
    const bool direct = direct_ok(g.a, g.lda, XA, g.M, g.K, dtype) && direct_ok(g.b, g.ldb, XB, g.N, g.K, dtype);
    int rc;
    if (p.bm == 128) rc = direct ? gemm_launch<T, XA, XB, 128, 64, true>(g, s) : gemm_launch<T, XA, XB, 128, 64, false>(g, s);
    else rc = direct ? gemm_launch<T, XA, XB, 64, 32, true>(g, s) : gemm_launch<T, XA, XB, 64, 32, false>(g, s);
    if (rc || p.splits == 1) return rc;
    const long long quads = (long long)g.M * ceil_div(g.N, 4);
    gemm_join_kernel<T><<<(unsigned)(quads < 256 * 4096 ? ceil_div(quads, 256) : 4096), 256, 0, s>>>(g);
    DMN_BLOCK_LAUNCH_CHECK();
    return DMN_OK;
}

constexpr int kMaxDzRuns = 64;
int dz_runs(int M) { return (int)(ceil_div(M, 64) < kMaxDzRuns ? ceil_div(M, 64) : kMaxDzRuns); }

int linear_check(const char* who, int64_t rows, int in, int out, int act, int dtype, int64_t ldx) {
    DMN_REQUIRE(dtype >= 0 && dtype <= 2, DMN_ERR_INVALID, "%s: dtype must be DMN_DT_F32, _BF16 or _F16", who);
    DMN_REQUIRE(act >= ACT_NONE && act <= ACT_GELU, DMN_ERR_INVALID, "%s: unknown activation %d", who, act);
    DMN_REQUIRE(rows >= 0 && in > 0 && out > 0, DMN_ERR_INVALID, "%s: rows must be >= 0, in and out > 0", who);
    DMN_REQUIRE(rows < (1 << 27) && in < (1 << 20) && out < (1 << 20) && rows * (in > out ? in : out) < ((int64_t)1 << 40), DMN_ERR_LIMIT,
                "%s: rows must be below 2^27, in and out below 2^20", who);
    DMN_REQUIRE(rows <= 1 || ldx >= in, DMN_ERR_INVALID, "%s: row stride of x below its width", who);
    DMN_REQUIRE(ldx < (1 << 20), DMN_ERR_LIMIT, "%s: row stride of x must be below 2^20 elements", who);
    return DMN_OK;
}

template <typename T>
int backward_run(const void* dy, long long lddy, const void* x, long long ldx, const void* w, const void* z, void* dx, void* dw, void* db,
                 int rows, int in, int out, int act, int dtype, char* ws, hipStream_t s) {
    if (rows == 0) {
        if (dw) zero_kernel<T><<<1024, 256, 0, s>>>((T*)dw, (long long)in * out);
        DMN_BLOCK_LAUNCH_CHECK();
        if (db) zero_kernel<T><<<64, 256, 0, s>>>((T*)db, out);
        DMN_BLOCK_LAUNCH_CHECK();
        return DMN_OK;
    }
    float* part = (float*)ws;
    const int runs = dz_runs(rows);
    ws += block_align256((size_t)runs * out * sizeof(float));
    const void* dz = dy;
    long long lddz = lddy;
    if (act != ACT_NONE || db) {
        DzArgs a{};
        a.dy = dy;
        a.z = z;
        a.lddy = lddy;
        a.dz = act != ACT_NONE ? ws : nullptr;
        a.part = db ? part : nullptr;
        a.M = rows;
        a.N = out;
        a.act = act;
        dz_kernel<T><<<dim3((unsigned)ceil_div(out, 16 * Pack<T>::N), runs), 256, 0, s>>>(a);
        DMN_BLOCK_LAUNCH_CHECK();
        if (db) {
            column_join_kernel<T><<<(unsigned)ceil_div(out, 32), 256, 0, s>>>(part, runs, out, (T*)db);
            DMN_BLOCK_LAUNCH_CHECK();
        }
        if (act != ACT_NONE) {
            dz = ws;
            lddz = out;
            ws += block_align256((size_t)rows * out * sizeof(T));
        }
    }
    int rc = DMN_OK;
    if (dx) {
        GemmArgs g{};
        g.a = dz;
        g.lda = lddz;
        g.b = w;
        g.ldb = in;
        g.M = rows;
        g.N = in;
        g.K = out;
        g.y = dx;
        rc = gemm_run<T, false, true>(g, dtype, ws, s);
    }
    if (dw && !rc) {
        GemmArgs g{};
        g.a = dz;
        g.lda = lddz;
        g.b = x;
        g.ldb = ldx;
        g.M = out;
        g.N = in;
        g.K = rows;
        g.y = dw;
        rc = gemm_run<T, true, true>(g, dtype, ws, s);
    }
    return rc;
}

}  // namespace

extern "C" size_t dmn_linear_forward_workspace_bytes(int64_t rows, int in, int out, int dtype) {
    if (rows <= 0 || rows >= (1 << 27) || in <= 0 || out <= 0 || dtype < 0 || dtype > 2) return 0;
    return gemm_workspace((int)rows, out, in, dtype);
}

extern "C" int dmn_linear_forward(const void* x, int64_t ldx, const void* weight, const void* bias, const void* residual, int64_t ldr,
                                  void* y, void* z, int64_t rows, int in, int out, int activation, int dtype, void* workspace,
                                  size_t workspace_bytes, void* stream) {
    int rc = linear_check("dmn_linear_forward", rows, in, out, activation, dtype, ldx);
    if (rc || rows == 0) return rc;
    DMN_REQUIRE(x && weight && y, DMN_ERR_INVALID, "dmn_linear_forward: null argument");
    DMN_REQUIRE(!residual || rows <= 1 || ldr >= out, DMN_ERR_INVALID, "dmn_linear_forward: row stride of the residual below its width");
    const size_t need = dmn_linear_forward_workspace_bytes(rows, in, out, dtype);
    DMN_REQUIRE(need == 0 || (workspace && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= need), DMN_ERR_WORKSPACE,
                "dmn_linear_forward: workspace of %zu bytes, %zu needed (16-byte aligned)", workspace_bytes, need);
    GemmArgs g{};
    g.a = x;
    g.lda = ldx;
    g.b = weight;
    g.ldb = in;
    g.M = (int)rows;
    g.N = out;
    g.K = in;
    g.bias = bias;
    g.res = residual;
    g.ldr = ldr;
    g.y = y;
    g.z = z;
    g.act = activation;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == DMN_DT_F32) return gemm_run<float, false, false>(g, dtype, workspace, s);
    if (dtype == DMN_DT_BF16) return gemm_run<__bf16, false, false>(g, dtype, workspace, s);
    return gemm_run<f16, false, false>(g, dtype, workspace, s);
}

extern "C" size_t dmn_linear_backward_workspace_bytes(int64_t rows, int in, int out, int activation, int dtype) {
    if (rows <= 0 || rows >= (1 << 27) || in <= 0 || out <= 0 || dtype < 0 || dtype > 2) return 0;
    const size_t dx = gemm_workspace((int)rows, in, out, dtype), dw = gemm_workspace(out, in, (int)rows, dtype);
    return block_align256((size_t)dz_runs((int)rows) * out * sizeof(float)) +
           (activation != ACT_NONE ? block_align256((size_t)rows * out * elem(dtype)) : 0) + (dx > dw ? dx : dw);
}

extern "C" int dmn_linear_backward(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* weight, const void* z, void* dx,
                                   void* dweight, void* dbias, int64_t rows, int in, int out, int activation, int dtype, void* workspace,
                                   size_t workspace_bytes, void* stream) {
    int rc = linear_check("dmn_linear_backward", rows, in, out, activation, dtype, ldx);
    if (rc) return rc;
    if (!dx && !dweight && !dbias) return DMN_OK;
    DMN_REQUIRE(rows == 0 || (dy && (!dx || weight) && (!dweight || x) && (activation == ACT_NONE || z)), DMN_ERR_INVALID,
                "dmn_linear_backward: null argument");
    DMN_REQUIRE(rows <= 1 || lddy >= out, DMN_ERR_INVALID, "dmn_linear_backward: row stride of dy below its width");
    DMN_REQUIRE(lddy < (1 << 20), DMN_ERR_LIMIT, "dmn_linear_backward: row stride of dy must be below 2^20 elements");
    const size_t need = dmn_linear_backward_workspace_bytes(rows, in, out, activation, dtype);
    DMN_REQUIRE(need == 0 || (workspace && (uintptr_t)workspace % 256 == 0 && workspace_bytes >= need), DMN_ERR_WORKSPACE,
                "dmn_linear_backward: workspace of %zu bytes, %zu needed (256-byte aligned)", workspace_bytes, need);
    hipStream_t s = (hipStream_t)stream;
    char* ws = (char*)workspace;
    if (dtype == DMN_DT_F32) return backward_run<float>(dy, lddy, x, ldx, weight, z, dx, dweight, dbias, (int)rows, in, out, activation, dtype, ws, s);
    if (dtype == DMN_DT_BF16) return backward_run<__bf16>(dy, lddy, x, ldx, weight, z, dx, dweight, dbias, (int)rows, in, out, activation, dtype, ws, s);
    return backward_run<f16>(dy, lddy, x, ldx, weight, z, dx, dweight, dbias, (int)rows, in, out, activation, dtype, ws, s);
}
