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
__device__ __forceinline__ float normal_bell(float z) { return __builtin_amdgcn_exp2f(-0.72134752f * z * z); }   // exp(-z^2 / 2)
// z Phi(z) as max(z, 0) - |z| Phi(-|z|): no cancellation, a NaN stays (through exp), and infinities give their limits (the
// factor |z| is held at 40, where Phi(-|z|) is zero in float32).
template <typename T> __device__ __forceinline__ float gelu(float z) {
    const float az = fminf(fabsf(z), 40.f), e = normal_bell(z);
    return __builtin_fmaf(-az, normal_tail_scaled<T>(az) * e, fmaxf(z, 0.f));
}
template <typename T> __device__ __forceinline__ float activate(float z, int act) {
    if (act == ACT_RELU) return z < 0.f ? 0.f : z;   // a NaN stays
    if (act == ACT_SILU) return z * __builtin_amdgcn_rcpf(1.0f + __expf(-z));
    if (act == ACT_GELU) return gelu<T>(z);
    return z;
}
// z is held within +-100, where the slopes have long been 0 and 1: an infinite z (a finite sum beyond the range of the type that
// kept it) would turn into 0 * inf. A NaN stays.
template <typename T> __device__ __forceinline__ float act_backward(float dy, float z, int act) {
    if (act == ACT_RELU) return z <= 0.f ? 0.f : dy;
    z = z < -100.f ? -100.f : z > 100.f ? 100.f : z;
    if (act == ACT_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.0f + __expf(-z));
        return dy * (s * __builtin_fmaf(z, 1.0f - s, 1.0f));
    }
    if (act == ACT_GELU) {
        const float e = normal_bell(z);
        return dy * __builtin_fmaf(z * 0.3989422804014327f, e, normal_cdf<T>(z, e));
    }
    return dy;
}

// ---- the product -----------------------------------------------------------------------------------------------------
struct GemmArgs {
    const void *a, *b;           // A(m, k): K: a[m * lda + k], X: a[k * lda + m]; B(n, k) alike
    const void* a2;              // null, or A's low part, laid out as a: A = (a + a2 / Parts::LOW) / Parts::PRE
    long long lda, ldb;
    int M, N, K;
    int splits, tiles_per_split; // the k tiles are shared out over so many workgroups
    float* part;                 // splits > 1: [splits][M][N] partial products; else the epilogue below
    const void* bias;            // [N] or null
    const void* res;             // [M][ldr] or null, added behind the activation
    long long ldr;
    void* y;                     // [M][N]
    void* z;                     // [M][N] or null: receives the value in front of the activation
    int z_exact;                 // z is float32, else of the operands' type
    int act;
};

// dz = dy act'(z) rounded to 16 bits is off by as much as dx and dW, rounded once, are themselves: their errors grow by sqrt 2
// (512 x 256 into 1024 GELU, relative, bf16 2.4e-3 instead of 1.7e-3), and far more in float16 where gradients are small (dy about
// 1e-6, of which the type keeps four bits: dW 2.5e-2 instead of 1.1e-3). So the products take dz as the sum of two numbers of the
// type, 16 bits of it (bf16) or 22 (float16): k is gone through twice, the low part first. float16's low part is stored 2^11
// times larger, or it would fall below the type's smallest step; both parts are halved, because a slope of up to 1.13 takes a
// large dy out of the type's range. The backward's matrix work doubles (training step of 4096 x 1024 into 4096 bf16 GELU: 131
// -> 217 us, of it dz 16 -> 31, the products 74 -> 148, the forward that keeps a float32 z 46 -> 48); a caller who does not want
// that leaves out DMN_LINEAR_EXACT: z and dz are rounded to the type.
template <typename T> struct Parts { static constexpr float PRE = 1.f, LOW = 1.f; };
template <> struct Parts<f16> { static constexpr float PRE = 0.5f, LOW = 2048.f; };
template <typename T> __device__ __forceinline__ void in_two(float d, T& high, T& low) {
    d *= Parts<T>::PRE;
    high = (T)d;
    const float rest = d - (float)high;   // exact
    low = (T)(fabsf((float)high) < INFINITY ? rest * Parts<T>::LOW : 0.f);   // an infinity or NaN stays what it is
}

// v_mfma on fragments of 16 bytes per lane: lane l holds row l & 15 of its operand; 16-bit types the eight k from 8 (l >> 4)
// of a step of 32, float32 the four k from 4 (l >> 4) of a step of 16 (four instructions, both operands in the same k
// order). The first operand's rows end up along a lane's four results, the second's across the lanes.
template <typename T> struct Frag;
template <> struct Frag<float> {
    typedef f32x4 type;
    static constexpr int KSTEP = 16, MMAS = 4;
    static __device__ __forceinline__ void mma(const type& p, const type& q, f32x4& c) {
#pragma unroll
        for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(p[s], q[s], c, 0, 0, 0);
    }
};
template <> struct Frag<__bf16> {
    typedef bf16x8 type;
    static constexpr int KSTEP = 32, MMAS = 1;
    static __device__ __forceinline__ void mma(const type& p, const type& q, f32x4& c) { c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(p, q, c, 0, 0, 0); }
};
template <> struct Frag<f16> {
    typedef f16x8 type;
    static constexpr int KSTEP = 32, MMAS = 1;
    static __device__ __forceinline__ void mma(const type& p, const type& q, f32x4& c) { c = __builtin_amdgcn_mfma_f32_16x16x32_f16(p, q, c, 0, 0, 0); }
};

// One operand's tile in LDS: R rows of m (or n) by KB bytes of k, in chunks of 16 bytes.
//   K tile: chunk (row, c): KB / 16 chunks per row, stored at row * (KB / 16) + (c ^ swizzle(row)). A fragment read is
//           served 16 lanes at a time, in the groups {0-3, 12-15, 20-23, 24-27}, {4-11, 16-19, 28-31} and these + 32
//           (found from the counted bank conflicts of four layouts): the swizzles make each group cover all 64 banks once.
//   X tile: chunk (k, c): R / E chunks per k row, stored at k * (R / E) + (c ^ swizzle(k)): the k rows that one read touches
//           lie in different banks.
template <typename T, bool X, int R, int KB> struct Tile {
    static constexpr int E = 16 / sizeof(T);               // elements per chunk
    static constexpr int BK = KB / sizeof(T);
    static constexpr int CHUNKS = R * KB / 16;
    static constexpr int CPR = X ? R / E : KB / 16;        // chunks per stored row
    static constexpr int READS = !X ? 1 : sizeof(T) == 4 ? 4 : 2;   // LDS instructions of one fragment
    static constexpr int SWZ16 = CPR >= 16 ? 7 : CPR / 2 - 1;

    static __device__ __forceinline__ int swizzle(int row) {
        if constexpr (!X) return KB == 128 ? (row >> 1) & 7 : -(row >> 2) & 3;
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
            return *(const frag*)(lds + row * KB + ((c ^ swizzle(row)) << 4));
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

// 16 bytes per lane from a buffer to LDS, lane l's at dst + 16 l. As assembly, because behind the builtin the compiler
// waits for ALL outstanding requests in front of every transposing LDS read, which leaves nothing in flight (the
// narrow dx product took 80 us instead of 41). The kernel waits for arrivals itself. The s_nop covers the wait states between a
// scalar write of m0 (or a vector write of the descriptor) and the request. m0 cannot be declared as overwritten (it is reserved);
// the build checks that nothing else in these kernels uses it (isa_check.py). The write to LDS is not declared either: a memory
// clobber here costs 1 % (8192 x 2048 into 8192 259 : 262 us). It is not needed, because between two of the kernel's barriers, which
// do carry one (the waits), requests go to a stage that no read touches: reads may pass requests, but never a barrier.
__device__ __forceinline__ void load_to_lds(u32x4 rsrc, unsigned offset, unsigned dst) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" : : "s"(dst), "v"(offset), "s"(rsrc));
}
__device__ __forceinline__ unsigned lds_address(const char* p) { return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const char*)p; }

// Staging of one operand from memory to LDS without registers, in 16-byte pieces through a buffer descriptor whose range
// check supplies the zeros outside the matrix. Base and row stride are multiples of 16 bytes; where a row ends inside a
// piece, the rest of the piece is there and, along k, holds zeros (pad_copy_kernel).
template <typename T, bool X, int R, int NT, int KB> struct Stager {
    typedef Tile<T, X, R, KB> Tl;
    static constexpr int PER = Tl::CHUNKS / NT;
    static_assert(Tl::CHUNKS % NT == 0, "whole chunks per thread");
    const T* next;        // first element of the k rows that the next request takes
    long long step;
    unsigned off[PER];

    __device__ __forceinline__ void start(const void* p, long long ld, int r0, int k0) {
        next = (const T*)p + (X ? (long long)k0 * ld + r0 : (long long)r0 * ld + k0);
    }
    __device__ __forceinline__ void init(const void* p, long long ld, int r0, int extent, int k0) {
        start(p, ld, r0, k0);
        step = X ? Tl::BK * ld : Tl::BK;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            int k, r;
            Tl::place(i * NT + threadIdx.x, k, r);
            off[i] = r0 + r < extent ? (unsigned)((X ? k * ld + r : r * ld + k) * (long long)sizeof(T)) : kOutOfRange;
        }
    }
    // the next tile, of whose k rows only `left` (or none, or all) exist, to LDS from address `dst` + 16 * lane of the wave
    __device__ __forceinline__ void fetch(int left, unsigned dst) {
        // raw buffer: address, no stride, bytes, flags
        const u32x4 rsrc = {(unsigned)(uintptr_t)next, (unsigned)((uintptr_t)next >> 32) & 0xffffu, 0x7fffffffu, 0x00020000u};
        next += step;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            unsigned o = off[i];
            if (left < Tl::BK) {
                int k, r;
                Tl::place(i * NT + threadIdx.x, k, r);
                if (k >= left) o = kOutOfRange;
            }
            load_to_lds(rsrc, o, dst + i * NT * 16);
        }
    }
};

template <typename T, bool EDGE> __device__ __forceinline__ typename Pack<T>::vec load_residual(const GemmArgs& g, int m, int n) {
    const T* p = (const T*)g.res + (long long)m * g.ldr;
    return EDGE ? load16_tail(p, n, g.N) : load16(p + n);
}
// Pack<T>::N neighbouring results of row m from column n < N, whose bias and (if there is one) residual are given. EDGE: the
// row may end among them.
template <typename T, bool RES, bool EDGE>
__device__ __forceinline__ void epilogue(const GemmArgs& g, int m, int n, const float* acc, const float* bias, typename Pack<T>::vec res, int act) {
    constexpr int V = Pack<T>::N;
    float z[V];
    typename Pack<T>::vec v;
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] = acc[i] + bias[i];
    if (g.z && sizeof(T) == 2 && !g.z_exact) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = (T)z[i];
        T* p = (T*)g.z + (long long)m * g.N;
        if (EDGE) store16_tail(p, n, g.N, v);
        else store16(p + n, v);
    } else if (g.z) {
        float* p = (float*)g.z + (long long)m * g.N;
#pragma unroll
        for (int e = 0; e < V; e += 4) {
            const f32x4 q = {z[e], z[e + 1], z[e + 2], z[e + 3]};
            if (!EDGE) store16(p + n + e, q);
            else if (n + e < g.N) store16_tail(p, n + e, g.N, q);
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] = activate<T>(z[i], act);
    if (RES && g.res) {
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] += (float)res[i];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (T)z[i];
    T* p = (T*)g.y + (long long)m * g.N;
    if (EDGE) store16_tail(p, n, g.N, v);
    else store16(p + n, v);
}
template <typename T> __device__ __forceinline__ void load_bias(const GemmArgs& g, int n, float* bias) {
#pragma unroll
    for (int i = 0; i < Pack<T>::N; ++i) bias[i] = 0.f;
    if (g.bias && n < g.N) {
        const auto v = load16_tail((const T*)g.bias, n, g.N);
#pragma unroll
        for (int i = 0; i < Pack<T>::N; ++i) bias[i] = (float)v[i];
    }
}

// Accumulators -> results. A lane holds four neighbouring columns of one of 16 rows; through LDS (two pieces of its own for
// every wave, in turn, 16 rows at a time) it comes to hold 16 bytes of a row, so that rows are read and written in whole
// pieces. The vector units do this while the matrix cores stand still, so it is kept short: a lane's columns stay the same
// (its bias is read once), and tiles inside the matrix check nothing. The residual's pieces are requested AHEAD pieces before
// they are added (8192 x 2048 into 8192 bf16: 273 -> 265 us, 4001 x 4096 into 1024 37.5 -> 36.9). RES: not in the backward.
template <typename T, bool RES, int FM, int FN, bool EDGE> __device__ __forceinline__ void store_rows(const GemmArgs& g, f32x4 (&acc)[FM][FN], int m0, int n0, int split, char* lds, int act) {
    constexpr int V = Pack<T>::N, WN = FN * 16, PITCH = WN + 4, LPR = WN / V, ROWS = 64 / LPR, EACH = 16 / ROWS;
    constexpr int AHEAD = FM * EACH < 4 ? FM * EACH : 4;
    const int lane = threadIdx.x & 63;
    const int c = lane % LPR * V, n = n0 + c;
    float bias[V];
    typename Pack<T>::vec res[AHEAD];
    auto fetch = [&](int q) {   // piece q: row m0 + q ROWS + lane / LPR
        const int m = m0 + q * ROWS + lane / LPR;
        if (RES && g.res && !(EDGE && (m >= g.M || n >= g.N))) res[q % AHEAD] = load_residual<T, EDGE>(g, m, n);
    };
    if (!g.part) {
        load_bias<T>(g, n, bias);
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) fetch(q);
    }
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        float* sh = (float*)lds + ((threadIdx.x >> 6) * 2 + (i & 1)) * 16 * PITCH;
#pragma unroll
        for (int j = 0; j < FN; ++j) *(f32x4*)(sh + (lane & 15) * PITCH + j * 16 + (lane >> 4) * 4) = acc[i][j];
#pragma unroll
        for (int r0 = 0; r0 < 16; r0 += ROWS) {
            const int r = r0 + lane / LPR, m = m0 + i * 16 + r;
            float v[V];
#pragma unroll
            for (int e = 0; e < V; e += 4) {
                const f32x4 q = *(const f32x4*)(sh + r * PITCH + c + e);
#pragma unroll
                for (int k = 0; k < 4; ++k) v[e + k] = q[k];
            }
            if (EDGE && (m >= g.M || n >= g.N)) continue;
            if (g.part) {
                float* p = g.part + ((long long)split * g.M + m) * g.N;
#pragma unroll
                for (int e = 0; e < V; e += 4) {
                    const f32x4 q = {v[e], v[e + 1], v[e + 2], v[e + 3]};
                    if (!EDGE) store16(p + n + e, q);
                    else if (n + e < g.N) store16_tail(p, n + e, g.N, q);
                }
            } else {
                const int q = i * EACH + r0 / ROWS;
                epilogue<T, RES, EDGE>(g, m, n, v, bias, res[q % AHEAD], act);
                if (q + AHEAD < FM * EACH) fetch(q + AHEAD);
            }
        }
    }
}
template <typename T, bool FORWARD, int FM, int FN> __device__ __forceinline__ void store_tile(const GemmArgs& g, f32x4 (&acc)[FM][FN], int m0, int n0, int split, char* lds) {
    if (m0 + FM * 16 > g.M || n0 + FN * 16 > g.N) store_rows<T, FORWARD, FM, FN, true>(g, acc, m0, n0, split, lds, FORWARD ? g.act : ACT_NONE);
    else if (FORWARD && g.act == ACT_GELU) store_rows<T, FORWARD, FM, FN, false>(g, acc, m0, n0, split, lds, ACT_GELU);
    else if (FORWARD && g.act == ACT_SILU) store_rows<T, FORWARD, FM, FN, false>(g, acc, m0, n0, split, lds, ACT_SILU);
    else if (FORWARD && g.act == ACT_RELU) store_rows<T, FORWARD, FM, FN, false>(g, acc, m0, n0, split, lds, ACT_RELU);
    else store_rows<T, FORWARD, FM, FN, false>(g, acc, m0, n0, split, lds, ACT_NONE);
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

template <int N> struct Int { static constexpr int value = N; };

// The product. S tiles of 128 bytes of k go round in LDS, each worked off in two steps; the fragments of the next step come out
// of LDS while the matrix cores work on the present one's, which are in registers. One barrier per tile, in front of its
// second step: behind it the tile's fragments of every wave are in registers, so that the request for the tile S further on
// may take its place, and the next tile has arrived (each wave has waited for its own part of it). Requests go on behind the
// last tile (they read nothing and give zeros), so that the count of outstanding ones is the same for every tile. With A in
// two parts (TWO; a kernel of its own, because the others would pay 3 % for the choice: 4001 x 4096 into 1024 training 118 : 121 us)
// the k tiles count twice, and at `turn` the requests go back to the first one, with the high part.
//
// Bound by the matrix cores where the large tile fills the chip: 8192^3 bf16 827 us forward, 824 dx, 855 dw (1330, 1335, 1286
// TFLOP/s; the card's own product library 715, 816, 930 us), float32 4096^3 960, 968, 984 us (143 to 140 TFLOP/s; library 914 to
// 918). Per step of 128
// bytes of k a 256 x 256 tile keeps them busy for 2048 cycles and brings 64 KB through the CU's first-level cache, 1024
// cycles at 64 bytes each; 128 x 128 brings half of that for a quarter of the products, which is why it stays below 1000
// TFLOP/s (4096 x 1024 out of k = 4096: 37 us). What reading the next fragments beside the products, counted waits and
// 128-byte rows in LDS (64-byte rows request half cache lines: 262 instead of 238 us) brought is the step from 366 to 238
// us for 8192 x 2048 into 8192.
template <typename T, bool XA, bool XB, bool TWO, int BM, int BN, int WM, int WN, int S>
__device__ __forceinline__ void product_tile(const GemmArgs& g, int tile, int split, char* lds) {
    constexpr int NT = (BM / WM) * (BN / WN) * 64, KB = 128;
    typedef Tile<T, XA, BM, KB> TA;
    typedef Tile<T, XB, BN, KB> TB;
    typedef Stager<T, XA, BM, NT, KB> SA;
    typedef Stager<T, XB, BN, NT, KB> SB;
    typedef typename Frag<T>::type frag;
    constexpr int BK = TA::BK, A_BYTES = BM * KB, STAGE = (BM + BN) * KB, FM = WM / 16, FN = WN / 16;
    constexpr int WAIT = (S - 2) * (SA::PER + SB::PER);
    static_assert(BK == 2 * Frag<T>::KSTEP && S >= 2 && WAIT + SA::PER + SB::PER < 64, "pipeline");
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = wave % (BM / WM) * WM, wn = wave / (BM / WM) * WN;
    int im, in;
    tile_of(tile, (g.M + BM - 1) / BM, (g.N + BN - 1) / BN, im, in);
    const int m0 = im * BM, n0 = in * BN;
    const int k_tiles = (g.K + BK - 1) / BK, all = TWO ? 2 * k_tiles : k_tiles, turn = TWO ? k_tiles : 0;
    const int t0 = split * g.tiles_per_split, t1 = t0 + g.tiles_per_split < all ? t0 + g.tiles_per_split : all;
    auto rows_to = [&](int tile) { return tile * BK < g.K ? tile * BK : g.K; };
    const bool high = !TWO || t0 >= turn;   // of the first request
    const int first = high ? t0 - turn : t0;
    int left = rows_to(high ? t1 - turn : t1 < turn ? t1 : turn) - first * BK;   // k rows that the next requests may still take
    int next = t0;                                                               // TWO: tile of the next request
    SA sa;
    SB sb;
    sa.init(high ? g.a : g.a2, g.lda, m0, g.M, first * BK);
    sb.init(g.b, g.ldb, n0, g.N, first * BK);
    const unsigned lds0 = __builtin_amdgcn_readfirstlane(lds_address(lds) + (threadIdx.x & ~63) * 16);
    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto scale = [&](float f) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] *= f;
    };
    auto fetch = [&](int stage) {
        if constexpr (TWO) {
            if (next == turn) {
                sa.start(g.a, g.lda, m0, 0);
                sb.start(g.b, g.ldb, n0, 0);
                left = rows_to(t1 - turn);   // none where the split ends here
            }
            ++next;
        }
        sa.fetch(left, lds0 + stage * STAGE);
        sb.fetch(left, lds0 + stage * STAGE + A_BYTES);
        left -= BK;
    };
    frag fa[2][FM], fb[2][FN];
    auto read = [&](auto step, int stage) {
        constexpr int P = decltype(step)::value;
        const char* cur = lds + stage * STAGE;
#pragma unroll
        for (int i = 0; i < FM; ++i) fa[P][i] = TA::read(cur, wm + i * 16, P, lane);
#pragma unroll
        for (int j = 0; j < FN; ++j) fb[P][j] = TB::read(cur + A_BYTES, wn + j * 16, P, lane);
    };
    auto multiply = [&](auto step) {
        constexpr int P = decltype(step)::value;
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) Frag<T>::mma(fb[P][j], fa[P][i], acc[i][j]);
        // LDS reads between the matrix instructions, not in front of them or (what the compiler would do) behind them
        constexpr int READS = FM * TA::READS + FN * TB::READS, MMAS = FM * FN * Frag<T>::MMAS, EACH = MMAS / READS > 0 ? MMAS / READS : 1;
#pragma unroll
        for (int i = 0; i < READS; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);      // a read of LDS
            __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);   // matrix instructions
        }
    };
#pragma unroll
    for (int i = 0; i < S; ++i) fetch(i);
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(WAIT + SA::PER + SB::PER) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
    read(Int<0>{}, 0);
    int stage = 0;
    for (int t = t0; t < t1; ++t) {
        if constexpr (TWO && Parts<T>::LOW != 1.f) {
            if (t == turn) scale(1.f / Parts<T>::LOW);
        }
        read(Int<1>{}, stage);
        multiply(Int<0>{});
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(WAIT) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" : : : "memory");
        fetch(stage);
        stage = stage + 1 == S ? 0 : stage + 1;
        read(Int<0>{}, stage);
        multiply(Int<1>{});
        __builtin_amdgcn_sched_barrier(0);
    }
    asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
    __syncthreads();   // the requests behind the end have landed, the tiles' memory is free
    if constexpr (TWO && Parts<T>::LOW != 1.f) {
        scale(t1 <= turn ? 1.f / (Parts<T>::LOW * Parts<T>::PRE) : 1.f / Parts<T>::PRE);
    }
    store_tile<T, !XB, FM, FN>(g, acc, m0 + wm, n0 + wn, split, lds);
}
template <typename T, bool XA, bool XB, bool TWO, int BM, int BN, int WM, int WN, int S>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64) void gemm_pipe_kernel(const GemmArgs g) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    product_tile<T, XA, XB, TWO, BM, BN, WM, WN, S>(g, blockIdx.x, blockIdx.y, lds);
}
// out[col] = sum over `parts` partial rows, in a fixed order: 32 columns per workgroup of NT threads, NT / 32 threads per column
struct ColumnJoin {
    const float* part;   // [parts][n]
    int parts, n;
    void* out;           // null: nothing to do
};
template <typename T, int NT> __device__ __forceinline__ void column_join(const ColumnJoin& j, int block, float* sh) {
    constexpr int G = NT / 32;
    const int c = threadIdx.x & 31, g = threadIdx.x >> 5, col = block * 32 + c;
    float s = 0.f;
    if (col < j.n) {
#pragma unroll 8
        for (int i = g; i < j.parts; i += G) s += j.part[(long long)i * j.n + col];
    }
    sh[g * 32 + c] = s;
    __syncthreads();
    if (g == 0 && col < j.n) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < G; ++i) t += sh[i * 32 + c];
        ((T*)j.out)[col] = (T)t;
    }
}
// Both of the backward's products in one launch: they read the same dz, and neither's tiles alone fill the chip evenly (one after
// the other each has its own first requests, last tiles and launch). The product with the longer tiles goes in front. Both
// products, one after the other and so (us, dz in one part): 4096 x 1024 into 4096 bf16 85 : 71, 2048 x 1024 into 1024 27 : 19, 4096 x 320 into
// 1280 29 : 19.5, 256 x 320 into 320 8.0 : 5.0, 16384 x 256 into 1024 float32 149 : 139; 4096^3 bf16, whose 256 x 256 tiles come
// out even, 214 : 265.
struct PairArgs {
    GemmArgs dx, dw;
    int dx_tiles, dw_tiles;   // of one split
    int dx_at, dw_at;         // first workgroup of each: one of them 0
    int db_at;                // the workgroups from here on join the column sums: a launch less, beside the last tiles (4096 x 1024
                              // into 4096, whole step: own launch 139 us, in front of the tiles 136, behind them 129)
    ColumnJoin db;
};
template <typename T, bool TWO, int BM, int BN, int WM, int WN, int S>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64) void gemm_pair_kernel(const PairArgs p) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int b = blockIdx.x;
    if (b >= p.db_at) {
        column_join<T, (BM / WM) * (BN / WN) * 64>(p.db, b - p.db_at, (float*)lds);
    } else if (p.dx_at ? b >= p.dx_at : b < p.dw_at) {
        const int i = b - p.dx_at, split = i / p.dx_tiles;
        product_tile<T, false, true, TWO, BM, BN, WM, WN, S>(p.dx, i - split * p.dx_tiles, split, lds);
    } else {
        const int i = b - p.dw_at, split = i / p.dw_tiles;
        product_tile<T, true, true, TWO, BM, BN, WM, WN, S>(p.dw, i - split * p.dw_tiles, split, lds);
    }
}

// The forward product for few rows (M <= 16 MF): bound by reading the weight once. A workgroup takes 16 NF columns; its waves
// share k out among themselves in runs of 128 bytes, each reading whole cache lines of 16 weight rows straight into
// matrix-core operands (x in the same k order; rows behind M repeat the last one and are dropped), several runs in flight.
// The waves' sums meet in LDS in a fixed order. Any alignment. One row through 2048 x 8192 bf16: 10.6 us with the weight out of
// the caches (3.2 TB/s; a launch with nothing in it and one trip to memory are 4 us of it), 8.2 us with it in them; 16 rows 12.5.
template <typename T, int MF, int NF, int WAVES> __global__ __launch_bounds__(WAVES * 64) void gemm_few_rows_kernel(const GemmArgs g) {
    typedef typename Pack<T>::vec vec;
    constexpr int V = Pack<T>::N, RUN = 8 * V, U = MF * NF >= 8 ? 1 : MF * NF >= 4 ? 2 : 4;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n0 = blockIdx.x * 16 * NF, kl = (lane >> 4) * 2 * V;
    const T *pw[NF], *px[MF];
#pragma unroll
    for (int j = 0; j < NF; ++j) {
        const int n = n0 + j * 16 + (lane & 15);
        pw[j] = (const T*)g.b + (long long)(n < g.N ? n : g.N - 1) * g.ldb;
    }
#pragma unroll
    for (int i = 0; i < MF; ++i) {
        const int m = i * 16 + (lane & 15);
        px[i] = (const T*)g.a + (long long)(m < g.M ? m : g.M - 1) * g.lda;
    }
    f32x4 acc[MF][NF];
#pragma unroll
    for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int j = 0; j < NF; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    vec fw[U][NF][2], fx[U][MF][2];
    auto multiply = [&](int u) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < MF; ++i)
#pragma unroll
                for (int j = 0; j < NF; ++j)
                    Frag<T>::mma(__builtin_bit_cast(typename Frag<T>::type, fw[u][j][h]), __builtin_bit_cast(typename Frag<T>::type, fx[u][i][h]), acc[i][j]);
    };
    const int runs = g.K / RUN;
    int run = wave;
    for (; run + (U - 1) * WAVES < runs; run += U * WAVES) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = (run + u * WAVES) * RUN + kl;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int j = 0; j < NF; ++j) fw[u][j][h] = load16(pw[j] + k + h * V);
#pragma unroll
                for (int i = 0; i < MF; ++i) fx[u][i][h] = load16(px[i] + k + h * V);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) multiply(u);
    }
    for (; run * RUN < g.K; run += WAVES) {   // the runs left over, the last of which may be short
        const int k = run * RUN + kl;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = k + h * V;
#pragma unroll
            for (int j = 0; j < NF; ++j) {
#pragma unroll
                for (int e = 0; e < V; ++e) fw[0][j][h][e] = (T)0.f;
                if (at < g.K) fw[0][j][h] = load16_tail(pw[j], at, g.K);
            }
#pragma unroll
            for (int i = 0; i < MF; ++i) {
#pragma unroll
                for (int e = 0; e < V; ++e) fx[0][i][h][e] = (T)0.f;
                if (at < g.K) fx[0][i][h] = load16_tail(px[i], at, g.K);
            }
        }
        multiply(0);
    }
    f32x4* sh = (f32x4*)lds;
#pragma unroll
    for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int j = 0; j < NF; ++j) sh[((wave * MF + i) * NF + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    for (int t = threadIdx.x; t < MF * NF * 64; t += WAVES * 64) {
        const int l = t & 63, j = t / 64 % NF, i = t / 64 / NF, m = i * 16 + (l & 15), n = n0 + j * 16 + (l >> 4) * 4;
        if (m >= g.M || n >= g.N) continue;
        f32x4 v = sh[t];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) v += sh[w * MF * NF * 64 + t];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (n + e >= g.N) break;
            float z = v[e] + (g.bias ? (float)((const T*)g.bias)[n + e] : 0.f);
            const long long at = (long long)m * g.N + n + e;
            if (g.z && sizeof(T) == 2 && !g.z_exact) ((T*)g.z)[at] = (T)z;
            else if (g.z) ((float*)g.z)[at] = z;
            z = activate<T>(z, g.act);
            if (g.res) z += (float)((const T*)g.res)[(long long)m * g.ldr + n + e];
            ((T*)g.y)[at] = (T)z;
        }
    }
}

// Joins the partial products of the k ranges and runs the epilogue: 256 / G pieces of a row per workgroup, G threads per piece
// that add every G-th range each and meet in LDS, in a fixed order.
template <typename T, int G> __global__ __launch_bounds__(256) void gemm_join_kernel(const GemmArgs g) {
    constexpr int V = Pack<T>::N, P = 256 / G;
    __shared__ float sh[G > 1 ? 256 * (V + 1) : 1];
    const int pieces = (g.N + V - 1) / V, group = threadIdx.x / P;
    const long long i = (long long)blockIdx.x * P + threadIdx.x % P, stride = (long long)g.M * g.N;
    const bool in = i < (long long)g.M * pieces;
    const int m = in ? (int)(i / pieces) : 0, n = in ? (int)(i % pieces) * V : 0;
    float v[V];
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = 0.f;
    if (in) {
        const float* p = g.part + (long long)m * g.N + group * stride;
#pragma unroll 4
        for (int s = group; s < g.splits; s += G, p += G * stride) {
#pragma unroll
            for (int e = 0; e < V; e += 4)
                if (n + e < g.N) {
                    const f32x4 w = load16_tail(p, n + e, g.N);
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[e + k] += w[k];
                }
        }
    }
    if constexpr (G > 1) {
#pragma unroll
        for (int e = 0; e < V; ++e) sh[threadIdx.x * (V + 1) + e] = v[e];
        __syncthreads();
        if (group) return;
#pragma unroll
        for (int s = 1; s < G; ++s)
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] += sh[(threadIdx.x + s * P) * (V + 1) + e];
    }
    if (!in) return;
    float bias[V];
    load_bias<T>(g, n, bias);
    epilogue<T, true, true>(g, m, n, v, bias, g.res ? load_residual<T, true>(g, m, n) : typename Pack<T>::vec{}, g.act);
}

// ---- what stands in front of the backward's products ------------------------------------------------------------------
// dz = dy act'(z), and partial column sums of dz: 16 threads of 16 bytes side by side, 16 rows at a time; workgroup
// (x, y) takes the y-th of gridDim.y runs of rows. EXACT (16-bit types): z is float32, dz leaves in two parts (`in_two`); else z is
// of the operands' type and dz is rounded to it. Bound by memory: 4096 x 4096 bf16 16 us (6.0 TB/s), EXACT 31 us (5.4 TB/s), 16384 x
// 1024 float32 40 us (5.0 TB/s).
struct DzArgs {
    const void *dy, *z;
    long long lddy;
    void* dz;             // [M][lddz], the rows' padding zero; null: only the column sums
    void* low;            // EXACT: the low part, alike
    long long lddz;
    float* part;          // [gridDim.y][N] or null
    int M, N, act;
};
template <typename T, bool EXACT> __global__ __launch_bounds__(256) void dz_kernel(const DzArgs a) {
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
            if (a.act != ACT_NONE) {
                float z[V];
                typename Pack<T>::vec low;
                if constexpr (EXACT) {
                    load_params<T, float>((const float*)a.z + (long long)m * a.N, n, a.N, z);
                } else {
                    const auto q = load16_tail((const T*)a.z + (long long)m * a.N, n, a.N);
#pragma unroll
                    for (int i = 0; i < V; ++i) z[i] = (float)q[i];
                }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float d = act_backward<T>((float)v[i], z[i], a.act);
                    sum[i] += d;
                    if constexpr (EXACT) {
                        T h, l;
                        in_two(d, h, l);
                        v[i] = h;
                        low[i] = l;
                    } else {
                        v[i] = (T)d;
                    }
                }
                if (a.dz) {   // behind the row's end dy and z read as zero, dz is
                    store16((T*)a.dz + (long long)m * a.lddz + n, v);
                    if constexpr (EXACT) store16((T*)a.low + (long long)m * a.lddz + n, low);
                }
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
template <typename T> __global__ __launch_bounds__(256) void column_join_kernel(const ColumnJoin j) {
    __shared__ float sh[256];
    column_join<T, 256>(j, blockIdx.x, sh);
}

template <typename T> __global__ __launch_bounds__(256) void zero_kernel(T* p, long long n) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) p[i] = (T)0.f;
}

// Copies of operands whose rows do not lie on 16-byte boundaries, rows padded with zeros to whole 16-byte pieces: the copy
// moves each element twice, where reading it unaligned into the tiles cost the products half of their rate and more
// (8191 x 2047 x 8191 bf16: 613 to 961 us).
struct CopyJob {
    const void* src;
    void* dst;
    long long ld;
    int rows, width, pitch;   // of src, in elements; of dst: rows x pitch
};
struct CopyArgs {
    CopyJob job[3];
};
template <typename T> __global__ __launch_bounds__(256) void pad_copy_kernel(const CopyArgs a) {
    constexpr int V = Pack<T>::N;
    const CopyJob& j = a.job[blockIdx.y];
    const int pieces = j.pitch / V;
    const long long total = (long long)j.rows * pieces;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const long long row = total < 0x7fffffff ? (int)i / pieces : i / pieces;
        const int at = (int)(i - row * pieces) * V;
        store16((T*)j.dst + row * j.pitch + at, load16_tail((const T*)j.src + row * j.ld, at, j.width));
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------------
inline int elem(int dtype) { return dtype == DMN_DT_F32 ? 4 : 2; }
inline long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// Tile and k split of a product, from its sizes and type alone, by the times that the tiles were measured to take (MI355X, us):
// `step` per 128 bytes of k and tile of a CU that works through several, `least` for a tile that is alone on its CU, `ends`
// for what stands around the steps (first requests, epilogue, launch); `together` tiles share a CU. The large tile moves the
// fewest bytes per product (8192^3 bf16 forward: 827 us; 128 x 128 with four stages 1078, with two 961, 64 x 64 1582), the others
// leave fewer CUs without work: 4096 x 1024 out of k = 4096 takes 88 us in 64 large tiles and 36 to 41 us in 256 tiles of 128 x
// 128 with four stages each, 43 with two; with 1024 such tiles it is the other way round (4096 x 4096 out of k = 1024: 46 with
// four stages, 38 with two, 34 in 256 large tiles). Where there are too few tiles for the CUs, k is split: the partial
// products are written and read again at some 4 TB/s, in one more launch. `ends` is one figure for every epilogue: a forward that
// keeps z or reads a residual takes longer than its estimate (4096 x 1024 into 4096 with GELU and z: 34 estimated, 48 measured);
// whether another tile would hide that better is not modelled.
struct GemmPlan {
    int tile, splits, per;   // index into kTiles; k tiles are counted in 128 bytes of k
    double us;
};
struct TileShape {
    int bm, bn, together;
    double step16, least16, ends16, step32, least32, ends32;
};
const TileShape kTiles[4] = {{256, 256, 1, 1.60, 1.12, 8.0, 7.4, 7.2, 22.0},
                             {128, 128, 1, 0.56, 0.45, 4.0, 2.0, 1.9, 8.0},
                             {128, 128, 2, 0.50, 0.68, 4.0, 1.9, 2.0, 9.0},
                             {64, 64, 4, 0.22, 0.28, 3.0, 0.55, 0.70, 6.0}};

double join_us(int splits, int M, int N) { return splits > 1 ? 3.0 + (double)splits * M * N * 8 / 4e6 : 0.0; }
GemmPlan gemm_plan(int M, int N, int K, int dtype, int parts) {   // parts of A: k is gone through so often
    const bool f32 = dtype == DMN_DT_F32;
    const long long kt = parts * ceil_div(K, 128 / elem(dtype));
    GemmPlan best{3, 1, (int)kt, 1e30};
    for (int i = 0; i < 4; ++i) {
        const TileShape& t = kTiles[i];
        const double step = f32 ? t.step32 : t.step16, least = f32 ? t.least32 : t.least16, ends = f32 ? t.ends32 : t.ends16;
        const long long tiles = ceil_div(M, t.bm) * ceil_div(N, t.bn);
        for (int splits = 1; splits <= 64 && (splits == 1 || kt / splits >= 4); splits *= 2) {
            const long long per = ceil_div(kt, splits), on_cu = ceil_div(tiles * splits, 256);
            const double all = tiles * splits > 128 ? on_cu * per * step : 0, one = per * least;
            const double us = (all > one ? all : one) + ends * ceil_div(on_cu, t.together) + join_us(splits, M, N);
            if (us < best.us) best = {i, (int)ceil_div(kt, per), (int)per, us};
        }
    }
    return best;
}
// dx and dw in one launch, where that is faster than one after the other: the CUs that one product's tiles leave without work
// take the other's, and tiles of both share a CU. The sum of their k tiles counts, and the longest one among its neighbours;
// the ends of all but the last lie beside other tiles' steps.
struct PairPlan {
    bool together;
    GemmPlan dx, dw;
};
PairPlan pair_plan(int rows, int in, int out, int dtype, int parts) {
    const bool f32 = dtype == DMN_DT_F32;
    const int bk = 128 / elem(dtype);
    const long long kx = parts * ceil_div(out, bk), kw = parts * ceil_div(rows, bk);
    PairPlan best{false, gemm_plan(rows, in, out, dtype, parts), gemm_plan(out, in, rows, dtype, parts)};
    double best_us = best.dx.us + best.dw.us;
    for (int i = 2; i < 4; ++i) {
        const TileShape& t = kTiles[i];
        const double step = f32 ? t.step32 : t.step16, least = f32 ? t.least32 : t.least16, ends = f32 ? t.ends32 : t.ends16;
        const long long tx = ceil_div(rows, t.bm) * ceil_div(in, t.bn), tw = ceil_div(out, t.bm) * ceil_div(in, t.bn);
        for (int sx = 1; sx <= 64 && (sx == 1 || kx / sx >= 4); sx *= 2)
            for (int sw = 1; sw <= 64 && (sw == 1 || kw / sw >= 4); sw *= 2) {
                const long long px = ceil_div(kx, sx), pw = ceil_div(kw, sw), longest = px > pw ? px : pw;
                const long long tiles = tx * sx + tw * sw, on_cu = ceil_div(tiles, 256);
                const double all = tiles > 128 ? step * on_cu * (tx * sx * px + tw * sw * pw) / tiles : 0;
                const double one = longest * (on_cu > 1 ? 2 * step : least);
                const double us = (all > one ? all : one) + ends + join_us(sx, rows, in) + join_us(sw, out, in);
                if (us < best_us) {
                    best_us = us;
                    best = {true, {i, (int)ceil_div(kx, px), (int)px, us}, {i, (int)ceil_div(kw, pw), (int)pw, us}};
                }
            }
    }
    return best;
}
size_t part_bytes(const GemmPlan& p, int M, int N) { return p.splits > 1 ? block_align256((size_t)p.splits * M * N * sizeof(float)) : 0; }
size_t gemm_workspace(int M, int N, int K, int dtype, int parts) {
    return part_bytes(gemm_plan(M, N, K, dtype, parts), M, N);
}
int activation_of(int flags) { return flags & ~DMN_LINEAR_EXACT; }
// Parts of dz, of which z is a float32 argument: see Parts.
int dz_parts(int flags, int dtype) { return dtype != DMN_DT_F32 && activation_of(flags) != ACT_NONE && (flags & DMN_LINEAR_EXACT) ? 2 : 1; }

// An operand in memory: rows of `width` elements, `ld` apart.
struct Operand {
    const void* p;
    long long ld;
    int rows, width;
};
int padded(int width, int dtype) { return (int)ceil_div(width, 16 / elem(dtype)) * (16 / elem(dtype)); }
// Bytes of the copy that the products need of it: none where its rows are whole 16-byte pieces.
size_t copy_bytes(const Operand& o, int dtype) {
    const int e = elem(dtype);
    if ((uintptr_t)o.p % 16 == 0 && (o.ld * e % 16 == 0 || o.rows <= 1) && (long long)o.width * e % 16 == 0) return 0;
    return block_align256((size_t)o.rows * padded(o.width, dtype) * e);
}
// Replaces the operands that need it by their copies, which take the workspace from `ws` on.
template <typename T> int copy_operands(Operand** list, int n, int dtype, char*& ws, hipStream_t s) {
    CopyArgs a{};
    int jobs = 0;
    long long most = 0;
    for (int i = 0; i < n; ++i) {
        Operand& o = *list[i];
        const size_t bytes = copy_bytes(o, dtype);
        if (!bytes) continue;
        const int pitch = padded(o.width, dtype);
        a.job[jobs++] = {o.p, ws, o.ld, o.rows, o.width, pitch};
        most = bytes / 16 > (size_t)most ? (long long)(bytes / 16) : most;
        o.p = ws;
        o.ld = pitch;
        ws += bytes;
    }
    if (!jobs) return DMN_OK;
    const long long blocks = ceil_div(most, 256);
    pad_copy_kernel<T><<<dim3((unsigned)(blocks < 4096 ? blocks : 4096), jobs), 256, 0, s>>>(a);
    DMN_BLOCK_LAUNCH_CHECK();
    return DMN_OK;
}

template <typename F> int allow_lds(F* kernel, int bytes) {
    if (bytes > 65536) DMN_HIP_CHECK(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    return DMN_OK;
}
template <typename T, bool XA, bool XB, bool TWO, int BM, int BN, int WM, int WN, int S> int pipe_launch(const GemmArgs& g, hipStream_t s) {
    constexpr int NT = (BM / WM) * (BN / WN) * 64, LDS = S * (BM + BN) * 128;
    static_assert((NT / 64) * 2 * 16 * (WN + 4) * 4 <= LDS, "the epilogue's pieces fit the tiles' memory");
    auto* kernel = gemm_pipe_kernel<T, XA, XB, TWO, BM, BN, WM, WN, S>;
    const int rc = allow_lds(kernel, LDS);
    if (rc) return rc;
    kernel<<<dim3((unsigned)(ceil_div(g.M, BM) * ceil_div(g.N, BN)), g.splits), NT, LDS, s>>>(g);
    DMN_BLOCK_LAUNCH_CHECK();
    return DMN_OK;
}
template <typename T, int G> int join_launch(const GemmArgs& g, hipStream_t s) {
    gemm_join_kernel<T, G><<<(unsigned)ceil_div((long long)g.M * ceil_div(g.N, Pack<T>::N), 256 / G), 256, 0, s>>>(g);
    DMN_BLOCK_LAUNCH_CHECK();
    return DMN_OK;
}
// Whether the forward takes the kernel for few rows. Its workgroups read all of x each, so x has to be small (us, this kernel
// against tiles, weights not in the caches: 64 x 2048 into 8192 bf16 17 : 25, 32 x 1000 into 1531 5 : 10, but 32 x 8192 into
// 2048 27 : 18 and 64 x 8192 42 : 19); and few columns of a long k leave it CUs without work (16 x 8192 into 2048 19 : 14,
// 16 x 4096 into 512 10 : 10; one row 13 : 14, in float32, where the tiles split k, 30 : 25).
// Where the weight's rows are off 16-byte boundaries the tiles would need a copy of it, and this kernel's loads are slow, the
// more so the more of x's rows there are; both sides are estimated in us from these times (this kernel : copy and tiles):
// bf16, k = 4095 into 4095, 1 row 17 : 27, 16 rows 28 : 28, 40 rows 52 : 31; 4095 into 1023, 1 row 17 : 17, 16 rows 28 : 18; 8191
// into 8191, 4 rows 76 : 83, 16 rows 100 : 86; float32, 4095 into 4095, 16 rows 25 : 49, 40 rows 42 : 50; 8191 into 2047, 8 rows
// 41 : 50, 40 rows 77 : 51. One estimate serves all types; it takes the slower side at float32 8191 into 8191 with 40 and 64 rows (131
// and 138 : 205) and, by less, at float32 4095 into 1023 with 8 (21 : 25).
bool few_rows(const Operand& w, int M, int dtype) {
    const int N = w.rows, K = w.width;
    const long long bytes = (long long)K * elem(dtype);
    if (M <= 64 && copy_bytes(w, dtype)) return 2.5 + K * 3.2e-3 * (1 + 0.055 * M) * (N > 4096 ? N / 4096. : 1.) < 11 + 0.55e-6 * bytes * N;
    return M <= 64 && M * bytes <= 256 * 1024 && (M < 8 || N >= 4096 || bytes < 8192);
}
template <typename T, int MF, int NF, int WAVES> int few_rows_launch(const GemmArgs& g, hipStream_t s) {
    constexpr int LDS = WAVES * MF * NF * 1024;
    static_assert(LDS <= 65536, "LDS without an attribute");
    gemm_few_rows_kernel<T, MF, NF, WAVES><<<(unsigned)ceil_div(g.N, 16 * NF), WAVES * 64, LDS, s>>>(g);
    DMN_BLOCK_LAUNCH_CHECK();
    return DMN_OK;
}
template <typename T> int few_rows_run(const GemmArgs& g, hipStream_t s) {
    // columns per workgroup: more of them read x less often, fewer fill the chip; waves: some sixteen per CU
    const long long cols = ceil_div(g.N, 16);
    if (g.M <= 16) return cols >= 256 ? few_rows_launch<T, 1, 1, 8>(g, s) : few_rows_launch<T, 1, 1, 16>(g, s);
    if (g.M <= 32) return cols >= 512 ? few_rows_launch<T, 2, 2, 8>(g, s) : few_rows_launch<T, 2, 1, 16>(g, s);
    return cols >= 1024 ? few_rows_launch<T, 4, 4, 4>(g, s) : cols >= 512 ? few_rows_launch<T, 4, 2, 8>(g, s) : few_rows_launch<T, 4, 1, 16>(g, s);
}

void set_plan(GemmArgs& g, const GemmPlan& p, void* ws) {
    g.splits = p.splits;
    g.tiles_per_split = p.per;
    g.part = p.splits > 1 ? (float*)ws : nullptr;
}
template <typename T> int join_run(const GemmArgs& g, hipStream_t s) {
    if (g.splits == 1) return DMN_OK;
    // eight threads per piece where there are few of them
    return g.splits >= 8 && (long long)g.M * g.N < (1 << 20) ? join_launch<T, 8>(g, s) : join_launch<T, 1>(g, s);
}
template <typename T, bool XA, bool XB, bool TWO> int tile_run(const GemmArgs& g, int tile, hipStream_t s) {
    if (tile == 0) return pipe_launch<T, XA, XB, TWO, 256, 256, 128, 64, 2>(g, s);
    if (tile == 1) return pipe_launch<T, XA, XB, TWO, 128, 128, 64, 32, 4>(g, s);
    if (tile == 2) return pipe_launch<T, XA, XB, TWO, 128, 128, 64, 32, 2>(g, s);
    return pipe_launch<T, XA, XB, TWO, 64, 64, 32, 32, 2>(g, s);
}
// C = sum_k A B with the operands on 16-byte boundaries (copy_operands).
template <typename T, bool XA, bool XB> int gemm_run(GemmArgs& g, int dtype, void* ws, hipStream_t s) {
    const GemmPlan p = gemm_plan(g.M, g.N, g.K, dtype, g.a2 ? 2 : 1);
    set_plan(g, p, ws);
    int rc = DMN_ERR_INVALID;
    if (!g.a2) rc = tile_run<T, XA, XB, false>(g, p.tile, s);
    else if constexpr (XB && sizeof(T) == 2) rc = tile_run<T, XA, XB, true>(g, p.tile, s);
    return rc ? rc : join_run<T>(g, s);
}
template <typename T, bool TWO, int BM, int BN, int WM, int WN, int S> int pair_launch(const PairArgs& a, hipStream_t s) {
    constexpr int NT = (BM / WM) * (BN / WN) * 64, LDS = S * (BM + BN) * 128;
    static_assert(LDS <= 65536, "LDS without an attribute");
    gemm_pair_kernel<T, TWO, BM, BN, WM, WN, S><<<(unsigned)(a.db_at + (a.db.out ? ceil_div(a.db.n, 32) : 0)), NT, LDS, s>>>(a);
    DMN_BLOCK_LAUNCH_CHECK();
    return DMN_OK;
}
template <typename T, bool TWO> int pair_tile_run(const PairArgs& a, int tile, hipStream_t s) {
    return tile == 2 ? pair_launch<T, TWO, 128, 128, 64, 32, 2>(a, s) : pair_launch<T, TWO, 64, 64, 32, 32, 2>(a, s);
}
// dx, dw and the join of db's partial sums; their partial products lie one behind the other in the workspace.
template <typename T> int pair_run(GemmArgs& dx, GemmArgs& dw, const ColumnJoin& db, const PairPlan& p, char* ws, hipStream_t s) {
    set_plan(dx, p.dx, ws);
    set_plan(dw, p.dw, ws + part_bytes(p.dx, dx.M, dx.N));
    const TileShape& t = kTiles[p.dx.tile];
    PairArgs a{dx, dw, (int)(ceil_div(dx.M, t.bm) * ceil_div(dx.N, t.bn)), (int)(ceil_div(dw.M, t.bm) * ceil_div(dw.N, t.bn)), 0, 0, 0, db};
    a.db_at = a.dx_tiles * dx.splits + a.dw_tiles * dw.splits;
    if (p.dx.per >= p.dw.per) a.dw_at = a.dx_tiles * dx.splits;
    else a.dx_at = a.dw_tiles * dw.splits;
    int rc = DMN_ERR_INVALID;
    if (!dx.a2) rc = pair_tile_run<T, false>(a, p.dx.tile, s);
    else if constexpr (sizeof(T) == 2) rc = pair_tile_run<T, true>(a, p.dx.tile, s);
    if (!rc) rc = join_run<T>(dx, s);
    return rc ? rc : join_run<T>(dw, s);
}

template <typename T> int forward_run(GemmArgs& g, int dtype, char* ws, hipStream_t s) {
    Operand x{g.a, g.lda, g.M, g.K}, w{g.b, g.ldb, g.N, g.K};
    if (few_rows(w, g.M, dtype)) return few_rows_run<T>(g, s);
    Operand* list[2] = {&x, &w};
    const int rc = copy_operands<T>(list, 2, dtype, ws, s);
    if (rc) return rc;
    g.a = x.p;
    g.lda = x.ld;
    g.b = w.p;
    g.ldb = w.ld;
    return gemm_run<T, false, false>(g, dtype, ws, s);
}

// Runs of rows that dz_kernel's workgroups take: more of them keep more CUs busy, and each leaves a partial row of column sums that
// the join has to read. dz's sums and their join, 16 : 64 : 256 : 1024 runs at most, us: 4096 x 4096 bf16 28 : 24 : 22 : 22, 4001 x 1024
// 23 : 10 : 12 : 12, 16384 x 1024 float32 59 : 23 : 25 : 29; narrow outputs, where 64 runs are 64 workgroups, would take more: 65536 x
// 64 bf16 305 : 80 : 27 : 17.
constexpr int kMaxDzRuns = 64;
int dz_runs(int M) { return (int)(ceil_div(M, 64) < kMaxDzRuns ? ceil_div(M, 64) : kMaxDzRuns); }

int linear_check(const char* who, int64_t rows, int in, int out, int act, int dtype, int64_t ldx) {
    DMN_REQUIRE(dtype >= 0 && dtype <= 2, DMN_ERR_INVALID, "%s: dtype must be DMN_DT_F32, _BF16 or _F16", who);
    DMN_REQUIRE(activation_of(act) >= ACT_NONE && activation_of(act) <= ACT_GELU, DMN_ERR_INVALID, "%s: unknown activation %d", who, act);
    DMN_REQUIRE(rows >= 0 && in > 0 && out > 0, DMN_ERR_INVALID, "%s: rows must be >= 0, in and out > 0", who);
    DMN_REQUIRE(rows < (1 << 27) && in < (1 << 20) && out < (1 << 20) && rows * (in > out ? in : out) < ((int64_t)1 << 40), DMN_ERR_LIMIT,
                "%s: rows must be below 2^27, in and out below 2^20", who);
    DMN_REQUIRE(rows <= 1 || ldx >= in, DMN_ERR_INVALID, "%s: row stride of x below its width", who);
    DMN_REQUIRE(ldx < (1 << 20), DMN_ERR_LIMIT, "%s: row stride of x must be below 2^20 elements", who);
    return DMN_OK;
}

template <typename T>
int backward_run(const void* dy, long long lddy, const void* x, long long ldx, const void* w, const void* z, void* dx, void* dw, void* db,
                 int rows, int in, int out, int flags, int dtype, char* ws, hipStream_t s) {
    if (rows == 0) {
        if (dw) zero_kernel<T><<<1024, 256, 0, s>>>((T*)dw, (long long)in * out);
        DMN_BLOCK_LAUNCH_CHECK();
        if (db) zero_kernel<T><<<64, 256, 0, s>>>((T*)db, out);
        DMN_BLOCK_LAUNCH_CHECK();
        return DMN_OK;
    }
    const int act = activation_of(flags), parts = dz_parts(flags, dtype);
    float* part = (float*)ws;
    const int runs = dz_runs(rows);
    ws += block_align256((size_t)runs * out * sizeof(float));
    ColumnJoin join{part, runs, out, nullptr};
    Operand z_{dy, lddy, rows, out}, w_{w, in, out, in}, x_{x, ldx, rows, in};
    const void* low = nullptr;
    if (act != ACT_NONE || db) {
        DzArgs a{};
        a.dy = dy;
        a.z = z;
        a.lddy = lddy;
        a.dz = act != ACT_NONE && (dx || dw) ? ws : nullptr;
        a.lddz = padded(out, dtype);
        const size_t dz_bytes = block_align256((size_t)rows * a.lddz * sizeof(T));
        a.low = parts == 2 ? ws + dz_bytes : nullptr;
        a.part = db ? part : nullptr;
        a.M = rows;
        a.N = out;
        a.act = act;
        const dim3 grid((unsigned)ceil_div(out, 16 * Pack<T>::N), runs);
        if (parts == 2) dz_kernel<T, sizeof(T) == 2><<<grid, 256, 0, s>>>(a);
        else dz_kernel<T, false><<<grid, 256, 0, s>>>(a);
        DMN_BLOCK_LAUNCH_CHECK();
        join.out = db;
        if (act != ACT_NONE) {
            z_.p = ws;
            z_.ld = a.lddz;
            z_.width = (int)a.lddz;
            low = a.low;
            ws += parts * dz_bytes;
        }
    }
    Operand* list[3];
    int n = 0;
    if (dx || dw) list[n++] = &z_;
    if (dx) list[n++] = &w_;
    if (dw) list[n++] = &x_;
    int rc = copy_operands<T>(list, n, dtype, ws, s);
    if (rc) return rc;
    GemmArgs gx{}, gw{};
    gx.a = gw.a = z_.p;
    gx.a2 = gw.a2 = low;
    gx.lda = gw.lda = z_.ld;
    gx.b = w_.p;
    gx.ldb = w_.ld;
    gx.M = rows;
    gx.K = out;
    gx.y = dx;
    gw.b = x_.p;
    gw.ldb = x_.ld;
    gw.M = out;
    gw.K = rows;
    gw.y = dw;
    gx.N = gw.N = in;
    if (dx && dw) {
        const PairPlan p = pair_plan(rows, in, out, dtype, parts);
        if (p.together) return pair_run<T>(gx, gw, join, p, ws, s);
    }
    if (join.out) {
        column_join_kernel<T><<<(unsigned)ceil_div(out, 32), 256, 0, s>>>(join);
        DMN_BLOCK_LAUNCH_CHECK();
    }
    if (dx) rc = gemm_run<T, false, true>(gx, dtype, ws, s);
    if (dw && !rc) rc = gemm_run<T, true, true>(gw, dtype, ws, s);
    return rc;
}

}  // namespace

extern "C" size_t dmn_linear_forward_workspace_bytes(const void* x, int64_t ldx, const void* weight, int64_t rows, int in, int out, int dtype) {
    if (rows <= 0 || rows >= (1 << 27) || in <= 0 || out <= 0 || dtype < 0 || dtype > 2) return 0;
    if (few_rows({weight, in, out, in}, (int)rows, dtype)) return 0;
    return gemm_workspace((int)rows, out, in, dtype, 1) + copy_bytes({x, ldx, (int)rows, in}, dtype) + copy_bytes({weight, in, out, in}, dtype);
}

extern "C" int dmn_linear_forward(const void* x, int64_t ldx, const void* weight, const void* bias, const void* residual, int64_t ldr,
                                  void* y, void* z, int64_t rows, int in, int out, int activation, int dtype, void* workspace,
                                  size_t workspace_bytes, void* stream) {
    int rc = linear_check("dmn_linear_forward", rows, in, out, activation, dtype, ldx);
    if (rc || rows == 0) return rc;
    DMN_REQUIRE(x && weight && y, DMN_ERR_INVALID, "dmn_linear_forward: null argument");
    DMN_REQUIRE(!residual || rows <= 1 || ldr >= out, DMN_ERR_INVALID, "dmn_linear_forward: row stride of the residual below its width");
    const size_t need = dmn_linear_forward_workspace_bytes(x, ldx, weight, rows, in, out, dtype);
    DMN_REQUIRE(need == 0 || (workspace && (uintptr_t)workspace % 256 == 0 && workspace_bytes >= need), DMN_ERR_WORKSPACE,
                "dmn_linear_forward: workspace of %zu bytes, %zu needed (256-byte aligned)", workspace_bytes, need);
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
    g.z_exact = (activation & DMN_LINEAR_EXACT) != 0;
    g.act = activation_of(activation);
    hipStream_t s = (hipStream_t)stream;
    char* ws = (char*)workspace;
    if (dtype == DMN_DT_F32) return forward_run<float>(g, dtype, ws, s);
    if (dtype == DMN_DT_BF16) return forward_run<__bf16>(g, dtype, ws, s);
    return forward_run<f16>(g, dtype, ws, s);
}

extern "C" size_t dmn_linear_backward_workspace_bytes(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* weight, int64_t rows,
                                                      int in, int out, int activation, int dtype) {
    if (rows <= 0 || rows >= (1 << 27) || in <= 0 || out <= 0 || dtype < 0 || dtype > 2) return 0;
    const int parts = dz_parts(activation, dtype);
    const size_t dx = gemm_workspace((int)rows, in, out, dtype, parts), dw = gemm_workspace(out, in, (int)rows, dtype, parts);
    const PairPlan p = pair_plan((int)rows, in, out, dtype, parts);
    const size_t pair = p.together ? part_bytes(p.dx, (int)rows, in) + part_bytes(p.dw, out, in) : 0, one = dx > dw ? dx : dw;
    const size_t dz = activation_of(activation) != ACT_NONE ? parts * block_align256((size_t)rows * padded(out, dtype) * elem(dtype)) : copy_bytes({dy, lddy, (int)rows, out}, dtype);
    return block_align256((size_t)dz_runs((int)rows) * out * sizeof(float)) + dz + copy_bytes({x, ldx, (int)rows, in}, dtype) +
           copy_bytes({weight, in, out, in}, dtype) + (pair > one ? pair : one);
}

extern "C" int dmn_linear_backward(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* weight, const void* z, void* dx,
                                   void* dweight, void* dbias, int64_t rows, int in, int out, int activation, int dtype, void* workspace,
                                   size_t workspace_bytes, void* stream) {
    int rc = linear_check("dmn_linear_backward", rows, in, out, activation, dtype, ldx);
    if (rc) return rc;
    if (!dx && !dweight && !dbias) return DMN_OK;
    DMN_REQUIRE(rows == 0 || (dy && (!dx || weight) && (!dweight || x) && (activation_of(activation) == ACT_NONE || z)), DMN_ERR_INVALID,
                "dmn_linear_backward: null argument");
    DMN_REQUIRE(rows <= 1 || lddy >= out, DMN_ERR_INVALID, "dmn_linear_backward: row stride of dy below its width");
    DMN_REQUIRE(lddy < (1 << 20), DMN_ERR_LIMIT, "dmn_linear_backward: row stride of dy must be below 2^20 elements");
    const size_t need = dmn_linear_backward_workspace_bytes(dy, lddy, x, ldx, weight, rows, in, out, activation, dtype);
    DMN_REQUIRE(need == 0 || (workspace && (uintptr_t)workspace % 256 == 0 && workspace_bytes >= need), DMN_ERR_WORKSPACE,
                "dmn_linear_backward: workspace of %zu bytes, %zu needed (256-byte aligned)", workspace_bytes, need);
    hipStream_t s = (hipStream_t)stream;
    char* ws = (char*)workspace;
    if (dtype == DMN_DT_F32) return backward_run<float>(dy, lddy, x, ldx, weight, z, dx, dweight, dbias, (int)rows, in, out, activation, dtype, ws, s);
    if (dtype == DMN_DT_BF16) return backward_run<__bf16>(dy, lddy, x, ldx, weight, z, dx, dweight, dbias, (int)rows, in, out, activation, dtype, ws, s);
    return backward_run<f16>(dy, lddy, x, ldx, weight, z, dx, dweight, dbias, (int)rows, in, out, activation, dtype, ws, s);
}

extern "C" int dmn_test_linear_plan(int64_t rows, int in, int out, int activation, int dtype, int alone, int* plan) {
    const int rc = linear_check("dmn_test_linear_plan", rows, in, out, activation, dtype, in);
    if (rc) return rc;
    DMN_REQUIRE(plan && rows > 0, DMN_ERR_INVALID, "dmn_test_linear_plan: null argument or no rows");
    const int parts = dz_parts(activation, dtype);
    const GemmPlan f = gemm_plan((int)rows, out, in, dtype, 1);
    PairPlan b = pair_plan((int)rows, in, out, dtype, parts);
    if (alone) b = {false, gemm_plan((int)rows, in, out, dtype, parts), gemm_plan(out, in, (int)rows, dtype, parts)};
    const bool few = few_rows({nullptr, in, out, in}, (int)rows, dtype);
    const int all[7] = {few ? -1 : f.tile, few ? 1 : f.splits, b.together, b.dx.tile, b.dx.splits, b.dw.tile, b.dw.splits};
    for (int i = 0; i < 7; ++i) plan[i] = all[i];
    return DMN_OK;
}
