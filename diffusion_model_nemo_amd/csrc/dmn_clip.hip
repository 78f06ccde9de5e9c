// Global norm of many gradient tensors, and clipping: norm = grad_scale sqrt(sum g^2) or grad_scale max |g| over all of
// them, c = min(1, max_norm / (norm + 1e-6)), dst = src * grad_scale * c.
//
// Bound by memory (and, for the usual few hundred small tensors, by launches): one launch reads every element once and
// leaves one partial per workgroup, one launch scales. Squares are added in float64, so a norm neither overflows nor
// loses small gradients beside large ones for any finite input, and the conversions and sums hide behind the loads (the
// part adds float64 at half its float32 rate, ten times what the memory delivers; with float32 sums the norm takes as long).
// 403 M bfloat16 elements: norm 127 us (6.3 TB/s), scaling into float32 490 us (4.9 TB/s); 256 tensors with 8 M elements: 8
// and 4 us. Every workgroup of the second launch
// adds the same partials in the same order: one norm, bit for bit, everywhere and on every run.
// The tensors' addresses travel in the kernel arguments (a launch carries as many as fit 4 KB), so nothing has to be copied
// to the device first and a captured call keeps the table it was captured with.
#include <math.h>
#include <stdlib.h>

#include "dmn_block.h"

namespace {

constexpr int kThreads = 256;
constexpr int kBlocks = 2048;       // workgroups of one launch: eight per CU, resident together
constexpr int64_t kKeep = 80 << 20;  // bytes that the cache behind the L2s is trusted to keep between the passes
constexpr int kPiece = 8192;        // elements that a workgroup takes at a time: neighbouring workgroups read neighbouring pieces

// Tensors of one launch: entry i owns the pieces [first[i], first[i + 1]). An entry takes twelve bytes, so that the default
// network's 256 gradients are one launch: where[i] is the address (47 bits, all that user space has), the types as source +
// 3 * destination (4 bits) and the elements of the last piece less one (13 bits).
template <bool OUT> struct ClipTable {
    static constexpr int K = OUT ? 196 : 330;
    int count, part_base;           // entries; index of the launch's first partial among all
    int first[K + 1];
    unsigned long long where[K];
    void* dst[OUT ? K : 1];
};
static_assert(sizeof(ClipTable<true>) <= 4000 && sizeof(ClipTable<false>) <= 4000 && kPiece == 1 << 13, "kernel arguments");

struct PieceOf {                    // one piece of an entry
    const void* src;
    int st, dt, len;
    long long at;                   // its first element
};
template <bool OUT> __device__ __forceinline__ PieceOf piece_of(const ClipTable<OUT>& t, int e, int p) {
    const unsigned long long w = t.where[e];
    const int types = (int)(w >> 47) & 15, last = (int)(w >> 51) + 1;
    return {(const void*)(w & ((1ull << 47) - 1)), types % 3, types / 3, p + 1 == t.first[e + 1] ? last : kPiece, (long long)(p - t.first[e]) * kPiece};
}

struct ClipScale {
    const double* part;
    int parts;
    int inf_norm, write_norm;
    float max_norm, grad_scale;
    float* norm;
};

__device__ __forceinline__ double max_nan(double a, double b) { return (b > a || b != b) ? b : a; }   // a NaN stays

// The sum (or maximum) over the workgroup, in every thread, in a fixed order.
__device__ __forceinline__ double block_join(double v, int inf_norm, double* sh) {
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        const double w = __shfl_xor(v, o);
        v = inf_norm ? max_nan(v, w) : v + w;
    }
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh[0];
#pragma unroll
    for (int i = 1; i < kThreads / 64; ++i) v = inf_norm ? max_nan(v, sh[i]) : v + sh[i];
    return v;
}

// STREAM: the data is not kept in the caches.
template <typename T, bool INF, bool STREAM> __device__ __forceinline__ double piece_norm(const T* p, int n) {
    constexpr int V = Pack<T>::N;
    double acc[4] = {0., 0., 0., 0.};
    auto add = [&](float x, int k) {
        if constexpr (INF) acc[k & 3] = max_nan(acc[k & 3], (double)fabsf(x));
        else acc[k & 3] = __builtin_fma((double)x, (double)x, acc[k & 3]);
    };
    int i = threadIdx.x * V;
    constexpr int STEP = kThreads * V;
    typedef typename Pack<T>::vec loose __attribute__((aligned(sizeof(T))));
    for (; i + 3 * STEP + V <= n; i += 4 * STEP) {
        typename Pack<T>::vec v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if constexpr (STREAM) v[k] = __builtin_nontemporal_load((const loose*)(p + i + k * STEP));
            else v[k] = load16(p + i + k * STEP);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) add((float)v[k][j], k);
    }
    for (; i < n; i += STEP) {
        if (i + V <= n) {
            const typename Pack<T>::vec v = load16(p + i);
#pragma unroll
            for (int j = 0; j < V; ++j) add((float)v[j], j);
        } else {
            for (int j = 0; i + j < n; ++j) add((float)p[i + j], 0);
        }
    }
    return INF ? max_nan(max_nan(acc[0], acc[1]), max_nan(acc[2], acc[3])) : (acc[0] + acc[1]) + (acc[2] + acc[3]);
}

// Entry of piece `p` (p < first[count]): binary search over scalars.
template <bool OUT> __device__ __forceinline__ int find_entry(const ClipTable<OUT>& t, int p) {
    int lo = 0, hi = t.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.first[mid] <= p) lo = mid;
        else hi = mid;
    }
    return lo;
}

template <bool INF, bool STREAM> __device__ __forceinline__ double piece_norm_of(const void* src, int dt, long long at, int n) {
    if (dt == DMN_DT_F32) return piece_norm<float, INF, STREAM>((const float*)src + at, n);
    if (dt == DMN_DT_BF16) return piece_norm<__bf16, INF, STREAM>((const __bf16*)src + at, n);
    return piece_norm<f16, INF, STREAM>((const f16*)src + at, n);
}
// Pieces below `stream_pieces` are read past the caches.
template <bool INF> __global__ __launch_bounds__(kThreads) void grad_norm_kernel(const ClipTable<false> t, double* part, int stream_pieces) {
    __shared__ double sh[kThreads / 64];
    const int pieces = t.first[t.count];
    double v = 0.;
    int e = find_entry(t, blockIdx.x);
    for (int p = blockIdx.x; p < pieces; p += gridDim.x) {
        while (t.first[e + 1] <= p) ++e;
        const PieceOf q = piece_of(t, e, p);
        const double w = p < stream_pieces ? piece_norm_of<INF, true>(q.src, q.st, q.at, q.len) : piece_norm_of<INF, false>(q.src, q.st, q.at, q.len);
        v = INF ? max_nan(v, w) : v + w;
    }
    v = block_join(v, INF, sh);
    if (threadIdx.x == 0) part[t.part_base + blockIdx.x] = v;
}

// The factor of every element from the partials of all launches.
__device__ __forceinline__ float clip_factor(const ClipScale& c, double* sh, float* norm_out) {
    double v = 0.;
    for (int i = threadIdx.x; i < c.parts; i += kThreads) v = c.inf_norm ? max_nan(v, c.part[i]) : v + c.part[i];
    v = block_join(v, c.inf_norm, sh);
    const double norm = (c.inf_norm ? v : sqrt(v)) * fabs((double)c.grad_scale);
    *norm_out = (float)norm;
    const double f = (double)c.max_norm / (norm + 1e-6);
    return (float)((f >= 1.0 ? 1.0 : f) * (double)c.grad_scale);   // a NaN stays
}

template <typename S, typename D> __device__ __forceinline__ void piece_scale(const S* src, D* dst, int n, float f) {
    constexpr int V = Pack<S>::N, W = Pack<D>::N, STEP = kThreads * V;
    auto put = [&](typename Pack<S>::vec v, int i) {
        if constexpr (V >= W) {
#pragma unroll
            for (int k = 0; k < V / W; ++k) {
                typename Pack<D>::vec o;
#pragma unroll
                for (int j = 0; j < W; ++j) o[j] = (D)((float)v[k * W + j] * f);
                store16(dst + i + k * W, o);
            }
        } else {   // float32 source, 16-bit destination: eight bytes
            D o[V];
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] = (D)((float)v[j] * f);
            __builtin_memcpy(dst + i, o, sizeof(o));
        }
    };
    int i = threadIdx.x * V;
    for (; i + 3 * STEP + V <= n; i += 4 * STEP) {
        typename Pack<S>::vec v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = load16(src + i + k * STEP);
#pragma unroll
        for (int k = 0; k < 4; ++k) put(v[k], i + k * STEP);
    }
    for (; i < n; i += STEP) {
        if (i + V <= n) put(load16(src + i), i);
        else
            for (int j = 0; i + j < n; ++j) dst[i + j] = (D)((float)src[i + j] * f);
    }
}

template <typename S> __device__ __forceinline__ void piece_scale_to(const void* src, void* dst, int dt, long long at, int n, float f) {
    const S* s = (const S*)src + at;
    if (dt == DMN_DT_F32) piece_scale(s, (float*)dst + at, n, f);
    else if (dt == DMN_DT_BF16) piece_scale(s, (__bf16*)dst + at, n, f);
    else piece_scale(s, (f16*)dst + at, n, f);
}

template <bool OUT> __global__ __launch_bounds__(kThreads) void grad_scale_kernel(const ClipTable<OUT> t, const ClipScale c) {
    __shared__ double sh[kThreads / 64];
    float norm;
    const float f = clip_factor(c, sh, &norm);
    if (c.write_norm && blockIdx.x == 0 && threadIdx.x == 0) *c.norm = norm;
    if (!OUT && f == 1.0f) return;    // in place and within the limit: the tensors are what they should be
    // from the end, which was read last and may still be in the cache
    int e = t.count - 1;
    for (int p = t.first[t.count] - 1 - (int)blockIdx.x; p >= 0; p -= gridDim.x) {
        while (t.first[e] > p) --e;
        const PieceOf q = piece_of(t, e, p);
        void* dst = OUT ? t.dst[e] : (void*)q.src;
        if (q.st == DMN_DT_F32) piece_scale_to<float>(q.src, dst, OUT ? q.dt : DMN_DT_F32, q.at, q.len, f);
        else if (q.st == DMN_DT_BF16) piece_scale_to<__bf16>(q.src, dst, OUT ? q.dt : DMN_DT_BF16, q.at, q.len, f);
        else piece_scale_to<f16>(q.src, dst, OUT ? q.dt : DMN_DT_F16, q.at, q.len, f);
    }
}

__global__ __launch_bounds__(kThreads) void grad_norm_only_kernel(const ClipScale c) {
    __shared__ double sh[kThreads / 64];
    float norm;
    (void)clip_factor(c, sh, &norm);
    if (threadIdx.x == 0) *c.norm = norm;
}

inline int dt_bytes(int dt) { return dt == DMN_DT_F32 ? 4 : 2; }

struct Range {
    uintptr_t from, to;
    int written;
};
int range_order(const void* a, const void* b) {
    const Range *x = (const Range*)a, *y = (const Range*)b;
    return x->from < y->from ? -1 : x->from > y->from ? 1 : 0;
}

// A written range may touch no other range: workgroups run in any order, so a gradient that is listed twice would be
// scaled once or twice as it falls. 0: fine, 1: overlap, 2: no memory.
int ranges_overlap(const DmnGradTensor* t, int n) {
    Range* r = (Range*)malloc(sizeof(Range) * 2 * (size_t)n);
    if (!r) return 2;
    int m = 0;
    for (int i = 0; i < n; ++i) {
        if (t[i].numel == 0) continue;
        const uintptr_t s = (uintptr_t)t[i].src, d = (uintptr_t)t[i].dst;
        r[m++] = {d, d + (uintptr_t)t[i].numel * dt_bytes(t[i].dst_dtype), 1};
        if (s != d || t[i].src_dtype != t[i].dst_dtype) r[m++] = {s, s + (uintptr_t)t[i].numel * dt_bytes(t[i].src_dtype), 0};
    }
    qsort(r, m, sizeof(Range), range_order);
    uintptr_t any = 0, written = 0;
    int bad = 0;
    for (int i = 0; i < m && !bad; ++i) {
        if (r[i].from < (r[i].written ? any : written)) bad = 1;
        if (r[i].to > any) any = r[i].to;
        if (r[i].written && r[i].to > written) written = r[i].to;
    }
    free(r);
    return bad;
}

// Workgroups of one of the launches that n tensors need (at most): fewer where there are many launches, because every
// workgroup of the second kind adds the partials of all of them.
int blocks_per_launch(int n) {
    const int launches = (n + ClipTable<false>::K - 1) / ClipTable<false>::K;
    return launches <= 4 ? kBlocks : launches <= 16 ? kBlocks / 4 : kBlocks / 16;
}

// Hands `emit` one launch's table after the other with its workgroups; the partials' indices run on over the launches.
// The third argument is the index of the last tensor in the table.
template <bool OUT, typename F> int for_tables(const DmnGradTensor* t, int n, F emit) {
    ClipTable<OUT> tab;
    tab.count = 0;
    tab.part_base = 0;
    tab.first[0] = 0;
    const int most = blocks_per_launch(n);
    int rc = DMN_OK;
    for (int i = 0; i < n && !rc; ++i) {
        if (t[i].numel > 0) {
            const int k = tab.count++;
            const int64_t pieces = (t[i].numel + kPiece - 1) / kPiece;
            tab.where[k] = (unsigned long long)(uintptr_t)t[i].src | (unsigned long long)(t[i].src_dtype + 3 * t[i].dst_dtype) << 47 |
                           (unsigned long long)(t[i].numel - (pieces - 1) * kPiece - 1) << 51;
            if (OUT) tab.dst[OUT ? k : 0] = t[i].dst;
            tab.first[k + 1] = tab.first[k] + (int)pieces;
        }
        if (tab.count == ClipTable<OUT>::K || (i == n - 1 && tab.count)) {
            const int pieces = tab.first[tab.count], blocks = pieces < most ? pieces : most;
            rc = emit(tab, blocks, i);
            tab.part_base += blocks;
            tab.count = 0;
        }
    }
    return rc;
}

}  // namespace

extern "C" size_t dmn_clip_grads_workspace_bytes(int n_tensors) {
    if (n_tensors < 0) return 0;
    const size_t launches = ((size_t)n_tensors + ClipTable<false>::K - 1) / ClipTable<false>::K;
    return launches * blocks_per_launch(n_tensors) * sizeof(double) + 256;
}

extern "C" int dmn_clip_grads(const DmnGradTensor* tensors, int n_tensors, int inf_norm, float max_norm, float grad_scale, float* norm,
                              void* workspace, size_t workspace_bytes, void* stream) {
    DMN_REQUIRE(norm && workspace && n_tensors >= 0 && (tensors || n_tensors == 0), DMN_ERR_INVALID, "dmn_clip_grads: null argument");
    DMN_REQUIRE(n_tensors <= (1 << 20), DMN_ERR_LIMIT, "dmn_clip_grads: more than 2^20 tensors");
    DMN_REQUIRE((inf_norm == 0 || inf_norm == 1) && max_norm >= 0.f && isfinite(grad_scale), DMN_ERR_INVALID,
                "dmn_clip_grads: inf_norm must be 0 or 1, max_norm >= 0 and grad_scale finite");
    DMN_REQUIRE((uintptr_t)workspace % 8 == 0 && workspace_bytes >= dmn_clip_grads_workspace_bytes(n_tensors), DMN_ERR_WORKSPACE,
                "dmn_clip_grads: workspace of %zu bytes, %zu needed (8-byte aligned)", workspace_bytes, dmn_clip_grads_workspace_bytes(n_tensors));
    int64_t total = 0, bytes = 0;
    int writes = 0, separate = 0;
    for (int i = 0; i < n_tensors; ++i) {
        const DmnGradTensor& t = tensors[i];
        DMN_REQUIRE(t.numel >= 0 && t.numel < ((int64_t)1 << 40) && t.src_dtype >= 0 && t.src_dtype <= 2 && t.dst_dtype >= 0 && t.dst_dtype <= 2,
                    DMN_ERR_INVALID, "dmn_clip_grads: tensor %d has a bad size or type", i);
        if (t.numel == 0) continue;
        DMN_REQUIRE(((uintptr_t)t.src | (uintptr_t)t.dst) >> 47 == 0, DMN_ERR_INVALID, "dmn_clip_grads: tensor %d has an impossible address", i);
        DMN_REQUIRE(t.src && (uintptr_t)t.src % dt_bytes(t.src_dtype) == 0 && (uintptr_t)t.dst % dt_bytes(t.dst_dtype) == 0, DMN_ERR_INVALID,
                    "dmn_clip_grads: tensor %d has no address, or one that is not aligned to its type", i);
        total += t.numel;
        bytes += t.numel * dt_bytes(t.src_dtype);
        writes += t.dst != nullptr;
        separate |= t.dst && (t.dst != t.src || t.dst_dtype != t.src_dtype);
    }
    int used = 0;
    for (int i = 0; i < n_tensors; ++i) used += tensors[i].numel > 0;
    DMN_REQUIRE(total < ((int64_t)1 << 43), DMN_ERR_LIMIT, "dmn_clip_grads: more than 2^43 elements");   // pieces count in 31 bits
    DMN_REQUIRE(writes == 0 || writes == used, DMN_ERR_INVALID, "dmn_clip_grads: either every tensor has a destination or none");
    if (writes) {
        const int bad = ranges_overlap(tensors, n_tensors);
        DMN_REQUIRE(bad != 2, DMN_ERR_LIMIT, "dmn_clip_grads: out of host memory");
        DMN_REQUIRE(bad == 0, DMN_ERR_INVALID, "dmn_clip_grads: a tensor that is written overlaps another one (or is listed twice)");
    }
    hipStream_t s = (hipStream_t)stream;
    double* part = (double*)workspace;
    ClipScale c{};
    c.part = part;
    c.inf_norm = inf_norm;
    c.max_norm = max_norm;
    c.grad_scale = grad_scale;
    c.norm = norm;
    // What the caches cannot hold until the second pass is read past them, all but the end, where that pass begins. Norm and
    // scaling of 403 M bfloat16 elements (0.8 GB) into float32, us: 125 + 499 with nothing kept, 130 + 490 with 80 MB, 156 +
    // 477 with 160 MB, 176 + 480 with everything through the caches.
    int64_t before = 0;
    int next = 0;   // tensor behind the launches so far
    int rc = for_tables<false>(tensors, n_tensors, [&](const ClipTable<false>& t, int blocks, int last) -> int {
        int stream = 0;
        for (int k = 0; next <= last; ++next) {
            if (tensors[next].numel == 0) continue;
            const int size = dt_bytes(tensors[next].src_dtype);
            if (before < bytes - kKeep) {
                before += tensors[next].numel * size;
                stream = t.first[k + 1];
                if (before > bytes - kKeep) stream -= (int)((before - (bytes - kKeep)) / size / kPiece);
            }
            ++k;
        }
        if (inf_norm) grad_norm_kernel<true><<<blocks, kThreads, 0, s>>>(t, part, stream);
        else grad_norm_kernel<false><<<blocks, kThreads, 0, s>>>(t, part, stream);
        c.parts = t.part_base + blocks;
        DMN_BLOCK_LAUNCH_CHECK();
        return DMN_OK;
    });
    if (rc) return rc;
    if (!writes) {
        grad_norm_only_kernel<<<1, kThreads, 0, s>>>(c);
        DMN_BLOCK_LAUNCH_CHECK();
        return DMN_OK;
    }
    c.write_norm = 1;
    auto scale = [&](const auto& t, int blocks, int) -> int {
        grad_scale_kernel<<<blocks, kThreads, 0, s>>>(t, c);
        c.write_norm = 0;
        DMN_BLOCK_LAUNCH_CHECK();
        return DMN_OK;
    };
    return separate ? for_tables<true>(tensors, n_tensors, scale) : for_tables<false>(tensors, n_tensors, scale);
}
