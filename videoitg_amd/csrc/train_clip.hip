// Global gradient norm over a list of tensors, and clipping.
//
//   norm  = |scale| * sqrt(sum over all tensors of g^2)
//   out_i = g_i * scale * min(1, max_norm / (norm + 1e-6))         (out_i may be g_i)
//
// Two passes over the data, each bound by HBM.  Pass 1: a fixed grid walks the 64 KiB pieces of up to 96 tensors (their addresses ride in the kernel
// arguments: nothing is uploaded, so a call can be captured into a graph) and leaves one sum per block; pass 2: every block adds the sums in the same
// order, so all blocks hold the same factor, and scales its pieces.  Squares are summed in fp64: the square of any fp32 / bf16 value is representable
// there, so neither large nor tiny gradients change the norm, and the fixed order gives the same bits on every call.  Pass 2 walks the pieces from the end: it
// begins with what pass 1 has left in the last-level cache.
//
// Measured: four decoder layers (1.86 GB, bf16 matrices and fp32 vectors): sums 299 us = 6.2 TB/s, scaling 716 us = 5.2 TB/s (a copy: 5.1);
// six tensors of a projector and a head (fp32, 68 MB): 14 + 24 us, mostly launch and the walk's tail.
#include "train_common.h"
#include <math.h>
#include <stdlib.h>

namespace vitg {

constexpr int CLIP_TENSORS = 96, CLIP_THREADS = 256, CLIP_PIECE = 65536;
struct ClipArgs {
    const void* in[CLIP_TENSORS];
    void* out[CLIP_TENSORS];
    long numel[CLIP_TENSORS];
    int piece0[CLIP_TENSORS + 1];             // first piece of each tensor
    unsigned char dtype[CLIP_TENSORS];
    int count;
};

// the tensor that holds piece p
__device__ __forceinline__ int clip_find(const ClipArgs& a, int p) {
    int lo = 0, hi = a.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.piece0[mid] <= p) lo = mid; else hi = mid - 1;
    }
    return lo;
}

template <typename T>
__device__ __forceinline__ double clip_sum_piece(const T* __restrict__ p, long count, int tid) {
    constexpr int V = 16 / sizeof(T);
    double s = 0.0;
    long done = 0;
    if (((uintptr_t)p & 15) == 0) {
        done = count / V * V;
        long i = (long)tid * V;
        double q[4] = {0.0, 0.0, 0.0, 0.0};
        for (; i + 3 * CLIP_THREADS * V < done; i += 4 * CLIP_THREADS * V) {       // four loads in flight, four chains of sums
            float v[4][V];
#pragma unroll
            for (int u = 0; u < 4; ++u) load_vec<T, V>(p + i + u * CLIP_THREADS * V, v[u]);
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int e = 0; e < V; ++e) q[u] += (double)v[u][e] * (double)v[u][e];
        }
        for (; i < done; i += CLIP_THREADS * V) {
            float v[V];
            load_vec<T, V>(p + i, v);
#pragma unroll
            for (int e = 0; e < V; ++e) q[0] += (double)v[e] * (double)v[e];
        }
        s = (q[0] + q[1]) + (q[2] + q[3]);
    }
    for (long i = done + tid; i < count; i += CLIP_THREADS) { const double v = (double)(float)p[i]; s += v * v; }
    return s;
}

__device__ __forceinline__ double block_sum_f64(double v, double* red) {      // every thread gets the sum; fixed order
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0] + red[1] + red[2] + red[3];
    __syncthreads();
    return v;
}

__global__ __launch_bounds__(CLIP_THREADS) void grad_sumsq_kernel(const ClipArgs a, double* __restrict__ sums) {
    __shared__ double red[4];
    const int pieces = a.piece0[a.count];
    double s = 0.0;
    for (int p = blockIdx.x; p < pieces; p += gridDim.x) {
        const int t = clip_find(a, p);
        const int esize = a.dtype[t] == DT_F32 ? 4 : 2;
        const long per = CLIP_PIECE / esize, at = (long)(p - a.piece0[t]) * per, count = min(per, a.numel[t] - at);
        if (a.dtype[t] == DT_BF16) s += clip_sum_piece((const bf16_t*)a.in[t] + at, count, threadIdx.x);
        else if (a.dtype[t] == DT_F16) s += clip_sum_piece((const f16_t*)a.in[t] + at, count, threadIdx.x);
        else s += clip_sum_piece((const float*)a.in[t] + at, count, threadIdx.x);
    }
    s = block_sum_f64(s, red);
    if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

// a factor below fp32's normal numbers (norms beyond 1e38, tiny limits) keeps its 24 bits as factor = first * second with a power of two for second: first * v does
// not overflow, and where it is subnormal the result is zero.  Ordinary factors have second = 1
struct ClipFactor { float first, second; };
__device__ __forceinline__ ClipFactor clip_factor(double f) {
    const double a = fabs(f);
    if (a < 0x1p-186) return {(float)(f * 0x1p126), 0x1p-126f};
    if (a < 0x1p-100) return {(float)(f * 0x1p64), 0x1p-64f};
    return {(float)f, 1.0f};
}

template <bool AROUND, typename T>
__device__ __forceinline__ void clip_scale_piece(const T* p, T* q, long count, const ClipFactor f, int tid) {
    constexpr int V = 16 / sizeof(T);
    long done = 0;
    if ((((uintptr_t)p | (uintptr_t)q) & 15) == 0) {
        done = count / V * V;
        long i = (long)tid * V;
        for (; i + 3 * CLIP_THREADS * V < done; i += 4 * CLIP_THREADS * V) {
            float v[4][V];
#pragma unroll
            for (int u = 0; u < 4; ++u) load_vec<T, V>(p + i + u * CLIP_THREADS * V, v[u]);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
#pragma unroll
                for (int e = 0; e < V; ++e) v[u][e] = v[u][e] * f.first * f.second;
                store_stream<T, V, AROUND>(q + i + u * CLIP_THREADS * V, v[u]);
            }
        }
        for (; i < done; i += CLIP_THREADS * V) {
            float v[V];
            load_vec<T, V>(p + i, v);
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = v[e] * f.first * f.second;
            store_vec<T, V>(q + i, v);
        }
    }
    for (long i = done + tid; i < count; i += CLIP_THREADS) q[i] = (T)((float)p[i] * f.first * f.second);
}

// the norm of all tensors from the sums of pass 1 (every block adds them in the same order)
__device__ __forceinline__ double clip_norm(const double* __restrict__ sums, int count, float scale, double* red) {
    double s = 0.0;
    for (int i = threadIdx.x; i < count; i += CLIP_THREADS) s += sums[i];
    return sqrt(block_sum_f64(s, red)) * fabs((double)scale);
}

template <bool AROUND>
__global__ __launch_bounds__(CLIP_THREADS) void grad_scale_kernel(const ClipArgs a, const double* __restrict__ sums, int nsums, float scale, float max_norm,
                                                                  float* __restrict__ norm_out) {
    __shared__ double red[4];
    const double norm = clip_norm(sums, nsums, scale, red);
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    // max_norm / inf = 0 and NaN stays NaN, as dividing by the norm says: an overflowed step shows in the norm AND in the gradients.  max_norm = inf: no limit
    const double clip = max_norm == INFINITY ? 1.0 : (double)max_norm / (norm + 1e-6);
    const ClipFactor factor = clip_factor((double)scale * (clip < 1.0 ? clip : clip != clip ? clip : 1.0));
    const int pieces = a.count ? a.piece0[a.count] : 0;
    // from the end: what pass 1 read last is still in the last-level cache
    for (int p = pieces - 1 - (int)blockIdx.x; p >= 0; p -= gridDim.x) {
        const int t = clip_find(a, p);
        if (factor.first == 1.0f && a.in[t] == a.out[t]) continue;              // in place and nothing to scale (second is 1 then)
        const int esize = a.dtype[t] == DT_F32 ? 4 : 2;
        const long per = CLIP_PIECE / esize, at = (long)(p - a.piece0[t]) * per, count = min(per, a.numel[t] - at);
        if (a.dtype[t] == DT_BF16) clip_scale_piece<AROUND>((const bf16_t*)a.in[t] + at, (bf16_t*)a.out[t] + at, count, factor, threadIdx.x);
        else if (a.dtype[t] == DT_F16) clip_scale_piece<AROUND>((const f16_t*)a.in[t] + at, (f16_t*)a.out[t] + at, count, factor, threadIdx.x);
        else clip_scale_piece<AROUND>((const float*)a.in[t] + at, (float*)a.out[t] + at, count, factor, threadIdx.x);
    }
}

__global__ __launch_bounds__(CLIP_THREADS) void grad_norm_kernel(const double* __restrict__ sums, int nsums, float scale, float* __restrict__ norm_out) {
    __shared__ double red[4];
    const double norm = clip_norm(sums, nsums, scale, red);
    if (threadIdx.x == 0) *norm_out = (float)norm;
}

// blocks per launch: at most 1 024 (four per CU), at most the pieces there are
static int clip_blocks(int pieces) { return pieces < 1024 ? pieces : 1024; }

// one launch takes the tensors [first, returned index): at most CLIP_TENSORS with elements (those without are passed over), fewer than 2^31 pieces
static int clip_span(int first, int count, const long* numel, const int* dtype, int* pieces) {
    long p = 0;
    int live = 0, i = first;
    for (; i < count; ++i) {
        if (numel[i] == 0) continue;
        const long per = CLIP_PIECE / dtype_size(dtype[i]), n = (numel[i] + per - 1) / per;
        if (live == CLIP_TENSORS || (live && p + n >= (1l << 31))) break;
        p += n;
        ++live;
    }
    *pieces = (int)p;
    return i;
}

static int clip_fill(ClipArgs& a, int first, int count, const void* const* in, void* const* out, const long* numel, const int* dtype) {
    int pieces = 0;
    const int end = clip_span(first, count, numel, dtype, &pieces);
    a.count = 0;
    pieces = 0;
    for (int i = first; i < end; ++i) {
        if (numel[i] == 0) continue;
        const long per = CLIP_PIECE / dtype_size(dtype[i]);
        a.in[a.count] = in[i]; a.out[a.count] = out ? out[i] : nullptr; a.numel[a.count] = numel[i]; a.dtype[a.count] = (unsigned char)dtype[i];
        a.piece0[a.count] = pieces;
        pieces += (int)((numel[i] + per - 1) / per);
        ++a.count;
    }
    a.piece0[a.count] = pieces;
    return end;
}

struct ClipSpan { uintptr_t begin, end; bool written; };
static int clip_span_order(const void* a, const void* b) {
    const uintptr_t x = ((const ClipSpan*)a)->begin, y = ((const ClipSpan*)b)->begin;
    return x < y ? -1 : x > y ? 1 : 0;
}
// whether memory that the call writes - outputs, norm, workspace - is also another tensor's (a shared byte would be scaled twice, or before another block has
// read it).  In order of their begins, a span that meets any earlier one meets the one that reaches furthest; if the pair in question is another one, that
// one and its partner have met before.
static bool clip_overlaps(int count, const void* const* in, void* const* out, const long* numel, const int* dtype, const void* norm, const void* ws, long ws_bytes,
                          bool* failed) {
    ClipSpan* const sp = (ClipSpan*)malloc(sizeof(ClipSpan) * (2 * (size_t)count + 2));
    *failed = sp == nullptr;
    if (!sp) return false;
    int n = 0;
    for (int i = 0; i < count; ++i) {
        const size_t bytes = (size_t)numel[i] * dtype_size(dtype[i]);
        if (!bytes) continue;
        sp[n++] = {(uintptr_t)in[i], (uintptr_t)in[i] + bytes, out && out[i] == in[i]};
        if (out && out[i] != in[i]) sp[n++] = {(uintptr_t)out[i], (uintptr_t)out[i] + bytes, true};
    }
    sp[n++] = {(uintptr_t)norm, (uintptr_t)norm + 4, true};
    sp[n++] = {(uintptr_t)ws, (uintptr_t)ws + (size_t)ws_bytes, true};
    qsort(sp, n, sizeof(ClipSpan), clip_span_order);
    bool meet = false;
    int far = 0;
    for (int i = 1; i < n && !meet; ++i) {
        meet = sp[i].begin < sp[far].end && (sp[i].written || sp[far].written);
        if (sp[i].end > sp[far].end) far = i;
    }
    free(sp);
    return meet;
}

static int clip_check(int count, const void* const* in, void* const* out, const long* numel, const int* dtype) {
    if (count < 0) return VITG_ERR_SHAPE;
    if (count && (!in || !numel || !dtype)) return VITG_ERR_ARG;
    for (int i = 0; i < count; ++i) {
        if (numel[i] < 0 || numel[i] >= (1l << 44)) return VITG_ERR_SHAPE;
        if (!dtype_ok(dtype[i])) return VITG_ERR_DTYPE;
        if (numel[i] && (!in[i] || (out && !out[i]))) return VITG_ERR_ARG;
        if (!aligned_to(in[i], dtype_size(dtype[i])) || (out && !aligned_to(out[i], dtype_size(dtype[i])))) return VITG_ERR_ALIGN;
    }
    return 0;
}

}  // namespace vitg

using namespace vitg;

extern "C" int vitg_clip_grad_plan(int count, const long* numel, const int* dtype, long* workspace_bytes) {
    if (!workspace_bytes || (count > 0 && (!numel || !dtype))) return VITG_ERR_ARG;
    if (count < 0) return VITG_ERR_SHAPE;
    for (int i = 0; i < count; ++i)
        if (numel[i] < 0 || numel[i] >= (1l << 44)) return VITG_ERR_SHAPE;
        else if (!dtype_ok(dtype[i])) return VITG_ERR_DTYPE;
    long blocks = 0;
    for (int at = 0; at < count;) {
        int pieces = 0;
        at = clip_span(at, count, numel, dtype, &pieces);
        blocks += clip_blocks(pieces);
    }
    *workspace_bytes = (blocks ? blocks : 1) * 8;
    return 0;
}

extern "C" int vitg_clip_grad(int count, const void* const* grads, void* const* outs, const long* numel, const int* dtype, float scale, float max_norm,
                              float* norm, void* workspace, long workspace_bytes, void* stream) {
    const int bad = clip_check(count, grads, outs, numel, dtype);
    if (bad) return bad;
    if (!norm || !workspace || !aligned_to(workspace, 8)) return VITG_ERR_ARG;
    if (outs && !(max_norm >= 0.f)) return VITG_ERR_ARG;
    long need = 0;
    (void)vitg_clip_grad_plan(count, numel, dtype, &need);
    if (workspace_bytes < need) return VITG_ERR_ARG;
    bool failed = false;
    if (clip_overlaps(count, grads, outs, numel, dtype, norm, workspace, need, &failed) || failed) return VITG_ERR_ARG;
    hipStream_t s = (hipStream_t)stream;
    double* const sums = (double*)workspace;
    ClipArgs a;
    int nsums = 0;
    for (int at = 0; at < count;) {
        at = clip_fill(a, at, count, grads, outs, numel, dtype);
        if (!a.count) break;
        const int blocks = clip_blocks(a.piece0[a.count]);
        hipLaunchKernelGGL(grad_sumsq_kernel, dim3(blocks), dim3(CLIP_THREADS), 0, s, a, sums + nsums);
        nsums += blocks;
    }
    if (!outs || nsums == 0) {
        hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(CLIP_THREADS), 0, s, sums, nsums, scale, norm);
        return launched();
    }
    long bytes = 0;
    for (int i = 0; i < count; ++i) bytes += numel[i] * dtype_size(dtype[i]);
    bool first = true;
    for (int at = 0; at < count; first = false) {
        at = clip_fill(a, at, count, grads, outs, numel, dtype);
        if (!a.count) break;
        with_flag(bytes > STREAM_BYTES, [&](auto around) {
            hipLaunchKernelGGL(grad_scale_kernel<decltype(around)::value>, dim3(clip_blocks(a.piece0[a.count])), dim3(CLIP_THREADS), 0, s, a, sums, nsums, scale, max_norm, first ? norm : (float*)nullptr);
        });
    }
    return launched();
}
