// The score head and the grounding loss with their gradients.
//
//   pooled[t] = mean_j h[t, j]                      z[t] = pooled[t] . w + b                              (vitg_pool_score, keeping pooled)
//   loss = mean_t [ pw y softplus(-z) + (1 - y) softplus(z) ],  pw = min(5, sqrt(neg / max(1, pos)))      (vitg_bce_loss)
//   dz[t] = scale / n * [ (1 - y) sigmoid(z) - pw y sigmoid(-z) ]
//   dh[t, j] = dz[t] / tokens * w       dw (+)= sum_t dz[t] pooled[t]       db (+)= sum_t dz[t]
//
// The backward of the mean needs no second look at h: the forward keeps the frame means (frames x D fp32, 1 / tokens of h), so a step reads h once and
// writes dh once - HBM-bound on both sides.
//
// Measured at D = 3584: 512 frames x 25 tokens, fp32 (184 MB): means and scores 32 us = 5.7 TB/s, gradients 29 us = 6.3 TB/s; 61 frames x 256 tokens, bf16
// (112 MB): means 18 us = 6.3 TB/s + scores 3 us, gradients 19 us = 5.9 TB/s; the loss 3 - 4 us, a launch.
#include "train_common.h"

namespace vitg {

// rows j0 .. j1-1 of one frame, V columns, summed
template <typename T, int V, bool AROUND>
__device__ __forceinline__ void sum_rows(const T* __restrict__ p, long ldh, int j0, int j1, float (&s)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] = 0.f;
#pragma unroll 5
    for (int j = j0; j < j1; ++j) {
        float v[V];
        load_stream<T, V, AROUND>(p + j * ldh, v);
#pragma unroll
        for (int e = 0; e < V; ++e) s[e] += v[e];
    }
}

// one block per frame: enough frames to fill the chip
template <typename T, int V, bool AROUND>
__global__ __launch_bounds__(1024) void pool_score_save_kernel(const T* __restrict__ h, long ldh, int tokens, int cv, const float* __restrict__ w,
                                                               const float* __restrict__ b, float* __restrict__ logits, float* __restrict__ pooled, long ldp) {
    __shared__ float part[16];
    const long t = blockIdx.x;
    const float inv = 1.0f / (float)tokens;
    float dot = 0.f;
    for (int c = threadIdx.x; c < cv; c += blockDim.x) {
        float s[V], ww[V];
        sum_rows<T, V, AROUND>(h + t * tokens * ldh + (long)c * V, ldh, 0, tokens, s);
        load_vec<float, V>(w + c * V, ww);
#pragma unroll
        for (int e = 0; e < V; ++e) { s[e] *= inv; dot += s[e] * ww[e]; }
        store_vec<float, V>(pooled + t * ldp + (long)c * V, s);
    }
    dot = wave_sum(dot);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = dot;
    __syncthreads();
    if (threadIdx.x == 0) {
        float sum = 0.f;
        for (int i = 0; i < (int)(blockDim.x >> 6); ++i) sum += part[i];
        logits[t] = sum + b[0];
    }
}

// few, long frames: a block takes 64 column groups of one frame, its four waves a quarter of the rows each (joined in order); pool_dot_kernel takes the
// scores from the means
template <typename T, int V, bool AROUND>
__global__ __launch_bounds__(256) void pool_mean_kernel(const T* __restrict__ h, long ldh, int tokens, int cv, float* __restrict__ pooled, long ldp) {
    __shared__ float part[3][64][V];
    const long t = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = blockIdx.y * 64 + lane;
    float s[V];
    if (c < cv) {
        sum_rows<T, V, AROUND>(h + t * tokens * ldh + (long)c * V, ldh, (int)((long)tokens * wave / 4), (int)((long)tokens * (wave + 1) / 4), s);
        if (wave) store_vec<float, V>(part[wave - 1][lane], s);
    }
    __syncthreads();
    if (wave || c >= cv) return;
    const float inv = 1.0f / (float)tokens;
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] = (((s[e] + part[0][lane][e]) + part[1][lane][e]) + part[2][lane][e]) * inv;
    store_vec<float, V>(pooled + t * ldp + (long)c * V, s);
}

__global__ __launch_bounds__(256) void pool_dot_kernel(const float* __restrict__ pooled, long ldp, int D, const float* __restrict__ w, const float* __restrict__ b,
                                                       float* __restrict__ logits) {
    __shared__ float part[4];
    const float* const p = pooled + (long)blockIdx.x * ldp;
    float dot = 0.f;
    for (int c = threadIdx.x * 4; c < D; c += 1024) {
        float v[4], ww[4];
        load_vec<float, 4>(p + c, v);
        load_vec<float, 4>(w + c, ww);
#pragma unroll
        for (int e = 0; e < 4; ++e) dot += v[e] * ww[e];
    }
    dot = wave_sum(dot);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = dot;
    __syncthreads();
    if (threadIdx.x == 0) logits[blockIdx.x] = part[0] + part[1] + part[2] + part[3] + b[0];
}

__device__ __forceinline__ double block_sum_1024(double v, double* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int i = 0; i < 16; ++i) v += red[i];
    __syncthreads();
    return v;
}

// one block: n is the number of frames of a batch (hundreds), the call is launch latency.  (long indices here and below: the last step past n must not wrap)
__global__ __launch_bounds__(1024) void bce_loss_backward_kernel(const float* __restrict__ z, const float* __restrict__ y, int n, float scale,
                                                                 float* __restrict__ out2, float* __restrict__ dz) {
    __shared__ double red[16];
    double pos = 0.0;
    for (long i = threadIdx.x; i < n; i += 1024) pos += y[i];
    pos = block_sum_1024(pos, red);
    const float fpos = (float)pos;
    const float pw = fminf(5.0f, sqrtf(((float)n - fpos) / fmaxf(1.0f, fpos)));
    const float g = scale / (float)n;
    double loss = 0.0;
    for (long i = threadIdx.x; i < n; i += 1024) {
        const float zi = z[i], yi = y[i];
        const float e = expf(-fabsf(zi)), r = 1.0f / (1.0f + e);
        const float p = zi >= 0.f ? r : e * r, q = zi >= 0.f ? e * r : r;        // sigmoid(z), sigmoid(-z): no cancellation on either side
        const float t = log1pf(e);                       // softplus(z) = t + max(z, 0), softplus(-z) = t + max(-z, 0): a sum of terms of one sign -
        loss += (1.0f - yi) * (t + fmaxf(zi, 0.0f)) + pw * yi * (t + fmaxf(-zi, 0.0f));      // (1 - y) z + softplus(-z) cancels where the scores are right
        dz[i] = g * ((1.0f - yi) * p - pw * yi * q);
    }
    loss = block_sum_1024(loss, red);
    if (threadIdx.x == 0) {
        out2[0] = (float)(loss / (double)n);
        out2[1] = pw;
    }
}

// blocks [0, wblocks): 64 columns of dw each (16 column quads x 16 frame groups) and, in block 0, db; the others: up to DH_ROWS rows of one frame of dh each
constexpr int DH_ROWS = 32;
template <typename T, int V>
__global__ __launch_bounds__(256) void pool_score_backward_kernel(const float* __restrict__ pooled, long ldp, int frames, int tokens, int D,
                                                                  const float* __restrict__ w, const float* __restrict__ dz, T* __restrict__ dh, long lddh,
                                                                  float* __restrict__ dw, float* __restrict__ db, int accumulate, int wblocks) {
    if ((int)blockIdx.x < wblocks) {
        __shared__ float part[16][64];
        __shared__ double red[4];
        const int q = threadIdx.x & 15, grp = threadIdx.x >> 4, c = blockIdx.x * 64 + q * 4;
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        if (c < D && dw) {
#pragma unroll 4
            for (long t = grp; t < frames; t += 16) {
                float v[4];
                load_vec<float, 4>(pooled + t * ldp + c, v);
                const float d = dz[t];
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[e] += d * v[e];
            }
        }
        store_vec<float, 4>(&part[grp][q * 4], acc);
        double sum = 0.0;
        if (db && blockIdx.x == 0)
            for (long t = threadIdx.x; t < frames; t += 256) sum += dz[t];
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
        __syncthreads();
        const int col = blockIdx.x * 64 + threadIdx.x;
        if (dw && threadIdx.x < 64 && col < D) {
            float s = 0.f;
            for (int i = 0; i < 16; ++i) s += part[i][threadIdx.x];
            dw[col] = accumulate ? dw[col] + s : s;
        }
        if (db && blockIdx.x == 0 && threadIdx.x == 0) {
            const float s = (float)(red[0] + red[1] + red[2] + red[3]);
            db[0] = accumulate ? db[0] + s : s;
        }
        return;
    }
    const int slices = (tokens + DH_ROWS - 1) / DH_ROWS, id = (int)blockIdx.x - wblocks;
    const long t = id / slices;
    const int j0 = id % slices * DH_ROWS, j1 = min(j0 + DH_ROWS, tokens);
    const float d = dz[t] / (float)tokens;
    for (long c = threadIdx.x * V; c < D; c += 256 * V) {
        float v[V];
        load_vec<float, V>(w + c, v);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] *= d;
        for (int j = j0; j < j1; ++j) store_vec<T, V>(dh + (t * tokens + j) * lddh + c, v);
    }
}

}  // namespace vitg

using namespace vitg;

extern "C" int vitg_pool_score_save(const void* h, int h_dtype, long ldh, int frames, int tokens_per_frame, int D, const float* w, const float* b,
                                    float* logits, float* pooled, long ldp, void* stream) {
    if (frames <= 0) return 0;
    if (!h || !w || !b || !logits || !pooled) return VITG_ERR_ARG;
    if (!dtype_ok(h_dtype)) return VITG_ERR_DTYPE;
    if (tokens_per_frame <= 0 || D <= 0 || ldh < D || ldp < D || frames >= (1 << 22)) return VITG_ERR_SHAPE;      // (a launch has fewer than 2^32 threads)
    if (D % 4 || ldh % 4 || ldp % 4 || !aligned_to(h, 4 * dtype_size(h_dtype)) || !aligned_to(w, 16) || !aligned_to(pooled, 16)) return VITG_ERR_ALIGN;
    const bool wide = h_dtype != DT_F32 && D % 8 == 0 && ldh % 8 == 0 && aligned_to(h, 16);
    const int cv = D / (wide ? 8 : 4);
    // One block per frame, or the rows of a frame over several blocks and a second launch for the scores: the second form where a frame is long and the frames'
    // waves (64 column groups each) are fewer than five a CU.  bf16, D = 3584, us: 8 x 196 14.6 against 11.0, 61 x 256 28.5 against 20.7, 128 x 196 34.6 against
    // 31.4; but 61 x 64 7.8 against 10.6 (the launch), 200 x 256 55 against 59, 512 x 256 143 against 152.  D = 1024: 160 x 196 20.9 against 13.8
    const bool few = (long)frames * cv < device_cu_count(current_device()) * 5l * 64 && tokens_per_frame >= 128 && cv > 64;
    const int threads = cv >= 1024 ? 1024 : (cv + 63) / 64 * 64;
    hipStream_t s = (hipStream_t)stream;
    with_dtype(h_dtype, [&](auto ti) {
        typedef decltype(ti) T;
        with_flag((long)frames * tokens_per_frame * D * (long)sizeof(T) > STREAM_BYTES, [&](auto around) {
            constexpr bool AROUND = decltype(around)::value;
            auto mean = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(frames, ceil_div(cv, 64)), dim3(256), 0, s, (const T*)h, ldh, tokens_per_frame, cv, pooled, ldp); };
            auto all = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(frames), dim3(threads), 0, s, (const T*)h, ldh, tokens_per_frame, cv, w, b, logits, pooled, ldp); };
            if (few) { if (wide) mean(pool_mean_kernel<T, 8, AROUND>); else mean(pool_mean_kernel<T, 4, AROUND>); }
            else if (wide) all(pool_score_save_kernel<T, 8, AROUND>);
            else all(pool_score_save_kernel<T, 4, AROUND>);
        });
    });
    if (few) hipLaunchKernelGGL(pool_dot_kernel, dim3(frames), dim3(256), 0, s, pooled, ldp, D, w, b, logits);
    return launched();
}

extern "C" int vitg_bce_loss_backward(const float* logits, const float* labels, int n, float scale, float* out2, float* dlogits, void* stream) {
    if (n <= 0 || !logits || !labels || !out2 || !dlogits) return VITG_ERR_ARG;
    hipLaunchKernelGGL(bce_loss_backward_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, logits, labels, n, scale, out2, dlogits);
    return launched();
}

extern "C" int vitg_pool_score_backward(const float* pooled, long ldp, int frames, int tokens_per_frame, int D, const float* w, const float* dlogits,
                                        void* dh, int dh_dtype, long lddh, float* dw, float* db, int accumulate, void* stream) {
    if (frames < 0 || tokens_per_frame <= 0 || D <= 0) return VITG_ERR_SHAPE;
    if (!w || (frames && !dlogits) || (dw && frames && !pooled)) return VITG_ERR_ARG;
    if (dh && !dtype_ok(dh_dtype)) return VITG_ERR_DTYPE;
    if ((dh && lddh < D) || (dw && frames && ldp < D)) return VITG_ERR_SHAPE;
    if (D % 4 || !aligned_to(w, 16) || (dw && (ldp % 4 || !aligned_to(pooled, 16))) || (dh && (lddh % 4 || !aligned_to(dh, 4 * dtype_size(dh_dtype))))) return VITG_ERR_ALIGN;
    const int wblocks = dw ? ceil_div(D, 64) : db ? 1 : 0;
    const long blocks = wblocks + (dh ? (long)frames * (((long)tokens_per_frame + DH_ROWS - 1) / DH_ROWS) : 0);
    if (!blocks) return 0;
    if (blocks >= (1l << 24)) return VITG_ERR_SHAPE;     // (a launch has fewer than 2^32 threads)
    const unsigned grid = (unsigned)blocks;
    const bool wide = dh && dh_dtype != DT_F32 && D % 8 == 0 && lddh % 8 == 0 && aligned_to(dh, 16);
    with_dtype(dh ? dh_dtype : (int)DT_F32, [&](auto ti) {
        typedef decltype(ti) T;
        auto run = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), 0, (hipStream_t)stream, pooled, ldp, frames, tokens_per_frame, D, w, dlogits, (T*)dh, lddh, dw, db, accumulate, wblocks);
        };
        if (wide) run(pool_score_backward_kernel<T, 8>); else run(pool_score_backward_kernel<T, 4>);
    });
    return launched();
}
