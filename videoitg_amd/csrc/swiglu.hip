// The gated feed-forward's first half for training:  [G | U] = X W^T (weight rows interleaved [32 gate | 32 up]),  H = silu(G) * U,  and its backward.
//
//   sig = 1 / (1 + e^-G)      dG = dH U sig (1 + G (1 - sig))      dU = dH G sig
//   dX = dGU W      dW (+)= dGU^T X
//
// Forward: one GEMM with the activation and the product in its epilogue; for training the epilogue also stores the 16-bit pre-activations (M x 2F), which
// costs their write instead of a second GEMM in the backward pass.
// Backward: dX runs on the GEMM form that takes W as it lies (contraction along W's rows); dW's contraction runs along the rows of both operands, so dGU comes
// out of its elementwise kernel in both orders and X passes through a tile transpose in front of the ordinary NT GEMM.  dGU is rounded to the 16-bit type once -
// the matrix pipe's operand type - and every sum over it is fp32.
//
// Measured at 3584 x 37888 (bf16; large library products of these shapes run at 1 307 - 1 436 TFLOP/s): one row 49 us = 5.6 TB/s of W (the kernel; 59 the call, back to back); 12 860 rows with
// pre-activations 2.67 ms = 1 309 TFLOP/s; their backward 5.73 ms: 0.80 in front (4.1 GB, 5.2 TB/s), dX and dW 2.46 each = 1 420 TFLOP/s; 1 607 rows (fp16)
// 0.88 ms: 0.08 + dX 0.43 (320-row tiles, K-major, three shares: 1 920 rows are multiplied) + dW 0.38 + the join 0.01.
#include "train_common.h"
#include "gemm_common.h"

namespace vitg {

// out[c, r] = in[r, c] for r < R, c < C; columns R .. Rp-1 of out are zero (K padding of the GEMM that reads it).  64 x 64 tiles through LDS.
constexpr int TR_LD = 72;                                // halfs per LDS row: 16-B aligned
template <typename T>
__device__ __forceinline__ void transpose_tile(T* tile, long r0, int c0, const T* __restrict__ in, long ldi, long R, int C, T* __restrict__ out, long ldo, long Rp) {
    typedef typename T16<T>::vec8 vec8;                  // tile: [c][r]
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int idx = i * 256 + threadIdx.x, r = idx >> 3, cq = (idx & 7) * 8;
        vec8 v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (T)0.f;
        if (r0 + r < R && c0 + cq < C) v = *(const vec8*)(in + (r0 + r) * ldi + c0 + cq);
#pragma unroll
        for (int e = 0; e < 8; ++e) tile[(cq + e) * TR_LD + r] = v[e];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int idx = i * 256 + threadIdx.x, c = idx >> 3, rq = (idx & 7) * 8;
        if (c0 + c < C && r0 + rq < Rp) *(vec8*)(out + (long)(c0 + c) * ldo + r0 + rq) = *(const vec8*)(tile + c * TR_LD + rq);
    }
}

// dGU from dH and the saved pre-activations, in both orders: dgu [M, 2F] (unless null) and dgut [2F, Mp] (unless null; columns M .. Mp-1 zero).
// One block: 64 rows x 32 features = 64 columns of gu.
template <typename T>
__device__ __forceinline__ void swiglu_grad_tile(T* tile, long r0, int n0, const T* __restrict__ dh, long lddh, const T* __restrict__ gu, long ldgu, long M, long Mp,
                                                 T* __restrict__ dgu, long lddgu, T* __restrict__ dgut) {
    typedef typename T16<T>::vec8 vec8;                  // tile: [column of gu][row]
    const int f0 = n0 / 2;
    {
        const int r = threadIdx.x >> 2, q = (threadIdx.x & 3) * 8;
        const long m = r0 + r;
        vec8 a, b;
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] = b[e] = (T)0.f;
        if (m < M) {
            const vec8 d = *(const vec8*)(dh + m * lddh + f0 + q), g = *(const vec8*)(gu + m * ldgu + n0 + q), u = *(const vec8*)(gu + m * ldgu + n0 + 32 + q);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float de = (float)d[e], ge = (float)g[e], ue = (float)u[e];
                const float sig = 1.0f / (1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * ge));
                a[e] = (T)(de * ue * sig * (1.0f + ge * (1.0f - sig)));
                b[e] = (T)(de * ge * sig);
            }
            if (dgu) {
                *(vec8*)(dgu + m * lddgu + n0 + q) = a;
                *(vec8*)(dgu + m * lddgu + n0 + 32 + q) = b;
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            tile[(q + e) * TR_LD + r] = a[e];
            tile[(32 + q + e) * TR_LD + r] = b[e];
        }
    }
    if (!dgut) return;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int idx = i * 256 + threadIdx.x, c = idx >> 3, rq = (idx & 7) * 8;
        *(vec8*)(dgut + (long)(n0 + c) * Mp + r0 + rq) = *(const vec8*)(tile + c * TR_LD + rq);
    }
}

// everything in front of the products in one launch: blocks [0, grad) dGU, then the tiles of X^T [K, Mp], then those of W^T [K, N] (64 x 64 each)
template <typename T>
struct SwigluPrep {
    const T* dh; long lddh; const T* gu; long ldgu; long M, Mp; T* dgu; long lddgu; T* dgut;
    const T* x; long ldx; T* xt; const T* w; long ldw; T* wt;
    int N, K; long grad, x_end;
};
template <typename T>
__global__ __launch_bounds__(256) void swiglu_prep_kernel(const SwigluPrep<T> a) {
    __shared__ __attribute__((aligned(16))) T tile[64 * TR_LD];
    const long mt = a.Mp / 64, id = blockIdx.x;
    if (id < a.grad) swiglu_grad_tile<T>(tile, id % mt * 64, (int)(id / mt) * 64, a.dh, a.lddh, a.gu, a.ldgu, a.M, a.Mp, a.dgu, a.lddgu, a.dgut);
    else if (id < a.x_end) transpose_tile<T>(tile, (id - a.grad) % mt * 64, (int)((id - a.grad) / mt) * 64, a.x, a.ldx, a.M, a.K, a.xt, a.Mp, a.Mp);
    else transpose_tile<T>(tile, (id - a.x_end) % (a.N / 64) * 64, (int)((id - a.x_end) / (a.N / 64)) * 64, a.w, a.ldw, a.N, a.K, a.wt, a.N, a.N);
}

// rows of `bytes` (a multiple of 16) set to zero, `pitch` bytes apart
__global__ __launch_bounds__(256) void zero_bytes_kernel(char* __restrict__ p, long pitch, long rows, long bytes) {
    for (long r = blockIdx.x; r < rows; r += gridDim.x)
        for (long c = threadIdx.x * 16l; c < bytes; c += 256 * 16) *(u32x4*)(p + r * pitch + c) = u32x4{0, 0, 0, 0};
}

// ---- few rows: every kernel below is a single pass over W or dW, bound by its bytes -----------------------------------------------------------------
//
// Forward, M <= 16: MFMA operands straight from global memory (nothing is shared between waves): A = 16 weight rows, B = the rows of X.  A block owns 16 gate
// rows and their 16 up rows; its four waves take a quarter of K each and their sums join through LDS as (w0 + w2) + (w1 + w3).
template <typename T>
__global__ __launch_bounds__(256) void swiglu_rows_kernel(const T* __restrict__ X, long ldx, const T* __restrict__ W, long ldw, int M, int K,
                                                          T* __restrict__ out, long ldo, T* __restrict__ gu, long ldgu) {
    typedef typename T16<T>::vec8 vec8;
    typedef typename T16<T>::vec4 vec4;
    constexpr int U = 4;                                 // k-steps of loads in flight
    __shared__ __attribute__((aligned(16))) f32x4 part[2][2][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, q = lane >> 4;
    const long group = blockIdx.x >> 1;                  // one [32 gate | 32 up] group, this block's half of it
    const int half = (blockIdx.x & 1) * 16;
    const T* const wg = W + (group * 64 + half + r16) * ldw + q * 8;
    const T* const wu = wg + 32 * ldw;
    const T* const xp = X + (long)min(r16, M - 1) * ldx + q * 8;
    f32x4 gate = {0.f, 0.f, 0.f, 0.f}, up = {0.f, 0.f, 0.f, 0.f};
    const int steps = K / 32, s0 = steps * wave / 4, s1 = steps * (wave + 1) / 4;
    for (int s = s0; s < s1; s += U) {
        vec8 a[U], b[U], x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long k = min(s + u, s1 - 1) * 32l;
            a[u] = *(const vec8*)(wg + k);
            b[u] = *(const vec8*)(wu + k);
            x[u] = *(const vec8*)(xp + k);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s + u >= s1) break;
            gate = T16<T>::mfma16(a[u], x[u], gate);
            up = T16<T>::mfma16(b[u], x[u], up);
        }
    }
    if (wave >= 2) { part[wave - 2][0][lane] = gate; part[wave - 2][1][lane] = up; }
    __syncthreads();
    if (wave < 2) { gate += part[wave][0][lane]; up += part[wave][1][lane]; }
    if (wave == 1) { part[1][0][lane] = gate; part[1][1][lane] = up; }
    __syncthreads();
    if (wave != 0 || r16 >= M) return;
    gate += part[1][0][lane];
    up += part[1][1][lane];
    const int m = r16, f = half + q * 4;                 // four features of one row per lane
    vec4 o, a, b;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        o[e] = (T)(silu_f(gate[e]) * up[e]);
        a[e] = (T)gate[e];
        b[e] = (T)up[e];
    }
    *(vec4*)(out + m * ldo + group * 32 + f) = o;
    if (gu) {
        *(vec4*)(gu + m * ldgu + group * 64 + f) = a;
        *(vec4*)(gu + m * ldgu + group * 64 + 32 + f) = b;
    }
}

// 8 x 8 block of 16-bit values in a lane's registers, transposed: in[i] = row i (8 columns), out[j] = column j (8 rows).  One v_perm_b32 per dword.
template <typename V8> __device__ __forceinline__ void transpose8(const V8 (&in)[8], V8 (&out)[8]) {
    u32x4 a[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = bitcast<u32x4>(in[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        u32x4 o;
#pragma unroll
        for (int t = 0; t < 4; ++t)
            o[t] = __builtin_amdgcn_perm(a[2 * t + 1][j >> 1], a[2 * t][j >> 1], (j & 1) ? 0x07060302u : 0x05040100u);
        out[j] = bitcast<V8>(o);
    }
}

// dX = dGU W, contraction along the ROWS of W: a lane loads an 8 x 8 block of W (8 rows, 16 B of each: a wave reads 4 x 256 B per instruction) and transposes
// it in registers into 8 MFMA operands - column d0 + 8 (lane & 15) + j of W is row (lane & 15) of operand j, so a lane's 8 accumulators are 32 consecutive
// columns of dX.  A block: 128 columns x one share of the rows, split over four waves, summed as (w0 + w2) + (w1 + w3) into part[share][m][K] (fp32).
template <typename T, int MT>
__device__ __forceinline__ void dx_rows_block(int column, int share, const T* __restrict__ dgu, long lddgu, const T* __restrict__ W, long ldw, int M, int N, int K,
                                              int shares, float* __restrict__ part) {
    typedef typename T16<T>::vec8 vec8;
    __shared__ __attribute__((aligned(16))) f32x4 red[2][8][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, q = lane >> 4;
    const int d0 = column * 128;
    const int col = min(d0 + ((r16 & 3) * 4 + (r16 >> 2)) * 8, K - 8);   // (the last block may hang over: its loads repeat, its stores are left out)
    const long steps = N / 32, ways = (long)shares * 4, way = (long)share * 4 + wave;
    const long s0 = steps * way / ways, s1 = steps * (way + 1) / ways;
    const T* const wp = W + (long)(q * 8) * ldw + col;
    const T* gp[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) gp[i] = dgu + (long)min(i * 16 + r16, M - 1) * lddgu + q * 8;
    f32x4 acc[MT][8];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
    for (long s = s0; s < s1; ++s) {
        vec8 w[8], f[8], g[MT];
        const T* const p = wp + s * 32 * ldw;
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = *(const vec8*)(p + i * ldw);
#pragma unroll
        for (int i = 0; i < MT; ++i) g[i] = *(const vec8*)(gp[i] + s * 32);
        transpose8(w, f);
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[i][j] = T16<T>::mfma16(f[j], g[i], acc[i][j]);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        __syncthreads();
        if (wave >= 2) {
#pragma unroll
            for (int j = 0; j < 8; ++j) red[wave - 2][j][lane] = acc[i][j];
        }
        __syncthreads();
        if (wave < 2) {
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[i][j] += red[wave][j][lane];
        }
        if (wave == 1) {
#pragma unroll
            for (int j = 0; j < 8; ++j) red[1][j][lane] = acc[i][j];
        }
        __syncthreads();
        const int m = i * 16 + r16;
        if (wave != 0 || m >= M) continue;
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[i][j] += red[1][j][lane];
        float* const o = part + ((long)share * M + m) * K;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int d = d0 + (r * 4 + q) * 8;
            if (d >= K) continue;
            *(f32x4*)(o + d) = f32x4{acc[i][0][r], acc[i][1][r], acc[i][2][r], acc[i][3][r]};
            *(f32x4*)(o + d + 4) = f32x4{acc[i][4][r], acc[i][5][r], acc[i][6][r], acc[i][7][r]};
        }
    }
}

// out[m, :] (+)= sum of the shares [share][M][K] in order, for one or two matrices (blocks [0, a_blocks) the first)
struct JoinArgs { const float* part; long M; int K, shares; void* out; long ldo; int accumulate; };
template <typename T>
__device__ __forceinline__ void join_quad(const JoinArgs& a, long i) {
    const long total = a.M * a.K;
    if (i >= total) return;
    f32x4 v = *(const f32x4*)(a.part + i);
#pragma unroll 8
    for (int s = 1; s < a.shares; ++s) v += *(const f32x4*)(a.part + s * total + i);
    T* const o = (T*)a.out + i / a.K * a.ldo + i % a.K;
    float w[4] = {0.f, 0.f, 0.f, 0.f};
    if (a.accumulate) load_vec<T, 4>(o, w);
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = a.accumulate ? w[e] + v[e] : v[e];
    store_vec<T, 4>(o, w);
}
template <typename TA, typename TB>
__global__ __launch_bounds__(256) void join_shares_kernel(const JoinArgs a, int a_blocks, const JoinArgs b) {
    if ((int)blockIdx.x < a_blocks) join_quad<TA>(a, ((long)blockIdx.x * 256 + threadIdx.x) * 4);
    else join_quad<TB>(b, ((long)((int)blockIdx.x - a_blocks) * 256 + threadIdx.x) * 4);
}
template <typename TA, typename TB = TA> static void join_shares(const JoinArgs& a, hipStream_t s, const JoinArgs& b = JoinArgs{}) {
    const int na = (int)((a.M * a.K / 4 + 255) / 256), nb = (int)((b.M * b.K / 4 + 255) / 256);
    hipLaunchKernelGGL((join_shares_kernel<TA, TB>), dim3(na + nb), dim3(256), 0, s, a, na, b);
}

// dW (+)= dGU^T X for M <= 32 rows: a wave owns 32 rows x 128 columns of dW.  A = X transposed in registers (as above), B = dGU^T rows from the transposed copy.
// Bound by the write of dW.
constexpr int DW_WAVE = 32;
template <typename T, typename TW, bool AROUND>
__device__ __forceinline__ void dw_rows_block(int column, int rows, const T* __restrict__ dgut, long Mp, const T* __restrict__ X, long ldx, int M, int N, int K,
                                              TW* __restrict__ dW, long lddw, int accumulate) {
    typedef typename T16<T>::vec8 vec8;
    constexpr int NT = DW_WAVE / 16;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, q = lane >> 4;
    const long n0 = ((long)rows * 4 + wave) * DW_WAVE;
    const int d0 = column * 128, col = min(d0 + ((r16 & 3) * 4 + (r16 >> 2)) * 8, K - 8);
    if (n0 >= N) return;
    f32x4 acc[NT][8];
    vec8 x[8], f[8], g[NT];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int m = q * 8 + i;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[i][e] = (T)0.f;
        if (m < M) x[i] = *(const vec8*)(X + (long)m * ldx + col);
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) g[i] = *(const vec8*)(dgut + (n0 + i * 16 + r16) * Mp + q * 8);
    transpose8(x, f);
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[i][j] = T16<T>::mfma16(f[j], g[i], f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int d = d0 + (r * 4 + q) * 8;
            if (d >= K) continue;
            TW* const o = dW + (n0 + i * 16 + r16) * lddw + d;
            float v[8];
            if (accumulate) load_vec<TW, 8>(o, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = accumulate ? v[j] + acc[i][j][r] : acc[i][j][r];
            store_stream<TW, 8, AROUND>(o, v);
        }
}

// both in one launch - dX reads W while dW is written: blocks [0, dx_blocks) dX (columns fastest), the others dW
template <typename T, typename TW, int MT, bool AROUND>
__global__ __launch_bounds__(256) void swiglu_rows_backward_kernel(const T* __restrict__ dgu, const T* __restrict__ W, long ldw, int M, int N, int K, int shares,
                                                                   float* __restrict__ part, int dx_blocks, const T* __restrict__ dgut, long Mp,
                                                                   const T* __restrict__ X, long ldx, TW* __restrict__ dW, long lddw, int accumulate) {
    const int columns = (K + 127) / 128, id = blockIdx.x;
    if (id < dx_blocks) dx_rows_block<T, MT>(id % columns, id / columns, dgu, N, W, ldw, M, N, K, shares, part);
    else dw_rows_block<T, TW, AROUND>((id - dx_blocks) % columns, (id - dx_blocks) / columns, dgut, Mp, X, ldx, M, N, K, dW, lddw, accumulate);
}

// rows that the three kernels take, against the GEMM forms beside them: whole calls back to back at 3584 x 37888, bf16, over weights that do not fit the last-level
// cache (us): forward 59 / 65 / 73 at 1 / 8 / 16 rows, the 128x128 tile 67 / 71 / 80 at 17 / 64 / 128; dX and dW of one call 154 at 1 - 32 rows, the GEMM forms 158 / 161
// at 33 / 64; with the fp32 dW added 314 - 324 against 362 - 364.  (dX alone: 69 - 82 at 1 - 32 against 60 at 33; dW alone 78 - 87 against 70.)
constexpr int FWD_ROWS = 16, BWD_ROWS = 32;

// shares of W's rows per 128 columns of dX: three blocks per CU, at least 4 steps of 32 rows per wave
static int dx_shares(int N, int K) {
    const int want = ceil_div(768, ceil_div(K, 128)), most = N / 32 / 16;
    return want < most ? want : most < 1 ? 1 : most;
}

// dX = dGU W for more rows: the GEMM with the K-major weight operand (gemm_mi16.hip), or a tile transpose of W in front of the NT GEMM, whose main loop is faster
// (12 860 rows: 2.43 + 0.12 ms against 2.78; 1 607 rows: 0.41 + 0.12 against 0.43).  Either may split its contraction (N) into fp32 partials where one round
// of tiles leaves CUs idle.  Estimated in microseconds: a 64-deep K-tile of a 256x256 tile takes 1.7 K-major and 1.48 NT (all CUs busy; the wide NT tiles are
// 10 % and 5 % better per flop), the transpose moves its bytes at 4.6 TB/s.  Small problems run on the ring kernel (gemm_ring.hip).  Most alternatives were
// forced in turn on 41 shapes (448 .. 3584 x 1024 .. 37888, 40 .. 4 096 rows; dX and dW): in 68 of 82 products the choice is among the five fastest and within
// 8 % of the best.  The others take a share count that the sweep left out, or lie behind it: 448 x 4544, 4 096 rows 15 % or more (K-major, eight shares, where the ring
// kernel in two takes 46 us - join_us prices 117 MB of partials as if they stayed in the cache).
enum { DX_KMAJOR, DX_TRANSPOSED, DX_RING };
struct DxPlan { int kind, bm, splits; };
// a 64-deep K-tile of the 128x128 ring kernel: 0.35 us alone, 0.7 with a block on every CU (L2)
static double ring_us(long tiles, int cus) { return 0.35 + 0.35 * (double)tiles / cus; }
// the partials' write and read, and a launch; up to ~120 MB they stay in the last-level cache
static double join_us(int splits, double rows, double cols) {
    const double bytes = splits * rows * cols * 8;
    return splits > 1 ? 3.0 + bytes / (bytes < 1.2e8 ? 10e6 : 5e6) : 0.0;
}
static DxPlan dx_plan(int M, int N, int K) {
    const int cus = device_cu_count(current_device()), kt = N / 64;
    DxPlan best = {DX_KMAJOR, 256, 1};
    double least = 1e30;
    auto consider = [&](int kind, int bm, int bn, int splits, double per_tile) {
        const long tiles = (long)ceil_div(M, bm) * ceil_div(K, bn) * splits;
        if (kind == DX_RING && tiles > cus) return;
        const double rounds = (double)((tiles + cus - 1) / cus);
        if (kind == DX_RING) per_tile = ring_us(tiles, cus);
        const double t = rounds * (ceil_div(kt, splits) * per_tile + 4.0) + join_us(splits, M, K) + (kind == DX_TRANSPOSED ? (double)N * K * 4 / 4.6e6 + 4.0 : 0.0);
        if (t < least) { least = t; best = {kind, bm, splits}; }
    };
    consider(DX_KMAJOR, 256, 256, 1, 1.7);
    consider(DX_TRANSPOSED, 256, 256, 1, 1.48);          // (vitg_gemm picks its own tile: the cheapest of these three)
    if (K >= 384) consider(DX_TRANSPOSED, 256, 384, 1, 1.48 * 1.5 / 1.1);
    if (M >= 384) consider(DX_TRANSPOSED, 384, 256, 1, 1.48 * 1.5 / 1.05);
    for (int sp = 1; sp <= 16 && sp <= kt; ++sp) {
        consider(DX_RING, 128, 128, sp, 0.0);
        if (sp < 2 || sp * 4 > kt) continue;
        consider(DX_KMAJOR, 256, 256, sp, 1.7);
        consider(DX_TRANSPOSED, 256, 256, sp, 1.48);
        if (M > 256) { consider(DX_KMAJOR, 320, 256, sp, 1.67 * 1.25); consider(DX_TRANSPOSED, 320, 256, sp, 1.45 * 1.25); }
    }
    return best;
}

// dW = dGU^T X has a long contraction (the rows) and, for narrow layers, few tiles: the same split, the same estimate
struct DwPlan { bool ring; int splits; };
static DwPlan dw_plan(long Mp, int N, int K) {
    const int cus = device_cu_count(current_device()), kt = (int)(Mp / 64);
    const long wide = (long)ceil_div(N, 256) * ceil_div(K, 256), small = (long)ceil_div(N, 128) * ceil_div(K, 128);
    DwPlan best = {false, 1};
    double least = 1e30;
    for (int sp = 1; sp <= 16 && sp <= kt; ++sp) {
        const double j = join_us(sp, N, K), tw = (double)((wide * sp + cus - 1) / cus) * (ceil_div(kt, sp) * 1.6 + 4.0) + j, tr = ceil_div(kt, sp) * ring_us(small * sp, cus) + 4.0 + j;
        if ((sp == 1 || sp * 4 <= kt) && tw < least) { least = tw; best = {false, sp}; }
        if (small * sp <= cus && tr < least) { least = tr; best = {true, sp}; }
    }
    return best;
}

static size_t pad256(size_t b) { return (b + 255) & ~(size_t)255; }
struct SwigluWorkspace { size_t dgu, dgut, xt, wt, part, bytes; long Mp; int dx_shares; DxPlan dx; DwPlan dw; bool pair; };
static SwigluWorkspace swiglu_workspace(int M, int N, int K, bool dx, bool dw) {
    SwigluWorkspace w = {};
    w.Mp = ((long)M + 63) / 64 * 64;
    size_t at = 0, part = 0;
    auto take = [&](size_t bytes) { const size_t a = at; at += pad256(bytes); return a; };
    if (dx) {
        w.dgu = take((size_t)M * N * 2);
        if (M <= BWD_ROWS) { w.dx_shares = dx_shares(N, K); part = (size_t)w.dx_shares * M * K * 4; }
        else {
            w.dx = dx_plan(M, N, K);
            if (w.dx.kind == DX_TRANSPOSED) w.wt = take((size_t)K * N * 2);
            if (w.dx.splits > 1) part = (size_t)w.dx.splits * M * K * 4;
        }
    }
    if (dw) {
        w.dgut = take((size_t)N * w.Mp * 2);
        if (M > BWD_ROWS) {
            w.xt = take((size_t)K * w.Mp * 2);
            w.dw = dw_plan(w.Mp, N, K);
            // (one share of the ring kernel needs a partial only where it is added to dW or shares a launch with dX)
            const size_t p = w.dw.splits > 1 || w.dw.ring ? (size_t)w.dw.splits * N * K * 4 : 0;
            // two ring products share one launch and one join: fewer launches, and the smaller one fills the CUs that the other leaves
            w.pair = dx && w.dw.ring && w.dx.kind == DX_RING;
            if (w.pair) part = (size_t)w.dx.splits * M * K * 4 + p;
            else if (p > part) part = p;                 // (dX's partials are joined before dW's are written)
        }
    }
    w.part = take(part);
    w.bytes = at;
    return w;
}

}  // namespace vitg

using namespace vitg;

// the GEMM kernels address a tile (up to 384 rows) with 32-bit byte offsets
static bool ld_ok(long ld) { return ld < (1l << 22); }

extern "C" int vitg_swiglu(const void* X, int ldx, const void* W, int ldw, int M, int N, int K, int dtype, void* out, int ldo, void* gu, int ldgu, void* stream) {
    if (M <= 0 || N <= 0) return 0;
    if (!X || !W || !out) return VITG_ERR_ARG;
    if (dtype != DT_BF16 && dtype != DT_F16) return VITG_ERR_DTYPE;
    if (K <= 0 || K % 64 || N % 64 || ldx < K || ldw < K || ldo < N / 2 || (gu && ldgu < N)) return VITG_ERR_SHAPE;
    if (M >= (1 << 30) || N >= (1 << 30) || !ld_ok(ldx) || !ld_ok(ldw) || !ld_ok(ldo) || (gu && !ld_ok(ldgu))) return VITG_ERR_SHAPE;
    if (ldx % 8 || ldw % 8 || ldo % 8 || (gu && ldgu % 8)) return VITG_ERR_ALIGN;
    if (!aligned_to(X, 16) || !aligned_to(W, 16) || !aligned_to(out, 16) || (gu && !aligned_to(gu, 16))) return VITG_ERR_ALIGN;
    hipStream_t s = (hipStream_t)stream;
    if (M <= FWD_ROWS) {
        auto run = [&](auto t) {
            typedef decltype(t) T;
            hipLaunchKernelGGL(swiglu_rows_kernel<T>, dim3(N / 32), dim3(256), 0, s, (const T*)X, (long)ldx, (const T*)W, (long)ldw, M, K, (T*)out, (long)ldo, (T*)gu, (long)ldgu);
        };
        if (dtype == DT_BF16) run(bf16_t{}); else run(f16_t{});
        return launched();
    }
    GemmArgs g = {};
    g.A = X; g.lda = ldx; g.W = W; g.ldw = ldw; g.M = M; g.N = N; g.K = K;
    g.out = out; g.ldo = ldo; g.gu = gu; g.ldgu = ldgu; g.split_k = 1;
    // at most one 128x128 tile per CU: the ring kernel (K = 1024, N = 4096, 512 rows: 12 us against 16 on the 128x128 tile and 23 on 256x256).  Up to 128 rows,
    // and with pre-activations up to two tiles per CU, the 128x128 tile at two blocks per CU (3584 x 37888, 128 rows: 73 against 100 us on a half-empty
    // 256-row tile; 2048 x 16384, 512 rows: 43 against 47); beyond that the 256-row tiles (1 024 rows: 57 against 80)
    const long tiles = (long)ceil_div(M, 128) * ceil_div(N, 128);
    const int cus = device_cu_count(current_device());
    int rc;
    if (tiles <= cus) rc = launch_gemm_ring(g, dtype, MODE_SWIGLU, false, s);
    else if (M <= 128 || (gu && tiles <= 2 * cus)) rc = launch_gemm128_swiglu(g, dtype, s);
    else if (gu) rc = launch_gemm_mi16_swiglu_save(g, dtype, s);
    else if (M < 256) rc = launch_gemm_mi16(g, dtype, MODE_SWIGLU, 6, s);
    else return vitg_gemm(X, ldx, W, ldw, M, N, K, dtype, VITG_GEMM_SWIGLU, nullptr, VITG_ACT_NONE, out, ldo, nullptr, 0, 0, stream);
    return rc == 0 ? 0 : VITG_ERR_LAUNCH;
}

extern "C" int vitg_swiglu_backward_plan(int M, int N, int K, int want_dx, int want_dw, long* workspace_bytes) {
    if (!workspace_bytes) return VITG_ERR_ARG;
    if (M < 0 || N <= 0 || K <= 0 || K % 64 || N % 64 || !ld_ok((long)M + 63) || !ld_ok(N)) return VITG_ERR_SHAPE;
    *workspace_bytes = M ? (long)swiglu_workspace(M, N, K, want_dx != 0, want_dw != 0).bytes : 0;
    return 0;
}

extern "C" int vitg_swiglu_backward(const void* dout, int lddo, const void* gu, int ldgu, const void* X, int ldx, const void* W, int ldw, int M, int N, int K,
                                    int dtype, void* dX, int lddx, void* dW, int lddw, int dw_dtype, int accumulate, void* workspace, long workspace_bytes,
                                    void* stream) {
    if (M < 0 || N <= 0 || K <= 0 || K % 64 || N % 64 || !ld_ok((long)M + 63) || !ld_ok(N)) return VITG_ERR_SHAPE;
    if (dtype != DT_BF16 && dtype != DT_F16) return VITG_ERR_DTYPE;
    if (!dX && !dW) return 0;
    if (dW && dw_dtype != dtype && dw_dtype != DT_F32) return VITG_ERR_DTYPE;
    if (dW && (lddw < K || lddw % 8 || !aligned_to(dW, 16))) return lddw < K ? VITG_ERR_SHAPE : VITG_ERR_ALIGN;
    hipStream_t s = (hipStream_t)stream;
    if (M == 0) {                                        // no rows: dW is zero (or what it was)
        if (dW && !accumulate) hipLaunchKernelGGL(zero_bytes_kernel, dim3(N < 4096 ? N : 4096), dim3(256), 0, s, (char*)dW, (long)lddw * dtype_size(dw_dtype), (long)N, (long)K * dtype_size(dw_dtype));
        return launched();
    }
    if (!dout || !gu || (dW && !X) || (dX && !W)) return VITG_ERR_ARG;
    if (lddo < N / 2 || ldgu < N || (dW && ldx < K) || (dX && (ldw < K || lddx < K))) return VITG_ERR_SHAPE;
    if (!ld_ok(lddo) || !ld_ok(ldgu) || (dW && (!ld_ok(ldx) || !ld_ok(lddw))) || (dX && (!ld_ok(ldw) || !ld_ok(lddx)))) return VITG_ERR_SHAPE;
    if (lddo % 8 || ldgu % 8 || (dW && ldx % 8) || (dX && (ldw % 8 || lddx % 8))) return VITG_ERR_ALIGN;
    if (!aligned_to(dout, 16) || !aligned_to(gu, 16) || (dW && !aligned_to(X, 16)) || (dX && (!aligned_to(W, 16) || !aligned_to(dX, 16)))) return VITG_ERR_ALIGN;
    const SwigluWorkspace ws = swiglu_workspace(M, N, K, dX != nullptr, dW != nullptr);
    if (!workspace || workspace_bytes < (long)ws.bytes || !aligned_to(workspace, 16)) return VITG_ERR_ARG;
    char* const base = (char*)workspace;
    void *const dgu = dX ? base + ws.dgu : nullptr, *const dgut = dW ? base + ws.dgut : nullptr, *const xt = base + ws.xt;
    float* const part = (float*)(base + ws.part);
    auto run = [&](auto t) -> int {
        typedef decltype(t) T;
        const bool few = M <= BWD_ROWS, pair = !few && dX && dW && ws.pair;
        {
            const long mt = ws.Mp / 64;
            SwigluPrep<T> a = {(const T*)dout, (long)lddo, (const T*)gu, (long)ldgu, (long)M, ws.Mp, (T*)dgu, (long)N, (T*)dgut,
                               (const T*)X, (long)ldx, (T*)xt, (const T*)W, (long)ldw, (T*)(base + ws.wt), N, K, mt * (N / 64), 0};
            a.x_end = a.grad + (dW && !few ? mt * (K / 64) : 0);
            const long blocks = a.x_end + (dX && !few && ws.dx.kind == DX_TRANSPOSED ? (long)(N / 64) * (K / 64) : 0);
            hipLaunchKernelGGL(swiglu_prep_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, s, a);
        }
        const JoinArgs join_dx = {part, M, K, few ? ws.dx_shares : ws.dx.splits, dX, lddx, 0};
        if (few) {
            const int columns = ceil_div(K, 128), nx = dX ? columns * ws.dx_shares : 0, nw = dW ? columns * ceil_div(N, 4 * DW_WAVE) : 0;
            auto go = [&](auto tw) {
                typedef decltype(tw) TW;
                auto launch = [&](auto kernel) {
                    hipLaunchKernelGGL(kernel, dim3(nx + nw), dim3(256), 0, s, (const T*)dgu, (const T*)W, (long)ldw, M, N, K, ws.dx_shares, part, nx, (const T*)dgut, ws.Mp, (const T*)X, (long)ldx, (TW*)dW, (long)lddw, accumulate);
                };
                with_flag((long)N * K * (long)sizeof(TW) > STREAM_BYTES, [&](auto around) {
                    constexpr bool AROUND = decltype(around)::value;
                    if (M <= 16) launch(swiglu_rows_backward_kernel<T, TW, 1, AROUND>); else launch(swiglu_rows_backward_kernel<T, TW, 2, AROUND>);
                });
            };
            if (dW && dw_dtype == DT_F32) go(float{}); else go(t);
            if (dX) join_shares<T>(join_dx, s);
            return launched();
        }
        GemmArgs gx = {}, gw = {};
        const int Mp = (int)ws.Mp;
        if (dX) {
            const DxPlan p = ws.dx;
            gx.A = dgu; gx.lda = N; gx.W = W; gx.ldw = ldw; gx.M = M; gx.N = K; gx.K = N; gx.split_k = p.splits;
            if (p.splits > 1 || pair) { gx.out = part; gx.ldo = K; gx.split_stride = (long)M * K; }
            else { gx.out = dX; gx.ldo = lddx; }
            if (p.kind == DX_TRANSPOSED) { gx.W = base + ws.wt; gx.ldw = N; }
        }
        if (dW) {
            gw.A = dgut; gw.lda = Mp; gw.W = xt; gw.ldw = Mp; gw.M = N; gw.N = K; gw.K = Mp; gw.split_k = ws.dw.splits;
            gw.out = pair ? part + (size_t)ws.dx.splits * M * K : part; gw.ldo = K; gw.split_stride = (long)N * K;
        }
        const JoinArgs join_dw = {(const float*)gw.out, N, K, ws.dw.splits, dW, lddw, accumulate};
        if (pair) {
            if (launch_gemm_ring_pair(gx, gw, dtype, s) != 0) return VITG_ERR_LAUNCH;
            if (dw_dtype == DT_F32) join_shares<T, float>(join_dx, s, join_dw); else join_shares<T, T>(join_dx, s, join_dw);
            return launched();
        }
        if (dX) {
            const DxPlan p = ws.dx;
            int rc;
            if (p.kind == DX_RING) rc = launch_gemm_ring(gx, dtype, p.splits > 1 ? MODE_F32 : MODE_STORE16, true, s);
            else if (p.kind == DX_KMAJOR) rc = launch_gemm_mi16_kmajor(gx, dtype, p.bm, s);
            else if (p.splits > 1) rc = launch_gemm_mi16(gx, dtype, MODE_F32, p.bm == 320 ? 12 : 6, s);
            else rc = vitg_gemm(dgu, N, gx.W, N, M, K, N, dtype, VITG_GEMM_STORE16, nullptr, VITG_ACT_NONE, dX, lddx, nullptr, 0, 0, stream);
            if (rc) return VITG_ERR_LAUNCH;
            if (p.splits > 1) join_shares<T>(join_dx, s);
        }
        if (dW) {
            const DwPlan p = ws.dw;
            if (p.ring && p.splits == 1 && !accumulate && dw_dtype != DT_F32) {
                gw.out = dW; gw.ldo = lddw;
                if (launch_gemm_ring(gw, dtype, MODE_STORE16, false, s) != 0) return VITG_ERR_LAUNCH;
            } else if (p.ring || p.splits > 1) {
                if ((p.ring ? launch_gemm_ring(gw, dtype, MODE_F32, false, s) : launch_gemm_mi16(gw, dtype, MODE_F32, 6, s)) != 0) return VITG_ERR_LAUNCH;
                if (dw_dtype == DT_F32) join_shares<float>(join_dw, s); else join_shares<T>(join_dw, s);
            } else if (accumulate && dw_dtype == DT_F32) {
                // added once, behind the sum, as join_quad does: a small step's sum keeps its bits beside a large running gradient on every route.  (Carried
                // in the accumulators instead: 0.2 % of the values a step off; 12 860 rows 3.05 ms against 3.10, 4 100 rows 1.08 against 1.14.  In 16 bits the old value
                // does start the accumulators, below: the result's rounding is 2^13 times theirs.)
                gw.out = dW; gw.ldo = lddw; gw.res = (const float*)dW; gw.ldr = lddw; gw.res_last = 1;
                const int cfg = gemm256_applicable(gw, MODE_F32) && gemm256_pick_cfg(gw, MODE_F32) == 9 ? 9 : 6;     // 256x384 or 256x256
                if (launch_gemm_mi16(gw, dtype, MODE_F32, cfg, s) != 0) return VITG_ERR_LAUNCH;
            } else {
                const int rc = dw_dtype == DT_F32
                    ? vitg_gemm(dgut, Mp, xt, Mp, N, K, Mp, dtype, VITG_GEMM_F32, nullptr, VITG_ACT_NONE, dW, lddw, nullptr, 0, 0, stream)
                    : accumulate ? vitg_gemm_res16(dgut, Mp, xt, Mp, N, K, Mp, dtype, nullptr, dW, lddw, dW, lddw, nullptr, 0, 0, stream)
                                 : vitg_gemm(dgut, Mp, xt, Mp, N, K, Mp, dtype, VITG_GEMM_STORE16, nullptr, VITG_ACT_NONE, dW, lddw, nullptr, 0, 0, stream);
                if (rc) return rc;
            }
        }
        return launched();
    };
    return dtype == DT_BF16 ? run(bf16_t{}) : run(f16_t{});
}
