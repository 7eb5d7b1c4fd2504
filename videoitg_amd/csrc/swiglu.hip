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
#include "train_common.h"
#include "gemm_common.h"

namespace vitg {

// out[c, r] = in[r, c] for r < R, c < C; columns R .. Rp-1 of out are zero (K padding of the GEMM that reads it).  64 x 64 tiles through LDS.
constexpr int TR_LD = 72;                                // halfs per LDS row: 16-B aligned
template <typename T>
__global__ __launch_bounds__(256) void transpose16_kernel(const T* __restrict__ in, long ldi, long R, int C, T* __restrict__ out, long ldo, long Rp) {
    typedef typename T16<T>::vec8 vec8;
    __shared__ __attribute__((aligned(16))) T tile[64 * TR_LD];          // [c][r]
    const long r0 = (long)blockIdx.x * 64;
    const int c0 = blockIdx.y * 64;
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
__global__ __launch_bounds__(256) void swiglu_grad_kernel(const T* __restrict__ dh, long lddh, const T* __restrict__ gu, long ldgu, long M, long Mp,
                                                          T* __restrict__ dgu, long lddgu, T* __restrict__ dgut) {
    typedef typename T16<T>::vec8 vec8;
    __shared__ __attribute__((aligned(16))) T tile[64 * TR_LD];          // [column of gu][row]
    const long r0 = (long)blockIdx.x * 64;
    const int f0 = blockIdx.y * 32, n0 = blockIdx.y * 64;
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
__global__ __launch_bounds__(256) void swiglu_dx_rows_kernel(const T* __restrict__ dgu, long lddgu, const T* __restrict__ W, long ldw, int M, int N, int K,
                                                             int shares, float* __restrict__ part) {
    typedef typename T16<T>::vec8 vec8;
    __shared__ __attribute__((aligned(16))) f32x4 red[2][8][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, q = lane >> 4;
    const int d0 = blockIdx.x * 128;
    const int col = min(d0 + ((r16 & 3) * 4 + (r16 >> 2)) * 8, K - 8);   // (the last block may hang over: its loads repeat, its stores are left out)
    const long steps = N / 32, ways = (long)shares * 4, way = (long)blockIdx.y * 4 + wave;
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
        float* const o = part + ((long)blockIdx.y * M + m) * K;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int d = d0 + (r * 4 + q) * 8;
            if (d >= K) continue;
            *(f32x4*)(o + d) = f32x4{acc[i][0][r], acc[i][1][r], acc[i][2][r], acc[i][3][r]};
            *(f32x4*)(o + d + 4) = f32x4{acc[i][4][r], acc[i][5][r], acc[i][6][r], acc[i][7][r]};
        }
    }
}

// out[m, :] (+)= sum of the shares [share][M][K] in order
template <typename T>
__global__ __launch_bounds__(256) void join_shares_kernel(const float* __restrict__ part, long M, int K, int shares, T* __restrict__ out, long ldo, int accumulate) {
    const long i = ((long)blockIdx.x * 256 + threadIdx.x) * 4, total = M * K;
    if (i >= total) return;
    f32x4 v = *(const f32x4*)(part + i);
#pragma unroll 8
    for (int s = 1; s < shares; ++s) v += *(const f32x4*)(part + s * total + i);
    T* const o = out + i / K * ldo + i % K;
    float w[4] = {0.f, 0.f, 0.f, 0.f};
    if (accumulate) load_vec<T, 4>(o, w);
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = accumulate ? w[e] + v[e] : v[e];
    store_vec<T, 4>(o, w);
}
template <typename T> static void join_shares(const float* part, long M, int K, int shares, void* out, long ldo, int accumulate, hipStream_t s) {
    hipLaunchKernelGGL(join_shares_kernel<T>, dim3((unsigned)((M * K / 4 + 255) / 256)), dim3(256), 0, s, part, M, K, shares, (T*)out, ldo, accumulate);
}

// dW (+)= dGU^T X for M <= 32 rows: a wave owns 64 rows x 128 columns of dW.  A = X transposed in registers (as above), B = dGU^T rows from the transposed copy.  Bound by the write of dW.
template <typename T, typename TW>
__global__ __launch_bounds__(256) void swiglu_dw_rows_kernel(const T* __restrict__ dgut, long Mp, const T* __restrict__ X, long ldx, int M, int N, int K,
                                                             TW* __restrict__ dW, long lddw, int accumulate) {
    typedef typename T16<T>::vec8 vec8;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, q = lane >> 4;
    const long n0 = ((long)blockIdx.y * 4 + wave) * 64;
    const int d0 = blockIdx.x * 128, col = min(d0 + ((r16 & 3) * 4 + (r16 >> 2)) * 8, K - 8);
    if (n0 >= N) return;
    f32x4 acc[4][8];
    vec8 x[8], f[8], g[4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int m = q * 8 + i;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[i][e] = (T)0.f;
        if (m < M) x[i] = *(const vec8*)(X + (long)m * ldx + col);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) g[i] = *(const vec8*)(dgut + (n0 + i * 16 + r16) * Mp + q * 8);
    transpose8(x, f);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[i][j] = T16<T>::mfma16(f[j], g[i], f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int d = d0 + (r * 4 + q) * 8;
            if (d >= K) continue;
            TW* const o = dW + (n0 + i * 16 + r16) * lddw + d;
            float v[8];
            if (accumulate) load_vec<TW, 8>(o, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = accumulate ? v[j] + acc[i][j][r] : acc[i][j][r];
            store_vec<TW, 8>(o, v);
        }
}

// rows that the three kernels take, against the GEMM forms at 3584 x 37888 (us): forward 61 - 74 at 1 - 16 rows, the 128-row tile 69 - 75 at 17 - 128;
// dX 70 - 83 at 1 - 32, 110 at 64, the K-major GEMM 91 at 65; dW 50 at 1 - 32, the GEMM 59 - 67 with a transpose of X in front
constexpr int FWD_ROWS = 16, DX_ROWS = 32, DW_ROWS = 32;

// shares of W's rows per 128 columns of dX: three blocks per CU, at least 4 steps of 32 rows per wave
static int dx_shares(int N, int K) {
    const int want = ceil_div(768, ceil_div(K, 128)), most = N / 32 / 16;
    return want < most ? want : most < 1 ? 1 : most;
}

// dX = dGU W for more rows: the GEMM with the K-major weight operand (gemm_mi16.hip), or a tile transpose of W in front of the NT GEMM, whose main loop is faster
// (12 860 rows: 2.43 + 0.12 ms against 2.78; 1 607 rows: 0.41 + 0.12 against 0.43).  Either may split its contraction (N) into fp32 partials where one round
// of tiles leaves CUs idle.  Estimated in microseconds: a 64-deep K-tile of a 256x256 tile takes 1.7 K-major and 1.48 NT (all CUs busy; the wide NT tiles are
// 10 % and 5 % better per flop), the transpose and the partials' write and read their bytes at 4.6 and 5 TB/s.
struct DxPlan { int bm, splits; bool transposed; };
static DxPlan dx_plan(int M, int N, int K) {
    const int cus = device_cu_count(current_device()), kt = N / 64;
    DxPlan best = {256, 1, false};
    double least = 1e30;
    auto consider = [&](int bm, int bn, int splits, bool transposed, double per_tile) {
        const double tiles = (double)ceil_div(M, bm) * ceil_div(K, bn) * splits;
        const double rounds = (double)(long)((tiles + cus - 1) / cus);
        const double t = rounds * (ceil_div(kt, splits) * per_tile * bm * bn / 65536.0 + 4.0) + (splits > 1 ? (double)splits * M * K * 8 / 5e6 + 6.0 : 0.0) +
                         (transposed ? (double)N * K * 4 / 4.6e6 + 4.0 : 0.0);
        if (t < least) { least = t; best = {bm, splits, transposed}; }
    };
    consider(256, 256, 1, false, 1.7);
    consider(256, 256, 1, true, 1.48);                   // (vitg_gemm picks its own tile: the cheapest of these three)
    if (K >= 384) consider(256, 384, 1, true, 1.48 / 1.1);
    if (M >= 384) consider(384, 256, 1, true, 1.48 / 1.05);
    for (int sp = 2; sp <= 16 && sp * 4 <= kt; ++sp) {
        consider(256, 256, sp, false, 1.7);
        consider(256, 256, sp, true, 1.48);
        if (M > 256) { consider(320, 256, sp, false, 1.67); consider(320, 256, sp, true, 1.45); }
    }
    return best;
}

// dW = dGU^T X has a long contraction (the rows) and, for narrow layers, few tiles: the same split, the same estimate
static int dw_splits(long Mp, int N, int K) {
    const int cus = device_cu_count(current_device());
    const long kt = Mp / 64, tiles = (long)ceil_div(N, 256) * ceil_div(K, 256);
    int best = 1;
    double least = 1e30;
    for (int sp = 1; sp <= 16 && (sp == 1 || sp * 4 <= kt); ++sp) {
        const double t = (double)((tiles * sp + cus - 1) / cus) * ((double)((kt + sp - 1) / sp) * 1.7 + 4.0) + (sp > 1 ? (double)sp * N * K * 8 / 5e6 + 6.0 : 0.0);
        if (t < least) { least = t; best = sp; }
    }
    return best;
}

static size_t pad256(size_t b) { return (b + 255) & ~(size_t)255; }
struct SwigluWorkspace { size_t dgu, dgut, xt, wt, part, bytes; long Mp; int dx_shares, dw_splits; DxPlan plan; };
static SwigluWorkspace swiglu_workspace(int M, int N, int K, bool dx, bool dw) {
    SwigluWorkspace w = {};
    w.Mp = ((long)M + 63) / 64 * 64;
    size_t at = 0, part = 0;
    auto take = [&](size_t bytes) { const size_t a = at; at += pad256(bytes); return a; };
    if (dx) {
        w.dgu = take((size_t)M * N * 2);
        if (M <= DX_ROWS) { w.dx_shares = dx_shares(N, K); part = (size_t)w.dx_shares * M * K * 4; }
        else {
            w.plan = dx_plan(M, N, K);
            if (w.plan.transposed) w.wt = take((size_t)K * N * 2);
            if (w.plan.splits > 1) part = (size_t)w.plan.splits * M * K * 4;
        }
    }
    if (dw) {
        w.dgut = take((size_t)N * w.Mp * 2);
        w.dw_splits = 1;
        if (M > DW_ROWS) {
            w.xt = take((size_t)K * w.Mp * 2);
            w.dw_splits = dw_splits(w.Mp, N, K);
            const size_t p = w.dw_splits > 1 ? (size_t)w.dw_splits * N * K * 4 : 0;
            if (p > part) part = p;                      // (dX's partials are joined before dW's are written)
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
    if (!ld_ok(ldx) || !ld_ok(ldw) || !ld_ok(ldo) || (gu && !ld_ok(ldgu))) return VITG_ERR_SHAPE;
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
    // the 128x128 tile while its tiles fit the chip once (K = 1024, N = 4096, 1 024 rows: 17.6 us against 23.5 on 256x256) and up to 128 rows (a 256-row tile
    // would be half empty: 73 against 100 us at 3584 x 37888); beyond that the 256-row tiles
    int rc;
    if (M <= 128 || (long)ceil_div(M, 128) * ceil_div(N, 128) <= device_cu_count(current_device())) rc = launch_gemm128_swiglu(g, dtype, s);
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
    void *dgu = dX ? base + ws.dgu : nullptr, *dgut = dW ? base + ws.dgut : nullptr, *xt = base + ws.xt;
    const unsigned mt = (unsigned)(ws.Mp / 64);
    float* const part = (float*)(base + ws.part);
    auto run = [&](auto t) -> int {
        typedef decltype(t) T;
        hipLaunchKernelGGL(swiglu_grad_kernel<T>, dim3(mt, N / 64), dim3(256), 0, s, (const T*)dout, (long)lddo, (const T*)gu, (long)ldgu, (long)M, ws.Mp, (T*)dgu, (long)N, (T*)dgut);
        if (dX && M <= DX_ROWS) {
            auto go = [&](auto kernel) {
                hipLaunchKernelGGL(kernel, dim3(ceil_div(K, 128), ws.dx_shares), dim3(256), 0, s, (const T*)dgu, (long)N, (const T*)W, (long)ldw, M, N, K, ws.dx_shares, part);
            };
            if (M <= 16) go(swiglu_dx_rows_kernel<T, 1>); else go(swiglu_dx_rows_kernel<T, 2>);
            join_shares<T>(part, M, K, ws.dx_shares, dX, lddx, 0, s);
        } else if (dX) {
            GemmArgs g = {};
            g.A = dgu; g.lda = N; g.W = W; g.ldw = ldw; g.M = M; g.N = K; g.K = N;
            g.split_k = ws.plan.splits;
            if (ws.plan.splits > 1) { g.out = part; g.ldo = K; g.split_stride = (long)M * K; }
            else { g.out = dX; g.ldo = lddx; }
            if (ws.plan.transposed) {
                hipLaunchKernelGGL(transpose16_kernel<T>, dim3(N / 64, K / 64), dim3(256), 0, s, (const T*)W, (long)ldw, (long)N, K, (T*)(base + ws.wt), (long)N, (long)N);
                g.W = base + ws.wt; g.ldw = N;
            }
            int rc;
            if (!ws.plan.transposed) rc = launch_gemm_mi16_kmajor(g, dtype, ws.plan.bm, s);
            else if (ws.plan.splits > 1) rc = launch_gemm_mi16(g, dtype, MODE_F32, ws.plan.bm == 320 ? 12 : 6, s);
            else rc = vitg_gemm(dgu, N, g.W, N, M, K, N, dtype, VITG_GEMM_STORE16, nullptr, VITG_ACT_NONE, dX, lddx, nullptr, 0, 0, stream);
            if (rc) return VITG_ERR_LAUNCH;
            if (ws.plan.splits > 1) join_shares<T>(part, M, K, ws.plan.splits, dX, lddx, 0, s);
        }
        if (dW && M <= DW_ROWS) {
            auto go = [&](auto tw) {
                typedef decltype(tw) TW;
                hipLaunchKernelGGL((swiglu_dw_rows_kernel<T, TW>), dim3(ceil_div(K, 128), ceil_div(N, 256)), dim3(256), 0, s, (const T*)dgut, ws.Mp, (const T*)X, (long)ldx, M, N, K, (TW*)dW, (long)lddw, accumulate);
            };
            if (dw_dtype == DT_F32) go(float{}); else go(t);
        } else if (dW) {
            void* const xt = base + ws.xt;
            const int Mp = (int)ws.Mp;
            hipLaunchKernelGGL(transpose16_kernel<T>, dim3(mt, K / 64), dim3(256), 0, s, (const T*)X, (long)ldx, (long)M, K, (T*)xt, ws.Mp, ws.Mp);
            if (ws.dw_splits > 1) {
                GemmArgs g = {};
                g.A = dgut; g.lda = Mp; g.W = xt; g.ldw = Mp; g.M = N; g.N = K; g.K = Mp;
                g.split_k = ws.dw_splits; g.out = part; g.ldo = K; g.split_stride = (long)N * K;
                if (launch_gemm_mi16(g, dtype, MODE_F32, 6, s) != 0) return VITG_ERR_LAUNCH;
                if (dw_dtype == DT_F32) join_shares<float>(part, N, K, ws.dw_splits, dW, lddw, accumulate, s);
                else join_shares<T>(part, N, K, ws.dw_splits, dW, lddw, accumulate, s);
            } else {
                const int rc = dw_dtype == DT_F32
                    ? vitg_gemm(dgut, Mp, xt, Mp, N, K, Mp, dtype, VITG_GEMM_F32, nullptr, VITG_ACT_NONE, dW, lddw, accumulate ? (const float*)dW : nullptr, lddw, 0, stream)
                    : accumulate ? vitg_gemm_res16(dgut, Mp, xt, Mp, N, K, Mp, dtype, nullptr, dW, lddw, dW, lddw, nullptr, 0, 0, stream)
                                 : vitg_gemm(dgut, Mp, xt, Mp, N, K, Mp, dtype, VITG_GEMM_STORE16, nullptr, VITG_ACT_NONE, dW, lddw, nullptr, 0, 0, stream);
                if (rc) return rc;
            }
        }
        return launched();
    };
    return dtype == DT_BF16 ? run(bf16_t{}) : run(f16_t{});
}
