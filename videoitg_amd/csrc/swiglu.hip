// The gated feed-forward's first half for training:  [G | U] = X W^T (weight rows interleaved [32 gate | 32 up]),  H = silu(G) * U,  and its backward.
//
//   sig = 1 / (1 + e^-G)      dG = dH U sig (1 + G (1 - sig))      dU = dH G sig
//   dX = dGU W      dW (+)= dGU^T X
//
// Forward: one GEMM with the activation and the product in its epilogue; for training the epilogue also stores the 16-bit pre-activations (M x 2F), which
// costs their write instead of a second GEMM in the backward pass.
// Backward: both products run on the NT GEMM kernels (contraction along both operands' rows), so the operands whose rows run the other way are
// transposed first: dGU comes out of its elementwise kernel in both orders, W and X pass through a tile transpose.  dGU is rounded to the 16-bit type once -
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

static size_t pad256(size_t b) { return (b + 255) & ~(size_t)255; }
struct SwigluWorkspace { size_t dgu, dgut, xt, wt, part, bytes; long Mp; int splits; };
static SwigluWorkspace swiglu_workspace(int M, int N, int K, bool dx, bool dw) {
    SwigluWorkspace w = {};
    w.Mp = ((long)M + 63) / 64 * 64;
    w.splits = 1;
    size_t at = 0;
    if (dx) { w.dgu = at; at += pad256((size_t)M * N * 2); w.wt = at; at += pad256((size_t)K * N * 2); }
    if (dw) { w.dgut = at; at += pad256((size_t)N * w.Mp * 2); w.xt = at; at += pad256((size_t)K * w.Mp * 2); }
    if (dx) {
        long part = 0;
        (void)vitg_gemm_splitk_plan(M, K, N, &w.splits, &part);
        w.part = at; at += pad256((size_t)part);
    }
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
    if (!gu) return vitg_gemm(X, ldx, W, ldw, M, N, K, dtype, VITG_GEMM_SWIGLU, nullptr, VITG_ACT_NONE, out, ldo, nullptr, 0, 0, stream);
    GemmArgs g = {};
    g.A = X; g.lda = ldx; g.W = W; g.ldw = ldw; g.M = M; g.N = N; g.K = K;
    g.out = out; g.ldo = ldo; g.gu = gu; g.ldgu = ldgu; g.split_k = 1;
    return launch_gemm_mi16_swiglu_save(g, dtype, (hipStream_t)stream) == 0 ? 0 : VITG_ERR_LAUNCH;
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
    void *dgu = dX ? base + ws.dgu : nullptr, *wt = base + ws.wt, *dgut = dW ? base + ws.dgut : nullptr, *xt = base + ws.xt;
    const unsigned mt = (unsigned)(ws.Mp / 64);
    auto run = [&](auto t) {
        typedef decltype(t) T;
        hipLaunchKernelGGL(swiglu_grad_kernel<T>, dim3(mt, N / 64), dim3(256), 0, s, (const T*)dout, (long)lddo, (const T*)gu, (long)ldgu, (long)M, ws.Mp, (T*)dgu, (long)N, (T*)dgut);
        if (dX) hipLaunchKernelGGL(transpose16_kernel<T>, dim3(N / 64, K / 64), dim3(256), 0, s, (const T*)W, (long)ldw, (long)N, K, (T*)wt, (long)N, (long)N);
        if (dW) hipLaunchKernelGGL(transpose16_kernel<T>, dim3(mt, K / 64), dim3(256), 0, s, (const T*)X, (long)ldx, (long)M, K, (T*)xt, ws.Mp, ws.Mp);
    };
    if (dtype == DT_BF16) run(bf16_t{}); else run(f16_t{});
    if (launched() != 0) return VITG_ERR_LAUNCH;
    if (dX) {
        const int rc = ws.splits > 1
            ? vitg_gemm_splitk16(dgu, N, wt, N, M, K, N, dtype, nullptr, dX, lddx, (float*)(base + ws.part), ws.splits, stream)
            : vitg_gemm(dgu, N, wt, N, M, K, N, dtype, VITG_GEMM_STORE16, nullptr, VITG_ACT_NONE, dX, lddx, nullptr, 0, 0, stream);
        if (rc) return rc;
    }
    if (dW) {
        const int Mp = (int)ws.Mp;
        if (dw_dtype == DT_F32)
            return vitg_gemm(dgut, Mp, xt, Mp, N, K, Mp, dtype, VITG_GEMM_F32, nullptr, VITG_ACT_NONE, dW, lddw, accumulate ? (const float*)dW : nullptr, lddw, 0, stream);
        if (accumulate) return vitg_gemm_res16(dgut, Mp, xt, Mp, N, K, Mp, dtype, nullptr, dW, lddw, dW, lddw, nullptr, 0, 0, stream);
        return vitg_gemm(dgut, Mp, xt, Mp, N, K, Mp, dtype, VITG_GEMM_STORE16, nullptr, VITG_ACT_NONE, dW, lddw, nullptr, 0, 0, stream);
    }
    return 0;
}
