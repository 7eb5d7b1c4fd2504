// C[M,N] = A[M,K] . W[N,K]^T (or A . W[K,N], WKM) for problems of at most one 128x128 tile per CU: latency, not the matrix pipe, is what they wait for.
//
// The wide tiles (gemm_mi16.hip) keep one K-tile in flight while one is multiplied; with few or narrow tiles a K-tile of work is shorter than a DMA round
// trip, and the loop runs at one K-tile per round trip.  Here a block keeps FOUR 64-deep K-tiles of 128 + 128 rows in LDS (128 KiB) and one in registers:
//   step t:  wait until this wave's DMA of tile t+1 has landed (three newer tiles stay in flight) and its fragment reads of tile t are done; barrier;
//            DMA of tile t+4 into the slot of tile t (every wave holds tile t in registers); fragment reads of tile t+1; the 32 MFMAs of tile t.
// Four waves as 2 x 2, 64 x 64 each, v_mfma_f32_16x16x32, MFMA "A" = weight rows (a lane holds 4 consecutive output features of one row).
// Measured: a step takes 0.35 us with one block on the chip (the barrier and the LDS reads), 0.7 us with a block on every CU (L2); K = 1024, N = 4096, 512 rows with
// the SwiGLU epilogue 12 us = 358 TFLOP/s, against 16 on the 128x128 tile of gemm.hip and 23 on the 256x256 one.
// LDS images and the XOR swizzles are those of gemm_mi16.hip (128-B rows, 16-B chunk ^ ((row >> 1) & 7); K-major weights: 256-B rows, 32-B chunk ^
// (((row >> 3) & 1) * 4 + (row & 3)), read with ds_read_b64_tr_b16).
#include "gemm_common.h"
#include "attn_common.h"

namespace vitg {

constexpr int RING_STAGES = 4, RING_TILE = 128, RING_STAGE = 2 * RING_TILE * 128, RING_THREADS = 256;

// one output tile: block `bid` of tiles_m * tiles_n, share `sp` of the contraction (mode F32)
template <typename T, int MODE, bool WKM>
__device__ __forceinline__ void ring_tile(const GemmArgs& g_, int bid, int sp, char* smem) {
    typedef typename T16<T>::vec8 vec8;
    typedef typename T16<T>::vec4 vec4;
    static_assert(!WKM || MODE != MODE_SWIGLU, "the K-major weight operand is combined with the plain forms only");
    GemmArgs g = g_;
    if (MODE == MODE_F32) {                              // its share of the K-tiles into its own partial
        const int nk = g.K / 64, per = nk / g.split_k, rem = nk % g.split_k, k0 = sp * per + min(sp, rem);
        g.A = (const char*)g.A + (size_t)k0 * 128;
        g.W = (const char*)g.W + (size_t)k0 * (WKM ? (size_t)g.ldw * 128 : (size_t)128);
        g.K = (per + (sp < rem ? 1 : 0)) * 64;
        g.out = (float*)g.out + (size_t)sp * g.split_stride;
    }
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave >> 1, wc = wave & 1, r16 = lane & 15, fq = lane >> 4;
    int tm, tn;
    block_to_tile(bid, g.tiles_m, g.tiles_n, g.group_m, tm, tn);
    const int m0 = tm * RING_TILE, n0 = tn * RING_TILE;

    // DMA: 16 instructions of 1 KiB per operand and K-tile, 4 per wave.  Rows / columns past the matrix repeat the last ones: their outputs are not stored.
    const char* const a_base = (const char*)g.A + (size_t)m0 * g.lda * 2;
    const char* const w_base = WKM ? (const char*)g.W + (size_t)n0 * 2 : (const char*)g.W + (size_t)n0 * g.ldw * 2;
    const size_t w_step = WKM ? (size_t)g.ldw * 128 : (size_t)128;
    unsigned a_off[4], w_off[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int row = (wave * 4 + j) * 8 + (lane >> 3), ch = (lane & 7) ^ ((row >> 1) & 7);
        a_off[j] = ((unsigned)(min(row, g.M - 1 - m0) * g.lda) + (unsigned)(ch * 8)) * 2u;
        if constexpr (WKM) {
            const int k = (wave * 4 + j) * 4 + (lane >> 4), slot = lane & 15;
            const int col = ((((slot >> 1) ^ (((k >> 3) & 1) * 4 + (k & 3))) << 1) + (slot & 1)) * 8;
            w_off[j] = ((unsigned)(k * g.ldw) + (unsigned)min(col, g.N - 8 - n0)) * 2u;
        } else w_off[j] = ((unsigned)(min(row, g.N - 1 - n0) * g.ldw) + (unsigned)(ch * 8)) * 2u;
    }
    auto issue = [&](int kt) {
        char* const st = smem + (kt & (RING_STAGES - 1)) * RING_STAGE + wave * 4096;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            lds_dma16(a_base + (size_t)kt * 128, a_off[j], st + j * 1024);
            lds_dma16(w_base + (size_t)kt * w_step, w_off[j], st + RING_STAGE / 2 + j * 1024);
        }
    };
    // fragment addresses inside a stage
    int a_rd[2], w_rd[WKM ? 4 : 2];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
        const int ch = ((ks * 4 + fq) ^ ((r16 >> 1) & 7)) << 4;
        a_rd[ks] = (wr * 64 + r16) * 128 + ch;
        if constexpr (!WKM) w_rd[ks] = RING_STAGE / 2 + (wc * 64 + r16) * 128 + ch;
    }
    if constexpr (WKM) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w_rd[i] = RING_STAGE / 2 + (fq * 8 + (r16 >> 2)) * 256 + (((wc * 4 + i) ^ ((fq & 1) * 4 + (r16 >> 2))) << 5) + (r16 & 3) * 8;
    }
    auto fragments = [&](int kt, vec8 (&fa)[2][4], vec8 (&fw)[2][4]) {
        const char* const st = smem + (kt & (RING_STAGES - 1)) * RING_STAGE;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (WKM) {
                    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
                    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(st + w_rd[i] + ks * (32 * 256)));
                    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(st + w_rd[i] + ks * (32 * 256) + 4 * 256));
                    fw[ks][i] = bitcast<vec8>(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
                } else fw[ks][i] = *(const vec8*)(st + w_rd[ks] + i * (16 * 128));
                fa[ks][i] = *(const vec8*)(st + a_rd[ks] + i * (16 * 128));
            }
        }
    };
    f32x4 acc[4][4];                                     // [weight tile][row tile]
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int nk = g.K / 64;
    constexpr int PER = 8;                               // DMA instructions per wave and K-tile
    auto landed = [&](int newer) {                       // all but the newest `newer` K-tiles of this wave's DMA have landed
        if (newer >= 3) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(3 * PER) : "memory");
        else if (newer == 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * PER) : "memory");
        else if (newer == 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PER) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    };
    auto barrier = [&]() {                               // nothing moves across it
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    auto multiply = [&](vec8 (&fa)[2][4], vec8 (&fw)[2][4]) {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = T16<T>::mfma16(fw[ks][i], fa[ks][j], acc[i][j]);
    };
    // step t < nk - 1: tile t is in (fa, fw), tile t + 1 goes to (na, nw)
    auto step = [&](int t, vec8 (&fa)[2][4], vec8 (&fw)[2][4], vec8 (&na)[2][4], vec8 (&nw)[2][4]) {
        landed(min(nk - 2 - t, 2));                      // tiles t+2, t+3 may still be in flight
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");          // tile t is in this wave's registers
        barrier();
        if (t + 4 < nk) issue(t + 4);
        fragments(t + 1, na, nw);
        multiply(fa, fw);
    };
#pragma unroll
    for (int t = 0; t < RING_STAGES; ++t)
        if (t < nk) issue(t);
    landed(min(nk - 1, 3));
    barrier();
    {
        vec8 fa0[2][4], fw0[2][4], fa1[2][4], fw1[2][4];
        fragments(0, fa0, fw0);
        int t = 0;
        for (; t + 2 < nk; t += 2) {
            step(t, fa0, fw0, fa1, fw1);
            step(t + 1, fa1, fw1, fa0, fw0);
        }
        if (t + 1 < nk) {
            step(t, fa0, fw0, fa1, fw1);
            multiply(fa1, fw1);
        } else multiply(fa0, fw0);
    }

    const int mw = m0 + wr * 64, nw = n0 + wc * 64;
    if constexpr (MODE == MODE_F32) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int m = mw + j * 16 + r16;
            if (m >= g.M) continue;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int n = nw + i * 16 + fq * 4;
                if (n < g.N) *(f32x4*)((float*)g.out + (size_t)m * g.ldo + n) = acc[i][j];
            }
        }
        return;
    }
    // 16-bit outputs: through a wave-private 8-KiB window (64 rows x 128 B) so that a lane stores 16 B of a row
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    barrier();                                           // every wave is done with the ring
    char* const win = smem + wave * 8192;
    // v(i, j) = the quad of column tile i (of TILES) and row tile j; columns [c0, c0 + 16 TILES) of out, at most `limit`
    auto store = [&](auto tiles_c, auto value, T* out, size_t ldo, int c0, int limit) {
        constexpr int TILES = decltype(tiles_c)::value, CH = TILES * 2, RB = TILES * 32, SH = CH == 4 ? 2 : 1;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < TILES; ++i) {
                const f32x4 v = value(i, j);
                vec4 o;
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = T16<T>::from_f32(v[e]);
                const int row = j * 16 + r16, c = i * 2 + (fq >> 1);
                *(vec4*)(win + row * RB + ((c ^ ((row >> SH) & (CH - 1))) << 4) + (fq & 1) * 8) = o;
            }
        // (the wave reads back what it wrote: LDS operations of one wave complete in order)
#pragma unroll
        for (int k = 0; k < CH; ++k) {
            const int idx = k * 64 + lane, row = idx / CH, c = idx % CH;
            const u32x4 v = *(const u32x4*)(win + row * RB + ((c ^ ((row >> SH) & (CH - 1))) << 4));
            if (mw + row < g.M && c0 + c * 8 < limit) *(u32x4*)(out + (size_t)(mw + row) * ldo + c0 + c * 8) = v;
        }
    };
    if constexpr (MODE == MODE_SWIGLU) {                 // column tiles 0, 1 gate, 2, 3 up ([32 gate | 32 up] weight rows)
        store(std::integral_constant<int, 2>{}, [&](int i, int j) {
            f32x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = silu_f(acc[i][j][e]) * acc[i + 2][j][e];
            return v;
        }, (T*)g.out, (size_t)g.ldo, nw / 2, g.N / 2);
        if (g.gu) store(std::integral_constant<int, 4>{}, [&](int i, int j) { return acc[i][j]; }, (T*)g.gu, (size_t)g.ldgu, nw, g.N);
    } else store(std::integral_constant<int, 4>{}, [&](int i, int j) { return acc[i][j]; }, (T*)g.out, (size_t)g.ldo, nw, g.N);
}

template <typename T, int MODE, bool WKM>
__global__ __launch_bounds__(RING_THREADS, 2) void gemm_ring_kernel(const GemmArgs g) {          // (2: at most 256 registers, no accumulation-file copies)
    extern __shared__ __attribute__((aligned(16))) char smem[];
    ring_tile<T, MODE, WKM>(g, blockIdx.x, blockIdx.y, smem);
}

// two independent products in one launch, both as fp32 partials: a's weight operand is K-major, b's is not
template <typename T>
__global__ __launch_bounds__(RING_THREADS, 2) void gemm_ring_pair_kernel(const GemmArgs a, const GemmArgs b) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int at = a.tiles_m * a.tiles_n, an = at * a.split_k, bt = b.tiles_m * b.tiles_n, id = blockIdx.x;
    if (id < an) ring_tile<T, MODE_F32, true>(a, id % at, id / at, smem);
    else ring_tile<T, MODE_F32, false>(b, (id - an) % bt, (id - an) / bt, smem);
}

constexpr int RING_LDS = RING_STAGES * RING_STAGE;
static void ring_grid(GemmArgs& g) { g.tiles_m = ceil_div(g.M, RING_TILE); g.tiles_n = ceil_div(g.N, RING_TILE); g.group_m = 4; }
template <typename K> static void ring_attribute(K kernel, std::atomic<unsigned>& done_mask) {
    const int dev = current_device();
    if (device_done(done_mask, dev)) return;
    (void)hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, RING_LDS);
    mark_device_done(done_mask, dev);
}

template <typename T, int MODE, bool WKM>
static int launch_ring(GemmArgs g, hipStream_t s) {
    static std::atomic<unsigned> done_mask{0};
    ring_attribute(gemm_ring_kernel<T, MODE, WKM>, done_mask);
    ring_grid(g);
    hipLaunchKernelGGL((gemm_ring_kernel<T, MODE, WKM>), dim3(g.tiles_m * g.tiles_n, MODE == MODE_F32 ? g.split_k : 1), dim3(RING_THREADS), RING_LDS, s, g);
    return (int)hipGetLastError();
}
template <typename T>
static int launch_ring_pair(GemmArgs a, GemmArgs b, hipStream_t s) {
    static std::atomic<unsigned> done_mask{0};
    ring_attribute(gemm_ring_pair_kernel<T>, done_mask);
    ring_grid(a);
    ring_grid(b);
    hipLaunchKernelGGL(gemm_ring_pair_kernel<T>, dim3(a.tiles_m * a.tiles_n * a.split_k + b.tiles_m * b.tiles_n * b.split_k), dim3(RING_THREADS), RING_LDS, s, a, b);
    return (int)hipGetLastError();
}

// mode SWIGLU (g.gu: pre-activations too), STORE16, or F32: raw fp32 partials of g.split_k shares of K, split_stride apart.  N and the leading dimensions
// multiples of 8, K of 64, pointers 16-byte aligned.
int launch_gemm_ring(const GemmArgs& g, int dtype, int mode, bool kmajor, hipStream_t s) {
    auto run = [&](auto t) {
        typedef decltype(t) T;
        if (mode == MODE_SWIGLU) return launch_ring<T, MODE_SWIGLU, false>(g, s);
        if (mode == MODE_F32) return kmajor ? launch_ring<T, MODE_F32, true>(g, s) : launch_ring<T, MODE_F32, false>(g, s);
        return kmajor ? launch_ring<T, MODE_STORE16, true>(g, s) : launch_ring<T, MODE_STORE16, false>(g, s);
    };
    return dtype == DT_BF16 ? run(bf16_t{}) : run(f16_t{});
}
// kmajor (K-major weight operand) and nt (ordinary) in one launch, both mode F32
int launch_gemm_ring_pair(const GemmArgs& kmajor, const GemmArgs& nt, int dtype, hipStream_t s) {
    return dtype == DT_BF16 ? launch_ring_pair<bf16_t>(kmajor, nt, s) : launch_ring_pair<f16_t>(kmajor, nt, s);
}

}  // namespace vitg
