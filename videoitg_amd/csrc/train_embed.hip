// Token embedding for training: lookup with a scale, and the gradient of the table.
//
//   out[i, :]      = scale * E[ids[i], :]                    ids outside [0, vocab): a zero row (image slots carry -200 in this framework, padding -1)
//   dE[v, :]  (+)= scale * sum over {i : ids[i] = v} of dout[i, :]
//
// The gradient sorts the tokens by id (stable: equal ids keep their order), cuts the sorted list into chunks of `chunk` tokens and lets a block sum the
// rows of one chunk: a run of equal ids that lies inside one chunk is finished there; a run that crosses chunks leaves fp32 partials, which a second
// kernel adds in chunk order.  No floating-point atomics: the order of every sum depends on the ids alone, so a repeated call gives the same bits.
//
// Measured at D = 3584 (a copy of 1 GiB runs at 5.1 TB/s here):
//   lookup     20 480 tokens (14 500 different), bf16: 49 us, 251 MB of rows, HBM; 60 tokens: 7 us, the call itself
//   gradient   5 003 tokens (3 060 different, one of them a third of the list) added to an fp32 table: sort 11 us, sums 27 us (157 MB, HBM), joins 7 us
//              20 480 tokens, dense bf16 table of 152 064 rows: 210 us of sort and zeroing (1.09 GB written, 5.2 TB/s), sums 42 us (246 MB), joins 7 us
#include "train_common.h"

namespace vitg {

// ---- lookup ------------------------------------------------------------------------------------------------------------------
template <typename TI, typename TO, int V>
__global__ void embed_lookup_kernel(const long long* __restrict__ ids, long n, const TI* __restrict__ table, long ldt, long vocab, int cv, float scale,
                                    TO* __restrict__ out, long ldo) {
    for (long row = (long)blockIdx.x * blockDim.y + threadIdx.y; row < n; row += (long)gridDim.x * blockDim.y) {
        const long long id = ids[row];
        const bool known = id >= 0 && id < vocab;
        for (int c = threadIdx.x; c < cv; c += blockDim.x) {
            float v[V];
            if (known) {
                load_vec<TI, V>(table + id * ldt + (long)c * V, v);
#pragma unroll
                for (int e = 0; e < V; ++e) v[e] *= scale;
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) v[e] = 0.f;
            }
            store_vec<TO, V>(out + row * ldo + (long)c * V, v);
        }
    }
}
constexpr long LOOKUP_BLOCKS = 1l << 20;                 // (a launch has fewer than 2^32 threads)

// ---- stable sort of (key, position); key = id, or vocab for a slot without a token (sorts behind every id) ------------------------
// The dense form also has to zero every row of the table (the rows of the batch's tokens are overwritten by the sums): a write of the whole table, which
// keeps HBM busy while the sort uses a few CUs.  So the zeroing rides along: each sort launch carries extra blocks behind its own that zero a share of the rows.
struct ZeroRows { void* table; long pitch, bytes, begin, end; int blocks; };      // rows [begin, end), `bytes` of every `pitch`, by the last `blocks` of the grid
// AROUND (the radix passes): non-temporal stores, which leave no dirty lines for the sums behind them to write back: 20 480 tokens of 3584 bf16 into 1 000 / 17 000 /
// 152 064 rows take 70 / 92 / 266 us against 70 / 101 / 286, and with a pass that reads the table behind them 78 / 121 / 485 against 78 / 128 / 499.  The short
// lists' single launch is over before HBM has taken that much, and the ordinary form wins there: 5 000 tokens, 17 000 rows 36 us against 42 (59 against 67 with the reader).
template <bool AROUND> __device__ __forceinline__ void zero_rows(const ZeroRows& z, int block) {
    auto run = [&](auto zero) {
        typedef decltype(zero) Z;
        for (long r = z.begin + block; r < z.end; r += z.blocks)
            for (long c = threadIdx.x * (long)sizeof(Z); c < z.bytes; c += blockDim.x * (long)sizeof(Z)) {
                Z* const p = (Z*)((char*)z.table + r * z.pitch + c);
                if constexpr (AROUND) __builtin_nontemporal_store(zero, p); else *p = zero;
            }
    };
    if ((z.pitch | z.bytes | (long)(uintptr_t)z.table) & 15) run(u32x2{0, 0}); else run(u32x4{0, 0, 0, 0});
}
__global__ __launch_bounds__(256) void zero_rows_kernel(const ZeroRows z) { zero_rows<true>(z, blockIdx.x); }

constexpr int SORT_BITS = 9, SORT_BINS = 1 << SORT_BITS, SORT_TILE = 2048, SORT_THREADS = 256;

__device__ __forceinline__ unsigned sort_key(long long id, unsigned vocab) { return id >= 0 && id < (long long)vocab ? (unsigned)id : vocab; }

// Short lists (n <= RANK_MAX): a token's place is the number of smaller keys plus the number of equal keys in front of it, counted against all keys in LDS.
// 64 tokens per block, its 16 waves count a sixteenth of the list each.  n^2 comparisons, two instructions each, on n / 64 blocks - and one launch.
// Added to a table (us, with the sums; ids spread / all equal) against the radix passes: 500 tokens 17 / 15 against 30 / 28, 5 000: 36 / 29 against 49 / 43,
// 15 360: 83 / 72 against 86 / 75 - about equal where the keys fill 60 KiB.
constexpr int RANK_MAX = 15360, RANK_WAVES = 16;
__global__ __launch_bounds__(RANK_WAVES * 64) void sort_rank_kernel(const long long* __restrict__ ids, int n, unsigned vocab, unsigned* __restrict__ key_out,
                                                                    unsigned* __restrict__ pos_out, int blocks, const ZeroRows z) {
    extern __shared__ __attribute__((aligned(16))) unsigned keys[];      // n keys, padded to a multiple of 16 with the largest value
    if ((int)blockIdx.x >= blocks) { zero_rows<false>(z, (int)blockIdx.x - blocks); return; }
    __shared__ unsigned part[64];
    const int padded = (n + 15) & ~15;
#pragma unroll 4
    for (int i = threadIdx.x; i < padded; i += RANK_WAVES * 64) keys[i] = i < n ? sort_key(ids[i], vocab) : 0xffffffffu;
    if (threadIdx.x < 64) part[threadIdx.x] = 0;
    __syncthreads();
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int i0 = blockIdx.x * 64, i = i0 + lane;
    const unsigned mine = keys[min(i, n - 1)];
    const int per = (padded / 16 + RANK_WAVES - 1) / RANK_WAVES * 16, lo = min(wave * per, padded), hi = min(lo + per, padded);
    unsigned count = 0;
    auto span = [&](int a, int b, auto f) {              // [a, b) of this wave's share; all bounds are multiples of 16
        for (int j = max(a, lo); j < min(b, hi); j += 16) {
            u32x4 k[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) k[u] = *(const u32x4*)(keys + j + u * 4);
#pragma unroll
            for (int e = 0; e < 16; ++e) count += f(k[e >> 2][e & 3], j + e) ? 1u : 0u;
        }
    };
    span(0, i0, [&](unsigned k, int) { return k <= mine; });
    span(i0, min(i0 + 64, padded), [&](unsigned k, int j) { return k < mine || (k == mine && j < i); });
    span(i0 + 64, padded, [&](unsigned k, int) { return k < mine; });
    atomicAdd(&part[lane], count);                       // whole numbers: the order does not matter
    __syncthreads();
    if (wave == 0 && i < n) {
        const unsigned at = part[lane];
        key_out[at] = mine;
        pos_out[at] = (unsigned)i;
    }
}

// Longer lists: radix passes, least significant digit first.  One pass = two launches: digit counts per tile of 2048 keys, then every tile scatters its keys behind the counts of the smaller
// digits and of the tiles in front of it.  FIRST: the keys are the ids themselves, the positions 0 .. n-1.
template <bool FIRST>
__global__ __launch_bounds__(SORT_THREADS) void sort_count_kernel(const long long* __restrict__ ids, const unsigned* __restrict__ key_in, long n, unsigned vocab,
                                                                  int shift, unsigned* __restrict__ counts, int tiles, const ZeroRows z) {
    if ((int)blockIdx.x >= tiles) { zero_rows<true>(z, (int)blockIdx.x - tiles); return; }
    __shared__ unsigned bins[SORT_BINS];
    for (int b = threadIdx.x; b < SORT_BINS; b += SORT_THREADS) bins[b] = 0;
    __syncthreads();
    const long base = (long)blockIdx.x * SORT_TILE;
    for (int k = threadIdx.x; k < SORT_TILE; k += SORT_THREADS) {
        const long i = base + k;
        if (i < n) atomicAdd(&bins[((FIRST ? sort_key(ids[i], vocab) : key_in[i]) >> shift) & (SORT_BINS - 1)], 1u);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < SORT_BINS; b += SORT_THREADS) counts[(size_t)blockIdx.x * SORT_BINS + b] = bins[b];
}

template <bool FIRST>
__global__ __launch_bounds__(SORT_THREADS) void sort_scatter_kernel(const long long* __restrict__ ids, const unsigned* __restrict__ key_in,
                                                                    const unsigned* __restrict__ pos_in, long n, unsigned vocab, int shift, int tiles,
                                                                    const unsigned* __restrict__ counts, unsigned* __restrict__ key_out, unsigned* __restrict__ pos_out,
                                                                    const ZeroRows z) {
    if ((int)blockIdx.x >= tiles) { zero_rows<true>(z, (int)blockIdx.x - tiles); return; }
    constexpr int WAVES = SORT_THREADS / 64, ROUNDS = SORT_TILE / SORT_THREADS, BPT = SORT_BINS / SORT_THREADS;
    __shared__ unsigned next[WAVES][SORT_BINS];          // next free slot of a digit for one wave's keys
    __shared__ unsigned wave_total[WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // thread t owns digits BPT t ..: keys with that digit in all tiles, and in the tiles in front of this one
    unsigned total[BPT], before[BPT], mine = 0;
#pragma unroll
    for (int d = 0; d < BPT; ++d) {
        total[d] = before[d] = 0;
        for (int t = 0; t < tiles; ++t) {
            const unsigned c = counts[(size_t)t * SORT_BINS + tid * BPT + d];
            total[d] += c;
            if (t < (int)blockIdx.x) before[d] += c;
        }
        mine += total[d];
    }
    unsigned scan = mine;                                // exclusive prefix over the threads (= over the digits)
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) { const unsigned up = __shfl_up(scan, o, 64); if (lane >= o) scan += up; }
    if (lane == 63) wave_total[wave] = scan;
    for (int b = tid; b < WAVES * SORT_BINS; b += SORT_THREADS) (&next[0][0])[b] = 0;
    __syncthreads();
    unsigned first = scan - mine;
    for (int w = 0; w < wave; ++w) first += wave_total[w];
    // this wave's keys: 64 consecutive ones per round, ROUNDS rounds; counts per digit
    unsigned key[ROUNDS], pos[ROUNDS];
    const long base = (long)blockIdx.x * SORT_TILE + wave * (ROUNDS * 64) + lane;
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const long i = base + r * 64;
        key[r] = 0; pos[r] = 0;
        if (i < n) {
            key[r] = FIRST ? sort_key(ids[i], vocab) : key_in[i];
            pos[r] = FIRST ? (unsigned)i : pos_in[i];
            atomicAdd(&next[wave][(key[r] >> shift) & (SORT_BINS - 1)], 1u);
        }
    }
    __syncthreads();
    // counts -> first slot: digits below, tiles in front, waves in front
#pragma unroll
    for (int d = 0; d < BPT; ++d) {
        unsigned at = first + before[d];
        first += total[d];
#pragma unroll
        for (int w = 0; w < WAVES; ++w) { const unsigned c = next[w][tid * BPT + d]; next[w][tid * BPT + d] = at; at += c; }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const bool live = base + r * 64 < n;
        const unsigned digit = (key[r] >> shift) & (SORT_BINS - 1);
        unsigned long long same = __ballot(live);        // lanes of this round with the same digit
#pragma unroll
        for (int b = 0; b < SORT_BITS; ++b) {
            const unsigned long long m = __ballot((digit >> b) & 1u);
            same &= ((digit >> b) & 1u) ? m : ~m;
        }
        const unsigned rank = __popcll(same & ((1ull << lane) - 1ull));
        // (one wave's LDS operations complete in order: every lane has read the slot before the first lane of its digit moves it on)
        volatile unsigned* const slot = &next[wave][digit];
        unsigned at = 0;
        if (live) at = *slot + rank;
        __builtin_amdgcn_wave_barrier();
        if (live && rank == 0) *slot = at + __popcll(same);
        __builtin_amdgcn_wave_barrier();
        if (live) { key_out[at] = key[r]; pos_out[at] = pos[r]; }
    }
}

// ---- the sums ----------------------------------------------------------------------------------------------------------------------
template <typename TT, int V>
__device__ __forceinline__ void finish_row(TT* __restrict__ row, int accumulate, float scale, const float (&acc)[V]) {
    float v[V];
    if (accumulate) load_vec<TT, V>(row, v);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = accumulate ? v[e] + scale * acc[e] : scale * acc[e];
    store_vec<TT, V>(row, v);
}

// partials: [chunk][2][cv * V] fp32 - slot 0: a run that began in an earlier chunk, slot 1: a run that begins here and goes on behind it
template <typename TD, typename TT, int V>
__global__ __launch_bounds__(256) void embed_grad_kernel(const unsigned* __restrict__ key, const unsigned* __restrict__ pos, long n, unsigned vocab, int chunk,
                                                         const TD* __restrict__ dout, long ldd, int cv, float scale, TT* __restrict__ table, long ldt,
                                                         int accumulate, float* __restrict__ partial) {
    const int c = blockIdx.y * 256 + threadIdx.x;
    if (c >= cv) return;
    const long e0 = (long)blockIdx.x * chunk, e1 = min(e0 + chunk, n);
    unsigned run = key[e0];
    if (run >= vocab) return;                            // nothing but slots without a token from here on
    bool began = e0 == 0 || key[e0 - 1] != run;
    float acc[V];
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.f;
    constexpr int G = 4;                                 // rows in flight
    for (long e4 = e0; e4 < e1; e4 += G) {
        float v[G][V];
        unsigned after[G];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const long e = min(e4 + g, e1 - 1);
            load_vec<TD, V>(dout + (long)pos[e] * ldd + (long)c * V, v[g]);
            after[g] = e + 1 < n ? key[e + 1] : vocab;
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            if (e4 + g >= e1) break;
#pragma unroll
            for (int k = 0; k < V; ++k) acc[k] += v[g][k];
            if (after[g] != run) {                       // the run ends with this token
                if (began) finish_row<TT, V>(table + (long)run * ldt + (long)c * V, accumulate, scale, acc);
                else store_vec<float, V>(partial + ((size_t)blockIdx.x * 2) * ((size_t)cv * V) + (size_t)c * V, acc);
                if (after[g] >= vocab || e4 + g + 1 == e1) return;      // no token is left, or the next run starts the next chunk
                run = after[g];
                began = true;
#pragma unroll
                for (int k = 0; k < V; ++k) acc[k] = 0.f;
            }
        }
    }
    // the run goes on in the next chunk
    store_vec<float, V>(partial + ((size_t)blockIdx.x * 2 + (began ? 1 : 0)) * ((size_t)cv * V) + (size_t)c * V, acc);
}

// runs across chunks: the partials of a run are added in chunk order by the wave (short lists) or the block (long ones) of the chunk in which it begins.  A block
// looks at 16 chunks, one per wave, and JOIN_COLS columns; a long list is cut into eight consecutive parts whose sums join through LDS in order.
constexpr int JOIN_PARTS = 8, JOIN_COLS = 512, JOIN_SHORT = 8;
template <typename TT>
__global__ __launch_bounds__(1024) void embed_join_kernel(const unsigned* __restrict__ key, long n, unsigned vocab, int chunk, int D, float scale,
                                                          TT* __restrict__ table, long ldt, int accumulate, const float* __restrict__ partial) {
    constexpr int V = 4;
    __shared__ float part[JOIN_PARTS][JOIN_COLS];
    __shared__ int items_of[16];
    const long chunks = (n + chunk - 1) / chunk;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, p = wave >> 1, c0 = blockIdx.y * JOIN_COLS;
    // item i of the run that begins in chunk b: the part that chunk b + i holds (slot 1 of the first, slot 0 of the others)
    auto item = [&](long b, long i, int c) { return partial + ((size_t)(b + i) * 2 + (i == 0 ? 1 : 0)) * (size_t)D + c; };
    auto add = [&](long b, long i0, long i1, int c, float (&acc)[V]) {
        for (long i = i0; i < i1; i += 8) {              // eight in flight; past the end the last one again, left out of the sum
            float v[8][V];
#pragma unroll
            for (int g = 0; g < 8; ++g) load_vec<float, V>(item(b, min(i + g, i1 - 1), c), v[g]);
#pragma unroll
            for (int g = 0; g < 8; ++g)
                if (i + g < i1)
#pragma unroll
                    for (int k = 0; k < V; ++k) acc[k] += v[g][k];
        }
    };
    const long mine = blockIdx.x * 16l + wave;
    int items = 0;                                       // parts of the run that begins in this wave's chunk and goes on behind it
    if (mine + 1 < chunks) {
        const unsigned run = key[(mine + 1) * chunk - 1];
        if (run < vocab && key[(mine + 1) * chunk] == run && !(mine > 0 && key[mine * chunk - 1] == run)) {
            items = 2;
            for (;;) {                                   // 64 chunks at a time: does the run reach into them
                const long j = mine + items + lane;
                const unsigned long long in = __ballot(j < chunks && key[min(j, chunks - 1) * chunk] == run);
                const int more = in == ~0ull ? 64 : __ffsll((unsigned long long)~in) - 1;
                items += more;
                if (more < 64) break;
            }
            if (items <= JOIN_SHORT)
                for (int c = c0 + lane * V; c < min(c0 + JOIN_COLS, D); c += 64 * V) {
                    float acc[V] = {0.f, 0.f, 0.f, 0.f};
                    add(mine, 0, items, c, acc);
                    finish_row<TT, V>(table + (long)run * ldt + c, accumulate, scale, acc);
                }
        }
    }
    if (lane == 0) items_of[wave] = items;
    __syncthreads();
    for (int w = 0; w < 16; ++w) {
        const int count = items_of[w];                   // (the same for every thread of the block)
        if (count <= JOIN_SHORT) continue;
        const long b = blockIdx.x * 16l + w;
        const int at = (wave & 1) * 256 + lane * V, c = c0 + at, per = (count + JOIN_PARTS - 1) / JOIN_PARTS;
        float acc[V] = {0.f, 0.f, 0.f, 0.f};
        if (c < D) add(b, p * per, min((p + 1) * per, count), c, acc);
        store_vec<float, V>(&part[p][at], acc);
        __syncthreads();
        if (p == 0 && c < D) {
            for (int q = 1; q < JOIN_PARTS; ++q)
#pragma unroll
                for (int k = 0; k < V; ++k) acc[k] += part[q][at + k];
            finish_row<TT, V>(table + (long)key[(b + 1) * chunk - 1] * ldt + c, accumulate, scale, acc);
        }
        __syncthreads();
    }
}

// Tokens per call: every tile of a radix pass reads the counts of all tiles, so a pass grows with the square of the list (2^24 tokens: 8 192 tiles, 137 GB of counts
// out of the caches).  Longer lists are added up over several calls with accumulate = 1.
constexpr long EMBED_TOKENS = 1l << 24;
// tokens per chunk: short chunks spread a short list over the CUs, long ones leave fewer partials to join.  bf16 rows of 3584 added to the table (us; ids spread over
// 150 000 rows / all equal), 16 - 32 - 64 tokens a chunk: 5 000 tokens 36 / 29 - 43 / 28; 10 000: 57 / 52 - 58 / 42; 20 480: 112 / 91 - 106 / 74 - 127 / 65;
// 32 768: 178 / 124 (32) - 179 / 89 (64); 131 072: 575 / 880 - 553 / 588 - 545 / 416
static int embed_chunk(long n) { return n >= 32768 ? 64 : n >= 8192 ? 32 : 16; }
static size_t round256(size_t b) { return (b + 255) & ~(size_t)255; }

struct EmbedWorkspace { size_t key[2], pos[2], counts, partial, bytes; int tiles, chunk; long chunks; };
static EmbedWorkspace embed_workspace(long n, int D) {
    EmbedWorkspace w = {};
    w.tiles = (int)((n + SORT_TILE - 1) / SORT_TILE);
    w.chunk = embed_chunk(n);
    w.chunks = (n + w.chunk - 1) / w.chunk;
    size_t at = 0;
    for (int i = 0; i < 2; ++i) { w.key[i] = at; at += round256((size_t)n * 4); w.pos[i] = at; at += round256((size_t)n * 4); }
    if (n > RANK_MAX) { w.counts = at; at += round256((size_t)w.tiles * SORT_BINS * 4); }
    w.partial = at; at += round256((size_t)w.chunks * 2 * D * 4);
    w.bytes = at;
    return w;
}

}  // namespace vitg

using namespace vitg;

extern "C" int vitg_embed_lookup(const long long* ids, long n, const void* table, int table_dtype, long ldt, long vocab, int D, float scale, void* out,
                                 int out_dtype, long ldo, void* stream) {
    if (n <= 0) return 0;
    if (!ids || !table || !out) return VITG_ERR_ARG;
    if (!dtype_ok(table_dtype) || !dtype_ok(out_dtype)) return VITG_ERR_DTYPE;
    if (vocab <= 0 || D <= 0 || n >= (1l << 31) || ldt < D || ldo < D) return VITG_ERR_SHAPE;
    if (D % 4 || ldt % 4 || ldo % 4 || !aligned_to(table, 4 * dtype_size(table_dtype)) || !aligned_to(out, 4 * dtype_size(out_dtype))) return VITG_ERR_ALIGN;
    const bool wide = D % 8 == 0 && ldt % 8 == 0 && ldo % 8 == 0 && aligned_to(table, 16) && aligned_to(out, 16);
    const int cv = D / (wide ? 8 : 4);
    const int tx = cv >= 512 ? 512 : (cv + 63) / 64 * 64, ty = tx >= 256 ? 1 : 256 / tx;
    const long blocks = (n + ty - 1) / ty;
    const dim3 grid((unsigned)(blocks < LOOKUP_BLOCKS ? blocks : LOOKUP_BLOCKS)), block(tx, ty);
    with_dtype(table_dtype, [&](auto ti) {
        typedef decltype(ti) TI;
        with_dtype(out_dtype, [&](auto to) {
            typedef decltype(to) TO;
            if (wide) hipLaunchKernelGGL((embed_lookup_kernel<TI, TO, 8>), grid, block, 0, (hipStream_t)stream, ids, n, (const TI*)table, ldt, vocab, cv, scale, (TO*)out, ldo);
            else hipLaunchKernelGGL((embed_lookup_kernel<TI, TO, 4>), grid, block, 0, (hipStream_t)stream, ids, n, (const TI*)table, ldt, vocab, cv, scale, (TO*)out, ldo);
        });
    });
    return launched();
}

extern "C" int vitg_embed_backward_plan(long n, int D, long* workspace_bytes) {
    if (!workspace_bytes) return VITG_ERR_ARG;
    if (n < 0 || n > EMBED_TOKENS || D <= 0) return VITG_ERR_SHAPE;
    *workspace_bytes = n ? (long)embed_workspace(n, D).bytes : 0;
    return 0;
}

extern "C" int vitg_embed_backward(const long long* ids, long n, const void* dout, int dout_dtype, long ldd, long vocab, int D, float scale, void* dtable,
                                   int table_dtype, long ldt, int accumulate, void* workspace, long workspace_bytes, void* stream) {
    if (n < 0 || vocab <= 0 || D <= 0 || n > EMBED_TOKENS || vocab >= (1l << 31) - 1 || ldt < D) return VITG_ERR_SHAPE;
    if (!dtable || (n && (!ids || !dout || !workspace))) return VITG_ERR_ARG;
    if (!dtype_ok(table_dtype) || !dtype_ok(dout_dtype)) return VITG_ERR_DTYPE;
    if (n && ldd < D) return VITG_ERR_SHAPE;
    if (D % 4 || ldt % 4 || (n && ldd % 4) || !aligned_to(dtable, 4 * dtype_size(table_dtype)) || (n && !aligned_to(dout, 4 * dtype_size(dout_dtype)))) return VITG_ERR_ALIGN;
    const EmbedWorkspace w = n ? embed_workspace(n, D) : EmbedWorkspace{};
    if (n && (workspace_bytes < (long)w.bytes || !aligned_to(workspace, 16))) return VITG_ERR_ARG;
    hipStream_t s = (hipStream_t)stream;
    const int tsize = dtype_size(table_dtype);
    if (n == 0) {
        const ZeroRows z = {dtable, ldt * tsize, (long)D * tsize, 0, vocab, 2048};
        if (!accumulate) hipLaunchKernelGGL(zero_rows_kernel, dim3(2048), dim3(256), 0, s, z);
        return launched();
    }
    char* const base = (char*)workspace;
    unsigned *key[2], *pos[2], *counts = (unsigned*)(base + w.counts);
    for (int i = 0; i < 2; ++i) { key[i] = (unsigned*)(base + w.key[i]); pos[i] = (unsigned*)(base + w.pos[i]); }
    float* const partial = (float*)(base + w.partial);
    int bits = 1;
    while ((vocab >> bits) != 0) ++bits;                 // keys 0 .. vocab
    const unsigned v = (unsigned)vocab;
    // launch i of the sort zeroes rows [i vocab / launches, (i + 1) vocab / launches)
    const int passes = (bits + SORT_BITS - 1) / SORT_BITS, launches = n <= RANK_MAX ? 1 : 2 * passes;
    auto zero = [&](int i) {
        ZeroRows z = {dtable, ldt * tsize, (long)D * tsize, vocab * i / launches, vocab * (i + 1) / launches, 0};
        if (!accumulate) z.blocks = (int)(z.end - z.begin < 2048 ? z.end - z.begin : 2048);
        return z;
    };
    int cur = 0;
    if (launches == 1) {
        const int blocks = (int)((n + 63) / 64);
        const ZeroRows z = zero(0);
        hipLaunchKernelGGL(sort_rank_kernel, dim3(blocks + z.blocks), dim3(RANK_WAVES * 64), (size_t)((n + 15) & ~15l) * 4, s, ids, (int)n, v, key[0], pos[0], blocks, z);
    } else
        for (int p = 0; p < passes; ++p) {
            const int to = cur ^ 1, shift = p * SORT_BITS;
            const ZeroRows z0 = zero(2 * p), z1 = zero(2 * p + 1);
            const dim3 g0(w.tiles + z0.blocks), g1(w.tiles + z1.blocks), t(SORT_THREADS);
            if (p == 0) {
                hipLaunchKernelGGL(sort_count_kernel<true>, g0, t, 0, s, ids, nullptr, n, v, shift, counts, w.tiles, z0);
                hipLaunchKernelGGL(sort_scatter_kernel<true>, g1, t, 0, s, ids, nullptr, nullptr, n, v, shift, w.tiles, counts, key[to], pos[to], z1);
            } else {
                hipLaunchKernelGGL(sort_count_kernel<false>, g0, t, 0, s, nullptr, key[cur], n, v, shift, counts, w.tiles, z0);
                hipLaunchKernelGGL(sort_scatter_kernel<false>, g1, t, 0, s, nullptr, key[cur], pos[cur], n, v, shift, w.tiles, counts, key[to], pos[to], z1);
            }
            cur = to;
        }
    const bool wide = D % 8 == 0 && ldt % 8 == 0 && ldd % 8 == 0 && aligned_to(dtable, 16) && aligned_to(dout, 16);
    const int cv = D / (wide ? 8 : 4);
    with_dtype(dout_dtype, [&](auto td) {
        typedef decltype(td) TD;
        with_dtype(table_dtype, [&](auto tt) {
            typedef decltype(tt) TT;
            const dim3 grid((unsigned)w.chunks, ceil_div(cv, 256));
            if (wide) hipLaunchKernelGGL((embed_grad_kernel<TD, TT, 8>), grid, dim3(256), 0, s, key[cur], pos[cur], n, v, w.chunk, (const TD*)dout, ldd, cv, scale, (TT*)dtable, ldt, accumulate, partial);
            else hipLaunchKernelGGL((embed_grad_kernel<TD, TT, 4>), grid, dim3(256), 0, s, key[cur], pos[cur], n, v, w.chunk, (const TD*)dout, ldd, cv, scale, (TT*)dtable, ldt, accumulate, partial);
        });
    });
    if (w.chunks > 1)
        with_dtype(table_dtype, [&](auto tt) {
            typedef decltype(tt) TT;
            hipLaunchKernelGGL((embed_join_kernel<TT>), dim3((unsigned)((w.chunks + 15) / 16), ceil_div(D, JOIN_COLS)), dim3(1024), 0, s, key[cur], n, v, w.chunk, D, scale, (TT*)dtable, ldt, accumulate, partial);
        });
    return launched();
}
