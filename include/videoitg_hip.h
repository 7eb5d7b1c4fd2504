/* videoitg_hip.h — C ABI of libvideoitg_hip.so, the gfx950 (MI355X) kernels under the VideoITG frame-selector
 * forward.
 *
 * The reference (NVlabs/VideoITG) has no native/FFI boundary of its own: it is pure Python and every arithmetic
 * op on this path executes inside third-party CUDA wheels.  Each entry point below therefore
 * cites the reference call site whose third-party kernel(s) it replaces.  All pointers are DEVICE pointers
 * (HBM) unless noted, sizes are plain ints, `stream` is a hipStream_t passed as void* (NULL = default stream);
 * every call is asynchronous on that stream, performs no allocation and no host synchronisation.
 * Return value: 0 on success, a negative VITG_ERR_* otherwise (nothing is launched on error).
 *
 * dtype codes: VITG_BF16 / VITG_F16 select the 16-bit storage type of activations and weights
 * (MFMA inputs); accumulation, residual stream, norm/softmax statistics are always fp32.
 */
#ifndef VIDEOITG_HIP_H
#define VIDEOITG_HIP_H

#ifdef __cplusplus
extern "C" {
#endif

#define VITG_BF16 0
#define VITG_F16 1
#define VITG_F32 2

#define VITG_ACT_NONE 0
#define VITG_ACT_GELU_TANH 1 /* SigLIP MLP: gelu_pytorch_tanh */
#define VITG_ACT_GELU_ERF 2  /* projector: nn.GELU() exact erf (mlp_proj.py:33) */

#define VITG_GEMM_STORE16 0 /* out16[m,n] = act(acc + bias) */
#define VITG_GEMM_F32 1     /* outf32[m,n] = act(acc + bias) + res[(m % res_mod), n]   (residual stream update) */
#define VITG_GEMM_SWIGLU 2  /* W rows interleaved [32 gate | 32 up]...: out16[m, n/2] = silu(gate) * up */

#define VITG_ERR_SHAPE (-1)
#define VITG_ERR_ALIGN (-2)
#define VITG_ERR_DTYPE (-3)
#define VITG_ERR_ARG (-4)
#define VITG_ERR_LAUNCH (-5)

/* Library / device identification.  vitg_version() needs no GPU. */
int vitg_version(void);
/* Fills name (<= name_len bytes, NUL terminated) with the gcnArchName of the current device and returns the
 * compute-unit count, or a negative error when no HIP device is usable. */
int vitg_device_info(char* name, int name_len);

/* Kernel-set selection for cross-check tests; 0 = the measured default everywhere.  FOUR keys, each a choice between the default and one
 * cross-check kernel set; the same values can come from the environment (VITG_<KEY IN CAPS>, read once).  Host-only, no GPU needed.
 *   gemm_tile   128  every GEMM on the 128x128 register-staged kernels (csrc/gemm.hip) | 256  never the 128-tile kernel where a 256-wide one applies
 *   gemm_cfg    2 | 6 | 9 | 10 | 12  force ONE shipped 256-wide tile shape (256x128x32 | 256x256x64 | 256x384x64 | 384x256x64 | 320x256x64) instead of the
 *               per-shape choice (csrc/gemm256.hip: choose_cfg) - lets a test reach every shipped kernel on a small shape (12 exists for the SwiGLU and
 *               fp32-residual GEMMs; other modes run 256x256 under it)
 *   attn_ab     2  head dim 72 on the per-tile kernel (csrc/attention.hip) instead of the half-tile-out-of-phase one (csrc/attention_ab.hip)
 *   attn_sp     2  head dim 128 on the per-tile kernel (csrc/attention.hip) instead of the 8-wave software-pipelined one (csrc/attention_sp.hip)
 *               (the one-wave-per-SIMD kernel of round 5, csrc/attention_w4.hip - +5 % in isolation, -4 % inside the step - lost its A/B where it runs
 *               and lives in the profiling library since round 6: attn_sp = 4 there)
 * Any other key or value returns VITG_ERR_ARG.  These are process-global test hooks: set them before the forward they should apply to, not from a
 * second thread while one runs.  tests/test_gpu_e2e.py::test_full_size_invariants runs the same video through (gemm_tile 128, attn_ab 2, attn_sp 2)
 * and through the defaults.
 * Everything that was an A/B switch in rounds 1-3 (gemm_flags, gemm_group, gemm_mi, gemm_mi_modes, gemm_pref, gemm_wm4, gemm_stagger, attn_waves,
 * attn_dma, attn_pipe, the other values of the four keys above) and every kernel variant that lost its A/B (32x32x16 wide tiles, 4 x 2 wave grid,
 * stream-K, hd-72 cross-tile / software-pipelined loops, 16-wave blocks, PV on 32x32x16, VALU row sums, hd-128 PV on 16x16x32, the round-1 research
 * configurations, the ablation switches that produce WRONG results by design) lives in libvideoitg_hip_prof.so only (build.sh --profiling,
 * include/videoitg_hip_profiling.h), which tools/ load and the product never does. */
int vitg_set_option(const char* key, int value);

/* A0[T*G*G, Kpad] (16-bit) = im2col of pixel_values [T,3,R,R] NCHW (pix_dtype VITG_F32/F16/BF16), k ordered
 * (c,ky,kx) like the conv weight [Dv,3,p,p] flattened, zero for k >= 3*p*p.
 * Replaces the unfold half of [3P] SiglipVisionEmbeddings.patch_embedding (cuDNN conv2d), reached from
 * /root/reference/eagle/model/multimodal_encoder/clip_encoder.py:146,151. */
int vitg_patchify(const void* pix, int pix_dtype, void* out, int T, int R, int patch, int Kpad, int dtype,
                  void* stream);

/* C = A[M,K] . W[N,K]^T with fused epilogue (mode VITG_GEMM_*).  A, W 16-bit row-major with leading dims
 * lda/ldw (elements, multiples of 8); K a multiple of 64 (callers zero-pad); bias fp32 [N] or NULL.
 * Replaces every cuBLAS GEMM of the path: SigLIP patch-embed/q/k/v/out/fc1/fc2 ([3P] modeling_siglip via
 * clip_encoder.py:146), projector Linear x2 (/root/reference/eagle/model/multimodal_projector/mlp_proj.py:31-35,72),
 * Qwen2 q/k/v/o/gate/up/down ([3P] modeling_qwen2 via
 * /root/reference/eagle/model/language_model/grounding_qwen2.py:135), including the bias add, GELU / SiLU*mul
 * activation and residual add that the reference runs as separate elementwise kernels. */
int vitg_gemm(const void* A, int lda, const void* W, int ldw, int M, int N, int K, int dtype, int mode,
              const float* bias, int act, void* out, int ldo, const float* res, int ldr, int res_mod,
              void* stream);

/* 16-bit residual stream (round 3).  The reference runs model.half() (/root/reference/eagle/model/builder.py:59, infer.py:21): its
 * residual adds happen on fp16 tensors.  vitg_gemm keeps the stream in fp32 (mode VITG_GEMM_F32); these three entry points run the
 * SigLIP tower's stream in the MFMA input type instead - half the bytes of every LayerNorm read, out-proj / fc2 read-modify-write -
 * with fp32 accumulation inside the epilogue and ONE rounding per residual update:
 *   vitg_gemm_res16:      out16[m,n] = round16( sum_k A[m,k] W[n,k] + bias[n] + res16[m,n] + res32[m % res_mod, n] )
 *                         res16 (16-bit, ld ldr16, may alias out) or res32 (fp32 table, e.g. the position embedding with res_mod = tokens
 *                         per frame) or neither.  Same call sites as vitg_gemm: SigLIP patch-embed (+ position table), out_proj, fc2.
 *   vitg_layernorm16:     LayerNorm of 16-bit rows -> 16-bit rows (same type), fp32 statistics; D, ldx, ldo multiples of 8.
 *   vitg_bilinear_pool16: vitg_bilinear_pool on 16-bit features.
 * The decoder's stream stays fp32 (12 860 rows: its norm traffic is 0.4 % of a step, and the 28-layer bidirectional stack is the
 * precision-sensitive part, profiles/r02_parity.md). */
int vitg_gemm_res16(const void* A, int lda, const void* W, int ldw, int M, int N, int K, int dtype, const float* bias, void* out,
                    int ldo, const void* res16, int ldr16, const float* res32, int ldr32, int res_mod, void* stream);
int vitg_layernorm16(const void* x, int ldx, const float* w, const float* b, void* out, int ldo, int dtype, long M, int D, float eps,
                     void* stream);

/* Patch embedding with the im2col INSIDE the GEMM's operand loader (round 4; north_star "coalesced ... patchify"): replaces the
 * stride-p convolution + position-embedding add of [3P] SiglipVisionEmbeddings (reached from
 * /root/reference/eagle/model/multimodal_encoder/clip_encoder.py:146) in ONE launch - no vitg_patchify pass, no im2col operand in HBM:
 *   out16[(t, py, px), n] = round16( sum_{c,ky,kx} pix[t, c, p py + ky, p px + kx] W[n, c, ky, kx] + bias[n] + pos[(py, px), n] )
 * pix: [T, 3, R, R] 16-bit NCHW (what the reference hands the tower, infer.py:55); rows/columns past p * (R / p) are ignored like the VALID
 * convolution ignores them.  Wf: the convolution weight re-laid ONCE at load to [N, ldw >= 64 ceil(3 p / 4)] in (c, ky)-pair order -
 * k = 16 (c p + ky) + slot; slot 0..7 = kx 0..7, slot 8..15 = kx p-8..p-1 with the slots of the re-read kx (p-8..7) zero; K-padding rows zero -
 * so that every 16-byte operand chunk is 8 consecutive pixels of one image row.  pos: fp32 [P, ldp] or null; bias fp32 [N] or null.
 * p even in 8..16, R even, N >= 256, T * 3 * R * R * 2 < 2^32; otherwise VITG_ERR_SHAPE (callers then use vitg_patchify + vitg_gemm_res16). */
int vitg_patch_embed16(const void* pix, int T, int R, int patch, const void* Wf, int ldw, int N, int dtype, const float* bias, void* out,
                       int ldo, const float* pos, int ldp, void* stream);
int vitg_bilinear_pool16(const void* x, int ldx, void* out, int ldo, int T, int G, int HW, int D, int dtype, const int* cmap, int Pc,
                         void* stream);

/* Deterministic split-K form of vitg_gemm(mode = VITG_GEMM_F32, act = none) for shapes with FEW output tiles and a long K - the
 * o / down projections of one rank of the context-parallel LLM (M = 12 860 / 8 rows: 98 tiles of 256 x 256 on 256 CUs).
 * vitg_gemm_splitk_plan tells how many splits pay off on this device (1 = use vitg_gemm) and how much fp32 workspace they need;
 * vitg_gemm_splitk runs `splits` blocks per output tile, each over its own K range into its own partial buffer, then
 * out[m,n] = partial_0 + partial_1 + ... + bias[n] + res[m,n] in that fixed order (no atomics: run-to-run bit-identical).
 * Same reference call sites as vitg_gemm (o_proj / down_proj + residual add, [3P] modeling_qwen2 via grounding_qwen2.py:135). */
int vitg_gemm_splitk_plan(int M, int N, int K, int* splits, long* workspace_bytes);
int vitg_gemm_splitk(const void* A, int lda, const void* W, int ldw, int M, int N, int K, int dtype, const float* bias, float* out,
                     int ldo, const float* res, int ldr, float* workspace, int splits, void* stream);
/* 16-bit-output form: out16 = round16(partial_0 + ... + bias) - the split-K form of vitg_gemm(mode = VITG_GEMM_STORE16, act = none) for the Q and K|V
 * projections of one context-parallel rank (q_proj / k_proj / v_proj + bias, [3P] modeling_qwen2 via grounding_qwen2.py:135; 98 / 28 output tiles on 256 CUs
 * where the plain launch leaves most of the chip idle for a whole K = 3584 tile).  Same plan function, same workspace rule, same fixed summation order. */
int vitg_gemm_splitk16(const void* A, int lda, const void* W, int ldw, int M, int N, int K, int dtype, const float* bias, void* out,
                       int ldo, float* workspace, int splits, void* stream);

/* ---- FP8 weight path (videoitg_amd/csrc/gemm_fp8.hip) ------------------------------------------------
 * The reference runs fp16 everywhere (/root/reference/eagle/model/builder.py:59), so this is an additional precision tier of the
 * same GEMM call sites as vitg_gemm: weights are stored as OCP e4m3fn bytes with one fp32 scale per OUTPUT CHANNEL (quantised
 * once at load time with vitg_quant_rows_fp8 on the [N,K] weight), activations are quantised PER TOKEN on the fly, and the
 * matrix pipe runs v_mfma_scale_f32_32x32x64_f8f6f4 (twice the 16-bit rate).  Accumulation, residual stream, norm and softmax
 * statistics stay fp32; attention stays 16-bit.
 *
 * vitg_quant_rows_fp8: out8[m, 0..ldo) = e4m3fn(x[m, :] / scale[m]) with scale[m] = max|x[m, :D]| / 448 (1 for an all-zero row),
 * round-to-nearest-even, columns D..ldo-1 zeroed.  x: in_dtype VITG_F32 / F16 / BF16, leading dimension ldx ELEMENTS; out8
 * leading dimension ldo BYTES (multiple of 16).
 * vitg_norm_quant_fp8: the same quantiser fused behind LayerNorm (b != NULL) or RMSNorm (b == NULL) of the fp32 residual row
 * (replaces vitg_layernorm / vitg_rmsnorm + a separate quantiser pass); D <= 4096.
 * vitg_gemm_fp8: out = epilogue( sa[m] * sw[n] * sum_k A8[m,k] W8[n,k] ), epilogue modes / bias / act / res exactly as vitg_gemm;
 * lda / ldw in BYTES (multiples of 16), K a multiple of 128 (callers zero-pad), N % 8 == 0; out_dtype = type of 16-bit outputs. */
int vitg_quant_rows_fp8(const void* x, long ldx, int in_dtype, void* out8, long ldo, float* scale, long M, int D, void* stream);
int vitg_norm_quant_fp8(const float* x, long ldx, const float* w, const float* b, void* out8, long ldo, float* scale, long M, int D,
                        float eps, void* stream);
int vitg_gemm_fp8(const void* A8, int lda, const float* sa, const void* W8, int ldw, const float* sw, int M, int N, int K,
                  int out_dtype, int mode, const float* bias, int act, void* out, int ldo, const float* res, int ldr, int res_mod,
                  void* stream);

/* The tower's 16-bit residual stream on the fp8 weight path (round 4): what vitg_gemm_res16 / vitg_layernorm16 are to vitg_gemm / vitg_layernorm.
 *   vitg_gemm_fp8_res16:   out16[m,n] = round16( scales * sum_k A8[m,k] W8[n,k] + bias[n] + res16[m,n] ); res16 (type `dtype`, may alias out) is
 *                          required; A8 carries per-token scales sa (a_mx == NULL) or MX block scales a_mx (sa ignored) as in vitg_gemm_fp8_mx.
 *   vitg_norm_quant_fp8_16: vitg_norm_quant_fp8 on 16-bit rows (in_dtype VITG_F16 / VITG_BF16).
 * Same call sites as vitg_gemm_res16 (SigLIP out_proj, fc2) and the LayerNorms in front of qkv / fc1. */
int vitg_gemm_fp8_res16(const void* A8, int lda, const float* sa, const void* a_mx, int ld_amx, const void* W8, int ldw, const float* sw, int M,
                        int N, int K, int dtype, const float* bias, void* out, int ldo, const void* res16, int ldr16, void* stream);
int vitg_norm_quant_fp8_16(const void* x, long ldx, int in_dtype, const float* w, const float* b, void* out8, long ldo, float* scale, long M,
                           int D, float eps, void* stream);

/* MX forms of vitg_gemm_fp8: activations that stay e4m3 BETWEEN two GEMMs carry OCP-MX block scales - one E8M0 byte (scale 2^(b-127)) per
 * 32 consecutive elements of a row, which v_mfma_scale_f32_32x32x64_f8f6f4 consumes as an operand - instead of a per-token fp32 scale
 * that only a separate pass over the finished row can compute.  Scale array layout: [K/128][ld][4] bytes, i.e. the four block scales
 * of the 128-deep K-tile kt of row m are the dword at byte ((kt * ld + m) * 4) (ld >= M).  Exactly one of a_mx / o_mx is non-NULL:
 *   o_mx (producer; mode VITG_GEMM_STORE16, or VITG_GEMM_SWIGLU with N/2 output columns): out = e4m3 bytes [M][ldo] (ldo BYTES, multiple
 *        of 128, columns past the last output column written as zeros)
 *        and, per 32-column block, the E8M0 exponent e = ceil(log2(max|v| / 448)) of v = act(sa*sw*acc + bias), out = e4m3(v * 2^-e)
 *        (round to nearest even, no saturation by construction); o_mx holds ldo/128 planes of ld_omx rows;
 *   a_mx (consumer; mode VITG_GEMM_F32, act none): A8 is such an output, a_mx its block scales (K/128 planes of ld_amx rows), sa is
 *        ignored; out = sw[n] * sum_k 2^(e[m,k/32]) A8[m,k] W8[n,k] + bias + res.
 * Used for both MLPs on the fp8 path (fc1 + GELU emits the operand of fc2: [3P] SiglipMLP via clip_encoder.py:146; gate/up + SwiGLU emits
 * the operand of down: [3P] Qwen2MLP via grounding_qwen2.py:135): removes the stand-alone quantiser pass over the hidden activation and
 * halves that tensor's bytes. */
int vitg_gemm_fp8_mx(const void* A8, int lda, const float* sa, const void* a_mx, int ld_amx, const void* W8, int ldw, const float* sw,
                     int M, int N, int K, int out_dtype, int mode, const float* bias, int act, void* out, int ldo, void* o_mx,
                     int ld_omx, const float* res, int ldr, void* stream);

/* Profiling aid (no reference counterpart, not on the product path): launches an MFMA-only kernel (blocks x 512 threads, 16
 * v_mfma_f32_32x32x16 per wave and iteration) whose operands are the 8 fragments of `pool` (8 x 64 lanes x 16 bytes, caller
 * filled: zeros, random, ...); *flops receives the flop count of the launch.  bench.py times it to report the MFMA rate the
 * device sustains on zero and on random operands (power-managed clock; videoitg_amd/csrc/probe.hip).  out: blocks*512 floats.
 * dtype 3 = the fp8 weight path's instruction (v_mfma_scale_f32_32x32x64_f8f6f4 on e4m3 bytes, 16 per wave and iteration). */
int vitg_mfma_probe(const void* pool, int dtype, int blocks, int iters, float* out, double* flops, void* stream);

/* out[m, 0..ldo) = LayerNorm(x[m, 0..D)) * w + b  (fp32 stats, eps inside rsqrt), columns D..ldo-1 zeroed.
 * out_dtype VITG_BF16/F16/F32.  Replaces [3P] SigLIP layer_norm1/2 (clip_encoder.py:146). */
int vitg_layernorm(const float* x, int ldx, const float* w, const float* b, void* out, int ldo, int out_dtype,
                   long M, int D, float eps, void* stream);

/* out = x * rsqrt(mean(x^2) + eps) * w.  Replaces [3P] Qwen2RMSNorm (grounding_qwen2.py:135). */
int vitg_rmsnorm(const float* x, int ldx, const float* w, void* out, int ldo, int out_dtype, long M, int D,
                 float eps, void* stream);

/* In-place rotary embedding (rotate_half layout) on `heads` consecutive heads of width head_dim starting at
 * qkv[n*ld]; cos/sin fp32 [N, head_dim/2].  Replaces [3P] apply_rotary_pos_emb (grounding_qwen2.py:135). */
int vitg_rope(void* qkv, int ld, const float* cos_t, const float* sin_t, long N, int heads, int head_dim, int dtype,
              void* stream);

/* Non-causal softmax(QK^T * scale) V, fp32 softmax, GQA (heads % kv_heads == 0), head_dim 72 or 128.
 * S queries attend to Sk keys (Sk == S on one GPU; Sk = all-gathered keys in the context-parallel LLM).  One (batch, kv head) slice of K / V must end
 * below 2 GiB - ((Sk rounded up to 64 - 1) * row stride + head_dim) * 2 bytes < 2^31, else VITG_ERR_SHAPE: the kernels stage it through 32-bit buffer
 * descriptors (whose range check turns the rows past the last key into zeros) with signed 32-bit lane offsets.
 * Strides in elements: *_bs batch, *_rs token row, *_hs head.  variant bit 0 = cross-check path that reads V from LDS with scalar
 * loads instead of ds_read_b64_tr_b16; variant bit 1 (value 2) = q already holds Q * scale * log2(e) (the producing projection carries the
 * factor in its q rows - what the engine does for the SigLIP tower): scores are exponentiated in base 2 with no further scaling, which lets
 * the head-dim-72 kernel take them from the matrix pipe ready for exp2 (no multiply, no max subtraction on the VALU).
 * Replaces flash-attn 2 fwd: SigLIP (clip_encoder.py:117 forces flash_attention_2) and the bidirectional
 * Qwen2 attention (grounding_qwen2.py:45-53, is_causal=False). */
int vitg_attention(const void* q, const void* k, const void* v, void* o, int batch, int heads, int kv_heads, int S,
                   int Sk, int head_dim, long q_bs, long k_bs, long v_bs, long o_bs, int q_rs, int k_rs, int v_rs, int o_rs,
                   int q_hs, int k_hs, int v_hs, int o_hs, float scale, int dtype, int variant, void* stream);

/* vitg_attention with the number of keys read from DEVICE memory at kernel start: keys [0, min(*kv_len_dev, Sk_max)) are attended,
 * rows beyond are ignored (their own outputs are still produced and are garbage-in/garbage-out for the caller to discard).
 * Launch geometry depends only on S, so one captured HIP graph serves every prompt length inside a padded bucket (SURVEY.md
 * section 7 hard part 6: "key-padding handled inside the attention kernel by length, not mask tensor").  Replaces the same
 * flash-attn call sites as vitg_attention; the reference strips padding on the host instead (eagle_archv1.py:272). */
int vitg_attention_dyn(const void* q, const void* k, const void* v, void* o, int batch, int heads, int kv_heads, int S,
                       int Sk_max, const int* kv_len_dev, int head_dim, long q_bs, long k_bs, long v_bs, long o_bs, int q_rs,
                       int k_rs, int v_rs, int o_rs, int q_hs, int k_hs, int v_hs, int o_hs, float scale, int dtype, int variant,
                       void* stream);

/* Bilinear G x G -> HW x HW token pool (align_corners=False, no antialias) of fp32 features [T*G*G, ldx] into
 * 16-bit [T*HW*HW, ldo]; HW == G is a plain cast.  cmap == NULL: x holds all G*G rows per frame; otherwise x holds Pc
 * compact rows per frame and cmap[y*G+x] is the compact row of token (y,x).  Replaces F.interpolate at mlp_proj.py:57-68. */
int vitg_bilinear_pool(const float* x, int ldx, void* out, int ldo, int T, int G, int HW, int D, int dtype,
                       const int* cmap, int Pc, void* stream);

/* out[b*n_idx + i, :] = src[b*rows_per_batch + idx[i], :] for b < batch (byte strides, 16-byte granules).  With
 * vitg_bilinear_pool's cmap (token y*G+x -> compact row, Pc rows per frame) this lets the LAST needed tower layer run its
 * Q projection, attention queries, out-proj and MLP only on the tokens the pool reads (81 of 729 at 27x27 -> 5x5): work
 * the reference performs and then discards (SURVEY.md 2.2 "only 81 of 729 source tokens have non-zero weight"). */
int vitg_gather_rows(const void* src, long ld_src_bytes, const int* idx, int n_idx, int rows_per_batch, int batch, void* out,
                     long ld_out_bytes, int row_bytes, void* stream);

/* out[i, :] = table[ids[i], :] (16-bit table -> fp32 rows).  Replaces embed_tokens at
 * /root/reference/eagle/model/eagle_archv1.py:310. */
int vitg_embed_gather(const long long* ids, int n, const void* table, int D, float* out, int ldo, int dtype,
                      void* stream);

/* logits[t] = mean_j h[t*tokens_per_frame + j, :] . w + b   (fp32).  Replaces grounding_qwen2.py:148-156. */
int vitg_pool_score(const float* h, int ldh, int frames, int tokens_per_frame, int D, const float* w,
                    const float* b, float* logits, void* stream);

/* scores[i] = sigmoid(logits[i]); order = argsort(scores) descending, ties by lower i (n <= 8192).
 * Replaces sigmoid + torch.sort at /root/reference/infer.py:72-74 and lmms_eval/models/videoitg.py:302-303
 * (whose tie order is unspecified; this one is deterministic). */
int vitg_rank(const float* logits, int n, float* scores, int* order, void* stream);

/* Grounding loss, forward value only: out2[0] = BCE-with-logits(logits, labels) with
 * pos_weight = min(5, sqrt(#neg / max(1, #pos))) = out2[1], mean over n (fp32).  Replaces the loss branch at
 * /root/reference/eagle/model/language_model/grounding_qwen2.py:159-169 (nn.BCEWithLogitsLoss). */
int vitg_bce_loss(const float* logits, const float* labels, int n, float* out2, void* stream);

/* Frame preprocessing in front of the tower.  Replaces the CPU call
 *   image_processor.preprocess(frames, return_tensors="pt")["pixel_values"]
 * at /root/reference/infer.py:55 and lmms_eval/models/videoitg.py:282,286 (third-party SiglipImageProcessor created at
 * eagle/model/multimodal_encoder/clip_encoder.py:115: Pillow BICUBIC resize on uint8, x * 1/255, (x - 0.5) / 0.5, HWC -> CHW).
 * frames: uint8 [T,H,W,3] device memory, strides in bytes (row_stride >= 3 W, frame_stride >= H row_stride);
 * out: [T,3,S,S] contiguous of out_dtype (VITG_F32 reproduces the reference's fp32 tensor bit for bit, VITG_F16 / VITG_BF16 its
 * .half() / .bfloat16()); tmp: scratch of vitg_preprocess_tmp_bytes bytes (may be null when that is 0).
 * The horizontal pass runs first, as Pillow's does - except that Pillow runs the VERTICAL pass first when an image more than 100 times taller than wide
 * is reduced in height (H > 100 W and S < H): that geometry returns VITG_ERR_SHAPE (W > 1, W != S); transpose the frames, call, transpose the result
 * (the two orders are each other's transposes - videoitg_amd/ops.py: preprocess_u8 does exactly that). */
int vitg_preprocess_tmp_bytes(int T, int H, int W, int S, long* bytes);
int vitg_preprocess_u8(const void* frames, int T, int H, int W, long frame_stride, int row_stride, void* out, int S,
                       int out_dtype, void* tmp, long tmp_bytes, void* stream);

/* ---- Operand-split precision tier (round 6; videoitg_amd/csrc/split.hip, engine option `operand_split`) ------------------------------
 * north_star compares with the reference's fp32 CPU path (|dscore| <= 1e-3); the reference's GPU path rounds every activation to fp16
 * (model.half(), /root/reference/eagle/model/builder.py:59) and so does the default path here.  On weights with massive-activation channels
 * 11-bit operands miss 1e-3 (profiles/r05_heavy_tail.md), so this tier carries every MFMA operand as a PAIR of fp16 values x = hi + lo
 * (hi = fp16(x), lo = fp16(x - hi): 22 bits; fp16 x fp16 products are exact in the fp32 accumulator).  A split operand of padded width Dp is one
 * fp16 matrix [M, >= 2 Dp]: hi in columns [0, Dp), lo in [lo_off, lo_off + Dp), pad columns zero; a GEMM consumes it through vitg_gemm with
 * K = 2 Dp against the weight laid twice side by side.  fp16 only.
 *
 * vitg_norm_split: LayerNorm (b != NULL) / RMSNorm (b == NULL) of fp32 rows -> split rows ([3P] SigLIP layer_norm1/2, Qwen2RMSNorm; the call
 *   sites vitg_layernorm / vitg_rmsnorm replace).  lo_off = padded payload width (multiple of 4, >= D), ldo >= 2 lo_off.
 * vitg_rope_split: vitg_rope on split q | k heads, in place (hi + lo is rotated in fp32 and split again).
 * vitg_bilinear_pool_split: vitg_bilinear_pool (mlp_proj.py:57-68) of fp32 features (dense, or compact with cmap / Pc as there) -> split rows.
 * vitg_gemm_split16: vitg_gemm's 16-bit-output modes (STORE16 with bias / activation, SWIGLU) writing (hi, lo) pairs: out[m, n] and
 *   out[m, n + lo_off]; N % 8 == 0, lo_off % 8 == 0, lo_off >= output width, ldo >= lo_off + output width.
 * vitg_attention_split: vitg_attention on split Q / K / V (lo planes at element offsets q_lo / k_lo / v_lo from the hi planes, same strides),
 *   S = Qh Kh^T + Qh Kl^T + Ql Kh^T, P split after the fp32 softmax, O = (Ph Vh + Ph Vl + Pl Vh) / l written as a split pair (o, o + o_lo).
 *   Replaces flash-attn at clip_encoder.py:117 / grounding_qwen2.py:45-53 for this tier; head_dim 72 or 128, GQA, non-causal. */
int vitg_norm_split(const float* x, int ldx, const float* w, const float* b, void* out, int ldo, int lo_off, long M, int D, float eps, void* stream);
int vitg_rope_split(void* qkv, int ld, long lo_off, const float* cos_t, const float* sin_t, long N, int heads, int head_dim, void* stream);
int vitg_bilinear_pool_split(const float* x, int ldx, void* out, int ldo, int lo_off, int T, int G, int HW, int D, const int* cmap, int Pc,
                             void* stream);
int vitg_gemm_split16(const void* A, int lda, const void* W, int ldw, int M, int N, int K, int mode, const float* bias, int act, void* out,
                      int ldo, long lo_off, void* stream);
int vitg_attention_split(const void* q, const void* k, const void* v, void* o, long q_lo, long k_lo, long v_lo, long o_lo, int batch, int heads,
                         int kv_heads, int S, int Sk, int head_dim, long q_bs, long k_bs, long v_bs, long o_bs, int q_rs, int k_rs, int v_rs,
                         int o_rs, int q_hs, int k_hs, int v_hs, int o_hs, float scale, void* stream);

/* ---- Training operators: what a fine-tuning step of the selector needs next to the forward (the reference trains it through autograd of the same modules:
 * eagle/model/language_model/grounding_qwen2.py:135-169 under train_itg.py).  Gradients never use floating-point atomics: the same call gives the same bits.
 * Workspaces belong to the call: two calls (or two captured graphs) that may run at the same time need one each.
 *
 * vitg_embed_lookup: out[i, :] = scale * table[ids[i], :] (table / out fp32, fp16 or bf16, one rounding); ids outside [0, vocab) - image slots, padding - give
 *   a zero row.  D, ldt, ldo multiples of 4.  (vitg_embed_gather without a scale, bounds or other types.)  embed_tokens at eagle/model/eagle_archv1.py:310.
 * vitg_embed_backward: dtable[v, :] = scale * sum over i with ids[i] = v of dout[i, :] for EVERY v < vocab (accumulate = 0: rows without a token are zero), or
 *   dtable[v, :] += that sum for the rows of the batch only (accumulate = 1).  ids outside the vocabulary contribute nothing.  fp32 sums.  Columns D .. ldt-1
 *   keep their contents.  At most 2^24 tokens a call.  workspace: vitg_embed_backward_plan bytes, 16-byte aligned. */
int vitg_embed_lookup(const long long* ids, long n, const void* table, int table_dtype, long ldt, long vocab, int D, float scale, void* out, int out_dtype,
                      long ldo, void* stream);
int vitg_embed_backward_plan(long n, int D, long* workspace_bytes);
int vitg_embed_backward(const long long* ids, long n, const void* dout, int dout_dtype, long ldd, long vocab, int D, float scale, void* dtable,
                        int table_dtype, long ldt, int accumulate, void* workspace, long workspace_bytes, void* stream);

/* The gated feed-forward's first half ([3P] Qwen2MLP gate_proj / up_proj / act via grounding_qwen2.py:135): [G | U] = X W^T with the weight rows interleaved
 * [32 gate | 32 up]... (the layout of VITG_GEMM_SWIGLU), out[M, N/2] = silu(G) * U.
 * vitg_swiglu: as vitg_gemm(mode = VITG_GEMM_SWIGLU); with gu != NULL it also stores [G | U] rounded to `dtype` in the weight rows' order ([M, N]) for the
 *   backward pass.  K % 64 == 0, N % 64 == 0, leading dimensions multiples of 8, 16-byte aligned pointers.
 * vitg_swiglu_backward: from dout = dL/d out and the saved gu: dX = dGU W (type dtype, overwritten) and dW (+)= dGU^T X (type dtype or fp32; accumulate = 1
 *   adds to what it holds), dGU rounded to dtype once - the matrix pipe's operand type (an fp16 value beyond 65 504 becomes infinite, one below 2^-25 zero, as in
 *   fp16 autograd: scale the loss for it); either of dX / dW may be NULL (then W / X is not read).  workspace: vitg_swiglu_backward_plan bytes, 16-byte
 *   aligned.  M = 0: dW becomes zero (accumulate = 0) or stays. */
int vitg_swiglu(const void* X, int ldx, const void* W, int ldw, int M, int N, int K, int dtype, void* out, int ldo, void* gu, int ldgu, void* stream);
int vitg_swiglu_backward_plan(int M, int N, int K, int want_dx, int want_dw, long* workspace_bytes);
int vitg_swiglu_backward(const void* dout, int lddo, const void* gu, int ldgu, const void* X, int ldx, const void* W, int ldw, int M, int N, int K, int dtype,
                         void* dX, int lddx, void* dW, int lddw, int dw_dtype, int accumulate, void* workspace, long workspace_bytes, void* stream);

/* The score head and grounding loss (grounding_qwen2.py:148-169) with their gradients.
 * vitg_pool_score_save: vitg_pool_score on fp32 / fp16 / bf16 rows (row t * tokens_per_frame + j, leading dimension ldh), keeping the frame means
 *   pooled[frames, ldp] (fp32).  Fewer than 2^22 frames.
 * vitg_bce_loss_backward: vitg_bce_loss (out2 = loss, pos_weight) and dlogits = scale * d loss / d logits.
 * vitg_pool_score_backward: dh[t * tokens_per_frame + j, :] = dlogits[t] / tokens_per_frame * w (fp32 / fp16 / bf16), dw (+)= sum_t dlogits[t] pooled[t, :],
 *   db (+)= sum_t dlogits[t]; each of dh / dw / db may be NULL; accumulate applies to dw and db.  Fewer than 2^24 slices of 32 tokens over all frames. */
int vitg_pool_score_save(const void* h, int h_dtype, long ldh, int frames, int tokens_per_frame, int D, const float* w, const float* b, float* logits,
                         float* pooled, long ldp, void* stream);
int vitg_bce_loss_backward(const float* logits, const float* labels, int n, float scale, float* out2, float* dlogits, void* stream);
int vitg_pool_score_backward(const float* pooled, long ldp, int frames, int tokens_per_frame, int D, const float* w, const float* dlogits, void* dh,
                             int dh_dtype, long lddh, float* dw, float* db, int accumulate, void* stream);

/* Global gradient norm over `count` tensors (HOST arrays of device pointers, element counts and dtype codes; contiguous tensors of fp32, fp16, bf16, mixed):
 * norm[0] = |scale| * sqrt(sum g^2) and, unless outs is NULL, outs[i] = grads[i] * scale * min(1, max_norm / (norm + 1e-6)); outs[i] may be grads[i], and
 * otherwise overlaps no tensor of the call.  Squares are summed in fp64.  An infinite norm gives factor 0, a NaN norm NaN, as the formula says (a finite
 * one beyond fp32 reads infinity in norm[0], while the factor comes from its fp64 value); max_norm = infinity scales only.  The addresses travel as kernel arguments: a captured call replays on the same tensors.  workspace: vitg_clip_grad_plan bytes,
 * 8-byte aligned.  (The reference's Trainer clips with max_grad_norm over all parameters of the model.) */
int vitg_clip_grad_plan(int count, const long* numel, const int* dtype, long* workspace_bytes);
int vitg_clip_grad(int count, const void* const* grads, void* const* outs, const long* numel, const int* dtype, float scale, float max_norm, float* norm,
                   void* workspace, long workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif
