/*
 * sf_hip.h — C-ABI of the MI355X (gfx950) kernel library `libsf_hip_kernels.so`.
 *
 * This is the drop-in boundary for the attention hot path of servoflow's
 * RDT-1B denoising loop.  Every entry point takes plain device pointers,
 * element strides and sizes, runs asynchronously on the given HIP stream,
 * never allocates or synchronises, and returns an `sf_status` code instead of
 * throwing.  All calls are capturable into a hipGraph.
 *
 * Reference interfaces replaced (paths relative to the servoflow tree):
 *   sf_attn_fwd            IBackend::attention
 *                          include/servoflow/backend/backend.h:105-110,
 *                          implemented by CUDABackend::attention
 *                          src/backend/cuda/cuda_backend.cu:470-501 and
 *                          cuda_ops::flash_attention
 *                          src/backend/cuda/ops/attention.cu:183-197.
 *   sf_attn_workspace_bytes the per-call workspace that
 *                          CUDABackend::attention sizes and allocates with
 *                          cudaMallocAsync (cuda_backend.cu:483-490); here the
 *                          caller owns it, so no allocation happens per call.
 *   sf_strerror            the message text of the std::runtime_error /
 *                          std::invalid_argument the reference throws
 *                          (cuda_backend.cu:22-40, 156-161).
 */
#ifndef SF_HIP_H_
#define SF_HIP_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes.  0 is success; errors are negative. */
typedef enum sf_status {
    SF_OK         = 0,
    SF_EINVAL     = -1,  /* bad shape, stride, alignment or argument       */
    SF_ENOTSUP    = -2,  /* valid request this library does not implement  */
    SF_EWORKSPACE = -3,  /* workspace missing or smaller than required     */
    SF_ELAUNCH    = -4,  /* kernel launch failed (hipGetLastError)         */
    SF_EDEVICE    = -5,  /* HIP runtime error outside a launch             */
    SF_ESCRATCH   = -6   /* request exceeds a fixed device scratch buffer  */
} sf_status;

/* Element types.  The numeric values equal servoflow's sf::DType
 * (include/servoflow/core/dtype.h:11-20) so a shim can cast directly. */
typedef enum sf_dtype {
    SF_F32  = 0,
    SF_F16  = 1,
    SF_BF16 = 2,
    SF_I8   = 3,
    SF_I32  = 5
} sf_dtype;

/*
 * Attention descriptor: out = softmax(Q·Kᵀ·scale) · V per (batch, head).
 *
 * Shapes: Q [B,H,Sq,D], K/V [B,H,Sk,D], out [B,H,Sq,D] addressed through
 * element strides (b, h, s); the head dimension d is contiguous (stride 1).
 * Writing out with o_stride = {Sq*H*D, D, H*D} stores [B,Sq,H*D] directly,
 * which is the layout the RDT block's output projection consumes
 * (replaces head_to_seq, src/backend/cuda/ops/split_ops.cuh:168-182).
 *
 * scale == 0 means 1/sqrt(D), as in attention.cu:150.
 * is_causal != 0 keeps key k for query q only when k <= q (top-left
 * alignment, attention.cu:117).
 * kv_valid_len: NULL (every key valid) or a DEVICE pointer to B int32
 * lengths; keys [valid_len[b], Sk) of batch b are ignored.  Lengths are
 * clamped to [0, Sk] on the device; a row with no valid key yields zeros.
 * kv_mask: NULL or a DEVICE pointer to a boolean key-padding mask, one byte
 * per key (nonzero = attend), batch b's row at kv_mask + b * kv_mask_stride
 * bytes (4-byte aligned, stride a multiple of 4, each row readable for Sk
 * rounded up to 4 bytes; bytes past Sk are ignored); combined with
 * kv_valid_len by AND.  This is the [B, Sk] key-padding form the RDT block
 * header documents (include/servoflow/models/rdt1b/dit_block.h:141) and the
 * mask argument of IBackend::attention (backend.h:104) that the reference
 * implementations ignore.
 * num_splits: 0 chooses the split-K factor automatically; n > 0 forces n
 * (at most 64).  Automatic: no split when B*H*ceil(Sq/80) fills the 256
 * CUs, none either when it does not and Sk <= 1024 (the call then runs one
 * workgroup per 16 query rows over all keys), key splits for about one
 * workgroup per CU otherwise.
 * exact_pv: 0 (default) runs the key-split kernel's (Sk > 128) P.V
 * contraction in fp16: a bf16 V converted with rounding to nearest, exact for
 * 2^-14 <= |v| < 2^16 (bf16's 8 significant bits fit fp16's 11; smaller
 * magnitudes round to fp16's subnormal grid, an absolute error of at most
 * 2^-25), and P rounded to the nearest fp16, ~2e-4 mean relative error on
 * the output.  A V element
 * with |v| >= 2^16 converts to +-inf, so the output column (head dim) it
 * belongs to becomes inf or NaN in every row that attends to its key, never
 * a saturated value; the other columns are unaffected.  A NaN or inf in V
 * behaves the same way.  1 keeps V in bf16 and P as a bf16 (hi, lo) pair
 * (~1e-5) for any finite V, at ~15% more time per key tile.
 * scale must be >= 0 (SF_ENOTSUP otherwise).
 *
 * in_dtype: SF_BF16, SF_F16 or SF_F32 for Q, K and V (the reference's
 * dispatch, attention.cu:183-197: fp16 -- its default compute dtype,
 * config.h:57 -- to flash attention, fp32 to the naive kernel).  fp16 runs
 * the same kernels with the fp16 MFMA for S = K.Q^T and V as loaded (exact_pv
 * then carries P as an fp16 hi/lo pair); fp32 runs a kernel on the fp32 MFMA
 * (v_mfma_f32_16x16x4_f32: nothing rounded below fp32; exact_pv ignored).
 * out_dtype: SF_BF16, SF_F16 or SF_F32 (rounded to nearest from fp32).
 *
 * Supported: D == 64, pointers 16-byte aligned, every stride a non-negative
 * multiple of 8 elements, s-strides >= D.
 */
typedef struct sf_attn_desc {
    int32_t B, H, Sq, Sk, D;
    float   scale;
    int32_t in_dtype;
    int32_t out_dtype;
    int32_t is_causal;
    int32_t num_splits;
    const int32_t* kv_valid_len;
    int64_t q_stride[3];
    int64_t k_stride[3];
    int64_t v_stride[3];
    int64_t o_stride[3];
    const uint8_t* kv_mask;
    int64_t kv_mask_stride;
    int32_t exact_pv;
    /* Optional (q_partials != NULL): Q given as the split-K partial sums of
     * its projection instead of q (which may then be NULL), the per-head
     * finish of the reference's q = gemm_bias_act(...), split and
     * apply_qk_norm (dit_block.cu:282-307) done inside the attention:
     * Q[b][h][s][d] = rmsnorm over d of (sum_j q_partials[j][b*Sq + s][n]
     * * q_scale[n] + q_bias[n]) * q_gamma[d], rounded to bf16, n = h*64 + d
     * (q_scale, q_bias, q_gamma each optional; q_eps the norm's epsilon).
     * q_partials: fp32 [q_splits][B*Sq][H*64] (sf_gemm's SF_EPI_PARTIALS
     * output), 1 <= q_splits <= 8, summed in ascending order.  bf16 inputs
     * on the query-block grid only (no key split, B*H*ceil(Sq/80) < 256 and
     * Sk <= 1024; such calls take that grid even for Sk <= 128); other calls
     * return SF_ENOTSUP.
     * Without q_partials, q_gamma and k_gamma (each optional, fp32 [64],
     * 16-byte aligned) apply the reference's per-head RMSNorm
     * (apply_qk_norm, dit_block.cu:185-196 and 262-272, called at 218-220
     * and 306-308; rms_norm_kernel_impl, norm.cuh:89-122) to every Q / K
     * row as it is loaded:
     * row[d] * (1 / sqrt(sum_d row[d]^2 / 64 + q_eps)) * gamma[d], rounded to
     * bf16 -- bit for bit what sf_gemm's per-head epilogue over a bf16
     * product (SF_EPI_HEADS above 160 rows) stores.  With q/k/v and their
     * strides pointing into a projection's 16-bit output (row b*S + s,
     * column section*H*64 + h*64 + d) this takes the place of split_qkv /
     * split_kv + apply_qk_norm.  bf16 or fp16 inputs (the normalised rows
     * are rounded to the input type; SF_ENOTSUP for fp32); k_gamma only on
     * the short-key path (Sk <= 128, no forced split). */
    const float* q_partials;
    int32_t q_splits;
    const float* q_bias;
    const float* q_scale;
    const float* q_gamma;
    float q_eps;
    const float* k_gamma;
    /* q_f16 != 0 (in_dtype SF_BF16, no q_partials): Q is given in fp16
     * while K and V are bf16 -- a projection's fp16 output rows against the
     * bf16 cross-attention K/V cache.  Each Q row is normalised with q_gamma
     * (when set) in fp32 and rounded to bf16 as it is loaded, so the
     * contraction is the bf16 one.  SF_ENOTSUP with another in_dtype or
     * with q_partials. */
    int32_t q_f16;
    /* With q_partials: q_row_ss != NULL says the projection's input rows
     * held x * gamma of a deferred RMSNorm (sf_gemm_desc.norm_ss); Q's row
     * b*Sq + s is then scaled by rsqrt(sum_t q_row_ss[t * B*Sq + b*Sq + s]
     * / q_row_n + q_row_eps) (q_row_tiles <= 64 tiles) after q_scale and
     * before q_bias -- as sf_gemm's a_row_ss does, bit for bit.
     * SF_EINVAL without q_partials. */
    const float* q_row_ss;
    int32_t q_row_tiles;
    int32_t q_row_n;
    float q_row_eps;
    /* v_f16 != 0 (in_dtype SF_BF16, exact_pv 0): V is given in fp16 while Q
     * and K are bf16 -- a cross-attention K/V cache whose V was converted
     * once (sf_bf16_to_f16_below) instead of per tile.  The fast P.V form
     * multiplies fp16 V by P rounded to fp16, exactly as it does after
     * converting a bf16 V itself, so a V converted with the same rounding
     * gives the same bits; the short-key kernel (Sk <= 128) takes fp16 V
     * with P as an fp16 (hi, lo) pair.  SF_ENOTSUP with another in_dtype or
     * with exact_pv. */
    int32_t v_f16;
    /* o_frag != 0: out is written as the [B*Sq][H*64] operand of
     * sf_gemm_frag in fragment order (row b*Sq + q, column h*64 + d; bf16 or
     * fp16) instead of through o_stride (ignored; SF_ENOTSUP for SF_F32). */
    int32_t o_frag;
    /* q_rows32 != NULL (in_dtype SF_BF16, no q_partials, no q_f16): Q given
     * as the fp32 rows [B*Sq][H*64] of a finished projection instead of q
     * (which may then be NULL): row b*Sq + s, column h*64 + d, normalised
     * with q_gamma (when set) and rounded to bf16 as it is loaded, on any
     * grid (key sets of at most 128 then run the ring kernel).  16-byte
     * aligned, at most 2 GB; SF_ENOTSUP with k_gamma. */
    const float* q_rows32;
} sf_attn_desc;

/* Fills a descriptor for contiguous [B,H,S,D] tensors (the layout
 * IBackend::attention documents at backend.h:103). */
void sf_attn_desc_init_bhsd(sf_attn_desc* desc, int32_t B, int32_t H,
                            int32_t Sq, int32_t Sk, int32_t D,
                            int32_t in_dtype, int32_t out_dtype);

/* Bytes of device workspace sf_attn_fwd needs for this descriptor: the
 * split-K partials (fp32 running max, running sum and unnormalised output),
 * 0 when the call needs no split.  Its contents need no initialisation;
 * calls that may run concurrently need separate workspaces. */
size_t sf_attn_workspace_bytes(const sf_attn_desc* desc);

/* Split-K factor sf_attn_fwd will use for this descriptor. */
int32_t sf_attn_num_splits(const sf_attn_desc* desc);

/* Enqueues the attention on `stream` (a hipStream_t; NULL = default). */
int sf_attn_fwd(const sf_attn_desc* desc, const void* q, const void* k,
                const void* v, void* out, void* workspace,
                size_t workspace_bytes, void* stream);

/* Allocation-free form of sf_attn_fwd.  No counterpart in the reference:
 * for callers that cannot allocate device memory (code under hipGraph
 * capture, tight serving loops, harnesses that forbid hipMalloc).  The
 * split-K partials go to a fixed device array of
 * SF_ATTN_NOALLOC_SCRATCH_BYTES held by the library on every GPU it runs on
 * until the process ends (looked up on the first call on each device: make
 * that first call outside a capture).  Same results as sf_attn_fwd with a
 * caller workspace.  A call whose partials (sf_attn_workspace_bytes) exceed
 * the array returns SF_ESCRATCH without launching anything; every split
 * count chosen automatically fits, only a large forced num_splits does not.
 * All calls on one GPU share its array and nothing in it needs to start at
 * zero: calls that may overlap on one GPU (different streams, or another
 * thread) race on it and must be serialised by the caller. */
#define SF_ATTN_NOALLOC_SCRATCH_BYTES (8u << 20)
int sf_attn_fwd_noalloc(const sf_attn_desc* desc, const void* q, const void* k,
                        const void* v, void* out, void* stream);

/* ---------------------------------------------------------------------------
 * Projections: C[M,N] = act(A[M,K] . W[N,K]^T + bias[N]).
 *
 * Replaces IBackend::gemm_bias_act as the RDT layers call it (trans_b = true;
 * backend.h:159-183, cuda_backend.cu:337-467; callers dit_block.cu:152-160,
 * 207, 233, 284, 291, 321) and folds in the ops around it:
 *   act: SF_ACT_GELU_TANH is GeluOp, SF_ACT_SILU is SiluOp
 *        (src/backend/cuda/ops/elementwise.cuh:35-68);
 *   epilogue SF_EPI_PLAIN: C (row stride ldc) in c_dtype; accumulate != 0
 *        adds into an fp32 C (the residual adds of dit_block.cu:372-384);
 *   epilogue SF_EPI_HEADS: the N columns are 1..3 sections of H*64 (Q|K|V or
 *        K|V, the order of split_qkv / split_kv, split_ops.cuh:62-84,
 *        210-226); section j goes to head_out[j][b][h][s][d] (bf16, element
 *        strides head_stride[j] = {b, h, s}) with row m = b*S + s (M need
 *        not be a multiple of S: the last batch element may be partial,
 *        e.g. the first L < S rows of one element), after an
 *        RMSNorm over the 64 head dims with head_gamma[j] when that pointer
 *        is non-NULL (q_norm / k_norm, dit_block.cu:219-220, 307-308);
 *   epilogue SF_EPI_ADD_NORM: C (fp32 residual) += result, then
 *        norm_out[m] = C[m] * rsqrt(mean(C[m]^2) + eps) * norm_gamma in
 *        norm_dtype (row stride norm_ldo): the branch add followed by the
 *        next RMSNorm, fused_add_rms_norm (norm.cuh:130-171,
 *        backend.h:127-134) as RDTBlock chains them (dit_block.cu:372-384);
 *        N <= 4096;
 *   w_dtype SF_I8: int8 weights with one fp32 scale per row (w_scale[N]),
 *        the weight-only dequant of quantization.cu:18-51 done in registers.
 * A and W rows must be 16-byte aligned (lda, ldw multiples of 8 elements),
 * K a multiple of 32; bias, w_scale, head_gamma, norm_gamma are fp32;
 * head_out must be 8-byte aligned with strides that are multiples of 4.
 *
 * workspace: scratch of sf_gemm_workspace_bytes().  M <= 160 (N a multiple
 * of 16): fp32 split-K partial sums, which spread one weight matrix over all
 * CUs.  M > 160: the library path -- hipBLASLt writes the fp32 product in
 * chunks of <= 8192 rows into the workspace (plus a bf16 copy of int8
 * weights and hipBLASLt's own scratch) and the epilogue kernels read it.
 * Two library-path cases store a bf16 product instead, with the bias (and
 * the int8 row scale) applied by hipBLASLt, as the reference's cuBLASLt
 * BIAS / GELU_BIAS epilogues return C in bf16 (cuda_backend.cu:414-447):
 *   - SF_EPI_PLAIN into a bf16 C without accumulate, act NONE or GELU_TANH:
 *     hipBLASLt writes C itself (GELU_BIAS for the GELU), one rounding as
 *     in the other paths, no epilogue kernel;
 *   - SF_EPI_HEADS / SF_EPI_ADD_NORM with round_product != 0: the per-head
 *     RMSNorm or the residual add + RMSNorm read bf16(A.W^T + bias) -- the
 *     reference's own storage point (the projection's bf16 output feeds
 *     split_qkv / fused_add_rms_norm) -- instead of the fp32 product.
 * int8 weights above 160 rows with no w_codes16 copy are read directly when
 * the call fits (sf_gemm_int8_direct): K = 2048, N a multiple of 256, ldw a
 * multiple of 16, fp16 activations, act NONE or GELU_TANH, and one of the
 * two 16-bit cases above in fp16 (an fp16 C, or round_product); the codes
 * are widened in registers and the product is stored in fp16 with the row
 * scale, bias and activation applied.
 * Other int8 calls there widen the codes into the workspace on every call.
 * With workspace == NULL a single-pass kernel runs instead and nothing
 * beyond A, W and the outputs is touched.  A non-NULL workspace that is too
 * small is SF_EWORKSPACE.  Calls that may run concurrently need separate
 * workspaces.
 * ------------------------------------------------------------------------- */
typedef enum sf_act { SF_ACT_NONE = 0, SF_ACT_GELU_TANH = 1, SF_ACT_SILU = 2 } sf_act;
typedef enum sf_epilogue {
    SF_EPI_PLAIN = 0,
    SF_EPI_HEADS = 1,
    SF_EPI_ADD_NORM = 2,
    /* The split-K path's fp32 K-slice sums stay in the workspace,
     * [sf_gemm_num_splits][M][N] (no bias, scale, activation; C not
     * written), for a consumer to finish -- the attention's q_partials.
     * Only for calls that run split-K (M <= 160 with a workspace); others
     * return SF_ENOTSUP. */
    SF_EPI_PARTIALS = 3
} sf_epilogue;

typedef struct sf_gemm_desc {
    int32_t M, N, K;
    const void* A;          /* [M][lda] bf16 */
    int64_t lda;
    int32_t a_dtype;
    const void* W;          /* [N][ldw] bf16 or int8 */
    int64_t ldw;
    int32_t w_dtype;
    const float* w_scale;   /* [N] for int8 weights */
    const float* bias;      /* [N] or NULL */
    int32_t act;
    int32_t epilogue;
    void* C;                /* SF_EPI_PLAIN output */
    int64_t ldc;
    int32_t c_dtype;
    int32_t accumulate;
    int32_t H, S;           /* SF_EPI_HEADS: heads per section, rows per batch */
    float eps;
    const float* head_gamma[3];
    void* head_out[3];
    int64_t head_stride[3][3];
    const float* norm_gamma; /* SF_EPI_ADD_NORM */
    void* norm_out;
    int64_t norm_ldo;
    int32_t norm_dtype;
    void* workspace;         /* split-K partial sums, or NULL */
    int64_t workspace_bytes;
    int32_t round_product;   /* M > 160, SF_EPI_HEADS / SF_EPI_ADD_NORM: bf16 product (see above) */
    const void* w_codes16;   /* int8 weights, optional: their codes as bf16 [N][K] (16-byte aligned,
                                sf_int8_codes_to_bf16); the library path reads this copy instead of
                                widening the codes itself on every call.  With w16_f16: an fp16
                                copy [N][K] of the weights (int8 codes or bf16 values,
                                sf_weights_to_f16) */
    int32_t w16_f16;         /* nonzero with a_dtype SF_F16: w_codes16 is the fp16 copy, and the
                                library path (M > 160) multiplies the fp16 activations by it in
                                fp16 -- no rounding of the activations to bf16 -- and its 16-bit
                                products (round_product, and a plain C written by hipBLASLt, which
                                must then be SF_F16) are fp16 (SF_EINVAL when w_codes16 is NULL on
                                this path).  The split-K path (M <= 160) reads the copy instead of
                                W when one is given: the operands it would otherwise form from W in
                                registers, so the same results without the conversion.  The
                                single-pass path reads W itself */
    /* Deferred RMSNorm (split-K path, M <= 160 with a workspace; SF_ENOTSUP
     * elsewhere; N a multiple of 64).  norm_ss (SF_EPI_ADD_NORM): instead of
     * the normalised row, norm_out[m] = C[m] * norm_gamma after the residual
     * add, and norm_ss[t * M + m] = the sum of C[m][n]^2 over the 64 columns
     * n of tile t (N / 64 tiles, fp32, 16-byte aligned) -- the row-wide
     * reduction is left to the consumer, so no workgroup waits for a whole
     * row.  a_row_ss (SF_EPI_PLAIN / SF_EPI_HEADS): A holds such rows; output
     * row m is scaled by rsqrt(sum_t a_row_ss[t * M + m] / a_row_n +
     * a_row_eps) (a_row_tiles tiles, <= 64) after the int8 scale and before
     * the bias: (s a) W^T = s (a W^T), the normalisation of
     * fused_add_rms_norm (norm.cuh:130-171) applied after the product. */
    float* norm_ss;
    const float* a_row_ss;
    int32_t a_row_tiles;
    int32_t a_row_n;
    float a_row_eps;
} sf_gemm_desc;

/* Bytes of workspace sf_gemm needs for this call (0: it always runs
 * single-pass): the split-K partials (M <= 160), or on the library path the
 * product buffer of the epilogue (none when hipBLASLt writes a plain bf16 C
 * itself), the int8 weights' bf16 copy and hipBLASLt's scratch. */
size_t sf_gemm_workspace_bytes(const sf_gemm_desc* desc);

int sf_gemm(const sf_gemm_desc* desc, void* stream);

/* K slices the split-K path uses for this shape (M, N, K, a_dtype), 0 when
 * the call does not run split-K. */
int32_t sf_gemm_num_splits(const sf_gemm_desc* desc);

/* 1 when sf_gemm multiplies this call's int8 weights directly above 160
 * rows (no 16-bit copy: w_codes16 NULL, the shape, types and epilogue
 * listed with the workspace above), else 0; pointers are not inspected.
 * Replaces the dequantize_int8_fp16_kernel pass (quantization.cu:18-51)
 * ahead of gemm_bias_act (cuda_backend.cu:337-467) for those calls. */
int32_t sf_gemm_int8_direct(const sf_gemm_desc* desc);

/* The SF_EPI_HEADS epilogue on a bf16 projection already in memory -- the
 * reference's split_qkv / split_kv followed by apply_qk_norm
 * (split_ops.cuh:62-84, dit_block.cu:185-196, 300-308) in one pass: row m of
 * P [M][ldp] (bias applied) is cut into N / (H*64) <= 3 sections of H heads,
 * each head's 64 values RMS-normalised with head_gamma[j] (when not NULL)
 * and written to head_out[j] at (m / S, h, m % S) with head_stride[j].
 * desc: M, N (a multiple of 64), H, S, eps, head_out, head_gamma,
 * head_stride as for sf_gemm; the GEMM fields are not read.  P 8-byte
 * aligned, ldp >= N a multiple of 4 (16 bytes and 8 take 16-byte loads).
 * Lets a caller run several projections as one GEMM (the runtime's K/V
 * cache: every layer's K/V weights in one matrix) and split per layer. */
int sf_heads_bf16(const sf_gemm_desc* desc, const void* P, int64_t ldp, void* stream);

/* Setup of the library path (M > 160) for this shape, once per shape and
 * process: for the fp32 product and the two bf16 products with bias (plain,
 * GELU) the hipBLASLt algorithm is chosen by timing its first 16
 * candidates on scratch buffers of the shape, each over weight copies
 * totalling 320 MB so that the weights stream from HBM as in a model step
 * (synchronous: allocates, launches on a private stream, frees).  sf_gemm
 * on a shape never prepared takes hipBLASLt's first candidate without
 * timing.  Call this before capturing a graph that contains the call. */
int sf_gemm_prepare(const sf_gemm_desc* desc);

/* Whether sf_gemm_prepare times hipBLASLt's candidates (timed = 1, the
 * default) or takes the first candidate of hipBLASLt's heuristic (0).  The
 * timed pick can differ from one process to the next, and with it the
 * bits of library-path products (M > 160); with 0 every process picks the
 * same algorithm for a given hipBLASLt, GPU and shape, so those products
 * are reproducible bit for bit, at up to ~35% more time per call.  Applies
 * to shapes prepared after the call (a shape keeps the algorithm it was
 * prepared with for the life of the process).  No counterpart in the
 * reference, whose cuBLASLt calls take cuBLASLt's heuristic choice
 * (cuda_backend.cu:414-447).  SF_EINVAL for other values. */
int sf_gemm_set_algo_timing(int32_t timed);

/* Which hipBLASLt algorithm the library path runs for this call's shape and
 * kind (M > 160; the first chunk of <= 8192 rows): *pick = its index in
 * hipBLASLt's heuristic list (0 = the heuristic's first choice),
 * *candidates = the usable candidates, *timed = 1 when the pick came from
 * timing them (sf_gemm_prepare with timing on), 0 otherwise.  SF_ENOTSUP
 * (pick -1) for a shape that is not on the library path or has not been
 * set up yet (sf_gemm_prepare or a first call).  No counterpart in the
 * reference: a record of what ran, for reproducibility reports. */
int sf_gemm_algo_pick(const sf_gemm_desc* desc, int32_t* pick, int32_t* candidates, int32_t* timed);

/* ---------------------------------------------------------------------------
 * Normalisation and dequant.
 * ------------------------------------------------------------------------- */
/* out[r] = x[r] * rsqrt(mean(x[r]^2) + eps) * gamma, fp32 accumulation
 * (rms_norm_kernel_impl, src/backend/cuda/ops/norm.cuh:89-122;
 * IBackend::rms_norm, backend.h:120-122).  x in SF_F32 or SF_BF16, out in
 * SF_BF16 or SF_F32, gamma fp32 [cols]. */
int sf_rmsnorm(const void* x, int32_t x_dtype, int64_t ldx, const float* gamma,
               void* out, int32_t out_dtype, int64_t ldo, int32_t rows,
               int32_t cols, float eps, void* stream);

/* Deferred RMSNorm of fp32 rows x (cols a multiple of 64, rows 16-byte
 * aligned): out[r] = x[r] * gamma (not yet normalised) and ss[t * rows + r]
 * = the sum of x[r][c]^2 over the 64 columns c of tile t, for a consumer
 * that applies rsqrt(sum_t ss / cols + eps) after its contraction
 * (sf_gemm_desc.a_row_ss, sf_attn_desc.q_row_ss) -- rms_norm_kernel_impl
 * (norm.cuh:89-122) with its row-wide step moved into the consumer. */
int sf_rmsnorm_deferred(const float* x, int64_t ldx, const float* gamma, void* out, int32_t out_dtype,
                        int64_t ldo, float* ss, int32_t rows, int32_t cols, void* stream);

/* residual[r] += delta[r]; out[r] = rmsnorm(residual[r]) * gamma
 * (fused_add_rms_norm_kernel, norm.cuh:130-171; IBackend::fused_add_rms_norm,
 * backend.h:127-134).  residual fp32 (kept in fp32 here), delta SF_F32 or
 * SF_BF16, out SF_BF16 or SF_F32. */
int sf_add_rmsnorm(const void* delta, int32_t delta_dtype, float* residual,
                   const float* gamma, void* out, int32_t out_dtype,
                   int32_t rows, int32_t cols, float eps, void* stream);

/* out[i] = float(q[i]) * scale[i / K] (per_channel != 0) or * scale[0],
 * q int8 [N][K] row-major (dequantize_int8_fp16_kernel,
 * src/backend/cuda/ops/quantization.cu:18-51; IBackend::dequantize,
 * backend.h:205-206).  out in SF_F32 or SF_BF16 (the reference writes fp16
 * with an fp16 scale; here the scale is fp32). */
int sf_dequant_int8(const int8_t* q, const float* scale, int32_t per_channel,
                    void* out, int32_t out_dtype, int64_t N, int64_t K,
                    void* stream);

/* Exact bf16 copies of int8 weight codes (no scale: |code| <= 128 fits
 * bf16's 8 significant bits), for up to SF_CODES_MAX_JOBS matrices in one
 * launch: job j widens q [N][ldq] into out [N][K].  The unpack of
 * dequantize_int8_fp16_kernel (quantization.cu:18-51) without its scale
 * multiply; the library path of sf_gemm (M > 160) takes such a copy as
 * w_codes16, so a caller running several int8 projections at a large batch
 * can widen their weights in one pass instead of one pass per call.  ldq
 * and K multiples of 16, pointers 16-byte aligned. */
#define SF_CODES_MAX_JOBS 8
typedef struct sf_codes_job {
    const int8_t* q;
    int64_t ldq;
    void* out;
    int32_t N, K;
} sf_codes_job;
int sf_int8_codes_to_bf16(const sf_codes_job* jobs, int32_t count, void* stream);

/* fp16 copies of projection weights for the library path's fp16 products
 * (sf_gemm_desc.w16_f16): job j converts w [N][ldw] -- int8 codes (exact,
 * no scale: the row scale stays with the GEMM) or bf16 values (rounded to
 * the nearest fp16: exact for 2^-14 <= |w| < 65520, within 2^-25 below,
 * +-inf at or above 65520) -- into out [N][K], up to SF_CODES_MAX_JOBS
 * matrices per launch.  K a multiple of 16, rows 16-byte aligned. */
typedef struct sf_w16_job {
    const void* w;
    int32_t w_dtype;   /* SF_I8 or SF_BF16 */
    int64_t ldw;       /* elements */
    void* out;
    int32_t N, K;
} sf_w16_job;
int sf_weights_to_f16(const sf_w16_job* jobs, int32_t count, void* stream);

/* ---------------------------------------------------------------------------
 * Fragment-ordered projections: one launch per projection.
 *
 * Fragment order of X[R][K] in 16 bits: blocks of 16 rows x 32 columns, block
 * (r / 16, k / 32) at index (r / 16) * (K / 32) + k / 32, 512 elements each;
 * inside a block, element (r, k) at (((k % 32) / 8) * 16 + r % 16) * 8 + k % 8.
 * R is padded to a multiple of 16; the padding rows are never written and may
 * hold anything.  int8: blocks of 16 rows x 64 columns, 1024 bytes, code
 * (r, k) at (((k % 32) / 8) * 16 + r % 16) * 16 + ((k % 64) / 32) * 8 + k % 8.
 * No counterpart in the reference: the layout lets a wave load an MFMA
 * operand as 1 KB of contiguous memory.
 * ------------------------------------------------------------------------- */
/* Elements of a fragment-ordered [rows][cols] buffer. */
size_t sf_frag_elems(int64_t rows, int64_t cols);

/* Row-major weights w [N][ldw] -> out in fragment order, up to
 * SF_CODES_MAX_JOBS matrices per launch: bf16 -> bf16, bf16 -> fp16 (rounded
 * as sf_weights_to_f16 does), fp16 -> fp16, int8 -> int8, int8 -> fp16
 * (exact, the row scale stays with the GEMM).  N a multiple of 16, K of 64, ldw of 8, pointers 16-byte aligned. */
typedef struct sf_frag_job {
    const void* w;
    int32_t w_dtype;
    int64_t ldw;
    void* out;
    int32_t out_dtype;
    int32_t N, K;
} sf_frag_job;
int sf_frag_pack(const sf_frag_job* jobs, int32_t count, void* stream);

/* RMSNorm of fp32 rows (cols a multiple of 64, at most 4096; rows and gamma
 * 16-byte aligned) into fragment order in SF_BF16 or SF_F16
 * (rms_norm_kernel_impl, norm.cuh:89-122).  ss != NULL: the deferred form of
 * sf_rmsnorm_deferred instead: x * gamma, and ss [rows][cols / 64] (row-major
 * here) the sums of squares of 64 columns; for SF_F16 with the marks of
 * sf_gemm_frag's SF_EPI_ADD_NORM. */
int sf_norm_frag(const float* x, int64_t ldx, const float* gamma, void* out, int32_t out_dtype, float* ss,
                 int32_t rows, int32_t cols, float eps, void* stream);

/* C = act((A . W^T) * w_scale * row scale + bias) (act with SF_EPI_PLAIN,
 * the row scale not with SF_EPI_ADD_NORM) with A and W in fragment
 * order, one launch, no workspace: sf_gemm's arithmetic (gemm_bias_act,
 * cuda_backend.cu:337-467) and epilogues over all of K in one workgroup.
 * N a multiple of 32, K of 64.  a_dtype SF_BF16 or SF_F16; w_dtype the same, or
 * SF_I8; w_scale [N] required for SF_I8, optional else.  Epilogues:
 *   SF_EPI_PLAIN     C row-major (ldc a multiple of 4) in c_dtype, with
 *                    accumulate for SF_F32; or, with c_frag, in fragment
 *                    order (SF_BF16 / SF_F16).
 *   SF_EPI_HEADS     as sf_gemm's: bf16 per-head outputs with the optional
 *                    per-head RMSNorm.
 *   SF_EPI_ADD_NORM  the deferred form only: C (fp32) += result, norm_out
 *                    (fragment order, norm_dtype) = C * norm_gamma, and
 *                    norm_ss[m * T + t] = the sum of C[m][n]^2 over tile t's
 *                    columns, T = sf_gemm_frag_ss_tiles(desc) <= 64 tiles.
 *                    SF_F16 marks: infinite where an element leaves fp16's
 *                    range, negated where the tile has no element of at least
 *                    sqrt(N) 2^-11 in magnitude.
 * a_row_ss (SF_EPI_PLAIN, SF_EPI_HEADS): as sf_gemm_desc's, but row-major,
 * [M][a_row_tiles].  SF_F16 rows need a_x (SF_EINVAL without) and are taken by
 * SF_EPI_PLAIN only (SF_ENOTSUP else): x * gamma can leave fp16's range or lie
 * in its subnormals.  Rows with an infinite sum, and rows of a mean square below
 * 1 whose sums are all negative, are normalised from the fp32 rows
 * a_x [M][a_x_ld] with a_x_gamma instead
 * (a_row_n == K).  Row m's result depends on row m, the weights and the
 * summation order that K fixes, not on M. */
typedef struct sf_frag_gemm_desc {
    int32_t M, N, K;
    const void* A;
    int32_t a_dtype;
    const void* W;
    int32_t w_dtype;
    const float* w_scale;
    const float* bias;
    int32_t act;
    int32_t epilogue;
    void* C;
    int64_t ldc;
    int32_t c_dtype;
    int32_t c_frag;
    int32_t accumulate;
    int32_t H, S;
    float eps;
    const float* head_gamma[3];
    void* head_out[3];
    int64_t head_stride[3][3];
    const float* norm_gamma;
    void* norm_out;
    int32_t norm_dtype;
    float* norm_ss;
    const float* a_row_ss;
    int32_t a_row_tiles;
    int32_t a_row_n;
    float a_row_eps;
    const float* a_x;
    int64_t a_x_ld;
    const float* a_x_gamma;
} sf_frag_gemm_desc;
int sf_gemm_frag(const sf_frag_gemm_desc* desc, void* stream);
/* Tile sums per row that SF_EPI_ADD_NORM writes for this call (M, N, a_dtype,
 * w_dtype are read). */
int32_t sf_gemm_frag_ss_tiles(const sf_frag_gemm_desc* desc);

/* ---------------------------------------------------------------------------
 * Projections over 4-bit weights with group scales.
 *
 * C[m][n] = act(sum_k A[m][k] * scale[n][k / group] * (code[n][k]
 * - zero[n][k / group]) + bias[n]): the weight form below the reference's
 * weight-only int8 (quantization.cu:18-51 ahead of gemm_bias_act,
 * cuda_backend.cu:337-467), which has no 4-bit form.  Codes are 0..15, group
 * 32, 64 or 128 inputs, K a multiple of the group, any N to 2^25, any M to
 * 2^21, lda to 2^23 (SF_ENOTSUP above).
 *
 * sf_w4_pack lays a checkpoint's codes and scales out once, in the order the
 * matrix operands are read; sf_gemm_w4 reads that.
 * ------------------------------------------------------------------------- */
typedef struct sf_w4_pack_desc {
    int32_t N, K, group;
    const uint8_t* codes;    /* [N][ldc] bytes: inputs 2 i (low half) and 2 i + 1 (high half) in byte i */
    int64_t ldc;             /* bytes, >= K / 2 */
    const void* scales;      /* [N][lds], K / group a row */
    int64_t lds;
    int32_t scale_dtype;     /* SF_F16 or SF_BF16, kept bit for bit */
    const uint8_t* zeros;    /* [N][ldz], one byte a group (0..255), or NULL: 8 */
    int64_t ldz;
} sf_w4_pack_desc;

/* Bytes of the packed form (0 for a shape that is not supported). */
size_t sf_w4_bytes(int32_t N, int32_t K, int32_t group);
/* out: sf_w4_bytes() bytes, 16-byte aligned. */
int sf_w4_pack(const sf_w4_pack_desc* desc, void* out, void* stream);

typedef struct sf_gemm_w4_desc {
    int32_t M, N, K, group;
    const void* A;           /* [M][lda] bf16 or fp16, rows 16-byte aligned (lda a multiple of 8) */
    int64_t lda;
    int32_t a_dtype;
    const void* W;           /* sf_w4_pack's output for the same N, K, group */
    int32_t scale_dtype;     /* as packed */
    const float* bias;       /* [N] or NULL */
    int32_t act;             /* sf_act */
    void* C;                 /* [M][ldc] */
    int64_t ldc;
    int32_t c_dtype;         /* SF_F32, SF_BF16 or SF_F16 */
    int32_t accumulate;      /* SF_F32 only: C += act(...) */
} sf_gemm_w4_desc;
/* One launch, no workspace.  Codes and activations meet exactly in fp32
 * accumulators; scale and zero point are applied to each group's sum in fp32.
 * The sums are of codes + 16: 31 times a group's sum of |A| has to be finite
 * (an infinity or a NaN in a row of A makes that row of C NaN).
 * C must not overlap A.
 * For few rows: from memory 16 x 8192 x 8192 takes 12 us where sf_gemm over 16-bit
 * weights takes 39, 134 rows 41 and 131.  From some 200 to 500 rows on (268 x 6144 x
 * 2048: 24 and 17; 536 x 2048 x 8192: 39 and 43; 1072 x 6144 x 2048: 67 and 32) the
 * 16-bit product is the faster one, up to 2.6 times. */
int sf_gemm_w4(const sf_gemm_w4_desc* desc, void* stream);

/* ---------------------------------------------------------------------------
 * 4-bit key / value cache: head norm + rotation into it, and attention over it.
 *
 * Format.  For every batch element, key head, token and group of 64 channels:
 * mid = bf16((max + min) / 2), a = max |x - mid|, s = (a rounded up to bf16)
 * / 8, code = clamp(floor((x - mid) / s) + 8, 0, 15); a code stands for
 * s (code - 7.5) + mid, so |value - x| <= s / 2.  s below 2^-126 counts as 0
 * (every code then stands for mid); a group with an infinity or a NaN reads
 * back as NaN, and only that group.  36 bytes for 64 channels of K or V,
 * against 128 in 16 bits.  The reference caches no keys: it projects them
 * again on every call (dit_block.cu:288-293).
 *
 * data: sf_kv4_bytes(B, H, capacity, D) bytes, 16-byte aligned, D 64 or 128;
 * it needs no initialisation.  Tokens are written one by one or many at a
 * time, each into its own bytes: writes to other slots never disturb a token,
 * so appending needs no order.
 * ------------------------------------------------------------------------- */
typedef struct sf_kv4_cache {
    void* data;
    int32_t B, H, capacity, D;
} sf_kv4_cache;
/* 0 for a shape that is not supported. */
size_t sf_kv4_bytes(int32_t B, int32_t H, int32_t capacity, int32_t D);

/* Query, key and value heads of B * S tokens: RMSNorm over each query and key
 * head's D channels (gamma[0], gamma[1]; NULL: none) -- apply_qk_norm,
 * dit_block.cu:185-196, 262-272 -- then the rotation of their first `rot`
 * channels by the token's position: channels (i, i + rot / 2), or (2 i,
 * 2 i + 1) with interleaved, turn by positions[m] * inv_freq[i] radians,
 * i < rot / 2 (the angle is formed in 64 bits).  rot a multiple of 16, 0 for
 * none.  Values pass unchanged.  All arithmetic in fp32, one rounding at the
 * end.
 *
 * Section j (0 query, 1 key, 2 value) has heads[j] heads (0: left out), reads
 * src[j] and writes out[j], both addressed as [B][heads][S][D] through element
 * strides {b, h, s}, channels contiguous: pointers 16-byte aligned, strides
 * non-negative multiples of 8.  A projection's output rows are three such
 * views (h stride D, s stride the row's).  out[j] may be src[j] itself (same
 * strides and type); otherwise they must not overlap.
 *
 * cache.data != NULL: keys and values go into the cache instead of out[1] and
 * out[2] (heads[1] == heads[2] == cache.H, cache.B == B, cache.D == D), token m
 * at slot slots[m], or at its position if slots is NULL.  A slot outside
 * [0, capacity) leaves the cache as it was.  The slots of one batch element
 * have to differ within a call; two tokens at one slot leave a mixture there,
 * and only there.
 * B * S is below 2^23 (SF_ENOTSUP above; sf_kv4_read likewise).
 * positions, slots: DEVICE [B * S]; positions NULL: token s of each batch
 * element is at s.  A token with a negative position is padding: nothing of it
 * is written. */
typedef struct sf_heads_rope_desc {
    int32_t B, S, D;
    int32_t heads[3];
    int32_t in_dtype, out_dtype;      /* SF_F32, SF_BF16 or SF_F16 */
    const void* src[3];
    int64_t src_stride[3][3];
    void* out[3];
    int64_t out_stride[3][3];
    const float* gamma[2];            /* [D] or NULL */
    float eps;
    const int32_t* positions;
    const double* inv_freq;           /* DEVICE [rot / 2] */
    int32_t rot, interleaved;
    sf_kv4_cache cache;               /* data NULL: none */
    const int32_t* slots;             /* only with a cache */
} sf_heads_rope_desc;
int sf_heads_rope(const sf_heads_rope_desc* desc, void* stream);

/* The values that cached tokens stand for: k and v [B][H][S][D] through
 * element strides {b, h, s} (as above) in out_dtype, token (b, s) from slot
 * slots[b * S + s] (DEVICE; NULL: slot s).  Zeros for a slot outside
 * [0, capacity). */
int sf_kv4_read(const sf_kv4_cache* cache, const int32_t* slots, int32_t S, void* k, const int64_t* k_stride, void* v,
                const int64_t* v_stride, int32_t out_dtype, void* stream);

/* out = softmax(Q K^T scale) V over the cache (IBackend::attention,
 * backend.h:105-110, on the values that the codes stand for).  Q and out
 * [B][Hq][Sq][D] through element strides {b, h, s}, channels contiguous,
 * pointers 16-byte aligned, strides non-negative multiples of 8; Hq a multiple
 * of cache.H, query head h reads key head h / (Hq / cache.H).
 * Sk: keys [0, Sk) are read at most (<= cache.capacity and 2^30).  kv_valid_len: NULL
 * or DEVICE [B]: keys from there on are not seen (clamped to [0, Sk]).
 * kv_mask: NULL or DEVICE bytes, [B] rows of Sk kv_mask_stride apart, nonzero
 * = seen.  is_causal: query s of Sq is the token at valid_len - Sq + s, and
 * sees the keys up to itself -- one new token, or a chunk behind what is
 * cached.  (sf_attn_fwd aligns causal rows at the other end, as
 * attention.cu:117 does.)  A row that sees nothing yields zeros.  Slots that
 * no row sees may hold anything.
 * scale 0: 1 / sqrt(D); negative: SF_ENOTSUP.  in_dtype SF_BF16 or SF_F16.
 * The softmax's maximum and sum are fp32; its weights enter the product with V
 * as bf16 (hi, lo) pairs, 2^-18 relative, and for an fp32 output as three bf16
 * terms, which leaves it within 1e-6 of its norm up to 16384 keys (as sums over
 * fp32 values).  Unless exact_pv is set, a bf16 output of more than 16 query rows
 * to a key head that all see the same tokens (no is_causal, or Sq 1), with at most
 * 2^15 keys to a split, takes weights and values as fp16, the values under a power of two
 * that keeps them in its range: 7 2^-12 of the largest value that the row sees,
 * beside the output's own rounding (6e-4 of the output's norm, where that rounding
 * is 1.7e-3; rows whose largest value is below 2^-100 lose bits).
 * Values are taken up to 2^100 in magnitude.  out may be Q itself
 * (same strides and type); otherwise they must not overlap.
 * num_splits: 0 chooses; n > 0 forces n key splits (at most 64; with more than
 * one of them B * Hq * Sq is below 2^24).  B * cache.H times the splits and the
 * groups of 16 or more query rows of a key head is below 2^23 (SF_ENOTSUP above
 * either). */
typedef struct sf_attn_kv4_desc {
    int32_t B, Hq, Sq, Sk;
    float scale;
    int32_t in_dtype, out_dtype;
    int32_t is_causal;
    int32_t num_splits;
    int32_t exact_pv;      /* weights as bf16 pairs, values as cached, for bf16 outputs of many rows too */
    const int32_t* kv_valid_len;
    const uint8_t* kv_mask;
    int64_t kv_mask_stride;
    int64_t q_stride[3];
    int64_t o_stride[3];
    sf_kv4_cache cache;
} sf_attn_kv4_desc;
/* Bytes of device workspace (the splits' partial sums), 0 where none is
 * needed.  No initialisation; calls that may run concurrently need separate
 * workspaces. */
size_t sf_attn_kv4_workspace_bytes(const sf_attn_kv4_desc* desc);
int sf_attn_kv4(const sf_attn_kv4_desc* desc, const void* q, void* out, void* workspace, size_t workspace_bytes,
                void* stream);

/* ---------------------------------------------------------------------------
 * A step that verifies a tree of drafted tokens over the 4-bit cache: the
 * tree's tables, attention of its nodes, the path that sampled tokens confirm,
 * and the cache with that path alone.
 *
 * Node 0 is the root, the last token already decided; parents[j] < j is node j's
 * parent, and any other value (node 0's too) counts as none: such a node has no
 * ancestors and is on no path.  `each` 0: one tree [T] for all batch elements;
 * otherwise a tree for each of them ([B][T]).  T to SF_TREE_MAX_NODES
 * (SF_ENOTSUP above).  All arrays are device memory.
 * ------------------------------------------------------------------------- */
#define SF_TREE_MAX_NODES 1024

/* masks [trees][T][ceil(T / 32)]: bit i of node j's row (word i / 32) is set
 * where i is j or an ancestor of j; the bits behind T are zero.  depth [trees][T]: a
 * node's number of ancestors (its position is the root's and that). */
int sf_tree_build(const int32_t* parents, int32_t trees, int32_t T, uint32_t* masks, int32_t* depth, void* stream);

typedef struct sf_draft_tree {
    const uint32_t* masks;   /* sf_tree_build's */
    int32_t T, each;
} sf_draft_tree;

/* sf_attn_kv4 for a tree: its T nodes are the last T of a sequence's cached
 * tokens (node i in slot valid_len - T + i; kv_valid_len NULL: Sk), the Sq <= T
 * queries the last Sq nodes.  A query sees every token before the nodes, itself
 * and its ancestors (of those, what kv_mask leaves).  Nodes before a sequence's
 * first token (valid_len < T) see nothing: zeros.  is_causal: SF_EINVAL.
 * Everything else as sf_attn_kv4, without the form in fp16. */
size_t sf_attn_kv4_tree_workspace_bytes(const sf_attn_kv4_desc* desc, const sf_draft_tree* tree);
int sf_attn_kv4_tree(const sf_attn_kv4_desc* desc, const sf_draft_tree* tree, const void* q, void* out, void* workspace,
                     size_t workspace_bytes, void* stream);

/* The path of drafted tokens that sampled ones confirm.  drafted [B][T]: the
 * nodes' tokens; sampled [B][T]: the token sampled behind each node.  From the
 * root on, the child whose drafted token is the node's sampled one follows, the
 * first such child by index, until there is none.  nodes, tokens [B][T]: the path
 * and the tokens sampled along it (one more than the drafted tokens confirmed), -1
 * behind the end; count [B]: the path's length, 1 at least.  Tokens sampled one by one
 * from the model give the same sequence.  drafted[b][0] is not read. */
int sf_tree_accept(const int32_t* parents, int32_t each, const int32_t* drafted, const int32_t* sampled, int32_t B,
                   int32_t T, int32_t* nodes, int32_t* count, int32_t* tokens, void* stream);

/* Keeps a path's tokens: for every batch element the cached token of slot first[b] +
 * nodes[b][i] moves to slot first[b] + i, as if all were read before any is
 * written.  nodes [B][n] (n to SF_TREE_MAX_NODES); a negative node, and one whose
 * slot or place is outside [0, capacity), is left out. */
int sf_kv4_keep(const sf_kv4_cache* cache, const int32_t* nodes, int32_t n, const int32_t* first, void* stream);

/* ---------------------------------------------------------------------------
 * One token from each row of logits, with given uniform numbers.
 *
 * With m the row's largest logit a token's weight is exp((l - m) / temperature),
 * held to 2^-44 of the largest.  In falling order of logits, ties by index: the
 * first top_k tokens (0 or less: all); of these the fewest whose weights reach
 * top_p of their sum (1 or more: all; one at least); of these the ones of at
 * least min_p times the largest weight (0: all; one at least).  The token is the
 * first whose running weight exceeds u times the sum of what is left, logprob the
 * logarithm of its share of that sum (near 0 to 1.02e-6 of itself, of which 2^-20 is that
 * weights are held to 2^-44, and V 2^-70, for fp32 rows with top_k V 2^-46: they
 * do not tell apart what is below).  temperature 0 or less: the first in order,
 * the lowest index of the largest logits.
 * A logit of -infinity is never taken; logits of +infinity share all the weight.
 * A row with a NaN, or without a logit above -infinity, gives token -1 and a NaN.
 * Sums are of whole numbers: a row's token depends on the row and its parameters
 * alone.
 * ------------------------------------------------------------------------- */
#define SF_SAMPLE_MAX_VOCAB (1 << 20)
typedef struct sf_sample_desc {
    int32_t rows, V;
    const void* logits;          /* [rows][ld], SF_F32, SF_BF16 or SF_F16, any alignment of the type */
    int64_t ld;
    int32_t dtype;
    const float* u;              /* DEVICE [rows], in [0, 1) */
    const float* temperature;    /* DEVICE [rows], or NULL: temperature_all; the others likewise */
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    float temperature_all;
    int32_t top_k_all;
    float top_p_all, min_p_all;
    int32_t* token;              /* [rows] */
    float* logprob;              /* [rows] or NULL */
} sf_sample_desc;
/* Bytes of device workspace (the sums of few long rows, which several workgroups share), 0 where none is needed;
 * 8-byte aligned, no initialisation; calls that may run concurrently need separate ones. */
size_t sf_sample_workspace_bytes(const sf_sample_desc* desc);
int sf_sample(const sf_sample_desc* desc, void* workspace, size_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------------------
 * Projections in 8-bit integers: activations with a scale for each row (token),
 * weights with one for each output channel.
 *
 * C[m][n] = act(a_scale[m] w_scale[n] sum_k a[m][k] w[n][k] + bias[n]), the sum exact
 * in 32 bits.  The reference's int8 is weight-only (quantization.cu:18-51); sf_gemm
 * with SF_I8 weights is that, and sf_gemm_i8 takes the same codes and scales.
 * K a multiple of 16 to 2^16, M to 2^22, N to 2^25, lda and ldw to 2^22; rows of A, W and
 * codes 16-byte aligned.
 * ------------------------------------------------------------------------- */

/* Rows of fp32, bf16 or fp16 (ldx in elements, rows 16-byte aligned) to codes
 * [rows][ldc] (8-byte aligned rows) and scale [rows]: scale = max |x| / 127, code = x / scale to
 * the nearest, ties to even, exactly.  A row of zeros has scale 0 and codes 0;
 * one with an infinity or a NaN has that scale, codes 0, and NaN products. */
int sf_quant_i8(const void* x, int64_t ldx, int32_t dtype, int32_t rows, int32_t cols, int8_t* codes, int64_t ldc,
                float* scale, void* stream);

typedef struct sf_gemm_i8_desc {
    int32_t M, N, K;
    const void* A;           /* [M][lda]: SF_I8 codes, or SF_F32, SF_BF16, SF_F16 rows to be quantised as sf_quant_i8 does */
    int64_t lda;
    int32_t a_dtype;
    const float* a_scale;    /* [M], with SF_I8 codes */
    const int8_t* W;         /* [N][ldw] */
    int64_t ldw;
    const float* w_scale;    /* [N] */
    const float* bias;       /* [N] or NULL */
    int32_t act;             /* sf_act */
    void* C;                 /* [M][ldc] */
    int64_t ldc;
    int32_t c_dtype;         /* SF_F32, SF_BF16 or SF_F16 */
    int32_t accumulate;      /* SF_F32 only: C += act(...) */
} sf_gemm_i8_desc;
/* Bytes of device workspace (the codes and scales of rows to be quantised; 0 for SF_I8 rows, and for up to 16
 * rows of 8192 inputs in all, which are quantised where they are multiplied), 16-byte aligned, no
 * initialisation; calls that may run concurrently need separate ones. */
size_t sf_gemm_i8_workspace_bytes(const sf_gemm_i8_desc* desc);
/* C must not overlap A. */
int sf_gemm_i8(const sf_gemm_i8_desc* desc, void* workspace, size_t workspace_bytes, void* stream);

/* Static text for a status code. */
const char* sf_strerror(int status);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif  /* SF_HIP_H_ */
