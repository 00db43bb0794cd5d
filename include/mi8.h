/*
 * mi8 - float8 linear path for gfx950 (MI355X): C ABI of libmi8.so.
 *
 * Every entry point is a plain C function over raw device pointers, sizes and a HIP stream handle.
 * Unless a function says otherwise it
 *   - returns MI8_OK (0) or a negative mi8_status; mi8_last_error() gives the text for the calling
 *     thread's most recent failure;
 *   - only enqueues work on `stream` (a hipStream_t passed as void*; NULL = the default stream): it never
 *     synchronises, never allocates or frees device memory, and keeps no state between calls that a caller could
 *     observe (the only memory of the library is per-device one-time set-up: a kernel's dynamic-LDS attribute and
 *     the compute-unit count, both latched with atomics, so first calls from several threads or on several
 *     devices are safe).  The one exception is mi8_cast_tensorwise_static, which works in a scratch array the
 *     library owns per GPU (see there);
 *   - requires every pointer to be 16-byte aligned device memory of at least the stated size.
 * All matrices are dense row-major with the row pitch given (or implied) in elements.
 *
 * The arithmetic these functions implement is the dynamic-scaling float8 training path the reference
 * reaches through torchao (reference: src/olmo_core/float8/__init__.py:133-150 converts every eligible
 * nn.Linear; src/olmo_core/float8/ao.py:152-186 carries the options).  The per-function comments cite
 * the reference interface each one stands in for.
 */
#ifndef MI8_H
#define MI8_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MI8_VERSION 100 /* major*10000 + minor*100 + patch */

typedef enum mi8_status {
    MI8_OK = 0,
    MI8_ERR_ARG = -1,         /* NULL pointer, negative size, unknown enum value */
    MI8_ERR_UNSUPPORTED = -2, /* shape or alignment outside what the kernels handle */
    MI8_ERR_LAUNCH = -3       /* HIP reported an error at launch */
} mi8_status;

/* float8 encodings (OCP): reference dtype names src/olmo_core/config.py:373-374 */
typedef enum mi8_fp8 { MI8_E4M3 = 0 /* float8_e4m3fn, max 448 */, MI8_E5M2 = 1 /* float8_e5m2, max 57344 */ } mi8_fp8;

/* high-precision element types accepted by the casts (src/olmo_core/config.py:370-372) */
typedef enum mi8_hp {
    MI8_BF16 = 0,
    MI8_F32 = 1,
    MI8_F16 = 2,  /* token permutation, routing, products of 16-bit operands, residual norms, dropout */
    MI8_RAW8 = 3, /* opaque 1-byte elements (fp8 rows): unweighted permutation only */
    MI8_F32_OF_BF16 = 4 /* GEMM outputs only: float32 that holds the values a bf16 output would (gradients of float32 weights) */
} mi8_hp;

/* flags shared by the cast entry points */
#define MI8_FLAG_POW2_SCALE 1u /* round every scale down to a power of two (ao.py:167 round_scales_to_power_of_2) */
#define MI8_FLAG_SW_CVT 2u     /* convert with integer arithmetic instead of v_cvt_pk_{fp8,bf8}_f32 (same bytes) */
#define MI8_FLAG_PAD_T128 8u   /* transposed copies of tensorwise casts: zero columns up to a multiple of 128 instead of 16 */
#define MI8_FLAG_READ_BY_FEW_ROWS 16u /* mi8_cast_rowwise: the copy is a weight that a product of at most 256 rows reads (same bytes) */
#define MI8_FLAG_AMAX_READY 4u /* grouped casts: the amax workspaces already hold the amax of x (see mi8_grouped_swiglu_*) */

/* Number of uint32 slots a tensorwise amax workspace must have. */
#define MI8_AMAX_SLOTS 2048

int mi8_version(void);
const char* mi8_last_error(void);

/* ---------------------------------------------------------------------------------------------
 * Tensorwise dynamic cast.   Stands in for torchao tensor_to_amax / amax_to_scale /
 * hp_tensor_and_scale_to_float8 as invoked by Float8Linear for TENSORWISE cast configs
 * (reference: the default AOCastConfig, src/olmo_core/float8/ao.py:76-86).
 * ------------------------------------------------------------------------------------------- */

/* Partial maxima of |x| over n contiguous elements.  Writes *n_slots_used (host int, may be NULL) and
 * fills slots[0 .. used) with the bit patterns of per-workgroup maxima (float32 bit pattern of |x|; a NaN
 * input yields a NaN pattern, which compares greatest).  slots must hold MI8_AMAX_SLOTS uint32.
 * The number of slots used depends only on n. */
int mi8_amax_partials(const void* x, int hp_dtype, int64_t n, uint32_t* slots, int32_t* n_slots_used, void* stream);

/* mi8_amax_partials for up to MI8_AMAX_BATCH tensors of one dtype in ONE launch (the input and the three weights of a
 * feed-forward block, whose tensorwise scales the reference reduces one after the other: torchao tensor_to_scale per
 * Float8Linear, reference src/olmo_core/float8/ao.py:76-86).  xs, ns, n_slots_used are HOST arrays of `count` entries;
 * tensor t's partials go to slots[t * MI8_AMAX_SLOTS ...], n_slots_used[t] (may be NULL) = mi8_amax_slots_for(ns[t]);
 * the values equal those of `count` separate mi8_amax_partials calls.  slots must hold count * MI8_AMAX_SLOTS uint32. */
#define MI8_AMAX_BATCH 8
int mi8_amax_partials_batch(const void* const* xs, const int64_t* ns, int32_t count, int hp_dtype, uint32_t* slots,
                            int32_t* n_slots_used, void* stream);

/* Number of slots mi8_amax_partials uses for n elements (host-side, no GPU work). */
int32_t mi8_amax_slots_for(int64_t n);

/* amax = max(slots[0..n_slots)), scale = float32(FP8_MAX * (1 / max(float64(amax), 1e-12))), optionally rounded
 * down to a power of two.  out[0] = scale, out[1] = amax (both float32, device). */
int mi8_scale_from_partials(const uint32_t* slots, int32_t n_slots, int fp8_dtype, uint32_t flags, float* out,
                            void* stream);

/* Tensorwise dynamic scales of many tensors in three launches: the once-per-optimizer-step refresh of all
 * float8 weight scales (reference: torchao precompute_float8_dynamic_scale_for_fsdp, called from
 * src/olmo_core/nn/transformer/model.py:1001-1008 when Float8Config.should_precompute_float8_dynamic_scale_for_fsdp,
 * src/olmo_core/float8/__init__.py:54-62).
 *   ptrs / numels: DEVICE arrays [n_tensors] of tensor base pointers (16-byte aligned) and element counts
 *   (multiples of 8 for bf16, 4 for float32); amax_workspace: uint32 [n_tensors] (overwritten);
 *   scales_out: float32 [n_tensors], the same values mi8_scale_from_partials gives tensor by tensor. */
int mi8_multi_tensor_scales(const void* const* ptrs, const int64_t* numels, int32_t n_tensors, int hp_dtype,
                            int fp8_dtype, uint32_t flags, uint32_t* amax_workspace, float* scales_out, void* stream);

/* Saturating cast of x[rows, cols] with one scale for the whole tensor.
 *   scale source: if slots != NULL the scale is reduced from slots[0..n_slots) exactly as
 *   mi8_scale_from_partials does (and written to scale_out[0] if scale_out != NULL);
 *   otherwise, if scale_in != NULL, it is read from scale_in[0] (device float32);
 *   with neither (tensors of at most 65536 elements, row-major output only: the activations of a generation
 *   step) one workgroup takes the amax, derives the scale and converts in a single launch.
 *   out   (may be NULL): fp8 [rows, ld_out], row-major with row pitch ld_out >= cols, ld_out % 16 == 0;
 *                        bytes cols..ld_out-1 of a row are not touched.
 *   out_t (may be NULL): fp8 [cols, ld_t], the transposed copy; ld_t >= rows, ld_t % 16 == 0; columns
 *                        rows..round_up(rows,16)-1 of out_t are written as zero (so that a GEMM may contract
 *                        over round_up(rows,16)), columns beyond are not touched.  With MI8_FLAG_PAD_T128 both
 *                        are multiples of 128: ld_t >= round_up(rows,128), zeros up to there (the persistent GEMM
 *                        contracts whole 128-byte steps).
 * cols % 16 == 0 is required.  The GEMMs accept any operand pitch that is a multiple of 16. */
int mi8_cast_tensorwise(const void* x, int hp_dtype, int64_t rows, int64_t cols, const uint32_t* slots,
                        int32_t n_slots, const float* scale_in, int fp8_dtype, uint32_t flags, void* out,
                        int64_t ld_out, void* out_t, int64_t ld_t, float* scale_out, void* stream);

/* mi8_cast_tensorwise for up to MI8_CAST_BATCH tensors (an input and the weights of a layer) in one launch, of bf16 and
 * float32 mixed.  A tensor with neither slots nor scale_in has its amax taken first, into amax_ws, in one more launch for
 * all of those.  Per tensor the arguments of mi8_cast_tensorwise (pad_t128: MI8_FLAG_PAD_T128 for this tensor; scale_out
 * is always written); bytes and scales are those of the separate calls. */
#define MI8_CAST_BATCH 8
typedef struct {
    const void* x;
    int64_t rows, cols;
    const uint32_t* slots;
    const float* scale_in;
    uint32_t* amax_ws; /* uint32 [MI8_AMAX_SLOTS], where slots and scale_in are NULL */
    void* out;
    int64_t ld_out;
    void* out_t;
    int64_t ld_t;
    float* scale_out;
    int32_t n_slots, hp_dtype, pad_t128;
} mi8_cast_item;
int mi8_cast_tensorwise_batch(const mi8_cast_item* items, int32_t count, int fp8_dtype, uint32_t flags, void* stream);

/* A scale per row with a row-major copy, and a scale per column with a transposed copy, of up to MI8_CAST_BATCH tensors:
 * per tensor the results of mi8_cast_rowwise and mi8_cast_colwise_t, two launches for all of them.
 *   out_rows: fp8 [rows, ld_rows]; row_scale: float32 [rows]; out_t: fp8 [cols, ld_t], ld_t >= round_up(rows, 128), zero
 *   from column `rows` to round_up(rows, 128) and not written beyond; col_scale: float32 [cols]; workspace: uint32 [mi8_two_cast_workspace_words(rows, cols)],
 *   16-byte aligned, contents on entry unimportant.  group_rows (0: rows): every group_rows rows, a multiple of 128 that
 *   divides rows, have column scales of their own, col_scale [rows / group_rows, cols] (the weights of experts). */
typedef struct {
    const void* x;
    int64_t rows, cols;
    void* out_rows;
    int64_t ld_rows;
    float* row_scale;
    void* out_t;
    int64_t ld_t;
    float* col_scale;
    uint32_t* workspace;
    int64_t group_rows;
    int32_t hp_dtype;
} mi8_two_cast_item;
int64_t mi8_two_cast_workspace_words(int64_t rows, int64_t cols);
int mi8_cast_rows_and_colwise_t_batch(const mi8_two_cast_item* items, int32_t count, int fp8_dtype, uint32_t flags, void* stream);

/* The dynamic tensorwise cast in one call for callers that cannot allocate device memory or hand over a
 * workspace (code under HIP graph capture, tight serving loops, harnesses that forbid hipMalloc): amax pass +
 * cast pass as mi8_amax_partials followed by mi8_cast_tensorwise(slots), with the partial maxima kept in an 8 KiB
 * array that is part of the library's device image (one copy per GPU, held until the process ends) instead of a
 * caller-owned workspace.  No counterpart in the reference.  Same outputs, bytes and scale as the two-call
 * route.  Limits: rows, cols <= MI8_STATIC_CAST_MAX_DIM and rows * cols <= MI8_STATIC_CAST_MAX_ELEMS, larger
 * inputs are refused with MI8_ERR_UNSUPPORTED.  All calls on one GPU share that GPU's array: calls that may
 * overlap on one GPU (different streams, different threads, replays of two captured graphs side by side) race and
 * nothing in the library guards against it; calls ordered on one stream do not.  The first call on a device looks
 * up the array's address (hipGetSymbolAddress, a host-side query that is no stream operation): make one call per
 * device outside of any stream capture before capturing calls into a graph. */
#define MI8_STATIC_CAST_MAX_DIM ((int64_t)1 << 22)
#define MI8_STATIC_CAST_MAX_ELEMS ((int64_t)1 << 32)
int mi8_cast_tensorwise_static(const void* x, int hp_dtype, int64_t rows, int64_t cols, int fp8_dtype, uint32_t flags,
                               void* out, int64_t ld_out, void* out_t, int64_t ld_t, float* scale_out, void* stream);


/* ---------------------------------------------------------------------------------------------
 * Axiswise ("rowwise" recipe) dynamic casts: AXISWISE cast configs of the rowwise recipes
 * (reference: AOFloat8LinearRecipe.rowwise / rowwise_with_gw_hp, src/olmo_core/float8/ao.py:100-109).
 * ------------------------------------------------------------------------------------------- */

/* One scale per row (amax over the last axis): out fp8 [rows, ld_out] (ld_out >= cols, ld_out % 16 == 0),
 * scale_out float32 [rows].  cols % 16 == 0, cols <= 65536. Single pass over x. */
int mi8_cast_rowwise(const void* x, int hp_dtype, int64_t rows, int64_t cols, int fp8_dtype, uint32_t flags,
                     void* out, int64_t ld_out, float* scale_out, void* stream);

/* The two per-row casts of an expert layer that is not differentiated, bf16 to e4m3, with the bytes and scales of the
 * separate steps.  gather_cast_rows: row r of out [tokens * top_k, ld_out] is row indices[r] / top_k of x
 * [tokens, cols] (an index outside [0, tokens * top_k): a row of zeros).  swiglu_cast_rows: rows of silu(x1) * x3,
 * rounded to bf16 first.  Same limits as mi8_cast_rowwise. */
int mi8_moe_gather_cast_rows(const void* x, int64_t tokens, int64_t cols, const int32_t* indices, int32_t top_k,
                             uint32_t flags, void* out, int64_t ld_out, float* scale_out, void* stream);
int mi8_swiglu_cast_rows(const void* x1, const void* x3, int64_t rows, int64_t cols, uint32_t flags, void* out,
                         int64_t ld_out, float* scale_out, void* stream);

/* Number of uint32 a column-amax workspace needs for a [rows, cols] input. */
int64_t mi8_colamax_workspace_slots(int64_t rows, int64_t cols);

/* One scale per column (amax over axis 0), output written TRANSPOSED: out_t fp8 [cols, ld_t] (pad columns
 * rows..round_up(rows,16)-1 zero), scale_out float32 [cols].  This is the operand layout the grad_weight GEMM and the
 * axiswise grad_input GEMM consume.  workspace: mi8_colamax_workspace_slots(rows, cols) uint32.
 * Two kernels: column amax, then cast + transpose. */
int mi8_cast_colwise_t(const void* x, int hp_dtype, int64_t rows, int64_t cols, int fp8_dtype, uint32_t flags,
                       uint32_t* workspace, void* out_t, int64_t ld_t, float* scale_out, void* stream);

/* ---------------------------------------------------------------------------------------------
 * Scaled float8 GEMM.  Stands in for torch._scaled_mm as driven by torchao's float8 mm dispatch
 * (the three GEMMs of one linear: output, grad_input, grad_weight).
 *   out[M, N] = bf16( (sum_k A[m,k] * B[n,k]) * (1/sa) * (1/sb) ), fp32 accumulation on fp8 MFMA.
 *   A: fp8 [M, lda] row-major, B: fp8 [N, ldb] row-major - both operands K-contiguous; K % 16 == 0,
 *   lda, ldb % 16 == 0.  a_dtype / b_dtype may differ (e5m2 x e4m3 for the gradient GEMMs).
 *   sa: quantisation scale(s) of A - one float32 if sa_rows == 0, else float32 [M]; sb likewise ([N]).
 *   out: [M, ldc] of out_dtype (MI8_BF16, MI8_F32 or MI8_F32_OF_BF16), ldc >= N.
 *   variant: -1 picks a tile configuration from the shape; 0..mi8_gemm_num_variants()-1 forces one.
 * ------------------------------------------------------------------------------------------- */
int mi8_gemm_fp8(const void* a, int a_dtype, int64_t lda, const void* b, int b_dtype, int64_t ldb, int64_t M,
                 int64_t N, int64_t K, const float* sa, int sa_is_vector, const float* sb, int sb_is_vector,
                 void* out, int out_dtype, int64_t ldc, int variant, void* stream);

/* out[M, N] += the product mi8_gemm_fp8 would write: the new term is rounded to out_dtype first and the sum of the
 * two is formed in float32 and rounded once, i.e. exactly what `out = out + gemm(...)` gives when both terms are
 * tensors of out_dtype.  This is how the grad_input of a block whose input feeds two linears (w1 and w3 of the
 * feed-forward block, src/olmo_core/nn/feed_forward.py:171) is summed by autograd; here the second GEMM adds into the
 * first one's output and the separate elementwise pass over [M, N] disappears.  Arguments as mi8_gemm_fp8 (the kernel
 * is chosen by shape), out_dtype MI8_BF16 or MI8_F32: MI8_F32_OF_BF16 is for products that are not added to anything, here
 * and in the other entry points that add. */
int mi8_gemm_fp8_accumulate(const void* a, int a_dtype, int64_t lda, const void* b, int b_dtype, int64_t ldb, int64_t M,
                            int64_t N, int64_t K, const float* sa, int sa_is_vector, const float* sb, int sb_is_vector,
                            void* out, int out_dtype, int64_t ldc, void* stream);

/* The two input projections of a SwiGLU feed-forward block and the activation between them and the output projection
 * in one launch (reference: src/olmo_core/nn/feed_forward.py:171, `self.w2(F.silu(self.w1(x)) * self.w3(x))`):
 *   x1[M, H] = bf16((A . B1^T) / sa / sb1),  x3[M, H] = bf16((A . B3^T) / sa / sb3)   (what mi8_gemm_fp8 writes, bit for bit)
 *   h[M, H]  = silu(x1) * x3                                                          (what mi8_swiglu_fwd writes, bit for bit)
 *   slots_h[0 .. *n_slots_used) = partial maxima of |h| as mi8_swiglu_fwd produces them for the cast of h that follows.
 * Every workgroup computes matching 128-column tiles of x1 and x3 and forms h in its epilogue, so x1 and x3 are written
 * once and never read back.  A fp8 [M, lda]; B1, B3 fp8 [H, ldb] of one type; single scales (float32 [1] each);
 * x1, x3, h bf16 [M, ldc]; slots_h must hold MI8_AMAX_SLOTS uint32.  Needs M >= 256, H >= 128, H % 8 == 0,
 * K % 128 == 0, ldc < 2^22 (MI8_ERR_UNSUPPORTED otherwise: run the three calls it stands for).
 * x_codes: NULL, or uint16[mi8_rowseg_code_count(M, H)] that receives the row-segment codes of the element-wise
 * larger of x1 and x3 (what mi8_rowseg_max_codes(x1, x3) computes; needs H % 64 == 0), for the backward pass's
 * mi8_swiglu_bwd_amax_from_codes. */
int mi8_gemm_fp8_swiglu_matches_separate(int64_t M, int64_t H, int64_t K); /* host only: 1 if the fused launch takes
    the shape, which has more than 96 tiles of 256 x 256: the library then cuts neither projection along K, so that the bits agree as well */
int mi8_gemm_fp8_swiglu_pays(int64_t M, int64_t H, int64_t K); /* host only: 1 for those shapes and, with K >= 512, for those of fewer
    tiles whose projections would not be cut along K */
int mi8_gemm_fp8_swiglu(const void* a, int a_dtype, int64_t lda, const void* b1, const void* b3, int b_dtype, int64_t ldb,
                        int64_t M, int64_t H, int64_t K, const float* sa, const float* sb1, const float* sb3, void* x1,
                        void* x3, void* h, int64_t ldc, uint32_t* slots_h, int32_t* n_slots_used, uint16_t* x_codes,
                        void* stream);

/* The same product with K cut into `splits` slices, for problems whose few output tiles would leave most of the
 * GPU idle (a few hundred rows of A against a weight matrix): every slice is summed by its own workgroups into
 * an fp32 plane of `workspace`, a second kernel adds the planes in slice order (results do not depend on
 * scheduling), applies the scales and rounds.  Arguments as mi8_gemm_fp8; splits in 1..min(64, ceil(K/128));
 * workspace: 16-byte aligned device memory of mi8_gemm_splitk_workspace_bytes(M, N, splits) bytes, owned by the
 * caller, free for reuse once the call's work on `stream` is done.  mi8_gemm_splitk_suggest returns the number
 * of slices the library would use for a shape (1: call mi8_gemm_fp8 instead).  Up to 64 rows K is summed in eighths
 * (slices of ceil(ceil(K / 128) / 8) steps) whichever entry point or kernel runs, mi8_few_rows_* included, so all of
 * them give one result.  Where one workgroup per tile adds the slices sooner, mi8_gemm_fp8_splitk does it that way (the
 * same sums; the workspace is then not touched).  No counterpart upstream: the reference leaves the choice of GEMM algorithm to torch._scaled_mm's backend. */
int mi8_gemm_fp8_splitk(const void* a, int a_dtype, int64_t lda, const void* b, int b_dtype, int64_t ldb,
                        int64_t M, int64_t N, int64_t K, const float* sa, int sa_is_vector, const float* sb,
                        int sb_is_vector, void* out, int out_dtype, int64_t ldc, int splits, void* workspace,
                        int64_t workspace_bytes, void* stream);
/* out += that product, summed as mi8_gemm_fp8_accumulate does. */
int mi8_gemm_fp8_splitk_accumulate(const void* a, int a_dtype, int64_t lda, const void* b, int b_dtype, int64_t ldb,
                                   int64_t M, int64_t N, int64_t K, const float* sa, int sa_is_vector, const float* sb,
                                   int sb_is_vector, void* out, int out_dtype, int64_t ldc, int splits, void* workspace,
                                   int64_t workspace_bytes, void* stream);
int mi8_gemm_splitk_suggest(int64_t M, int64_t N, int64_t K);
int64_t mi8_gemm_splitk_workspace_bytes(int64_t M, int64_t N, int splits);

/* Up to MI8_GEMM_BATCH products of one pair of fp8 types in ONE launch, each as mi8_gemm_fp8 (or, where the library cuts
 * the product along K, mi8_gemm_fp8_splitk with the suggested slices) gives it, bit for bit.  add_to_previous: the product
 * is added to the output of the one before it (same M, N, out, ldc, out_dtype), as mi8_gemm_fp8_accumulate does; otherwise
 * outputs must not overlap.  For the products of a layer of ordinary size, which fill a part of the chip each: whether
 * one launch is estimated faster than one per product is what mi8_gemm_fp8_batch_pays returns (1 or 0; 0 for what
 * mi8_gemm_fp8_batch refuses). */
#define MI8_GEMM_BATCH 8
typedef struct {
    const void* a;
    int64_t lda;
    const void* b;
    int64_t ldb;
    int64_t M, N, K;
    const float* sa;
    const float* sb;
    void* out;
    int64_t ldc;
    int32_t sa_is_vector, sb_is_vector, out_dtype, add_to_previous;
} mi8_gemm_product;
int mi8_gemm_fp8_batch_pays(const mi8_gemm_product* products, int32_t count);
int mi8_gemm_fp8_batch(const mi8_gemm_product* products, int32_t count, int a_dtype, int b_dtype, void* stream);

/* Number of GEMM kernel variants compiled in (variant ids 0..n-1; -1 lets the library choose by shape).  Which id is
 * which kernel may change with the library: look a variant up by its name. */
int mi8_gemm_num_variants(void);
const char* mi8_gemm_variant_name(int variant);
/* Host only: the variant that -1 stands for in mi8_gemm_fp8 (accumulate != 0: in mi8_gemm_fp8_accumulate) when ldc == N, the
 * pointers are 16-byte aligned and the scales of one kind; -1 for an empty product and for a sum in MI8_F32_OF_BF16. */
int mi8_gemm_variant_for(int64_t M, int64_t N, int64_t K, int out_dtype, int accumulate);

/* ---------------------------------------------------------------------------------------------
 * Ragged grouped operations for the dropless-MoE expert layer.  The reference runs this layer in bf16 through
 * grouped_gemm.ops.gmm(x, w, batch_sizes, trans_b) or a per-expert loop (src/olmo_core/nn/moe/mlp.py:256-270);
 * these entry points are its float8 counterpart with the axiswise recipe applied to every expert's slice
 * independently.  Rows of the activation matrix form consecutive groups; group_sizes is an int64 device array
 * (as DroplessMoEMLP.forward receives it, mlp.py:272-280) that is never copied to the host.
 * ------------------------------------------------------------------------------------------- */

/* Upper bound of the padded token axis used by the grouped transposed layouts: every group's segment starts at a
 * multiple of 128 (T rounded up to 128, plus 128 per group after the first). */
int64_t mi8_grouped_padded_rows(int64_t T, int32_t num_groups);

/* Per-group, per-column dynamic cast with transposed output: for group e (rows R_e of x[T, cols]) the scale of
 * column c is taken over R_e only; out_t[c, 128 * tiles_before(e) + (r - first row of e)] holds the bytes, the
 * rest of each 128-aligned segment is zero.  amax_ws: uint32 [num_groups * cols], ZERO on entry.
 * scale_out: float32 [num_groups, cols] (rows of empty groups are not written).
 * ld_t >= mi8_grouped_padded_rows(T, num_groups), ld_t % 16 == 0.  With equal group sizes that are multiples of
 * 128 this is a batched transpose-cast (used for the expert weights). */
int mi8_grouped_cast_colwise_t(const void* x, int hp_dtype, int64_t T, int64_t cols, const int64_t* group_sizes,
                               int32_t num_groups, int fp8_dtype, uint32_t flags, uint32_t* amax_ws, void* out_t,
                               int64_t ld_t, float* scale_out, void* stream);

/* The same two passes (amax, cast) also produce the per-row cast of x that the forward / grad_input GEMMs take:
 * out_rows fp8 [T, ld_rows] row-major with one scale per row (row_scale_out float32 [T], the values
 * mi8_cast_rowwise gives), saving the separate pass over x.  row_amax_ws: uint32 [T], ZERO on entry.  Both
 * products use fp8_dtype and flags.  Rows beyond the last group (if the sizes sum to less than T) are not
 * written. */
int mi8_grouped_cast_rows_and_colwise_t(const void* x, int hp_dtype, int64_t T, int64_t cols,
                                        const int64_t* group_sizes, int32_t num_groups, int fp8_dtype, uint32_t flags,
                                        uint32_t* amax_ws, void* out_t, int64_t ld_t, float* scale_out,
                                        uint32_t* row_amax_ws, void* out_rows, int64_t ld_rows, float* row_scale_out,
                                        void* stream);

/* h = silu(x1) * x2 of the expert layer (src/olmo_core/nn/moe/mlp.py:286-291; bf16 [T, cols], the rounding points
 * of mi8_swiglu_fwd) together with the amax pass of the cast that follows: amax_ws (uint32 [num_groups * cols]) and
 * row_amax_ws (uint32 [T]), both ZERO on entry, receive the per-(group, column) and per-row amax of h, so that
 * mi8_grouped_cast_rows_and_colwise_t(h, ..., flags | MI8_FLAG_AMAX_READY, ...) skips its own first pass.  Rows
 * beyond the last group are not written.  The backward form writes the gradients g1 (of x1) and g2 (of x2) of that
 * product for the incoming gradient gh, each with its own pair of amax workspaces. */
int mi8_grouped_swiglu_fwd(const void* x1, const void* x2, int64_t T, int64_t cols, const int64_t* group_sizes,
                           int32_t num_groups, void* h, uint32_t* amax_ws, uint32_t* row_amax_ws, void* stream);
int mi8_grouped_swiglu_bwd(const void* x1, const void* x2, const void* gh, int64_t T, int64_t cols,
                           const int64_t* group_sizes, int32_t num_groups, void* g1, void* g2, uint32_t* amax_ws1,
                           uint32_t* row_amax_ws1, uint32_t* amax_ws2, uint32_t* row_amax_ws2, void* stream);

/* out[R_e, :N] = (A[R_e, :K] . B_e[:N, :K]^T) / sa[r] / sb_e[n]   for every group e.
 *   A fp8 [T, lda]; B_e = b + e * b_group_stride (bytes), N rows of pitch ldb; sa float32 [T];
 *   sb_e = sb + e * sb_group_stride (floats), N values; out [T, ldc] of out_dtype.
 *   lda < 2^27, or T * lda < 2^32. */
int mi8_grouped_gemm_fp8(const void* a, int a_dtype, int64_t lda, const void* b, int b_dtype, int64_t ldb,
                         int64_t b_group_stride, const int64_t* group_sizes, int32_t num_groups, int64_t T, int64_t N,
                         int64_t K, const float* sa, const float* sb, int64_t sb_group_stride, void* out,
                         int out_dtype, int64_t ldc, void* stream);

/* out[R_e, :N] += that product, summed as mi8_gemm_fp8_accumulate does (the two grad_input terms of the expert
 * layer, src/olmo_core/nn/moe/mlp.py:286-291). */
int mi8_grouped_gemm_fp8_accumulate(const void* a, int a_dtype, int64_t lda, const void* b, int b_dtype, int64_t ldb,
                                    int64_t b_group_stride, const int64_t* group_sizes, int32_t num_groups, int64_t T,
                                    int64_t N, int64_t K, const float* sa, const float* sb, int64_t sb_group_stride,
                                    void* out, int out_dtype, int64_t ldc, void* stream);

/* out[rows of group e, :N] = (a1 . B1_e^T) / sa1 / sb1_e + (a2 . B2_e^T) / sa2 / sb2_e, both products summed in one
 * float32 accumulation and rounded once to bf16: the grad_input of an expert layer whose input feeds two projections
 * (gx = g1 . W1 + g2 . W3, src/olmo_core/nn/moe/mlp.py:272-292 in backward) as one launch instead of
 * mi8_grouped_gemm_fp8 + mi8_grouped_gemm_fp8_accumulate, without the read-modify-write of the output.  a1 [T, K1] and
 * a2 [T, K2] share the row pitch lda; B1_e [N, K1] and B2_e [N, K2] the row pitch ldb and the group stride; sa1, sa2:
 * float32 [T]; sb1, sb2: float32, group e at + e * sb_group_stride, N values.  EVERY SCALE MUST BE AN EXACT POWER OF TWO
 * (what the casts write under MI8_FLAG_POW2_SCALE): the scales are applied inside the matrix instructions as exponents,
 * a mantissa is ignored.  The sum differs from the two-call route by one rounding (that route rounds each product to bf16
 * before adding).  Shapes: mi8_grouped_gemm_fp8_dual_supported (T, N >= 256, N % 8 == 0, K1 and K2 multiples of 256);
 * out: bf16 [T, ldc], ldc % 8 == 0. */
int mi8_grouped_gemm_fp8_dual_supported(int64_t T, int64_t N, int64_t K1, int64_t K2);
int mi8_grouped_gemm_fp8_dual(const void* a1, const void* a2, int a_dtype, int64_t lda, const void* b1, const void* b2,
                              int b_dtype, int64_t ldb, int64_t b_group_stride, const int64_t* group_sizes,
                              int32_t num_groups, int64_t T, int64_t N, int64_t K1, int64_t K2, const float* sa1,
                              const float* sa2, const float* sb1, const float* sb2, int64_t sb_group_stride, void* out,
                              int64_t ldc, void* stream);

/* out[e, :N, :Kl] = (A_t[:N, S_e] . B_t[:Kl, S_e]^T) / sa[e, n] / sb[e, k]: the contraction runs over group e's
 * 128-aligned segment S_e of the padded token axis (layout written by mi8_grouped_cast_colwise_t; both operands
 * have pitch ld_t).  Empty groups produce zeros.  out is [num_groups, N, Kl] contiguous. */
int mi8_grouped_wgrad_fp8(const void* a_t, int a_dtype, const void* b_t, int b_dtype, int64_t ld_t,
                          const int64_t* group_sizes, int32_t num_groups, int64_t T, int64_t N, int64_t Kl,
                          const float* sa, const float* sb, void* out, int out_dtype, void* stream);

/* A generation step of a SwiGLU block (tensorwise e4m3, evaluation): h = silu(x1) * x3 in bf16 [M, H], x1 = x B1^T,
 * x3 = x B3^T, with the partial maxima of |h| (slots_h: uint32 [MI8_AMAX_SLOTS], *n_slots_used of them written), in one
 * launch; x1 and x3 are not written.  1 <= M <= 64, H % 8 == 0 and H <= 16 * MI8_AMAX_SLOTS, K % 16 == 0, pitches multiples
 * of 16, pointers 16-byte aligned.
 *   x_is_fp8 != 0: x is e4m3 [M, lda] with its scale sx; otherwise bf16, contiguous (lda == K), at most 16 rows and 16384
 *   elements: every workgroup then takes the amax and quantises (flags: MI8_FLAG_POW2_SCALE) what it reads. */
int mi8_few_rows_swiglu(const void* x, int x_is_fp8, int64_t lda, const float* sx, const void* b1, const void* b3,
                        int64_t ldb, int64_t M, int64_t H, int64_t K, const float* sb1, const float* sb3, uint32_t flags,
                        void* h, uint32_t* slots_h, int32_t* n_slots_used, void* stream);

/* out[M, ldc] (bf16) = q(x) B^T scaled, x bf16 [M, lda], M <= 16, quantised to e4m3 by the launch with the scale of the
 * partial maxima `slots` (mi8_scale_from_partials): the bits of mi8_cast_tensorwise followed by mi8_gemm_fp8.
 * M * K <= 65536, N % 8 == 0, K % 16 == 0, lda % 8 == 0, ldb % 16 == 0, ldc % 4 == 0, pointers 16-byte aligned. */
int mi8_few_rows_cast_gemm(const void* x, int64_t lda, const uint32_t* slots, int32_t n_slots, const void* b, int64_t ldb,
                           int64_t M, int64_t N, int64_t K, const float* sb, uint32_t flags, void* out, int64_t ldc,
                           void* stream);

/* ---------------------------------------------------------------------------------------------
 * SwiGLU pointwise kernels between the projections of the feed-forward block
 * (reference: src/olmo_core/nn/feed_forward.py:171  w2(silu(w1 x) * w3 x)).
 *   forward : h = bf16(bf16(silu(x1)) * x3), optionally also the amax partials of h.
 *   backward: given gh, g1 = gh * x3 * silu'(x1), g3 = gh * silu(x1), evaluated with bf16 roundings of
 *             torch's elementwise autograd formulas; optionally amax partials of g1 and g3.
 * All tensors bf16, n elements, n % 8 == 0.
 * ------------------------------------------------------------------------------------------- */
int mi8_swiglu_fwd(const void* x1, const void* x3, void* h, int64_t n, uint32_t* slots_h, void* stream);
int mi8_swiglu_bwd(const void* x1, const void* x3, const void* gh, void* g1, void* g3, int64_t n,
                   uint32_t* slots_g1, uint32_t* slots_g3, void* stream);

/* The feed-forward block's backward needs g1 and g3 only as fp8 operands.  Two passes that never write them in bf16:
 * mi8_swiglu_bwd with g1 = g3 = NULL leaves just the amax partials of what it would have written; this entry point
 * then recomputes the gradients tile by tile and writes the tensorwise casts of both (row-major [rows, ld_out]
 * and/or transposed [cols, ld_t] copies, the layouts of mi8_cast_tensorwise; the same layouts for both outputs) with
 * the scales taken from those partials.  Bytes and scales equal mi8_swiglu_bwd + mi8_cast_tensorwise on each output. */
int mi8_swiglu_bwd_cast(const void* x1, const void* x3, const void* gh, int64_t rows, int64_t cols,
                        const uint32_t* slots_g1, const uint32_t* slots_g3, int32_t n_slots, int fp8_dtype, uint32_t flags,
                        void* out1, void* out3, int64_t ld_out, void* out1_t, void* out3_t, int64_t ld_t,
                        float* scale_out1, float* scale_out3, void* stream);

/* The amax of g1 and g3 without computing every element (the tensorwise scale of the gradient operands,
 * torchao tensor_to_amax over what src/olmo_core/nn/feed_forward.py:171 back-propagates).
 *
 * A row segment is 64 consecutive columns of a row (the last one of a row may be shorter).  Its code is the largest
 * magnitude in it as a 16-bit integer: the exponent and mantissa bits of the bf16 value, which grow with the
 * magnitude and add like logarithms.  codes = uint16[mi8_rowseg_code_count(rows, cols)], segment (r, c / 64) at
 * index (c / 64) * rows + r.  mi8_rowseg_max_codes computes them for one tensor, or for the element-wise larger of
 * two (b may be NULL); mi8_gemm_fp8_codes and mi8_gemm_fp8_swiglu write them for the tensors they produce.
 *
 * The sum of a segment's codes in gh and in (x1, x3) bounds log2 of both gradients on all its elements.
 * mi8_swiglu_bwd_amax_from_codes computes exactly only the segments whose bound could still raise the maxima (all
 * segments that may hold a non-finite input among them) and leaves state[0] = amax bits of g1, state[1] = of g3
 * (float32 bit patterns, the values mi8_swiglu_bwd's partials reduce to; pass them to mi8_swiglu_bwd_cast with
 * n_slots = 1); state is uint32[mi8_swiglu_amax_state_words(rows, cols)], overwritten (nothing to clear beforehand).
 * Tensors are bf16 [rows, cols] contiguous, cols % 8 == 0; the code arrays 16-byte aligned. */
int64_t mi8_rowseg_code_count(int64_t rows, int64_t cols);
int64_t mi8_swiglu_amax_state_words(int64_t rows, int64_t cols);
int mi8_rowseg_max_codes(const void* a, const void* b, int64_t rows, int64_t cols, uint16_t* codes, void* stream);
int mi8_swiglu_bwd_amax_from_codes(const void* x1, const void* x3, const void* gh, int64_t rows, int64_t cols,
                                   const uint16_t* gh_codes, const uint16_t* x_codes, uint32_t* state, void* stream);
/* out = mi8_gemm_fp8(a, b) for single scales and a bf16 output, with the row-segment codes of out written by the
 * epilogue (the gradient reaching h = silu(x1) * x3, grad_h = grad_y W2 of src/olmo_core/nn/feed_forward.py:171, is
 * produced this way).  mi8_gemm_fp8_codes_supported: shapes it takes (those mi8_gemm_fp8 runs on the same kernel, so
 * out has the same bits; N % 64 == 0; ldc < 2^22). */
int mi8_gemm_fp8_codes_supported(int64_t M, int64_t N, int64_t K);
int mi8_gemm_fp8_codes(const void* a, int a_dtype, int64_t lda, const void* b, int b_dtype, int64_t ldb, int64_t M, int64_t N,
                       int64_t K, const float* sa, const float* sb, void* out, int64_t ldc, uint16_t* codes, void* stream);

/* ---------------------------------------------------------------------------------------------
 * Token permutation around the expert GEMMs of a mixture-of-experts layer.  These replace the copy kernels of
 * src/olmo_core/kernels/moe.py (gather :101-139, padded_scatter / scatter :142-192, scatter_wgrad :251-298,
 * binned_gather :377-406, binned_scatter :409-441, binned_scatter_wgrad :512-537), which the autograd functions
 * of src/olmo_core/ops/moe.py:26-205 call.
 *
 *   tokens, hidden : x is [tokens, hidden]; every token has top_k slots, slot s belongs to token s / top_k.
 *   indices        : int32 [tokens * top_k], the slot held by each row of the expert-sorted side
 *                    (argsort of the flattened expert assignment, ops/moe.py / parallel_mlp.py:102-125).
 *   weights        : [tokens * top_k] of w_dtype (MI8_BF16 / MI8_F16 / MI8_F32) indexed by slot, or NULL.
 *   bins           : int32 [experts], inclusive prefix sums of the tokens per expert (binned forms).
 * Products are formed in float32 and rounded once to the element type, as the reference kernels do.  Rows are
 * moved with 16-byte accesses when hidden * element size is a multiple of 16 and the buffers are 16-byte
 * aligned, element by element otherwise.  An index outside [0, tokens * top_k) is treated as a dropped token.
 * ------------------------------------------------------------------------------------------- */

/* indices [n]: the slots 0..n-1 stably sorted by expert id (ids: int32 or int64 [n], taken modulo 2^32); bin_ids [n]:
 * their ids; bins [experts]: inclusive prefix sums of sizes.  n up to mi8_moe_sort_slots_max(). */
int64_t mi8_moe_sort_slots_max(void);
int mi8_moe_sort_slots(const void* ids, int ids_are_64, int64_t n, const int64_t* sizes, int32_t experts, int32_t* indices,
                       int32_t* bin_ids, int32_t* bins, void* stream);

/* The same for more slots and up to 256 experts, as long as ceil(n / 1024)^2 * (experts + 2) <= 3e8 (2^20 slots of 256 experts,
 * 2^21 of 64).  workspace: int32 [mi8_moe_sort_workspace_words(n, experts)] (0: not taken), overwritten. */
int64_t mi8_moe_sort_workspace_words(int64_t n, int32_t experts);
int mi8_moe_sort_many_slots(const void* ids, int ids_are_64, int64_t n, const int64_t* sizes, int32_t experts, int32_t* workspace,
                            int32_t* indices, int32_t* bin_ids, int32_t* bins, void* stream);

/* out[i, :] = x[indices[i] / top_k, :] * weights[indices[i]]           out: [tokens * top_k, hidden] */
int mi8_moe_gather(const void* x, int dtype, int64_t tokens, int64_t hidden, const int32_t* indices,
                   const void* weights, int w_dtype, int32_t top_k, void* out, void* stream);

/* mi8_moe_gather (weights NULL: unweighted) followed by mi8_grouped_cast_rows_and_colwise_t, without the gathered high-precision
 * tensor in between: the token rows are read through `indices` in both passes (x stays cache resident: every token
 * row is read top_k times), and only the float8 products are written - the per-row cast [tokens * top_k, ld_rows]
 * with its scales and the per-(group, column) transposed cast with its scales, i.e. the operands of the expert
 * GEMMs of a dropless mixture-of-experts layer (the copy kernel of src/olmo_core/kernels/moe.py:42-139 fused with the
 * quantisation that follows it in a float8 expert layer; its backward stays mi8_moe_scatter).  With weights (the
 * backward of the weighted scatter: grad_output rows times the router weight of the slot) every product is rounded to
 * the element type before it is quantised, as mi8_moe_gather writes it.  A slot index outside
 * [0, tokens * top_k) reads as a row of zeros.  Workspaces, outputs and group semantics as
 * mi8_grouped_cast_rows_and_colwise_t with T = tokens * top_k; bytes and scales equal the two-call route. */
int mi8_moe_gather_cast_rows_and_colwise_t(const void* x, int hp_dtype, int64_t tokens, int64_t cols,
                                           const int32_t* indices, int32_t top_k, const void* weights, int w_dtype,
                                           const int64_t* group_sizes,
                                           int32_t num_groups, int fp8_dtype, uint32_t flags, uint32_t* amax_ws,
                                           void* out_t, int64_t ld_t, float* scale_out, uint32_t* row_amax_ws,
                                           void* out_rows, int64_t ld_rows, float* row_scale_out, void* stream);

/* out[e, j, :] = the j-th token row of expert e (scaled), zero rows beyond the expert's token count; tokens
 * beyond `capacity` are dropped.                                          out: [experts, capacity, hidden] */
int mi8_moe_binned_gather(const void* x, int dtype, int64_t tokens, int64_t hidden, const int32_t* indices,
                          const void* weights, int w_dtype, const int32_t* bins, int32_t experts, int64_t capacity,
                          int32_t top_k, void* out, void* stream);

/* out[t, :] = sum over the top_k slots s of token t of round(x[row holding s, :] * weights[s]), summed in float32
 * in slot order and rounded once (top_k == 1: a pure move).  x: [tokens * top_k, hidden], out: [tokens, hidden].
 * inverse_workspace: int32 [tokens * top_k], overwritten. */
int mi8_moe_scatter(const void* x, int dtype, int64_t tokens, int64_t hidden, const int32_t* indices,
                    const void* weights, int w_dtype, int32_t top_k, int32_t* inverse_workspace, void* out,
                    void* stream);

/* The same from the binned layout x: [experts, capacity, hidden]; dropped tokens contribute zero. */
int mi8_moe_binned_scatter(const void* x, int dtype, int64_t tokens, int64_t hidden, const int32_t* indices,
                           const void* weights, int w_dtype, const int32_t* bins, int32_t experts, int64_t capacity,
                           int32_t top_k, int32_t* inverse_workspace, void* out, void* stream);

/* Gradient of the scatter weights: out[indices[i]] = dot(x[i, :], grad[indices[i] / top_k, :]) accumulated in
 * float32.  x: [tokens * top_k, hidden], grad: [tokens, hidden], out: [tokens * top_k] of dtype. */
int mi8_moe_scatter_wgrad(const void* x, const void* grad, int dtype, int64_t tokens, int64_t hidden,
                          const int32_t* indices, int32_t top_k, void* out, void* stream);

/* The same from the binned layout; slots of dropped tokens get zero. */
int mi8_moe_binned_scatter_wgrad(const void* x, const void* grad, int dtype, int64_t tokens, int64_t hidden,
                                 const int32_t* indices, const int32_t* bins, int32_t experts, int64_t capacity,
                                 int32_t top_k, void* out, void* stream);

/* A sequence of calls of this library made by one call: the launches of a layer whose kernels are shorter than the calls from
 * an interpreter that make them.  `words`: per call the number mi8_plan_function(name) gives (-1: cannot be planned) and
 * the call's arguments in order, one word each: a number; for an address 0 (NULL), -1 (the stream), -2
 * (n_slots_used: not wanted) or (buffer + 1) << 48 | offset into buffers[buffer]; for an array of items (mi8_cast_item, mi8_two_cast_item,
 * mi8_gemm_product) their number and their fields in order.  Ends with the first
 * call that fails, returning its status.  Nothing is kept between calls; buffers must outlive the work on `stream`. */
int mi8_plan_function(const char* name);
int mi8_run_plan(const int64_t* words, int64_t n_words, const void* const* buffers, int32_t n_buffers, void* stream);
/* partial maxima that mi8_gemm_fp8_swiglu writes for these sizes on the current device (its *n_slots_used) */
int32_t mi8_gemm_fp8_swiglu_slots(int64_t M, int64_t H, int64_t K);
int32_t mi8_few_rows_swiglu_slots(int64_t M, int64_t H, int64_t K, int x_is_fp8); /* (of mi8_few_rows_swiglu, operands without padding: lda = ldb = K) */

/* ---------------------------------------------------------------------------------------------
 * Block scales: float8 (e4m3) with one power-of-two scale per 128 elements of the contracted axis.  No counterpart in the
 * reference, whose recipes scale whole tensors, rows or columns (src/olmo_core/float8/ao.py:76-109).
 *
 * An operand [rows, K] is float8 rows of round_up(K, 128) bytes or more (zero from K on) and one exponent byte per row and
 * block of 128: an element is q * 2^(byte - 127).  The byte of row r and block k is at
 *     scales[k * round_up(rows, 128) + 128 * (r / 128) + 8 * (r % 16) + r % 128 / 16]
 * in an array of mi8_block_scale_bytes(rows, K) bytes.  The scale of a block is the largest power of two that keeps its
 * largest magnitude times the scale within 448, at most 2^120; a block that holds an infinity or a NaN is NaN throughout.
 * ------------------------------------------------------------------------------------------- */
int64_t mi8_block_scale_bytes(int64_t rows, int64_t K); /* host only */

/* Casts of x[matrices * rows, cols] (contiguous, cols % 16 == 0), `matrices` matrices (at most 65535) of equal size one after the other:
 *   out (may be NULL):   [matrices * rows, ld_out] and scales [matrices][mi8_block_scale_bytes(rows, cols)]: blocks of 128 along a row
 *   out_t (may be NULL): [matrices][cols, ld_t] and scales_t [matrices][mi8_block_scale_bytes(cols, rows)]: the transposed copy,
 *                        blocks of 128 along a column, zero from column `rows` up to round_up(rows, 128)
 *   square != 0: the blocks are 128 x 128 (weights) and both copies hold the same values. */
int mi8_cast_block(const void* x, int hp_dtype, int64_t rows, int64_t cols, int32_t matrices, int32_t square, void* out, int64_t ld_out,
                   void* scales, void* out_t, int64_t ld_t, void* scales_t, void* stream);

/* The same for rows in consecutive groups (device int64 sizes, clamped as in mi8_grouped_gemm_fp8): out rows stay where they are in x
 * [T, ld_out], but the scales of both copies and the columns of the transposed one lie on an axis of A = mi8_grouped_padded_rows(T,
 * num_groups) rows on which every group starts at the next multiple of 128 (as in mi8_grouped_wgrad_fp8):
 * scales [ceil(cols / 128)][A], out_t [cols, ld_t >= A], scales_t [A / 128][round_up(cols, 128)].  Rows behind the last group are not touched. */
int mi8_grouped_cast_block(const void* x, int hp_dtype, int64_t T, int64_t cols, const int64_t* group_sizes, int32_t num_groups, void* out,
                           int64_t ld_out, void* scales, void* out_t, int64_t ld_t, void* scales_t, void* stream);

/* Up to MI8_BLOCK_CAST_BATCH casts of one input type in one launch: the arguments and results of mi8_cast_block (group_sizes NULL, num_groups 0) or
 * mi8_grouped_cast_block (group_sizes set, matrices 1, square 0; rows is T). */
#define MI8_BLOCK_CAST_BATCH 8
typedef struct {
    const void* x;
    int64_t rows, cols;
    void* out;
    int64_t ld_out;
    void* scales;
    void* out_t;
    int64_t ld_t;
    void* scales_t;
    const int64_t* group_sizes;
    int32_t num_groups, matrices, square, hp_dtype;
} mi8_block_cast_item;
int mi8_cast_block_batch(const mi8_block_cast_item* items, int32_t count, void* stream);

/* out[M, N] = A . B^T over ceil(K / 128) blocks: float32 accumulation, the scales applied inside the matrix instructions.
 * N % 8 == 0, ldc % 8 == 0, operand pitches multiples of 16, below 2^24 and at least round_up(K, 128); out bf16 or float32.
 * variant: -1 chooses by the sizes; 0 to 3 tiles of 64 x 64, 128 x 64, 64 x 128, 256 x 256 (bf16 output only): same sums in the
 * same order. */
int mi8_gemm_fp8_block(const void* a, int64_t lda, const void* a_scales, const void* b, int64_t ldb, const void* b_scales, int64_t M, int64_t N,
                       int64_t K, void* out, int out_dtype, int64_t ldc, int variant, void* stream);

/* Up to MI8_BLOCK_GEMM_BATCH such products that do not need one another: the results of the calls one by one, in one launch where none of
 * them would take the 256 x 256 tiles. */
#define MI8_BLOCK_GEMM_BATCH 8
typedef struct {
    const void* a;
    int64_t lda;
    const void* a_scales;
    const void* b;
    int64_t ldb;
    const void* b_scales;
    int64_t M, N, K;
    void* out;
    int64_t ldc;
    int32_t out_dtype, reserved; /* reserved: 0 */
} mi8_block_product;
int mi8_gemm_fp8_block_batch(const mi8_block_product* items, int32_t count, void* stream);

/* out[rows of e] = A[rows of e] . B_e^T, A and its scales from mi8_grouped_cast_block, B_e = b + e * b_group_stride with the scales
 * b_scales + e * mi8_block_scale_bytes(N, K).  Rows behind the last group become zero. */
int mi8_grouped_gemm_fp8_block(const void* a, int64_t lda, const void* a_scales, const void* b, int64_t ldb, int64_t b_group_stride,
                               const void* b_scales, const int64_t* group_sizes, int32_t num_groups, int64_t T, int64_t N, int64_t K, void* out,
                               int out_dtype, int64_t ldc, void* stream);

/* out[M, N] (the type of x) = q(x) . B^T for a few rows of x [M, K] (bf16 or float32, contiguous), which are quantised in the same launch
 * as mi8_cast_block does; b [N, ldb] and b_scales of mi8_cast_block.  At most mi8_block_rows_max(0) rows.  num_groups > 0: rows in
 * groups as in mi8_grouped_gemm_fp8_block, at most mi8_block_rows_max(num_groups) in all. */
int64_t mi8_block_rows_max(int32_t num_groups); /* host only */
int mi8_block_rows(const void* x, int hp_dtype, int64_t M, const void* b, int64_t ldb, int64_t b_group_stride, const void* b_scales,
                   const int64_t* group_sizes, int32_t num_groups, int64_t N, int64_t K, void* out, void* stream);

/* out[e] [N, Kl] = A_t[:, tokens of e] . B_t[:, tokens of e]^T, transposed copies of mi8_grouped_cast_block with one pitch; zeros for an
 * empty group. */
int mi8_grouped_wgrad_fp8_block(const void* a_t, const void* a_scales, const void* b_t, const void* b_scales, int64_t ld_t,
                                const int64_t* group_sizes, int32_t num_groups, int64_t T, int64_t N, int64_t Kl, void* out, int out_dtype,
                                void* stream);

/* Host only: which of mi8_gemm_fp8_block's variants these sizes take in the grouped products above, with operands and outputs without padding
 * between their rows (-1: an empty problem).  All give the same bits. */
int32_t mi8_grouped_gemm_fp8_block_variant(int64_t T, int64_t N, int64_t K, int32_t num_groups, int out_dtype);
int32_t mi8_grouped_wgrad_fp8_block_variant(int64_t T, int64_t N, int64_t Kl, int32_t num_groups, int out_dtype);

/* ---------------------------------------------------------------------------------------------
 * Routing to experts.  From logits [tokens, experts] (bf16, float16 or float32; at most 512 experts) to the top_k (at most 64) experts of
 * every token: scores s = softmax or sigmoid of the logits, chosen by c = s + bias (bias may be NULL; it is no part of the weights),
 * the largest first, the lowest index of equal ones.  groups > 1: of that many (at most 32) equal groups of consecutive experts only the
 * groups_kept with the largest sum of their two largest c are chosen from.  weights[t][j] = scale * s_j, with normalize divided by the sum of the
 * token's chosen s (0 where all of them are below 2^-1024).  The choice is that of 64-bit scores (without a bias or
 * groups that of the logits themselves); a NaN comes last.  counts[e]: slots of expert e.
 * workspace: int32 [mi8_moe_route_workspace_words()], contents on entry unimportant; may be NULL where that is 0.
 * Stands beside the permutation above, whose expert ids and batch sizes it makes (reference: the router's part of
 * src/olmo_core/nn/moe/parallel_mlp.py:102-183's inputs).
 * ------------------------------------------------------------------------------------------- */
int64_t mi8_moe_route_workspace_words(int64_t tokens, int32_t experts); /* host only */
int mi8_moe_route(const void* logits, int hp_dtype, int64_t tokens, int32_t experts, int32_t top_k, int32_t softmax, const float* bias,
                  int32_t groups, int32_t groups_kept, int32_t normalize, float scale, int32_t* workspace, float* weights, int64_t* indices,
                  int64_t* counts, void* stream);

/* grad_logits (the logits' type) from grad, the gradient of the weights [tokens, top_k], and what mi8_moe_route gave. */
int mi8_moe_route_grad(const void* logits, int hp_dtype, int64_t tokens, int32_t experts, int32_t top_k, int32_t softmax, int32_t normalize,
                       float scale, const float* weights, const int64_t* indices, const float* grad, void* grad_logits, void* stream);

/* ---------------------------------------------------------------------------------------------
 * Products in the model's own type (bf16 or float16, both operands and the output), summed in float32 and rounded once:
 *     C [M, N] = act(A . B^T + bias) + residual
 * a_by_k / b_by_k = 0: the operand lies [rows, K], 1: [K, rows].  A by K goes with B by K only (a weight gradient).  Pitches are multiples of 8
 * elements up to 2^22; in [rows, K] operands the elements from K up to the next multiple of 8 are zeros.
 * C, z and the residual may have any pitch and alignment of their type.
 * (Stand beside the float8 products, for layers that are not converted; reference: the bf16 nn.Linear calls and grouped_gemm.ops.gmm of
 * src/olmo_core/nn/feed_forward.py:114-171 and src/olmo_core/nn/moe/mlp.py:177-292.)
 * ------------------------------------------------------------------------------------------- */
typedef enum mi8_activation {
    MI8_ACT_NONE = 0,
    MI8_ACT_RELU = 1,
    MI8_ACT_SILU = 2,
    MI8_ACT_GELU = 3,     /* x times the normal distribution function of x */
    MI8_ACT_GELU_TANH = 4 /* its approximation x (1 + tanh(sqrt(2 / pi) (x + 0.044715 x^3))) / 2 */
} mi8_activation;

/* Which kernel a product takes; MI8_HALF_ANY: the library chooses, by the sizes.  (The tiles sum K in one order, their results have the same bits; a few rows and
 * products of few tiles sum slices of K.) */
typedef enum mi8_half_variant {
    MI8_HALF_ANY = 0,
    MI8_HALF_256 = 1, /* tiles of 256 x 256 */
    MI8_HALF_128 = 2, /* 128 x 128, two workgroups on a compute unit */
    MI8_HALF_64 = 3,  /* 64 x 64 */
    MI8_HALF_ROWS = 4, /* up to 16 rows of A, both operands [rows, K] */
    MI8_HALF_192 = 5  /* 192 x 256, A [rows, K]; not for groups */
} mi8_half_variant;

typedef struct mi8_half_epilogue {
    const void* bias;     /* [N], or NULL */
    const void* residual; /* [M, N] of the operands' type, or NULL */
    int64_t ld_residual;
    void* z;              /* NULL, or where A . B^T + bias goes (of the operands' type) */
    int64_t ld_z;
    int32_t bias_dtype;   /* the operands' type or MI8_F32 */
    int32_t activation;   /* mi8_activation */
} mi8_half_epilogue;

int mi8_gemm_half(int hp_dtype, const void* a, int64_t lda, int a_by_k, const void* b, int64_t ldb, int b_by_k, int64_t M, int64_t N, int64_t K,
                  const mi8_half_epilogue* epilogue /* NULL: none */, void* out, int64_t ldc, int variant, void* workspace, void* stream);

/* Host only: bytes that `workspace` above needs where the library chooses (0: none; with NULL it chooses without slices of K), which variant these sizes take with
 * it, in how many slices of K, and the variants of the grouped products below (-1: an empty product). */
int64_t mi8_gemm_half_workspace_bytes(int64_t M, int64_t N, int64_t K, int a_by_k, int b_by_k);
int mi8_gemm_half_variant(int64_t M, int64_t N, int64_t K, int a_by_k, int b_by_k, int32_t* slices);
int mi8_grouped_gemm_half_variant(int64_t T, int64_t N, int64_t K, int32_t num_groups);
int mi8_grouped_wgrad_half_variant(int64_t T, int64_t M, int64_t N, int32_t num_groups);

/* Rows of A and C in consecutive groups of group_sizes[e] rows (device int64): group e times B + e * b_group_stride (elements).  Sizes count up to T in
 * all; rows behind the last group give zeros. */
int mi8_grouped_gemm_half(int hp_dtype, const void* a, int64_t lda, const void* b, int64_t ldb, int b_by_k, int64_t b_group_stride,
                          const int64_t* group_sizes, int32_t num_groups, int64_t T, int64_t N, int64_t K, void* out, int64_t ldc, int variant,
                          void* stream);

/* out[e] [M, N] = A[rows of e]^T . B[rows of e], A [T, M] and B [T, N]; zeros for an empty group. */
int mi8_grouped_wgrad_half(int hp_dtype, const void* a, int64_t lda, const void* b, int64_t ldb, const int64_t* group_sizes, int32_t num_groups, int64_t T,
                           int64_t M, int64_t N, void* out, int variant, void* stream);

/* out [rows, ld_out] = x [rows, cols] of 16-bit elements at any pitch and alignment, zeros from cols to ld_out: an operand for the products above. */
int mi8_half_pad(const void* x, int64_t ld_x, int64_t rows, int64_t cols, void* out, int64_t ld_out, void* stream);

/* The epilogue's gradient: dz [M, ld_dz] = grad * act'(z) (dz, z NULL: no activation, dz is not written; columns N .. ld_dz are zeroed) and
 * bias_grad [N] = the column sums of grad * act'(z) (NULL: not wanted), summed in float32 in an order that the sizes decide.
 * workspace: float32 [mi8_half_epilogue_grad_workspace_words(M, N)] where bias_grad is wanted. */
int64_t mi8_half_epilogue_grad_workspace_words(int64_t M, int64_t N); /* host only */
int mi8_half_epilogue_grad(int hp_dtype, const void* grad, int64_t ld_grad, const void* z, int64_t ld_z, int activation, int64_t M, int64_t N, void* dz,
                           int64_t ld_dz, void* bias_grad, int bias_dtype, float* workspace, void* stream);

/* ---------------------------------------------------------------------------------------------
 * Dropout from a counter: element i of a tensor of n (bf16, float16 or float32, in the order of memory) takes 16 bits, the (i % 8)-th of Philox-4x32 with 7 rounds,
 * counter (i / 8, offset), key seed (seed_on_device[0] where that is not NULL, read when the kernel runs), 64 bits each and low word first.
 * y = x * factor where they are at least `threshold` (0 .. 65536), else 0.  The gradient is the same map.
 * (reference: the nn.Dropout calls of src/olmo_core/nn/transformer/block.py)
 * ------------------------------------------------------------------------------------------- */
int mi8_dropout(const void* x, int hp_dtype, int64_t n, uint32_t threshold, float factor, uint64_t seed, const int64_t* seed_on_device, uint64_t offset,
                void* y, void* stream);

/* A block's output on its way into the residual stream and the norm in front of the next one, rows of `features` (at most 16384) elements:
 *     stream = residual_scale * residual + scale * gate * drop(norm(branch) * post),    normed = norm(stream) * pre,
 *     norm(a) = a / sqrt(mean(a^2) + eps)
 * Sums and the stream inside are float32.  residual, stream and residual_grad have stream_dtype (the branch's or float32), branch, normed and branch_grad
 * the branch's; stream, normed, branch_grad and residual_grad are contiguous.  drop: as in mi8_dropout, with the rows one after the other; threshold 0: none.
 * (reference: the norms and residual additions of src/olmo_core/nn/transformer/block.py, src/olmo_core/nn/layer_norm.py) */
typedef struct mi8_residual_norm {
    const void* branch;    /* backward: NULL without a norm or gate on it; given, the stream is made again from it and the residual */
    const void* residual;  /* NULL: none */
    void* stream;          /* forward: NULL if not wanted; backward: read where normed_grad is given and branch is NULL */
    void* normed;          /* forward, with pre_norm */
    const void* post;      /* [features], or NULL: 1 (the same for pre and gate) */
    const void* pre;
    const void* gate;
    float* branch_rstd;    /* [rows] 1 / sqrt(..) of either norm: written by the forward unless NULL, read by the backward */
    float* stream_rstd;
    const int64_t* seed_on_device;
    /* backward: gradients in (NULL: zero) and out (NULL: not wanted; the weights' have their weights' types) */
    const void* stream_grad;
    const void* normed_grad;
    void* branch_grad;
    void* residual_grad;
    void* post_grad;
    void* pre_grad;
    void* gate_grad;
    uint64_t seed;
    uint64_t offset;
    int64_t rows;
    int64_t features;
    int64_t ld_branch, ld_residual, ld_stream_grad, ld_normed_grad; /* elements between rows */
    int32_t branch_dtype, stream_dtype;
    int32_t post_dtype, pre_dtype, gate_dtype; /* the branch's or MI8_F32 */
    int32_t post_norm, pre_norm;               /* whether there is that norm */
    uint32_t threshold;
    float factor;
    float scale, residual_scale, eps;
} mi8_residual_norm;

int mi8_residual_norm_forward(const mi8_residual_norm* args, void* stream);

/* workspace: float32 [mi8_residual_norm_workspace_words(rows, features)] where a weight's gradient is wanted.  Column sums are added in an order that the
 * sizes decide. */
int64_t mi8_residual_norm_workspace_words(int64_t rows, int64_t features); /* host only */
int mi8_residual_norm_backward(const mi8_residual_norm* args, float* workspace, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* MI8_H */
