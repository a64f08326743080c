/*
 * fp4attn.h -- C ABI of libfp4attn.so, the sm_100a (B200) FP4 fused attention.
 *
 * Drop-in boundary for the reference florianmattana/fp4-fused-attention-sm120.
 * The reference exposes no library: its public surface is the header
 * common.h -- the encoders encode_fp4_e2m1 / compute_scale_ue8m0
 * (common.h:21-48), the kernel template
 *     template<int HEAD_DIM> __global__ void fused_fp4_attention(
 *         const float* Q, const float* K, float* Out, const float* V,
 *         int seq_q, int seq_k, int heads)                      (common.h:68-77)
 * launched as <<<batch*heads, NUM_THREADS>>> (tests/test_attention.cu:160-161),
 * and the constants BLOCK_ELEMENT / BQ (common.h:15, :18).  Each entry point
 * below names the reference interface it replaces.
 *
 * Conventions: all pointers are device pointers unless stated; tensors are
 * contiguous [batch, heads, seq, head_dim] (the reference layout,
 * common.h:99-102); `stream` is a cudaStream_t (0 = legacy default stream).
 * Every call is asynchronous on `stream` and returns an fp4attn_status code;
 * a non-zero code means nothing was launched.  The library keeps no state
 * between calls except, per device, its first-use set-up (the device check
 * and the SM count; kernel attributes per device context), an error word
 * (fp4attn_status_query), the fp4attn_forward_noalloc scratch, and per host
 * thread a cache of recently encoded TMA descriptors.  Calls on different
 * streams may run concurrently; the caller owns all buffers.  The attention
 * kernel of a call is launched as the programmatic dependent of the launch
 * before it in the stream (normally this call's quantiser): it starts while
 * that launch finishes and waits for it before reading the workspace.
 */
#ifndef FP4ATTN_H
#define FP4ATTN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- constants kept from the reference (common.h:12, :15, :18) ---------- */
#define FP4ATTN_BLOCK_ELEMENT 32 /* elements per UE8M0 scale (BLOCK_ELEMENT) */
#define FP4ATTN_BQ 64            /* the reference's fixed Q tile (BQ)         */

/* ---- status codes ------------------------------------------------------- */
typedef enum {
    FP4ATTN_OK = 0,
    FP4ATTN_EINVAL = 1,       /* bad shape, dtype, pointer alignment or size  */
    FP4ATTN_EUNSUPPORTED = 2, /* head_dim not compiled / no sm_100 device     */
    FP4ATTN_ECUDA = 3,        /* a CUDA runtime or driver call failed          */
    FP4ATTN_ETIMEOUT = 4,     /* a kernel's bounded wait expired (reported by  */
                              /* fp4attn_status_query after the stream syncs) */
    FP4ATTN_EWORKSPACE = 5,   /* workspace missing or too small               */
    FP4ATTN_EINDEX = 6        /* a position, page, sequence or length that a  */
                              /* kernel read was out of range (reported by    */
                              /* fp4attn_status_query after the stream syncs) */
} fp4attn_status;

/* ---- element types ------------------------------------------------------ */
typedef enum { FP4ATTN_F32 = 0, FP4ATTN_F16 = 1 } fp4attn_dtype;

/* ---- UE8M0 scale rules -------------------------------------------------- */
typedef enum {
    /* The reference rule, bit-exact with compute_scale_ue8m0 (common.h:39-48)
     * as built on the host with glibc: byte = (uint8)(ceil(log2(max|x|)) + 127),
     * an all-zero block gives 127. */
    FP4ATTN_SCALE_REFERENCE = 0,
    /* OCP-MX style: byte = (uint8)(ceil(log2(max|x| / 6)) + 127).  Not part of
     * the reference; offered because it uses the full E2M1 range. */
    FP4ATTN_SCALE_OCP = 1
} fp4attn_scale_mode;

/* ---- attention masks ------------------------------------------------------ */
typedef enum {
    FP4ATTN_MASK_NONE = 0,   /* every query sees every key (the reference's only mode) */
    /* Causal, bottom-right aligned: query i sees keys j <= i + seq_k - seq_q, so
     * with seq_q == seq_k row i sees keys 0..i.  A query that sees no key
     * (only possible when seq_q > seq_k) gets a zero output row. */
    FP4ATTN_MASK_CAUSAL = 1
} fp4attn_mask;

/* ---- layouts of quantised output ---------------------------------------- */
typedef enum {
    /* codes: rows x head_dim/2 bytes, two E2M1 codes per byte, element 2i in
     * the low nibble; scales: rows x head_dim/32 bytes, row-major. */
    FP4ATTN_LAYOUT_ROWMAJOR = 0
} fp4attn_layout;

/* Quantise `rows` rows of `head_dim` elements (head_dim % 32 == 0) to E2M1
 * codes plus one UE8M0 scale per 32 elements.
 * Replaces: the per-tile quantisation inside the reference kernel
 * (common.h:108-124 for Q, :159-169 for K) built from encode_fp4_e2m1 and
 * compute_scale_ue8m0 (common.h:21-48).  The reference returns each code in an
 * 8-bit container (code << 2, common.h:35); this packs two codes per byte.
 * x: device, dtype elements; codes: rows*head_dim/2 bytes; scales:
 * rows*head_dim/32 bytes. */
int fp4attn_quantize(const void* x, int dtype, int64_t rows, int head_dim, uint8_t* codes,
                     uint8_t* scales, int scale_mode, int layout, void* stream);

/* Bytes of device workspace fp4attn_forward needs for this problem (the
 * quantised Q/K tiles, their scale tiles, an FP16 copy of V when V is FP32,
 * and, for a small problem whose keys are split over several CTAs, the
 * partial results of the key partitions and their arrival counters).  The
 * same for every mask mode.  Returns 0 for an invalid shape. */
size_t fp4attn_workspace_size(int batch, int heads, int seq_q, int seq_k, int head_dim, int in_dtype);

/* Out = softmax(Q K^T * softmax_scale) V per (batch, head) slice, with Q and K
 * quantised to E2M1 + UE8M0 (block 32 along head_dim) and V, P in FP16 on the
 * tensor cores (FP32 accumulation).
 * Replaces: fused_fp4_attention<HEAD_DIM><<<batch*heads, 128>>>(Q, K, Out, V,
 * seq_q, seq_k, heads) (common.h:68-77; tests/test_attention.cu:160-161).
 * Differences, by design: any seq_q >= 1 (the reference computes only the
 * first 64 query rows, common.h:96-102) and any seq_k >= 1 (the reference
 * needs seq_k % 64 == 0, common.h:67); head_dim is a runtime argument among
 * {32, 64, 96, 128, 160, 256}; inputs and output may be FP32 (as in the
 * reference) or FP16.
 * Q: [batch, heads, seq_q, head_dim]; K, V: [batch, heads, seq_k, head_dim];
 * Out: [batch, heads, seq_q, head_dim] of out_dtype; all 16-byte aligned.
 * softmax_scale <= 0 selects 1/sqrt(head_dim) (common.h:130).
 * workspace: device memory of at least fp4attn_workspace_size(...) bytes,
 * 256-byte aligned; it must not be used by another call in flight. */
int fp4attn_forward(const void* Q, const void* K, const void* V, void* Out, int in_dtype, int out_dtype,
                    int batch, int heads, int seq_q, int seq_k, int head_dim, float softmax_scale,
                    int scale_mode, void* workspace, size_t workspace_bytes, void* stream);

/* The two halves of fp4attn_forward, for callers that quantise once and
 * attend many times (e.g. a fixed K/V) or time the attention kernel alone.
 * fp4attn_prepare quantises Q and K into `workspace` (and, for FP32 input,
 * stores an FP16 copy of V there).  Replaces: the quantisation prologue of the
 * reference kernel (common.h:108-124 for Q, :146-169 for K and V). */
int fp4attn_prepare(const void* Q, const void* K, const void* V, int in_dtype, int batch, int heads, int seq_q,
                    int seq_k, int head_dim, int scale_mode, void* workspace, size_t workspace_bytes, void* stream);

/* Runs the attention kernel on a workspace filled by fp4attn_prepare with the
 * same shape and in_dtype.  V is read directly when in_dtype is FP16.  May be
 * called any number of times on one prepared workspace (one call at a time);
 * after a call that reported FP4ATTN_ETIMEOUT, prepare the workspace again.
 * Replaces: the main loop of the reference kernel (common.h:140-327). */
int fp4attn_attend(const void* V, void* Out, int in_dtype, int out_dtype, int batch, int heads, int seq_q, int seq_k,
                   int head_dim, float softmax_scale, const void* workspace, size_t workspace_bytes, void* stream);

/* fp4attn_forward and fp4attn_attend with a mask (fp4attn_mask).  With
 * FP4ATTN_MASK_NONE they are those calls; with FP4ATTN_MASK_CAUSAL each query
 * tile also stops reading keys after the last one it can see, so a causal
 * problem costs about half the unmasked one.  The workspace is the same.
 * No counterpart in the reference, which has no mask (common.h:228-265
 * softmaxes every key of every tile). */
int fp4attn_forward_masked(const void* Q, const void* K, const void* V, void* Out, int in_dtype, int out_dtype,
                           int batch, int heads, int seq_q, int seq_k, int head_dim, float softmax_scale,
                           int scale_mode, int mask_mode, void* workspace, size_t workspace_bytes, void* stream);
int fp4attn_attend_masked(const void* V, void* Out, int in_dtype, int out_dtype, int batch, int heads, int seq_q,
                          int seq_k, int head_dim, float softmax_scale, int mask_mode, const void* workspace,
                          size_t workspace_bytes, void* stream);

/* fp4attn_forward with Q quantised inside the attention kernel instead of in
 * the pre-pass launch, as the reference quantises its Q tile inside its own
 * kernel (common.h:108-124): the pre-pass quantises only K, and the attention
 * kernel reads FP16 Q and encodes it with the same encoder, so the codes,
 * scales and output are those of fp4attn_forward, bit for bit.  Applies to
 * FP16 input with head_dim <= 128, seq_k >= 3008 (48 key tiles of 64) on the
 * large-problem schedule (seq_q > 128 and at least 75 query groups of 256
 * rows); any other problem runs the fp4attn_forward path.  Same arguments and
 * workspace as fp4attn_forward.
 * Replaces: the quantisation prologue of fused_fp4_attention (common.h:108-124). */
int fp4attn_forward_fused_q(const void* Q, const void* K, const void* V, void* Out, int in_dtype, int out_dtype,
                            int batch, int heads, int seq_q, int seq_k, int head_dim, float softmax_scale,
                            int scale_mode, void* workspace, size_t workspace_bytes, void* stream);

/* fp4attn_forward for callers that cannot allocate device memory (code running
 * during CUDA graph capture, runtimes that own all device memory, loops that
 * must not block on an allocation): the same computation, with the workspace
 * taken from a 64 MiB scratch array the library holds on each device from the
 * first call (or from context creation under CUDA_MODULE_LOADING=EAGER) until
 * the process exits.  Problems whose fp4attn_workspace_size exceeds 64 MiB are
 * rejected with FP4ATTN_EWORKSPACE.  The first call on a device looks up the
 * scratch's device address (again after a device reset, which moves it); make
 * it before any stream capture.  All calls on a
 * device share the scratch: calls that may overlap on the GPU must be
 * serialised by the caller.  No counterpart in the reference (its kernel keeps
 * everything in shared memory and needs no workspace). */
int fp4attn_forward_noalloc(const void* Q, const void* K, const void* V, void* Out, int in_dtype, int out_dtype,
                            int batch, int heads, int seq_q, int seq_k, int head_dim, float softmax_scale,
                            int scale_mode, void* stream);

/* fp4attn_forward_masked that also writes, per query row, the natural-log
 * log-sum-exp of the scaled scores, lse[b][h][i] = ln(sum_j exp(scale * S_ij))
 * over the keys the row sees (FP32 [batch, heads, seq_q]; +inf for a row that
 * sees no key) -- the statistic the backward pass rebuilds the probabilities
 * from.  head_dim 32, 64, 96 and 128.  Same workspace as fp4attn_forward.  No
 * counterpart in the reference (forward only; its row max and sum stay in
 * registers, common.h:228-265). */
int fp4attn_forward_lse(const void* Q, const void* K, const void* V, void* Out, float* lse, int in_dtype,
                        int out_dtype, int batch, int heads, int seq_q, int seq_k, int head_dim, float softmax_scale,
                        int scale_mode, int mask_mode, void* workspace, size_t workspace_bytes, void* stream);

/* Workspace bytes fp4attn_backward needs for this shape and input type (0 if
 * unsupported). */
size_t fp4attn_backward_workspace_size(int batch, int heads, int seq_q, int seq_k, int head_dim, int in_dtype);

/* Gradient of the FP4 fused attention.  Inputs: the forward's Q, K, V and
 * dOut (the gradient of Out), all of in_dtype (FP16 or FP32; FP32 V and dOut
 * are rounded to FP16 for the tensor cores, as the forward rounds V), its
 * output Out (out_dtype FP16 or FP32) and the lse rows of
 * fp4attn_forward_lse (same shape, scale, scale_mode and mask).  Outputs: FP32 dQ, dK, dV in the layout of Q, K, V.  The quantiser
 * is treated as a straight-through estimator: with Qq, Kq the dequantised
 * codes the forward multiplied and P its probabilities,
 *   dV = P^T dOut,  dZ = P o (dOut V^T - rowsum(dOut o Out)),
 *   dQ = scale * dZ Kq,  dK = scale * dZ^T Qq.
 * head_dim 32, 64, 96 and 128.  Every byte of dQ, dK and dV is written.  No
 * counterpart in the reference, which is inference-only. */
int fp4attn_backward(const void* Q, const void* K, const void* V, const void* Out, const void* dOut, const float* lse,
                     float* dQ, float* dK, float* dV, int in_dtype, int out_dtype, int batch, int heads, int seq_q,
                     int seq_k, int head_dim, float softmax_scale, int scale_mode, int mask_mode, void* workspace,
                     size_t workspace_bytes, void* stream);

/* The two halves of fp4attn_backward (as fp4attn_prepare / fp4attn_attend
 * are of fp4attn_forward).  fp4attn_backward_prepare quantises Q and K into
 * the workspace (codes, scale tiles and the dequantised values as BF16), for
 * FP32 input stores FP16 copies of V and dOut there, forms the per-row
 * statistics of dOut, Out and lse, and clears dQ;
 * fp4attn_backward_attend runs the backward kernel on that workspace, adding
 * into dQ and writing dK and dV.  Same shapes, alignment and workspace as
 * fp4attn_backward. */
int fp4attn_backward_prepare(const void* Q, const void* K, const void* V, const void* Out, const void* dOut,
                             const float* lse, float* dQ, int in_dtype, int out_dtype, int batch, int heads, int seq_q,
                             int seq_k, int head_dim, int scale_mode, void* workspace, size_t workspace_bytes,
                             void* stream);
int fp4attn_backward_attend(const void* V, const void* dOut, float* dQ, float* dK, float* dV, int in_dtype, int batch,
                            int heads, int seq_q, int seq_k, int head_dim, float softmax_scale, int mask_mode,
                            const void* workspace, size_t workspace_bytes, void* stream);

/* Self-test of the backward kernel's failure path (the counterpart of
 * fp4attn_selftest_abort): fp4attn_backward_prepare, then the head_dim 64
 * backward kernel in a test instantiation where one gradient thread withholds
 * its first arrival, with every wait bounded by timeout_us.  The wait runs
 * out, every role of every CTA leaves its loop, in-flight copies and MMAs are
 * drained, TMEM is freed; fp4attn_status_query then reports
 * FP4ATTN_ETIMEOUT and the context stays usable.  FP16 inputs, seq_q > 64.
 * dQ, dK and dV hold no result afterwards. */
int fp4attn_selftest_backward_abort(const void* Q, const void* K, const void* V, const void* Out, const void* dOut,
                                    const float* lse, float* dQ, float* dK, float* dV, int batch, int heads, int seq_q,
                                    int seq_k, void* workspace, size_t workspace_bytes, unsigned timeout_us,
                                    void* stream);

/* S = Q K^T (no softmax scale) on the FP4-quantised Q and K of one problem,
 * written as FP32 [batch, heads, seq_q, seq_k].  Because FP4 products with
 * power-of-two scales are exact, S is checkable bit for bit.
 * Replaces: the reference's debug kernel debug_mma (common.h:331-398), which
 * computes one 64x64 tile of Q K^T on FP4 codes. */
int fp4attn_debug_scores(const void* Q, const void* K, float* S, int in_dtype, int batch, int heads,
                         int seq_q, int seq_k, int head_dim, int scale_mode, void* workspace,
                         size_t workspace_bytes, void* stream);

/* Reads and clears the device error word that kernels set when a bounded
 * wait expires or an index is out of range.  Synchronises `stream` first.
 * Returns FP4ATTN_OK, FP4ATTN_ETIMEOUT or FP4ATTN_EINDEX (or FP4ATTN_ECUDA if the query itself fails).  The word is
 * one per device, shared by every stream: a kernel still running on another
 * stream may set it after this call returns (it is then reported by the next
 * query), and a timeout raised on another stream is reported by whichever
 * query reads the word first.  To attribute a timeout to one stream's work,
 * synchronise the other streams that run this library's kernels (or the
 * device) before querying.  The reference has no device-side error reporting
 * (callers only poll cudaGetLastError, tests/test_attention.cu:103-105). */
int fp4attn_status_query(void* stream);

/* Test hook for the failure path: launches one CTA that waits on an mbarrier
 * nothing will complete, with the given bound, so that the bounded wait runs
 * out and sets the error word.  No fault, trap or hang is involved. */
int fp4attn_selftest_timeout(unsigned timeout_us, void* stream);

/* Test hook for the attention kernel's own failure path: runs the
 * head_dim-64, FP32-output attention kernel (seq_q > 128, a problem without
 * key partitions) over a workspace filled by fp4attn_prepare (FP16 input), in
 * a build in which one softmax thread never makes its first "S copied"
 * arrival.  The kernel's bounded wait for it expires after timeout_us; every
 * role then leaves its loop, drains its in-flight copies and MMAs, frees its
 * tensor memory and returns, and fp4attn_status_query reports
 * FP4ATTN_ETIMEOUT.  No fault, trap or hang is involved; later calls on the
 * same context run normally.  No counterpart in the reference. */
int fp4attn_selftest_abort(const void* V, void* Out, int batch, int heads, int seq_q, int seq_k,
                           const void* workspace, size_t workspace_bytes, unsigned timeout_us, void* stream);

/* Test hook: y[i] = 2^x[i] computed by the FMA-pipe polynomial the softmax
 * uses for part of its exponentials (n even, 16-byte aligned device arrays).
 * No counterpart in the reference, whose softmax calls expf (common.h:236). */
int fp4attn_selftest_exp2(const float* x, float* y, int64_t n, void* stream);

/* ---- serving: rotary positions, the paged cache, attention over it --------
 * The reference has none of these (it attends over whole K and V tensors,
 * common.h:68-77).  All are asynchronous on `stream`, keep nothing between
 * calls and may be captured into CUDA graphs.  Positions, pages, sequence
 * numbers and lengths that a kernel reads from device memory are checked
 * there: what is out of range is not accessed, and the next
 * fp4attn_status_query reports FP4ATTN_EINDEX. */

/* table[p][j] = factor * (cos, sin)(p * freqs[j]) as FP32, [max_positions]
 * [pairs][2], the angles in 64 bits.  freqs: `pairs` doubles (1 to 128) in
 * host memory.  Long-context scalings change freqs and factor. */
int fp4attn_rotary_table(const double* freqs, int pairs, int64_t max_positions, double factor, float* table,
                         void* stream);

/* Rotary positions: y = x with the first rotary_dim (even) elements of every
 * row turned pair by pair by the angles of the row's position, the rest
 * copied.  Pairs are (2j, 2j+1) when `interleaved`, else (j, j+rotary_dim/2).
 * x, y: [batch, heads, seq, head_dim] with element strides {batch, head, seq}
 * (the last dimension contiguous), F16 or F32; y may be x itself (with the
 * same strides).  positions: [batch][seq] with positions_stride elements from
 * one batch entry to the next (0: shared), or null for 0 .. seq-1; a position
 * outside [0, max_positions) gives a row of zeros and FP4ATTN_EINDEX.
 * inverse: turned back by the same angles (the transpose), which is the
 * gradient: dx = fp4attn_rotary(dy, inverse).  Products and sums are rounded
 * to FP32 one by one and the result once to the tensor's type. */
int fp4attn_rotary(const void* x, void* y, int dtype, int batch, int heads, int seq, int head_dim,
                   const int64_t* x_strides, const int64_t* y_strides, const float* table, int rotary_dim,
                   int64_t max_positions, const int32_t* positions, int64_t positions_stride, int interleaved,
                   int inverse, void* stream);

/* One layer's paged cache: keys as E2M1 codes with UE8M0 scales (the
 * row-major forms of fp4attn_quantize, but with 255 stored as 254), values as
 * FP16.  Within a page everything is contiguous; the strides (bytes from one
 * page to the next, multiples of 16) let a page hold several layers.
 * page_size: 16, 32, 64 or 128 tokens; pointers 16-byte aligned. */
typedef struct {
    uint8_t* k_codes;  /* [pages][kv_heads][page_size][head_dim / 2]  */
    uint8_t* k_scales; /* [pages][kv_heads][page_size][head_dim / 32] */
    void* v;           /* [pages][kv_heads][page_size][head_dim] FP16 */
    int64_t k_codes_stride, k_scales_stride, v_stride;
    int pages, page_size, kv_heads, head_dim;
} fp4attn_cache;

/* Puts new tokens into a cache: each key is rotated (when `table` is given),
 * rounded to its type and quantised by scale_mode; each value is rounded to
 * FP16; and, when Q is given, each query is rotated into Q_out.  K, V:
 * [tokens, kv_heads, head_dim], Q: [tokens, q_heads, head_dim], with element
 * strides {token, head}; Q_out: the same, contiguous.
 * Token i is token positions[i] of sequence seq_ids[i] (null: sequence i), and
 * lies in page block_table[seq * table_stride + position / page_size].  A
 * negative position marks padding: it leaves the cache alone and gives a zero
 * query row; so does a position beyond the rotary table, as FP4ATTN_EINDEX.
 * The codes and scales are byte for byte those of fp4attn_rotary followed by
 * fp4attn_quantize.  No two tokens of a call may have the same place in the
 * cache, and Q_out must not overlap Q.  One block a token in parallel: rows are
 * fastest 16-byte aligned (pointers and strides), with rotary_dim a multiple of
 * 64 or interleaved pairs; rows that are not aligned are taken element by
 * element. */
int fp4attn_cache_append(const fp4attn_cache* cache, const void* K, const void* V, const void* Q, void* Q_out,
                         int dtype, int tokens, int q_heads, const int64_t* k_strides, const int64_t* v_strides,
                         const int64_t* q_strides, const int32_t* block_table, int64_t table_stride, int seqs,
                         int max_pages, const int32_t* seq_ids, const int32_t* positions, const float* table,
                         int rotary_dim, int64_t max_positions, int interleaved, int scale_mode, void* stream);

/* Reads tokens back: K and V [seqs, heads, max_length, head_dim] of dtype get
 * the values of tokens starts[s] .. starts[s]+lengths[s]-1 (starts null: 0) of
 * every sequence, zeros behind them; heads is a multiple of kv_heads, each
 * key/value head repeated for its query heads.  For attention over a cached
 * prefix by fp4attn_forward_masked. A key above FP16's range is infinite there. */
int fp4attn_cache_gather(const fp4attn_cache* cache, const int32_t* block_table, int64_t table_stride, int seqs,
                         int max_pages, const int32_t* starts, const int32_t* lengths, int max_length, int heads,
                         void* K, void* V, int dtype, void* stream);

/* Workspace bytes of fp4attn_paged_attention (0 for an invalid shape); it does
 * not depend on the lengths. */
size_t fp4attn_paged_attention_workspace_size(int batch, int q_heads, int kv_heads, int head_dim);

/* Attention of one new token per sequence over the cache: Out[b][h] =
 * softmax(softmax_scale * Qq Kq^T) V over the first seq_lens[b] tokens of
 * sequence b (its own included, once appended), what fp4attn_forward gives for
 * that one query row.  Q: [batch, q_heads, head_dim] of in_dtype with element
 * strides {batch, head}; query head h reads key/value head
 * h / (q_heads / kv_heads).  Out: [batch, q_heads, head_dim] of out_dtype,
 * lse (or null): [batch, q_heads] natural log-sum-exp.  A sequence of length
 * 0 gives zeros and +inf.  Several new tokens of one sequence are as many
 * rows that share its pages, with lengths that grow by one.
 * softmax_scale <= 0 selects 1/sqrt(head_dim).  With either output type the
 * probabilities keep 22 bits down to 2^-21 of the largest, and those below lose
 * at most 2^-43 of it; FP16 output is the FP32 output rounded once.
 * A length beyond the block table counts as the table's, and a page outside the
 * cache as page 0 (FP4ATTN_EINDEX either way; the other sequences keep their
 * results).  max_pages * page_size is at most 2^30.  Results repeat bit for bit
 * for the same lengths; they depend on the lengths of the other sequences in the
 * last bits, by where long sequences are divided.  workspace: as
 * fp4attn_paged_attention_workspace_size says, 256-byte aligned, any content;
 * not shared with another call in flight. */
int fp4attn_paged_attention(const fp4attn_cache* cache, const void* Q, void* Out, float* lse, int in_dtype,
                            int out_dtype, int batch, int q_heads, const int64_t* q_strides,
                            const int32_t* block_table, int64_t table_stride, int max_pages, const int32_t* seq_lens,
                            float softmax_scale, int scale_mode, void* workspace, size_t workspace_bytes,
                            void* stream);

/* Test hook for paged attention's failure path (the counterpart of
 * fp4attn_selftest_abort): the head_dim 64, FP32-output kernel in a build in
 * which one thread of its first block never reports its first weights, every
 * wait bounded by timeout_us.  That wait runs out, the block's roles leave their
 * loops and drain what is in flight, and the join joins what there is:
 * nothing outside Out and the workspace is written, fp4attn_status_query
 * reports FP4ATTN_ETIMEOUT, and the sequences of that block hold no result.
 * Q: [batch, q_heads, 64] FP16, contiguous; at most four query heads a
 * key/value head; with a first sequence of 640 tokens a block and more the block
 * leaves in mid-sequence. */
int fp4attn_selftest_paged_abort(const fp4attn_cache* cache, const void* Q, float* Out, int batch, int q_heads,
                                 const int32_t* block_table, int64_t table_stride, int max_pages, const int32_t* seq_lens,
                                 void* workspace, size_t workspace_bytes, unsigned timeout_us, void* stream);

/* Copies whole pages, src[i] to dst[i], within each of n_caches caches (the
 * layers of a model share one page numbering).  src, dst: host memory, read
 * before the call returns.  A page may be copied to several, but none is
 * written twice or both read and written (FP4ATTN_EINVAL). */
int fp4attn_copy_pages(const fp4attn_cache* caches, int n_caches, const int32_t* src, const int32_t* dst, int n,
                       void* stream);

/* Static description of a status code. */
const char* fp4attn_error_string(int status);

/* Detail of the last failure on the calling host thread ("" if none). */
const char* fp4attn_last_error(void);

/* Head dims compiled into this library, written to `dims` (up to `cap`);
 * returns how many there are. */
int fp4attn_supported_head_dims(int* dims, int cap);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* FP4ATTN_H */
