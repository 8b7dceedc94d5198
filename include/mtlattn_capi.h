/*
 * mtlattn C ABI -- the drop-in boundary of the MI355X (gfx950) varlen
 * flash-attention library libmtlattn_hip.so.
 *
 * Every entry point replaces one export of the reference's pybind11 module
 * `mtlattn._C` (src/ext.mm:784-811). Signatures use plain pointers, sizes and
 * an opaque stream handle only (no torch types), so any FFI can bind them; the
 * torch extension mtlattn_amd/csrc/torch_ext.cpp is one such binder.
 *
 * Conventions shared by all entry points:
 *  - Tensors are device pointers. q/k/v/out/dout are [tokens, heads, D] with
 *    the last two dims contiguous (head stride == D) and a free row stride
 *    (in elements), as src/ext.mm:322-325 requires.
 *  - cu_seqlens_{q,kv} are device int32 [num_seqs + 1] cumulative offsets.
 *    Sequence bounds are clamped to [0, total] on the device, so malformed
 *    offsets never address outside the tensors.
 *  - Causal masking is end-aligned: query i sees key j iff
 *    j <= i + (kv_len - q_len); window W > 0 adds j > i + (kv_len - q_len) - W.
 *  - GQA: query head h reads kv head h / (Hq / Hkv).
 *  - The library never allocates device memory. Callers pass scratch space
 *    sized by the matching *_workspace_size() query.
 *  - Work is enqueued on `stream` (a hipStream_t; NULL = the default stream)
 *    of the current device; nothing synchronises with the host.
 *  - Return value: MTLATTN_OK (0) or a negative MTLATTN_ERR_*; the message is
 *    available from mtlattn_last_error() on the calling thread.
 */
#ifndef MTLATTN_CAPI_H
#define MTLATTN_CAPI_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MTLATTN_ABI_VERSION 2

/* element types of q/k/v/out/dout/dq/dk/dv */
enum {
    MTLATTN_DTYPE_F32 = 0,
    MTLATTN_DTYPE_F16 = 1,
    MTLATTN_DTYPE_BF16 = 2
};

enum {
    MTLATTN_OK = 0,
    MTLATTN_ERR_INVALID = -1,     /* bad argument (shape, stride, null pointer) */
    MTLATTN_ERR_UNSUPPORTED = -2, /* valid request this build has no kernel for */
    MTLATTN_ERR_WORKSPACE = -3,   /* workspace missing or too small */
    MTLATTN_ERR_LAUNCH = -4       /* HIP reported an error at launch */
};

/*
 * Problem description shared by every entry point. Mirrors the scalar part
 * of the reference's kernel argument block `Params` (src/ext.mm:44-57) plus
 * the bias strides of src/ext.mm:348-365.
 */
typedef struct mtlattn_problem {
    int32_t dtype;            /* MTLATTN_DTYPE_* of q/k/v */
    int32_t num_seqs;         /* B; cu_seqlens have B + 1 entries */
    int64_t total_q;          /* rows of q / out / dout */
    int64_t total_kv;         /* rows of k / v */
    int32_t num_heads_q;      /* Hq */
    int32_t num_heads_kv;     /* Hkv; Hq % Hkv == 0 */
    int32_t head_dim;         /* D */
    int32_t max_seqlen_q;     /* caller's bound on q lengths: up to 16 routes to decode. Too
                               * small a bound: rows past a sequence's first 16 / (heads per
                               * group) are computed slowly on calls that decode runs one
                               * workgroup per item (fewer than 2048 keys a sequence, or K
                               * and V below 0.9 GB), and left unwritten on the others */
    float scale;              /* logit = scale * q.k (+ bias) */
    int32_t causal;           /* 0 / 1 */
    int32_t window;           /* <= 0: no sliding window */
    const int32_t* cu_seqlens_q;   /* device int32 [B + 1] */
    const int32_t* cu_seqlens_kv;  /* device int32 [B + 1] */
    const float* bias;        /* optional fp32 additive mask, NULL = none */
    int64_t bias_q_stride;    /* elements between query rows of bias */
    int64_t bias_h_stride;    /* elements between heads; 0 = broadcast over heads */
    int64_t bias_kv_cols;     /* size of bias's key dim; keys beyond read as 0 */
    /* Row addressing of bias (no counterpart in the reference, which indexes
     * by global query row): 0 = row of global query r at r * bias_q_stride;
     * 1 = row of query i of sequence s at s * bias_seq_stride +
     * min(i, bias_seq_rows - 1) * bias_q_stride (a dense [B or 1, H or 1,
     * Nq, Nkv] mask used in place, stride 0 for a broadcast batch dim). */
    int32_t bias_seq_local;
    int64_t bias_seq_stride;
    int64_t bias_seq_rows;
} mtlattn_problem;

/* Version of this header the library was built from (== MTLATTN_ABI_VERSION). */
int mtlattn_abi_version(void);

/* Message describing the last failure on this thread ("" if none). */
const char* mtlattn_last_error(void);

/* Compute-unit count of `device` (256 on MI355X); <= 0 on error.
 * Replaces _C.gpu_core_count (src/ext.mm:785). */
int mtlattn_gpu_core_count(int device);

/*
 * Forward: out = softmax(scale * q k^T + bias + mask) v per sequence, plus the
 * natural-log LSE per (row, head) when `lse` is non-NULL.
 * Replaces _C.varlen_attention (src/ext.mm:293-489) including its routing:
 * few-query / long-KV calls go to split-KV decode + combine
 * (src/ext.mm:367-390; here also with a window or a bias, which the
 * reference sends to its flash forward), everything else to the flash
 * forward.
 *   out : contiguous [total_q, Hq, D], same dtype as q
 *   lse : NULL or fp32 [total_q, Hq] (rows with no allowed key get -inf)
 * Workspace: the split-KV partials of calls routed to decode (few-query calls
 * of fewer than 2048 keys a sequence run without one, one workgroup per
 * sequence and kv head); fp32 partials of O and the LSE for fp16/bf16 problems
 * with few query rows against many keys (none needed: unsplit); for fp32
 * problems on the fp32 matrix-core kernels whose grid would leave CUs idle,
 * fp32 partials of 2-8 key splits (a smaller workspace runs them unsplit);
 * otherwise none.
 */
size_t mtlattn_varlen_fwd_workspace_size(const mtlattn_problem* p);
int mtlattn_varlen_fwd(const mtlattn_problem* p,
                       const void* q, int64_t q_row_stride,
                       const void* k, int64_t k_row_stride,
                       const void* v, int64_t v_row_stride,
                       void* out, float* lse,
                       void* workspace, size_t workspace_bytes,
                       void* stream);

/*
 * The forward above, allocating nothing and taking no workspace. No
 * counterpart in the reference: for callers that cannot allocate device
 * memory -- code under HIP graph capture, tight serving (decode) loops,
 * harnesses that forbid allocation. Same routing, kernels and results as
 * mtlattn_varlen_fwd (bitwise); the split-KV partials of calls routed to
 * decode, and the key-split partials of fp32 and 16-bit forwards on small
 * grids (sized to fit it), live in a static device array of MTLATTN_NOALLOC_SCRATCH_BYTES per
 * GPU, set up on the first call on each GPU (do that call outside capture)
 * and held until the process ends. Calls whose partials would exceed it
 * (mtlattn_varlen_fwd_workspace_size(p) > MTLATTN_NOALLOC_SCRATCH_BYTES)
 * return MTLATTN_ERR_WORKSPACE. Every call on a GPU shares that GPU's
 * array: calls that overlap on one GPU (other streams, other threads) race
 * and must be serialised by the caller. Each call rewrites every partial it
 * reads, so nothing carries over from earlier calls.
 */
#define MTLATTN_NOALLOC_SCRATCH_BYTES (64ll << 20)
int mtlattn_varlen_fwd_noalloc(const mtlattn_problem* p,
                               const void* q, int64_t q_row_stride,
                               const void* k, int64_t k_row_stride,
                               const void* v, int64_t v_row_stride,
                               void* out, float* lse,
                               void* stream);

/*
 * Dense forward for the SDPA adapter: q [B, Hq, Nq, D], k / v [B, Hkv, Nkv, D]
 * read in place through element strides of their B, H and N dims (D contiguous),
 * out contiguous [B, Hq, Nq, D]. No counterpart in the reference, whose adapter
 * copies all four into packed rows (mtlattn/__init__.py:162-181). `p` gives
 * dtype, num_seqs (= B), the head counts, head_dim, scale, causal and a bias
 * with bias_seq_local; its cu_seqlens, token totals and window are not read.
 * lens: NULL, or device int32 [B] (Nq == Nkv): tokens past lens[b] (clamped to
 * [0, Nq]) are padding -- not attended, their output rows 0. fp16/bf16,
 * D in {64, 80, 88, 96, 128}, scale > 0, 16-byte aligned rows, and shapes that
 * mtlattn_varlen_fwd runs on its unsplit flash kernels; otherwise
 * MTLATTN_ERR_UNSUPPORTED with nothing launched (pack the rows and call
 * mtlattn_varlen_fwd). Same values as that. No workspace.
 */
int mtlattn_dense_fwd(const mtlattn_problem* p, int32_t Nq, int32_t Nkv,
                      const void* q, int64_t q_batch_stride, int64_t q_head_stride, int64_t q_row_stride,
                      const void* k, int64_t k_batch_stride, int64_t k_head_stride, int64_t k_row_stride,
                      const void* v, int64_t v_batch_stride, int64_t v_head_stride, int64_t v_row_stride,
                      const int32_t* lens, void* out, void* stream);

/*
 * Backward: (dq, dk, dv) of the forward above given dout and the forward's
 * out and lse. dk/dv of a kv head are summed over its Hq/Hkv query heads
 * inside the kernels (no atomics; bitwise run-to-run deterministic).
 * Replaces _C.varlen_attention_bwd (src/ext.mm:502-594). The reference needs
 * contiguous inputs (mtlattn/__init__.py:42-45); this entry also takes row
 * strides. dq/dk/dv are written contiguous in the input dtype. The
 * workspace (fp32 [total_q, Hq]) holds delta = rowsum(dO * O) of every row a
 * sequence owns when the call returns; at head dims 64 and 128 the dQ kernel
 * computes it (no separate preprocess launch), bitwise equal to
 * mtlattn_bwd_preprocess. On the fp32 matrix-core kernels the dQ kernel
 * computes delta too (equal to the preprocess up to fp32 rounding); for fp32
 * problems whose dQ or dK/dV grid would leave CUs idle, the size query adds
 * room (after delta, 256-byte aligned) for fp32 partials of 2-8 splits,
 * summed in a fixed order; a workspace of only the delta size runs unsplit.
 * The same holds for the dK/dV of fp16/bf16 problems whose key blocks would
 * leave CUs idle (up to 1 GiB of fp32 partials, by the number of tokens).
 */
size_t mtlattn_varlen_bwd_workspace_size(const mtlattn_problem* p);
int mtlattn_varlen_bwd(const mtlattn_problem* p,
                       const void* q, int64_t q_row_stride,
                       const void* k, int64_t k_row_stride,
                       const void* v, int64_t v_row_stride,
                       const void* out, int64_t out_row_stride,
                       const void* dout, int64_t dout_row_stride,
                       const float* lse,
                       void* dq, void* dk, void* dv,
                       void* workspace, size_t workspace_bytes,
                       void* stream);

/*
 * The backward above with row strides (elements) for dq and for dk and dv, so
 * that the gradients of a packed qkv or kv tensor are written in place. No
 * counterpart in the reference (its wrappers stack the three). fp16/bf16 on
 * the matrix-core kernels with 8-byte aligned rows; otherwise
 * MTLATTN_ERR_UNSUPPORTED before anything is launched. Same workspace,
 * kernels and values as mtlattn_varlen_bwd.
 */
int mtlattn_varlen_bwd_strided(const mtlattn_problem* p,
                               const void* q, int64_t q_row_stride,
                               const void* k, int64_t k_row_stride,
                               const void* v, int64_t v_row_stride,
                               const void* out, int64_t out_row_stride,
                               const void* dout, int64_t dout_row_stride,
                               const float* lse,
                               void* dq, int64_t dq_row_stride,
                               void* dk, void* dv, int64_t dkv_row_stride,
                               void* workspace, size_t workspace_bytes,
                               void* stream);

/*
 * delta[row, h] = sum_d dout[row, h, d] * out[row, h, d] in fp32.
 * Replaces the torch reduction at src/ext.mm:518 / bwd_delta_impl
 * (src/attention.metal:724-733). delta: fp32 [total_q, Hq].
 */
int mtlattn_bwd_preprocess(const mtlattn_problem* p,
                           const void* out, int64_t out_row_stride,
                           const void* dout, int64_t dout_row_stride,
                           float* delta, void* stream);

/*
 * dQ alone (test entry). Replaces _C.mpp_bwd_dq (src/ext.mm:656-711).
 * dq_dtype: MTLATTN_DTYPE_F32 (as the reference returns) or p->dtype.
 */
int mtlattn_bwd_dq(const mtlattn_problem* p,
                   const void* q, int64_t q_row_stride,
                   const void* k, int64_t k_row_stride,
                   const void* v, int64_t v_row_stride,
                   const void* dout, int64_t dout_row_stride,
                   const float* lse, const float* delta,
                   void* dq, int32_t dq_dtype, void* stream);

/*
 * dK and dV alone (test entry). Replaces _C.mpp_bwd_dkv (src/ext.mm:597-653).
 * dkv_dtype: MTLATTN_DTYPE_F32 (as the reference returns) or p->dtype.
 */
int mtlattn_bwd_dkv(const mtlattn_problem* p,
                    const void* q, int64_t q_row_stride,
                    const void* k, int64_t k_row_stride,
                    const void* v, int64_t v_row_stride,
                    const void* dout, int64_t dout_row_stride,
                    const float* lse, const float* delta,
                    void* dk, void* dv, int32_t dkv_dtype, void* stream);

/*
 * Split-KV decode with an explicit split count (test entry): each split
 * attends one chunk of every sequence's keys and writes a normalised fp32
 * partial O and its LSE; a combine kernel merges them and also writes the
 * final LSE when `lse` is non-NULL. num_splits == 1 is a plain forward.
 * Replaces _C.attn_splitkv (src/ext.mm:716-773; kernels
 * src/attn_mpp.metal:384-535). Requires fp16/bf16, D in {64, 128},
 * max_seqlen_q <= 16 (query rows of a kv head handled in groups of 16).
 * Bias and window are honoured (the reference's split path has neither);
 * with a window the splits divide only the keys the sequence's rows can see.
 * Workspace: fp32 partial rows of D values plus one LSE each, 16 rows per
 * (kv head, head group, sequence, split).
 */
size_t mtlattn_attn_splitkv_workspace_size(const mtlattn_problem* p, int32_t num_splits);
int mtlattn_attn_splitkv(const mtlattn_problem* p,
                         const void* q, int64_t q_row_stride,
                         const void* k, int64_t k_row_stride,
                         const void* v, int64_t v_row_stride,
                         void* out, float* lse, int32_t num_splits,
                         void* workspace, size_t workspace_bytes,
                         void* stream);

/*
 * Decode over a paged KV cache. No counterpart in the reference (it has no
 * paged KV); the layout is FlashAttention's varlen call with a block table.
 * Same computation as the forward (causal, window, bias, LSE) for
 * max_seqlen_q <= 16, fp16/bf16, D in {64, 128}, through split-KV + combine.
 *   k_cache / v_cache : [num_pages, page_size, Hkv, D], token row strides
 *                       k_row_stride / v_row_stride (elements); a page is
 *                       page_size consecutive token rows
 *   block_table       : int32 [num_seqs, block_table_stride] on the device
 *                       (block_table_stride entries per sequence, all of
 *                       them readable); logical key j of sequence s is row
 *                       j % page_size of page
 *                       block_table[s * block_table_stride + min(j / page_size,
 *                       block_table_stride - 1)] (page indices are clamped
 *                       to [0, num_pages)), so the table needs
 *                       ceil(kv_len / page_size) entries per sequence
 *   p->cu_seqlens_kv  : logical KV lengths (prefix sums); p->total_kv is an
 *                       upper bound on cu_seqlens_kv[num_seqs], the sum of
 *                       the logical lengths (pages may be shared between
 *                       sequences, so it can exceed the cache capacity)
 *   page_size         : a multiple of 16
 *   max_seqlen_kv     : bound on the logical KV lengths (sizes the window
 *                       splits)
 * Work split: fixed KV chunks numbered by the logical prefix sums (slots for
 * p->total_kv keys) as on the contiguous decode path; with a window, equal
 * splits of each sequence's band.
 * Workspace: mtlattn_paged_decode_workspace_size(p, max_seqlen_kv) bytes.
 */
size_t mtlattn_paged_decode_workspace_size(const mtlattn_problem* p, int64_t max_seqlen_kv);
int mtlattn_paged_decode(const mtlattn_problem* p,
                         const void* q, int64_t q_row_stride,
                         const void* k_cache, int64_t k_row_stride,
                         const void* v_cache, int64_t v_row_stride,
                         int32_t page_size, int64_t num_pages,
                         const int32_t* block_table, int64_t block_table_stride,
                         int64_t max_seqlen_kv,
                         void* out, float* lse,
                         void* workspace, size_t workspace_bytes,
                         void* stream);

/*
 * A paged KV cache held in 8 bits. No counterpart in the reference. Pages,
 * token rows and the block table as for mtlattn_paged_decode; an element is a
 * code, and a value is its code times the scale of its block of tokens and kv
 * head. Codes: e4m3 (sign, 4 exponent and 3 mantissa bits, +-448 at most, one
 * NaN) or int8 (-127 .. 127).
 *   k, v            : codes [num_pages, page_size, Hkv, D], token row strides
 *                     k_row_stride / v_row_stride (elements), rows and strides
 *                     16-byte aligned (8-byte for writing and reading back)
 *   k_scale, v_scale: fp32 [num_pages, page_size / block, Hkv], contiguous
 *   block           : tokens that share a scale: 16, 32, 64, 128 or 256, and a
 *                     divisor of page_size
 * Writing and reading back take D a multiple of 8 in [16, 256] and
 * Hkv * D <= 65536; attention D in {64, 128}.
 */
enum {
    MTLATTN_CODE_E4M3 = 3,
    MTLATTN_CODE_INT8 = 4
};

typedef struct mtlattn_cache8 {
    int32_t code;             /* MTLATTN_CODE_* */
    int32_t page_size;
    int32_t block;
    int32_t num_heads_kv;
    int32_t head_dim;
    int64_t num_pages;
    void* k;
    int64_t k_row_stride;
    void* v;
    int64_t v_row_stride;
    float* k_scale;
    float* v_scale;
    const int32_t* block_table;    /* device int32 [num_seqs, block_table_stride] */
    int64_t block_table_stride;
} mtlattn_cache8;

/*
 * Writes rows k, v [total, Hkv, D] (dtype fp32 / fp16 / bf16, row strides in
 * elements, 16-byte aligned rows) into the cache: sequence s's rows
 * cu_seqlens[s] .. cu_seqlens[s + 1] become its last logical tokens, whose count
 * cu_seqlens_kv (prefix sums, with the new tokens) gives -- the offsets that the
 * attention over the cache then takes for its queries and keys.
 * For each block and kv head that gets rows, with a = the largest magnitude
 * among their finite values (at least 2^-92): need = the smallest power of two
 * with a <= 448 need (e4m3), a * fp32(1 / 127) (int8). A block that already
 * holds tokens of the sequence keeps a larger scale; a smaller one grows to
 * `need`, and the earlier tokens' codes are rounded to it. Codes are the nearest to value /
 * scale, ties to even; infinities take the largest code, NaN stays NaN in e4m3
 * and is 0 in int8. Nothing else of the cache changes.
 * Rows whose logical position is negative (more rows than tokens), or whose
 * table column or page does not exist, are not written. Blocks that get rows
 * must stand once in the block tables. Codes and scales must share memory neither
 * with each other nor with the rows (K and V side by side in the token rows of one
 * buffer, at the same stride, do not); such calls are refused.
 * No workspace; deterministic.
 */
int mtlattn_cache8_write(const mtlattn_cache8* c, int32_t dtype,
                         const void* k, int64_t k_row_stride,
                         const void* v, int64_t v_row_stride,
                         int64_t total, int32_t num_seqs,
                         const int32_t* cu_seqlens, const int32_t* cu_seqlens_kv,
                         void* stream);

/*
 * Reads the last tokens of each sequence back: rows cu_seqlens[s] ..
 * cu_seqlens[s + 1] of k and v (contiguous [total, Hkv, D], 16-byte aligned, of
 * type dtype) are its last logical tokens, code * scale in fp32, rounded to it. With
 * cu_seqlens = cu_seqlens_kv: all of them. Table columns and pages are clamped
 * as in the attention; rows of no sequence and of negative positions are 0.
 */
int mtlattn_cache8_read(const mtlattn_cache8* c, int32_t dtype,
                        void* k, void* v,
                        int64_t total, int32_t num_seqs,
                        const int32_t* cu_seqlens, const int32_t* cu_seqlens_kv,
                        void* stream);

/*
 * mtlattn_paged_decode over an 8-bit cache: same computation, options and
 * limits (p->dtype is the type of q and out), on values code * scale. Query rows
 * past the 16 / (heads per group) that p->max_seqlen_q promised come back NaN.
 * Rows of no sequence are left as they were. Keys that a row does not see (for
 * their place, the causal mask or the window) do not reach it, whatever their codes
 * and scales; those that it sees do as the definition says: an infinite v_scale makes
 * infinities, or NaN where signs meet or a code or a weight is 0. max_seqlen_kv
 * shapes the launch only; p->total_kv bounds the logical lengths.
 * Workspace: mtlattn_decode8_workspace_size(p, max_seqlen_kv) bytes.
 */
size_t mtlattn_decode8_workspace_size(const mtlattn_problem* p, int64_t max_seqlen_kv);
int mtlattn_decode8(const mtlattn_problem* p,
                    const void* q, int64_t q_row_stride,
                    const mtlattn_cache8* c, int64_t max_seqlen_kv,
                    void* out, float* lse,
                    void* workspace, size_t workspace_bytes,
                    void* stream);

/*
 * How mtlattn_decode8 would lay out `p` on the current device (256 CUs are assumed
 * without one): `waves` per workgroup, which take `heads` kv heads, waves / heads of
 * them each; the work in `pieces` pieces with partial results (0: a workgroup takes
 * whole sequences).
 */
int mtlattn_decode8_layout(const mtlattn_problem* p, int64_t max_seqlen_kv,
                           int32_t* waves, int32_t* heads, int32_t* pieces);

/*
 * Position rotation of queries and keys, with their per-head norms in the same
 * pass. No counterpart in the reference. For each row and head, x of D values:
 *   xh = x / sqrt(mean(x^2) + eps) * weight      (xh = x without weights)
 *   y_a = scale (a cos t - b sin t), y_b = scale (b cos t + a sin t),
 *   t = positions[row] * inv_freq[i]
 * for the pairs (a, b) = (xh[i], xh[i + rotary_dim / 2]), or, interleaved,
 * (xh[2 i], xh[2 i + 1]), i < rotary_dim / 2; elements from rotary_dim on are xh.
 * Angles are formed in 64 bits, all else in fp32, rounded once.
 */
typedef struct mtlattn_rotary {
    int32_t dtype;            /* MTLATTN_DTYPE_* of the rows */
    int32_t num_heads_q;
    int32_t num_heads_kv;
    int32_t head_dim;         /* D, 1 .. 256 */
    int32_t rotary_dim;       /* even, 0 (no rotation) .. D */
    int32_t interleaved;      /* 0 / 1 */
    float scale;
    float eps;                /* finite, >= 0 (not read without weights) */
    int64_t total;            /* rows */
    const int32_t* positions;      /* device int32 [total] */
    const float* inv_freq;         /* device fp32 [rotary_dim / 2] */
    const void* q_weight;          /* device [D], both or neither (NULL: no norms) */
    const void* k_weight;
    int32_t weight_dtype;     /* MTLATTN_DTYPE_F32, or dtype */
} mtlattn_rotary;

/*
 * q [total, Hq, D] and k [total, Hkv, D] into q_out and k_out (row strides in
 * elements). q_out may be q, k_out may be k (same pointer and stride);
 * otherwise outputs share memory with nothing. No workspace.
 * D and rotary_dim multiples of 16 and 16-byte aligned rows take the fast kernel.
 */
int mtlattn_rotary_fwd(const mtlattn_rotary* r,
                       const void* q, int64_t q_row_stride,
                       const void* k, int64_t k_row_stride,
                       void* q_out, int64_t q_out_row_stride,
                       void* k_out, int64_t k_out_row_stride,
                       void* stream);

/*
 * Its backward: from dq_out and dk_out, the gradients dq and dk of q and k and,
 * with norms, of the weights (dq_weight, dk_weight [D] of weight_dtype; NULL:
 * not wanted). q and k are read with norms only. Outputs share memory with
 * nothing. Workspace (with norms): fp32 sums of the weights' gradients, added in
 * a fixed order: the same results from run to run.
 */
size_t mtlattn_rotary_bwd_workspace_size(const mtlattn_rotary* r);
int mtlattn_rotary_bwd(const mtlattn_rotary* r,
                       const void* q, int64_t q_row_stride,
                       const void* k, int64_t k_row_stride,
                       const void* dq_out, int64_t dq_out_row_stride,
                       const void* dk_out, int64_t dk_out_row_stride,
                       void* dq, int64_t dq_row_stride,
                       void* dk, int64_t dk_row_stride,
                       void* dq_weight, void* dk_weight,
                       void* workspace, size_t workspace_bytes,
                       void* stream);

/*
 * New rows into the 16-bit paged cache of mtlattn_paged_decode: sequence s's rows
 * cu_seqlens[s] .. cu_seqlens[s + 1] of k and v [r->total, Hkv, D] become its last
 * logical tokens, whose count cu_seqlens_kv (prefix sums, with the new tokens)
 * gives. k is normed and rotated on the way as r says (rotary_dim 0, k_weight NULL:
 * copied), and so is q, when it is not NULL, into q_out. r->positions NULL: a
 * token's place in its sequence. With q NULL, q_weight and num_heads_q are
 * not used. dtype fp16 or bf16, any page_size >= 1.
 * Rows whose logical position is negative, or whose table column or page does not
 * exist, are not written to the cache (their q is still turned); q_out rows of no
 * sequence are 0. Nothing else of the cache changes. Cache rows that get tokens must
 * stand once in the block tables. q_out may be q; otherwise caches, q_out and the rows
 * must not share memory (K and V side by side in the token rows of one buffer do not);
 * such calls are refused. No workspace; deterministic.
 */
int mtlattn_cache_append(const mtlattn_rotary* r,
                         const void* q, int64_t q_row_stride,
                         void* q_out, int64_t q_out_row_stride,
                         const void* k, int64_t k_row_stride,
                         const void* v, int64_t v_row_stride,
                         void* k_cache, int64_t k_cache_row_stride,
                         void* v_cache, int64_t v_cache_row_stride,
                         int32_t page_size, int64_t num_pages,
                         const int32_t* block_table, int64_t block_table_stride,
                         int32_t num_seqs,
                         const int32_t* cu_seqlens, const int32_t* cu_seqlens_kv,
                         void* stream);

/*
 * Attention of a tree of drafted tokens over the cache of mtlattn_paged_decode. No
 * counterpart in the reference. Sequence s's queries, rows cu_seqlens_q[s] ..
 * cu_seqlens_q[s + 1], are its last logical tokens, whose keys are in the cache
 * already (mtlattn_cache_append); query i sees every key before them, and of them
 * token j iff tree_mask's byte j of the query's row is not 0 (j < tree_cols; itself
 * included only if the mask says so).
 *   out[row] = sum_j softmax_j(p->scale * q k_j) v_j over the seen keys, lse as for the
 *   forward; rows that see no key: 0 and -inf. Keys that a row does not see do not reach
 *   it, whatever their values. Scores, softmax and sums are fp32; the weights multiply V
 *   with 16 bits (bf16: two bf16 numbers each) or 22 (fp16); the result is rounded once.
 *   p            : dtype fp16/bf16, D in {64, 128}, cu_seqlens_kv the logical lengths
 *                  (prefix sums); total_kv, causal, window and bias are not read.
 *                  max_seqlen_q shapes the launch only, and so does max_seqlen_kv
 *   tree_mask    : bytes [total_q, tree_cols], row stride in bytes, tree_cols in [1, 256]
 *   the cache    : as for mtlattn_paged_decode, page_size a multiple of 16
 * Rows of no sequence are left as they were. Deterministic.
 * Workspace: mtlattn_tree_decode_workspace_size(p, max_seqlen_kv) bytes, 16-byte aligned.
 */
size_t mtlattn_tree_decode_workspace_size(const mtlattn_problem* p, int64_t max_seqlen_kv);
int mtlattn_tree_decode(const mtlattn_problem* p,
                        const void* q, int64_t q_row_stride,
                        const void* k_cache, int64_t k_row_stride,
                        const void* v_cache, int64_t v_row_stride,
                        int32_t page_size, int64_t num_pages,
                        const int32_t* block_table, int64_t block_table_stride,
                        int64_t max_seqlen_kv,
                        const uint8_t* tree_mask, int64_t tree_mask_row_stride, int32_t tree_cols,
                        void* out, float* lse,
                        void* workspace, size_t workspace_bytes,
                        void* stream);

/* Number of split-KV work-item slots per (kv head, head group) the forward's
 * decode routing would use for `p` (0 = the call is not routed to split-KV).
 * The automatic path cuts each sequence's KV into fixed-length chunks (about
 * 18 work items of one wave per CU, or 3 of one workgroup on short streams) rather than a fixed number of splits per sequence,
 * so ragged KV lengths stay balanced; with a window each sequence gets a
 * fixed number of equal splits of its window band instead (slots =
 * num_seqs * splits). Retunes src/ext.mm:372-388. */
int32_t mtlattn_decode_num_splits(const mtlattn_problem* p);

/*
 * Key-padding pack / unpack for the SDPA adapter. No counterpart in the
 * reference's _C: its adapter (mtlattn/__init__.py:202-249) copies each
 * batch's valid prefix in Python after pulling the lengths to the host; these
 * do it on the device with no host synchronisation.
 *
 * mtlattn_pack_padded: dense src [B, H, N, D] (element strides sb, sh, sn of
 * the B, H, N dims; D contiguous) -> packed rows dst [B * N, H, D]. Batch b's
 * first lens[b] tokens (clamped to [0, N]) go to rows cu[b] + n, where
 * cu = prefix sums of the lengths, written to cu_out [B + 1] (int32, device);
 * the padded tokens follow all valid ones. Use dst with cu_out as the varlen
 * q/k/v and cu_seqlens (rows past cu_out[B] belong to no sequence).
 * mtlattn_unpack_padded: packed rows src [B * N, H, D] -> dense dst
 * [B, H, N, D] (strides sb, sh, sn): token (b, n) takes row cu[b] + n when
 * n < lens[b], zeros otherwise.
 * dtype is MTLATTN_DTYPE_*; all pointers are device pointers.
 */
int mtlattn_pack_padded(int32_t dtype, int32_t B, int32_t N, int32_t H, int32_t D,
                        const void* src, int64_t sb, int64_t sh, int64_t sn,
                        const int32_t* lens, int32_t* cu_out, void* dst, void* stream);
int mtlattn_unpack_padded(int32_t dtype, int32_t B, int32_t N, int32_t H, int32_t D,
                          const void* src, const int32_t* lens, const int32_t* cu,
                          void* dst, int64_t sb, int64_t sh, int64_t sn, void* stream);

/*
 * Sets *flag = 1 if any of the `bytes` bytes at a and b (device pointers)
 * differ, else leaves it; flag is an int32 that the device can write, such as
 * pinned host memory, cleared by the caller. For the SDPA adapter, which keeps
 * what it decided about a mask only while the mask's content stays.
 */
int mtlattn_content_differs(const void* a, const void* b, int64_t bytes, int32_t* flag, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MTLATTN_CAPI_H */
