/*
 * flexatt.h — C ABI of the MI355X (gfx950) flash-attention library
 * (libflexatt.so).
 *
 * The reference (dropletzhu/npu-flex-att) has no C ABI: its host wrappers in
 * npu_flash_attention.py launch Triton kernels directly.  Each entry point
 * below replaces one such launch (or one torch op of the wrapper) and is what
 * a foreign-function binding of that wrapper calls; the Python host layer of
 * this repository binds them with ctypes.
 *
 * Conventions
 *  - Tensors are 4-D [B, H, S, D] views: a device pointer plus element
 *    strides.  The innermost stride must be 1 and every row must start on a
 *    16-byte boundary (data pointer and the b/h/s strides times the element
 *    size are multiples of 16 bytes).  Batch and head strides may be 0
 *    (broadcast).
 *  - q, o, dout and dq have shape [B, Hq, Sq, D]; k, v, dk and dv have shape
 *    [B, Hkv, Skv, D]; Hq is a multiple of Hkv and query head h reads KV head
 *    h / (Hq / Hkv).
 *  - lse and delta are contiguous fp32 [B, Hq, Sq]; lse is the natural-log
 *    log-sum-exp of the masked, scaled (and soft-capped, ALiBi-biased) scores.
 *  - All work is enqueued on `stream` (a hipStream_t; NULL = the null
 *    stream) and is asynchronous.  Nothing is allocated or freed: the caller
 *    owns every buffer (flexatt_fwd_decode_noalloc alone uses a fixed
 *    library-owned device buffer instead of a workspace argument).  Results
 *    are bitwise deterministic.
 *  - Return value: FLEXATT_OK, a negative FLEXATT_E* code for a rejected
 *    argument (nothing is launched), or a positive hipError_t from a launch.
 */
#ifndef FLEXATT_H_
#define FLEXATT_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element type of q/k/v/o/dout/dq/dk/dv. */
enum flexatt_dtype { FLEXATT_F32 = 0, FLEXATT_F16 = 1, FLEXATT_BF16 = 2 };

/* Status codes (negative: argument rejected before any launch). */
enum flexatt_status {
  FLEXATT_OK = 0,
  FLEXATT_EINVAL = -1,     /* null pointer, non-positive size, bad flag */
  FLEXATT_EDTYPE = -2,     /* unknown dtype */
  FLEXATT_EHEADDIM = -3,   /* head_dim not in {32, 64, 128, 256} */
  FLEXATT_ESHAPE = -4,     /* heads_q % heads_kv != 0, or sizes overflow */
  FLEXATT_ELAYOUT = -5,    /* innermost stride != 1 or a row not 16-byte aligned */
  FLEXATT_ERANGE = -6,     /* problem outside an entry point's range (see its comment) */
  FLEXATT_ESCRATCH = -7    /* problem needs more than the fixed scratch buffer of a no-alloc entry point */
};

/* One [B, H, S, D] tensor: device pointer and element strides. */
typedef struct flexatt_tensor {
  void* data;
  int64_t stride_b, stride_h, stride_s, stride_d;
} flexatt_tensor;

/* The attention problem: sizes and the mask primitives.
 * npu_flash_attention.py:606-616 (forward signature) and :659-668 (backward)
 * carry the same fields as Python arguments; block_m / block_n are tiling
 * hints there and have no counterpart here. */
typedef struct flexatt_problem {
  int32_t dtype;          /* enum flexatt_dtype */
  int32_t batch;          /* B */
  int32_t heads_q;        /* Hq */
  int32_t heads_kv;       /* Hkv */
  int32_t seqlen_q;       /* Sq */
  int32_t seqlen_kv;      /* Skv (any value >= 1; no tile-multiple requirement) */
  int32_t head_dim;       /* D in {32, 64, 128, 256} */
  float scale;            /* softmax scale (the caller applies the 1/sqrt(D) default) */
  int32_t causal;         /* 1: keep j <= i (top-left aligned) */
  int32_t sliding_window; /* W > 0: keep i - j <= W; 0: off */
  float soft_cap;         /* c > 0: x -> c * tanh(x / c); 0: off */
  const float* alibi_slopes; /* device fp32 [Hq]: x += slope[h] * (i - j); NULL: off */
  /* Interval masks (no counterpart in the reference, which lists document
   * masking and PrefixLM as future work, README.md:219, DESIGN.md:374):
   * device int32 [B, Sq, 2] holding, for query row i of batch b, the range
   * [lo, hi) of keys it may attend, on top of the other primitives.  Both
   * bounds must be non-decreasing in i.  A document mask is symmetric: the
   * range of positions of i's document (then col_bounds may stay NULL and
   * seqlen_q == seqlen_kv).  NULL: off. */
  const int32_t* doc_bounds;
  /* The transpose of doc_bounds for a mask that is not symmetric (PrefixLM):
   * device int32 [B, Skv, 2], for key j the range [lo, hi) of query rows
   * that may attend it, both non-decreasing in j; it must describe the same
   * mask as doc_bounds.  NULL: doc_bounds is symmetric and read as both. */
  const int32_t* col_bounds;
  /* Block-sparse mask (the reference lists the block-sparse BlockMask index
   * format as unsupported, README.md:198): device uint8 [B, block_heads,
   * ceil(Sq / 128), ceil(Skv / 128)]; a zero entry removes the 128 x 128
   * block of (query rows, keys) from the attention of those heads, on top of
   * the other primitives.  block_heads is 1 (one map for every head) or
   * heads_q; ceil(Skv / 128) <= 2048.  NULL: off. */
  const uint8_t* block_map;
  int32_t block_heads;
  int32_t reserved; /* 0 */
} flexatt_problem;

/* The interval bounds of a document mask (flexatt_problem.doc_bounds) from
 * document ids: `ids` is a contiguous device array [batch, seqlen] of integers
 * of ids_bytes (1, 2, 4 or 8) bytes, and bounds[b][s] receives the range
 * [lo, hi) of the maximal run of equal ids that holds position s.  No
 * counterpart in the reference. */
int flexatt_document_bounds(const void* ids, int ids_bytes, int batch, int seqlen, int32_t* bounds, void* stream);

/* Forward: o = softmax(mask(score(q k^T))) v and lse.
 * Replaces the flash_attn_fwd_kernel launch of npu_flash_attention_forward,
 * npu_flash_attention.py:634-652. */
int flexatt_fwd(const flexatt_problem* p, const flexatt_tensor* q, const flexatt_tensor* k,
                const flexatt_tensor* v, const flexatt_tensor* o, float* lse, void* stream);

/* flexatt_fwd without its choice by size: the kernels of large problems, which
 * small ones otherwise leave for the split ones (to compare the two). */
int flexatt_fwd_regular(const flexatt_problem* p, const flexatt_tensor* q, const flexatt_tensor* k,
                        const flexatt_tensor* v, const flexatt_tensor* o, float* lse, void* stream);

/* Split-KV decode forward (flash-decoding): the results of flexatt_fwd for
 * problems with few query rows per KV head, computed by splitting the KV
 * range over many workgroups.  Range: fp16/bf16, head_dim <= 128 and
 * (heads_q / heads_kv) * seqlen_q <= 32; otherwise FLEXATT_ERANGE.
 * `workspace` is caller-owned device memory of at least
 * flexatt_fwd_decode_workspace(p) bytes, 16-byte aligned; it holds partial
 * results between the two kernels of this call and may be reused once the
 * call's work on `stream` is done.  Same o / lse as flexatt_fwd up to the
 * rounding of a different summation order; bitwise deterministic.
 * Replaces the unused split-KV pair flash_attn_fwd_split_kv_kernel /
 * flash_attn_fwd_reduce_kernel, npu_flash_attention.py:169-293. */
size_t flexatt_fwd_decode_workspace(const flexatt_problem* p); /* 0: outside the range */
int flexatt_fwd_decode(const flexatt_problem* p, const flexatt_tensor* q, const flexatt_tensor* k,
                       const flexatt_tensor* v, const flexatt_tensor* o, float* lse, void* workspace,
                       size_t workspace_bytes, void* stream);

/* The split-KV forward over its whole range: that of flexatt_fwd_decode and
 * head_dim 256 (else FLEXATT_ERANGE, and 0 bytes); otherwise as
 * flexatt_fwd_decode. */
size_t flexatt_fwd_split_workspace(const flexatt_problem* p); /* 0: outside the range */
int flexatt_fwd_split(const flexatt_problem* p, const flexatt_tensor* q, const flexatt_tensor* k,
                      const flexatt_tensor* v, const flexatt_tensor* o, float* lse, void* workspace,
                      size_t workspace_bytes, void* stream);

/* Split-KV decode forward that allocates nothing.  No counterpart in the
 * reference: it is for callers that cannot allocate device memory or pass a
 * workspace (code under HIP graph capture, tight serving loops, harnesses
 * that forbid hipMalloc).  Same kernels, split plan and results as
 * flexatt_fwd_decode (bitwise equal), with the partial results in a
 * library-owned device buffer of FLEXATT_NOALLOC_SCRATCH_BYTES per GPU,
 * held until the process ends; nothing is allocated or freed per call.
 * Range: that of flexatt_fwd_decode (else FLEXATT_ERANGE), and
 * flexatt_fwd_decode_workspace(p) <= FLEXATT_NOALLOC_SCRATCH_BYTES (else
 * FLEXATT_ESCRATCH, checked before any GPU work).  `stream` must belong to
 * the current device.  Every call on one GPU shares that GPU's buffer:
 * calls that overlap on one GPU (on different streams or host threads)
 * race, so the caller serialises them; calls in order on one stream are
 * safe (each one overwrites every partial it reads). */
#define FLEXATT_NOALLOC_SCRATCH_BYTES (16u << 20)
int flexatt_fwd_decode_noalloc(const flexatt_problem* p, const flexatt_tensor* q, const flexatt_tensor* k,
                               const flexatt_tensor* v, const flexatt_tensor* o, float* lse, void* stream);

/* Backward pre-pass: delta[b,h,i] = sum_d o * dout in fp32.
 * Replaces the torch op at npu_flash_attention.py:681-685. */
int flexatt_bwd_delta(const flexatt_problem* p, const flexatt_tensor* o, const flexatt_tensor* dout,
                      float* delta, void* stream);

/* Backward dQ (needs lse and delta).
 * Replaces the flash_attn_bwd_dq_kernel launch, npu_flash_attention.py:695-712. */
int flexatt_bwd_dq(const flexatt_problem* p, const flexatt_tensor* q, const flexatt_tensor* k,
                   const flexatt_tensor* v, const flexatt_tensor* dout, const float* lse,
                   const float* delta, const flexatt_tensor* dq, void* stream);

/* Backward Delta and dQ in one pass where the dQ kernel can form Delta itself
 * (fp16/bf16, head_dim 64 or 128, no interval or block mask; otherwise the Delta
 * pass then dQ): delta (the caller's fp32 [B,Hq,Sq] buffer) receives sum_d o * dout,
 * for flexatt_bwd_dkdv after it.  Replaces the Delta op and the
 * flash_attn_bwd_dq_kernel launch of npu_flash_attention_backward,
 * npu_flash_attention.py:681-712. */
int flexatt_bwd_dq_delta(const flexatt_problem* p, const flexatt_tensor* q, const flexatt_tensor* k,
                         const flexatt_tensor* v, const flexatt_tensor* o, const flexatt_tensor* dout,
                         const float* lse, float* delta, const flexatt_tensor* dq, void* stream);

/* Backward dK/dV with the GQA group sum folded in: dk/dv are [B, Hkv, Skv, D].
 * Replaces the flash_attn_bwd_dkdv_kernel launch plus the group sum,
 * npu_flash_attention.py:714-737. */
int flexatt_bwd_dkdv(const flexatt_problem* p, const flexatt_tensor* q, const flexatt_tensor* k,
                     const flexatt_tensor* v, const flexatt_tensor* dout, const float* lse,
                     const float* delta, const flexatt_tensor* dk, const flexatt_tensor* dv,
                     void* stream);

/* Whole backward: delta (into the caller's fp32 [B,Hq,Sq] `delta` buffer)
 * and dQ (flexatt_bwd_dq_delta), then dK/dV.  Replaces the kernel launches and torch ops of
 * npu_flash_attention_backward, npu_flash_attention.py:659-739. */
int flexatt_bwd(const flexatt_problem* p, const flexatt_tensor* q, const flexatt_tensor* k,
                const flexatt_tensor* v, const flexatt_tensor* o, const flexatt_tensor* dout,
                const float* lse, float* delta, const flexatt_tensor* dq, const flexatt_tensor* dk,
                const flexatt_tensor* dv, void* stream);

/* Bytes of work-queue counters at the end of the staged-dS workspace. */
#define FLEXATT_BWD_QUEUE_BYTES 256

/* Backward with dS staged through HBM (fp16/bf16 at head_dim 64, 128 or
 * 256; fp32 at every head_dim).  The dK/dV kernel already forms dS
 * for every attended pair; it writes those values (rounded to the input
 * dtype, as its own dK MFMAs consume them) to a caller-owned workspace, and
 * the dQ kernel forms dQ = scale * dS K from them instead of recomputing S
 * and dP.  The workspace holds 2 bytes (fp32: 4 bytes) per attended (query
 * row, KV row) pair of each query head, in 32 x 128 units over the causal /
 * window band (interval and block masks keep that layout; masked pairs hold
 * zeros, and the units of removed 128 x 128 blocks, or fp16/bf16 units whose
 * keys an interval mask keeps from the tile's rows, are neither written nor
 * read), followed by FLEXATT_BWD_QUEUE_BYTES of
 * work-queue counters:
 * flexatt_bwd_workspace(p) bytes in all (0: the problem is outside this
 * range), 16-byte aligned, not zeroed, reusable once the call's work on
 * `stream` is done.  Same results as flexatt_bwd up to fp32 summation
 * order; bitwise deterministic.
 *
 * flexatt_bwd_ws: the whole backward (replaces the Delta op, both kernel
 * launches and the group sum of npu_flash_attention_backward,
 * npu_flash_attention.py:681-737): the Delta pass into `delta`, dK/dV
 * writing dS, then dQ.  Past the first workgroup per CU, the dK/dV and dQ
 * workgroups take the longest remaining work items from the queue counters
 * (which the Delta pass clears), so that faster XCDs take more work (fp16/
 * bf16); with a workspace of only the dS band's size the static order is
 * kept.  Outside
 * the range it runs flexatt_bwd and the workspace may be NULL.
 *
 * Bounded memory.  The band grows as Sq * Skv (about 1 byte per (query row,
 * KV row) pair of each query head for causal fp16/bf16, 1.1 GB at B=2 Hq=32
 * S=4096), while the reference's backward needs O(S) memory
 * (npu_flash_attention.py:675-685).  flexatt_bwd_ws therefore also accepts:
 *  - a workspace smaller than the whole band but holding the band of at
 *    least one (batch, KV head) group (G = heads_q / heads_kv query heads):
 *    the staged backward then runs in passes over chunks of whole groups
 *    (whole batches when one fits, else KV heads of one batch), reusing the
 *    workspace pass after pass on `stream`; smaller: FLEXATT_EINVAL;
 *  - workspace == NULL with workspace_bytes == 0: the recomputing backward
 *    (flexatt_bwd), O(S) memory.
 * flexatt_bwd_workspace_limited(p, limit) is the size to allocate under a
 * byte budget: the whole band (plus the queue counters) when it fits, else
 * the most whole groups that fit, else 0 (no staging: pass NULL, 0).  Passes
 * give the same results as one pass up to fp32 summation order. */
size_t flexatt_bwd_workspace(const flexatt_problem* p);
size_t flexatt_bwd_workspace_limited(const flexatt_problem* p, size_t limit_bytes);
/* Whether staging pays for p: 1 when p is in the staged range and the staged
 * backward measured faster than the recomputing one on MI355X, 0 otherwise
 * (out of range, or fp16/bf16 at head_dim 64 without soft-cap and without
 * document, prefix or block-map masks, where the recomputing backward is
 * 2-15% faster).  Advisory: flexatt_bwd_ws stages whenever it is given a
 * workspace.  No counterpart in the reference, which has one backward. */
int flexatt_bwd_prefers_staging(const flexatt_problem* p);
int flexatt_bwd_ws(const flexatt_problem* p, const flexatt_tensor* q, const flexatt_tensor* k,
                   const flexatt_tensor* v, const flexatt_tensor* o, const flexatt_tensor* dout,
                   const float* lse, float* delta, const flexatt_tensor* dq, const flexatt_tensor* dk,
                   const flexatt_tensor* dv, void* workspace, size_t workspace_bytes, void* stream);

/* Whole backward for problems that fill few workgroups of the other two: the
 * Delta pass into `delta`, then dK/dV and dQ in one launch whose items split
 * their streams of tiles over the waves of a workgroup, and the long dK/dV
 * streams over several workgroups (fp32 sums in the workspace, added by one
 * more launch).  Range: head_dim <= 128 without a block map (else
 * FLEXATT_ERANGE).  `workspace`: flexatt_bwd_split_workspace(p) bytes, 16-byte
 * aligned, not zeroed, reusable once the call's work on `stream` is done; NULL
 * when that is 0.  Same results as flexatt_bwd up to fp32 summation order;
 * bitwise deterministic.  flexatt_bwd_prefers_split(p): 1 where it measured
 * faster on MI355X than the staged and the recomputing backward, else 0. */
int flexatt_bwd_prefers_split(const flexatt_problem* p);
size_t flexatt_bwd_split_workspace(const flexatt_problem* p);
int flexatt_bwd_split(const flexatt_problem* p, const flexatt_tensor* q, const flexatt_tensor* k,
                      const flexatt_tensor* v, const flexatt_tensor* o, const flexatt_tensor* dout,
                      const float* lse, float* delta, const flexatt_tensor* dq, const flexatt_tensor* dk,
                      const flexatt_tensor* dv, void* workspace, size_t workspace_bytes, void* stream);

/* Bytes worth adding to a whole-band workspace of flexatt_bwd_ws (after the
 * queue counters): where a KV block per CU leaves the dK/dV launch waiting for
 * its longest blocks, flexatt_bwd_ws then shares each block's query tiles
 * between workgroups and adds their fp32 sums from there, the same results up
 * to summation order.  0: nothing to gain. */
size_t flexatt_bwd_ws_parts_bytes(const flexatt_problem* p);

/* The two kernels of flexatt_bwd_ws on their own (FLEXATT_ERANGE outside
 * its range).  flexatt_bwd_dkdv_ds replaces the flash_attn_bwd_dkdv_kernel
 * launch and the group sum (npu_flash_attention.py:714-737) and also fills
 * the workspace; flexatt_bwd_dq_ds replaces the flash_attn_bwd_dq_kernel
 * launch (:695-712) and reads the workspace a flexatt_bwd_dkdv_ds call on
 * the same problem wrote before it on the stream.  Both keep the static work
 * order (the queue counters are not used). */
int flexatt_bwd_dkdv_ds(const flexatt_problem* p, const flexatt_tensor* q, const flexatt_tensor* k,
                        const flexatt_tensor* v, const flexatt_tensor* dout, const float* lse,
                        const float* delta, const flexatt_tensor* dk, const flexatt_tensor* dv,
                        void* workspace, size_t workspace_bytes, void* stream);
int flexatt_bwd_dq_ds(const flexatt_problem* p, const flexatt_tensor* k, const void* workspace,
                      size_t workspace_bytes, const flexatt_tensor* dq, void* stream);

/* ---------------------------------------------------------------- positions
 * and the K/V cache.  None of the entry points below has a counterpart in the
 * reference, whose inputs are already positioned and which keeps no cache.
 * `cache` tensors are [B, Hkv, cache_rows, D] views like any other; `lengths`
 * is device int32 [B], the rows of each sequence that are in use. */

/* Rotary positions.  Pair i of the first rotary_dim elements of a head, elements
 * (i, i + rotary_dim / 2), or (2i, 2i + 1) when interleaved, is turned by
 * position * inv_freq[i] radians (the product in 64 bits) and scaled by
 * magnitude; the other elements are copied.  Rounded once. */
typedef struct flexatt_rotary {
  int32_t dtype;        /* enum flexatt_dtype */
  int32_t batch;        /* B */
  int32_t heads_q;      /* Hq >= 1; in flexatt_rotary_append also 0: no q */
  int32_t heads_kv;     /* Hkv >= 0; 0: no k */
  int32_t seqlen;       /* S, new tokens per sequence (FLEXATT_ERANGE: more than a launch has work-items,
                         * 2^32 - 1, of which B S D / 2 are taken at most) */
  int32_t head_dim;     /* D in {32, 64, 128, 256} */
  int32_t rotary_dim;   /* even, 0 .. D; 0: nothing is turned and inv_freq may be NULL */
  int32_t interleaved;  /* 1: neighbouring elements are pairs */
  int32_t inverse;      /* 1: turned backwards (the gradient) */
  float magnitude;
  const double* inv_freq; /* device [rotary_dim / 2] */
  /* Position of token (b, s): positions[b * position_stride_b + s *
   * position_stride_s], device integers of position_bytes (4 or 8) bytes.  NULL
   * with position_bytes 0: s, or lengths[b] + s in flexatt_rotary_append. */
  const void* positions;
  int64_t position_stride_b, position_stride_s;
  int32_t position_bytes;
  int32_t reserved;     /* 0 */
} flexatt_rotary;

/* q_out = turned q [B, Hq, S, D] and k_out = turned k [B, Hkv, S, D] (both NULL
 * when heads_kv is 0).  An output may be its own input. */
int flexatt_rotary_apply(const flexatt_rotary* r, const flexatt_tensor* q, const flexatt_tensor* k,
                         const flexatt_tensor* q_out, const flexatt_tensor* k_out, void* stream);

/* q_out = turned q, and the rows lengths[b] .. lengths[b] + S - 1 of the cache
 * receive turned k and v [B, Hkv, S, D] (q and q_out NULL when heads_q is 0).  A row
 * outside [0, cache_rows) is not written.  `lengths` is not changed.  q, q_out, k, v
 * and lengths may not lie within the span of the cache; k_cache and v_cache may share a
 * buffer side by side (the same strides), not memory. */
int flexatt_rotary_append(const flexatt_rotary* r, const flexatt_tensor* q, const flexatt_tensor* k,
                          const flexatt_tensor* v, const flexatt_tensor* q_out, const flexatt_tensor* k_cache,
                          const flexatt_tensor* v_cache, int32_t cache_rows, const int32_t* lengths, void* stream);

/* Attention of `tokens` (T) drafted tokens per sequence over the cache.  The keys
 * of drafted token t of sequence b with n = lengths[b]: the cached rows j < n (with
 * a window, n + depths[b][t] - j <= W), and the rows n + u, u < T, that hold the
 * drafted tokens themselves, where tree_mask[b][t][u] is not 0 (no mask: u <= t).
 * Scores, soft-cap, softmax and LSE as flexatt_fwd; a row without keys is 0 with
 * LSE -inf.  A sequence with n < 0 or n + T > cache_rows gets NaN (o and lse).
 * Rows of the cache from n + T on are not read.  Values of rows that a token does not see
 * have weight 0 in its sum, so they must be finite.  Rows of k_cache and v_cache lie less
 * than 2^26 bytes apart (else FLEXATT_ERANGE). */
typedef struct flexatt_tree {
  int32_t dtype;
  int32_t batch;
  int32_t heads_q;
  int32_t heads_kv;
  int32_t tokens;         /* T >= 1; (Hq / Hkv) T at most 2^20 and B Hq T at most 2^23 (else FLEXATT_ERANGE) */
  int32_t cache_rows;     /* >= 1 */
  int32_t head_dim;
  float scale;
  float soft_cap;         /* 0: off */
  int32_t sliding_window; /* W > 0; 0: off */
  int32_t mask_batch;     /* tree_mask: 1 (one tree for all sequences) or batch; 0 with NULL */
  int32_t reserved;       /* 0 */
  const uint8_t* tree_mask; /* device [mask_batch][T][T], or NULL */
  /* device int32 [B][T], depth of each token in its tree (0: directly behind the
   * cached ones; less counts as 0); read with a window only.  NULL: t, which a
   * window takes with a NULL tree_mask only. */
  const int32_t* depths;
  const int32_t* lengths;   /* device int32 [B] */
} flexatt_tree;

/* o [B, Hq, T, D] and lse fp32 [B, Hq, T].  `workspace`:
 * flexatt_tree_fwd_workspace(p) bytes, 16-byte aligned, not zeroed, reusable once
 * the call's work on `stream` is done; NULL when that is 0 (SIZE_MAX: p is
 * rejected). */
size_t flexatt_tree_fwd_workspace(const flexatt_tree* p);
int flexatt_tree_fwd(const flexatt_tree* p, const flexatt_tensor* q, const flexatt_tensor* k_cache,
                     const flexatt_tensor* v_cache, const flexatt_tensor* o, float* lse, void* workspace,
                     size_t workspace_bytes, void* stream);

/* The attention weight each key has received: sums[b][hk][j] = sum over the G
 * query heads of KV head hk and the query rows i of exp(x_ij - lse_i), with the
 * scores of flexatt_fwd; a masked pair and a row with lse -inf give 0.  Query row i
 * of sequence b is at position start + i, start = query_starts[b] (NULL:
 * query_start); causal keeps j <= start + i, a window start + i - j <= W.  Keys
 * from lengths[b] on (NULL: seqlen_kv; values outside [0, seqlen_kv] count as the
 * nearer end) get 0, with `accumulate` nothing.  FLEXATT_ERANGE: more blocks of 256 keys
 * (of 128 with rows of 1 KB), B Hkv of each, than a launch has workgroups, 2^24 - 1. */
typedef struct flexatt_weights {
  int32_t dtype;
  int32_t batch;
  int32_t heads_q;
  int32_t heads_kv;
  int32_t seqlen_q;
  int32_t seqlen_kv;
  int32_t head_dim;
  float scale;
  float soft_cap;         /* 0: off */
  int32_t causal;
  int32_t sliding_window; /* 0: off */
  int32_t query_start;
  int32_t accumulate;     /* 1: added to sums */
  int32_t reserved;       /* 0 */
  const int32_t* query_starts; /* device int32 [B], or NULL */
  const int32_t* lengths;      /* device int32 [B], or NULL */
} flexatt_weights;

/* sums: contiguous fp32 [B, Hkv, seqlen_kv], not within the span of an input.
 * `workspace` as in flexatt_tree_fwd. */
size_t flexatt_weight_sums_workspace(const flexatt_weights* p);
int flexatt_weight_sums(const flexatt_weights* p, const flexatt_tensor* q, const flexatt_tensor* k, const float* lse,
                        float* sums, void* workspace, size_t workspace_bytes, void* stream);

/* Eviction.  Of the n = lengths[b] rows (clamped to [0, cache_rows]) of each KV
 * head, n > keep, the first `sinks`, the last `recent` and the keep - sinks -
 * recent others with the largest scores stay (of equal ones the lowest rows; NaN is
 * the largest score), in row order; n <= keep: all stay.  They are copied to the
 * first rows of k_out and v_out, their scores to scores_out, their rows' numbers
 * to slots (-1 behind), and min(n, keep) to lengths_out.  Rows of k_out and v_out
 * behind them are left as they were, or with `fill` zeroed up to row keep - 1;
 * scores_out is 0 behind them.  FLEXATT_ERANGE: B Hkv of 2^24 or more. */
typedef struct flexatt_evict {
  int32_t dtype;
  int32_t batch;
  int32_t heads_kv;
  int32_t cache_rows;
  int32_t head_dim;
  int32_t keep;      /* >= 1 */
  int32_t recent;    /* >= 0 */
  int32_t sinks;     /* >= 0; recent + sinks <= keep */
  int32_t out_rows;  /* rows of k_out, v_out and scores_out, >= keep */
  int32_t fill;
  const int32_t* lengths; /* device int32 [B] */
} flexatt_evict;

/* scores: contiguous fp32 [B, Hkv, cache_rows]; scores_out [B, Hkv, out_rows];
 * slots int32 [B, Hkv, keep]; lengths_out int32 [B].  No output may
 * lie within the span of an input or of another output; k_out and v_out may share a
 * buffer side by side (the same strides), not memory. */
int flexatt_evict_rows(const flexatt_evict* p, const flexatt_tensor* k_cache, const flexatt_tensor* v_cache,
                       const float* scores, const flexatt_tensor* k_out, const flexatt_tensor* v_out,
                       float* scores_out, int32_t* slots, int32_t* lengths_out, void* stream);

/* Queries and keys normalised for each head, then turned: y = R (x w / sqrt(mean x^2 +
 * eps)), the mean over the head's D elements in 32 bits (of a row whose mean passes them,
 * scaled by a power of two), R the rotation of flexatt_rotary (inverse 0).  Rounded once. */
typedef struct flexatt_norm {
  int32_t weight_dtype; /* FLEXATT_F32, or the call's dtype */
  float eps;            /* a normal number above 0 */
  const void* q_weight; /* device [D]; NULL when heads_q is 0 */
  const void* k_weight; /* device [D]; NULL when heads_kv is 0 */
} flexatt_norm;

/* As flexatt_rotary_apply (FLEXATT_ERANGE: also more than 2^30 heads).  An output may be its
 * own input. */
int flexatt_norm_rotary_apply(const flexatt_rotary* r, const flexatt_norm* n, const flexatt_tensor* q,
                              const flexatt_tensor* k, const flexatt_tensor* q_out, const flexatt_tensor* k_out,
                              void* stream);

/* Its gradients (FLEXATT_ERANGE alike): dq, dk and the weights' (device [D] of weight_dtype,
 * sums over all rows in 32 bits) from q, k and the gradients of q_out and k_out.  k, k_grad,
 * dk and dk_weight are NULL when heads_kv is 0.  `workspace` as in flexatt_tree_fwd.  No
 * output, nor the workspace, may lie within an input or another of them. */
size_t flexatt_norm_rotary_grad_workspace(const flexatt_rotary* r);
int flexatt_norm_rotary_grad(const flexatt_rotary* r, const flexatt_norm* n, const flexatt_tensor* q,
                             const flexatt_tensor* k, const flexatt_tensor* q_grad, const flexatt_tensor* k_grad,
                             const flexatt_tensor* dq, const flexatt_tensor* dk, void* dq_weight, void* dk_weight,
                             void* workspace, size_t workspace_bytes, void* stream);

/* As flexatt_rotary_append; weights, inv_freq and positions may not lie within the span of
 * the cache either. */
int flexatt_norm_rotary_append(const flexatt_rotary* r, const flexatt_norm* n, const flexatt_tensor* q,
                               const flexatt_tensor* k, const flexatt_tensor* v, const flexatt_tensor* q_out,
                               const flexatt_tensor* k_cache, const flexatt_tensor* v_cache, int32_t cache_rows,
                               const int32_t* lengths, void* stream);

/* Caches of 8 bits.  A row (one position of one head) is D codes and one fp32 scale s =
 * max(amax, 2^-100) / top, of its values' largest size amax and the largest code top:
 * codes are y / s to the nearest, of two the even one, and stand for code * s.  y, amax and
 * y / s are in 64 bits (for e4m3 the quotient is rounded to 32 on its way).  A row with an
 * infinity, NaN or a value beyond 32 bits has codes 0 and scale NaN.
 * Code tensors are [B, Hkv, cache_rows, D] views of bytes (strides in bytes, multiples of
 * 16), scales contiguous fp32 [B, Hkv, cache_rows]. */
enum flexatt_code {
  FLEXATT_E4M3 = 1, /* fp8, 4 bits of exponent, 3 of mantissa, no infinity; top 448 */
  FLEXATT_INT8 = 2  /* top 127 */
};

/* flexatt_rotary_append, or with a norm (n, may be NULL) flexatt_norm_rotary_append, into
 * such a cache; q_out is of the call's dtype.  The cache and its scales lie apart from
 * each other (k_cache and v_cache may share a buffer side by side) and from the rest. */
int flexatt_quant_append(const flexatt_rotary* r, const flexatt_norm* n, int32_t code, const flexatt_tensor* q,
                         const flexatt_tensor* k, const flexatt_tensor* v, const flexatt_tensor* q_out,
                         const flexatt_tensor* k_cache, const flexatt_tensor* v_cache, float* k_scales,
                         float* v_scales, int32_t cache_rows, const int32_t* lengths, void* stream);

/* The values of the first lengths[b] rows (clamped to [0, cache_rows]) of such a cache,
 * rounded to dtype, into k_out and v_out [B, Hkv, cache_rows, D]; the rows behind them are
 * left as they were, or with `fill` zeroed.  FLEXATT_ERANGE: more than a launch has
 * work-items. */
typedef struct flexatt_dequant {
  int32_t dtype;
  int32_t code;       /* enum flexatt_code */
  int32_t batch;
  int32_t heads_kv;
  int32_t cache_rows;
  int32_t head_dim;
  int32_t fill;
  int32_t reserved;   /* 0 */
  const int32_t* lengths; /* device int32 [B] */
} flexatt_dequant;
int flexatt_dequant_rows(const flexatt_dequant* p, const flexatt_tensor* k_cache, const flexatt_tensor* v_cache,
                         const float* k_scales, const float* v_scales, const flexatt_tensor* k_out,
                         const flexatt_tensor* v_out, void* stream);

/* flexatt_tree_fwd over such a cache, for dtype fp16 and bf16 (else FLEXATT_EDTYPE), a
 * tree_mask for up to 2^15 tokens, and no more workgroups than a launch can have (else
 * FLEXATT_ERANGE).  The scores are q . code times the key's scale; weights times the values'
 * scales, relative to the largest of these that the row sees, are rounded to fp16 for the
 * second product (for fp16, to two numbers of it). */
size_t flexatt_quant_tree_fwd_workspace(const flexatt_tree* p);
int flexatt_quant_tree_fwd(const flexatt_tree* p, int32_t code, const flexatt_tensor* q, const flexatt_tensor* k_cache,
                           const flexatt_tensor* v_cache, const float* k_scales, const float* v_scales,
                           const flexatt_tensor* o, float* lse, void* workspace, size_t workspace_bytes, void* stream);

/* flexatt_tree_fwd behind a prefix of `prefix_rows` rows (>= 1; with cache_rows at most
 * 2^30, else FLEXATT_ESHAPE; FLEXATT_ERANGE: also more workgroups than a launch can have)
 * that all sequences share: the keys of a token are the prefix's, then those flexatt_tree_fwd
 * gives it.  A cached row j of sequence b is at position prefix_rows + j, a row of the prefix
 * at its own: a window leaves the rows of the prefix with prefix_rows + n + depths[b][t] - j
 * <= W.  prefix_k and prefix_v are [Hkv, prefix_rows, D] views (stride_b is not used), of rows
 * as those of the cache. */
size_t flexatt_prefix_fwd_workspace(const flexatt_tree* p, int32_t prefix_rows);
int flexatt_prefix_fwd(const flexatt_tree* p, int32_t prefix_rows, const flexatt_tensor* q,
                       const flexatt_tensor* prefix_k, const flexatt_tensor* prefix_v, const flexatt_tensor* k_cache,
                       const flexatt_tensor* v_cache, const flexatt_tensor* o, float* lse, void* workspace,
                       size_t workspace_bytes, void* stream);

/* Human-readable text for a status code (static storage). */
const char* flexatt_status_string(int status);

/* ABI version of this header (bumped on any signature change). */
int flexatt_abi_version(void);

#define FLEXATT_ABI_VERSION 10

#ifdef __cplusplus
}
#endif

#endif /* FLEXATT_H_ */
