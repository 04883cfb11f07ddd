#ifndef YB_LM_H
#define YB_LM_H

/* Text-decoder operators on device buffers, for programs that run a decoder
 * beside the detector (captions of detections, questions about an image): the
 * norm and rotation of queries and keys with the write into the cache,
 * attention over that cache, and token sampling.  No counterpart in the
 * reference (phucb2/yolo-baremetal has no text model); they stand beside the
 * PSA attention (layers.c:310-405) and the Detect top-k (detect.c:63-166).
 *
 * All tensors live in the memory of one device.  The calls enqueue on `stream`
 * (a cudaStream_t; NULL = the default stream) and do not synchronize; they can
 * be captured into a CUDA graph once one call has run on the device before
 * (which loads the kernels).  Strides are in elements and non-negative, given
 * as [batch, row, head]; the last dimension is contiguous.  Pointers lie on
 * their elements' boundaries (others are refused).  Lengths and positions are
 * read on the device, so that a captured graph follows them.  No operator has
 * a gradient. */

#include <stddef.h>

#include "status.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef enum { YB_F32 = 0, YB_F16 = 1, YB_BF16 = 2 } yb_dtype;

/* ------------------------------------------------------------- attention
 * For query row i of sequence b and head h, at position
 * pos = k_len[b] - q_len[b] + i (the last row meets the last key):
 *   s_j = scale * q . k_j
 *   s_j = cap * tanh(s_j / cap)               when cap > 0
 *   s_j = s_j - slopes[h] * |pos - j|         when slopes
 *   o   = sum_j softmax(s)_j v_j  over the visible keys j:
 *         0 <= j < k_len[b],
 *         key_range[b][i][0] <= j < key_range[b][i][1]   when key_range
 *           (a document mask: the first key and the end of the row's document),
 *         j <= pos, or j < prefix[b] when prefix         when causal.
 * Key head h / (Hq / Hkv).  A row that sees no key gives zeros, as does one
 * whose visible scores are all -infinity.  Rows i >= q_len[b] of o keep their
 * contents.  Keys that a row does not see do not touch it, whatever they hold
 * (infinities and NaN included; a row that shares a block with such values is
 * computed twice, slowly).  A visible s_j of NaN or +infinity makes the row NaN.
 * Scores, sums and o are formed in fp32.  A capped score is within 16 2^-24 of
 * its value, or within 2^-22 of the cap where that is more than 2^20 times below
 * the scale, or more than 2^20 times above it and the score past 4e-4 of it.  The
 * weights enter the second product rounded to dtype. */
typedef struct {
    const void* q; /* [B, Sq, Hq, D]  */
    const void* k; /* [B, Sk, Hkv, D] */
    const void* v; /* [B, Sk, Hkv, D] */
    void* o;       /* [B, Sq, Hq, D]; must not overlap the inputs */
    const int* q_len;     /* [B] rows in use, clamped to [0, Sq]; NULL: Sq */
    const int* k_len;     /* [B] keys in use, clamped to [0, Sk]; NULL: Sk */
    const int* prefix;    /* [B]; NULL: none.  Only with causal */
    const int* key_range; /* [B, Sq, 2]; NULL: all keys */
    const float* slopes;  /* [Hq]; NULL: none */
    long long q_stride[3], k_stride[3], v_stride[3], o_stride[3];
    int dtype; /* yb_dtype: YB_F16 or YB_BF16 */
    int B, Sq, Sk, Hq, Hkv, D;
    int causal;
    float scale; /* finite, > 0 */
    float cap;   /* finite, >= 0; 0 = no cap */
} yb_attn_args;

/* A handle holds the error word of the kernels' bounded waits; it may be used
 * from any number of streams at once.  Create it outside stream captures, and
 * keep it while a graph that holds its runs is replayed. */
status_t yb_attn_create(int device, void** attn);

/* Scratch bytes that yb_attn_run needs for these sizes (may be 0).  Calls that
 * can overlap in time need scratch of their own. */
status_t yb_attn_workspace(void* attn, const yb_attn_args* a, size_t* bytes);

/* D a multiple of 8 in [8, 128]; Hq a multiple of Hkv.  q, k, v, o 16-byte
 * aligned with strides that are multiples of 8 elements; only the batch
 * strides of q, k and v may be 0 (one tensor for all sequences).  key_range
 * 8-byte aligned.  workspace:
 * 16-byte aligned, at least yb_attn_workspace bytes. */
status_t yb_attn_run(void* attn, const yb_attn_args* a, void* workspace, size_t workspace_bytes, void* stream);

/* Synchronizes the device, reads and clears the error word.  ERROR_DEVICE: a
 * kernel gave up a wait (2 s, and 32 us a key, a minute at most) since the last
 * check, and rows of its output are wrong; nothing else tells. */
status_t yb_attn_check(void* attn);
status_t yb_attn_destroy(void* attn);

/* Test hook of the bounded waits, as yb_conv_debug_withhold: the next
 * yb_attn_run issues no load and bounds its waits to 1 ms; it records the
 * error, frees its tensor memory and ends, so that yb_attn_check reports
 * ERROR_DEVICE and later runs are unaffected. */
status_t yb_attn_debug_withhold(void* attn);

/* --------------------------------------- norm and rotation of queries, keys
 * For each head x [D] of token t (t < length[b]) of sequence b:
 *   y_d = x_d / sqrt(mean(x^2) + eps) * (weight_d + weight_add)
 * then pair i of the first R dimensions is rotated by the angle
 * positions[b][t] * inv_freq[i] (radians; formed and reduced to one turn in 64
 * bits): pairs (i, i + R/2), or (2i, 2i + 1) when interleaved.  fp32 between
 * the load and the store (a sum of squares above its range gives zeros; with
 * eps = 0 one that vanishes gives infinities or NaN).
 * q -> q_out[b][t]; k -> k_out[b][start[b] + t], and v, unchanged, to the same
 * row of v_out: rows of a cache.  Rows outside [0, cache_rows) are not
 * written; nothing else of the outputs is touched.  q_out may be q, and, when
 * start is NULL, k_out may be k and v_out v (with the same strides); other
 * overlaps are not allowed. */
typedef struct {
    const void* q; /* [B, S, Hq, D]  */
    const void* k; /* [B, S, Hkv, D] */
    const void* v; /* [B, S, Hkv, D], or NULL */
    void* q_out;   /* [B, S, Hq, D] */
    void* k_out;   /* [B, cache_rows, Hkv, D] */
    void* v_out;   /* [B, cache_rows, Hkv, D], or NULL */
    const float* q_weight; /* [D]; NULL: ones */
    const float* k_weight; /* [D]; NULL: ones */
    const double* inv_freq; /* [R / 2] */
    const int* start;     /* [B]; NULL: 0 */
    const int* length;    /* [B] tokens in use, clamped to [0, S]; NULL: S */
    const int* positions; /* [B, S]; NULL: start[b] + t */
    long long q_stride[3], k_stride[3], v_stride[3], q_out_stride[3], k_out_stride[3], v_out_stride[3];
    int dtype; /* yb_dtype */
    int B, S, cache_rows, Hq, Hkv, D, R;
    int interleaved;
    float eps;        /* finite, >= 0 */
    float weight_add; /* added to both weights (1 for weights stored around 0) */
} yb_qk_args;

/* D even, in [2, 256]; R even, in [0, D]; Hkv may be 0 (queries alone). */
status_t yb_qk_norm_rope(const yb_qk_args* a, void* stream);

/* --------------------------------------------------------------- sampling
 * For row b, with w_i = exp((logit_i - max) / temperature): tokens in order of
 * falling logit, equal ones by rising index;
 *   top_k > 0: the first top_k of them;
 *   top_p < 1: of these, each whose forerunners hold less than top_p of their
 *              whole weight (the first one always);
 *   min_p > 0: of these, each with w_i >= min_p (above 1 it counts as 1);
 * token[b] is the first of the kept ones, by rising index, whose running sum
 * of weights exceeds u[b] times their whole weight, and logprob[b] the log of
 * its share of that weight (from its logit, in 64 bits).  temperature <= 0 or
 * NaN: the largest logit, with logprob 0.  Logits of -infinity or NaN are never
 * chosen, +infinity counts as the largest finite float; a row without any other
 * logit gives token -1 and logprob -infinity.  u is clamped to [0, 1).  Weights are held as whole
 * numbers of 2^-44, so that sums do not depend on their order; a token below
 * 2^-45 of the largest weight is never chosen. */
typedef struct {
    const void* logits;       /* [B, V] */
    const float* u;           /* [B] */
    const float* temperature; /* [B]; NULL: 1 */
    const int* top_k;         /* [B]; NULL, or <= 0: off */
    const float* top_p;       /* [B]; NULL, or >= 1, or NaN: off */
    const float* min_p;       /* [B]; NULL, or <= 0, or NaN: off */
    int* token;               /* [B] */
    float* logprob;           /* [B], or NULL */
    long long row_stride;
    int dtype; /* yb_dtype */
    int B, V;  /* V <= YB_SAMPLE_MAX_VOCAB */
} yb_sample_args;

#define YB_SAMPLE_MAX_VOCAB 262144

status_t yb_sample(const yb_sample_args* a, void* stream);

#ifdef __cplusplus
}
#endif

#endif
