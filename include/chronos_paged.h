/*
 * chronos_paged.h — C ABI of the paged key-value cache and of the attention
 * that serves a ragged batch from it.
 *
 *   chronos_paged_append      new key/value rows of every sequence into its pages
 *   chronos_paged_decode      attention of one new token per sequence over the
 *                             pages, optionally under a sliding window with first
 *                             tokens that stay visible, optionally adding every
 *                             slot's attention weight to running sums
 *   chronos_paged_evict       the cache cut down to a budget of slots per
 *                             (sequence, kv head): what gathered least attention goes
 *   chronos_window_attention  causal attention of packed prompts (or of the newest
 *                             part of longer ones), optional window and first tokens
 *
 * The one-token kernels of chronos_attention.h serve contiguous caches whose
 * rows all stand at the same position; here every sequence has its own length,
 * its slots lie in pages of `page_size` slots named by `page_table`, and keys
 * are stored rotated, so attention does not depend on the order of the slots.
 *
 * Conventions as in chronos_moe.h: DEVICE pointers, the caller allocates, calls
 * are ordered on the given stream, nothing synchronises the host, no function
 * aborts.  Strides are in elements; the innermost dimension is contiguous.
 * Lengths and page numbers are read on the device.  A length beyond the table
 * (or the running sums) is cut to it, a page number outside [0, num_pages) is
 * never dereferenced (its slots count as hidden, an append to it is dropped);
 * both are reported as CHRONOS_ERR_INVALID_ARG in the status word.
 */
#ifndef CHRONOS_PAGED_H_
#define CHRONOS_PAGED_H_

#include <stddef.h>
#include <stdint.h>

#include "chronos_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

#define CHRONOS_PAGED_MAX_HEAD_DIM 256

/* The pages of one layer and the sequences' page tables. */
typedef struct ChronosPagedCache {
    int32_t batch;             /* B sequences; 0 is allowed */
    int32_t kv_heads;          /* G */
    int32_t head_dim;          /* D, 1..256 */
    int32_t dtype;             /* CHRONOS_DTYPE_* of the pages, q, the new rows and out */
    int32_t num_pages;
    int32_t page_size;         /* slots per page, >= 1 */
    int32_t table_width;       /* pages a sequence may have */
    int32_t reserved;
    void* k_pages;             /* [num_pages, page_size, G, D] by the strides below */
    void* v_pages;
    int64_t k_page_stride, k_slot_stride, k_head_stride;
    int64_t v_page_stride, v_slot_stride, v_head_stride;
    const int32_t* page_table; /* [B, table_width], rows page_table_stride apart */
    int64_t page_table_stride;
    const int32_t* lens;       /* [B] slots in use (decode: the new token included; append:
                                  before the append) */
} ChronosPagedCache;

/* Token t of sequence b (tokens [cu_seqlens[b], cu_seqlens[b+1]) of the packed
 * rows, in order; without cu_seqlens one token per sequence) goes to slot
 * lens[b] + i.  With `weights`, weights[b, g, slot] = 0; with `positions`,
 * positions[b, g, slot] = seen[b] + i.  Rows behind the last sequence are not
 * read.  With `lens_out`, lens_out[b] = lens[b] + the tokens of sequence b stored
 * before its first dropped one, and seen_out[b] = seen[b] + the same number;
 * lens_out may be lens and seen_out may be seen, any other overlap is refused. */
typedef struct ChronosPagedAppendArgs {
    ChronosPagedCache cache;
    int64_t num_tokens;        /* rows of k and v */
    const void* k;             /* [num_tokens, G, D] */
    const void* v;
    int64_t k_row_stride, k_head_stride, v_row_stride, v_head_stride;
    const int32_t* cu_seqlens; /* [B + 1] or NULL (num_tokens == B) */
    const int32_t* seen;       /* [B] tokens seen before (positions), or NULL */
    float* weights;            /* [B, G, slot_cap] or NULL */
    int32_t* positions;        /* [B, G, slot_cap] or NULL */
    int64_t slot_cap;
    int32_t* lens_out;         /* [B] or NULL */
    int32_t* seen_out;         /* [B] or NULL (needs seen) */
    int32_t* status;           /* device status word, or NULL */
} ChronosPagedAppendArgs;

/* One new token per sequence, whose own slot is lens[b] - 1:
 *     visible(j) = j < len and (window == 0 or j >= len - window or j < sinks)
 *     s_j = scale q . k_j,  p_j = exp(s_j - lse) over visible j,  out = sum_j p_j v_j
 * A sequence of length 0 gets zeros and lse = -inf.  With `weights`,
 *     weights_out[b, g, j] = weights[b, g, j] + sum over the group's heads of p_j
 * for every j < len (hidden ones add nothing); slots behind are left as they
 * are; weights_out may be weights, any other overlap of the two is refused.  The workspace of a call with weights then
 * holds 4 bytes per query head and slot that a row can see (by table_width and
 * slot_cap, or window), up to 2^28 bytes or one sequence's: beyond that the call
 * runs over groups of sequences.  The choice of kernel and grid goes by the same
 * sizes: a table far wider than the rows costs a second kernel. */
typedef struct ChronosPagedDecodeArgs {
    ChronosPagedCache cache;
    int32_t heads;             /* H, a multiple of G */
    int32_t window;            /* 0: no window */
    int32_t sinks;             /* first slots that stay visible under a window */
    float scale;               /* > 0 */
    const void* q;             /* [B, H, D] */
    int64_t q_row_stride, q_head_stride;
    void* out;                 /* [B, H, D] */
    int64_t out_row_stride, out_head_stride;
    float* lse;                /* [B, H] or NULL */
    const float* weights;      /* [B, G, slot_cap] or NULL */
    float* weights_out;
    int64_t slot_cap;
    void* workspace;           /* chronos_paged_decode_workspace bytes, 256-byte aligned; NULL for 0 */
    size_t workspace_bytes;
    int32_t* status;
} ChronosPagedDecodeArgs;

/* For every (b, g) with n = lens[b] > budget slots: keep `budget` of them: those
 * at a position < sinks or >= seen[b] - recent, then the largest weights (NaN
 * above every number, -0 = 0, equal ones by the lower slot).  Kept slots below
 * `budget` stay where they are; the i-th kept slot at or beyond it moves into
 * the i-th slot below it that was given up: K and V rows in the pages, weight
 * and position into weights_out / positions_out (which may be the inputs, but not
 * overlap them otherwise).
 *     src[b, g, j] = slot that now sits in slot j (j itself where it stayed),
 *     -1 for j >= min(n, budget);  lens_out[b] = min(n, budget)
 * Slots of weights_out / positions_out from lens_out on are left as they are. */
typedef struct ChronosPagedEvictArgs {
    ChronosPagedCache cache;
    int32_t budget;            /* >= 1 */
    int32_t sinks;             /* >= 0, sinks + recent <= budget */
    int32_t recent;            /* >= 0 */
    int32_t reserved;
    const int32_t* seen;       /* [B] tokens seen so far: positions are below it */
    const float* weights;      /* [B, G, slot_cap] */
    const int32_t* positions;  /* [B, G, slot_cap] */
    float* weights_out;
    int32_t* positions_out;
    int64_t slot_cap;
    int32_t* lens_out;         /* [B]; may be cache.lens or seen */
    int32_t* src;              /* [B, G, budget] */
    void* workspace;           /* chronos_paged_evict_workspace bytes, 256-byte aligned */
    size_t workspace_bytes;
    int32_t* status;
} ChronosPagedEvictArgs;

/* Sequence b has the query rows [cu_q[b], cu_q[b+1]) and the key rows
 * [cu_k[b], cu_k[b+1]); its i-th query stands at position t = lk - lq + i and sees
 *     key j <= t with (window == 0 or j > t - window or j < sinks).
 * A row that sees nothing (t < 0) gets zeros and lse = -inf.  Query rows behind
 * the last sequence are left as they are, key rows behind it are not used.
 * Offsets that do not ascend or leave the rows are reported as
 * CHRONOS_ERR_INVALID_ARG in the status word; what the results are is not said then.
 * out may be q, but not k or v. */
typedef struct ChronosWindowAttnArgs {
    int32_t batch;
    int32_t heads;             /* H, a multiple of kv_heads */
    int32_t kv_heads;
    int32_t head_dim;          /* 1..256 */
    int32_t dtype;
    int32_t window;            /* 0: no window */
    int32_t sinks;
    float scale;               /* > 0 */
    int64_t num_q;             /* rows of q and out */
    int64_t num_k;             /* rows of k and v */
    const void* q;             /* [num_q, H, D] */
    const void* k;             /* [num_k, G, D] */
    const void* v;
    void* out;                 /* [num_q, H, D] */
    int64_t q_row_stride, q_head_stride, k_row_stride, k_head_stride;
    int64_t v_row_stride, v_head_stride, out_row_stride, out_head_stride;
    const int32_t* cu_q;       /* [B + 1], ascending from 0 */
    const int32_t* cu_k;       /* [B + 1] */
    float* lse;                /* [num_q, H] or NULL */
    int32_t* status;
} ChronosWindowAttnArgs;

CHRONOS_API int chronos_paged_append(const ChronosPagedAppendArgs* args, void* cuda_stream);
CHRONOS_API int chronos_paged_decode(const ChronosPagedDecodeArgs* args, void* cuda_stream);
CHRONOS_API int chronos_paged_evict(const ChronosPagedEvictArgs* args, void* cuda_stream);
CHRONOS_API int chronos_window_attention(const ChronosWindowAttnArgs* args, void* cuda_stream);

/* Workspace bytes of a call, from its shapes and the alignment of its buffers (set
 * them as for the call); 0 where it needs none, and, with chronos_moe_last_error
 * set, for an invalid shape. */
CHRONOS_API size_t chronos_paged_decode_workspace(const ChronosPagedDecodeArgs* args);
CHRONOS_API size_t chronos_paged_evict_workspace(const ChronosPagedEvictArgs* args);

CHRONOS_API size_t chronos_paged_append_args_size(void);
CHRONOS_API size_t chronos_paged_decode_args_size(void);
CHRONOS_API size_t chronos_paged_evict_args_size(void);
CHRONOS_API size_t chronos_window_attn_args_size(void);

#ifdef __cplusplus
}
#endif

#endif /* CHRONOS_PAGED_H_ */
