/*
 * chronos_paged4.h — C ABI of what a server needs around the paged key-value
 * cache of chronos_paged.h: the append that rotates queries and keys on the way,
 * pages of 4-bit values with the attention that reads them, and attention over
 * the pages that a score selects for each query.
 *
 *   chronos_paged_append_rope  new rows into the pages, keys and queries rotated
 *   chronos_paged_gather       rows of the cache, packed one after the other
 *   chronos_paged_decode4      one-token attention over pages of 4-bit values
 *   chronos_paged_bounds       smallest and largest key of every page and column
 *   chronos_paged_select       the pages that each query's bounds rank highest
 *   chronos_paged_sparse       attention over the slots of selected pages
 *
 * Conventions as in chronos_paged.h.  Results may not overlap each other, the cache or
 * another input, but where a call names it: such calls are refused.
 *
 * Packed pages (4-bit values).  With P = head_dim rounded up to 64, 128 or 256 a
 * page of a kv head is page_size / 16 records of 9 P bytes (page_size is a multiple of
 * 16), one after the other.  A record holds 16 slots: first their codes, P / 2 bytes a
 * slot (byte i: column 2i in the low half, 2i + 1 in the high one), then their
 * scales, P / 16 bytes a slot (one for 16 columns).  A code is e2m1 (sign and one of 0,
 * 0.5, 1, 1.5, 2, 3, 4, 6), a scale e4m3 without sign, and
 *     value = code * scale * k_scale (v_scale; both between 2^-126 and 2^126).
 * Of 16 columns x_i, y_i = x_i / k_scale, the append stores
 *     scale = e4m3(min(fp32(max |y_i| / 6), 448)),  code_i = e2m1(y_i / scale)
 * to the nearest, ties to the even code, as exact arithmetic on the inputs and the
 * tables decides; magnitudes beyond 6 scale take 6.  A scale of zero has codes of
 * zero.  Where one of the 16 is NaN or infinite the scale is NaN (and the 16 values
 * with it).  Columns behind head_dim are zeros.
 * In the cache structs of packed calls `dtype` is the type of the rows outside the
 * pages, k_page_stride and k_head_stride count bytes, multiples of 16, and
 * k_slot_stride is not used; likewise for v.  The pages start on 16 bytes.
 */
#ifndef CHRONOS_PAGED4_H_
#define CHRONOS_PAGED4_H_

#include "chronos_paged.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Token t of sequence b, its i-th (tokens as in chronos_paged_append), stands at
 * position seen[b] + i.  Of a key or query row x, with c = cos[position], s =
 * sin[position], r = rope_dim, columns counted from rope_start and j < r / 2:
 *     y_j = x_j c_j - x_{j + r/2} s_j,   y_{j + r/2} = x_{j + r/2} c_{j + r/2} + x_j s_{j + r/2}
 * the other columns as they are.  k goes to the pages (and k_out) so, v as it is, q to
 * q_out.  With rope_dim 0 nothing is rotated.  Weights, positions, lens_out and
 * seen_out as in chronos_paged_append; a token whose position lies outside the
 * tables is dropped like one without a page (and its rows of q_out and k_out are
 * zeros; those of a token that only lacks a page are rotated all the same).  Rows
 * behind the last sequence are not written; they may be read, and what they hold does
 * not matter.  q_out may be q and k_out may be k (with the same strides). */
typedef struct ChronosPagedRopeArgs {
    ChronosPagedCache cache;   /* lens: before the append */
    int32_t packed;            /* 1: pages of 4-bit values */
    int32_t heads;             /* query heads of q, 0 without q */
    int32_t rope_dim;          /* even, rope_start + rope_dim <= head_dim */
    int32_t rope_start;
    int32_t table_len;         /* rows of cos and sin */
    int32_t table_dtype;       /* fp32, or cache.dtype */
    float k_scale, v_scale;    /* packed: 2^-126 to 2^126 */
    int64_t num_tokens;
    const void* k;             /* [num_tokens, G, D] */
    const void* v;
    const void* q;             /* [num_tokens, heads, D] or NULL */
    void* q_out;
    void* k_out;               /* [num_tokens, G, D] or NULL */
    int64_t k_row_stride, k_head_stride, v_row_stride, v_head_stride, q_row_stride, q_head_stride;
    int64_t q_out_row_stride, q_out_head_stride, k_out_row_stride, k_out_head_stride;
    const void* cos;           /* [table_len, rope_dim] */
    const void* sin;
    int64_t cos_row_stride, sin_row_stride;
    const int32_t* cu_seqlens; /* [B + 1] or NULL */
    const int32_t* seen;       /* [B]; NULL only without rotation and positions */
    float* weights;
    int32_t* positions;
    int64_t slot_cap;
    int32_t* lens_out;
    int32_t* seen_out;
    int32_t* status;
} ChronosPagedRopeArgs;

/* Row cu_seqlens[b] + i of k_out and v_out = slot first[b] + i of sequence b (without
 * `first`: its newest slots, those that end at lens[b]).  A slot outside [0, lens[b])
 * or without a page gives zeros and is reported.  Rows behind the last sequence are
 * left as they are. */
typedef struct ChronosPagedGatherArgs {
    ChronosPagedCache cache;
    int32_t packed;
    int32_t reserved;
    float k_scale, v_scale;
    int64_t num_tokens;        /* rows of k_out and v_out */
    void* k_out;               /* [num_tokens, G, D] */
    void* v_out;
    int64_t k_row_stride, k_head_stride, v_row_stride, v_head_stride;
    const int32_t* cu_seqlens; /* [B + 1] */
    const int32_t* first;      /* [B] or NULL */
    int32_t* status;
} ChronosPagedGatherArgs;

/* chronos_paged_decode over packed pages, without running sums.  out may be q (with the
 * same strides). */
typedef struct ChronosPagedDecode4Args {
    ChronosPagedCache cache;
    int32_t heads;
    int32_t window;
    int32_t sinks;
    float scale;               /* > 0; scale * k_scale 2^-126 to 2^126 */
    float k_scale, v_scale;    /* 2^-126 to 2^126 */
    const void* q;             /* [B, H, D] */
    int64_t q_row_stride, q_head_stride;
    void* out;                 /* [B, H, D] */
    int64_t out_row_stride, out_head_stride;
    float* lse;                /* [B, H] or NULL */
    void* workspace;           /* chronos_paged_decode4_workspace bytes, 256-byte aligned; NULL for 0 */
    size_t workspace_bytes;
    int32_t* status;
} ChronosPagedDecode4Args;

/* bounds[page, 0, g, d] and [page, 1, g, d] = smallest and largest key of column d over the
 * page's slots in use (of 4-bit pages, whose values may have more bits than the layer
 * type, the smallest rounded down and the largest up); NaN where one of them is.  Brought
 * up to date: the pages of the newest tokens (one per sequence, or cu_seqlens[b + 1] -
 * cu_seqlens[b]), whose older slots are in the bounds already; with `full` every page of
 * every sequence, from its slots alone. */
typedef struct ChronosPagedBoundsArgs {
    ChronosPagedCache cache;   /* lens: the newest tokens included; v is not used */
    int32_t packed;
    int32_t full;
    float k_scale;
    int32_t reserved;
    int64_t num_tokens;        /* new tokens of all sequences, with cu_seqlens */
    const int32_t* cu_seqlens; /* [B + 1] or NULL */
    void* bounds;              /* [num_pages, 2, G, D], contiguous, of cache.dtype */
    int32_t* status;
} ChronosPagedBoundsArgs;

/* Token t is one of its sequence's newest (cu_seqlens as above, without it one per
 * sequence): n = lens[b] - (cu_seqlens[b + 1] - 1 - t) slots are at or before it, in
 * m = ceil(n / page_size) pages.  For each kv head, pages[t, g, :] = ascending, the pages
 * j < first and j >= m - last, and of the others those with the highest
 *     score_j = sum over the group's heads h and d of max(q_hd bounds[j,0,g,d], q_hd bounds[j,1,g,d])
 * (0 times infinity and a maximum with NaN are NaN; NaN above every number, equal ones
 * by the lower page), min(topk, m) in all, -1 behind.  Scores are sums in 64 bits.  The rows of tokens behind the last sequence are
 * left as they are.  A page number that is none ranks last, a lens[b] beyond the table is
 * cut to it; both are reported. */
typedef struct ChronosPagedSelectArgs {
    ChronosPagedCache cache;   /* k_pages and v_pages are not used */
    int32_t heads;
    int32_t topk;              /* >= first + last */
    int32_t first;             /* >= 0 */
    int32_t last;              /* >= 1: a token's own page is always in */
    int64_t num_tokens;
    const void* q;             /* [num_tokens, H, D] */
    int64_t q_row_stride, q_head_stride;
    const void* bounds;        /* [num_pages, 2, G, D], contiguous */
    const int32_t* cu_seqlens;
    int32_t* pages;            /* [num_tokens, G, topk] */
    void* workspace;           /* chronos_paged_select_workspace bytes, 256-byte aligned */
    size_t workspace_bytes;
    int32_t* status;
} ChronosPagedSelectArgs;

/* Attention of token t (n slots at or before it, as above) over the slots j < n of the
 * pages pages[t, g, :]; entries below 0 or at or beyond m are passed over, a page that is
 * named twice counts twice.  Nothing visible: zeros and lse = -inf.  Rows of tokens behind
 * the last sequence are left as they are.  out may be q (with the same strides). */
typedef struct ChronosPagedSparseArgs {
    ChronosPagedCache cache;
    int32_t packed;
    int32_t heads;
    int32_t topk;              /* entries of pages per token and kv head */
    float scale;
    float k_scale, v_scale;    /* packed: as in chronos_paged_decode4 */
    int64_t num_tokens;
    const void* q;             /* [num_tokens, H, D] */
    int64_t q_row_stride, q_head_stride;
    void* out;
    int64_t out_row_stride, out_head_stride;
    float* lse;                /* [num_tokens, H] or NULL */
    const int32_t* pages;      /* [num_tokens, G, topk] */
    const int32_t* cu_seqlens;
    int32_t* status;
} ChronosPagedSparseArgs;

CHRONOS_API int chronos_paged_append_rope(const ChronosPagedRopeArgs* args, void* cuda_stream);
CHRONOS_API int chronos_paged_gather(const ChronosPagedGatherArgs* args, void* cuda_stream);
CHRONOS_API int chronos_paged_decode4(const ChronosPagedDecode4Args* args, void* cuda_stream);
CHRONOS_API int chronos_paged_bounds(const ChronosPagedBoundsArgs* args, void* cuda_stream);
CHRONOS_API int chronos_paged_select(const ChronosPagedSelectArgs* args, void* cuda_stream);
CHRONOS_API int chronos_paged_sparse(const ChronosPagedSparseArgs* args, void* cuda_stream);

/* Workspace bytes, from the shapes; 0 where a call needs none, and, with
 * chronos_moe_last_error set, for an invalid shape. */
CHRONOS_API size_t chronos_paged_decode4_workspace(const ChronosPagedDecode4Args* args);
CHRONOS_API size_t chronos_paged_select_workspace(const ChronosPagedSelectArgs* args);

CHRONOS_API size_t chronos_paged_rope_args_size(void);
CHRONOS_API size_t chronos_paged_gather_args_size(void);
CHRONOS_API size_t chronos_paged_decode4_args_size(void);
CHRONOS_API size_t chronos_paged_bounds_args_size(void);
CHRONOS_API size_t chronos_paged_select_args_size(void);
CHRONOS_API size_t chronos_paged_sparse_args_size(void);

#ifdef __cplusplus
}
#endif

#endif /* CHRONOS_PAGED4_H_ */
