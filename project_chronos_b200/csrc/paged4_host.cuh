// paged4_host.cuh — argument checks that the calls of include/chronos_paged4.h share.
#pragma once

#include <iterator>

#include "chronos_paged4.h"
#include "fp4.cuh"
#include "paged_host.cuh"

namespace chronos {

constexpr int kPaged4MaxRep = 256;   // query heads per kv head

inline int check_heads(int heads, const ChronosPagedCache& c, const char* what) {
    if (heads < 1 || heads % c.kv_heads || heads / c.kv_heads > kPaged4MaxRep)
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: heads %d must be 1..%d times kv_heads %d", what, heads, kPaged4MaxRep, c.kv_heads);
    return CHRONOS_OK;
}
inline int check_positive(const char* name, float x, const char* what) {
    if (!(x > 0.0f) || !std::isfinite(x)) return fail(CHRONOS_ERR_INVALID_ARG, "%s: %s %g must be positive", what, name, x);
    return CHRONOS_OK;
}
inline int check_tokens(int64_t tokens, const int32_t* cu, const ChronosPagedCache& c, const char* what) {
    if (tokens < 0 || tokens * c.kv_heads > INT32_MAX / 16)
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: num_tokens %lld", what, static_cast<long long>(tokens));
    if (cu == nullptr && tokens != c.batch)
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: %lld rows for %d sequences without cu_seqlens", what, static_cast<long long>(tokens), c.batch);
    return CHRONOS_OK;
}
// The factor of a cache: values are multiplied by its reciprocal in fp32, which has to be as exact as
// any (neither infinite nor with fewer bits).
inline int check_factor(const char* name, float x, const char* what) {
    if (!(x >= 0x1p-126f && x <= 0x1p126f))
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: %s %g must lie between 2^-126 and 2^126", what, name, x);
    return CHRONOS_OK;
}
// The factor of the scores over 4-bit pages, held in fp32 as well.
inline int check_scores(float scale, float k_scale, const char* what) {
    const double x = static_cast<double>(scale) * k_scale;
    if (!(x >= 0x1p-126 && x <= 0x1p126))
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: scale %g * k_scale %g must lie between 2^-126 and 2^126", what, scale, k_scale);
    return CHRONOS_OK;
}
// Rows of heads, strides in bytes.
struct RowsOf {
    const void* at;
    int64_t rows, row, heads, head, bytes;
};
inline RowsOf rows_of(const void* at, int dtype, int64_t rows, int64_t row, int64_t heads, int64_t head, int64_t dim) {
    const int64_t es = static_cast<int64_t>(elem_bytes(dtype));
    return RowsOf{at, at == nullptr ? 0 : rows, row * es, heads, head * es, dim * es};
}
// Whether the two may share a byte.  Rows side by side in one array (parts of a projection,
// heads in turn) do not.
inline bool rows_meet(const RowsOf& a, const RowsOf& b) {
    if (a.rows <= 0 || b.rows <= 0 || a.heads <= 0 || b.heads <= 0) return false;
    const int64_t ea = (a.heads - 1) * a.head + a.bytes, eb = (b.heads - 1) * b.head + b.bytes;
    const int64_t at_a = static_cast<int64_t>(reinterpret_cast<uintptr_t>(a.at)), at_b = static_cast<int64_t>(reinterpret_cast<uintptr_t>(b.at));
    if (at_a + (a.rows - 1) * a.row + ea <= at_b || at_b + (b.rows - 1) * b.row + eb <= at_a) return false;
    const auto apart = [&](int64_t step, int64_t na, int64_t nb) {   // all of a lies in [0, na) modulo step, b in [d, d + nb)
        const int64_t d = ((at_b - at_a) % step + step) % step;
        return d >= na && d + nb <= step;
    };
    if (a.row == b.row && a.row > 0 && apart(a.row, ea, eb)) return false;
    return !(a.row == b.row && a.head == b.head && a.head > 0 && a.row % a.head == 0 && apart(a.head, a.bytes, b.bytes));
}
// Whether the two are the same rows.
inline bool rows_same(const RowsOf& a, const RowsOf& b) {
    return a.at == b.at && (a.row == b.row || a.rows <= 1) && (a.head == b.head || a.heads <= 1);
}
// n numbers of `size` bytes, one after the other.
inline RowsOf array_of(const void* at, int64_t n, int64_t size) { return RowsOf{at, at == nullptr ? 0 : 1, 0, 1, 0, n * size}; }
// The pages of K or V, each as one stretch.
inline RowsOf pages_of(const ChronosPagedCache& c, bool packed, const void* at, int64_t page, int64_t slot, int64_t head) {
    const int64_t es = packed ? 1 : static_cast<int64_t>(elem_bytes(c.dtype));
    const int64_t bytes = packed ? static_cast<int64_t>(c.page_size) / 16 * fp4_record(fp4_columns(c.head_dim)) : c.head_dim * es;
    const int64_t slots = packed ? 0 : (c.page_size - 1) * slot;
    return RowsOf{at, at == nullptr ? 0 : c.num_pages, page * es, 1, 0, (slots + (c.kv_heads - 1) * head) * es + bytes};
}
// A call's results overlap nothing that it reads (`inputs`, the cache) and not each other.
inline int check_apart(const char* what, const ChronosPagedCache& c, bool packed, std::initializer_list<RowsOf> results,
                       std::initializer_list<RowsOf> inputs) {
    const RowsOf cache[] = {pages_of(c, packed, c.k_pages, c.k_page_stride, c.k_slot_stride, c.k_head_stride),
                            pages_of(c, packed, c.v_pages, c.v_page_stride, c.v_slot_stride, c.v_head_stride),
                            RowsOf{c.page_table, c.page_table == nullptr ? 0 : c.batch, c.page_table_stride * 4, 1, 0, c.table_width * int64_t{4}},
                            array_of(c.lens, c.batch, 4)};
    for (const RowsOf* r = results.begin(); r != results.end(); ++r) {
        const auto meets = [&](const RowsOf& x) { return rows_meet(*r, x); };
        if (std::any_of(std::begin(cache), std::end(cache), meets) || std::any_of(inputs.begin(), inputs.end(), meets) ||
            std::any_of(r + 1, results.end(), meets))
            return fail(CHRONOS_ERR_INVALID_ARG, "%s: results overlap each other, the cache or other inputs", what);
    }
    return CHRONOS_OK;
}
// The results of an attention call: `out` may be `q`.
inline int check_results(const char* what, const ChronosPagedCache& c, bool packed, int64_t rows, int heads, const void* q, int64_t q_row,
                         int64_t q_head, const void* out, int64_t out_row, int64_t out_head, const float* lse, const RowsOf& list, const RowsOf& cu) {
    const RowsOf in = rows_of(q, c.dtype, rows, q_row, heads, q_head, c.head_dim), to = rows_of(out, c.dtype, rows, out_row, heads, out_head, c.head_dim),
                 sums = array_of(lse, rows * heads, 4);
    if (rows_same(to, in) ? rows_meet(sums, in) : rows_meet(to, in) || rows_meet(sums, in))
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: out may be q, with the same strides; results overlap no other input", what);
    return check_apart(what, c, packed, {to, sums}, {list, cu});
}

// Pages of 4-bit values.
inline int check_packed(const ChronosPagedCache& c, float k_scale, float v_scale, const char* what) {
    if (c.page_size % 16) return fail(CHRONOS_ERR_INVALID_ARG, "%s: 4-bit pages need a page_size that is a multiple of 16, got %d", what, c.page_size);
    if (!multiples(16, {c.k_page_stride, c.k_head_stride, c.v_page_stride, c.v_head_stride}) || !aligned(c.k_pages, 16) || !aligned(c.v_pages, 16))
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: 4-bit pages and their strides must be multiples of 16 bytes", what);
    if (c.k_page_stride < 0 || c.v_page_stride < 0 || c.k_page_stride > UINT32_MAX || c.v_page_stride > UINT32_MAX ||
        static_cast<int64_t>(c.page_size) * 144 > INT32_MAX)
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: 4-bit pages of %d slots, %lld and %lld bytes apart", what, c.page_size,
                    static_cast<long long>(c.k_page_stride), static_cast<long long>(c.v_page_stride));
    if (int rc = check_factor("k_scale", k_scale, what)) return rc;
    return check_factor("v_scale", v_scale, what);
}

}  // namespace chronos
