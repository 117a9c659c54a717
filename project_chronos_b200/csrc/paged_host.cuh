// paged_host.cuh — argument checks and sizes that the C ABI's calls on the paged cache share.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <initializer_list>

#include "chronos_paged.h"
#include "host.cuh"

namespace chronos {

inline size_t elem_bytes(int dtype) { return dtype == CHRONOS_DTYPE_FP32 ? 4 : 2; }
inline bool dtype_known(int d) { return d == CHRONOS_DTYPE_BF16 || d == CHRONOS_DTYPE_FP16 || d == CHRONOS_DTYPE_FP32; }
inline size_t round_up(size_t v, size_t a) { return (v + a - 1) / a * a; }
inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
inline bool multiples(int64_t of, std::initializer_list<int64_t> v) {
    return std::all_of(v.begin(), v.end(), [of](int64_t x) { return x % of == 0; });
}

inline int check_cache(const ChronosPagedCache& c, const char* what) {
    if (c.batch < 0 || c.kv_heads < 1 || c.head_dim < 1 || c.head_dim > CHRONOS_PAGED_MAX_HEAD_DIM ||
        !dtype_known(c.dtype))
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: batch %d, kv_heads %d, head_dim %d (1..%d), dtype %d", what, c.batch,
                    c.kv_heads, c.head_dim, CHRONOS_PAGED_MAX_HEAD_DIM, c.dtype);
    if (c.num_pages < 0 || c.page_size < 1 || c.table_width < 0)
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: num_pages %d, page_size %d (>= 1), table_width %d", what, c.num_pages,
                    c.page_size, c.table_width);
    if (static_cast<int64_t>(c.batch) * c.kv_heads > (1 << 20))
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: batch %d * kv_heads %d too large", what, c.batch, c.kv_heads);
    return CHRONOS_OK;
}
inline int check_cache_pointers(const ChronosPagedCache& c, const char* what) {
    if (c.batch > 0 && (c.lens == nullptr || (c.table_width > 0 && c.page_table == nullptr) ||
                        (c.num_pages > 0 && (c.k_pages == nullptr || c.v_pages == nullptr))))
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: lens, page_table, k_pages and v_pages are required", what);
    return CHRONOS_OK;
}
// Whether two arrays of n numbers overlap (`same`: other than as one).
template <typename T>
inline bool cross(const T* a, const T* b, int64_t n, bool same) {
    return a != nullptr && b != nullptr && a < b + n && b < a + n && !(same && a == b);
}
// Numbers of a per-slot array.
inline int64_t slots_of(const ChronosPagedCache& c, int64_t slot_cap) { return static_cast<int64_t>(c.batch) * c.kv_heads * slot_cap; }
// A window (or number of first tokens) as the kernels take it: rows have at most 2^30
// keys, so a longer one hides nothing, and positions minus it stay within 32 bits.
inline int cut_window(int window) { return std::min(window, 1 << 30); }
// Slots a sequence can have: what its table (and the per-slot arrays, when there are any) hold.
inline int slot_limit(const ChronosPagedCache& c, int64_t slot_cap, bool has_cap) {
    int64_t n = static_cast<int64_t>(c.table_width) * c.page_size;
    if (has_cap) n = std::min(n, slot_cap);
    return static_cast<int>(std::min<int64_t>(n, (1 << 30)));
}

// Bytes of the widest unit that every row can be copied in: 16, or one element.
inline bool copies16(const ChronosPagedCache& c) {
    const int64_t n = 16 / static_cast<int64_t>(elem_bytes(c.dtype));
    return c.head_dim % n == 0 && aligned(c.k_pages, 16) && aligned(c.v_pages, 16) &&
           multiples(n, {c.k_page_stride, c.k_slot_stride, c.k_head_stride, c.v_page_stride, c.v_slot_stride, c.v_head_stride});
}
// log2 of the page size, -1 where it is no power of two.
inline int page_shift_of(const ChronosPagedCache& c) {
    if ((c.page_size & (c.page_size - 1)) != 0) return -1;
    int s = 0;
    while ((1 << s) < c.page_size) ++s;
    return s;
}

}  // namespace chronos
