// chronos_paged4.cu — the C ABI of include/chronos_paged4.h but for its attention calls:
// argument checks, choice of kernel and launches.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "chronos_paged4.h"
#include "paged4_host.cuh"
#include "paged_rope.cuh"
#include "paged_select.cuh"

namespace chronos {
namespace {

bool power_of_two(float x) {
    int e;
    return std::frexp(x, &e) == 0.5f;
}

// Rows that are read and written 8 columns at a time (16 bytes of 16-bit types, 32 of fp32).
bool rows8(int dtype, std::initializer_list<const void*> at, std::initializer_list<int64_t> strides) {
    return std::all_of(at.begin(), at.end(), [](const void* p) { return aligned(p, 16); }) &&
           multiples(dtype == CHRONOS_DTYPE_FP32 ? 4 : 8, strides);
}
bool pages8(const ChronosPagedCache& c) {
    return rows8(c.dtype, {c.k_pages, c.v_pages},
                 {c.k_page_stride, c.k_slot_stride, c.k_head_stride, c.v_page_stride, c.v_slot_stride, c.v_head_stride});
}

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
template <typename T, typename TT, bool PACKED>
auto rope_kernel(int lanes, bool vec) -> void (*)(PagedRopeParams) {
    return !vec ? paged_rope_kernel<T, TT, 32, false, PACKED>
           : lanes == 8 ? paged_rope_kernel<T, TT, 8, true, PACKED>
           : lanes == 16 ? paged_rope_kernel<T, TT, 16, true, PACKED> : paged_rope_kernel<T, TT, 32, true, PACKED>;
}

template <typename T, typename TT>
int launch_rope(PagedRopeParams p, bool packed, bool vec, cudaStream_t st) {
    const int lanes = vec ? fp4_columns(p.c.head_dim) / 8 : 32, rows = 2 * p.c.kv_heads + p.heads;
    // Warps per token: more while SMs would be idle and every one has rows of its own.
    p.slices = 1;
    while (p.slices < kRopeWarps && p.slices * (32 / lanes) < rows && p.tokens * p.slices < 16 * static_cast<int64_t>(sm_count())) p.slices *= 2;
    const int per = kRopeWarps / p.slices;
    auto kernel = packed ? rope_kernel<T, TT, true>(lanes, vec) : rope_kernel<T, TT, false>(lanes, vec);
    const int smem = vec && sizeof(T) == 2 ? kRopeWarps * kRopeRing * 512 : 0;
    if (p.tokens > 0) {
        CHRONOS_CUDA_CHECK(launch_kernel(kernel, dim3(static_cast<unsigned>((p.tokens + per - 1) / per)), dim3(kRopeThreads), smem, st, false, p));
    }
    if (p.cu != nullptr && (p.lens_out != nullptr || p.seen_out != nullptr))
        CHRONOS_CUDA_CHECK(launch_kernel(paged_rope_advance_kernel, dim3((p.c.batch + kRopeWarps - 1) / kRopeWarps), dim3(kRopeThreads), 0,
                                         st, p.tokens > 0, p));
    return CHRONOS_OK;
}

template <typename T, bool PACKED>
auto gather_kernel(int lanes, bool vec) -> void (*)(PagedGatherParams) {
    return !vec ? paged_gather_kernel<T, 32, false, PACKED>
           : lanes == 8 ? paged_gather_kernel<T, 8, true, PACKED>
           : lanes == 16 ? paged_gather_kernel<T, 16, true, PACKED> : paged_gather_kernel<T, 32, true, PACKED>;
}
template <typename T, bool PACKED>
auto bounds_kernel(int lanes, bool vec) -> void (*)(PagedBoundsParams) {
    return !vec ? paged_bounds_kernel<T, 32, false, PACKED>
           : lanes == 8 ? paged_bounds_kernel<T, 8, true, PACKED>
           : lanes == 16 ? paged_bounds_kernel<T, 16, true, PACKED> : paged_bounds_kernel<T, 32, true, PACKED>;
}
template <typename F>
int by_dtype(int dtype, F f) {
    switch (dtype) {
        case CHRONOS_DTYPE_BF16: return f(__nv_bfloat16{});
        case CHRONOS_DTYPE_FP16: return f(__half{});
        default: return f(float{});
    }
}

// ---------------------------------------------------------------------------
// selection
// ---------------------------------------------------------------------------
constexpr size_t kSelectBytes = size_t{1} << 28;   // of keys at a time

int check_select(const ChronosPagedSelectArgs* a) {
    const char* what = "chronos_paged_select";
    if (a == nullptr) return fail(CHRONOS_ERR_INVALID_ARG, "%s: args is NULL", what);
    if (int rc = check_cache(a->cache, what)) return rc;
    if (int rc = check_heads(a->heads, a->cache, what)) return rc;
    if (a->first < 0 || a->last < 1 || a->topk < 1 || static_cast<int64_t>(a->first) + a->last > a->topk)
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: topk %d must hold first %d (>= 0) and last %d (>= 1)", what, a->topk, a->first, a->last);
    return check_tokens(a->num_tokens, a->cu_seqlens, a->cache, what);
}
// Tokens whose keys are held at a time.
int64_t select_group(const ChronosPagedSelectArgs* a) {
    const size_t one = static_cast<size_t>(a->cache.kv_heads) * std::max(1, a->cache.table_width) * 8;
    int64_t n = static_cast<int64_t>(std::max<size_t>(1, kSelectBytes / one));
    if (n >= kSelectTokens) n -= n % kSelectTokens;
    return std::max<int64_t>(1, std::min(a->num_tokens, n));
}
size_t select_bytes(const ChronosPagedSelectArgs* a) {
    if (a->cache.table_width <= a->topk) return 0;   // every row takes all its pages
    return static_cast<size_t>(select_group(a)) * a->cache.kv_heads * a->cache.table_width * 8;
}

}  // namespace
}  // namespace chronos

extern "C" int chronos_paged_append_rope(const ChronosPagedRopeArgs* a, void* stream) {
    using namespace chronos;
    g_last_error.clear();
    const char* what = "chronos_paged_append_rope";
    if (a == nullptr) return fail(CHRONOS_ERR_INVALID_ARG, "%s: args is NULL", what);
    if (int rc = check_cache(a->cache, what)) return rc;
    if (int rc = check_tokens(a->num_tokens, a->cu_seqlens, a->cache, what)) return rc;
    const bool has_q = a->heads > 0;
    if (a->heads < 0 || a->heads > 65536) return fail(CHRONOS_ERR_INVALID_ARG, "%s: heads %d", what, a->heads);
    if (a->rope_dim < 0 || a->rope_dim % 2 || a->rope_start < 0 || static_cast<int64_t>(a->rope_start) + a->rope_dim > a->cache.head_dim)
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: columns %d + %d (even) of rotation in a head of %d", what, a->rope_start, a->rope_dim,
                    a->cache.head_dim);
    if (a->rope_dim > 0 && (a->table_len < 0 || (a->table_dtype != CHRONOS_DTYPE_FP32 && a->table_dtype != a->cache.dtype)))
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: table_len %d, table_dtype %d (fp32 or the layer's)", what, a->table_len, a->table_dtype);
    if ((a->rope_dim > 0 || a->positions != nullptr || a->seen_out != nullptr) && a->seen == nullptr)
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: the rotation, positions and seen_out need seen", what);
    if ((a->weights != nullptr || a->positions != nullptr) && a->slot_cap < 0)
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: slot_cap %lld", what, static_cast<long long>(a->slot_cap));
    const int n = a->cache.batch;
    if (cross(a->lens_out, a->cache.lens, n, true) || cross(a->seen_out, a->seen, n, true) ||
        cross(a->lens_out, a->seen, n, false) || cross(a->seen_out, a->cache.lens, n, false) ||
        cross(a->lens_out, a->seen_out, n, false))
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: lens_out may be lens, seen_out may be seen, and they overlap nothing else", what);
    const int dt = a->cache.dtype, G = a->cache.kv_heads, D = a->cache.head_dim;
    const RowsOf k = rows_of(a->k, dt, a->num_tokens, a->k_row_stride, G, a->k_head_stride, D),
                 v = rows_of(a->v, dt, a->num_tokens, a->v_row_stride, G, a->v_head_stride, D),
                 q = rows_of(a->q, dt, a->num_tokens, a->q_row_stride, a->heads, a->q_head_stride, D),
                 qo = rows_of(a->q_out, dt, a->num_tokens, a->q_out_row_stride, a->heads, a->q_out_head_stride, D),
                 ko = rows_of(a->k_out, dt, a->num_tokens, a->k_out_row_stride, G, a->k_out_head_stride, D);
    if (rows_meet(qo, k) || rows_meet(qo, v) || rows_meet(qo, ko) || rows_meet(ko, v) || rows_meet(ko, q) ||
        (!rows_same(qo, q) && rows_meet(qo, q)) || (!rows_same(ko, k) && rows_meet(ko, k)))
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: q_out may be q and k_out k, with the same strides; they overlap nothing else", what);
    if (a->packed)
        if (int rc = check_packed(a->cache, a->k_scale, a->v_scale, what)) return rc;
    {
        const int64_t es = a->table_dtype == CHRONOS_DTYPE_FP32 ? 4 : 2;
        const auto table = [&](const void* at, int64_t row) {
            return RowsOf{at, at == nullptr || a->rope_dim == 0 ? 0 : a->table_len, row * es, 1, 0, a->rope_dim * es};
        };
        const RowsOf cos = table(a->cos, a->cos_row_stride), sin = table(a->sin, a->sin_row_stride), cu = array_of(a->cu_seqlens, n + int64_t{1}, 4),
                     seen = array_of(a->seen, n, 4);
        if (int rc = check_apart(what, a->cache, a->packed != 0, {qo, ko}, {cos, sin, cu, seen})) return rc;
        // (lens_out and seen_out among themselves and against lens and seen: above)
        ChronosPagedCache rest = a->cache;
        rest.lens = nullptr;
        for (const void* out : {a->lens_out, a->seen_out})
            if (int rc = check_apart(what, rest, a->packed != 0, {array_of(out, n, 4)}, {k, v, q, cos, sin, cu, qo, ko})) return rc;
    }
    const bool counts = a->lens_out != nullptr || a->seen_out != nullptr;
    if (n == 0 || (a->num_tokens == 0 && !counts)) return CHRONOS_OK;
    if (int rc = check_cache_pointers(a->cache, what)) return rc;
    if (a->num_tokens > 0 && (a->k == nullptr || a->v == nullptr || (has_q && (a->q == nullptr || a->q_out == nullptr)) ||
                              (a->rope_dim > 0 && a->table_len > 0 && (a->cos == nullptr || a->sin == nullptr))))
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: k, v, q and q_out (with heads), cos and sin (with rope_dim) are required", what);
    PagedRopeParams p{};
    p.c = a->cache;
    p.tokens = a->num_tokens;
    p.heads = a->heads;
    p.dim = a->rope_dim;
    p.start = a->rope_start;
    p.table_len = a->table_len;
    p.columns = fp4_columns(a->cache.head_dim);
    p.k = a->k;
    p.v = a->v;
    p.q = a->q;
    p.q_out = a->q_out;
    p.k_out = a->k_out;
    p.k_row = a->k_row_stride;
    p.k_head = a->k_head_stride;
    p.v_row = a->v_row_stride;
    p.v_head = a->v_head_stride;
    p.q_row = a->q_row_stride;
    p.q_head = a->q_head_stride;
    p.qo_row = a->q_out_row_stride;
    p.qo_head = a->q_out_head_stride;
    p.ko_row = a->k_out_row_stride;
    p.ko_head = a->k_out_head_stride;
    p.cos = a->cos;
    p.sin = a->sin;
    p.cos_row = a->cos_row_stride;
    p.sin_row = a->sin_row_stride;
    p.cu = a->cu_seqlens;
    p.seen = a->seen;
    p.weights = a->weights;
    p.positions = a->positions;
    p.slot_cap = a->slot_cap;
    p.max_slots = slot_limit(a->cache, a->slot_cap, a->weights != nullptr || a->positions != nullptr);
    p.lens_out = a->lens_out;
    p.seen_out = a->seen_out;
    p.k_scale = a->packed ? a->k_scale : 1.0f;
    p.v_scale = a->packed ? a->v_scale : 1.0f;
    p.k_unit = 1.0f / p.k_scale;
    p.v_unit = 1.0f / p.v_scale;
    p.k_exact = power_of_two(p.k_scale);
    p.v_exact = power_of_two(p.v_scale);
    p.status = a->status;
    bool vec = a->cache.head_dim % 8 == 0 && p.dim % 16 == 0 && p.start % 8 == 0 && (a->packed || pages8(a->cache)) &&
               rows8(dt, {p.k, p.v}, {p.k_row, p.k_head, p.v_row, p.v_head});
    if (has_q) vec = vec && rows8(dt, {p.q, p.q_out}, {p.q_row, p.q_head, p.qo_row, p.qo_head});
    if (p.k_out != nullptr) vec = vec && rows8(dt, {p.k_out}, {p.ko_row, p.ko_head});
    if (p.dim > 0) vec = vec && rows8(a->table_dtype, {p.cos, p.sin}, {p.cos_row, p.sin_row});
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return by_dtype(dt, [&](auto x) {
        using T = decltype(x);
        if (p.dim > 0 && a->table_dtype == dt) return launch_rope<T, T>(p, a->packed != 0, vec, st);
        return launch_rope<T, float>(p, a->packed != 0, vec, st);
    });
}

extern "C" int chronos_paged_gather(const ChronosPagedGatherArgs* a, void* stream) {
    using namespace chronos;
    g_last_error.clear();
    const char* what = "chronos_paged_gather";
    if (a == nullptr) return fail(CHRONOS_ERR_INVALID_ARG, "%s: args is NULL", what);
    if (int rc = check_cache(a->cache, what)) return rc;
    if (a->num_tokens < 0 || a->num_tokens > INT32_MAX)
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: num_tokens %lld", what, static_cast<long long>(a->num_tokens));
    if (a->packed)
        if (int rc = check_packed(a->cache, a->k_scale, a->v_scale, what)) return rc;
    if (a->cache.batch == 0 || a->num_tokens == 0) return CHRONOS_OK;
    if (int rc = check_cache_pointers(a->cache, what)) return rc;
    if (a->k_out == nullptr || a->v_out == nullptr || a->cu_seqlens == nullptr)
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: k_out, v_out and cu_seqlens are required", what);
    const ChronosPagedCache& c = a->cache;
    if (int rc = check_apart(what, c, a->packed != 0,
                             {rows_of(a->k_out, c.dtype, a->num_tokens, a->k_row_stride, c.kv_heads, a->k_head_stride, c.head_dim),
                              rows_of(a->v_out, c.dtype, a->num_tokens, a->v_row_stride, c.kv_heads, a->v_head_stride, c.head_dim)},
                             {array_of(a->cu_seqlens, c.batch + int64_t{1}, 4), array_of(a->first, c.batch, 4)}))
        return rc;
    PagedGatherParams p{};
    p.c = a->cache;
    p.tokens = a->num_tokens;
    p.columns = fp4_columns(a->cache.head_dim);
    p.k_scale = a->k_scale;
    p.v_scale = a->v_scale;
    p.k = a->k_out;
    p.v = a->v_out;
    p.k_row = a->k_row_stride;
    p.k_head = a->k_head_stride;
    p.v_row = a->v_row_stride;
    p.v_head = a->v_head_stride;
    p.cu = a->cu_seqlens;
    p.first = a->first;
    p.max_slots = slot_limit(a->cache, 0, false);
    p.status = a->status;
    const int dt = a->cache.dtype;
    const bool vec = a->cache.head_dim % 8 == 0 && (a->packed || pages8(a->cache)) &&
                     rows8(dt, {p.k, p.v}, {p.k_row, p.k_head, p.v_row, p.v_head});
    // as many tokens per block as leave every SM four blocks
    p.block = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kGatherTokens, p.tokens / (4 * sm_count()))));
    const dim3 grid(static_cast<unsigned>((p.tokens + p.block - 1) / p.block));
    return by_dtype(dt, [&](auto x) {
        using T = decltype(x);
        auto kernel = a->packed ? gather_kernel<T, true>(p.columns / 8, vec) : gather_kernel<T, false>(p.columns / 8, vec);
        CHRONOS_CUDA_CHECK(launch_kernel(kernel, grid, dim3(kRopeThreads), 0, static_cast<cudaStream_t>(stream), false, p));
        return static_cast<int>(CHRONOS_OK);
    });
}

extern "C" int chronos_paged_bounds(const ChronosPagedBoundsArgs* a, void* stream) {
    using namespace chronos;
    g_last_error.clear();
    const char* what = "chronos_paged_bounds";
    if (a == nullptr) return fail(CHRONOS_ERR_INVALID_ARG, "%s: args is NULL", what);
    if (int rc = check_cache(a->cache, what)) return rc;
    if (a->num_tokens < 0 || a->num_tokens > INT32_MAX)
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: num_tokens %lld", what, static_cast<long long>(a->num_tokens));
    if (a->packed) {
        ChronosPagedCache c = a->cache;
        c.v_pages = c.k_pages;
        c.v_page_stride = c.k_page_stride;
        c.v_head_stride = c.k_head_stride;
        if (int rc = check_packed(c, a->k_scale, 1.0f, what)) return rc;
    }
    const ChronosPagedCache& c = a->cache;
    if (c.batch == 0 || c.table_width == 0 || c.num_pages == 0) return CHRONOS_OK;
    if (c.lens == nullptr || c.page_table == nullptr || c.k_pages == nullptr || a->bounds == nullptr)
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: lens, page_table, k_pages and bounds are required", what);
    {
        ChronosPagedCache keys = c;
        keys.v_pages = nullptr;
        if (int rc = check_apart(what, keys, a->packed != 0, {array_of(a->bounds, c.num_pages * int64_t{2} * c.kv_heads * c.head_dim, elem_bytes(c.dtype))},
                                 {array_of(a->cu_seqlens, c.batch + int64_t{1}, 4)}))
            return rc;
    }
    PagedBoundsParams p{};
    p.c = c;
    p.packed = a->packed;
    p.columns = fp4_columns(c.head_dim);
    p.full = a->full;
    p.k_scale = a->k_scale;
    p.tokens = a->num_tokens;
    p.cu = a->cu_seqlens;
    p.bounds = a->bounds;
    p.max_slots = slot_limit(c, 0, false);
    p.status = a->status;
    // pages of a sequence that a call can touch; the blocks of a row take them in turn
    const int64_t rows = static_cast<int64_t>(c.batch) * c.kv_heads;
    int64_t pages = c.table_width;
    if (!a->full) pages = std::min<int64_t>(pages, a->cu_seqlens == nullptr ? 1 : (a->num_tokens + c.page_size - 1) / c.page_size + 1);
    pages = std::max<int64_t>(1, std::min<int64_t>(pages, 8 * static_cast<int64_t>(sm_count()) / rows));
    const unsigned by = static_cast<unsigned>(std::min<int64_t>(rows, 32768)), bz = static_cast<unsigned>((rows + by - 1) / by);
    const int es = static_cast<int>(elem_bytes(c.dtype));
    const bool vec = c.head_dim % 8 == 0 &&
                     (a->packed || (aligned(c.k_pages, 16) && multiples(16 / es, {c.k_page_stride, c.k_slot_stride, c.k_head_stride})));
    return by_dtype(c.dtype, [&](auto x) {
        using T = decltype(x);
        auto kernel = a->packed ? bounds_kernel<T, true>(p.columns / 8, vec) : bounds_kernel<T, false>(p.columns / 8, vec);
        CHRONOS_CUDA_CHECK(launch_kernel(kernel, dim3(static_cast<unsigned>(pages), by, bz), dim3(kBoundThreads), 0,
                                         static_cast<cudaStream_t>(stream), false, p));
        return static_cast<int>(CHRONOS_OK);
    });
}

extern "C" size_t chronos_paged_select_workspace(const ChronosPagedSelectArgs* a) {
    using namespace chronos;
    g_last_error.clear();
    if (check_select(a)) return 0;
    return select_bytes(a);
}

extern "C" int chronos_paged_select(const ChronosPagedSelectArgs* a, void* stream) {
    using namespace chronos;
    g_last_error.clear();
    const char* what = "chronos_paged_select";
    if (int rc = check_select(a)) return rc;
    const ChronosPagedCache& c = a->cache;
    if (c.batch == 0 || a->num_tokens == 0) return CHRONOS_OK;
    const size_t bytes = select_bytes(a);
    if (c.lens == nullptr || a->q == nullptr || a->pages == nullptr ||
        (bytes > 0 && (c.page_table == nullptr || (c.num_pages > 0 && a->bounds == nullptr))))
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: lens, page_table, q, bounds and pages are required", what);
    {
        ChronosPagedCache table = c;
        table.k_pages = table.v_pages = nullptr;
        if (int rc = check_apart(what, table, false, {array_of(a->pages, a->num_tokens * c.kv_heads * a->topk, 4)},
                                 {rows_of(a->q, c.dtype, a->num_tokens, a->q_row_stride, a->heads, a->q_head_stride, c.head_dim),
                                  array_of(a->bounds, c.num_pages * int64_t{2} * c.kv_heads * c.head_dim, elem_bytes(c.dtype)),
                                  array_of(a->cu_seqlens, c.batch + int64_t{1}, 4)}))
            return rc;
    }
    if (bytes > 0 && (a->workspace == nullptr || !aligned(a->workspace, 256) || a->workspace_bytes < bytes))
        return fail(CHRONOS_ERR_WORKSPACE_TOO_SMALL, "%s: workspace of %zu bytes, %zu (256-byte aligned) needed", what,
                    a->workspace == nullptr ? size_t{0} : a->workspace_bytes, bytes);
    PagedSelectParams p{};
    p.c = c;
    p.heads = a->heads;
    p.rep = a->heads / c.kv_heads;
    p.topk = a->topk;
    p.first = a->first;
    p.last = a->last;
    p.q = a->q;
    p.q_row = a->q_row_stride;
    p.q_head = a->q_head_stride;
    p.bounds = a->bounds;
    p.cu = a->cu_seqlens;
    p.pages = a->pages;
    p.max_slots = slot_limit(c, 0, false);
    p.width = c.table_width;
    p.keys = static_cast<unsigned long long*>(a->workspace);
    p.status = a->status;
    // rows of D elements of the bounds, one after the other
    const bool vec = c.head_dim % 8 == 0 && aligned(a->bounds, 16);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int64_t group = select_group(a);
    const int per = p.cu == nullptr ? 1 : kSelectTokens, smem = bytes > 0 ? kSelectKeys * 8 : 0;
    for (int64_t t0 = 0; t0 < a->num_tokens; t0 += group) {
        p.token0 = t0;
        p.tokens = std::min(group, a->num_tokens - t0);
        // (of a packed call every sequence may have a tile that is not full)
        const int64_t tiles = p.cu == nullptr ? p.tokens : p.tokens / per + std::min<int64_t>(c.batch, p.tokens);
        // Blocks per tile and kv head: a cluster, as long as each has a round of pages and the blocks fit
        // the SMs (of a packed call about half of them find no tile).  32 rows of 512 pages and 8 heads: 75 us
        // of the whole step with one block each, 78 with two; 34 tokens of 8 rows: 79 with two, 65 with eight.
        p.cluster = 1;
        while (p.cluster < 8 && p.cluster * 64 < c.table_width && c.table_width > p.topk &&
               2 * p.cluster * tiles * c.kv_heads <= (per == 1 ? 3 : 6) * static_cast<int64_t>(sm_count()))
            p.cluster *= 2;
        const int rc = by_dtype(c.dtype, [&](auto x) {
            using T = decltype(x);
            auto kernel = per == 1 ? (vec ? paged_select_kernel<T, true, 1> : paged_select_kernel<T, false, 1>)
                                   : (vec ? paged_select_kernel<T, true, kSelectTokens> : paged_select_kernel<T, false, kSelectTokens>);
            if (int rc = set_smem(kernel, kSelectKeys * 8)) return rc;
            CHRONOS_CUDA_CHECK(launch_cluster(kernel, dim3(static_cast<unsigned>(tiles * c.kv_heads * p.cluster)), dim3(kSelectThreads), smem,
                                              st, p.cluster, p));
            return static_cast<int>(CHRONOS_OK);
        });
        if (rc) return rc;
    }
    return CHRONOS_OK;
}

extern "C" size_t chronos_paged_rope_args_size(void) { return sizeof(ChronosPagedRopeArgs); }
extern "C" size_t chronos_paged_gather_args_size(void) { return sizeof(ChronosPagedGatherArgs); }
extern "C" size_t chronos_paged_decode4_args_size(void) { return sizeof(ChronosPagedDecode4Args); }
extern "C" size_t chronos_paged_bounds_args_size(void) { return sizeof(ChronosPagedBoundsArgs); }
extern "C" size_t chronos_paged_select_args_size(void) { return sizeof(ChronosPagedSelectArgs); }
extern "C" size_t chronos_paged_sparse_args_size(void) { return sizeof(ChronosPagedSparseArgs); }
