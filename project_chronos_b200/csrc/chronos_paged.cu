// chronos_paged.cu — the C ABI of include/chronos_paged.h: argument checks,
// workspace layout, choice of kernel and launches.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "chronos_paged.h"
#include "common.cuh"
#include "host.cuh"
#include "paged.cuh"
#include "window_attention.cuh"

namespace chronos {
namespace {

size_t elem_bytes(int dtype) { return dtype == CHRONOS_DTYPE_FP32 ? 4 : 2; }
bool dtype_known(int d) { return d == CHRONOS_DTYPE_BF16 || d == CHRONOS_DTYPE_FP16 || d == CHRONOS_DTYPE_FP32; }
size_t round_up(size_t v, size_t a) { return (v + a - 1) / a * a; }
bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
bool multiples(int64_t of, std::initializer_list<int64_t> v) {
    return std::all_of(v.begin(), v.end(), [of](int64_t x) { return x % of == 0; });
}

int check_cache(const ChronosPagedCache& c, const char* what) {
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
int check_cache_pointers(const ChronosPagedCache& c, const char* what) {
    if (c.batch > 0 && (c.lens == nullptr || (c.table_width > 0 && c.page_table == nullptr) ||
                        (c.num_pages > 0 && (c.k_pages == nullptr || c.v_pages == nullptr))))
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: lens, page_table, k_pages and v_pages are required", what);
    return CHRONOS_OK;
}
// Whether two arrays of n numbers overlap (`same`: other than as one).
template <typename T>
bool cross(const T* a, const T* b, int64_t n, bool same) {
    return a != nullptr && b != nullptr && a < b + n && b < a + n && !(same && a == b);
}
// Numbers of a per-slot array.
int64_t slots_of(const ChronosPagedCache& c, int64_t slot_cap) { return static_cast<int64_t>(c.batch) * c.kv_heads * slot_cap; }
// A window (or number of first tokens) as the kernels take it: rows have at most 2^30
// keys, so a longer one hides nothing, and positions minus it stay within 32 bits.
int cut_window(int window) { return std::min(window, 1 << 30); }
// Slots a sequence can have: what its table (and the per-slot arrays, when there are any) hold.
int slot_limit(const ChronosPagedCache& c, int64_t slot_cap, bool has_cap) {
    int64_t n = static_cast<int64_t>(c.table_width) * c.page_size;
    if (has_cap) n = std::min(n, slot_cap);
    return static_cast<int>(std::min<int64_t>(n, (1 << 30)));
}

// ---------------------------------------------------------------------------
// one-token attention
// ---------------------------------------------------------------------------
// Blocks of 64 places that a block of a cluster takes at most, where the clusters leave
// more than half of the grid idle / where they do not.  (8 each: one row set of 4096 slots
// on 64 of 296 blocks 16.4 us, 12.3 us by the work list; 64 rows up to 2048 slots on 256
// blocks 16.4 us, 18.4 us by the list; 256 rows up to 512 slots 12.4 and 20.5 us.)
constexpr int kPdClusterBlocks = 6, kPdClusterBlocksFull = 8;

// Bytes of scores that a call with running sums keeps at a time (or one sequence's, where
// those are more): it runs over groups of sequences.  64 rows under a table of 131072 slots,
// 32 / 8 heads of 128 in bf16: with 500 slots each 123 us in four groups, 91 us at once with
// 1.07 GB of scores; with 8000 slots each 468 and 427 us.
constexpr size_t kPdScoreBytes = size_t{1} << 28;

struct DecodePlan {
    int group;           // sequences at a time
    bool mma;
    int dp;              // padded head dimension of the tensor-core path
    bool one_page;       // 16 consecutive aligned slots lie in one page
    int per_sm;          // blocks an SM holds
    int cluster;         // blocks per row in one cluster; 0: the work list and a second kernel
    int rows, parts, grid, part_stride, max_vis;
    int64_t score_stride;
    size_t o_part_o, o_part_ml, o_lse2, o_scores, total;
};

int check_decode(const ChronosPagedDecodeArgs* a) {
    const char* what = "chronos_paged_decode";
    if (a == nullptr) return fail(CHRONOS_ERR_INVALID_ARG, "%s: args is NULL", what);
    if (int rc = check_cache(a->cache, what)) return rc;
    if (a->heads < 1 || a->heads % a->cache.kv_heads || a->heads / a->cache.kv_heads > kPdMaxRep)
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: heads %d must be 1..%d times kv_heads %d", what, a->heads, kPdMaxRep,
                    a->cache.kv_heads);
    if (a->window < 0 || a->sinks < 0)
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: window %d, sinks %d must not be negative", what, a->window, a->sinks);
    if (!(a->scale > 0.0f) || !std::isfinite(a->scale))
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: scale %g must be positive", what, a->scale);
    if ((a->weights == nullptr) != (a->weights_out == nullptr))
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: weights and weights_out go together", what);
    if (a->weights != nullptr && a->slot_cap < 0)
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: slot_cap %lld", what, static_cast<long long>(a->slot_cap));
    if (cross<float>(a->weights, a->weights_out, slots_of(a->cache, a->slot_cap), true))
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: weights_out overlaps weights other than as the same array", what);
    return CHRONOS_OK;
}

// The tensor-core path: rows that can be copied 16 bytes at a time (fp32: up to 128
// columns), q and out in pairs.
bool decode_uses_mma(const ChronosPagedDecodeArgs* a) {
    const ChronosPagedCache& c = a->cache;
    const int64_t n = 16 / static_cast<int64_t>(elem_bytes(c.dtype));
    return (c.dtype != CHRONOS_DTYPE_FP32 || c.head_dim <= 128) && c.head_dim % n == 0 && aligned(c.k_pages, 16) &&
           aligned(c.v_pages, 16) && aligned(a->q, 8) && aligned(a->out, 8) &&
           multiples(n, {c.k_page_stride, c.k_slot_stride, c.k_head_stride, c.v_page_stride, c.v_slot_stride, c.v_head_stride}) &&
           multiples(2, {a->q_row_stride, a->q_head_stride, a->out_row_stride, a->out_head_stride});
}

// Blocks per row when a cluster joins them, 0 when the work list is cut evenly instead.
int decode_cluster(const ChronosPagedDecodeArgs* a, const DecodePlan& d, int64_t blocks) {
    if (!d.mma || a->weights != nullptr) return 0;
    const int64_t rows = static_cast<int64_t>(d.group) * a->cache.kv_heads * d.parts;
    const int64_t room = static_cast<int64_t>(d.per_sm) * sm_count();
    int size = 1;
    while (size < 8 && size < blocks) size *= 2;
    while (size > 1 && rows * size > room) size /= 2;
    const int64_t most = 2 * rows * size > room ? kPdClusterBlocksFull : kPdClusterBlocks;
    return rows * size <= room && blocks <= most * size ? size : 0;
}

// The plan of a group of `group` sequences (0: as many as the call takes at a time).
DecodePlan decode_plan(const ChronosPagedDecodeArgs* a, int group = 0) {
    const ChronosPagedCache& c = a->cache;
    DecodePlan d{};
    d.mma = decode_uses_mma(a);
    d.dp = c.head_dim <= 64 ? 64 : c.head_dim <= 128 ? 128 : 256;
    d.per_sm = !d.mma ? 4 : d.dp * elem_bytes(c.dtype) == 128 ? 3 : 2;   // PagedMma::kBlocksPerSm
    d.rows = d.mma && c.dtype != CHRONOS_DTYPE_FP32 ? 16 : 8;
    const int rep = a->heads / c.kv_heads;
    d.parts = (rep + d.rows - 1) / d.rows;
    const int limit = slot_limit(c, a->slot_cap, a->weights != nullptr);
    // places of a row: both runs of visible slots start at a multiple of 16
    d.max_vis = a->window > 0 ? static_cast<int>(std::min<int64_t>(limit, static_cast<int64_t>(a->window) + a->sinks + 32)) : limit;
    d.one_page = c.page_size % kPdTile == 0;
    d.score_stride = a->weights != nullptr ? round_up(d.max_vis, kPdBlock) : 0;
    d.group = group > 0 ? group : c.batch;
    const size_t scores = static_cast<size_t>(a->heads) * d.score_stride * 4;   // of a sequence
    if (group == 0 && scores > 0 && scores * c.batch > kPdScoreBytes) {
        const int most = static_cast<int>(std::max<size_t>(1, kPdScoreBytes / scores));
        const int groups = (c.batch + most - 1) / most;
        d.group = (c.batch + groups - 1) / groups;
    }
    const int64_t blocks = (static_cast<int64_t>(d.max_vis) + kPdBlock - 1) / kPdBlock;
    const int64_t units = std::max<int64_t>(1, blocks) * d.group * c.kv_heads * d.parts;
    d.grid = static_cast<int>(std::min<int64_t>({units, static_cast<int64_t>(d.per_sm) * sm_count(), kPdMaxGrid}));
    d.cluster = decode_cluster(a, d, blocks);
    d.part_stride = d.mma ? d.dp : static_cast<int>(round_up(c.head_dim, 4));
    size_t at = 0;
    auto take = [&at](size_t bytes) {
        const size_t o = at;
        at = round_up(at + bytes, 256);
        return o;
    };
    const size_t slots = d.cluster > 0 ? 0 : 2 * static_cast<size_t>(d.grid) * d.rows;
    d.o_part_o = take(slots * d.part_stride * 4);
    d.o_part_ml = take(slots * 8);
    if (a->weights != nullptr) {
        d.o_lse2 = take(static_cast<size_t>(d.group) * a->heads * 4);
        d.o_scores = take(scores * d.group);
    }
    d.total = d.cluster > 0 ? 0 : std::max<size_t>(at, 256);   // a cluster needs none
    return d;
}

using DecodeKernel = void (*)(PagedDecodeParams);
template <typename T, int DP, int NT>
DecodeKernel decode_kernel(bool one_page, bool cluster) {
    if (cluster) return one_page ? paged_decode_mma_kernel<T, DP, NT, true, true> : paged_decode_mma_kernel<T, DP, NT, false, true>;
    return one_page ? paged_decode_mma_kernel<T, DP, NT, true, false> : paged_decode_mma_kernel<T, DP, NT, false, false>;
}

template <typename T, int DP>
int launch_decode_mma(const PagedDecodeParams& p, const DecodePlan& d, cudaStream_t st) {
    using S = PagedMma<T, DP>;
    DecodeKernel kernel = decode_kernel<T, DP, 1>(d.one_page, d.cluster > 0);
    if constexpr (sizeof(T) == 2)
        if (p.rep > 8) kernel = decode_kernel<T, DP, 2>(d.one_page, d.cluster > 0);
    if (int rc = set_smem(kernel, S::kSmem)) return rc;
    if (d.cluster == 0) {
        CHRONOS_CUDA_CHECK(launch_kernel(kernel, dim3(p.grid), dim3(kPdThreads), S::kSmem, st, false, p));
        return CHRONOS_OK;
    }
    CHRONOS_CUDA_CHECK(launch_cluster(kernel, dim3(static_cast<unsigned>(p.c.batch) * p.c.kv_heads * p.parts * d.cluster),
                                      dim3(kPdThreads), S::kSmem, st, d.cluster, p));
    return CHRONOS_OK;
}

template <typename T>
int launch_decode(const PagedDecodeParams& p, const DecodePlan& d, bool vec, cudaStream_t st) {
    if (d.mma) {
        int rc;
        if constexpr (sizeof(T) == 2)
            rc = d.dp == 64 ? launch_decode_mma<T, 64>(p, d, st)
                            : d.dp == 128 ? launch_decode_mma<T, 128>(p, d, st) : launch_decode_mma<T, 256>(p, d, st);
        else
            rc = d.dp == 64 ? launch_decode_mma<T, 64>(p, d, st) : launch_decode_mma<T, 128>(p, d, st);
        if (rc || d.cluster > 0) return rc;
    }
    if (!d.mma)
        CHRONOS_CUDA_CHECK(launch_kernel(vec ? paged_decode_simt_kernel<T, true> : paged_decode_simt_kernel<T, false>,
                                         dim3(p.grid), dim3(kPdThreads), 0, st, false, p));
    // rows of one unit are never cut: then there is nothing to join
    const bool joins = d.max_vis > kPdBlock;
    PagedDecodeParams j = p;
    j.join_blocks = joins ? p.c.batch * p.heads : 0;
    j.weight_chunks = (p.max_slots + kPdWeightSlots - 1) / kPdWeightSlots;
    const int64_t blocks = j.join_blocks + (p.weights != nullptr ? static_cast<int64_t>(p.c.batch) * p.c.kv_heads * j.weight_chunks : 0);
    if (blocks > 0)
        CHRONOS_CUDA_CHECK(launch_kernel(paged_join_kernel<T>, dim3(static_cast<unsigned>(blocks)), dim3(kPdJoinThreads), 0,
                                         st, true, j));
    return CHRONOS_OK;
}

// The sequences from b0 on that plan `d` is of.
int decode_group(const ChronosPagedDecodeArgs* a, const DecodePlan& d, int b0, int limit, cudaStream_t st) {
    const int64_t es = static_cast<int64_t>(elem_bytes(a->cache.dtype));
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    PagedDecodeParams p{};
    p.c = a->cache;
    p.c.batch = d.group;
    p.c.lens += b0;
    p.c.page_table += b0 * a->cache.page_table_stride;
    p.heads = a->heads;
    p.rep = a->heads / a->cache.kv_heads;
    p.rows = d.rows;
    p.parts = d.parts;
    p.window = cut_window(a->window);
    p.sinks = a->window > 0 ? cut_window(a->sinks) : 0;
    p.max_slots = limit;
    p.page_shift = -1;
    if ((a->cache.page_size & (a->cache.page_size - 1)) == 0)
        for (p.page_shift = 0; (1 << p.page_shift) < a->cache.page_size;) ++p.page_shift;
    p.cluster = d.cluster;
    p.sl2 = static_cast<float>(static_cast<double>(a->scale) * 1.4426950408889634);
    p.q = static_cast<const uint8_t*>(a->q) + b0 * a->q_row_stride * es;
    p.q_row = a->q_row_stride;
    p.q_head = a->q_head_stride;
    p.out = static_cast<uint8_t*>(a->out) + b0 * a->out_row_stride * es;
    p.out_row = a->out_row_stride;
    p.out_head = a->out_head_stride;
    if (a->lse != nullptr) p.lse = a->lse + static_cast<int64_t>(b0) * a->heads;
    if (a->weights != nullptr) {
        const int64_t at = static_cast<int64_t>(b0) * a->cache.kv_heads * a->slot_cap;
        p.weights = a->weights + at;
        p.weights_out = a->weights_out + at;
    }
    p.slot_cap = a->slot_cap;
    p.grid = d.grid;
    p.part_stride = d.part_stride;
    p.part_o = reinterpret_cast<float*>(ws + d.o_part_o);
    p.part_ml = reinterpret_cast<float*>(ws + d.o_part_ml);
    if (a->weights != nullptr) {
        p.lse2 = reinterpret_cast<float*>(ws + d.o_lse2);
        p.scores = reinterpret_cast<float*>(ws + d.o_scores);
        p.score_stride = d.score_stride;
    }
    p.status = a->status;
    const int64_t ve = a->cache.dtype == CHRONOS_DTYPE_FP32 ? 16 : 8;
    const bool vec = a->cache.head_dim % 4 == 0 && aligned(a->cache.k_pages, ve) && aligned(a->cache.v_pages, ve) &&
                     multiples(4, {a->cache.k_page_stride, a->cache.k_slot_stride, a->cache.k_head_stride,
                                   a->cache.v_page_stride, a->cache.v_slot_stride, a->cache.v_head_stride});
    switch (a->cache.dtype) {
        case CHRONOS_DTYPE_BF16: return launch_decode<__nv_bfloat16>(p, d, vec, st);
        case CHRONOS_DTYPE_FP16: return launch_decode<__half>(p, d, vec, st);
        default: return launch_decode<float>(p, d, vec, st);
    }
}

// ---------------------------------------------------------------------------
// eviction
// ---------------------------------------------------------------------------
constexpr int kEvictKeyBytes = 192 * 1024;   // of shared memory for the keys of a row
static_assert(kEvictKeyBytes / 4 / 32 <= 3 * kEvictBins / 2, "the bits of such a row fit the counters' place");

struct EvictPlan {
    int64_t max_moves;
    int64_t bit_words;      // 0 where a row's keys (and then its bits) fit shared memory
    size_t o_moves, o_counts, o_lens, o_bits, total;
};

int check_evict(const ChronosPagedEvictArgs* a) {
    const char* what = "chronos_paged_evict";
    if (a == nullptr) return fail(CHRONOS_ERR_INVALID_ARG, "%s: args is NULL", what);
    if (int rc = check_cache(a->cache, what)) return rc;
    if (a->budget < 1 || a->sinks < 0 || a->recent < 0 ||
        static_cast<int64_t>(a->sinks) + a->recent > a->budget)
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: budget %d must be >= 1 and >= sinks %d + recent %d", what, a->budget,
                    a->sinks, a->recent);
    if (a->slot_cap < 0) return fail(CHRONOS_ERR_INVALID_ARG, "%s: slot_cap %lld", what, static_cast<long long>(a->slot_cap));
    const int64_t n = slots_of(a->cache, a->slot_cap);
    if (cross<float>(a->weights, a->weights_out, n, true) || cross<int32_t>(a->positions, a->positions_out, n, true))
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: weights_out and positions_out overlap their inputs other than as the same arrays",
                    what);
    return CHRONOS_OK;
}

EvictPlan evict_plan(const ChronosPagedEvictArgs* a) {
    EvictPlan e{};
    const int limit = slot_limit(a->cache, a->slot_cap, true);
    e.max_moves = std::max(0, std::min(a->budget, limit - a->budget));
    const size_t rows = static_cast<size_t>(a->cache.batch) * a->cache.kv_heads;
    e.o_moves = 0;
    e.o_counts = round_up(rows * e.max_moves * 8, 256);
    e.o_lens = e.o_counts + round_up(rows * 4, 256);
    e.o_bits = e.o_lens + round_up(static_cast<size_t>(a->cache.batch) * 4, 256);
    e.bit_words = static_cast<int64_t>(limit) * 4 <= kEvictKeyBytes ? 0 : (limit + 31) / 32;
    e.total = e.o_bits + rows * e.bit_words * 8 + 256;
    return e;
}

// Bytes of the widest unit that every row can be copied in: 16, or one element.
bool copies16(const ChronosPagedCache& c) {
    const int64_t n = 16 / static_cast<int64_t>(elem_bytes(c.dtype));
    return c.head_dim % n == 0 && aligned(c.k_pages, 16) && aligned(c.v_pages, 16) &&
           multiples(n, {c.k_page_stride, c.k_slot_stride, c.k_head_stride, c.v_page_stride, c.v_slot_stride, c.v_head_stride});
}

// ---------------------------------------------------------------------------
// prompt attention
// ---------------------------------------------------------------------------
template <typename T, bool VEC>
auto window_simt_pick(int dim) -> void (*)(WindowParams) {
    return dim <= 64 ? window_simt_kernel<T, 1, VEC>
           : dim <= 128 ? window_simt_kernel<T, 2, VEC>
           : dim <= 192 ? window_simt_kernel<T, 3, VEC> : window_simt_kernel<T, 4, VEC>;
}

template <typename T>
int launch_window_simt(const WindowParams& p, cudaStream_t st) {
    const size_t four = 4 * sizeof(T);
    const bool vec = p.dim % 4 == 0 && aligned(p.q, four) && aligned(p.k, four) && aligned(p.v, four) &&
                     multiples(4, {p.q_row, p.q_head, p.k_row, p.k_head, p.v_row, p.v_head});
    void (*kernel)(WindowParams) = vec ? window_simt_pick<T, true>(p.dim) : window_simt_pick<T, false>(p.dim);
    const int smem = window_simt_smem(p.dim);
    if (int rc = set_smem(kernel, smem)) return rc;
    const int64_t tiles = (p.num_q + kWsRows - 1) / kWsRows + p.batch;   // one more than there are, at least
    CHRONOS_CUDA_CHECK(launch_kernel(kernel, dim3(static_cast<unsigned>(tiles * p.heads)), dim3(kWsThreads), smem, st, false, p));
    return CHRONOS_OK;
}

// Tensor map of rows of 16-bit vectors: `dims` outermost last, `strides` in
// elements (of dims[1..]), box of 64 elements by box[1..], 128-byte swizzle.
bool encode_rows(CUtensorMap* m, int dtype, const void* base, int rank, const uint64_t* dims, const int64_t* strides,
                 const uint32_t* box) {
    EncodeTiledFn enc = get_encode_fn();
    if (enc == nullptr) return false;
    cuuint64_t d[4], s[3];
    cuuint32_t b[4], e[4] = {1, 1, 1, 1};
    for (int i = 0; i < rank; ++i) {
        d[i] = dims[i];
        b[i] = box[i];
        if (i > 0) s[i - 1] = static_cast<cuuint64_t>(strides[i - 1]) * 2;
    }
    return enc(m, dtype == CHRONOS_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
               static_cast<cuuint32_t>(rank), const_cast<void*>(base), d, s, b, e, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// What the loads and the 16-byte stores of the tensor-core path need.  A tensor map steps by
// at least one element: rows or heads read several times (a stride of zero) have no map.
bool window_uses_tc(const WindowParams& p) {
    if ((p.num_q > 1 && p.q_row == 0) || (p.heads > 1 && p.q_head == 0) || (p.num_k > 1 && (p.k_row == 0 || p.v_row == 0)) ||
        (p.kv_heads > 1 && (p.k_head == 0 || p.v_head == 0)))
        return false;
    return p.dim % 8 == 0 && p.dim <= 128 && p.num_k > 0 && aligned(p.q, 16) && aligned(p.k, 16) && aligned(p.v, 16) &&
           aligned(p.out, 16) &&
           multiples(8, {p.q_row, p.q_head, p.k_row, p.k_head, p.v_row, p.v_head, p.o_row, p.o_head});
}

template <typename T, int DP>
int launch_window_tc(const WindowParams& p, int dtype, bool* taken, cudaStream_t st) {
    // rows of a block: the query heads of a kv head side by side where their number divides a tile
    int rp_log2 = 0;
    if ((p.rep & (p.rep - 1)) == 0 && p.rep <= 16)
        while ((1 << rp_log2) < p.rep) ++rp_log2;
    const int rp = 1 << rp_log2, groups = p.heads / rp;
    const uint64_t dq[4] = {static_cast<uint64_t>(p.dim), static_cast<uint64_t>(rp), static_cast<uint64_t>(groups),
                            static_cast<uint64_t>(p.num_q)};
    const uint64_t dk[3] = {static_cast<uint64_t>(p.dim), static_cast<uint64_t>(p.kv_heads), static_cast<uint64_t>(p.num_k)};
    const int64_t sq[3] = {p.q_head, p.q_head * rp, p.q_row}, sk[2] = {p.k_head, p.k_row}, sv[2] = {p.v_head, p.v_row};
    const uint32_t bq[4] = {64, static_cast<uint32_t>(rp), 1, static_cast<uint32_t>(128 / rp)}, bk[3] = {64, 1, kWtKeys};
    CUtensorMap mq, mk, mv;
    *taken = encode_rows(&mq, dtype, p.q, 4, dq, sq, bq) && encode_rows(&mk, dtype, p.k, 3, dk, sk, bk) &&
             encode_rows(&mv, dtype, p.v, 3, dk, sv, bk);
    if (!*taken) return CHRONOS_OK;   // strides the maps cannot hold
    using C = WindowTc<DP>;
    const int tokens = 256 / rp;
    const int64_t tiles = (p.num_q + static_cast<int64_t>(p.batch) * (tokens - 1)) / tokens;   // at most
    const int64_t blocks = tiles * groups;
    // Split the keys over a cluster while SMs are idle and the sequences' mean length leaves each
    // block two tiles or more; not below 8 tiles, where the join costs what the split gains (517
    // keys on two blocks 16.5 us, split 23; 1500 keys on 64 blocks 29 us, split 24.7; 64 queries
    // on 8064 keys 119 us, split over 8 blocks 36).
    const int64_t mean = p.num_k / p.batch;
    const int64_t keys = p.window > 0 ? std::min<int64_t>(mean, static_cast<int64_t>(p.window) + p.sinks + tokens) : mean;
    int splits = 1;   // (and one tile's blocks that check the offsets)
    while (splits < 8 && blocks * splits * 2 <= sm_count() && keys >= std::max(8, 4 * splits) * kWtKeys) splits *= 2;
    if (splits == 1) {
        if (int rc = set_smem(window_tc_kernel<T, DP, false>, C::kSmem)) return rc;
        CHRONOS_CUDA_CHECK(launch_kernel(window_tc_kernel<T, DP, false>, dim3(static_cast<unsigned>(blocks + 1)), dim3(kWtThreads),
                                         C::kSmem, st, false, p, mq, mk, mv, rp_log2, groups, 1));
        return CHRONOS_OK;
    }
    if (int rc = set_smem(window_tc_kernel<T, DP, true>, C::kSplitSmem)) return rc;
    CHRONOS_CUDA_CHECK(launch_cluster(window_tc_kernel<T, DP, true>, dim3(static_cast<unsigned>((blocks + 1) * splits)), dim3(kWtThreads),
                                      C::kSplitSmem, st, splits, p, mq, mk, mv, rp_log2, groups, splits));
    return CHRONOS_OK;
}

template <typename T>
int window_impl(WindowParams p, int dtype, cudaStream_t st) {
    if constexpr (sizeof(T) == 2) {
        if (window_uses_tc(p)) {
            // no step is ever taken in a dimension of one: any stride will do
            if (p.num_q == 1) p.q_row = p.dim;
            if (p.heads == 1) p.q_head = p.dim;
            if (p.num_k == 1) p.k_row = p.v_row = p.dim;
            if (p.kv_heads == 1) p.k_head = p.v_head = p.dim;
            bool taken = false;
            const int rc = p.dim <= 64 ? launch_window_tc<T, 64>(p, dtype, &taken, st) : launch_window_tc<T, 128>(p, dtype, &taken, st);
            if (rc || taken) return rc;
        }
    }
    return launch_window_simt<T>(p, st);
}

}  // namespace
}  // namespace chronos

extern "C" size_t chronos_paged_decode_workspace(const ChronosPagedDecodeArgs* a) {
    using namespace chronos;
    g_last_error.clear();
    if (check_decode(a)) return 0;
    return decode_plan(a).total;
}

extern "C" int chronos_paged_decode(const ChronosPagedDecodeArgs* a, void* stream) {
    using namespace chronos;
    g_last_error.clear();
    const char* what = "chronos_paged_decode";
    if (int rc = check_decode(a)) return rc;
    if (a->cache.batch == 0) return CHRONOS_OK;
    if (int rc = check_cache_pointers(a->cache, what)) return rc;
    if (a->q == nullptr || a->out == nullptr) return fail(CHRONOS_ERR_INVALID_ARG, "%s: q and out are required", what);
    const DecodePlan d = decode_plan(a);
    const int64_t units = (static_cast<int64_t>(d.max_vis) / kPdBlock + 1) * a->cache.batch * a->cache.kv_heads * d.parts;
    const int limit = slot_limit(a->cache, a->slot_cap, a->weights != nullptr);
    const int64_t adds = static_cast<int64_t>(a->cache.batch) * a->heads +
                         static_cast<int64_t>(a->cache.batch) * a->cache.kv_heads * (limit / kPdWeightSlots + 1);
    if (units >= (1 << 30) || adds >= INT32_MAX)
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: batch %d * heads * slots %d too large", what, a->cache.batch, limit);
    if (d.total > 0 && (a->workspace == nullptr || !aligned(a->workspace, 256) || a->workspace_bytes < d.total))
        return fail(CHRONOS_ERR_WORKSPACE_TOO_SMALL, "%s: workspace of %zu bytes, %zu (256-byte aligned) needed", what,
                    a->workspace == nullptr ? size_t{0} : a->workspace_bytes, d.total);
    for (int b0 = 0; b0 < a->cache.batch; b0 += d.group) {
        const int n = std::min(d.group, a->cache.batch - b0);
        if (int rc = decode_group(a, n == d.group ? d : decode_plan(a, n), b0, limit, static_cast<cudaStream_t>(stream))) return rc;
    }
    return CHRONOS_OK;
}

extern "C" int chronos_paged_append(const ChronosPagedAppendArgs* a, void* stream) {
    using namespace chronos;
    g_last_error.clear();
    const char* what = "chronos_paged_append";
    if (a == nullptr) return fail(CHRONOS_ERR_INVALID_ARG, "%s: args is NULL", what);
    if (int rc = check_cache(a->cache, what)) return rc;
    if (a->num_tokens < 0 || a->num_tokens > INT32_MAX)
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: num_tokens %lld", what, static_cast<long long>(a->num_tokens));
    if (a->cu_seqlens == nullptr && a->num_tokens != a->cache.batch)
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: %lld rows for %d sequences without cu_seqlens", what,
                    static_cast<long long>(a->num_tokens), a->cache.batch);
    if (a->positions != nullptr && a->seen == nullptr)
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: positions need seen", what);
    const bool arrays = a->weights != nullptr || a->positions != nullptr;
    if (arrays && a->slot_cap < 0)
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: slot_cap %lld", what, static_cast<long long>(a->slot_cap));
    if (a->seen_out != nullptr && a->seen == nullptr)
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: seen_out needs seen", what);
    const int n = a->cache.batch;
    if (cross(a->lens_out, a->cache.lens, n, true) || cross(a->seen_out, a->seen, n, true) ||
        cross(a->lens_out, a->seen, n, false) || cross(a->seen_out, a->cache.lens, n, false) ||
        cross(a->lens_out, a->seen_out, n, false))
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: lens_out may be lens, seen_out may be seen, and they overlap nothing else", what);
    const bool counts = a->lens_out != nullptr || a->seen_out != nullptr;
    if (a->cache.batch == 0 || (a->num_tokens == 0 && !counts)) return CHRONOS_OK;
    if (int rc = check_cache_pointers(a->cache, what)) return rc;
    if (a->num_tokens > 0 && (a->k == nullptr || a->v == nullptr)) return fail(CHRONOS_ERR_INVALID_ARG, "%s: k and v are required", what);
    PagedAppendParams p{};
    p.c = a->cache;
    p.tokens = a->num_tokens;
    p.k = a->k;
    p.v = a->v;
    p.k_row = a->k_row_stride;
    p.k_head = a->k_head_stride;
    p.v_row = a->v_row_stride;
    p.v_head = a->v_head_stride;
    p.cu = a->cu_seqlens;
    p.seen = a->seen;
    p.weights = a->weights;
    p.positions = a->positions;
    p.slot_cap = a->slot_cap;
    p.max_slots = slot_limit(a->cache, a->slot_cap, arrays);
    p.lens_out = a->lens_out;
    p.seen_out = a->seen_out;
    p.status = a->status;
    const int es = static_cast<int>(elem_bytes(a->cache.dtype));
    const bool wide = copies16(a->cache) && aligned(a->k, 16) && aligned(a->v, 16) &&
                      multiples(16 / es, {a->k_row_stride, a->k_head_stride, a->v_row_stride, a->v_head_stride});
    const int per = wide ? 16 / es : 1;
    const int units = a->cache.head_dim / per;
    const int64_t blocks = (a->num_tokens + kAppendThreads / 32 - 1) / (kAppendThreads / 32);
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(blocks, 64 * static_cast<int64_t>(sm_count()))));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a->num_tokens > 0) {
        if (wide) CHRONOS_CUDA_CHECK(launch_kernel(paged_append_kernel<uint4>, grid, dim3(kAppendThreads), 0, st, false, p, units, per));
        else if (es == 2) CHRONOS_CUDA_CHECK(launch_kernel(paged_append_kernel<uint16_t>, grid, dim3(kAppendThreads), 0, st, false, p, units, per));
        else CHRONOS_CUDA_CHECK(launch_kernel(paged_append_kernel<uint32_t>, grid, dim3(kAppendThreads), 0, st, false, p, units, per));
    }
    if (counts && a->cu_seqlens != nullptr)
        CHRONOS_CUDA_CHECK(launch_kernel(paged_advance_kernel, dim3((n + kAppendThreads / 32 - 1) / (kAppendThreads / 32)),
                                         dim3(kAppendThreads), 0, st, a->num_tokens > 0, p));
    return CHRONOS_OK;
}

extern "C" size_t chronos_paged_evict_workspace(const ChronosPagedEvictArgs* a) {
    using namespace chronos;
    g_last_error.clear();
    if (check_evict(a)) return 0;
    return evict_plan(a).total;
}

extern "C" int chronos_paged_evict(const ChronosPagedEvictArgs* a, void* stream) {
    using namespace chronos;
    g_last_error.clear();
    const char* what = "chronos_paged_evict";
    if (int rc = check_evict(a)) return rc;
    if (a->cache.batch == 0) return CHRONOS_OK;
    if (int rc = check_cache_pointers(a->cache, what)) return rc;
    if (a->seen == nullptr || a->weights == nullptr || a->positions == nullptr || a->weights_out == nullptr ||
        a->positions_out == nullptr || a->lens_out == nullptr || a->src == nullptr)
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: seen, weights, positions, their outputs, lens_out and src are required", what);
    const int rows = a->cache.batch * a->cache.kv_heads;
    const EvictPlan e = evict_plan(a);
    if (a->workspace == nullptr || !aligned(a->workspace, 256) || a->workspace_bytes < e.total)
        return fail(CHRONOS_ERR_WORKSPACE_TOO_SMALL, "%s: workspace of %zu bytes, %zu (256-byte aligned) needed", what,
                    a->workspace == nullptr ? size_t{0} : a->workspace_bytes, e.total);
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    PagedEvictParams p{};
    p.c = a->cache;
    p.budget = a->budget;
    p.sinks = a->sinks;
    p.recent = a->recent;
    p.seen = a->seen;
    p.weights = a->weights;
    p.positions = a->positions;
    p.weights_out = a->weights_out;
    p.positions_out = a->positions_out;
    p.slot_cap = a->slot_cap;
    p.lens_out = a->lens_out;
    p.src = a->src;
    p.max_slots = slot_limit(a->cache, a->slot_cap, true);
    p.moves = reinterpret_cast<int32_t*>(ws + e.o_moves);
    p.counts = reinterpret_cast<int32_t*>(ws + e.o_counts);
    p.lens_copy = reinterpret_cast<int32_t*>(ws + e.o_lens);
    p.max_moves = e.max_moves;
    p.status = a->status;
    const int64_t key_bytes = static_cast<int64_t>(p.max_slots) * 4;
    p.keys_in_smem = key_bytes <= kEvictKeyBytes;
    p.bits = reinterpret_cast<uint32_t*>(ws + e.o_bits);
    p.bit_words = e.bit_words;
    const int smem = p.keys_in_smem ? static_cast<int>(key_bytes) : 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (int rc = set_smem(paged_evict_select_kernel, kEvictKeyBytes)) return rc;
    const int es = static_cast<int>(elem_bytes(a->cache.dtype));
    const bool wide = copies16(a->cache);
    const int per = wide ? 16 / es : 1;
    const int units = a->cache.head_dim / per;
    // Few moves per row (a cache that gives up a page's slots at a time): the selecting block
    // makes them, without the second kernel.  Not where lens_out lies over lens or seen, which
    // the other kv heads' blocks still read.
    p.move_here = wide && e.max_moves <= kEvictMovesHere && !cross(a->lens_out, a->cache.lens, a->cache.batch, false) &&
                  !cross(a->lens_out, a->seen, a->cache.batch, false);
    CHRONOS_CUDA_CHECK(launch_kernel(paged_evict_select_kernel, dim3(rows), dim3(kEvictThreads), smem, st, false, p, units, per));
    if (p.move_here) return CHRONOS_OK;
    const int64_t bx = std::max<int64_t>(1, std::min<int64_t>((e.max_moves + kEvictMovesPerBlock - 1) / kEvictMovesPerBlock, 4096));
    const unsigned by = std::min(rows, 32768), bz = (rows + by - 1) / by;   // rows, up to 2^20
    const dim3 grid(static_cast<unsigned>(bx), by, bz), block(kEvictMoveThreads);
    if (wide) CHRONOS_CUDA_CHECK(launch_kernel(paged_evict_move_kernel<uint4>, grid, block, 0, st, true, p, units, per));
    else if (es == 2) CHRONOS_CUDA_CHECK(launch_kernel(paged_evict_move_kernel<uint16_t>, grid, block, 0, st, true, p, units, per));
    else CHRONOS_CUDA_CHECK(launch_kernel(paged_evict_move_kernel<uint32_t>, grid, block, 0, st, true, p, units, per));
    return CHRONOS_OK;
}

extern "C" int chronos_window_attention(const ChronosWindowAttnArgs* a, void* stream) {
    using namespace chronos;
    g_last_error.clear();
    const char* what = "chronos_window_attention";
    if (a == nullptr) return fail(CHRONOS_ERR_INVALID_ARG, "%s: args is NULL", what);
    if (a->batch < 0 || a->kv_heads < 1 || a->heads < 1 || a->heads % a->kv_heads || a->head_dim < 1 ||
        a->head_dim > CHRONOS_PAGED_MAX_HEAD_DIM || !dtype_known(a->dtype))
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: batch %d, heads %d, kv_heads %d (divides heads), head_dim %d (1..%d), dtype %d",
                    what, a->batch, a->heads, a->kv_heads, a->head_dim, CHRONOS_PAGED_MAX_HEAD_DIM, a->dtype);
    if (a->window < 0 || a->sinks < 0)
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: window %d, sinks %d must not be negative", what, a->window, a->sinks);
    if (!(a->scale > 0.0f) || !std::isfinite(a->scale))
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: scale %g must be positive", what, a->scale);
    if (a->num_q < 0 || a->num_k < 0 || a->num_q > (1 << 30) || a->num_k > (1 << 30) ||
        ((a->num_q + kWsRows - 1) / kWsRows + a->batch) * a->heads >= INT32_MAX)
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: %lld query rows, %lld key rows", what, static_cast<long long>(a->num_q),
                    static_cast<long long>(a->num_k));
    if (a->batch == 0 || a->num_q == 0) return CHRONOS_OK;
    if (a->q == nullptr || a->out == nullptr || a->cu_q == nullptr || a->cu_k == nullptr ||
        (a->num_k > 0 && (a->k == nullptr || a->v == nullptr)))
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: q, k, v, out, cu_q and cu_k are required", what);
    if (a->num_k > 0 && (a->out == a->k || a->out == a->v))
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: out may be q, but not k or v", what);
    WindowParams p{};
    p.batch = a->batch;
    p.heads = a->heads;
    p.kv_heads = a->kv_heads;
    p.rep = a->heads / a->kv_heads;
    p.dim = a->head_dim;
    p.window = cut_window(a->window);
    p.sinks = a->window > 0 ? cut_window(a->sinks) : 0;
    p.sl2 = static_cast<float>(static_cast<double>(a->scale) * 1.4426950408889634);
    p.num_q = a->num_q;
    p.num_k = a->num_k;
    p.q = a->q;
    p.k = a->k;
    p.v = a->v;
    p.out = a->out;
    p.q_row = a->q_row_stride;
    p.q_head = a->q_head_stride;
    p.k_row = a->k_row_stride;
    p.k_head = a->k_head_stride;
    p.v_row = a->v_row_stride;
    p.v_head = a->v_head_stride;
    p.o_row = a->out_row_stride;
    p.o_head = a->out_head_stride;
    p.cu_q = a->cu_q;
    p.cu_k = a->cu_k;
    p.lse = a->lse;
    p.status = a->status;
    if (p.k_head == 0 && p.v_head == 0) {   // one kv head read as several
        p.kv_heads = 1;
        p.rep = p.heads;
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (a->dtype) {
        case CHRONOS_DTYPE_BF16: return window_impl<__nv_bfloat16>(p, a->dtype, st);
        case CHRONOS_DTYPE_FP16: return window_impl<__half>(p, a->dtype, st);
        default: return window_impl<float>(p, a->dtype, st);
    }
}

extern "C" size_t chronos_paged_append_args_size(void) { return sizeof(ChronosPagedAppendArgs); }
extern "C" size_t chronos_paged_decode_args_size(void) { return sizeof(ChronosPagedDecodeArgs); }
extern "C" size_t chronos_paged_evict_args_size(void) { return sizeof(ChronosPagedEvictArgs); }
extern "C" size_t chronos_window_attn_args_size(void) { return sizeof(ChronosWindowAttnArgs); }
