// chronos_decode4.cu — chronos_paged_decode4 (include/chronos_paged4.h): argument checks,
// workspace layout, choice of kernel and launches.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "paged4.cuh"
#include "paged4_host.cuh"

namespace chronos {
namespace {

// Blocks of 64 slots that a block of a cluster takes at most: where the clusters leave half of the
// grid idle / do not / where the rows alone fill it (clusters of one, also more of them than run at
// once).  Beyond that the work list, which cuts all rows evenly but costs a second kernel and joins.
// Heads of 128, list against cluster: 1 row of 4096 slots, 2 kv heads (8 blocks each) 11.8 and 14.4 us;
// 16 rows up to 1500 slots, 8 kv heads (12 each) 19.1 and 15.9 us, 20 rows up to 4000 (32 each) 29.0 and
// 35.6 us; 48 rows up to 1500 (24 each) 37.9 and 28.9 us, 128 rows up to 500 57 and 34 us, 100 rows up to
// 4000 (63 each) 115 and 124 us.
constexpr int kP4ClusterBlocks = 6, kP4ClusterBlocksFull = 16, kP4RowBlocks = 24;
// Tiles of 16 slots that a warp takes of a unit of the work list.
constexpr int kP4ListTiles = 4;

struct Decode4Plan {
    int dp, parts, grid, cluster, max_vis;
    size_t o_part_ml, total;
};

int check_decode4(const ChronosPagedDecode4Args* a) {
    const char* what = "chronos_paged_decode4";
    if (a == nullptr) return fail(CHRONOS_ERR_INVALID_ARG, "%s: args is NULL", what);
    if (int rc = check_cache(a->cache, what)) return rc;
    if (int rc = check_heads(a->heads, a->cache, what)) return rc;
    if (a->window < 0 || a->sinks < 0)
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: window %d, sinks %d must not be negative", what, a->window, a->sinks);
    if (int rc = check_positive("scale", a->scale, what)) return rc;
    if (int rc = check_packed(a->cache, a->k_scale, a->v_scale, what)) return rc;
    return check_scores(a->scale, a->k_scale, what);
}

template <typename T, int DP, int NT>
int blocks_per_sm() {
    return Paged4<T, DP, NT>::kBlocksPerSm;
}
template <typename T>
int blocks_per_sm(int dp, int rep) {
    if (rep > 8) return dp == 64 ? blocks_per_sm<T, 64, 2>() : dp == 128 ? blocks_per_sm<T, 128, 2>() : blocks_per_sm<T, 256, 2>();
    return dp == 64 ? blocks_per_sm<T, 64, 1>() : dp == 128 ? blocks_per_sm<T, 128, 1>() : blocks_per_sm<T, 256, 1>();
}

Decode4Plan decode4_plan(const ChronosPagedDecode4Args* a) {
    const ChronosPagedCache& c = a->cache;
    Decode4Plan d{};
    d.dp = fp4_columns(c.head_dim);
    const int rep = a->heads / c.kv_heads;
    d.parts = (rep + 15) / 16;
    const int per_sm = c.dtype == CHRONOS_DTYPE_FP32 ? blocks_per_sm<float>(d.dp, rep) : blocks_per_sm<__half>(d.dp, rep);
    const int limit = slot_limit(c, 0, false);
    d.max_vis = a->window > 0 ? static_cast<int>(std::min<int64_t>(limit, static_cast<int64_t>(a->window) + a->sinks + 32)) : limit;
    const int64_t blocks = (static_cast<int64_t>(d.max_vis) + kPdBlock - 1) / kPdBlock;
    const int64_t rows = static_cast<int64_t>(c.batch) * c.kv_heads * d.parts, room = static_cast<int64_t>(per_sm) * sm_count();
    const int64_t units = std::max<int64_t>(1, (blocks + kP4ListTiles - 1) / kP4ListTiles) * rows;
    d.grid = static_cast<int>(std::min<int64_t>({units, room, kPdMaxGrid}));
    int size = 1;
    while (size < 8 && size < blocks) size *= 2;
    while (size > 1 && rows * size > room) size /= 2;
    const int64_t most = size == 1 && 2 * rows > room ? kP4RowBlocks : 2 * rows * size > room ? kP4ClusterBlocksFull : kP4ClusterBlocks;
    d.cluster = blocks <= most * size ? size : 0;
    const size_t slots = d.cluster > 0 ? 0 : 2 * static_cast<size_t>(d.grid) * 16;
    d.o_part_ml = round_up(slots * d.dp * 4, 256);
    d.total = d.cluster > 0 ? 0 : d.o_part_ml + round_up(slots * 8, 256);
    return d;
}

template <typename T, int DP, int NT>
int launch_decode4(const PagedDecodeParams& p, const Decode4Plan& d, cudaStream_t st) {
    using S = Paged4<T, DP, NT>;
    if (d.cluster > 0) {
        auto kernel = paged_decode4_kernel<T, DP, NT, 1, true, false>;
        if (int rc = set_smem(kernel, S::kSmem)) return rc;
        CHRONOS_CUDA_CHECK(launch_cluster(kernel, dim3(static_cast<unsigned>(p.c.batch) * p.c.kv_heads * p.parts * d.cluster),
                                          dim3(kPdThreads), S::kSmem, st, d.cluster, p));
        return CHRONOS_OK;
    }
    auto kernel = paged_decode4_kernel<T, DP, NT, kP4ListTiles, false, false>;
    if (int rc = set_smem(kernel, S::kSmem)) return rc;
    CHRONOS_CUDA_CHECK(launch_kernel(kernel, dim3(p.grid), dim3(kPdThreads), S::kSmem, st, false, p));
    // (the list begins at 25 blocks of 64 slots a row: there are rows that may be cut)
    CHRONOS_CUDA_CHECK(launch_kernel(paged_join_kernel<T, kP4ListTiles * kPdBlock>, dim3(static_cast<unsigned>(p.join_blocks)), dim3(kPdJoinThreads), 0, st, true, p));
    return CHRONOS_OK;
}
template <typename T>
int launch_decode4(const PagedDecodeParams& p, const Decode4Plan& d, cudaStream_t st) {
    if (p.rep > 8)
        return d.dp == 64 ? launch_decode4<T, 64, 2>(p, d, st)
                          : d.dp == 128 ? launch_decode4<T, 128, 2>(p, d, st) : launch_decode4<T, 256, 2>(p, d, st);
    return d.dp == 64 ? launch_decode4<T, 64, 1>(p, d, st)
                      : d.dp == 128 ? launch_decode4<T, 128, 1>(p, d, st) : launch_decode4<T, 256, 1>(p, d, st);
}

}  // namespace
}  // namespace chronos

extern "C" size_t chronos_paged_decode4_workspace(const ChronosPagedDecode4Args* a) {
    using namespace chronos;
    g_last_error.clear();
    if (check_decode4(a)) return 0;
    return decode4_plan(a).total;
}

extern "C" int chronos_paged_decode4(const ChronosPagedDecode4Args* a, void* stream) {
    using namespace chronos;
    g_last_error.clear();
    const char* what = "chronos_paged_decode4";
    if (int rc = check_decode4(a)) return rc;
    if (a->cache.batch == 0) return CHRONOS_OK;
    if (int rc = check_cache_pointers(a->cache, what)) return rc;
    if (a->q == nullptr || a->out == nullptr) return fail(CHRONOS_ERR_INVALID_ARG, "%s: q and out are required", what);
    if (int rc = check_results(what, a->cache, true, a->cache.batch, a->heads, a->q, a->q_row_stride, a->q_head_stride, a->out, a->out_row_stride,
                               a->out_head_stride, a->lse, RowsOf{}, RowsOf{}))
        return rc;
    const Decode4Plan d = decode4_plan(a);
    const int64_t units = (static_cast<int64_t>(d.max_vis) / kPdBlock + 1) * a->cache.batch * a->cache.kv_heads * d.parts;
    if (units >= (1 << 30) || static_cast<int64_t>(a->cache.batch) * a->heads >= INT32_MAX / 8)
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: batch %d * heads * slots %d too large", what, a->cache.batch, d.max_vis);
    if (d.total > 0 && (a->workspace == nullptr || !aligned(a->workspace, 256) || a->workspace_bytes < d.total))
        return fail(CHRONOS_ERR_WORKSPACE_TOO_SMALL, "%s: workspace of %zu bytes, %zu (256-byte aligned) needed", what,
                    a->workspace == nullptr ? size_t{0} : a->workspace_bytes, d.total);
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    PagedDecodeParams p{};
    p.c = a->cache;
    p.heads = a->heads;
    p.rep = a->heads / a->cache.kv_heads;
    p.rows = 16;
    p.parts = d.parts;
    p.window = cut_window(a->window);
    p.sinks = a->window > 0 ? cut_window(a->sinks) : 0;
    p.max_slots = slot_limit(a->cache, 0, false);
    p.page_shift = page_shift_of(a->cache);
    p.cluster = d.cluster;
    p.sl2 = static_cast<float>(static_cast<double>(a->scale) * a->k_scale * 1.4426950408889634);
    p.v_scale = a->v_scale;
    p.q = a->q;
    p.q_row = a->q_row_stride;
    p.q_head = a->q_head_stride;
    p.out = a->out;
    p.out_row = a->out_row_stride;
    p.out_head = a->out_head_stride;
    p.lse = a->lse;
    p.grid = d.grid;
    p.part_stride = d.dp;
    p.part_o = reinterpret_cast<float*>(ws);
    p.part_ml = reinterpret_cast<float*>(ws + d.o_part_ml);
    p.join_blocks = a->cache.batch * a->heads;
    p.status = a->status;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (a->cache.dtype) {
        case CHRONOS_DTYPE_BF16: return launch_decode4<__nv_bfloat16>(p, d, st);
        case CHRONOS_DTYPE_FP16: return launch_decode4<__half>(p, d, st);
        default: return launch_decode4<float>(p, d, st);
    }
}
