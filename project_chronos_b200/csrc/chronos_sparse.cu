// chronos_sparse.cu — chronos_paged_sparse (include/chronos_paged4.h): argument checks,
// choice of kernel and launches.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "paged4.cuh"
#include "paged4_host.cuh"

namespace chronos {
namespace {

// Blocks per (token, group of query heads): a cluster, as long as the SMs hold all of them.
int sparse_cluster(const PagedDecodeParams& p, int64_t rows, int per_sm) {
    const int64_t blocks = (static_cast<int64_t>(p.topk) * p.c.page_size + kPdBlock - 1) / kPdBlock;
    const int64_t room = static_cast<int64_t>(per_sm) * sm_count();
    int size = 1;
    while (size < 8 && size < blocks) size *= 2;
    while (size > 1 && rows * size > room) size /= 2;
    return size;
}

template <typename K>
int launch_sparse_kernel(K kernel, int smem, int per_sm, PagedDecodeParams p, int64_t tokens, cudaStream_t st) {
    const int64_t rows = tokens * p.c.kv_heads * p.parts;
    p.cluster = sparse_cluster(p, rows, per_sm);
    if (int rc = set_smem(kernel, smem)) return rc;
    CHRONOS_CUDA_CHECK(launch_cluster(kernel, dim3(static_cast<unsigned>(rows * p.cluster)), dim3(kPdThreads), smem, st, p.cluster, p));
    return CHRONOS_OK;
}

template <typename T, int DP, int NT>
int launch_sparse4(const PagedDecodeParams& p, int64_t tokens, cudaStream_t st) {
    using S = Paged4<T, DP, NT>;
    return launch_sparse_kernel(paged_decode4_kernel<T, DP, NT, 1, true, true>, S::kSmem, S::kBlocksPerSm, p, tokens, st);
}
template <typename T>
int launch_sparse4(const PagedDecodeParams& p, int dp, int64_t tokens, cudaStream_t st) {
    if (p.rep > 8)
        return dp == 64 ? launch_sparse4<T, 64, 2>(p, tokens, st)
                        : dp == 128 ? launch_sparse4<T, 128, 2>(p, tokens, st) : launch_sparse4<T, 256, 2>(p, tokens, st);
    return dp == 64 ? launch_sparse4<T, 64, 1>(p, tokens, st)
                    : dp == 128 ? launch_sparse4<T, 128, 1>(p, tokens, st) : launch_sparse4<T, 256, 1>(p, tokens, st);
}

template <typename T, int DP, int NT>
int launch_sparse_mma(const PagedDecodeParams& p, int64_t tokens, cudaStream_t st) {
    using S = PagedMma<T, DP>;
    auto kernel = p.c.page_size % kPdTile == 0 ? paged_decode_mma_kernel<T, DP, NT, true, true, true>
                                               : paged_decode_mma_kernel<T, DP, NT, false, true, true>;
    return launch_sparse_kernel(kernel, S::kSmem, S::kBlocksPerSm, p, tokens, st);
}
template <typename T, int NT>
int launch_sparse_mma(const PagedDecodeParams& p, int dp, int64_t tokens, cudaStream_t st) {
    if (dp == 64) return launch_sparse_mma<T, 64, NT>(p, tokens, st);
    if constexpr (sizeof(T) == 2)
        if (dp == 256) return launch_sparse_mma<T, 256, NT>(p, tokens, st);
    return launch_sparse_mma<T, 128, NT>(p, tokens, st);
}

template <typename T>
int launch_sparse(PagedDecodeParams p, int dp, bool packed, int64_t tokens, cudaStream_t st) {
    if (packed) {
        p.rows = 16;
        p.parts = (p.rep + 15) / 16;
        return launch_sparse4<T>(p, dp, tokens, st);
    }
    const ChronosPagedCache& c = p.c;
    const int64_t n = 16 / static_cast<int64_t>(sizeof(T));
    if ((sizeof(T) == 2 || c.head_dim <= 128) && c.head_dim % n == 0 && copies16(c) && aligned(p.q, 8) && aligned(p.out, 8) &&
        multiples(2, {p.q_row, p.q_head, p.out_row, p.out_head})) {
        p.rows = sizeof(T) == 2 ? 16 : 8;
        p.parts = (p.rep + p.rows - 1) / p.rows;
        if constexpr (sizeof(T) == 2)
            if (p.rep > 8) return launch_sparse_mma<T, 2>(p, dp, tokens, st);
        return launch_sparse_mma<T, 1>(p, dp, tokens, st);
    }
    p.rows = kPdSimtRows;
    p.parts = (p.rep + p.rows - 1) / p.rows;
    const size_t four = 4 * sizeof(T);
    const bool vec = c.head_dim % 4 == 0 && aligned(c.k_pages, four) && aligned(c.v_pages, four) &&
                     multiples(4, {c.k_page_stride, c.k_slot_stride, c.k_head_stride, c.v_page_stride, c.v_slot_stride, c.v_head_stride});
    CHRONOS_CUDA_CHECK(launch_kernel(vec ? paged_decode_simt_kernel<T, true, true> : paged_decode_simt_kernel<T, false, true>,
                                     dim3(static_cast<unsigned>(tokens * c.kv_heads * p.parts)), dim3(kPdThreads), 0, st, false, p));
    return CHRONOS_OK;
}

}  // namespace
}  // namespace chronos

extern "C" int chronos_paged_sparse(const ChronosPagedSparseArgs* a, void* stream) {
    using namespace chronos;
    g_last_error.clear();
    const char* what = "chronos_paged_sparse";
    if (a == nullptr) return fail(CHRONOS_ERR_INVALID_ARG, "%s: args is NULL", what);
    if (int rc = check_cache(a->cache, what)) return rc;
    if (int rc = check_heads(a->heads, a->cache, what)) return rc;
    if (int rc = check_positive("scale", a->scale, what)) return rc;
    if (int rc = check_tokens(a->num_tokens, a->cu_seqlens, a->cache, what)) return rc;
    // a block's places are 32-bit numbers, and so are the blocks of a launch
    if (a->topk < 0 || static_cast<int64_t>(a->topk) * a->cache.page_size >= (1 << 30))
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: topk %d pages of %d slots", what, a->topk, a->cache.page_size);
    if (a->num_tokens * a->heads >= INT32_MAX / 8)
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: %lld tokens of %d heads", what, static_cast<long long>(a->num_tokens), a->heads);
    if (a->packed) {
        if (int rc = check_packed(a->cache, a->k_scale, a->v_scale, what)) return rc;
        if (int rc = check_scores(a->scale, a->k_scale, what)) return rc;
    }
    if (a->cache.batch == 0 || a->num_tokens == 0) return CHRONOS_OK;
    if (int rc = check_cache_pointers(a->cache, what)) return rc;
    if (a->q == nullptr || a->out == nullptr || (a->topk > 0 && a->pages == nullptr))
        return fail(CHRONOS_ERR_INVALID_ARG, "%s: q, out and pages are required", what);
    if (int rc = check_results(what, a->cache, a->packed != 0, a->num_tokens, a->heads, a->q, a->q_row_stride, a->q_head_stride, a->out, a->out_row_stride,
                               a->out_head_stride, a->lse, array_of(a->pages, a->num_tokens * a->cache.kv_heads * a->topk, 4),
                               array_of(a->cu_seqlens, a->cache.batch + int64_t{1}, 4)))
        return rc;
    PagedDecodeParams p{};
    p.c = a->cache;
    p.heads = a->heads;
    p.rep = a->heads / a->cache.kv_heads;
    p.max_slots = slot_limit(a->cache, 0, false);
    p.page_shift = page_shift_of(a->cache);
    p.sl2 = static_cast<float>(static_cast<double>(a->scale) * (a->packed ? a->k_scale : 1.0f) * 1.4426950408889634);
    p.v_scale = a->v_scale;
    p.q = a->q;
    p.q_row = a->q_row_stride;
    p.q_head = a->q_head_stride;
    p.out = a->out;
    p.out_row = a->out_row_stride;
    p.out_head = a->out_head_stride;
    p.lse = a->lse;
    p.sel = a->pages;
    p.topk = a->topk;
    p.cu = a->cu_seqlens;
    p.status = a->status;
    const int dp = fp4_columns(a->cache.head_dim);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (a->cache.dtype) {
        case CHRONOS_DTYPE_BF16: return launch_sparse<__nv_bfloat16>(p, dp, a->packed != 0, a->num_tokens, st);
        case CHRONOS_DTYPE_FP16: return launch_sparse<__half>(p, dp, a->packed != 0, a->num_tokens, st);
        default: return launch_sparse<float>(p, dp, a->packed != 0, a->num_tokens, st);
    }
}
