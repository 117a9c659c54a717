// window_attention.cuh — causal attention of a packed batch of prompts, with an
// optional sliding window and first tokens that stay visible
// (include/chronos_paged.h, chronos_window_attention).
//
// Row t of a sequence sees the keys j <= t with window == 0, j > t - window or
// j < sinks.  One pass over the visible key tiles with a running maximum and
// sum: out = sum 2^(x_j - m) v_j / sum 2^(x_j - m), x_j = scale log2(e) q.k_j.
#pragma once

#include <cooperative_groups.h>

#include "chronos_paged.h"
#include "common.cuh"
#include "paged.cuh"

namespace chronos {

struct WindowParams {
    int batch, heads, kv_heads, rep, dim, window, sinks;
    float sl2;
    int64_t num_q, num_k;
    const void* q;
    const void* k;
    const void* v;
    void* out;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head;
    const int32_t* cu_q;
    const int32_t* cu_k;
    float* lse;
    int32_t* status;
};

// The row tile a block works on: `rows` queries of sequence b from its query m0 on.
struct WindowTile {
    int b, m0;
    int q0, k0;         // first rows of the sequence in q and k
    int lq, lk;
};

// Report offsets that do not ascend or leave q or k: the last block does, for which offsets
// that ascend leave no tile.  A function of its own, called where a block has no tile: inlined
// at the start it made the tensor-core path spill (32 prompts of 512 39.1 -> 42.6 us).
__device__ __noinline__ void window_check_offsets(const WindowParams& p) {
    for (int b = threadIdx.x; b < p.batch; b += blockDim.x) {
        const int q0 = p.cu_q[b], q1 = p.cu_q[b + 1], k0 = p.cu_k[b], k1 = p.cu_k[b + 1];
        if (q0 < 0 || q1 < q0 || q1 > p.num_q || k0 < 0 || k1 < k0 || k1 > p.num_k) report_status(p.status, CHRONOS_ERR_INVALID_ARG);
    }
}

// Tile number `x` of all sequences' tiles of `rows` queries (a whole warp calls
// this; false behind the last one).  Within a sequence the last tile comes
// first: under a causal mask it has the most keys.  A sequence whose offsets
// leave q or k, or do not ascend, is left out: no access leaves them.  (Offsets
// that descend can give more tiles than there are blocks: they are reported here, too.)
__device__ __forceinline__ bool window_tile(const WindowParams& p, int64_t x, int rows, int lane, WindowTile& t) {
    int64_t before = 0;
    for (int base = 0; base < p.batch; base += 32) {
        const int b = base + lane;
        int64_t n = 0;
        if (b < p.batch) {
            const int lq = p.cu_q[b + 1] - p.cu_q[b];
            if (lq < 0) report_status(p.status, CHRONOS_ERR_INVALID_ARG);
            n = (max(0, min(lq, static_cast<int>(p.num_q))) + rows - 1) / rows;
        }
        int64_t inc = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t u = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += u;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, before + inc > x);
        if (past) {
            const int l = __ffs(past) - 1;
            const int64_t start = before + __shfl_sync(0xffffffffu, inc - n, l);
            const int64_t cnt = __shfl_sync(0xffffffffu, n, l);
            t.b = base + l;
            t.q0 = p.cu_q[t.b];
            t.k0 = p.cu_k[t.b];
            t.lq = p.cu_q[t.b + 1] - p.cu_q[t.b];
            t.lk = p.cu_k[t.b + 1] - p.cu_k[t.b];
            if (t.q0 < 0 || static_cast<int64_t>(t.q0) + t.lq > p.num_q || t.k0 < 0 || t.lk < 0 ||
                static_cast<int64_t>(t.k0) + t.lk > p.num_k)
                return false;
            t.m0 = static_cast<int>((start + cnt - 1 - x) * rows);
            return true;
        }
        before += __shfl_sync(0xffffffffu, inc, 31);
    }
    return false;
}

// ---------------------------------------------------------------------------
// general path: fp32 products (fp32 layers; head dimensions or strides the
// tensor-core path cannot take).  64 queries x 64 keys per step, 256 threads as
// 16 x 16: a thread forms 4 x 4 scores and 4 rows x D/16 columns of the output from
// tiles in shared memory.  Bound by the fp32 pipes and the tiles' loads, which nothing
// overlaps: 22 TFLOP/s for 8 fp32 prompts of 512 (8 / 2 heads of 128), 33 for 4 of 1024
// on 1024 earlier keys (32 / 8 heads of 64).
// ---------------------------------------------------------------------------
constexpr int kWsThreads = 256;
constexpr int kWsRows = 64;
constexpr int kWsKeys = 64;

__host__ __device__ constexpr int window_simt_dim(int dim) { return (dim + 63) / 64 * 64; }
__host__ __device__ constexpr int window_simt_smem(int dim) {
    return (kWsRows + 2 * kWsKeys) * (window_simt_dim(dim) + 4) * 4 + kWsRows * (kWsKeys + 4) * 4;
}

// NC: groups of 64 output columns (head_dim <= 64 * NC); VEC: rows of 4 elements on
// boundaries of 4.
template <typename T, int NC, bool VEC>
__global__ void __launch_bounds__(kWsThreads) window_simt_kernel(const __grid_constant__ WindowParams p) {
    constexpr int DP = 64 * NC, LD = DP + 4;      // row stride: float4 reads of 16 rows on different banks
    extern __shared__ __align__(16) float wsm[];
    float* s_q = wsm;
    float* s_k = s_q + kWsRows * LD;
    float* s_v = s_k + kWsKeys * LD;
    float* s_p = s_v + kWsKeys * LD;              // [64][68]
    constexpr int LP = kWsKeys + 4;
    const int lane = threadIdx.x & 31;
    const int head = blockIdx.x % p.heads, g = head / p.rep;
    WindowTile t;
    if (!window_tile(p, blockIdx.x / p.heads, kWsRows, lane, t)) {
        if (blockIdx.x == gridDim.x - 1) window_check_offsets(p);
        return;
    }
    const int rows = min(kWsRows, t.lq - t.m0);
    const int t0 = t.lk - t.lq + t.m0;            // position of the first row
    const int hi = min(t.lk, t0 + rows);          // keys [lo, hi) and the first ones
    const int lo = p.window > 0 ? max(0, t0 - p.window + 1) : 0;
    const int ns = p.window > 0 ? (max(0, min(p.sinks, hi)) + kWsKeys - 1) / kWsKeys : 0;
    const int w0 = max(ns * kWsKeys, lo);
    const int nt = ns + (hi > w0 ? (hi - w0 + kWsKeys - 1) / kWsKeys : 0);
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;

    auto stage = [&](float* dst, const T* src, int64_t row_stride, int n) {
#pragma unroll 4
        for (int i = threadIdx.x; i < kWsRows * (DP / 4); i += kWsThreads) {
            const int r = i / (DP / 4), d = i % (DP / 4) * 4;
            float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (r < n && d < p.dim) load4<T, VEC>(src + r * row_stride, d, p.dim, v);
            *reinterpret_cast<float4*>(dst + r * LD + d) = make_float4(v[0], v[1], v[2], v[3]);
        }
    };
    stage(s_q, static_cast<const T*>(p.q) + static_cast<int64_t>(t.q0 + t.m0) * p.q_row + head * p.q_head, p.q_row, rows);
    float m[4], l[4], o[4][NC * 4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.0f;
#pragma unroll
        for (int c = 0; c < NC * 4; ++c) o[r][c] = 0.0f;
    }
    for (int it = 0; it < nt; ++it) {
        const int j0 = it < ns ? it * kWsKeys : w0 + (it - ns) * kWsKeys;
        const int n = min(kWsKeys, t.lk - j0);
        __syncthreads();
        stage(s_k, static_cast<const T*>(p.k) + static_cast<int64_t>(t.k0 + j0) * p.k_row + g * p.k_head, p.k_row, n);
        stage(s_v, static_cast<const T*>(p.v) + static_cast<int64_t>(t.k0 + j0) * p.v_row + g * p.v_head, p.v_row, n);
        __syncthreads();
        float s[4][4];
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < 4; ++c) s[r][c] = 0.0f;
#pragma unroll 4
        for (int d = 0; d < DP; d += 4) {
            float4 a[4], b[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) a[r] = *reinterpret_cast<const float4*>(s_q + (ty * 4 + r) * LD + d);
#pragma unroll
            for (int c = 0; c < 4; ++c) b[c] = *reinterpret_cast<const float4*>(s_k + (tx + 16 * c) * LD + d);
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    s[r][c] = fmaf(a[r].x, b[c].x, fmaf(a[r].y, b[c].y, fmaf(a[r].z, b[c].z, fmaf(a[r].w, b[c].w, s[r][c]))));
        }
        bool hidden = false;   // some weight of this thread's rows is masked
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int tr = t0 + ty * 4 + r;
            float n0 = -INFINITY;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int j = j0 + tx + 16 * c;
                const bool on = j <= tr && j < t.lk && (p.window == 0 || j > tr - p.window || j < p.sinks);
                s[r][c] = on ? s[r][c] * p.sl2 : -INFINITY;
                n0 = fmaxf(n0, s[r][c]);
            }
#pragma unroll
            for (int x = 1; x < 16; x <<= 1) n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, x));
            n0 = fmaxf(n0, m[r]);
            const float u = n0 == -INFINITY ? 0.0f : n0;
            const float c0 = exp2_fast(m[r] - u);
            m[r] = n0;
            float sum = 0.0f;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float e = exp2_fast(s[r][c] - u);
                sum += e;
                s_p[(ty * 4 + r) * LP + tx + 16 * c] = e;
            }
            l[r] = l[r] * c0 + sum;
#pragma unroll
            for (int c = 0; c < NC * 4; ++c) o[r][c] *= c0;
            const bool full = j0 + kWsKeys - 1 <= tr && (p.window == 0 || j0 > tr - p.window);
            hidden |= !full;
        }
        __syncwarp();   // a row's 16 threads lie in one warp
        // masked keys add nothing, even where their values are not finite
        if (__any_sync(0xffffffffu, hidden)) {
            for (int j = 0; j < kWsKeys; ++j) {
                float pr[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) pr[r] = s_p[(ty * 4 + r) * LP + j];
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const float4 v = *reinterpret_cast<const float4*>(s_v + j * LD + c * 64 + tx * 4);
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (pr[r] != 0.0f) {
                            o[r][4 * c] = fmaf(pr[r], v.x, o[r][4 * c]);
                            o[r][4 * c + 1] = fmaf(pr[r], v.y, o[r][4 * c + 1]);
                            o[r][4 * c + 2] = fmaf(pr[r], v.z, o[r][4 * c + 2]);
                            o[r][4 * c + 3] = fmaf(pr[r], v.w, o[r][4 * c + 3]);
                        }
                }
            }
        } else {
#pragma unroll 2
            for (int j = 0; j < kWsKeys; j += 4) {
                float4 pr[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) pr[r] = *reinterpret_cast<const float4*>(s_p + (ty * 4 + r) * LP + j);
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int c = 0; c < NC; ++c) {
                        const float4 v = *reinterpret_cast<const float4*>(s_v + (j + e) * LD + c * 64 + tx * 4);
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float x = e == 0 ? pr[r].x : e == 1 ? pr[r].y : e == 2 ? pr[r].z : pr[r].w;
                            o[r][4 * c] = fmaf(x, v.x, o[r][4 * c]);
                            o[r][4 * c + 1] = fmaf(x, v.y, o[r][4 * c + 1]);
                            o[r][4 * c + 2] = fmaf(x, v.z, o[r][4 * c + 2]);
                            o[r][4 * c + 3] = fmaf(x, v.w, o[r][4 * c + 3]);
                        }
                    }
            }
        }
        __syncwarp();
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
#pragma unroll
        for (int x = 1; x < 16; x <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], x);
        const int row = ty * 4 + r;
        if (row >= rows) continue;
        const float inv = l[r] > 0.0f ? 1.0f / l[r] : l[r];   // 0 for a row that saw nothing; NaN stays
        T* out = static_cast<T*>(p.out) + static_cast<int64_t>(t.q0 + t.m0 + row) * p.o_row + head * p.o_head;
#pragma unroll
        for (int c = 0; c < NC * 4; ++c) {
            const int d = (c >> 2) * 64 + tx * 4 + (c & 3);
            if (d < p.dim) out[d] = from_f32<T>(o[r][c] * inv);
        }
        if (tx == 0 && p.lse != nullptr)
            p.lse[static_cast<int64_t>(t.q0 + t.m0 + row) * p.heads + head] = l[r] != 0.0f ? (m[r] + log2f(l[r])) * kLn2 : -INFINITY;
    }
}

// ---------------------------------------------------------------------------
// tensor-core path: bf16 / fp16, head_dim a multiple of 8 up to 128
// ---------------------------------------------------------------------------
// Bound: the tensor cores (4 D flops per visible pair and head) and, as closely,
// the 16 exponentials a cycle of an SM's special-function units.  A block holds
// 256 query rows as two tiles of 128, each with a warpgroup of its own, so one
// tile's exponentials run while the other's products do.  Accumulators live in
// TMEM: scores S (128 columns per tile), over which the weights P are written in
// the layer type as the first operand of the second product, and the output O
// (DP columns per tile).  A row belongs to one thread, so its maximum and sum
// need no exchange.  With several query heads per kv head (a power of two up to
// 16) the 256 rows are 256 / rep tokens times rep heads: keys and values are
// loaded once for all of them, and a window has fewer tiles with hidden pairs.
//
//   warps 0-3, 4-7   softmax of tile 0 / 1, rescaling of O, output
//   warp 8           TMA loads of Q, K, V (128-byte swizzle, no multicast)
//   warp 9           tcgen05.mma issue, TMEM allocation
//   warps 10, 11     V tiles with hidden keys: rows behind the sequence become
//                    zero (0 * NaN would reach every row), and so do rows that
//                    are not finite, in which case the block computes its rows
//                    again pair by pair at the end (right, not fast: one infinity near
//                    the end of 8192 keys takes 4 x 2048 queries from 0.77 to 141 ms)
//
// Measured, 32 / 8 heads of 128: 4 x 1793 to 2048 queries on up to 8192 keys in bf16 770 to
// 788 us in long runs, which the power cap holds (1020 TFLOP/s, 73 % of the library product's
// sustained rate), 673 us in short ones (71 % of its burst rate); one prompt of 8191 under a
// window of 1024 with 4 first tokens in fp16 203 to 209 us.  A tile's chain bounds it: maximum and exponentials of its 128 x 128 scores about 2000
// cycles, then both products 1400 (1040 by themselves), and two such chains per SM
// overlap to 3500 cycles per 128 keys where either unit alone needs 2050.
//
// Few row tiles and many keys (SPLIT): a thread-block cluster shares a row tile, block r
// of it the r-th part of the key tiles; every block leaves its rows' (m, l, O) in its
// shared memory and joins its share of the rows through distributed shared memory.
//
// O is rescaled only when a row's maximum grew by more than 2^8 in weight: until
// then weights are taken against the older maximum, at most 256 times too large,
// which the fp32 sums and both 16-bit formats hold without loss (fp16 weights also
// carry 2^7, see WeightLift).
constexpr int kWtThreads = 384;
constexpr int kWtKeys = 128;
constexpr float kWtRescaleLog2 = 8.0f;
constexpr uint64_t kWtLimitNs = 2000000000ull;

template <int DP>
struct WindowTc {
    static constexpr int kHalves = DP / 64;
    static constexpr int kTileBytes = 128 * DP * 2;         // 128 rows of K, V or Q
    static constexpr int kStages = DP == 64 ? 3 : 2;        // of K and of V
    static constexpr int kBarriers = 2 + 5 * kStages + 2 + 4 + 2 + 1;
    static constexpr int kSmem = 1024 + (2 + 2 * kStages) * kTileBytes + 8 * kBarriers + 32;
    static constexpr int kSplitSmem = kSmem + 256 * 8;      // and (m, l) of every row
    static_assert(256 * DP * 4 <= (2 + kStages) * kTileBytes, "fp32 rows fit the buffers of Q and K");
    static constexpr int kSCol = 0, kOCol = 256;            // S of tile w at 128 w, O at 256 + DP w
};

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
            smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2,
                                            int c3) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::
            "r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
        : "memory");
}

// D[tmem] (+)= A[tmem] * B[smem desc], kind::f16.
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
        "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Descriptor of an operand stored along its N dimension (128-byte swizzle: rows
// of 64 elements along N, one row per k, atoms of 8 rows = 1024 bytes): leading
// byte offset between 64-element groups of N, stride byte offset between groups
// of 8 k.
__device__ __forceinline__ uint64_t sdesc_mn_sw128(uint32_t smem_addr, uint32_t group_bytes) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((smem_addr >> 4) & 0x3FFFu);
    d |= static_cast<uint64_t>((group_bytes >> 4) & 0x3FFFu) << 16;
    d |= static_cast<uint64_t>(1024u >> 4) << 32;
    d |= static_cast<uint64_t>(1u) << 46;
    d |= static_cast<uint64_t>(2u) << 61;
    return d;
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const float* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]),
        "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tmem_st16u(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}

// 32 bytes in one store (a whole DRAM sector; 32-byte aligned).
__device__ __forceinline__ void store32(void* p, const uint32_t (&x)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(x[0]), "r"(x[1]), "r"(x[2]),
                 "r"(x[3]), "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7])
                 : "memory");
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(p));
    return p != 0;
}

// Two fp32 operations per instruction, and the largest of three (NaN if one is).
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<uint64_t&>(d))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t&>(d))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// One row pair by pair (a whole warp): only visible keys are touched.
template <typename T>
__device__ __noinline__ void window_row_exact(const WindowParams& p, const WindowTile& t, int token, int head, int lane) {
    const int tr = t.lk - t.lq + token;
    const T* q = static_cast<const T*>(p.q) + static_cast<int64_t>(t.q0 + token) * p.q_row + head * p.q_head;
    const T* k = static_cast<const T*>(p.k) + static_cast<int64_t>(t.k0) * p.k_row + (head / p.rep) * p.k_head;
    const T* v = static_cast<const T*>(p.v) + static_cast<int64_t>(t.k0) * p.v_row + (head / p.rep) * p.v_head;
    float m = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const int lo = p.window > 0 ? max(0, tr - p.window + 1) : 0;
    const int first = min(p.sinks, lo);
    for (int i = 0; i < first + tr + 1 - lo; ++i) {
        const int64_t j = i < first ? i : lo + i - first;
        float x = 0.0f;
        for (int d = lane; d < p.dim; d += 32) x = fmaf(to_f32<T>(q[d]), to_f32<T>(k[j * p.k_row + d]), x);
        x = warp_sum(x) * p.sl2;
        const float n = fmaxf(m, x), u = n == -INFINITY ? 0.0f : n;
        const float c = exp2_fast(m - u), e = exp2_fast(x - u);
        m = n;
        l = l * c + e;
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            const int d = lane + 32 * a;
            if (d < p.dim) o[a] = fmaf(e, to_f32<T>(v[j * p.v_row + d]), o[a] * c);
        }
    }
    const float inv = l > 0.0f ? 1.0f / l : l;
    T* out = static_cast<T*>(p.out) + static_cast<int64_t>(t.q0 + token) * p.o_row + head * p.o_head;
#pragma unroll
    for (int a = 0; a < 4; ++a)
        if (lane + 32 * a < p.dim) out[lane + 32 * a] = from_f32<T>(o[a] * inv);
    if (lane == 0 && p.lse != nullptr)
        p.lse[static_cast<int64_t>(t.q0 + token) * p.heads + head] = l != 0.0f ? (m + log2f(l)) * kLn2 : -INFINITY;
}

template <typename T>
__device__ __forceinline__ bool any_not_finite(const uint4& u) {
    constexpr uint32_t E = sizeof(T) == 2 && AbFormat<T>::value == 1 ? 0x7f80u : 0x7c00u;
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) bad |= (w[i] & E) == E || (w[i] & (E << 16)) == (E << 16);
    return bad;
}

// The rows of a split row tile (256, fp32 and swizzled in every block's `part`, (m, l) in
// `ml`) that fall to this block, eight warps.  Lane x holds what the x-th of the warp's rows
// needs of every part; then four rows at a time are read and joined, in the order of the
// keys.  A function of its own: inlined, its registers made the main loop spill.
template <typename T, int DP>
__device__ __noinline__ void window_cluster_join(const WindowParams& p, const WindowTile& t, float* s_part, float* s_ml,
                                                 const int* not_finite, int hg, int rows, int rp_log2, int rank,
                                                 int splits, int warp, int lane) {
    cooperative_groups::cluster_group cl = cooperative_groups::this_cluster();
    constexpr int NV = DP / 32, R = 4;
    bool again = false;
    for (int q = 0; q < splits; ++q) again |= *static_cast<const volatile int*>(cl.map_shared_rank(not_finite, q)) != 0;
    auto row_of = [&](int x) { return (x * splits + rank) * 8 + warp; };
    const int n = 32 / splits;
    float c[8], M = -INFINITY, L = 0.0f;
    const int mine = min(row_of(lane), 255);
#pragma unroll
    for (int q = 0; q < 8; ++q) {
        c[q] = q < splits ? cl.map_shared_rank(s_ml, q)[mine * 2] : -INFINITY;
        M = max3(M, c[q], M);
    }
    const float u = M == -INFINITY ? 0.0f : M;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
        c[q] = exp2_fast(c[q] - u);
        if (q < splits) L += cl.map_shared_rank(s_ml, q)[mine * 2 + 1] * c[q];
    }
    const float inv = L > 0.0f ? 1.0f / L : L, lg = L != 0.0f ? (u + log2f(L)) * kLn2 : -INFINITY;
    for (int x0 = 0; x0 < n && (row_of(x0) >> rp_log2) < rows; x0 += R) {
        float acc[R][NV];
#pragma unroll
        for (int y = 0; y < R; ++y)
#pragma unroll
            for (int e = 0; e < NV; ++e) acc[y][e] = 0.0f;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            if (q >= splits) break;
            const float* part = cl.map_shared_rank(s_part, q);
#pragma unroll
            for (int y = 0; y < R; ++y) {
                const int row = row_of(x0 + y);
                const float w = __shfl_sync(0xffffffffu, c[q], x0 + y);
#pragma unroll
                for (int e = 0; e < NV; ++e) {
                    const int d = lane + 32 * e;
                    acc[y][e] = fmaf(w, part[row * DP + ((d / 4) ^ (row & 7)) * 4 + (d & 3)], acc[y][e]);
                }
            }
        }
#pragma unroll
        for (int y = 0; y < R; ++y) {
            const int row = row_of(x0 + y);
            const int token = row >> rp_log2, head = (hg << rp_log2) + (row & ((1 << rp_log2) - 1));
            const float f = __shfl_sync(0xffffffffu, inv, x0 + y), e0 = __shfl_sync(0xffffffffu, lg, x0 + y);
            if (token >= rows) continue;
            if (again) {
                window_row_exact<T>(p, t, t.m0 + token, head, lane);
                continue;
            }
            const int64_t qrow = t.q0 + t.m0 + token;
            T* out = static_cast<T*>(p.out) + qrow * p.o_row + head * p.o_head;
#pragma unroll
            for (int e = 0; e < NV; ++e)
                if (lane + 32 * e < p.dim) out[lane + 32 * e] = from_f32<T>(acc[y][e] * f);
            if (lane == 0 && p.lse != nullptr) p.lse[qrow * p.heads + head] = e0;
        }
    }
}

// rp: heads per row group (1 << rp_log2), the query heads of one kv head or 1.
template <typename T, int DP, bool SPLIT>
__global__ void __launch_bounds__(kWtThreads, 1) window_tc_kernel(const __grid_constant__ WindowParams p,
                                                                  const __grid_constant__ CUtensorMap tm_q,
                                                                  const __grid_constant__ CUtensorMap tm_k,
                                                                  const __grid_constant__ CUtensorMap tm_v, int rp_log2,
                                                                  int groups, int splits) {
    using C = WindowTc<DP>;
    constexpr int NS = C::kStages;
    extern __shared__ uint8_t dyn[];
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    if (warp == 8 && lane == 0) {
        prefetch_tmap(&tm_q);
        prefetch_tmap(&tm_k);
        prefetch_tmap(&tm_v);
    }
    const int block = SPLIT ? static_cast<int>(blockIdx.x) / splits : static_cast<int>(blockIdx.x);
    const int hg = block % groups;
    const int tokens = 256 >> rp_log2;            // tokens of the block
    WindowTile t;
    if (!window_tile(p, block / groups, tokens, lane, t)) {
        if (blockIdx.x == gridDim.x - 1) window_check_offsets(p);
        return;
    }
    const int rows = min(tokens, t.lq - t.m0);
    const int t0 = t.lk - t.lq + t.m0;            // position of the first token
    const int hi = min(t.lk, t0 + rows);          // keys [lo, hi) and the first ones
    const int lo = p.window > 0 ? max(0, t0 - p.window + 1) : 0;
    const int ns = p.window > 0 ? (max(0, min(p.sinks, hi)) + kWtKeys - 1) / kWtKeys : 0;
    const int w0 = max(ns * kWtKeys, lo);
    const int all = ns + (hi > w0 ? (hi - w0 + kWtKeys - 1) / kWtKeys : 0);
    // this block's key tiles
    const int rank = SPLIT ? static_cast<int>(blockIdx.x) % splits : 0;
    const int i0 = SPLIT ? all * rank / splits : 0, nt = SPLIT ? all * (rank + 1) / splits - i0 : all;
    auto tile_base = [&](int i) {
        if (SPLIT) i += i0;
        return i < ns ? i * kWtKeys : w0 + (i - ns) * kWtKeys;
    };

    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~uintptr_t{1023});
    uint8_t* s_q = smem;
    uint8_t* s_k = s_q + 2 * C::kTileBytes;
    uint8_t* s_v = s_k + NS * C::kTileBytes;
    uint64_t* bars = reinterpret_cast<uint64_t*>(s_v + NS * C::kTileBytes);
    uint64_t* q_full = bars;
    uint64_t* k_full = q_full + 2;                // q_full [2]: by tile
    uint64_t* k_empty = k_full + NS;
    uint64_t* v_full = k_empty + NS;
    uint64_t* v_ok = v_full + NS;
    uint64_t* v_empty = v_ok + NS;
    uint64_t* s_full = v_empty + NS;              // [2]
    uint64_t* p_ready = s_full + 2;               // [2][2]: tile, half of its keys
    uint64_t* o_done = p_ready + 4;               // [2]
    uint64_t* drained = o_done + 2;
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(drained + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(s_tmem + 1);
    volatile int* not_finite = abort_flag + 1;
    float* s_ml = reinterpret_cast<float*>(bars + C::kBarriers + 4);   // [256][2], SPLIT only
    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        mbar_init(q_full + 1, 1);
        for (int i = 0; i < NS; ++i) {
            mbar_init(k_full + i, 1);
            mbar_init(k_empty + i, 1);
            mbar_init(v_full + i, 1);
            mbar_init(v_ok + i, 2);
            mbar_init(v_empty + i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(s_full + i, 1);
            mbar_init(p_ready + 2 * i, 4);
            mbar_init(p_ready + 2 * i + 1, 4);
            mbar_init(o_done + i, 1);
        }
        mbar_init(drained, 1);
        *abort_flag = 0;
        *not_finite = 0;
        fence_mbar_init();
    }
    if (warp == 9) {
        tmem_alloc(s_tmem, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        // the timer of the bounded wait costs more than most of these waits: look at it late
        for (int i = 0; i < 256; ++i)
            if (mbar_try_wait(bar, parity)) return true;
        if (mbar_wait_bounded(bar, parity, kWtLimitNs, const_cast<volatile int*>(abort_flag))) return true;
        *abort_flag = 1;
        report_status(p.status, CHRONOS_ERR_PIPELINE_TIMEOUT);
        return false;
    };

    if (warp >= 8) {
        // the block launched with 384 * 168 registers: 256 * 200 + 128 * 104 (the issuing warp
        // spills with fewer: 72 cost 2 %, 56 cost 7 %)
        asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
        if (warp == 8 && lane == 0 && nt > 0) {
            // ------------------------------ loads ------------------------------
            const int g = groups == p.kv_heads ? hg : hg / p.rep;
            auto load_q = [&](int w) {
                mbar_arrive_expect_tx(q_full + w, C::kTileBytes);
                for (int h = 0; h < C::kHalves; ++h)
                    tma_load_4d(s_q + w * C::kTileBytes + h * 16384, &tm_q, q_full + w, h * 64, 0, hg,
                                t.q0 + t.m0 + w * (128 >> rp_log2));
            };
            load_q(0);
            int i = 0;
            for (; i < nt; ++i) {
                const int st = i % NS;
                const uint32_t ph = (i / NS) & 1;
                const int row = t.k0 + tile_base(i);
                if (!wait(k_empty + st, ph ^ 1u)) break;
                mbar_arrive_expect_tx(k_full + st, C::kTileBytes);
                for (int h = 0; h < C::kHalves; ++h)
                    tma_load_3d(s_k + st * C::kTileBytes + h * 16384, &tm_k, k_full + st, h * 64, g, row);
                if (i == 0) load_q(1);
                if (!wait(v_empty + st, ph ^ 1u)) {
                    ++i;   // this tile's K copy is in flight (its V barrier is not waited for below)
                    break;
                }
                mbar_arrive_expect_tx(v_full + st, C::kTileBytes);
                for (int h = 0; h < C::kHalves; ++h)
                    tma_load_3d(s_v + st * C::kTileBytes + h * 16384, &tm_v, v_full + st, h * 64, g, row);
            }
            if (*abort_flag) {
                // the copies in flight land before the block's shared memory is given up
                volatile int go = 0;
                mbar_wait_bounded(q_full, 0, kWtLimitNs, &go);
                mbar_wait_bounded(q_full + 1, 0, kWtLimitNs, &go);
                for (int j = max(0, i - NS); j < i; ++j) {
                    mbar_wait_bounded(k_full + j % NS, (j / NS) & 1, kWtLimitNs, &go);
                    mbar_wait_bounded(v_full + j % NS, (j / NS) & 1, kWtLimitNs, &go);
                }
            }
        } else if (warp == 9 && nt > 0) {
            // ------------------------------ products ------------------------------
            // The whole warp walks the loop and one elected lane issues: descriptors are one
            // addition to a warp-uniform base (built one by one by a single lane, the products
            // alone took 1.59 us per 128 keys, so 1.45).
            constexpr uint32_t ID_QK = idesc_f16(128, kWtKeys, AbFormat<T>::value);
            constexpr uint32_t ID_PV = idesc_f16(128, DP, AbFormat<T>::value) | (1u << 16);   // B along N
            const bool leader = elect_one();
            const uint64_t dq = sdesc_k_sw128(smem_u32(s_q)), dk = sdesc_k_sw128(smem_u32(s_k));
            const uint64_t dv = sdesc_mn_sw128(smem_u32(s_v), 16384);
            constexpr uint32_t TILE = C::kTileBytes >> 4;   // descriptors count 16 bytes
            auto qk = [&](int w, int st) {
                const uint64_t a = dq + w * TILE, b = dk + st * TILE;
                if (leader) {
#pragma unroll
                    for (int kk = 0; kk < DP / 16; ++kk) {
                        constexpr int H = 16384 >> 4;
                        umma_f16(tmem + C::kSCol + 128 * w, a + (kk / 4) * H + (kk % 4) * 2, b + (kk / 4) * H + (kk % 4) * 2,
                                 ID_QK, kk > 0);
                    }
                    umma_commit(s_full + w);
                }
            };
            auto pv = [&](int w, int st, int half, bool first) {
                const uint64_t b = dv + st * TILE;
                if (leader)
#pragma unroll
                    for (int kk = 0; kk < kWtKeys / 32; ++kk) {
                        const int k = half * (kWtKeys / 32) + kk;
                        umma_f16_ts(tmem + C::kOCol + DP * w, tmem + C::kSCol + 128 * w + k * 8, b + k * (2048 >> 4), ID_PV,
                                    !first || k > 0);
                    }
            };
            auto until = [&](uint64_t* bar, uint32_t parity) {
                const bool ok = __all_sync(0xffffffffu, wait(bar, parity));
                tc_fence_after();
                return ok;
            };
            bool ok = until(q_full, 0) && until(k_full, 0);
            if (ok) qk(0, 0);
            ok = ok && until(q_full + 1, 0);
            if (ok) {
                qk(1, 0);
                if (leader) umma_commit(k_empty);
            }
            // the weights of tile w overwrite its scores: the next scores are issued behind the product
            // that reads them, and products of one thread run in order
            int st = 0;
            uint32_t ph = 0;
            ok = ok && until(v_ok, 0);
            for (int i = 0; i < nt && ok; ++i) {
                const int sn = st + 1 == NS ? 0 : st + 1;
                const uint32_t pn = st + 1 == NS ? ph ^ 1u : ph;
                const bool more = i + 1 < nt;
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    if (!(ok = until(p_ready + 2 * w, i & 1))) break;
                    pv(w, st, 0, i == 0);   // the first half of the keys while the second is still exponentiated
                    if (!(ok = until(p_ready + 2 * w + 1, i & 1))) break;
                    pv(w, st, 1, false);
                    if (w == 1 && leader) umma_commit(v_empty + st);
                    if (more) {
                        // waits for loads stand behind queued products
                        if (w == 0 && !(ok = until(k_full + sn, pn))) break;
                        qk(w, sn);
                    } else if (leader) {
                        umma_commit(o_done + w);
                    }
                }
                if (ok && more) {
                    if (leader) umma_commit(k_empty + sn);
                    ok = until(v_ok + sn, pn);
                }
                st = sn;
                ph = pn;
            }
            if (!ok && leader) {
                volatile int go = 0;
                umma_commit(drained);
                mbar_wait_bounded(drained, 0, kWtLimitNs, &go);
            }
        } else if (warp >= 10) {
            // ------------------------------ V tiles with hidden keys ------------------------------
            const int tl = hi - 1;   // position of the last token (or the last key)
            for (int i = 0; i < nt; ++i) {
                const int st = i % NS, base = tile_base(i);
                if (!wait(v_full + st, (i / NS) & 1)) break;
                if (base + kWtKeys - 1 > t0 || (p.window > 0 && base <= tl - p.window)) {
                    const int n = t.lk - base;   // keys of the sequence in this tile
                    for (int r = threadIdx.x - 320; r < kWtKeys; r += 64) {
                        uint8_t* row = s_v + st * C::kTileBytes + r * 128;
                        bool zero = r >= n;
                        if (!zero) {
                            bool bad = false;
#pragma unroll 4
                            for (int c = 0; c < 8 * C::kHalves; ++c)
                                bad |= any_not_finite<T>(*reinterpret_cast<const uint4*>(
                                    row + (c >> 3) * 16384 + (((c + r) & 7) << 4)));
                            if (bad) *not_finite = 1;
                            zero = bad;
                        }
                        if (zero)
#pragma unroll 4
                            for (int c = 0; c < 8 * C::kHalves; ++c)
                                *reinterpret_cast<uint4*>(row + (c >> 3) * 16384 + (((c + r) & 7) << 4)) = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async_smem();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(v_ok + st);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
        // ------------------------------ softmax and output ------------------------------
        const int w = warp >> 2;
        const int r = (warp & 3) * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lanes + C::kSCol + 128 * w, to = tmem + lanes + C::kOCol + DP * w;
        const int per = 128 >> rp_log2;
        const int local = w * per + (r >> rp_log2);          // token within the block
        const int head = (hg << rp_log2) + (r & ((1 << rp_log2) - 1));
        const int tr = t0 + local;                            // this row's position
        const int ta = t0 + w * per, tb = min(ta + per, hi) - 1;   // the tile's first and last positions
        constexpr float kLift = WeightLift<T>::value;
        float m = -INFINITY, l = 0.0f;
        bool ok = true;
        for (int i = 0; i < nt; ++i) {
            ok = wait(s_full + w, i & 1);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            float s[kWtKeys];
#pragma unroll
            for (int c = 0; c < kWtKeys; c += 32) tmem_ld32(ts + c, s + c);
            tmem_wait_ld();
            const int base = tile_base(i);
            const bool edge = base + kWtKeys - 1 > ta || (p.window > 0 && base <= tb - p.window);
            if (edge) {
                const int last = tr - base, from = p.window > 0 ? last - p.window + 1 : 0, first = p.sinks - base;
#pragma unroll
                for (int c = 0; c < kWtKeys; c += 32) {
                    const uint32_t on = ones_below(last + 1 - c) & (~ones_below(from - c) | ones_below(first - c));
                    if (__any_sync(0xffffffffu, on != 0xffffffffu))
#pragma unroll
                        for (int e = 0; e < 32; ++e) s[c + e] = (on >> e) & 1u ? s[c + e] : -INFINITY;
                }
            }
            // the running maximum; a NaN score makes it NaN, and with it the whole row
            float mx[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) mx[e] = max3(s[e], s[8 + e], s[16 + e]);
#pragma unroll
            for (int c = 24; c < kWtKeys - 8; c += 16)
#pragma unroll
                for (int e = 0; e < 8; ++e) mx[e] = max3(mx[e], s[c + e], s[c + 8 + e]);
#pragma unroll
            for (int e = 0; e < 8; e += 2) mx[e] = max3(mx[e], s[kWtKeys - 8 + e], max3(mx[e + 1], s[kWtKeys - 7 + e], m));
            const float n = max3(max3(mx[0], mx[2], mx[4]), mx[6], m);
            if (i == 0) {
                m = n;
            } else {
                const bool grow = n != m && !((n - m) * p.sl2 <= kWtRescaleLog2);
                if (__any_sync(0xffffffffu, grow)) {
                    // the scores' barrier also covers the second product before them: O is complete
                    const float f = grow ? exp2_fast((m - n) * p.sl2) : 1.0f;
                    if (grow) m = n;
                    l *= f;
#pragma unroll
                    for (int c = 0; c < DP; c += 16) {   // 16 columns at a time beside the 128 scores
                        float o[16];
                        tmem_ld16(to + c, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] *= f;
                        tmem_st16(to + c, o);
                    }
                }
            }
            const float u = m == -INFINITY ? 0.0f : m * p.sl2 - kLift;
            const float2 scale = make_float2(p.sl2, p.sl2), shift = make_float2(-u, -u);
            float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
            for (int c = 0; c < kWtKeys; c += 32) {
                uint32_t x[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    float2 a = fma2(make_float2(s[c + 2 * e], s[c + 2 * e + 1]), scale, shift);
                    a.x = exp2_fast(a.x);
                    a.y = exp2_fast(a.y);
                    sum[e & 1] = add2(sum[e & 1], a);
                    x[e] = pack2<T>(a.x, a.y);   // weights in T for the second product; the sum keeps fp32
                }
                tmem_st16u(ts + c / 2, x);
                if (c & 32) {
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(p_ready + 2 * w + c / 64);
                }
            }
            l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        }
        if (m == INFINITY) l = NAN;   // inf - inf
        // every V tile has been looked through when the last one has; a row is either stored here or
        // computed again from q, which out may be (seen while the last product runs)
        bool again = false;
        if (!SPLIT && nt > 0 && ok) {
            ok = wait(v_ok + (nt - 1) % NS, ((nt - 1) / NS) & 1);
            again = *not_finite != 0;
        }
        if (nt > 0) ok = __all_sync(0xffffffffu, ok && wait(o_done + w, 0));
        tc_fence_after();
        if constexpr (SPLIT) {
            // unnormalised, in fp32, 16-byte chunks swizzled by row; the products with Q and K are complete
            float* part = reinterpret_cast<float*>(s_q) + (w * 128 + r) * DP;
#pragma unroll
            for (int c = 0; c < DP; c += 32) {
                float o[32];
                if (nt > 0) {
                    tmem_ld32(to + c, o);
                    tmem_wait_ld();
                }
#pragma unroll
                for (int e = 0; e < 32; e += 4)
                    *reinterpret_cast<float4*>(part + (((c + e) / 4) ^ (r & 7)) * 4) =
                        nt > 0 ? make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
            s_ml[(w * 128 + r) * 2] = m == -INFINITY ? m : m * p.sl2 - kLift;
            s_ml[(w * 128 + r) * 2 + 1] = l;
        }
        const bool mine = !SPLIT && ok && !again && local < rows;
        const int64_t qrow = t.q0 + t.m0 + local;
        const float inv = l > 0.0f ? 1.0f / l : l;
        T* out = static_cast<T*>(p.out) + qrow * p.o_row + head * p.o_head;
        const bool wide = (reinterpret_cast<uintptr_t>(out) & 31) == 0;
#pragma unroll
        for (int c = 0; c < DP; c += 32) {
            float o[32];
            if (!SPLIT && nt > 0) {
                tmem_ld32(to + c, o);
                tmem_wait_ld();
            }
            if (mine)
#pragma unroll
                for (int e = 0; e < 32; e += 16) {
                    uint32_t x[8];
#pragma unroll
                    for (int y = 0; y < 8; ++y)
                        x[y] = nt > 0 ? pack2<T>(o[e + 2 * y] * inv, o[e + 2 * y + 1] * inv) : 0u;
                    if (wide && c + e + 16 <= p.dim) {
                        store32(out + c + e, x);
                    } else {
                        if (c + e < p.dim) *reinterpret_cast<uint4*>(out + c + e) = make_uint4(x[0], x[1], x[2], x[3]);
                        if (c + e + 8 < p.dim) *reinterpret_cast<uint4*>(out + c + e + 8) = make_uint4(x[4], x[5], x[6], x[7]);
                    }
                }
        }
        if (mine && p.lse != nullptr)
            p.lse[qrow * p.heads + head] = l != 0.0f ? ((m == -INFINITY ? 0.0f : m * p.sl2 - kLift) + log2f(l)) * kLn2 : -INFINITY;
        if (again && ok)
            for (int x = warp; x < 256; x += 8) {
                const int tok = x >> rp_log2;
                if (tok < rows) window_row_exact<T>(p, t, t.m0 + tok, (hg << rp_log2) + (x & ((1 << rp_log2) - 1)), lane);
            }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
    if constexpr (SPLIT) {
        cooperative_groups::this_cluster().sync();
        // (the softmax warps: the others gave their registers up)
        if (warp < 8)
            window_cluster_join<T, DP>(p, t, reinterpret_cast<float*>(s_q), s_ml, const_cast<const int*>(not_finite), hg, rows,
                                       rp_log2, rank, splits, warp, lane);
        __syncwarp();
        cooperative_groups::this_cluster().sync();   // nobody leaves while its part is read
    }
}

}  // namespace chronos
