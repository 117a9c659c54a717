// window_attention.cuh — causal attention of a packed batch of prompts, with an
// optional sliding window and first tokens that stay visible
// (include/chronos_paged.h, chronos_window_attention).
//
// Row t of a sequence sees the keys j <= t with window == 0, j > t - window or
// j < sinks.  One pass over the visible key tiles with a running maximum and
// sum: out = sum 2^(x_j - m) v_j / sum 2^(x_j - m), x_j = scale log2(e) q.k_j.
#pragma once

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
    int64_t q0, k0;     // first rows of the sequence in q and k
    int lq, lk;
};

// Tile number `x` of all sequences' tiles of `rows` queries (a whole warp calls
// this; false behind the last one).  Within a sequence the last tile comes
// first: under a causal mask it has the most keys.  Offsets that do not ascend
// or leave q or k are cut so that no access leaves them, and reported.
__device__ __forceinline__ bool window_tile(const WindowParams& p, int64_t x, int rows, int lane, WindowTile& t) {
    int64_t before = 0;
    for (int base = 0; base < p.batch; base += 32) {
        const int b = base + lane;
        int64_t n = 0;
        if (b < p.batch) n = (max(0, min(p.cu_q[b + 1] - p.cu_q[b], static_cast<int>(p.num_q))) + rows - 1) / rows;
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
            if (t.q0 < 0 || t.q0 + t.lq > p.num_q || t.k0 < 0 || t.lk < 0 || t.k0 + t.lk > p.num_k) {
                if (lane == 0) report_status(p.status, CHRONOS_ERR_INVALID_ARG);
                return false;
            }
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
// 16 x 16: a thread forms 4 x 4 scores and 4 rows x D/16 columns of the output.
// ---------------------------------------------------------------------------
constexpr int kWsThreads = 256;
constexpr int kWsRows = 64;
constexpr int kWsKeys = 64;

__host__ __device__ constexpr int window_simt_dim(int dim) { return (dim + 63) / 64 * 64; }
__host__ __device__ constexpr int window_simt_smem(int dim) {
    return (kWsRows + 2 * kWsKeys) * (window_simt_dim(dim) + 4) * 4 + kWsRows * (kWsKeys + 4) * 4;
}

// NC: groups of 64 output columns (head_dim <= 64 * NC).
template <typename T, int NC>
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
    if (!window_tile(p, blockIdx.x / p.heads, kWsRows, lane, t)) return;
    const int rows = min(kWsRows, t.lq - t.m0);
    const int t0 = t.lk - t.lq + t.m0;            // position of the first row
    const int hi = min(t.lk, t0 + rows);          // keys [lo, hi) and the first ones
    const int lo = p.window > 0 ? max(0, t0 - p.window + 1) : 0;
    const int ns = p.window > 0 ? (max(0, min(p.sinks, hi)) + kWsKeys - 1) / kWsKeys : 0;
    const int w0 = max(ns * kWsKeys, lo);
    const int nt = ns + (hi > w0 ? (hi - w0 + kWsKeys - 1) / kWsKeys : 0);
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;

    auto stage = [&](float* dst, const T* src, int64_t row_stride, int n) {
        for (int i = threadIdx.x; i < kWsRows * DP; i += kWsThreads) {
            const int r = i / DP, d = i % DP;
            dst[r * LD + d] = r < n && d < p.dim ? to_f32<T>(src[r * row_stride + d]) : 0.0f;
        }
    };
    stage(s_q, static_cast<const T*>(p.q) + (t.q0 + t.m0) * p.q_row + head * p.q_head, p.q_row, rows);
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
        stage(s_k, static_cast<const T*>(p.k) + (t.k0 + j0) * p.k_row + g * p.k_head, p.k_row, n);
        stage(s_v, static_cast<const T*>(p.v) + (t.k0 + j0) * p.v_row + g * p.v_head, p.v_row, n);
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
        T* out = static_cast<T*>(p.out) + (t.q0 + t.m0 + row) * p.o_row + head * p.o_head;
#pragma unroll
        for (int c = 0; c < NC * 4; ++c) {
            const int d = (c >> 2) * 64 + tx * 4 + (c & 3);
            if (d < p.dim) out[d] = from_f32<T>(o[r][c] * inv);
        }
        if (tx == 0 && p.lse != nullptr)
            p.lse[(t.q0 + t.m0 + row) * p.heads + head] = l[r] != 0.0f ? (m[r] + log2f(l[r])) * kLn2 : -INFINITY;
    }
}

}  // namespace chronos
