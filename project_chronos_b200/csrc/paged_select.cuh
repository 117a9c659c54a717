// paged_select.cuh — which pages of a long cache a query looks at: bounds of every page's
// keys, the scores they give, and the highest of them (include/chronos_paged4.h).
//
// No key k of a page gives q.k above sum_d max(q_d lo_d, q_d hi_d).  Summed over the query
// heads of a kv head that is one product,
//     score = sum_d up_d hi_d + down_d lo_d,   up = sum_h max(q_h, 0), down = sum_h min(q_h, 0),
// whatever the number of heads: 2 D products per page for 2 D elements read.  It is summed
// in 64 bits, whose rate (half of fp32's) the reading does not leave behind: pages that a
// sum in 32 bits would mix up keep the order that their exact scores have.
#pragma once

#include "chronos_paged4.h"
#include "fp4.cuh"
#include "paged.cuh"
#include "paged_rope.cuh"

namespace chronos {

struct PagedBoundsParams {
    ChronosPagedCache c;
    int packed, columns, full;
    float k_scale;
    int64_t tokens;
    const int32_t* cu;
    void* bounds;
    int max_slots;
    int32_t* status;
};

constexpr int kBoundThreads = 128;

// NaN where one of the two is.
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// A block per (sequence, kv head) and page in turn: LPR lanes hold a slot's columns, 8 each,
// the block's other groups take the next slots; the groups meet in shared memory.
template <typename T, int LPR, bool VEC, bool PACKED>
__global__ void __launch_bounds__(kBoundThreads) paged_bounds_kernel(const __grid_constant__ PagedBoundsParams p) {
    constexpr int GROUPS = kBoundThreads / LPR;
    __shared__ float s_x[2][GROUPS][LPR * 8];
    const int G = p.c.kv_heads, D = p.c.head_dim, size = p.c.page_size;
    const int64_t row = static_cast<int64_t>(blockIdx.z) * gridDim.y + blockIdx.y;
    const int b = static_cast<int>(row / G), g = static_cast<int>(row % G);
    if (b >= p.c.batch) return;
    const int raw = p.c.lens[b], len = min(max(raw, 0), p.max_slots);
    if (raw != len && g == 0 && blockIdx.x == 0 && threadIdx.x == 0) report_status(p.status, CHRONOS_ERR_INVALID_ARG);
    // the newest slots: [from, len).  Tokens that were dropped make it begin earlier, which does no harm.
    const int fresh = p.full ? len : p.cu == nullptr ? 1 : max(p.cu[b + 1] - p.cu[b], 0);
    const int from = max(len - fresh, 0);
    if (from >= len) return;
    const int group = threadIdx.x / LPR, col = threadIdx.x % LPR * 8;
    for (int j = from / size + blockIdx.x; j * static_cast<int64_t>(size) < len; j += gridDim.x) {
        const int page = p.c.page_table[b * p.c.page_table_stride + j];
        if (page < 0 || page >= p.c.num_pages) {
            if (threadIdx.x == 0) report_status(p.status, CHRONOS_ERR_INVALID_ARG);
            continue;
        }
        const int start = j * size, stop = min(len - start, size);   // of the page's slots
        int at = max(from - start, 0);
        float lo[8], hi[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            lo[e] = INFINITY;
            hi[e] = -INFINITY;
        }
        if (col < D) {
#pragma unroll 4
            for (int i = at + group; i < stop; i += GROUPS) {
                float x[8];
                if constexpr (PACKED) {
                    const uint8_t* record = static_cast<const uint8_t*>(p.c.k_pages) + page * p.c.k_page_stride + g * p.c.k_head_stride +
                                            (i >> 4) * fp4_record(p.columns);
                    fp4_load8(record, i & 15, col, p.columns, p.k_scale, x);
                } else {
                    const T* k = static_cast<const T*>(p.c.k_pages) + page * p.c.k_page_stride + i * p.c.k_slot_stride + g * p.c.k_head_stride;
                    if constexpr (VEC) {
                        load8<T>(k + col, x);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] = col + e < D ? to_f32<T>(k[col + e]) : 0.0f;
                    }
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    lo[e] = min_nan(lo[e], x[e]);
                    hi[e] = max_nan(hi[e], x[e]);
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            s_x[0][group][col + e] = lo[e];
            s_x[1][group][col + e] = hi[e];
        }
        __syncthreads();
        T* out = static_cast<T*>(p.bounds) + (static_cast<int64_t>(page) * 2 * G + g) * D;
        for (int i = threadIdx.x; i < 2 * LPR * 8; i += kBoundThreads) {
            const int d = i % (LPR * 8), which = i / (LPR * 8);
            if (d >= D) continue;
            float v = s_x[which][0][d];
            const int used = min(GROUPS, stop - at);
            for (int k = 1; k < used; ++k) v = which ? max_nan(v, s_x[1][k][d]) : min_nan(v, s_x[0][k][d]);
            T* to = out + static_cast<int64_t>(which) * G * D + d;
            if (at > 0) {   // older slots are in the bounds already
                const float old = to_f32<T>(*to);
                v = which ? max_nan(v, old) : min_nan(v, old);
            }
            *to = from_f32<T>(v);
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------
// scores
// ---------------------------------------------------------------------------
struct PagedSelectParams {
    ChronosPagedCache c;
    int heads, rep, topk, first, last;
    int64_t token0, tokens;     // tokens [token0, token0 + tokens) of the call
    const void* q;
    int64_t q_row, q_head;
    const void* bounds;
    const int32_t* cu;
    int32_t* pages;
    int max_slots;
    int64_t width;              // keys per token and kv head
    unsigned long long* keys;   // [tokens][kv heads][width]
    int chunk;                  // pages of a block
    int32_t* status;
};

// A token's sequence (-1: none), the slots at or before it and their pages.
struct SelectToken {
    int seq, len, pages;
};
__device__ __forceinline__ SelectToken select_token(const PagedSelectParams& p, int64_t t, int lane) {
    SelectToken r{};
    r.seq = p.cu == nullptr ? static_cast<int>(t) : paged_sequence(p.cu, p.c.batch, t, lane);
    if (r.seq >= p.c.batch || (p.cu != nullptr && t < p.cu[r.seq])) {
        r.seq = -1;
        return r;
    }
    r.len = min(max(p.c.lens[r.seq], 0), p.max_slots);
    if (p.cu != nullptr) r.len = static_cast<int>(max(int64_t{0}, r.len - (static_cast<int64_t>(p.cu[r.seq + 1]) - 1 - t)));
    r.pages = (r.len + p.c.page_size - 1) / p.c.page_size;
    return r;
}

// A score's place in the order of numbers: -0 as 0, NaN above every number, and room above
// for the pages that are always in (and 0 for a page that is none).
__device__ __forceinline__ unsigned long long select_key(double x) {
    if (x != x) return ~0ull - 1;
    const unsigned long long u = static_cast<unsigned long long>(__double_as_longlong(x + 0.0));
    return (u >> 63) ? ~u : (u | (1ull << 63));
}

constexpr int kScoreThreads = 256;
constexpr int kScoreTokens = 8;     // tokens of one sequence that share the reading of a page

// Bound by reading the bounds.  8 lanes share a page; each takes every eighth group of 8
// columns of lo and hi, and the partial sums meet in three shuffles.  Block: a chunk of
// pages, a kv head, up to 8 tokens (split where their sequences differ).
template <typename T, bool VEC>
__global__ void __launch_bounds__(kScoreThreads) paged_score_kernel(const __grid_constant__ PagedSelectParams p) {
    constexpr int MAXD = CHRONOS_PAGED_MAX_HEAD_DIM;
    __shared__ __align__(16) double s_q[kScoreTokens][2][MAXD];   // down, up
    __shared__ SelectToken s_t[kScoreTokens];
    const int G = p.c.kv_heads, D = p.c.head_dim, g = blockIdx.y;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t t0 = static_cast<int64_t>(blockIdx.z) * kScoreTokens;
    const int n = static_cast<int>(min(int64_t{kScoreTokens}, p.tokens - t0));
    if (warp < n) {
        const SelectToken r = select_token(p, p.token0 + t0 + warp, lane);
        if (lane == 0) s_t[warp] = r;
    }
    __syncthreads();
    const int j0 = blockIdx.x * p.chunk;
    bool any = false;   // tokens with no more pages than they may take need no scores
    for (int i = 0; i < n; ++i) any |= s_t[i].pages > p.topk && s_t[i].pages > j0;
    if (!any) return;
    const int D8 = (D + 7) & ~7;
    for (int i = threadIdx.x; i < n * D8; i += kScoreThreads) {
        const int t = i / D8, d = i % D8;
        double up = 0.0, down = 0.0;
        if (d < D && s_t[t].pages > p.topk) {
            const T* q = static_cast<const T*>(p.q) + (p.token0 + t0 + t) * p.q_row + static_cast<int64_t>(g) * p.rep * p.q_head + d;
            for (int h = 0; h < p.rep; ++h) {
                const float x = to_f32<T>(q[h * p.q_head]);
                if (x > 0.0f) up += x;
                else down += x;   // and NaN
            }
        }
        s_q[t][0][d] = down;
        s_q[t][1][d] = up;
    }
    __syncthreads();
    const int part = threadIdx.x & 7;
    for (int i0 = 0; i0 < n;) {
        // tokens i0 .. i1 - 1 share a sequence
        int i1 = i0 + 1;
        const int seq = s_t[i0].seq;
        while (i1 < n && s_t[i1].seq == seq) ++i1;
        const int most = s_t[i1 - 1].pages;   // the last of them sees most
        if (seq >= 0 && most > p.topk) {
            const int32_t* table = p.c.page_table + seq * p.c.page_table_stride;
            for (int j = j0 + (threadIdx.x >> 3); j - static_cast<int>(threadIdx.x >> 3) < min(j0 + p.chunk, most); j += kScoreThreads / 8) {
                const bool in = j < min(j0 + p.chunk, most);
                int page = in ? table[j] : -1;
                if (in && (page < 0 || page >= p.c.num_pages)) {
                    report_status(p.status, CHRONOS_ERR_INVALID_ARG);
                    page = -1;
                }
                double acc[kScoreTokens];
#pragma unroll
                for (int t = 0; t < kScoreTokens; ++t) acc[t] = 0.0;
                if (page >= 0) {
                    const T* lo = static_cast<const T*>(p.bounds) + (static_cast<int64_t>(page) * 2 * G + g) * D;
                    const T* hi = lo + static_cast<int64_t>(G) * D;
                    for (int d = part * 8; d < D; d += 64) {
                        float a[8], c[8];
                        if constexpr (VEC) {
                            load8<T>(lo + d, a);
                            load8<T>(hi + d, c);
                        } else {
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                a[e] = d + e < D ? to_f32<T>(lo[d + e]) : 0.0f;
                                c[e] = d + e < D ? to_f32<T>(hi[d + e]) : 0.0f;
                            }
                        }
                        double wa[8], wc[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            wa[e] = a[e];
                            wc[e] = c[e];
                        }
#pragma unroll
                        for (int t = 0; t < kScoreTokens; ++t) {
                            if (i0 + t >= i1) break;
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                acc[t] = fma(s_q[i0 + t][0][d + e], wa[e], acc[t]);
                                acc[t] = fma(s_q[i0 + t][1][d + e], wc[e], acc[t]);
                            }
                        }
                    }
                }
#pragma unroll
                for (int t = 0; t < kScoreTokens; ++t) {
                    if (i0 + t >= i1) break;
                    double x = acc[t];
#pragma unroll
                    for (int o = 1; o < 8; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
                    if (part == 0 && in && j < s_t[i0 + t].pages)
                        p.keys[((t0 + i0 + t) * G + g) * p.width + j] = page < 0 ? 0ull : select_key(x);
                }
            }
        }
        i0 = i1;
    }
}

// ---------------------------------------------------------------------------
// selection
// ---------------------------------------------------------------------------
constexpr int kSelectThreads = 512;
constexpr int kSelectWarps = kSelectThreads / 32;
constexpr int kSelectBits = 11, kSelectBins = 1 << kSelectBits;
constexpr int kSelectKeys = 6144;   // keys that shared memory holds (48 KB of them)

// Inclusive sum over the block's threads of their counts (x: kSelectWarps ints of shared
// memory, free before and after); total: of all.
__device__ __forceinline__ int select_scan(int mine, int* x, int warp, int lane, int& total) {
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
    }
    __syncthreads();
    if (lane == 31) x[warp] = inc;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kSelectWarps; ++w) {
        before += w < warp ? x[w] : 0;
        total += x[w];
    }
    return before + inc;
}

// A block per (token, kv head): the topk-th largest key by radix selection, 11 bits at a time
// from the highest bit in which the keys differ, then the pages above it and the first of
// those equal to it, in their order.
__global__ void __launch_bounds__(kSelectThreads) paged_select_kernel(const __grid_constant__ PagedSelectParams p) {
    extern __shared__ unsigned long long s_keys[];   // [kSelectKeys]
    __shared__ int s_hist[kSelectBins];
    __shared__ int s_x[kSelectWarps];
    __shared__ unsigned long long s_y[2][kSelectWarps];
    __shared__ int s_digit, s_above, s_same;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = p.c.kv_heads;
    const int64_t t = blockIdx.x / G;   // of this launch
    const int g = blockIdx.x % G;
    const SelectToken tok = select_token(p, p.token0 + t, lane);
    pdl_wait();
    if (tok.seq < 0) return;
    int32_t* out = p.pages + ((p.token0 + t) * G + g) * p.topk;
    const int n = tok.pages;
    if (g == 0 && threadIdx.x == 0 && (p.c.lens[tok.seq] < 0 || p.c.lens[tok.seq] > p.max_slots))
        report_status(p.status, CHRONOS_ERR_INVALID_ARG);
    if (n <= p.topk) {
        for (int i = threadIdx.x; i < p.topk; i += kSelectThreads) out[i] = i < n ? i : -1;
        return;
    }
    unsigned long long* mine = p.keys + (t * G + g) * p.width;
    unsigned long long* keys = n <= kSelectKeys ? s_keys : mine;
    unsigned long long all = ~0ull, some = 0ull;
    for (int j = threadIdx.x; j < n; j += kSelectThreads) {
        const unsigned long long k = j < p.first || j >= n - p.last ? ~0ull : mine[j];
        keys[j] = k;
        all &= k;
        some |= k;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        all &= __shfl_xor_sync(0xffffffffu, all, o);
        some |= __shfl_xor_sync(0xffffffffu, some, o);
    }
    if (lane == 0) {
        s_y[0][warp] = all;
        s_y[1][warp] = some;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSelectWarps; ++w) {
        all &= s_y[0][w];
        some |= s_y[1][w];
    }
    // bits from `top` on differ somewhere
    int top = 64 - __clzll(static_cast<long long>(all ^ some));   // 0: all equal
    unsigned long long known = top == 64 ? 0ull : ~0ull << top, prefix = all & known;
    int want = p.topk;
    bool ties = true;   // more keys equal the threshold than are wanted
    while (top > 0) {
        const int shift = max(0, top - kSelectBits), bits = top - shift;
        const unsigned long long mask = (1ull << bits) - 1;
        for (int i = threadIdx.x; i < kSelectBins; i += kSelectThreads) s_hist[i] = 0;
        __syncthreads();
        for (int j = threadIdx.x; j < n; j += kSelectThreads) {
            const unsigned long long k = keys[j];
            if ((k & known) == prefix) atomicAdd(&s_hist[(k >> shift) & mask], 1);
        }
        __syncthreads();
        // thread i holds the digits from kSelectBins - 1 - 4 i down
        int h[4], sum = 0, total;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += h[i] = s_hist[kSelectBins - 1 - 4 * threadIdx.x - i];
        int above = select_scan(sum, s_x, warp, lane, total) - sum;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (above < want && above + h[i] >= want) {
                s_digit = kSelectBins - 1 - 4 * threadIdx.x - i;
                s_above = above;
                s_same = h[i];
            }
            above += h[i];
        }
        __syncthreads();
        prefix |= static_cast<unsigned long long>(s_digit) << shift;
        known |= mask << shift;
        want -= s_above;
        top = shift;
        if (s_same == want) {   // all of them: the bits below do not matter
            ties = false;
            break;
        }
        __syncthreads();
    }
    // pages in order: above the threshold, or one of the first `want` equal to it
    int same = 0, kept = 0;
    for (int j0 = 0; j0 < n; j0 += kSelectThreads) {
        const int j = j0 + threadIdx.x;
        const unsigned long long k = j < n ? keys[j] & known : 0ull;
        const bool eq = j < n && k == prefix, gt = j < n && k > prefix;
        bool take = gt || eq;
        int total;
        if (ties) {
            const int at = select_scan(eq ? 1 : 0, s_x, warp, lane, total);
            take = gt || (eq && same + at <= want);
            same += total;
        }
        const int at = select_scan(take ? 1 : 0, s_x, warp, lane, total);
        if (take) out[kept + at - 1] = j;
        kept += total;
    }
}

}  // namespace chronos
