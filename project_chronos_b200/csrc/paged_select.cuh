// paged_select.cuh — which pages of a long cache a query looks at: bounds of every page's
// keys, the scores they give, and the highest of them (include/chronos_paged4.h).
//
// No key k of a page gives q.k above sum_d max(q_d lo_d, q_d hi_d).  Summed over the query
// heads of a kv head that is one product,
//     score = sum_d up_d hi_d + down_d lo_d,   up = sum_h max(q_h, 0), down = sum_h min(q_h, 0),
// whatever the number of heads: 2 D products per page for 2 D elements read.  It is summed
// in 64 bits, which does not bound it (the FP64 pipe is 9 % busy): pages that a
// sum in 32 bits would mix up keep the order that their exact scores have.  That holds for
// finite bounds and queries: where an infinity meets up or down = 0 (no query of that sign) the
// product is NaN and the maximum need not be.  Any bound or query that is not finite makes the
// sum infinite or NaN, so those few pages are found by their scores and done again head by head.
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

// A smallest or largest value of codes and scales as it is stored: times the cache's factor, whose
// product has more bits than 16-bit types (than fp32, too), rounded outwards, so that no key lies outside.
template <typename T>
__device__ __forceinline__ T bound_outwards(float x, float unit, bool largest) {
    const float y = largest ? __fmul_ru(x, unit) : __fmul_rd(x, unit);
    if constexpr (std::is_same<T, float>::value) return y;
    else if constexpr (std::is_same<T, __half>::value) return largest ? __float2half_ru(y) : __float2half_rd(y);
    else return largest ? __float2bfloat16_ru(y) : __float2bfloat16_rd(y);
}

// A block per (sequence, kv head) and page in turn: LPR lanes hold a slot's columns, 8 each,
// the block's other groups take the next slots; the groups meet in shared memory.  One new token
// per sequence is bound by latency (32 rows of 8 heads 3 us), since older slots are not read again.
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
                    fp4_load8(record, i & 15, col, p.columns, 1.0f, x);   // (the factor, a positive one, comes last)
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
            if constexpr (PACKED) v = to_f32<T>(bound_outwards<T>(v, p.k_scale, which != 0));
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
    int cluster;                // blocks per tile and kv head
    int32_t* status;
};

// A score's place in the order of numbers: -0 as 0, NaN above every number (and 0 for a page
// that is none).
__device__ __forceinline__ unsigned long long select_key(double x) {
    if (x != x) return ~0ull - 1;
    const unsigned long long u = static_cast<unsigned long long>(__double_as_longlong(x + 0.0));
    return (u >> 63) ? ~u : (u | (1ull << 63));
}

constexpr int kSelectThreads = 256;
constexpr int kSelectWarps = kSelectThreads / 32;
constexpr int kSelectTokens = 8;    // tokens of one sequence that share the reading of a page
constexpr int kSelectPages = 512;   // pages whose numbers a block holds at a time
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

struct SelectShared {
    __align__(16) int hist[kSelectBins];
    int scan[kSelectWarps];
    unsigned long long ends[2][kSelectWarps];
    int digit, above, same;
};

// The scores of a token's pages [lo, hi) that are infinite or NaN, again from the formula as it stands: NaN where
// a product or a maximum is.  (Only they can be wrong: a sum of minus infinity is an infinite query's, below
// bounds that are finite.)  What is finite is summed as paged_select_kernel sums it, so that equal
// scores stay equal.  Whole blocks call it; 8 lanes take a page.  Rare: one column at a time, in few registers.
template <typename T>
__device__ __forceinline__ void select_again(const PagedSelectParams& p, unsigned long long* keys, int64_t token, int g, int seq, int lo, int hi) {
    const uint32_t lanes = 0xffu << (threadIdx.x & 24);
    const T* q = static_cast<const T*>(p.q) + token * p.q_row + static_cast<int64_t>(g) * p.rep * p.q_head;
    const int G = p.c.kv_heads, D = p.c.head_dim;
#pragma unroll 1
    for (int j = lo + (threadIdx.x >> 3); j < hi; j += kSelectThreads / 8) {
        if (keys[j] < select_key(INFINITY)) continue;
        const T* bounds = static_cast<const T*>(p.bounds) + (static_cast<int64_t>(p.c.page_table[seq * p.c.page_table_stride + j]) * 2 * G + g) * D;
        double x = 0.0, odd = 0.0;
#pragma unroll 1
        for (int i = 0; i < 16 * ((D + 63) / 64); ++i) {   // 8 columns' lower, then their upper bounds
            const bool upper = (i & 8) != 0;
            const int d = (i >> 4) * 64 + (threadIdx.x & 7) * 8 + (i & 7);
            if (d >= D) continue;
            const float low = to_f32<T>(bounds[d]), high = to_f32<T>(bounds[static_cast<int64_t>(G) * D + d]);
            double sum = 0.0, side = 0.0;   // of the column's maxima, of its queries on this side
#pragma unroll 1
            for (int h = 0; h < p.rep; ++h) {
                const float v = to_f32<T>(q[h * p.q_head + d]);
                const double a = static_cast<double>(v) * low, b = static_cast<double>(v) * high;
                sum += a != a || a > b ? a : b;   // NaN where one is
                if ((v > 0.0f) == upper) side += v;
            }
            const float bound = upper ? high : low;
            if (!(fabs(sum) < INFINITY)) odd += upper ? 0.0 : sum;
            else if (fabsf(bound) < INFINITY) x = fma(side, static_cast<double>(bound), x);   // (an infinity is on the side that no query takes)
        }
        x += odd;
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) x += __shfl_xor_sync(lanes, x, o);
        if ((threadIdx.x & 7) == 0) keys[j] = select_key(x);
    }
}

// The pages of one token and kv head, by a block.  Of the pages that are not always in, the
// `want`-th largest key by radix selection, 11 bits at a time of what the keys are above the
// smallest one (scores lie in a few binades: their upper bits alone would tell nothing), then the
// pages above it and the first of those equal to it, in their order.  n: the token's pages.
template <typename T>
__device__ __forceinline__ void select_row(const PagedSelectParams& p, SelectShared& s, unsigned long long* held, unsigned long long* mine,
                                           int32_t* out, int n, int64_t token, int g, int seq) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (n <= p.topk) {
        for (int i = threadIdx.x; i < p.topk; i += kSelectThreads) out[i] = i < n ? i : -1;
        return;
    }
    // pages [lo, hi) compete for `want` places (first + last <= topk < n: there are some)
    const int lo = p.first, hi = n - p.last;
    int want = p.topk - p.first - p.last;
    const bool fits = n <= kSelectKeys;
    for (int i = threadIdx.x; i < kSelectBins; i += kSelectThreads) s.hist[i] = 0;
    unsigned long long low, high;
    for (bool again = false;; again = true) {
        low = ~0ull;
        high = 0ull;
#pragma unroll 4
        for (int j = lo + threadIdx.x; j < hi; j += kSelectThreads) {
            const unsigned long long k = mine[j];
            if (fits) held[j] = k;
            low = min(low, k);
            high = max(high, k);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            low = min(low, __shfl_xor_sync(0xffffffffu, low, o));
            high = max(high, __shfl_xor_sync(0xffffffffu, high, o));
        }
        if (lane == 0) {
            s.ends[0][warp] = low;
            s.ends[1][warp] = high;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kSelectWarps; ++w) {
            low = min(low, s.ends[0][w]);
            high = max(high, s.ends[1][w]);
        }
        if (again || high < select_key(INFINITY)) break;
        select_again<T>(p, mine, token, g, seq, lo, hi);
        __syncthreads();
    }
    auto key = [&](int j) { return (fits ? held[j] : mine[j]) - low; };
    // what the keys are above the smallest has `top` bits
    int top = 64 - __clzll(static_cast<long long>(high - low));
    unsigned long long known = top == 64 ? 0ull : ~0ull << top, prefix = 0ull;
    if (want == 0) prefix = known = ~0ull, top = 0;   // none of them: no key is above or equal (they are below 2^64 - 1)
    for (bool fresh = true; top > 0; fresh = false) {
        const int shift = max(0, top - kSelectBits), bits = top - shift;
        const unsigned long long mask = (1ull << bits) - 1;
        if (!fresh) {
            for (int i = threadIdx.x; i < kSelectBins; i += kSelectThreads) s.hist[i] = 0;
            __syncthreads();
        }
        for (int j = lo + threadIdx.x; j < hi; j += kSelectThreads) {
            const unsigned long long k = key(j);
            if ((k & known) == prefix) atomicAdd(&s.hist[(k >> shift) & mask], 1);
        }
        __syncthreads();
        // thread i holds the digits from kSelectBins - 1 - PER i down
        constexpr int PER = kSelectBins / kSelectThreads;
        static_assert(PER % 4 == 0, "whole vectors");
        int h[PER], sum = 0, total;
#pragma unroll
        for (int i = 0; i < PER / 4; ++i) {
            const int4 four = *reinterpret_cast<const int4*>(&s.hist[kSelectBins - PER * threadIdx.x - 4 * i - 4]);
            h[4 * i] = four.w; h[4 * i + 1] = four.z; h[4 * i + 2] = four.y; h[4 * i + 3] = four.x;
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) sum += h[i];
        int above = select_scan(sum, s.scan, warp, lane, total) - sum;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (above < want && above + h[i] >= want) {
                s.digit = kSelectBins - 1 - PER * threadIdx.x - i;
                s.above = above;
                s.same = h[i];
            }
            above += h[i];
        }
        __syncthreads();
        prefix |= static_cast<unsigned long long>(s.digit) << shift;
        known |= mask << shift;
        want -= s.above;
        top = shift;
        if (s.same == want) break;   // all of them: the bits below do not matter
    }
    // pages in order: always in, above the threshold, or one of the first `want` equal to it
    int more = 0, same = 0;   // pages before this round's: taken whatever comes, equal to the threshold
    for (int j0 = 0; j0 < n; j0 += kSelectThreads) {
        const int j = j0 + threadIdx.x;
        const bool inside = j >= lo && j < hi, always = j < n && !inside;
        const unsigned long long k = inside ? key(j) & known : 0ull;
        const bool eq = inside && k == prefix, gt = always || (inside && k > prefix);
        int total;
        const int at = select_scan((gt ? 1 << 16 : 0) | (eq ? 1 : 0), s.scan, warp, lane, total);
        const int rank = same + (at & 0xffff);   // among the equal ones, from 1 on
        if (gt || (eq && rank <= want)) out[more + (at >> 16) + min(rank, want) - 1] = j;
        more += total >> 16;
        same += total & 0xffff;
    }
}

// Bound by reading the bounds.  A cluster of p.cluster blocks per TOKENS tokens of a sequence (1
// where every sequence has one) and kv head.  Scores: the blocks share the pages, 8 lanes a
// page, two pages at a time (16-bit types), whose loads all go out before the first is used; each
// lane takes every eighth group of 8 columns of lo and hi, and the partial sums meet in three
// shuffles.  The queries' sums lie in shared memory so that the 8 lanes' parts are side by side,
// the pages' numbers beside them: both are fetched at once.  Then the blocks share the tokens'
// selections.  32 rows of 256 to 512 pages, 8 heads of 128: 52 us with a look-up before every
// page, 19 without, the selection included (50 MB of bounds, 8 us at HBM's rate; the FP64 pipe is 9 % busy, 34 %
// of issue slots are used: a block's few warps wait for its rounds of loads, then for the selection's
// rounds of counting).
template <typename T, bool VEC, int TOKENS>
__global__ void __launch_bounds__(kSelectThreads, TOKENS == 1 ? 3 : 2) paged_select_kernel(const __grid_constant__ PagedSelectParams p) {
    constexpr int MAXD = CHRONOS_PAGED_MAX_HEAD_DIM, GROUPS = kSelectThreads / 8;
    constexpr int PAGES = sizeof(T) == 2 && VEC ? 2 : 1, CHUNKS = PAGES;   // pages and 64 columns that are in flight at once
    constexpr int ROUND = PAGES * GROUPS;                                  // pages of a block at once
    extern __shared__ unsigned long long s_keys[];                         // [kSelectKeys]
    __shared__ __align__(16) double2 s_q[TOKENS][2][MAXD / 2];   // down, up; columns 64 c + 8 part + 2 e, + 1 at (4 c + e) * 8 + part
    __shared__ int s_page[kSelectPages];
    __shared__ SelectShared s_sel;
    const int G = p.c.kv_heads, D = p.c.head_dim, C = p.cluster;
    const int rank = blockIdx.x % C, g = blockIdx.x / C % G, tile = blockIdx.x / C / G;
    const int lane = threadIdx.x & 31;
    // the tokens: [t0, t0 + n) of sequence seq, the last of which sees `len` slots
    int64_t t0 = p.token0 + tile;
    int seq = static_cast<int>(t0), n = 1;
    if (p.cu != nullptr) {
        // `tile` of the list of all sequences' tiles of TOKENS tokens (this launch has tokens token0 ..)
        int before = 0;
        seq = -1;
        for (int base = 0; base < p.c.batch && seq < 0; base += 32) {
            const int b = base + lane;
            int64_t lo = 0, hi = 0;
            if (b < p.c.batch) {
                lo = max(static_cast<int64_t>(p.cu[b]), p.token0);
                hi = min(static_cast<int64_t>(p.cu[b + 1]), p.token0 + p.tokens);
            }
            const int mine = hi > lo ? static_cast<int>((hi - lo + TOKENS - 1) / TOKENS) : 0;
            int inc = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += v;
            }
            const uint32_t past = __ballot_sync(0xffffffffu, before + inc > tile);
            if (past != 0u) {
                const int l = __ffs(past) - 1;
                const int in = tile - before - __shfl_sync(0xffffffffu, inc - mine, l);
                t0 = __shfl_sync(0xffffffffu, lo, l) + static_cast<int64_t>(in) * TOKENS;
                n = static_cast<int>(min(int64_t{TOKENS}, __shfl_sync(0xffffffffu, hi, l) - t0));
                seq = base + l;
            }
            before += __shfl_sync(0xffffffffu, inc, 31);
        }
        if (seq < 0) return;   // more clusters than tiles
    }
    const int raw = p.c.lens[seq], cut = min(max(raw, 0), p.max_slots);
    if (raw != cut && blockIdx.x % (C * G) == 0 && threadIdx.x == 0) report_status(p.status, CHRONOS_ERR_INVALID_ARG);
    const int len = p.cu == nullptr ? cut : static_cast<int>(max(int64_t{0}, cut - (static_cast<int64_t>(p.cu[seq + 1]) - (t0 + n))));
    const int most = (len + p.c.page_size - 1) / p.c.page_size;
    unsigned long long* keys = p.keys + ((t0 - p.token0) * G + g) * p.width;   // of token t: t * G * width on
    auto pages_of = [&](int t) { return TOKENS == 1 ? most : (max(len - (n - 1 - t), 0) + p.c.page_size - 1) / p.c.page_size; };
    if (most > p.topk) {   // (else all pages are taken: no scores)
        const int D64 = (D + 63) & ~63;
        for (int i = threadIdx.x; i < n * D64; i += kSelectThreads) {
            const int t = i / D64, d = i % D64;
            double up = 0.0, down = 0.0;
            if (d < D) {
                const T* q = static_cast<const T*>(p.q) + (t0 + t) * p.q_row + static_cast<int64_t>(g) * p.rep * p.q_head + d;
#pragma unroll 4
                for (int h = 0; h < p.rep; ++h) {
                    const float x = to_f32<T>(q[h * p.q_head]);
                    if (x > 0.0f) up += x;
                    else down += x;   // and NaN
                }
            }
            const int at = 2 * (((d >> 6) * 4 + ((d & 7) >> 1)) * 8 + ((d >> 3) & 7)) + (d & 1);
            reinterpret_cast<double*>(s_q[t][0])[at] = down;
            reinterpret_cast<double*>(s_q[t][1])[at] = up;
        }
        const int part = threadIdx.x & 7, group = threadIdx.x >> 3;
        // rounds of ROUND pages go to the blocks in turn, kSelectPages / ROUND rounds of this block at a time
        constexpr int ROUNDS = kSelectPages / ROUND;
        for (int r0 = 0; (r0 * C + rank) * ROUND < most; r0 += ROUNDS) {
            if (r0 > 0) __syncthreads();   // the numbers before are read
            for (int i = threadIdx.x; i < kSelectPages; i += kSelectThreads) {
                const int64_t j = (static_cast<int64_t>(r0 + i / ROUND) * C + rank) * ROUND + i % ROUND;
                int page = -1;
                if (j < most) {
                    page = p.c.page_table[seq * p.c.page_table_stride + j];
                    if (page < 0 || page >= p.c.num_pages) {
                        report_status(p.status, CHRONOS_ERR_INVALID_ARG);
                        page = -1;
                    }
                }
                s_page[i] = page;
            }
            __syncthreads();
            for (int r = 0; r < ROUNDS && ((r0 + r) * C + rank) * ROUND < most; ++r) {
                const int j0 = ((r0 + r) * C + rank) * ROUND + group;
                double acc[TOKENS][PAGES];
                int page[PAGES];
#pragma unroll
                for (int k = 0; k < PAGES; ++k) {
                    page[k] = s_page[r * ROUND + k * GROUPS + group];
#pragma unroll
                    for (int t = 0; t < TOKENS; ++t) acc[t][k] = 0.0;
                }
                for (int c0 = 0; c0 * 64 < D; c0 += CHUNKS) {
                    RopeRow<T, VEC> x[PAGES][2][CHUNKS];   // page, lo or hi, 64 columns
#pragma unroll
                    for (int k = 0; k < PAGES; ++k)
#pragma unroll
                        for (int w = 0; w < 2; ++w)
#pragma unroll
                            for (int c = 0; c < CHUNKS; ++c) {
                                const int d = (c0 + c) * 64 + part * 8;
                                const T* row = static_cast<const T*>(p.bounds) + ((static_cast<int64_t>(page[k]) * 2 + w) * G + g) * D;
                                x[k][w][c].load(row, d, page[k] >= 0 && d < D, D, 0, 0);
                            }
#pragma unroll
                    for (int c = 0; c < CHUNKS; ++c) {
                        if ((c0 + c) * 64 >= D) break;
#pragma unroll
                        for (int w = 0; w < 2; ++w) {
                            float a[PAGES][8];
#pragma unroll
                            for (int k = 0; k < PAGES; ++k) x[k][w][c].values(a[k]);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                double v[PAGES][2];
#pragma unroll
                                for (int k = 0; k < PAGES; ++k) {
                                    v[k][0] = a[k][2 * e];
                                    v[k][1] = a[k][2 * e + 1];
                                }
#pragma unroll
                                for (int t = 0; t < TOKENS; ++t) {
                                    if (TOKENS > 1 && t >= n) break;
                                    const double2 q = s_q[t][w][((c0 + c) * 4 + e) * 8 + part];
#pragma unroll
                                    for (int k = 0; k < PAGES; ++k) acc[t][k] = fma(q.y, v[k][1], fma(q.x, v[k][0], acc[t][k]));
                                }
                            }
                        }
                    }
                }
#pragma unroll
                for (int t = 0; t < TOKENS; ++t) {
                    if (TOKENS > 1 && t >= n) break;
                    const int pages = pages_of(t);
#pragma unroll
                    for (int k = 0; k < PAGES; ++k) {
                        double x = acc[t][k];
#pragma unroll
                        for (int o = 1; o < 8; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
                        const int j = j0 + k * GROUPS;
                        if (part == 0 && j < pages) keys[t * G * p.width + j] = page[k] < 0 ? 0ull : select_key(x);
                    }
                }
            }
        }
    }
    // every block's keys are written (they are read from global memory, by blocks of this cluster only)
    if (C > 1) cooperative_groups::this_cluster().sync();
    else __syncthreads();
    for (int t = rank; t < n; t += C) {
        select_row<T>(p, s_sel, s_keys, keys + t * G * p.width, p.pages + ((t0 + t) * G + g) * p.topk, pages_of(t), t0 + t, g, seq);
        __syncthreads();   // the next one writes where this one reads
    }
}

}  // namespace chronos
