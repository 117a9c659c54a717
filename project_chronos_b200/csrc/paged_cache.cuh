// paged_cache.cuh — the append that fills the pages of the key-value cache and the
// eviction that empties them (include/chronos_paged.h).
#pragma once

#include "chronos_paged.h"
#include "common.cuh"
#include "paged.cuh"

namespace chronos {

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
struct PagedAppendParams {
    ChronosPagedCache c;
    int64_t tokens;
    const void* k;
    const void* v;
    int64_t k_row, k_head, v_row, v_head;
    const int32_t* cu;
    const int32_t* seen;
    float* weights;
    int32_t* positions;
    int64_t slot_cap;
    int max_slots;
    int32_t* lens_out;
    int32_t* seen_out;
    int32_t* status;
};

constexpr int kAppendThreads = 256;

// Sequence b's new length: `stored` tokens were.  One lane calls it, after the whole warp
// has read the sequence's old ones.
__device__ __forceinline__ void paged_advance(const PagedAppendParams& p, int b, int stored) {
    if (p.lens_out != nullptr) p.lens_out[b] = p.c.lens[b] + stored;
    if (p.seen_out != nullptr) p.seen_out[b] = p.seen[b] + stored;
}

// Copies: 4 * G * D * size bytes of traffic per token.  One warp per token: it
// finds the sequence with one ballot per 32 offsets, then its lanes copy the
// token's K and V rows in units of V bytes (16, or one element where the
// strides forbid more), four loads in flight before the first store.  8 prompts of up
// to 8192 tokens, 8 heads of 128 in bf16: 57 us, 5.6 TB/s read and written.
// Without offsets a warp has a sequence to itself and advances its length, too.
template <typename V>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const __grid_constant__ PagedAppendParams p,
                                                                      int units_per_head, int elems_per_unit) {
    const int lane = threadIdx.x & 31;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * (kAppendThreads / 32);
    const int G = p.c.kv_heads, n = G * units_per_head;
    for (int64_t t = static_cast<int64_t>(blockIdx.x) * (kAppendThreads / 32) + (threadIdx.x >> 5); t < p.tokens; t += warps) {
        int b = 0;
        int64_t i = 0;
        if (p.cu == nullptr) {
            b = static_cast<int>(t);
        } else {
            // sequences whose end is <= t come before token t's (ends ascend)
            for (int base = 0; base < p.c.batch; base += 32) {
                const bool before = base + lane < p.c.batch && p.cu[base + lane + 1] <= t;
                const int cnt = __popc(__ballot_sync(0xffffffffu, before));
                b += cnt;
                if (cnt < 32) break;
            }
            if (b >= p.c.batch) continue;   // a row behind the last sequence
            i = t - p.cu[b];
            if (i < 0) continue;
        }
        const int64_t slot = p.c.lens[b] + i;
        const bool fits = slot >= 0 && slot < p.max_slots;
        const int page = fits ? p.c.page_table[b * p.c.page_table_stride + slot / p.c.page_size] : -1;
        if (page < 0 || page >= p.c.num_pages) {
            if (p.cu == nullptr) __syncwarp();
            if (lane == 0) {
                report_status(p.status, CHRONOS_ERR_INVALID_ARG);
                if (p.cu == nullptr) paged_advance(p, b, 0);
            }
            continue;
        }
        const int64_t in_page = slot % p.c.page_size;
        const char* ks = static_cast<const char*>(p.k);
        const char* vs = static_cast<const char*>(p.v);
        char* kd = static_cast<char*>(p.c.k_pages);
        char* vd = static_cast<char*>(p.c.v_pages);
        const int es = static_cast<int>(sizeof(V)) / elems_per_unit;
        for (int u0 = lane; u0 < n; u0 += 64) {
            V x[4];
            int64_t dk[2], dv[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int u = u0 + 32 * j;
                if (u < n) {
                    const int64_t g = u / units_per_head, e = static_cast<int64_t>(u % units_per_head) * elems_per_unit;
                    x[2 * j] = *reinterpret_cast<const V*>(ks + (t * p.k_row + g * p.k_head + e) * es);
                    x[2 * j + 1] = *reinterpret_cast<const V*>(vs + (t * p.v_row + g * p.v_head + e) * es);
                    dk[j] = (page * p.c.k_page_stride + in_page * p.c.k_slot_stride + g * p.c.k_head_stride + e) * es;
                    dv[j] = (page * p.c.v_page_stride + in_page * p.c.v_slot_stride + g * p.c.v_head_stride + e) * es;
                }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
                if (u0 + 32 * j < n) {
                    *reinterpret_cast<V*>(kd + dk[j]) = x[2 * j];
                    *reinterpret_cast<V*>(vd + dv[j]) = x[2 * j + 1];
                }
        }
        for (int g = lane; g < G; g += 32) {
            const int64_t at = (static_cast<int64_t>(b) * G + g) * p.slot_cap + slot;
            if (p.weights != nullptr) p.weights[at] = 0.0f;
            if (p.positions != nullptr) p.positions[at] = static_cast<int32_t>(p.seen[b] + i);
        }
        if (p.cu == nullptr) {
            __syncwarp();
            if (lane == 0) paged_advance(p, b, 1);
        }
    }
}

// The lengths after a packed append, one warp per sequence: its tokens up to the first that
// had no slot or no page (the pages its new slots lie in, 32 at a time).
__global__ void __launch_bounds__(kAppendThreads) paged_advance_kernel(const __grid_constant__ PagedAppendParams p) {
    const int lane = threadIdx.x & 31;
    const int b = blockIdx.x * (kAppendThreads / 32) + (threadIdx.x >> 5);
    if (b >= p.c.batch) return;
    pdl_wait();   // the rows are stored by the old lengths
    const int64_t first = p.cu[b], last = min(static_cast<int64_t>(p.cu[b + 1]), p.tokens);
    if (lane == 0 && (first < 0 || p.cu[b + 1] < first || p.cu[b + 1] > p.tokens)) report_status(p.status, CHRONOS_ERR_INVALID_ARG);
    const int64_t from = p.c.lens[b], size = p.c.page_size;
    int64_t n = from >= 0 && first >= 0 ? max(int64_t{0}, min(last - first, p.max_slots - from)) : 0;
    if (n > 0)
        for (int64_t p0 = from / size; p0 * size < from + n; p0 += 32) {
            const int64_t at = p0 + lane;
            bool none = false;
            if (at * size < from + n) {
                const int page = p.c.page_table[b * p.c.page_table_stride + at];
                none = page < 0 || page >= p.c.num_pages;
            }
            const uint32_t gone = __ballot_sync(0xffffffffu, none);
            if (gone) {
                n = max(int64_t{0}, (p0 + __ffs(gone) - 1) * size - from);
                break;
            }
        }
    __syncwarp();
    if (lane == 0) paged_advance(p, b, static_cast<int>(n));
}

// ---------------------------------------------------------------------------
// eviction
// ---------------------------------------------------------------------------
struct PagedEvictParams {
    ChronosPagedCache c;
    int budget, sinks, recent;
    const int32_t* seen;
    const float* weights;
    const int32_t* positions;
    float* weights_out;
    int32_t* positions_out;
    int64_t slot_cap;
    int32_t* lens_out;
    int32_t* src;
    int max_slots;
    int keys_in_smem;      // 1: a row's keys fit shared memory, else they are formed again from the inputs
    uint32_t* bits;        // [B * G][2][bit_words] for rows whose keys do not fit
    int64_t bit_words;
    int32_t* moves;        // [B * G][max_moves][2]: (slot given up, slot that moves there)
    int32_t* counts;       // [B * G]
    int32_t* lens_copy;    // [B] lens_out may be the caller's lens
    int64_t max_moves;
    int move_here;         // 1: the selecting block moves the rows (16-byte units) and writes lens_out
    int32_t* status;
};

// Slots beyond the budget up to which the selecting block moves the rows itself: 32 warps
// with four rows each.
constexpr int kEvictMovesHere = 128;
constexpr int kEvictThreads = 1024;
constexpr int kEvictWarps = kEvictThreads / 32;
constexpr int kEvictBins = 2048;   // 11 + 11 + 10 bits of the key

// A weight's place in the order of floats as an unsigned number: larger weights
// first, -0 as 0, NaN above every number; what is kept anyway above all.
__device__ __forceinline__ uint32_t evict_key(float w, int pos, int sinks, int64_t newest) {
    if (pos < sinks || pos >= newest) return 0xffffffffu;
    if (w != w) return 0xfffffffeu;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// The K and V rows of the moves, read once and written once: a warp takes four moves at
// a time (all four rows' loads in flight before the first store: 230 MB of K and V rows
// of 256 bytes in 45 us, 5.1 TB/s; one move at a time 53 us).  Sources (slots >=
// budget) and targets (slots < budget) never overlap, so the order does not matter.
template <typename V>
__device__ __forceinline__ void paged_move_rows(const PagedEvictParams& p, int b, int g, const int32_t* mv, int count,
                                                int warp, int warps, int lane, int units, int elems_per_unit) {
    constexpr int M = 4;
    const int32_t* table = p.c.page_table + b * p.c.page_table_stride;
    const int es = static_cast<int>(sizeof(V)) / elems_per_unit;
    char* kp = static_cast<char*>(p.c.k_pages);
    char* vp = static_cast<char*>(p.c.v_pages);
    for (int i0 = warp * M; i0 < count; i0 += warps * M) {
        // lanes 2m and 2m + 1: target and source of move m, as offsets of their K and V rows
        int64_t ko = 0, vo = 0;
        bool ok = false;
        if (lane < 2 * M && i0 + lane / 2 < count) {
            const int slot = mv[2 * i0 + lane];
            const int page = table[slot / p.c.page_size];
            const int64_t in = slot % p.c.page_size;
            ok = page >= 0 && page < p.c.num_pages;
            if (!ok) report_status(p.status, CHRONOS_ERR_INVALID_ARG);
            ko = (page * p.c.k_page_stride + in * p.c.k_slot_stride + g * p.c.k_head_stride) * es;
            vo = (page * p.c.v_page_stride + in * p.c.v_slot_stride + g * p.c.v_head_stride) * es;
        }
        const uint32_t good = __ballot_sync(0xffffffffu, ok);
        for (int u0 = 0; u0 < 2 * units; u0 += 32) {
            const int u = u0 + lane;
            const bool isv = u >= units;
            const int64_t e = static_cast<int64_t>(isv ? u - units : u) * elems_per_unit * es;
            V x[M];
            char* to[M];
#pragma unroll
            for (int m = 0; m < M; ++m) {
                const int64_t kt = __shfl_sync(0xffffffffu, ko, 2 * m), kf = __shfl_sync(0xffffffffu, ko, 2 * m + 1);
                const int64_t vt = __shfl_sync(0xffffffffu, vo, 2 * m), vf = __shfl_sync(0xffffffffu, vo, 2 * m + 1);
                to[m] = nullptr;
                if (u < 2 * units && ((good >> (2 * m)) & 3u) == 3u) {
                    to[m] = (isv ? vp + vt : kp + kt) + e;
                    x[m] = *reinterpret_cast<const V*>((isv ? vp + vf : kp + kf) + e);
                }
            }
#pragma unroll
            for (int m = 0; m < M; ++m)
                if (to[m] != nullptr) *reinterpret_cast<V*>(to[m]) = x[m];
        }
    }
}

// Sum of the values that the warps before this one left in x[kEvictWarps] (whole warps
// call it; `total`: of all warps).
__device__ __forceinline__ int evict_before(const int* x, int warp, int lane, int* total = nullptr) {
    const int v = x[lane];
    int inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += t;
    }
    if (total != nullptr) *total = __shfl_sync(0xffffffffu, inc, 31);
    return __shfl_sync(0xffffffffu, inc - v, warp);
}

// One block per (sequence, kv head).  The budget-th largest key by radix
// selection (three counting passes over 11, 11 and 10 bits, counters in shared
// memory, the first pass while the keys are formed), then one bit per slot for
// what is kept, and scans of their counts, which give every hole and every slot that
// moves its rank.  Bound by latency: a row's 8 bytes per slot
// pass one SM (64 rows of 2049 slots 10 us, of up to 32768 slots 36 us).
__global__ void __launch_bounds__(kEvictThreads) paged_evict_select_kernel(const __grid_constant__ PagedEvictParams p,
                                                                              int units, int elems_per_unit) {
    extern __shared__ uint32_t s_keys[];   // [max_slots] when keys_in_smem
    __shared__ int s_hist[3][kEvictBins];
    __shared__ int s_a[3][kEvictWarps], s_b[kEvictWarps];
    __shared__ int s_digit[3], s_above[3];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row = blockIdx.x, b = row / p.c.kv_heads;
    const int raw = p.c.lens[b];
    const int64_t newest = static_cast<int64_t>(p.seen[b]) - p.recent;
    const int n = min(max(raw, 0), p.max_slots);
    if (threadIdx.x == 0 && raw != n) report_status(p.status, CHRONOS_ERR_INVALID_ARG);
    const int64_t base = row * p.slot_cap;
    const float* w = p.weights + base;
    const int32_t* pos = p.positions + base;
    int32_t* src = p.src + static_cast<int64_t>(row) * p.budget;
    if (row % p.c.kv_heads == 0 && threadIdx.x == 0) {
        if (p.move_here) p.lens_out[b] = min(n, p.budget);
        else p.lens_copy[b] = n;
    }
    if (n <= p.budget) {
        for (int j = threadIdx.x; j < p.budget; j += kEvictThreads) src[j] = j < n ? j : -1;
        for (int j = threadIdx.x; j < n; j += kEvictThreads) {
            const float a = w[j];
            const int c = pos[j];
            p.weights_out[base + j] = a;
            p.positions_out[base + j] = c;
        }
        if (threadIdx.x == 0) p.counts[row] = 0;
        return;
    }
    auto key = [&](int j) -> uint32_t {
        return p.keys_in_smem ? s_keys[j] : evict_key(w[j], pos[j], p.sinks, newest);
    };
    for (int i = threadIdx.x; i < 3 * kEvictBins; i += kEvictThreads) (&s_hist[0][0])[i] = 0;
    __syncthreads();
    auto first = [&](int j, float a, int c) {
        const uint32_t k = evict_key(a, c, p.sinks, newest);
        if (p.keys_in_smem) s_keys[j] = k;
        atomicAdd(&s_hist[0][k >> 21], 1);
    };
    const bool vec = (p.slot_cap & 3) == 0 &&
                     ((reinterpret_cast<uintptr_t>(p.weights) | reinterpret_cast<uintptr_t>(p.positions)) & 15) == 0;
    const int whole = vec ? n / 4 : 0;
#pragma unroll 4
    for (int i = threadIdx.x; i < whole; i += kEvictThreads) {
        const float4 a = reinterpret_cast<const float4*>(w)[i];
        const int4 c = reinterpret_cast<const int4*>(pos)[i];
        first(4 * i, a.x, c.x);
        first(4 * i + 1, a.y, c.y);
        first(4 * i + 2, a.z, c.z);
        first(4 * i + 3, a.w, c.w);
    }
    for (int j = 4 * whole + threadIdx.x; j < n; j += kEvictThreads) first(j, w[j], pos[j]);
    // radix selection: `prefix` the digits found, `want` the rank still to find below it
    uint32_t prefix = 0, known = 0;
    int want = p.budget;
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
        const uint32_t mask = (1u << bits) - 1u;
        if (pass > 0)
            for (int j = threadIdx.x; j < n; j += kEvictThreads) {
                const uint32_t k = key(j);
                if ((k & known) == prefix) atomicAdd(&s_hist[pass][(k >> shift) & mask], 1);
            }
        __syncthreads();
        // digit d such that fewer than `want` keys lie above it, and with it at least `want`:
        // thread i holds the two highest digits not yet held by threads before it
        const int d0 = kEvictBins - 1 - 2 * threadIdx.x;
        const int h0 = s_hist[pass][d0], h1 = s_hist[pass][d0 - 1];
        int inc = h0 + h1;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, inc, x);
            if (lane >= x) inc += t;
        }
        if (lane == 31) s_a[pass][warp] = inc;
        __syncthreads();
        const int above = inc - h0 - h1 + evict_before(s_a[pass], warp, lane);
        if (above < want && above + h0 >= want) {
            s_digit[pass] = d0;
            s_above[pass] = above;
        } else if (above + h0 < want && above + h0 + h1 >= want) {
            s_digit[pass] = d0 - 1;
            s_above[pass] = above + h0;
        }
        __syncthreads();
        prefix |= static_cast<uint32_t>(s_digit[pass]) << shift;
        known |= mask << shift;
        want -= s_above[pass];
    }
    // kept: keys above `prefix`, and the first `want` slots whose key equals it.  One pass over
    // the keys leaves both as bits; from there on a thread owns contiguous words of 32 slots.
    const int words = (n + 31) / 32;
    uint32_t* more = p.keys_in_smem ? reinterpret_cast<uint32_t*>(&s_hist[0][0])
                                    : p.bits + static_cast<int64_t>(row) * 2 * p.bit_words;
    uint32_t* same = more + (p.keys_in_smem ? 3 * kEvictBins / 2 : p.bit_words);
#pragma unroll 4
    for (int j = warp * 32 + lane; j - lane < n; j += kEvictThreads) {
        const bool in = j < n;
        const uint32_t k = key(min(j, n - 1));
        const uint32_t gt = __ballot_sync(0xffffffffu, in && k > prefix), eq = __ballot_sync(0xffffffffu, in && k == prefix);
        if (lane == 0) {
            more[j >> 5] = gt;
            same[j >> 5] = eq;
        }
    }
    __syncthreads();
    const int per = (words + kEvictThreads - 1) / kEvictThreads;
    const int w0 = min(words, static_cast<int>(threadIdx.x) * per), w1 = min(words, w0 + per);
    // exclusive prefix of a thread's count, over the block
    auto before = [&](int mine, int* x, int* total) {
        int inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += t;
        }
        if (lane == 31) x[warp] = inc;
        __syncthreads();
        return inc - mine + evict_before(x, warp, lane, total);
    };
    int eq = 0;
    for (int i = w0; i < w1; ++i) eq += __popc(same[i]);
    int rank = before(eq, s_a[0], nullptr);
    int holes = 0, movers = 0, count = 0;
    for (int i = w0; i < w1; ++i) {
        uint32_t take = same[i];
        const int room = max(0, want - rank);
        rank += __popc(take);
        while (__popc(take) > room) take &= ~(0x80000000u >> __clz(take));   // the lower slots first
        const uint32_t keep = more[i] | take, low = ones_below(p.budget - 32 * i);
        more[i] = keep;
        holes += __popc(~keep & low & ones_below(n - 32 * i));
        movers += __popc(keep & ~low);
    }
    int h = before(holes, s_a[1], &count), m = before(movers, s_b, nullptr);
    int32_t* mv = p.moves + static_cast<int64_t>(row) * p.max_moves * 2;
    for (int i = w0; i < w1; ++i) {
        const uint32_t keep = more[i], low = ones_below(p.budget - 32 * i);
        for (uint32_t x = ~keep & low & ones_below(n - 32 * i); x; x &= x - 1) mv[2 * h++] = 32 * i + __ffs(x) - 1;
        for (uint32_t x = keep & ~low; x; x &= x - 1) mv[2 * m++ + 1] = 32 * i + __ffs(x) - 1;
    }
#pragma unroll 4
    for (int j = threadIdx.x; j < p.budget; j += kEvictThreads) {
        src[j] = j;
        if (p.weights_out != p.weights) p.weights_out[base + j] = w[j];
        if (p.positions_out != p.positions) p.positions_out[base + j] = pos[j];
    }
    if (threadIdx.x == 0) p.counts[row] = count;
    __syncthreads();   // the lists and the copies above are written
#pragma unroll 4
    for (int i = threadIdx.x; i < count; i += kEvictThreads) {
        const int2 move = reinterpret_cast<const int2*>(mv)[i];
        src[move.x] = move.y;
        p.weights_out[base + move.x] = w[move.y];
        p.positions_out[base + move.x] = pos[move.y];
    }
    if (p.move_here) paged_move_rows<uint4>(p, b, row % p.c.kv_heads, mv, count, warp, kEvictWarps, lane, units, elems_per_unit);
}

constexpr int kEvictMoveThreads = 256;
constexpr int kEvictMovesPerBlock = kEvictMoveThreads / 32 * 4;

template <typename V>
__global__ void __launch_bounds__(kEvictMoveThreads) paged_evict_move_kernel(const __grid_constant__ PagedEvictParams p,
                                                                             int units, int elems_per_unit) {
    const int row = blockIdx.z * gridDim.y + blockIdx.y, b = row / p.c.kv_heads, g = row % p.c.kv_heads;
    if (b >= p.c.batch) return;
    pdl_wait();
    if (g == 0 && blockIdx.x == 0 && threadIdx.x == 0) p.lens_out[b] = min(p.lens_copy[b], p.budget);
    paged_move_rows<V>(p, b, g, p.moves + static_cast<int64_t>(row) * p.max_moves * 2, p.counts[row],
                       blockIdx.x * (kEvictMoveThreads / 32) + (threadIdx.x >> 5), gridDim.x * (kEvictMoveThreads / 32),
                       threadIdx.x & 31, units, elems_per_unit);
}

}  // namespace chronos
