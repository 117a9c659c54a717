// paged_rope.cuh — rows into the pages of the key-value cache with the rotation of
// queries and keys on the way, into pages of the layer type or of 4-bit values, and
// rows back out of the pages (include/chronos_paged4.h).
//
// Bound by HBM for prompts (every row read once, written once) and by latency for one
// token per sequence.  A warp owns a token, or a slice of its rows where tokens are few:
// the angles of its columns stay in registers for all heads, a lane holds 8 columns, so a
// row of 128 takes half a warp.  8 prompts up to 8192 tokens, 32 / 8 heads of 128 in bf16: 154 us,
// 6.3 TB/s read and written (partner columns by a second load, two rows in flight: 375 us); 32 rows of
// one token 3.0 us.
//
// 4-bit rows: 193 instructions per 256 values of K, V and q bound them (77 % of issue slots, DRAM 36 % busy;
// 8 prompts up to 4096 tokens, 16 / 8 heads of 128 in fp16 75 us for 244 MB).  The code of a value and the scale of a block are decided as exact
// arithmetic decides: the fp32 value y is off by at most 2^-22 (|x c| + |x' s|), so a
// code (scale) is taken where the values that much above and below it give the same
// one, and computed in 64 bits where they do not (of rotated normal values about one block of 16 in
// 2000, so about one unit of a warp, 16 blocks, in 125: a step of 128 rows and 8 kv heads has some).  Values that
// are exact in 16 bits (v, columns that are not rotated) lie on a border or at least 2^-13
// of a scale away from it: there y / scale is rounded to 2^-17, which restores what lay on it.
#pragma once

#include "chronos_paged4.h"
#include "fp4.cuh"
#include "paged.cuh"

namespace chronos {

struct PagedRopeParams {
    ChronosPagedCache c;
    int64_t tokens;
    int heads;                  // query heads, 0 without queries
    int dim, start, table_len;  // rotated columns, where they begin, rows of the tables
    int columns;                // packed: stored columns of a slot
    const void* k;
    const void* v;
    const void* q;
    void* q_out;
    void* k_out;
    int64_t k_row, k_head, v_row, v_head, q_row, q_head, qo_row, qo_head, ko_row, ko_head;
    const void* cos;
    const void* sin;
    int64_t cos_row, sin_row;
    const int32_t* cu;
    const int32_t* seen;
    float* weights;
    int32_t* positions;
    int64_t slot_cap;
    int max_slots;
    int32_t* lens_out;
    int32_t* seen_out;
    float k_unit, v_unit;       // 1 / k_scale, 1 / v_scale in fp32
    float k_scale, v_scale;
    int k_exact, v_exact;       // the scale is a power of two: x / scale is exact
    int slices;                 // warps per token: 1, 2, 4 or 8
    int32_t* status;
};

constexpr int kRopeThreads = 256;
constexpr int kRopeWarps = kRopeThreads / 32;
constexpr int kRopeRing = 8;   // units of rows (512 bytes of 16-bit types) that a warp's ring holds

// Column that column d turns with (d itself where it is not rotated).
__device__ __forceinline__ int rope_partner(int d, int start, int dim) {
    const int j = d - start;
    return j < 0 || j >= dim ? d : j < dim / 2 ? d + dim / 2 : d - dim / 2;
}

// A lane's 8 columns of a row as they are loaded.  VEC: 16-byte words; else numbers, with the
// columns they turn with beside them.
template <typename T, bool VEC>
struct RopeRow {
    uint4 w[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* row, int col, bool on, int, int, int) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i)
            w[i] = on ? reinterpret_cast<const uint4*>(row + col)[i] : make_uint4(0u, 0u, 0u, 0u);
    }
    __device__ __forceinline__ void values(float (&x)[8]) const { load8<T>(reinterpret_cast<const T*>(w), x); }
    __device__ __forceinline__ void store(T* row, int col, int) const {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(row + col)[i] = w[i];
    }
    // Columns that lane `lane` has, zeros for those that do not turn.  Whole warps call it.
    __device__ __forceinline__ void partner(float (&x)[8], int lane, bool turns) const {
        RopeRow r;
        auto take = [&](uint32_t v) {
            const uint32_t g = __shfl_sync(0xffffffffu, v, lane);
            return turns ? g : 0u;
        };
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.w[i] = make_uint4(take(w[i].x), take(w[i].y), take(w[i].z), take(w[i].w));
        r.values(x);
    }
    __device__ __forceinline__ void read(uint32_t at) {   // from shared memory
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i)
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[i].x), "=r"(w[i].y), "=r"(w[i].z), "=r"(w[i].w) : "r"(at + i * 16));
    }
};
template <typename T>
struct RopeRow<T, false> {
    float x[8], with[8];
    __device__ __forceinline__ void load(const T* row, int col, bool on, int D, int start, int dim) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[j] = with[j] = 0.0f;
            if (on && col + j < D) {
                x[j] = to_f32<T>(row[col + j]);
                const int w = rope_partner(col + j, start, dim);
                if (w != col + j) with[j] = to_f32<T>(row[w]);
            }
        }
    }
    __device__ __forceinline__ void values(float (&v)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = x[j];
    }
    __device__ __forceinline__ void store(T* row, int col, int D) const {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (col + j < D) row[col + j] = from_f32<T>(x[j]);
    }
};
template <typename T, bool VEC>
__device__ __forceinline__ void rope_store(T* row, const float (&y)[8], int col, int D) {
    if constexpr (VEC) {
        store8<T>(row + col, y);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (col + j < D) row[col + j] = from_f32<T>(y[j]);
    }
}

// What a lane's 8 values are made of, for the computation in 64 bits: the row (NULL: zeros)
// and the angles of its position (NULL: not rotated).
template <typename T, typename TT>
struct RopeSource {
    const T* row;
    const TT* cos;
    const TT* sin;
    int col, D, start, dim;
    float scale;   // the cache's factor
    __device__ __forceinline__ double value(int j) const {
        const int d = col + j;
        if (row == nullptr || d >= D) return 0.0;
        double v = to_f32<T>(row[d]);
        const int w = cos != nullptr ? rope_partner(d, start, dim) : d;
        if (w != d) {
            const double turned = static_cast<double>(to_f32<T>(row[w])) * to_f32<TT>(sin[d - start]);
            v = v * to_f32<TT>(cos[d - start]) + (w > d ? -turned : turned);
        }
        return scale == 1.0f ? v : v / static_cast<double>(scale);
    }
};
// Codes and scale in 64 bits.  Whole warps call it.
template <typename T, typename TT>
__device__ __forceinline__ uint32_t fp4_block_exact(const RopeSource<T, TT>& src, uint32_t& scale) {
    double x[8], t = 0.0;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        x[j] = src.value(j);
        const double d = fabs(x[j]);
        bad |= !(d < INFINITY);
        t = fmax(t, d);
    }
    t = fmax(t, __shfl_xor_sync(0xffffffffu, t, 1));
    bad |= __shfl_xor_sync(0xffffffffu, bad ? 1 : 0, 1) != 0;
    const float t6 = static_cast<float>(t / 6.0);
    const uint32_t e = bad ? kFp8Nan : fp8_scales(t6, t6) & 0xffu;
    scale = e;
    if (bad || e == 0u) return 0u;
    const double z = fp8_value(e);
    uint32_t c = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const double d = x[j], m = fabs(d);
        const uint32_t level = (m > 0.25 * z) + (m >= 0.75 * z) + (m > 1.25 * z) + (m >= 1.75 * z) + (m > 2.5 * z) +
                               (m >= 3.5 * z) + (m > 5.0 * z);
        c |= (level | (signbit(d) ? 8u : 0u)) << (4 * j);
    }
    return c;
}

// Codes of a lane's 8 values y (in units of the cache's factor; top: the largest magnitude, NaN
// where one is) and the scale of its block of 16 (two lanes).  off: no value of the lane is off by more than 2^-22 off; 0 where all are
// what they are.  open: the block has to be decided in 64 bits (codes and scale are then not).  Whole warps call it.
template <typename T>
__device__ __forceinline__ uint32_t fp4_block(const float (&y)[8], float top, float off, uint32_t& scale, bool& open) {
    // here and in what follows: NaN where one of the 16 is
    const float a = max_magnitude(top, __shfl_xor_sync(0xffffffffu, top, 1));
    const bool exact = off == 0.0f;
    off = fmaxf(off, __shfl_xor_sync(0xffffffffu, off, 1));
    const bool finite = a < INFINITY;
    // exact magnitudes are divided as they are (16-bit ones lie on the middle of two scales or at
    // least 2^-12 of it away: rounding the quotient to 15 bits restores what lay there); the others
    // open the scale where a little more or less of them gives another one
    uint32_t two;
    if (off != 0.0f) {
        const float a6 = a * (1.0f / 6.0f), d6 = fmaxf(off, a) * 0x1p-21f;
        two = fp8_scales(fmaxf(a6 - d6, 0.0f), a6 + d6);
    } else {
        float a6;
        if constexpr (sizeof(T) == 2) a6 = __uint_as_float((__float_as_uint(a * (1.0f / 6.0f)) + 0x80u) & 0xffffff00u);
        else a6 = a / 6.0f;
        two = fp8_scales(a6, a6);
    }
    const float s = fp8_value(two);
    const float r = s > 0.0f ? reciprocal(s) : 0.0f;
    uint32_t codes;
    open = (two & 0xffu) != two >> 8;
    float u[8];
    if (sizeof(T) == 2 && exact) {
        // 96 + 2^-17 z: values of 64 to 128 have 17 bits behind the point
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = copysignf(fmaf(y[j], r, 96.0f) - 96.0f, y[j]);
        codes = fp4_codes(u);
    } else {
        const float d = exact ? 0.0f : fmaxf(off, a) * r * 0x1p-21f;   // with what r and the product are off 7 of these 8 times 2^-24; exact: zeros
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = fmaf(y[j], r, -d);
        codes = fp4_codes(u);
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = fmaf(y[j], r, d);
        // a sign that differs is one of values next to zero: decided like the codes
        open |= codes != fp4_codes(u);
    }
    scale = two & 0xffu;
    // NaN and infinities of the inputs, or finite values that pass fp32 on the way (a sum of the
    // rotation, a quotient by a small factor): 64 bits tell which
    open |= !finite;
    codes = finite && scale != 0u ? codes : 0u;
    if (!finite) scale = kFp8Nan;
    return codes;
}

// Where a slot's codes of the columns from `col` on lie in its record (the first of 16), and their scale.
__device__ __forceinline__ int fp4_codes_at(int line, int col, int columns) { return line * (columns / 2) + col / 2; }
__device__ __forceinline__ int fp4_scale_at(int line, int col, int columns) { return 8 * columns + line * (columns / 16) + col / 16; }

// A token's place in the pages and its position.
struct RopePlace {
    int t, page, in_page;
    int64_t at;
    bool placed;
};
// What a warp's rows of 4 bits leave to the end: units (again: bits n % 32 of K's, of V's) with blocks that are
// decided in 64 bits, and the rows of k_out, which may be k.  Not inlined: its registers stay out of the
// common path.  Whole warps call it.
template <typename T, typename TT, int LPR, bool VEC>
__device__ __noinline__ void rope4_rest(const PagedRopeParams& p, const RopePlace w, int slice, int slice_v, uint32_t again_k, uint32_t again_v) {
    constexpr int RPW = 32 / LPR;
    const int lane = threadIdx.x & 31, sub = lane / LPR, col = lane % LPR * 8, G = p.c.kv_heads, D = p.c.head_dim;
    const int uk = (G + RPW - 1) / RPW;
    const bool turned = p.dim > 0 && w.placed;
    const TT* cos = static_cast<const TT*>(p.cos) + w.at * p.cos_row;
    const TT* sin = static_cast<const TT*>(p.sin) + w.at * p.sin_row;
    for (int of_v = 0; of_v < 2; ++of_v) {
        const uint32_t again = of_v ? again_v : again_k;
        if (again == 0u) continue;
        const T* src = of_v ? static_cast<const T*>(p.v) + w.t * p.v_row : static_cast<const T*>(p.k) + w.t * p.k_row;
        uint8_t* to = (of_v ? static_cast<uint8_t*>(p.c.v_pages) + w.page * p.c.v_page_stride : static_cast<uint8_t*>(p.c.k_pages) + w.page * p.c.k_page_stride) +
                      static_cast<int64_t>(w.in_page >> 4) * fp4_record(p.columns);
        const int64_t from_head = of_v ? p.v_head : p.k_head, to_head = of_v ? p.c.v_head_stride : p.c.k_head_stride;
        for (int u = of_v ? slice_v : slice, n = 0; u < uk; u += p.slices, ++n) {
            if (((again >> (n & 31)) & 1u) == 0u) continue;
            const int row = u * RPW + sub;
            const RopeSource<T, TT> exact{row < G ? src + row * from_head : nullptr, turned && !of_v ? cos : nullptr, sin, col, D, p.start, p.dim,
                                          of_v ? p.v_scale : p.k_scale};
            uint32_t scale;
            const uint32_t codes = fp4_block_exact<T, TT>(exact, scale);
            if (row < G && col < p.columns) {
                uint8_t* record = to + row * to_head;
                *reinterpret_cast<uint32_t*>(record + fp4_codes_at(w.in_page & 15, col, p.columns)) = codes;
                if ((col & 8) == 0) record[fp4_scale_at(w.in_page & 15, col, p.columns)] = static_cast<uint8_t>(scale);
            }
        }
    }
    if (p.k_out == nullptr) return;
    __syncwarp();   // the rows are read
    for (int u = slice; u < uk; u += p.slices) {
        const int row = u * RPW + sub;
        const bool has = row < G && col < D;
        const T* k = static_cast<const T*>(p.k) + w.t * p.k_row + row * p.k_head;
        T* out = static_cast<T*>(p.k_out) + w.t * p.ko_row + row * p.ko_head;
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            y[j] = 0.0f;
            const int d = col + j;
            if (!has || d >= D || !w.placed) continue;
            y[j] = to_f32<T>(k[d]);
            const int with = rope_partner(d, p.start, p.dim), r = d - p.start;
            if (with != d) {
                const float s = to_f32<TT>(sin[r]);
                y[j] = fmaf(y[j], to_f32<TT>(cos[r]), to_f32<T>(k[with]) * (with > d ? -s : s));
            }
        }
        __syncwarp();
        if (has) rope_store<T, VEC>(out, y, col, D);
    }
}

// LPR lanes hold a row (8 columns each).  VEC: rows, halves and tables can be read 8
// columns at a time.  Rows of 16-bit types then come through a ring in shared memory, so that all of a
// token's are on their way at once (loads next to their uses left warps waiting for memory 43 % of the
// time: 4-bit prompts and their rows back 112 us for 100); fp32 rows, twice the bytes per unit, come one unit ahead in registers
// (24 chunks up to 257 tokens: 12.3 us for 14.2 through the ring).
template <typename T, typename TT, int LPR, bool VEC, bool PACKED>
__global__ void __launch_bounds__(kRopeThreads, !VEC ? 1 : PACKED && sizeof(T) == 4 ? 2 : 3) paged_rope_kernel(const __grid_constant__ PagedRopeParams p) {
    constexpr int RPW = 32 / LPR;                       // rows of a warp at once: a unit
    constexpr int W = sizeof(T) / 2;                    // 16-byte words of 8 columns (VEC)
    constexpr int UNIT = W * 512, NS = kRopeRing;
    constexpr bool RING = VEC && W == 1;
    extern __shared__ __align__(16) uint4 s_ring[];     // [warp][NS][UNIT / 16]
    __shared__ uint4 s_zero;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int slice = warp & (p.slices - 1), shift = __popc(p.slices - 1);
    const int t = static_cast<int>(blockIdx.x) * (kRopeWarps >> shift) + (warp >> shift);   // (tokens are below 2^28)
    const int G = p.c.kv_heads, D = p.c.head_dim;
    const int sub = lane / LPR, col = lane % LPR * 8;
    const bool on = col < D;
    // units of one kind: this warp's rows begin at `sub + slice * RPW` and lie `step` apart
    const int uk = (G + RPW - 1) / RPW, uq = (p.heads + RPW - 1) / RPW, step = p.slices * RPW;
    const int row0 = slice * RPW + sub;
    // V's begin half the warps further: where a token's rows of a kind are fewer than its warps, others take them
    const int slice_v = (slice + p.slices / 2) & (p.slices - 1), row0_v = slice_v * RPW + sub;
    const T* src_k = static_cast<const T*>(p.k) + t * p.k_row;
    const T* src_v = static_cast<const T*>(p.v) + t * p.v_row;
    const T* src_q = static_cast<const T*>(p.q) + t * p.q_row;
    // this warp's units: nk of K, then nv of V, then nq of Q (slices is a power of two)
    const bool some = t < p.tokens;
    const int nk = some ? (uk - slice + p.slices - 1) >> shift : 0, nv = some ? (uk - slice_v + p.slices - 1) >> shift : 0,
              nq = some ? (uq - slice + p.slices - 1) >> shift : 0;
    const uint32_t ring = smem_u32(s_ring) + warp * NS * UNIT, mine = ring + lane * 16;
    // Where unit m's rows begin for this lane (NULL: it has none of them).
    auto source = [&](int m) -> const T* {
        const T* src = src_k;
        int row = row0, rows = G;
        int64_t head = p.k_head;
        if (m >= nk + nv) {
            m -= nk + nv;
            src = src_q, row = row0, rows = m < nq ? p.heads : 0, head = p.q_head;
        } else if (m >= nk) {
            m -= nk;
            src = src_v, row = row0_v, head = p.v_head;
        }
        row += m * step;
        return on && row < rows ? src + row * head : nullptr;
    };
    auto issue = [&](int m) {
        if constexpr (RING) {
            if (m < nk + nv + nq)
                if (const T* row = source(m)) cp_async16(mine + (m & (NS - 1)) * UNIT, row + col, true);
            cp_async_commit();
        }
    };
    // the first rows are on their way while the token's place is looked up
    RopeRow<T, VEC> ahead;   // fp32: the next unit
    if constexpr (RING) {
#pragma unroll
        for (int m = 0; m < NS - 1; ++m) issue(m);
        if (!on)   // columns behind the row's end
#pragma unroll
            for (int i = 0; i < NS; ++i) s_ring[(warp * NS + i) * 32 + lane] = make_uint4(0u, 0u, 0u, 0u);
        if (lane == 0) s_zero = make_uint4(0u, 0u, 0u, 0u);   // (every warp writes what it reads)
    } else if constexpr (VEC) {
        const T* row = source(0);
        ahead.load(row, col, row != nullptr, D, 0, 0);
    }

    int b = -1, page = -1, in_page = 0;
    int64_t i = 0, slot = 0, at = 0;
    bool placed = false;    // at a position of the tables
    if (t < p.tokens) {
        b = p.cu == nullptr ? t : paged_sequence(p.cu, p.c.batch, t, lane);
        if (b >= p.c.batch) b = -1;   // a row behind the last sequence
        if (b >= 0 && p.cu != nullptr) {
            i = t - p.cu[b];
            if (i < 0) b = -1;
        }
    }
    if (b >= 0) {
        slot = p.c.lens[b] + i;
        at = p.seen != nullptr ? p.seen[b] + i : 0;
        placed = p.dim == 0 || (at >= 0 && at < p.table_len);
        if (placed && slot >= 0 && slot < p.max_slots) {
            const int size = p.c.page_size, j = static_cast<int>(slot) / size;
            in_page = static_cast<int>(slot) - j * size;
            page = p.c.page_table[b * p.c.page_table_stride + j];
        }
        if (page < 0 || page >= p.c.num_pages) {
            page = -1;
            if (lane == 0) report_status(p.status, CHRONOS_ERR_INVALID_ARG);
        }
    }
    if (p.cu == nullptr) {
        __syncthreads();   // every slice of a token has read its sequence's lengths
        if (b >= 0 && slice == 0 && lane == 0) {
            if (p.lens_out != nullptr) p.lens_out[b] = static_cast<int32_t>(slot) + (page >= 0 ? 1 : 0);
            if (p.seen_out != nullptr) p.seen_out[b] = static_cast<int32_t>(at) + (page >= 0 ? 1 : 0);
        }
    }
    if (b < 0) {
        cp_async_wait<0>();
        return;
    }
    if (slice == 0 && page >= 0 && (p.weights != nullptr || p.positions != nullptr))
        for (int g = lane; g < G; g += 32) {
            const int64_t w = (static_cast<int64_t>(b) * G + g) * p.slot_cap + slot;
            if (p.weights != nullptr) p.weights[w] = 0.0f;
            if (p.positions != nullptr) p.positions[w] = static_cast<int32_t>(at);
        }

    // angles of this lane's columns; the sine carries the sign of its half
    float cs[8], sn[8];
    bool turns = false;
    const TT* cos = static_cast<const TT*>(p.cos) + at * p.cos_row;
    const TT* sin = static_cast<const TT*>(p.sin) + at * p.sin_row;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        cs[j] = 1.0f;
        sn[j] = -0.0f;   // x c - 0 is x, its sign included
    }
    if (on && p.dim > 0 && placed) {
        if constexpr (VEC) {
            const int j = col - p.start;
            turns = j >= 0 && j < p.dim;
            if (turns) {
                load8<TT>(cos + j, cs);
                load8<TT>(sin + j, sn);
                if (j < p.dim / 2)
#pragma unroll
                    for (int e = 0; e < 8; ++e) sn[e] = -sn[e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int j = col + e - p.start;
                if (col + e < D && j >= 0 && j < p.dim) {
                    turns = true;
                    cs[e] = to_f32<TT>(cos[j]);
                    sn[e] = to_f32<TT>(sin[j]);
                    if (j < p.dim / 2) sn[e] = -sn[e];
                }
            }
        }
    }
    // where the columns these turn with are: in the unit another lane's, zeros for those that do not turn
    const int other = VEC ? lane - lane % LPR + rope_partner(col, p.start, turns ? p.dim : 0) / 8 : lane;
    uint32_t from = 0, from_stage = 0;
    if constexpr (RING) {
        from = turns ? ring + other * 16 : smem_u32(&s_zero);
        from_stage = turns ? UNIT : 0;
    }

    int m = 0;   // units taken
    // The next unit's rows (has: this lane's is one).
    auto next = [&](RopeRow<T, VEC>& x, const T* src, bool has) {
        if constexpr (RING) {
            __syncwarp();   // every lane has read the unit before
            issue(m + NS - 1);
            cp_async_wait<NS - 1>();
        } else if constexpr (VEC) {
            x = ahead;
            const T* row = source(m + 1);
            ahead.load(row, col, row != nullptr, D, 0, 0);
        } else {
            x.load(src, col, on && has, D, p.start, p.dim);
        }
        __syncwarp();   // (a row is read before it is written over: q_out may be q, k_out k)
        if constexpr (RING) x.read(mine + (m & (NS - 1)) * UNIT);
        ++m;
    };
    // ... of the unit taken last
    auto rotate = [&](const RopeRow<T, VEC>& x, float (&y)[8], float& most) {
        float w[8];
        x.values(y);
        if constexpr (VEC && !RING) {
            x.partner(w, other, turns);
        } else if constexpr (RING) {
            RopeRow<T, true> r;
            r.read(from + ((m - 1) & (NS - 1)) * from_stage);
            r.values(w);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = x.with[j];
        }
        most = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            w[j] *= sn[j];
            if constexpr (PACKED) most = fmaxf(most, fabsf(w[j]));
            y[j] = fmaf(y[j], cs[j], w[j]);
        }
    };
    // where this lane's part of the slot's first row lies
    const int line = in_page & 15;
    uint8_t *kp, *vp;   // packed: codes (and `to_scale` on from there the scales); else columns
    int64_t kh = p.c.k_head_stride, vh = p.c.v_head_stride;
    const int to_scale = 8 * p.columns + line * (p.columns / 16) + col / 16 - (line * (p.columns / 2) + col / 2);
    if constexpr (PACKED) {
        const int64_t in = static_cast<int64_t>(in_page >> 4) * fp4_record(p.columns) + line * (p.columns / 2) + col / 2;
        kp = static_cast<uint8_t*>(p.c.k_pages) + page * p.c.k_page_stride + in + row0 * kh;
        vp = static_cast<uint8_t*>(p.c.v_pages) + page * p.c.v_page_stride + in + row0_v * vh;
    } else {
        kh *= sizeof(T);
        vh *= sizeof(T);
        kp = reinterpret_cast<uint8_t*>(static_cast<T*>(p.c.k_pages) + page * p.c.k_page_stride + in_page * p.c.k_slot_stride) + row0 * kh;
        vp = reinterpret_cast<uint8_t*>(static_cast<T*>(p.c.v_pages) + page * p.c.v_page_stride + in_page * p.c.v_slot_stride) + row0_v * vh;
    }
    auto put4 = [&](uint32_t codes, uint32_t scale, uint8_t* to, bool has) {
        if (has && col < p.columns) {
            *reinterpret_cast<uint32_t*>(to) = codes;
            if ((col & 8) == 0) to[to_scale] = static_cast<uint8_t>(scale);
        }
    };
    // rows of K or V into their records; true where a block has to be done in 64 bits
    auto store4 = [&](float (&y)[8], float most, bool turned, bool whole, float unit, uint8_t* to, bool has) {
        if (unit != 1.0f) {
            most *= unit;
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] *= unit;
        }
        float top = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max_magnitude(top, y[j]);
        // |x c| + |x' s| <= |y| + 2 |x' s|; fp32 values that are exact need the room of r and the product only
        const float off = turned || !whole || sizeof(T) == 4 ? fmaf(2.0f, most, top) : 0.0f;
        uint32_t scale;
        bool open;
        const uint32_t codes = fp4_block<T>(y, top, off, scale, open);
        put4(codes, scale, to, has);
        return __any_sync(0xffffffffu, open && has) != 0;
    };
    auto clear = [&](float (&y)[8]) {   // stored nowhere: q_out and k_out are zeros
        if (!placed)
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = 0.0f;
    };

    // units with blocks that are left to 64 bits (of 32 and more units some are done that need not)
    uint32_t again_k = 0, again_v = 0;
    for (int n = 0, row = row0; n < nk; ++n, row += step) {
        RopeRow<T, VEC> x;
        float y[8], most;
        next(x, src_k + row * p.k_head, row < G);
        rotate(x, y, most);
        if constexpr (PACKED) {
            if (page >= 0 && store4(y, most, turns, p.k_exact, p.k_unit, kp + n * step * kh, row < G)) again_k |= 1u << (n & 31);
        } else {
            if (page >= 0 && on && row < G) rope_store<T, VEC>(reinterpret_cast<T*>(kp + n * step * kh), y, col, D);
            if (p.k_out != nullptr) {
                clear(y);
                if (on && row < G) rope_store<T, VEC>(static_cast<T*>(p.k_out) + t * p.ko_row + row * p.ko_head, y, col, D);
            }
        }
    }
    for (int n = 0, row = row0_v; n < nv; ++n, row += step) {
        const bool has = row < G && page >= 0;
        RopeRow<T, VEC> x;
        next(x, src_v + row * p.v_head, has);
        if constexpr (PACKED) {
            float y[8];
            x.values(y);
            if (store4(y, 0.0f, false, p.v_exact, p.v_unit, vp + n * step * vh, has)) again_v |= 1u << (n & 31);
        } else if (on && has) {
            x.store(reinterpret_cast<T*>(vp + n * step * vh), col, D);
        }
    }
    T* q_out = static_cast<T*>(p.q_out) + t * p.qo_row + row0 * p.qo_head;
    for (int n = 0, row = row0; n < nq; ++n, row += step) {
        const bool has = row < p.heads;
        RopeRow<T, VEC> x;
        float y[8], most;
        next(x, src_q + row * p.q_head, has);
        rotate(x, y, most);
        clear(y);
        if (on && has) rope_store<T, VEC>(q_out, y, col, D);
        q_out += step * p.qo_head;
    }
    if constexpr (RING) cp_async_wait<0>();
    if constexpr (PACKED)
        if ((again_k | again_v) != 0u || p.k_out != nullptr)
            rope4_rest<T, TT, LPR, VEC>(p, RopePlace{t, page, in_page, at, placed}, slice, slice_v, again_k, again_v);
}

// The lengths after a packed append, one warp per sequence: its tokens up to the first that
// had no slot, no page or no position.
__global__ void __launch_bounds__(kRopeThreads) paged_rope_advance_kernel(const __grid_constant__ PagedRopeParams p) {
    const int lane = threadIdx.x & 31;
    const int b = blockIdx.x * kRopeWarps + (threadIdx.x >> 5);
    if (b >= p.c.batch) return;
    pdl_wait();   // the rows are stored by the old lengths
    const int64_t first = p.cu[b], last = min(static_cast<int64_t>(p.cu[b + 1]), p.tokens);
    if (lane == 0 && (first < 0 || p.cu[b + 1] < first || p.cu[b + 1] > p.tokens)) report_status(p.status, CHRONOS_ERR_INVALID_ARG);
    const int64_t from = p.c.lens[b], size = p.c.page_size, at = p.seen != nullptr ? p.seen[b] : 0;
    int64_t n = from >= 0 && first >= 0 ? max(int64_t{0}, min(last - first, p.max_slots - from)) : 0;
    if (p.dim > 0) n = at >= 0 ? max(int64_t{0}, min(n, p.table_len - at)) : 0;
    if (n > 0)
        for (int64_t p0 = from / size; p0 * size < from + n; p0 += 32) {
            const int64_t j = p0 + lane;
            bool none = false;
            if (j * size < from + n) {
                const int page = p.c.page_table[b * p.c.page_table_stride + j];
                none = page < 0 || page >= p.c.num_pages;
            }
            const uint32_t gone = __ballot_sync(0xffffffffu, none);
            if (gone) {
                n = max(int64_t{0}, (p0 + __ffs(gone) - 1) * size - from);
                break;
            }
        }
    __syncwarp();
    if (lane == 0) {
        if (p.lens_out != nullptr) p.lens_out[b] = static_cast<int32_t>(from + n);
        if (p.seen_out != nullptr) p.seen_out[b] = static_cast<int32_t>(at + n);
    }
}

// ---------------------------------------------------------------------------
// rows out of the pages
// ---------------------------------------------------------------------------
struct PagedGatherParams {
    ChronosPagedCache c;
    int64_t tokens;
    int columns;
    float k_scale, v_scale;
    void* k;
    void* v;
    int64_t k_row, k_head, v_row, v_head;
    const int32_t* cu;
    const int32_t* first;
    int max_slots;
    int block;                  // tokens of a block, up to kGatherTokens
    int32_t* status;
};

// The 8 values of codes with their scale.
__device__ __forceinline__ void fp4_values8(uint32_t codes, uint32_t scale, float unit, float (&v)[8]) {
    const uint32_t s = fp8_halves(scale | scale << 8);
    uint32_t h[4];
    fp4_halves(codes, h);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        h[j] = mul_halves(h[j], s);   // 6 bits of at most 2688: exact in halves
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
        v[2 * j] = f.x;
        v[2 * j + 1] = f.y;
    }
    if (unit != 1.0f)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= unit;
}
// The 8 values that a stored slot of 4 bits has from column `col` on.
__device__ __forceinline__ void fp4_load8(const uint8_t* record, int line, int col, int columns, float unit, float (&v)[8]) {
    fp4_values8(*reinterpret_cast<const uint32_t*>(record + line * (columns / 2) + col / 2),
                record[8 * columns + line * (columns / 16) + col / 16], unit, v);
}

// A block takes p.block consecutive tokens (up to 32): one lane of each warp looks up where a
// token's slot lies, then the warps take a token's K or V rows in turn, 8 columns per lane and
// several rows' loads in flight.  Rows that are none are zeros.  19525 tokens of 8 heads of 128 from
// 4 bits to fp16 26 us (3.9 TB/s read and written; 59 % of issue slots, warps wait for loads the rest: no
// unit is full); a warp per token left HBM idle for the chain of look-ups: 40 us.  From bf16 pages 39049 tokens
// 58 us (5.5 TB/s).
constexpr int kGatherTokens = 32;

template <typename T, int LPR, bool VEC, bool PACKED>
__global__ void __launch_bounds__(kRopeThreads) paged_gather_kernel(const __grid_constant__ PagedGatherParams p) {
    constexpr int RPW = 32 / LPR, U = sizeof(T) == 2 && VEC ? 4 : 2;
    __shared__ int64_t s_k[kGatherTokens], s_v[kGatherTokens];   // where the token's slot lies, -1: nowhere, -2: no row
    __shared__ int s_line[kGatherTokens];
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.block;
    const int G = p.c.kv_heads, D = p.c.head_dim;
    const int sub = lane / LPR, col = lane % LPR * 8;
    for (int n = warp; n < p.block; n += kRopeWarps) {
        const int64_t t = t0 + n;
        int64_t k = -2, v = -2;
        int line = 0;
        const int b = t < p.tokens ? paged_sequence(p.cu, p.c.batch, t, lane) : p.c.batch;
        if (b < p.c.batch && t >= p.cu[b]) {
            k = v = -1;
            const int64_t len = min(p.c.lens[b], p.max_slots);
            const int64_t slot = p.first != nullptr ? p.first[b] + t - p.cu[b] : p.c.lens[b] - (static_cast<int64_t>(p.cu[b + 1]) - t);
            int page = -1;
            int in = 0;
            if (slot >= 0 && slot < len) {
                const int j = static_cast<int>(slot) / p.c.page_size;
                in = static_cast<int>(slot) - j * p.c.page_size;
                page = p.c.page_table[b * p.c.page_table_stride + j];
            }
            if (page >= 0 && page < p.c.num_pages) {
                k = page * p.c.k_page_stride + (PACKED ? static_cast<int64_t>(in >> 4) * fp4_record(p.columns) : in * p.c.k_slot_stride);
                v = page * p.c.v_page_stride + (PACKED ? static_cast<int64_t>(in >> 4) * fp4_record(p.columns) : in * p.c.v_slot_stride);
                line = in & 15;
            } else if (lane == 0) {
                report_status(p.status, CHRONOS_ERR_INVALID_ARG);
            }
        }
        if (lane == 0) {
            s_k[n] = k;
            s_v[n] = v;
            s_line[n] = line;
        }
    }
    __syncthreads();
    if (col >= D) return;
    // a token's K rows, then its V rows, RPW at a time
    const int uk = (G + RPW - 1) / RPW;
    auto rows = [&](int n, bool is_k) {
        const int64_t at = is_k ? s_k[n] : s_v[n];
        if (at == -2) return;
        const int64_t head = is_k ? p.c.k_head_stride : p.c.v_head_stride;
        const float unit = is_k ? p.k_scale : p.v_scale;
        T* to = is_k ? static_cast<T*>(p.k) + (t0 + n) * p.k_row + sub * p.k_head : static_cast<T*>(p.v) + (t0 + n) * p.v_row + sub * p.v_head;
        const int64_t to_head = is_k ? p.k_head : p.v_head;
        const int line = s_line[n];
        const uint8_t* record = static_cast<const uint8_t*>(is_k ? p.c.k_pages : p.c.v_pages) + at + sub * head;   // packed
        const T* row = static_cast<const T*>(is_k ? p.c.k_pages : p.c.v_pages) + at + sub * head;                  // not
        for (int u0 = 0; u0 < uk; u0 += U) {
            uint32_t codes[PACKED ? U : 1], scale[PACKED ? U : 1];
            RopeRow<T, VEC> x[PACKED ? 1 : U];
#pragma unroll
            for (int m = 0; m < U; ++m) {
                const int g = (u0 + m) * RPW;
                const bool live = at >= 0 && g + sub < G;
                if constexpr (PACKED) {
                    codes[m] = scale[m] = 0u;
                    if (live) {
                        codes[m] = *reinterpret_cast<const uint32_t*>(record + g * head + line * (p.columns / 2) + col / 2);
                        scale[m] = record[g * head + 8 * p.columns + line * (p.columns / 16) + col / 16];
                    }
                } else {
                    x[m].load(row + g * head, col, live, D, 0, 0);
                }
            }
#pragma unroll
            for (int m = 0; m < U; ++m) {
                const int g = (u0 + m) * RPW;
                if (g + sub >= G) break;
                float y[8];
                if constexpr (PACKED) fp4_values8(codes[m], scale[m], unit, y);
                else x[m].values(y);
                rope_store<T, VEC>(to + g * to_head, y, col, D);
            }
        }
    };
    for (int n = warp; n < 2 * p.block; n += kRopeWarps) rows(n >> 1, (n & 1) == 0);
}

}  // namespace chronos
