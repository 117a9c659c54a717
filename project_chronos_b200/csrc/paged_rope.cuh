// paged_rope.cuh — rows into the pages of the key-value cache with the rotation of
// queries and keys on the way, into pages of the layer type or of 4-bit values, and
// rows back out of the pages (include/chronos_paged4.h).
//
// Bound by HBM for prompts (every row read once, written once) and by latency for one
// token per sequence.  A warp owns a token, or a slice of its rows where tokens are few:
// the angles of its columns stay in registers for all heads, a lane holds 8 columns, so a
// row of 128 takes half a warp.
//
// 4-bit rows.  The code of a value and the scale of a block are decided as exact
// arithmetic decides: the fp32 value y is off by at most 2^-22 (|x c| + |x' s|), so a
// code (scale) is taken where the values that much above and below it give the same
// one, and computed in 64 bits where they do not (a warp in some thousand).  Values that
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

// Column that column d turns with (d itself where it is not rotated).
__device__ __forceinline__ int rope_partner(int d, int start, int dim) {
    const int j = d - start;
    return j < 0 || j >= dim ? d : j < dim / 2 ? d + dim / 2 : d - dim / 2;
}

// A lane's 8 columns of a row as they are loaded.  VEC: 16-byte words (the columns they turn
// with come from the lane that has them); else numbers, with those columns beside them.
template <typename T, bool VEC>
struct RopeRow {
    uint4 w[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* row, int col, bool on, int, int, int) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i)
            w[i] = on ? reinterpret_cast<const uint4*>(row + col)[i] : make_uint4(0u, 0u, 0u, 0u);
    }
    __device__ __forceinline__ void values(float (&x)[8]) const { load8<T>(reinterpret_cast<const T*>(w), x); }
    // Whole warps call it.
    __device__ __forceinline__ void partner(float (&x)[8], int lane) const {
        RopeRow r;
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) {
            r.w[i].x = __shfl_sync(0xffffffffu, w[i].x, lane);
            r.w[i].y = __shfl_sync(0xffffffffu, w[i].y, lane);
            r.w[i].z = __shfl_sync(0xffffffffu, w[i].z, lane);
            r.w[i].w = __shfl_sync(0xffffffffu, w[i].w, lane);
        }
        r.values(x);
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
    __device__ __forceinline__ void partner(float (&v)[8], int) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = with[j];
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
        return v / static_cast<double>(scale);
    }
};
// Codes and scale in 64 bits.  two: the scale's candidates, the lower one in the low byte.
// Whole warps call it.  Not inlined: its registers stay out of the common path.
template <typename T, typename TT>
__device__ __noinline__ uint32_t fp4_block_exact(const RopeSource<T, TT> src, uint32_t two, uint32_t* scale) {
    double t = 0.0;
    for (int j = 0; j < 8; ++j) t = fmax(t, fabs(src.value(j)));
    t = fmax(t, __shfl_xor_sync(0xffffffffu, t, 1));
    uint32_t lo = two & 0xffu;
    if (lo != two >> 8) lo = fp8_scales(static_cast<float>(t / 6.0), 0.0f) & 0xffu;
    *scale = lo;
    const double z = fp8_value(lo);
    uint32_t c = 0;
    for (int j = 0; j < 8; ++j) {
        const double d = src.value(j), m = fabs(d);
        const uint32_t level = (m > 0.25 * z) + (m >= 0.75 * z) + (m > 1.25 * z) + (m >= 1.75 * z) + (m > 2.5 * z) +
                               (m >= 3.5 * z) + (m > 5.0 * z);
        c |= (level | (signbit(d) ? 8u : 0u)) << (4 * j);
    }
    return c;
}

// Codes of a lane's 8 values and the scale of its block of 16 (two lanes).  y: the values in
// units of the cache's factor; off: what y may be off by at most, in 2^-20 (rotated or
// divided values; `exact` ones are what they are).  Whole warps call it.
template <typename T, typename TT>
__device__ __forceinline__ uint32_t fp4_block(const float (&y)[8], const float (&off)[8], bool exact, uint32_t& scale,
                                              const RopeSource<T, TT>& src) {
    constexpr float kOff = 0x1p-20f;
    uint32_t top = 0;
    float most = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        top = max(top, __float_as_uint(y[j]) & 0x7fffffffu);
        most = fmaxf(most, off[j]);
    }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));   // 0: all 16 are exact
    const bool finite = top < 0x7f800000u;
    const float a = finite ? __uint_as_float(top) : 0.0f;
    // exact magnitudes are divided as they are; the others open the scale where a little more or
    // less of them gives another one
    uint32_t two;
    if (most == 0.0f) {
        const float a6 = a / 6.0f;
        two = fp8_scales(a6, a6);
    } else {
        const float a6 = a * (1.0f / 6.0f), d6 = fmaxf(most, a) * (kOff / 2);
        two = fp8_scales(fmaxf(a6 - d6, 0.0f), a6 + d6);
    }
    const float s = fp8_value(two);
    const float r = s > 0.0f ? __frcp_rn(s) : 0.0f;
    uint32_t codes;
    bool open = (two & 0xffu) != two >> 8;
    float u[8];
    if (sizeof(T) == 2 && exact) {
        // 96 + 2^-17 z: values of 64 to 128 have 17 bits behind the point
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = copysignf(fmaf(y[j], r, 96.0f) - 96.0f, y[j]);
        codes = fp4_codes(u);
    } else {
        const float d = r * kOff;
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = fmaf(exact ? fabsf(y[j]) : off[j], -d, y[j] * r);
        codes = fp4_codes(u);
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = fmaf(exact ? fabsf(y[j]) : off[j], d, y[j] * r);
        open |= codes != fp4_codes(u);
    }
    scale = two & 0xffu;
    open &= finite;
    if (__any_sync(0xffffffffu, open)) codes = fp4_block_exact<T, TT>(src, two, &scale);
    codes = finite && scale != 0u ? codes : 0u;
    if (!finite) scale = kFp8Nan;
    return codes;
}

// LPR lanes hold a row (8 columns each).  VEC: rows, halves and tables can be read 8
// columns at a time.
template <typename T, typename TT, int LPR, bool VEC, bool PACKED>
__global__ void __launch_bounds__(kRopeThreads, !VEC ? 1 : PACKED || sizeof(T) == 4 ? 2 : 3) paged_rope_kernel(const __grid_constant__ PagedRopeParams p) {
    constexpr int RPW = 32 / LPR;                       // rows of a warp at once
    constexpr int U = sizeof(T) == 2 && VEC ? 4 : 2;    // ... and so many times that in flight
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int slice = warp % p.slices;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * (kRopeWarps / p.slices) + warp / p.slices;
    const int G = p.c.kv_heads, D = p.c.head_dim, rows = 2 * G + p.heads;
    const int sub = lane / LPR, col = lane % LPR * 8;
    const bool on = col < D;
    const int stride = p.slices * RPW;
    auto source = [&](int r) {
        return r < G ? static_cast<const T*>(p.k) + t * p.k_row + r * p.k_head
                     : r < 2 * G ? static_cast<const T*>(p.v) + t * p.v_row + (r - G) * p.v_head
                                 : static_cast<const T*>(p.q) + t * p.q_row + (r - 2 * G) * p.q_head;
    };
    // the first rows are on their way while the token's place is looked up
    RopeRow<T, VEC> x[U];
    int r0 = slice * RPW;
#pragma unroll
    for (int n = 0; n < U; ++n) {
        const int r = r0 + n * stride + sub;
        x[n].load(source(r), col, on && r < rows && t < p.tokens, D, p.start, p.dim);
    }

    int b = -1, page = -1;
    int64_t i = 0, slot = 0, at = 0;
    bool placed = false;    // at a position of the tables
    if (t < p.tokens) {
        b = p.cu == nullptr ? static_cast<int>(t) : paged_sequence(p.cu, p.c.batch, t, lane);
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
        if (placed && slot >= 0 && slot < p.max_slots) page = p.c.page_table[b * p.c.page_table_stride + slot / p.c.page_size];
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
    if (b < 0) return;
    const int in_page = static_cast<int>(slot % p.c.page_size);
    if (slice == 0 && page >= 0)
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
        sn[j] = 0.0f;
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
    const int from = VEC ? lane - lane % LPR + rope_partner(col, p.start, turns ? p.dim : 0) / 8 : lane;   // the lane that has what these turn with

    for (; r0 < rows; r0 += stride * U) {
        if (r0 != slice * RPW)
#pragma unroll
            for (int n = 0; n < U; ++n) {
                const int r = r0 + n * stride + sub;
                x[n].load(source(r), col, on && r < rows, D, p.start, p.dim);
            }
        __syncwarp();   // q_out may be q, k_out k: a row is read before it is written over
#pragma unroll
        for (int n = 0; n < U; ++n) {
            const int base = r0 + n * stride, r = base + sub;
            if (base >= rows) break;
            const bool is_k = r < G, is_v = !is_k && r < 2 * G, turned = turns && !is_v;
            float y[8], w[8];
            x[n].values(y);
            x[n].partner(w, from);
            float off[PACKED ? 8 : 1];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                w[j] *= sn[j];
                if constexpr (PACKED) off[j] = turned ? fmaf(fabsf(y[j]), fabsf(cs[j]), fabsf(w[j])) : fabsf(y[j]);
                y[j] = turned ? fmaf(y[j], cs[j], w[j]) : y[j];
            }
            uint32_t codes = 0, scale = 0;
            const bool store4 = PACKED && page >= 0 && base < 2 * G;   // a row of the group is one of K or V
            if constexpr (PACKED) {
                if (store4) {
                    const float unit = is_k ? p.k_unit : p.v_unit;
                    const bool exact = !turned && (is_k ? p.k_exact : p.v_exact);
                    float z[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        z[j] = y[j] * unit;
                        off[j] = exact ? 0.0f : off[j] * unit;
                    }
                    const RopeSource<T, TT> src{r < 2 * G ? source(r) : nullptr, turned ? cos : nullptr, sin, col, D, p.start, p.dim,
                                                is_k ? p.k_scale : p.v_scale};
                    codes = fp4_block<T, TT>(z, off, exact, scale, src);
                    __syncwarp();   // the rows may be read there
                }
            }
            if (on && r < rows) {
                if (!placed)   // stored nowhere: q_out and k_out are zeros
#pragma unroll
                    for (int j = 0; j < 8; ++j) y[j] = 0.0f;
                if (!is_k && !is_v)
                    rope_store<T, VEC>(static_cast<T*>(p.q_out) + t * p.qo_row + (r - 2 * G) * p.qo_head, y, col, D);
                else if (is_k && p.k_out != nullptr)
                    rope_store<T, VEC>(static_cast<T*>(p.k_out) + t * p.ko_row + r * p.ko_head, y, col, D);
                if (!PACKED && page >= 0) {
                    if (is_k)
                        rope_store<T, VEC>(static_cast<T*>(p.c.k_pages) + page * p.c.k_page_stride + in_page * p.c.k_slot_stride +
                                               r * p.c.k_head_stride, y, col, D);
                    else if (is_v)
                        rope_store<T, VEC>(static_cast<T*>(p.c.v_pages) + page * p.c.v_page_stride + in_page * p.c.v_slot_stride +
                                               (r - G) * p.c.v_head_stride, y, col, D);
                }
            }
            if (store4 && r < 2 * G && col < p.columns) {
                const int g = is_k ? r : r - G, line = in_page & 15;
                uint8_t* record = static_cast<uint8_t*>(is_k ? p.c.k_pages : p.c.v_pages) +
                                  page * (is_k ? p.c.k_page_stride : p.c.v_page_stride) +
                                  g * (is_k ? p.c.k_head_stride : p.c.v_head_stride) + (in_page >> 4) * fp4_record(p.columns);
                *reinterpret_cast<uint32_t*>(record + line * (p.columns / 2) + col / 2) = codes;
                if ((col & 8) == 0) record[8 * p.columns + line * (p.columns / 16) + col / 16] = static_cast<uint8_t>(scale);
            }
        }
    }
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
    int32_t* status;
};

// The 8 values that a stored slot of 4 bits has from column `col` on.
__device__ __forceinline__ void fp4_load8(const uint8_t* record, int line, int col, int columns, float unit, float (&v)[8]) {
    const uint32_t codes = *reinterpret_cast<const uint32_t*>(record + line * (columns / 2) + col / 2);
    const float s = fp8_value(record[8 * columns + line * (columns / 16) + col / 16]);
    uint32_t h[4];
    fp4_halves(codes, h);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
        v[2 * j] = f.x * s * unit;   // code * scale is exact
        v[2 * j + 1] = f.y * s * unit;
    }
}

// A warp per token, 8 columns per lane; rows that are none are zeros.
template <typename T, int LPR, bool VEC, bool PACKED>
__global__ void __launch_bounds__(kRopeThreads) paged_gather_kernel(const __grid_constant__ PagedGatherParams p) {
    constexpr int RPW = 32 / LPR, U = 4;
    const int lane = threadIdx.x & 31;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * kRopeWarps + (threadIdx.x >> 5);
    if (t >= p.tokens) return;
    const int b = paged_sequence(p.cu, p.c.batch, t, lane);
    if (b >= p.c.batch) return;
    const int64_t i = t - p.cu[b];
    if (i < 0) return;
    const int64_t len = min(p.c.lens[b], p.max_slots);
    const int64_t slot = p.first != nullptr ? p.first[b] + i : p.c.lens[b] - (static_cast<int64_t>(p.cu[b + 1]) - t);
    int page = -1;
    if (slot >= 0 && slot < len) page = p.c.page_table[b * p.c.page_table_stride + slot / p.c.page_size];
    if (page < 0 || page >= p.c.num_pages) {
        page = -1;
        if (lane == 0) report_status(p.status, CHRONOS_ERR_INVALID_ARG);
    }
    const int in_page = page >= 0 ? static_cast<int>(slot % p.c.page_size) : 0;
    const int G = p.c.kv_heads, D = p.c.head_dim;
    const int sub = lane / LPR, col = lane % LPR * 8;
    if (col >= D) return;
    for (int r0 = 0; r0 < 2 * G; r0 += RPW * U) {
        float x[U][8];
#pragma unroll
        for (int n = 0; n < U; ++n) {
            const int r = r0 + n * RPW + sub;
#pragma unroll
            for (int j = 0; j < 8; ++j) x[n][j] = 0.0f;
            if (r >= 2 * G || page < 0) continue;
            const bool is_k = r < G;
            const int g = is_k ? r : r - G;
            if constexpr (PACKED) {
                const uint8_t* record = static_cast<const uint8_t*>(is_k ? p.c.k_pages : p.c.v_pages) +
                                        page * (is_k ? p.c.k_page_stride : p.c.v_page_stride) +
                                        g * (is_k ? p.c.k_head_stride : p.c.v_head_stride) + (in_page >> 4) * fp4_record(p.columns);
                fp4_load8(record, in_page & 15, col, p.columns, is_k ? p.k_scale : p.v_scale, x[n]);
            } else {
                const T* row = is_k ? static_cast<const T*>(p.c.k_pages) + page * p.c.k_page_stride + in_page * p.c.k_slot_stride + g * p.c.k_head_stride
                                    : static_cast<const T*>(p.c.v_pages) + page * p.c.v_page_stride + in_page * p.c.v_slot_stride + g * p.c.v_head_stride;
                if constexpr (VEC) {
                    load8<T>(row + col, x[n]);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (col + j < D) x[n][j] = to_f32<T>(row[col + j]);
                }
            }
        }
#pragma unroll
        for (int n = 0; n < U; ++n) {
            const int r = r0 + n * RPW + sub;
            if (r >= 2 * G) continue;
            T* to = r < G ? static_cast<T*>(p.k) + t * p.k_row + r * p.k_head : static_cast<T*>(p.v) + t * p.v_row + (r - G) * p.v_head;
            rope_store<T, VEC>(to, x[n], col, D);
        }
    }
}

}  // namespace chronos
