// paged4.cuh — one-token attention over pages of 4-bit values, of whole sequences or of
// selected pages (include/chronos_paged4.h).  Work split, running maxima and joins as in
// paged.cuh.
#pragma once

#include "fp4.cuh"
#include "paged.cuh"

namespace chronos {

// The place of slot m of a tile in the products: with it, and the 16-byte pieces of the
// slots' codes moved by paged4_turn, neither product's reads of shared memory collide
// (K: 8 slots' quarters at once; V: an eighth of four slots each).
__device__ __forceinline__ int paged4_place(int m) { return m ^ (((m >> 1) ^ (m >> 2)) & 1); }
template <int DP>
__device__ __forceinline__ int paged4_turn(int slot) {
    return DP == 64 ? 0 : DP == 128 ? ((slot >> 2) & 1) << 1 : slot & 7;
}

template <typename T, int DP, int NT>
struct Paged4 {
    static constexpr int kSlotBytes = DP / 2;                  // codes
    static constexpr int kRecord = fp4_record(DP);             // 16 slots of K or V
    static constexpr int kStages = 4;
    static constexpr int kStageBytes = kPdWarps * 2 * kRecord;
    static constexpr int kOStride = DP + 4;
    static constexpr int kMergeBytes = kPdWarps * 8 * kOStride * 4;
    static constexpr int kSmem = kStages * kStageBytes + kMergeBytes + kPdWarps * 16 * 4 + kStages * kPdWarps * 4;
    static constexpr int kTerms = sizeof(T) == 4 ? 2 : 1;      // halves that a query or weight is split into
    static constexpr int kBlocksPerSm = DP == 256 || (DP == 128 && NT * kTerms > 2) ? 2 : DP == 128 && NT * kTerms > 1 ? 3 : 4;
    static constexpr int kPartBytes = (16 * DP + 32) * 4;      // what a cluster's block leaves for the join
    static_assert(kPartBytes <= kStages * kStageBytes, "the part takes the copies' place");
};

// A query column in halves: in units of 2^-k of its head, and for fp32 layers the rest.
template <int TERMS>
__device__ __forceinline__ void paged4_halves(float a, float b, uint32_t (&r)[TERMS]) {
    const __half2 h = __floats2half2_rn(a, b);
    r[0] = *reinterpret_cast<const uint32_t*>(&h);
    if constexpr (TERMS == 2) {
        const float2 f = __half22float2(h);
        const float x = a - f.x, y = b - f.y;   // what is not finite has no rest
        const __half2 l = __floats2half2_rn(x == x ? x : 0.0f, y == y ? y : 0.0f);
        r[1] = *reinterpret_cast<const uint32_t*>(&l);
    }
}

// HBM bound as long as the products are fed: 9/8 D bytes per slot and kv head.  Codes become
// halves, times the scales of their blocks (code * scale has 6 bits: exact), and go through
// the products of paged.cuh, S^T = K Q^T and O^T = V^T P^T, in fp16 whatever the layer:
// queries in units of a power of two of their head (all their bits but of columns below
// 2^-14 of the largest), weights of up to 2^15.  fp32 layers split queries and weights
// into two halves each (22 bits).  The order of the columns inside a product is free: a
// lane takes a contiguous quarter of a K slot and a contiguous eighth of a V slot, so a
// tile's codes are read by one wide load per slot.  V's halves come in pairs of columns and
// are paired by slots with one byte permutation each.
template <typename T, int DP, int NT, bool CL, bool SEL>
__global__ void __launch_bounds__(kPdThreads, Paged4<T, DP, NT>::kBlocksPerSm) paged_decode4_kernel(
    const __grid_constant__ PagedDecodeParams p) {
    using S = Paged4<T, DP, NT>;
    constexpr int NS = S::kStages, RB = S::kSlotBytes, REC = S::kRecord, TERMS = S::kTerms;
    constexpr int PIECES = 2 * REC / 16, PER = (PIECES + 31) / 32;   // 16-byte copies of a tile, per lane
    constexpr int KW = DP / 32, VW = DP / 64;                        // words of 8 codes per slot and lane
    constexpr float kGrow = 8.0f, kLift = 7.0f;                      // see WeightLift
    static_assert(!SEL || CL, "selected pages: a cluster per row");
    extern __shared__ __align__(128) uint8_t smem[];
    float* s_o = reinterpret_cast<float*>(smem + NS * S::kStageBytes);   // [warp][8 heads][kOStride]
    float* s_ml = s_o + S::kMergeBytes / 4;                              // [warp][8][2]
    uint32_t* s_vis = reinterpret_cast<uint32_t*>(s_ml + kPdWarps * 16); // [stage][warp]
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int quad = lane >> 2, qc = lane & 3;

    int end;
    PagedIter ld;
    const int rank = CL ? static_cast<int>(blockIdx.x) % p.cluster : 0;
    if constexpr (CL) {
        const int row = blockIdx.x / p.cluster, per = p.c.kv_heads * p.parts;
        ld.u = 0;
        ld.b = row / per;
        ld.v = row % per;
        ld.blk = rank;
        if constexpr (SEL) {
            ld.r = paged_row_sel(p, ld.b, lane);
            if (ld.r.seq < 0) return;
        } else {
            ld.r = paged_row(p, ld.b);
        }
        end = ld.r.nblk > rank ? (ld.r.nblk - rank + p.cluster - 1) / p.cluster : 0;
        if (!SEL && blockIdx.x == 0) paged_check_lens(p);
    } else {
        const int total = paged_total(p, lane);
        const int share = paged_share(p, total);
        const int begin = static_cast<int>(blockIdx.x) * share;
        end = min(total, begin + share);
        if (blockIdx.x == 0) paged_check_lens(p);
        if (begin >= end) return;
        ld = paged_seek(p, begin, lane);
    }
    auto advance = [&](PagedIter& it) {
        if constexpr (CL) {
            ++it.u;
            it.blk += p.cluster;
        } else {
            it.advance(p, end);
        }
    };
    PagedIter cp = ld;
    PagedLook look = paged_look_at<SEL, true>(p, ld, end, warp, lane);

    // a tile: K's record, V's record, as they lie in the pages but for the turned pieces
    uint32_t to[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int n = lane + 32 * i, c = n < REC / 16 ? n : n - REC / 16;
        const int slot = c / (RB / 16), piece = c % (RB / 16);
        to[i] = static_cast<uint32_t>((n - c) * 16 + (c < RB ? slot * RB + ((piece ^ paged4_turn<DP>(slot)) << 4) : c * 16));
    }
    auto issue = [&](int stage) {
        uint32_t vis = look.vis;
        if (look.page < 0) vis = 0u;
        if (vis) {
            const int64_t g = ld.v / p.parts, at = static_cast<int64_t>(look.slot >> 4) * REC;
            const uint8_t* k = static_cast<const uint8_t*>(p.c.k_pages) + look.page * p.c.k_page_stride + g * p.c.k_head_stride + at;
            const uint8_t* v = static_cast<const uint8_t*>(p.c.v_pages) + look.page * p.c.v_page_stride + g * p.c.v_head_stride + at;
            const uint32_t st = smem_u32(smem + stage * S::kStageBytes + warp * 2 * REC);
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int n = lane + 32 * i;
                if (n < PIECES) cp_async16(st + to[i], n < REC / 16 ? k + n * 16 : v + (n * 16 - REC), true);
            }
        }
        if (lane == 0) s_vis[stage * kPdWarps + warp] = vis;
    };
#pragma unroll
    for (int s = 0; s < NS - 1; ++s) {
        if (ld.u < end) {
            issue(s);
            advance(ld);
            look = paged_look_at<SEL, true>(p, ld, end, warp, lane);
        }
        cp_async_commit();
    }

    const int kslot = paged4_place(quad);            // and 8 on
    const int v0 = paged4_place(2 * qc), v1 = paged4_place(2 * qc + 1);
    uint32_t qb[NT][DP / 16][2][TERMS];
    float unit[NT][2];          // of the scores of heads 2 qc and 2 qc + 1
    float o[NT][DP / 16][4];
    float m[NT][2], l[NT][2];
    bool fresh = true;          // the next unit opens a new part or row
    int part_blk = 0;           // the block it opened with
    int stage = 0;
    while (cp.u < end || (CL && fresh)) {
        const int kvh = cp.v / p.parts, h0 = (cp.v % p.parts) * 16;
        const int nh = min(16, p.rep - h0);          // query heads of this unit
        if (fresh) {
            fresh = false;
            part_blk = cp.blk;
            const T* q = static_cast<const T*>(p.q) + cp.b * p.q_row + static_cast<int64_t>(kvh * p.rep + h0) * p.q_head;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                m[t][0] = m[t][1] = -INFINITY;
                l[t][0] = l[t][1] = 0.0f;
#pragma unroll
                for (int i = 0; i < DP / 16; ++i) o[t][i][0] = o[t][i][1] = o[t][i][2] = o[t][i][3] = 0.0f;
                // a head's columns in units of a power of two: the largest is 2^8 to 2^9
                const int row = t * 8 + quad;
                const T* head = q + row * p.q_head + qc * (DP / 4);
                const bool on = row < nh;
                uint32_t top = 0;
#pragma unroll
                for (int d = 0; d < DP / 4; ++d)
                    if (on && qc * (DP / 4) + d < p.c.head_dim) top = max(top, __float_as_uint(to_f32<T>(head[d])) & 0x7fffffffu);
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const int k = min(max(8 - (static_cast<int>(top >> 23) - 127), -110), 110);
                const float up = __uint_as_float(static_cast<uint32_t>(127 + k) << 23), down = __uint_as_float(static_cast<uint32_t>(127 - k) << 23);
#pragma unroll
                for (int i = 0; i < DP / 16; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int d = i * 4 + j * 2, c = qc * (DP / 4) + d;
                        const float a = on && c < p.c.head_dim ? to_f32<T>(head[d]) * up : 0.0f;
                        const float b = on && c + 1 < p.c.head_dim ? to_f32<T>(head[d + 1]) * up : 0.0f;
                        paged4_halves<TERMS>(a, b, qb[t][i][j]);
                    }
#pragma unroll
                for (int j = 0; j < 2; ++j) unit[t][j] = p.sl2 * __shfl_sync(0xffffffffu, down, (2 * qc + j) * 4);
            }
        }
        if (ld.u < end) {
            issue(stage == 0 ? NS - 1 : stage - 1);
            advance(ld);
            look = paged_look_at<SEL, true>(p, ld, end, warp, lane);
        }
        cp_async_commit();
        cp_async_wait<NS - 1>();
        __syncwarp();
        const uint8_t* st = smem + stage * S::kStageBytes + warp * 2 * REC;
        const uint32_t vis = cp.u < end ? s_vis[stage * kPdWarps + warp] : 0u;
        if (vis) {
            float s[NT][4];
#pragma unroll
            for (int t = 0; t < NT; ++t) s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.0f;
            {
                // this lane's quarter of slots kslot and kslot + 8
                uint32_t w[2][KW], sc[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const uint8_t* slot = st + (kslot + 8 * r) * RB;
                    const uint8_t* scales = st + 16 * RB + (kslot + 8 * r) * (DP / 16);
                    if constexpr (DP == 64) {
                        const uint2 x = *reinterpret_cast<const uint2*>(slot + qc * 8);
                        w[r][0] = x.x; w[r][1] = x.y;
                        sc[r] = scales[qc];
                    } else if constexpr (DP == 128) {
                        const uint4 x = *reinterpret_cast<const uint4*>(slot + ((qc ^ paged4_turn<DP>(kslot)) << 4));
                        w[r][0] = x.x; w[r][1] = x.y; w[r][2] = x.z; w[r][3] = x.w;
                        sc[r] = *reinterpret_cast<const uint16_t*>(scales + qc * 2);
                    } else {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const uint4 x = *reinterpret_cast<const uint4*>(slot + (((2 * qc + i) ^ paged4_turn<DP>(kslot)) << 4));
                            w[r][4 * i] = x.x; w[r][4 * i + 1] = x.y; w[r][4 * i + 2] = x.z; w[r][4 * i + 3] = x.w;
                        }
                        sc[r] = *reinterpret_cast<const uint32_t*>(scales + qc * 4);
                    }
                }
#pragma unroll
                for (int i = 0; i < KW; ++i) {   // 8 columns of both slots: two pieces of 16 in the product's order
                    uint32_t x[2][4];
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        fp4_halves(w[r][i], x[r]);
                        const uint32_t two = fp8_halves(sc[r] >> (16 * (i / 4)));
                        const uint32_t one = __byte_perm(two, two, (i / 2) % 2 == 0 ? 0x1010 : 0x3232);
#pragma unroll
                        for (int j = 0; j < 4; ++j) x[r][j] = mul_halves(x[r][j], one);
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t a[4] = {x[0][2 * j], x[1][2 * j], x[0][2 * j + 1], x[1][2 * j + 1]};
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int e = TERMS - 1; e >= 0; --e)
                                mma_16816<__half>(s[t], a, qb[t][2 * i + j][0][e], qb[t][2 * i + j][1][e]);
                    }
                }
            }
            // s[t][0..1]: slot kslot, heads 8t + 2qc, + 1; s[t][2..3]: slot kslot + 8
            const bool on0 = (vis >> kslot) & 1u, on1 = (vis >> (kslot + 8)) & 1u;
            bool grow = false;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[t][j] = (j < 2 ? on0 : on1) ? s[t][j] * unit[t][j & 1] : -INFINITY;
                    grow |= s[t][j] > m[t][j & 1] + kGrow;
                }
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float n = fmaxf(s[t][j], s[t][2 + j]);
#pragma unroll
                        for (int x = 4; x < 32; x <<= 1) n = fmaxf(n, __shfl_xor_sync(0xffffffffu, n, x));
                        n = fmaxf(n, m[t][j]);
                        const float c = n == -INFINITY ? 1.0f : exp2_fast(m[t][j] - n);
                        m[t][j] = n;
                        l[t][j] *= c;
#pragma unroll
                        for (int i = 0; i < DP / 16; ++i) {
                            o[t][i][j] *= c;
                            o[t][i][2 + j] *= c;
                        }
                    }
            }
            uint32_t pb[NT][2][TERMS];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const float u0 = m[t][0] == -INFINITY ? 0.0f : m[t][0] - kLift, u1 = m[t][1] == -INFINITY ? 0.0f : m[t][1] - kLift;
                const float a = exp2_fast(s[t][0] - u0), b = exp2_fast(s[t][1] - u1);
                const float c = exp2_fast(s[t][2] - u0), d = exp2_fast(s[t][3] - u1);
                l[t][0] += a + c;
                l[t][1] += b + d;
                // weights in halves for the second product; the sum keeps fp32
                uint32_t x[TERMS], y[TERMS];
                paged4_halves<TERMS>(a, b, x);
                paged4_halves<TERMS>(c, d, y);
#pragma unroll
                for (int e = 0; e < TERMS; ++e) {
                    pb[t][0][e] = transpose8x8(x[e]);
                    pb[t][1][e] = transpose8x8(y[e]);
                }
            }
            // this lane's eighth of four slots of V: the products' rows 2 qc, 2 qc + 1 and 8 on
            uint32_t w[4][VW], sc[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int sl = ((r & 1) ? v1 : v0), at = sl + (r >> 1) * 8;
                const uint8_t* slot = st + REC + at * RB;
                const uint8_t* scales = st + REC + 16 * RB + at * (DP / 16);
                if constexpr (DP == 64) {
                    w[r][0] = *reinterpret_cast<const uint32_t*>(slot + quad * 4);
                    sc[r] = scales[quad >> 1];
                } else if constexpr (DP == 128) {
                    const uint2 x = *reinterpret_cast<const uint2*>(slot + (((quad >> 1) ^ paged4_turn<DP>(sl)) << 4) + (quad & 1) * 8);
                    w[r][0] = x.x; w[r][1] = x.y;
                    sc[r] = scales[quad];
                } else {
                    const uint4 x = *reinterpret_cast<const uint4*>(slot + ((quad ^ paged4_turn<DP>(sl)) << 4));
                    w[r][0] = x.x; w[r][1] = x.y; w[r][2] = x.z; w[r][3] = x.w;
                    sc[r] = *reinterpret_cast<const uint16_t*>(scales + quad * 2);
                }
                sc[r] = fp8_halves(sc[r]);
                if (vis != 0xffffu && !((vis >> at) & 1u)) sc[r] = 0u;   // what lies behind the length may be anything
            }
#pragma unroll
            for (int i = 0; i < VW; ++i) {
                uint32_t x[4][4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    fp4_halves(w[r][i], x[r]);
                    const uint32_t one = __byte_perm(sc[r], sc[r], DP < 256 || i < 2 ? 0x1010 : 0x3232);
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[r][j] = mul_halves(x[r][j], one);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {   // columns 2j and 2j + 1 of the word: the rows quad and quad + 8 of a product
                    const uint32_t a[4] = {__byte_perm(x[0][j], x[1][j], 0x5410), __byte_perm(x[0][j], x[1][j], 0x7632),
                                           __byte_perm(x[2][j], x[3][j], 0x5410), __byte_perm(x[2][j], x[3][j], 0x7632)};
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int e = TERMS - 1; e >= 0; --e) mma_16816<__half>(o[t][4 * i + j], a, pb[t][0][e], pb[t][1][e]);
                }
            }
        }
        __syncwarp();   // every lane has read the tile before its stage is filled again
        stage = stage == NS - 1 ? 0 : stage + 1;

        if (CL ? cp.u + 1 >= end : (cp.blk + 1 == cp.r.nblk || cp.u + 1 == end)) {
            // the row (or this block's part of it) is complete: join the four warps, 8 heads at a time
            fresh = !CL;
            const bool whole = CL ? p.cluster == 1 : part_blk == 0 && cp.blk + 1 == cp.r.nblk;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                if (t * 8 >= nh) break;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) l[t][j] += __shfl_xor_sync(0xffffffffu, l[t][j], x);
                    if (quad == 0)
                        *reinterpret_cast<float2*>(s_ml + (warp * 8 + qc * 2 + j) * 2) = make_float2(m[t][j] - kLift, l[t][j]);
                    float* dst = s_o + (warp * 8 + qc * 2 + j) * S::kOStride + quad * (DP / 8);
#pragma unroll
                    for (int i = 0; i < DP / 16; ++i)
                        *reinterpret_cast<float2*>(dst + 2 * i) = make_float2(o[t][i][j], o[t][i][2 + j]);
                }
                __syncthreads();
                for (int h = warp; h < 8 && t * 8 + h < nh; h += kPdWarps) {
                    float M = -INFINITY, L = 0.0f, c[kPdWarps];
#pragma unroll
                    for (int w = 0; w < kPdWarps; ++w) M = fmaxf(M, s_ml[(w * 8 + h) * 2]);
                    const float u = M == -INFINITY ? 0.0f : M;
#pragma unroll
                    for (int w = 0; w < kPdWarps; ++w) {
                        c[w] = exp2_fast(s_ml[(w * 8 + h) * 2] - u);
                        L += s_ml[(w * 8 + h) * 2 + 1] * c[w];
                    }
                    const float inv = (whole ? (L > 0.0f ? 1.0f / L : L) : 1.0f) * p.v_scale;
                    const int row = t * 8 + h, head = kvh * p.rep + h0 + row;
                    const int64_t part = (2 * static_cast<int64_t>(blockIdx.x) + (part_blk == 0 ? 1 : 0)) * 16 + row;
                    T* out = static_cast<T*>(p.out) + cp.b * p.out_row + head * p.out_head;
                    // a cluster's block leaves its part where the copies were (they are all consumed)
                    float* po = CL ? reinterpret_cast<float*>(smem) + row * DP : p.part_o + part * p.part_stride;
                    for (int d = lane * 2; d < DP; d += 64) {
                        float a = 0.0f, b = 0.0f;
#pragma unroll
                        for (int w = 0; w < kPdWarps; ++w) {
                            const float2 v = *reinterpret_cast<const float2*>(s_o + (w * 8 + h) * S::kOStride + d);
                            a = fmaf(v.x, c[w], a);
                            b = fmaf(v.y, c[w], b);
                        }
                        a *= inv;
                        b *= inv;
                        if (!whole) {
                            *reinterpret_cast<float2*>(po + d) = make_float2(a, b);
                        } else {
                            if (d < p.c.head_dim) out[d] = from_f32<T>(a);
                            if (d + 1 < p.c.head_dim) out[d + 1] = from_f32<T>(b);
                        }
                    }
                    if (lane == 0) {
                        if (!whole) {
                            float* ml = CL ? reinterpret_cast<float*>(smem) + 16 * DP + row * 2 : p.part_ml + part * 2;
                            *reinterpret_cast<float2*>(ml) = make_float2(M, L);
                        } else if (p.lse != nullptr) {
                            p.lse[static_cast<int64_t>(cp.b) * p.heads + head] = L != 0.0f ? (u + log2f(L)) * kLn2 : -INFINITY;
                        }
                    }
                }
                if (NT > 1 || !CL) __syncthreads();
            }
            if (CL) break;
        }
        advance(cp);
    }
    cp_async_wait<0>();
    if constexpr (CL)
        if (p.cluster > 1) {
            const int kvh = cp.v / p.parts, h0 = (cp.v % p.parts) * 16;
            paged_cluster_join<T>(p, smem, DP, rank, cp.b, kvh * p.rep + h0, min(16, p.rep - h0), warp, lane);
        }
}

}  // namespace chronos
