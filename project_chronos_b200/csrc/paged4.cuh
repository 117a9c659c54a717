// paged4.cuh — one-token attention over pages of 4-bit values, of whole sequences or of
// selected pages (include/chronos_paged4.h).  Work split, running maxima and joins as in
// paged.cuh.
#pragma once

#include <type_traits>

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
    static constexpr int kSmem = kStages * kStageBytes + kMergeBytes + kPdWarps * 16 * 4;
    static constexpr int kTerms = sizeof(T) == 4 ? 2 : 1;      // halves that a query is split into
    // four blocks of 128 registers measured 2 to 7 % slower than three for heads of 128
    static constexpr int kBlocksPerSm = DP == 256 || (DP == 128 && NT * kTerms > 2) ? 2 : DP == 128 ? 3 : 4;
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

// Shared memory at an address the compiler keeps in a register (it would work the address out again
// for every tile), with what is added at compile time in the instruction.
template <int N>
__device__ __forceinline__ void lds_words(uint32_t (&r)[N], uint32_t at, int off) {
    if constexpr (N == 1)
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(r[0]) : "r"(at + off));
    else if constexpr (N == 2)
        asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(at + off));
    else
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at + off));
}
// N bytes (1, 2 or 4) with zeros above.
template <int N>
__device__ __forceinline__ uint32_t lds_bytes(uint32_t at, int off) {
    uint32_t r;
    if constexpr (N == 1) asm volatile("ld.shared.u8 %0, [%1];" : "=r"(r) : "r"(at + off));
    else if constexpr (N == 2) asm volatile("{\n\t.reg .u16 t;\n\tld.shared.u16 t, [%1];\n\tcvt.u32.u16 %0, t;\n\t}" : "=r"(r) : "r"(at + off));
    else asm volatile("ld.shared.b32 %0, [%1];" : "=r"(r) : "r"(at + off));
    return r;
}
__device__ __forceinline__ uint32_t kept(uint32_t x) {
    uint32_t r;
    asm volatile("mov.b32 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

// HBM bound as long as the products are fed: 9/8 D bytes per slot and kv head.  Codes become
// halves, times the scales of their blocks (code * scale has 6 bits: exact), and go through
// the products of paged.cuh, S^T = K Q^T and O^T = V^T P^T, in fp16 whatever the layer:
// queries in units of a power of two of their head (all their bits but of columns below
// 2^-22 of the largest), weights of up to 2^15.  fp32 layers split queries and weights
// into two halves each (22 bits).  The order of the columns inside a product is free: a
// lane takes a contiguous quarter of a K slot and a contiguous eighth of a V slot, so a
// tile's codes are read by one wide load per slot.  V's halves come in pairs of columns; the
// multiplications by two slots' scales pair them by slots.
//
// A warp takes TILES tiles of 16 slots of a unit (4 * TILES tiles), one after the other; its lanes
// look up the pages of a unit's tiles at once, a unit ahead.
//
// Measured, 32 / 8 heads of 128: 4 rows of 100003 to 131072 slots in fp16 138 us, 4.1 TB/s of 4-bit
// records (the 16-bit cache: 291 to 310 us); 32 ragged rows up to 8192 slots 58 us.  348 instructions per
// tile, of which 64 conversions, 96 scale products and 16 tensor products are the format's.  No unit
// is full (60 % of issue slots, ALU 43 %, FMA 39 %): a scheduler's three warps each follow one chain of
// dependent steps per tile.  16 slots per look-up and unit: 206 us.
template <typename T, int DP, int NT, int TILES, bool CL, bool SEL>
__global__ void __launch_bounds__(kPdThreads, Paged4<T, DP, NT>::kBlocksPerSm) paged_decode4_kernel(
    const __grid_constant__ PagedDecodeParams p) {
    using S = Paged4<T, DP, NT>;
    constexpr int NS = S::kStages, RB = S::kSlotBytes, REC = S::kRecord, TERMS = S::kTerms, BLOCK = TILES * kPdBlock;
    constexpr int KW = DP / 32, VW = DP / 64;                        // words of 8 codes per slot and lane
    constexpr float kGrow = 8.0f, kLift = 7.0f;                      // see WeightLift
    // Halves that a weight is split into; the sum of weights is fp32 whatever it is.  One is off by up to
    // 2^-11, an eighth of what a bf16 result's own rounding is, and as much as an fp16 result's: 4 fp16 rows of
    // 100003 to 131072 slots are 2.4e-4 off with one and 2.1e-4 with two (fp32 weights: 2.1e-4), in
    // 140 and 160 us, so whole sequences of fp16 layers take one.  Selected pages, few slots whose
    // look-ups bound the call, take two; so do fp32 layers (22 bits).
    constexpr int WT = TERMS == 2 || (SEL && std::is_same<T, __half>::value) ? 2 : 1;
    static_assert(!SEL || CL, "selected pages: a cluster per row");
    extern __shared__ __align__(128) uint8_t smem[];
    float* s_o = reinterpret_cast<float*>(smem + NS * S::kStageBytes);   // [warp][8 heads][kOStride]
    float* s_ml = s_o + S::kMergeBytes / 4;                              // [warp][8][2]
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int quad = lane >> 2, qc = lane & 3;

    int end;
    PagedIter pf;   // the unit that is looked up next
    const int rank = CL ? static_cast<int>(blockIdx.x) % p.cluster : 0;
    if constexpr (CL) {
        const int row = blockIdx.x / p.cluster, per = p.c.kv_heads * p.parts;
        pf.u = 0;
        pf.b = row / per;
        pf.v = row % per;
        pf.blk = rank;
        if constexpr (SEL) {
            pf.r = paged_row_sel<BLOCK>(p, pf.b, lane);
            if (pf.r.seq < 0) return;
        } else {
            pf.r = paged_row<BLOCK>(p, pf.b);
        }
        end = pf.r.nblk > rank ? (pf.r.nblk - rank + p.cluster - 1) / p.cluster : 0;
        if (!SEL && blockIdx.x == 0) paged_check_lens(p);
    } else {
        const int total = paged_total<BLOCK>(p, lane);
        const int share = paged_share(p, total);
        const int begin = static_cast<int>(blockIdx.x) * share;
        end = min(total, begin + share);
        if (blockIdx.x == 0) paged_check_lens(p);
        if (begin >= end) return;
        pf = paged_seek<BLOCK>(p, begin, lane);
    }
    auto advance = [&](PagedIter& it) {
        if constexpr (CL) {
            ++it.u;
            it.blk += p.cluster;
        } else {
            it.template advance<BLOCK>(p, end);
        }
    };
    auto kv_head = [&](int v) { return p.parts == 1 ? v : v / p.parts; };
    // lane j (and j + TILES, ...) has tile j of the unit
    auto look_up = [&]() {
        const int place = pf.blk * BLOCK + (warp * TILES + (lane & (TILES - 1))) * kPdTile;
        if constexpr (SEL) return paged_look_sel<true>(p, pf, pf.u < end, place, lane);
        else return paged_look_place<true>(p, pf, pf.u < end, place, lane);
    };
    PagedIter cp = pf;
    PagedLook look = look_up();
    int head = kv_head(pf.v), left = end - pf.u;   // the unit that is being copied, units left
    advance(pf);
    PagedLook ahead = look_up();
    int head_ahead = kv_head(pf.v);

    // a tile: K's record, V's record, as they lie in the pages but for the turned pieces: codes
    // (CODES pieces of 16 bytes each) by all lanes, both scales (DP / 16 pieces each) by DP / 8 lanes
    constexpr int CODES = DP / 2, SCALES = DP / 16;
    const uint32_t ring = smem_u32(smem) + warp * 2 * REC;
    uint32_t to[CODES / 32];
#pragma unroll
    for (int i = 0; i < CODES / 32; ++i) {
        const int n = lane + 32 * i, slot = n / (RB / 16), piece = n % (RB / 16);
        to[i] = ring + static_cast<uint32_t>(slot * RB + ((piece ^ paged4_turn<DP>(slot)) << 4));
    }
    const bool of_v = (lane & (SCALES - 1)) != lane;   // the scales of V
    const uint32_t to_scale = ring + static_cast<uint32_t>((of_v ? REC : 0) + 16 * (CODES + (lane & (SCALES - 1))));
    const uint8_t *k_row = nullptr, *v_row = nullptr;
    auto row_pointers = [&]() {
        k_row = static_cast<const uint8_t*>(p.c.k_pages) + head * p.c.k_head_stride + lane * 16;
        v_row = static_cast<const uint8_t*>(p.c.v_pages) + head * p.c.v_head_stride + lane * 16;
    };
    row_pointers();
    uint32_t shows[NS];   // which slots of the tile in a stage are visible
    // Copies tile `tile` of the unit `look` is of into a stage (both known at compile time).
    auto issue = [&](int stage, int tile) {
        shows[stage] = 0u;
        if (left > 0) {
            int page = look.page;
            uint32_t at = static_cast<uint32_t>(look.slot >> 4) * REC, vis = look.vis;   // of a page: 32 bits
            if constexpr (TILES > 1) {
                page = __shfl_sync(0xffffffffu, page, tile);
                at = __shfl_sync(0xffffffffu, at, tile);
                vis = __shfl_sync(0xffffffffu, vis, tile);
            }
            if (page >= 0 && vis != 0u) {
                shows[stage] = vis;
                // page strides fit 32 bits (the host sees to it): one multiplication per pointer
                const uint8_t* k = k_row + static_cast<uint64_t>(static_cast<uint32_t>(page)) * static_cast<uint32_t>(p.c.k_page_stride) + at;
                const uint8_t* v = v_row + static_cast<uint64_t>(static_cast<uint32_t>(page)) * static_cast<uint32_t>(p.c.v_page_stride) + at;
#pragma unroll
                for (int i = 0; i < CODES / 32; ++i) {
                    cp_async16(to[i] + stage * S::kStageBytes, k + i * 512, true);
                    cp_async16(to[i] + stage * S::kStageBytes + REC, v + i * 512, true);
                }
                const uint8_t* s = of_v ? v - SCALES * 16 : k;
                if (lane < 2 * SCALES) cp_async16(to_scale + stage * S::kStageBytes, s + CODES * 16, true);
            }
            if (tile == TILES - 1) {   // on to the next unit
                --left;
                look = ahead;
                if (head != head_ahead) {
                    head = head_ahead;
                    row_pointers();
                }
                advance(pf);
                ahead = look_up();
                head_ahead = kv_head(pf.v);
            }
        }
        cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < NS - 1; ++s) issue(s, s % TILES);

    const int kslot = paged4_place(quad);            // and 8 on
    const int v0 = paged4_place(2 * qc), v1 = paged4_place(2 * qc + 1);
    uint32_t qb[NT][DP / 16][2][TERMS];
    float unit[NT][2];               // of the scores of heads 2 qc and 2 qc + 1
    float o[NT][DP / 16][4];
    float base[NT][2], l[NT][2];     // what is taken off the scores: the maximum as it lags, less kLift
    // where this lane finds its parts of a tile (slots + 8: 8 slots on)
    constexpr int SB = DP / 16;                      // scales of a slot
    const uint32_t k_at = kept(ring + kslot * RB + (DP == 64 ? qc * 8 : ((DP == 128 ? qc : 2 * qc) ^ paged4_turn<DP>(kslot)) << 4));
    const uint32_t k_at2 = DP < 256 ? 0u : kept(ring + kslot * RB + (((2 * qc + 1) ^ paged4_turn<DP>(kslot)) << 4));
    const uint32_t ks_at = kept(ring + 16 * RB + kslot * SB + qc * (SB / 4));
    uint32_t v_at[2], vs_at[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int sl = r ? v1 : v0;
        v_at[r] = kept(ring + REC + sl * RB + (DP == 64 ? quad * 4 : DP == 128 ? (((quad >> 1) ^ paged4_turn<DP>(sl)) << 4) + (quad & 1) * 8
                                                                              : (quad ^ paged4_turn<DP>(sl)) << 4));
        vs_at[r] = kept(ring + REC + 16 * RB + sl * SB + (DP == 64 ? quad >> 1 : DP == 128 ? quad : quad * 2));
    }

    // A row's (or part's) beginning: kv head kvh, query heads from h0 on.
    auto open_row = [&](int kvh, int h0, int nh) {
        const T* q = static_cast<const T*>(p.q) + cp.b * p.q_row + static_cast<int64_t>(kvh * p.rep + h0) * p.q_head;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            base[t][0] = base[t][1] = -INFINITY;
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
    };

    // The tile in a stage.
    auto take = [&](auto stage_of) {
        constexpr int stage = decltype(stage_of)::value, at = stage * S::kStageBytes;
        const uint32_t vis = shows[stage];
        if (vis == 0u) return;
        float s[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t) s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.0f;
        {
            // this lane's quarter of slots kslot and kslot + 8
            uint32_t w[2][KW], two[2][(KW + 3) / 4];
            if constexpr (DP < 256) {
                lds_words<KW>(w[0], k_at, at);
                lds_words<KW>(w[1], k_at, at + 8 * RB);
                two[0][0] = fp8_halves(lds_bytes<SB / 4>(ks_at, at));
                two[1][0] = fp8_halves(lds_bytes<SB / 4>(ks_at, at + 8 * SB));
            } else {
                uint32_t x[4];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    if (r == 0) lds_words<4>(x, k_at, at);
                    else lds_words<4>(x, k_at, at + 8 * RB);
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[r][i] = x[i];
                    if (r == 0) lds_words<4>(x, k_at2, at);
                    else lds_words<4>(x, k_at2, at + 8 * RB);
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[r][4 + i] = x[i];
                    const uint32_t sc = r == 0 ? lds_bytes<4>(ks_at, at) : lds_bytes<4>(ks_at, at + 8 * SB);
                    two[r][0] = fp8_halves(sc);
                    two[r][1] = fp8_halves(sc >> 16);
                }
            }
#pragma unroll
            for (int i = 0; i < KW; ++i) {   // 8 columns of both slots: two pieces of 16 in the product's order
                uint32_t x[2][4];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    fp4_halves(w[r][i], x[r]);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        x[r][j] = (i / 2) % 2 == 0 ? mul_low(x[r][j], two[r][i / 4]) : mul_high(x[r][j], two[r][i / 4]);
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
        if (vis != 0xffffu) {
            const bool on0 = (vis >> kslot) & 1u, on1 = (vis >> (kslot + 8)) & 1u;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[t][j] = (j < 2 ? on0 : on1) ? s[t][j] : -INFINITY;
        }
        // logarithms of the weights; a row's first tile finds base at -inf and grows
        float x[NT][4];
        bool grow = false;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[t][j] = fmaf(s[t][j], unit[t][j & 1], -base[t][j & 1]);
                grow |= x[t][j] > kGrow + kLift;
            }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float n = fmaxf(s[t][j], s[t][2 + j]) * unit[t][j];
#pragma unroll
                    for (int y = 4; y < 32; y <<= 1) n = fmaxf(n, __shfl_xor_sync(0xffffffffu, n, y));
                    n = fmaxf(n - kLift, base[t][j]);
                    const float c = n == -INFINITY ? 1.0f : exp2_fast(base[t][j] - n);
                    base[t][j] = n;
                    l[t][j] *= c;
                    x[t][j] = n == -INFINITY ? s[t][j] : fmaf(s[t][j], unit[t][j], -n);   // -inf or NaN as it is
                    x[t][2 + j] = n == -INFINITY ? s[t][2 + j] : fmaf(s[t][2 + j], unit[t][j], -n);
#pragma unroll
                    for (int i = 0; i < DP / 16; ++i) {
                        o[t][i][j] *= c;
                        o[t][i][2 + j] *= c;
                    }
                }
        }
        uint32_t pb[NT][2][WT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const float a = exp2_fast(x[t][0]), b = exp2_fast(x[t][1]), c = exp2_fast(x[t][2]), d = exp2_fast(x[t][3]);
            l[t][0] += a + c;
            l[t][1] += b + d;
            // weights in halves for the second product; the sum keeps fp32
            uint32_t y[WT], z[WT];
            paged4_halves<WT>(a, b, y);
            paged4_halves<WT>(c, d, z);
#pragma unroll
            for (int e = 0; e < WT; ++e) {
                pb[t][0][e] = transpose8x8(y[e]);
                pb[t][1][e] = transpose8x8(z[e]);
            }
        }
        // this lane's eighth of four slots of V: the products' rows 2 qc, 2 qc + 1 and 8 on
        uint32_t w[4][VW], sc[4];
        constexpr int VB = DP == 256 ? 2 : 1;
        lds_words<VW>(w[0], v_at[0], at);
        lds_words<VW>(w[1], v_at[1], at);
        lds_words<VW>(w[2], v_at[0], at + 8 * RB);
        lds_words<VW>(w[3], v_at[1], at + 8 * RB);
        sc[0] = lds_bytes<VB>(vs_at[0], at);
        sc[1] = lds_bytes<VB>(vs_at[1], at);
        sc[2] = lds_bytes<VB>(vs_at[0], at + 8 * SB);
        sc[3] = lds_bytes<VB>(vs_at[1], at + 8 * SB);
        if (vis != 0xffffu)   // what lies behind the length may be anything
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (!((vis >> (((r & 1) ? v1 : v0) + (r >> 1) * 8)) & 1u)) sc[r] = 0u;
#pragma unroll
        for (int i = 0; i < VW; ++i) {
            uint32_t y[4][4], one[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                fp4_halves(w[r][i], y[r]);
                // (scale, 0) of the even slots, (0, scale) of the odd ones
                const uint32_t e = DP < 256 ? sc[r] : i < 2 ? sc[r] & 0xffu : sc[r] >> 8;
                one[r] = fp8_halves((r & 1) ? e * 256u : e);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {   // columns 2j and 2j + 1 of the word: the rows quad and quad + 8 of a product
                uint32_t a[4];
                pair_scaled(y[0][j], y[1][j], one[0], one[1], a[0], a[1]);
                pair_scaled(y[2][j], y[3][j], one[2], one[3], a[2], a[3]);
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int e = WT - 1; e >= 0; --e) mma_16816<__half>(o[t][4 * i + j], a, pb[t][0][e], pb[t][1][e]);
            }
        }
    };

    // The end of a row (`whole`) or of this block's part of it: join the four warps, 8 heads at a time.
    auto close_row = [&](int kvh, int h0, int nh, bool whole, bool first) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if (t * 8 >= nh) break;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l[t][j] += __shfl_xor_sync(0xffffffffu, l[t][j], x);
                if (quad == 0)
                    *reinterpret_cast<float2*>(s_ml + (warp * 8 + qc * 2 + j) * 2) = make_float2(base[t][j], l[t][j]);
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
                const int row = t * 8 + h, qh = kvh * p.rep + h0 + row;
                const int64_t part = (2 * static_cast<int64_t>(blockIdx.x) + (first ? 1 : 0)) * 16 + row;
                T* out = static_cast<T*>(p.out) + cp.b * p.out_row + qh * p.out_head;
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
                        p.lse[static_cast<int64_t>(cp.b) * p.heads + qh] = L != 0.0f ? (u + log2f(L)) * kLn2 : -INFINITY;
                    }
                }
            }
            if (NT > 1 || !CL) __syncthreads();
        }
    };

    // The next tile's copies, `tile` of its unit, and the tile in stage `step`.
    static_assert(NS == 4, "the steps below");
    auto run = [&](auto step, int tile) {
        issue((decltype(step)::value + NS - 1) % NS, tile);
        cp_async_wait<NS - 1>();
        __syncwarp();
        take(step);
        __syncwarp();   // every lane has read the tile before its stage is filled again
    };
    if constexpr (CL) {
        const int kvh = kv_head(cp.v), h0 = (cp.v - kvh * p.parts) * 16, nh = min(16, p.rep - h0);
        open_row(kvh, h0, nh);
        for (int n = 0; n < end; n += NS) {
            run(std::integral_constant<int, 0>{}, 0);
            if (n + 1 < end) run(std::integral_constant<int, 1>{}, 0);
            if (n + 2 < end) run(std::integral_constant<int, 2>{}, 0);
            if (n + 3 < end) run(std::integral_constant<int, 3>{}, 0);
        }
        close_row(kvh, h0, nh, p.cluster == 1, false);
    } else {
        static_assert(CL || TILES == NS, "the tiles of a unit are the stages");
        bool fresh = true;    // the next unit opens a new part or row
        bool first = false;   // ... the row itself
        while (cp.u < end) {
            const int kvh = kv_head(cp.v), h0 = (cp.v - kvh * p.parts) * 16;
            const int nh = min(16, p.rep - h0);          // query heads of this unit
            if (fresh) {
                fresh = false;
                first = cp.blk == 0;
                open_row(kvh, h0, nh);
            }
            run(std::integral_constant<int, 0>{}, 3);
            run(std::integral_constant<int, 1>{}, 0);
            run(std::integral_constant<int, 2>{}, 1);
            run(std::integral_constant<int, 3>{}, 2);
            const bool last = cp.blk + 1 == cp.r.nblk;
            if (last || cp.u + 1 == end) {
                fresh = true;
                close_row(kvh, h0, nh, first && last, first);
            }
            advance(cp);
        }
    }
    cp_async_wait<0>();
    if constexpr (CL)
        if (p.cluster > 1) {
            const int kvh = kv_head(cp.v), h0 = (cp.v - kvh * p.parts) * 16;
            paged_cluster_join<T>(p, smem, DP, rank, cp.b, kvh * p.rep + h0, min(16, p.rep - h0), warp, lane);
        }
}

}  // namespace chronos
