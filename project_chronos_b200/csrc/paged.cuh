// paged.cuh — the paged key-value cache: attention of one new token per
// sequence over its pages, the append that fills them and the eviction that
// empties them (include/chronos_paged.h).
//
// One-token attention.  With x_j = scale * log2(e) * q.k_j over the visible
// slots, any set of slots is summarised by
//     m = max x_j,  l = sum 2^(x_j - m),  o = sum 2^(x_j - m) v_j
// and two such triples join as m = max(m1, m2), l = l1 2^(m1-m) + l2 2^(m2-m),
// o likewise.  So every warp runs once over its slots with a running (m, l, o)
// in registers, warps join through shared memory, blocks through a workspace.
//
// Work split.  The visible slots of every (sequence, group of query heads) are
// cut into blocks of 64, all blocks of all sequences are numbered in one list
// and block c of the grid takes the c-th equal share of the list, read from the
// lengths on the device (a captured graph replays while the lengths grow).  A
// share holds whole rows, which it finishes itself, and at most two parts of
// rows (its first and its last), which a second kernel joins in the order of
// the list: the result does not depend on which block ran first.
#pragma once

#include <cooperative_groups.h>

#include "chronos_paged.h"
#include "common.cuh"

namespace chronos {

constexpr int kPdWarps = 4;
constexpr int kPdThreads = 32 * kPdWarps;
constexpr int kPdTile = 16;                     // slots a warp takes at a time
constexpr int kPdBlock = kPdTile * kPdWarps;    // slots of one unit of the work list
constexpr int kPdMaxGrid = 1024;
constexpr int kPdMaxRep = 256;                  // query heads per kv head

// Bits 0..n-1 set (none for n <= 0, all for n >= 32).
__device__ __forceinline__ uint32_t ones_below(int n) {
    return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
}

struct PagedDecodeParams {
    ChronosPagedCache c;
    int heads, rep;        // query heads, query heads per kv head
    int rows;              // query heads a unit computes at once (16 on the tensor cores, 8 without)
    int parts;             // ceil(rep / rows): units per kv head
    int window, sinks;
    int max_slots;         // lengths are cut to this
    int page_shift;        // log2(page_size), -1 where it is no power of two
    int cluster;           // blocks per row (cluster kernels)
    float sl2;             // scale * log2(e)
    const void* q;
    int64_t q_row, q_head;
    void* out;
    int64_t out_row, out_head;
    float* lse;
    const float* weights;
    float* weights_out;
    int64_t slot_cap;
    int grid;              // blocks of the first kernel
    int part_stride;       // floats per head of a part
    float* part_o;         // [2 * grid][rows][part_stride]
    float* part_ml;        // [2 * grid][rows][2]
    float* lse2;           // [B * H] log2 of the softmax sum (rows one block finished); weights only
    float* scores;         // [B * H][score_stride] x_j by visible index, or NULL; weights only
    int64_t score_stride;
    int join_blocks;       // blocks of the second kernel that join rows (the others add weights)
    int weight_chunks;     // blocks per (sequence, kv head) that add weights
    int32_t* status;
};

// The visible slots of sequence b, [0, first) and [lo, len), as a list of n places
// that starts every run of slots at a multiple of 16: place i is slot i before
// `front`, slot i + skip from there on.  Places before lo or at first.. are hidden.
struct PagedRow {
    int len, lo, first, front, skip, n, nblk;
    __device__ __forceinline__ int slot(int place) const { return place < front ? place : place + skip; }
    // Which of the 16 slots from `slot0` on are visible.
    __device__ __forceinline__ uint32_t visible16(int slot0) const {
        return (ones_below(first - slot0) | (ones_below(len - slot0) & ~ones_below(lo - slot0))) & 0xffffu;
    }
};
__device__ __forceinline__ PagedRow paged_row(const PagedDecodeParams& p, int b) {
    PagedRow r;
    r.len = min(max(p.c.lens[b], 0), p.max_slots);
    r.lo = p.window > 0 ? max(0, r.len - p.window) : 0;
    r.first = min(p.sinks, r.lo);
    r.front = (r.first + 15) & ~15;
    r.skip = max(0, (r.lo & ~15) - r.front);
    r.n = r.len - r.skip;
    r.nblk = max(1, (r.n + kPdBlock - 1) / kPdBlock);   // an empty row still has its zeros written
    return r;
}

// A place in the work list: unit u is block `blk` of row (b, v), v = kv head and part.
struct PagedIter {
    int u, b, v, blk;
    PagedRow r;
    __device__ __forceinline__ void advance(const PagedDecodeParams& p, int end) {
        ++u;
        if (++blk < r.nblk) return;
        blk = 0;
        if (++v < p.c.kv_heads * p.parts) return;
        v = 0;
        ++b;
        if (u < end) r = paged_row(p, b);
    }
};

// Report lengths that the table (or the running sums) cannot hold; one block does.
__device__ __forceinline__ void paged_check_lens(const PagedDecodeParams& p) {
    for (int b = threadIdx.x; b < p.c.batch; b += blockDim.x)
        if (p.c.lens[b] < 0 || p.c.lens[b] > p.max_slots) report_status(p.status, CHRONOS_ERR_INVALID_ARG);
}

// Number of units of all sequences (every lane of a warp gets it).
__device__ __forceinline__ int paged_total(const PagedDecodeParams& p, int lane) {
    int s = 0;
    for (int b = lane; b < p.c.batch; b += 32) s += paged_row(p, b).nblk;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s * p.c.kv_heads * p.parts;
}
// Units per block of the grid.
__device__ __forceinline__ int paged_share(const PagedDecodeParams& p, int total) {
    return max(1, (total + p.grid - 1) / p.grid);
}
// First unit of sequence b / the sequence that holds unit u (whole warps call these).
__device__ __forceinline__ int paged_first_unit(const PagedDecodeParams& p, int b, int lane) {
    int s = 0;
    for (int i = lane; i < b; i += 32) s += paged_row(p, i).nblk;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s * p.c.kv_heads * p.parts;
}
__device__ __forceinline__ PagedIter paged_seek(const PagedDecodeParams& p, int u, int lane) {
    const int per = p.c.kv_heads * p.parts;
    PagedIter it{};
    it.u = u;
    int before = 0;
    for (int base = 0; base < p.c.batch; base += 32) {
        const int b = base + lane;
        const int n = b < p.c.batch ? paged_row(p, b).nblk * per : 0;
        int inc = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += t;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, before + inc > u);
        if (past) {
            const int l = __ffs(past) - 1;
            const int start = before + __shfl_sync(0xffffffffu, inc - n, l);
            it.b = base + l;
            it.r = paged_row(p, it.b);
            it.v = (u - start) / it.r.nblk;
            it.blk = (u - start) % it.r.nblk;
            return it;
        }
        before += __shfl_sync(0xffffffffu, inc, 31);
    }
    return it;   // not reached for u < total
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float kLn2 = 0.6931471805599453f;
// log2 of the factor that weights carry when they are rounded to T for the second product
// (and with them their sum: it cancels).  fp16 has no numbers below 2^-25: without it a slot
// 2^-26 as heavy as the heaviest counted in the sum but not in the product, which cost
// 0.2 % where 131072 such slots followed one.  Maxima lag by up to 2^8, so 2^15 is reached.
template <typename T>
struct WeightLift {
    static constexpr float value = 0.0f;
};
template <>
struct WeightLift<__half> {
    static constexpr float value = 7.0f;
};

__device__ __forceinline__ void paged_split(const PagedDecodeParams& p, int slot, int& page, int& in_page) {
    if (p.page_shift >= 0) {
        page = slot >> p.page_shift;
        in_page = slot & (p.c.page_size - 1);
    } else {
        page = slot / p.c.page_size;
        in_page = slot - page * p.c.page_size;
    }
}

// The 16 places a warp takes next: which are visible, and their page and slot (lane i
// and i + 16 hold place i; all lanes hold place 0's where page_size is a multiple of
// 16: then all 16 lie in one page).  A page that is none hides its places.
struct PagedLook {
    int page, slot;
    uint32_t vis;
};
template <bool ONE_PAGE>
__device__ __forceinline__ PagedLook paged_look(const PagedDecodeParams& p, const PagedIter& it, int end, int warp,
                                                int lane) {
    PagedLook k{-1, 0, 0u};
    const int place = it.blk * kPdBlock + warp * kPdTile;
    if (it.u < end && place < it.r.n) {
        const int slot0 = it.r.slot(place);
        k.vis = it.r.visible16(slot0);
        const bool mine = ONE_PAGE || (k.vis >> (lane & 15)) & 1u;
        int page = 0;
        if (mine && k.vis) {
            paged_split(p, slot0 + (ONE_PAGE ? 0 : lane & 15), page, k.slot);
            k.page = p.c.page_table[it.b * p.c.page_table_stride + page];
            if (k.page < 0 || k.page >= p.c.num_pages) {
                report_status(p.status, CHRONOS_ERR_INVALID_ARG);
                k.page = -1;
            }
        }
    }
    return k;
}

// ---------------------------------------------------------------------------
// tensor-core path: bf16 / fp16, up to 16 query heads of a kv head at once
// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                                         uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// fp32 operands by two tf32 terms each, x = hi + lo: hi is x rounded to 11 bits, lo the
// rest, of which the tensor core takes the first 11 bits, so hi + lo is off by 2^-21 |x|
// at most, and hi hi + hi lo + lo hi leaves out a term below 2^-22.  What is not finite
// has no rest and stays out of the small terms (infinity times a rest of zero).
struct Tf32Pair {
    uint32_t hi, lo;
};
struct Tf32Value : Tf32Pair {
    uint32_t cross;   // hi in the small terms
};
__device__ __forceinline__ Tf32Pair tf32_split(float x) {
    Tf32Pair r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r.hi) : "f"(x));
    const float lo = x - __uint_as_float(r.hi);
    r.lo = lo == lo ? __float_as_uint(lo) : 0u;
    return r;
}
__device__ __forceinline__ Tf32Value tf32_value(float x) {
    Tf32Value r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r.hi) : "f"(x));
    const float lo = x - __uint_as_float(r.hi);
    const bool finite = lo == lo;
    r.lo = finite ? __float_as_uint(lo) : 0u;
    r.cross = finite ? r.hi : 0u;
    return r;
}
__device__ __forceinline__ void mma_1688_tf32(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                              uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// d += a * (b0, b1) for a 16 x 8 piece of K or V^T and the two rows of a split operand.
// The tensor core cuts its sums instead of rounding them: each piece is summed from
// zero, small terms first, and added to d in fp32 (a running sum on the tensor core was
// 2.8e-6 off where this is 4e-7).
__device__ __forceinline__ void mma_fp32(float (&d)[4], const float (&a)[4], const Tf32Pair& b0, const Tf32Pair& b1) {
    const Tf32Value x0 = tf32_value(a[0]), x1 = tf32_value(a[1]), x2 = tf32_value(a[2]), x3 = tf32_value(a[3]);
    float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    mma_1688_tf32(t, x0.cross, x1.cross, x2.cross, x3.cross, b0.lo, b1.lo);
    mma_1688_tf32(t, x0.lo, x1.lo, x2.lo, x3.lo, b0.hi, b1.hi);
    mma_1688_tf32(t, x0.hi, x1.hi, x2.hi, x3.hi, b0.hi, b1.hi);
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i] += t[i];
}
template <bool TRANS>
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
    if (TRANS)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                     : "r"(addr)
                     : "memory");
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                     : "r"(addr)
                     : "memory");
}
// Two fp32 values rounded to T, `lo` in the low half.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// 16 bytes global -> shared, zeros instead where !valid (src is not read then).
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
    const int n = valid ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// The parts of a row's `nh` heads (from `head0` on) that the blocks of a cluster hold in
// their shared memory, o [16][stride] fp32 and then (m, l) [16][2]: every block joins
// its share of the heads, in the order of the blocks.
template <typename T>
__device__ __forceinline__ void paged_cluster_join(const PagedDecodeParams& p, void* part, int stride, int rank, int b,
                                                   int head0, int nh, int warp, int lane) {
    namespace cg = cooperative_groups;
    cg::cluster_group cl = cg::this_cluster();
    cl.sync();
    const float* mine = static_cast<const float*>(part);
    for (int row = rank * kPdWarps + warp; row < nh; row += p.cluster * kPdWarps) {
        float M = -INFINITY, L = 0.0f;
        const float* peer = cl.map_shared_rank(mine, lane < p.cluster ? lane : 0) + 16 * stride + row * 2;
        const float pm = lane < p.cluster ? peer[0] : -INFINITY, pl = lane < p.cluster ? peer[1] : 0.0f;
        M = pm;
#pragma unroll
        for (int x = 4; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
        M = __shfl_sync(0xffffffffu, M, 0);
        const float u = M == -INFINITY ? 0.0f : M;
        const float c = exp2_fast(pm - u);
        L = pl * c;
#pragma unroll
        for (int x = 4; x > 0; x >>= 1) L += __shfl_xor_sync(0xffffffffu, L, x);
        L = __shfl_sync(0xffffffffu, L, 0);
        const float inv = L > 0.0f ? 1.0f / L : L;
        T* out = static_cast<T*>(p.out) + b * p.out_row + (head0 + row) * p.out_head;
        float acc[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
        for (int r = 0; r < p.cluster; ++r) {
            const float* po = cl.map_shared_rank(mine, r) + row * stride;
            const float w = __shfl_sync(0xffffffffu, c, r);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (lane + 32 * i < p.c.head_dim) acc[i] = fmaf(w, po[lane + 32 * i], acc[i]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (lane + 32 * i < p.c.head_dim) out[lane + 32 * i] = from_f32<T>(acc[i] * inv);
        if (lane == 0 && p.lse != nullptr)
            p.lse[static_cast<int64_t>(b) * p.heads + head0 + row] = L != 0.0f ? (u + log2f(L)) * kLn2 : -INFINITY;
    }
    cl.sync();   // nobody leaves while its part is read
}

// Swaps rows and columns of an 8 x 8 matrix of 16-bit values held by a warp.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// DP: the head dimension rounded up to 64, 128 or 256 (columns behind it are zero).
template <typename T, int DP>
struct PagedMma {
    static constexpr int kRowBytes = DP * static_cast<int>(sizeof(T));
    // Rows of 512 bytes have one stage, K and V of which are filled again separately as
    // soon as each is read: two blocks per SM then hide each other's waits (three stages
    // and one block per SM: 168 against 117 us for 16 x 16384 slots in fp32).
    static constexpr int kStages = kRowBytes == 512 ? 1 : 3;
    static constexpr int kTileBytes = kPdTile * kRowBytes;                    // K or V of one warp's tile
    static constexpr int kStageBytes = kPdWarps * 2 * kTileBytes;
    static constexpr int kOStride = DP + 4;                                   // fp32; four heads on different banks
    static constexpr int kMergeBytes = kPdWarps * 8 * kOStride * 4;
    static constexpr int kSmem = kStages * kStageBytes + kMergeBytes + kPdWarps * 8 * 2 * 4 + kStages * kPdWarps * 4;
    static constexpr int kBlocksPerSm = kRowBytes == 128 ? 3 : 2;
    static constexpr int kRows = sizeof(T) == 4 ? 8 : 16;                     // query heads of a unit at most
};

// HBM bound: 2 * D elements per visible slot and kv head against 4 * D flops per query
// head (fp32 layers by three tf32 products each).  Transposed products, S^T = K Q^T (16 slots x 8 heads) and
// O^T = V^T P^T (16 columns x 8 heads), take the query heads of a kv head as the
// 8-wide operand: no row of the 16-wide one is wasted, and one movmatrix turns the
// weights from the first product's result into the second's operand.  A warp owns 16
// slots at a time and its own ring of asynchronous copies (K and V rows go to shared
// memory 16 bytes at a time, swizzled against bank conflicts), so warps never wait for
// each other inside a row.  The maximum moves only when a score exceeds it by more
// than 2^8 in weight, which one vote per tile finds out.
//
// Measured, 32 / 8 heads of 128: 4 rows of 100003 to 131072 slots in fp16 291 to 310 us on
// different boxes, 6.4 to 6.8 TB/s (16-wide rows of heads, maxima and page lookups per row of
// slots: 418 us).  16 rows of 16384 slots in bf16: 32 / 8 heads of 64 105 us (5.1 TB/s), of 128
// 172 us (6.2), of 256 311 us (6.9); 8 / 2 heads of 64 35 us (3.8), of 128 54 us (5.0), of 256
// 89 us (6.0).  In fp32, heads of 128: 8 / 2 126 us (4.2 TB/s), 32 / 8 460 us (4.7), bound by
// the splitting into tf32.
//
// NT: groups of 8 query heads (1 or 2).  CL: a cluster of p.cluster blocks per row
// shares its blocks of 64 places and joins through distributed shared memory;
// otherwise block c takes the c-th share of the work list.
template <typename T, int DP, int NT, bool ONE_PAGE, bool CL>
__global__ void __launch_bounds__(kPdThreads, PagedMma<T, DP>::kBlocksPerSm) paged_decode_mma_kernel(
    const __grid_constant__ PagedDecodeParams p) {
    using S = PagedMma<T, DP>;
    constexpr int NS = S::kStages;
    constexpr int EPC = 16 / static_cast<int>(sizeof(T));   // elements of a 16-byte chunk
    constexpr int CPR = DP / EPC;          // chunks per row
    constexpr int RB = S::kRowBytes;
    constexpr int RPI = 32 / CPR;          // rows a warp copies per instruction
    constexpr float kGrow = 8.0f, kLift = WeightLift<T>::value;
    extern __shared__ __align__(128) uint8_t smem[];
    float* s_o = reinterpret_cast<float*>(smem + NS * S::kStageBytes);         // [warp][8 heads][kOStride]
    float* s_ml = s_o + S::kMergeBytes / 4;                                    // [warp][8][2]
    uint32_t* s_vis = reinterpret_cast<uint32_t*>(s_ml + kPdWarps * 16);       // [stage][warp]
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int quad = lane >> 2, qc = lane & 3;   // a product's row (slot, column of V) and pair of heads

    int end;
    PagedIter ld;
    const int rank = CL ? static_cast<int>(blockIdx.x) % p.cluster : 0;
    if constexpr (CL) {
        const int row = blockIdx.x / p.cluster, per = p.c.kv_heads * p.parts;
        ld.u = 0;
        ld.b = row / per;
        ld.v = row % per;
        ld.blk = rank;
        ld.r = paged_row(p, ld.b);
        end = ld.r.nblk > rank ? (ld.r.nblk - rank + p.cluster - 1) / p.cluster : 0;
        if (blockIdx.x == 0) paged_check_lens(p);
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
    PagedLook look = paged_look<ONE_PAGE>(p, ld, end, warp, lane);

    const int ch = lane % CPR, lrow = lane / CPR;
    const bool col = ch * EPC < p.c.head_dim;
    // what: 1 = K, 2 = V, 3 = both
    auto issue = [&](int stage, int what) {
        const uint32_t sk = smem_u32(smem + stage * S::kStageBytes + warp * 2 * S::kTileBytes);
        const int64_t g = ld.v / p.parts;
        uint32_t vis = look.vis;
        if (ONE_PAGE) {
            if (look.page < 0) vis = 0u;
            // one page: the rows stand a slot stride apart
            const T* ks = static_cast<const T*>(p.c.k_pages) + g * p.c.k_head_stride + ch * EPC;
            const T* vs = static_cast<const T*>(p.c.v_pages) + g * p.c.v_head_stride + ch * EPC;
            if (vis) {
                ks += look.page * p.c.k_page_stride + (look.slot + lrow) * p.c.k_slot_stride;
                vs += look.page * p.c.v_page_stride + (look.slot + lrow) * p.c.v_slot_stride;
            }
            const int64_t kstep = vis ? RPI * p.c.k_slot_stride : 0, vstep = vis ? RPI * p.c.v_slot_stride : 0;
#pragma unroll
            for (int i = 0; i < kPdTile / RPI; ++i) {
                const int r = i * RPI + lrow;
                const bool ok = col && ((vis >> r) & 1u);
                const uint32_t off = static_cast<uint32_t>(r * RB + ((ch ^ (r & 7)) << 4));
                if (what & 1) cp_async16(sk + off, ok ? ks : p.c.k_pages, ok);
                if (what & 2) cp_async16(sk + S::kTileBytes + off, ok ? vs : p.c.v_pages, ok);
                ks += kstep;
                vs += vstep;
            }
        } else {
            vis &= __ballot_sync(0xffffffffu, look.page >= 0) & 0xffffu;
            const T* kb = static_cast<const T*>(p.c.k_pages) + g * p.c.k_head_stride + ch * EPC;
            const T* vb = static_cast<const T*>(p.c.v_pages) + g * p.c.v_head_stride + ch * EPC;
#pragma unroll
            for (int i = 0; i < kPdTile / RPI; ++i) {
                const int r = i * RPI + lrow;
                const int page = __shfl_sync(0xffffffffu, look.page, r);
                const int64_t slot = __shfl_sync(0xffffffffu, look.slot, r);
                const bool ok = col && ((vis >> r) & 1u);
                const uint32_t off = static_cast<uint32_t>(r * RB + ((ch ^ (r & 7)) << 4));
                if (what & 1)
                    cp_async16(sk + off, ok ? kb + page * p.c.k_page_stride + slot * p.c.k_slot_stride : p.c.k_pages, ok);
                if (what & 2)
                    cp_async16(sk + S::kTileBytes + off, ok ? vb + page * p.c.v_page_stride + slot * p.c.v_slot_stride : p.c.v_pages, ok);
            }
        }
        if (NS > 1 && lane == 0) s_vis[stage * kPdWarps + warp] = vis;
        return vis;
    };
    uint32_t vis_next = 0u;     // one stage: what the tile in it shows
    if constexpr (NS == 1) {
        if (ld.u < end) vis_next = issue(0, 1);
        cp_async_commit();
        if (ld.u < end) issue(0, 2);
        cp_async_commit();
        if (ld.u < end) {
            advance(ld);
            look = paged_look<ONE_PAGE>(p, ld, end, warp, lane);
        }
    }
#pragma unroll
    for (int s = 0; s < NS - 1; ++s) {
        if (ld.u < end) {
            issue(s, 3);
            advance(ld);
            look = paged_look<ONE_PAGE>(p, ld, end, warp, lane);
        }
        cp_async_commit();
    }

    // where ldmatrix finds this lane's row of a 16 x 16 piece of K (rows: slots) or V
    uint32_t koff[4], voff[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int kr = (lane & 7) + ((lane >> 3) & 1) * 8, vr = (lane & 7) + (lane >> 4) * 8;
        koff[i] = static_cast<uint32_t>(kr * RB + (((2 * i + (lane >> 4)) ^ (lane & 7)) << 4));
        voff[i] = static_cast<uint32_t>(S::kTileBytes + vr * RB + (((2 * i + ((lane >> 3) & 1)) ^ (lane & 7)) << 4));
    }
    constexpr bool F32 = sizeof(T) == 4;
    static_assert(!F32 || NT == 1, "fp32 units have 8 heads");
    uint32_t qb[NT][F32 ? 1 : DP / 16][2];
    Tf32Pair qf[F32 ? DP / 8 : 1][2];
    float o[NT][DP / 16][4];
    float m[NT][2], l[NT][2];
    bool fresh = true;          // the next unit opens a new part or row
    int part_blk = 0;           // the block it opened with
    int stage = 0;
    while (cp.u < end || (CL && fresh)) {
        const int kvh = cp.v / p.parts, h0 = (cp.v % p.parts) * S::kRows;
        const int nh = min(S::kRows, p.rep - h0);             // query heads of this unit
        if (fresh) {
            fresh = false;
            part_blk = cp.blk;
            const T* q = static_cast<const T*>(p.q) + cp.b * p.q_row + static_cast<int64_t>(kvh * p.rep + h0) * p.q_head;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                m[t][0] = m[t][1] = -INFINITY;
                l[t][0] = l[t][1] = 0.0f;
#pragma unroll
                for (int i = 0; i < DP / 16; ++i) {
                    o[t][i][0] = o[t][i][1] = o[t][i][2] = o[t][i][3] = 0.0f;
#pragma unroll
                    for (int j = 0; j < 2 && !F32; ++j) {
                        const int row = t * 8 + quad, d = i * 16 + qc * 2 + j * 8;
                        qb[t][i][j] = row < nh && d < p.c.head_dim
                                          ? *reinterpret_cast<const uint32_t*>(q + row * p.q_head + d) : 0u;
                    }
                }
            }
            if constexpr (F32)
#pragma unroll
                for (int i = 0; i < DP / 8; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int d = i * 8 + qc + j * 4;
                        qf[i][j] = tf32_split(quad < nh && d < p.c.head_dim ? to_f32<T>(q[quad * p.q_head + d]) : 0.0f);
                    }
        }
        if constexpr (NS > 1) {
            if (ld.u < end) {
                issue(stage == 0 ? NS - 1 : stage - 1, 3);
                advance(ld);
                look = paged_look<ONE_PAGE>(p, ld, end, warp, lane);
            }
            cp_async_commit();
            cp_async_wait<NS - 1>();
        } else {
            cp_async_wait<1>();   // K; V of the tile may still be on its way
        }
        __syncwarp();
        const uint32_t st = smem_u32(smem + stage * S::kStageBytes + warp * 2 * S::kTileBytes);
        const uint32_t vis = NS == 1 ? vis_next : cp.u < end ? s_vis[stage * kPdWarps + warp] : 0u;
        const bool computes = vis || (p.scores != nullptr && cp.u < end);   // with running sums, hidden slots' scores are written too
        float s[NT][4];
        if (computes) {
#pragma unroll
            for (int t = 0; t < NT; ++t) s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.0f;
#pragma unroll
            for (int kk = 0; kk < RB / 32; ++kk) {   // 32 bytes of every slot's row at a time
                uint32_t ka[4];
                ldmatrix_x4<false>(ka, st + koff[kk & 3] + (kk >> 2) * 128);
                if constexpr (F32) {
                    const float a[4] = {__uint_as_float(ka[0]), __uint_as_float(ka[1]), __uint_as_float(ka[2]),
                                        __uint_as_float(ka[3])};
                    mma_fp32(s[0], a, qf[kk][0], qf[kk][1]);
                } else {
#pragma unroll
                    for (int t = 0; t < NT; ++t) mma_16816<T>(s[t], ka, qb[t][kk][0], qb[t][kk][1]);
                }
            }
        }
        if constexpr (NS == 1) {
            __syncwarp();   // K is read
            vis_next = ld.u < end ? issue(0, 1) : 0u;
            cp_async_commit();
            cp_async_wait<1>();   // V
            __syncwarp();
        }
        if (computes) {
            // s[t][0..1]: slot quad, heads 8t + 2qc, + 1; s[t][2..3]: slot quad + 8
            const bool on0 = (vis >> quad) & 1u, on1 = (vis >> (quad + 8)) & 1u;
            bool grow = false;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[t][j] = (j < 2 ? on0 : on1) ? s[t][j] * p.sl2 : -INFINITY;
                    grow |= s[t][j] > m[t][j & 1] + kGrow;
                }
            if (p.scores != nullptr) {
                const int idx = cp.blk * kPdBlock + warp * kPdTile + quad;
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int h = t * 8 + qc * 2 + j;
                        if (h < nh) {
                            float* sc = p.scores + (static_cast<int64_t>(cp.b) * p.heads + kvh * p.rep + h0 + h) * p.score_stride + idx;
                            sc[0] = s[t][j];
                            sc[8] = s[t][2 + j];
                        }
                    }
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
            uint32_t pb[NT][2];
            Tf32Pair pf[F32 ? 4 : 1];   // [8 slots][2 rows of 4]
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const float u0 = m[t][0] == -INFINITY ? 0.0f : m[t][0] - kLift, u1 = m[t][1] == -INFINITY ? 0.0f : m[t][1] - kLift;
                const float a = exp2_fast(s[t][0] - u0), b = exp2_fast(s[t][1] - u1);
                const float c = exp2_fast(s[t][2] - u0), d = exp2_fast(s[t][3] - u1);
                l[t][0] += a + c;
                l[t][1] += b + d;
                if constexpr (F32) {
                    // row k of 8 slots, head quad: held by the lane of slot k and pair quad / 2
                    const float w[4] = {a, b, c, d};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int src = (qc + (i & 1) * 4) * 4 + (quad >> 1);
                        const float x = __shfl_sync(0xffffffffu, w[(i >> 1) * 2], src);
                        const float y = __shfl_sync(0xffffffffu, w[(i >> 1) * 2 + 1], src);
                        pf[i] = tf32_split((quad & 1) ? y : x);
                    }
                    continue;
                }
                // weights in T for the second product; the sum keeps fp32
                pb[t][0] = transpose8x8(pack2<T>(a, b));
                pb[t][1] = transpose8x8(pack2<T>(c, d));
            }
#pragma unroll
            for (int dd = 0; dd < DP / 16; ++dd) {
                if constexpr (F32) {
                    const uint8_t* v = smem + stage * S::kStageBytes + warp * 2 * S::kTileBytes + S::kTileBytes;
#pragma unroll
                    for (int k = 0; k < 2; ++k) {   // slots 8k .. 8k + 7
                        float a[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int slot = k * 8 + qc + (i >> 1) * 4, d = dd * 16 + quad + (i & 1) * 8;
                            a[i] = *reinterpret_cast<const float*>(v + slot * RB + (((d >> 2) ^ (slot & 7)) << 4) + (d & 3) * 4);
                        }
                        mma_fp32(o[0][dd], a, pf[2 * k], pf[2 * k + 1]);
                    }
                } else {
                    uint32_t va[4];
                    ldmatrix_x4<true>(va, st + voff[dd & 3] + (dd >> 2) * 128);
#pragma unroll
                    for (int t = 0; t < NT; ++t) mma_16816<T>(o[t][dd], va, pb[t][0], pb[t][1]);
                }
            }
        }
        __syncwarp();   // every lane has read the tile before its stage is filled again
        if constexpr (NS == 1) {
            if (ld.u < end) {
                issue(0, 2);
                advance(ld);
                look = paged_look<ONE_PAGE>(p, ld, end, warp, lane);
            }
            cp_async_commit();
        }
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
#pragma unroll
                    for (int i = 0; i < DP / 16; ++i) {
                        float* dst = s_o + (warp * 8 + qc * 2 + j) * S::kOStride + i * 16 + quad;
                        dst[0] = o[t][i][j];
                        dst[8] = o[t][i][2 + j];
                    }
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
                    const float inv = whole ? (L > 0.0f ? 1.0f / L : L) : 1.0f;
                    const int row = t * 8 + h, head = kvh * p.rep + h0 + row;
                    const int64_t part = (2 * static_cast<int64_t>(blockIdx.x) + (part_blk == 0 ? 1 : 0)) * S::kRows + row;
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
                        if (!whole) *reinterpret_cast<float2*>(po + d) = make_float2(a, b);
                        else if (d < p.c.head_dim) {
                            if constexpr (F32) *reinterpret_cast<float2*>(out + d) = make_float2(a * inv, b * inv);
                            else *reinterpret_cast<uint32_t*>(out + d) = pack2<T>(a * inv, b * inv);
                        }
                    }
                    if (lane == 0) {
                        if (!whole) {
                            float* ml = CL ? reinterpret_cast<float*>(smem) + 16 * DP + row * 2 : p.part_ml + part * 2;
                            *reinterpret_cast<float2*>(ml) = make_float2(M, L);
                        } else {
                            const float lg = L != 0.0f ? u + log2f(L) : -INFINITY;
                            if (p.lse != nullptr) p.lse[static_cast<int64_t>(cp.b) * p.heads + head] = lg * kLn2;
                            if (p.scores != nullptr) p.lse2[static_cast<int64_t>(cp.b) * p.heads + head] = lg;
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
            const int kvh = cp.v / p.parts, h0 = (cp.v % p.parts) * S::kRows;
            paged_cluster_join<T>(p, smem, DP, rank, cp.b, kvh * p.rep + h0, min(S::kRows, p.rep - h0), warp, lane);
        }
}

// ---------------------------------------------------------------------------
// general path: head dimensions or strides the copies above cannot take, fp32 heads
// of more than 128.  Same work list; 8 query
// heads at once, fp32 products.  K: four lanes share a slot (their partial dot
// products meet in two shuffles), two slots per lane in flight; V: the lanes
// split the columns and run over the warp's 16 slots.
// ---------------------------------------------------------------------------
constexpr int kPdSimtRows = 8;

template <typename T, bool VEC>
__device__ __forceinline__ void load4(const T* p, int d, int dim, float (&v)[4]) {
    if (VEC) {
        if constexpr (sizeof(T) == 4) {
            const float4 f = *reinterpret_cast<const float4*>(p + d);
            v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
        } else {
            const uint2 u = *reinterpret_cast<const uint2*>(p + d);
            const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = to_f32<T>(t[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = d + i < dim ? to_f32<T>(p[d + i]) : 0.0f;
    }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kPdThreads) paged_decode_simt_kernel(const __grid_constant__ PagedDecodeParams p) {
    constexpr int R = kPdSimtRows, MAXD = CHRONOS_PAGED_MAX_HEAD_DIM;
    __shared__ __align__(16) float s_q[R][MAXD];
    __shared__ __align__(16) float s_o[kPdWarps - 1][R][MAXD];
    __shared__ __align__(16) float s_p[kPdWarps][kPdTile][R];
    __shared__ float s_c[kPdWarps][R];
    __shared__ float s_ml[kPdWarps][R][2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int D = p.c.head_dim, D4 = (D + 3) / 4;
    const int slot_lane = lane >> 2, part = lane & 3;

    const int total = paged_total(p, lane);
    const int share = paged_share(p, total);
    const int begin = static_cast<int>(blockIdx.x) * share, end = min(total, begin + share);
    if (blockIdx.x == 0) paged_check_lens(p);
    if (begin >= end) return;
    PagedIter cp = paged_seek(p, begin, lane);
    PagedLook look = paged_look<false>(p, cp, end, warp, lane);
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};   // heads 2 * part, 2 * part + 1
    float o[R][8];
    bool fresh = true;
    int part_blk = 0;
    while (cp.u < end) {
        const int kvh = cp.v / p.parts, h0 = (cp.v % p.parts) * R;
        const int nh = min(R, p.rep - h0);
        if (fresh) {
            fresh = false;
            part_blk = cp.blk;
            m[0] = m[1] = -INFINITY;
            l[0] = l[1] = 0.0f;
#pragma unroll
            for (int h = 0; h < R; ++h)
#pragma unroll
                for (int i = 0; i < 8; ++i) o[h][i] = 0.0f;
            __syncthreads();
            const T* q = static_cast<const T*>(p.q) + cp.b * p.q_row + static_cast<int64_t>(kvh * p.rep + h0) * p.q_head;
            for (int i = threadIdx.x; i < R * MAXD; i += kPdThreads) {
                const int h = i / MAXD, d = i % MAXD;
                s_q[h][d] = h < nh && d < D ? to_f32<T>(q[h * p.q_head + d]) : 0.0f;
            }
            __syncthreads();
        }
        PagedIter nx = cp;
        nx.advance(p, end);
        const PagedLook cur = look;
        look = paged_look<false>(p, nx, end, warp, lane);
        const uint32_t vis = __ballot_sync(0xffffffffu, cur.page >= 0) & 0xffffu;
        if (vis || p.scores != nullptr) {
            // scores of slots slot_lane and slot_lane + 8
            const int pg0 = __shfl_sync(0xffffffffu, cur.page, slot_lane), pg1 = __shfl_sync(0xffffffffu, cur.page, slot_lane + 8);
            const int64_t sl0 = __shfl_sync(0xffffffffu, cur.slot, slot_lane), sl1 = __shfl_sync(0xffffffffu, cur.slot, slot_lane + 8);
            const T* kb = static_cast<const T*>(p.c.k_pages) + kvh * p.c.k_head_stride;
            const T* k0 = kb + (pg0 >= 0 ? pg0 * p.c.k_page_stride + sl0 * p.c.k_slot_stride : 0);
            const T* k1 = kb + (pg1 >= 0 ? pg1 * p.c.k_page_stride + sl1 * p.c.k_slot_stride : 0);
            float s0[R], s1[R];
#pragma unroll
            for (int h = 0; h < R; ++h) s0[h] = s1[h] = 0.0f;
#pragma unroll 4
            for (int c = part; c < D4; c += 4) {
                float a[4] = {0.0f, 0.0f, 0.0f, 0.0f}, b[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                if (pg0 >= 0) load4<T, VEC>(k0, c * 4, D, a);
                if (pg1 >= 0) load4<T, VEC>(k1, c * 4, D, b);
#pragma unroll
                for (int h = 0; h < R; ++h) {
                    const float4 qv = *reinterpret_cast<const float4*>(&s_q[h][c * 4]);
                    s0[h] = fmaf(a[0], qv.x, fmaf(a[1], qv.y, fmaf(a[2], qv.z, fmaf(a[3], qv.w, s0[h]))));
                    s1[h] = fmaf(b[0], qv.x, fmaf(b[1], qv.y, fmaf(b[2], qv.z, fmaf(b[3], qv.w, s1[h]))));
                }
            }
#pragma unroll
            for (int h = 0; h < R; ++h) {
#pragma unroll
                for (int x = 1; x < 4; x <<= 1) {
                    s0[h] += __shfl_xor_sync(0xffffffffu, s0[h], x);
                    s1[h] += __shfl_xor_sync(0xffffffffu, s1[h], x);
                }
            }
            // lane `part` of a slot's four keeps heads 2 * part and 2 * part + 1
            float x[2][2];
#pragma unroll
            for (int h = 0; h < R; ++h)
                if ((h >> 1) == part) {
                    x[h & 1][0] = pg0 >= 0 ? s0[h] * p.sl2 : -INFINITY;
                    x[h & 1][1] = pg1 >= 0 ? s1[h] * p.sl2 : -INFINITY;
                }
            const int idx = cp.blk * kPdBlock + warp * kPdTile + slot_lane;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int h = 2 * part + j;
                if (p.scores != nullptr && h < nh) {
                    float* sc = p.scores + (static_cast<int64_t>(cp.b) * p.heads + kvh * p.rep + h0 + h) * p.score_stride + idx;
                    sc[0] = x[j][0];
                    sc[8] = x[j][1];
                }
                float n = fmaxf(x[j][0], x[j][1]);
#pragma unroll
                for (int t = 4; t < 32; t <<= 1) n = fmaxf(n, __shfl_xor_sync(0xffffffffu, n, t));
                n = fmaxf(n, m[j]);
                const float u = n == -INFINITY ? 0.0f : n;
                const float c = exp2_fast(m[j] - u);
                m[j] = n;
                const float a = exp2_fast(x[j][0] - u), b = exp2_fast(x[j][1] - u);
                l[j] = l[j] * c + a + b;
                s_p[warp][slot_lane][h] = a;
                s_p[warp][slot_lane + 8][h] = b;
                if (slot_lane == 0) s_c[warp][h] = c;
            }
            __syncwarp();
#pragma unroll
            for (int h = 0; h < R; ++h) {
                const float c = s_c[warp][h];
#pragma unroll
                for (int i = 0; i < 8; ++i) o[h][i] *= c;
            }
            const T* vb = static_cast<const T*>(p.c.v_pages) + kvh * p.c.v_head_stride;
#pragma unroll 8
            for (int t = 0; t < kPdTile; ++t) {
                const int page = __shfl_sync(0xffffffffu, cur.page, t);
                const int64_t slot = __shfl_sync(0xffffffffu, cur.slot, t);
                if (page < 0) continue;
                const T* v = vb + page * p.c.v_page_stride + slot * p.c.v_slot_stride;
                const float4 pa = *reinterpret_cast<const float4*>(&s_p[warp][t][0]);
                const float4 pb = *reinterpret_cast<const float4*>(&s_p[warp][t][4]);
                const float ph[R] = {pa.x, pa.y, pa.z, pa.w, pb.x, pb.y, pb.z, pb.w};
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int d = lane * 4 + 128 * i;
                    if (d < D) {
                        float a[4];
                        load4<T, VEC>(v, d, D, a);
#pragma unroll
                        for (int h = 0; h < R; ++h)
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[h][i * 4 + e] = fmaf(ph[h], a[e], o[h][i * 4 + e]);
                    }
                }
            }
            __syncwarp();
        }
        if (cp.blk + 1 == cp.r.nblk || cp.u + 1 == end) {
            fresh = true;
            const bool whole = part_blk == 0 && cp.blk + 1 == cp.r.nblk;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int t = 4; t < 32; t <<= 1) l[j] += __shfl_xor_sync(0xffffffffu, l[j], t);
                if (slot_lane == 0) {
                    s_ml[warp][2 * part + j][0] = m[j];
                    s_ml[warp][2 * part + j][1] = l[j];
                }
            }
            __syncthreads();
            float M[R], L[R];
#pragma unroll
            for (int h = 0; h < R; ++h) {
                M[h] = -INFINITY;
                L[h] = 0.0f;
#pragma unroll
                for (int w = 0; w < kPdWarps; ++w) M[h] = fmaxf(M[h], s_ml[w][h][0]);
                const float u = M[h] == -INFINITY ? 0.0f : M[h];
#pragma unroll
                for (int w = 0; w < kPdWarps; ++w) L[h] += s_ml[w][h][1] * exp2_fast(s_ml[w][h][0] - u);
                const float c = exp2_fast(s_ml[warp][h][0] - u);
#pragma unroll
                for (int i = 0; i < 8; ++i) o[h][i] *= c;
            }
            if (warp > 0)
#pragma unroll
                for (int h = 0; h < R; ++h)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        *reinterpret_cast<float4*>(&s_o[warp - 1][h][lane * 4 + 128 * i]) =
                            make_float4(o[h][4 * i], o[h][4 * i + 1], o[h][4 * i + 2], o[h][4 * i + 3]);
            __syncthreads();
            if (warp == 0) {
#pragma unroll
                for (int h = 0; h < R; ++h) {
                    if (h >= nh) break;
                    const float inv = whole ? (L[h] > 0.0f ? 1.0f / L[h] : L[h]) : 1.0f;
                    const int64_t slot = (2 * static_cast<int64_t>(blockIdx.x) + (part_blk == 0 ? 1 : 0)) * R + h;
                    const int head = kvh * p.rep + h0 + h;
                    T* out = static_cast<T*>(p.out) + cp.b * p.out_row + head * p.out_head;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int d = lane * 4 + 128 * (i >> 2) + (i & 3);
                        if (d < D) {
                            float a = o[h][i];
#pragma unroll
                            for (int w = 0; w < kPdWarps - 1; ++w) a += s_o[w][h][d];
                            if (whole) out[d] = from_f32<T>(a * inv);
                            else p.part_o[slot * p.part_stride + d] = a;
                        }
                    }
                    if (lane == 0) {
                        if (!whole) {
                            p.part_ml[slot * 2] = M[h];
                            p.part_ml[slot * 2 + 1] = L[h];
                        } else {
                            const float lg = L[h] != 0.0f ? (M[h] == -INFINITY ? 0.0f : M[h]) + log2f(L[h]) : -INFINITY;
                            if (p.lse != nullptr) p.lse[static_cast<int64_t>(cp.b) * p.heads + head] = lg * kLn2;
                            if (p.scores != nullptr) p.lse2[static_cast<int64_t>(cp.b) * p.heads + head] = lg;
                        }
                    }
                }
            }
        }
        cp = nx;
    }
}

// ---------------------------------------------------------------------------
// join of the parts, and the running sums of the attention weights
// ---------------------------------------------------------------------------
constexpr int kPdJoinThreads = 256;
constexpr int kPdWeightSlots = 4 * kPdJoinThreads;   // slots per block that adds weights

// The parts of row (b, v): blocks c0..c1 of the grid; part(c) its place in the workspace.
struct PagedParts {
    int c0, c1;
    __device__ __forceinline__ int64_t part(int c) const { return 2 * static_cast<int64_t>(c) + (c == c0 ? 1 : 0); }
};
__device__ __forceinline__ PagedParts paged_parts(const PagedDecodeParams& p, int b, int v, int lane) {
    const int share = paged_share(p, paged_total(p, lane));
    const int nblk = paged_row(p, b).nblk;
    const int s = paged_first_unit(p, b, lane) + v * nblk;
    return PagedParts{s / share, (s + nblk - 1) / share};
}

template <typename T>
__global__ void __launch_bounds__(kPdJoinThreads) paged_join_kernel(const __grid_constant__ PagedDecodeParams p) {
    constexpr int W = kPdJoinThreads / 32;
    __shared__ float s_w[kPdMaxGrid];
    __shared__ float s_red[W];
    __shared__ float s_o[W][CHRONOS_PAGED_MAX_HEAD_DIM];
    __shared__ float s_lse[kPdMaxRep];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    if (static_cast<int>(blockIdx.x) < p.join_blocks) {
        const int b = blockIdx.x / p.heads, head = blockIdx.x % p.heads;
        const int kvh = head / p.rep, hr = head % p.rep;
        const PagedParts pp = paged_parts(p, b, kvh * p.parts + hr / p.rows, lane);
        if (pp.c0 == pp.c1) return;   // one block finished the row
        const int n = pp.c1 - pp.c0 + 1, row = hr % p.rows;
        float M = -INFINITY;
        for (int i = threadIdx.x; i < n; i += kPdJoinThreads)
            M = fmaxf(M, p.part_ml[(pp.part(pp.c0 + i) * p.rows + row) * 2]);
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
        if (lane == 0) s_red[warp] = M;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) M = fmaxf(M, s_red[w]);
        const float u = M == -INFINITY ? 0.0f : M;
        float L = 0.0f;
        for (int i = threadIdx.x; i < n; i += kPdJoinThreads) {
            const float* ml = p.part_ml + (pp.part(pp.c0 + i) * p.rows + row) * 2;
            const float c = exp2_fast(ml[0] - u);
            s_w[i] = c;
            L += ml[1] * c;
        }
        L = warp_sum(L);
        __syncthreads();
        if (lane == 0) s_red[warp] = L;
        __syncthreads();
        L = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) L += s_red[w];
        // warps take every W-th part, lanes 4 columns (twice for more than 128)
        float acc[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
        const int D = p.c.head_dim;
#pragma unroll 4
        for (int i = warp; i < n; i += W) {
            const float* po = p.part_o + (pp.part(pp.c0 + i) * p.rows + row) * p.part_stride;
            const float c = s_w[i];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int d = lane * 4 + 128 * j;
                if (d < D) {
                    const float4 f = *reinterpret_cast<const float4*>(po + d);
                    acc[4 * j] = fmaf(c, f.x, acc[4 * j]);
                    acc[4 * j + 1] = fmaf(c, f.y, acc[4 * j + 1]);
                    acc[4 * j + 2] = fmaf(c, f.z, acc[4 * j + 2]);
                    acc[4 * j + 3] = fmaf(c, f.w, acc[4 * j + 3]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) s_o[warp][lane * 4 + 128 * (i >> 2) + (i & 3)] = acc[i];
        __syncthreads();
        const float inv = L > 0.0f ? 1.0f / L : L;   // 0 where nothing was visible; NaN stays
        T* out = static_cast<T*>(p.out) + b * p.out_row + head * p.out_head;
        for (int d = threadIdx.x; d < D; d += kPdJoinThreads) {
            float a = 0.0f;
#pragma unroll
            for (int w = 0; w < W; ++w) a += s_o[w][d];
            out[d] = from_f32<T>(a * inv);
        }
        if (threadIdx.x == 0 && p.lse != nullptr)
            p.lse[static_cast<int64_t>(b) * p.heads + head] = L != 0.0f ? (u + log2f(L)) * kLn2 : -INFINITY;
        return;
    }
    // weights_out[b, g, j] = weights[b, g, j] + sum_h 2^(x_hj - lse2_h)
    int i = static_cast<int>(blockIdx.x) - p.join_blocks;
    const int chunk = i % p.weight_chunks;
    i /= p.weight_chunks;
    const int g = i % p.c.kv_heads, b = i / p.c.kv_heads;
    const PagedRow r = paged_row(p, b);
    if (chunk * kPdWeightSlots >= r.len) return;
    const int64_t hb = static_cast<int64_t>(b) * p.heads + g * p.rep;
    for (int h = warp; h < p.rep; h += W) {
        const PagedParts pp = paged_parts(p, b, g * p.parts + h / p.rows, lane);
        float lg;
        if (pp.c0 == pp.c1) {
            lg = p.lse2[hb + h];
        } else {
            const int row = h % p.rows;
            float M = -INFINITY;
            for (int c = pp.c0 + lane; c <= pp.c1; c += 32) M = fmaxf(M, p.part_ml[(pp.part(c) * p.rows + row) * 2]);
#pragma unroll
            for (int x = 16; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
            const float u = M == -INFINITY ? 0.0f : M;
            float L = 0.0f;
            for (int c = pp.c0 + lane; c <= pp.c1; c += 32) {
                const float* ml = p.part_ml + (pp.part(c) * p.rows + row) * 2;
                L += ml[1] * exp2_fast(ml[0] - u);
            }
            L = warp_sum(L);
            lg = L != 0.0f ? u + log2f(L) : INFINITY;   // nothing readable: weights of zero
        }
        if (lane == 0) s_lse[h] = lg == -INFINITY ? INFINITY : lg;
    }
    __syncthreads();
    const int64_t wb = (static_cast<int64_t>(b) * p.c.kv_heads + g) * p.slot_cap;
    const int j0 = chunk * kPdWeightSlots + threadIdx.x * 4;
    const float* sc = p.scores + hb * p.score_stride;
    const bool vec = r.skip == 0 && r.first == r.lo && j0 + 4 <= r.len && (p.slot_cap & 3) == 0 &&
                     ((reinterpret_cast<uintptr_t>(p.weights) | reinterpret_cast<uintptr_t>(p.weights_out)) & 15) == 0;
    if (vec) {   // every slot visible: index = slot
        float4 w = *reinterpret_cast<const float4*>(p.weights + wb + j0);
        for (int h = 0; h < p.rep; ++h) {
            const float4 x = *reinterpret_cast<const float4*>(sc + h * p.score_stride + j0);
            const float lg = s_lse[h];
            w.x += exp2_fast(x.x - lg);
            w.y += exp2_fast(x.y - lg);
            w.z += exp2_fast(x.z - lg);
            w.w += exp2_fast(x.w - lg);
        }
        *reinterpret_cast<float4*>(p.weights_out + wb + j0) = w;
    } else {
        for (int j = j0; j < min(j0 + 4, r.len); ++j) {
            float w = p.weights[wb + j];
            const int idx = j < r.front ? j : j - r.skip;   // its place, if it has one
            if (j < r.first || j >= r.lo)
                for (int h = 0; h < p.rep; ++h) w += exp2_fast(sc[h * p.score_stride + idx] - s_lse[h]);
            p.weights_out[wb + j] = w;
        }
    }
}

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
