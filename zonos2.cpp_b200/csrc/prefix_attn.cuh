// prefix_attn.cuh — what the kernels of prefix_attention share (k_prefix_attn.cu,
// k_prefix_tc.cu): the launch's parameters, the cutting of the line of units, and small
// device helpers.
#pragma once

#include "ops.cuh"
#include "ops.h"
#include "tc05.cuh"

#include <atomic>

namespace z2b {

constexpr int TC_ROWS = 256, TC_KEYS = 128;    // rows of a segment and keys of a unit on tcgen05
constexpr int MIN_UNITS = 2;           // line positions per worker at least, before more workers are used
// Line positions that a segment takes ahead of its units: what a worker spends on a segment
// besides its units (queries, the partial result), so that ranges of short segments are not
// the longest ones.
constexpr int SEG_COST = 1, TC_SEG_COST = 3;
// The reference m of a row's probabilities 2^(s - m) is its maximum less P_SHIFT, and stays until
// the maximum is LAG above it: probabilities lie below 2^15, within f16, sums and O are f32, so
// nothing overflows (bf16 values of V below 2^80: 2^15 of each of 2^30 keys), rescaling O becomes rare, and the shift keeps small probabilities of f16
// caches off the bottom of its range (2^-31 of the largest is still there).
constexpr float P_SHIFT = 7.0f, LAG = 15.0f;

struct AttnP {
    const void* q;
    long long q_row, q_head, table_stride;
    const int *row_off, *seq_len, *table, *prefix_pages;
    uint32_t* err;
    int n_rows, n_seq, nkv, G, page_len, n_pages, max_pages, prefix_len;
    uint32_t g_mul;                    // ceil(2^32 / G), for quotients by G of numbers x with x G < 2^32
    int box_rows, box_halves;          // rows of one TMA box (a power of two that divides page_len, at most a
                                       // unit's keys), and how many 64-dim halves it holds
    float scale2;                      // scale * log2(e)
    int pf_row_tiles;                  // row tiles of the prefix in this launch (0: none)
    int after_prefix;                  // 1: the launch before is the prefix's, which this one runs beside
    int early, head_start;             // CTAs that find an SM while that one runs, and line positions each gets through meanwhile
    float* part_o;                     // [slots][rows of a segment][head_dim]
    float2* part_ml;                   // [slots][rows of a segment] (m in log2 units, l)
    uint32_t polls;                    // limit of a wait
    int* plan;                         // [2][n_seq + 1] unit and segment offsets of the streams, written for the join
};

__device__ __forceinline__ int div_g(const AttnP& p, int x) { return p.G == 1 ? x : (int)__umulhi((uint32_t)x, p.g_mul); }
__device__ __forceinline__ int cdiv(int a, int b) { return (a + b - 1) / b; }

// One stream's extent, with offsets and lengths that are out of range cut to nothing. Where no
// stream's offsets drop, the streams' rows are disjoint, which bounds all sums over them; where one
// does, no stream's rows are taken.
struct SeqInfo { int lo, n, len, nt, qt; bool bad, drops; };
template <int MT, int KU> __device__ __forceinline__ SeqInfo seq_info(const AttnP& p, int b, bool l2) {
    SeqInfo s;
    const int lo = ld_word(p.row_off + b, l2), hi = ld_word(p.row_off + b + 1, l2), len = ld_word(p.seq_len + b, l2);
    const long long cap = (long long)p.max_pages * p.page_len;
    s.drops = hi < lo;
    s.bad = lo < 0 || hi < lo || hi > p.n_rows || len < 0 || len > cap;
    s.lo = lo;
    s.n = s.bad ? 0 : hi - lo;
    s.len = s.bad ? 0 : len;
    s.nt = s.n ? cdiv(s.len, KU) : 0;
    s.qt = cdiv(s.n * p.G, MT);
    return s;
}

// A line of W positions cut into equal ranges: worker i's begins at floor(W i / workers). W is
// below 2^31 and workers at most 2^11, so 32-bit arithmetic is exact: W i / workers =
// i (W / workers) + i (W % workers) / workers, and the last quotient, of a number x with
// x workers < 2^32, is the high word of x ceil(2^32 / workers).
struct Cut {
    int workers, each, rest;
    uint32_t inv;
    __device__ __forceinline__ Cut(int W, int most) {
        workers = max(1, min(most, W / MIN_UNITS));
        each = (int)((unsigned)W / (unsigned)workers);
        rest = W - each * workers;
        inv = workers > 1 ? 0xffffffffu / (unsigned)workers + 1u : 0u;
    }
    __device__ __forceinline__ Cut() {}
    __device__ __forceinline__ int begin(int i) const { return i * each + (int)__umulhi((unsigned)(i * rest), inv); }
    // The worker that holds position u: an f32 guess, off by one at most, put right exactly.
    __device__ __forceinline__ int owner(int u, int W) const {
        int i = min(workers - 1, (int)__fdividef((float)u * (float)workers, (float)W));
        while (begin(i) > u) --i;
        while (begin(i + 1) <= u) ++i;
        return i;
    }
};

// The line of the own kernel: workers of the first p.early CTAs take [0, mid), which their head
// start makes longer ranges, the others [mid, W). Worker numbers go along the line.
struct Cuts {
    Cut a, b;
    int W, mid, na;
    __device__ __forceinline__ Cuts(const AttnP& p, int W_, int ctas, int warps) : W(W_), mid(0), na(0) {
        if (p.early > 0) {
            const long long lead = (long long)p.early * p.head_start;
            mid = W <= lead ? W : (int)(lead + (W - lead) * p.early / ctas);
            a = Cut(mid, p.early * warps);
            na = a.workers;
        }
        b = Cut(W - mid, (ctas - p.early) * warps);
    }
    __device__ __forceinline__ int owner(int u) const { return u < mid ? a.owner(u, mid) : na + b.owner(u - mid, W - mid); }
};

template <typename T> __device__ __forceinline__ void mma_t(float* d, const uint32_t* a, uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma_t<__half>(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    mma16816(d, a[0], a[1], a[2], a[3], b0, b1);
}
template <> __device__ __forceinline__ void mma_t<__nv_bfloat16>(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
        "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
// Transpose of an 8 x 8 tile of 16-bit values held two to a lane.
__device__ __forceinline__ uint32_t movm(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
// True in one thread of a whole converged warp, the same one at every call. Under this
// predicate the compiler issues a copy or a product once; under a plain lane test it must
// allow for several lanes and loops over them, moving every operand again (measured: some
// 120 cycles a product).
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(one));
    return one != 0;
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* m) {
    asm volatile("prefetch.tensormap [%0];" :: "l"(reinterpret_cast<uint64_t>(m)) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// One box of a page: rows [row, row + box_rows) of key head h, dims from 64 half on. The view is
// [page][head][half][row][up to 64 dims], so one box can bring both halves of a tile's rows.
__device__ __forceinline__ void tma_load_page(uint32_t dst, const CUtensorMap* map, int row, int half, int h, int page, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
        :: "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(row), "r"(half), "r"(h), "r"(page), "r"(smem_u32(bar))
        : "memory");
}

// How a tile of `keys` rows is cut into boxes: runs of rows that stay within a page, both halves
// of head_dim 128 in one box when a run is the whole tile.
inline void cut_boxes(AttnP& p, int keys, int hd) {
    const int pow2 = p.page_len & -p.page_len;
    p.box_rows = pow2 > keys ? keys : pow2;
    p.box_halves = hd > 64 && p.box_rows == keys ? 2 : 1;
}

inline bool make_page_map(CUtensorMap* m, const void* base, const z2b_paged_kv& c, const AttnP& p) {
    auto enc = tensor_map_encoder();
    if (!enc) return false;
    const int inner = c.head_dim < 64 ? c.head_dim : 64;
    const cuuint64_t dims[5] = {(cuuint64_t)inner, (cuuint64_t)c.page_len, (cuuint64_t)(c.head_dim / inner), (cuuint64_t)c.n_head_kv,
                                (cuuint64_t)c.n_pages};
    const cuuint64_t strides[4] = {(cuuint64_t)c.row_stride * 2, 128, (cuuint64_t)c.head_stride * 2, (cuuint64_t)c.page_stride * 2};
    const cuuint32_t box[5] = {(cuuint32_t)inner, (cuuint32_t)p.box_rows, (cuuint32_t)p.box_halves, 1, 1}, one[5] = {1, 1, 1, 1, 1};
    const CUtensorMapSwizzle sw = inner == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : inner == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B;
    return enc(m, c.type == Z2B_TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5,
               const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, sw,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The prefix on tcgen05 (k_prefix_tc.cu): segments of TC_ROWS rows, units of TC_KEYS keys.
// head_dim 64 or 128.
template <typename T, int HD>
cudaError_t launch_prefix_tc(const AttnP& p, const CUtensorMap& km, const CUtensorMap& vm, int grid, cudaStream_t s);

}  // namespace z2b
