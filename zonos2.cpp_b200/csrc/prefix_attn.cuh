// prefix_attn.cuh — what the kernels of prefix_attention share (k_prefix_attn.cu,
// k_prefix_tc.cu): the launch's parameters, the cutting of the line of units, and small
// device helpers.
#pragma once

#include "ops.cuh"
#include "ops.h"
#include "tc05.cuh"

#include <atomic>

namespace z2b {

constexpr int KU = 32;                 // keys of a unit on the warp-level kernel
constexpr int TC_ROWS = 256, TC_KEYS = 128;    // rows of a segment and keys of a unit on tcgen05
constexpr int MIN_UNITS = 2;           // units per worker at least, before more workers are used

struct AttnP {
    const void* q;
    long long q_row, q_head, table_stride;
    const int *row_off, *seq_len, *table, *prefix_pages;
    uint32_t* err;
    int n_rows, n_seq, nkv, G, page_len, n_pages, max_pages, prefix_len;
    int box_rows;                      // rows of one TMA box: a power of two that divides page_len, at most a unit's keys
    float scale2;                      // scale * log2(e)
    int pf_row_tiles;                  // row tiles of the prefix in this launch (0: none)
    int max_slots;
    int after_prefix;                  // 1: the launch before is the prefix's, which this one runs beside
    float* part_o;                     // [max_slots][rows of a segment][head_dim]
    float2* part_ml;                   // [max_slots][rows of a segment] (m in log2 units, l)
    int* plan;                         // [2][n_seq + 1] unit and segment offsets of the streams, written for the join
};

__device__ __forceinline__ int cdiv(int a, int b) { return (a + b - 1) / b; }

// One stream's extent, with offsets and lengths that are out of range cut to nothing.
struct SeqInfo { int lo, n, len, nt, qt; bool bad; };
template <int MT> __device__ __forceinline__ SeqInfo seq_info(const AttnP& p, int b) {
    SeqInfo s;
    const int lo = p.row_off[b], hi = p.row_off[b + 1], len = p.seq_len[b];
    const long long cap = (long long)p.max_pages * p.page_len;
    s.bad = lo < 0 || hi < lo || hi > p.n_rows || len < 0 || len > cap;
    s.lo = lo;
    s.n = s.bad ? 0 : hi - lo;
    s.len = s.bad ? 0 : len;
    s.nt = s.n ? cdiv(s.len, KU) : 0;
    s.qt = cdiv(s.n * p.G, MT);
    return s;
}

// Which of `workers` holds unit u of a line of W: the i with W i / workers <= u < W (i + 1) / workers.
__device__ __forceinline__ int unit_owner(long long u, long long W, int workers) {
    return (int)(((u + 1) * workers - 1) / W);
}
__device__ __forceinline__ int line_workers(long long W, int most) {
    return (int)max(1ll, min((long long)most, W / MIN_UNITS));
}

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
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
        :: "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar)) : "memory");
}

// The prefix on tcgen05 (k_prefix_tc.cu): segments of TC_ROWS rows, units of TC_KEYS keys.
// head_dim 64 or 128.
template <typename T, int HD>
cudaError_t launch_prefix_tc(const AttnP& p, const CUtensorMap& km, const CUtensorMap& vm, int grid, cudaStream_t s);

}  // namespace z2b
