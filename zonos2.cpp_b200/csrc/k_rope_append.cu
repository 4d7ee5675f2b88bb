// k_rope_append.cu — rotate the new rows' queries and keys and append keys and values to a
// paged cache, in one launch (sm_100a; include/z2b_ops.h).
//
// Pair (a, b) of a head at position s turns by s * w_i:  a' = m (a cos - b sin),
// b' = m (b cos + a sin). The table holds w_i as a 64-bit fraction of a turn, so s * step
// wraps modulo one turn and the product is exact: no position is too far for f32 angles
// (an f32 product s * w is off by 0.06 rad at one million).
//
// Bound: bytes (every element is read and written once) for prompts, launch and load
// latency for decode rows. A warp takes one row: its lanes hold VEC pairs each, several heads
// side by side, and walk the heads with the same pairs, so a lane computes its sines once
// (they cost about as many instructions as rotating a head). The loads of BATCH heads are in
// flight together: 16384 rows of 32 + 2 x 8 heads of 128 dims, bf16, 403 MB, take 67 us (6.0
// TB/s, 92% of the measured copy), against 83 us with two; a warp that takes four rows in
// turn, their places looked up side by side, 76 us. Few rows spread a row's heads over several
// warps (blockIdx.y) until the device is full.
#include "launch.cuh"
#include "ops.cuh"
#include "ops.h"

namespace z2b {
namespace {

struct RopeP {
    z2b_rope rope;
    const void *q, *k, *v;
    void *q_out, *kc, *vc;
    long long q_row, q_head, o_row, o_head, k_row, k_head, v_row, v_head;
    long long page_stride, row_stride, head_stride, table_stride;
    const int *row_off, *seq_len, *table, *pos;
    uint32_t* err;
    int n_rows, n_seq, nh, nkv, hd, page_len, n_pages, max_pages, prefix_len;
};

// VEC consecutive elements, by 16-byte accesses when VEC is 8.
template <typename T, int VEC> struct Run {
    T e[VEC];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (VEC == 8) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(e)[i] = reinterpret_cast<const uint4*>(p)[i];
        } else e[0] = p[0];
    }
};

template <typename T, int VEC> __device__ __forceinline__ void store_vec(T* p, const float (&x)[VEC]) {
    if constexpr (VEC == 8 && sizeof(T) == 4) {
        *(float4*)p = make_float4(x[0], x[1], x[2], x[3]);
        *(float4*)(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
    } else if constexpr (VEC == 8) {
        uint4 u;
        T* e = reinterpret_cast<T*>(&u);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(x[i]);
        *(uint4*)p = u;
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) p[i] = from_f32<T>(x[i]);
    }
}

constexpr int WARPS = 4;                // of a block

// TI: type of q, k, v; TC: of the cache. A unit is VEC pairs of one head: two runs of VEC
// elements (at a0 and b0) in every layout. VEC 1 takes any alignment and dims.
template <typename TI, typename TC, int VEC>
__global__ void __launch_bounds__(32 * WARPS) rope_append_ops_kernel(const __grid_constant__ RopeP p) {
    constexpr int BATCH = VEC == 1 ? 1 : sizeof(TI) == 4 ? 3 : 6;    // heads whose loads are in flight together
    const int lane = threadIdx.x & 31, t = blockIdx.x * WARPS + (threadIdx.x >> 5);
    pdl_wait();
    pdl_release();
    if (t >= p.n_rows) return;
    const int total = p.row_off[p.n_seq];
    const int b = warp_find_seq(p.row_off, p.n_seq, t);
    const int lo = p.row_off[b], hi = p.row_off[b + 1], len = p.seq_len[b];
    if (p.err && t == 0 && blockIdx.y == 0) {                        // offsets that no row need come across
        bool bad = lane == 0 && (p.row_off[0] < 0 || total > p.n_rows);
        for (int i = lane; i < p.n_seq; i += 32) bad |= p.row_off[i + 1] < p.row_off[i];
        if (bad) atomicOr(p.err, Z2B_OPS_BAD_INDEX);
    }
    // a stream whose offsets cannot be is left out whole; offsets that descend may still name a row
    // for a stream whose own are sound
    const bool broken = lo < 0 || hi < lo || hi > total || hi > p.n_rows || (t < lo && b > 0);
    const long long r = (long long)len - hi + t;                     // cache row
    if (broken || t < lo || t >= hi || r < 0 || (p.k && r >= (long long)p.max_pages * p.page_len)) {
        // rows ahead of the first stream and padding stay as they are
        if ((broken || (t >= lo && t < total)) && lane == 0 && p.err) atomicOr(p.err, Z2B_OPS_BAD_INDEX);
        return;
    }
    const long long at = p.pos ? (long long)p.pos[t] : (long long)p.prefix_len + r;
    long long crow = 0;
    bool store = p.k != nullptr;
    if (store) {
        const int pi = (int)(r / p.page_len), page = p.table[(long long)b * p.table_stride + pi];
        store = page >= 0 && page < p.n_pages;
        if (!store && lane == 0 && p.err) atomicOr(p.err, Z2B_OPS_BAD_PAGE);
        crow = (long long)page * p.page_stride + (r - (long long)pi * p.page_len) * p.row_stride;
    }

    const int rot = p.rope.rot_dim, half = rot >> 1;
    const int ur = half / VEC;                                       // rotated units of a head
    const int units = ur + (p.hd - rot + 2 * VEC - 1) / (2 * VEC);
    const int side = max(1, 32 / units);                             // heads side by side in a warp
    const int step = gridDim.y * side;
    const TI *q = (const TI*)p.q, *k = (const TI*)p.k, *v = (const TI*)p.v;
    const int heads = p.nh + (store ? 2 * p.nkv : 0);
    for (int u0 = 0; u0 < units; u0 += 32) {
        const int u = units > 32 ? u0 + lane : lane % units;
        const int h0 = units > 32 ? 0 : lane / units;
        const bool idle = u >= units || h0 >= side;
        const bool turns = u < ur;
        int a0, b0;
        float cs[VEC], sn[VEC];
        if (turns) {
            if (p.rope.layout == Z2B_ROPE_HALF) { a0 = u * VEC; b0 = half + u * VEC; }
            else { a0 = 2 * u * VEC; b0 = a0 + VEC; }
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                // signed top half of the wrapped phase: half-turns in [-1, 1)
                const int top = (int)(((unsigned long long)at * p.rope.step[u * VEC + e]) >> 32);
                float s, c;
                sincospif((float)top * 4.6566128730773926e-10f, &s, &c);     // 2^-31
                cs[e] = c * p.rope.mag;
                sn[e] = s * p.rope.mag;
            }
        } else {
            a0 = rot + 2 * (u - ur) * VEC;
            b0 = a0 + VEC;
        }
        const bool has_b = VEC > 1 || turns || b0 < p.hd;
        for (int hb = idle ? heads : h0 + blockIdx.y * side; hb < heads; hb += BATCH * step) {
            Run<TI, VEC> rx[BATCH], ry[BATCH];
#pragma unroll
            for (int j = 0; j < BATCH; ++j) {
                const int h = hb + j * step;
                if (h >= heads) break;
                const TI* src = h < p.nh ? q + (long long)t * p.q_row + h * p.q_head
                              : h < p.nh + p.nkv ? k + (long long)t * p.k_row + (h - p.nh) * p.k_head
                                                 : v + (long long)t * p.v_row + (h - p.nh - p.nkv) * p.v_head;
                rx[j].load(src + a0);
                if (has_b) ry[j].load(src + b0);
            }
#pragma unroll
            for (int j = 0; j < BATCH; ++j) {
                const int h = hb + j * step;
                if (h >= heads) break;
                float x[VEC], y[VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    x[e] = to_f32(rx[j].e[e]);
                    y[e] = has_b ? to_f32(ry[j].e[e]) : 0.0f;
                }
                if (turns && h < p.nh + p.nkv) {
                    if (p.rope.layout == Z2B_ROPE_HALF || VEC == 1) {
#pragma unroll
                        for (int e = 0; e < VEC; ++e) {
                            const float f = x[e], g = y[e];
                            x[e] = f * cs[e] - g * sn[e];
                            y[e] = g * cs[e] + f * sn[e];
                        }
                    } else if constexpr (VEC > 1) {
                        // the 2 VEC elements are consecutive: pair e is (2e, 2e + 1)
#pragma unroll
                        for (int e = 0; e < VEC / 2; ++e) {
                            const float f = x[2 * e], g = x[2 * e + 1], f2 = y[2 * e], g2 = y[2 * e + 1];
                            x[2 * e] = f * cs[e] - g * sn[e];
                            x[2 * e + 1] = g * cs[e] + f * sn[e];
                            y[2 * e] = f2 * cs[e + VEC / 2] - g2 * sn[e + VEC / 2];
                            y[2 * e + 1] = g2 * cs[e + VEC / 2] + f2 * sn[e + VEC / 2];
                        }
                    }
                }
                if (h < p.nh) {
                    TI* dst = (TI*)p.q_out + (long long)t * p.o_row + h * p.o_head;
                    store_vec<TI, VEC>(dst + a0, x);
                    if (has_b) store_vec<TI, VEC>(dst + b0, y);
                } else {
                    const bool isk = h < p.nh + p.nkv;
                    TC* dst = (TC*)(isk ? p.kc : p.vc) + crow + (h - p.nh - (isk ? 0 : p.nkv)) * p.head_stride;
                    store_vec<TC, VEC>(dst + a0, x);
                    if (has_b) store_vec<TC, VEC>(dst + b0, y);
                }
            }
        }
    }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename TI, typename TC> cudaError_t go(const RopeP& p, bool vec, dim3 grid, cudaStream_t s) {
    return vec ? launch_pdl(rope_append_ops_kernel<TI, TC, 8>, grid, dim3(32 * WARPS), 0, s, p)
               : launch_pdl(rope_append_ops_kernel<TI, TC, 1>, grid, dim3(32 * WARPS), 0, s, p);
}

}  // namespace

cudaError_t launch_rope_append(const z2b_rope_append_args& a, cudaStream_t s) {
    RopeP p{};
    const z2b_paged_kv& c = *a.kv;
    if (a.rope) p.rope = *a.rope;
    p.q = a.q; p.k = a.k; p.v = a.v; p.q_out = a.q_out; p.kc = c.k; p.vc = c.v;
    p.q_row = a.q_row; p.q_head = a.q_head; p.o_row = a.o_row; p.o_head = a.o_head;
    p.k_row = a.k_row; p.k_head = a.k_head; p.v_row = a.v_row; p.v_head = a.v_head;
    p.page_stride = c.page_stride; p.row_stride = c.row_stride; p.head_stride = c.head_stride;
    p.table_stride = a.table_stride;
    p.row_off = a.row_off; p.seq_len = a.seq_len; p.table = a.page_table; p.pos = a.pos; p.err = a.err;
    p.n_rows = a.n_rows; p.n_seq = a.n_seq; p.nh = a.n_head; p.nkv = c.n_head_kv; p.hd = c.head_dim;
    p.page_len = c.page_len; p.n_pages = c.n_pages; p.max_pages = a.max_pages; p.prefix_len = a.prefix_len;

    // 16-byte accesses when every run of 8 elements is aligned for both types
    const long long eight = p.q_row | p.q_head | p.o_row | p.o_head | p.k_row | p.k_head | p.v_row | p.v_head |
                            p.page_stride | p.row_stride | p.head_stride;
    const bool vec = p.rope.rot_dim % 16 == 0 && (p.hd - p.rope.rot_dim) % 16 == 0 && eight % 8 == 0 &&
                     aligned16(p.q) && aligned16(p.k) && aligned16(p.v) && aligned16(p.q_out) && aligned16(p.kc) &&
                     aligned16(p.vc);
    const int VEC = vec ? 8 : 1;
    const int units = (p.rope.rot_dim / 2) / VEC + (p.hd - p.rope.rot_dim + 2 * VEC - 1) / (2 * VEC);
    const int side = units >= 32 ? 1 : 32 / units;
    const int heads = p.nh + (p.k ? 2 * p.nkv : 0);
    const int iters = (heads + side - 1) / side;
    // a row's heads over `split` warps while that finds idle schedulers (four warps an SM). Rows of
    // 32 + 2 x 8 heads of 128 dims, one warp each / split, in us: 1: 5.6 / 3.1, 64: 6.1 / 3.9, 256: 6.2 /
    // 4.6; up to eight warps an SM instead, 1024 rows: 7.4 / 8.4
    int split = 1;
    while (split < iters && (long long)p.n_rows * split < 148 * 4) ++split;
    const dim3 grid((p.n_rows + WARPS - 1) / WARPS, split);
    if (a.type == Z2B_TYPE_F32)
        return c.type == Z2B_TYPE_F16 ? go<float, __half>(p, vec, grid, s) : go<float, __nv_bfloat16>(p, vec, grid, s);
    if (a.type == Z2B_TYPE_F16)
        return c.type == Z2B_TYPE_F16 ? go<__half, __half>(p, vec, grid, s) : go<__half, __nv_bfloat16>(p, vec, grid, s);
    return c.type == Z2B_TYPE_F16 ? go<__nv_bfloat16, __half>(p, vec, grid, s)
                                  : go<__nv_bfloat16, __nv_bfloat16>(p, vec, grid, s);
}

}  // namespace z2b
