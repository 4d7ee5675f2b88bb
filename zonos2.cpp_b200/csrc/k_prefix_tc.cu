// k_prefix_tc.cu — the shared prefix of prefix_attention on the fifth-generation tensor
// cores (sm_100a): the rows of all streams against the prefix, one tall product.
//
// A segment is 256 rows (query heads of one key head, over the streams) of one key head, a
// unit 128 keys. One CTA per SM walks its range of the line (prefix_attn.cuh):
//   warp 8   TMA: K and V tiles of 128 keys through a ring, boxes by page, 128-byte swizzle;
//   warp 9   one thread issues S_t = Q_t K^T (both operands in shared memory) and O_t += P_t V
//            (P_t from TMEM, V as it lies in the cache: N-major);
//   warps 0-3 and 4-7: softmax of row tile t = 0, 1. A thread holds one row: no shuffles. It
//            reads S_t from TMEM, takes the running maximum, and writes P_t, rounded to the
//            cache's type, over S_t. The first half of P_t is handed over while the second is
//            taken.
// TMEM (512 columns): S_0, S_1 of 128 each, O_0, O_1 of head_dim each. While one tile's
// probabilities are taken the tensor core works on the other's products.
//
// O is rescaled (through registers) only when a row's maximum has run ahead of the one in use
// (LAG). l sums the unrounded probabilities.
//
// Bound: per unit the products of both tiles take 2048 cycles at head_dim 128, and the
// 2 x 128^2 exponentials the same at 16 per cycle and SM; under the load the SMs run at about
// 1.5 GHz. 1024 rows of each of 8 key heads over 32768 keys (137 GFLOP) take 125 us on
// all SMs, 1.1 PFLOP/s, 67% of measured cuBLAS bf16. Tried on that case and slower: two blocks of 64 scores
// a tile in place of one of 128, so that scores never wait for the product that frees them
// (+14 us: 64 keys are fed at 3/4 rate, 6 KB of operands per 32 cycles from shared memory);
// reading the scores twice to spare registers (+10 us); a quarter of the exponentials by a
// polynomial on the multiply-add pipe (+8 us); issuing whichever tile's product is ready
// instead of in turn (+20 us: the polling warp takes issue slots).
#include "launch.cuh"
#include "prefix_attn.cuh"

namespace z2b {
namespace {

// Three warpgroups: two of softmax, one of TMA (warp 8) and MMA (warp 9). Launched at 168
// registers a thread (384 x 168 = 64512); the third keeps 80 and the softmax rows, which hold 128
// scores each, get 208: 256 x 208 + 128 x 80 = 63488. At head_dim 128 that still leaves 52 bytes a thread
// in local memory (112 read back), 8 at 64.
constexpr int TC_THREADS = 384;

__device__ __forceinline__ uint32_t idesc_t(bool bf16, int n, bool b_mn) {
    return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(128 >> 4) << 24);
}

// Shared-memory descriptor of V as B operand, N-major with the 128-byte swizzle: rows are
// keys, 64 dims (128 bytes) each; 8-key groups 1024 B apart, the second 64 dims 16 KB apart.
__device__ __forceinline__ uint64_t desc_v(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(16384 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) |
           (2ull << 61);
}

__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
        :: "r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}

#define R4(x, i) "=r"(x[i]), "=r"(x[i + 1]), "=r"(x[i + 2]), "=r"(x[i + 3])
#define V4(x, i) "r"(x[i]), "r"(x[i + 1]), "r"(x[i + 2]), "r"(x[i + 3])
// 32 f32 columns of this thread's lane, without waiting.
__device__ __forceinline__ void tmem_ld32(uint32_t a, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : R4(r, 0), R4(r, 4), R4(r, 8), R4(r, 12), R4(r, 16), R4(r, 20), R4(r, 24), R4(r, 28) : "r"(a));
}
__device__ __forceinline__ void tmem_st32(uint32_t a, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
        :: V4(r, 0), V4(r, 4), V4(r, 8), V4(r, 12), V4(r, 16), V4(r, 20), V4(r, 24), V4(r, 28), "r"(a) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t a, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
        :: V4(r, 0), V4(r, 4), V4(r, 8), V4(r, 12), "r"(a) : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Pairs of f32 for the two-wide multiply-adds.
__device__ __forceinline__ uint64_t f2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void un2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// Row tiles (of 128) of segment row tile j that hold live rows.
__device__ __forceinline__ int live_tiles(int j, int live_rows) {
    return max(0, min(2, cdiv(live_rows - j * TC_ROWS, 128)));
}

// K or V tiles in the ring: what 227 KB hold beside the two Q tiles, a power of two.
__host__ __device__ constexpr int ring_stages(int hd) { return hd == 128 ? 4 : 8; }

template <typename T, int HD>
__global__ void __launch_bounds__(TC_THREADS, 1) prefix_tc_kernel(const __grid_constant__ AttnP p,
                                                                 const __grid_constant__ CUtensorMap kmap,
                                                                 const __grid_constant__ CUtensorMap vmap) {
    constexpr int HALVES = HD / 64, TILE = HALVES * 16384;       // 128 rows x HD of 16 bits
    constexpr int stages = ring_stages(HD);
    constexpr uint32_t TMEM_COLS = 512, S_COL = 0, O_COL = 256;
    constexpr bool BF = sizeof(T) == 2 && !std::is_same<T, __half>::value;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* ring = smem + 2 * TILE;
    __shared__ __align__(8) uint64_t kv_full[stages], kv_empty[stages], q_full[2], s_full[2], p_full[2][2], pv_done[2], fin;
    __shared__ uint32_t tmem_base;
    __shared__ volatile int s_abort;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     :: "r"(smem_u32(&tmem_base)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < stages; ++i) { mbar_init(&kv_full[i], 1); mbar_init(&kv_empty[i], 1); }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&q_full[t], 4);
            mbar_init(&s_full[t], 1);
            mbar_init(&p_full[t][0], 4);
            mbar_init(&p_full[t][1], 4);
            mbar_init(&pv_done[t], 1);
        }
        mbar_init(&fin, 1);
        s_abort = 0;
        fence_mbar_init();
        prefetch_map(&kmap);
        prefetch_map(&vmap);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tm = tmem_base;
    pdl_wait();
    pdl_release();

    const int live_rows = max(0, min(p.n_rows, p.row_off[p.n_seq])) * p.G;
    const int nt = cdiv(p.prefix_len, TC_KEYS), size = nt + TC_SEG_COST;   // line positions of a segment
    const int W = p.pf_row_tiles * p.nkv * size;
    const Cut cut(W, gridDim.x);
    int u0 = 0, u1 = 0;
    if ((int)blockIdx.x < cut.workers) {
        u0 = cut.begin(blockIdx.x);
        u1 = cut.begin(blockIdx.x + 1);
    }

    if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == 8) {
        // ---- TMA producer: lane i looks up run i's page, one lane issues the boxes
        const int nb = TC_KEYS / p.box_rows;                     // at most 16
        int it = 0;
        bool ok = true;
        for (int u = u0; u < u1 && ok;) {
            const int seg = u / size, end = min(u1, (seg + 1) * size), unit0 = seg * size + TC_SEG_COST, h = seg % p.nkv;
            if (live_tiles(seg / p.nkv, live_rows) == 0) { u = end; continue; }
            for (u = max(u, unit0); u < end && ok; ++u) {
                const int key = (u - unit0) * TC_KEYS + lane * p.box_rows, row = key % p.page_len;
                int page = p.n_pages;                            // out of the view: zeros
                if (lane < nb && key < p.prefix_len) {
                    page = p.prefix_pages[key / p.page_len];
                    if (page < 0 || page >= p.n_pages) {
                        page = p.n_pages;
                        if (p.err) atomicOr(p.err, Z2B_OPS_BAD_PAGE);
                    }
                }
#pragma unroll 1
                for (int isv = 0; isv < 2 && ok; ++isv) {
                    const int st = it % stages, use = it / stages;
                    ok = __all_sync(0xffffffffu, use == 0 || wait_ab(&kv_empty[st], (use - 1) & 1, p.err, &s_abort, p.polls));
                    if (!ok) break;
                    if (lane == 0) mbar_expect_tx(&kv_full[st], TILE);
                    __syncwarp();
                    for (int i = 0; i < nb; ++i) {
                        const int pg = __shfl_sync(0xffffffffu, page, i), pr = __shfl_sync(0xffffffffu, row, i);
                        if (elect_one())
                            for (int half = 0; half < HALVES; half += p.box_halves)
                                tma_load_page(smem_u32(ring) + st * TILE + half * 16384 + i * p.box_rows * 128, isv ? &vmap : &kmap, pr,
                                              half, h, pg, &kv_full[st]);
                    }
                    __syncwarp();
                    ++it;
                }
            }
        }
        // copies in flight land in this CTA's memory, also where another warp's wait has run out and
        // nobody reads them any more: the CTA outlives them
        if (lane == 0)
            for (int k = max(0, it - stages); k < it; ++k) mbar_wait(&kv_full[k % stages], (k / stages) & 1, nullptr, 1u << 16);
        __syncwarp();
    } else if (warp == 9) {
        // ---- MMA issuer: the warp walks together, one thread issues
        const uint32_t id_s = idesc_t(BF, TC_KEYS, false), id_o = idesc_t(BF, HD, true);
        const uint64_t qd = umma_desc_sw128(smem_u32(smem)), kd = umma_desc_sw128(smem_u32(ring)), vd = desc_v(smem_u32(ring));
        int c = 0;                                               // units done
        int segs[2] = {0, 0}, ct[2] = {0, 0};                    // segments and units done of each row tile
        bool ok = true;
        auto wait = [&](uint64_t* bar, int phase) {
            if (ok) ok = __all_sync(0xffffffffu, wait_ab(bar, phase & 1, p.err, &s_abort, p.polls));
            return ok;
        };
        auto scores = [&](int t, int idx, bool last) {           // S_t = Q_t K^T; `last`: K's stage is free after it
            const uint64_t da = qd + (uint64_t)(t * (TILE >> 4)), db = kd + (uint64_t)((idx % stages) * (TILE >> 4));
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < HD / 16; ++k)                // 32 bytes a step, 16 KB a half
                    umma_f16(tm + S_COL + t * 128, da + ((k >> 2) * 1024 + (k & 3) * 2), db + ((k >> 2) * 1024 + (k & 3) * 2), id_s, k > 0);
                umma_commit(&s_full[t]);
                if (last) umma_commit(&kv_empty[idx % stages]);
            }
            __syncwarp();
        };
        for (int u = u0; u < u1 && ok;) {
            const int seg = u / size, end = min(u1, (seg + 1) * size), n = end - max(u, seg * size + TC_SEG_COST);
            const int nl = live_tiles(seg / p.nkv, live_rows);
            u = end;
            if (nl == 0 || n <= 0) continue;
            wait(&kv_full[2 * c % stages], 2 * c / stages);
            for (int t = 0; t < nl; ++t) {
                wait(&q_full[t], segs[t]++);
                if (!ok) break;
                tc_fence_after();
                scores(t, 2 * c, t == nl - 1);
            }
            for (int j = 0; j < n && ok; ++j, ++c) {
                const int vi = 2 * c + 1, ki = 2 * c + 2;
                for (int t = 0; t < nl && ok; ++t) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        wait(&p_full[t][half], ct[t]);
                        if (half == 0 && t == 0) wait(&kv_full[vi % stages], vi / stages);
                        if (!ok) break;
                        tc_fence_after();
                        const uint64_t db = vd + (uint64_t)((vi % stages) * (TILE >> 4) + half * 512);
                        if (elect_one()) {
#pragma unroll
                            for (int k = 0; k < 4; ++k)          // O_t += P_t V, 2 KB a step of 16 keys
                                umma_ts(tm + O_COL + t * HD, tm + S_COL + t * 128 + half * 32 + k * 8, db + k * 128, id_o, j > 0 || half > 0 || k > 0);
                            if (half == 1) {
                                umma_commit(&pv_done[t]);
                                if (t == nl - 1) umma_commit(&kv_empty[vi % stages]);
                            }
                        }
                        __syncwarp();
                    }
                    if (j + 1 < n) {
                        // the next scores overwrite P_t: they wait for the product that reads it
                        if (t == 0) wait(&kv_full[ki % stages], ki / stages);
                        wait(&pv_done[t], ct[t]);
                        if (!ok) break;
                        tc_fence_after();
                        scores(t, ki, t == nl - 1);
                    }
                    ++ct[t];
                }
            }
        }
        // every product issued completes before the block gives its memory back
        if (elect_one()) umma_commit(&fin);
        __syncwarp();
        (void)mbar_wait(&fin, 0, nullptr, 1u << 16);
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        // ---- softmax: thread = row
        const int t = warp >> 2, row = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;       // 32 (warp % 4) lanes, in the address's upper half
        const uint32_t ts = tm + lanes + S_COL + t * 128, to = tm + lanes + O_COL + t * HD;
        uint8_t* qt = smem + t * TILE;
        const bool flip = p.scale2 < 0.0f;                       // the maximum of s * scale is taken on s: negate Q instead
        const bool flat = p.scale2 == 0.0f;                      // all scores equal: zero Q, so that masked keys stay apart
        const float sc = flat ? 1.0f : fabsf(p.scale2);
        const bool q16 = ((reinterpret_cast<uintptr_t>(p.q) | (uintptr_t)(p.q_row * 2) | (uintptr_t)(p.q_head * 2)) & 15) == 0;
        int c = 0, ct = 0;
        bool ok = true;
        for (int u = u0; u < u1;) {
            const int seg = u / size, end = min(u1, (seg + 1) * size), unit0 = seg * size + TC_SEG_COST;
            const int n = end - max(u, unit0), key_first = (max(u, unit0) - unit0) * TC_KEYS;
            const int j = seg / p.nkv, h = seg % p.nkv, nl = live_tiles(j, live_rows);
            u = end;
            if (n <= 0) continue;
            if (t >= nl) { c += nl ? n : 0; continue; }
            // Q_t: this thread's row, swizzled by 16-byte chunks
            const int r = j * TC_ROWS + t * 128 + row;
            const bool live = r < live_rows;
            const size_t at = (size_t)(seg + (int)blockIdx.x) * TC_ROWS + t * 128 + row;         // of this row's partial result
            auto missing = [&] { if (live) p.part_ml[at] = make_float2(NAN, NAN); };            // a wait ran out
            if (!ok) { missing(); continue; }
            {
                const T* src = (const T*)p.q + (long long)(r / p.G) * p.q_row + (long long)(h * p.G + r % p.G) * p.q_head;
#pragma unroll
                for (int k = 0; k < HD / 8; ++k) {
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (live && !flat && q16) v = *(const uint4*)(src + k * 8);
                    else if (live && !flat) {
                        const uint32_t* w = (const uint32_t*)(src + k * 8);
                        v = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                    if (flip) { v.x ^= 0x80008000u; v.y ^= 0x80008000u; v.z ^= 0x80008000u; v.w ^= 0x80008000u; }
                    *(uint4*)(qt + (k >> 3) * 16384 + row * 128 + (((k & 7) ^ (row & 7)) << 4)) = v;
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[t]);
            float m = -INFINITY, l = 0.0f;
            for (int i = 0; i < n; ++i, ++c) {
                ok = __all_sync(0xffffffffu, wait_ab(&s_full[t], ct & 1, p.err, &s_abort, p.polls));
                if (!ok) break;
                ++ct;
                tc_fence_after();
                const int keys = p.prefix_len - key_first - i * TC_KEYS;
                if (keys < TC_KEYS) {
                    // V rows behind the last key may hold anything: zero times that is not zero. Each tile
                    // clears them before its go-ahead, whichever comes first.
                    const int vi = 2 * c + 1;
                    ok = __all_sync(0xffffffffu, wait_ab(&kv_full[vi % stages], (vi / stages) & 1, p.err, &s_abort, p.polls));
                    if (!ok) break;
                    if (row >= keys)
#pragma unroll
                        for (int k = 0; k < HD / 8; ++k)
                            *(uint4*)(ring + (vi % stages) * TILE + (k >> 3) * 16384 + row * 128 + ((k & 7) << 4)) = make_uint4(0, 0, 0, 0);
                    fence_proxy_async();
                }
                uint32_t s[TC_KEYS];
#pragma unroll
                for (int k = 0; k < TC_KEYS; k += 32) tmem_ld32(ts + k, s + k);
                tmem_wait_ld();
                if (keys < TC_KEYS) {
#pragma unroll
                    for (int k = 0; k < TC_KEYS; ++k)
                        if (k >= keys) s[k] = 0xff800000u;       // -inf
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < TC_KEYS; e += 2)
                    mx[(e >> 1) & 3] = max3(mx[(e >> 1) & 3], __uint_as_float(s[e]), __uint_as_float(s[e + 1]));
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sc;
                const bool raise = top > m + LAG;
                if (__any_sync(0xffffffffu, raise)) {
                    const float f = raise ? ex2(m - (top - P_SHIFT)) : 1.0f;
                    if (raise) m = top - P_SHIFT;
                    l *= f;
                    if (i > 0) {                                 // these scores were issued after the last O was done
#pragma unroll
                        for (int k = 0; k < HD; k += 32) {
                            uint32_t o[32];
                            tmem_ld32(to + k, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            tmem_st32(to + k, o);
                        }
                    }
                }
                uint64_t sum[2] = {0, 0};
                const uint64_t sc2 = f2(sc, sc), m2 = f2(-m, -m);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint32_t pk[16];
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        float x, y;
                        un2(fma2(f2(__uint_as_float(s[k * 32 + e]), __uint_as_float(s[k * 32 + e + 1])), sc2, m2), x, y);
                        x = ex2(x);
                        y = ex2(y);
                        sum[(e >> 1) & 1] = add2(sum[(e >> 1) & 1], f2(x, y));
                        pk[e / 2] = pack2<T>(x, y);
                    }
                    tmem_st16(ts + k * 16, pk);
                    if (k & 1) {
                        tmem_wait_st();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&p_full[t][k >> 1]);
                    }
                }
                float x, y;
                un2(add2(sum[0], sum[1]), x, y);
                l += x + y;
            }
            if (ok) ok = __all_sync(0xffffffffu, wait_ab(&pv_done[t], (ct - 1) & 1, p.err, &s_abort, p.polls));
            if (!ok) { missing(); continue; }
            tc_fence_after();
            float* po = p.part_o + at * HD;
#pragma unroll
            for (int k = 0; k < HD; k += 32) {
                uint32_t o[32];
                tmem_ld32(to + k, o);
                tmem_wait_ld();
                if (live)
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        *(uint4*)(po + k + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            }
            if (live) p.part_ml[at] = make_float2(m, l);
            tc_fence_before();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tm), "r"(TMEM_COLS) : "memory");
    }
}

}  // namespace

template <typename T, int HD>
cudaError_t launch_prefix_tc(const AttnP& p, const CUtensorMap& km, const CUtensorMap& vm, int grid, cudaStream_t s) {
    constexpr int TILE = HD / 64 * 16384;
    constexpr int smem = 1024 + (2 + ring_stages(HD)) * TILE;
    static std::atomic<uint64_t> opted{0};                       // devices whose shared-memory opt-in is done
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(opted.load(std::memory_order_relaxed) >> dev & 1)) {
        e = cudaFuncSetAttribute(prefix_tc_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        if (dev < 64) opted.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    return launch_pdl(prefix_tc_kernel<T, HD>, dim3(grid), dim3(TC_THREADS), smem, s, p, km, vm);
}

template cudaError_t launch_prefix_tc<__half, 64>(const AttnP&, const CUtensorMap&, const CUtensorMap&, int, cudaStream_t);
template cudaError_t launch_prefix_tc<__half, 128>(const AttnP&, const CUtensorMap&, const CUtensorMap&, int, cudaStream_t);
template cudaError_t launch_prefix_tc<__nv_bfloat16, 64>(const AttnP&, const CUtensorMap&, const CUtensorMap&, int, cudaStream_t);
template cudaError_t launch_prefix_tc<__nv_bfloat16, 128>(const AttnP&, const CUtensorMap&, const CUtensorMap&, int, cudaStream_t);

}  // namespace z2b
