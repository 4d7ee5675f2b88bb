// k_prefix_attn.cu — attention of many streams over one shared prefix and each stream's own
// paged rows (sm_100a; include/z2b_ops.h).
//
// out = softmax(scale q K^T) V over the union of two key sets, each handled where it is
// cheapest and joined by their softmax statistics:
//   out = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i ,  M = max m_i
// over partial results i with O_i = sum_k p_k v_k, l_i = sum_k p_k, p_k = 2^(s_k - m_i).
//   prefix: the rows of ALL streams form one tall query matrix per key head, so the prefix is
//           read once per row tile instead of once per stream;
//   own:    each stream's rows (its query heads of one key head side by side) over its pages.
// Bound: the own part by HBM bytes, the prefix by tensor-core rate once the rows are many.
//
// Work split: a unit is 64 keys of one segment (row tile x key head). All units form one line
// that is cut into equal contiguous ranges, one per CTA, whatever the lengths; a CTA streams
// K and V tiles through a TMA ring across segment borders and leaves one partial result per
// segment it touches. Partial slots are segment + CTA: going along the line every new partial
// advances one of the two, so slots never collide and their number is bounded by
// segments + CTAs. Nothing is accumulated by atomics: the same call gives the same bits.
#include "launch.cuh"
#include "ops.h"
#include "prefix_attn.cuh"

#include <atomic>

namespace z2b {
namespace {

constexpr int COMPUTE_WARPS = 4;
constexpr int THREADS = 32 * (COMPUTE_WARPS + 1);
constexpr int MAX_SMEM = 200 * 1024;   // dynamic shared memory a launch may ask for

// Shared-memory tile of 64 rows of one key head: rows of RB bytes (at most 128: head_dim 128
// is two halves), 16-byte chunks XOR-swizzled as the TMA box writes them.
template <int HD> struct Tile {
    static constexpr int INNER = HD < 64 ? HD : 64;              // elements of one box row
    static constexpr int HALVES = HD / INNER;
    static constexpr int RB = INNER * 2;
    static constexpr int BYTES = KT * HD * 2;
    __device__ static __forceinline__ uint32_t chunk(int row, int c) {   // byte offset of 8 elements
        constexpr int PER = RB / 16;
        const int half = c / PER, cc = c % PER;
        const int x = PER == 8 ? (row & 7) : PER == 4 ? ((row >> 1) & 3) : ((row >> 2) & 1);
        return half * (KT * RB) + row * RB + ((cc ^ x) << 4);
    }
};

// One segment of the line, as the producer and the compute warps both walk it.
struct Seg {
    int h, j, seg, unit0, nt;          // key head, row tile, segment id, first unit, units
    int b, lo, n, klen, lim_max;       // stream (-1: the prefix), first row, rows, keys, keys its last row sees
};

template <int MT>
__device__ __forceinline__ Seg find_seg(const AttnP& p, const int* s_unit, const int* s_seg, int pf_nt, int pf_units,
                                        int total_rows, int u) {
    Seg g;
    if (u < pf_units) {
        g.seg = u / pf_nt;
        g.unit0 = g.seg * pf_nt;
        g.nt = pf_nt;
        g.j = g.seg / p.nkv;
        g.h = g.seg % p.nkv;
        g.b = -1;
        g.lo = 0;
        g.n = total_rows;
        g.klen = g.lim_max = p.prefix_len;
        return g;
    }
    const int v = u - pf_units;
    int lo = 0, hi = p.n_seq - 1;                                // last b with s_unit[b] <= v
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s_unit[mid] <= v) lo = mid; else hi = mid - 1;
    }
    const SeqInfo s = seq_info<MT>(p, lo);
    const int js = (v - s_unit[lo]) / s.nt;
    g.seg = p.pf_row_tiles * p.nkv + s_seg[lo] + js;
    g.unit0 = pf_units + s_unit[lo] + js * s.nt;
    g.nt = s.nt;
    g.j = js / p.nkv;
    g.h = js % p.nkv;
    g.b = lo;
    g.lo = s.lo;
    g.n = s.n;
    g.klen = s.len;
    const int last = min(s.n - 1, (g.j * MT + MT - 1) / p.G);
    g.lim_max = min(s.len, s.len - s.n + last + 1);
    return g;
}

// MT = 16 WM rows per segment; the four compute warps are WM row groups x WN shares of the
// unit's keys. Few rows (decode: the query heads of one key head) put all warps on the keys.
template <typename T, int HD, int WM>
__global__ void __launch_bounds__(THREADS) prefix_attn_kernel(const __grid_constant__ AttnP p,
                                                              const __grid_constant__ CUtensorMap kmap,
                                                              const __grid_constant__ CUtensorMap vmap) {
    constexpr int WN = COMPUTE_WARPS / WM, MT = 16 * WM, KW = KT / WN;
    constexpr int KS = HD / 16, NT = KW / 8, DT = HD / 8;
    constexpr int STAGE = 2 * Tile<HD>::BYTES;
    constexpr int RS = HD + 4;                                   // padded row of the cross-warp sum
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    float* s_red = (float*)(smem + (size_t)p.stages * STAGE);    // [WN][MT][RS] when WN > 1
    int* s_unit = (int*)(s_red + (WN > 1 ? WN * MT * RS : 0));
    int* s_seg = s_unit + p.n_seq + 1;
    __shared__ __align__(8) uint64_t s_full[8], s_empty[8];
    __shared__ float2 s_ml[WN][MT];
    __shared__ int s_scan[2][THREADS / 32];
    __shared__ volatile int s_abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < p.stages; ++i) { mbar_init(&s_full[i], 1); mbar_init(&s_empty[i], COMPUTE_WARPS); }
        fence_mbar_init();
        s_abort = 0;
    }
    if (!p.after_prefix) { pdl_wait(); pdl_release(); }

    // ---- the line: offsets of every stream's units and segments, by a block scan
    const int total_rows = max(0, min(p.n_rows, p.row_off[p.n_seq]));
    const int pf_nt = cdiv(p.prefix_len, KT), pf_units = p.pf_row_tiles * p.nkv * pf_nt;
    if (p.own) {
        const int per = cdiv(p.n_seq, THREADS);
        const int b0 = min(p.n_seq, (int)threadIdx.x * per), b1 = min(p.n_seq, b0 + per);
        int su = 0, sg = 0;
        for (int b = b0; b < b1; ++b) {
            const SeqInfo s = seq_info<MT>(p, b);
            if (s.bad && blockIdx.x == 0 && p.err) atomicOr(p.err, Z2B_OPS_BAD_INDEX);
            s_unit[b] = su;
            s_seg[b] = sg;
            su += s.qt * p.nkv * s.nt;
            sg += s.qt * p.nkv;
        }
        int iu = su, ig = sg;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int a = __shfl_up_sync(0xffffffffu, iu, o), c = __shfl_up_sync(0xffffffffu, ig, o);
            if (lane >= o) { iu += a; ig += c; }
        }
        if (lane == 31) { s_scan[0][warp] = iu; s_scan[1][warp] = ig; }
        __syncthreads();
        int eu = iu - su, eg = ig - sg;
        for (int w = 0; w < warp; ++w) { eu += s_scan[0][w]; eg += s_scan[1][w]; }
        for (int b = b0; b < b1; ++b) { s_unit[b] += eu; s_seg[b] += eg; }
        if (threadIdx.x == THREADS - 1) { s_unit[p.n_seq] = eu + su; s_seg[p.n_seq] = eg + sg; }
    }
    __syncthreads();
    if (p.own && blockIdx.x == 0)
        for (int b = threadIdx.x; b <= p.n_seq; b += THREADS) { p.plan[b] = s_unit[b]; p.plan[p.n_seq + 1 + b] = s_seg[b]; }
    const long long W = (long long)pf_units + (p.own ? s_unit[p.n_seq] : 0);
    const int ctas = line_ctas(W, gridDim.x);
    int u0 = 0, u1 = 0;
    if ((int)blockIdx.x < ctas) {
        u0 = (int)(W * blockIdx.x / ctas);
        u1 = (int)(W * (blockIdx.x + 1) / ctas);
    }

    if (warp == COMPUTE_WARPS) {
        // ---- producer warp: one TMA box per lane, pages looked up a unit ahead of the copy
        const int nb = KT / p.box_rows, jobs = 2 * nb * Tile<HD>::HALVES;
        int it = 0;
        for (int u = u0; u < u1 && !s_abort;) {
            const Seg g = find_seg<MT>(p, s_unit, s_seg, pf_nt, pf_units, total_rows, u);
            const int end = min(u1, g.unit0 + g.nt);
            const int* pages = g.b < 0 ? p.prefix_pages : p.table + (long long)g.b * p.table_stride;
            for (; u < end; ++u) {
                const int key0 = (u - g.unit0) * KT;
                if (key0 >= g.lim_max) continue;                 // no row of the tile sees these keys
                const int st = it % p.stages, use = it / p.stages;
                bool ok = true;
                for (int base = 0; base < jobs; base += 32) {
                    const int i = base + lane;
                    const int rb = i % nb, rest = i / nb;        // rest: half, then K or V
                    const int key = key0 + rb * p.box_rows;
                    int page = p.n_pages;                        // out of the view: the box fills with zeros
                    if (i < jobs && key < g.klen) {
                        page = pages[key / p.page_len];
                        if (page < 0 || page >= p.n_pages) {
                            page = p.n_pages;
                            if (p.err) atomicOr(p.err, Z2B_OPS_BAD_PAGE);
                        }
                    }
                    if (base == 0) {
                        if (lane == 0) {
                            ok = use == 0 || wait_ab(&s_empty[st], (use - 1) & 1, p.err, &s_abort);
                            if (ok) mbar_expect_tx(&s_full[st], STAGE);
                        }
                        ok = __shfl_sync(0xffffffffu, ok, 0);
                        if (!ok) break;
                    }
                    if (i < jobs) {
                        const int half = rest % Tile<HD>::HALVES, isv = rest / Tile<HD>::HALVES;
                        const uint32_t dst = smem_u32(smem) + st * STAGE + isv * Tile<HD>::BYTES +
                                             half * (KT * Tile<HD>::RB) + rb * p.box_rows * Tile<HD>::RB;
                        tma_load_4d(dst, isv ? &vmap : &kmap, half * 64, g.h, key % p.page_len, page, &s_full[st]);
                    }
                }
                if (!ok) { u = u1; break; }
                ++it;
            }
        }
        // after a wait that ran out, the copies in flight still land in this CTA's memory
        if (lane == 0 && s_abort)
            for (int k = max(0, it - p.stages); k < it; ++k) mbar_wait(&s_full[k % p.stages], (k / p.stages) & 1, p.err);
    } else {
        // ---- compute warps
        const int wr = warp / WN, wc = warp % WN, r0 = lane >> 2, quad = lane & 3, kb = wc * KW;
        int it = 0;
        bool dead = false;                                       // a wait ran out: walk on, touching no tile,
        for (int u = u0; u < u1;) {                              // so that all four warps meet at the barriers
            const Seg g = find_seg<MT>(p, s_unit, s_seg, pf_nt, pf_units, total_rows, u);
            const int end = min(u1, g.unit0 + g.nt);
            // this lane's two rows
            int lim[2];
            uint32_t qa[KS][4];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int rr = g.j * MT + wr * 16 + r0 + 8 * x, i = rr / p.G;
                const bool live = i < g.n;
                lim[x] = !live ? 0 : g.b < 0 ? g.klen : min(g.klen, g.klen - g.n + i + 1);
                const T* qp = (const T*)p.q + (long long)(g.lo + i) * p.q_row + (long long)(g.h * p.G + rr % p.G) * p.q_head + quad * 2;
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    qa[k][x] = live ? *(const uint32_t*)(qp + k * 16) : 0u;
                    qa[k][x + 2] = live ? *(const uint32_t*)(qp + k * 16 + 8) : 0u;
                }
            }
            const int lim_min = min(lim[0], lim[1]);
            float o[DT][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.0f;

            for (; u < end; ++u) {
                const int key0 = (u - g.unit0) * KT;
                if (key0 >= g.lim_max) continue;
                const int st = it % p.stages, use = it / p.stages;
                ++it;
                if (!dead) dead = !wait_ab(&s_full[st], use & 1, p.err, &s_abort);
                dead = __any_sync(0xffffffffu, dead);
                if (dead) continue;
                uint8_t* kt = smem + (size_t)st * STAGE;
                const uint32_t ks = smem_u32(kt), vs = ks + Tile<HD>::BYTES;
                const bool tail = key0 + KT > g.klen;
                if (tail) {
                    // rows behind the last key may hold anything: zero times that is not zero
                    for (int i = lane; i < KW * (HD / 8); i += 32) {
                        const int row = kb + i / (HD / 8);
                        if (key0 + row >= g.klen)
                            *(uint4*)(kt + Tile<HD>::BYTES + Tile<HD>::chunk(row, i % (HD / 8))) = make_uint4(0, 0, 0, 0);
                    }
                    __syncwarp();
                }
                float s[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
#pragma unroll
                for (int k = 0; k < KS; ++k) {
#pragma unroll
                    for (int n = 0; n < NT; n += 2) {
                        uint32_t r[4];
                        ldsm4(ks + Tile<HD>::chunk(kb + n * 8 + ((lane >> 4) << 3) + (lane & 7), 2 * k + ((lane >> 3) & 1)), r);
                        mma_t<T>(s[n], qa[k], r[0], r[1]);
                        mma_t<T>(s[n + 1], qa[k], r[2], r[3]);
                    }
                }
                const bool cut = key0 + kb + KW > lim_min;
                float mx[2] = {m[0], m[1]};
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[n][e] *= p.scale2;
                        if (cut && key0 + kb + n * 8 + quad * 2 + (e & 1) >= lim[e >> 1]) s[n][e] = -INFINITY;
                        mx[e >> 1] = fmaxf(mx[e >> 1], s[n][e]);
                    }
                float f[2], base[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 1));
                    mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 2));
                    base[x] = mx[x] == -INFINITY ? 0.0f : mx[x];         // a row that has seen no key yet
                    f[x] = ex2(m[x] - base[x]);
                    m[x] = mx[x];
                    l[x] *= f[x];
                }
#pragma unroll
                for (int d = 0; d < DT; ++d) { o[d][0] *= f[0]; o[d][1] *= f[0]; o[d][2] *= f[1]; o[d][3] *= f[1]; }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[n][e] = ex2(s[n][e] - base[e >> 1]);
                        l[e >> 1] += s[n][e];
                    }
#pragma unroll
                for (int k = 0; k < KW / 16; ++k) {
                    // the probabilities rounded (to nearest) to the cache's type: the tensor core's operand
                    const uint32_t pa[4] = {pack2<T>(s[2 * k][0], s[2 * k][1]), pack2<T>(s[2 * k][2], s[2 * k][3]),
                                            pack2<T>(s[2 * k + 1][0], s[2 * k + 1][1]), pack2<T>(s[2 * k + 1][2], s[2 * k + 1][3])};
#pragma unroll
                    for (int d = 0; d < DT; d += 2) {
                        uint32_t r[4];
                        ldsm4t(vs + Tile<HD>::chunk(kb + k * 16 + (lane & 15), d + (lane >> 4)), r);
                        mma_t<T>(o[d], pa, r[0], r[1]);
                        mma_t<T>(o[d + 1], pa, r[2], r[3]);
                    }
                }
                if (tail) fence_proxy_async();                   // this stage's zeros before the next copy into it
                __syncwarp();
                if (lane == 0) mbar_arrive(&s_empty[st]);
            }

            // ---- the segment's (or the range's) end: one partial result
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
                l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
            }
            const int slot = g.seg + (int)blockIdx.x;
            const bool fits = slot < p.max_slots;                // false only for offsets that do not ascend
            if (!fits && p.err && threadIdx.x == 0) atomicOr(p.err, Z2B_OPS_BAD_INDEX);
            const int rows = min(MT, g.n * p.G - g.j * MT);      // live rows of the tile
            float* po = p.part_o + (size_t)slot * MT * HD;
            float2* pm = p.part_ml + (size_t)slot * MT;
            if constexpr (WN == 1) {
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int row = wr * 16 + r0 + 8 * x;
                    if (!fits || row >= rows) continue;
#pragma unroll
                    for (int d = 0; d < DT; ++d)
                        *(float2*)(po + (size_t)row * HD + d * 8 + quad * 2) = make_float2(o[d][2 * x], o[d][2 * x + 1]);
                    if (quad == 0) pm[row] = make_float2(m[x], l[x]);
                }
            } else {
                if (quad == 0) {
                    s_ml[wc][wr * 16 + r0] = make_float2(m[0], l[0]);
                    s_ml[wc][wr * 16 + r0 + 8] = make_float2(m[1], l[1]);
                }
                compute_sync();
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int row = wr * 16 + r0 + 8 * x;
                    if (row >= rows) continue;
                    float M = -INFINITY;
#pragma unroll
                    for (int w = 0; w < WN; ++w) M = fmaxf(M, s_ml[w][row].x);
                    const float f = m[x] == -INFINITY ? 0.0f : ex2(m[x] - M);
                    float* dst = s_red + (size_t)(wc * MT + row) * RS + quad * 2;
#pragma unroll
                    for (int d = 0; d < DT; ++d) *(float2*)(dst + d * 8) = make_float2(o[d][2 * x] * f, o[d][2 * x + 1] * f);
                }
                compute_sync();
                for (int i = threadIdx.x; fits && i < rows * (HD / 4); i += 32 * COMPUTE_WARPS) {
                    const int row = i / (HD / 4), c = i % (HD / 4) * 4;
                    float4 a = *(const float4*)(s_red + (size_t)row * RS + c);
#pragma unroll
                    for (int w = 1; w < WN; ++w) {
                        const float4 b = *(const float4*)(s_red + (size_t)(w * MT + row) * RS + c);
                        a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
                    }
                    *(float4*)(po + (size_t)row * HD + c) = a;
                    if (c == 0) {
                        float M = -INFINITY, L = 0.0f;
#pragma unroll
                        for (int w = 0; w < WN; ++w) M = fmaxf(M, s_ml[w][row].x);
#pragma unroll
                        for (int w = 0; w < WN; ++w)
                            if (s_ml[w][row].x != -INFINITY) L += s_ml[w][row].y * ex2(s_ml[w][row].x - M);
                        pm[row] = make_float2(M, L);
                    }
                }
                compute_sync();                                  // s_ml and s_red are free again
            }
        }
    }
    // beside a prefix launch: the join that follows waits for this grid, so this grid ends after that one
    if (p.after_prefix) { pdl_release(); pdl_wait(); }
}

// ---- join ---------------------------------------------------------------------------------
struct PartSet {                        // partial results of one launch
    const float* o;
    const float2* ml;
    int mt, kt, grid, max_slots;       // rows of a partial, keys of a unit
};
struct JoinP {
    AttnP a;
    PartSet pf, own;                    // pf.o null: the prefix's partials are in `own` (or there is none)
    void* out;
    float* lse;
    long long o_row, o_head;
};

// One warp per (row, head): lanes gather the statistics of up to 32 partials at a time, then
// the weighted outputs are summed with each lane on its own dims.
template <typename T, int HD, int MT>
__global__ void __launch_bounds__(256) prefix_attn_join_kernel(const __grid_constant__ JoinP p) {
    constexpr int DPL = HD >= 32 ? HD / 32 : 1;
    const AttnP& a = p.a;
    const int lane = threadIdx.x & 31, nh = a.nkv * a.G;
    const int w = blockIdx.x * 8 + (threadIdx.x >> 5), t = w / nh, head = w % nh;
    pdl_wait();
    pdl_release();
    if (t >= a.n_rows || t >= a.row_off[a.n_seq]) return;        // padding stays as it is
    const int h = head / a.G, g = head % a.G;
    const int b = warp_find_seq(a.row_off, a.n_seq, t);
    if (b < 0) return;
    const SeqInfo s = seq_info<MT>(a, b);
    const int i = t - s.lo;
    if (s.bad || i >= s.n) return;

    float M = -INFINITY, L = 0.0f, acc[DPL];
#pragma unroll
    for (int d = 0; d < DPL; ++d) acc[d] = 0.0f;
    const bool has = lane * DPL < HD;
    auto add = [&](const PartSet& ps, long long W, long long first, int nt, int seg, int row) {
        if (nt == 0) return;
        const int ctas = line_ctas(W, ps.grid);
        const int c0 = unit_owner(first, W, ctas), c1 = unit_owner(first + nt - 1, W, ctas);
        for (int base = c0; base <= c1; base += 32) {
            const int slot = seg + base + lane;
            float2 ml = make_float2(-INFINITY, 0.0f);
            if (base + lane <= c1 && slot < ps.max_slots) ml = ps.ml[(size_t)slot * ps.mt + row];
            const float top = fmaxf(M, warp_max(ml.x));
            if (top == -INFINITY) continue;
            const float f = ex2(M - top);
            M = top;
            const float wt = ex2(ml.x - top);
            L = L * f + warp_sum(ml.y * wt);
#pragma unroll
            for (int d = 0; d < DPL; ++d) acc[d] *= f;
            const int n = min(32, c1 - base + 1);
#pragma unroll 4
            for (int k = 0; k < n; ++k) {
                const float wk = __shfl_sync(0xffffffffu, wt, k);
                const int sl = seg + base + k;
                if (wk == 0.0f || !has || sl >= ps.max_slots) continue;
                const float* src = ps.o + ((size_t)sl * ps.mt + row) * HD + lane * DPL;
                if constexpr (DPL == 4) {
                    const float4 v = *(const float4*)src;
                    acc[0] += wk * v.x; acc[1] += wk * v.y; acc[2] += wk * v.z; acc[3] += wk * v.w;
                } else if constexpr (DPL == 2) {
                    const float2 v = *(const float2*)src;
                    acc[0] += wk * v.x; acc[1] += wk * v.y;
                } else {
                    acc[0] += wk * src[0];
                }
            }
        }
    };
    const int pf_units = a.pf_row_tiles * a.nkv * cdiv(a.prefix_len, KT);
    const int* units = a.plan;
    const long long W = (long long)pf_units + units[a.n_seq];
    {
        const PartSet& ps = p.pf.o ? p.pf : p.own;
        const int r = t * a.G + g, seg = (r / ps.mt) * a.nkv + h, pf_nt = cdiv(a.prefix_len, ps.kt);
        const long long Wp = p.pf.o ? (long long)cdiv(a.n_rows * a.G, ps.mt) * a.nkv * pf_nt : W;
        add(ps, Wp, (long long)seg * pf_nt, pf_nt, seg, r % ps.mt);
    }
    {
        const int r = i * a.G + g, js = (r / MT) * a.nkv + h;
        add(p.own, W, (long long)pf_units + units[b] + (long long)js * s.nt, s.nt,
            a.pf_row_tiles * a.nkv + a.plan[a.n_seq + 1 + b] + js, r % MT);
    }
    const float inv = L > 0.0f ? 1.0f / L : 0.0f;
    if (has) {
        T* dst = (T*)p.out + (long long)t * p.o_row + (long long)head * p.o_head + lane * DPL;
        if constexpr (DPL == 1) *dst = from_f32<T>(acc[0] * inv);
        else {
#pragma unroll
            for (int d = 0; d < DPL; d += 2) *(uint32_t*)(dst + d) = pack2<T>(acc[d] * inv, acc[d + 1] * inv);
        }
    }
    // ln(sum) = (M + log2 L) ln 2
    if (lane == 0 && p.lse) p.lse[(long long)t * nh + head] = L > 0.0f ? (M + log2f(L)) * 0.6931471805599453f : -INFINITY;
}

// ---- host -----------------------------------------------------------------------------------
struct HostPlan {
    int G, wm, mt;                      // own rows per segment
    int grid, own_slots, pf_rt;         // pf_rt > 0: prefix row tiles inside the own launch
    bool pf_apart;                      // the prefix has a launch of its own
    bool pf_tc;                         // ... on the tcgen05 kernel
    int pf_mt, pf_kt, pf_tiles, pf_grid, pf_slots;
    size_t off_own_ml, off_own_o, off_pf_ml, off_pf_o, bytes;
};

size_t up(size_t x) { return (x + 255) & ~(size_t)255; }

HostPlan host_plan(const z2b_prefix_attn_args& a) {
    HostPlan h{};
    const int nkv = a.kv->n_head_kv, hd = a.kv->head_dim;
    h.G = a.n_head / nkv;
    // rows of one stream and key head, on average: the smallest tile that holds them
    const long long rows = (long long)((a.n_rows + a.n_seq - 1) / a.n_seq) * h.G;
    h.wm = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    h.mt = 16 * h.wm;
    h.grid = 148 * 2;
    const long long R = (long long)a.n_rows * h.G;
    if (a.prefix_len > 0) {
        const long long rt = (R + h.mt - 1) / h.mt;
        if (rt <= 2) h.pf_rt = (int)rt;
        else {
            h.pf_apart = true;
            // more rows than one warp-level tile holds: 256-row tiles on tcgen05 (one CTA per SM)
            h.pf_tc = hd >= 64 && R > 64 && a.scale != 0.0f;
            h.pf_mt = h.pf_tc ? TC_ROWS : 64;
            h.pf_kt = h.pf_tc ? TC_KEYS : KT;
            h.pf_tiles = (int)((R + h.pf_mt - 1) / h.pf_mt);
            h.pf_grid = h.pf_tc ? 148 : 148 * 2;
            h.pf_slots = h.pf_tiles * nkv + h.pf_grid;
        }
    }
    const long long segs = ((R + h.mt - 1) / h.mt + a.n_seq + h.pf_rt) * nkv;
    h.own_slots = (int)(segs + h.grid);
    size_t n = up((size_t)2 * (a.n_seq + 1) * 4);
    h.off_own_ml = n; n += up((size_t)h.own_slots * h.mt * 8);
    h.off_own_o = n; n += up((size_t)h.own_slots * h.mt * hd * 4);
    h.off_pf_ml = n; n += up((size_t)h.pf_slots * h.pf_mt * 8);
    h.off_pf_o = n; n += up((size_t)h.pf_slots * h.pf_mt * hd * 4);
    h.bytes = n;
    return h;
}

bool make_map(CUtensorMap* m, const void* base, const z2b_paged_kv& c, int box_rows, int inner) {
    auto enc = tensor_map_encoder();
    if (!enc) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)c.head_dim, (cuuint64_t)c.n_head_kv, (cuuint64_t)c.page_len, (cuuint64_t)c.n_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)c.head_stride * 2, (cuuint64_t)c.row_stride * 2, (cuuint64_t)c.page_stride * 2};
    const cuuint32_t box[4] = {(cuuint32_t)inner, 1, (cuuint32_t)box_rows, 1}, one[4] = {1, 1, 1, 1};
    const CUtensorMapSwizzle sw = inner == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : inner == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B;
    return enc(m, c.type == Z2B_TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
               const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, sw,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int HD, int WM>
cudaError_t go_attn(AttnP p, const CUtensorMap& km, const CUtensorMap& vm, int grid, cudaStream_t s) {
    constexpr int WN = COMPUTE_WARPS / WM, MT = 16 * WM, STAGE = 2 * Tile<HD>::BYTES;
    p.stages = 65536 / STAGE > 8 ? 8 : 65536 / STAGE;
    const size_t smem = 1024 + (size_t)p.stages * STAGE + (WN > 1 ? (size_t)WN * MT * (HD + 4) * 4 : 0) +
                        (p.own ? (size_t)2 * (p.n_seq + 1) * 4 : 0);
    static std::atomic<uint64_t> opted{0};                       // devices whose shared-memory opt-in is done
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(opted.load(std::memory_order_relaxed) >> dev & 1)) {
        e = cudaFuncSetAttribute(prefix_attn_kernel<T, HD, WM>, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SMEM);
        if (e != cudaSuccess) return e;
        if (dev < 64) opted.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    return launch_pdl(prefix_attn_kernel<T, HD, WM>, dim3(grid), dim3(THREADS), smem, s, p, km, vm);
}

template <typename T, int HD>
cudaError_t go_all(const z2b_prefix_attn_args& a, const HostPlan& h, cudaStream_t s) {
    const z2b_paged_kv& c = *a.kv;
    AttnP p{};
    p.q = a.q; p.q_row = a.q_row; p.q_head = a.q_head; p.table_stride = a.table_stride;
    p.row_off = a.row_off; p.seq_len = a.seq_len; p.table = a.page_table; p.prefix_pages = a.prefix_pages; p.err = a.err;
    p.n_rows = a.n_rows; p.n_seq = a.n_seq; p.nkv = c.n_head_kv; p.G = h.G; p.page_len = c.page_len; p.n_pages = c.n_pages;
    p.max_pages = a.max_pages; p.prefix_len = a.prefix_len;
    p.box_rows = c.page_len & -c.page_len;
    if (p.box_rows > KT) p.box_rows = KT;
    p.scale2 = a.scale * 1.4426950408889634f;
    CUtensorMap km, vm;
    if (!make_map(&km, c.k, c, p.box_rows, Tile<HD>::INNER) || !make_map(&vm, c.v, c, p.box_rows, Tile<HD>::INNER))
        return cudaErrorNotSupported;
    uint8_t* ws = (uint8_t*)a.workspace;
    p.plan = (int*)ws;
    cudaError_t e;
    if (h.pf_apart) {
        AttnP f = p;
        f.pf_row_tiles = h.pf_tiles;
        f.max_slots = h.pf_slots;
        f.part_ml = (float2*)(ws + h.off_pf_ml);
        f.part_o = (float*)(ws + h.off_pf_o);
        if constexpr (HD >= 64) e = h.pf_tc ? launch_prefix_tc<T, HD>(f, km, vm, h.pf_grid, s) : go_attn<T, HD, 4>(f, km, vm, h.pf_grid, s);
        else e = go_attn<T, HD, 4>(f, km, vm, h.pf_grid, s);
        if (e != cudaSuccess) return e;
    }
    p.own = 1;
    p.pf_row_tiles = h.pf_rt;
    p.after_prefix = h.pf_apart;
    p.max_slots = h.own_slots;
    p.part_ml = (float2*)(ws + h.off_own_ml);
    p.part_o = (float*)(ws + h.off_own_o);
    e = h.wm == 1 ? go_attn<T, HD, 1>(p, km, vm, h.grid, s) : h.wm == 2 ? go_attn<T, HD, 2>(p, km, vm, h.grid, s)
                                                                       : go_attn<T, HD, 4>(p, km, vm, h.grid, s);
    if (e != cudaSuccess) return e;
    JoinP j{};
    j.a = p;
    j.own = PartSet{p.part_o, p.part_ml, h.mt, KT, h.grid, h.own_slots};
    if (h.pf_apart) j.pf = PartSet{(float*)(ws + h.off_pf_o), (float2*)(ws + h.off_pf_ml), h.pf_mt, h.pf_kt, h.pf_grid, h.pf_slots};
    j.out = a.out; j.o_row = a.o_row; j.o_head = a.o_head; j.lse = a.lse;
    const dim3 grid((unsigned)(((long long)a.n_rows * a.n_head + 7) / 8));
    if (h.wm == 1) return launch_pdl(prefix_attn_join_kernel<T, HD, 16>, grid, dim3(256), 0, s, j);
    if (h.wm == 2) return launch_pdl(prefix_attn_join_kernel<T, HD, 32>, grid, dim3(256), 0, s, j);
    return launch_pdl(prefix_attn_join_kernel<T, HD, 64>, grid, dim3(256), 0, s, j);
}

template <typename T> cudaError_t go_type(const z2b_prefix_attn_args& a, const HostPlan& h, cudaStream_t s) {
    switch (a.kv->head_dim) {
        case 16: return go_all<T, 16>(a, h, s);
        case 32: return go_all<T, 32>(a, h, s);
        case 64: return go_all<T, 64>(a, h, s);
        case 128: return go_all<T, 128>(a, h, s);
    }
    return cudaErrorInvalidValue;
}

}  // namespace

size_t prefix_attention_bytes(const z2b_prefix_attn_args& a) { return host_plan(a).bytes; }

cudaError_t launch_prefix_attention(const z2b_prefix_attn_args& a, cudaStream_t s) {
    const HostPlan h = host_plan(a);
    return a.kv->type == Z2B_TYPE_F16 ? go_type<__half>(a, h, s) : go_type<__nv_bfloat16>(a, h, s);
}

}  // namespace z2b
