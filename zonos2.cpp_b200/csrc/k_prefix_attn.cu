// k_prefix_attn.cu — attention of many streams over one shared prefix and each stream's own
// paged rows (sm_100a; include/z2b_ops.h).
//
// out = softmax(scale q K^T) V over the union of two key sets, each handled where it is
// cheapest and joined by their softmax statistics:
//   out = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i ,  M = max m_i
// over partial results i with O_i = sum_k p_k v_k, l_i = sum_k p_k, p_k = 2^(s_k - m_i).
//   prefix: the rows of ALL streams form one tall query matrix per key head, so the prefix is
//           read once per row tile instead of once per stream (k_prefix_tc.cu when they are many);
//   own:    each stream's rows (its query heads of one key head side by side) over its pages.
// Bound: the own part by HBM bytes, the prefix by tensor-core rate once the rows are many.
//
// Probabilities are rounded to the cache's type for their product with V, since the tensor cores take
// 16-bit operands; taking them as a sum of two such would double those products. Against 64 bits the
// result is 1.2 to 1.4 times as far off as with f32 probabilities (bf16 0.0023 of the output's size to
// 0.0017, f16 0.00026 to 0.00021), the last rounding included. Sums and statistics are f32.
//
// Made for decode and draft rows. Prompt rows are right but far from the tensor cores' rate: their own
// keys come here too, read again from L2 for every row tile. 2048 rows of one stream over themselves, 32
// heads of 128 dims, take 394 us (87 TFLOP/s; the operations alone 21); 8 x 256 rows behind a prefix of
// 8192, which k_prefix_tc.cu takes, 370 us (765 TFLOP/s). head_dim 16 and 32 never take that path: 64
// streams of 16 heads behind a prefix of 8192 take 44 us with either, 26 with 64 dims.
//
// Work split: a unit is KU keys of one segment (row tile x key head). All units form one line
// that is cut into equal contiguous ranges, one per worker, whatever the lengths; a worker
// leaves one partial result per segment it touches. Partial slots are segment + worker: going
// along the line every new partial advances one of the two, so slots never collide and their
// number is bounded by segments + workers. Nothing is accumulated by atomics: the same call
// gives the same bits.
//
// A worker is ONE WARP with a TMA ring of its own, so that no barrier ties warps together and
// the loads of a warp's next units stay in flight while it finishes a segment or fetches the
// next one's queries; together the rings of an SM hold 192 KB.
#include "launch.cuh"
#include "ops.h"
#include "prefix_attn.cuh"
#include "../../include/z2b_tools.h"

namespace z2b {
namespace {

// Keys of a unit, ring stages of a warp (of 16, 8, 4 and 2 KB), and warps of a CTA (one CTA per
// SM): as many as registers and shared memory hold.
__host__ __device__ constexpr int unit_keys(int hd) { return 32; }
__host__ __device__ constexpr int ring_stages(int hd) { return hd == 128 ? 2 : hd == 64 ? 3 : hd == 32 ? 6 : 8; }
__host__ __device__ constexpr int max_warps(int hd) { return hd == 128 ? 6 : 8; }
constexpr int MAX_SMEM = 226 * 1024;   // dynamic shared memory of a launch
constexpr int CTAS = 148;              // one per SM

// Shared-memory tile of KU rows of one key head: rows of RB bytes (at most 128: head_dim 128
// is two halves), 16-byte chunks XOR-swizzled as the TMA box writes them.
template <int HD> struct Tile {
    static constexpr int KU = unit_keys(HD);
    static constexpr int INNER = HD < 64 ? HD : 64;              // elements of one box row
    static constexpr int HALVES = HD / INNER;
    static constexpr int RB = INNER * 2;
    static constexpr int BYTES = KU * HD * 2;
    __device__ static __forceinline__ uint32_t chunk(int row, int c) {   // byte offset of 8 elements
        constexpr int PER = RB / 16;
        const int half = c / PER, cc = c % PER;
        const int x = PER == 8 ? (row & 7) : PER == 4 ? ((row >> 1) & 3) : ((row >> 2) & 1);
        return half * (KU * RB) + row * RB + ((cc ^ x) << 4);
    }
};

// The line's streams in shared memory, and one segment of it.
struct Line {
    const int4* rec;                   // [n_seq + 1] first unit, first segment, first row, rows
    const int* len;                    // [n_seq]
    int pf_nt, pf_units, total_rows;   // units of a prefix segment, line positions of all of them
};
struct Seg {
    int h, j, seg, unit0, nt;          // key head, row tile, segment id, position of its first unit, units
    int lo, n, klen, lim_max;          // first row, rows, keys, keys that the tile's last row sees
    const int* pages;
    bool prefix;
};

template <int MT, int KU> __device__ __forceinline__ Seg find_seg(const AttnP& p, const Line& ln, int u) {
    Seg g;
    if (u < ln.pf_units) {
        const int size = ln.pf_nt + SEG_COST;
        g.seg = u / size;
        g.unit0 = g.seg * size + SEG_COST;
        g.nt = ln.pf_nt;
        g.prefix = true;
        g.h = g.seg / p.pf_row_tiles;
        g.j = g.seg % p.pf_row_tiles;
        g.lo = 0;
        g.n = ln.total_rows;
        g.klen = g.lim_max = p.prefix_len;
        g.pages = p.prefix_pages;
        return g;
    }
    const int v = u - ln.pf_units;
    int lo = 0, hi = p.n_seq - 1;                                // the last stream that starts at or before v
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (ln.rec[mid].x <= v) lo = mid; else hi = mid - 1;
    }
    const int4 r = ln.rec[lo];
    g.lo = r.z;
    g.n = r.w;
    g.klen = ln.len[lo];
    g.nt = cdiv(g.klen, KU);
    g.prefix = false;
    const int size = g.nt + SEG_COST, qt = cdiv(g.n * p.G, MT), js = (v - r.x) / size;
    g.seg = p.pf_row_tiles * p.nkv + r.y + js;
    g.unit0 = ln.pf_units + r.x + js * size + SEG_COST;
    g.h = js / qt;
    g.j = js % qt;
    const int last = min(g.n - 1, div_g(p, g.j * MT + MT - 1));
    g.lim_max = min(g.klen, g.klen - g.n + last + 1);
    g.pages = p.table + (long long)lo * p.table_stride;
    return g;
}

// A segment has MT = 8 NB rows. The products are taken transposed, keys and dims on the tensor
// core's 16-row side and the rows on its 8-column side, since decode has few rows:
//   S^T[16 keys][8 rows] = K Q^T ,  O^T[16 dims][8 rows] += V^T P^T .
// P^T comes out of S^T's accumulator layout by one 8 x 8 transpose per tile.
template <typename T, int HD, int NB>
__global__ void __launch_bounds__(32 * max_warps(HD), 1) prefix_attn_kernel(const __grid_constant__ AttnP p,
                                                                           const __grid_constant__ CUtensorMap kmap,
                                                                           const __grid_constant__ CUtensorMap vmap) {
    constexpr int MT = 8 * NB, KU = unit_keys(HD), KS = HD / 16, KM = KU / 16, DT = HD / 16;
    constexpr int STAGE = 2 * Tile<HD>::BYTES, NS = ring_stages(HD);
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) uint64_t s_full[max_warps(HD)][NS];
    __shared__ int s_scan[2][max_warps(HD)];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    uint8_t* ring = smem + (size_t)warp * NS * STAGE;
    uint8_t* s_q = smem + (size_t)nw * NS * STAGE + (size_t)warp * MT * HD * 2;
    int4* s_rec = (int4*)(smem + (size_t)nw * (NS * STAGE + MT * HD * 2));
    int* s_len = (int*)(s_rec + p.n_seq + 1);
    uint64_t* full = s_full[warp];

    if (lane == 0) {
        for (int i = 0; i < NS; ++i) mbar_init(&full[i], 1);
        fence_mbar_init();
    }
    if (threadIdx.x == 0) { prefetch_map(&kmap); prefetch_map(&vmap); }
    if (!p.after_prefix) pdl_wait();
    pdl_release();                                               // the join reads its streams' extents meanwhile
    const int last_off = ld_word(p.row_off + p.n_seq, p.after_prefix);

    // ---- the line: offsets of every stream's units and segments, by a block scan
    {
        const int per = cdiv(p.n_seq, blockDim.x);
        const int b0 = min(p.n_seq, (int)threadIdx.x * per), b1 = min(p.n_seq, b0 + per);
        unsigned su = 0, sg = 0;
        int drops = 0;
        for (int b = b0; b < b1; ++b) {
            const SeqInfo s = seq_info<MT, KU>(p, b, p.after_prefix);
            drops |= s.drops;
            if (s.bad && blockIdx.x == 0 && p.err) atomicOr(p.err, Z2B_OPS_BAD_INDEX);
            s_rec[b] = make_int4(su, sg, s.lo, s.n);
            s_len[b] = s.len;
            su += s.nt ? s.qt * p.nkv * (s.nt + SEG_COST) : 0;
            sg += s.qt * p.nkv;
        }
        unsigned iu = su, ig = sg;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned a = __shfl_up_sync(0xffffffffu, iu, o), c = __shfl_up_sync(0xffffffffu, ig, o);
            if (lane >= o) { iu += a; ig += c; }
        }
        if (lane == 31) { s_scan[0][warp] = iu; s_scan[1][warp] = ig; }
        drops = __syncthreads_or(drops);
        unsigned eu = iu - su, eg = ig - sg;
        for (int w = 0; w < warp; ++w) { eu += s_scan[0][w]; eg += s_scan[1][w]; }
        for (int b = b0; b < b1; ++b) {
            s_rec[b].x += eu;
            s_rec[b].y += eg;
            if (blockIdx.x == 0) { p.plan[b] = s_rec[b].x; p.plan[p.n_seq + 1 + b] = s_rec[b].y; }
        }
        if (threadIdx.x == blockDim.x - 1) {
            s_rec[p.n_seq] = make_int4(drops ? 0 : eu + su, 0, 0, 0);
            if (blockIdx.x == 0) p.plan[p.n_seq] = drops ? -1 : (int)(eu + su);
        }
    }
    Line ln;
    ln.rec = s_rec;
    ln.len = s_len;
    ln.total_rows = max(0, min(p.n_rows, last_off));
    ln.pf_nt = cdiv(p.prefix_len, KU);
    ln.pf_units = p.pf_row_tiles * p.nkv * (ln.pf_nt + SEG_COST);
    __syncthreads();
    const int W = ln.pf_units + s_rec[p.n_seq].x;
    const Cuts cuts(p, W, gridDim.x, nw);
    int me, u = 0, u1 = 0;                                       // few workers: one per SM first
    if ((int)blockIdx.x < p.early) {
        me = warp * p.early + blockIdx.x;
        if (me < cuts.a.workers) {
            u = cuts.a.begin(me);
            u1 = cuts.a.begin(me + 1);
        }
    } else {
        const int i = warp * (gridDim.x - p.early) + blockIdx.x - p.early;
        me = cuts.na + i;
        if (i < cuts.b.workers) {
            u = cuts.mid + cuts.b.begin(i);
            u1 = cuts.mid + cuts.b.begin(i + 1);
        }
    }

    // ---- the copies, NS units ahead of the products: a box of K and one of V per run of rows
    // that stays within a page; lane i looks up run i's page
    const int nb = KU / p.box_rows;                              // at most 4
    Seg gi;                            // segment of the next unit to copy
    gi.unit0 = -1;
    gi.nt = 0;
    int ui = u, issued = 0, page = 0, pidx = 0, prow = 0;        // this lane's box: page id, its index, row in it
    bool wanted = false;
    auto look_up = [&] {               // move ui to the next unit that some row sees; this lane's page of it
        prow += KU;
        while (prow >= p.page_len) { prow -= p.page_len; ++pidx; }
        while (ui < u1) {
            if (ui >= gi.unit0 + gi.nt) {
                gi = find_seg<MT, KU>(p, ln, ui);
                ui = max(ui, gi.unit0);
                const int key = (ui - gi.unit0) * KU + lane * p.box_rows;
                pidx = key / p.page_len;
                prow = key % p.page_len;
            }
            if ((ui - gi.unit0) * KU < gi.lim_max) break;
            ui = gi.unit0 + gi.nt;                               // keys only rise: behind an unseen unit all are
        }
        if (ui >= u1) return;
        page = p.n_pages;                                        // out of the view: the box fills with zeros
        wanted = false;
        if (lane < nb && (ui - gi.unit0) * KU + lane * p.box_rows < gi.klen) {
            page = ld_word(gi.pages + pidx, p.after_prefix);     // on its way until copy() checks it
            wanted = true;
        }
    };
    auto copy = [&] {
        if (ui >= u1) return;
        const int st = issued % NS;
        const uint32_t dst = smem_u32(ring) + st * STAGE;
        if (wanted && (page < 0 || page >= p.n_pages)) {
            page = p.n_pages;
            if (p.err) atomicOr(p.err, Z2B_OPS_BAD_PAGE);
        }
        if (lane == 0) mbar_expect_tx(&full[st], STAGE);
        __syncwarp();
        for (int i = 0; i < nb; ++i) {
            const int pg = __shfl_sync(0xffffffffu, page, i), pr = __shfl_sync(0xffffffffu, prow, i);
            if (elect_one())
                for (int half = 0; half < Tile<HD>::HALVES; half += p.box_halves) {
                    const uint32_t d = dst + half * (KU * Tile<HD>::RB) + i * p.box_rows * Tile<HD>::RB;
                    tma_load_page(d, &kmap, pr, half, gi.h, pg, &full[st]);
                    tma_load_page(d + Tile<HD>::BYTES, &vmap, pr, half, gi.h, pg, &full[st]);
                }
        }
        __syncwarp();
        ++issued;
        ++ui;
        look_up();
    };
    look_up();
    for (int i = 0; i < NS; ++i) copy();

    // ---- the queries of the next segment, on their way while this one is worked on
    const bool q16 = ((reinterpret_cast<uintptr_t>(p.q) | (uintptr_t)(p.q_row * 2) | (uintptr_t)(p.q_head * 2)) & 15) == 0;
    auto fetch_q = [&](const Seg& g) {
        for (int i = lane; i < MT * (HD / 8); i += 32) {
            const int row = i / (HD / 8), c = i % (HD / 8), rr = g.j * MT + row, t = div_g(p, rr);
            const bool live = t < g.n;
            const T* src = (const T*)p.q + (live ? (long long)(g.lo + t) * p.q_row + (long long)(g.h * p.G + rr - t * p.G) * p.q_head + c * 8 : 0);
            uint8_t* dst = s_q + row * (HD * 2) + ((c ^ (row & (HD / 8 - 1) & 7)) << 4);
            if (q16) cp_async16(dst, src, live);
            else
#pragma unroll
                for (int e = 0; e < 4; ++e) ((uint32_t*)dst)[e] = live ? (uint32_t)ld_word((const int*)(src + 2 * e), p.after_prefix) : 0u;
        }
        cp_async_commit();
    };
    const bool flat = p.scale2 == 0.0f;                          // all scores equal: zero queries, so that masked keys stay apart
    const float sc = flat ? 1.0f : fabsf(p.scale2);              // the maximum is taken before the scale: a negative one
    const uint32_t q_and = flat ? 0u : 0xffffffffu, q_xor = p.scale2 < 0.0f ? 0x80008000u : 0u;     // negates the queries
    // byte offsets of this lane's 16-byte chunks in a K and a V tile, for four steps of 32 bytes:
    // K as rows (A of S^T), V transposed on the way (A of O^T)
    constexpr int OFFS = HD >= 64 ? 4 : HD / 16;
    uint32_t koff[OFFS], voff[OFFS];
#pragma unroll
    for (int k = 0; k < OFFS; ++k) {
        koff[k] = Tile<HD>::chunk(lane & 15, 2 * k + (lane >> 4));
        voff[k] = Tile<HD>::BYTES + Tile<HD>::chunk(((lane >> 4) << 3) + (lane & 7), 2 * k + ((lane >> 3) & 1));
    }
    const int key_l = lane >> 2, row_l = (lane & 3) * 2;         // this lane's key and first row in an accumulator tile

    int it = 0;
    bool dead = false;                                           // a wait ran out
    const bool quick = p.polls > 0;                              // read here, not on the first wait's way
    Seg g;
    if (u < u1) {
        g = find_seg<MT, KU>(p, ln, u);
        u = max(u, g.unit0);
        if (u < u1) fetch_q(g);
    }
    while (u < u1) {
        const int end = min(u1, g.unit0 + g.nt);
        cp_async_wait_0();
        __syncwarp();
        uint32_t qb[NB][KS][2];                                  // Q^T as B operand
#pragma unroll
        for (int nb_ = 0; nb_ < NB; ++nb_)
#pragma unroll
            for (int k = 0; k < KS; k += 2) {
                const int row = nb_ * 8 + (lane & 7), c = 2 * k + (lane >> 3);
                uint32_t r[4];
                ldsm4(smem_u32(s_q) + row * (HD * 2) + (((KS > 1 ? c : c & 1) ^ (row & (HD / 8 - 1) & 7)) << 4), r);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (k + e / 2 < KS) qb[nb_][k + e / 2][e & 1] = (r[e] & q_and) ^ q_xor;
            }
        __syncwarp();
        Seg gn;
        if (end < u1) {
            gn = find_seg<MT, KU>(p, ln, end);
            if (gn.unit0 < u1) fetch_q(gn);
        }
        int lim[NB][2], lim_min = 0x7fffffff;                    // keys that this lane's rows see
#pragma unroll
        for (int nb_ = 0; nb_ < NB; ++nb_)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int i = div_g(p, g.j * MT + nb_ * 8 + row_l + x);
                lim[nb_][x] = i >= g.n ? 0 : g.prefix ? g.klen : min(g.klen, g.klen - g.n + i + 1);
                if (i < g.n) lim_min = min(lim_min, lim[nb_][x]);        // rows that do not exist are never stored
            }
        float o[NB][DT][4], m[NB][2], l[NB][2];
#pragma unroll
        for (int nb_ = 0; nb_ < NB; ++nb_) {
            m[nb_][0] = m[nb_][1] = -INFINITY;
            l[nb_][0] = l[nb_][1] = 0.0f;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[nb_][d][0] = o[nb_][d][1] = o[nb_][d][2] = o[nb_][d][3] = 0.0f;
        }

        for (; u < end; ++u) {
            const int key0 = (u - g.unit0) * KU;
            if (key0 >= g.lim_max) { u = end; break; }           // no row of the tile sees the rest
            const int st = it % NS;
            if (!dead)
                dead = __any_sync(0xffffffffu, !((quick && mbar_try_wait(&full[st], (it / NS) & 1)) || mbar_wait(&full[st], (it / NS) & 1, p.err, p.polls)));
            if (dead) {                                          // this and the range's other segments: not numbers
#pragma unroll
                for (int nb_ = 0; nb_ < NB; ++nb_) l[nb_][0] = l[nb_][1] = NAN;
                u = end;
                break;
            }
            ++it;
            uint8_t* kt = ring + (size_t)st * STAGE;
            const uint32_t ks = smem_u32(kt);
            const bool tail = key0 + KU > g.klen;
            if (tail) {
                // rows behind the last key may hold anything: zero times that is not zero
                for (int i = lane; i < KU * (HD / 8); i += 32)
                    if (key0 + i / (HD / 8) >= g.klen)
                        *(uint4*)(kt + Tile<HD>::BYTES + Tile<HD>::chunk(i / (HD / 8), i % (HD / 8))) = make_uint4(0, 0, 0, 0);
                __syncwarp();
            }
            float s[NB][KM][4];
#pragma unroll
            for (int nb_ = 0; nb_ < NB; ++nb_)
#pragma unroll
                for (int n = 0; n < KM; ++n) s[nb_][n][0] = s[nb_][n][1] = s[nb_][n][2] = s[nb_][n][3] = 0.0f;
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int n = 0; n < KM; ++n) {
                    uint32_t r[4];
                    ldsm4(ks + koff[k % OFFS] + (k / OFFS) * (KU * Tile<HD>::RB) + n * 16 * Tile<HD>::RB, r);
#pragma unroll
                    for (int nb_ = 0; nb_ < NB; ++nb_) mma_t<T>(s[nb_][n], r, qb[nb_][k][0], qb[nb_][k][1]);
                }
            if (__any_sync(0xffffffffu, key0 + KU > lim_min)) {  // some row does not see all of the unit
#pragma unroll
                for (int nb_ = 0; nb_ < NB; ++nb_)
#pragma unroll
                    for (int n = 0; n < KM; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (key0 + n * 16 + key_l + (e >> 1) * 8 >= lim[nb_][e & 1]) s[nb_][n][e] = -INFINITY;
            }
            float top[NB][2];
            bool raise = false;
#pragma unroll
            for (int nb_ = 0; nb_ < NB; ++nb_)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    float mx = fmaxf(s[nb_][0][x], s[nb_][0][2 + x]);
#pragma unroll
                    for (int n = 1; n < KM; ++n) mx = fmaxf(mx, fmaxf(s[nb_][n][x], s[nb_][n][2 + x]));
                    top[nb_][x] = mx;
                }
            // maxima over the lanes that share the rows
#pragma unroll
            for (int w = 4; w < 32; w <<= 1)
#pragma unroll
                for (int nb_ = 0; nb_ < NB; ++nb_)
#pragma unroll
                    for (int x = 0; x < 2; ++x) top[nb_][x] = fmaxf(top[nb_][x], __shfl_xor_sync(0xffffffffu, top[nb_][x], w));
#pragma unroll
            for (int nb_ = 0; nb_ < NB; ++nb_)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    top[nb_][x] *= sc;
                    raise |= top[nb_][x] > m[nb_][x] + LAG;
                }
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int nb_ = 0; nb_ < NB; ++nb_) {
                    float f[2];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        f[x] = 1.0f;
                        if (top[nb_][x] > m[nb_][x] + LAG) {
                            const float to = top[nb_][x] - P_SHIFT;
                            f[x] = ex2(m[nb_][x] - to);
                            m[nb_][x] = to;
                        }
                        l[nb_][x] *= f[x];
                    }
#pragma unroll
                    for (int d = 0; d < DT; ++d) { o[nb_][d][0] *= f[0]; o[nb_][d][1] *= f[1]; o[nb_][d][2] *= f[0]; o[nb_][d][3] *= f[1]; }
                }
            }
            uint32_t pb[NB][KM][2];                              // P^T as B operand
#pragma unroll
            for (int nb_ = 0; nb_ < NB; ++nb_) {
                // a row that has seen no key yet has a maximum of -infinity, and no probability
                const float b0 = m[nb_][0] == -INFINITY ? 0.0f : -m[nb_][0], b1 = m[nb_][1] == -INFINITY ? 0.0f : -m[nb_][1];
#pragma unroll
                for (int n = 0; n < KM; ++n) {
                    float* x = s[nb_][n];
                    x[0] = ex2(fmaf(x[0], sc, b0));
                    x[1] = ex2(fmaf(x[1], sc, b1));
                    x[2] = ex2(fmaf(x[2], sc, b0));
                    x[3] = ex2(fmaf(x[3], sc, b1));
                    l[nb_][0] += x[0] + x[2];
                    l[nb_][1] += x[1] + x[3];
                    // rounded (to nearest) to the cache's type: the tensor core's operand
                    pb[nb_][n][0] = movm(pack2<T>(x[0], x[1]));
                    pb[nb_][n][1] = movm(pack2<T>(x[2], x[3]));
                }
            }
#pragma unroll
            for (int n = 0; n < KM; ++n)
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    uint32_t r[4];
                    ldsm4t(ks + voff[d % OFFS] + (d / OFFS) * (KU * Tile<HD>::RB) + n * 16 * Tile<HD>::RB, r);
#pragma unroll
                    for (int nb_ = 0; nb_ < NB; ++nb_) mma_t<T>(o[nb_][d], r, pb[nb_][n][0], pb[nb_][n][1]);
                }
            if (tail) fence_proxy_async();                       // this stage's zeros before the next copy into it
            __syncwarp();
            copy();
        }

        // ---- the segment's (or the range's) end: one partial result
        const int slot = g.seg + me;
        const int rows = min(MT, g.n * p.G - g.j * MT);          // live rows of the tile
        float* po = p.part_o + (size_t)slot * MT * HD;
        float2* pm = p.part_ml + (size_t)slot * MT;
#pragma unroll
        for (int nb_ = 0; nb_ < NB; ++nb_)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                float sum = l[nb_][x];
#pragma unroll
                for (int w = 4; w < 32; w <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
                const int row = nb_ * 8 + row_l + x;
                if (row >= rows) continue;
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    po[(size_t)row * HD + d * 16 + key_l] = o[nb_][d][x];
                    po[(size_t)row * HD + d * 16 + 8 + key_l] = o[nb_][d][2 + x];
                }
                if (key_l == 0) pm[row] = make_float2(m[nb_][x], sum);
            }
        if (end < u1) u = max(end, gn.unit0);
        g = gn;
    }
    cp_async_wait_0();
    // after a wait that ran out, the copies in flight still land in this CTA's memory
    if (dead)
        for (int k = it; k < issued; ++k) mbar_wait(&full[k % NS], (k / NS) & 1, nullptr, 1u << 16);
    // beside a prefix launch: the join that follows waits for this grid, so this grid ends after that one
    if (p.after_prefix) pdl_wait();
}

// ---- join ---------------------------------------------------------------------------------
struct PartSet {                        // partial results of one launch
    const float* o;
    const float2* ml;
    int mt, keys, workers, slots, row_tiles;       // rows of a partial, keys of a unit, ..., row tiles of the prefix in it
};
struct JoinP {
    AttnP a;
    PartSet pf, own;                    // pf: the launch that took the prefix (own's when it took both)
    int pf_apart;
    void* out;
    float* lse;
    long long o_row, o_head;
};

// Where the partial results of one head of a row lie: n0 in the prefix's set from slot0 on, n1 in
// the stream's own, each at its row of a slot.
struct Parts { int n0, n1, slot0, slot1, row0, row1; };

// One row's stream, found ahead of the launch's wait (the launches ahead release this one once
// their own predecessors are done, so the call's inputs are there; they are read past L1), and the
// offsets of its units and segments on the line: read from the plan after the wait, or (EARLY)
// summed by the warp from the inputs, and the caller waits.
struct RowInfo { SeqInfo s; int i; unsigned own_units, unit_b, seg_b; bool taken, live; };
template <int MT, int KU, bool EARLY> __device__ __forceinline__ RowInfo row_info(const AttnP& a, int t) {
    const int lane = threadIdx.x & 31;
    RowInfo x;
    const int total = ld_word(a.row_off + a.n_seq, true);
    const int b = warp_find_seq(a.row_off, a.n_seq, t, true);
    x.s = seq_info<MT, KU>(a, b, true);
    if constexpr (EARLY) {
        x.own_units = x.unit_b = x.seg_b = 0;
        bool drops = false;
        for (int c = lane; c < a.n_seq; c += 32) {
            const SeqInfo y = seq_info<MT, KU>(a, c, true);
            drops |= y.drops;
            const unsigned segs = y.qt * a.nkv, units = y.nt ? segs * (y.nt + SEG_COST) : 0u;
            x.own_units += units;
            if (c < b) { x.unit_b += units; x.seg_b += segs; }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            x.own_units += __shfl_xor_sync(0xffffffffu, x.own_units, o);
            x.unit_b += __shfl_xor_sync(0xffffffffu, x.unit_b, o);
            x.seg_b += __shfl_xor_sync(0xffffffffu, x.seg_b, o);
        }
        x.taken = !__any_sync(0xffffffffu, drops);
    } else {
        pdl_wait();
        x.own_units = a.plan[a.n_seq];
        x.taken = a.plan[a.n_seq] >= 0;
        x.unit_b = a.plan[b];
        x.seg_b = a.plan[a.n_seq + 1 + b];
    }
    x.i = t - x.s.lo;
    x.live = x.taken && t < total && !x.s.bad && x.i >= 0 && x.i < x.s.n;   // else padding, which stays as it is
    return x;
}

template <int MT, int KU> __device__ __forceinline__ Parts find_parts(const JoinP& p, const RowInfo& x, int t, int head) {
    const AttnP& a = p.a;
    const int h = div_g(a, head), g = head - h * a.G;
    const int pf_units = a.pf_row_tiles * a.nkv * (cdiv(a.prefix_len, KU) + SEG_COST);
    const int positions = pf_units + x.own_units;
    const Cuts cuts(a, positions, CTAS, p.own.workers / CTAS);
    Parts r{0, 0, 0, 0, 0, 0};
    if (a.prefix_len > 0) {
        const int nt = cdiv(a.prefix_len, p.pf.keys), row = t * a.G + g, j = row / p.pf.mt, seg = p.pf_apart ? j * a.nkv + h : h * p.pf.row_tiles + j;
        const int cost = p.pf_apart ? TC_SEG_COST : SEG_COST, first = seg * (nt + cost) + cost;
        int c0, c1;
        if (p.pf_apart) {
            const int Wp = p.pf.row_tiles * a.nkv * (nt + cost);
            const Cut cp(Wp, p.pf.workers);
            c0 = cp.owner(first, Wp);
            c1 = cp.owner(first + nt - 1, Wp);
        } else {
            c0 = cuts.owner(first);
            c1 = cuts.owner(first + nt - 1);
        }
        r.n0 = c1 - c0 + 1;
        r.slot0 = seg + c0;
        r.row0 = row - j * p.pf.mt;
    }
    if (x.s.nt > 0) {
        const int row = x.i * a.G + g, js = h * x.s.qt + row / MT;
        const int first = pf_units + x.unit_b + js * (x.s.nt + SEG_COST) + SEG_COST;
        const int c0 = cuts.owner(first);
        r.n1 = cuts.owner(first + x.s.nt - 1) - c0 + 1;
        r.slot1 = a.pf_row_tiles * a.nkv + x.seg_b + js + c0;
        r.row1 = row % MT;
    }
    return r;
}

// Statistics and address of partial k of a head.
template <int HD> __device__ __forceinline__ void part(const JoinP& p, const Parts& r, int k, float2& ml, const float*& src) {
    ml = make_float2(-INFINITY, 0.0f);
    src = p.own.o;
    if (k < r.n0 + r.n1) {
        const PartSet& ps = k < r.n0 ? p.pf : p.own;
        const size_t at = k < r.n0 ? (size_t)(r.slot0 + k) * ps.mt + r.row0 : (size_t)(r.slot1 + k - r.n0) * ps.mt + r.row1;
        ml = ps.ml[at];
        src = ps.o + at * HD;
    }
}

template <int DPL, int HD> __device__ __forceinline__ void load_dims(const float* src, int lane, float (&v)[DPL]) {
    if constexpr (DPL == 4) {
        const float4 x = *(const float4*)(src + lane * 4);
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    } else if constexpr (DPL == 2) {
        const float2 x = *(const float2*)(src + lane * 2);
        v[0] = x.x; v[1] = x.y;
    } else {
        v[0] = HD >= 32 || lane < HD ? src[lane] : 0.0f;
    }
}

template <typename T, int DPL, int HD>
__device__ __forceinline__ void put_row(const JoinP& p, int t, int head, int lane, float M, float L, const float (&acc)[DPL]) {
    // a row that saw no key has a sum of 0; one that is not a number (a query's, or a partial result that
    // is missing) makes all of the row so
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    if (HD >= 32 || lane < HD) {
        T* dst = (T*)p.out + (long long)t * p.o_row + (long long)head * p.o_head + lane * DPL;
        if constexpr (DPL == 1) *dst = from_f32<T>(acc[0] * inv);
        else {
#pragma unroll
            for (int d = 0; d < DPL; d += 2) *(uint32_t*)(dst + d) = pack2<T>(acc[d] * inv, acc[d + 1] * inv);
        }
    }
    // ln(sum) = (M + log2 L) ln 2
    if (lane == 0 && p.lse) p.lse[(long long)t * (p.a.nkv * p.a.G) + head] = L == 0.0f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
}

// Many rows: a warp per row and four heads. Lane 8 g + k takes the statistics of partial k of
// head g (8 at a time), then the outputs are summed with each lane on its own dims: those of
// four heads and KB partials in flight together, and the first ahead of the weights. Bound: the
// chain of dependent loads (statistics, outputs) and the bytes of the partials.
template <typename T, int HD, int MT>
__global__ void __launch_bounds__(128, 4) prefix_attn_join_kernel(const __grid_constant__ JoinP p) {
    constexpr int DPL = HD >= 32 ? HD / 32 : 1, KU = unit_keys(HD), GH = 4, KB = DPL == 4 ? 4 : 8;
    const AttnP& a = p.a;
    const int lane = threadIdx.x & 31, nh = a.nkv * a.G, groups = cdiv(nh, GH);
    const int item = blockIdx.x * 4 + (threadIdx.x >> 5), t = item / groups, head0 = (item - t * groups) * GH;
    if (t >= a.n_rows) { pdl_wait(); return; }
    const RowInfo x = row_info<MT, KU, false>(a, t);
    pdl_release();
    if (!x.live) return;
    const int g = lane >> 3, k_l = lane & 7;
    Parts r{0, 0, 0, 0, 0, 0};
    if (head0 + g < nh) r = find_parts<MT, KU>(p, x, t, head0 + g);
    const int n = r.n0 + r.n1;
    int most = n;
#pragma unroll
    for (int o = 8; o < 32; o <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    float M = -INFINITY, L = 0.0f, acc[GH][DPL];                 // M, L: of head g
#pragma unroll
    for (int h = 0; h < GH; ++h)
#pragma unroll
        for (int d = 0; d < DPL; ++d) acc[h][d] = 0.0f;
    for (int base = 0; base < most; base += 8) {
        float2 ml;
        const float* src;
        part<HD>(p, r, base + k_l, ml, src);
        const int cnt = min(8, most - base);
        float wt = 0.0f;
        for (int k0 = 0; k0 < cnt; k0 += KB) {
            float v[KB][GH][DPL];
#pragma unroll
            for (int e = 0; e < KB; ++e)
#pragma unroll
                for (int h = 0; h < GH; ++h) {
                    const int from = h * 8 + min(k0 + e, 7);
                    const float* sp = (const float*)__shfl_sync(0xffffffffu, (unsigned long long)src, from);
                    const bool has = k0 + e < 8 && base + k0 + e < __shfl_sync(0xffffffffu, n, h * 8);
#pragma unroll
                    for (int d = 0; d < DPL; ++d) v[e][h][d] = 0.0f;
                    if (has) load_dims<DPL, HD>(sp, lane, v[e][h]);
                }
            if (k0 == 0) {
                float top = ml.x, sum;
#pragma unroll
                for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                top = fmaxf(M, top);
                const float to = top == -INFINITY ? 0.0f : top;  // no partial has seen a key
                const float f = ex2(M - to);
                wt = ex2(ml.x - to);
                sum = ml.y * wt;
#pragma unroll
                for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                M = top;
                L = L * f + sum;
#pragma unroll
                for (int h = 0; h < GH; ++h) {
                    const float fh = __shfl_sync(0xffffffffu, f, h * 8);
#pragma unroll
                    for (int d = 0; d < DPL; ++d) acc[h][d] *= fh;
                }
            }
#pragma unroll
            for (int e = 0; e < KB; ++e)
#pragma unroll
                for (int h = 0; h < GH; ++h) {                   // outputs that are not there are zeros
                    const float wk = __shfl_sync(0xffffffffu, wt, h * 8 + min(k0 + e, 7));
#pragma unroll
                    for (int d = 0; d < DPL; ++d) acc[h][d] += wk * v[e][h][d];
                }
        }
    }
#pragma unroll
    for (int h = 0; h < GH; ++h) {
        const float Mh = __shfl_sync(0xffffffffu, M, h * 8), Lh = __shfl_sync(0xffffffffu, L, h * 8);
        if (head0 + h < nh) put_row<T, DPL, HD>(p, t, head0 + h, lane, Mh, Lh, acc[h]);
    }
}

// Few rows, whose keys then lie with many workers: a block of eight warps per row and head, warp
// w taking the partials w, w + 8, ... All blocks are resident while the launch ahead still runs,
// so warp 0 finds the head's parts meanwhile, where the streams are few enough to sum (each word
// asked for once a block: by every warp, the words' L2 slice takes 3 us more on 16 streams).
template <typename T, int HD, int MT>
__global__ void __launch_bounds__(256, 4) prefix_attn_join_few_kernel(const __grid_constant__ JoinP p) {
    constexpr int DPL = HD >= 32 ? HD / 32 : 1, KU = unit_keys(HD), W = 8;
    const AttnP& a = p.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nh = a.nkv * a.G;
    const int t = blockIdx.x / nh, head = blockIdx.x - t * nh;
    __shared__ Parts s_parts;
    __shared__ bool s_live;
    const bool early = a.n_seq <= 256;
    if (!early) pdl_wait();
    if (warp == 0) {
        const RowInfo x = early ? row_info<MT, KU, true>(a, t) : row_info<MT, KU, false>(a, t);
        Parts y{0, 0, 0, 0, 0, 0};
        if (x.live) y = find_parts<MT, KU>(p, x, t, head);
        if (lane == 0) { s_parts = y; s_live = x.live; }
    }
    __syncthreads();
    const Parts r = s_parts;
    if (early) pdl_wait();
    pdl_release();
    if (!s_live) return;
    const int n = r.n0 + r.n1;
    float M = -INFINITY, L = 0.0f, acc[DPL];
#pragma unroll
    for (int d = 0; d < DPL; ++d) acc[d] = 0.0f;
    for (int base = warp; base < n; base += 32 * W) {
        float2 ml;
        const float* src;
        part<HD>(p, r, base + lane * W, ml, src);
        const int cnt = min(32, cdiv(n - base, W));
        float wt = 0.0f;
        for (int k0 = 0; k0 < cnt; k0 += 4) {
            float v[4][DPL];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                load_dims<DPL, HD>((const float*)__shfl_sync(0xffffffffu, (unsigned long long)src, min(k0 + e, cnt - 1)), lane, v[e]);
            if (k0 == 0) {                                       // the weights, with the first outputs on their way
                const float top = fmaxf(M, warp_max(ml.x));
                const float to = top == -INFINITY ? 0.0f : top;
                const float f = ex2(M - to);
                wt = ex2(ml.x - to);
                M = top;
                L = L * f + warp_sum(ml.y * wt);
#pragma unroll
                for (int d = 0; d < DPL; ++d) acc[d] *= f;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float wk = __shfl_sync(0xffffffffu, wt, min(k0 + e, cnt - 1));
                if (k0 + e >= cnt) wk = 0.0f;
#pragma unroll
                for (int d = 0; d < DPL; ++d) acc[d] += wk * v[e][d];
            }
        }
    }
    __shared__ float s_acc[W][HD + 2];                           // the block's warps, in a fixed order
    if (lane == 0) { s_acc[warp][HD] = M; s_acc[warp][HD + 1] = L; }
    if (HD >= 32 || lane < HD)
#pragma unroll
        for (int d = 0; d < DPL; ++d) s_acc[warp][lane * DPL + d] = acc[d];
    __syncthreads();
    if (warp > 0) return;
    for (int w = 1; w < W; ++w) {
        const float top = fmaxf(M, s_acc[w][HD]);
        const float to = top == -INFINITY ? 0.0f : top;          // no key seen
        const float f = ex2(M - to), fw = ex2(s_acc[w][HD] - to);
        M = top;
        L = L * f + s_acc[w][HD + 1] * fw;
        if (HD >= 32 || lane < HD)
#pragma unroll
            for (int d = 0; d < DPL; ++d) acc[d] = acc[d] * f + s_acc[w][lane * DPL + d] * fw;
    }
    put_row<T, DPL, HD>(p, t, head, lane, M, L, acc);
}

// ---- host -----------------------------------------------------------------------------------
struct HostPlan {
    int G, nb, warps;                   // blocks of 8 rows in an own segment, warps of a CTA
    PartSet own, pf;                    // pointers unset
    int early, head_start;              // as in AttnP
    bool pf_tc;                         // the prefix has a launch of its own, on tcgen05
    size_t off_own_ml, off_own_o, off_pf_ml, off_pf_o, bytes;
};

// Rings, queries and the line's streams (20 bytes each; OPS_MAX_SEQ of them leave room for four warps).
size_t attn_smem(int hd, int nb, int warps, int n_seq) {
    return 1024 + (size_t)warps * (ring_stages(hd) * 2 * unit_keys(hd) * hd * 2 + 8 * nb * hd * 2) + (size_t)(n_seq + 1) * 20;
}

size_t up(size_t x) { return (x + 255) & ~(size_t)255; }

// The prefix on tcgen05 fills an SM, its own keys' kernel another's: the first is kept to all SMs but
// PF_LEAVES, where the second starts beside it (the tensor cores are power-bound and lose less than
// their share of SMs, HBM would idle). While a CTA there takes one of its units an early CTA takes
// some OWN_PER_PF; what the early ones do not get through, all SMs share when the prefix is done.
// None / 36 left, us: 256 streams, 32 heads of 128, prefix 32768, own up to 600: 197 / 173 (216 / 202
// over hundreds of passes, when the clocks have fallen); 64, 16 heads, 8192, up to 200: 47 / 38; up to
// 4000: 102 / 92; 64 x 5 rows of 64 dims, 4097, up to 300: 41 / 38. With next to no own keys 64 dims
// lose (256, 16 heads, 32768, up to 8: 70 / 78; 128 dims: 93 / 91): the host does not see the lengths, and
// the number stays one. 16, 24, 32, 40 left, the first of these at 12 units: 219 (the early CTAs end
// last), 214, 182, 181 where 36 took 177. Where the early CTAs get through the whole line, the others
// start behind the prefix all the same, find nothing and end.
constexpr int PF_LEAVES = 36, OWN_PER_PF = 16;

std::atomic<int> g_polls{-1};           // limit of a wait set by a test, or negative

HostPlan host_plan(const z2b_prefix_attn_args& a) {
    HostPlan h{};
    const int nkv = a.kv->n_head_kv, hd = a.kv->head_dim;
    h.G = a.n_head / nkv;
    // rows of one stream and key head, on average: the smallest tile that holds them (32 streams of up
    // to 3000 keys, 16 rows each, tiles of 8 / 16: 30 / 27 us at head_dim 64, 40 / 37 at 128; 32 rows,
    // tiles of 8 / 32 at 64: 34 / 29, of 8 / 16 at 128: 51 / 38). head_dim 128 keeps 16: 32 rows do not
    // fit the registers, a second row tile finds its keys in L2
    const long long rows = (long long)((a.n_rows + a.n_seq - 1) / a.n_seq) * h.G;
    h.nb = rows <= 8 ? 1 : rows <= 16 || hd > 64 ? 2 : 4;
    h.warps = max_warps(hd);                                     // fewer where the line's streams need the room
    while (attn_smem(hd, h.nb, h.warps, a.n_seq) > MAX_SMEM) --h.warps;
    const long long R = (long long)a.n_rows * h.G;
    const int mt = 8 * h.nb;
    // The prefix on tcgen05 costs a launch and its filling (6 us), on the line a read of its keys per
    // row tile. Calls of 4 key heads, up to 8 own keys, head_dim 128, line / tcgen05 in us, R rows a key
    // head, prefixes of 512, 2048, 8192, 32768: R 16: 9 / 14, 11 / 14, 15 / 16, 27 / 29; R 32: 10 / 14,
    // 11 / 14, 17 / 16, 42 / 30; R 64: 11 / 15, 13 / 15, 25 / 17, 74 / 31; R 256: 17 / 27, 31 / 25, 84 / 36,
    // 293 / 52; and at head_dim 64: R 32: 8 / 12, 9 / 12, 13 / 14, 26 / 25; R 64: 10 / 12, 10 / 13, 17 / 15,
    // 46 / 25; R 256: 15 / 22, 23 / 19, 55 / 25, 180 / 38
    h.pf_tc = hd >= 64 && R >= 32 && (double)a.n_rows * a.n_head * a.prefix_len >= 2097152.0;
    const int pf_tiles = a.prefix_len > 0 && !h.pf_tc ? (int)((R + mt - 1) / mt) : 0;
    h.own = PartSet{nullptr, nullptr, mt, unit_keys(hd), CTAS * h.warps, 0, pf_tiles};
    const long long segs = ((R + mt - 1) / mt + a.n_seq + pf_tiles) * nkv;
    h.own.slots = (int)(segs + h.own.workers);
    h.pf = h.own;
    size_t n = up((size_t)2 * (a.n_seq + 1) * 4);
    h.off_own_ml = n; n += up((size_t)h.own.slots * mt * 8);
    h.off_own_o = n; n += up((size_t)h.own.slots * mt * hd * 4);
    if (h.pf_tc) {
        const int tiles = (int)((R + TC_ROWS - 1) / TC_ROWS);
        // a multiple of the row tiles, where that leaves few SMs idle: the row tiles are cut alike then,
        // so the CTAs that read the same keys do so at the same time and all but one find them in L2
        const int most = CTAS - PF_LEAVES, ctas = tiles <= most && most % tiles * 20 <= most ? most - most % tiles : most;
        h.early = CTAS - ctas;
        h.head_start = (int)((long long)OWN_PER_PF * tiles * nkv * ((a.prefix_len + TC_KEYS - 1) / TC_KEYS + TC_SEG_COST) / ctas);
        h.pf = PartSet{nullptr, nullptr, TC_ROWS, TC_KEYS, ctas, tiles * nkv + ctas, tiles};
        h.off_pf_ml = n; n += up((size_t)h.pf.slots * TC_ROWS * 8);
        h.off_pf_o = n; n += up((size_t)h.pf.slots * TC_ROWS * hd * 4);
    }
    h.bytes = n;
    return h;
}

template <typename T, int HD, int NB>
cudaError_t go_attn(const AttnP& p, const CUtensorMap& km, const CUtensorMap& vm, int warps, cudaStream_t s) {
    static std::atomic<uint64_t> opted{0};                       // devices whose shared-memory opt-in is done
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(opted.load(std::memory_order_relaxed) >> dev & 1)) {
        e = cudaFuncSetAttribute(prefix_attn_kernel<T, HD, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SMEM);
        if (e != cudaSuccess) return e;
        if (dev < 64) opted.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    return launch_pdl(prefix_attn_kernel<T, HD, NB>, dim3(CTAS), dim3(32 * warps),
                      attn_smem(HD, NB, warps, p.n_seq), s, p, km, vm);
}

template <typename T, int HD, int MT>
cudaError_t go_join(const JoinP& j, const z2b_prefix_attn_args& a, cudaStream_t s) {
    // a block per row and head, or a warp per four heads of a row: streams of 16 heads with up to 200
    // own keys, block / warp, in us: 32 items 8.9 / 11.4, 512: 11 / 13.3, 1024: 16.7 / 16.0, 2048: 28 / 19;
    // with up to 4000: 512: 30 / 36, 1024: 55 / 55, 2048: 101 / 93
    const long long items = (long long)a.n_rows * a.n_head;
    if (items <= 148 * 6) return launch_pdl(prefix_attn_join_few_kernel<T, HD, MT>, dim3((unsigned)items), dim3(256), 0, s, j);
    const long long warps = (long long)a.n_rows * ((a.n_head + 3) / 4);
    return launch_pdl(prefix_attn_join_kernel<T, HD, MT>, dim3((unsigned)((warps + 3) / 4)), dim3(128), 0, s, j);
}

template <typename T, int HD>
cudaError_t go_all(const z2b_prefix_attn_args& a, HostPlan h, cudaStream_t s) {
    const z2b_paged_kv& c = *a.kv;
    AttnP p{};
    p.q = a.q; p.q_row = a.q_row; p.q_head = a.q_head; p.table_stride = a.table_stride;
    p.row_off = a.row_off; p.seq_len = a.seq_len; p.table = a.page_table; p.prefix_pages = a.prefix_pages; p.err = a.err;
    p.n_rows = a.n_rows; p.n_seq = a.n_seq; p.nkv = c.n_head_kv; p.G = h.G; p.page_len = c.page_len; p.n_pages = c.n_pages;
    p.max_pages = a.max_pages; p.prefix_len = a.prefix_len;
    p.g_mul = (uint32_t)((0x100000000ull + h.G - 1) / h.G);
    const int polls = g_polls.load(std::memory_order_relaxed);
    p.polls = polls < 0 ? kMaxWaitPolls : (uint32_t)polls;
    p.scale2 = a.scale * 1.4426950408889634f;
    uint8_t* ws = (uint8_t*)a.workspace;
    p.plan = (int*)ws;
    CUtensorMap km, vm;
    cudaError_t e;
    if constexpr (HD >= 64) {
        if (h.pf_tc) {
            AttnP f = p;
            cut_boxes(f, TC_KEYS, HD);
            f.pf_row_tiles = h.pf.row_tiles;
            h.pf.ml = f.part_ml = (float2*)(ws + h.off_pf_ml);
            h.pf.o = f.part_o = (float*)(ws + h.off_pf_o);
            if (!make_page_map(&km, c.k, c, f) || !make_page_map(&vm, c.v, c, f)) return cudaErrorNotSupported;
            if ((e = launch_prefix_tc<T, HD>(f, km, vm, h.pf.workers, s)) != cudaSuccess) return e;
        }
    }
    cut_boxes(p, unit_keys(HD), HD);
    if (!make_page_map(&km, c.k, c, p) || !make_page_map(&vm, c.v, c, p))
        return cudaErrorNotSupported;
    p.pf_row_tiles = h.own.row_tiles;
    p.after_prefix = h.pf_tc;
    p.early = h.early;
    p.head_start = h.head_start;
    h.own.ml = p.part_ml = (float2*)(ws + h.off_own_ml);
    h.own.o = p.part_o = (float*)(ws + h.off_own_o);
    e = h.nb == 1 ? go_attn<T, HD, 1>(p, km, vm, h.warps, s) : cudaSuccess;
    if (h.nb == 2) e = go_attn<T, HD, 2>(p, km, vm, h.warps, s);
    if constexpr (HD <= 64)
        if (h.nb == 4) e = go_attn<T, HD, 4>(p, km, vm, h.warps, s);
    if (e != cudaSuccess) return e;
    const JoinP j{p, h.pf_tc ? h.pf : h.own, h.own, h.pf_tc, a.out, a.lse, a.o_row, a.o_head};
    if constexpr (HD <= 64)
        if (h.nb == 4) return go_join<T, HD, 32>(j, a, s);
    return h.nb == 1 ? go_join<T, HD, 8>(j, a, s) : go_join<T, HD, 16>(j, a, s);
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

extern "C" void z2b_test_attn_wait_polls(int polls) { z2b::g_polls.store(polls, std::memory_order_relaxed); }
