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
// Work split: a unit is KU keys of one segment (row tile x key head). All units form one line
// that is cut into equal contiguous ranges, one per worker, whatever the lengths; a worker
// leaves one partial result per segment it touches. Partial slots are segment + worker: going
// along the line every new partial advances one of the two, so slots never collide and their
// number is bounded by segments + workers. Nothing is accumulated by atomics: the same call
// gives the same bits.
//
// A worker is ONE WARP with a TMA ring of its own, so that no barrier ties warps together and
// the loads of a warp's next units stay in flight while it finishes a segment or fetches the
// next one's queries; together the rings of an SM hold 192 KB in flight.
#include "launch.cuh"
#include "ops.h"
#include "prefix_attn.cuh"

namespace z2b {
namespace {

// Warps of a CTA (one CTA per SM) and ring stages of a warp: 16, 8, 4 and 2 KB stages.
__host__ __device__ constexpr int max_warps(int hd) { return hd == 128 ? 6 : 8; }
__host__ __device__ constexpr int ring_stages(int hd) { return hd == 128 ? 2 : hd == 64 ? 3 : hd == 32 ? 6 : 8; }

// Shared-memory tile of KU rows of one key head: rows of RB bytes (at most 128: head_dim 128
// is two halves), 16-byte chunks XOR-swizzled as the TMA box writes them.
template <int HD> struct Tile {
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
    int pf_nt, pf_units, total_rows;
};
struct Seg {
    int h, j, seg, unit0, nt;          // key head, row tile, segment id, first unit, units
    int lo, n, klen, lim_max;          // first row, rows, keys, keys that the tile's last row sees
    const int* pages;
};

template <int MT> __device__ __forceinline__ Seg find_seg(const AttnP& p, const Line& ln, int u) {
    Seg g;
    if (u < ln.pf_units) {
        g.seg = u / ln.pf_nt;
        g.unit0 = g.seg * ln.pf_nt;
        g.nt = ln.pf_nt;
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
    const int qt = cdiv(g.n * p.G, MT), js = (v - r.x) / g.nt;
    g.seg = p.pf_row_tiles * p.nkv + r.y + js;
    g.unit0 = ln.pf_units + r.x + js * g.nt;
    g.h = js / qt;
    g.j = js % qt;
    const int last = min(g.n - 1, (g.j * MT + MT - 1) / p.G);
    g.lim_max = min(g.klen, g.klen - g.n + last + 1);
    g.pages = p.table + (long long)lo * p.table_stride;
    return g;
}

// M16 blocks of 16 rows per segment: 2 when a stream has more than 16 rows of a key head, so
// that its keys are read once for all of them.
template <typename T, int HD, int M16>
__global__ void __launch_bounds__(32 * max_warps(HD), 1) prefix_attn_kernel(const __grid_constant__ AttnP p,
                                                                           const __grid_constant__ CUtensorMap kmap,
                                                                           const __grid_constant__ CUtensorMap vmap) {
    constexpr int MT = 16 * M16, KS = HD / 16, NT = KU / 8, DT = HD / 8;
    constexpr int STAGE = 2 * Tile<HD>::BYTES, NS = ring_stages(HD);
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) uint64_t s_full[max_warps(HD)][NS];
    __shared__ int s_scan[2][max_warps(HD)];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    uint8_t* ring = smem + (size_t)warp * NS * STAGE;
    int4* s_rec = (int4*)(smem + (size_t)nw * NS * STAGE);
    int* s_len = (int*)(s_rec + p.n_seq + 1);
    uint64_t* full = s_full[warp];

    if (lane == 0) {
        for (int i = 0; i < NS; ++i) mbar_init(&full[i], 1);
        fence_mbar_init();
    }
    if (!p.after_prefix) { pdl_wait(); pdl_release(); }

    // ---- the line: offsets of every stream's units and segments, by a block scan
    {
        const int per = cdiv(p.n_seq, blockDim.x);
        const int b0 = min(p.n_seq, (int)threadIdx.x * per), b1 = min(p.n_seq, b0 + per);
        int su = 0, sg = 0;
        for (int b = b0; b < b1; ++b) {
            const SeqInfo s = seq_info<MT>(p, b);
            if (s.bad && blockIdx.x == 0 && p.err) atomicOr(p.err, Z2B_OPS_BAD_INDEX);
            s_rec[b] = make_int4(su, sg, s.lo, s.n);
            s_len[b] = s.len;
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
        for (int b = b0; b < b1; ++b) {
            s_rec[b].x += eu;
            s_rec[b].y += eg;
            if (blockIdx.x == 0) { p.plan[b] = s_rec[b].x; p.plan[p.n_seq + 1 + b] = s_rec[b].y; }
        }
        if (threadIdx.x == blockDim.x - 1) {
            s_rec[p.n_seq] = make_int4(eu + su, eg + sg, 0, 0);
            if (blockIdx.x == 0) { p.plan[p.n_seq] = eu + su; p.plan[2 * p.n_seq + 1] = eg + sg; }
        }
    }
    Line ln;
    ln.rec = s_rec;
    ln.len = s_len;
    ln.total_rows = max(0, min(p.n_rows, p.row_off[p.n_seq]));
    ln.pf_nt = cdiv(p.prefix_len, KU);
    ln.pf_units = p.pf_row_tiles * p.nkv * ln.pf_nt;
    __syncthreads();
    const long long W = (long long)ln.pf_units + s_rec[p.n_seq].x;
    const int workers = line_workers(W, gridDim.x * nw);
    const int me = warp * gridDim.x + blockIdx.x;                // few workers: one per SM first
    int u = 0, u1 = 0;
    if (me < workers) {
        u = (int)(W * me / workers);
        u1 = (int)(W * (me + 1) / workers);
    }

    // ---- the copies, NS units ahead of the products: one TMA box per lane
    const int nb = KU / p.box_rows, jobs = 2 * nb * Tile<HD>::HALVES;   // at most 16
    const int rb = lane % nb, half = lane / nb % Tile<HD>::HALVES, isv = lane / nb / Tile<HD>::HALVES;
    const uint32_t box_dst = smem_u32(ring) + isv * Tile<HD>::BYTES + half * (KU * Tile<HD>::RB) + rb * p.box_rows * Tile<HD>::RB;
    Seg gi;                            // segment of the next unit to copy
    gi.unit0 = -1;
    gi.nt = 0;
    int ui = u, issued = 0, page = 0;
    auto look_up = [&] {               // move ui to the next unit that some row sees; this lane's page of it
        for (; ui < u1; ui = gi.unit0 + gi.nt) {                 // keys only rise: behind an unseen unit all are
            if (ui >= gi.unit0 + gi.nt) gi = find_seg<MT>(p, ln, ui);
            if ((ui - gi.unit0) * KU < gi.lim_max) break;
        }
        if (ui >= u1) return;
        const int key = (ui - gi.unit0) * KU + rb * p.box_rows;
        page = p.n_pages;                                        // out of the view: the box fills with zeros
        if (lane < jobs && key < gi.klen) page = gi.pages[key / p.page_len];
    };
    auto copy = [&] {
        if (ui >= u1) return;
        const int st = issued % NS, key = (ui - gi.unit0) * KU + rb * p.box_rows;
        if (page < 0 || page > p.n_pages || (page == p.n_pages && lane < jobs && key < gi.klen)) {
            page = p.n_pages;
            if (p.err) atomicOr(p.err, Z2B_OPS_BAD_PAGE);
        }
        if (lane == 0) mbar_expect_tx(&full[st], STAGE);
        __syncwarp();
        if (lane < jobs)
            tma_load_4d(box_dst + st * STAGE, isv ? &vmap : &kmap, half * 64, gi.h, key % p.page_len, page, &full[st]);
        ++issued;
        ++ui;
        look_up();
    };
    look_up();
    for (int i = 0; i < NS; ++i) copy();

    int it = 0;
    bool dead = false;                                           // a wait ran out
    while (u < u1 && !dead) {
        const Seg g = find_seg<MT>(p, ln, u);
        const int end = min(u1, g.unit0 + g.nt);
        // this lane's rows: two of each block of 16
        int lim[M16][2], lim_min = 0x7fffffff;
        uint32_t qa[M16][KS][4];
#pragma unroll
        for (int mb = 0; mb < M16; ++mb)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int rr = g.j * MT + mb * 16 + (lane >> 2) + 8 * x, i = rr / p.G;
                const bool live = i < g.n;
                lim[mb][x] = !live ? 0 : u < ln.pf_units ? g.klen : min(g.klen, g.klen - g.n + i + 1);
                lim_min = min(lim_min, lim[mb][x]);
                const T* qp = (const T*)p.q + (long long)(g.lo + i) * p.q_row + (long long)(g.h * p.G + rr % p.G) * p.q_head + (lane & 3) * 2;
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    qa[mb][k][x] = live ? *(const uint32_t*)(qp + k * 16) : 0u;
                    qa[mb][k][x + 2] = live ? *(const uint32_t*)(qp + k * 16 + 8) : 0u;
                }
            }
        float o[M16][DT][4], m[M16][2], l[M16][2];
#pragma unroll
        for (int mb = 0; mb < M16; ++mb) {
            m[mb][0] = m[mb][1] = -INFINITY;
            l[mb][0] = l[mb][1] = 0.0f;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[mb][d][0] = o[mb][d][1] = o[mb][d][2] = o[mb][d][3] = 0.0f;
        }

        for (; u < end; ++u) {
            const int key0 = (u - g.unit0) * KU;
            if (key0 >= g.lim_max) { u = end; break; }           // no row of the tile sees the rest
            const int st = it % NS;
            dead = __any_sync(0xffffffffu, !mbar_wait(&full[st], (it / NS) & 1, p.err));
            if (dead) break;
            ++it;
            uint8_t* kt = ring + (size_t)st * STAGE;
            const uint32_t ks = smem_u32(kt), vs = ks + Tile<HD>::BYTES;
            const bool tail = key0 + KU > g.klen;
            if (tail) {
                // rows behind the last key may hold anything: zero times that is not zero
                for (int i = lane; i < KU * (HD / 8); i += 32)
                    if (key0 + i / (HD / 8) >= g.klen)
                        *(uint4*)(kt + Tile<HD>::BYTES + Tile<HD>::chunk(i / (HD / 8), i % (HD / 8))) = make_uint4(0, 0, 0, 0);
                __syncwarp();
            }
            float s[M16][NT][4];
#pragma unroll
            for (int mb = 0; mb < M16; ++mb)
#pragma unroll
                for (int n = 0; n < NT; ++n) s[mb][n][0] = s[mb][n][1] = s[mb][n][2] = s[mb][n][3] = 0.0f;
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int n = 0; n < NT; n += 2) {
                    uint32_t r[4];
                    ldsm4(ks + Tile<HD>::chunk(n * 8 + ((lane >> 4) << 3) + (lane & 7), 2 * k + ((lane >> 3) & 1)), r);
#pragma unroll
                    for (int mb = 0; mb < M16; ++mb) {
                        mma_t<T>(s[mb][n], qa[mb][k], r[0], r[1]);
                        mma_t<T>(s[mb][n + 1], qa[mb][k], r[2], r[3]);
                    }
                }
            const bool cut = key0 + KU > lim_min;
#pragma unroll
            for (int mb = 0; mb < M16; ++mb) {
                float mx[2] = {m[mb][0], m[mb][1]}, f[2], base[2];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[mb][n][e] *= p.scale2;
                        if (cut && key0 + n * 8 + (lane & 3) * 2 + (e & 1) >= lim[mb][e >> 1]) s[mb][n][e] = -INFINITY;
                        mx[e >> 1] = fmaxf(mx[e >> 1], s[mb][n][e]);
                    }
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 1));
                    mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 2));
                    base[x] = mx[x] == -INFINITY ? 0.0f : mx[x];         // a row that has seen no key yet
                    f[x] = ex2(m[mb][x] - base[x]);
                    m[mb][x] = mx[x];
                    l[mb][x] *= f[x];
                }
#pragma unroll
                for (int d = 0; d < DT; ++d) { o[mb][d][0] *= f[0]; o[mb][d][1] *= f[0]; o[mb][d][2] *= f[1]; o[mb][d][3] *= f[1]; }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[mb][n][e] = ex2(s[mb][n][e] - base[e >> 1]);
                        l[mb][e >> 1] += s[mb][n][e];
                    }
            }
#pragma unroll
            for (int k = 0; k < KU / 16; ++k) {
                // the probabilities rounded (to nearest) to the cache's type: the tensor core's operand
                uint32_t pa[M16][4];
#pragma unroll
                for (int mb = 0; mb < M16; ++mb) {
                    pa[mb][0] = pack2<T>(s[mb][2 * k][0], s[mb][2 * k][1]);
                    pa[mb][1] = pack2<T>(s[mb][2 * k][2], s[mb][2 * k][3]);
                    pa[mb][2] = pack2<T>(s[mb][2 * k + 1][0], s[mb][2 * k + 1][1]);
                    pa[mb][3] = pack2<T>(s[mb][2 * k + 1][2], s[mb][2 * k + 1][3]);
                }
#pragma unroll
                for (int d = 0; d < DT; d += 2) {
                    uint32_t r[4];
                    ldsm4t(vs + Tile<HD>::chunk(k * 16 + (lane & 15), d + (lane >> 4)), r);
#pragma unroll
                    for (int mb = 0; mb < M16; ++mb) {
                        mma_t<T>(o[mb][d], pa[mb], r[0], r[1]);
                        mma_t<T>(o[mb][d + 1], pa[mb], r[2], r[3]);
                    }
                }
            }
            if (tail) fence_proxy_async();                       // this stage's zeros before the next copy into it
            __syncwarp();
            copy();
        }
        if (dead) break;

        // ---- the segment's (or the range's) end: one partial result
        const int slot = g.seg + me;
        const bool fits = slot < p.max_slots;                    // false only for offsets that do not ascend
        if (!fits && p.err && lane == 0) atomicOr(p.err, Z2B_OPS_BAD_INDEX);
        const int rows = fits ? min(MT, g.n * p.G - g.j * MT) : 0;       // live rows of the tile
        float* po = p.part_o + (size_t)slot * MT * HD;
        float2* pm = p.part_ml + (size_t)slot * MT;
#pragma unroll
        for (int mb = 0; mb < M16; ++mb)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                float sum = l[mb][x];
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                const int row = mb * 16 + (lane >> 2) + 8 * x;
                if (row >= rows) continue;
#pragma unroll
                for (int d = 0; d < DT; ++d)
                    *(float2*)(po + (size_t)row * HD + d * 8 + (lane & 3) * 2) = make_float2(o[mb][d][2 * x], o[mb][d][2 * x + 1]);
                if ((lane & 3) == 0) pm[row] = make_float2(m[mb][x], sum);
            }
    }
    // after a wait that ran out, the copies in flight still land in this CTA's memory
    if (dead)
        for (int k = it; k < issued; ++k) mbar_wait(&full[k % NS], (k / NS) & 1, nullptr, 1u << 16);
    // beside a prefix launch: the join that follows waits for this grid, so this grid ends after that one
    if (p.after_prefix) { pdl_release(); pdl_wait(); }
}

// ---- join ---------------------------------------------------------------------------------
struct PartSet {                        // partial results of one launch
    const float* o;
    const float2* ml;
    int mt, keys, workers, max_slots, row_tiles;   // rows of a partial, keys of a unit, ..., row tiles of the prefix in it
};
struct JoinP {
    AttnP a;
    PartSet pf, own;                    // pf: the launch that took the prefix (own's when it took both)
    int pf_apart;
    void* out;
    float* lse;
    long long o_row, o_head;
};

// One warp per (row, head). The partials of both sets are numbered through; lanes take the
// statistics of 32 at a time, then the weighted outputs are summed with each lane on its own
// dims, four loads in flight. Bound: the chain of dependent loads (offsets, statistics, outputs).
template <typename T, int HD, int MT>
__global__ void __launch_bounds__(256) prefix_attn_join_kernel(const __grid_constant__ JoinP p) {
    constexpr int DPL = HD >= 32 ? HD / 32 : 1;
    const AttnP& a = p.a;
    const int lane = threadIdx.x & 31, nh = a.nkv * a.G;
    const int w = blockIdx.x * 8 + (threadIdx.x >> 5), t = w / nh, head = w % nh;
    const int h = head / a.G, g = head % a.G;
    pdl_wait();
    pdl_release();
    if (t >= a.n_rows) return;
    const int total = a.row_off[a.n_seq], own_units = a.plan[a.n_seq];
    const int b = warp_find_seq(a.row_off, a.n_seq, t);
    if (t >= total || b < 0) return;                             // padding stays as it is
    const int unit_b = a.plan[b], seg_b = a.plan[a.n_seq + 1 + b];
    const SeqInfo s = seq_info<MT>(a, b);
    const int i = t - s.lo;
    if (s.bad || i >= s.n) return;

    // the workers that hold this row's segment of the prefix, and of the stream's own rows
    const int pf_units = a.pf_row_tiles * a.nkv * cdiv(a.prefix_len, KU);
    const long long W = (long long)pf_units + own_units;
    int n0 = 0, n1 = 0, slot0 = 0, slot1 = 0, row0 = 0, row1 = 0;
    if (a.prefix_len > 0) {
        const int nt = cdiv(a.prefix_len, p.pf.keys), r = t * a.G + g, seg = h * p.pf.row_tiles + r / p.pf.mt;
        const long long Wp = p.pf_apart ? (long long)p.pf.row_tiles * a.nkv * nt : W, first = (long long)seg * nt;
        const int workers = line_workers(Wp, p.pf.workers), c0 = unit_owner(first, Wp, workers);
        n0 = unit_owner(first + nt - 1, Wp, workers) - c0 + 1;
        slot0 = seg + c0;
        row0 = r % p.pf.mt;
        if (slot0 + n0 > p.pf.max_slots) n0 = 0;
    }
    if (s.nt > 0) {
        const int r = i * a.G + g, js = h * s.qt + r / MT;
        const long long first = (long long)pf_units + unit_b + (long long)js * s.nt;
        const int workers = line_workers(W, p.own.workers), c0 = unit_owner(first, W, workers);
        n1 = unit_owner(first + s.nt - 1, W, workers) - c0 + 1;
        slot1 = a.pf_row_tiles * a.nkv + seg_b + js + c0;
        row1 = r % MT;
        if (slot1 + n1 > p.own.max_slots) n1 = 0;                // only for offsets that do not ascend
    }
    const int n = n0 + n1;
    float M = -INFINITY, L = 0.0f, acc[DPL];
#pragma unroll
    for (int d = 0; d < DPL; ++d) acc[d] = 0.0f;
    for (int base = 0; base < n; base += 32) {
        const int k = base + lane;
        float2 ml = make_float2(-INFINITY, 0.0f);
        const float* src = p.own.o;
        if (k < n) {
            const PartSet& ps = k < n0 ? p.pf : p.own;
            const size_t at = k < n0 ? (size_t)(slot0 + k) * ps.mt + row0 : (size_t)(slot1 + k - n0) * ps.mt + row1;
            ml = ps.ml[at];
            src = ps.o + at * HD;
        }
        const float top = fmaxf(M, warp_max(ml.x));
        if (top == -INFINITY) continue;
        const float f = ex2(M - top), wt = ex2(ml.x - top);
        M = top;
        L = L * f + warp_sum(ml.y * wt);
#pragma unroll
        for (int d = 0; d < DPL; ++d) acc[d] *= f;
        const int cnt = min(32, n - base);
        for (int k0 = 0; k0 < cnt; k0 += 4) {
            float v[4][DPL], wk[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int from = min(k0 + e, cnt - 1);
                const float* sp = (const float*)__shfl_sync(0xffffffffu, (unsigned long long)src, from);
                wk[e] = __shfl_sync(0xffffffffu, wt, from);
                if (k0 + e >= cnt) wk[e] = 0.0f;
                if (HD >= 32 || lane < HD) {
                    if constexpr (DPL == 4) {
                        const float4 x = *(const float4*)(sp + lane * 4);
                        v[e][0] = x.x; v[e][1] = x.y; v[e][2] = x.z; v[e][3] = x.w;
                    } else if constexpr (DPL == 2) {
                        const float2 x = *(const float2*)(sp + lane * 2);
                        v[e][0] = x.x; v[e][1] = x.y;
                    } else {
                        v[e][0] = sp[lane];
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int d = 0; d < DPL; ++d) acc[d] += wk[e] * v[e][d];
        }
    }
    const float inv = L > 0.0f ? 1.0f / L : 0.0f;
    if (HD >= 32 || lane < HD) {
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
    int G, m16, warps;                  // blocks of 16 rows in an own segment, warps of a CTA
    PartSet own, pf;                    // pointers unset
    bool pf_tc;                         // the prefix has a launch of its own, on tcgen05
    size_t off_own_ml, off_own_o, off_pf_ml, off_pf_o, bytes;
};

size_t up(size_t x) { return (x + 255) & ~(size_t)255; }

HostPlan host_plan(const z2b_prefix_attn_args& a) {
    HostPlan h{};
    const int nkv = a.kv->n_head_kv, hd = a.kv->head_dim;
    h.G = a.n_head / nkv;
    // rows of one stream and key head, on average; head_dim 128 keeps 16 (32 rows do not fit the
    // registers), a second row tile then finds its keys in L2
    h.m16 = hd > 64 || (long long)((a.n_rows + a.n_seq - 1) / a.n_seq) * h.G <= 16 ? 1 : 2;
    h.warps = a.n_seq > 1024 ? 4 : max_warps(hd);                // room for the line's streams beside the rings
    const long long R = (long long)a.n_rows * h.G;
    const int mt = 16 * h.m16;
    h.pf_tc = a.prefix_len > 0 && hd >= 64 && R > 64;
    const int pf_tiles = a.prefix_len > 0 && !h.pf_tc ? (int)((R + mt - 1) / mt) : 0;
    h.own = PartSet{nullptr, nullptr, mt, KU, 148 * h.warps, 0, pf_tiles};
    const long long segs = ((R + mt - 1) / mt + a.n_seq + pf_tiles) * nkv;
    h.own.max_slots = (int)(segs + h.own.workers);
    h.pf = h.own;
    size_t n = up((size_t)2 * (a.n_seq + 1) * 4);
    h.off_own_ml = n; n += up((size_t)h.own.max_slots * mt * 8);
    h.off_own_o = n; n += up((size_t)h.own.max_slots * mt * hd * 4);
    if (h.pf_tc) {
        const int tiles = (int)((R + TC_ROWS - 1) / TC_ROWS);
        h.pf = PartSet{nullptr, nullptr, TC_ROWS, TC_KEYS, 148, tiles * nkv + 148, tiles};
        h.off_pf_ml = n; n += up((size_t)h.pf.max_slots * TC_ROWS * 8);
        h.off_pf_o = n; n += up((size_t)h.pf.max_slots * TC_ROWS * hd * 4);
    }
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

template <typename T, int HD, int M16>
cudaError_t go_attn(const AttnP& p, const CUtensorMap& km, const CUtensorMap& vm, int warps, cudaStream_t s) {
    constexpr int STAGE = 2 * Tile<HD>::BYTES;
    constexpr int most = 224 * 1024;
    const size_t smem = 1024 + (size_t)warps * ring_stages(HD) * STAGE + (size_t)(p.n_seq + 1) * 20;
    static std::atomic<uint64_t> opted{0};                       // devices whose shared-memory opt-in is done
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(opted.load(std::memory_order_relaxed) >> dev & 1)) {
        e = cudaFuncSetAttribute(prefix_attn_kernel<T, HD, M16>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        if (e != cudaSuccess) return e;
        if (dev < 64) opted.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    return launch_pdl(prefix_attn_kernel<T, HD, M16>, dim3(148), dim3(32 * warps), smem, s, p, km, vm);
}

template <typename T, int HD>
cudaError_t go_all(const z2b_prefix_attn_args& a, HostPlan h, cudaStream_t s) {
    const z2b_paged_kv& c = *a.kv;
    AttnP p{};
    p.q = a.q; p.q_row = a.q_row; p.q_head = a.q_head; p.table_stride = a.table_stride;
    p.row_off = a.row_off; p.seq_len = a.seq_len; p.table = a.page_table; p.prefix_pages = a.prefix_pages; p.err = a.err;
    p.n_rows = a.n_rows; p.n_seq = a.n_seq; p.nkv = c.n_head_kv; p.G = h.G; p.page_len = c.page_len; p.n_pages = c.n_pages;
    p.max_pages = a.max_pages; p.prefix_len = a.prefix_len;
    const int page_pow2 = c.page_len & -c.page_len;
    p.scale2 = a.scale * 1.4426950408889634f;
    uint8_t* ws = (uint8_t*)a.workspace;
    p.plan = (int*)ws;
    CUtensorMap km, vm;
    cudaError_t e;
    if constexpr (HD >= 64) {
        if (h.pf_tc) {
            AttnP f = p;
            f.box_rows = page_pow2 > TC_KEYS ? TC_KEYS : page_pow2;
            f.pf_row_tiles = h.pf.row_tiles;
            f.max_slots = h.pf.max_slots;
            h.pf.ml = f.part_ml = (float2*)(ws + h.off_pf_ml);
            h.pf.o = f.part_o = (float*)(ws + h.off_pf_o);
            if (!make_map(&km, c.k, c, f.box_rows, 64) || !make_map(&vm, c.v, c, f.box_rows, 64)) return cudaErrorNotSupported;
            if ((e = launch_prefix_tc<T, HD>(f, km, vm, h.pf.workers, s)) != cudaSuccess) return e;
        }
    }
    p.box_rows = page_pow2 > KU ? KU : page_pow2;
    if (!make_map(&km, c.k, c, p.box_rows, Tile<HD>::INNER) || !make_map(&vm, c.v, c, p.box_rows, Tile<HD>::INNER))
        return cudaErrorNotSupported;
    p.pf_row_tiles = h.own.row_tiles;
    p.after_prefix = h.pf_tc;
    p.max_slots = h.own.max_slots;
    h.own.ml = p.part_ml = (float2*)(ws + h.off_own_ml);
    h.own.o = p.part_o = (float*)(ws + h.off_own_o);
    if constexpr (HD > 64) e = go_attn<T, HD, 1>(p, km, vm, h.warps, s);
    else e = h.m16 == 1 ? go_attn<T, HD, 1>(p, km, vm, h.warps, s) : go_attn<T, HD, 2>(p, km, vm, h.warps, s);
    if (e != cudaSuccess) return e;
    const JoinP j{p, h.pf_tc ? h.pf : h.own, h.own, h.pf_tc, a.out, a.lse, a.o_row, a.o_head};
    const dim3 grid((unsigned)(((long long)a.n_rows * a.n_head + 7) / 8));
    if constexpr (HD <= 64)
        if (h.m16 == 2) return launch_pdl(prefix_attn_join_kernel<T, HD, 32>, grid, dim3(256), 0, s, j);
    return launch_pdl(prefix_attn_join_kernel<T, HD, 16>, grid, dim3(256), 0, s, j);
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
