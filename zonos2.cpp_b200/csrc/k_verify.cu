// k_verify.cu — verification of drafted frames against the target's probabilities
// (sm_100a; include/z2b_ops.h).
//
// A drafted token x of frame i, codebook c is kept when u q(x) < p(x). The run ends at the
// first frame with a refused token; there each refused token becomes a draw from
// max(p - q, 0), and after a run without refusals one more frame is drawn from p. A draw is
// the first v whose running sum exceeds r * total.
//
// Bound: latency for frame-sized vocabularies, else the bytes of one row of p and of q per
// drawn token: the kept tokens cost one gathered value each, and no other row is read. One
// cluster of CTAs takes one (stream, codebook): every CTA finds the run's end for itself
// (a handful of gathers), then the row is split over the cluster, each warp summing one
// contiguous share; the totals are exchanged through distributed shared memory, and the
// one CTA whose range holds the target walks the one warp's share that does.
//
// The sums are f64 over exact differences of the inputs, so where they are split does not
// move a draw except within 1e-15 of a border; u * q and the comparison are f64 as well.
#include "launch.cuh"
#include "ops.cuh"
#include "ops.h"

#include <cooperative_groups.h>

namespace z2b {
namespace {

namespace cg = cooperative_groups;

constexpr int WARPS = 8, THREADS = 32 * WARPS;
constexpr int MAX_CLUSTER = 8;          // CTAs per row: the portable cluster size

struct VerifyP {
    z2b_verify_args a;
    int cluster;
};

// Probability mass left for a draw at v: p, less q where there is one, less all of it at
// the drafted token where the draft had no probabilities. Not-a-number counts as zero
// (fmax returns its other operand).
template <typename T, bool HAS_Q, bool SUB>
__device__ __forceinline__ double left_at(const T* __restrict__ p, const T* __restrict__ q, int v, int drafted) {
    const double x = (double)to_f32(p[v]);
    if constexpr (SUB && HAS_Q) return fmax(x - (double)to_f32(q[v]), 0.0);
    else if constexpr (SUB) return v == drafted ? fmax(x - 1.0, 0.0) : fmax(x, 0.0);
    else return fmax(x, 0.0);
}

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

struct DrawShared {
    double warp_tot[WARPS];
    double cta_tot;                     // read by the cluster's other CTAs
    double scan[WARPS];
    int found, last;
};

// The drawn token, or -1 when the mass is zero everywhere. Called by every thread of the
// cluster; all get the same `total`, only the CTA whose range holds the target a token
// (the others -2).
template <typename T, bool HAS_Q, bool SUB>
__device__ int draw(const T* p, const T* q, int V, int drafted, double r, int rank, int n_cta, DrawShared& sh) {
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int shares = n_cta * WARPS;
    const int per = (V + shares - 1) / shares;
    const int share = rank * WARPS + w;
    const int lo = min(V, share * per), hi = min(V, lo + per);
    double s0 = 0.0, s1 = 0.0;
    int v = lo + lane;
    for (; v + 7 * 32 < hi; v += 8 * 32) {                       // eight loads of each row in flight
        double x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = left_at<T, HAS_Q, SUB>(p, q, v + j * 32, drafted);
#pragma unroll
        for (int j = 0; j < 8; j += 2) { s0 += x[j]; s1 += x[j + 1]; }
    }
#pragma unroll 4
    for (; v < hi; v += 32) s0 += left_at<T, HAS_Q, SUB>(p, q, v, drafted);
    const double ws = warp_sum_f64(s0 + s1);
    __syncthreads();                                             // sh from an earlier draw
    if (lane == 0) sh.warp_tot[w] = ws;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int i = 0; i < WARPS; ++i) t += sh.warp_tot[i];
        sh.cta_tot = t;
        sh.found = 0x7fffffff;
        sh.last = -1;
    }
    cg::cluster_group cl = cg::this_cluster();
    if (n_cta > 1) cl.sync(); else __syncthreads();
    double base = 0.0, total = 0.0;
    int owner = -1, tail = -1;                                   // the range that holds the target
    double cta[MAX_CLUSTER];
#pragma unroll
    for (int i = 0; i < MAX_CLUSTER; ++i) {
        cta[i] = i >= n_cta ? 0.0 : n_cta > 1 ? *cl.map_shared_rank(&sh.cta_tot, i) : sh.cta_tot;
        total += cta[i];
    }
    if (n_cta > 1) cl.sync();                                    // no CTA leaves or reuses its total before all read it
    if (!(total > 0.0)) return -1;
    const double target = r * total;
    double run = 0.0;
#pragma unroll
    for (int i = 0; i < MAX_CLUSTER; ++i) {
        if (cta[i] > 0.0) tail = i;
        if (owner < 0 && run + cta[i] > target) { owner = i; base = run; }
        run += cta[i];
    }
    const bool past = owner < 0;                                 // rounding left the target at the total
    if (past) owner = tail;
    if (owner != rank) return -2;
    int share_w = -1, tail_w = 0;
    double run_w = base;
    for (int i = 0; i < WARPS; ++i) {
        if (sh.warp_tot[i] > 0.0) tail_w = i;
        if (share_w < 0 && !past && run_w + sh.warp_tot[i] > target) { share_w = i; base = run_w; }
        run_w += sh.warp_tot[i];
    }
    const bool past_w = share_w < 0;
    if (past_w) share_w = tail_w;
    // the whole CTA walks that share: a run of consecutive entries per thread
    const int slo = min(V, (rank * WARPS + share_w) * per), shi = min(V, slo + per);
    const int each = (shi - slo + THREADS - 1) / THREADS;
    const int tlo = min(shi, slo + (int)threadIdx.x * each), thi = min(shi, tlo + each);
    double mine = 0.0;
    int last = -1;
    for (int i = tlo; i < thi; ++i) {
        const double x = left_at<T, HAS_Q, SUB>(p, q, i, drafted);
        if (x > 0.0) last = i;
        mine += x;
    }
    double inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
    }
    if (lane == 31) sh.scan[w] = inc;
    __syncthreads();
    double before = past_w ? 0.0 : base;
    for (int i = 0; i < w; ++i) before += sh.scan[i];
    before += inc - mine;
    if (last >= 0) atomicMax(&sh.last, last);
    if (!past_w && mine > 0.0 && before + mine > target) {
        double c = before;
        for (int i = tlo; i < thi; ++i) {
            c += left_at<T, HAS_Q, SUB>(p, q, i, drafted);
            if (c > target) { atomicMin(&sh.found, i); break; }
        }
    }
    __syncthreads();
    // rounding may leave the target at the very end of the share: its last entry with mass
    return sh.found != 0x7fffffff ? sh.found : sh.last;
}

template <typename T, bool HAS_Q>
__global__ void __launch_bounds__(THREADS) verify_kernel(const __grid_constant__ VerifyP P) {
    const z2b_verify_args& a = P.a;
    __shared__ DrawShared sh;
    __shared__ int s_end;
    const int n_cta = P.cluster, rank = blockIdx.x % n_cta;
    const int item = blockIdx.x / n_cta, b = item / a.n_codebooks, c = item % a.n_codebooks;
    const int C = a.n_codebooks, N = a.max_draft, V = a.vocab;
    pdl_wait();
    pdl_release();
    int n = a.n_draft ? a.n_draft[b] : N;
    if (n < 0 || n > N) {
        if (threadIdx.x == 0 && a.err) atomicOr(a.err, Z2B_OPS_BAD_INDEX);
        n = n < 0 ? 0 : N;
    }
    const int32_t* draft = a.draft + (long long)b * N * C;
    const T* p = (const T*)a.p + (long long)b * a.p_seq;
    const T* q = HAS_Q ? (const T*)a.q + (long long)b * a.q_seq : nullptr;
    auto kept = [&](int f, int cb) {
        const int x = draft[f * C + cb];
        if (x < 0 || x >= V) {
            if (a.err) atomicOr(a.err, Z2B_OPS_BAD_INDEX);
            return false;
        }
        const double u = a.u_accept[((long long)b * N + f) * C + cb];
        const double pt = (double)to_f32(p[f * a.p_frame + cb * a.p_book + x]);
        const double qt = HAS_Q ? (double)to_f32(q[f * a.q_frame + cb * a.q_book + x]) : 1.0;
        return u * qt < pt;
    };
    if (threadIdx.x == 0) s_end = n;
    __syncthreads();
    for (int i = threadIdx.x; i < n * C; i += THREADS)
        if (!kept(i / C, i % C)) atomicMin(&s_end, i / C);
    __syncthreads();
    const int end = s_end;
    int32_t* out = a.tokens + (long long)b * (N + 1) * C + c;
    if (rank == 0) {
        for (int f = threadIdx.x; f <= N; f += THREADS)
            if (f != end) out[f * C] = f < end ? draft[f * C + c] : -1;
        if (c == 0 && threadIdx.x == 0) a.n_accepted[b] = end;
    }
    // uniform over the cluster from here on
    const int x = end < n ? draft[end * C + c] : -1;
    if (end < n && kept(end, c)) {
        if (rank == 0 && threadIdx.x == 0) out[end * C] = x;
        return;
    }
    const double r = a.u_draw[((long long)b * (N + 1) + end) * C + c];
    const T* pr = p + end * a.p_frame + c * a.p_book;
    int tok = -1;
    if (end < n) {
        const T* qr = HAS_Q ? q + end * a.q_frame + c * a.q_book : nullptr;
        tok = draw<T, HAS_Q, true>(pr, qr, V, x, r, rank, n_cta, sh);
    }
    if (tok == -1) tok = draw<T, HAS_Q, false>(pr, nullptr, V, -1, r, rank, n_cta, sh);
    // -1: a row without any mass has no token; its first CTA says so
    if (threadIdx.x == 0 && (tok >= 0 || (tok == -1 && rank == 0))) out[end * C] = tok;
}

template <typename T> cudaError_t go(const VerifyP& P, bool has_q, dim3 grid, cudaStream_t s) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(THREADS);
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = P.cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    return has_q ? cudaLaunchKernelEx(&cfg, verify_kernel<T, true>, P) : cudaLaunchKernelEx(&cfg, verify_kernel<T, false>, P);
}

}  // namespace

cudaError_t launch_verify(const z2b_verify_args& a, cudaStream_t s) {
    VerifyP P{a, 1};
    // CTAs per row: enough that one CTA's share is a few thousand entries, while the
    // clusters of all rows still fit the device about twice over (148 SMs)
    const long long items = (long long)a.n_seq * a.n_codebooks;
    while (P.cluster < MAX_CLUSTER && a.vocab / P.cluster > 2048 && items * P.cluster < 296) P.cluster *= 2;
    const dim3 grid((unsigned)(items * P.cluster));
    if (a.type == Z2B_TYPE_F32) return go<float>(P, a.q != nullptr, grid, s);
    if (a.type == Z2B_TYPE_F16) return go<__half>(P, a.q != nullptr, grid, s);
    return go<__nv_bfloat16>(P, a.q != nullptr, grid, s);
}

}  // namespace z2b
