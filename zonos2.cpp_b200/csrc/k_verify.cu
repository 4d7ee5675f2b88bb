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
// CTA, or a cluster of them for large vocabularies, takes one (stream, codebook): every CTA
// finds the run's end for itself (a handful of gathers). Then
//   small rows: a thread holds up to EACH consecutive entries; one block scan finds the draw (1026
//   entries: 3.0 us, where a first pass for the sum and a second for the draw took 4.6);
//   large rows: the row is split over the cluster, each warp summing one contiguous share with
//   lanes side by side; the totals are exchanged through distributed shared memory, and the one
//   CTA whose range holds the target scans the one warp's share that does.
//
// The sums are f64 over exact differences of the inputs, so where they are split does not
// move a draw except within 1e-15 of a border, and never to an entry without mass; u * q and the
// comparison are f64 as well.
#include "launch.cuh"
#include "ops.cuh"
#include "ops.h"

#include <cooperative_groups.h>

namespace z2b {
namespace {

namespace cg = cooperative_groups;

constexpr int MAX_CLUSTER = 8;          // CTAs per row: the portable cluster size
constexpr int EACH = 8;                 // entries of a small row that a thread holds
constexpr int SMALL_WARPS = 8, LARGE_WARPS = 12;
// A draw's answer where it is no token: the row has no mass at all, or another CTA has the token.
constexpr int NO_MASS = -1, ELSEWHERE = -2;

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

// A number drawn with, in [0, 1]: below, the first token with mass is drawn, else out of range the last.
__device__ __forceinline__ double unit(double r) { return r < 0.0 ? 0.0 : r < 1.0 ? r : 1.0; }

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <int WARPS> struct DrawShared {
    double warp_tot[WARPS];
    double cta[2][MAX_CLUSTER];         // the cluster's totals, each CTA's pushed by itself; one set per draw
    double scan[WARPS];
    int found, last;
};

// The drawn token of a row of at most 32 WARPS EACH entries, or NO_MASS. Called by the
// whole CTA; all threads get it.
template <typename T, bool HAS_Q, bool SUB, int WARPS>
__device__ int draw_small(const T* p, const T* q, int V, int drafted, double r, DrawShared<WARPS>& sh) {
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, each = (V + 32 * WARPS - 1) / (32 * WARPS);
    const int lo = min(V, (int)threadIdx.x * each);
    double x[EACH], mine = 0.0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) x[i] = i < each && lo + i < V ? left_at<T, HAS_Q, SUB>(p, q, lo + i, drafted) : 0.0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) mine += x[i];
    double inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
    }
    __syncthreads();                                             // sh from an earlier draw
    if (lane == 31) sh.warp_tot[w] = inc;
    if (threadIdx.x == 0) { sh.found = 0x7fffffff; sh.last = -1; }
    __syncthreads();
    double before = 0.0, total = 0.0;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
        if (i == w) before = total;
        total += sh.warp_tot[i];
    }
    if (!(total > 0.0)) return NO_MASS;
    const double target = unit(r) * total;
    before += inc - mine;
    if (mine > 0.0) {
        int last = -1, first = 0x7fffffff;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            before += x[i];
            if (!(x[i] > 0.0)) continue;                         // rounding may leave `before` past the target here already
            last = lo + i;
            if (before > target && first == 0x7fffffff) first = lo + i;
        }
        if (first != 0x7fffffff) atomicMin(&sh.found, first);
        else atomicMax(&sh.last, last);                          // rounding may leave the target at the total
    }
    __syncthreads();
    return sh.found != 0x7fffffff ? sh.found : sh.last;
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// The drawn token. Called by every thread of the cluster, all of whose CTAs have
// started. NO_MASS comes from the cluster's total alone, so that its CTAs agree whether another draw
// (with its barriers) follows; else the CTA whose range holds the target gets the token and the others
// ELSEWHERE. That range has mass: the target is at least 0, so a range whose sum takes the running
// total past it adds to it. `set`: 0 for a cluster's first draw, 1 for its second.
template <typename T, bool HAS_Q, bool SUB, int WARPS>
__device__ int draw_large(const T* p, const T* q, int V, int drafted, double r, int rank, int n_cta, int set, DrawShared<WARPS>& sh) {
    constexpr int THREADS = 32 * WARPS;
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int shares = n_cta * WARPS;
    const int per = (V + shares - 1) / shares;
    const int share = rank * WARPS + w;
    const int lo = min(V, share * per), hi = min(V, lo + per);
    double s0 = 0.0, s1 = 0.0;
    for (int v = lo + lane; v < hi; v += 8 * 32) {               // eight loads of each row in flight
        double x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = v + j * 32 < hi ? left_at<T, HAS_Q, SUB>(p, q, v + j * 32, drafted) : 0.0;
#pragma unroll
        for (int j = 0; j < 8; j += 2) { s0 += x[j]; s1 += x[j + 1]; }
    }
    const double ws = warp_sum_f64(s0 + s1);
    __syncthreads();                                             // sh from an earlier draw
    if (lane == 0) sh.warp_tot[w] = ws;
    __syncthreads();
    if (threadIdx.x < n_cta) {                                   // thread i hands this CTA's total to CTA i
        double t = 0.0;
        for (int i = 0; i < WARPS; ++i) t += sh.warp_tot[i];
        if (n_cta > 1) *cg::this_cluster().map_shared_rank(&sh.cta[set][rank], threadIdx.x) = t;
        else sh.cta[set][0] = t;
        if (threadIdx.x == 0) { sh.found = 0x7fffffff; sh.last = -1; }
    }
    if (n_cta > 1) { cluster_arrive(); cluster_wait(); } else __syncthreads();
    double base = 0.0, total = 0.0;
    int owner = -1, tail = -1;                                   // the range that holds the target
    double cta[MAX_CLUSTER];
#pragma unroll
    for (int i = 0; i < MAX_CLUSTER; ++i) {
        cta[i] = i < n_cta ? sh.cta[set][i] : 0.0;
        total += cta[i];
    }
    if (!(total > 0.0)) return NO_MASS;
    const double target = unit(r) * total;
    double run = 0.0;
#pragma unroll
    for (int i = 0; i < MAX_CLUSTER; ++i) {
        if (cta[i] > 0.0) tail = i;
        if (owner < 0 && run + cta[i] > target) { owner = i; base = run; }
        run += cta[i];
    }
    const bool past = owner < 0;                                 // rounding left the target at the total
    if (past) owner = tail;
    if (owner != rank) return ELSEWHERE;
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
    double mine = 0.0, x[EACH];
    int last = -1;
#pragma unroll
    for (int i = 0; i < EACH; ++i) x[i] = tlo + i < thi ? left_at<T, HAS_Q, SUB>(p, q, tlo + i, drafted) : 0.0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        if (x[i] > 0.0) last = tlo + i;
        mine += x[i];
    }
    for (int i = tlo + EACH; i < thi; ++i) {                     // vocabularies beyond what the threads hold
        const double y = left_at<T, HAS_Q, SUB>(p, q, i, drafted);
        if (y > 0.0) last = i;
        mine += y;
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
        int first = 0x7fffffff;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            before += x[i];
            if (x[i] > 0.0 && before > target && first == 0x7fffffff) first = tlo + i;
        }
        for (int i = tlo + EACH; i < thi && first == 0x7fffffff; ++i) {
            const double y = left_at<T, HAS_Q, SUB>(p, q, i, drafted);
            before += y;
            if (y > 0.0 && before > target) first = i;
        }
        atomicMin(&sh.found, first);
    }
    __syncthreads();
    // rounding may leave the target at the very end of the share: its last entry with mass
    return sh.found != 0x7fffffff ? sh.found : sh.last;
}

template <typename T, bool HAS_Q, int WARPS>
__global__ void __launch_bounds__(32 * WARPS) verify_kernel(const __grid_constant__ VerifyP P) {
    constexpr int THREADS = 32 * WARPS;
    const z2b_verify_args& a = P.a;
    __shared__ DrawShared<WARPS> sh;
    __shared__ int s_end;
    const int n_cta = P.cluster, rank = blockIdx.x % n_cta;
    const int item = blockIdx.x / n_cta, b = item / a.n_codebooks, c = item % a.n_codebooks;
    const int C = a.n_codebooks, N = a.max_draft, V = a.vocab;
    if (n_cta > 1) cluster_arrive();                             // waited for before the first total is handed over
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
        const double u = a.u_accept[((long long)b * N + f) * C + cb];
        if (f >= n) return true;                                 // not drafted: decides nothing
        if (x < 0 || x >= V) {
            if (a.err) atomicOr(a.err, Z2B_OPS_BAD_INDEX);
            return false;
        }
        const double pt = (double)to_f32(p[f * a.p_frame + cb * a.p_book + x]);
        const double qt = HAS_Q ? (double)to_f32(q[f * a.q_frame + cb * a.q_book + x]) : 1.0;
        return u * qt < pt;
    };
    if (threadIdx.x == 0) s_end = n;
    __syncthreads();
    for (int i = threadIdx.x; i < N * C; i += THREADS)           // all N: not waiting for n to load the drafts
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
    const bool keep = end < n && kept(end, c);
    if (n_cta > 1) cluster_wait();
    if (keep) {
        if (rank == 0 && threadIdx.x == 0) out[end * C] = x;
        return;
    }
    const double r = a.u_draw[((long long)b * (N + 1) + end) * C + c];
    const T* pr = p + end * a.p_frame + c * a.p_book;
    const T* qr = HAS_Q && end < n ? q + end * a.q_frame + c * a.q_book : nullptr;
    int tok = NO_MASS;
    if constexpr (WARPS == SMALL_WARPS) {
        if (end < n) tok = draw_small<T, HAS_Q, true, WARPS>(pr, qr, V, x, r, sh);
        if (tok == NO_MASS) tok = draw_small<T, HAS_Q, false, WARPS>(pr, nullptr, V, -1, r, sh);
    } else {
        if (end < n) tok = draw_large<T, HAS_Q, true, WARPS>(pr, qr, V, x, r, rank, n_cta, 0, sh);
        if (tok == NO_MASS) tok = draw_large<T, HAS_Q, false, WARPS>(pr, nullptr, V, -1, r, rank, n_cta, 1, sh);
    }
    // looked at last: the rows are not to wait for it
    if (rank == 0 && threadIdx.x == 0 && a.err && !(r >= 0.0 && r < 1.0)) atomicOr(a.err, Z2B_OPS_BAD_INDEX);
    // a row without any mass has no token (-1); its first CTA says so
    if (threadIdx.x == 0 && (tok >= 0 || (tok == NO_MASS && rank == 0))) out[end * C] = tok;
}

template <typename T, int WARPS> cudaError_t go(const VerifyP& P, bool has_q, dim3 grid, cudaStream_t s) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(32 * WARPS);
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = P.cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = P.cluster > 1 ? 2 : 1;
    return has_q ? cudaLaunchKernelEx(&cfg, verify_kernel<T, true, WARPS>, P) : cudaLaunchKernelEx(&cfg, verify_kernel<T, false, WARPS>, P);
}

template <typename T> cudaError_t go_type(VerifyP P, cudaStream_t s) {
    const z2b_verify_args& a = P.a;
    const long long items = (long long)a.n_seq * a.n_codebooks;
    if (a.vocab <= 32 * SMALL_WARPS * EACH) return go<T, SMALL_WARPS>(P, a.q != nullptr, dim3((unsigned)items), s);
    // CTAs per row: enough that one CTA's share is a few thousand entries, while all clusters
    // are resident together (two CTAs an SM, 148 SMs). One CTA / a cluster by this rule, in us:
    // 1 stream, vocabulary 10007: 6.6 / 5.4, 50021: 14.7 / 6.4, 200003: 42 / 9.2; 32 streams, 10007:
    // 6.6 / 5.7, 50021: 15 / 8.4; 128 streams, 50021: 26 / 17.5, 10007: 6.8 / 7.5 (four each: 12)
    while (P.cluster < MAX_CLUSTER && a.vocab / P.cluster > 4096 && items * P.cluster * 2 <= 296) P.cluster *= 2;
    return go<T, LARGE_WARPS>(P, a.q != nullptr, dim3((unsigned)(items * P.cluster)), s);
}

}  // namespace

cudaError_t launch_verify(const z2b_verify_args& a, cudaStream_t s) {
    const VerifyP P{a, 1};
    return a.type == Z2B_TYPE_F32 ? go_type<float>(P, s) : a.type == Z2B_TYPE_F16 ? go_type<__half>(P, s) : go_type<__nv_bfloat16>(P, s);
}

}  // namespace z2b
