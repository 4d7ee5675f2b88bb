// capi_ops.cpp — extern "C" entry points declared in include/z2b_ops.h: argument checks and
// the device switch around the launches of ops.h.
#include "ops.h"
#include "runtime.h"

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <initializer_list>
#include <string>
#include <utility>

using namespace z2b;

namespace {

// The calling thread's device, put back when the call ends.
struct DeviceGuard {
    int prev = -1;
    cudaError_t rc;
    explicit DeviceGuard(int device) {
        rc = cudaGetDevice(&prev);
        if (rc == cudaSuccess && prev != device) rc = cudaSetDevice(device);
        else if (rc == cudaSuccess) prev = -1;
    }
    ~DeviceGuard() { if (prev >= 0) cudaSetDevice(prev); }
};

// No exception leaves a C entry point, not even for want of memory for the message.
int fail(int rc, const char* what, const char* more = "") {
    try { set_error(std::string(what) + more); } catch (...) {}
    return rc;
}
int bad(const char* what) { return fail(Z2B_ERR_ARG, what); }
int unsupported(const char* what) { return fail(Z2B_ERR_UNSUPPORTED, what); }

int launched(cudaError_t e, const char* op) {
    if (e == cudaSuccess) return Z2B_OK;
    cudaGetLastError();                                  // a refused launch leaves nothing behind
    return fail(e == cudaErrorNotSupported ? Z2B_ERR_UNSUPPORTED : Z2B_ERR_CUDA, op, cudaGetErrorString(e));
}

bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
unsigned type_size(int t) { return t == Z2B_TYPE_F32 ? 4 : 2; }
bool act_type(int t) { return t == Z2B_TYPE_F32 || t == Z2B_TYPE_F16 || t == Z2B_TYPE_BF16; }

// ---- shared memory. An array is a box of elements at sum of i_d * stride_d, 0 <= i_d < n_d; two of
// its elements, or elements of two arrays, are the same where the differences x_d of their indices
// solve sum of stride_d x_d = delta. The strides of usual arrays nest (each is at least what the smaller
// ones span), which leaves a candidate or two per dim; others are searched, up to a limit.
struct Var { long long stride, lo, hi; };       // a difference of indices and its range

// Whether var[0..n) (strides descending, positive) reach delta. Out of `steps`: taken as no.
bool reaches(const Var* v, int n, long long delta, int* steps) {
    if (n == 0) return delta == 0;
    long long lo = 0, hi = 0;                    // what the later ones span
    for (int i = 1; i < n; ++i) { lo += v[i].stride * v[i].lo; hi += v[i].stride * v[i].hi; }
    const long long s = v->stride, a = delta - hi, b = delta - lo;
    long long x = a > 0 ? (a + s - 1) / s : -(-a / s), end = b >= 0 ? b / s : -((-b + s - 1) / s);
    x = std::max(x, v->lo);
    end = std::min(end, v->hi);
    for (; x <= end; ++x) {
        if (--*steps < 0) return false;
        if (reaches(v + 1, n - 1, delta - s * x, steps)) return true;
    }
    return false;
}

struct Box {
    const void* p;
    int n = 0, size;
    bool back[4];                                // a dim that runs backwards: taken from its other end
    long long stride[4], len[4], first = 0, last = 0;       // elements from p to the lowest one, from that to the highest
    bool real;                                   // false: it spans more than addresses do, there is nothing to compare
    // `size` bytes an element, aligned to it
    Box(const void* p_, int size_, std::initializer_list<std::pair<long long, long long>> dims) : p(p_), size(size_) {
        __int128 low = 0, span = 0;
        for (const auto& d : dims) {
            if (d.second <= 1) continue;         // a dim of one has no stride
            const __int128 far = (__int128)d.first * (d.second - 1);
            back[n] = far < 0;
            if (far < 0) low += far;
            span += far < 0 ? -far : far;
            stride[n] = far < 0 ? -d.first : d.first;
            len[n++] = d.second;
        }
        real = span < 1ll << 56;
        if (real) { first = (long long)low; last = (long long)span; }
    }
    bool same_place(const Box& o) const {
        return p == o.p && n == o.n && std::equal(stride, stride + n, o.stride) && std::equal(back, back + n, o.back) &&
               std::equal(len, len + n, o.len);
    }
};
bool steeper(const Var& a, const Var& b) { return a.stride > b.stride; }

// Some element has two indices.
bool shares_itself(const Box& b) {
    Var v[4];
    for (int i = 0; i < b.n; ++i) {
        if (b.stride[i] == 0) return true;
        v[i] = Var{b.stride[i], 1 - b.len[i], b.len[i] - 1};
    }
    if (!b.real) return false;
    std::sort(v, v + b.n, steeper);
    long long span = 0;
    bool nest = true;
    for (int i = b.n - 1; i >= 0; --i) { nest &= v[i].stride > span; span += v[i].stride * v[i].hi; }
    if (nest) return false;
    int steps = 1 << 16;
    for (int i = 0; i < b.n; ++i) {              // the first dim in which the two indices differ
        const Var all = v[i];
        v[i].lo = 1;
        if (reaches(v + i, b.n - i, 0, &steps)) return true;
        v[i] = all;
    }
    return false;
}

// Some element of one is an element of the other, of the same size.
bool share(const Box& a, const Box& b) {
    const long long d = (long long)((uintptr_t)b.p - (uintptr_t)a.p) / a.size + b.first - a.first;
    if (!a.real || !b.real || d > a.last || -d > b.last) return false;
    Var v[8];
    int n = 0;
    for (int i = 0; i < a.n; ++i) if (a.stride[i]) v[n++] = Var{a.stride[i], 0, a.len[i] - 1};
    for (int i = 0; i < b.n; ++i) {
        if (!b.stride[i]) continue;              // an input's dim without a stride stays where it is
        int j = 0;
        while (j < n && v[j].stride != b.stride[i]) ++j;
        if (j == n) v[n++] = Var{b.stride[i], 0, 0};
        v[j].lo -= b.len[i] - 1;                 // equal strides: one difference
    }
    std::sort(v, v + n, steeper);
    int steps = 1 << 16;
    return reaches(v, n, d, &steps);
}

// What both cache operators ask of the view; empty when it is sound.
const char* check_kv(const z2b_paged_kv* c) {
    if (!c) return "kv: null argument";
    if (!c->k || !c->v) return "kv: null cache";
    if (c->type != Z2B_TYPE_F16 && c->type != Z2B_TYPE_BF16) return "kv: type must be Z2B_TYPE_F16 or Z2B_TYPE_BF16";
    if (c->n_pages < 1 || c->page_len < 1 || c->n_head_kv < 1 || c->head_dim < 1) return "kv: sizes must be positive";
    if (c->page_stride < 0 || c->row_stride < 0 || c->head_stride < 0) return "kv: strides must not be negative";
    if (!aligned(c->k, 2) || !aligned(c->v, 2)) return "kv: misaligned cache";
    return "";
}

// The stream metadata of a call with rows.
const char* check_rows(int n_seq, const int32_t* row_off, const int32_t* seq_len, const int32_t* table, int64_t table_stride,
                       int max_pages) {
    if (!row_off || !seq_len) return "null row_off or seq_len";
    if (max_pages < 0 || (max_pages > 0 && !table)) return "null page_table";
    if (max_pages > 0 && n_seq > 1 && table_stride < max_pages) return "table_stride is less than max_pages";
    if (!aligned(row_off, 4) || !aligned(seq_len, 4) || !aligned(table, 4)) return "misaligned int32 array";
    return "";
}

}  // namespace

extern "C" {

int z2b_rope_init(z2b_rope* out, int rot_dim, int layout, double base, int scaling, double factor, int orig_ctx) {
    if (!out) return bad("rope_init: null argument");
    if (rot_dim < 2 || rot_dim > Z2B_ROPE_MAX_DIM || rot_dim % 2) return bad("rope_init: rot_dim must be even, 2..Z2B_ROPE_MAX_DIM");
    if (layout != Z2B_ROPE_INTERLEAVED && layout != Z2B_ROPE_HALF) return bad("rope_init: unknown layout");
    if (!(base > 1.0) || !std::isfinite(base)) return bad("rope_init: base must be above 1");
    if (scaling < Z2B_ROPE_SCALE_NONE || scaling > Z2B_ROPE_SCALE_BY_PARTS) return bad("rope_init: unknown scaling");
    if (!(factor > 0.0) || !std::isfinite(factor)) return bad("rope_init: factor must be positive");
    if (scaling == Z2B_ROPE_SCALE_NONE && factor != 1.0) return bad("rope_init: factor needs a scaling");
    if (scaling == Z2B_ROPE_SCALE_NTK && rot_dim <= 2) return bad("rope_init: SCALE_NTK needs rot_dim above 2");
    if (scaling == Z2B_ROPE_SCALE_BY_PARTS && orig_ctx <= 0) return bad("rope_init: SCALE_BY_PARTS needs orig_ctx");
    const double two_pi = 6.283185307179586476925286766559;
    if (scaling == Z2B_ROPE_SCALE_NTK) base *= std::pow(factor, (double)rot_dim / (rot_dim - 2));
    if (!(base > 0.0) || !std::isfinite(base)) return bad("rope_init: the factor takes the base out of range");
    z2b_rope r{};
    r.rot_dim = rot_dim;
    r.layout = layout;
    r.mag = scaling == Z2B_ROPE_SCALE_BY_PARTS ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
    if (!(r.mag > 0.0f)) return bad("rope_init: the factor leaves no positive magnitude");
    for (int i = 0; i < rot_dim / 2; ++i) {
        double w = std::pow(base, -2.0 * i / rot_dim);           // radians per position
        if (scaling == Z2B_ROPE_SCALE_LINEAR) w /= factor;
        else if (scaling == Z2B_ROPE_SCALE_BY_PARTS) {
            const double turns = orig_ctx * w / two_pi;
            const double keep = std::min(1.0, std::max(0.0, (turns - 1.0) / (32.0 - 1.0)));
            w = w / factor * (1.0 - keep) + w * keep;
        }
        double t = w / two_pi;
        if (!std::isfinite(t)) return bad("rope_init: the factor takes a frequency out of range");
        t -= std::floor(t);                                      // whole turns change nothing
        const double top = std::ldexp(t, 64);                    // exact: a power of two
        r.step[i] = top >= 18446744073709551616.0 ? 0 : (uint64_t)top;
    }
    *out = r;
    return Z2B_OK;
}

int z2b_rope_append(const z2b_rope_append_args* args, void* stream) {
    if (!args) return bad("rope_append: null argument");
    const z2b_rope_append_args& a = *args;
    const char* m = check_kv(a.kv);
    if (*m) return bad(m);
    if (!act_type(a.type)) return bad("rope_append: type must be Z2B_TYPE_F32, F16 or BF16");
    if (a.n_rows < 0 || a.n_seq < 0 || a.n_head < 0 || a.prefix_len < 0) return bad("rope_append: negative size");
    if (a.n_head > 0 && a.n_rows > 0 && (!a.q || !a.q_out)) return bad("rope_append: null q or q_out");
    if ((a.k == nullptr) != (a.v == nullptr)) return bad("rope_append: k and v come together");
    if (a.rope && (a.rope->rot_dim < 2 || a.rope->rot_dim > Z2B_ROPE_MAX_DIM || a.rope->rot_dim % 2 ||
                   a.rope->rot_dim > a.kv->head_dim || (a.rope->layout != Z2B_ROPE_INTERLEAVED && a.rope->layout != Z2B_ROPE_HALF)))
        return bad("rope_append: the rotation does not fit head_dim");
    if (a.kv->head_dim > 1024) return unsupported("rope_append: head_dim above 1024");
    if (a.n_seq > OPS_MAX_SEQ) return unsupported("rope_append: more than 4096 streams");
    if (a.n_rows > (1 << 30) || a.n_head > (1 << 20) || a.kv->n_head_kv > (1 << 20))    // row and head numbers are 32-bit
        return unsupported("rope_append: too many rows or heads for one call");
    const int e = (int)type_size(a.type);
    if (!aligned(a.q, e) || !aligned(a.q_out, e) || !aligned(a.k, e) || !aligned(a.v, e) || !aligned(a.pos, 4))
        return bad("rope_append: misaligned array");
    if (a.n_rows == 0 || a.n_seq == 0 || (a.n_head == 0 && !a.k)) return Z2B_OK;
    m = check_rows(a.n_seq, a.row_off, a.seq_len, a.page_table, a.table_stride, a.max_pages);
    if (*m) return bad(m);
    // rows are turned and stored at the same time, in any order
    const z2b_paged_kv& c = *a.kv;
    const Box out(a.n_head ? a.q_out : nullptr, e, {{a.o_row, a.n_rows}, {a.o_head, a.n_head}, {1, c.head_dim}});
    if (out.p) {
        const Box q(a.q, e, {{a.q_row, a.n_rows}, {a.q_head, a.n_head}, {1, c.head_dim}});
        if (shares_itself(out)) return bad("rope_append: rows or heads of q_out share memory");
        if (!out.same_place(q) && share(out, q)) return bad("rope_append: q_out lies across q");
    }
    if (a.k) {
        const Box k(a.k, e, {{a.k_row, a.n_rows}, {a.k_head, c.n_head_kv}, {1, c.head_dim}});
        const Box v(a.v, e, {{a.v_row, a.n_rows}, {a.v_head, c.n_head_kv}, {1, c.head_dim}});
        if (out.p && (share(out, k) || share(out, v))) return bad("rope_append: q_out lies across k or v");
        const Box kc(c.k, 2, {{c.page_stride, c.n_pages}, {c.row_stride, c.page_len}, {c.head_stride, c.n_head_kv}, {1, c.head_dim}});
        const Box vc(c.v, 2, {{c.page_stride, c.n_pages}, {c.row_stride, c.page_len}, {c.head_stride, c.n_head_kv}, {1, c.head_dim}});
        if (shares_itself(kc) || share(kc, vc)) return bad("rope_append: pages, rows, heads or keys and values of the cache share memory");
    }
    DeviceGuard g(a.device);
    if (g.rc != cudaSuccess) return launched(g.rc, "rope_append: device: ");
    return launched(launch_rope_append(a, (cudaStream_t)stream), "rope_append: ");
}

static const char* check_attn(const z2b_prefix_attn_args& a, int* rc) {
    *rc = Z2B_ERR_ARG;
    const char* m = check_kv(a.kv);
    if (*m) return m;
    const z2b_paged_kv& c = *a.kv;
    if (a.n_rows < 0 || a.n_seq < 0 || a.prefix_len < 0 || a.max_pages < 0) return "prefix_attention: negative size";
    if (a.n_head < 1 || a.n_head % c.n_head_kv) return "prefix_attention: n_head must be a multiple of the cache's heads";
    *rc = Z2B_ERR_UNSUPPORTED;
    if (c.head_dim != 16 && c.head_dim != 32 && c.head_dim != 64 && c.head_dim != 128)
        return "prefix_attention: head_dim must be 16, 32, 64 or 128";
    if (c.page_len % 8) return "prefix_attention: page_len must be a multiple of 8";
    if (a.n_seq > OPS_MAX_SEQ) return "prefix_attention: more than 4096 streams";
    // unit and slot numbers are 32-bit; rows x heads of a key head, and head numbers, are divided by the
    // group size G by a 32-bit multiplication that is exact while number x G is below 2^32
    const long long G = a.n_head / c.n_head_kv, tiles = ((long long)a.n_rows * G + 7) / 8;
    const long long own = ((long long)a.max_pages * c.page_len + 31) / 32 + 1, pf = ((long long)a.prefix_len + 31) / 32 + 1;
    if (tiles * c.n_head_kv > (1 << 24) || (long long)a.n_seq * c.n_head_kv > (1 << 24) || own > (1 << 24) || pf > (1 << 24) ||
        ((long long)a.n_rows + 32) * G * G > 0xffffffffll || a.n_head * G > 0xffffffffll || ((tiles + a.n_seq) * own + (tiles + 1) * pf) * c.n_head_kv > 0x7fffffffll)
        return "prefix_attention: too many rows, streams or pages for one call";
    return "";
}

size_t z2b_prefix_attention_workspace(const z2b_prefix_attn_args* args) {
    int rc;
    if (!args) { bad("prefix_attention: null argument"); return 0; }
    const char* m = check_attn(*args, &rc);
    if (*m) { fail(rc, m); return 0; }
    if (args->n_rows == 0 || args->n_seq == 0) return 256;
    return prefix_attention_bytes(*args);
}

int z2b_prefix_attention(const z2b_prefix_attn_args* args, void* stream) {
    if (!args) return bad("prefix_attention: null argument");
    const z2b_prefix_attn_args& a = *args;
    int rc;
    const char* m = check_attn(a, &rc);
    if (*m) return fail(rc, m);
    const z2b_paged_kv& c = *a.kv;
    if (!aligned(c.k, 16) || !aligned(c.v, 16) || (c.page_stride | c.row_stride | c.head_stride) % 8)
        return bad("prefix_attention: the cache must be 16-byte aligned with strides that are multiples of 8");
    if (!std::isfinite(a.scale * 2.0f)) return bad("prefix_attention: scale must be finite, and twice it");
    if (a.n_rows == 0 || a.n_seq == 0) return Z2B_OK;
    if (!a.q || !a.out) return bad("prefix_attention: null q or out");
    if (!aligned(a.q, 4) || !aligned(a.out, 4) || (a.q_row | a.q_head | a.o_row | a.o_head) % 2 || !aligned(a.lse, 4))
        return bad("prefix_attention: q and out must be 4-byte aligned with even strides");
    m = check_rows(a.n_seq, a.row_off, a.seq_len, a.page_table, a.table_stride, a.max_pages);
    if (*m) return bad(m);
    if (a.prefix_len > 0 && !a.prefix_pages) return bad("prefix_attention: null prefix_pages");
    if (!a.workspace || !aligned(a.workspace, 16)) return bad("prefix_attention: the workspace must be 16-byte aligned");
    if (a.workspace_bytes < prefix_attention_bytes(a)) return bad("prefix_attention: the workspace is too small");
    if (shares_itself(Box(a.out, 2, {{a.o_row, a.n_rows}, {a.o_head, a.n_head}, {1, c.head_dim}})))
        return bad("prefix_attention: rows or heads of out share memory");
    DeviceGuard g(a.device);
    if (g.rc != cudaSuccess) return launched(g.rc, "prefix_attention: device: ");
    return launched(launch_prefix_attention(a, (cudaStream_t)stream), "prefix_attention: ");
}

int z2b_verify_drafts(const z2b_verify_args* args, void* stream) {
    if (!args) return bad("verify_drafts: null argument");
    const z2b_verify_args& a = *args;
    if (!act_type(a.type)) return bad("verify_drafts: type must be Z2B_TYPE_F32, F16 or BF16");
    if (a.n_seq < 0 || a.max_draft < 0 || a.n_codebooks < 1 || a.vocab < 1) return bad("verify_drafts: bad size");
    if (a.n_seq == 0) return Z2B_OK;
    if (!a.p || !a.u_draw || !a.tokens || !a.n_accepted) return bad("verify_drafts: null argument");
    if (a.max_draft > 0 && (!a.draft || !a.u_accept)) return bad("verify_drafts: null draft or u_accept");
    if (a.vocab > (1 << 30) || (long long)a.n_seq * a.n_codebooks > (1 << 27) || a.max_draft > (1 << 20) / a.n_codebooks)
        return unsupported("verify_drafts: too many rows for one call");
    const unsigned e = type_size(a.type);
    if (!aligned(a.p, e) || !aligned(a.q, e) || !aligned(a.draft, 4) || !aligned(a.n_draft, 4) || !aligned(a.u_accept, 8) ||
        !aligned(a.u_draw, 8) || !aligned(a.tokens, 4) || !aligned(a.n_accepted, 4))
        return bad("verify_drafts: misaligned array");
    DeviceGuard g(a.device);
    if (g.rc != cudaSuccess) return launched(g.rc, "verify_drafts: device: ");
    return launched(launch_verify(a, (cudaStream_t)stream), "verify_drafts: ");
}

}  // extern "C"
