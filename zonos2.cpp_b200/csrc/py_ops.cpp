// py_ops.cpp — the Python binding of include/z2b_ops.h for torch tensors (module z2b._ops,
// imported by z2b.ops): checks the tensors, allocates results and workspace through torch, and
// calls the C entry points on torch's current stream.
//
// Compiled against torch, unlike the rest of the binding, because the small calls are bound by
// it: taking some forty sizes, strides and addresses from tensors in Python costs 9 us beside
// the 2 us of a launch, here 1.
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/z2b_ops.h"

#include <limits>
#include <string>

extern "C" const char* z2b_last_error(void);

namespace {

PyObject* g_error = nullptr;            // z2b.runtime.Z2BError(rc, message)

struct Refused { int rc; std::string msg; };
[[noreturn]] void refuse(const std::string& msg) { throw Refused{1, msg}; }

void raise(const Refused& r) {
    PyObject* e = PyObject_CallFunction(g_error, "is", r.rc, r.msg.c_str());
    if (e) { PyErr_SetObject(g_error, e); Py_DECREF(e); }
}

int64_t integer(PyObject* o, const char* what, int64_t most = std::numeric_limits<int32_t>::max()) {
    const long long v = PyLong_Check(o) ? PyLong_AsLongLong(o) : -1;
    if (PyErr_Occurred()) { PyErr_Clear(); refuse(std::string(what) + ": the number is out of range"); }
    if (!PyLong_Check(o) || v < 0 || v > most) refuse(std::string(what) + ": a number from 0 to 2^31 - 1 is wanted");
    return v;
}

const at::Tensor& tensor(PyObject* o, const char* what) {
    if (!THPVariable_Check(o)) refuse(std::string(what) + ": a tensor is wanted");
    return THPVariable_Unpack(o);
}
const at::Tensor* maybe(PyObject* o, const char* what) { return o == Py_None ? nullptr : &tensor(o, what); }

int type_code(at::ScalarType t, const char* what) {
    switch (t) {
        case at::kFloat: return Z2B_TYPE_F32;
        case at::kHalf: return Z2B_TYPE_F16;
        case at::kBFloat16: return Z2B_TYPE_BF16;
        default: refuse(std::string(what) + ": f32, f16 or bf16 is wanted");
    }
}

int device_of(const at::Tensor& t, const char* what) {
    if (!t.is_cuda()) refuse(std::string(what) + ": a CUDA tensor is wanted");
    return t.device().index();
}
void same_device(const at::Tensor& t, int device, const char* what) {
    if (!t.is_cuda() || t.device().index() != device) refuse(std::string(what) + ": not on the call's device");
}
// Gradients of either mode; forward mode has no switch to call under, its tensors are taken apart first.
void no_grad(const at::Tensor& t, const char* what) {
    if (t.requires_grad() && at::GradMode::is_enabled()) refuse(std::string(what) + ": there is no backward pass; call under torch.no_grad()");
    if (t._fw_grad(0).defined()) refuse(std::string(what) + ": there is no forward-mode gradient; pass the tensor without its tangent");
}

// A contiguous array of `dtype` and that shape.
void* array(const at::Tensor& t, at::ScalarType dtype, at::IntArrayRef shape, int device, const char* what) {
    same_device(t, device, what);
    if (t.scalar_type() != dtype || t.sizes() != shape || !t.is_contiguous())
        refuse(std::string(what) + ": a contiguous " + std::string(c10::toString(dtype)) + " tensor of another shape is wanted");
    return t.data_ptr();
}
const int32_t* ints(const at::Tensor& t, int64_t n, int device, const char* what) {
    return (const int32_t*)array(t, at::kInt, {n}, device, what);
}
uint32_t* err_word(PyObject* o, int device) {
    return o == Py_None ? nullptr : (uint32_t*)array(tensor(o, "err"), at::kInt, {1}, device, "err");
}

// Rows [n][heads][head_dim] of `dtype`.
void* rows(const at::Tensor& t, int64_t n, int64_t heads, int64_t hd, at::ScalarType dtype, int device, const char* what, int64_t* row,
           int64_t* head) {
    same_device(t, device, what);
    if (t.dim() != 3 || t.size(0) != n || t.size(1) != heads || t.size(2) != hd) refuse(std::string(what) + ": [rows][heads][head_dim] do not match");
    if (t.scalar_type() != dtype || (t.stride(2) != 1 && hd > 1)) refuse(std::string(what) + ": wrong type, or the dims of a head are not contiguous");
    *row = t.stride(0);
    *head = t.stride(1);
    return t.data_ptr();
}

const int32_t* page_table(const at::Tensor& t, int64_t n_seq, int device, int64_t* stride, int32_t* pages) {
    same_device(t, device, "page_table");
    if (t.scalar_type() != at::kInt || t.dim() != 2 || t.size(0) != n_seq || (t.size(1) > 1 && t.stride(1) != 1) || t.size(1) > INT32_MAX)
        refuse("page_table: an int32 tensor [streams][pages], the pages of a stream contiguous, is wanted");
    *stride = t.stride(0);
    *pages = (int32_t)t.size(1);
    return (const int32_t*)t.data_ptr();
}

at::Tensor fresh(at::IntArrayRef shape, at::ScalarType dtype, int device) {
    return at::detail::empty_cuda(shape, dtype, at::Device(at::kCUDA, (c10::DeviceIndex)device), std::nullopt);
}

void* stream_of(int device) { return (void*)c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }

// Calls without the interpreter's lock; a refusal becomes Z2BError.
template <typename F> void call(F f) {
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = f();
    Py_END_ALLOW_THREADS
    if (rc) throw Refused{rc, z2b_last_error()};
}

void want(Py_ssize_t got, Py_ssize_t n) {
    if (got != n) refuse("wrong number of arguments");
}

#define GUARDED(...)                                   \
    HANDLE_TH_ERRORS                                   \
    try { __VA_ARGS__ } catch (const Refused& r) { raise(r); return nullptr; } \
    END_HANDLE_TH_ERRORS

int32_t as_int(int64_t v, const char* what) {
    if (v > INT32_MAX) refuse(std::string(what) + ": too large");
    return (int32_t)v;
}

// rope_append(rope address or 0, kv address, device, q, k, v, row_off, seq_len, page_table, prefix_len, pos, out, err)
PyObject* rope_append(PyObject*, PyObject* const* v, Py_ssize_t n_args) {
    GUARDED(
        want(n_args, 13);
        z2b_rope_append_args a{};
        a.rope = (const z2b_rope*)integer(v[0], "rope", INT64_MAX);
        a.kv = (const z2b_paged_kv*)integer(v[1], "kv", INT64_MAX);
        a.device = (int32_t)integer(v[2], "device");
        const at::Tensor *q = maybe(v[3], "q"), *k = maybe(v[4], "k"), *val = maybe(v[5], "v"), *out = maybe(v[11], "out");
        if ((!q && !k) || !k != !val) refuse("rope_append: q, or k and v, or all three");
        const at::Tensor& lead = q ? *q : *k;
        if (lead.dim() != 3) refuse("rope_append: rows [rows][heads][head_dim] are wanted");
        const at::ScalarType dt = lead.scalar_type();
        a.type = type_code(dt, "rope_append");
        const int64_t n = lead.size(0);
        const int64_t hd = a.kv->head_dim;
        a.n_rows = as_int(n, "rows");
        at::Tensor made;
        if (q) {
            no_grad(*q, "q");
            a.n_head = as_int(q->size(1), "heads");
            a.q = rows(*q, n, a.n_head, hd, dt, a.device, "q", &a.q_row, &a.q_head);
            if (!out) {
                made = fresh({n, a.n_head, hd}, dt, a.device);
                out = &made;
            }
            a.q_out = rows(*out, n, a.n_head, hd, dt, a.device, "out", &a.o_row, &a.o_head);
            no_grad(*out, "out");
        } else if (out) refuse("rope_append: out without q");
        if (k) {
            no_grad(*k, "k");
            no_grad(*val, "v");
            a.k = rows(*k, n, a.kv->n_head_kv, hd, dt, a.device, "k", &a.k_row, &a.k_head);
            a.v = rows(*val, n, a.kv->n_head_kv, hd, dt, a.device, "v", &a.v_row, &a.v_head);
            if (!n) a.k = a.v = nullptr;
        }
        const at::Tensor& lens = tensor(v[7], "seq_len");
        a.n_seq = as_int(lens.numel(), "streams");
        a.row_off = ints(tensor(v[6], "row_off"), (int64_t)a.n_seq + 1, a.device, "row_off");
        a.seq_len = ints(lens, a.n_seq, a.device, "seq_len");
        a.page_table = page_table(tensor(v[8], "page_table"), a.n_seq, a.device, &a.table_stride, &a.max_pages);
        a.prefix_len = (int32_t)integer(v[9], "prefix_len");
        if (v[10] != Py_None) a.pos = ints(tensor(v[10], "pos"), n, a.device, "pos");
        a.err = err_word(v[12], a.device);
        void* s = stream_of(a.device);
        call([&] { return z2b_rope_append(&a, s); });
        if (!q) Py_RETURN_NONE;
        if (made.defined()) return THPVariable_Wrap(made);
        Py_INCREF(v[11]);
        return v[11];
    )
}

// prefix_attention(kv address, device, q, row_off, seq_len, page_table, prefix_pages, prefix_len, scale, out, lse, err)
PyObject* prefix_attention(PyObject*, PyObject* const* v, Py_ssize_t n_args) {
    GUARDED(
        want(n_args, 12);
        z2b_prefix_attn_args a{};
        a.kv = (const z2b_paged_kv*)integer(v[0], "kv", INT64_MAX);
        a.device = (int32_t)integer(v[1], "device");
        const at::Tensor& q = tensor(v[2], "q");
        if (q.dim() != 3) refuse("q: rows [rows][heads][head_dim] are wanted");
        no_grad(q, "q");
        const at::ScalarType dt = a.kv->type == Z2B_TYPE_F16 ? at::kHalf : at::kBFloat16;
        const int64_t n = q.size(0);
        const int64_t nh = q.size(1);
        const int64_t hd = a.kv->head_dim;
        a.n_rows = as_int(n, "rows");
        a.n_head = as_int(nh, "heads");
        a.q = rows(q, n, nh, hd, dt, a.device, "q", &a.q_row, &a.q_head);
        const at::Tensor& lens = tensor(v[4], "seq_len");
        a.n_seq = as_int(lens.numel(), "streams");
        a.row_off = ints(tensor(v[3], "row_off"), (int64_t)a.n_seq + 1, a.device, "row_off");
        a.seq_len = ints(lens, a.n_seq, a.device, "seq_len");
        a.page_table = page_table(tensor(v[5], "page_table"), a.n_seq, a.device, &a.table_stride, &a.max_pages);
        a.prefix_len = (int32_t)integer(v[7], "prefix_len");
        if (a.prefix_len > 0) {
            if (v[6] == Py_None) refuse("prefix_pages: missing");
            const at::Tensor& pages = tensor(v[6], "prefix_pages");
            a.prefix_pages = ints(pages, pages.numel(), a.device, "prefix_pages");
            if (pages.numel() < ((int64_t)a.prefix_len + a.kv->page_len - 1) / a.kv->page_len)
                refuse("prefix_pages: a page for every page_len rows of the prefix is wanted");
        }
        const double scale = PyFloat_AsDouble(v[8]);
        if (PyErr_Occurred()) { PyErr_Clear(); refuse("scale: a number is wanted"); }
        a.scale = (float)scale;
        at::Tensor made; at::Tensor made_lse;
        const at::Tensor* out = maybe(v[9], "out");
        if (!out) {
            made = fresh({n, nh, hd}, dt, a.device);
            out = &made;
        }
        a.out = rows(*out, n, nh, hd, dt, a.device, "out", &a.o_row, &a.o_head);
        no_grad(*out, "out");
        const bool want_lse = v[10] == Py_True;
        if (want_lse) {
            made_lse = fresh({n, nh}, at::kFloat, a.device);
            a.lse = (float*)made_lse.data_ptr();
        } else if (v[10] != Py_None && v[10] != Py_False) {
            a.lse = (float*)array(tensor(v[10], "lse"), at::kFloat, {n, nh}, a.device, "lse");
            no_grad(tensor(v[10], "lse"), "lse");
        }
        a.err = err_word(v[11], a.device);
        a.workspace_bytes = z2b_prefix_attention_workspace(&a);      // 0: the call below says what is wrong with the sizes
        const at::Tensor ws = fresh({(int64_t)a.workspace_bytes}, at::kByte, a.device);
        a.workspace = ws.data_ptr();
        void* s = stream_of(a.device);
        call([&] { return z2b_prefix_attention(&a, s); });
        PyObject* o = v[9];
        if (made.defined()) { o = THPVariable_Wrap(made); if (!o) return nullptr; } else Py_INCREF(o);
        if (v[10] == Py_None || v[10] == Py_False) return o;
        PyObject* l = v[10];
        if (want_lse) { l = THPVariable_Wrap(made_lse); if (!l) { Py_DECREF(o); return nullptr; } } else Py_INCREF(l);
        PyObject* both = PyTuple_Pack(2, o, l);
        Py_DECREF(o);
        Py_DECREF(l);
        return both;
    )
}

// verify_drafts(p, q, draft, u_accept, u_draw, n_draft, err)
PyObject* verify_drafts(PyObject*, PyObject* const* v, Py_ssize_t n_args) {
    GUARDED(
        want(n_args, 7);
        z2b_verify_args a{};
        const at::Tensor& p = tensor(v[0], "p");
        a.device = device_of(p, "p");
        a.type = type_code(p.scalar_type(), "p");
        no_grad(p, "p");
        if (p.dim() != 4 || p.size(1) < 1) refuse("p: [streams][drafts + 1][codebooks][vocab] is wanted");
        const int64_t B = p.size(0);
        const int64_t N = p.size(1) - 1;
        const int64_t C = p.size(2);
        const int64_t V = p.size(3);
        if (p.stride(3) != 1 && V > 1) refuse("p: the vocabulary must be contiguous");
        a.n_seq = as_int(B, "streams");
        a.max_draft = as_int(N, "drafts");
        a.n_codebooks = as_int(C, "codebooks");
        a.vocab = as_int(V, "vocab");
        a.p = p.data_ptr();
        a.p_seq = p.stride(0); a.p_frame = p.stride(1); a.p_book = p.stride(2);
        if (const at::Tensor* q = maybe(v[1], "q")) {
            same_device(*q, a.device, "q");
            no_grad(*q, "q");
            if (q->dim() != 4 || q->size(0) != B || q->size(1) != N || q->size(2) != C || q->size(3) != V || q->scalar_type() != p.scalar_type() ||
                (q->stride(3) != 1 && V > 1))
                refuse("q: [streams][drafts][codebooks][vocab] of p's type is wanted, the vocabulary contiguous");
            if (N > 0) a.q = q->data_ptr();
            a.q_seq = q->stride(0); a.q_frame = q->stride(1); a.q_book = q->stride(2);
        }
        a.draft = (const int32_t*)array(tensor(v[2], "draft"), at::kInt, {B, N, C}, a.device, "draft");
        a.u_accept = (const double*)array(tensor(v[3], "u_accept"), at::kDouble, {B, N, C}, a.device, "u_accept");
        a.u_draw = (const double*)array(tensor(v[4], "u_draw"), at::kDouble, {B, N + 1, C}, a.device, "u_draw");
        if (v[5] != Py_None) a.n_draft = ints(tensor(v[5], "n_draft"), B, a.device, "n_draft");
        a.err = err_word(v[6], a.device);
        const at::Tensor tokens = fresh({B, N + 1, C}, at::kInt, a.device);
        const at::Tensor kept = fresh({B}, at::kInt, a.device);
        a.tokens = (int32_t*)tokens.data_ptr();
        a.n_accepted = (int32_t*)kept.data_ptr();
        void* s = stream_of(a.device);
        call([&] { return z2b_verify_drafts(&a, s); });
        PyObject* t = THPVariable_Wrap(tokens);
        PyObject* n = t ? THPVariable_Wrap(kept) : nullptr;
        PyObject* both = n ? PyTuple_Pack(2, t, n) : nullptr;
        Py_XDECREF(t);
        Py_XDECREF(n);
        return both;
    )
}

// The class that refusals raise.
PyObject* set_error_class(PyObject*, PyObject* cls) {
    Py_INCREF(cls);
    Py_XSETREF(g_error, cls);
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"rope_append", (PyCFunction)(void*)rope_append, METH_FASTCALL, nullptr},
    {"prefix_attention", (PyCFunction)(void*)prefix_attention, METH_FASTCALL, nullptr},
    {"verify_drafts", (PyCFunction)(void*)verify_drafts, METH_FASTCALL, nullptr},
    {"set_error_class", set_error_class, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops(void) { return PyModule_Create(&module); }
