"""The operators of include/z2b_ops.h on torch CUDA tensors.

``rope_append``, ``prefix_attention`` and ``verify_drafts`` run on the tensors' device, on
torch's current stream of that device, allocate their outputs (and workspace) through torch
and neither synchronise nor copy to the host, so they can be captured into CUDA graphs.
Every refusal raises ``Z2BError``, as in ``z2b.runtime``. ``err``, where given, is an int32
tensor of one element on the device that the kernels OR ``BAD_INDEX``, ``BAD_PAGE`` and
``TIMEOUT`` into; ``check(err)`` reads it (which synchronises) and raises.

Rows are packed over the streams: stream b owns rows [row_off[b], row_off[b + 1]) of q
[rows][heads][head_dim], rows from row_off[-1] on are padding and stay as they are, seq_len[b]
counts the stream's cached rows with the new ones, and page_table[b] lists its pages.
"""
from __future__ import annotations

import ctypes
import math
import struct

import torch

from .runtime import Z2BError, lib

TIMEOUT, BAD_INDEX, BAD_PAGE = 1, 2, 4
_TYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
_LAYOUT = {"interleaved": 0, "half": 1}
_SCALING = {"none": 0, "linear": 1, "ntk": 2, "by_parts": 3}

_I, _L, _P, _F, _Z = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p, ctypes.c_float, ctypes.c_size_t


class RopeTable(ctypes.Structure):
    """z2b_rope."""
    _fields_ = [("rot_dim", _I), ("layout", _I), ("mag", _F), ("reserved", _I), ("step", ctypes.c_uint64 * 128)]


class PagedKVView(ctypes.Structure):
    """z2b_paged_kv."""
    _fields_ = [("k", _P), ("v", _P), ("type", _I), ("n_pages", _I), ("page_len", _I), ("n_head_kv", _I),
                ("head_dim", _I), ("page_stride", _L), ("row_stride", _L), ("head_stride", _L)]


class RopeAppendArgs(ctypes.Structure):
    """z2b_rope_append_args."""
    _fields_ = [("device", _I), ("type", _I), ("n_rows", _I), ("n_seq", _I), ("n_head", _I), ("prefix_len", _I),
                ("rope", _P), ("kv", _P), ("q", _P), ("q_out", _P), ("k", _P), ("v", _P)] + \
               [(n, _L) for n in ("q_row", "q_head", "o_row", "o_head", "k_row", "k_head", "v_row", "v_head")] + \
               [("row_off", _P), ("seq_len", _P), ("page_table", _P), ("table_stride", _L), ("max_pages", _I),
                ("pos", _P), ("err", _P)]


class PrefixAttnArgs(ctypes.Structure):
    """z2b_prefix_attn_args."""
    _fields_ = [("device", _I), ("n_rows", _I), ("n_seq", _I), ("n_head", _I), ("prefix_len", _I), ("scale", _F),
                ("kv", _P), ("q", _P), ("out", _P), ("lse", _P), ("q_row", _L), ("q_head", _L), ("o_row", _L),
                ("o_head", _L), ("row_off", _P), ("seq_len", _P), ("page_table", _P), ("table_stride", _L),
                ("max_pages", _I), ("prefix_pages", _P), ("workspace", _P), ("workspace_bytes", _Z), ("err", _P)]


class VerifyArgs(ctypes.Structure):
    """z2b_verify_args."""
    _fields_ = [("device", _I), ("type", _I), ("n_seq", _I), ("max_draft", _I), ("n_codebooks", _I), ("vocab", _I),
                ("p", _P), ("q", _P), ("draft", _P), ("n_draft", _P), ("u_accept", _P), ("u_draw", _P), ("tokens", _P),
                ("n_accepted", _P)] + [(n, _L) for n in ("p_seq", "p_frame", "p_book", "q_seq", "q_frame", "q_book")] + \
               [("err", _P)]


def _packer(cls):
    """struct packer of an argument structure: a quarter of the time its constructor takes, which
    is a good part of a small call."""
    code = {_I: "i", _L: "q", _P: "P", _F: "f", _Z: "N"}
    pack = struct.Struct("@" + "".join(code[f] for _, f in cls._fields_)).pack

    def packed(*values):
        try:
            return pack(*values)
        except struct.error as e:
            _refuse(f"a number is out of range or not one: {e}")
    return packed


_pack_append, _pack_attn, _pack_verify = _packer(RopeAppendArgs), _packer(PrefixAttnArgs), _packer(VerifyArgs)
_F16, _BF16, _F32, _F64, _I32, _U8 = torch.float16, torch.bfloat16, torch.float32, torch.float64, torch.int32, torch.uint8
_empty_like = torch.empty_like
# the raw handle of torch's current stream without building a Stream object, where torch has it
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
_fn = None


def _lib():
    global _fn
    if _fn is None:
        L = lib()
        L.z2b_rope_init.argtypes = [_P, ctypes.c_int, ctypes.c_int, ctypes.c_double, ctypes.c_int, ctypes.c_double, ctypes.c_int]
        for f in (L.z2b_rope_append, L.z2b_prefix_attention, L.z2b_verify_drafts):
            f.argtypes, f.restype = [_P, _P], ctypes.c_int
        L.z2b_prefix_attention_workspace.argtypes, L.z2b_prefix_attention_workspace.restype = [_P], _Z
        _fn = L
    return _fn


def _raise(rc):
    raise Z2BError(rc, _lib().z2b_last_error().decode(errors="replace"))


def _refuse(msg):
    raise Z2BError(1, msg)


def _ints(t, n, idx, what):
    """Address of an int32 array of n on device idx, without gaps."""
    if t.dtype is _I32 and t.get_device() == idx and t.is_contiguous() and t.dim() == 1 and t.numel() == n:
        return t.data_ptr()
    _refuse(f"{what}: a contiguous int32 tensor of {n} on device {idx} is wanted")


def check(err):
    """Raise Z2BError when a kernel has recorded a finding in `err` (synchronises)."""
    bits = int(err.item())
    if bits:
        names = [n for b, n in ((TIMEOUT, "a bounded wait ran out"), (BAD_INDEX, "an offset, length or token id out of range"),
                                (BAD_PAGE, "a page id outside the cache")) if bits & b]
        raise Z2BError(6, ", ".join(names))


class Rope:
    """A rotation of the first rot_dim dims of a head: pairs (2i, 2i + 1) ("interleaved") or
    (i, i + rot_dim / 2) ("half"), position s turning pair i by s * base^(-2i / rot_dim), scaled for
    long contexts by "linear", "ntk" or "by_parts" (z2b_ops.h). Host data, usable on any device."""

    def __init__(self, rot_dim: int, base: float = 10000.0, layout: str = "interleaved", scaling: str = "none",
                 factor: float = 1.0, orig_ctx: int = 0):
        if layout not in _LAYOUT or scaling not in _SCALING:
            _refuse("rope: layout is 'interleaved' or 'half', scaling 'none', 'linear', 'ntk' or 'by_parts'")
        self.table = RopeTable()
        self._at = ctypes.addressof(self.table)
        rc = _lib().z2b_rope_init(self._at, int(rot_dim), _LAYOUT[layout], float(base),
                                  _SCALING[scaling], float(factor), int(orig_ctx))
        if rc:
            _raise(rc)


class PagedKV:
    """The K and V pages of one layer: tensors [pages][page_len][kv heads][head_dim] (any strides
    with the dims of a head together), f16 or bf16, of the same strides."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        if k.dim() != 4 or k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype or k.device != v.device:
            _refuse("kv: k and v must be 4-dimensional and alike in shape, strides, type and device")
        if k.dtype not in (torch.float16, torch.bfloat16) or not k.is_cuda:
            _refuse("kv: f16 or bf16 CUDA tensors are wanted")
        if k.stride(3) != 1 or 0 in k.shape:
            _refuse("kv: the dims of a head must be contiguous, and no size zero")
        self.k, self.v, self.device, self.dtype = k, v, k.device, k.dtype
        self.n_pages, self.page_len, self.n_head_kv, self.head_dim = k.shape
        # a stride along a dimension of one says nothing: it reads as if packed
        sp, sr, sh, _ = k.stride()
        sh = sh if self.n_head_kv > 1 else self.head_dim
        sr = sr if self.page_len > 1 else sh * self.n_head_kv
        sp = sp if self.n_pages > 1 else self.page_len * self.n_head_kv * self.head_dim
        self.view = PagedKVView(k.data_ptr(), v.data_ptr(), _TYPE[k.dtype], *k.shape, sp, sr, sh)
        self._idx, self._at, self._scale = k.get_device(), ctypes.addressof(self.view), 1.0 / math.sqrt(self.head_dim)
        self._bytes = {}                # workspace bytes by sizes


def _rows(t, n, heads, kv, dtype, what):
    """Strides and address of rows [n][heads][head_dim] on the cache's device."""
    s, r = t.shape, t.stride()
    if len(s) != 3 or s[0] != n or s[1] != heads or s[2] != kv.head_dim:
        _refuse(f"{what}: [{n}][{heads}][{kv.head_dim}] is wanted")
    if r[2] != 1 or t.dtype is not dtype or t.get_device() != kv._idx:
        _refuse(f"{what}: wrong device or type, or the dims of a head are not contiguous")
    return r[0], r[1], t.data_ptr()


def _table(t, n_seq, idx):
    s = t.shape
    if t.dtype is not _I32 or t.get_device() != idx or len(s) != 2 or s[0] != n_seq:
        _refuse(f"page_table: an int32 tensor [{n_seq}][pages] on device {idx} is wanted")
    r = t.stride()
    if r[1] != 1 and s[1] > 1:
        _refuse("page_table: the pages of a stream must be contiguous")
    return t.data_ptr(), r[0], s[1]


def rope_append(rope: Rope | None, kv: PagedKV, q, k, v, row_off, seq_len, page_table, prefix_len: int = 0, pos=None,
                out=None, err=None):
    """Rotate q and k and append k and v to the pages (z2b_rope_append); returns the rotated q
    (`out` when given, which may be q). q may be None (nothing returned), k and v may be None (only
    q turns); rope None stores unrotated keys. `pos` [rows] int32 replaces the positions prefix_len +
    cache row. A new result's padding rows are not written."""
    lead = q if q is not None else k
    if lead is None or (k is None) != (v is None):
        _refuse("rope_append: q, or k and v, or all three")
    if lead.dim() != 3:
        _refuse("rope_append: rows [rows][heads][head_dim] are wanted")
    idx, dt, n, nh = kv._idx, lead.dtype, lead.shape[0], 0
    code = _TYPE.get(dt)
    if code is None:
        _refuse("rope_append: f32, f16 or bf16 rows are wanted")
    n_seq = seq_len.numel()
    qr = qh = qp = outr = outh = outp = kr = kh = kp = vr = vh = vp = 0
    if q is not None:
        nh = q.shape[1]
        qr, qh, qp = _rows(q, n, nh, kv, dt, "q")
        if out is None:
            out = _empty_like(q)
            outr, outh, _ = out.stride()
            outp = out.data_ptr()
        else:
            outr, outh, outp = _rows(out, n, nh, kv, dt, "out")
    elif out is not None:
        _refuse("rope_append: out without q")
    if k is not None:
        kr, kh, kp = _rows(k, n, kv.n_head_kv, kv, dt, "k")
        vr, vh, vp = _rows(v, n, kv.n_head_kv, kv, dt, "v")
    tab, tstride, pages = _table(page_table, n_seq, idx)
    rc = _lib().z2b_rope_append(
        _pack_append(idx, code, n, n_seq, nh, prefix_len, rope._at if rope is not None else 0, kv._at, qp, outp, kp, vp,
                     qr, qh, outr, outh, kr, kh, vr, vh, _ints(row_off, n_seq + 1, idx, "row_off"),
                     _ints(seq_len, n_seq, idx, "seq_len"), tab, tstride, pages,
                     0 if pos is None else _ints(pos, n, idx, "pos"), 0 if err is None else _ints(err, 1, idx, "err")),
        _raw_stream(idx))
    if rc:
        _raise(rc)
    return out


def prefix_attention(kv: PagedKV, q, row_off, seq_len, page_table, prefix_pages=None, prefix_len: int = 0, scale=None,
                     out=None, lse=None, err=None):
    """Attention of every row over the shared prefix (`prefix_pages`, `prefix_len` rows) and its
    stream's own rows up to its own (z2b_prefix_attention). q [rows][heads][head_dim] of the cache's
    type; scale defaults to 1 / sqrt(head_dim). Returns out, or (out, lse) when lse is True or an f32
    tensor [rows][heads]. Padding rows of new results are not written."""
    if q.dim() != 3:
        _refuse("q: rows [rows][heads][head_dim] are wanted")
    idx, n_seq = kv._idx, seq_len.numel()
    n, nh, _ = q.shape
    qr, qh, qp = _rows(q, n, nh, kv, kv.dtype, "q")
    if out is None:
        out = _empty_like(q)
        outr, outh, _ = out.stride()
        outp = out.data_ptr()
    else:
        outr, outh, outp = _rows(out, n, nh, kv, kv.dtype, "out")
    if lse is True:
        lse = q.new_empty((n, nh), dtype=_F32)
    elif lse is False:
        lse = None
    elif lse is not None and (lse.dtype is not _F32 or lse.shape != (n, nh) or lse.get_device() != idx or not lse.is_contiguous()):
        _refuse("lse: a contiguous f32 tensor [rows][heads] on the cache's device is wanted")
    shared = 0
    if prefix_len > 0:
        if prefix_pages is None or prefix_pages.numel() * kv.page_len < prefix_len:
            _refuse("prefix_pages: a page for every page_len rows of the prefix is wanted")
        shared = _ints(prefix_pages, prefix_pages.numel(), idx, "prefix_pages")
    tab, tstride, pages = _table(page_table, n_seq, idx)
    if scale is None:
        scale = kv._scale
    off, lens, flag = _ints(row_off, n_seq + 1, idx, "row_off"), _ints(seq_len, n_seq, idx, "seq_len"), 0 if err is None else _ints(err, 1, idx, "err")
    L = _lib()
    need = kv._bytes.get((n, n_seq, nh, prefix_len, pages))
    if need is None:
        need = L.z2b_prefix_attention_workspace(
            _pack_attn(idx, n, n_seq, nh, prefix_len, scale, kv._at, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, pages, 0, 0, 0, 0))
        if len(kv._bytes) > 1000:
            kv._bytes.clear()
        kv._bytes[(n, n_seq, nh, prefix_len, pages)] = need
    ws = q.new_empty((need,), dtype=_U8)            # 0: the call below says what is wrong with the sizes
    rc = L.z2b_prefix_attention(
        _pack_attn(idx, n, n_seq, nh, prefix_len, scale, kv._at, qp, outp, 0 if lse is None else lse.data_ptr(), qr, qh, outr,
                   outh, off, lens, tab, tstride, pages, shared, ws.data_ptr(), need, flag), _raw_stream(idx))
    if rc:
        _raise(rc)
    return out if lse is None else (out, lse)


def verify_drafts(p, q, draft, u_accept, u_draw, n_draft=None, err=None):
    """Keep or replace drafted frames (z2b_verify_drafts). p [streams][drafts + 1][codebooks][vocab]:
    the target's probabilities; q [streams][drafts][codebooks][vocab]: the draft's, or None when it put
    all on the drafted token; draft int32 and u_accept float64 [streams][drafts][codebooks]; u_draw
    float64 [streams][drafts + 1][codebooks]; n_draft [streams] int32. Returns (tokens int32
    [streams][drafts + 1][codebooks], accepted frames int32 [streams]); tokens behind the frame after
    the accepted ones are -1."""
    idx, code, dt = p.get_device(), _TYPE.get(p.dtype), p.dtype
    if p.dim() != 4 or idx < 0 or code is None or p.shape[1] < 1:
        _refuse("p: a CUDA tensor [streams][drafts + 1][codebooks][vocab], f32, f16 or bf16, is wanted")
    B, N1, C, V = p.shape
    N, ps, qs, qp = N1 - 1, p.stride(), (0, 0, 0), 0
    if ps[3] != 1 and V > 1:
        _refuse("p: the vocabulary must be contiguous")
    if q is not None:
        qs, qp = q.stride(), q.data_ptr()
        if q.shape != (B, N, C, V) or q.dtype is not dt or q.get_device() != idx or (qs[3] != 1 and V > 1):
            _refuse(f"q: [{B}][{N}][{C}][{V}] of p's type is wanted, the vocabulary contiguous")
    if draft.dtype is not _I32 or draft.get_device() != idx or draft.shape != (B, N, C) or not draft.is_contiguous():
        _refuse(f"draft: a contiguous int32 tensor [{B}][{N}][{C}] is wanted")
    if u_accept.dtype is not _F64 or u_accept.get_device() != idx or u_accept.shape != (B, N, C) or not u_accept.is_contiguous():
        _refuse(f"u_accept: a contiguous float64 tensor [{B}][{N}][{C}] is wanted")
    if u_draw.dtype is not _F64 or u_draw.get_device() != idx or u_draw.shape != (B, N1, C) or not u_draw.is_contiguous():
        _refuse(f"u_draw: a contiguous float64 tensor [{B}][{N1}][{C}] is wanted")
    tokens = _empty_like(u_draw, dtype=_I32)
    kept = draft.new_empty((B,))
    rc = _lib().z2b_verify_drafts(
        _pack_verify(idx, code, B, N, C, V, p.data_ptr(), qp, draft.data_ptr(),
                     0 if n_draft is None else _ints(n_draft, B, idx, "n_draft"), u_accept.data_ptr(), u_draw.data_ptr(),
                     tokens.data_ptr(), kept.data_ptr(), ps[0], ps[1], ps[2], qs[0], qs[1], qs[2],
                     0 if err is None else _ints(err, 1, idx, "err")), _raw_stream(idx))
    if rc:
        _raise(rc)
    return tokens, kept
