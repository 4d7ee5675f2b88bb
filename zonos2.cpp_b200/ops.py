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


def _ints(t, shape, device, what):
    """Address of an int32 array on the device, of that shape and without gaps."""
    if t.dtype != torch.int32 or t.shape != shape or t.device != device or not t.is_contiguous():
        _refuse(f"{what}: a contiguous int32 tensor {tuple(shape)} on {device} is wanted")
    return t.data_ptr()


def _err(err, device):
    return None if err is None else _ints(err, (1,), device, "err")


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


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
        rc = _lib().z2b_rope_init(ctypes.addressof(self.table), int(rot_dim), _LAYOUT[layout], float(base),
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
        self.view = PagedKVView(k.data_ptr(), v.data_ptr(), _TYPE[k.dtype], *k.shape, *k.stride()[:3])


def _rows(t, heads, kv, what, dtype=None):
    if t.dim() != 3 or t.shape[2] != kv.head_dim or (heads is not None and t.shape[1] != heads):
        _refuse(f"{what}: [rows][{heads or 'heads'}][{kv.head_dim}] is wanted")
    if t.device != kv.device or t.stride(2) != 1 or (dtype is not None and t.dtype != dtype):
        _refuse(f"{what}: wrong device or type, or the dims of a head are not contiguous")


def _table(page_table, n_seq, kv):
    if page_table.dim() != 2 or page_table.shape[0] != n_seq or page_table.dtype != torch.int32 or \
            page_table.device != kv.device or (page_table.shape[1] > 1 and page_table.stride(1) != 1):
        _refuse("page_table: an int32 tensor [streams][pages] on the cache's device is wanted")
    return page_table.data_ptr(), page_table.stride(0), page_table.shape[1]


def rope_append(rope: Rope | None, kv: PagedKV, q, k, v, row_off, seq_len, page_table, prefix_len: int = 0, pos=None,
                out=None, err=None):
    """Rotate q and k and append k and v to the pages (z2b_rope_append); returns the rotated q
    (`out` when given, which may be q). q may be None (nothing returned), k and v may be None (only
    q turns); rope None stores unrotated keys. `pos` [rows] int32 replaces the positions prefix_len +
    cache row. A new result's padding rows are not written."""
    lead = q if q is not None else k
    if lead is None or (k is None) != (v is None):
        _refuse("rope_append: q, or k and v, or all three")
    dev, n, dt = kv.device, lead.shape[0], lead.dtype
    if dt not in _TYPE:
        _refuse("rope_append: f32, f16 or bf16 rows are wanted")
    n_seq = seq_len.shape[0]
    qs = os_ = ks = vs = (0, 0)
    nh = 0
    if q is not None:
        _rows(q, None, kv, "q")
        nh = q.shape[1]
        if out is None:
            out = torch.empty(q.shape, dtype=dt, device=dev)
        else:
            _rows(out, nh, kv, "out", dt)
            if out.shape[0] != n:
                _refuse("out: as many rows as q are wanted")
        qs, os_ = q.stride(), out.stride()
    elif out is not None:
        _refuse("rope_append: out without q")
    if k is not None:
        _rows(k, kv.n_head_kv, kv, "k", dt)
        _rows(v, kv.n_head_kv, kv, "v", dt)
        if k.shape[0] != n or v.shape[0] != n:
            _refuse("rope_append: q, k and v must have the same rows")
        ks, vs = k.stride(), v.stride()
    tab, tstride, pages = _table(page_table, n_seq, kv)
    a = RopeAppendArgs(
        dev.index, _TYPE[dt], n, n_seq, nh, prefix_len, ctypes.addressof(rope.table) if rope is not None else None,
        ctypes.addressof(kv.view), q.data_ptr() if nh else None, out.data_ptr() if nh else None,
        k.data_ptr() if k is not None else None, v.data_ptr() if v is not None else None,
        qs[0], qs[1], os_[0], os_[1], ks[0], ks[1], vs[0], vs[1],
        _ints(row_off, (n_seq + 1,), dev, "row_off"), _ints(seq_len, (n_seq,), dev, "seq_len"), tab, tstride, pages,
        None if pos is None else _ints(pos, (n,), dev, "pos"), _err(err, dev))
    rc = _lib().z2b_rope_append(ctypes.addressof(a), _stream(dev))
    if rc:
        _raise(rc)
    return out


def prefix_attention(kv: PagedKV, q, row_off, seq_len, page_table, prefix_pages=None, prefix_len: int = 0, scale=None,
                     out=None, lse=None, err=None):
    """Attention of every row over the shared prefix (`prefix_pages`, `prefix_len` rows) and its
    stream's own rows up to its own (z2b_prefix_attention). q [rows][heads][head_dim] of the cache's
    type; scale defaults to 1 / sqrt(head_dim). Returns out, or (out, lse) when lse is True or an f32
    tensor [rows][heads]. Padding rows of new results are not written."""
    dev, n_seq = kv.device, seq_len.shape[0]
    _rows(q, None, kv, "q", kv.dtype)
    n, nh, _ = q.shape
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    else:
        _rows(out, nh, kv, "out", q.dtype)
        if out.shape[0] != n:
            _refuse("out: as many rows as q are wanted")
    if lse is True:
        lse = torch.empty((n, nh), dtype=torch.float32, device=dev)
    elif lse is False:
        lse = None
    if lse is not None and (lse.dtype != torch.float32 or lse.shape != (n, nh) or lse.device != dev or not lse.is_contiguous()):
        _refuse("lse: a contiguous f32 tensor [rows][heads] on the cache's device is wanted")
    need = -(-prefix_len // kv.page_len)
    if prefix_len > 0 and (prefix_pages is None or prefix_pages.dim() != 1 or prefix_pages.shape[0] < need):
        _refuse("prefix_pages: a page for every page_len rows of the prefix is wanted")
    tab, tstride, pages = _table(page_table, n_seq, kv)
    qs, os_ = q.stride(), out.stride()
    a = PrefixAttnArgs(
        dev.index, n, n_seq, nh, prefix_len, 1.0 / math.sqrt(kv.head_dim) if scale is None else scale,
        ctypes.addressof(kv.view), q.data_ptr(), out.data_ptr(), None if lse is None else lse.data_ptr(), qs[0], qs[1],
        os_[0], os_[1], _ints(row_off, (n_seq + 1,), dev, "row_off"), _ints(seq_len, (n_seq,), dev, "seq_len"), tab,
        tstride, pages, _ints(prefix_pages, prefix_pages.shape, dev, "prefix_pages") if prefix_len > 0 else None,
        None, 0, _err(err, dev))
    L, at = _lib(), ctypes.addressof(a)
    a.workspace_bytes = L.z2b_prefix_attention_workspace(at)
    if a.workspace_bytes:
        ws = torch.empty(a.workspace_bytes, dtype=torch.uint8, device=dev)
        a.workspace = ws.data_ptr()
    rc = L.z2b_prefix_attention(at, _stream(dev))
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
    dev = p.device
    if p.dim() != 4 or not p.is_cuda or p.dtype not in _TYPE or (p.shape[3] > 1 and p.stride(3) != 1):
        _refuse("p: a CUDA tensor [streams][drafts + 1][codebooks][vocab], f32, f16 or bf16, is wanted")
    B, N1, C, V = p.shape
    N = N1 - 1
    if N < 0:
        _refuse("p: at least one frame is wanted")
    qs = (0, 0, 0)
    if q is not None:
        if q.shape != (B, N, C, V) or q.dtype != p.dtype or q.device != dev or (V > 1 and q.stride(3) != 1):
            _refuse("q: [streams][drafts][codebooks][vocab] of p's type is wanted")
        qs = q.stride()
    for t, shape, what in ((u_accept, (B, N, C), "u_accept"), (u_draw, (B, N1, C), "u_draw")):
        if t.dtype != torch.float64 or t.shape != shape or t.device != dev or not t.is_contiguous():
            _refuse(f"{what}: a contiguous float64 tensor {shape} on {dev} is wanted")
    ps = p.stride()
    tokens = torch.empty((B, N1, C), dtype=torch.int32, device=dev)
    kept = torch.empty((B,), dtype=torch.int32, device=dev)
    a = VerifyArgs(dev.index, _TYPE[p.dtype], B, N, C, V, p.data_ptr(), q.data_ptr() if q is not None and N else None,
                   _ints(draft, (B, N, C), dev, "draft"), None if n_draft is None else _ints(n_draft, (B,), dev, "n_draft"),
                   u_accept.data_ptr(), u_draw.data_ptr(), tokens.data_ptr(), kept.data_ptr(), ps[0], ps[1], ps[2],
                   qs[0], qs[1], qs[2], _err(err, dev))
    rc = _lib().z2b_verify_drafts(ctypes.addressof(a), _stream(dev))
    if rc:
        _raise(rc)
    return tokens, kept
