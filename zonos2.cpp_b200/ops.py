"""The operators of include/z2b_ops.h on torch CUDA tensors.

``rope_append``, ``prefix_attention`` and ``verify_drafts`` run on the tensors' device, on
torch's current stream of that device, allocate their outputs (and workspace) through torch
and neither synchronise nor copy to the host, so they can be captured into CUDA graphs.
Every refusal raises ``Z2BError``, as in ``z2b.runtime``. ``err``, where given, is an int32
tensor of one element on the device that the kernels OR ``BAD_INDEX``, ``BAD_PAGE`` and
``TIMEOUT`` into; ``check(err)`` reads it (which synchronises) and raises.

Rows are packed over the streams: stream b owns rows [row_off[b], row_off[b + 1]) of q
[rows][heads][head_dim], rows ahead of row_off[0] and from row_off[-1] on are padding and stay as they
are, seq_len[b] counts the stream's cached rows with the new ones, and page_table[b] lists its pages.
There is no backward pass and no forward-mode gradient: tensors that want one or carry a tangent are
refused, and autograd does not see what is written in place (the pages, `out`, `lse`).
"""
from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd import forward_ad

try:
    from . import _ops                  # the compiled binding, built with the library
except ImportError as e:
    raise ImportError(f"z2b.ops: its compiled binding _ops.so is missing or was built against another torch ({e}); "
                      "build it with `python zonos2.cpp_b200/build.py ops`") from e
from .runtime import Z2BError, lib

TIMEOUT, BAD_INDEX, BAD_PAGE = 1, 2, 4
_TYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
_LAYOUT = {"interleaved": 0, "half": 1}
_SCALING = {"none": 0, "linear": 1, "ntk": 2, "by_parts": 3}

_I, _L, _P, _F = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p, ctypes.c_float


class RopeTable(ctypes.Structure):
    """z2b_rope."""
    _fields_ = [("rot_dim", _I), ("layout", _I), ("mag", _F), ("reserved", _I), ("step", ctypes.c_uint64 * 128)]


class PagedKVView(ctypes.Structure):
    """z2b_paged_kv."""
    _fields_ = [("k", _P), ("v", _P), ("type", _I), ("n_pages", _I), ("page_len", _I), ("n_head_kv", _I),
                ("head_dim", _I), ("page_stride", _L), ("row_stride", _L), ("head_stride", _L)]


_rope_append, _prefix_attention, _verify_drafts = _ops.rope_append, _ops.prefix_attention, _ops.verify_drafts
_ops.set_error_class(Z2BError)


def _refuse(msg):
    raise Z2BError(1, msg)


def check(err):
    """Raise Z2BError when a kernel has recorded a finding in `err` (synchronises)."""
    bits = int(err.item())
    if bits:
        names = [n for b, n in ((TIMEOUT, "a bounded wait ran out"), (BAD_INDEX, "an offset, length, token id or number drawn with out of range"),
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
        if not all(-2 ** 31 <= int(x) < 2 ** 31 for x in (rot_dim, orig_ctx)):      # ctypes would wrap them
            _refuse("rope: rot_dim and orig_ctx are 32-bit numbers")
        self.table = RopeTable()
        self._at = ctypes.addressof(self.table)
        f = lib().z2b_rope_init
        f.argtypes = [_P, ctypes.c_int, ctypes.c_int, ctypes.c_double, ctypes.c_int, ctypes.c_double, ctypes.c_int]
        rc = f(self._at, int(rot_dim), _LAYOUT[layout], float(base), _SCALING[scaling], float(factor), int(orig_ctx))
        if rc:
            raise Z2BError(rc, lib().z2b_last_error().decode(errors="replace"))
        self._args = (rot_dim, base, layout, scaling, factor, orig_ctx)

    def __reduce__(self):               # a copy has a table, and its address, of its own
        return Rope, self._args


class PagedKV:
    """The K and V pages of one layer: tensors [pages][page_len][kv heads][head_dim] (any strides
    with the dims of a head together), f16 or bf16, of the same strides. What rope_append stores to must
    not share memory: neither keys with values nor expanded pages."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        if k.dim() != 4 or k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype or k.device != v.device:
            _refuse("kv: k and v must be 4-dimensional and alike in shape, strides, type and device")
        if k.dtype not in (torch.float16, torch.bfloat16) or not k.is_cuda:
            _refuse("kv: f16 or bf16 CUDA tensors are wanted")
        if k.stride(3) != 1 or 0 in k.shape:
            _refuse("kv: the dims of a head must be contiguous, and no size zero")
        if k.requires_grad or v.requires_grad or any(forward_ad.unpack_dual(x).tangent is not None for x in (k, v)):
            _refuse("kv: the pages are written in place, without a gradient")
        self.k, self.v, self.device, self.dtype = k, v, k.device, k.dtype
        self.n_pages, self.page_len, self.n_head_kv, self.head_dim = k.shape
        # a stride along a dimension of one says nothing: it reads as if packed
        sp, sr, sh, _ = k.stride()
        sh = sh if self.n_head_kv > 1 else self.head_dim
        sr = sr if self.page_len > 1 else sh * self.n_head_kv
        sp = sp if self.n_pages > 1 else self.page_len * self.n_head_kv * self.head_dim
        self.view = PagedKVView(k.data_ptr(), v.data_ptr(), _TYPE[k.dtype], *k.shape, sp, sr, sh)
        self._idx, self._at, self._scale = k.get_device(), ctypes.addressof(self.view), 1.0 / math.sqrt(self.head_dim)

    def __reduce__(self):               # a copy's view is of the copied tensors
        return PagedKV, (self.k, self.v)


def rope_append(rope: Rope | None, kv: PagedKV, q, k, v, row_off, seq_len, page_table, prefix_len: int = 0, pos=None,
                out=None, err=None):
    """Rotate q and k and append k and v to the pages (z2b_rope_append); returns the rotated q
    (`out` when given, which may be q, or lie apart from q, k and v). q may be None (nothing returned), k
    and v may be None (only q turns); rope None stores unrotated keys. `pos` [rows] int32 replaces the
    positions prefix_len + cache row. A new result is contiguous, and its padding rows are not written."""
    return _rope_append(rope._at if rope is not None else 0, kv._at, kv._idx, q, k, v, row_off, seq_len, page_table, prefix_len,
                        pos, out, err)


def prefix_attention(kv: PagedKV, q, row_off, seq_len, page_table, prefix_pages=None, prefix_len: int = 0, scale=None,
                     out=None, lse=None, err=None):
    """Attention of every row over the shared prefix (`prefix_pages`, `prefix_len` rows) and its
    stream's own rows up to its own (z2b_prefix_attention). q [rows][heads][head_dim] of the cache's
    type; scale defaults to 1 / sqrt(head_dim); out may be q. Returns out, or (out, lse) when lse is
    True or an f32 tensor [rows][heads]. New results are contiguous, and their padding rows are not
    written."""
    return _prefix_attention(kv._at, kv._idx, q, row_off, seq_len, page_table, prefix_pages, prefix_len,
                             kv._scale if scale is None else scale, out, lse, err)


def verify_drafts(p, q, draft, u_accept, u_draw, n_draft=None, err=None):
    """Keep or replace drafted frames (z2b_verify_drafts). p [streams][drafts + 1][codebooks][vocab]:
    the target's probabilities; q [streams][drafts][codebooks][vocab]: the draft's, or None when it put
    all on the drafted token; draft int32 and u_accept float64 [streams][drafts][codebooks]; u_draw
    float64 [streams][drafts + 1][codebooks], both in [0, 1); n_draft [streams] int32. Returns (tokens int32
    [streams][drafts + 1][codebooks], accepted frames int32 [streams]); tokens behind the frame after
    the accepted ones are -1."""
    return _verify_drafts(p, q, draft, u_accept, u_draw, n_draft, err)
