"""The argument structures of include/z2b_ops.h for ctypes, to call the C entries directly."""
from __future__ import annotations

import ctypes

import z2b.runtime as R

_I, _L, _P, _F, _Z = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p, ctypes.c_float, ctypes.c_size_t


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


def library():
    L = R.lib()
    for f in (L.z2b_rope_append, L.z2b_prefix_attention, L.z2b_verify_drafts):
        f.argtypes, f.restype = [_P, _P], ctypes.c_int
    L.z2b_prefix_attention_workspace.argtypes, L.z2b_prefix_attention_workspace.restype = [_P], _Z
    return L
