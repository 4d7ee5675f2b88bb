"""Refusals of the device-buffer operators (include/z2b_ops.h) at the edges of what their arguments
allow, on the host."""
from __future__ import annotations

import ctypes
import math

import pytest

torch = pytest.importorskip("torch")

import z2b.ops as ops
import z2b.runtime as R
from tests import ops_args as args
from tests.test_ops_refusals import ARG, BUF, UNSUPPORTED, _append, _attn, _call, _view


@pytest.mark.parametrize("kw", [
    dict(rot_dim=4, scaling="ntk", factor=1e-200), dict(rot_dim=4, scaling="ntk", factor=1e200),     # base 0, infinite
    dict(scaling="linear", factor=5e-324), dict(scaling="linear", factor=1e-320),                    # frequencies overflow
    dict(scaling="by_parts", factor=1e-320, orig_ctx=8192),
    dict(scaling="by_parts", factor=1e-5, orig_ctx=8192),                                            # cos and sin times -0.15
    dict(base=math.inf), dict(scaling="linear", factor=math.inf)], ids=str)
def test_rotations_that_overflow(kw):
    with pytest.raises(R.Z2BError) as e:
        ops.Rope(**{"rot_dim": 64, **kw})
    assert e.value.rc == ARG


@pytest.mark.parametrize("kw", [dict(scaling="ntk", factor=0.5), dict(rot_dim=4, scaling="ntk", factor=1e-3), dict(scaling="linear", factor=1e-6), dict(scaling="linear", factor=1e300),
                                dict(scaling="by_parts", factor=0.5, orig_ctx=8192), dict(base=1e300),
                                dict(scaling="by_parts", factor=1e300, orig_ctx=8192)], ids=str)
def test_rotations_at_the_edge(kw):
    """Factors below 1 and far ones that still have a table."""
    t = ops.Rope(**{"rot_dim": 64, **kw}).table
    assert t.rot_dim == kw.get("rot_dim", 64) and math.isfinite(t.mag) and t.mag > 0


@pytest.mark.parametrize("kw", [dict(rot_dim=2 ** 32 + 64), dict(rot_dim=-2 ** 32 + 64), dict(scaling="by_parts", factor=2.0, orig_ctx=2 ** 32 + 8192),
                                dict(scaling="by_parts", factor=2.0, orig_ctx=2 ** 64)], ids=str)
def test_rotation_sizes_beyond_32_bits(kw):
    """Numbers that would wrap to others on their way into C."""
    with pytest.raises(R.Z2BError):
        ops.Rope(**{"rot_dim": 64, **kw})


def test_head_numbers_that_32_bits_do_not_divide():
    """Head numbers are divided by the group size in 32 bits: n_head times the group stays below 2^32.
    8191 query heads to each of 64 key heads still fit, of 65 they do not."""
    L = args.library()
    for nkv, fits in ((64, True), (65, False)):
        n = 8191 * nkv
        a = _attn(_view(n_head_kv=nkv, head_dim=16, row_stride=16 * nkv, head_stride=16, page_stride=256 * nkv), n_rows=1, n_seq=1,
                  n_head=n, q_row=16 * n, q_head=16, o_row=16 * n, o_head=16)
        assert (L.z2b_prefix_attention_workspace(ctypes.addressof(a)) > 0) == fits
        if not fits:
            assert _call("z2b_prefix_attention", a)[0] == UNSUPPORTED
