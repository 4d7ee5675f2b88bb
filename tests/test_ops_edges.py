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


# ------------------------------------------------------------------------- shared memory
NO_DEVICE = 1 << 20                 # what is not refused ends at the device, which is not there


def _elements(at, dims):
    """Element numbers of a box as a list."""
    out = [at]
    for stride, n in dims:
        out = [x + stride * i for x in out for i in range(n)]
    return out


def _append_boxes(q, o, k, v, kc, vc, kv_strides, rows=3, heads=2, nkv=2, hd=4, pages=2, page_len=3):
    """rope_append with arrays (first element, row stride, head stride) of f16 in one address space of
    elements, the cache's two (first element) with strides (page, row, head)."""
    at = lambda e: (1 << 30) + 2 * e  # noqa: E731
    ps, rs, hs = kv_strides
    view = ops.PagedKVView(k=at(kc), v=at(vc), type=1, n_pages=pages, page_len=page_len, n_head_kv=nkv, head_dim=hd,
                           page_stride=ps, row_stride=rs, head_stride=hs)
    a = args.RopeAppendArgs(device=NO_DEVICE, type=1, n_rows=rows, n_seq=1, n_head=heads, kv=ctypes.addressof(view), q=at(q[0]),
                            q_out=at(o[0]), k=at(k[0]), v=at(v[0]), q_row=q[1], q_head=q[2], o_row=o[1], o_head=o[2], k_row=k[1],
                            k_head=k[2], v_row=v[1], v_head=v[2], row_off=BUF, seq_len=BUF, page_table=BUF, table_stride=2, max_pages=2)
    rc, msg = _call("z2b_rope_append", a)
    qe, oe = (_elements(x[0], [(x[1], rows), (x[2], heads), (1, hd)]) for x in (q, o))
    ke, ve = (_elements(x[0], [(x[1], rows), (x[2], nkv), (1, hd)]) for x in (k, v))
    ce, de = (_elements(x, [(ps, pages), (rs, page_len), (hs, nkv), (1, hd)]) for x in (kc, vc))
    shared = len(set(oe)) < len(oe) or (qe != oe and set(qe) & set(oe)) or set(oe) & set(ke + ve) or len(set(ce)) < len(ce) or set(ce) & set(de)
    return rc, msg, bool(shared)


def test_append_refuses_shared_memory_and_nothing_else():
    """Against a count of the elements themselves: boxes at random places and strides, nested and not."""
    import random
    rng = random.Random(5)
    seen = {True: 0, False: 0}
    for n in range(4000):
        pick = lambda far: (rng.randrange(far), rng.choice((0, 4, 5, 8, 12, 16, 24, 40, 100)), rng.choice((0, 3, 4, 8, 12, 13, 50)))  # noqa: E731
        q = (rng.randrange(40), rng.choice((8, 16, 24, 32)), rng.choice((4, 8, 12, 24)))
        o = q if n % 4 == 0 else pick(120) if n % 4 == 1 else (q[0] + rng.randrange(-8, 300), q[1], q[2])
        k, v = ((rng.randrange(60, 400), q[1], 4) for _ in range(2))
        cache = rng.choice(((24, 8, 4), (48, 16, 4), (24, 4, 12), (48, 8, 4), (20, 8, 4), (0, 8, 4), (7, 21, 4), (26, 9, 4), (9, 18, 4)))
        rc, msg, shared = _append_boxes(q, o, k, v, 1000, 1000 + rng.choice((0, 4, 8, 12, 24, 48, 100, -24, 23)), cache)
        seen[shared] += 1
        assert (rc == ARG) == shared, (q, o, k, v, cache, msg)
        assert not shared or "share memory" in msg or "lies across" in msg
    assert min(seen.values()) > 300


def test_append_takes_slices_of_one_buffer():
    """q turned in place, k and v beside it, and keys and values of one cache buffer in turn: by page, by row, by head."""
    q, k, v = (0, 24, 4), (8, 24, 4), (16, 24, 4)
    for cache, apart in (((48, 8, 4), 24), ((48, 16, 4), 8), ((48, 16, 8), 4), ((24, 8, 4), 48)):
        rc, msg, shared = _append_boxes(q, q, k, v, 1000, 1000 + apart, cache)
        assert not shared and rc != ARG, msg


def test_attention_refuses_results_that_share_memory():
    view = dict(n_head_kv=2, head_dim=64)
    for (row, head), ok in (((256, 64), True), ((64, 192), True), ((192, 128), True), ((128, 64), True), ((96, 64), False), ((64, 128), False), ((0, 64), False), ((256, 32), False)):
        a = _attn(_view(**view), device=NO_DEVICE, n_rows=3, n_head=2, o_row=row, o_head=head, workspace_bytes=1 << 40)
        rc, msg = _call("z2b_prefix_attention", a)
        assert (rc == ARG) == (not ok), (row, head, msg)
    # the keys may be the values there, and pages may repeat: they are only read
    a = _attn(_view(page_stride=0, **view), device=NO_DEVICE, workspace_bytes=1 << 40)
    assert _call("z2b_prefix_attention", a)[0] != ARG


def test_append_takes_rows_that_run_backwards():
    """Negative strides of q, q_out, k and v name the same boxes from their other end."""
    import random
    rng = random.Random(6)
    seen = {True: 0, False: 0}
    for _ in range(3000):
        pick = lambda: (rng.randrange(200, 360), rng.choice((-24, -8, 8, 16, 24)), rng.choice((-12, -4, 4, 8, 12)))  # noqa: E731
        q, o, k, v = pick(), pick(), pick(), pick()
        o = q if rng.random() < 0.2 else o
        rc, msg, shared = _append_boxes(q, o, k, v, 1000, 1024, (48, 8, 4))
        seen[shared] += 1
        assert (rc == ARG) == shared, (q, o, k, v, msg)
    assert min(seen.values()) > 300
    for row, head, ok in ((-256, 64, True), (-256, -64, True), (-64, 64, False), (-96, -64, False)):
        a = _attn(_view(), device=NO_DEVICE, n_rows=3, n_head=2, o_row=row, o_head=head, workspace_bytes=1 << 40)
        assert (_call("z2b_prefix_attention", a)[0] == ARG) == (not ok)


def test_a_context_that_is_not_read_may_be_anything():
    assert ops.Rope(64, orig_ctx=-1).table.step[1] == ops.Rope(64).table.step[1]
