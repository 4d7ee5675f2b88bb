"""Argument checks of the device-buffer operators (include/z2b_ops.h) and the rotation table,
on the host: every refusal returns its code before a device is touched, and
z2b_last_error() names the fault. The table is checked against 50-digit arithmetic."""
from __future__ import annotations

import ctypes
import decimal
import math

import pytest

torch = pytest.importorskip("torch")

import z2b.ops as ops
import z2b.runtime as R
from tests import ops_args as args

ARG, UNSUPPORTED = 1, 7
BUF = 1 << 20                       # an address that is aligned and never read


def _call(fn, a):
    L = args.library()
    return getattr(L, fn)(ctypes.addressof(a), None), L.z2b_last_error().decode()


def _view(**kw):
    d = dict(k=BUF, v=BUF, type=1, n_pages=4, page_len=16, n_head_kv=2, head_dim=64, page_stride=16 * 2 * 64,
             row_stride=128, head_stride=64)
    d.update(kw)
    return ops.PagedKVView(**d)


def _append(view=None, rope=None, **kw):
    v = view or _view()
    d = dict(device=0, type=1, n_rows=3, n_seq=2, n_head=4, prefix_len=0, kv=ctypes.addressof(v), q=BUF, q_out=BUF, k=BUF,
             v=BUF, row_off=BUF, seq_len=BUF, page_table=BUF, table_stride=2, max_pages=2,
             rope=None if rope is None else ctypes.addressof(rope))
    d.update(kw)
    a = args.RopeAppendArgs(**d)
    a._keep = (v, rope)
    return a


def _attn(view=None, **kw):
    v = view or _view()
    d = dict(device=0, n_rows=3, n_seq=2, n_head=4, prefix_len=5, scale=0.1, kv=ctypes.addressof(v), q=BUF, out=BUF,
             q_row=256, q_head=64, o_row=256, o_head=64, row_off=BUF, seq_len=BUF, page_table=BUF, table_stride=2, max_pages=2,
             prefix_pages=BUF, workspace=BUF, workspace_bytes=1 << 40)
    d.update(kw)
    a = args.PrefixAttnArgs(**d)
    a._keep = v
    return a


def _verify(**kw):
    d = dict(device=0, type=0, n_seq=2, max_draft=3, n_codebooks=2, vocab=100, p=BUF, q=BUF, draft=BUF, u_accept=BUF,
             u_draw=BUF, tokens=BUF, n_accepted=BUF)
    d.update(kw)
    return args.VerifyArgs(**d)


BAD_VIEWS = [dict(k=None), dict(v=None), dict(type=0), dict(type=5), dict(n_pages=0), dict(page_len=0), dict(n_head_kv=0),
             dict(head_dim=0), dict(page_stride=-1), dict(k=BUF + 1)]


@pytest.mark.parametrize("bad", BAD_VIEWS, ids=str)
def test_cache_view_refusals(bad):
    for fn, a in (("z2b_rope_append", _append(_view(**bad))), ("z2b_prefix_attention", _attn(_view(**bad)))):
        rc, msg = _call(fn, a)
        assert rc == ARG and msg.startswith("kv:"), msg


@pytest.mark.parametrize("bad,rc", [
    (dict(type=2), ARG), (dict(n_rows=-1), ARG), (dict(n_seq=-1), ARG), (dict(prefix_len=-1), ARG), (dict(q=None), ARG),
    (dict(q_out=None), ARG), (dict(k=None), ARG), (dict(v=None), ARG), (dict(row_off=None), ARG), (dict(seq_len=None), ARG),
    (dict(page_table=None), ARG), (dict(table_stride=1), ARG), (dict(q=BUF + 1), ARG), (dict(row_off=BUF + 2), ARG),
    (dict(kv=None), ARG), (dict(n_seq=4097), UNSUPPORTED)], ids=str)
def test_append_refusals(bad, rc):
    got, msg = _call("z2b_rope_append", _append(**bad))
    assert got == rc and msg


def test_append_refuses_a_rotation_wider_than_the_head():
    r = ops.Rope(128).table
    got, msg = _call("z2b_rope_append", _append(rope=r))
    assert got == ARG and "head_dim" in msg


@pytest.mark.parametrize("view,bad,rc", [
    ({}, dict(n_head=3), ARG), ({}, dict(n_head=0), ARG), ({}, dict(n_rows=-1), ARG), ({}, dict(prefix_len=-1), ARG),
    ({}, dict(q=None), ARG), ({}, dict(out=None), ARG), ({}, dict(q=BUF + 2), ARG), ({}, dict(q_head=65), ARG),
    ({}, dict(prefix_pages=None), ARG), ({}, dict(workspace=None), ARG), ({}, dict(workspace=BUF + 8), ARG),
    ({}, dict(workspace_bytes=64), ARG), ({}, dict(scale=math.nan), ARG), ({}, dict(scale=math.inf), ARG),
    ({}, dict(page_table=None), ARG), ({}, dict(n_seq=4097), UNSUPPORTED),
    ({}, dict(max_pages=1 << 30, table_stride=1 << 30), UNSUPPORTED),
    (dict(head_dim=80), {}, UNSUPPORTED), (dict(head_dim=256), {}, UNSUPPORTED), (dict(page_len=12), {}, UNSUPPORTED),
    (dict(k=BUF + 8), {}, ARG), (dict(row_stride=132), {}, ARG)], ids=str)
def test_attention_refusals(view, bad, rc):
    got, msg = _call("z2b_prefix_attention", _attn(_view(**view), **bad))
    assert got == rc and msg


@pytest.mark.parametrize("bad,rc", [
    (dict(type=3), ARG), (dict(n_seq=-1), ARG), (dict(max_draft=-1), ARG), (dict(n_codebooks=0), ARG), (dict(vocab=0), ARG),
    (dict(p=None), ARG), (dict(draft=None), ARG), (dict(u_accept=None), ARG), (dict(u_draw=None), ARG),
    (dict(tokens=None), ARG), (dict(n_accepted=None), ARG), (dict(u_draw=BUF + 4), ARG), (dict(p=BUF + 2), ARG),
    (dict(vocab=(1 << 30) + 1), UNSUPPORTED), (dict(n_seq=1 << 30), UNSUPPORTED)], ids=str)
def test_verify_refusals(bad, rc):
    got, msg = _call("z2b_verify_drafts", _verify(**bad))
    assert got == rc and msg


def test_nothing_to_do_is_not_an_error():
    """No rows or no streams: the calls return before they need a device."""
    assert _call("z2b_rope_append", _append(n_rows=0))[0] == 0
    assert _call("z2b_rope_append", _append(n_seq=0))[0] == 0
    assert _call("z2b_rope_append", _append(n_head=0, q=None, q_out=None, k=None, v=None))[0] == 0
    assert _call("z2b_prefix_attention", _attn(n_rows=0))[0] == 0
    assert _call("z2b_verify_drafts", _verify(n_seq=0))[0] == 0


def test_null_arguments():
    L = args.library()
    for fn in ("z2b_rope_append", "z2b_prefix_attention", "z2b_verify_drafts"):
        assert getattr(L, fn)(None, None) == ARG
    assert L.z2b_prefix_attention_workspace(None) == 0
    a = _attn(n_head=3)
    assert L.z2b_prefix_attention_workspace(ctypes.addressof(a)) == 0


def test_workspace_grows_with_the_call():
    L = args.library()

    def size(**kw):
        a = _attn(**kw)
        return L.z2b_prefix_attention_workspace(ctypes.addressof(a))

    assert 0 < size() <= size(n_rows=64, n_seq=64) <= size(n_rows=4096, n_seq=64)


@pytest.mark.parametrize("kw", [
    dict(rot_dim=0), dict(rot_dim=3), dict(rot_dim=258), dict(base=1.0), dict(base=math.nan), dict(layout="other"),
    dict(scaling="other"), dict(scaling="linear", factor=0.0), dict(factor=2.0), dict(scaling="ntk", factor=2.0, rot_dim=2),
    dict(scaling="by_parts", factor=2.0, orig_ctx=0)], ids=str)
def test_rope_refusals(kw):
    with pytest.raises(R.Z2BError):
        ops.Rope(**{"rot_dim": 64, **kw})


@pytest.mark.parametrize("kw", [dict(), dict(base=1e6, rot_dim=128), dict(scaling="linear", factor=4.0),
                                dict(scaling="ntk", factor=2.0), dict(scaling="by_parts", factor=16.0, orig_ctx=8192),
                                dict(rot_dim=2), dict(rot_dim=256, layout="half")], ids=str)
def test_rope_table_against_decimals(kw):
    """Each step is the pair's turns per position: within 2^-52 of it relatively (a few f64
    roundings of pow, of the division by 2 pi and of the scaling: 16 of 2^-53 at most)."""
    kw = {"rot_dim": 64, "base": 10000.0, **kw}
    t = ops.Rope(**kw).table
    d, f = kw["rot_dim"], decimal.Decimal(kw.get("factor", 1.0))
    with decimal.localcontext() as c:
        c.prec = 50
        two_pi = 2 * decimal.Decimal("3.14159265358979323846264338327950288419716939937510")
        base = decimal.Decimal(kw["base"])
        if kw.get("scaling") == "ntk":
            base *= (f.ln() * d / (d - 2)).exp()
        for i in range(d // 2):
            w = (base.ln() * -2 * i / d).exp()
            if kw.get("scaling") == "linear":
                w /= f
            elif kw.get("scaling") == "by_parts":
                keep = min(decimal.Decimal(1), max(decimal.Decimal(0), (kw["orig_ctx"] * w / two_pi - 1) / 31))
                w = w / f * (1 - keep) + w * keep
            want = w / two_pi * 2 ** 64
            # pow amplifies a base's rounding by the exponent (at most 1 here; ln(base) < 16 bounds the rest)
            assert abs(decimal.Decimal(int(t.step[i])) - want) <= want * decimal.Decimal(16 * 2.0 ** -53) + 1
    assert t.mag == pytest.approx(0.1 * math.log(16.0) + 1.0 if kw.get("scaling") == "by_parts" else 1.0, rel=2.0 ** -23)



def test_sizes_that_32_bits_do_not_number():
    """Rows, heads, and the prefix's and the streams' units together."""
    for bad in (dict(n_rows=(1 << 30) + 1), dict(n_head=(1 << 20) + 1)):
        assert _call("z2b_rope_append", _append(**bad))[0] == UNSUPPORTED
    # 2048 tiles of 8 rows, and 2^19 units of 32 keys: 2049 (2^19 + 1) > 2^30 for the prefix or the pages, both over 2^31
    half = dict(n_rows=1 << 13, n_seq=1, n_head=2, max_pages=1, table_stride=1 << 20, prefix_len=1 << 24)
    both = dict(half, max_pages=1 << 20)
    L = args.library()
    for kw, fits in ((half, True), (both, False)):
        a = _attn(_view(n_head_kv=1), **kw)
        assert (L.z2b_prefix_attention_workspace(ctypes.addressof(a)) > 0) == fits
    assert _call("z2b_prefix_attention", _attn(_view(n_head_kv=1), **both))[0] == UNSUPPORTED
    assert _call("z2b_prefix_attention", _attn(scale=3e38))[0] == ARG
