"""The device-buffer operators (include/z2b_ops.h) against plain 64-bit restatements, at the
sizes, layouts and masks where they can go wrong, and their findings on bad metadata."""
from __future__ import annotations

import copy
import math

import pytest

torch = pytest.importorskip("torch")

import z2b.ops as ops
import z2b.runtime as R
from tests import ops_ref

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
DEV = "cuda:0"


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _i32(x):
    return torch.as_tensor(x, dtype=torch.int32, device=DEV)


class Streams:
    """Paged streams on the device: caches filled with NaN except the rows before each length."""

    def __init__(self, counts, lens, page, nkv, hd, dtype, prefix=0, heads_first=False, seed=0, pad=0, filled=True):
        g = _gen(seed)
        B = len(counts)
        self.counts, self.lens, self.page, self.prefix = list(counts), list(lens), page, prefix
        self.off = [0]
        for n in counts:
            self.off.append(self.off[-1] + n)
        self.total, self.rows = self.off[-1], self.off[-1] + pad
        per = max(1, -(-max([*lens, 1]) // page))
        np_ = -(-prefix // page)
        order = torch.randperm(B * per + np_ + 2, generator=g)
        self.table = order[: B * per].reshape(B, per).to(torch.int32)
        self.shared = order[B * per: B * per + np_].to(torch.int32)
        shape = (B * per + np_ + 2, page, nkv, hd)
        self.kc, self.vc = (torch.full(shape, math.nan) for _ in range(2))
        for c in (self.kc, self.vc):
            for b in range(B):
                for j in range(lens[b] if filled else 0):
                    c[self.table[b, j // page], j % page] = torch.randn((nkv, hd), generator=g)
            for j in range(prefix):
                c[self.shared[j // page], j % page] = torch.randn((nkv, hd), generator=g)
        self.kc, self.vc = self.kc.to(dtype), self.vc.to(dtype)
        if heads_first:
            dk, dv = (x.transpose(1, 2).contiguous().to(DEV).transpose(1, 2) for x in (self.kc, self.vc))
        else:
            dk, dv = self.kc.to(DEV), self.vc.to(DEV)
        self.kv = ops.PagedKV(dk, dv)
        self.d_off, self.d_lens, self.d_table, self.d_shared = _i32(self.off), _i32(self.lens), self.table.to(DEV), self.shared.to(DEV)
        self.err = torch.zeros(1, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------------- rope_append
def _check_append(s, q, k, v, out, rope_kw, layout, dtype, cdtype, pos=None, qin=None):
    """q in `dtype`, cache in `cdtype`: half a step of the type (eps / 2 of the value), and for the
    f32 arithmetic 2^-20 of |a| + |b|: 1.9e-7 rad of angle (2^-24 half-turns), 1.2e-7 of the sine,
    four f32 roundings (2.4e-7); and |position| 2^-51 of it for the f64 frequency and product on
    both sides. Rows of other streams' pages stay bit for bit."""
    w, mag = ops_ref.freqs(**rope_kw) if rope_kw else (torch.zeros(0, dtype=torch.float64), 1.0)
    kc, vc = s.kc.double().clone(), s.vc.double().clone()
    touched = torch.zeros(s.kc.shape[:2], dtype=torch.bool)

    def near(got, want, src, t, at):
        size = src.double().abs()
        # |a| + |b| of a pair, bounded by the two largest of the head
        slack = size.topk(min(2, size.shape[-1]), -1).values.sum(-1, keepdim=True) * mag * (2.0 ** -20 + abs(at) * 2.0 ** -51)
        tol = want.abs() * torch.finfo(t).eps / 2 + slack + torch.finfo(t).smallest_normal * torch.finfo(t).eps
        assert ((got.double() - want).abs() <= tol).all()

    for b, n in enumerate(s.counts):
        for i in range(n):
            t, r = s.off[b] + i, s.lens[b] - n + i
            at = float(pos[t]) if pos is not None else s.prefix + r
            if q is not None:
                near(out[t].cpu(), ops_ref.rotate(qin[t].cpu().double(), at, w, mag, layout), qin[t].cpu(), dtype, at)
            if k is not None:
                pg = int(s.table[b, r // s.page])
                near(s.kv.k[pg, r % s.page].cpu(), ops_ref.rotate(k[t].cpu().double(), at, w, mag, layout), k[t].cpu(), cdtype, at)
                assert torch.equal(s.kv.v[pg, r % s.page].cpu(), v[t].cpu().to(cdtype))
                touched[pg, r % s.page] = True
    for got, was in ((s.kv.k.cpu(), s.kc), (s.kv.v.cpu(), s.vc)):
        assert torch.equal(torch.nan_to_num(got[~touched], 7.0), torch.nan_to_num(was[~touched], 7.0))


def _rows(s, heads, hd, dtype, seed):
    return torch.randn((s.rows, heads, hd), generator=_gen(seed)).to(dtype).to(DEV)


APPENDS = [
    # counts, lens, page, nh, nkv, hd, type, cache, rope, layout, prefix, heads_first, pad
    ([1], [1], 256, 16, 4, 128, F16, F16, dict(rot=128, base=1e6), "interleaved", 0, False, 0),
    ([5, 0, 3, 1], [9, 4, 3, 33], 16, 8, 2, 64, BF16, BF16, dict(rot=32), "half", 100003, False, 3),
    ([2, 7], [8, 7], 7, 3, 3, 64, F32, F16, dict(rot=64, scaling="linear", factor=4.0), "interleaved", 257, True, 1),
    ([40, 1], [40, 50], 48, 6, 1, 80, F32, BF16, dict(rot=48, scaling="ntk", factor=2.0), "half", 0, False, 0),
    ([3], [10], 5, 2, 1, 20, F16, BF16, dict(rot=10), "interleaved", 12, False, 2),       # one pair at a time
    ([2], [2], 8, 1, 1, 7, F32, F16, dict(rot=4), "half", 3, False, 0),                   # odd head, odd tail
    ([1] * 70, list(range(1, 71)), 32, 4, 2, 32, BF16, F16, dict(rot=32, scaling="by_parts", factor=16.0, orig_ctx=2048), "half",
     5, False, 0),
    ([0, 0, 4, 0], [0, 5, 4, 0], 16, 4, 4, 128, F16, F16, None, "interleaved", 0, False, 1),   # no rotation
    ([300, 200], [300, 900], 64, 4, 1, 256, BF16, BF16, dict(rot=256), "half", 2 ** 31 - 2000, False, 0),
    ([1], [1], 1, 1, 1, 2, F32, BF16, dict(rot=2), "half", 1, False, 0),
]


@pytest.mark.parametrize("case", APPENDS, ids=str)
def test_rope_append(case):
    counts, lens, page, nh, nkv, hd, dtype, cdtype, rkw, layout, prefix, hf, pad = case
    s = Streams(counts, lens, page, nkv, hd, cdtype, heads_first=hf, pad=pad, filled=False)
    s.prefix = prefix
    q, k, v = _rows(s, nh, hd, dtype, 1), _rows(s, nkv, hd, dtype, 2), _rows(s, nkv, hd, dtype, 3)
    rope = ops.Rope(rkw["rot"], layout=layout, **{a: b for a, b in rkw.items() if a != "rot"}) if rkw else None
    out = torch.full_like(q, 5.0)
    got = ops.rope_append(rope, s.kv, q, k, v, s.d_off, s.d_lens, s.d_table, prefix_len=prefix, out=out, err=s.err)
    assert got is out
    ops.check(s.err)
    _check_append(s, q, k, v, out, rkw, layout, dtype, cdtype, qin=q)
    assert (out[s.total:] == 5.0).all()                      # padding stays


def test_rope_append_strides_in_place_positions():
    """q, k and v as slices of one buffer at an odd offset, q turned in place, positions given."""
    s = Streams([4, 2], [6, 2], 16, 2, 64, F16, filled=False)
    for lead in (0, 8, 1):                                    # 16-byte runs, then not
        buf = torch.randn((s.rows, lead + (4 + 2 + 2) * 64 + 8), generator=_gen(9)).to(F16).to(DEV)
        q, k, v = (buf[:, lead + a * 64: lead + b * 64].unflatten(1, (-1, 64)) for a, b in ((0, 4), (4, 6), (6, 8)))
        was = q.clone()
        pos = _i32([0, 5, 2 ** 31 - 1, 7, -3, 1000000])
        rope = ops.Rope(64, layout="half")
        assert ops.rope_append(rope, s.kv, q, k, v, s.d_off, s.d_lens, s.d_table, pos=pos, out=q, err=s.err) is q
        ops.check(s.err)
        _check_append(s, q, k, v, q, dict(rot=64), "half", F16, F16, pos=pos.cpu(), qin=was)


def test_rope_append_parts():
    """Only q (the pages stay), then only k and v."""
    s = Streams([3], [5], 8, 2, 32, F16, filled=False)
    q, k, v = _rows(s, 4, 32, F16, 1), _rows(s, 2, 32, F16, 2), _rows(s, 2, 32, F16, 3)
    rope = ops.Rope(32)
    out = ops.rope_append(rope, s.kv, q, None, None, s.d_off, s.d_lens, s.d_table)
    _check_append(s, q, None, None, out, dict(rot=32), "interleaved", F16, F16, qin=q)
    assert ops.rope_append(rope, s.kv, None, k, v, s.d_off, s.d_lens, s.d_table) is None
    _check_append(s, None, k, v, None, dict(rot=32), "interleaved", F16, F16)


def test_rope_append_bad_metadata():
    """A page id outside the cache, a length below the row count and one past the table: recorded,
    those rows skipped, the others stored."""
    s = Streams([1, 2, 1, 1], [3, 2, 4, 4], 4, 1, 32, F16, filled=False)
    q, k, v = _rows(s, 2, 32, F16, 1), _rows(s, 1, 32, F16, 2), _rows(s, 1, 32, F16, 3)
    rope = ops.Rope(32)
    for bad in (-1, s.kv.n_pages, 2 ** 31 - 1):
        s.err.zero_()
        t = s.d_table.clone()
        t[0, 0] = bad
        ops.rope_append(rope, s.kv, q, k, v, s.d_off, s.d_lens, t, err=s.err)
        assert int(s.err) == ops.BAD_PAGE
        with pytest.raises(R.Z2BError):
            ops.check(s.err)
    for lens in ([3, 1, 4, 4], [3, 2, 5, 4], [3, 2, -1, 4], [3, 2, 2 ** 31 - 1, 4]):
        s.err.zero_()
        ops.rope_append(rope, s.kv, q, k, v, s.d_off, _i32(lens), s.d_table, err=s.err)
        assert int(s.err) & ops.BAD_INDEX
    assert torch.equal(s.kv.v[s.table[3, 0], 3].cpu(), v[4].cpu())
    assert torch.isnan(s.kv.v[s.table[0, 0]]).sum() > 0


# ------------------------------------------------------------------------- prefix_attention
def _check_attention(s, q, out, lse, scale=None):
    """Each probability rounded by half a step (eps / 2) for its product with V, the result by half a
    step again; scores off by 2 hd 2^-24 of sum |q k| (f32 accumulation, doubled for the tensor
    core's alignment), which moves a probability by that much twice (numerator and sum); 2^-18 for
    ex2, the joins and the division."""
    dt, hd = s.kv.dtype, s.kv.head_dim
    want, wlse, spread, most = ops_ref.attention(q.cpu(), s.kv.k.cpu(), s.kv.v.cpu(), s.off, s.lens, s.table, s.shared, s.prefix,
                                                 hd ** -0.5 if scale is None else scale)
    n = s.total
    half, delta = torch.finfo(dt).eps / 2, 4 * hd * 2.0 ** -24 * most + 2.0 ** -18
    got = out[:n].cpu().double()
    assert torch.isfinite(got).all()
    tol = (half + delta) * spread[:n] + half * want[:n].abs() + torch.finfo(dt).smallest_normal
    assert ((got - want[:n]).abs() <= tol).all(), float(((got - want[:n]).abs() - tol).max())
    gl = lse[:n].cpu().double()
    empty = wlse[:n] == -math.inf
    assert torch.equal(gl == -math.inf, empty)
    assert ((gl - wlse[:n]).abs()[~empty] <= delta + wlse[:n].abs()[~empty] * 2.0 ** -22).all()


ATTNS = [
    # counts, lens, page, nh, nkv, hd, type, prefix, heads_first, pad
    ([1], [1], 256, 16, 4, 128, F16, 0, False, 0),                       # one key
    ([1], [1], 256, 16, 4, 128, F16, 1, False, 0),
    ([1, 1], [5, 3], 256, 16, 4, 128, F16, 67, False, 0),
    ([1, 1, 1], [64, 65, 63], 16, 4, 4, 64, BF16, 64, False, 2),         # unit borders
    ([1] * 16, [1 + 37 * i for i in range(16)], 32, 16, 4, 128, F16, 200, False, 0),
    ([5] * 6, [5, 9, 70, 130, 6, 64], 16, 6, 2, 64, BF16, 129, True, 0), # drafts, three heads a key head
    ([3, 0, 1, 2], [200, 0, 40, 2], 48, 8, 1, 32, F16, 65, False, 3),    # ragged, a stream without rows
    ([2, 0, 3], [2, 70, 3], 8, 2, 2, 16, BF16, 33, False, 0),            # small head, pages of 8
    ([40, 1], [100, 300], 24, 4, 2, 64, F16, 10, False, 1),              # a prompt chunk beside a decode row
    ([4, 3], [2, 0], 16, 4, 2, 32, F16, 0, False, 0),                    # rows that see no key at all
    ([4, 3], [2, 0], 16, 4, 2, 32, F16, 9, False, 0),                    # ... and see the prefix alone
    ([1] * 40, [3] * 40, 64, 8, 1, 128, BF16, 300, True, 0),             # many rows of one key head
    ([7] * 3, [7, 20, 64], 16, 7, 1, 128, F16, 17, False, 0),
    ([1], [5000], 64, 2, 1, 128, F16, 0, False, 0),                      # one long stream over many CTAs
    ([20] * 4, [20, 33, 90, 64], 16, 2, 1, 128, BF16, 500, False, 0),
    ([9, 17], [64, 128], 40, 12, 2, 16, F16, 0, False, 0),
    # prefixes of many rows
    ([1] * 20, [2] * 20, 256, 16, 4, 128, F16, 128, False, 0),           # 80 rows a key head, one unit
    ([1] * 33, [1] * 33, 64, 16, 2, 64, BF16, 129, False, 5),            # 264 rows: eight in the second tile
    ([5] * 13, [70] * 13, 16, 6, 2, 64, F16, 257, True, 0),              # 195 rows, pages of 16
    ([1] * 100, [3] * 100, 8, 6, 1, 128, BF16, 1000, False, 0),          # 600 rows, pages of 8
    ([3, 0, 90], [3, 9, 95], 48, 4, 1, 128, F16, 127, False, 9),         # a prompt chunk over the prefix
    ([1] * 65, [1] * 65, 32, 1, 1, 64, BF16, 3000, False, 0),            # one head; 65 rows
]


@pytest.mark.parametrize("case", ATTNS, ids=str)
def test_prefix_attention(case):
    counts, lens, page, nh, nkv, hd, dtype, prefix, hf, pad = case
    s = Streams(counts, lens, page, nkv, hd, dtype, prefix=prefix, heads_first=hf, pad=pad, seed=4)
    q = (torch.randn((s.rows, nh, hd), generator=_gen(5)) * 1.5).to(dtype).to(DEV)
    out, lse = torch.full_like(q, 5.0), torch.full((s.rows, nh), 5.0, device=DEV)
    got = ops.prefix_attention(s.kv, q, s.d_off, s.d_lens, s.d_table, s.d_shared, prefix, out=out, lse=lse, err=s.err)
    assert got[0] is out and got[1] is lse
    ops.check(s.err)
    _check_attention(s, q, out, lse)
    assert (out[s.total:] == 5.0).all() and (lse[s.total:] == 5.0).all()
    again, alse = ops.prefix_attention(s.kv, q, s.d_off, s.d_lens, s.d_table, s.d_shared, prefix, lse=True)
    assert torch.equal(out[: s.total], again[: s.total]) and torch.equal(lse[: s.total], alse[: s.total])


def test_prefix_attention_strides_scale_and_peaks():
    """q and out as slices of wider buffers, a scale of its own, scores far apart (one key takes all)."""
    s = Streams([2, 1], [30, 100], 16, 2, 64, F16, prefix=50, seed=6)
    wide = torch.randn((s.rows, 3, 4, 64), generator=_gen(7)).to(F16).to(DEV) * 8
    q, out = wide[:, 1], torch.zeros((s.rows, 8, 64), dtype=F16, device=DEV)[:, ::2]
    lse = torch.zeros((s.rows, 4), device=DEV)
    ops.prefix_attention(s.kv, q, s.d_off, s.d_lens, s.d_table, s.d_shared, 50, scale=0.7, out=out, lse=lse, err=s.err)
    ops.check(s.err)
    _check_attention(s, q, out, lse, scale=0.7)


def test_prefix_attention_equals_a_private_copy():
    """Streams that share a prefix give what the same streams give with the prefix in their own pages."""
    g = _gen(11)
    lens, P, page, nkv, hd, nh = [3, 20, 64], 80, 16, 2, 64, 4
    s = Streams([1, 2, 1], lens, page, nkv, hd, F16, prefix=P, seed=12)
    q = torch.randn((4, nh, hd), generator=g).to(F16).to(DEV)
    out, lse = ops.prefix_attention(s.kv, q, s.d_off, s.d_lens, s.d_table, s.d_shared, P, lse=True)
    table = torch.cat((s.d_shared[None].expand(3, -1), s.d_table), 1).contiguous()     # P is whole pages
    own, olse = ops.prefix_attention(s.kv, q, s.d_off, s.d_lens + P, table, lse=True)
    # both within the bound of the 64-bit value; here their distance: two roundings each
    assert (out - own).abs().max() <= 4 * torch.finfo(F16).eps and (lse - olse).abs().max() <= 1e-5


def test_prefix_attention_bad_metadata():
    """Bad pages read as zeros, bad lengths and offsets drop their stream: recorded, the others stay."""
    s = Streams([1, 1, 1], [40, 40, 40], 16, 2, 64, F16, prefix=40, seed=8)
    q = torch.randn((3, 4, 64), generator=_gen(1)).to(F16).to(DEV)
    good = ops.prefix_attention(s.kv, q, s.d_off, s.d_lens, s.d_table, s.d_shared, 40)
    for bad in (-1, s.kv.n_pages, 2 ** 31 - 1):
        t = s.d_table.clone()
        t[1, 1] = bad
        s.err.zero_()
        out = ops.prefix_attention(s.kv, q, s.d_off, s.d_lens, t, s.d_shared, 40, err=s.err)
        assert int(s.err) == ops.BAD_PAGE and torch.equal(out[[0, 2]], good[[0, 2]])
        sh = s.d_shared.clone()
        sh[0] = bad
        s.err.zero_()
        ops.prefix_attention(s.kv, q, s.d_off, s.d_lens, s.d_table, sh, 40, err=s.err)
        assert int(s.err) == ops.BAD_PAGE
    for lens in ([40, -1, 40], [40, 49, 40], [40, 2 ** 31 - 1, 40]):
        s.err.zero_()
        out = torch.full_like(q, 5.0)
        ops.prefix_attention(s.kv, q, s.d_off, _i32(lens), s.d_table, s.d_shared, 40, out=out, err=s.err)
        assert int(s.err) == ops.BAD_INDEX and torch.equal(out[[0, 2]], good[[0, 2]])
        assert (out[1] == 5.0).all()
    for off in ([0, 1, 0, 3], [-1, 1, 2, 3], [0, 3, 0, 3], [0, 1, 2, 4]):
        s.err.zero_()
        ops.prefix_attention(s.kv, q, _i32(off), s.d_lens, s.d_table, s.d_shared, 40, err=s.err)
        assert int(s.err) == ops.BAD_INDEX
    torch.cuda.synchronize()


# ------------------------------------------------------------------------- verify_drafts
def _verify_inputs(B, N, C, V, dtype, apart, seed, certain=False):
    g = _gen(seed)
    base = torch.randn((B, N + 1, C, V), generator=g) * 2
    p = torch.softmax(base, -1).to(dtype)
    far = base[:, :N] + apart * torch.randn((B, N, C, V), generator=g)
    q = torch.softmax(far, -1)
    draft = torch.multinomial(q.reshape(-1, V), 1, generator=g).reshape(B, N, C).to(torch.int32) if N else torch.zeros((B, 0, C), dtype=torch.int32)
    u = torch.rand((B, N, C), generator=g, dtype=torch.float64)
    r = torch.rand((B, N + 1, C), generator=g, dtype=torch.float64)
    return p, None if certain else q.to(dtype), draft, u, r


def _verify(p, q, draft, u, r, n=None, err=None):
    d = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    return [x.cpu() for x in ops.verify_drafts(d(p), d(q), d(draft), d(u), d(r), n_draft=d(n), err=err)]


@pytest.mark.parametrize("B,N,C,V,dtype,apart,certain,ragged", [
    (1, 4, 9, 1026, F32, 0.5, False, False), (3, 3, 9, 1026, F32, 0.1, True, True), (5, 2, 1, 5000, F16, 0.7, False, True),
    (2, 6, 2, 40001, F32, 0.3, False, False), (1, 1, 1, 131071, BF16, 0.5, False, False), (40, 3, 9, 257, F32, 0.3, False, True),
    (4, 5, 3, 1, F32, 0.0, False, False), (4, 2, 1, 2, F32, 1.0, False, False), (6, 0, 4, 300, F32, 0.0, True, False),
    (2, 3, 1, 33, F16, 0.0, False, False), (1, 8, 33, 70, F32, 0.05, False, False), (200, 2, 1, 4099, F32, 0.4, True, False)], ids=str)
def test_verify_drafts(B, N, C, V, dtype, apart, certain, ragged):
    p, q, draft, u, r = _verify_inputs(B, N, C, V, dtype, apart, 3, certain)
    n = torch.randint(0, N + 1, (B,), generator=_gen(2)).to(torch.int32) if ragged else None
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = _verify(p, q, draft, u, r, n, err)
    ops.check(err)
    want = ops_ref.verify(p, q, draft, u, r, n)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_verify_borders():
    """Exact borders in dyadic probabilities: a draw takes the first token whose sum EXCEEDS the
    target, a draft is kept below p and refused at it; numbers at 0 and just below 1."""
    p = torch.tensor([0.25, 0.0, 0.25, 0.5, 0.0]).repeat(1, 2, 1, 1)
    draft = torch.zeros((1, 1, 1), dtype=torch.int32)
    one = 1.0 - 2.0 ** -53
    for u in (0.0, 0.25, 0.25 - 2.0 ** -54, one):
        for r in (0.0, 0.25, 0.5, one, 1.0):
            a = (p, None, draft, torch.full((1, 1, 1), u, dtype=torch.float64), torch.full((1, 2, 1), r, dtype=torch.float64))
            got, want = _verify(*a), ops_ref.verify(*a, None)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_verify_equal_rows_and_empty_mass():
    """p = q keeps every draft; q above p everywhere else leaves no mass, so the draw is from p; a row
    without mass has no token (-1); entries that are not numbers count as zero."""
    V = 3000
    p, _, draft, u, r = _verify_inputs(2, 2, 3, V, F32, 0.0, 5)
    got = _verify(p, p[:, :2].contiguous(), draft, u, r)
    assert (got[1] == 2).all() and torch.equal(got[0][:, :2], draft)
    q = p[:, :2] * 2 + 1
    u.fill_(0.9)
    got, want = _verify(p, q, draft, u, r), ops_ref.verify(p, q, draft, u, r, None)
    assert torch.equal(got[0], want[0]) and (got[1] == 0).all()
    z = torch.zeros_like(p)
    got = _verify(z, None, draft, u, r)
    assert (got[0] == -1).all() and (got[1] == 0).all()
    z[..., 17] = 0.5
    z[..., 5] = math.nan
    z[..., 2900] = math.nan
    draft.fill_(5)
    assert (_verify(z, None, draft, u, r)[0][:, 0] == 17).all()


def test_verify_bad_tokens():
    """Token ids and counts out of range are recorded; the token is refused."""
    p, q, draft, u, r = _verify_inputs(3, 2, 2, 100, F32, 0.0, 6)
    u.zero_()
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    for bad in (-1, 100, 2 ** 31 - 1):
        err.zero_()
        d = draft.clone()
        d[1, 1, 0] = bad
        tok, kept = _verify(p, q, d, u, r, None, err)
        assert int(err) == ops.BAD_INDEX and kept.tolist() == [2, 1, 2] and 0 <= int(tok[1, 1, 0]) < 100
    err.zero_()
    kept = _verify(p, q, draft, u, r, torch.tensor([1, -1, 9], dtype=torch.int32), err)[1]
    assert int(err) == ops.BAD_INDEX and kept.tolist() == [1, 0, 2]


def test_verify_strides():
    """Probabilities as slices of wider buffers (a padded vocabulary)."""
    p, q, draft, u, r = _verify_inputs(3, 3, 2, 777, F32, 0.4, 8)
    wp, wq = torch.full((3, 5, 2, 801), 9.0), torch.full((3, 3, 4, 777), 9.0)
    wp[:, :4, :, :777], wq[:, :, 1:3] = p, q
    got = ops.verify_drafts(wp.to(DEV)[:, :4, :, :777], wq.to(DEV)[:, :, 1:3], draft.to(DEV), u.to(DEV), r.to(DEV))
    want = ops_ref.verify(p, q, draft, u, r, None)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


# ------------------------------------------------------------------------- together
def _step(rope, s, x, lens, P, head, drafts, u, r):
    """One pass of one layer: rotate and append, attend, probabilities of every row, verify."""
    q, k, v = x
    B, N = drafts.shape[:2]
    qr = ops.rope_append(rope, s.kv, q, k, v, s.d_off, lens, s.d_table, prefix_len=P)
    out = ops.prefix_attention(s.kv, qr, s.d_off, lens, s.d_table, s.d_shared, P)
    p = torch.softmax(out.flatten(1).float() @ head, -1).reshape(B, N + 1, 3, -1)
    return (out, p) + ops.verify_drafts(p, None, drafts, u, r)


def _step_inputs():
    P, B, N, nh, nkv, hd, V = 40, 5, 3, 4, 2, 64, 50
    s = Streams([N + 1] * B, [N + 1 + 7 * b for b in range(B)], 16, nkv, hd, F16, prefix=P, seed=21)
    g = _gen(22)
    mk = lambda h: torch.randn((s.rows, h, hd), generator=g).to(F16).to(DEV)  # noqa: E731
    x = mk(nh), mk(nkv), mk(nkv)
    head = torch.randn((nh * hd, 3 * V), generator=g).to(DEV) * 0.2
    drafts = torch.randint(0, V, (B, N, 3), generator=g).to(torch.int32).to(DEV)
    u = (torch.rand((B, N, 3), generator=g, dtype=torch.float64) * 0.02).to(DEV)
    r = torch.rand((B, N + 1, 3), generator=g, dtype=torch.float64).to(DEV)
    return s, x, P, head, drafts, u, r


def test_step_together():
    """The three operators as one decode pass over streams with a shared prefix and drafts."""
    s, x, P, head, drafts, u, r = _step_inputs()
    rope = ops.Rope(64, layout="half")
    out, p, tok, kept = _step(rope, s, x, s.d_lens, P, head, drafts, u, r)
    qr = ops.rope_append(rope, s.kv, x[0], None, None, s.d_off, s.d_lens, s.d_table, prefix_len=P)
    lse = ops.prefix_attention(s.kv, qr, s.d_off, s.d_lens, s.d_table, s.d_shared, P, lse=True)[1]
    _check_attention(s, qr, out, lse)
    want = ops_ref.verify(p.cpu(), None, drafts.cpu(), u.cpu(), r.cpu(), None)
    assert torch.equal(tok.cpu(), want[0]) and torch.equal(kept.cpu(), want[1])


def test_step_captured_and_on_other_streams():
    """The pass captured into two graphs that share a memory pool and replayed in turn with new
    lengths, and run on a side stream, gives what the eager pass gives, bit for bit."""
    s, x, P, head, drafts, u, r = _step_inputs()
    rope = ops.Rope(64, layout="half")
    lens = s.d_lens.clone()
    pool = torch.cuda.graph_pool_handle()
    _step(rope, s, x, lens, P, head, drafts, u, r)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            res = _step(rope, s, x, lens, P, head, drafts, u, r)
        graphs.append((g, res))
    for shift in (0, 3, -2):
        lens.copy_((s.d_lens + shift).clamp(min=4, max=int(s.table.shape[1]) * 16))
        for g, res in graphs:
            g.replay()
            got = [t.clone() for t in res]
            torch.cuda.synchronize()
            want = _step(rope, s, x, lens, P, head, drafts, u, r)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _step(rope, s, x, lens, P, head, drafts, u, r)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_calls_at_once():
    """Two streams running the operator at the same time, each with its own workspace."""
    a = Streams([1] * 8, [200] * 8, 16, 2, 128, F16, prefix=300, seed=31)
    q = torch.randn((8, 8, 128), generator=_gen(1)).to(F16).to(DEV)
    want = ops.prefix_attention(a.kv, q, a.d_off, a.d_lens, a.d_table, a.d_shared, 300)
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(20):
        for st in sides:
            with torch.cuda.stream(st):
                got.append(ops.prefix_attention(a.kv, q, a.d_off, a.d_lens, a.d_table, a.d_shared, 300))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)


def test_python_refusals():
    """What the binding refuses before the library sees it."""
    s = Streams([1], [4], 16, 2, 64, F16)
    q = torch.zeros((1, 4, 64), dtype=F16, device=DEV)
    k = torch.zeros((1, 2, 64), dtype=F16, device=DEV)
    meta = (s.d_off, s.d_lens, s.d_table)
    bad = [
        lambda: ops.PagedKV(s.kv.k, s.kv.v.float()), lambda: ops.PagedKV(s.kv.k.cpu(), s.kv.v.cpu()),
        lambda: ops.rope_append(None, s.kv, None, None, None, *meta), lambda: ops.rope_append(None, s.kv, q, k, None, *meta),
        lambda: ops.rope_append(None, s.kv, q.double(), k, k, *meta), lambda: ops.rope_append(None, s.kv, q, k.float(), k, *meta),
        lambda: ops.rope_append(None, s.kv, q[..., :32], k, k, *meta), lambda: ops.rope_append(ops.Rope(128), s.kv, q, k, k, *meta),
        lambda: ops.prefix_attention(s.kv, q.bfloat16(), *meta), lambda: ops.prefix_attention(s.kv, q[:, :3], *meta),
        lambda: ops.prefix_attention(s.kv, q, s.d_off.long(), *meta[1:]), lambda: ops.prefix_attention(s.kv, q, *meta, prefix_len=5),
        lambda: ops.prefix_attention(s.kv, q, s.d_off[:1], *meta[1:]), lambda: ops.prefix_attention(s.kv, q, *meta, lse=q),
        lambda: ops.prefix_attention(s.kv, q, *meta[:2], s.d_table[0]), lambda: ops.prefix_attention(s.kv, q, *meta, err=q),
    ]
    for f in bad:
        with pytest.raises(R.Z2BError):
            f()
    grad = q.clone().requires_grad_()                        # no operator has a backward pass
    for f in (lambda: ops.prefix_attention(s.kv, grad, *meta), lambda: ops.rope_append(None, s.kv, grad, None, None, *meta),
              lambda: ops.verify_drafts(torch.ones((1, 1, 1, 4), device=DEV, requires_grad=True), None, s.d_lens.new_zeros((1, 0, 1)),
                                        torch.zeros((1, 0, 1), dtype=torch.float64, device=DEV),
                                        torch.zeros((1, 1, 1), dtype=torch.float64, device=DEV))):
        with pytest.raises(R.Z2BError):
            f()
        with torch.no_grad():
            f()
    none = ops.prefix_attention(s.kv, q[:0], _i32([0, 0]), s.d_lens, s.d_table)
    assert none.shape == (0, 4, 64)


@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0], ids=str)
def test_prefix_attention_scales(scale):
    """A scale of zero (all keys alike) and a negative one, few rows and many."""
    for B, P in ((2, 140), (30, 8800)):
        s = Streams([1] * B, [3] * B, 16, 2, 64, F16, prefix=P, seed=14)
        q = torch.randn((B, 8, 64), generator=_gen(15)).to(F16).to(DEV)
        out, lse = ops.prefix_attention(s.kv, q, s.d_off, s.d_lens, s.d_table, s.d_shared, P, scale=scale, lse=True, err=s.err)
        ops.check(s.err)
        _check_attention(s, q, out, lse, scale=scale)


def test_prefix_attention_many_streams():
    """More streams than one block holds records for at full width."""
    B = 1500
    s = Streams([1 if b % 3 else 0 for b in range(B)], [1 + b % 70 for b in range(B)], 16, 1, 64, F16, prefix=20, seed=16)
    q = torch.randn((s.rows, 2, 64), generator=_gen(17)).to(F16).to(DEV)
    out, lse = ops.prefix_attention(s.kv, q, s.d_off, s.d_lens, s.d_table, s.d_shared, 20, lse=True, err=s.err)
    ops.check(s.err)
    _check_attention(s, q, out, lse)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
@pytest.mark.parametrize("B,P", [(2, 4001), (40, 14001)], ids=str)
def test_prefix_attention_small_probabilities(dtype, B, P):
    """One key takes nearly all, thousands of others 2^-27 of it each: their share is not lost below f16's
    range. The probabilities are held times 2^7, so one of 2^-27 is a multiple of 2^-24 off by 2^-25
    at most: 2^-5 of it; the result (3e-5) by another half step of its type."""
    s = Streams([1] * B, [1] * B, 16, 1, 64, dtype, prefix=P, seed=18)
    for c in (s.kv.k, s.kv.v):
        c.zero_()
    s.kv.v.fill_(1.0)
    first = int(s.shared[0])
    s.kv.k[first, 0, 0, 0] = 4.6875
    s.kv.v[first, 0] = 0.0
    q = torch.zeros((B, 4, 64), dtype=dtype, device=DEV)
    q[:, :, 0] = 4.0
    out = ops.prefix_attention(s.kv, q, s.d_off, s.d_lens, s.d_table, s.d_shared, P, scale=1.0, err=s.err)
    ops.check(s.err)
    small = (P - 1 + 1) * math.exp(-18.75)                   # the prefix's other keys and the stream's own
    want = small / (1 + small)
    assert ((out.double() - want).abs() <= want * 2.0 ** -5 + max(2.0 ** -25, torch.finfo(dtype).eps / 2 * want)).all()


def test_binding_refuses_numbers_out_of_range():
    s = Streams([1], [4], 16, 2, 64, F16)
    q = torch.zeros((1, 4, 64), dtype=F16, device=DEV)
    for n in (-1, 2 ** 40):
        with pytest.raises(R.Z2BError):
            ops.prefix_attention(s.kv, q, s.d_off, s.d_lens, s.d_table, s.shared.new_zeros(1 << 4).to(DEV), n)
        with pytest.raises(R.Z2BError):
            ops.rope_append(None, s.kv, q, None, None, s.d_off, s.d_lens, s.d_table, prefix_len=n)


def test_cache_of_one_head_or_page_in_any_order():
    """Strides along dimensions of one (a transposed view's) say nothing."""
    g = _gen(19)
    k, v = (torch.randn((1, 32, 64), generator=g).to(F16).to(DEV).as_strided((1, 32, 1, 64), (3, 64, 5, 1)) for _ in range(2))
    kv = ops.PagedKV(k, v)
    q = torch.randn((1, 4, 64), generator=g).to(F16).to(DEV)
    out, lse = ops.prefix_attention(kv, q, _i32([0, 1]), _i32([20]), _i32([[0]]), lse=True)
    plain = ops.PagedKV(k.contiguous().view(1, 32, 1, 64).clone(), v.contiguous().view(1, 32, 1, 64).clone())
    want, wlse = ops.prefix_attention(plain, q, _i32([0, 1]), _i32([20]), _i32([[0]]), lse=True)
    assert torch.equal(out, want) and torch.equal(lse, wlse)


def test_prefix_attention_unaligned_queries_and_in_place():
    """q at an odd pair of elements (no 16-byte rows), few rows and many; out may be q itself."""
    for B, P in ((3, 150), (40, 6600)):
        s = Streams([1] * B, [5] * B, 16, 2, 64, BF16, prefix=P, seed=20)
        buf = torch.randn((B, 2 + 8 * 64), generator=_gen(21)).to(BF16).to(DEV)
        q = buf[:, 2:].unflatten(1, (8, 64))
        kept = q.clone()
        lse = torch.zeros((B, 8), device=DEV)
        assert ops.prefix_attention(s.kv, q, s.d_off, s.d_lens, s.d_table, s.d_shared, P, out=q, lse=lse, err=s.err)[0] is q
        ops.check(s.err)
        _check_attention(s, kept, q, lse)


@pytest.mark.parametrize("counts,page,nh,nkv,hd,dtype,prefix,pad", [
    ([1] * 8, 64, 16, 4, 128, F16, 16400, 0),                # 32 rows a key head: one tile half full
    ([1] * 40, 256, 16, 4, 64, BF16, 3300, 3),               # 160 rows: two tiles, the second a quarter full
    ([5] * 13, 16, 6, 2, 64, F16, 13500, 0),                 # 195 rows, pages of 16, the last unit of 60 keys
    ([1] * 100, 8, 6, 1, 128, BF16, 3501, 0),                # 600 rows: three segments of the one head, pages of 8
    ([3, 0, 90], 48, 4, 1, 128, F16, 5700, 9),               # a prompt chunk over the prefix
    ([1] * 65, 32, 2, 1, 64, BF16, 16200, 0),                # 130 rows: two of them in the second tile
    ([1] * 700, 16, 32, 8, 64, F16, 100, 0),                 # 2800 rows over less than one unit
], ids=str)
def test_prefix_attention_long_prefix(counts, page, nh, nkv, hd, dtype, prefix, pad):
    """Prefixes long enough for the 256-row tiles of the tensor cores, at tile and unit borders."""
    s = Streams(counts, [n + i % 5 for i, n in enumerate(counts)], page, nkv, hd, dtype, prefix=1, pad=pad, seed=23)
    s.prefix, need = prefix, -(-prefix // page)              # one page after another, drawn at once
    k, v = (torch.randn((need + s.kv.n_pages, page, nkv, hd), generator=_gen(24 + i)).to(dtype).to(DEV) for i in range(2))
    for new, old in ((k, s.kv.k), (v, s.kv.v)):
        new[need:] = old
        tail = need * page - prefix
        if tail:
            new[need - 1, page - tail:] = math.nan
    s.kv = ops.PagedKV(k, v)
    s.table, s.shared = s.table + need, torch.arange(need, dtype=torch.int32)
    s.d_table, s.d_shared = s.table.to(DEV), s.shared.to(DEV)
    q = (torch.randn((s.rows, nh, hd), generator=_gen(26)) * 1.5).to(dtype).to(DEV)
    out, lse = torch.full_like(q, 5.0), torch.full((s.rows, nh), 5.0, device=DEV)
    ops.prefix_attention(s.kv, q, s.d_off, s.d_lens, s.d_table, s.d_shared, prefix, out=out, lse=lse, err=s.err)
    ops.check(s.err)
    pick = [0, s.total // 2, s.total - 1]                    # rows checked against 64 bits
    b_of = [next(b for b in range(len(counts)) if s.off[b + 1] > t) for t in pick]
    for t, b in zip(pick, b_of):
        one = Streams([1], [1], page, nkv, hd, dtype)
        one.kc, one.prefix, one.kv = s.kc, prefix, s.kv
        sees = s.lens[b] - counts[b] + (t - s.off[b]) + 1
        one.off, one.lens, one.total = [0, 1], [sees], 1
        one.table, one.shared = s.table[b:b + 1], s.shared
        _check_attention(one, q[t:t + 1], out[t:t + 1], lse[t:t + 1])
    # the other rows: the same rows as calls of three (whose prefix the warp-level kernel takes) agree
    for t, b in ((s.total // 3, None), (s.total - 2, None)):
        b = next(b for b in range(len(counts)) if s.off[b + 1] > t)
        sees = s.lens[b] - counts[b] + (t - s.off[b]) + 1
        want, wl = ops.prefix_attention(s.kv, q[t:t + 1], _i32([0, 1]), _i32([sees]), s.d_table[b:b + 1], s.d_shared, prefix, lse=True)
        spread = 4 * torch.finfo(dtype).eps * want.double().abs().amax() + 2e-3      # two roundings of P and of the result each
        assert (out[t].double() - want[0].double()).abs().max() <= spread and (lse[t] - wl[0]).abs().max() <= 1e-3
    assert (out[s.total:] == 5.0).all() and (lse[s.total:] == 5.0).all()
    again = ops.prefix_attention(s.kv, q, s.d_off, s.d_lens, s.d_table, s.d_shared, prefix)
    assert torch.equal(out[: s.total], again[: s.total])


@pytest.mark.parametrize("B,pages", [(4, 2), (300, 2), (512, 4096)], ids=str)
def test_prefix_attention_descending_offsets(B, pages):
    """Offsets that rise and drop by turns name every row many times over (the largest case: more units
    of work than 32 bits count). Recorded, and no row is written, few streams and many."""
    rows = 4096 if pages > 2 else 24
    kv = ops.PagedKV(*(torch.zeros((3, 64, 8, 16), dtype=F16, device=DEV) for _ in range(2)))
    q = torch.zeros((rows, 64 if pages > 2 else 8, 16), dtype=F16, device=DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    off = _i32([0, rows] * (B // 2) + [0])
    lens, table = _i32([pages * 64] * B), torch.zeros((B, pages), dtype=torch.int32, device=DEV)
    for last in (0, rows):
        off[-1] = last
        for prefix in (0, 100):
            err.zero_()
            out = torch.full_like(q, 5.0)
            lse = torch.full(q.shape[:2], 6.0, device=DEV)
            ops.prefix_attention(kv, q, off, lens, table, _i32([1, 2]), prefix, out=out, lse=lse, err=err)
            assert int(err) == ops.BAD_INDEX
            assert (out == 5.0).all() and (lse == 6.0).all()


def test_copies_of_views_and_rotations():
    """A copied cache view is of the copied tensors, a copied rotation outlives its original."""
    s = Streams([3], [5], 8, 2, 32, F16, filled=False)
    q, k, v = _rows(s, 4, 32, F16, 1), _rows(s, 2, 32, F16, 2), _rows(s, 2, 32, F16, 3)
    rope, kv = copy.deepcopy(ops.Rope(32, base=500.0)), copy.deepcopy(s.kv)
    before = s.kv.k.clone()
    got = ops.rope_append(rope, kv, q, k, v, s.d_off, s.d_lens, s.d_table)
    assert torch.equal(s.kv.k.view(torch.int16), before.view(torch.int16))
    want = ops.rope_append(ops.Rope(32, base=500.0), s.kv, q, k, v, s.d_off, s.d_lens, s.d_table)
    assert torch.equal(got, want) and torch.equal(kv.k.view(torch.int16), s.kv.k.view(torch.int16))


def test_rotating_queries_without_pages():
    """With no keys to store the table may be empty."""
    s = Streams([3, 2], [5, 9], 8, 2, 32, F16, filled=False)
    q = _rows(s, 4, 32, F16, 1)
    got = ops.rope_append(ops.Rope(32), s.kv, q, None, None, s.d_off, s.d_lens, s.d_table[:, :0], err=s.err)
    ops.check(s.err)
    assert torch.equal(got, ops.rope_append(ops.Rope(32), s.kv, q, None, None, s.d_off, s.d_lens, s.d_table))


def test_results_that_share_memory_or_want_gradients():
    s = Streams([2], [4], 16, 2, 64, F16)
    q = torch.zeros((2, 4, 64), dtype=F16, device=DEV)
    meta = (s.d_off, s.d_lens, s.d_table)
    for out in (q[:1].expand(2, 4, 64), q[:, :1].expand(2, 4, 64), q.clone().requires_grad_()):
        with pytest.raises(R.Z2BError):
            ops.prefix_attention(s.kv, q, *meta, out=out)
        with pytest.raises(R.Z2BError):
            ops.rope_append(None, s.kv, q, None, None, *meta, out=out)
    with pytest.raises(R.Z2BError):
        ops.PagedKV(s.kv.k.clone().requires_grad_(), s.kv.v.clone().requires_grad_())


@pytest.mark.parametrize("lens", [[30001, 27000], [5000, 3], [1, 1]], ids=str)
def test_prefix_attention_long_own_behind_long_prefix(lens):
    """A prefix with a launch of its own, and own keys that outlast it, end with it and hardly are there."""
    s = Streams([1, 1], lens, 64, 1, 64, BF16, prefix=32768, seed=40)
    q = torch.randn((2, 32, 64), generator=_gen(41)).to(BF16).to(DEV)
    out, lse = ops.prefix_attention(s.kv, q, s.d_off, s.d_lens, s.d_table, s.d_shared, 32768, lse=True, err=s.err)
    ops.check(s.err)
    _check_attention(s, q, out, lse)
