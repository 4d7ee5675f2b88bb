"""The device-buffer operators (include/z2b_ops.h) at the edges of what their documentation allows:
numbers and offsets out of range, borders of a draw, results and inputs that share memory, waits that
run out, and the kernels that only large calls reach, against plain 64-bit restatements."""
from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

import z2b.ops as ops
import z2b.runtime as R
from tests import ops_ref

pytestmark = pytest.mark.gpu
F32, F16, BF16, F64 = torch.float32, torch.float16, torch.bfloat16, torch.float64
DEV = "cuda:0"


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _i32(x):
    return torch.as_tensor(x, dtype=torch.int32, device=DEV)


def _word():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------------- verify_drafts
def _dev(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


@pytest.mark.parametrize("V", [300, 20001, 131075], ids=str)      # one CTA; clusters of eight
@pytest.mark.parametrize("residual", ["late", "none"])
def test_verify_numbers_out_of_range(V, residual):
    """A u_draw outside [0, 1) is recorded; below 0 it draws the first token with mass, else the last. The
    mass lies in the last eighth of the row, so the first ranges and warps of a split row have none;
    where q is above p everywhere the draw is from p itself."""
    lo = V - V // 8
    p = torch.zeros((1, 2, 1, V))
    p[..., lo:V - 3] = 1.0 / (V - 3 - lo)
    q = torch.zeros((1, 1, 1, V)) if residual == "late" else p[:, :1] * 2 + 1
    draft = torch.zeros((1, 1, 1), dtype=torch.int32)             # p is zero there: refused
    u = torch.full((1, 1, 1), 0.5, dtype=F64)
    for r, want in ((-0.5, lo), (-1e300, lo), (-math.inf, lo), (-5e-324, lo), (1.0, V - 4), (7.0, V - 4), (math.inf, V - 4),
                    (math.nan, V - 4)):
        err = _word()
        tok, kept = ops.verify_drafts(*_dev(p, q, draft, u, torch.full((1, 2, 1), r, dtype=F64)), err=err)
        assert int(err) == ops.BAD_INDEX and tok.tolist() == [[[want], [-1]]] and kept.tolist() == [0]
        with pytest.raises(R.Z2BError):
            ops.check(err)
    for r in (0.0, -0.0, 1.0 - 2.0 ** -53):
        err = _word()
        ops.verify_drafts(*_dev(p, q, draft, u, torch.full((1, 2, 1), r, dtype=F64)), err=err)
        ops.check(err)


@pytest.mark.parametrize("B,C", [(1, 1), (3, 2), (30, 1)], ids=str)
def test_verify_second_draw_of_a_cluster(B, C):
    """q above p everywhere leaves nothing to draw from: rows that a cluster shares draw again, from p."""
    V, g = 40007, _gen(4)
    p = torch.softmax(torch.randn((B, 3, C, V), generator=g) * 2, -1)
    draft = torch.randint(0, V, (B, 2, C), generator=g).to(torch.int32)
    u, r = torch.full((B, 2, C), 0.9, dtype=F64), torch.rand((B, 3, C), generator=g, dtype=F64)
    q = p[:, :2] * 2 + 1
    tok, kept = ops.verify_drafts(*_dev(p, q, draft, u, r))
    want = ops_ref.verify(p, q, draft, u, r, None)
    assert (want[1] == 0).all() and torch.equal(tok.cpu(), want[0]) and torch.equal(kept.cpu(), want[1])


@pytest.mark.parametrize("V", [1026, 5000, 40007], ids=str)       # rows in threads, in one CTA, in a cluster
def test_verify_never_draws_a_token_without_mass(V):
    """Numbers at every border of the running sums: whichever side of it rounding puts a sum, the token
    drawn has mass, and is one of the two that meet there. Probabilities over 40 orders of magnitude, so that
    the order of the sums does round."""
    g = _gen(V)
    p = torch.softmax(torch.randn(V, generator=g) * 12, -1)
    q = torch.softmax(torch.randn(V, generator=g) * 12, -1)
    left = (p.double() - q.double()).clamp(min=0)
    some = left.nonzero().flatten()
    pick = some[torch.linspace(0, len(some) - 1, 500).long()]
    r0 = left.cumsum(0)[pick] / left.sum()
    r = torch.cat([(r0 + k * 2.0 ** -53).clamp(0, 1 - 2.0 ** -53) for k in (-2, -1, 0, 1, 2)])
    B = len(r)
    p2, q2 = (x.to(DEV).expand(B, n, 1, V) for x, n in ((p, 2), (q, 1)))
    draft = torch.full((B, 1, 1), int(q.argmax()), dtype=torch.int32)
    u, rr = torch.ones((B, 1, 1), dtype=F64), torch.zeros((B, 2, 1), dtype=F64)
    rr[:, 0, 0] = r
    assert p[q.argmax()] <= q.max()                           # u = 1 refuses it
    tok, kept = ops.verify_drafts(p2, q2, *_dev(draft, u, rr))
    tok = tok[:, 0, 0].cpu().long()
    assert (kept == 0).all() and (left[tok] > 0).all()
    # the sum up to the token, and ahead of it, against the target: off by V roundings of 2^-53 of the total
    cum, slack = left.cumsum(0), V * 2.0 ** -53 * left.sum()
    target = r * left.sum()
    assert (cum[tok] >= target - slack).all() and (cum[tok] - left[tok] <= target + slack).all()


# ------------------------------------------------------------------------- rope_append
def _three_streams():
    g = _gen(3)
    k, v = (torch.randn((8, 4, 1, 32), generator=g).to(F16).to(DEV) for _ in range(2))
    q, kn, vn = (torch.randn((4, h, 32), generator=g).to(F16).to(DEV) for h in (2, 1, 1))
    return ops.PagedKV(k, v), _i32([6, 7, 8]), _i32([[0, 1], [2, 3], [4, 5]]), q, kn, vn


@pytest.mark.parametrize("off,stored", [
    # offsets; (row, stream, cache row) of the rows of streams whose own offsets are sound
    ([0, 1, 2, 5], [(0, 0, 5), (1, 1, 6)]),                  # the last stream ends behind the rows
    ([0, 1, 9, 12], [(0, 0, 5)]), ([0, 4, 4, 6], [(0, 0, 2), (1, 0, 3), (2, 0, 4), (3, 0, 5)]),
    ([-1, 1, 2, 3], [(1, 1, 6), (2, 2, 7)]),                 # the first begins ahead of them
    ([0, 2, 1, 1], []), ([0, 2, 1, 4], [(0, 0, 4), (2, 2, 6), (3, 2, 7)]), ([2, 1, 0, 0], []),      # descending
    ([0, 1, 2, -5], []), ([0, 9, 9, 9], []), ([-9, -8, -7, -6], []), ([5, 4, 4, 4], []),
    ([0, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1], []), ([-2 ** 31, 1, 2, 3], [(1, 1, 6), (2, 2, 7)])], ids=str)
def test_rope_append_bad_offsets(off, stored):
    """Offsets out of range or descending are recorded; the rows of streams that they belong to turn
    nothing and store nothing, and no cached row changes but those of the sound streams."""
    kv, lens, table, q, k, v = _three_streams()
    want_k, want_v, want_q = kv.k.clone(), kv.v.clone(), torch.full_like(q, 5.0)
    for t, b, r in stored:
        page = int(table[b, r // 4])
        want_k[page, r % 4], want_v[page, r % 4], want_q[t] = k[t], v[t], q[t]
    for err in (_word(), None):                              # the same rows with and without the word
        out = torch.full_like(q, 5.0)
        ops.rope_append(None, kv, q, k, v, _i32(off), lens, table, out=out, err=err)
        assert torch.equal(kv.k, want_k) and torch.equal(kv.v, want_v) and torch.equal(out, want_q)
        assert err is None or int(err) == ops.BAD_INDEX


def test_rope_append_many_bad_offsets():
    """One descent among many streams, wherever it lies, is recorded."""
    B = 300
    kv = ops.PagedKV(*(torch.zeros((3, 4, 1, 32), dtype=F16, device=DEV) for _ in range(2)))
    q = torch.zeros((B, 1, 32), dtype=F16, device=DEV)
    for at in (0, 1, 31, 32, 150, 298, 299):
        off = torch.arange(B + 1)
        off[at + 1:] -= 2
        if at == 0:
            off[0] = 1
        off.clamp_(min=0)
        err = _word()
        ops.rope_append(None, kv, q, None, None, _i32(off), _i32([4] * B), _i32([[1]] * B), err=err)
        assert int(err) == (ops.BAD_INDEX if (off[1:] < off[:-1]).any() else 0), at


def test_rope_append_rows_ahead_of_the_first_stream():
    """row_off[0] above 0: the rows ahead of it belong to no stream, which is no fault."""
    kv, lens, table, q, k, v = _three_streams()
    was, err, out = kv.k.clone(), _word(), torch.full_like(q, 5.0)
    ops.rope_append(None, kv, q, k, v, _i32([1, 2, 2, 3]), lens, table, out=out, err=err)
    ops.check(err)
    assert (out[0] == 5).all() and (out[3] == 5).all() and torch.equal(out[1:3], q[1:3])
    was[1, 1], was[5, 3] = k[1], k[2]
    assert torch.equal(kv.k, was)
    pages = ops.PagedKV(*(x.reshape(4, 8, 1, 32) for x in (kv.k, kv.v)))        # pages of 8 for the attention
    o, lse = ops.prefix_attention(pages, q, _i32([1, 2, 2, 3]), lens, _i32([[0], [1], [2]]), out=torch.full_like(q, 5.0),
                                  lse=torch.full((4, 2), 6.0, device=DEV), err=err)
    ops.check(err)
    assert (o[0] == 5).all() and (o[3] == 5).all() and (lse[0] == 6).all() and (lse[3] == 6).all()


# ------------------------------------------------------------------------- prefix_attention
@pytest.mark.parametrize("B,P", [(3, 40), (200, 40), (40, 8800)], ids=str)        # joined by blocks, by warps; tall prefix
def test_prefix_attention_of_queries_that_are_not_numbers(B, P):
    """A query with an entry that is not a number has a result and an lse that are not, and no other row does."""
    g, page = _gen(5), 16
    np_ = -(-P // page)
    k, v = (torch.randn((np_ + B, page, 2, 64), generator=g).to(F16).to(DEV) for _ in range(2))
    q = torch.randn((B, 8, 64), generator=g).to(F16).to(DEV)
    args = (_i32(range(B + 1)), _i32([5] * B), _i32(range(np_, np_ + B))[:, None], _i32(range(np_)), P)
    out, lse = ops.prefix_attention(ops.PagedKV(k, v), q, *args, lse=True)
    q[1, 3, 5] = math.nan
    got, glse = ops.prefix_attention(ops.PagedKV(k, v), q, *args, lse=True)
    assert torch.isnan(got[1, 3]).all() and torch.isnan(glse[1, 3])
    rest = torch.ones((B, 8), dtype=torch.bool, device=DEV)
    rest[1, 3] = False
    assert torch.equal(got[rest], out[rest]) and torch.equal(glse[rest], lse[rest])


def _many(B, P, hd=64, nh=8, nkv=2, own=5, dtype=F16, page=16, seed=6):
    """B decode rows behind one prefix: cache, queries and the arguments after them."""
    g, np_, per = _gen(seed), -(-P // page), -(-own // page)
    k, v = (torch.randn((np_ + B * per, page, nkv, hd), generator=g).to(dtype).to(DEV) for _ in range(2))
    q = torch.randn((B, nh, hd), generator=g).to(dtype).to(DEV)
    table = torch.arange(np_, np_ + B * per, dtype=torch.int32, device=DEV).reshape(B, per)
    return ops.PagedKV(k, v), q, (_i32(range(B + 1)), _i32([own] * B), table, _i32(range(np_)), P)


@pytest.fixture
def wait_polls():
    f = R.lib().z2b_test_attn_wait_polls
    yield f
    torch.cuda.synchronize()
    f(-1)


# joined by blocks, by warps; a tall prefix of few and of many units a CTA, with and without own keys
WAITS = [(2, 40, 64, 5), (3, 0, 32, 900), (200, 40, 128, 5), (40, 6600, 64, 5), (40, 6600, 128, 300), (200, 16000, 128, 40)]


@pytest.mark.parametrize("B,P,hd,own", WAITS, ids=str)
def test_prefix_attention_waits_that_run_out(wait_polls, B, P, hd, own):
    """Every wait gives up at once: TIMEOUT is recorded, the call ends with its copies and products done,
    and the next one is right."""
    kv, q, args = _many(B, P, hd, own=own)
    want = ops.prefix_attention(kv, q, *args)
    torch.cuda.synchronize()
    for _ in range(3):
        err = _word()
        wait_polls(0)
        ops.prefix_attention(kv, q, *args, err=err)
        wait_polls(-1)
        assert int(err) == ops.TIMEOUT
        with pytest.raises(R.Z2BError):
            ops.check(err)
        assert torch.equal(ops.prefix_attention(kv, q, *args), want)


@pytest.mark.parametrize("B,P,hd,own", WAITS, ids=str)
def test_prefix_attention_results_of_waits_that_run_out(wait_polls, B, P, hd, own):
    """What a wait that ran out leaves cannot pass for a result, also without the error word, and whatever
    the workspace held before."""
    kv, q, args = _many(B, P, hd, own=own)
    for _ in range(2):                                       # the second with the first's good partial results
        wait_polls(0)
        out, lse = ops.prefix_attention(kv, q, *args, lse=True)
        wait_polls(-1)
        assert torch.isnan(out).all() and torch.isnan(lse).all()
        ops.prefix_attention(kv, q, *args)


# ------------------------------------------------------------------------- gradients
def test_gradients_of_either_mode_are_refused():
    """A tangent would be lost without a word; so would the gradient of an lse."""
    from torch.autograd import forward_ad
    kv, lens, table, q, k, v = _three_streams()
    pages = ops.PagedKV(*(x.reshape(4, 8, 1, 32) for x in (kv.k, kv.v)))
    off, eight = _i32([0, 2, 3, 4]), _i32([[0], [1], [2]])
    p, draft = torch.full((1, 2, 1, 4), 0.25, device=DEV), torch.zeros((1, 1, 1), dtype=torch.int32, device=DEV)
    u, r = torch.zeros((1, 1, 1), dtype=F64, device=DEV), torch.zeros((1, 2, 1), dtype=F64, device=DEV)
    calls = [                                                # each with the tensor that carries the tangent
        (q, lambda x: ops.prefix_attention(pages, x, off, lens, eight)), (q, lambda x: ops.rope_append(None, kv, x, k, v, off, lens, table)),
        (k, lambda x: ops.rope_append(None, kv, q, x, v, off, lens, table)), (v, lambda x: ops.rope_append(None, kv, q, k, x, off, lens, table)),
        (q, lambda x: ops.rope_append(None, kv, q, k, v, off, lens, table, out=x)),
        (q, lambda x: ops.prefix_attention(pages, q, off, lens, eight, out=x)),
        (torch.zeros((4, 2), device=DEV), lambda x: ops.prefix_attention(pages, q, off, lens, eight, lse=x)),
        (p, lambda x: ops.verify_drafts(x, None, draft, u, r)), (p[:, :1], lambda x: ops.verify_drafts(p, x, draft, u, r)),
        (pages.k, lambda x: ops.PagedKV(x, pages.v)), (pages.v, lambda x: ops.PagedKV(pages.k, x))]
    for x, f in calls:
        f(x)
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(x, torch.ones_like(x))
            with pytest.raises(R.Z2BError):
                f(dual)
            with torch.no_grad(), pytest.raises(R.Z2BError):     # which forward mode does not heed
                f(dual)
            f(forward_ad.unpack_dual(dual).primal)
    with pytest.raises(R.Z2BError):
        calls[6][1](torch.zeros((4, 2), device=DEV, requires_grad=True))


# ------------------------------------------------------------------------- shared memory
def test_tensors_that_share_memory():
    """What rope_append writes shares no memory with what it reads or writes beside it; slices of one buffer
    pass, and pages that are only read may be anything."""
    g = _gen(9)
    kv, lens, table, q, k, v = _three_streams()
    meta = (_i32([0, 2, 3, 4]), lens, table)
    buf = torch.randn(4096, generator=g).to(F16).to(DEV)
    pages = buf[:2048].view(8, 2, 4, 1, 32)
    one = ops.PagedKV(pages[:, 0], pages[:, 1])              # keys and values by turns
    for f in (lambda: ops.rope_append(None, kv, q, None, None, *meta, out=buf.as_strided((4, 2, 32), (48, 32, 1))),
              lambda: ops.rope_append(None, kv, buf[:256].view(4, 2, 32), None, None, *meta, out=buf[64:320].view(4, 2, 32)),
              lambda: ops.rope_append(None, kv, q, buf[:128].view(4, 1, 32), v, *meta, out=buf[:256].view(4, 2, 32)),
              lambda: ops.rope_append(None, ops.PagedKV(kv.k, kv.k), q, k, v, *meta),
              lambda: ops.rope_append(None, ops.PagedKV(*(buf[x:x + 1024].view(8, 4, 1, 32) for x in (0, 32))), q, k, v, *meta),
              lambda: ops.rope_append(None, ops.PagedKV(*(x[:1].expand(8, -1, -1, -1) for x in (kv.k, kv.v))), q, k, v, *meta)):
        with pytest.raises(R.Z2BError):
            f()
    want = ops.rope_append(ops.Rope(32), kv, q, k, v, *meta)
    fused = torch.cat((q, k, v), 1)                          # rows of [q | k | v], q turned in place
    got = ops.rope_append(ops.Rope(32), one, fused[:, :2], fused[:, 2:3], fused[:, 3:], *meta, out=fused[:, :2])
    assert torch.equal(got, want) and torch.equal(fused[:, 2:3], k)
    for b, r in ((0, 4), (0, 5), (1, 6), (2, 7)):
        at = int(table[b, r // 4]), r % 4
        assert torch.equal(one.k[at], kv.k[at]) and torch.equal(one.v[at], kv.v[at])
    same = ops.PagedKV(*(x.reshape(4, 8, 1, 32)[:1].expand(4, -1, -1, -1) for x in (kv.k, kv.k)))
    a = ops.prefix_attention(same, q, meta[0], lens, _i32([[0], [1], [2]]))
    b = ops.prefix_attention(ops.PagedKV(*(same.k.contiguous() for _ in range(2))), q, meta[0], lens, _i32([[0], [1], [2]]))
    assert torch.equal(a, b)
