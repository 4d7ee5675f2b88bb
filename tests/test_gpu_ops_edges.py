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


# ------------------------------------------------------------------------- large calls against 64 bits
class Paged:
    """Streams of uneven lengths with pages in random order behind one prefix, on the device: the pages a
    stream does not need have ids out of range, cache rows that no stream has are not numbers."""

    def __init__(self, counts, lens, page, nkv, hd, dtype, prefix, ahead=0, pad=0, seed=0):
        g = _gen(seed)
        need = [-(-n // page) for n in lens]
        np_, B = -(-prefix // page), len(counts)
        order = torch.randperm(sum(need) + np_ + 2, generator=g).to(torch.int32)
        self.table = torch.full((B, max([*need, 1])), -1, dtype=torch.int32)
        at = np_
        for b, n in enumerate(need):
            self.table[b, :n] = order[at: at + n]
            at += n
        self.shared, self.prefix, self.page = order[:np_], prefix, page
        dg = torch.Generator(device=DEV)
        dg.manual_seed(seed)
        k, v = (torch.randn((len(order), page, nkv, hd), generator=dg, device=DEV).to(dtype) for _ in range(2))
        for pages, n in [(self.shared, prefix)] + [(self.table[b, :m], lens[b]) for b, m in enumerate(need)]:
            if n % page:
                k[pages[-1], n % page:] = math.nan
                v[pages[-1], n % page:] = math.nan
        self.kv, self.lens, self.counts = ops.PagedKV(k, v), list(lens), list(counts)
        self.off = [ahead]
        for n in counts:
            self.off.append(self.off[-1] + n)
        self.rows = self.off[-1] + pad
        self.args = (_i32(self.off), _i32(lens), self.table.to(DEV), self.shared.to(DEV), prefix)

    def queries(self, nh, seed=1, by=1.5):
        g = torch.Generator(device=DEV)
        g.manual_seed(seed)
        return (torch.randn((self.rows, nh, self.kv.head_dim), generator=g, device=DEV) * by).to(self.kv.dtype)

    def exact(self, q, scale):
        """out, lse, sum of p |v|, largest sum of |q k| scale, in 64 bits; rows of no stream are 5."""
        nkv, hd = self.kv.n_head_kv, self.kv.head_dim
        G = q.shape[1] // nkv
        out, lse, spread = (torch.full(s, 5.0, dtype=F64, device=DEV) for s in (q.shape, q.shape[:2], q.shape))
        most, pk, pv = 0.0, *self._rows(self.shared, self.prefix)
        for b, n in enumerate(self.counts):
            if n == 0:
                continue
            lo, L = self.off[b], self.lens[b]
            if self.prefix + L == 0:
                out[lo: lo + n], spread[lo: lo + n], lse[lo: lo + n] = 0.0, 0.0, -math.inf
                continue
            ok, ov = self._rows(self.table[b], L)
            k, v = torch.cat((pk, ok), 1), torch.cat((pv, ov), 1)             # [nkv][keys][hd]
            x = q[lo: lo + n].double().reshape(n, nkv, G, hd).permute(1, 0, 2, 3).reshape(nkv, n * G, hd)
            most = max(most, float((x.abs() @ k.abs().transpose(1, 2)).max()) * abs(scale))
            s = (x @ k.transpose(1, 2)).reshape(nkv, n, G, -1) * scale
            sees = torch.arange(k.shape[1], device=DEV)[None] < self.prefix + (L - n + 1 + torch.arange(n, device=DEV)[:, None]).clamp(min=0)
            s = s.masked_fill(~sees[None, :, None], -math.inf)
            p = torch.softmax(s, -1).nan_to_num(0.0).reshape(nkv, n * G, -1)      # a row that sees no key: zeros
            back = lambda y: y.reshape(nkv, n, G, -1).permute(1, 0, 2, 3).reshape(n, nkv * G, -1)  # noqa: E731
            out[lo: lo + n], spread[lo: lo + n] = back(p @ v), back(p @ v.abs())
            lse[lo: lo + n] = back(torch.logsumexp(s, -1)[..., None])[..., 0]
        return out, lse, spread, most

    def _rows(self, pages, n):
        p = pages[: -(-n // self.page)].long().to(DEV)
        return (x[p].flatten(0, 1)[:n].double().transpose(0, 1) for x in (self.kv.k, self.kv.v))

    def check(self, q, out, lse, scale=None):
        """Every row. Each probability rounded by half a step of the type (eps / 2) for its product with V, the
        result by half a step again; scores off by 2 hd 2^-24 of sum |q k| (f32 sums, doubled for the tensor
        cores' alignment), which moves a probability by that much twice (numerator and sum); 2^-18 for ex2,
        the joins and the division; a probability below the type's normal range by half its smallest step."""
        scale = self.kv.head_dim ** -0.5 if scale is None else scale
        want, wlse, spread, most = self.exact(q, scale)
        dt = self.kv.dtype
        half, delta = torch.finfo(dt).eps / 2, 4 * self.kv.head_dim * 2.0 ** -24 * most + 2.0 ** -18
        tol = (half + delta) * spread + half * want.abs() + torch.finfo(dt).smallest_normal
        off = (out.double() - want).abs() - tol
        assert torch.isfinite(out).all() and (off <= 0).all(), float(off.max())
        empty = wlse == -math.inf
        assert torch.equal(lse == -math.inf, empty)
        assert ((lse.double() - wlse).abs()[~empty] <= delta + wlse.abs()[~empty] * 2.0 ** -22).all()


def _attend(s, q, scale=None):
    out, lse, err = torch.full_like(q, 5.0), torch.full(q.shape[:2], 5.0, device=DEV), _word()
    ops.prefix_attention(s.kv, q, *s.args, scale=scale, out=out, lse=lse, err=err)
    ops.check(err)
    return out, lse


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
@pytest.mark.parametrize("hd", [16, 32, 64, 128])
@pytest.mark.parametrize("nh,nkv,prefix", [(7, 7, 40), (6, 2, 300), (16, 4, 0)], ids=str)
def test_join_of_many_rows(hd, dtype, nh, nkv, prefix):
    """More rows x heads than are joined by blocks, head counts that four do not divide, and a stream so much
    longer than the others that its heads are spread over many partial results."""
    B = -(-900 // nh) + 3
    counts = [1 + (b % 11 == 5) for b in range(B)]
    lens = [2 + 7 * b % 90 for b in range(B)]
    lens[B // 2], lens[3] = 20011, 0 if counts[3] == 1 else 1
    s = Paged(counts, lens, 16, nkv, hd, dtype, prefix, ahead=1, pad=2, seed=hd + nh)
    q = s.queries(nh)
    assert s.off[-1] * nh > 888
    s.check(q, *_attend(s, q))


TALL = [  # counts, lens, page, nh, nkv, hd, prefix, ahead, pad
    ([1] * 64, [5 + 3 * b for b in range(64)], 16, 16, 4, 128, 3001, 0, 0),                # 256 rows a key head
    ([1] * 65, [1] * 65, 64, 16, 4, 128, 2500, 0, 3),                                      # 260: four in a second segment
    ([5] * 13, [70] * 13, 16, 6, 2, 64, 13501, 0, 0),
    ([1] * 33, [40] * 33, 256, 12, 1, 128, 6017, 3, 1),                                    # 396 + rows ahead: 432
    ([1] * 32, [9] * 32, 8, 1, 1, 64, 65541, 0, 0),                                        # 32 rows, many CTAs a segment
    ([3, 0, 90, 1], [3, 9, 4000, 2], 48, 4, 1, 128, 5700, 0, 9),
    ([1] * 150, [300 + b for b in range(150)], 32, 8, 8, 64, 2000, 1, 0),                  # own keys through all SMs
]


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
@pytest.mark.parametrize("case", TALL, ids=str)
def test_tall_prefix_every_row(case, dtype):
    """Prefixes that the tensor cores take in 256-row tiles: every row, row tile borders among them."""
    counts, lens, page, nh, nkv, hd, prefix, ahead, pad = case
    s = Paged(counts, lens, page, nkv, hd, dtype, prefix, ahead, pad, seed=hd)
    q = s.queries(nh)
    assert hd >= 64 and s.rows * nh // nkv >= 32 and s.rows * nh * prefix >= 1 << 21
    s.check(q, *_attend(s, q))


@pytest.mark.parametrize("scale", [0.0, -0.11, 0.9], ids=str)
@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
def test_tall_prefix_scales(scale, dtype):
    """head_dim 128: all keys alike, a negative scale, and one where a few keys take all and the maximum runs ahead."""
    s = Paged([1] * 40, [30] * 40, 16, 2, 128, dtype, 4100, seed=2)
    q = s.queries(8)
    s.check(q, *_attend(s, q, scale), scale)


def test_tall_values():
    """bf16 values of up to 2^79 in V: sums over thousands of keys and probabilities held above 1 stay finite."""
    for counts, prefix in (([1] * 3, 3000), ([1] * 40, 6600)):
        s = Paged(counts, [40] * len(counts), 16, 2, 64, BF16, prefix, seed=3)
        q = s.queries(8)
        out, lse = _attend(s, q)
        big = torch.tensor(2.0 ** 76, dtype=BF16, device=DEV)
        s.kv.v.mul_(big)
        got, glse = _attend(s, q)
        assert torch.equal(got, out * big) and torch.equal(lse, glse)     # powers of two: the same bits


# ------------------------------------------------------------------------- a prefix launch and what runs beside it
def _layer(x, rope, s, i, wait):
    """One layer of a decode pass: rotate and append, then attend; `wait` after each where given."""
    q, k, v = x[i]
    kv, lens = s.layers[i], s.d_lens
    q = ops.rope_append(rope, kv, q, k, v, s.args[0], lens, s.args[2], prefix_len=s.prefix)
    wait()
    out, lse = ops.prefix_attention(kv, q, s.args[0], lens, *s.args[2:], lse=True)
    wait()
    return out, lse, q


def _two_layers(hd, nh, nkv, B, prefix, own, dtype):
    s = Paged([2] * B, [own] * B, 16, nkv, hd, dtype, prefix, seed=8)
    k, v = (torch.nan_to_num(t, 0.5) for t in (s.kv.k, s.kv.v))
    s.layers = [ops.PagedKV(k.clone(), v.clone()), ops.PagedKV(v.clone(), k.clone())]
    s.d_lens = s.args[1].clone()
    assert s.rows * nh * prefix >= 1 << 21
    x = [[torch.zeros((s.rows, h, hd), dtype=dtype, device=DEV) for h in (nh, nkv, nkv)] for _ in range(2)]
    return s, x


def _fill(s, x, step):
    g = torch.Generator(device=DEV)
    g.manual_seed(step)
    for t in (t for layer in x for t in layer):
        t.copy_(torch.randn(t.shape, generator=g, device=DEV))
    s.d_lens.copy_((s.args[1] - 5 * step).clamp_(min=2))


SIZES = [(64, 8, 2, 40, 6600, 30), (128, 16, 4, 33, 4000, 700), (128, 8, 8, 64, 9000, 14)]


@pytest.mark.parametrize("hd,nh,nkv,B,prefix,own", SIZES, ids=str)
def test_tall_prefix_straight_behind_the_append(hd, nh, nkv, B, prefix, own):
    """Two layers back to back, eagerly, on a side stream, and as two graphs that share a memory pool replayed
    in turn on changing inputs: the bits of a run that waits after every call."""
    s, x = _two_layers(hd, nh, nkv, B, prefix, own, BF16)
    rope, none = ops.Rope(hd, layout="half"), lambda: None
    run = lambda wait=none: [t for i in range(2) for t in _layer(x, rope, s, i, wait)]  # noqa: E731
    was = [(kv.k.clone(), kv.v.clone()) for kv in s.layers]

    def reset():
        for kv, (k, v) in zip(s.layers, was):
            kv.k.copy_(k)
            kv.v.copy_(v)

    want = []
    for step in range(4):
        reset()
        _fill(s, x, step)
        torch.cuda.synchronize()
        want.append([t.clone() for t in run(torch.cuda.synchronize)])
    for a, b in zip(want, want[1:]):
        assert not torch.equal(a[0], b[0])
    pool, graphs = torch.cuda.graph_pool_handle(), []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            res = run()
        graphs.append((g, res))
    side = torch.cuda.Stream()
    for step in (3, 0, 2, 1, 0, 3):
        reset()
        _fill(s, x, step)
        got = run()
        assert all(torch.equal(a, b) for a, b in zip(got, want[step]))
        for g, res in graphs:
            reset()
            g.replay()
            got = [t.clone() for t in res]
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want[step]))
        reset()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = run()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(got, want[step]))


@pytest.mark.parametrize("hd,nh,nkv,B,prefix,own", SIZES, ids=str)
def test_two_tall_calls_at_once(hd, nh, nkv, B, prefix, own):
    """Two streams, each with calls of its own back to back."""
    cases = [Paged([1] * B, [own + 9 * i] * B, 16, nkv, hd, F16, prefix + 100 * i, seed=i) for i in range(2)]
    qs = [s.queries(nh) for s in cases]
    want = [_attend(s, q) for s, q in zip(cases, qs)]
    torch.cuda.synchronize()
    sides, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(10):
        for s, q, w, st in zip(cases, qs, want, sides):
            with torch.cuda.stream(st):
                got.append((ops.prefix_attention(s.kv, q, *s.args, lse=True), w))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g, w in got for a, b in zip(g, w))


# ------------------------------------------------------------------------- the distribution of verified frames
def test_verified_frames_follow_the_target():
    """Drafts drawn from q and verified: the first frame's two tokens are distributed as p's product, the second's,
    where there is one, again. 200000 streams a case: a count differs from n p by six sigma at most (2e-9 a cell)."""
    V, C, B, g = 5, 2, 200000, _gen(12)
    p1 = torch.softmax(torch.randn((3, C, V), generator=g), -1)
    q1 = torch.softmax(torch.randn((2, C, V), generator=g), -1)
    for q in (q1, None):
        draft = torch.stack([torch.multinomial(q1[f, c].double(), B, True, generator=g) for f in range(2) for c in range(C)], 1)
        draft = draft.reshape(B, 2, C).to(torch.int32)
        if q is None:                                        # a certain draft: any token, here always the same
            draft = torch.tensor([[[1, 3], [0, 2]]], dtype=torch.int32).expand(B, 2, C).contiguous()
        u, r = torch.rand((B, 2, C), generator=g, dtype=F64), torch.rand((B, 3, C), generator=g, dtype=F64)
        tok, kept = ops.verify_drafts(p1.to(DEV).expand(B, 3, C, V), None if q is None else q.to(DEV).expand(B, 2, C, V), *_dev(draft, u, r))
        tok, kept = tok.cpu().long(), kept.cpu()
        for f in range(3):
            has = kept >= f
            n = int(has.sum())
            cells = torch.bincount(tok[has, f, 0] * V + tok[has, f, 1], minlength=V * V).double()
            want = (p1[f, 0].double()[:, None] * p1[f, 1].double()).flatten()
            assert n > 100 and ((cells - n * want).abs() <= 6 * (n * want * (1 - want)).sqrt() + 1).all(), (f, n)


# ------------------------------------------------------------------------- the largest numbers
@pytest.mark.parametrize("hd,nh,nkv", [(16, 8, 1), (64, 16, 2), (128, 4, 1)], ids=str)
def test_as_many_streams_as_a_call_takes(hd, nh, nkv):
    """4096 streams, whose records leave the least room for the copies, behind a short and a tall prefix."""
    B = 4096
    for prefix in (20, 300):
        s = Paged([1 if b % 8 else 0 for b in range(B)], [1 + b % 70 for b in range(B)], 16, nkv, hd, BF16, prefix, seed=hd)
        q = s.queries(nh)
        out, lse = _attend(s, q)
        pick = list(range(0, B, 61)) + [B - 1]               # some of the streams against 64 bits
        rows = [s.off[b] for b in pick if s.counts[b]]
        t = Paged([1], [1], 16, nkv, hd, BF16, 0)
        t.kv, t.prefix, t.shared = s.kv, prefix, s.shared
        t.table, t.lens, t.counts = s.table[pick], [s.lens[b] for b in pick], [s.counts[b] for b in pick]
        t.off = [sum(t.counts[:i]) for i in range(len(pick) + 1)]
        t.check(q[rows], out[rows], lse[rows])


def test_offsets_beyond_32_bits():
    """Pages more than 2^32 elements apart, rows of q as well: appended and read back."""
    hd, far = 64, (1 << 32) + 64
    big = [torch.zeros(far + 32 * hd, dtype=F16, device=DEV) for _ in range(2)]
    kv = ops.PagedKV(*(x.as_strided((2, 16, 2, hd), (far, 2 * hd, hd, 1)) for x in big))
    g = _gen(30)
    q, k, v = (torch.randn((2, h, hd), generator=g).to(F16).to(DEV) for h in (4, 2, 2))
    wide = torch.zeros(far + 4 * hd, dtype=F16, device=DEV)
    qs = wide.as_strided((2, 4, hd), (far, hd, 1))
    qs.copy_(q)
    small = ops.PagedKV(*(torch.zeros((2, 16, 2, hd), dtype=F16, device=DEV) for _ in range(2)))
    meta = (_i32([0, 1, 2]), _i32([7, 9]), _i32([[0], [1]]))
    rope = ops.Rope(hd)
    want = ops.rope_append(rope, small, q, k, v, *meta)
    assert torch.equal(ops.rope_append(rope, kv, qs, k, v, *meta, out=qs), want)
    for a, b in ((kv.k, small.k), (kv.v, small.v)):
        assert torch.equal(a, b)
    o = ops.prefix_attention(small, want, *meta, _i32([1]), 12)
    assert torch.equal(ops.prefix_attention(kv, qs, *meta, _i32([1]), 12, out=qs), o)
    del big, wide, kv, qs
    torch.cuda.empty_cache()
