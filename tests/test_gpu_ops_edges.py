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
