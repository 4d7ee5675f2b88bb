"""Cases of the paged-cache operators: rope_append, prefix_attention and verify_drafts.

They are the three steps of one pass over streams that share a prompt and carry drafted
tokens: rotate the new rows and append them to the paged cache, attend over the shared
prefix and each stream's own rows, and check the drafts against the target's
probabilities. `own` selects the framework's kernels; otherwise `run` computes the same
with elementary torch operations.

Shapes used throughout: rows of all streams are packed, stream b owns the rows
[row_off[b], row_off[b + 1]) of a [T][heads][head_dim] tensor, its cached rows (the new
ones included) are lens[b], and row i of its n new rows sits at cache row lens[b] - n + i
and at position prefix_len + that. Rows from row_off[-1] on are padding.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _ops():
    """The package's operators (its folder name is not an identifier, so it is loaded as z2b)."""
    if "z2b" not in sys.modules:
        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "zonos2.cpp_b200")
        spec = importlib.util.spec_from_file_location("z2b", os.path.join(pkg, "__init__.py"),
                                                      submodule_search_locations=[pkg])
        sys.modules["z2b"] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules["z2b"])
    return importlib.import_module("z2b.ops")


# ---------------------------------------------------------------------------- cases
def _append(name, **kw):
    d = dict(op="append", seqs=1, rows=1, ragged=False, pad=0, past=128, prefix=0, heads=16, kv_heads=4, head_dim=128,
             rot=128, layout="interleaved", base=1e6, scaling="none", factor=1.0, orig=8192, page=256, heads_first=False,
             type="f16", cache="f16")
    d.update(kw)
    return dict(d, name=name) if name else d


def _attn(name, **kw):
    d = dict(op="attention", seqs=1, rows=1, ragged=False, pad=0, prefix=64, own_min=1, own_max=64, heads=16, kv_heads=4,
             head_dim=128, page=256, heads_first=False, type="f16")
    d.update(kw)
    return dict(d, name=name) if name else d


def _verify(name, **kw):
    d = dict(op="verify", seqs=1, drafts=4, ragged=False, codebooks=9, vocab=1026, type="f32", draft_probs=True, apart=0.7)
    d.update(kw)
    return dict(d, name=name) if name else d


def listed():
    return [
        # one stream, one new row, the backbone's own shape: nothing but latency
        _append("append_decode_1"),
        # 64 streams with 4 drafted tokens each behind a long shared prompt: half layout, half of
        # the head rotated, frequencies scaled for a context beyond the trained one
        _append("append_drafts_64x5", seqs=64, rows=5, past=700, prefix=100003, heads=32, kv_heads=8, rot=64,
                layout="half", scaling="by_parts", factor=16.0, page=16, type="bf16", cache="bf16"),
        # ragged rows and a padded batch, f32 activations as the step's projections leave them,
        # into an f16 cache of small odd pages
        _append("append_f32_ragged", seqs=33, rows=61, ragged=True, pad=7, past=1000, prefix=257, heads=12, kv_heads=4,
                head_dim=64, rot=64, base=1e4, scaling="linear", factor=4.0, page=48, heads_first=True, type="f32",
                cache="f16"),
        # prompts of new streams, 16k rows in one call: bandwidth
        _append("append_prompts_16k", seqs=8, rows=2048, past=0, prefix=0, heads=32, kv_heads=8, layout="half",
                scaling="ntk", factor=2.0, page=64, type="bf16", cache="bf16"),
        # two streams of one short prompt at their first tokens
        _attn("attn_first_tokens_2", seqs=2, prefix=67, own_max=5),
        # 16 streams of the backbone's shape that share a prompt, contexts to 2048
        _attn("attn_streams_16", seqs=16, prefix=1000, own_max=1048),
        # 64 streams with 4 drafts each, three query heads to a key head, small pages
        _attn("attn_drafts_64x5", seqs=64, rows=5, prefix=4097, own_min=5, own_max=300, heads=24, kv_heads=8, head_dim=64,
              page=16, type="bf16"),
        # few streams whose own contexts are long and uneven, behind a short prompt; rows ragged
        _attn("attn_long_own_7", seqs=7, rows=3, ragged=True, pad=2, prefix=129, own_max=30011, kv_heads=4, page=64,
              heads_first=True, type="bf16"),
        # the largest: 256 streams over one 32k document
        _attn("attn_document_256", seqs=256, prefix=32768, own_max=600, heads=32, kv_heads=8, page=64, type="bf16"),
        # one stream's drafted frames, nine codebooks each
        _verify("verify_frames_1"),
        # 64 streams, drafts without probabilities of their own (greedy drafts)
        _verify("verify_frames_64", seqs=64, drafts=3, ragged=True, draft_probs=False),
        # text-sized vocabulary, odd
        _verify("verify_vocab_32", seqs=32, drafts=5, codebooks=1, vocab=128003),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {c["name"]: c for c in listed()}
    top = {"append": work(most["append_prompts_16k"]), "attention": work(most["attn_document_256"]),
           "verify": work(most["verify_vocab_32"])}
    while True:
        op = rng.choice(("append", "attention", "verify"))
        half = rng.choice(("f16", "bf16"))
        kv = rng.choice((1, 2, 4, 8))
        common = dict(seqs=_log(rng, 1, 256), ragged=rng.random() < 0.5, pad=rng.choice((0, 0, 3)),
                      heads=kv * rng.choice((1, 2, 3, 4, 7, 8)), kv_heads=kv, page=rng.choice((16, 32, 48, 64, 128, 256)),
                      heads_first=rng.random() < 0.3)
        if op == "append":
            hd = rng.choice((32, 64, 128))
            wide = rng.random() < 0.3
            c = _append(None, **dict(common, rows=_log(rng, 1, 2048), past=_log(rng, 1, 1000), prefix=rng.choice((0, _log(rng, 1, 500000))),
                                     head_dim=hd, rot=rng.choice((hd, hd // 2)), layout=rng.choice(("interleaved", "half")),
                                     base=rng.choice((1e4, 1e6)), scaling=rng.choice(("none", "linear", "ntk", "by_parts")),
                                     factor=rng.choice((2.0, 4.0, 16.0)), orig=rng.choice((2048, 8192)),
                                     type="f32" if wide else half, cache=half))
            if c["scaling"] == "none":
                c["factor"] = 1.0
            fits = c["seqs"] * c["rows"] <= 16384
        elif op == "attention":
            rows = rng.choice((1, 1, _log(rng, 1, 8)))
            c = _attn(None, **dict(common, rows=rows, prefix=rng.choice((0, _log(rng, 1, 32768), _log(rng, 1, 32768))),
                                   own_min=rows, own_max=max(rows, _log(rng, 1, 30000)), head_dim=rng.choice((32, 64, 128)), type=half))
            # what the plain form holds at a time stays within the largest listed case's
            scores = c["seqs"] * rows * c["heads"] * (c["prefix"] + c["own_max"])
            fits = scores <= 3e8 and c["seqs"] * c["own_max"] * c["kv_heads"] * c["head_dim"] <= 2e8
        else:
            books = rng.choice((1, 1, 4, 9))
            c = _verify(None, seqs=_log(rng, 1, 128), drafts=_log(rng, 1, 8), ragged=rng.random() < 0.5, codebooks=books,
                        vocab=_log(rng, 300, 200000), type=rng.choice(("f32", "f32", "bf16")), draft_probs=rng.random() < 0.7,
                        apart=rng.choice((0.3, 0.7, 1.5)))
            fits = c["seqs"] * (c["drafts"] + 1) * books * c["vocab"] <= 32 * 6 * 128003
        w = work(c)
        if fits and w["bytes"] <= top[op]["bytes"] and w["flops"] <= max(top[op]["flops"], 1):
            return c


# ---------------------------------------------------------------------------- inputs
def _gen(seed, salt=0):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1000003 + salt) & 0x7FFFFFFFFFFF)
    return g


def _host(seed):
    g = torch.Generator()
    g.manual_seed((int(seed) * 7919 + 13) & 0x7FFFFFFFFFFF)
    return g


def _row_counts(c):
    """New rows of each stream: all `rows`, or ragged from 0 (one stream has the most); the case's
    own, so that a case has one shape."""
    n = torch.full((c["seqs"],), c["rows"])
    if c["ragged"]:
        g = torch.Generator()
        g.manual_seed(c["seqs"] * 100003 + c["rows"])
        n = torch.randint(0, c["rows"] + 1, (c["seqs"],), generator=g)
        n[c["seqs"] // 2] = c["rows"]
    return n


def _layout(c, most, g, more=0):
    """Page tables of the streams (and `more` further pages), a random order of a pool a little larger."""
    per = max(1, -(-most // c["page"]))
    used = c["seqs"] * per + more
    order = torch.randperm(used + 3, generator=g).to(torch.int32)
    return order[: c["seqs"] * per].reshape(c["seqs"], per).to(DEV), order[c["seqs"] * per: used].to(DEV), used + 3


def _cache(c, pages, dtype, g):
    shape = (pages, c["kv_heads"], c["page"], c["head_dim"]) if c["heads_first"] else (pages, c["page"], c["kv_heads"], c["head_dim"])
    t = [torch.randn(shape, generator=g, device=DEV, dtype=dtype) for _ in range(2)]
    return [x.transpose(1, 2) if c["heads_first"] else x for x in t]


def _off(n):
    return torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(n, 0)]).to(torch.int32).to(DEV)


def _freqs(c):
    """Radians per position of each rotated pair, and the factor on cos and sin (64 bits)."""
    d = c["rot"]
    i = torch.arange(d // 2, dtype=torch.float64)
    base, f, mag = c["base"], c["factor"], 1.0
    if c["scaling"] == "ntk":
        base = base * f ** (d / (d - 2))
    w = base ** (-2 * i / d)
    if c["scaling"] == "linear":
        w = w / f
    elif c["scaling"] == "by_parts":
        turns = c["orig"] * w / (2 * math.pi)           # turns within the trained context
        keep = torch.clamp((turns - 1.0) / (32.0 - 1.0), 0, 1)
        w = w / f * (1 - keep) + w * keep
        mag = 0.1 * math.log(f) + 1.0
    return w.to(DEV), mag


def prepare(case, seed):
    c, s = dict(case), {"case": dict(case)}
    if c["op"] == "verify":
        return _prepare_verify(c, s, seed)
    h, g = _host(seed), _gen(seed)
    n = _row_counts(c)
    T = int(n.sum())
    dtype = TYPES[c["type"]]
    if c["op"] == "append":
        lens = torch.randint(0, c["past"] + 1, (c["seqs"],), generator=h) + n
        table, _, pages = _layout(c, c["past"] + c["rows"], h)
        k, v = _cache(c, pages, TYPES[c["cache"]], g)
        def mk(heads):
            return torch.randn((T + c["pad"], heads, c["head_dim"]), generator=g, device=DEV, dtype=torch.float32).to(dtype)
        s.update(q=mk(c["heads"]), k=mk(c["kv_heads"]), v=mk(c["kv_heads"]))
        s["w"], s["mag"] = _freqs(c)
        if own:     # the rotation's table and the view of the cache, which a program makes once
            ops = _ops()
            s["rope"] = ops.Rope(c["rot"], base=c["base"], layout=c["layout"], scaling=c["scaling"], factor=c["factor"],
                                 orig_ctx=c["orig"])
    else:
        lens = torch.randint(c["own_min"], c["own_max"] + 1, (c["seqs"],), generator=h)
        lens[0] = c["own_max"]
        lens = torch.maximum(lens, n)
        more = -(-c["prefix"] // c["page"])
        table, shared, pages = _layout(c, max(c["own_max"], c["rows"]), h, more)
        k, v = _cache(c, pages, dtype, g)
        q = torch.randn((T + c["pad"], c["heads"], c["head_dim"]), generator=g, device=DEV, dtype=torch.float32)
        s.update(q=(q * 1.5).to(dtype), shared=shared)
    if own:
        s["cache"] = _ops().PagedKV(k, v)
    s.update(k_cache=k, v_cache=v, table=table, lens=lens.to(torch.int32).to(DEV), off=_off(n), total=T, max_rows=max(1, int(n.max())),
             max_own=int(lens.max()))
    return s


def _prepare_verify(c, s, seed):
    g, h = _gen(seed), _host(seed)
    B, N, C, V, dt = c["seqs"], c["drafts"], c["codebooks"], c["vocab"], TYPES[c["type"]]
    base = torch.randn((B, N + 1, C, V), generator=g, device=DEV) * 2.5
    s["p"] = torch.softmax(base, -1).to(dt)
    far = base[:, :N] + c["apart"] * torch.randn((B, N, C, V), generator=g, device=DEV)
    del base
    # drafts drawn from the draft's own distribution
    noise = torch.empty_like(far).exponential_(generator=g)
    s["draft"] = (far - noise.log()).argmax(-1).to(torch.int32)
    s["q"] = torch.softmax(far, -1).to(dt) if c["draft_probs"] else None
    s["u"] = torch.rand((B, N, C), generator=g, device=DEV, dtype=torch.float64)
    s["r"] = torch.rand((B, N + 1, C), generator=g, device=DEV, dtype=torch.float64)
    s["n"] = torch.randint(0, N + 1, (B,), generator=h).to(torch.int32).to(DEV) if c["ragged"] else None
    return s


# ---------------------------------------------------------------------------- a pass
def run(s):
    c = s["case"]
    if c["op"] == "append":
        return _run_append(s, c)
    if c["op"] == "attention":
        return _run_attention(s, c)
    return _run_verify(s, c)


def _row_places(s):
    """Stream, new-row index and cache row of each of the `total` rows."""
    t = torch.arange(s["total"], device=DEV)
    off = s["off"].long()
    b = torch.searchsorted(off[1:].contiguous(), t, right=True)
    i = t - off[b]
    return b, i, s["lens"].long()[b] - (off[b + 1] - off[b]) + i


def _rotate(x, cos, sin, rot, layout):
    a = x[..., :rot]
    if layout == "half":
        e, o = a[..., : rot // 2], a[..., rot // 2:]
    else:
        e, o = a[..., 0::2], a[..., 1::2]
    r = (e * cos - o * sin, o * cos + e * sin)
    a = torch.cat(r, -1) if layout == "half" else torch.stack(r, -1).flatten(-2)
    return torch.cat((a, x[..., rot:]), -1)


def _run_append(s, c):
    if own:
        q = _ops().rope_append(s["rope"], s["cache"], s["q"], s["k"], s["v"], s["off"], s["lens"], s["table"],
                               prefix_len=c["prefix"])
        return {"q": q[: s["total"]], "k": s["k_cache"], "v": s["v_cache"]}
    T = s["total"]
    b, _, at = _row_places(s)
    angle = (at + c["prefix"]).double()[:, None] * s["w"]
    cos, sin = ((f(angle) * s["mag"]).float()[:, None] for f in (torch.cos, torch.sin))
    page = s["table"][b, at // c["page"]].long()
    q = _rotate(s["q"][:T].float(), cos, sin, c["rot"], c["layout"]).to(s["q"].dtype)
    s["k_cache"][page, at % c["page"]] = _rotate(s["k"][:T].float(), cos, sin, c["rot"], c["layout"]).to(s["k_cache"].dtype)
    s["v_cache"][page, at % c["page"]] = s["v"][:T].to(s["v_cache"].dtype)
    return {"q": q, "k": s["k_cache"], "v": s["v_cache"]}


def _run_attention(s, c):
    if own:
        out, lse = _ops().prefix_attention(s["cache"], s["q"], s["off"], s["lens"], s["table"], s["shared"],
                                           prefix_len=c["prefix"], lse=True)
        return {"out": out[: s["total"]], "lse": lse[: s["total"]]}
    T, kv, hd, per, most = s["total"], c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"], s["max_own"]
    b, i, at = _row_places(s)
    q = s["q"][:T].float().reshape(T, kv, per, hd) * hd ** -0.5
    kp, vp = (x[s["shared"].long()].flatten(0, 1)[: c["prefix"]].float().transpose(0, 1) for x in (s["k_cache"], s["v_cache"]))
    sp = torch.matmul(q.permute(1, 0, 2, 3).reshape(kv, T * per, hd), kp.transpose(1, 2))           # [kv][T per][prefix]
    j = torch.arange(most, device=DEV)
    page = s["table"].long()[:, j // c["page"]]
    ko, vo = (x[page, j % c["page"]].float().permute(0, 2, 1, 3) for x in (s["k_cache"], s["v_cache"]))  # [B][kv][most][hd]
    # the streams' rows side by side, as many as the stream with the most has
    rows = s["max_rows"]
    qo = torch.zeros((c["seqs"], rows, kv, per, hd), device=DEV)
    qo[b, i] = q
    so = torch.matmul(qo.permute(0, 2, 1, 3, 4).reshape(c["seqs"], kv, rows * per, hd), ko.transpose(2, 3))
    so = so.reshape(c["seqs"], kv, rows, per, most)[b, :, i]                                         # [T][kv][per][most]
    so = so.masked_fill((j[None] > at[:, None])[:, None, None], -math.inf)
    sp = sp.reshape(kv, T, per, -1).permute(1, 0, 2, 3)
    m = so.amax(-1, keepdim=True)
    if c["prefix"]:
        m = torch.maximum(m, sp.amax(-1, keepdim=True))
    m = torch.where(m == -math.inf, 0.0, m)
    eo, ep = torch.exp(so - m), torch.exp(sp - m)
    total = eo.sum(-1, keepdim=True) + ep.sum(-1, keepdim=True)
    po = torch.zeros((c["seqs"], rows, kv, per, most), device=DEV)
    po[b, i] = eo
    oo = torch.matmul(po.permute(0, 2, 1, 3, 4).reshape(c["seqs"], kv, rows * per, most), vo)
    oo = oo.reshape(c["seqs"], kv, rows, per, hd)[b, :, i]
    op = torch.matmul(ep.permute(1, 0, 2, 3).reshape(kv, T * per, -1), vp).reshape(kv, T, per, hd).permute(1, 0, 2, 3)
    out = torch.where(total > 0, (oo + op) / total, 0.0)
    lse = (m + torch.log(total)).squeeze(-1)
    return {"out": out.reshape(T, c["heads"], hd).to(s["q"].dtype), "lse": lse.reshape(T, c["heads"])}


def _run_verify(s, c):
    if own:
        frames, kept = _ops().verify_drafts(s["p"], s["q"], s["draft"], s["u"], s["r"], n_draft=s["n"])
        return {"frames": frames, "accepted": kept}
    p, q, draft = s["p"], s["q"], s["draft"].long()
    B, N, C = draft.shape
    pt = p[:, :N].gather(-1, draft[..., None]).squeeze(-1).double()
    qt = q.gather(-1, draft[..., None]).squeeze(-1).double() if q is not None else torch.ones_like(pt)
    ok = s["u"] * qt < pt
    n = s["n"].long() if s["n"] is not None else torch.full((B,), N, device=DEV)
    i = torch.arange(N, device=DEV)
    kept = (ok.all(-1) & (i[None] < n[:, None])).long().cumprod(-1).sum(-1)
    rows = torch.arange(B, device=DEV)
    last = kept == n                                    # every draft kept: one more frame from the target
    at = kept.clamp(max=N - 1)
    pr = p[rows, kept].double()                         # [B][C][V]
    if q is not None:
        qr = q[rows, at].double()
    else:
        qr = torch.zeros_like(pr).scatter_(-1, draft[rows, at][..., None], 1.0)
    left = (pr - qr).clamp_(min=0)
    use = (~last)[:, None, None] & (left.sum(-1, keepdim=True) > 0)
    left = torch.where(use, left, pr)
    cum = left.cumsum(-1)
    r = s["r"][rows, kept] * cum[..., -1]
    drawn = (cum <= r[..., None]).sum(-1)
    where = torch.arange(left.shape[-1], device=DEV)
    drawn = torch.minimum(drawn, torch.where(left > 0, where, 0).amax(-1))
    tok = torch.where(ok[rows, at] & ~last[:, None], draft[rows, at], drawn)
    frames = torch.full((B, N + 1, C), -1, dtype=torch.int64, device=DEV)
    frames[:, :N] = torch.where(i[None, :, None] < kept[:, None, None], draft, -1)
    frames[rows, kept] = tok
    return {"frames": frames.to(torch.int32), "accepted": kept.to(torch.int32)}


# ---------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    c = dict(case)
    if c["op"] == "verify":
        return None                                     # whole numbers only
    s = prepare(c, seed)
    off, lens, hd = s["off"].tolist(), s["lens"].tolist(), c["head_dim"]

    def turn(x, pos):
        x, d = x.double(), c["rot"]
        pairs = x[..., :d].unflatten(-1, (2, d // 2)).transpose(-1, -2) if c["layout"] == "half" else x[..., :d].unflatten(-1, (d // 2, 2))
        angle = pos[:, None] * s["w"]
        z = torch.complex(pairs[..., 0], pairs[..., 1]) * torch.polar(torch.full_like(angle, s["mag"]), angle)[:, None]
        z = torch.view_as_real(z)
        return torch.cat((z.transpose(-1, -2).flatten(-2) if c["layout"] == "half" else z.flatten(-2), x[..., d:]), -1)

    if c["op"] == "append":
        q, k, v = [], s["k_cache"].double(), s["v_cache"].double()
        for b in range(c["seqs"]):
            lo, hi = off[b], off[b + 1]
            at = torch.arange(lens[b] - (hi - lo), lens[b], device=DEV)
            pos = (at + c["prefix"]).double()
            q.append(turn(s["q"][lo:hi], pos))
            page = s["table"][b].long()[at // c["page"]]
            k[page, at % c["page"]] = turn(s["k"][lo:hi], pos)
            v[page, at % c["page"]] = s["v"][lo:hi].double()
        return {"q": torch.cat(q), "k": k, "v": v}

    per = c["heads"] // c["kv_heads"]
    out = torch.zeros((s["total"], c["heads"], hd), dtype=torch.float64, device=DEV)
    lse = torch.full((s["total"], c["heads"]), -math.inf, dtype=torch.float64, device=DEV)
    shared = [x[s["shared"].long()].flatten(0, 1)[: c["prefix"]].double() for x in (s["k_cache"], s["v_cache"])]
    for b in range(c["seqs"]):
        lo, n = off[b], off[b + 1] - off[b]
        if n == 0:
            continue
        mine = [x[s["table"][b].long()].flatten(0, 1)[: lens[b]].double() for x in (s["k_cache"], s["v_cache"])]
        k, v = (torch.cat((x, y)) for x, y in zip(shared, mine))                    # [L][kv][hd]
        q = s["q"][lo: lo + n].double().unflatten(1, (c["kv_heads"], per))
        x = torch.einsum("nkgd,lkd->nkgl", q, k) / math.sqrt(hd)
        sees = torch.arange(k.shape[0], device=DEV)[None] < c["prefix"] + lens[b] - n + 1 + torch.arange(n, device=DEV)[:, None]
        x = x.masked_fill(~sees[:, None, None], -math.inf)
        lse[lo: lo + n] = torch.logsumexp(x, -1).flatten(1)
        out[lo: lo + n] = torch.einsum("nkgl,lkd->nkgd", torch.softmax(x, -1), v).flatten(1, 2)
    return {"out": out, "lse": lse}


# ---------------------------------------------------------------------------- work
def work(case):
    c = dict(case)
    rows = c["seqs"] * (c.get("rows", 0) / 2 if c["ragged"] else c.get("rows", 0))  # the expected ones where ragged
    if c["op"] == "append":
        e, z = SIZE[c["type"]], SIZE[c["cache"]]
        per = c["head_dim"] * (c["heads"] * 2 * e + c["kv_heads"] * 2 * (e + z))
        return {"bytes": rows * per + c["seqs"] * 12, "flops": rows * (c["heads"] + c["kv_heads"]) * c["rot"] * 3}
    if c["op"] == "attention":
        z, hd = SIZE[c["type"]], c["head_dim"]
        mine = c["seqs"] * (c["own_min"] + c["own_max"]) / 2
        keys = rows * (c["prefix"] + (c["own_min"] + c["own_max"]) / 2)
        return {"bytes": (c["prefix"] + mine) * c["kv_heads"] * hd * 2 * z + rows * c["heads"] * (hd * 2 * z + 4),
                "flops": 4.0 * keys * c["heads"] * hd}
    # the drafted tokens' probabilities, and the target's and the draft's row of each draw: a
    # frame ends the run where one of its codebooks was refused, and only those are drawn
    keep = {0.3: 0.88, 0.7: 0.72, 1.5: 0.45}.get(c["apart"], 0.7) if c["draft_probs"] else 0.3
    n, C = c["drafts"] / (2 if c["ragged"] else 1), c["codebooks"]
    full = keep ** (C * n)
    drawn = C * (full + (1 - full) * (1 - keep) / (1 - keep ** C))
    both = 2 if c["draft_probs"] else 1
    return {"bytes": c["seqs"] * (n * C * (both * SIZE[c["type"]] + 12) + drawn * (c["vocab"] * SIZE[c["type"]] * both + 8)
                                  + (c["drafts"] + 1) * C * 4),
            "flops": c["seqs"] * drawn * c["vocab"] * 2}
