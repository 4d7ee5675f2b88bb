"""Plain 64-bit restatements of the device-buffer operators (include/z2b_ops.h), row by row on
the CPU, for the GPU tests."""
from __future__ import annotations

import math

import torch


def freqs(rot, base=10000.0, scaling="none", factor=1.0, orig_ctx=0):
    i = torch.arange(rot // 2, dtype=torch.float64)
    mag = 1.0
    if scaling == "ntk":
        base = base * factor ** (rot / (rot - 2))
    w = base ** (-2 * i / rot)
    if scaling == "linear":
        w = w / factor
    if scaling == "by_parts":
        keep = torch.clamp((orig_ctx * w / (2 * math.pi) - 1) / 31, 0, 1)
        w = w / factor * (1 - keep) + w * keep
        mag = 0.1 * math.log(factor) + 1
    return w, mag


def rotate(x, pos, w, mag, layout):
    """x [heads][hd] (f64) at position pos."""
    rot = 2 * len(w)
    a, b = (x[:, : rot // 2], x[:, rot // 2: rot]) if layout == "half" else (x[:, 0:rot:2], x[:, 1:rot:2])
    c, s = torch.cos(pos * w) * mag, torch.sin(pos * w) * mag
    e, o = a * c - b * s, b * c + a * s
    y = x.clone()
    if layout == "half":
        y[:, : rot // 2], y[:, rot // 2: rot] = e, o
    else:
        y[:, 0:rot:2], y[:, 1:rot:2] = e, o
    return y


def attention(q, k_cache, v_cache, off, lens, table, prefix_pages, prefix_len, scale):
    """(out, lse, sum of p |v|, largest sum of |q k| scale): f64, rows behind off[-1] are NaN."""
    q, kc, vc = q.double(), k_cache.double(), v_cache.double()
    page, nkv = kc.shape[1], kc.shape[2]
    per = q.shape[1] // nkv
    out = torch.full(q.shape, math.nan, dtype=torch.float64)
    lse = torch.full(q.shape[:2], math.nan, dtype=torch.float64)
    spread = torch.full(q.shape, math.nan, dtype=torch.float64)
    most = 0.0

    def rows(pages, n):
        if n == 0:
            return kc.new_zeros((0, nkv, kc.shape[3])), vc.new_zeros((0, nkv, kc.shape[3]))
        p = pages[: -(-n // page)].long()
        return kc[p].flatten(0, 1)[:n], vc[p].flatten(0, 1)[:n]

    kp, vp = rows(prefix_pages, prefix_len) if prefix_len else rows(None, 0)
    for b in range(len(lens)):
        n = off[b + 1] - off[b]
        ko, vo = rows(table[b], lens[b])
        for i in range(n):
            t = off[b] + i
            sees = max(0, lens[b] - n + i + 1)
            k, v = torch.cat((kp, ko[:sees])), torch.cat((vp, vo[:sees]))
            for h in range(q.shape[1]):
                x = (k[:, h // per] @ q[t, h]) * scale
                if len(x) == 0:
                    out[t, h], lse[t, h], spread[t, h] = 0.0, -math.inf, 0.0
                    continue
                p = torch.softmax(x, 0)
                lse[t, h] = torch.logsumexp(x, 0)
                out[t, h] = p @ v[:, h // per]
                spread[t, h] = p @ v[:, h // per].abs()
                most = max(most, float((k[:, h // per].abs() @ q[t, h].abs()).max() * abs(scale)))
    return out, lse, spread, most


def verify(p, q, draft, u, r, n_draft):
    """Tokens and kept counts; p, q as given (any type), q None for a certain draft."""
    B, N1, C, V = p.shape
    tokens = torch.full((B, N1, C), -1, dtype=torch.int32)
    kept = torch.zeros(B, dtype=torch.int32)
    for b in range(B):
        n = int(n_draft[b]) if n_draft is not None else N1 - 1
        for f in range(n + 1):
            refused = []
            for c in range(C):
                x = int(draft[b, f, c]) if f < n else -1
                if f < n:
                    qx = float(q[b, f, c, x]) if q is not None else 1.0
                    if float(u[b, f, c]) * qx < float(p[b, f, c, x]):
                        tokens[b, f, c] = x
                        continue
                refused.append(c)
                row = p[b, f, c].double()
                left = row.clamp(min=0)
                if f < n:
                    take = q[b, f, c].double() if q is not None else torch.nn.functional.one_hot(torch.tensor(x), V).double()
                    rest = (row - take).clamp(min=0)
                    if float(rest.sum()) > 0:
                        left = rest
                cum = left.cumsum(0)
                if not float(cum[-1]) > 0:
                    tokens[b, f, c] = -1
                    continue
                past = (cum > float(r[b, f, c]) * cum[-1]).nonzero()
                tokens[b, f, c] = int(past[0]) if len(past) else int((left > 0).nonzero()[-1])
            if refused or f == n:
                kept[b] = f
                break
    return tokens, kept
