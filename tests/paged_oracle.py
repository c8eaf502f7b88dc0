"""The paged cache, its attention and the verification of drafts in 64 bits, token by token or sequence by sequence, from the definitions alone."""
import math

import torch

EPS = 2.0 ** -23
HALF = 2.0 ** -8                       # a rounding to bf16 is off by this much of the value at most


def i32(v, dev="cpu"):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def rotated(x, c, s):
    """``x [.., D]`` rotated and normalised, fp64, and how far fp32 arithmetic may be from it: three roundings of each product's size."""
    d = x.shape[-1] // 2
    a, b = x[..., :d].double(), x[..., d:].double()
    c, s = c.double(), s.double()
    y = torch.cat([a * c + b * s, b * c - a * s], -1)
    size = torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()], -1)
    r = 1.0 / (y.square().mean(-1, keepdim=True) + EPS).sqrt()
    return y * r, size * r * 2.0 ** -21


def pieces(starts, pos):
    st = starts.tolist()
    return [(st[b], st[b + 1] - st[b], p) for b, p in enumerate(pos.tolist())]


def append(qkv, cos, sin, cache, table, starts, pos):
    """``(q, k, v)`` in fp64 as a call leaves them, and the tolerances of q and k (values are copied)."""
    k, v = (x.double().clone() for x in cache)
    n_pages, h, page, d = k.shape
    n = qkv.shape[0]
    q, qt, kt = torch.zeros(n, h, d, dtype=torch.float64, device=qkv.device), torch.zeros(n, h, d, dtype=torch.float64, device=qkv.device), torch.zeros_like(k)
    x = qkv.view(n, 3, h, d)
    for b, (a, m, p0) in enumerate(pieces(starts, pos)):
        for i in range(m):
            p = p0 + i
            if p0 < 0 or p >= min(table.shape[1] * page, cos.shape[0]):
                continue
            y, t = rotated(x[a + i, :2], cos[p], sin[p])
            q[a + i], qt[a + i] = y[0], HALF * y[0].abs() + t[0]
            at = int(table[b, p // page])
            if 0 <= at < n_pages:
                k[at, :, p % page], kt[at, :, p % page] = y[1], HALF * y[1].abs() + t[1]
                v[at, :, p % page] = x[a + i, 2].double()
    return (q.view(n, -1), k, v), (qt.view(n, -1), kt)


def first_key(p, start, window):
    return max(start, (p // 128 - (window // 128 - 1)) * 128 if window else 0, 0)


def attend(q, cache, table, starts, pos, scale, doc_start, window):
    """``y [N, H*D]`` in fp64 and its tolerance: probabilities and the result are rounded to bf16 once each, the exponentials and sums are
    fp32 (2^-16 of the weights' sum covers them)."""
    k, v = cache
    n_pages, h, page, d = k.shape
    n = q.shape[0]
    y, tol = torch.zeros(n, h, d, dtype=torch.float64, device=q.device), torch.zeros(n, h, d, dtype=torch.float64, device=q.device)
    for b, (a, m, p0) in enumerate(pieces(starts, pos)):
        live = 0 if p0 < 0 else min(m, max(0, table.shape[1] * page - p0))
        if not live:
            continue
        ids = table[b].long()[:-(-(p0 + live) // page)]
        there = ((ids >= 0) & (ids < n_pages)).repeat_interleave(page)[:p0 + live]
        kk, vv = (x[ids.clamp(0, n_pages - 1)].double().transpose(0, 1).reshape(h, -1, d)[:, :p0 + live] for x in (k, v))
        j = torch.arange(p0 + live, device=q.device)
        for i in range(live):
            p = p0 + i
            seen = torch.nonzero((j >= first_key(p, int(doc_start[a + i]) if doc_start is not None else 0, window)) & (j <= p) & there)[:, 0]
            if seen.numel() == 0:
                continue
            w = torch.softmax(torch.einsum("hd,hnd->hn", q[a + i].double().view(h, d), kk[:, seen]) * scale, -1)
            y[a + i] = torch.einsum("hn,hnd->hd", w, vv[:, seen])
            tol[a + i] = (HALF + 2.0 ** -16) * torch.einsum("hn,hnd->hd", w, vv[:, seen].abs()) + HALF * y[a + i].abs()
    return y.view(n, -1), tol.view(n, -1)


def world(b, h, d, page, lens, pos, dev="cpu", seed=0, spare=2, room=0):
    """A pool of pages in no order, a table and pieces: ``cache`` (normalised keys, values at random), ``table`` (-1 behind what a sequence needs),
    ``starts``, ``pos``."""
    from them_bones_b200 import ops
    g = torch.Generator().manual_seed(seed)
    need = [max(0, -(-(max(p, 0) + n) // page)) for p, n in zip(pos, lens)]
    m = max(1, max(need) + room)
    pages = sum(need) + spare
    c = ops.paged_cache(pages, h, d, page, dev)
    k = torch.randn(pages, h, page, d, generator=g)
    c.k.copy_(k / k.square().mean(-1, keepdim=True).sqrt())
    c.v.copy_(torch.randn(pages, h, page, d, generator=g))
    order, table, at = torch.randperm(pages, generator=g), torch.full((b, m), -1, dtype=torch.int32), 0
    for i, x in enumerate(need):
        table[i, :x] = order[at:at + x].int()
        at += x
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    return c, table.to(dev), i32(starts, dev), i32(pos, dev)


def queries(n, h, d, dev="cpu", seed=1):
    x = torch.randn(n, h, d, generator=torch.Generator().manual_seed(seed))
    return (x / x.square().mean(-1, keepdim=True).sqrt()).to(torch.bfloat16).view(n, h * d).to(dev)


def angles(rows, d, dev="cpu"):
    a = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    return a.cos().float().to(dev), a.sin().float().to(dev)


def law(row, t):
    """exp of differences in 64 bits by Python's own arithmetic; None for a row without a number."""
    z = [float(x) for x in row]
    m = max((x for x in z if x == x), default=-math.inf)
    if any(x != x for x in z) or m in (math.inf, -math.inf):
        return None
    e = [math.exp((x - m) / t) for x in z]
    s = math.fsum(e)
    return [x / s for x in e]


def verify(logits, ids, starts, uniforms, draft, t, vocab):
    """``[(accepted, token)]``, and for each sequence how near the closest decision was to its border (relative; 64-bit sums of 10^5 terms are off by 10^-12 at most)."""
    out, near = [], []
    st, ids = starts.tolist(), ids.tolist()
    u = uniforms.double().tolist() if uniforms is not None else None
    for a, e in zip(st, st[1:]):
        got, token, close = 0, -1, 1.0
        for r in range(a, e):
            p, x, more = law(logits[r, :vocab].tolist(), t or 1.0), ids[r + 1] if r + 1 < e else -1, r + 1 < e
            if p is None:
                break
            if t == 0:
                best = max(range(vocab), key=lambda i: (float(logits[r, i]), -i))
                if more and best == x:
                    got += 1
                    continue
                token = best
                break
            w = p
            if more:
                q = law(draft[r, :vocab].tolist(), t) if draft is not None else [0.0] * vocab
                if q is not None and 0 <= x < vocab:
                    if draft is None:
                        q[x] = 1.0
                    most = max(u[r][0] * q[x], p[x])
                    close = min(close, abs(u[r][0] * q[x] - p[x]) / most if most > 0 else 1.0)
                    if u[r][0] * q[x] < p[x]:
                        got += 1
                        continue
                if q is not None:
                    w = [max(pp - qq, 0.0) for pp, qq in zip(p, q)]
                    w = w if math.fsum(w) > 1e-12 else p        # q is p, or as good as
            total, c = math.fsum(w), 0.0
            for i, x in enumerate(w):
                c += x
                if x > 0:
                    token = i
                    close = min(close, abs(c - u[r][1] * total) / total)
                    if c > u[r][1] * total:
                        break
            break
        out.append((got, token))
        near.append(close)
    return out, near
