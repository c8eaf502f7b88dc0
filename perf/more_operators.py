"""The operators of serving from a paged cache and of drafted tokens, as measurable cases.

Three entry points of ``them_bones_b200.ops``: ``paged_append`` (RoPE and norm of the new queries and keys, keys and values into
their pages), ``paged_attention`` (pieces of new tokens, from one token a sequence to whole prompts, against the pages) and
``verify_drafts`` (which of a sequence's drafted tokens the target's logits let stand, and the token behind them).  The sizes are
those of the benchmark models (10 heads of 128, vocabulary 65536, sequences of 2048, 64 sequences a decode step), of the tiny
model (4 heads of 64, vocabulary 8192) and of caches far longer than the training sequence.

``listed`` gives the fixed cases, ``draw`` further ones of the same ranges, ``prepare`` what a program holds before the call, ``run``
the call (in plain torch where ``own`` is false), ``work`` the bytes and operations it cannot do without and ``exact`` the results
in 64 bits.

The new tokens of all sequences lie one after another: sequence b's are the rows ``starts[b] .. starts[b + 1]``, at the positions
from ``pos[b]`` on.  A cache is two tensors ``[pages, H, P, D]`` of P tokens a page; position p of sequence b is in page
``table[b, p // P]``.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BF16 = torch.bfloat16
EPS = 2.0 ** -23


# -- the cases ---------------------------------------------------------------------------------------------------------
def listed():
    return [
        # a batch of prompts of one length goes into an empty cache
        dict(name="append_prompts", kind="append", b=8, heads=10, head_dim=128, page=64, tokens=2048, ragged=False, held=0, spread="same"),
        # a decode step of 64 sequences: latency
        dict(name="append_step", kind="append", b=64, heads=10, head_dim=128, page=64, tokens=1, ragged=False, held=2047, spread="even"),
        # pieces of prompts of odd lengths, the tiny model's heads, small pages, some sequences without a token
        dict(name="append_pieces", kind="append", b=24, heads=4, head_dim=64, page=16, tokens=333, ragged=True, held=1024, spread="even"),
        # one user, a short answer: latency
        dict(name="attend_one", kind="attend", b=1, heads=10, head_dim=128, page=64, tokens=1, ragged=False, held=299, spread="same", docs=False, window=0),
        # a decode step of 64 sequences of up to 2048 tokens in documents
        dict(name="attend_step", kind="attend", b=64, heads=10, head_dim=128, page=64, tokens=1, ragged=False, held=2047, spread="even", docs=True, window=0),
        # a step that verifies up to four drafts a sequence
        dict(name="attend_drafts", kind="attend", b=32, heads=10, head_dim=128, page=64, tokens=5, ragged=True, held=1500, spread="even", docs=False, window=0),
        # few sequences, a long cache
        dict(name="attend_long", kind="attend", b=4, heads=10, head_dim=128, page=128, tokens=1, ragged=False, held=131071, spread="even", docs=False, window=0),
        # prompts from their first token on
        dict(name="attend_prompts", kind="attend", b=8, heads=10, head_dim=128, page=64, tokens=2048, ragged=False, held=0, spread="same", docs=False, window=0),
        # the last piece of one long prompt
        dict(name="attend_piece", kind="attend", b=1, heads=10, head_dim=128, page=128, tokens=512, ragged=False, held=15900, spread="same", docs=False, window=0),
        # pieces of every length in one call, a banded layer of the tiny model's heads, small pages
        dict(name="attend_mixed", kind="attend", b=24, heads=4, head_dim=64, page=16, tokens=700, ragged=True, held=1800, spread="even", docs=True, window=512),
        # what the target's logits say of up to four drafts for each of 64 sequences, drawn from a smaller model
        dict(name="verify_step", kind="verify", b=64, drafts=4, ragged=True, vocab=65536, columns=65536, dtype="bf16", model=True, temperature=1.0),
        # one user, seven drafts looked up in the text, an odd vocabulary in padded rows
        dict(name="verify_one", kind="verify", b=1, drafts=7, ragged=False, vocab=8191, columns=8192, dtype="fp32", model=False, temperature=0.7),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(["append", "attend", "attend", "attend", "attend", "verify", "verify"])
    if kind == "verify":
        vocab = rng.choice([65536, 65536, 8192, 8 * rng.randint(100, 8000), rng.randint(200, 65535)])
        drafts, dtype = rng.randint(1, 12), rng.choice(["bf16", "bf16", "fp32"])
        b = _log_int(rng, 1, max(1, min(128, 320 * 65536 // ((drafts + 1) * vocab * (2 if dtype == "fp32" else 1)))))
        return dict(kind=kind, b=b, drafts=drafts, ragged=rng.random() < 0.5, vocab=vocab, columns=-(-vocab // 64) * 64 if rng.random() < 0.8 else vocab,
                    dtype=dtype, model=rng.random() < 0.6, temperature=rng.choice([1.0, 1.0, 0.7, 1.5, 0.0]))
    heads, head_dim = rng.choice([(10, 128), (10, 128), (4, 64), (16, 128), (5, 128), (3, 64)])
    page, tokens = rng.choice([16, 32, 64, 64, 128]), _log_int(rng, 1, 2048)
    case = dict(kind=kind, heads=heads, head_dim=head_dim, page=page, tokens=tokens, ragged=rng.random() < 0.6)
    if kind == "append":
        case.update(b=_log_int(rng, 1, max(1, min(64, 16384 * 10 * 128 // (tokens * heads * head_dim)))), held=rng.choice([0, rng.randint(1, 2000)]),
                    spread=rng.choice(["same", "even"]))
        return case
    held = _log_int(rng, 1, 131071 if tokens <= 16 else max(64, min(16384, 4096 * 2048 // tokens - tokens)))
    # bounded by the keys of a step and by the pairs of a piece
    pairs, keys = heads * tokens * (held + tokens), heads * head_dim * (held + tokens)
    b = _log_int(rng, 1, max(1, min(96, 4 * 10 * 2048 * 2048 // pairs, 2 * 10 * 128 * 131072 // keys)))
    case.update(b=b, held=held, spread=rng.choice(["same", "even", "even"]), docs=rng.random() < 0.5, window=rng.choice([0, 0, 128, 512]))
    return case


# -- lengths: the same set for every seed, in another order -------------------------------------------------------------
def _pieces(case):
    """``[(tokens held before, new tokens)]``, some sequences of a ragged case without a new token."""
    out = []
    for i in range(case["b"]):
        n = max(1, case["tokens"] * ((3 * i + 2) % 7 + 1) // 7) if case["ragged"] else case["tokens"]
        n = 0 if case["ragged"] and i % 7 == 3 else n
        out.append((case["held"] if case["spread"] == "same" else case["held"] * (i + 1) // case["b"], n))
    return out


def _document(i, p):
    """Start of the document that position p of the i-th sequence is in."""
    length = 190 + 173 * (i % 7)
    return p // length * length


def _first(case, i, p):
    lo = _document(i, p) if case["docs"] else 0
    return max(lo, (p // 128 - (case["window"] // 128 - 1)) * 128) if case["window"] else lo


def _drafts(case):
    return [(5 * i + 3) % (case["drafts"] + 1) if case["ragged"] else case["drafts"] for i in range(case["b"])]


# -- what a program holds before the call -------------------------------------------------------------------------------
def _normal(gen, *shape):
    return torch.randn(*shape, device=gen.device, dtype=BF16, generator=gen)


def _prepare_rows(st, case, gen, order):
    dev = gen.device
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    h, d, page = case["heads"], case["head_dim"], case["page"]
    pieces = [_pieces(case)[i] for i in order]
    n = sum(x for _, x in pieces)
    starts = [0]
    for _, x in pieces:
        starts.append(starts[-1] + x)
    need = [-(-(p + x) // page) for p, x in pieces]
    most, pages = max(1, max(need)), sum(need) + 3
    # pages as a program that has run for a while hands them out: in no order, the rest of a row without one
    slot = torch.randperm(pages, device=dev, generator=gen)
    row = torch.arange(most, device=dev)[None, :]
    need, base = torch.tensor(need, device=dev)[:, None], torch.tensor([sum(need[:i]) for i in range(len(need))], device=dev)[:, None]
    st["table"] = torch.where(row < need, slot[(base + row).clamp(max=pages - 1)], torch.full_like(row, -1)).to(torch.int32).contiguous()
    st["starts"], st["pos"] = ints(starts), ints([p for p, _ in pieces])
    st["longest"], st["length"] = max(x for _, x in pieces), max(p + x for p, x in pieces)
    st["n"] = n
    st["k"], st["v"] = _normal(gen, pages, h, page, d), _normal(gen, pages, h, page, d)
    if case["kind"] == "append":
        st["qkv"] = _normal(gen, n, 3 * h * d)
        angle = torch.arange(st["length"], device=dev, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, d, 2, device=dev, dtype=torch.float64) / d)
        st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
        return
    # queries and keys behind the norm, as `paged_append` leaves them
    q = _normal(gen, n, h, d).float()
    st["q"] = (q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS)).to(BF16).view(n, h * d)
    for part in st["k"].split(1024):
        part.copy_(part.float() * torch.rsqrt(part.float().square().mean(-1, keepdim=True) + EPS))
    st["doc_start"] = ints([_document(i, p + j) for i, (p, x) in zip(order, pieces) for j in range(x)]) if case["docs"] else None
    st["scale"], st["window"] = 1.0 / math.sqrt(d), case["window"]


def _prepare_drafts(st, case, gen, order):
    dev = gen.device
    count = [_drafts(case)[i] for i in order]
    n, v, c = sum(count) + len(count), case["vocab"], case["columns"]
    starts = torch.zeros(len(count) + 1, dtype=torch.int32, device=dev)
    starts[1:] = torch.tensor(count, device=dev).add(1).cumsum(0)
    spread = torch.exp(torch.rand(n, 1, device=dev, generator=gen) * 2.0 - 0.5)                   # flat rows and peaked ones
    z = 15.0 * torch.tanh(torch.randn(n, c, device=dev, generator=gen) * spread / 15.0)
    near = 15.0 * torch.tanh((z + 0.4 * torch.randn(n, c, device=dev, generator=gen)) / 15.0)       # a smaller model's view of the same text
    dt = torch.float32 if case["dtype"] == "fp32" else BF16
    z, near = z.to(dt), near.to(dt)
    # each draft from the smaller model at this temperature (or its best), as a program has them
    t = case["temperature"]
    noise = -torch.log(-torch.log(torch.rand(n, v, device=dev, generator=gen).clamp(1e-12, 1 - 1e-7))) if t else 0.0
    drawn = ((near[:, :v].float() / t if t else near[:, :v].float()) + noise).argmax(1)
    ids = torch.randint(0, v, (n,), device=dev, generator=gen)
    ids[1:] = torch.where(torch.isin(torch.arange(1, n, device=dev), starts[:-1].long()), ids[1:], drawn[:-1])
    st.update(logits=z, draft=near if case["model"] else None, ids=ids, starts=starts, uniforms=torch.rand(n, 2, device=dev, generator=gen))


def prepare(case, seed):
    gen = torch.Generator(device=torch.device("cuda")).manual_seed(seed)
    order = list(range(case["b"]))
    random.Random(seed).shuffle(order)
    st = dict(case=case)
    (_prepare_drafts if case["kind"] == "verify" else _prepare_rows)(st, case, gen, order)
    return st


# -- the plain forms -----------------------------------------------------------------------------------------------------
def _owner(starts, n):
    """Sequence of each row and its place in the piece."""
    row = torch.arange(n, device=starts.device)
    b = torch.searchsorted(starts.long(), row, right=True) - 1
    return b, row - starts.long()[b]


def _turn(x, c, s):
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    y = torch.cat([a * c + b * s, b * c - a * s], -1)
    return y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS)


def _plain_append(st):
    k, v, n = st["k"], st["v"], st["n"]
    _, h, page, d = k.shape
    b, i = _owner(st["starts"], n)
    p = st["pos"].long()[b] + i
    x = st["qkv"].float().view(n, 3, h, d)
    y = _turn(x[:, :2], st["cos"][p][:, None, None], st["sin"][p][:, None, None]).to(BF16)
    at = st["table"].long()[b, p // page]
    k[at, :, p % page] = y[:, 1]
    v[at, :, p % page] = x[:, 2].to(BF16)
    return [y[:, 0].reshape(n, h * d), k, v]


def _plain_attend(st):
    q, k, v, starts, pos, n = st["q"], st["k"], st["v"], st["starts"], st["pos"].long(), st["n"]
    _, h, page, d = k.shape
    dev, nseq, t = q.device, pos.shape[0], st["longest"]
    # every sequence's keys and values side by side [B, H, L, D], and its new tokens in rows of one length
    table = st["table"].long()
    at = table.clamp(min=0)
    length = table.shape[1] * page
    keys = k[at].float().transpose(1, 2).reshape(nseq, h, length, d)
    scores_at = torch.arange(t, device=dev)[None, :]
    rows = (starts.long()[:-1, None] + scores_at).clamp(max=max(n - 1, 0))
    real = scores_at < (starts[1:] - starts[:-1]).long()[:, None]
    p = pos[:, None] + scores_at
    lo = torch.zeros_like(p) if st["doc_start"] is None else st["doc_start"].long()[rows]
    if st["window"]:
        lo = torch.maximum(lo, (p // 128 - (st["window"] // 128 - 1)) * 128)
    j = torch.arange(length, device=dev)
    seen = ((j >= lo[..., None]) & (j <= p[..., None]) & real[..., None])[:, None]
    scores = torch.matmul(q.view(n, h, d).float()[rows].transpose(1, 2), keys.transpose(-1, -2)).mul_(st["scale"])
    scores.masked_fill_(~seen, -1e30)
    del keys
    scores -= scores.amax(-1, keepdim=True)
    w = scores.exp_().masked_fill_(~seen, 0.0)
    values = v[at].float().transpose(1, 2).reshape(nseq, h, length, d)
    y = torch.matmul(w, values) / w.sum(-1, keepdim=True).clamp(min=1e-30)
    return y.transpose(1, 2)[real].reshape(n, h * d).to(BF16)


def _softmax(z, t):
    e = torch.exp((z - z.amax(-1, keepdim=True)) / t)
    return e / e.sum(-1, keepdim=True)


def _plain_verify(st):
    case, v, t = st["case"], st["case"]["vocab"], st["case"]["temperature"]
    logits, ids, starts = st["logits"][:, :v], st["ids"], st["starts"].long()
    n, dev = logits.shape[0], logits.device
    b, i = _owner(st["starts"], n)
    following = torch.cat([ids[1:], ids[:1]])
    drafted = torch.arange(n, device=dev) + 1 < starts[b + 1]
    if t == 0.0:
        best = torch.max(logits, 1).indices
        stands = drafted & (best == following)
    else:
        # 64 bits: a probability next to its border decides between whole numbers
        z = logits.double()
        z = (z - z.amax(1, keepdim=True)) / t
        lse = torch.log(torch.exp(z).sum(1))
        px = torch.exp(z.gather(1, following[:, None])[:, 0] - lse)
        del z
        qx = torch.ones_like(px)
        if st["draft"] is not None:
            z = st["draft"][:, :v].double()
            z = (z - z.amax(1, keepdim=True)) / t
            qx = torch.exp(z.gather(1, following[:, None])[:, 0] - torch.log(torch.exp(z).sum(1)))
            del z
        stands = drafted & (st["uniforms"][:, 0].double() * qx < px)
    # the first row of each sequence that does not stand
    miss = torch.where(stands, n, torch.arange(n, device=dev))
    last = torch.full((starts.shape[0] - 1,), n, device=dev).scatter_reduce(0, b, miss, "amin")
    accepted = (last - starts[:-1]).to(torch.int32)
    if t == 0.0:
        return [accepted, best[last]]
    w = _softmax(logits[last].double(), t)
    refused = last + 1 < starts[1:]
    if st["draft"] is not None:
        w = torch.where(refused[:, None], (w - _softmax(st["draft"][last, :v].double(), t)).clamp(min=0.0), w)
    else:
        x = following[last][:, None]
        w.scatter_(1, x, torch.where(refused[:, None], torch.zeros_like(w[:, :1]), w.gather(1, x)))
    total = w.cumsum(1)
    token = torch.searchsorted(total, st["uniforms"][last, 1:2].double() * total[:, -1:], right=True)[:, 0]
    return [accepted, token.clamp(max=v - 1)]


# -- one pass -------------------------------------------------------------------------------------------------------------
def run(st):
    kind = st["case"]["kind"]
    if not own:
        return _plain_append(st) if kind == "append" else _plain_attend(st) if kind == "attend" else _plain_verify(st)
    from them_bones_b200 import ops
    if kind == "append":
        q = ops.paged_append(st["qkv"], st["cos"], st["sin"], ops.PagedKV(st["k"], st["v"]), st["table"], st["starts"], st["pos"])
        return [q, st["k"], st["v"]]
    if kind == "attend":
        return ops.paged_attention(st["q"], ops.PagedKV(st["k"], st["v"]), st["table"], st["starts"], st["pos"], st["scale"], doc_start=st["doc_start"],
                                   window=st["window"], longest=st["longest"])
    return list(ops.verify_drafts(st["logits"], st["ids"], st["starts"], st["uniforms"], draft_logits=st["draft"], temperature=st["case"]["temperature"],
                                  vocab=st["case"]["vocab"]))


def work(case):
    if case["kind"] == "verify":
        rows, drafted = sum(_drafts(case)) + case["b"], sum(_drafts(case))
        size = case["vocab"] * (4 if case["dtype"] == "fp32" else 2)
        n = rows + (drafted if case["model"] and case["temperature"] else 0)
        return {"bytes": n * size + 24 * rows + 12 * case["b"], "flops": 6 * n * case["vocab"]}
    hd, n = case["heads"] * case["head_dim"], sum(x for _, x in _pieces(case))
    if case["kind"] == "append":
        return {"bytes": 12 * hd * n + 4 * case["head_dim"] * n, "flops": 2 * hd * n * 8}
    keys = pairs = 0
    for i, (p, x) in enumerate(_pieces(case)):
        if x:
            keys += p + x - _first(case, i, p)
            pairs += sum(p + j + 1 - _first(case, i, p + j) for j in range(x))
    return {"bytes": 4 * hd * (n + keys), "flops": 4 * hd * pairs}


# -- the definitions in 64 bits ---------------------------------------------------------------------------------------------
def _exact_append(st):
    k, v = st["k"].double(), st["v"].double()
    _, h, page, d = k.shape
    out, starts = [], st["starts"].tolist()
    for b, p0 in enumerate(st["pos"].tolist()):
        a, e = starts[b], starts[b + 1]
        x = st["qkv"][a:e].double().view(e - a, 3, h, d)
        c, s = (st[name][p0:p0 + e - a].double()[:, None, None] for name in ("cos", "sin"))
        z = torch.complex(x[:, :2, :, :d // 2], x[:, :2, :, d // 2:]) * torch.complex(c, -s)             # a rotation by the negative angle
        z = torch.cat([z.real, z.imag], -1)
        z = z / torch.sqrt(z.square().mean(-1, keepdim=True) + EPS)
        out.append(z[:, 0].reshape(e - a, h * d))
        for f in range(p0 // page, -(-(p0 + e - a) // page)):                                             # a page at a time
            lo, hi = max(f * page, p0), min((f + 1) * page, p0 + e - a)
            at = int(st["table"][b, f])
            k[at, :, lo - f * page:hi - f * page] = z[lo - p0:hi - p0, 1].transpose(0, 1)
            v[at, :, lo - f * page:hi - f * page] = x[lo - p0:hi - p0, 2].transpose(0, 1)
    return [torch.cat(out), k, v]


def _exact_attend(st):
    q, k, v = st["q"], st["k"], st["v"]
    _, h, page, d = k.shape
    y, starts = torch.zeros(st["n"], h, d, dtype=torch.float64, device=q.device), st["starts"].tolist()
    for b, p0 in enumerate(st["pos"].tolist()):
        a, e = starts[b], starts[b + 1]
        if a == e:
            continue
        at = st["table"][b, :-(-(p0 + e - a) // page)].long()
        for g in range(h):
            kk, vv = (x[at, g].double().reshape(-1, d)[:p0 + e - a] for x in (k, v))
            for r in range(a, e, 512):
                m = min(r + 512, e)
                p = torch.arange(p0 + r - a, p0 + m - a, device=q.device)
                lo = st["doc_start"][r:m].long() if st["doc_start"] is not None else torch.zeros_like(p)
                if st["window"]:
                    lo = torch.maximum(lo, (p // 128 + 1) * 128 - st["window"])
                j = torch.arange(kk.shape[0], device=q.device)[None, :]
                s = (q[r:m].double().view(m - r, h, d)[:, g] @ kk.T) * st["scale"]
                s = torch.where((j < lo[:, None]) | (j > p[:, None]), torch.full_like(s, -math.inf), s)
                y[r:m, g] = torch.softmax(s, 1) @ vv
    return y.view(-1, h * d)


def _exact_verify(st):
    v, t, starts, ids = st["case"]["vocab"], st["case"]["temperature"], st["starts"].tolist(), st["ids"].tolist()
    law = lambda z, r: torch.log_softmax(z[r, :v].double() / t, 0).exp()  # noqa: E731
    accepted, tokens = [], []
    for a, e in zip(starts, starts[1:]):
        for r in range(a, e):
            more = r + 1 < e
            if t == 0.0:
                token = int(st["logits"][r, :v].max(0).indices)
                if more and token == ids[r + 1]:
                    continue
                break
            p = law(st["logits"], r)
            if more:
                x, (u, _) = ids[r + 1], st["uniforms"][r].tolist()
                q = torch.zeros_like(p)
                if st["draft"] is not None:
                    q = law(st["draft"], r)
                else:
                    q[x] = 1.0
                if u * float(q[x]) < float(p[x]):
                    continue
                p = torch.relu(p - q)
            below = p.cumsum(0) <= float(st["uniforms"][r, 1]) * p.sum()
            token = min(int(below.sum()), v - 1)
            break
        accepted.append(r - a)
        tokens.append(token)
    dev = st["ids"].device
    return [torch.tensor(accepted, dtype=torch.int32, device=dev), torch.tensor(tokens, device=dev)]


def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "verify": _exact_verify}[case["kind"]](st)
