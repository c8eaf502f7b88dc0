"""The operators of low-memory serving and of what a model's answers are worth, as measurable cases.

Four entry points of ``them_bones_b200.ops``: ``kv8_append`` and ``kv8_read`` (keys and values into an 8-bit cache with a
scale for each block of 64 tokens and head, and back), ``kv8_attention`` (one token a sequence against such a cache:
RoPE and norm of the new query and key, append, attention) and ``token_logprobs`` (log-probability of given tokens,
entropy and the most probable alternatives of each row of logits, and the gradient).  The sizes are those of the
benchmark models (10 heads of 128, vocabulary 65536, sequences of 2048, 64 sequences a decode step), of the tiny model
(4 heads of 64, vocabulary 8192) and of caches far longer than the training sequence.

``listed`` gives the fixed cases, ``draw`` further ones of the same ranges, ``prepare`` what a program holds before the
call, ``run`` the call (in plain 32-bit torch where ``own`` is false), ``work`` the bytes and operations it cannot do
without and ``exact`` the results in 64 bits.

A cache is six tensors: codes of the keys ``[B, H, T, D]`` and of the values ``[B, H, T/64, D, 64]`` (int8, the values of
a block transposed), their scales ``[B, H, T/64]`` and the open block, whose tokens are kept in bf16 until it is full,
``[B, H, 64, D]``.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BF16 = torch.bfloat16
BLOCK = 64
EPS = 2.0 ** -23


# -- the cases ---------------------------------------------------------------------------------------------------------
def listed():
    return [
        # a batch of prompts of one length goes into an empty cache
        dict(name="fill_prompts", kind="fill", b=8, heads=10, head_dim=128, held=0, tokens=2048, ragged=False),
        # a further piece of every prompt, of another length in each sequence, behind what the cache holds
        dict(name="fill_pieces", kind="fill", b=24, heads=4, head_dim=64, held=1024, tokens=333, ragged=True),
        # one user, a short answer: latency
        dict(name="attend_one", kind="attend", b=1, heads=10, head_dim=128, length=300, spread="same", docs=False, window=0, idle=False),
        # a decode step of 64 sequences of up to 2048 tokens in documents
        dict(name="attend_step", kind="attend", b=64, heads=10, head_dim=128, length=2048, spread="even", docs=True, window=0, idle=False),
        # the tiny model's heads in a banded layer, some sequences of the batch done
        dict(name="attend_banded", kind="attend", b=37, heads=4, head_dim=64, length=2000, spread="even", docs=True, window=512, idle=True),
        # a step in which every sequence fills its block
        dict(name="attend_closing", kind="attend", b=32, heads=10, head_dim=128, length=1536, spread="closing", docs=False, window=0, idle=False),
        # few sequences, a long cache
        dict(name="attend_long", kind="attend", b=4, heads=10, head_dim=128, length=131072, spread="even", docs=False, window=0, idle=False),
        # what a decode step's logits say about its 64 answers
        dict(name="score_step", kind="score", rows=64, vocab=65536, columns=65536, dtype="bf16", topk=8, backward=False),
        # and about one
        dict(name="score_one", kind="score", rows=1, vocab=65536, columns=65536, dtype="bf16", topk=20, backward=False),
        # two windows of text scored from the model's fp32 logits
        dict(name="score_text", kind="score", rows=4096, vocab=65536, columns=65536, dtype="fp32", topk=5, backward=False),
        # a block of rows of a policy's step: log-probability and entropy, and the gradient of both
        dict(name="train_policy", kind="score", rows=4096, vocab=65536, columns=65536, dtype="bf16", topk=0, backward=True),
        # a small odd vocabulary in padded rows, with a gradient to the alternatives as in distillation
        dict(name="train_odd", kind="score", rows=777, vocab=8191, columns=8192, dtype="fp32", topk=3, backward=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(["fill", "attend", "attend", "attend", "score", "score", "train"])
    if kind in ("fill", "attend"):
        heads, head_dim = rng.choice([(10, 128), (10, 128), (4, 64), (16, 128), (5, 128), (3, 64)])
    if kind == "fill":
        tokens, held = _log_int(rng, 1, 4096), rng.choice([0, BLOCK * _log_int(rng, 1, 32), rng.randint(1, 2000)])
        b = _log_int(rng, 1, max(1, min(64, 16384 * 10 * 128 // (max(tokens + held, 256) * heads * head_dim))))
        return dict(kind=kind, b=b, heads=heads, head_dim=head_dim, held=held, tokens=tokens, ragged=rng.random() < 0.6)
    if kind == "attend":
        length = _log_int(rng, 1, 131072)
        b = _log_int(rng, 1, max(1, min(128, 4 * 10 * 128 * 131072 // (length * heads * head_dim))))
        spread = rng.choice(["same", "even", "even", "closing"])
        return dict(kind=kind, b=b, heads=heads, head_dim=head_dim, length=-(-length // BLOCK) * BLOCK if spread == "closing" else length, spread=spread,
                    docs=rng.random() < 0.5, window=rng.choice([0, 0, 128, 512]), idle=spread != "same" and b > 2 and rng.random() < 0.3)
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    rows, vocab = _log_int(rng, 1, 2048 if dtype == "fp32" else 4096), rng.choice([65536, 65536, 8192, 8 * rng.randint(100, 8000), rng.randint(200, 65535)])
    topk = rng.choice([0, 1, 4, rng.randint(2, 32)])
    return dict(kind="score", rows=rows, vocab=vocab, columns=-(-vocab // 64) * 64 if rng.random() < 0.8 else vocab, dtype=dtype,
                topk=topk, backward=kind == "train")


# -- positions: the same set for every seed, in another order ---------------------------------------------------------
def _positions(case):
    """``[(position of the new token, first visible one)]`` of an ``attend`` case; an idle sequence is at -1."""
    b, length, out = case["b"], case["length"], []
    for i in range(b):
        pos = length - 1 if case["spread"] == "same" else max(0, length * (i + 1) // b - 1)
        if case["spread"] == "closing":
            pos = pos // BLOCK * BLOCK + BLOCK - 1
        start = pos * (5 * i % 8) // 8 if case["docs"] else 0
        if case["docs"] and i % 16 == 7:
            start = pos
        out.append((-1, 0) if case["idle"] and i % 5 == 2 else (pos, start))
    return out


def _first_key(pos, start, window):
    return max(start, (pos // 128 - (window // 128 - 1)) * 128 if window else 0, 0)


def _pieces(case):
    """``[(tokens held, tokens to add)]`` of a ``fill`` case.  A piece that goes over the end of a block begins with one (a call can
    then be made again on the same cache)."""
    out = []
    for i in range(case["b"]):
        held = case["held"] - (BLOCK * (i % 4) if case["ragged"] and case["held"] >= 4 * BLOCK else 0)
        n = max(1, case["tokens"] * ((3 * i + 2) % 7 + 1) // 7) if case["ragged"] else case["tokens"]
        n = 0 if case["ragged"] and i % 7 == 3 else n
        if held % BLOCK + n > BLOCK:
            held -= held % BLOCK
        out.append((held, n))
    return out


# -- what a program holds before the call -------------------------------------------------------------------------------
def _capacity(n):
    return max(1, -(-n // BLOCK)) * BLOCK


def _cache(gen, b, heads, head_dim, capacity):
    """A cache of keys and values whose entries are spread like those behind a norm, the scales those of their largest ones."""
    dev = gen.device
    codes = lambda *shape: (torch.randn(*shape, device=dev, dtype=torch.float16, generator=gen) * 32).round_().clamp_(-127, 127).to(torch.int8)  # noqa: E731
    nb = capacity // BLOCK
    scales = lambda: (3.5 + torch.rand(b, heads, nb, device=dev, generator=gen)) / 127  # noqa: E731
    tail = lambda: torch.randn(b, heads, BLOCK, head_dim, device=dev, generator=gen).to(BF16)  # noqa: E731
    return (codes(b, heads, capacity, head_dim), codes(b, heads, nb, head_dim, BLOCK), scales(), scales(), tail(), tail())


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    order = list(range(case.get("b", 0)))
    random.Random(seed).shuffle(order)
    st = dict(case=case)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    if case["kind"] == "attend":
        b, h, d = case["b"], case["heads"], case["head_dim"]
        at = [_positions(case)[i] for i in order]
        cap = _capacity(case["length"])
        st["cache"] = _cache(gen, b, h, d, cap)
        st["qkv"] = torch.randn(b, 3 * h * d, device=dev, generator=gen).to(BF16)
        angle = torch.arange(cap, device=dev, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, d, 2, device=dev, dtype=torch.float64) / d)
        st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
        st["pos"] = ints([case["length"] - 1]) if case["spread"] == "same" else ints([p for p, _ in at])
        st["doc_start"] = ints([s for _, s in at]) if case["docs"] else None
        st["scale"], st["window"] = 1.0 / math.sqrt(d), case["window"]
        if case["spread"] == "closing":
            st["row"], st["block"] = torch.arange(b, device=dev), ints([max(p, 0) // BLOCK for p, _ in at]).long()
    elif case["kind"] == "fill":
        b, h, d, t = case["b"], case["heads"], case["head_dim"], case["tokens"]
        pieces = [_pieces(case)[i] for i in order]
        st["length"] = max(p + n for p, n in pieces)
        st["cache"] = _cache(gen, b, h, d, _capacity(st["length"]))
        packed = torch.randn(b, t, 3 * h * d, device=dev, generator=gen).to(BF16)       # keys and values lie as a projection leaves them
        st["k"], st["v"] = (packed[..., i * h * d:(i + 1) * h * d].view(b, t, h, d) for i in (1, 2))
        st["pos"], st["lens"] = ints([p for p, _ in pieces]), ints([n for _, n in pieces])
        st["held"] = st["pos"] + st["lens"]
    else:
        rows, v, c, k = case["rows"], case["vocab"], case["columns"], case["topk"]
        spread = torch.exp(torch.rand(rows, 1, device=dev, generator=gen) * 2.0 - 0.5)            # flat rows and peaked ones
        z = 15.0 * torch.tanh(torch.randn(rows, c, device=dev, generator=gen) * spread / 15.0)
        st["logits"] = (z if case["dtype"] == "fp32" else z.to(BF16)).requires_grad_(case["backward"])
        tokens = torch.randint(0, v, (rows,), device=dev, generator=gen)
        best = z[:, :v].argmax(1)
        i = torch.arange(rows, device=dev)
        tokens = torch.where(i % 3 == 1, best, tokens)
        st["tokens"] = torch.where(i % 16 == 9, torch.full_like(tokens, -1), tokens)
        if case["backward"]:
            st["grads"] = [torch.randn(rows, device=dev, generator=gen) / rows, 0.1 * torch.randn(rows, device=dev, generator=gen) / rows]
            if k:
                st["grads"].append(torch.randn(rows, k, device=dev, generator=gen) / rows)
    return st


# -- the plain forms -----------------------------------------------------------------------------------------------------
def _quantise(x):
    """``x [.., 64, D]`` as codes and the block's scale."""
    most = x.abs().amax((-1, -2), keepdim=True)
    return torch.round(x * (127.0 / most)).clamp(-127, 127).to(torch.int8), (most / 127.0)[..., 0, 0]


def _plain_fill(k, v, cache, pos, lens, held, length):
    k8, v8, ks, vs, kt, vt = cache
    b, t, h, d = k.shape
    dev, nb = k.device, k8.shape[2] // BLOCK
    span = (t + 2 * BLOCK - 2) // BLOCK + 1                                    # blocks that a piece can touch
    first = pos.long() // BLOCK
    at = torch.arange(span * BLOCK, device=dev)[None, :]                       # from the start of the first block
    old, end = (pos.long() % BLOCK)[:, None], (pos.long() % BLOCK + lens.long())[:, None]
    rows = torch.arange(b, device=dev)[:, None]
    for new, tail, codes, scales in ((k, kt, k8, ks), (v, vt, v8, vs)):
        x = new[rows, (at - old).clamp(0, t - 1)].float().transpose(1, 2)      # [B, H, span * 64, D]
        x[:, :, :BLOCK] = torch.where((at < old)[:, None, :BLOCK, None], tail.float(), x[:, :, :BLOCK])
        x = torch.where((at < end)[:, None, :, None], x, torch.zeros((), device=dev))
        blocks = x.view(b, h, span, BLOCK, d)
        q, s = _quantise(blocks)
        rel = torch.arange(nb, device=dev)[None, :] - first[:, None]           # a block of the cache among those of the piece
        full = ((rel >= 0) & ((rel + 1) * BLOCK <= end) & (end > old))[:, None, :]
        rel = rel.clamp(0, span - 1)[:, None, :].expand(b, h, nb)
        scales.copy_(torch.where(full, s.gather(2, rel), scales))
        full, rel = full[..., None, None], rel[..., None, None].expand(b, h, nb, BLOCK, d)
        if codes is k8:
            old8 = codes.view(b, h, nb, BLOCK, d)
            old8.copy_(torch.where(full, q.gather(2, rel), old8))
        else:
            codes.copy_(torch.where(full, q.gather(2, rel).transpose(-1, -2), codes))
        last = (end // BLOCK)[:, 0]                                            # the block that stays open, if a token is in it
        keep = torch.arange(BLOCK, device=dev)[None, :] < end - last[:, None] * BLOCK
        fresh = blocks[torch.arange(b, device=dev), :, last.clamp(max=span - 1)]
        tail.copy_(torch.where((keep & (lens.long() > 0)[:, None])[:, None, :, None], fresh, tail.float()))
    return _plain_read(cache, held, length) + (ks, vs, kt, vt)


def _assemble(cache, blk, n):
    """Keys and values ``[B, H, n, D]`` in 32 bits: the codes times their scales, block ``blk[b]`` from the open one."""
    k8, v8, ks, vs, kt, vt = cache
    b, h, _, d = k8.shape
    nb = n // BLOCK
    k = (k8[:, :, :n].reshape(b, h, nb, BLOCK, d).float() * ks[:, :, :nb, None, None]).view(b, h, n, d)
    v = (v8[:, :, :nb].float() * vs[:, :, :nb, None, None]).transpose(-1, -2).reshape(b, h, n, d)
    at = (blk[:, None] * BLOCK + torch.arange(BLOCK, device=k.device)[None, :])[:, None, :, None]
    ok = at < n
    at = at.clamp(max=n - 1).expand(b, h, BLOCK, d)
    k.scatter_(2, at, torch.where(ok, kt.float(), k.gather(2, at)))
    v.scatter_(2, at, torch.where(ok, vt.float(), v.gather(2, at)))
    return k, v


def _plain_read(cache, held, length):
    k, v = _assemble(cache, held.long() // BLOCK, cache[0].shape[2])
    live = (torch.arange(length, device=k.device)[None, :] < held[:, None])[:, :, None, None]
    return tuple(torch.where(live, x[:, :, :length].transpose(1, 2), torch.zeros((), device=k.device)).to(BF16) for x in (k, v))


def _turn(x, c, s):
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    y = torch.cat([a * c + b * s, b * c - a * s], -1)
    return y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS)


def _plain_attend(qkv, cos, sin, cache, pos, scale, doc_start, window, length):
    k8, v8, ks, vs, kt, vt = cache
    b, h, _, d = k8.shape
    dev = qkv.device
    p = pos.long().expand(b)
    live, p = p >= 0, p.clamp(min=0)
    q, k, v = qkv.float().view(b, 3, h, d).unbind(1)
    c, s = cos[p][:, None], sin[p][:, None]
    q, k = _turn(q, c, s), _turn(k, c, s)
    rows, slot, blk = torch.arange(b, device=dev), p % BLOCK, p // BLOCK
    on = live[:, None, None]
    kt[rows, :, slot] = torch.where(on, k.to(BF16), kt[rows, :, slot])
    vt[rows, :, slot] = torch.where(on, v.to(BF16), vt[rows, :, slot])
    n = _capacity(length)
    keys, values = _assemble(cache, blk, n)
    scores = (keys * q[:, :, None, :]).sum(-1) * scale
    j = torch.arange(n, device=dev)[None, :]
    lo = torch.zeros_like(p) if doc_start is None else doc_start.long()
    if window:
        lo = torch.maximum(lo, (p // 128 - (window // 128 - 1)) * 128)
    seen = ((j >= lo[:, None]) & (j <= p[:, None]) & live[:, None])[:, None, :]
    top = torch.where(seen, scores, torch.full((), -1e30, device=dev)).amax(-1, keepdim=True)
    w = torch.where(seen, torch.exp(scores - top), torch.zeros((), device=dev))
    y = (w[..., None] * values).sum(2) / w.sum(-1, keepdim=True).clamp(min=1e-30)
    # a full block becomes codes
    full = live & (slot == BLOCK - 1)
    kq, kscale = _quantise(kt.float())
    vq, vscale = _quantise(vt.float())
    k5 = k8.view(b, h, -1, BLOCK, d)
    k5[rows, :, blk] = torch.where(full[:, None, None, None], kq, k5[rows, :, blk])
    v8[rows, :, blk] = torch.where(full[:, None, None, None], vq.transpose(-1, -2), v8[rows, :, blk])
    ks[rows, :, blk] = torch.where(full[:, None], kscale, ks[rows, :, blk])
    vs[rows, :, blk] = torch.where(full[:, None], vscale, vs[rows, :, blk])
    return y.reshape(b, h * d).to(BF16)


def _closed(st):
    """The blocks that an ``attend`` case fills, as the values that their codes stand for."""
    k8, v8, ks, vs, _, _ = st["cache"]
    b, h, _, d = k8.shape
    i, blk = st["row"], st["block"]
    return [(k8.view(b, h, -1, BLOCK, d)[i, :, blk] * ks[i, :, blk][..., None, None]).to(BF16), (v8[i, :, blk] * vs[i, :, blk][..., None, None]).to(BF16)]


def _plain_logprobs(logits, tokens, topk, vocab):
    z = logits[:, :vocab].float()
    z = z - z.amax(1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    logp = z - torch.log(total)
    p = e / total
    entropy = -(p * logp).sum(1)
    given = logp.gather(1, tokens.clamp(min=0)[:, None])[:, 0] * (tokens >= 0)
    if not topk:
        return given, entropy, logp[:, :0], tokens[:, None][:, :0], p, logp
    ids = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :topk]
    return given, entropy, logp.gather(1, ids), ids, p, logp


def _plain_score(st):
    case, tokens = st["case"], st["tokens"]
    given, entropy, top, ids, p, logp = _plain_logprobs(st["logits"].detach(), tokens, case["topk"], case["vocab"])
    if not case["backward"]:
        return [given, entropy, top, ids] if case["topk"] else [given, entropy]
    g, gh = st["grads"][0] * (tokens >= 0), st["grads"][1]
    pull = g + (st["grads"][2].sum(1) if case["topk"] else 0)
    d = -p * (pull[:, None] + gh[:, None] * (logp + entropy[:, None]))
    d.scatter_add_(1, tokens.clamp(min=0)[:, None], g[:, None])
    if case["topk"]:
        d.scatter_add_(1, ids, st["grads"][2])
    dz = torch.zeros_like(st["logits"])
    dz[:, :case["vocab"]] = d.to(dz.dtype)
    return [given, entropy] + ([top, ids] if case["topk"] else []) + [dz]


# -- one pass -------------------------------------------------------------------------------------------------------------
def run(st):
    case = st["case"]
    if case["kind"] == "fill":
        if not own:
            return list(_plain_fill(st["k"], st["v"], st["cache"], st["pos"], st["lens"], st["held"], st["length"]))
        from them_bones_b200 import ops
        cache = ops.KV8(*st["cache"])
        ops.kv8_append(cache, st["k"], st["v"], st["pos"], st["lens"])
        return list(ops.kv8_read(cache, st["held"], st["length"])) + list(cache[2:])
    if case["kind"] == "attend":
        if not own:
            y = _plain_attend(st["qkv"], st["cos"], st["sin"], st["cache"], st["pos"], st["scale"], st["doc_start"], st["window"], case["length"])
        else:
            from them_bones_b200 import ops
            y = ops.kv8_attention(st["qkv"], st["cos"], st["sin"], ops.KV8(*st["cache"]), st["pos"], st["scale"], st["doc_start"], st["window"])
        return [y, st["cache"][4], st["cache"][5]] + (_closed(st) if case["spread"] == "closing" else [])
    if not own:
        return _plain_score(st)
    from them_bones_b200 import ops
    r = ops.token_logprobs(st["logits"], st["tokens"], case["topk"], case["vocab"])
    out = [r.logprob, r.entropy] + ([r.top_logprob, r.top_id] if case["topk"] else [])
    if case["backward"]:
        at = [r.logprob, r.entropy] + ([r.top_logprob] if case["topk"] else [])
        out = [x.detach() for x in out] + list(torch.autograd.grad(at, [st["logits"]], st["grads"]))
    return out


def work(case):
    if case["kind"] == "fill":
        hd, t = case["heads"] * case["head_dim"], sum(n for _, n in _pieces(case))
        length = max(p + n for p, n in _pieces(case))
        held = sum(p for p, _ in _pieces(case))
        # new tokens are read in bf16 and written in 8 bits; what was held is read in 8 bits; everything is written out in bf16
        return {"bytes": 2 * hd * (t * 2 + t + held + case["b"] * length * 2), "flops": 2 * hd * (3 * t + held + t)}
    if case["kind"] == "attend":
        hd, keys, open_keys, live = case["heads"] * case["head_dim"], 0, 0, 0
        for pos, start in _positions(case):
            if pos < 0:
                continue
            lo = _first_key(pos, start, case["window"])
            live += 1
            keys += pos + 1 - lo
            open_keys += pos - max(lo, pos // BLOCK * BLOCK)           # behind the new token, in bf16
        closing = case["spread"] == "closing"
        return {"bytes": 2 * hd * (keys - open_keys - live) + 4 * hd * open_keys + 2 * hd * (3 * live + case["b"]) + 4 * hd * live
                + (live * 2 * hd * BLOCK if closing else 0), "flops": 4 * hd * keys}
    size = 4 if case["dtype"] == "fp32" else 2
    n = case["rows"] * case["vocab"]
    return {"bytes": n * size * (2 if case["backward"] else 1) + case["rows"] * (16 + 12 * case["topk"]), "flops": n * (14 if case["backward"] else 6)}


# -- the definitions in 64 bits ---------------------------------------------------------------------------------------------
def _exact_score(st):
    case = st["case"]
    v, k = case["vocab"], case["topk"]
    outs = []
    for r in range(0, case["rows"], 512):
        z = st["logits"].detach()[r:r + 512, :v].double()
        t = st["tokens"][r:r + 512]
        lse = torch.logsumexp(z, 1)
        p = torch.softmax(z, 1)
        mean = (p * z).sum(1)
        ent = lse - mean
        some = t >= 0
        one = torch.zeros_like(z)
        one[torch.nonzero(some)[:, 0], t[some]] = 1.0
        row = [(one * z).sum(1) - lse * some, ent]
        best = torch.topk(z, k, 1) if k else None
        if k:
            row += [best.values - lse[:, None]]
        if case["backward"]:
            g, gh = (x[r:r + 512].double() for x in st["grads"][:2])
            # d lse / dz = p;  d (sum p z) / dz_v = p_v (1 + z_v - mean);  d z_t / dz = one
            d = one * g[:, None] + p * (gh - g * some)[:, None] - gh[:, None] * p * (1 + z - mean[:, None])
            if k:
                gt = st["grads"][2][r:r + 512].double()
                ids = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :k]
                pick = torch.zeros_like(z).scatter_(1, ids, gt)
                d = d + pick - p * gt.sum(1, keepdim=True)
            dz = z.new_zeros(z.shape[0], case["columns"])
            dz[:, :v] = d
            row.append(dz)
        outs.append(row)
    got = [torch.cat(x) for x in zip(*outs)]
    if k:
        got.insert(3, None)
    return got


def _exact_block(x):
    """``x [H, 64, D]`` in 64 bits as the values that its 8-bit form stands for, and the scale."""
    s = x.abs().flatten(1).amax(1) / 127.0
    return torch.round(x / s[:, None, None]).clamp(-127, 127) * s[:, None, None], s


def _exact_fill(st):
    k8, v8, ks, vs, kt, vt = (x.clone() for x in st["cache"])
    scales, tails, reads = [ks.double(), vs.double()], [kt.double(), vt.double()], []
    for which, (codes, new) in enumerate(((k8, st["k"]), (v8, st["v"]))):
        out = torch.zeros(k8.shape[0], st["length"], k8.shape[1], k8.shape[3], dtype=torch.float64, device=k8.device)
        for b, (p, n) in enumerate(zip(st["pos"].tolist(), st["lens"].tolist())):
            q = codes[b].double() if which == 0 else codes[b].double().transpose(-1, -2).reshape(k8.shape[1:])
            line = q * scales[which][b].repeat_interleave(BLOCK, 1)[..., None]                     # [H, T, D]
            first = p // BLOCK * BLOCK
            line[:, first:p] = tails[which][b, :, :p - first]
            line[:, p:p + n] = new[b, :n].double().transpose(0, 1)
            end = p + n
            if n:
                m = end // BLOCK * BLOCK
                tails[which][b, :, :end - m] = line[:, m:end]
                for f in range(first, m, BLOCK):
                    line[:, f:f + BLOCK], scales[which][b, :, f // BLOCK] = _exact_block(line[:, f:f + BLOCK])
            out[b, :end] = line[:, :end].transpose(0, 1)
        reads.append(out)
    return reads + scales + tails


def _exact_attend(st):
    case = st["case"]
    k8, v8, ks, vs, kt, vt = st["cache"]
    nseq, h, _, d = k8.shape
    half = d // 2
    ys, kts, vts, closed = [], kt.double(), vt.double(), ([], [])
    pos = st["pos"].tolist() * (nseq if st["pos"].numel() == 1 else 1)
    for b, p in enumerate(pos):
        y = torch.zeros(h, d, dtype=torch.float64, device=k8.device)
        if p >= 0:
            x = st["qkv"][b].double().view(3, h, d)
            c, s = st["cos"][p].double(), st["sin"][p].double()
            z = torch.complex(x[:2, :, :half], x[:2, :, half:]) * torch.complex(c, -s)              # a rotation by the negative angle
            z = torch.cat([z.real, z.imag], -1)
            z = z / torch.sqrt(z.square().mean(-1, keepdim=True) + EPS)
            kts[b, :, p % BLOCK], vts[b, :, p % BLOCK] = z[1].to(BF16).double(), x[2]
            m = p // BLOCK * BLOCK
            lo = _first_key(p, int(st["doc_start"][b]) if st["doc_start"] is not None else 0, st["window"])
            scores, parts = [], []
            a = lo // BLOCK * BLOCK
            if a < m:
                kk = k8[b, :, a:m].double() * ks[b, :, a // BLOCK:m // BLOCK].double().repeat_interleave(BLOCK, 1)[..., None]
                vv = (v8[b, :, a // BLOCK:m // BLOCK].double() * vs[b, :, a // BLOCK:m // BLOCK].double()[..., None, None]).transpose(-1, -2).reshape(h, m - a, d)
                scores.append(torch.einsum("hd,hnd->hn", z[0], kk)[:, lo - a:])
                parts.append(vv[:, lo - a:])
            f = max(lo - m, 0)
            scores.append(torch.einsum("hd,hnd->hn", z[0], kts[b, :, f:p - m + 1]))
            parts.append(vts[b, :, f:p - m + 1])
            w = torch.softmax(torch.cat(scores, 1) * st["scale"], 1)
            y = torch.einsum("hn,hnd->hd", w, torch.cat(parts, 1))
        if case["spread"] == "closing":
            blk = max(p, 0) // BLOCK
            if p >= 0:
                closed[0].append(_exact_block(kts[b])[0])
                closed[1].append(_exact_block(vts[b])[0].transpose(-1, -2))
            else:
                closed[0].append(k8[b].view(h, -1, BLOCK, d)[:, blk].double() * ks[b, :, blk].double()[:, None, None])
                closed[1].append(v8[b, :, blk].double() * vs[b, :, blk].double()[:, None, None])
        ys.append(y.reshape(-1))
    return [torch.stack(ys), kts, vts] + ([torch.stack(x) for x in closed] if closed[0] else [])


def exact(case, seed):
    st = prepare(case, seed)
    return {"fill": _exact_fill, "attend": _exact_attend, "score": _exact_score}[case["kind"]](st)
