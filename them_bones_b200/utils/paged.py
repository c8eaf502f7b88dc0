"""Decoding from a paged cache: prompts of any lengths in pieces, sampling, and drafted tokens that the model verifies.

A forward pass takes pieces of new tokens, packed one after another (``forward_pieces``): whole prompts, pieces of them, one token a
sequence, or a token and the drafts behind it.  Keys and values go to pages that all sequences share (``ops.paged_append``), the
pieces see them from there (``ops.paged_attention``), and one call decides what the next token of each sequence is, drawn or the most probable
one, and how many of its drafts stand (``ops.verify_drafts``).  The drafts come from a smaller model with a cache of its own, or from the text
itself (the tokens that followed the last occurrence of the newest ones); whichever it is, answers are distributed as without them.

When which pays: prompts of more than 512 tokens, which go by pieces here and token by token with the other caches, and batches of unequal lengths; for short prompts the other
caches' step is the shorter one (one sequence 0.55 for 1.6 ms at 20 layers of 1280).  A call captures its graphs anew, 10 to 20 ms.  Drafts pay where most of them stand and
the draft model is much the smaller; looking them up in the text is the host's work, in proportion to the texts: 2 / 13 / 25 ms a step for 64 texts of 200 / 1000 / 2000 tokens, so there it
costs more than it can save.

The reference scores teacher-forced full sequences only (round2/submission/inference.py:26-27).
"""
from __future__ import annotations

import contextlib

import torch

from .. import ops
from ..models.moe import MoeMLP

PIECE = 4096                  # tokens of a prompt that a pass takes of all sequences together
LOOKUP = 3                    # newest tokens that a lookup goes by at most


def check_model(model):
    """Raises for models that decode from other caches or from none."""
    if getattr(model, "os1", None) is not None or model.tables is not None or any(blk.attn is None for blk in model.transformer.h):
        raise ValueError("paged decoding has no form with an output table, hashed tables or attention-free blocks")
    if any(isinstance(blk.mlp, MoeMLP) and blk.mlp.ep_world > 1 for blk in model.transformer.h):
        raise ValueError("paged decoding keeps all experts on one rank")


class PagedCache:
    """One pool of pages a layer and one table for all layers.  ``lens``: tokens that each sequence may grow to."""

    def __init__(self, model, lens, page: int = 64):
        cfg = model.config
        w = model.lm_head.weight
        need = [max(1, -(-n // page)) for n in lens]
        self.layers = [ops.paged_cache(sum(need), cfg.n_head, cfg.head_dim, page, w.device, w.dtype) for _ in model.transformer.h]
        table, at = torch.full((len(need), max(need)), -1, dtype=torch.int32), 0
        for row, n in zip(table, need):
            row[:n] = torch.arange(at, at + n, dtype=torch.int32)
            at += n
        self.table = table.to(w.device)
        self.pos = torch.zeros(len(need), dtype=torch.int32, device=w.device)               # tokens held; -1: a sequence that is done
        self.doc_start = torch.zeros(len(need), dtype=torch.int32, device=w.device)         # of the last token held


def _starts(lens, device):
    out = torch.zeros(len(lens) + 1, dtype=torch.int32)
    out[1:] = torch.tensor(lens, dtype=torch.int32).cumsum(0)
    return out.to(device)


def _documents(cfg, ids, starts, cache):
    """Start of the document that each new token is in, from the last start tokens before or at it, and from what the sequence held."""
    row = torch.arange(ids.shape[0], device=ids.device)
    b = (torch.searchsorted(starts.long(), row, right=True) - 1).clamp(0, starts.shape[0] - 2)
    pos = cache.pos.long()[b] + row - starts.long()[b]
    far = 1 << 32                                            # above any position: a sequence's marks stay above all before it
    mark = torch.where(ids == cfg.bos_id, pos, cache.doc_start.long()[b])
    return (torch.cummax(b * far + mark, 0).values - b * far).to(torch.int32)


@torch.no_grad()
def forward_pieces(model, ids, cache: PagedCache, starts, longest: int):
    """New tokens ``ids [N]`` (rows ``starts[b] .. starts[b + 1]`` are sequence b's, behind the ``cache.pos[b]`` it holds) through the model; keys and values go
    to the cache, whose ``pos`` and ``doc_start`` the caller moves on.  -> ``(normed hidden rows [N, C], document starts [N] or None)``."""
    cfg = model.config
    doc = _documents(cfg, ids, starts, cache) if cfg.doc_mask else None
    x = ops.rms_norm(ops.embedding(ids, model.transformer.wte.weight, model.cos_dtype()))
    x0, skips = x, []
    n_layer, n_skip = cfg.n_layer, model.n_skip
    for i, blk in enumerate(model.transformer.h):
        if n_skip and i >= n_layer - n_skip:
            x = x + model.skip_lambda[i - (n_layer - n_skip)].to(x.dtype) * skips.pop()
        x, xn = ops.resid_mix_norm(x, x0, blk.resid_lambda, blk.x0_lambda)
        at = blk.attn
        qkv = ops.linear_qkv(xn, at.c_q.weight, at.c_k.weight, at.c_v.weight, precision=at.precision)
        if model.value_embeds is not None and str(i) in model.value_embeds:
            ve = ops.embedding(ids, model.value_embeds[str(i)].weight, x.dtype)
            a = ve.shape[1]
            qkv = torch.cat([qkv[:, :2 * a], qkv[:, 2 * a:] + blk.ve_lambda.to(qkv.dtype) * ve], 1)
        q = ops.paged_append(qkv, model.cos, model.sin, cache.layers[i], cache.table, starts, cache.pos)
        y = ops.paged_attention(q, cache.layers[i], cache.table, starts, cache.pos, at.scale, doc, at.window, longest)
        x, xn = ops.norm_split(ops.linear(y, at.c_proj.weight, residual=x, precision=at.precision))
        if isinstance(blk.mlp, MoeMLP):                      # a sequence of one token each: no token loses its expert to another
            x = blk.mlp(xn.unsqueeze(1), residual=x.unsqueeze(1)).squeeze(1)
        else:
            x = blk.mlp(xn, residual=x)
        if n_skip and i < n_skip:
            skips.append(x)
    return ops.rms_norm(x), doc


def _logits(model, x):
    return ops.lmhead_logits(x, model.lm_head.weight, model.config.vocab_size, model.config.softcap)


class _Step:
    """A pass over at most ``width`` tokens of each sequence, of fixed shapes: on a GPU the first call runs, the second is captured into a CUDA graph and all
    from then on are replayed.  It takes ``ids`` (packed by ``starts``) and ``uniforms``, and leaves ``logits`` and ``out`` (``ops.Verified``).  With drafts
    (``verify``) all rows count, ``draft`` their logits where a model drew them; else the token behind each sequence's last one is drawn.
    ``after``: what else belongs to the pass."""

    def __init__(self, model, cache: PagedCache, width: int, temperature: float, verify=False, draft=None, after=None):
        b, dev = cache.pos.shape[0], cache.pos.device
        self.model, self.cache, self.width, self.temperature, self.verify, self.draft, self.after = model, cache, width, temperature, verify, draft, after
        self.ids = torch.zeros(b * width, dtype=torch.int64, device=dev)
        self.starts = _starts([width] * b, dev)
        self.each = self.starts if verify else _starts([1] * b, dev)
        self.given = self.ids if verify else torch.zeros(b, dtype=torch.int64, device=dev)
        self.uniforms = torch.zeros(self.given.shape[0], 2, dtype=torch.float32, device=dev)
        self.graph, self.calls = None, 0

    def _pass(self):
        x, self.doc = forward_pieces(self.model, self.ids, self.cache, self.starts, self.width)
        if not self.verify and self.width > 1:
            x = x[(self.starts[1:].long() - 1).clamp(min=0)]
        self.logits = ops.lmhead_logits(x, self.model.lm_head.weight, self.model.config.vocab_size, self.model.config.softcap)
        self.out = ops.verify_drafts(self.logits, self.given, self.each, self.uniforms if self.temperature else None, self.draft, self.temperature)
        if self.after is not None:
            self.after(self)

    def __call__(self, gen):
        if self.temperature:
            torch.rand(self.uniforms.shape, generator=gen, out=self.uniforms)
        self.calls += 1
        if self.calls == 1 or not self.ids.is_cuda or ops.reference_path():
            return self._pass()
        if self.graph is None:
            torch.cuda.synchronize()
            self.graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side), torch.cuda.graph(self.graph, stream=side):
                self._pass()
            torch.cuda.current_stream().wait_stream(side)
        self.graph.replay()

    def advance(self, taken):
        """The cache holds ``taken [B]`` (int32, on the device) more tokens of each piece; a sequence that is done (-1) stays so."""
        c = self.cache
        if self.doc is not None:
            last = (self.starts[:-1] + taken - 1).long().clamp(min=0)
            c.doc_start.copy_(torch.where((taken > 0) & (c.pos >= 0), self.doc[last], c.doc_start))
        c.pos.add_(torch.where(c.pos >= 0, taken, torch.zeros_like(taken)))


def _prefill(model, cache: PagedCache, texts):
    """All but the last token of each text into the cache, at most ``PIECE`` tokens of all together a pass."""
    held, dev = [0] * len(texts), cache.pos.device
    while any(h < len(t) - 1 for h, t in zip(held, texts)):
        room, lens = PIECE, []
        for h, t in zip(held, texts):
            lens.append(min(room, len(t) - 1 - h))
            room -= lens[-1]
        ids = torch.tensor([x for h, n, t in zip(held, lens, texts) for x in t[h:h + n]], dtype=torch.int64, device=dev)
        starts = _starts(lens, dev)
        _, doc = forward_pieces(model, ids, cache, starts, max(lens))
        new = starts[1:] - starts[:-1]
        if doc is not None:
            cache.doc_start.copy_(torch.where(new > 0, doc[(starts[1:].long() - 1).clamp(min=0)], cache.doc_start))
        cache.pos.add_(new)
        held = [h + n for h, n in zip(held, lens)]


def lookup(text, k: int):
    """The ``k`` tokens at most that followed the last occurrence of the text's newest tokens (``LOOKUP`` of them, or as few as one) in the text before.  Goes through the
    text token by token: 0.4 ms for 2000 tokens in which the newest have not been before."""
    for n in range(min(LOOKUP, len(text) - 1), 0, -1):
        tail = text[-n:]
        for i in range(len(text) - n - 1, -1, -1):
            if text[i:i + n] == tail:
                return text[i + n:i + n + k]
    return []


class _ModelDrafts:
    """Drafts from a smaller model with a cache of its own: a pass over what it has not seen (the last draft, where all stood, and the token behind), then one
    over each draft but the last.  ``logits``: of each draft at the row in front of it, where the verification reads them."""

    def __init__(self, model, texts, lens, drafts: int, temperature: float):
        self.cache, self.k = PagedCache(model, lens), drafts
        _prefill(model, self.cache, texts)
        b, w = len(texts), model.lm_head.weight
        self.logits = torch.zeros(b * (drafts + 1), model.config.vocab_size, dtype=torch.float32, device=w.device)
        self.held = [len(t) - 1 for t in texts]
        self.docs = None                                       # [drafts, B]: start of the document behind each pass, of one draft more each
        self.first, self.next = _Step(model, self.cache, 2, temperature), _Step(model, self.cache, 1, temperature)

    def draw(self, texts, done, gen):
        """``[B, k]`` tokens behind the texts, of which the cache lacks one or two tokens each."""
        b, dev, step = len(texts), self.cache.pos.device, self.first
        lens = [0 if d else len(t) - h for t, h, d in zip(texts, self.held, done)]
        self.cache.pos.copy_(torch.tensor([-1 if d else h for h, d in zip(self.held, done)], dtype=torch.int32))
        step.starts.copy_(_starts(lens, dev))
        packed = [x for t, n in zip(texts, lens) for x in (t[len(t) - n:] if n else ())]
        step.ids.copy_(torch.tensor(packed + [0] * (2 * b - len(packed)), dtype=torch.int64))
        out, docs = [], []
        for i in range(self.k):
            step(gen)
            out.append(step.out.token.clamp(min=0))
            self.logits[i::self.k + 1].copy_(step.logits)
            step.advance(step.starts[1:] - step.starts[:-1])
            docs.append(self.cache.doc_start.clone())
            step = self.next
            step.ids.copy_(out[-1])
        self.held = [h if d else len(t) + self.k - 1 for h, t, d in zip(self.held, texts, done)]
        self.docs = torch.stack(docs)
        return torch.stack(out, 1)

    def forget(self, texts, accepted):
        """Of the drafts only ``accepted`` stand: what the cache holds of the others is written over by what comes there, and a document that began among
        them did not."""
        last = torch.tensor([min(a, self.k - 1) for a in accepted], device=self.docs.device)
        self.cache.doc_start.copy_(self.docs.gather(0, last[None])[0])
        self.held = [min(h, n + a) for h, n, a in zip(self.held, texts, accepted)]


@torch.no_grad()
def paged_decode(model, prompts, n_new: int, temperature: float = 0.0, drafts: int = 0, draft=None, seed: int = 0, page: int = 64):
    """``prompts`` (``[B, P]`` or a list of B rows of tokens of any lengths) and ``n_new`` tokens behind each, by arg-max (``temperature=0``) or drawn.
    ``drafts``: how many tokens are drafted and verified a step, by ``draft``, a smaller model of the same vocabulary, or without one
    looked up in the text; the answers are those of the model all the same: the same tokens at temperature 0 (but for the rounding of products of other
    shapes), the same distribution above.  ``seed``: of the random numbers.  -> ``[B, P + n_new]``, or a list of rows."""
    check_model(model)
    cfg, dev = model.config, model.lm_head.weight.device
    texts = [[int(x) for x in t] for t in (prompts.tolist() if isinstance(prompts, torch.Tensor) else prompts)]
    if not texts or not all(texts) or n_new < 0 or max(map(len, texts)) + n_new > cfg.sequence_len:
        raise ValueError("prompts of one token or more, which with the new tokens fit the model's sequence length")
    if any(not 0 <= x < cfg.vocab_size for t in texts for x in t):
        raise ValueError(f"prompts hold tokens outside the vocabulary of {cfg.vocab_size}")
    if not 0 <= drafts <= 64 or temperature < 0 or (draft is not None and not drafts):
        raise ValueError(f"{drafts} drafts (0 to 64; some, if there is a model for them), temperature {temperature}")
    if draft is not None:
        check_model(draft)
        if draft.config.vocab_size != cfg.vocab_size or draft.config.sequence_len < cfg.sequence_len or draft.lm_head.weight.device != dev:
            raise ValueError("a draft model has the model's vocabulary, its sequence length and its device")
    goal = [len(t) + n_new for t in texts]
    gen = torch.Generator(device=dev).manual_seed(seed)
    with torch.cuda.device(dev) if dev.type == "cuda" else contextlib.nullcontext():          # streams and graphs are the current device's
        if n_new:
            cache = PagedCache(model, goal, page)
            _prefill(model, cache, texts)
            if drafts:
                _drafted(model, cache, texts, goal, temperature, drafts, draft, gen)
            else:
                for t, new in zip(texts, _plain(model, cache, texts, n_new, temperature, gen)):
                    t.extend(new)
        if dev.type == "cuda" and not ops.reference_path():
            from ..ops import _lib as L
            L.check_error_word()
    rows = [torch.tensor(t, dtype=torch.int64, device=dev) for t in texts]
    return torch.stack(rows) if isinstance(prompts, torch.Tensor) else rows


def _plain(model, cache, texts, n_new, temperature, gen):
    """One token a step, nothing read by the host in between."""
    b, dev = len(texts), cache.pos.device
    new, one = torch.zeros(b, n_new, dtype=torch.int64, device=dev), torch.ones(b, dtype=torch.int32, device=dev)
    at = torch.zeros(1, dtype=torch.int64, device=dev)

    def after(step):
        new.index_copy_(1, at, step.out.token[:, None])
        at.add_(1)
        step.ids.copy_(step.out.token.clamp(min=0))
        step.advance(one)

    step = _Step(model, cache, 1, temperature, after=after)
    step.ids.copy_(torch.tensor([t[-1] for t in texts]))
    for _ in range(n_new):
        step(gen)
    return _numbers(new)


def _numbers(new):
    out = new.tolist()
    if min(min(row) for row in out) < 0:
        raise RuntimeError("the model's logits hold no number")
    return out


def _drafted(model, cache, texts, goal, temperature, k, draft, gen):
    """A token and ``k`` drafts a step; the texts grow by what stands and the token behind it."""
    b, dev = len(texts), cache.pos.device
    source = _ModelDrafts(draft, texts, goal, k, temperature) if draft is not None else None
    step = _Step(model, cache, k + 1, temperature, verify=True, draft=source.logits if source is not None and temperature else None)
    ids = step.ids.view(b, k + 1)
    while True:
        done = [len(t) >= n for t, n in zip(texts, goal)]
        if all(done):
            return
        ids[:, 0].copy_(torch.tensor([t[-1] for t in texts]))
        if source is not None:
            ids[:, 1:].copy_(source.draw(texts, done, gen))
        else:
            ids[:, 1:].copy_(torch.tensor([(x + [0] * k)[:k] for x in (lookup(t, k) for t in texts)]))
        cache.pos.masked_fill_(torch.tensor(done, device=dev), -1)
        step(gen)
        step.advance(step.out.accepted + 1)
        accepted, token, tried = step.out.accepted.tolist(), step.out.token.tolist(), ids[:, 1:].tolist()
        before = [len(t) for t in texts]
        for i, t in enumerate(texts):
            if done[i]:
                continue
            if token[i] < 0:
                raise RuntimeError("the model's logits hold no number")
            t.extend((tried[i][:accepted[i]] + [token[i]])[:goal[i] - len(t)])
        if source is not None:
            source.forget(before, accepted)
