"""Log-probabilities of given tokens, entropy and the most probable alternatives of rows of logits: checks and the native body
(``csrc/logprobs.cu``), an autograd ``Function`` whose gradient reaches the logits through all three."""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import _lib as L
from . import COUNTS
from ..ref import functional as RF

TOP_MAX = 32


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor         # fp32 [..]: of the given token; 0 where there is none
    entropy: torch.Tensor         # fp32 [..], nats
    top_logprob: torch.Tensor     # fp32 [.., topk], descending
    top_id: torch.Tensor          # int64 [.., topk]


def check(logits, tokens, topk, vocab):
    if logits.dim() < 1 or not logits.is_floating_point():
        raise ValueError(f"token_logprobs: logits {logits.dtype} {tuple(logits.shape)}")
    if tokens.shape != logits.shape[:-1] or tokens.dtype not in (torch.int64, torch.int32) or tokens.device != logits.device:
        raise ValueError(f"token_logprobs: tokens {tokens.dtype} {tuple(tokens.shape)} on {tokens.device}, expected int64 or int32 {tuple(logits.shape[:-1])} on {logits.device}")
    if not 1 <= vocab <= logits.shape[-1]:
        raise ValueError(f"token_logprobs: a vocabulary of {vocab} in {logits.shape[-1]} columns")
    if not 0 <= topk <= min(TOP_MAX, vocab):
        raise ValueError(f"token_logprobs: topk {topk}, at most {min(TOP_MAX, vocab)}")


def check_head(x, w, tokens, topk, vocab, cap):
    if x.dim() < 1 or w.dim() != 2 or x.shape[-1] != w.shape[1] or not x.is_floating_point() or w.device != x.device:
        raise ValueError(f"lmhead_logprobs: rows {tuple(x.shape)} on {x.device}, head {tuple(w.shape)} on {w.device}")
    if tokens.shape != x.shape[:-1] or tokens.dtype not in (torch.int64, torch.int32) or tokens.device != x.device:
        raise ValueError(f"lmhead_logprobs: tokens {tokens.dtype} {tuple(tokens.shape)} on {tokens.device}, expected int64 or int32 {tuple(x.shape[:-1])} on {x.device}")
    if not 1 <= vocab <= w.shape[0] or not 0 <= topk <= min(TOP_MAX, vocab):
        raise ValueError(f"lmhead_logprobs: a vocabulary of {vocab} in {w.shape[0]} rows, topk {topk} (at most {TOP_MAX})")
    if not 0 < cap < float("inf"):
        raise ValueError(f"lmhead_logprobs: a soft-cap of {cap}")


def statement(logits, tokens, topk, vocab) -> TokenLogprobs:
    shp = logits.shape[:-1]
    g, h, t, i = RF.token_logprobs(logits.reshape(-1, logits.shape[-1]), tokens.reshape(-1).to(torch.int64), topk, vocab)
    return TokenLogprobs(g.view(shp), h.view(shp), t.view(*shp, topk), i.view(*shp, topk))


def _forward(z, tokens, topk, vocab, want_stats):
    rows = z.shape[0]
    given = torch.empty(rows, dtype=torch.float32, device=z.device)
    entropy, top, ids = given.new_empty(rows), given.new_empty((rows, topk)), tokens.new_empty((rows, topk))
    stats = given.new_empty((rows, 4)) if want_stats else None
    with L.device(z.get_device()):
        L.call("bones_logprobs_fwd", z.data_ptr(), z.stride(0), int(z.dtype is torch.float32), rows, vocab, tokens.data_ptr(), topk, given.data_ptr(),
               entropy.data_ptr(), top.data_ptr(), ids.data_ptr(), stats.data_ptr() if want_stats else 0, L.raw_stream())
    COUNTS["token_logprobs"] += 1
    return given, entropy, top, ids, stats


def has_tangent(*xs) -> bool:
    """Whether one of the tensors (or None) carries a tangent of forward-mode differentiation; kernels that go by address would drop it."""
    return forward_ad._current_level >= 0 and any(x is not None and forward_ad.unpack_dual(x).tangent is not None for x in xs)


def _as_kernel(gs):
    """Gradients as the kernel reads them, fp32 and contiguous, and their addresses (0: none); None where one has no address (a batched
    gradient) or a tangent, or a graph is being recorded: then the statement's own operators."""
    if torch.is_grad_enabled() or has_tangent(*gs):
        return None
    try:
        gs = [g if g is None or (g.dtype is torch.float32 and g.is_contiguous()) else g.float().contiguous() for g in gs]
        return gs, [0 if g is None else g.data_ptr() for g in gs]
    except RuntimeError:
        return None


def _backward(z, tokens, ids, stats, vocab, at, dz, cap):
    L.call("bones_logprobs_bwd", z.data_ptr(), z.stride(0), int(z.dtype is torch.float32), z.shape[0], vocab, z.shape[1], tokens.data_ptr(), ids.shape[1],
           ids.data_ptr(), stats.data_ptr(), at[0], at[1], at[2], dz.data_ptr(), dz.stride(0), cap, L.raw_stream())


class _LogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, tokens, topk, vocab):
        given, entropy, top, ids, stats = _forward(z, tokens, topk, vocab, True)
        ctx.save_for_backward(z, tokens, ids, stats)
        ctx.vocab = vocab
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(ids)
        return given, entropy, top, ids

    @staticmethod
    def backward(ctx, g_given, g_entropy, g_top, _g_ids):
        z, tokens, ids, stats = ctx.saved_tensors
        gs = [g_given, g_entropy, g_top if ids.shape[1] else None]
        if g_given is None and g_entropy is None and gs[2] is None:
            return None, None, None, None
        ready = _as_kernel(gs)
        if ready is None:
            return _statement_grad(*_settled(z, ctx.vocab), tokens, ids, ctx.vocab, *gs), None, None, None
        dz = torch.empty(z.shape, dtype=z.dtype, device=z.device)
        with L.device(z.get_device()):
            _backward(z, tokens, ids, stats, ctx.vocab, ready[1], dz, 0.0)
        return dz, None, None, None


def _settled(z, vocab):
    """``z`` with zeros for its rows without a number, and which ones they are."""
    bad = RF.rows_without_number(z[:, :vocab].float())
    return torch.where(bad[:, None], torch.zeros_like(z), z), bad


def _statement_grad(z, bad, tokens, ids, vocab, g_given, g_entropy, g_top):
    """The gradient in PyTorch operators (differentiable, batchable); ``z`` is the saved input itself, but for ``_settled``: a row without a
    number has NaN for its gradient where something depends on it, and 0 where nothing does, not NaN times 0."""
    logp = torch.log_softmax(z[:, :vocab].float(), -1)
    gone = logp == float("-inf")
    p, logp0 = logp.exp(), logp.masked_fill(gone, 0.0)
    some = (tokens >= 0) & (tokens < vocab)
    d, used = torch.zeros_like(p), torch.zeros_like(bad)
    if g_given is not None:
        g = torch.where(some, g_given, torch.zeros_like(g_given))
        used = used | (g != 0)
        one = torch.zeros_like(p).scatter(1, torch.where(some, tokens, torch.zeros_like(tokens))[:, None], 1.0)
        d = d + g[:, None] * (one - p)
    if g_entropy is not None:
        used = used | (g_entropy != 0)
        entropy = -(p * logp0).sum(-1)
        d = d - g_entropy[:, None] * p * (logp0 + entropy[:, None])
    if g_top is not None:
        used = used | (g_top != 0).any(-1)
        d = d - p * g_top.sum(-1, keepdim=True)
        for j in range(ids.shape[1]):
            d = d + g_top[:, j:j + 1] * torch.zeros_like(p).scatter(1, ids[:, j:j + 1], 1.0)
    d = torch.where((bad & used)[:, None], torch.full_like(p, float("nan")), d)
    return torch.nn.functional.pad(d, (0, z.shape[1] - vocab)).to(z.dtype)


def native(logits, tokens, topk, vocab) -> TokenLogprobs:
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"native token_logprobs does not cover this call: dtype {logits.dtype} (bf16 and fp32)")
    rows = logits.dim() == 2
    z = logits if rows else logits.reshape(-1, logits.shape[-1])
    if z.stride(1) != 1:
        z = z.contiguous()
    tk = tokens if rows and tokens.dtype is torch.int64 and tokens.is_contiguous() else tokens.reshape(-1).to(torch.int64).contiguous()
    # a tangent goes to the function too, which has no forward mode and says so
    recorded = (torch.is_grad_enabled() and logits.requires_grad) or has_tangent(logits)
    r = _LogprobsFn.apply(z, tk, topk, vocab) if recorded else _forward(z, tk, topk, vocab, False)[:4]
    if rows:
        return TokenLogprobs(*r)
    shp = logits.shape[:-1]
    return TokenLogprobs(r[0].view(shp), r[1].view(shp), r[2].view(*shp, topk), r[3].view(*shp, topk))


# -- from the last hidden rows ---------------------------------------------------------------------------------------
def head_statement(x, w, tokens, topk, vocab, cap) -> TokenLogprobs:
    z = RF.softcap_logits(torch.nn.functional.linear(x, w.to(x.dtype))[..., :vocab], cap)
    return statement(z, tokens, topk, vocab)


class _HeadLogprobsFn(torch.autograd.Function):
    """The head in blocks of rows: the logits of a block are made, looked at and dropped, and made again for their gradient, so that only
    one ``[rows, V]`` block exists at a time.  A head that owns its gradient (``main_grad``) gets it by accumulation."""

    @staticmethod
    def forward(ctx, x, w, tokens, topk, vocab, cap, want_grad):
        from . import cuda as C
        m, dev = x.shape[0], x.device
        given, entropy = torch.empty(m, dtype=torch.float32, device=dev), torch.empty(m, dtype=torch.float32, device=dev)
        top, ids = torch.empty((m, topk), dtype=torch.float32, device=dev), torch.empty((m, topk), dtype=torch.int64, device=dev)
        stats = torch.empty((m, 4), dtype=torch.float32, device=dev)
        buf = torch.empty(min(C.LOSS_ROWS, m), w.shape[0], dtype=torch.bfloat16, device=dev)
        for a in range(0, m, C.LOSS_ROWS):
            n = min(C.LOSS_ROWS, m - a)
            _capped(x[a:a + n], w, cap, buf[:n])
            L.call("bones_logprobs_fwd", buf.data_ptr(), buf.stride(0), 0, n, vocab, tokens[a:a + n].data_ptr(), topk, given[a:a + n].data_ptr(),
                   entropy[a:a + n].data_ptr(), top[a:a + n].data_ptr(), ids[a:a + n].data_ptr(), stats[a:a + n].data_ptr(), L.raw_stream())
        COUNTS["lmhead_logprobs"] += 1
        if want_grad:
            ctx.save_for_backward(x, w, tokens, ids, stats)
            ctx.vocab, ctx.cap, ctx.main_grad = vocab, cap, getattr(w, "main_grad", None)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(ids)
        return given, entropy, top, ids

    @staticmethod
    def backward(ctx, g_given, g_entropy, g_top, _g_ids):
        from . import cuda as C
        x, w, tokens, ids, stats = ctx.saved_tensors
        gs = [g_given, g_entropy, g_top if ids.shape[1] else None]
        none = (None,) * 5
        if all(g is None for g in gs):
            return None, None, *none
        ready, m = _as_kernel(gs), x.shape[0]
        if ready is None:
            z, bad = _settled(RF.softcap_logits(torch.nn.functional.linear(x.float(), w.float()), ctx.cap), ctx.vocab)
            d = _statement_grad(z, bad, tokens, ids, ctx.vocab, *gs) * (1 - (z / ctx.cap).square())
            return (d @ w.float()).to(x.dtype), (d.transpose(-1, -2) @ x.float()).to(w.dtype), *none
        gs = ready[0]
        need_x, need_w = ctx.needs_input_grad[:2]
        dx = torch.zeros(x.shape, dtype=torch.float32, device=x.device) if need_x else None
        dw = ctx.main_grad if ctx.main_grad is not None or not need_w else torch.zeros(w.shape, dtype=torch.float32, device=w.device)
        buf = torch.empty(min(C.LOSS_ROWS, m), w.shape[0], dtype=torch.bfloat16, device=x.device)
        with L.device(x.get_device()):
            for a in range(0, m, C.LOSS_ROWS):
                n = min(C.LOSS_ROWS, m - a)
                z = buf[:n]
                _capped(x[a:a + n], w, ctx.cap, z)
                _backward(z, tokens[a:a + n], ids[a:a + n], stats[a:a + n], ctx.vocab, [0 if g is None else g[a:a + n].data_ptr() for g in gs], z, ctx.cap)
                if need_x:
                    C.mm_nn_acc(z, w, dx[a:a + n])
                if need_w:
                    C.mm_tn_acc(z, x[a:a + n], dw)
        return dx.to(x.dtype) if need_x else None, dw.to(w.dtype) if need_w and ctx.main_grad is None else None, *none


def _capped(x, w, cap, out):
    from . import cuda as C
    C.mm_nt(x, w, out=out, epi=L.EPI_SOFTCAP, alpha=1.0 / cap, beta=cap)


def head_native(x, w, tokens, topk, vocab, cap) -> TokenLogprobs:
    from .cuda import _c
    if x.dtype != torch.bfloat16 or w.dtype != torch.bfloat16 or x.shape[-1] % 8 or w.shape[0] % 8:
        raise ValueError(f"native lmhead_logprobs does not cover this call: {x.dtype} {tuple(x.shape)}, head {w.dtype} {tuple(w.shape)} "
                         "(bf16, rows of whole 16 bytes)")
    shp, x2, tk = x.shape[:-1], _c(x).view(-1, x.shape[-1]), tokens.reshape(-1).to(torch.int64).contiguous()
    x2 = x2 if x2.data_ptr() % 16 == 0 else x2.clone()
    if w.stride(1) != 1 or w.stride(0) % 8 or w.data_ptr() % 16:
        own, w = getattr(w, "main_grad", None), w.clone(memory_format=torch.contiguous_format)
        if own is not None:
            w.main_grad = own
    with L.device(x.get_device()):
        r = _HeadLogprobsFn.apply(x2, w, tk, topk, vocab, float(cap), torch.is_grad_enabled() and (x.requires_grad or w.requires_grad))
    return TokenLogprobs(r[0].view(shp), r[1].view(shp), r[2].view(*shp, topk), r[3].view(*shp, topk))
