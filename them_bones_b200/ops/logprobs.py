"""Log-probabilities of given tokens, entropy and the most probable alternatives of rows of logits: checks and the native body
(``csrc/logprobs.cu``), an autograd ``Function`` whose gradient reaches the logits through all three."""
from __future__ import annotations

from typing import NamedTuple

import torch

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


def statement(logits, tokens, topk, vocab) -> TokenLogprobs:
    shp = logits.shape[:-1]
    g, h, t, i = RF.token_logprobs(logits.reshape(-1, logits.shape[-1]), tokens.reshape(-1).to(torch.int64), topk, vocab)
    return TokenLogprobs(g.view(shp), h.view(shp), t.view(*shp, topk), i.view(*shp, topk))


def _forward(z, tokens, topk, vocab, want_stats):
    rows, dev = z.shape[0], z.device
    given, entropy = torch.empty(rows, dtype=torch.float32, device=dev), torch.empty(rows, dtype=torch.float32, device=dev)
    top, ids = torch.empty((rows, topk), dtype=torch.float32, device=dev), torch.empty((rows, topk), dtype=torch.int64, device=dev)
    stats = torch.empty((rows, 4), dtype=torch.float32, device=dev) if want_stats else None
    with L.device(z.get_device()):
        L.call("bones_logprobs_fwd", z.data_ptr(), z.stride(0), int(z.dtype is torch.float32), rows, vocab, tokens.data_ptr(), topk, given.data_ptr(),
               entropy.data_ptr(), top.data_ptr(), ids.data_ptr(), stats.data_ptr() if want_stats else 0, L.raw_stream())
    COUNTS["token_logprobs"] += 1
    return given, entropy, top, ids, stats


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
        from .cuda import _by_address
        z, tokens, ids, stats = ctx.saved_tensors
        k = ids.shape[1]
        gs = [g_given, g_entropy, g_top if k else None]
        if all(g is None for g in gs):
            return None, None, None, None
        if not all(_by_address(g) for g in gs + [z] if g is not None):
            # batched gradients, or a graph recorded through this one: the statement's own operators
            return _statement_grad(z, tokens, ids, ctx.vocab, *gs), None, None, None
        gs = [g.float().contiguous() if g is not None else None for g in gs]
        g0, g1, g2 = (0 if g is None else g.data_ptr() for g in gs)
        dz = torch.empty(z.shape, dtype=z.dtype, device=z.device)
        with L.device(z.get_device()):
            L.call("bones_logprobs_bwd", z.data_ptr(), z.stride(0), int(z.dtype == torch.float32), z.shape[0], ctx.vocab, z.shape[1], tokens.data_ptr(), k,
                   ids.data_ptr(), stats.data_ptr(), g0, g1, g2, dz.data_ptr(), z.shape[1], L.raw_stream())
        return dz, None, None, None


def _statement_grad(z, tokens, ids, vocab, g_given, g_entropy, g_top):
    """The gradient in PyTorch operators (differentiable, batchable); ``z`` is the saved input itself."""
    logp = torch.log_softmax(z[:, :vocab].float(), -1)
    gone = logp == float("-inf")
    p, logp0 = logp.exp(), logp.masked_fill(gone, 0.0)
    some = (tokens >= 0) & (tokens < vocab)
    d = torch.zeros_like(p)
    if g_given is not None:
        g = (g_given * some)[:, None]
        one = torch.zeros_like(p).scatter(1, torch.where(some, tokens, torch.zeros_like(tokens))[:, None], 1.0)
        d = d + g * (one - p)
    if g_entropy is not None:
        entropy = -(p * logp0).sum(-1)
        d = d - g_entropy[:, None] * p * (logp0 + entropy[:, None])
    if g_top is not None:
        d = d - p * g_top.sum(-1, keepdim=True)
        for j in range(ids.shape[1]):
            d = d + g_top[:, j:j + 1] * torch.zeros_like(p).scatter(1, ids[:, j:j + 1], 1.0)
    return torch.nn.functional.pad(d, (0, z.shape[1] - vocab)).to(z.dtype)


def native(logits, tokens, topk, vocab) -> TokenLogprobs:
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"native token_logprobs does not cover this call: dtype {logits.dtype} (bf16 and fp32)")
    rows = logits.dim() == 2
    z = logits if rows else logits.reshape(-1, logits.shape[-1])
    if z.stride(1) != 1:
        z = z.contiguous()
    tk = tokens if rows and tokens.dtype is torch.int64 and tokens.is_contiguous() else tokens.reshape(-1).to(torch.int64).contiguous()
    r = _LogprobsFn.apply(z, tk, topk, vocab) if torch.is_grad_enabled() and logits.requires_grad else _forward(z, tk, topk, vocab, False)[:4]
    if rows:
        return TokenLogprobs(*r)
    shp = logits.shape[:-1]
    return TokenLogprobs(r[0].view(shp), r[1].view(shp), r[2].view(*shp, topk), r[3].view(*shp, topk))
