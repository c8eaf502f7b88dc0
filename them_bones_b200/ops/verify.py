"""Verification of drafted tokens: the checks of its call and the native body (``csrc/verify.cu``)."""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib as L
from . import COUNTS
from .logprobs import has_tangent

COLDEST, WARMEST = 1e-6, 1e6  # temperatures but 0


class Verified(NamedTuple):
    accepted: torch.Tensor        # int32 [B]: how many of the sequence's drafts stand
    token: torch.Tensor           # int64 [B]: the token behind them; -1 where there is none


def check(logits, ids, starts, uniforms, draft, temperature, vocab):
    if logits.dim() != 2 or not logits.is_floating_point() or logits.shape[0] >= 1 << 26:
        raise ValueError(f"verify_drafts: logits {logits.dtype} {tuple(logits.shape)}, expected [N, C] of fewer than 2^26 rows")
    n, dev = logits.shape[0], logits.device
    if ids.shape != (n,) or ids.dtype is not torch.int64 or ids.device != dev or not ids.is_contiguous():
        raise ValueError(f"verify_drafts: ids {ids.dtype} {tuple(ids.shape)} on {ids.device}, expected contiguous int64 [{n}] on {dev}")
    if starts.dim() != 1 or not 2 <= starts.shape[0] <= 65536 or starts.dtype is not torch.int32 or starts.device != dev or not starts.is_contiguous():
        raise ValueError(f"verify_drafts: starts {starts.dtype} {tuple(starts.shape)} on {starts.device}, expected contiguous int32 [B + 1] on {dev}, B from 1 to 65535")
    if not 1 <= vocab <= logits.shape[1] or vocab > 1 << 30:
        raise ValueError(f"verify_drafts: a vocabulary of {vocab} in {logits.shape[1]} columns")
    if temperature != 0 and not COLDEST <= temperature <= WARMEST:
        raise ValueError(f"verify_drafts: temperature {temperature} (0, or {COLDEST} to {WARMEST})")
    if temperature != 0 and (uniforms is None or uniforms.shape != (n, 2) or uniforms.dtype is not torch.float32 or uniforms.device != dev or not uniforms.is_contiguous()):
        have = None if uniforms is None else f"{uniforms.dtype} {tuple(uniforms.shape)} on {uniforms.device}"
        raise ValueError(f"verify_drafts: uniforms {have}, expected contiguous fp32 [{n}, 2] on {dev}")
    if draft is not None and (draft.dim() != 2 or draft.shape[0] != n or draft.shape[1] < vocab or draft.dtype is not logits.dtype or draft.device != dev):
        raise ValueError(f"verify_drafts: draft logits {draft.dtype} {tuple(draft.shape)} on {draft.device}, expected {logits.dtype} [{n}, {vocab} or more] on {dev}")
    if torch.is_grad_enabled() and (logits.requires_grad or (draft is not None and draft.requires_grad)):
        raise ValueError("verify_drafts: it has no gradient; call it under torch.no_grad()")
    if has_tangent(logits, draft):
        raise ValueError("verify_drafts: it has no forward-mode differentiation")


def _rows(x):
    """``x [N, C]`` with consecutive values in a row."""
    return x if x.stride(1) == 1 and (x.shape[0] <= 1 or x.stride(0) >= x.shape[1]) else x.contiguous()


def short(logits, ids, starts, uniforms, draft, temperature, vocab):
    """The call by the short way (``csrc/calls.cpp``), or None where its tensors are not as the kernels want them."""
    out = L.calls().verify_drafts(logits, ids, starts, uniforms, draft, temperature, vocab, COLDEST, WARMEST)
    if out is None:
        return None
    L.LAUNCHES[0] += 2
    COUNTS["verify_drafts"] += 1
    return Verified(*out)


def native(logits, ids, starts, uniforms, draft, temperature, vocab) -> Verified:
    if logits.dtype is not torch.bfloat16 and logits.dtype is not torch.float32:
        raise ValueError(f"native verify_drafts does not cover this call: logits of {logits.dtype} (bf16 and fp32)")
    n, b, dev = logits.shape[0], starts.shape[0] - 1, logits.get_device()
    accepted, token = torch.empty(b, dtype=torch.int32, device=logits.device), torch.empty(b, dtype=torch.int64, device=logits.device)
    z, q = _rows(logits), None if draft is None or temperature == 0 else _rows(draft)
    stats = torch.empty((max(n, 1), 2, 2), dtype=torch.float64, device=logits.device)           # of each row: target's and draft's
    with L.device(dev):
        L.call("bones_verify", z.data_ptr(), z.stride(0), 0 if q is None else q.data_ptr(), 0 if q is None else q.stride(0), int(z.dtype is torch.float32), ids.data_ptr(),
               starts.data_ptr(), 0 if uniforms is None else uniforms.data_ptr(), b, n, vocab, temperature, stats.data_ptr(), accepted.data_ptr(), token.data_ptr(),
               L.raw_stream(), launches=2)
    COUNTS["verify_drafts"] += 1
    return Verified(accepted, token)
