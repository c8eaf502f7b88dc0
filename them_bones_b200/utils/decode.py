"""Greedy decoding with a KV cache.

The reference scores teacher-forced full sequences only (round2/submission/inference.py:26-27); autoregressive decoding
is an added capability.  The cache stores, per layer, keys *after* RoPE and QK-norm and raw values, so a decode step
rotates only the new token (RoPE at its absolute position) and attends over the cached prefix restricted to the current
document and the layer's window.  It holds them in bf16 or, with close to half the memory and half the bytes of a step in long
caches, in 8 bits (``kv="int8"``: ``ops.kv8_cache``).  A decoder can also say what each of its answers was worth
(``logprobs=k``: ``ops.token_logprobs`` of every generated token).

When 8 bits pay: the tokens of the open block are held in bf16 beside the codes, so a cache of 64 tokens takes 1.5 times the bf16 one's
memory, one of 128 as much, one of 2048 0.53 of it.  ``NativeDecoder``'s step reads the codes themselves and is the faster one from a few hundred
tokens on (at 64 tokens it costs 0.5 to 2 us a layer).  The plain route (``_forward_cached``: prompts of more than 512 tokens, models whose heads
are not of 128, models on the CPU) turns the codes into fp32 numbers at every call: there only the memory is saved.
"""
from __future__ import annotations

import ctypes

import torch
import torch.nn.functional as F

from .. import ops
from ..models.moe import MoeMLP
from ..ref import functional as RF

_I = ctypes.c_int


def L_check():
    from ..ops import _lib as L
    L.check_error_word()


KV_TYPES = ("bf16", "int8")


class KVCache:
    """``kv="bf16"``: keys and values ``[layers, B, T, H, D]`` in the model's type; ``"int8"``: a ``KV8`` for each layer in ``kv8``."""

    def __init__(self, model, batch: int, max_len: int, kv: str = "bf16"):
        cfg = model.config
        dev, dt = model.lm_head.weight.device, model.lm_head.weight.dtype
        if kv not in KV_TYPES:
            raise ValueError(f"key/value cache {kv!r} (one of {KV_TYPES})")
        self.max_len, self.k, self.v, self.kv8 = max_len, None, None, None
        if kv == "int8":
            self.kv8 = [ops.kv8_cache(batch, max_len, cfg.n_head, cfg.head_dim, dev) for _ in range(cfg.n_layer)]
        else:
            shape = (cfg.n_layer, batch, max_len, cfg.n_head, cfg.head_dim)
            self.k = torch.zeros(shape, dtype=dt, device=dev)
            self.v = torch.zeros(shape, dtype=dt, device=dev)
        self.doc_start = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.len = 0
        self.tokens = None          # token history [batch, max_len], kept when the model has hashed tables


def _attend(q, k, v, scale, lo):
    """q ``[B,H,1,D]``, k/v ``[B,L,H,D]``; keys at positions < ``lo[b]`` are masked."""
    b, l = k.shape[0], k.shape[1]
    s = torch.einsum("bhqd,blhd->bhql", q.float(), k.float()) * scale
    pos = torch.arange(l, device=k.device)[None, None, None, :]
    s = s.masked_fill(pos < lo[:, None, None, None], float("-inf"))
    return torch.einsum("bhql,blhd->bqhd", torch.softmax(s, -1), v.float())


@torch.no_grad()
def _forward_cached(model, idx, cache: KVCache):
    """Run ``idx [B, t]`` (the whole prompt at prefill, one token afterwards), appending to the cache.  Returns the
    logits of the last position ``[B, V]``."""
    cfg = model.config
    b, t = idx.shape
    p0 = cache.len
    dev = idx.device
    pos = torch.arange(p0, p0 + t, device=dev)
    # document starts: most recent BOS at or before each new position
    if cfg.doc_mask:
        marks = torch.where(idx == cfg.bos_id, pos[None, :].expand(b, t).to(torch.int32),
                            torch.zeros(b, t, dtype=torch.int32, device=dev))
        ds = torch.maximum(torch.cummax(marks, 1).values, cache.doc_start[:, None])
        cache.doc_start = ds[:, -1].clone()
    else:
        ds = torch.zeros(b, t, dtype=torch.int32, device=dev)
    cos, sin = model.cos[p0:p0 + t], model.sin[p0:p0 + t]
    x = F.embedding(idx, model.transformer.wte.weight)
    if model.tables is not None:
        # rows keyed by the last `order` tokens: the cache keeps the token history for contexts that start before this call
        if cache.tokens is None:
            cache.tokens = torch.zeros(b, cache.max_len, dtype=torch.int64, device=dev)
        cache.tokens[:, p0:p0 + t] = idx
        hist, tb = cache.tokens[:, :p0 + t], model.tables
        ids = torch.stack([RF.ngram_rows(hist, o, tb.rows, tb.seed + j, _doc_start_full(hist, cfg) if cfg.doc_mask else None)[:, p0:]
                           for j, o in enumerate(tb.orders)])
        x = tb.add_lookup(x, idx, None, model.table_lambda, rows=ids)
    x = RF.rms_norm(x)
    x0 = x
    skips = []
    n_layer, n_skip = cfg.n_layer, model.n_skip
    for i, blk in enumerate(model.transformer.h):
        if n_skip and i >= n_layer - n_skip:
            x = x + model.skip_lambda[i - (n_layer - n_skip)].to(x.dtype) * skips.pop()
        x = RF.resid_mix(x, x0, blk.resid_lambda, blk.x0_lambda)
        xn = RF.rms_norm(x)
        at = blk.attn
        q = F.linear(xn, at.c_q.weight).view(b, t, at.n_head, at.head_dim)
        k = F.linear(xn, at.c_k.weight).view(b, t, at.n_head, at.head_dim)
        v = F.linear(xn, at.c_v.weight).view(b, t, at.n_head, at.head_dim)
        if model.value_embeds is not None and str(i) in model.value_embeds:
            ve = F.embedding(idx, model.value_embeds[str(i)].weight).view(b, t, at.n_head, at.head_dim)
            v = v + blk.ve_lambda.to(v.dtype) * ve.to(v.dtype)
        q = RF.rms_norm(_rope_at(q, cos, sin))
        k = RF.rms_norm(_rope_at(k, cos, sin))
        if cache.kv8 is not None:
            # a token sees the block it is in as it came and the ones before it from their codes, as it does token by token
            c8, b0 = cache.kv8[i], p0 // RF.KV8_BLOCK * RF.KV8_BLOCK
            new = [x.to(c8.k_open.dtype) for x in (k, v)]
            exact = [torch.cat([old[:, :, :p0 - b0], x.transpose(1, 2)], 2) for old, x in zip((c8.k_open, c8.v_open), new)]       # from b0 on
            ops.kv8_append(c8, *new, p0)
            lines = RF.kv8_coded(c8, b0 // RF.KV8_BLOCK, p0 + t - b0)
            held = [x.transpose(1, 2) for x in lines]
        else:
            cache.k[i, :, p0:p0 + t] = k
            cache.v[i, :, p0:p0 + t] = v
            held = cache.k[i], cache.v[i]
        ys = []
        for j in range(t):                                   # prefill is short in decode benchmarks; one row at a time
            cur = p0 + j
            lo = ds[:, j].to(torch.int64)
            if at.window:
                lo = torch.maximum(lo, torch.full_like(lo, max(0, (cur // 128 - (at.window // 128 - 1)) * 128)))
            if cache.kv8 is not None and (j == 0 or cur % RF.KV8_BLOCK == 0):       # a block's tokens as they came, the one before it from its codes
                first = cur // RF.KV8_BLOCK * RF.KV8_BLOCK
                for line, own in zip(lines, exact):
                    line[:, :, first:first + RF.KV8_BLOCK] = own[:, :, first - b0:first - b0 + RF.KV8_BLOCK]
                if j and first:
                    n8, full = first // RF.KV8_BLOCK - 1, slice(first - RF.KV8_BLOCK, first)
                    lines[0][:, :, full] = RF.kv8_values(c8.k[:, :, full], c8.k_scale[:, :, n8])
                    lines[1][:, :, full] = RF.kv8_values(c8.v[:, :, n8].transpose(-1, -2), c8.v_scale[:, :, n8])
            ys.append(_attend(q[:, j:j + 1].transpose(1, 2), *(x[:, :cur + 1] for x in held), at.scale, lo))
        y = torch.cat(ys, 1).reshape(b, t, -1).to(x.dtype)
        x = x + F.linear(y, at.c_proj.weight)
        xn = RF.rms_norm(x)
        if isinstance(blk.mlp, MoeMLP):
            x = blk.mlp(xn, residual=x)
        else:
            x = x + RF.mlp(xn, blk.mlp.c_fc.weight, blk.mlp.c_proj.weight)
        if n_skip and i < n_skip:
            skips.append(x)
    cache.len = p0 + t
    x = RF.rms_norm(x[:, -1])
    return RF.softcap_logits(F.linear(x, model.lm_head.weight)[..., :cfg.vocab_size], cfg.softcap)


def _doc_start_full(hist, cfg):
    return RF.doc_start_positions(hist, cfg.bos_id)


def _rope_at(x, cos, sin):
    d = x.shape[-1] // 2
    x1, x2 = x[..., :d].float(), x[..., d:].float()
    c, s = cos[None, :, None, :].float(), sin[None, :, None, :].float()
    return torch.cat([x1 * c + x2 * s, -x1 * s + x2 * c], -1).to(x.dtype)


def _token_rows(out, b, device) -> bool:
    """Whether ``out`` is what the fused step's last kernel reads forced tokens from and writes generated ones to by address:
    ``b`` rows of int64 on the model's device, each contiguous, any distance apart that keeps them disjoint."""
    return (out.dim() == 2 and out.shape[0] == b and out.dtype == torch.int64 and out.device == device and out.stride(1) == 1
            and (b == 1 or out.stride(0) >= out.shape[1]))


def projection_splits(b, n, k, residual, sms):
    """CTAs of a cluster that share the contraction of each 128-column tile of a decode projection (``n`` columns, ``k`` long).

    Doubled while a CTA keeps a K block of 64, up to what the batch makes worth while and what the ``sms`` SMs take in one go.
    A CTA finishes at least four sequences: up to 16 of them 4 CTAs (8 pad the sequences to 32), up to 32 8 CTAs.  Above, the exchange
    of the partial sums (32 KB a CTA) costs as much as the loads: 2 CTAs, except that the residual epilogue (out, c_proj: few columns,
    and per sequence a residual, x0 and sums of squares to handle) is shorter the fewer sequences a CTA finishes: 16, and 8 above
    64 sequences, where an SM holds one CTA.  Room: two CTAs of up to 64 sequences fit an SM, but clusters leave gaps: 1.6 CTAs an
    SM, 1.25 where clusters of 8 meet 17 to 32 sequences, one above 64 sequences and 0.8 of clusters of four or more (16 tiles
    by 8 CTAs: 524 us where 4 take 480).

    Six layers, us a step, all layers on this kernel, this rule against 2 CTAs for every projection of more than ten tiles and at most 160
    CTAs (``use_rows`` takes 1280 and 1408 wide up to 64 sequences to the other kernel, where they are faster still): 1280 wide the
    same (batch 64 242, batch 24 186, batch 8 171); 1408 wide 256 for 342 at batch 64, 336 for 399 at 128; 2048 wide 349 for 441, 437 for 515,
    246 for 253 at batch 8; 256 wide 145 for 148 and 204 for 212; 512 to 1152 wide the same.
    """
    tiles, kb = n // 128, k // 64
    most = 4 if b <= 16 else 8 if b <= 32 else 2 if not residual else 16 if b <= 64 else 8
    splits = 1
    while splits < most and splits * 2 <= kb:
        room = 1.6 if b <= 16 or 32 < b <= 64 else 1.25 if b <= 32 else 1.0 if splits == 1 else 0.8
        if tiles * splits * 2 > room * sms:
            break
        splits *= 2
    return splits


# What a projection brings to L2 ahead of the next one at most: a layer's largest weights with room to spare (13 MB at width 1280); of
# the head's 168 MB only as much as is read first.
AHEAD_LIMIT = 16 << 20


def rows_plan(b, n, k, sms):
    """``(columns of a tile, CTAs that share its contraction)`` of a projection on ``csrc/decode_rows.cu``, or None where it does not apply:
    more than 64 sequences (its MMA has 64 rows), too few or too many columns for one wave.

    A CTA fills an SM's shared memory, so a plan is one wave: at most ``sms`` CTAs, 0.9 of them in clusters of four or more, which leave
    gaps.  The contraction is shared until a CTA's part is 1536 at most (a chain of 96 MMAs, 2 us) and tiles of 32 columns or more
    occupy half of the SMs.  Within that, wide tiles (all CTAs read the same rows of X from L2: fewer of them, less traffic), but narrow
    ones in clusters of four or more, where a CTA's weights and its exchange count for more.  20 layers, 1280 wide, us a step, all else equal:
    qkv at batch 64 / 40 / 16 / 4 in tiles of 64 637 / 607 / 549 / 528, 48 644 / 607 / 545 / 520, 32 650 / 605 / 560 / 530, 64 by two CTAs
    654 / 633 / 568 / 523; out 32 by two 636 / 605 / 544 / 520, 16 by one 643 / 593 / 556 / 550; c_fc 64 634 / 597 / 534 / 518, 32 655 / 614 /
    569 / 543; c_proj 40 by four 634 / 594 / 534 / 517, 64 by four 660 / 597 / 536 / 517, 32 by two 661 / 621 / 560 / 548.
    """
    if b > 64 or k % 128:
        return None
    for s in (1, 2, 4, 8):
        if s > k // 128 or (k > 1536 * s and s < 8):
            continue
        fit = [nt for nt in (64, 48, 40, 32) if n % nt == 0 and sms // 2 <= n // nt * s <= (sms if s < 4 else int(0.9 * sms))]
        if fit:
            return (fit[0] if s < 4 else fit[-1]), s
    # few columns: the most CTAs with parts of 256 or more (256 wide: 115 us a step of six layers for 145 at batch 64, 103 for 106 at 8)
    few = [(n // nt * s, -s, nt) for nt in (16, 32, 64) for s in (1, 2, 4, 8)
           if n % nt == 0 and (s == 1 or k >= 256 * s) and k <= 1536 * s and n // nt * s < sms // 2]
    return (max(few)[2], -max(few)[1]) if few else None


def use_rows(b, c, a, hidden, sms):
    """Whether the layers' projections run on ``csrc/decode_rows.cu``: all four or none, since two of its CTAs, or one and one of the other
    kernel's, do not share an SM (2048 wide, ``out`` alone on it: 10 to 15 % slower).  Between 256 and 896 wide, models with few sequences
    stay on the other kernel, whose clusters split their contractions further.  Six layers, us a step here / there: 128 wide at batch 1 / 8 /
    16 88 / 93, 92 / 98, 94 / 100; 256 98 / 98, 103 / 106, 105 / 108; 384 113 / 107, 116 / 116, 118 / 118, at 20 121 / 128; 512 121 / 115, 125 / 121,
    127 / 126, at 20 132 / 132; 640 125 / 124, 129 / 131, 131 / 135; 768 134 / 133, 138 / 141, 137 / 141; 896 138 / 144, 138 / 149, 142 / 153."""
    if 256 < c < 896 and b <= 16:
        return False
    return all(rows_plan(b, n, k, sms) is not None for n, k in ((3 * a, c), (c, a), (hidden, c), (c, hidden)))


def head_on_rows(b, n, k):
    """Whether the head ``[n, k]`` of a step whose layers run on ``csrc/decode_rows.cu`` runs there too, its tiles walked by one CTA an SM.

    Above 32 sequences the other kernel pads to 64 and holds one CTA an SM; up to 16 it is the faster everywhere.  Between, what counts is
    the head's bytes.  A tile of a short contraction costs more here than there.  us a step of four layers here / there: 1280 x 65536 at
    batch 12 142.0 / 141.6, 20 143.8 / 142.5, 28 145.8 / 144.7, 33 148 / 158, 40 149 / 156, 64 157 / 160; 1024 x 32768 at 20 115.5 / 114.5, 33
    117.6 / 118.9, 64 125 / 127; 1536 x 65536 at 18 164.7 / 165.8, 28 169 / 170.5, 33 166 / 176; 1024 x 131072 at 18 158 / 162, 28 161 / 168, 64 169 /
    190.  Of six layers: 256 x 65536 at 20 129 / 122, 64 133.5 / 130, 256 x 8192 at 64 the same; 768 x 32768 at 40 160.5 / 158."""
    return (b > 32 and (k >= 1024 or n <= 16384)) or (b > 16 and n * k >= 100_000_000)


class NativeDecoder:
    """One decode step as a CUDA graph over the native kernels: embedding, fused norms, tcgen05 GEMMs, the two decode
    kernels (``csrc/decode.cu``: RoPE + QK-norm + cache append, cached attention), soft-capped logits, arg-max.  The
    position, the per-sequence document starts, the current tokens and the output buffer live on the device and are
    advanced inside the graph, so generating ``n`` tokens is ``n`` graph replays with no host synchronisation.
    Eligible: bf16 models on CUDA whose blocks all have attention with head_dim 128.  MoE blocks run their routed experts
    inside the graph (router, slotting, grouped expert GEMMs, combine: all device-side, a decode step uses one slot per
    sequence and expert); hashed input tables are looked up from row ids hashed on the device from the token history.
    With a cache in 8 bits the attention is ``ops.kv8_attention``.  ``logprobs=k``: ``report`` holds, for each position of ``out``, what the
    logits that it was chosen from say of the token there (a forced one's too), their entropy and k alternatives."""

    @staticmethod
    def eligible(model) -> bool:
        cfg = model.config
        w = model.lm_head.weight
        tables_ok = model.tables is None or model.tables.dtype == torch.bfloat16
        return (w.is_cuda and w.dtype == torch.bfloat16 and cfg.head_dim == 128 and tables_ok and getattr(model, "os1", None) is None
                and not ops.reference_path() and all(blk.attn is not None for blk in model.transformer.h))

    def __init__(self, model, cache: KVCache, first_tokens: torch.Tensor, out: torch.Tensor, prompt_len: int = 0, logprobs: int | None = None):
        # positions below ``prompt_len`` are teacher-forced from ``out`` (stepwise prefill through the same graph)
        self.model, self.cache, self.out = model, cache, out
        dev = first_tokens.device
        self.report = None if logprobs is None else _empty_report(first_tokens.shape[0], out.shape[1], logprobs, dev)
        self.prompt_len = torch.tensor([prompt_len], dtype=torch.int32, device=dev)
        self.tok = first_tokens.clone().to(torch.int64)
        self.pos = torch.tensor([cache.len], dtype=torch.int32, device=dev)
        self.graph = None
        cfg = model.config
        b, a = self.tok.shape[0], cfg.n_head * cfg.head_dim
        self.qbuf = torch.empty(b, a, dtype=torch.bfloat16, device=dev)
        self.y = torch.empty(b, a, dtype=torch.bfloat16, device=dev)
        # With few rows a projection has too few output tiles to pull its weights at memory speed, so its contraction
        # runs as a batch of products over K chunks of 256, each into its own fp32 slice, which the finishing kernel
        # adds in a fixed order (no atomics: a step is reproducible bit for bit).
        self.split = b <= 128 and cfg.n_embd % 256 == 0 and a % 256 == 0
        self.dense = [not isinstance(blk.mlp, MoeMLP) for blk in model.transformer.h]
        self.fused = self._fused_ok()
        if self.fused:
            c, f32, bf = cfg.n_embd, torch.float32, torch.bfloat16
            self.wqkv = [torch.cat([blk.attn.c_q.weight, blk.attn.c_k.weight, blk.attn.c_v.weight]) for blk in model.transformer.h]
            self.x0, self.xa, self.xb = (torch.empty(b, c, dtype=bf, device=dev) for _ in range(3))
            self.qkv = torch.empty(b, 3 * a, dtype=bf, device=dev)
            self.h = torch.empty(b, cfg.mlp_ratio * c, dtype=bf, device=dev)
            self.ssq_a, self.ssq_b = (torch.empty(c // 16, b, dtype=f32, device=dev) for _ in range(2))
            self.sms = torch.cuda.get_device_properties(dev).multi_processor_count
            self.rows = use_rows(b, c, a, cfg.mlp_ratio * c, self.sms)
            self.ticket = torch.zeros(1, dtype=torch.int32, device=dev)
            self.last_logits = torch.empty(b, model.lm_head.weight.shape[0], dtype=bf, device=dev)
        elif self.split:
            self.wqkv = [torch.cat([blk.attn.c_q.weight, blk.attn.c_k.weight, blk.attn.c_v.weight]).contiguous()
                         for blk in model.transformer.h]
            ws = self.wqkv + [blk.attn.c_proj.weight for blk in model.transformer.h]
            ws += [w for blk, dense in zip(model.transformer.h, self.dense) if dense for w in (blk.mlp.c_fc.weight, blk.mlp.c_proj.weight)]
            self.split = all(w.shape[1] % 256 == 0 for w in ws)
            self.part = torch.empty(max(b * w.shape[0] * (w.shape[1] // 256) for w in ws), dtype=torch.float32, device=dev)

    def _fused_ok(self) -> bool:
        """Whether the step runs on the kernels of ``csrc/decode_gemm.cu``: a plain dense decoder with at most 128 sequences.
        Any other ``out`` goes through the indexed reads and writes of the general step, which take or refuse it."""
        model, cfg = self.model, self.model.config
        ws = [w for blk, dense in zip(model.transformer.h, self.dense) if dense
              for w in (blk.attn.c_q.weight, blk.attn.c_k.weight, blk.attn.c_v.weight, blk.attn.c_proj.weight, blk.mlp.c_fc.weight, blk.mlp.c_proj.weight)]
        ws += [model.lm_head.weight, model.transformer.wte.weight]
        scalars = [v for blk in model.transformer.h for v in (blk.resid_lambda, blk.x0_lambda)]
        return (self.tok.shape[0] <= 128 and all(self.dense) and model.tables is None and model.value_embeds is None and not model.n_skip
                and len(model.transformer.h) > 0 and cfg.n_embd % 128 == 0 and _token_rows(self.out, self.tok.shape[0], self.tok.device)
                and all(w.dtype == torch.bfloat16 and w.is_contiguous() and w.data_ptr() % 16 == 0 and w.shape[0] % 128 == 0 and w.shape[1] % 64 == 0 for w in ws)
                and all(v.dtype == torch.float32 for v in scalars) and model.cos.dtype == torch.float32 and model.sin.dtype == torch.float32)

    def _proj(self, x, w, out, epi, ssq=None, n_ssq=0, res=None, mix=None, ssq_out=None, nxt=None):
        """One projection of the fused step, ``nxt`` the weights that it reads next; returns how many partial sums of squares a sequence has in ``ssq_out``."""
        from ..ops import _lib as L
        b, (n, k) = x.shape[0], w.shape
        x0, ma, mb = (self.x0, mix[0], mix[1]) if mix is not None else (None, None, None)
        head = epi == 3
        plan = None if not self.rows else rows_plan(b, n, k, self.sms) if not head else (64, 1) if head_on_rows(b, n, k) else None
        cap = ctypes.c_float(self.model.config.softcap)
        if plan is not None:
            nt, splits = plan
            L.call("bones_decode_rows", L.ptr(x), L.ptr(w), L.ptr(out), _I(b), _I(n), _I(k), _I(nt), _I(splits), _I(self.sms if head else 0), _I(epi), L.ptr(ssq), _I(n_ssq), L.ptr(res),
                   L.ptr(x0), L.ptr(ma), L.ptr(mb), L.ptr(ssq_out), cap, L.ptr(nxt),
                   ctypes.c_longlong(0 if nxt is None else min(2 * nxt.numel(), AHEAD_LIMIT)), _I(1), L.stream())
            return n // nt
        splits = projection_splits(b, n, k, res is not None, self.sms)
        L.call("bones_decode_gemm", L.ptr(x), L.ptr(w), L.ptr(out), _I(b), _I(n), _I(k), _I(splits), _I(epi), L.ptr(ssq), _I(n_ssq), L.ptr(res),
               L.ptr(x0), L.ptr(ma), L.ptr(mb), L.ptr(ssq_out), cap, _I(1), L.stream())
        return n // 128

    def _step_fused(self):
        """Five kernels a layer (qkv, attention, out, c_fc, c_proj), one before the first and two after the last; the norms,
        the residual mix, ReLU^2 and the soft-cap are in the projections' epilogues."""
        from ..ops import _lib as L, kv8 as KV8
        model, cache, cfg = self.model, self.cache, self.model.config
        tok, pos, b, c = self.tok, self.pos, self.tok.shape[0], cfg.n_embd
        ds = cache.doc_start if cfg.doc_mask else None
        hs = model.transformer.h
        w = model.transformer.wte.weight
        L.call("bones_decode_begin", L.ptr(tok), L.ptr(pos), L.ptr(ds), ctypes.c_longlong(cfg.bos_id), L.ptr(w), ctypes.c_longlong(w.shape[0]), _I(c),
               L.ptr(hs[0].resid_lambda), L.ptr(hs[0].x0_lambda), L.ptr(self.x0), L.ptr(self.xa), L.ptr(self.ssq_a), _I(b), L.stream())
        n_ssq = 1
        for i, blk in enumerate(hs):
            at = blk.attn
            self._proj(self.xa, self.wqkv[i], self.qkv, 0, ssq=self.ssq_a, n_ssq=n_ssq, nxt=at.c_proj.weight)
            if cache.kv8 is not None:
                dims = KV8.check_attention(self.qkv, model.cos, model.sin, cache.kv8[i], pos, ds, at.window)
                KV8.launch(self.qkv, model.cos, model.sin, dims, pos, at.scale, ds, at.window, self.y, pdl=1)
            else:
                L.call("bones_decode_attn_step", L.ptr(self.qkv), L.ptr(model.cos), L.ptr(model.sin), L.ptr(cache.k[i]), L.ptr(cache.v[i]), L.ptr(pos), L.ptr(ds),
                       L.ptr(self.y), _I(b), _I(at.n_head), _I(cache.max_len), ctypes.c_float(at.scale), _I(at.window // 128), L.stream())
            n_ssq = self._proj(self.y, at.c_proj.weight, self.xb, 2, res=self.xa, ssq_out=self.ssq_b, nxt=blk.mlp.c_fc.weight)
            self._proj(self.xb, blk.mlp.c_fc.weight, self.h, 1, ssq=self.ssq_b, n_ssq=n_ssq, nxt=blk.mlp.c_proj.weight)
            nxt = hs[i + 1] if i + 1 < len(hs) else None
            mix = (nxt.resid_lambda, nxt.x0_lambda) if nxt is not None else None
            n_ssq = self._proj(self.h, blk.mlp.c_proj.weight, self.xa, 2, res=self.xb, mix=mix, ssq_out=self.ssq_a,
                               nxt=self.wqkv[i + 1] if nxt is not None else model.lm_head.weight)
        self._proj(self.xa, model.lm_head.weight, self.last_logits, 3, ssq=self.ssq_a, n_ssq=n_ssq)
        L.call("bones_decode_end", L.ptr(self.last_logits), ctypes.c_longlong(self.last_logits.shape[1]), _I(cfg.vocab_size), L.ptr(pos),
               L.ptr(self.prompt_len), L.ptr(self.out), ctypes.c_longlong(self.out.stride(0)), _I(self.out.shape[1]), L.ptr(tok), L.ptr(self.ticket), _I(b),
               L.stream())

    def _lin(self, x, w, mode=0, residual=None):
        """``x [b, k] @ w[n, k]^T`` as ``k / 256`` batched partial products into fp32 slices, then their ordered sum as
        bf16 (mode 0), through ReLU^2 (2) or ``+ residual`` (1)."""
        from ..ops import _lib as L
        b, k = x.shape
        n = w.shape[0]
        splits = k // 256
        part = self.part[:splits * b * n]
        L.gemm(x, w, part, m=b, n=n, k=256, lda=x.stride(0), ldb=w.stride(0), ldd=n, epi=L.EPI_F32, force_bn=128, pair=False,
               batch=splits, stride_a=256, stride_b=256, stride_d=b * n)
        out = torch.empty(b, n, dtype=torch.bfloat16, device=x.device)
        L.call("bones_acc_finish", L.ptr(part), ctypes.c_int(splits), ctypes.c_longlong(b * n), L.ptr(residual), L.ptr(out),
               ctypes.c_longlong(b * n), ctypes.c_int(mode), L.stream())
        return out

    def _step(self):
        from ..ops import _lib as L
        from ..ops import cuda as C
        if self.fused:
            self._step_fused()
            return self._note()
        model, cache, cfg = self.model, self.cache, self.model.config
        tok, pos = self.tok, self.pos
        b, tmax = tok.shape[0], cache.max_len
        if cfg.doc_mask:
            cache.doc_start.copy_(torch.where(tok == cfg.bos_id, pos.expand(b), cache.doc_start))
        x = ops.embedding(tok, model.transformer.wte.weight, torch.bfloat16)
        if model.tables is not None:
            tb = model.tables
            ds = cache.doc_start if cfg.doc_mask else None
            for j, o in enumerate(tb.orders):
                rows = RF.ngram_rows_at(self.out, pos, o, tb.rows, tb.seed + j, ds)
                x = x + model.table_lambda[j].to(x.dtype) * tb.gather(j, rows)
        x = ops.rms_norm(x)
        x0 = x
        skips = []
        n_layer, n_skip = cfg.n_layer, model.n_skip
        for i, blk in enumerate(model.transformer.h):
            if n_skip and i >= n_layer - n_skip:
                x = x + model.skip_lambda[i - (n_layer - n_skip)].to(x.dtype) * skips.pop()
            x, xn = ops.resid_mix_norm(x, x0, blk.resid_lambda, blk.x0_lambda)
            at = blk.attn
            qkv = self._lin(xn, self.wqkv[i]) if self.split else ops.linear_qkv(xn, at.c_q.weight, at.c_k.weight, at.c_v.weight)
            ve = lam = None
            if model.value_embeds is not None and str(i) in model.value_embeds:
                ve = ops.embedding(tok, model.value_embeds[str(i)].weight, torch.bfloat16)
                lam = blk.ve_lambda.detach().float()
            if cache.kv8 is not None:
                if ve is not None:
                    qkv[:, 2 * ve.shape[1]:].add_(lam.to(qkv.dtype) * ve)          # as in training: both factors and the product in bf16
                y = ops.kv8_attention(qkv, model.cos, model.sin, cache.kv8[i], pos, at.scale, cache.doc_start if cfg.doc_mask else None, at.window)
            else:
                y = self.y
                L.call("bones_decode_qkv", L.ptr(qkv), L.ptr(model.cos), L.ptr(model.sin), L.ptr(ve), L.ptr(lam), L.ptr(self.qbuf),
                       L.ptr(cache.k[i]), L.ptr(cache.v[i]), L.ptr(pos), C._I(b), C._I(at.n_head), C._I(tmax), L.stream())
                L.call("bones_decode_attn", L.ptr(self.qbuf), L.ptr(cache.k[i]), L.ptr(cache.v[i]), L.ptr(pos),
                       L.ptr(cache.doc_start if cfg.doc_mask else None), L.ptr(y), C._I(b), C._I(at.n_head), C._I(tmax),
                       C._F(at.scale), C._I(at.window // 128), L.stream())
            if self.split:
                x = self._lin(y, at.c_proj.weight, 1, x)
                x, xn = ops.norm_split(x)
                if self.dense[i]:
                    x = self._lin(self._lin(xn, blk.mlp.c_fc.weight, 2), blk.mlp.c_proj.weight, 1, x)
                else:
                    x = blk.mlp(xn.view(b, 1, -1), residual=x.view(b, 1, -1)).view(b, -1)
            else:
                x = ops.linear(y, at.c_proj.weight, residual=x)
                x, xn = ops.norm_split(x)
                x = blk.mlp(xn.view(b, 1, -1), residual=x.view(b, 1, -1)).view(b, -1) if not self.dense[i] else blk.mlp(xn, residual=x)
            if n_skip and i < n_skip:
                skips.append(x)
        xn = ops.rms_norm(x)
        logits = C.mm_nt(xn, model.lm_head.weight, epi=L.EPI_SOFTCAP, alpha=1.0 / cfg.softcap, beta=cfg.softcap)
        self.last_logits = logits                                          # [B, padded vocab] bf16, soft-capped
        nxt = logits[:, :cfg.vocab_size].float().argmax(-1)
        pos.add_(1)
        at = pos.to(torch.int64)
        forced = self.out.index_select(1, at)[:, 0]
        nxt = torch.where((pos < self.prompt_len).expand_as(nxt), forced, nxt)
        self.out.index_copy_(1, at, nxt[:, None])                         # token at position pos (after the increment)
        tok.copy_(nxt)
        self._note()

    def _note(self):
        """What this step's logits say of the token that now stands at ``pos``; a step past the end of ``out`` leaves the last place."""
        if self.report is None:
            return
        k = self.report.top_id.shape[2]
        at = self.pos.to(torch.int64).clamp(max=self.report.logprob.shape[1] - 1)
        for kept, new in zip(self.report, ops.token_logprobs(self.last_logits, self.tok, k, self.model.config.vocab_size)):
            kept.index_copy_(1, at, new[:, None])

    @torch.no_grad()
    def run(self, n_steps: int):
        """``n_steps`` decode steps; the first one runs eagerly (it also warms every kernel up), the rest replay the graph."""
        if n_steps <= 0:
            return
        self._step()
        if n_steps == 1:
            return
        if self.graph is None:
            torch.cuda.synchronize()
            self.graph = torch.cuda.CUDAGraph()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                with torch.cuda.graph(self.graph, stream=side):
                    self._step()
            torch.cuda.current_stream().wait_stream(side)       # capturing does not execute the step
        for _ in range(n_steps - 1):
            self.graph.replay()


def _empty_report(b: int, length: int, k: int, dev) -> ops.TokenLogprobs:
    """Zeros for ``length`` positions, and one place more for what a step past the end writes."""
    z = lambda dt, *shape: torch.zeros(b, length + 1, *shape, dtype=dt, device=dev)  # noqa: E731
    return ops.TokenLogprobs(z(torch.float32), z(torch.float32), z(torch.float32, k), z(torch.int64, k))


def _with_report(out, report, p: int):
    """What ``greedy_decode`` returns: the tokens, and where it was asked for what the new ones were worth."""
    return out if report is None else (out, ops.TokenLogprobs(*(x[:, p:out.shape[1]].contiguous() for x in report)))


def _noted(model, logits, nxt, k, report: list):
    if k is not None:
        report.append(ops.token_logprobs(logits, nxt, k, model.config.vocab_size))


def _stacked(report: list, b: int, k, dev):
    if k is None:
        return None
    return ops.TokenLogprobs(*(torch.stack(x, 1) for x in zip(*report))) if report else ops.TokenLogprobs(*(x[:, :0] for x in _empty_report(b, 0, k, dev)))


@torch.no_grad()
def greedy_decode(model, prompts: torch.Tensor, n_new: int, kv: str = "bf16", logprobs: int | None = None):
    """``prompts [B, P]`` -> ``[B, P + n_new]`` by arg-max decoding.  ``kv``: how the cache holds keys and values, ``"bf16"`` or ``"int8"`` (for
    long answers; see the module's text).
    ``logprobs=k``: ``(tokens, TokenLogprobs)`` with the log-probability, the entropy and k alternatives of each new token ``[B, n_new]``."""
    b, p = prompts.shape
    if p + n_new > model.config.sequence_len:
        raise ValueError("prompt + new tokens exceed the model's sequence length")
    if kv not in KV_TYPES:
        raise ValueError(f"key/value cache {kv!r} (one of {KV_TYPES})")
    if logprobs is not None and not 0 <= logprobs <= min(ops._logprobs.TOP_MAX, model.config.vocab_size):
        raise ValueError(f"{logprobs} alternatives (0 to {min(ops._logprobs.TOP_MAX, model.config.vocab_size)})")
    if getattr(model, "os1", None) is not None or any(blk.attn is None for blk in model.transformer.h):
        if kv != "bf16":
            raise ValueError("models with an output table or attention-free blocks decode without a cache")
        return greedy_decode_full(model, prompts, n_new, logprobs)          # cache-free route
    cache = KVCache(model, b, p + n_new, kv)
    if NativeDecoder.eligible(model) and n_new >= 1:
        out = torch.zeros(b, p + n_new, dtype=torch.int64, device=prompts.device)
        out[:, :p] = prompts
        if p <= 512:
            # short prompts are pre-filled token by token through the same graph (teacher-forced), then decoded
            dec = NativeDecoder(model, cache, prompts[:, 0], out, prompt_len=p, logprobs=logprobs)
            dec.run(p + n_new - 1)
            report = dec.report
        else:
            # long prompts: prefill on the cached PyTorch route, then one graph replay per generated token
            logits = _forward_cached(model, prompts, cache)
            first = logits.argmax(-1)
            out[:, p] = first
            report = None if logprobs is None else _empty_report(b, p + n_new, logprobs, prompts.device)
            if n_new > 1:
                dec = NativeDecoder(model, cache, first, out, logprobs=logprobs)
                dec.run(n_new - 1)
                report = dec.report
            if report is not None:
                for kept, new in zip(report, ops.token_logprobs(logits, first, logprobs, model.config.vocab_size)):
                    kept[:, p] = new
        L_check()
        return _with_report(out, report, p)
    out, report = [prompts], []
    logits = _forward_cached(model, prompts, cache)
    for _ in range(n_new):
        nxt = logits.argmax(-1, keepdim=True)
        out.append(nxt)
        _noted(model, logits, nxt[:, 0], logprobs, report)
        if cache.len >= p + n_new:
            break
        logits = _forward_cached(model, nxt, cache)
    out, report = torch.cat(out, 1)[:, :p + n_new], _stacked(report, b, logprobs, prompts.device)
    return out if report is None else (out, report)


@torch.no_grad()
def greedy_decode_full(model, prompts: torch.Tensor, n_new: int, logprobs: int | None = None):
    """Cache-free decoding (re-runs the full forward per token); the oracle for the cached path and the route used
    when hashed tables are attached."""
    seq, report = prompts, []
    for _ in range(n_new):
        logits = model(seq)[:, -1]
        nxt = logits.argmax(-1, keepdim=True)
        _noted(model, logits, nxt[:, 0], logprobs, report)
        seq = torch.cat([seq, nxt], 1)
    report = _stacked(report, prompts.shape[0], logprobs, prompts.device)
    return seq if report is None else (seq, report)
