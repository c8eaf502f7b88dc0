"""Decoding with a cache in 8 bits and with what the answers were worth, on the CPU."""
import pytest
import torch


def _model(**kw):
    from them_bones_b200.config import GPTConfig
    from them_bones_b200.models.gpt import GPT
    torch.manual_seed(3)
    cfg = GPTConfig(**{**dict(sequence_len=160, vocab_size=97, n_layer=2, n_head=2, n_embd=128, head_dim=64, doc_mask=True), **kw})
    model = GPT(cfg)
    model.init_weights()
    for p in model.parameters():
        if p.dim() == 2:
            torch.nn.init.normal_(p, std=0.08)
    return model.eval()


@pytest.mark.parametrize("kw", [{}, dict(attn_window=128, attn_long=(1,)), dict(value_embeds=1), dict(unet=True)])
def test_a_prompt_at_once_or_token_by_token(kw):
    """The cache holds the same either way, so the logits differ by the rounding of products of other shapes alone."""
    from them_bones_b200.utils import decode as D
    model, b, n = _model(**kw), 3, 150
    toks = torch.randint(1, 97, (b, n))
    toks[:, 0] = 0
    toks[1, 70] = toks[2, 64] = toks[2, 149] = 0
    whole, parts, bf16 = D.KVCache(model, b, n, "int8"), D.KVCache(model, b, n, "int8"), D.KVCache(model, b, n)
    a = D._forward_cached(model, toks, whole)
    for i in range(n):
        c = D._forward_cached(model, toks[:, i:i + 1], parts)
    # keys and values of unit size pass through bf16 (a rounding that falls the other way moves one by 2^-7) and 7 bits; logits of size 1
    assert float((a - c).abs().max()) < 2 ** -7
    same = sum(int((x != y).sum()) for p, q in zip(whole.kv8, parts.kv8) for x, y in zip(p[:2], q[:2]))
    assert same <= 2e-3 * sum(x.numel() for p in whole.kv8 for x in p[:2])
    exact = D._forward_cached(model, toks, bf16)
    assert 0 < float((a - exact).norm() / exact.norm()) < 2e-2          # a code is off by 1/254 of its block's largest value at most


@pytest.mark.parametrize("kv", ["bf16", "int8"])
def test_greedy_decode_tells_what_its_answers_were_worth(kv):
    from them_bones_b200 import ops
    from them_bones_b200.utils import decode as D
    model = _model()
    prompts = torch.randint(1, 97, (2, 70))
    plain = D.greedy_decode(model, prompts, 12, kv=kv)
    out, r = D.greedy_decode(model, prompts, 12, kv=kv, logprobs=4)
    assert torch.equal(plain, out) and out.shape == (2, 82)
    assert r.logprob.shape == r.entropy.shape == (2, 12) and r.top_id.shape == r.top_logprob.shape == (2, 12, 4)
    assert torch.equal(r.top_id[..., 0], out[:, 70:]) and torch.equal(r.top_logprob[..., 0], r.logprob)
    with torch.no_grad():
        want = ops.token_logprobs(model(out)[:, 69:-1], out[:, 70:], 4)
    tol = 1e-4 if kv == "bf16" else 2e-2                                # fp32 products of other shapes; codes of 7 bits
    assert float((r.logprob - want.logprob).abs().max()) < tol and float((r.entropy - want.entropy).abs().max()) < tol
    none = D.greedy_decode(model, prompts, 0, kv=kv, logprobs=2)[1]
    assert none.logprob.shape == (2, 0) and none.top_id.shape == (2, 0, 2)


def test_cache_free_models_and_refusals():
    from them_bones_b200.utils import decode as D
    model = _model(attn_layers=(1,))
    prompts = torch.randint(1, 97, (2, 5))
    out, r = D.greedy_decode(model, prompts, 3, logprobs=1)
    assert torch.equal(r.top_id[..., 0], out[:, 5:])
    with pytest.raises(ValueError):
        D.greedy_decode(model, prompts, 3, kv="int8")
    model = _model()
    for kw in (dict(kv="fp8"), dict(logprobs=-1), dict(logprobs=33)):
        with pytest.raises(ValueError):
            D.greedy_decode(model, prompts, 3, **kw)
    with pytest.raises(ValueError):
        D.greedy_decode(_model(n_head=4, head_dim=32), prompts, 3, kv="int8")
    with pytest.raises(ValueError):
        D.KVCache(model, 2, 8, "int4")


def test_scores_token_by_token():
    from them_bones_b200.utils.evalbpb import report_continuations, score_continuations
    model = _model()
    toks = torch.randint(1, 97, (3, 40))
    ctx, total = torch.tensor([5, 39, 1]), torch.tensor([20, 40, 40])
    r = report_continuations(model, toks, ctx, total, 3)
    s = score_continuations(model, toks, ctx, total)
    assert r.logprob.shape == (3, 40) and r.top_id.shape == (3, 40, 3)
    assert float((r.logprob.sum(1) - s).abs().max()) < 1e-4             # 39 fp32 terms of size 5
    pos = torch.arange(40)[None]
    keep = (pos >= ctx[:, None]) & (pos < total[:, None])
    assert not r.logprob[~keep].any() and not r.entropy[~keep].any() and not r.top_id[~keep].any() and bool((r.entropy[keep] > 0).all())
    best = model(toks).argmax(-1)
    assert torch.equal(r.top_id[:, 1:, 0][keep[:, 1:]], best[:, :-1][keep[:, 1:]])


def test_gradient_through_the_model():
    """Log-probability and entropy of given tokens as a loss: the same gradient as from the loss head and from the logits."""
    from them_bones_b200 import ops
    model = _model()
    idx = torch.randint(1, 97, (2, 30))
    tokens = torch.randint(0, 97, (2, 30))
    tokens[0, 3] = -1
    r = model.token_logprobs(idx, tokens)
    ps = [p for p in model.parameters() if p.dim() == 2]
    a = torch.autograd.grad(-r.logprob.sum(), ps, retain_graph=True)
    b = torch.autograd.grad(model(idx, tokens, loss_reduction="sum"), ps)
    for x, y in zip(a, b):
        assert float((x - y).norm()) <= 1e-5 * float(y.norm()) + 1e-7
    c = torch.autograd.grad(r.entropy.sum(), ps)
    d = torch.autograd.grad(ops.token_logprobs(model(idx), tokens).entropy.sum(), ps)
    for x, y in zip(c, d):
        assert float((x - y).norm()) <= 1e-5 * float(y.norm()) + 1e-7
    model.os1 = object()
    with pytest.raises(ValueError):
        model.token_logprobs(idx, tokens)


def test_head_refusals():
    from them_bones_b200 import ops
    x, w, t = torch.randn(3, 16), torch.randn(24, 16), torch.zeros(3, dtype=torch.int64)
    for args in ((x, w[:, :8], t, 20, 15.0), (x, w, t[:2], 20, 15.0), (x, w, t, 25, 15.0), (x, w, t, 0, 15.0), (x, w, t, 20, 15.0, 21), (x, w, t.float(), 20, 15.0)):
        with pytest.raises(ValueError):
            ops.lmhead_logprobs(*args)
