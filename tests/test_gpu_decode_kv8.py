"""The decode step with a cache in 8 bits, and with what its answers were worth."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(n_embd=256, n_layer=2, seq=256, **kw):
    from them_bones_b200.config import GPTConfig
    from them_bones_b200.models.gpt import GPT
    torch.manual_seed(3)
    cfg = GPTConfig(**{**dict(sequence_len=seq, vocab_size=1024, n_layer=n_layer, n_head=n_embd // 128, n_embd=n_embd, head_dim=128, doc_mask=True), **kw})
    with torch.device("cuda"):
        model = GPT(cfg)
    model.init_weights()
    for p in model.parameters():
        if p.dim() >= 2:
            torch.nn.init.normal_(p, std=0.05)
    return model.cast_compute(torch.bfloat16).eval()


def _tokens(b, n, docs=True):
    toks = torch.randint(1, 1000, (b, n), device="cuda")
    if docs:
        toks[torch.rand(b, n, device="cuda") < 0.03] = 0
    toks[:, 0] = 0
    return toks


@pytest.mark.parametrize("b,kw,fused", [(64, {}, True), (7, dict(attn_window=128, attn_long=(1,)), True), (1, {}, True), (100, dict(n_embd=384), True), (130, {}, False),
                                        (5, dict(value_embeds=1), False), (4, dict(unet=True), False), (6, dict(n_embd=640, n_layer=1), True)])
def test_step_with_an_8_bit_cache(b, kw, fused):
    from them_bones_b200.utils import decode as D
    model, n = _model(**kw), 150
    toks = _tokens(b, n)
    toks[: b // 2, n - 1] = 0
    out = torch.cat([toks, torch.zeros(b, 1, dtype=torch.int64, device="cuda")], 1)
    with torch.no_grad():
        cache = D.KVCache(model, b, n + 1, "int8")
        dec = D.NativeDecoder(model, cache, toks[:, 0], out, prompt_len=n, logprobs=4)
        assert dec.fused == fused
        dec.run(n)
        got = dec.last_logits[:, :1024].float()
        ref_cache = D.KVCache(model, b, n + 1, "int8")
        ref = D._forward_cached(model, toks, ref_cache)
        bf16 = D._forward_cached(model, toks, D.KVCache(model, b, n + 1))
    D.L_check()
    rel = (got - ref).norm(dim=1) / ref.norm(dim=1)
    assert float(rel.max()) < 6e-2, rel                     # bf16 activations of the layers, row by row, as with a bf16 cache
    assert float((ref - bf16).norm() / bf16.norm()) < 6e-2
    # what the first layer's cache holds comes from the same inputs up to bf16 activations: keys of unit size, a bf16 step or two and a code apart
    for x, y, scale in zip(cache.kv8[0][:2], ref_cache.kv8[0][:2], cache.kv8[0][2:4]):
        assert float((x.float() - y.float())[..., :128, :].abs().mean()) < 2.0
    assert not any(bool(s.signbit().any()) for layer in cache.kv8 for s in layer[2:4])
    # the last position's report is that of the logits that stand there
    from them_bones_b200 import ops
    want = ops.token_logprobs(dec.last_logits, out[:, n], 4, 1024)
    assert all(torch.equal(x[:, n], y) for x, y in zip(dec.report, want)) and torch.equal(dec.report.top_id[:, n, 0], out[:, n])
    assert bool((dec.report.logprob[:, 1:n] < 0).all()) and not dec.report.logprob[:, 0].any() and not dec.report.logprob[:, n + 1].any()


def test_report_of_forced_tokens_matches_the_scores():
    """Teacher-forced positions: the step's log-probabilities against the batched scoring path's."""
    from them_bones_b200.utils import decode as D
    from them_bones_b200.utils.evalbpb import report_continuations, score_continuations
    model, b, n = _model(), 9, 140
    toks = _tokens(b, n, docs=False)
    out = torch.cat([toks, torch.zeros(b, 1, dtype=torch.int64, device="cuda")], 1)
    with torch.no_grad():
        dec = D.NativeDecoder(model, D.KVCache(model, b, n + 1), toks[:, 0], out, prompt_len=n, logprobs=2)
        dec.run(n)
        r = report_continuations(model, toks, torch.ones(b, dtype=torch.int64, device="cuda"), torch.full((b,), n, device="cuda"), 2)
        s = score_continuations(model, toks, torch.ones(b, dtype=torch.int64, device="cuda"), torch.full((b,), n, device="cuda"))
    # logits of size 3 that went through bf16 activations on two routes: a few percent of them
    assert float((dec.report.logprob[:, 1:n] - r.logprob[:, 1:]).abs().max()) < 0.3
    assert float((dec.report.logprob[:, 1:n] - r.logprob[:, 1:]).abs().mean()) < 0.03
    assert float((r.logprob.sum(1) - s).abs().max()) < 139 * 2 ** -7       # bf16 logits of size 3 here, fp32 sums there


@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("p", [5, 600])
def test_greedy_decode(kv, p):
    """Prompts that are fed token by token, and long ones that go through the other route first."""
    from them_bones_b200.utils import decode as D
    model = _model(n_layer=1, seq=1024)
    prompts = _tokens(2, p)
    plain = D.greedy_decode(model, prompts, 70, kv=kv)
    out, r = D.greedy_decode(model, prompts, 70, kv=kv, logprobs=3)
    assert torch.equal(plain, out) and torch.equal(out[:, :p], prompts)
    assert r.logprob.shape == (2, 70) and torch.equal(r.top_id[..., 0], out[:, p:]) and torch.equal(r.top_logprob[..., 0], r.logprob)
    one, q = D.greedy_decode(model, prompts, 1, kv=kv, logprobs=0)
    assert torch.equal(one, out[:, :p + 1]) and q.top_id.shape == (2, 1, 0) and torch.equal(q.logprob, r.logprob[:, :1])


def test_steps_past_the_end_and_two_decoders():
    from them_bones_b200.utils import decode as D
    model, b, n = _model(), 3, 20
    toks = _tokens(b, n)
    outs = []
    with torch.no_grad():
        decs = []
        for _ in range(2):
            out = torch.cat([toks[:, :8], torch.zeros(b, n - 8, dtype=torch.int64, device="cuda")], 1)
            decs.append(D.NativeDecoder(model, D.KVCache(model, b, n, "int8"), toks[:, 0], out, prompt_len=8, logprobs=2))
            outs.append(out)
        for _ in range(5):                                   # in turn: the graphs share nothing
            for d in decs:
                d.run(3)
        alone = torch.cat([toks[:, :8], torch.zeros(b, n - 8, dtype=torch.int64, device="cuda")], 1)
        dec = D.NativeDecoder(model, D.KVCache(model, b, n, "int8"), toks[:, 0], alone, prompt_len=8, logprobs=2)
        dec.run(15)
    D.L_check()
    assert torch.equal(outs[0], alone) and torch.equal(outs[1], alone)
    assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(dec.report, decs[0].report, decs[1].report))
    kept = [x.clone() for x in dec.report]
    dec.run(4)
    assert torch.equal(alone[:, :16], outs[0][:, :16]) and all(torch.equal(x[:, :16], y[:, :16]) for x, y in zip(dec.report, kept))


def test_long_cache_step(monkeypatch):
    """The step over a cache in which all heads share the CTAs, against the same step with a cluster for each: a document that begins within the
    step is seen by both, and later tokens see no other document's."""
    from them_bones_b200 import ops
    from them_bones_b200.utils import decode as D
    model, b, n = _model(seq=16384), 3, 140
    toks = _tokens(b, n)
    toks[0, 70], toks[1, 128], toks[2, n - 1] = 0, 0, 0
    logits, caches = [], []
    for long in (ops._kv8.LONG, 1 << 40):
        monkeypatch.setattr(ops._kv8, "LONG", long)
        out = torch.cat([toks, torch.zeros(b, 1, dtype=torch.int64, device="cuda")], 1)
        with torch.no_grad():
            cache = D.KVCache(model, b, 16384, "int8")
            dec = D.NativeDecoder(model, cache, toks[:, 0], out, prompt_len=n)
            assert dec.fused
            dec.run(n)
        logits.append(dec.last_logits[:, :1024].float())
        caches.append(cache)
    D.L_check()
    # two orders of summation, rounded to bf16: a step of it here and there, through two layers
    assert float((logits[0] - logits[1]).norm() / logits[1].norm()) < 2e-2
    for x, y in zip(caches[0].kv8[0], caches[1].kv8[0]):                     # the first layer's keys and values do not depend on it
        assert torch.equal(x, y)
    assert torch.equal(caches[0].doc_start, caches[1].doc_start)


def test_moe_step():
    from them_bones_b200.config import moe_capacity_for
    from them_bones_b200.utils import decode as D
    model = _model(moe_layers=(1,), moe_experts=4, moe_topk=2, moe_hidden=256, moe_capacity=moe_capacity_for(1.25, 256, 2, 4))
    prompts = _tokens(4, 6)
    out, r = D.greedy_decode(model, prompts, 80, kv="int8", logprobs=2)
    assert torch.equal(r.top_id[..., 0], out[:, 6:]) and bool(r.logprob.isfinite().all())


# -- the head ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("m,c,vocab,padded,topk", [(1, 64, 100, 128, 3), (5, 256, 1000, 1024, 0), (300, 128, 8192, 8192, 8), (130, 64, 509, 512, 32)])
def test_head_against_64_bits(m, c, vocab, padded, topk, monkeypatch):
    from them_bones_b200 import ops
    from them_bones_b200.ops import cuda as C
    monkeypatch.setattr(C, "LOSS_ROWS", 128)                 # several blocks of rows
    torch.manual_seed(m)
    x = torch.randn(m, c, device="cuda").bfloat16().requires_grad_()
    w = (0.3 * torch.randn(padded, c, device="cuda")).bfloat16().requires_grad_()
    tokens = torch.randint(-1, vocab, (m,), device="cuda")
    r = ops.lmhead_logprobs(x, w, tokens, vocab, 15.0, topk)
    # by the same blocks: how many CTAs share a row, and with it the order of its sum, goes by the number of rows
    blocks = [C.mm_nt(x.detach()[a:a + 128], w.detach(), epi=C.L.EPI_SOFTCAP, alpha=1 / 15.0, beta=15.0) for a in range(0, m, 128)]
    want = [ops.token_logprobs(z, t, topk, vocab) for z, t in zip(blocks, tokens.split(128))]
    assert all(torch.equal(a, torch.cat(b)) for a, b in zip(r, zip(*want)))
    z = torch.cat(blocks)
    gs = [torch.randn(m, device="cuda"), torch.randn(m, device="cuda"), torch.randn(m, topk, device="cuda")]
    at = [r.logprob, r.entropy] + ([r.top_logprob] if topk else [])
    dx, dw = torch.autograd.grad(at, [x, w], gs[:len(at)])
    # the gradient's own formula from the bf16 logits, in 64 bits
    z64 = z[:, :vocab].double()
    logp = torch.log_softmax(z64, -1)
    p, h = logp.exp(), -(logp.exp() * logp).sum(-1, keepdim=True)
    g = (gs[0] * (tokens >= 0)).double()[:, None]
    d = -p * (g + gs[2].double().sum(1, keepdim=True) + gs[1].double()[:, None] * (logp + h))
    d.scatter_add_(1, tokens.clamp_min(0)[:, None], g)
    if topk:
        d.scatter_add_(1, r.top_id, gs[2].double())
    d = d * (1 - (z64 / 15.0).square())
    dx64, dw64 = d @ w.detach().double()[:vocab], d.T @ x.detach().double()
    # bf16 logit gradients (2^-9 of each on average) summed at random, then one rounding of the result to bf16
    rel = lambda a, b: float((a.double() - b).norm() / b.norm())  # noqa: E731
    assert rel(dx, dx64) < 2 ** -7 and rel(dw[:vocab], dw64) < 2 ** -7 and not dw[vocab:].any()


def test_head_gradient_that_the_weight_owns():
    from them_bones_b200 import ops
    torch.manual_seed(0)
    x, w = torch.randn(40, 64, device="cuda").bfloat16(), (0.3 * torch.randn(256, 64, device="cuda")).bfloat16()
    tokens = torch.randint(0, 250, (40,), device="cuda")
    own, plain = (w.clone().requires_grad_() for _ in range(2))
    own.main_grad = torch.ones(256, 64, device="cuda")
    a = ops.lmhead_logprobs(x.requires_grad_(), own, tokens, 250, 15.0)
    a.logprob.sum().backward()
    b = ops.lmhead_logprobs(x.detach().clone().requires_grad_(), plain, tokens, 250, 15.0)
    b.logprob.sum().backward()
    assert own.grad is None and float((own.main_grad - 1 - plain.grad.float()).norm()) < 2 ** -7 * float(plain.grad.float().norm())
    with torch.no_grad():
        assert not ops.lmhead_logprobs(x, w, tokens, 250, 15.0).logprob.requires_grad


def test_head_rows_and_weights_that_lie_anywhere():
    from them_bones_b200 import ops
    torch.manual_seed(2)
    x, w = torch.randn(2, 9, 65, device="cuda").bfloat16(), (0.3 * torch.randn(65, 129, device="cuda")).bfloat16()
    tokens = torch.randint(0, 120, (2, 9), device="cuda")
    for xv, wv in ((x[:, ::2, 1:], w[:64, :128].T), (x[..., :64].transpose(0, 1).transpose(0, 1), w[1:, 1:].T), (x[:, :, :64], w.T[:128, 1:])):
        leaves = [t.detach().requires_grad_() for t in (xv, wv)]
        plain = [t.detach().clone(memory_format=torch.contiguous_format).requires_grad_() for t in (xv, wv)]
        tk = tokens[:, :xv.shape[1]]
        a, b = (ops.lmhead_logprobs(*t, tk, 120, 15.0, 3) for t in (leaves, plain))
        assert a.logprob.shape == tk.shape and all(torch.equal(p, q) for p, q in zip(a, b))
        for p, q in zip(torch.autograd.grad(a.logprob.sum(), leaves), torch.autograd.grad(b.logprob.sum(), plain)):
            assert p.shape == q.shape and float((p.float() - q.float()).norm()) <= 2 ** -8 * float(q.float().norm())


def test_head_of_no_rows():
    from them_bones_b200 import ops
    x, w = torch.randn(0, 64, device="cuda").bfloat16().requires_grad_(), torch.randn(128, 64, device="cuda").bfloat16().requires_grad_()
    r = ops.lmhead_logprobs(x, w, torch.zeros(0, dtype=torch.int64, device="cuda"), 120, 15.0, 2)
    dx, dw = torch.autograd.grad(r.entropy.sum(), [x, w])
    assert r.top_id.shape == (0, 2) and dx.shape == (0, 64) and not dw.any()


def test_head_batched_and_recorded_gradients():
    from them_bones_b200 import ops
    torch.manual_seed(1)
    x, w = torch.randn(6, 64, device="cuda").bfloat16().requires_grad_(), (0.3 * torch.randn(128, 64, device="cuda")).bfloat16().requires_grad_()
    r = ops.lmhead_logprobs(x, w, torch.randint(0, 120, (6,), device="cuda"), 120, 15.0, 2)
    rows = torch.eye(6, device="cuda")
    batched, = torch.autograd.grad(r.logprob, [x], rows, is_grads_batched=True, retain_graph=True)
    single = torch.stack([torch.autograd.grad(r.logprob, [x], e, retain_graph=True)[0] for e in rows])
    assert float((batched.float() - single.float()).norm() / single.float().norm()) < 2e-2          # one route's logits are bf16
    d, = torch.autograd.grad(r.entropy.sum(), [x], create_graph=True)
    dd, = torch.autograd.grad(d.float().square().sum(), [w])
    assert bool(dd.isfinite().all()) and dd.any()


def test_model_gradient_on_the_native_path():
    """A policy's step through the whole model: the head's gradient against the loss head's on the same tokens."""
    model = _model(n_layer=2).train()
    idx = _tokens(2, 128)
    tokens = torch.roll(idx, -1, 1)
    ps = [p for p in model.parameters() if p.dim() == 2]
    r = model.token_logprobs(idx, tokens)
    a = torch.autograd.grad(-r.logprob.mean(), ps, allow_unused=True)
    b = torch.autograd.grad(model(idx, tokens), ps, allow_unused=True)
    for x, y in zip(a, b):
        assert (x is None) == (y is None)
        if x is not None and float(y.float().norm()) > 0:
            assert float((x.float() - y.float()).norm() / y.float().norm()) < 3e-2      # bf16 roundings of the same gradient on two routes


def test_head_native_refusals():
    from them_bones_b200 import ops
    x, w, t = torch.randn(3, 64, device="cuda").bfloat16(), torch.randn(128, 64, device="cuda").bfloat16(), torch.zeros(3, dtype=torch.int64, device="cuda")
    for args in ((x.float(), w, t, 100, 15.0), (x, w.float(), t, 100, 15.0), (x, w, t, 100, 0.0), (x[:, :60], w[:, :60], t, 100, 15.0)):
        with pytest.raises(ValueError):
            ops.lmhead_logprobs(*args)
