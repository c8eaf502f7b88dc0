"""The log-probability kernels against 64 bits and against the statement, on the rows where they can go wrong."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _exact(z, tokens, topk, vocab):
    z = z.detach()[:, :vocab].double()
    logp = torch.log_softmax(z, -1)
    gone = logp == float("-inf")
    lp0 = logp.masked_fill(gone, 0.0)
    h = -(logp.exp() * lp0).sum(-1)
    some = (tokens >= 0) & (tokens < vocab)
    given = torch.where(some, logp.gather(1, tokens.clamp(0, vocab - 1)[:, None])[:, 0], torch.zeros((), dtype=torch.float64, device=z.device))
    ids = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :topk]
    return given, h, logp.gather(1, ids), ids, logp, lp0, some


def _exact_grad(z, tokens, topk, vocab, gs):
    _, h, _, ids, logp, lp0, some = _exact(z, tokens, topk, vocab)
    p = logp.exp()
    d = torch.zeros_like(p)
    if gs[0] is not None:
        g = gs[0].double() * some
        d -= g[:, None] * p
        d.scatter_add_(1, tokens.clamp(0, vocab - 1)[:, None], g[:, None])
    if gs[1] is not None:
        d -= gs[1].double()[:, None] * p * (lp0 + h[:, None])
    if gs[2] is not None and topk:
        d -= gs[2].double().sum(1, keepdim=True) * p
        d.scatter_add_(1, ids, gs[2].double())
    return torch.nn.functional.pad(d, (0, z.shape[1] - vocab)), p


def _logits(rows, cols, dtype, seed=0, spread=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = spread * torch.randn(rows, cols, device="cuda", generator=g)
    return (15 * torch.tanh(z / 15)).to(dtype)


SHAPES = [(1, 65536, 65536, 20), (3, 1, 1, 1), (2, 2, 8, 2), (5, 7, 7, 3), (4, 33, 64, 32), (64, 65536, 65536, 8), (7, 50257, 50304, 5), (9, 50257, 50257, 32), (130, 8191, 8192, 1),
          (300, 1000, 1000, 0), (2, 200000, 200064, 4), (150, 65536, 65600, 16), (1, 511, 512, 32), (2000, 513, 520, 2)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab,cols,topk", SHAPES)
def test_forward(rows, vocab, cols, topk, dtype):
    from them_bones_b200 import ops
    z = _logits(rows, cols, dtype, seed=rows)
    z[:, vocab:] = 100.0                                               # behind the vocabulary: never looked at
    tokens = torch.randint(-1, vocab, (rows,), device="cuda")
    tokens[0] = vocab - 1
    r = ops.token_logprobs(z, tokens, topk, vocab)
    given, h, top, ids, _, _, _ = _exact(z, tokens, topk, vocab)
    assert torch.equal(r.top_id, ids) and r.top_id.dtype == torch.int64
    # z - max is exact to a rounding of 30 at most; sums of up to 2^18 terms in parts of 2^9 and their logarithm: 2^9 + 2^9 roundings of relative size 2^-24
    tol = 30 * 2 ** -24 * 2 + 2 ** 10 * 2 ** -24
    for got, want in ((r.logprob, given), (r.entropy, h), (r.top_logprob, top)):
        assert got.dtype == torch.float32 and float((got.double() - want).abs().max() if got.numel() else 0) <= tol
    assert not r.logprob[tokens < 0].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab,cols,topk", SHAPES)
@pytest.mark.parametrize("which", ["all", "given", "entropy", "top"])
def test_backward(rows, vocab, cols, topk, dtype, which):
    from them_bones_b200 import ops
    if which == "top" and not topk:
        pytest.skip("no alternatives")
    z = _logits(rows, cols, dtype, seed=rows).requires_grad_()
    tokens = torch.randint(-1, vocab, (rows,), device="cuda")
    r = ops.token_logprobs(z, tokens, topk, vocab)
    if topk:
        tokens[::2] = r.top_id[::2, -1]                                # the given token among the alternatives
        r = ops.token_logprobs(z, tokens, topk, vocab)
    g = torch.Generator(device="cuda").manual_seed(5)
    gs = [torch.randn(rows, device="cuda", generator=g), torch.randn(rows, device="cuda", generator=g), torch.randn(rows, topk, device="cuda", generator=g)]
    use = {"all": [0, 1] + ([2] if topk else []), "given": [0], "entropy": [1], "top": [2]}[which]
    d, = torch.autograd.grad([r[i] for i in use], [z], [gs[i] for i in use])
    want, p = _exact_grad(z, tokens, topk, vocab, [gs[i] if i in use else None for i in range(3)])
    assert d.dtype == dtype and d.shape == z.shape and not d[:, vocab:].any()
    # half a step of the type, and fp32 factors: each term is a product of p (relative error 2^-24 * (30 + 2^10)) and sums of up to 34 numbers
    pull = sum(gs[i].abs().double().reshape(rows, -1).sum(1) * (30.0 if i == 1 else 1.0) for i in use)[:, None]
    fp32 = 2 ** -12 * pull * torch.nn.functional.pad(p, (0, cols - vocab)) + 2 ** -20 * pull
    assert bool(((d.double() - want).abs() <= torch.finfo(dtype).eps / 2 * want.abs() + fp32).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(2, 65536), (200, 65536), (5, 999), (3, 131072)])
@pytest.mark.parametrize("what", ["equal", "ascending", "descending", "few", "blocks", "infinite"])
def test_order_of_alternatives(rows, vocab, what, dtype):
    """Rows on which a selection by parts has to keep more than it usually does."""
    from them_bones_b200 import ops
    i = torch.arange(vocab, device="cuda", dtype=torch.float32)
    row = {"equal": torch.full_like(i, 2.5), "ascending": i / vocab, "descending": -i / vocab, "few": (i % 3 == 1).float(), "blocks": (i // 1000) % 7,
           "infinite": torch.where(i % 5 == 0, float("-inf"), -(i % 1024) / 1024)}[what]
    z = row.to(dtype).expand(rows, vocab).contiguous()
    z[-1] = z[-1].flip(0)
    tokens = torch.full((rows,), 1, device="cuda")
    r = ops.token_logprobs(z, tokens, 32, vocab)
    given, h, top, ids, _, _, _ = _exact(z, tokens, 32, vocab)
    assert torch.equal(r.top_id, ids)
    tol = 2 ** 10 * 2 ** -24 + 2 ** -20
    for got, want in ((r.logprob, given), (r.entropy, h), (r.top_logprob, top)):
        same = got.double() == want                                    # infinities
        assert bool((same | ((got.double() - want).abs() <= tol)).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [5, 3000, 65536])
def test_rows_without_a_number(vocab, dtype):
    from them_bones_b200 import ops
    inf, nan = float("inf"), float("nan")
    z = _logits(8, vocab, dtype)
    z[0, 3] = nan
    z[1, 4] = inf
    z[2] = -inf
    z[3] = nan
    z[4, 1] = inf
    z[4, 2] = nan
    z[5, :] = -inf
    z[5, 2] = 1.0
    z[6, 0] = 3e38
    z[6, 1] = -3e38
    z.requires_grad_()
    tokens = torch.tensor([0, 4, 1, 2, 1, 2, 0, 1], device="cuda")
    k = min(vocab, 6)
    r = ops.token_logprobs(z, tokens, k)
    w = ops._logprobs.statement(z, tokens, k, vocab)
    assert torch.equal(r.top_id, w.top_id)
    for a, b in ((r.logprob, w.logprob), (r.entropy, w.entropy), (r.top_logprob, w.top_logprob)):
        assert bool(a[:5].isnan().all()) and bool(b[:5].isnan().all()) and not a[5:].isnan().any()
        assert torch.equal(a.isinf(), b.isinf()) and torch.allclose(a[5:].nan_to_num(), b[5:].nan_to_num(), rtol=2e-6, atol=2e-5)
    assert not r.entropy[5:7].any() and not r.logprob[5].any()
    d, = torch.autograd.grad(r.logprob.nansum() + r.entropy.nansum(), [z])
    assert bool(d[5:].isfinite().all())
    keep = torch.tensor([0, 0, 0, 0, 0, 1, 1, 1.0], device="cuda")
    r = ops.token_logprobs(z, tokens)
    d, = torch.autograd.grad([r.logprob, r.entropy], [z], [keep, keep])
    assert bool(d.isfinite().all()) and not d[:5].any()                # rows that nothing depends on


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 300])
def test_columns_masked_with_the_lowest_number(rows, dtype):
    """Masks of -inf and of the type's lowest value hide columns alike; rows of nothing but the lowest value are uniform."""
    from them_bones_b200 import ops
    low = torch.finfo(dtype).min
    z = _logits(rows, 20000, dtype, seed=2)
    keep = torch.rand(20000, device="cuda") < 0.3
    tokens = torch.full((rows,), int(keep.nonzero()[7]), device="cuda")
    a, b = (ops.token_logprobs(torch.where(keep, z, torch.full((), m, dtype=dtype, device="cuda")), tokens, 32) for m in (float("-inf"), low))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    few = torch.full((rows, 20000), float("-inf"), dtype=dtype, device="cuda")
    few[:, 17000:17040] = low                                          # 40 of them behind nothing, in one thread's reach or in many
    r = ops.token_logprobs(few, torch.full((rows,), 17003, device="cuda"), 32)
    assert torch.equal(r.top_id, torch.arange(17000, 17032, device="cuda").expand(rows, 32))
    assert float((r.entropy - 3.6888795).abs().max()) < 1e-5 and float((r.logprob + 3.6888795).abs().max()) < 1e-5


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 300])
@pytest.mark.parametrize("mask", [-1e4, -1e7, -2e7, -9e7, -2e8, -1e9, -1e10, -1e20, -1e30, -3e38])
def test_masks_of_any_depth(mask, rows, dtype):
    """Threads that find nothing but masked columns for a while, and then others."""
    from them_bones_b200 import ops
    z = _logits(rows, 65536, dtype, seed=4)
    z[:, :40000] = mask
    z[:, 50000:65000] = mask
    tokens = torch.full((rows,), 41000, device="cuda")
    r = ops.token_logprobs(z, tokens, 5)
    given, h, top, ids, _, _, _ = _exact(z, tokens, 5, 65536)
    assert torch.equal(r.top_id, ids)
    tol = 30 * 2 ** -24 * 2 + 2 ** 10 * 2 ** -24                           # as in `test_forward`
    for got, want in ((r.logprob, given), (r.entropy, h), (r.top_logprob, top)):
        assert float((got.double() - want).abs().max()) <= tol


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 300])
@pytest.mark.parametrize("size", [1e3, 3e6, 1.1e7, 1e8, 1e9, 1e12, 1e25, 1e30, 3e37, -1e3, -3e6, -1.1e7, -1e9, -1e12, -1e30, -3e37])
def test_logits_of_any_size(size, rows, dtype):
    """Rows around a large number: what counts is the distance from the largest, whatever it is."""
    from them_bones_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(1)
    step = 2.0 ** (torch.tensor(abs(size), dtype=torch.float64).log2().floor() - (7 if dtype == torch.bfloat16 else 23))       # of the type there
    k = torch.randint(0, 9, (rows, 20000), device="cuda", generator=g)
    z = (size - step * k).to(dtype)
    assert torch.equal(z.double(), (size - step * k).to(dtype).double())
    tokens = torch.randint(0, 20000, (rows,), device="cuda", generator=g)
    x = z.clone().requires_grad_()
    r = ops.token_logprobs(x, tokens, 5)
    given, h, top, ids, _, _, _ = _exact(z, tokens, 5, 20000)
    assert torch.equal(r.top_id, ids)
    tol = 2 ** 10 * 2 ** -24 + 2 ** -18                                     # sums as in `test_forward`; distances are exact, and beyond 20 their exponentials count for nothing
    for got, want in ((r.logprob, given), (r.entropy, h), (r.top_logprob, top)):
        got, want = got.detach().double(), want
        assert bool(((got - want).abs() <= tol + 2 ** -22 * want.abs()).all()), float((got - want).abs().max())
    d, = torch.autograd.grad(r.logprob.sum() + r.entropy.sum(), [x])
    want, p = _exact_grad(z, tokens, 0, 20000, [torch.ones(rows, device="cuda"), torch.ones(rows, device="cuda"), None])
    assert bool(d.isfinite().all()) and bool(((d.double() - want).abs() <= torch.finfo(dtype).eps / 2 * want.abs() + 2 ** -12 * 31 * p + 2 ** -20).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_that_lie_anywhere(dtype):
    from them_bones_b200 import ops
    big = _logits(12, 2011, dtype)
    for view in (big[:, 1:], big[::3, 2:1003], big[1:2], big[:, ::2], big.T[:100], big[:1].expand(6, -1), big.view(3, 4, -1)[:, 1:3, 5:]):
        leaf = view.detach().clone().requires_grad_()
        x = view.detach().requires_grad_()
        tokens = torch.randint(0, 11, view.shape[:-1], device="cuda", dtype=torch.int32)
        a, b = (ops.token_logprobs(t, tokens, 4, view.shape[-1] - 1 if view.shape[-1] > 12 else None) for t in (x, leaf))
        assert torch.equal(a.top_id, b.top_id) and a.logprob.shape == view.shape[:-1]
        # the row's parts begin at its first 16-byte boundary, so two alignments add in two orders: each is within the bound of `test_forward`
        # of the exact value, 30 * 2^-23 + 2^-14, and they are within twice that of one another
        tol = 2 * (30 * 2 ** -23 + 2 ** -14)
        assert all(float((p - q).detach().abs().max()) <= tol for p, q in zip(a[:3], b[:3]))
        da, db = (torch.autograd.grad(r.logprob.sum() + 0.5 * r.entropy.sum() + r.top_logprob[..., 1].sum(), [t])[0] for r, t in ((a, x), (b, leaf)))
        # a probability is off by `tol` of itself (at most 1), times the sum of 1 + 1 + 0.5 * (1 + 30) for the three gradients; one step of the type
        assert bool(((da.double() - db.double()).abs() <= torch.finfo(dtype).eps * db.double().abs() + tol * 18).all())


def test_none_and_one():
    from them_bones_b200 import ops
    z = _logits(4, 100, torch.float32).view(2, 2, 100)
    r = ops.token_logprobs(z[:0], torch.zeros(0, 2, dtype=torch.int64, device="cuda"), 3)
    assert r.logprob.shape == (0, 2) and r.top_id.shape == (0, 2, 3)
    r = ops.token_logprobs(z[0, 0], torch.tensor(5, device="cuda"), 3)
    assert r.logprob.shape == () and r.top_id.shape == (3,)
    x = z[:0].clone().requires_grad_()
    d, = torch.autograd.grad(ops.token_logprobs(x, torch.zeros(0, 2, dtype=torch.int64, device="cuda"), 3).entropy.sum(), [x])
    assert d.shape == x.shape


def test_tokens_outside_the_vocabulary():
    from them_bones_b200 import ops
    z = _logits(5, 64, torch.bfloat16).requires_grad_()
    tokens = torch.tensor([-1, 50, 49, 1 << 40, -(1 << 40)], device="cuda")
    r = ops.token_logprobs(z, tokens, 0, 50)
    assert r.logprob[[0, 1, 3, 4]].eq(0).all() and float(r.logprob[2].detach()) < 0
    d, = torch.autograd.grad(r.logprob.sum(), [z])
    assert not d[[0, 1, 3, 4]].any() and d[2, :50].any() and not d[:, 50:].any()


def test_batched_and_recorded_gradients():
    from them_bones_b200 import ops
    z = _logits(6, 40, torch.float32).requires_grad_()
    tokens = torch.tensor([0, 5, -1, 39, 2, 2], device="cuda")
    r = ops.token_logprobs(z, tokens, 3)
    rows = torch.eye(6, device="cuda")
    batched, = torch.autograd.grad(r.logprob, [z], rows, is_grads_batched=True, retain_graph=True)
    single = torch.stack([torch.autograd.grad(r.logprob, [z], e, retain_graph=True)[0] for e in rows])
    assert torch.allclose(batched, single, rtol=1e-5, atol=1e-6)

    def f(x):
        q = ops.token_logprobs(x, tokens, 3)
        return q.logprob.sum() + q.entropy.square().sum() + q.top_logprob[:, 1].sum()
    d, = torch.autograd.grad(f(z), [z], create_graph=True)
    plain, = torch.autograd.grad(f(z), [z])
    assert torch.allclose(d, plain, rtol=1e-5, atol=1e-6)
    dd, = torch.autograd.grad(d.square().sum(), [z])
    y = z.detach().double().requires_grad_()

    def f64(x):
        logp = torch.log_softmax(x, -1)
        ids = r.top_id[:, 1:2]
        g = torch.where(tokens >= 0, logp.gather(1, tokens.clamp_min(0)[:, None])[:, 0], torch.zeros((), dtype=torch.float64, device="cuda"))
        return g.sum() + (-(logp.exp() * logp).sum(-1)).square().sum() + logp.gather(1, ids).sum()
    e, = torch.autograd.grad(f64(y), [y], create_graph=True)
    ee, = torch.autograd.grad(e.square().sum(), [y])
    assert float((dd.double() - ee).norm() / ee.norm()) < 1e-4


@pytest.mark.parametrize("topk", [0, 3])
def test_captured_with_its_gradient(topk):
    from them_bones_b200 import ops
    torch.manual_seed(1)
    z = _logits(70, 3001, torch.bfloat16)
    x = z.clone().requires_grad_()
    tokens = torch.randint(0, 3001, (70,), device="cuda")
    g = torch.randn(70, device="cuda")

    def step(t):
        r = ops.token_logprobs(t, tokens, topk)
        return r, torch.autograd.grad([r.logprob, r.entropy], [t], [g, g])[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(x)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r, d = step(x)
    for seed in (3, 4):
        new = _logits(70, 3001, torch.bfloat16, seed=seed)
        with torch.no_grad():
            x.copy_(new)
        graph.replay()
        w, dw = step(new.clone().requires_grad_())
        assert all(torch.equal(a, b) for a, b in zip(r, w)) and torch.equal(d, dw)


def test_offsets_past_32_bits():
    from them_bones_b200 import ops
    rows, cols = 33000, 65600
    z = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    assert z.numel() > 1 << 31
    z[-1, :65536] = _logits(1, 65536, torch.bfloat16)[0]
    z.requires_grad_()
    tokens = torch.full((rows,), 7, device="cuda")
    r = ops.token_logprobs(z, tokens, 2, 65536)
    one = z.detach()[-1:].clone().requires_grad_()
    w = ops.token_logprobs(one, tokens[:1], 2, 65536)
    for a, b in zip(r, w):
        assert torch.allclose(a[-1:].double(), b.double(), rtol=1e-6, atol=1e-5)
    assert r.top_id[:-1].eq(torch.tensor([0, 1], device="cuda")).all()
    d, = torch.autograd.grad(r.logprob.sum(), [z])
    dw, = torch.autograd.grad(w.logprob.sum(), [one])
    assert torch.allclose(d[-1:].float(), dw.float(), rtol=2 ** -7, atol=1e-9) and not d[:, 65536:].any()
    assert float(d[123, 7]) == pytest.approx(1 - 2 ** -16, rel=2 ** -7) and float(d[123, 8]) == pytest.approx(-2 ** -16, rel=2 ** -7)


def test_native_refusals():
    from them_bones_b200 import ops
    with pytest.raises(ValueError):
        ops.token_logprobs(torch.randn(3, 8, device="cuda").half(), torch.zeros(3, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError):
        ops.token_logprobs(torch.randn(3, 8, device="cuda"), torch.zeros(3, dtype=torch.int64))
