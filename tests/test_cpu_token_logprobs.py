"""Log-probabilities of tokens on the CPU: the statement against 64 bits and its refusals."""
import pytest
import torch


def test_against_64_bits_and_differences():
    from them_bones_b200 import ops
    torch.manual_seed(0)
    z = (3 * torch.randn(4, 11, dtype=torch.float64)).requires_grad_()
    tokens = torch.tensor([3, -1, 8, 9])
    g, h, t, i = ops.token_logprobs(z, tokens, 4, 9)
    logp = torch.log_softmax(z.detach()[:, :9], -1)
    want_h = -(logp.exp() * logp).sum(-1)
    # fp32 values of size 12 at most behind sums of 9
    assert float((g.detach().double() - torch.stack([logp[0, 3], logp[1, 0] * 0, logp[2, 8], logp[3, 0] * 0])).abs().max()) < 12 * 2 ** -21
    assert float((h.detach().double() - want_h).abs().max()) < 12 * 2 ** -21
    top = logp.sort(-1, descending=True)
    assert torch.equal(i, top.indices[:, :4]) and float((t.detach().double() - top.values[:, :4]).abs().max()) < 12 * 2 ** -21
    weights = [torch.randn(4), torch.randn(4), torch.randn(4, 4)]
    d, = torch.autograd.grad([g, h, t], [z], weights)
    f = lambda x: (ops.token_logprobs(x, tokens, 4, 9)[0].double() * weights[0]).sum() + (ops.token_logprobs(x, tokens, 4, 9)[1].double() * weights[1]).sum() + (
        ops.token_logprobs(x, tokens, 4, 9)[2].double() * weights[2]).sum()  # noqa: E731
    step = 2 ** -6
    for r, c in ((0, 3), (0, 5), (1, 2), (2, 8), (3, 0), (3, 10)):
        e = torch.zeros_like(z)
        e[r, c] = step
        num = (f(z.detach() + e) - f(z.detach() - e)) / (2 * step)
        # third derivatives of size 20 at most times step^2 / 6, and fp32 differences
        assert abs(float(num - d[r, c])) < 20 * step ** 2 + 40 * 2 ** -22 / step


def test_ties_infinities_and_rows_without_a_number():
    from them_bones_b200 import ops
    inf, nan = float("inf"), float("nan")
    z = torch.tensor([[1.0, 2.0, 2.0, 0.0, 2.0], [-inf, 0.0, -inf, 0.0, -inf], [-inf] * 5, [0.0, nan, 1.0, nan, 2.0], [0.0, inf, 1.0, inf, 2.0], [0.0, -0.0, 0.0, -0.0, -1.0]])
    g, h, t, i = ops.token_logprobs(z, torch.tensor([1, 1, 0, 0, 0, 1]), 5)
    assert i.tolist() == [[1, 2, 4, 0, 3], [1, 3, 0, 2, 4], [0, 1, 2, 3, 4], [1, 3, 4, 2, 0], [1, 3, 4, 2, 0], [0, 1, 2, 3, 4]]
    assert abs(float(h[1]) - 0.6931472) < 1e-6 and float(t[1, 2]) == -inf and abs(float(g[1]) + 0.6931472) < 1e-6
    assert all(bool(x[2:5].isnan().all()) for x in (g, h, t))
    y = z.clone().requires_grad_()
    r = ops.token_logprobs(y, torch.tensor([1, 1, 0, 0, 0, 1]))
    d, = torch.autograd.grad(r.logprob[1] + r.entropy[1], [y])
    assert bool(d[[0, 1, 5]].isfinite().all()) and not d[0].any() and not d[1, [0, 2, 4]].any()
    assert r.top_id.shape == (6, 0) and r.top_logprob.shape == (6, 0)


def test_shapes():
    from them_bones_b200 import ops
    z = torch.randn(2, 3, 10)
    r = ops.token_logprobs(z, torch.zeros(2, 3, dtype=torch.int32), 2, 7)
    assert r.logprob.shape == r.entropy.shape == (2, 3) and r.top_id.shape == r.top_logprob.shape == (2, 3, 2) and int(r.top_id.max()) < 7
    one = ops.token_logprobs(z[0, 0], torch.tensor(1), 3)
    assert one.logprob.shape == () and one.top_id.shape == (3,)
    none = ops.token_logprobs(z[:0], torch.zeros(0, 3, dtype=torch.int64), 2)
    assert none.logprob.shape == (0, 3) and none.top_id.shape == (0, 3, 2)


def test_refusals():
    from them_bones_b200 import ops
    z, t = torch.randn(3, 10), torch.zeros(3, dtype=torch.int64)
    for args in ((z, t[:2]), (z, t.float()), (z.int(), t), (z, t, 11), (z, t, -1), (z, t, 8, 7), (z, t, 0, 0), (z, t, 0, 11), (torch.randn(3, 100), t, 33),
                 (torch.tensor(1.0), torch.tensor(0))):
        with pytest.raises(ValueError):
            ops.token_logprobs(*args)


def test_head_refusals():
    from them_bones_b200 import ops
    x, w, t = torch.randn(3, 16), torch.randn(40, 16), torch.zeros(3, dtype=torch.int64)
    assert ops.lmhead_logprobs(x, w, t, 40, 15.0, 2).top_id.shape == (3, 2)
    for args in ((x, w, t[:2], 40, 15.0), (x, w, t.float(), 40, 15.0), (x[:, :8], w, t, 40, 15.0), (x.int(), w, t, 40, 15.0), (x, w[0], t, 40, 15.0), (x, w, t, 41, 15.0),
                 (x, w, t, 0, 15.0), (x, w, t, 40, 15.0, 33), (x, w, t, 4, 15.0, 5), (x, w, t, 40, 0.0), (x, w, t, 40, -15.0), (x, w, t, 40, float("inf")),
                 (x, w, t, 40, float("nan"))):
        with pytest.raises(ValueError):
            ops.lmhead_logprobs(*args)
