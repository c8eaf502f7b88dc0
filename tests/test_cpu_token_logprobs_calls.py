"""The native log-probabilities' way through autograd, on the CPU: the kernels' entries are stood in for by the statement."""
import pytest
import torch
from torch.autograd import forward_ad


@pytest.fixture
def native(monkeypatch):
    """``ops.token_logprobs`` by the native body whose forward kernel is the statement."""
    from them_bones_b200 import ops
    from them_bones_b200.ref import functional as RF

    def forward(z, tokens, topk, vocab, want_stats):
        given, h, top, ids = RF.token_logprobs(z.detach(), tokens, topk, vocab)
        return given, h, top, ids, torch.zeros(z.shape[0], 4)

    def no_kernel(*args):
        raise AssertionError("the gradient's kernel was to run")
    monkeypatch.setattr(ops._logprobs, "_forward", forward)
    monkeypatch.setattr(ops._logprobs, "_backward", no_kernel)
    return lambda z, tokens, topk=0: ops._logprobs.native(z, tokens, topk, z.shape[-1])


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("shape", [(3,), (2, 3)])
def test_a_tangent_is_not_dropped(native, grad, shape):
    z, tokens = torch.randn(*shape, 7), torch.zeros(shape, dtype=torch.int64)
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            native(forward_ad.make_dual(z, torch.ones_like(z)), tokens, 2)
        assert not native(z, tokens, 2).logprob.requires_grad          # another tensor's level does not matter


def test_a_tangent_of_the_gradient_is_not_dropped(native):
    """Differentiation forward through the backward pass: the gradient is linear in what comes from above."""
    torch.manual_seed(0)
    z, tokens = torch.randn(3, 7, requires_grad=True), torch.tensor([1, -1, 6])
    r = native(z, tokens, 2)
    g, t = torch.randn(2, 3)
    with forward_ad.dual_level():
        d, = torch.autograd.grad(r.logprob, [z], forward_ad.make_dual(g, t), retain_graph=True)
        tangent = forward_ad.unpack_dual(d).tangent
    want, = torch.autograd.grad(r.logprob, [z], t, create_graph=True)
    # products and sums of three numbers of size 5 at most in fp32
    assert tangent is not None and float((tangent - want).detach().abs().max()) < 15 * 2 ** -22


def _rows_of_all_kinds():
    """Seven rows, the first five without a number, and their tokens."""
    inf, nan = float("inf"), float("nan")
    torch.manual_seed(2)
    z = torch.randn(7, 9)
    z[0, 3], z[1, 4], z[2], z[3], z[4, 1], z[4, 2] = nan, inf, -inf, nan, inf, nan
    z[5, :4] = -inf
    return z, torch.tensor([0, 4, 1, -1, 1, 5, 2])


@pytest.mark.parametrize("route", ["statement", "native"])
@pytest.mark.parametrize("how", ["recorded", "batched", "plain", "tokens"])
def test_rows_without_a_number_that_nothing_depends_on(route, how, native):
    """Zeros for them however the gradient is taken, NaN where something does depend on them, and the others' gradients untouched."""
    from them_bones_b200 import ops
    z, tokens = _rows_of_all_kinds()
    z.requires_grad_()
    f = native if route == "native" else lambda a, t, k=0: ops._logprobs.statement(a, t, k, a.shape[-1])
    r = f(z, tokens, 2)
    if how == "plain" and route == "native":
        pytest.skip("the kernel's")
    outs = [r.logprob, r.entropy, r.top_logprob]
    keep = torch.tensor([0, 0, 0, 0, 0, 1.0, 2.0])
    gs = [keep, -keep, torch.stack([keep, 3 * keep], 1)]
    alone, = torch.autograd.grad(list(f(z[5:], tokens[5:], 2)[:3]), [z], [g[5:] for g in gs], create_graph=True)
    alone = alone.detach()
    if how == "recorded":
        d, = torch.autograd.grad(outs, [z], gs, create_graph=True)
        second, = torch.autograd.grad(d[5:].square().sum(), [z], retain_graph=True)
        assert bool(second[5:].isfinite().all()) and second[6].any()
    elif how == "batched":
        d = torch.autograd.grad(outs, [z], [torch.stack([g, 0 * g]) for g in gs], is_grads_batched=True)[0]
        assert not d[1].any()
        d = d[0]
    elif how == "tokens":                                           # row 3 has no token: what comes from above its log-probability counts for nothing
        g = keep.clone()
        g[3] = 1
        d, = torch.autograd.grad([r.logprob], [z], [g], create_graph=True)
        alone, = torch.autograd.grad([f(z[5:], tokens[5:], 2).logprob], [z], [g[5:]], create_graph=True)
    else:
        d, = torch.autograd.grad(outs, [z], gs)
    d = d.detach()
    assert not d[:5].any() and not d[:5].isnan().any()
    assert float((d[5:] - alone[5:]).detach().abs().max()) < 2 ** -20          # sums of a few numbers of size 3 in another order
    gs = [x.clone() for x in (torch.zeros(7), keep, gs[2])]
    gs[1][1] = 1.0
    d, = torch.autograd.grad([x for x in f(z, tokens, 2)[:3]], [z], gs, create_graph=True)
    assert bool(d[1].isnan().any()) and not d[[0, 2, 3, 4]].detach().any() and bool(d[5:].isfinite().all())


def test_rows_without_a_number_in_the_head(monkeypatch):
    """The head's recorded gradient: a row of the input that nothing depends on leaves its own gradient at zero."""
    from them_bones_b200 import ops
    torch.manual_seed(1)
    x, w, tokens = torch.randn(4, 8), torch.randn(16, 8, requires_grad=True), torch.tensor([1, 2, -1, 3])
    x[0, 2], x[2, 1] = float("nan"), float("nan")
    x.requires_grad_()

    class Ctx:
        needs_input_grad, vocab, cap, main_grad = (True, True), 12, 15.0, None
        saved_tensors = (x, w, tokens, torch.tensor([[1], [2], [0], [3]]), torch.zeros(4, 4))
    with torch.enable_grad():
        dx, _ = ops._logprobs._HeadLogprobsFn.backward(Ctx, torch.tensor([0, 1.0, 1.0, 1.0]), torch.tensor([0, 1.0, 0, 0.0]), None, None)[:2]
    assert not dx[[0, 2]].detach().any() and bool(dx[[1, 3]].isfinite().all()) and dx[1].detach().any()


@pytest.mark.parametrize("mode", ["func.grad", "vmap", "jvp"])
def test_function_transforms_of_the_statement(mode):
    from them_bones_b200 import ops
    z, tokens = _rows_of_all_kinds()
    f = lambda a: ops.token_logprobs(a, tokens, 2).logprob[5:].sum()  # noqa: E731
    y = z.clone().requires_grad_()
    want, = torch.autograd.grad(f(y), [y])
    if mode == "func.grad":
        got = torch.func.grad(f)(z)
    elif mode == "vmap":
        one = lambda a, t: ops.token_logprobs(a, t, 2).logprob  # noqa: E731
        got = torch.cat([torch.zeros(5, 9), torch.func.vmap(torch.func.grad(one))(z[5:], tokens[5:])])
    else:
        t = torch.randn(7, 9)
        got = torch.func.jvp(f, (z,), (t,))[1]
        want = (want * t)[5:].sum()
    assert float((got - want).abs().max()) < 2 ** -18 and not want.isnan().any()
