"""Calls of the log-probabilities that go around the kernels' plain way: forward-mode differentiation, recorded and batched gradients."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("grad", [True, False])
def test_a_tangent_is_not_dropped(grad):
    from them_bones_b200 import ops
    z, tokens = torch.randn(3, 64, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    x, w = torch.randn(3, 64, device="cuda").bfloat16(), torch.randn(128, 64, device="cuda").bfloat16()
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            ops.token_logprobs(forward_ad.make_dual(z, torch.ones_like(z)), tokens, 2)
        for args in ((forward_ad.make_dual(x, torch.ones_like(x)), w), (x, forward_ad.make_dual(w, torch.ones_like(w)))):
            with pytest.raises(NotImplementedError):
                ops.lmhead_logprobs(*args, tokens, 128, 15.0)


def test_a_tangent_of_the_gradient():
    from them_bones_b200 import ops
    torch.manual_seed(0)
    z, tokens = torch.randn(3, 64, device="cuda", requires_grad=True), torch.tensor([1, -1, 6], device="cuda")
    r = ops.token_logprobs(z, tokens, 2)
    g, t = torch.randn(2, 3, device="cuda")
    with forward_ad.dual_level():
        d, = torch.autograd.grad(r.logprob, [z], forward_ad.make_dual(g, t), retain_graph=True)
        tangent = forward_ad.unpack_dual(d).tangent
    want, = torch.autograd.grad(r.logprob, [z], t)
    # the gradient is linear in what comes from above: p of it, p off by a few roundings of exponents up to 30
    assert float((tangent - want).abs().max()) < float(t.abs().max()) * 30 * 2 ** -22


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("how", ["plain", "recorded", "batched", "plain operators"])
def test_rows_without_a_number_that_nothing_depends_on(how, dtype):
    """Zeros for them however the gradient is taken, and NaN for one that something depends on."""
    from them_bones_b200 import ops
    inf, nan = float("inf"), float("nan")
    torch.manual_seed(2)
    z = torch.randn(7, 520, device="cuda").to(dtype)
    z[0, 3], z[1, 4], z[2], z[3], z[4, 1], z[4, 2] = nan, inf, -inf, nan, inf, nan
    z[5, :300] = -inf
    z.requires_grad_()
    tokens = torch.tensor([0, 4, 1, -1, 1, 505, 2], device="cuda")
    keep = torch.tensor([0, 0, 0, 0, 0, 1.0, 2.0], device="cuda")
    gs = [keep, -keep, torch.stack([keep, 3 * keep], 1)]
    gs[0] = keep.clone()
    gs[0][3] = 1.0                                                  # row 3 has no token: this counts for nothing
    ops.set_reference_path(how == "plain operators")
    try:
        r = ops.token_logprobs(z, tokens, 2, 515)
        outs = [r.logprob, r.entropy, r.top_logprob]
        if how == "batched":
            d = torch.autograd.grad(outs, [z], [torch.stack([0 * g, g]) for g in gs], is_grads_batched=True, retain_graph=True)[0][1]
        else:
            d, = torch.autograd.grad(outs, [z], gs, create_graph=how == "recorded", retain_graph=True)
        gs[1] = gs[1].clone()
        gs[1][2] = 1.0
        e, = torch.autograd.grad(outs, [z], gs, create_graph=how != "plain")
    finally:
        ops.set_reference_path(False)
    d, e = d.detach(), e.detach()
    want, = torch.autograd.grad(ops.token_logprobs(z, tokens, 2, 515)[:3], [z], [gs[0], -keep, gs[2]])
    assert not d[:5].any() and not d[:5].isnan().any() and not d[:, 515:].any()
    # fp32 products and sums of numbers of size 20 at most, and a rounding to the type that may fall the other way
    assert bool(((d - want)[5:].float().abs() <= torch.finfo(dtype).eps * want[5:].float().abs() + 20 * 2 ** -18).all())
    assert bool(e[2, :515].isnan().all()) and not e[[0, 1, 3, 4]].any() and bool(e[5:].isfinite().all())


@pytest.mark.parametrize("form", ["turned", "odd rows", "odd address"])
def test_a_head_that_owns_its_gradient_and_lies_anywhere(form):
    """The kernels take a copy of such a weight; its gradient goes where the weight's owner wants it all the same."""
    from them_bones_b200 import ops
    torch.manual_seed(0)
    x, flat = torch.randn(40, 64, device="cuda").bfloat16(), (0.3 * torch.randn(256 * 64 + 256, device="cuda")).bfloat16()
    w = {"turned": lambda: flat[:256 * 64].view(64, 256).T, "odd rows": lambda: flat[:256 * 65].view(256, 65)[:, :64], "odd address": lambda: flat[3:256 * 64 + 3].view(256, 64)}[form]()
    tokens = torch.randint(0, 250, (40,), device="cuda")
    own, plain = w.detach().requires_grad_(), w.detach().clone(memory_format=torch.contiguous_format).requires_grad_()
    own.main_grad = torch.ones(256, 64, device="cuda")
    a, b = (ops.lmhead_logprobs(x, t, tokens, 250, 15.0) for t in (own, plain))
    assert torch.equal(a.logprob, b.logprob)
    a.logprob.sum().backward()
    b.logprob.sum().backward()
    # one is fp32, the other rounded to bf16
    assert own.grad is None and float((own.main_grad - 1 - plain.grad.float()).norm()) < 2 ** -7 * float(plain.grad.float().norm())
