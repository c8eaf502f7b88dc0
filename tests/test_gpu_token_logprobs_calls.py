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
