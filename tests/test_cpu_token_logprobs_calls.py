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
