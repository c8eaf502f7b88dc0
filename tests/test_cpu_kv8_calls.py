"""Calls of the 8-bit cache that its documentation allows or excludes and that are easy to get wrong, on the CPU."""
import pytest
import torch
from torch.autograd import forward_ad


def test_a_tangent_is_refused():
    from them_bones_b200 import ops
    c = ops.kv8_cache(1, 64, 1, 64)
    k, qkv, cos = torch.randn(1, 2, 1, 64), torch.randn(1, 192), torch.ones(64, 32)
    for grad in (True, False):
        with torch.set_grad_enabled(grad), forward_ad.dual_level():
            dual = forward_ad.make_dual(k, torch.ones_like(k))
            for args in ((dual, k), (k, dual)):
                with pytest.raises(ValueError):
                    ops.kv8_append(c, *args, 0)
            with pytest.raises(ValueError):
                ops.kv8_attention(forward_ad.make_dual(qkv, torch.ones_like(qkv)), cos, cos, c, 0, 1.0)
            assert not any(x.any() for x in c)
            ops.kv8_append(c, k[:, :0], k[:, :0], 0)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size", [3e17, 1e19, 1e25, 3e37, 1e-12, 1e-30])
@pytest.mark.parametrize("which", ["query", "key", "both"])
def test_norm_of_large_and_small_rows(which, size, d):
    """Rows whose squares leave fp32 are normalised as any others; far below the norm's epsilon they come out as zeros."""
    from tests import kv8_oracle as O
    from them_bones_b200 import ops
    from them_bones_b200.ref import functional as RF
    torch.manual_seed(7)
    b, h, n = 2, 2, 100
    cos, sin = (x.to("cpu") for x in RF.rotary_tables(n + 1, d, 10000.0))
    cache = ops.kv8_cache(b, n + 1, h, d, "cpu")
    k, v = torch.randn(2, b, n, h, d, device="cpu").bfloat16()
    ops.kv8_append(cache, k, v, 0)
    before = [x.clone() for x in cache]
    qkv = torch.randn(b, 3, h, d, device="cpu").clamp(-4, 4)
    if which != "key":
        qkv[:, 0] *= size
    if which != "query":
        qkv[:, 1] *= size
    qkv[1, :2, 0] /= qkv[1, :2, 0].abs().amax(-1, keepdim=True) if size > 1 else 1.0          # a row of the largest there are beside smaller ones
    if size > 1:
        qkv[1, :2, 0] *= 3e38
    qkv = qkv.bfloat16().view(b, -1)
    y = ops.kv8_attention(qkv, cos, sin, cache, n, 0.09).double().view(b, h, d)
    new_k = cache.k_open[:, :, n % 64]
    for i in range(b):
        want = O.new_rows(qkv[i], cos, sin, n, h, d)[1]
        # a rounding to bf16 behind a few of fp32 at most; 2^-133 is half of bf16's smallest step
        assert bool(((new_k[i].double() - want).abs() <= (2 ** -8 + 2 ** -18) * want.abs() + 2.0 ** -133).all())
    want, most = O.attend(qkv, cos, sin, before, new_k, [n] * b, 0.09, None, 0)
    # as in the kernels' own tests: a rounding to bf16, fp32 scores of 0.09 * 16 d at most off by 32 roundings, probabilities of 11 bits
    tol = 2 ** -8 * want.abs() + (2 * 0.09 * 16 * d * 32 * 2 ** -24 + 2 ** -11) * most[:, None, None]
    assert bool(y.isfinite().all()) and bool(((y - want).abs() <= tol).all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_rows_that_are_not_finite(bad):
    """A query with such a value has no result; a key with one has none for who sees it."""
    from them_bones_b200 import ops
    torch.manual_seed(8)
    cos = torch.ones(64, 32, device="cpu")
    for part in (0, 1):
        cache = ops.kv8_cache(2, 64, 2, 64, "cpu")
        qkv = torch.randn(2, 3, 2, 64, device="cpu").bfloat16()
        qkv[1, part, 1, 5] = bad
        y = ops.kv8_attention(qkv.view(2, -1), cos, 0 * cos, cache, 0, 0.1).view(2, 2, 64)
        assert bool(y[0].isfinite().all()) and bool(y[1, 0].isfinite().all()) and bool(y[1, 1].isnan().all())
