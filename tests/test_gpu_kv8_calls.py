"""Calls of the 8-bit cache that its documentation allows and that are easy to get wrong: foreign strides, large values, roundings, far offsets."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _same(a, b):
    return all(torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8)) for x, y in zip(a, b))


def _lone(form, h, d):
    """One token of one sequence (or of one head) whose distances are no multiples of eight values where nothing lies at that distance."""
    x = torch.randn(4, 5, 3 * h * d + 1, device="cuda").bfloat16()
    if form == "odd rows":
        return x.as_strided((1, 1, h, d), (x.stride(0), x.stride(1), d, 1))
    if form == "contiguous":
        return x[:3, 0, :h * d].contiguous().view(3, h, d, 1).permute(0, 3, 1, 2)
    if form == "one head":
        return x[:1, :1, None, :d]
    return x[0, 0, :h * d].view(h, d).as_strided((1, 1, h, d), (3, 1, d, 1))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("form", ["odd rows", "contiguous", "one head", "any"])
@pytest.mark.parametrize("pos", [0, 63])
def test_append_of_one_token_with_any_distance(form, d, pos):
    from them_bones_b200 import ops
    torch.manual_seed(1)
    k, v = _lone(form, 2, d), _lone(form, 2, d)
    b, _, h, _ = k.shape
    assert k.stride(1) % 8
    got, want = (ops.kv8_cache(b, 128, h, d, "cuda") for _ in range(2))
    for c in (got, want):
        c.k_open[:, :, :pos] = 0.5
        c.v_open[:, :, :pos] = -0.25
    ops.kv8_append(got, k, v, pos)
    ops.kv8_append(want, *(torch.empty(b, 1, h, d, device="cuda", dtype=torch.bfloat16).copy_(x) for x in (k, v)), pos)
    assert _same(got, want)
    if pos == 0:
        assert torch.equal(got.k_open[:, :, 0], k[:, 0]) and torch.equal(got.v_open[:, :, 0], v[:, 0])
    else:
        assert bool((got.k_scale[:, :, 0] > 0).all()) and got.k[:, :, 63].any() and got.v[:, :, 0, :, 63].any()
