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
