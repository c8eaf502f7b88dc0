"""The 8-bit cache where offsets pass 31 and 32 bits: codes, read-back, inputs and rotary tables that lie far from their tensors' begin."""
import pytest
import torch

from tests import kv8_oracle as O

pytestmark = pytest.mark.gpu


def _close(y, qkv, cos, sin, at, cache, small, skip, start, h, d, scale=0.1):
    """Attention of one sequence at ``at`` over what ``small`` holds from position ``skip`` on, seen from ``start``."""
    q, _, vn = O.new_rows(qkv, cos, sin, at, h, d)
    ks, vs = O.held(small, 0, at - skip)
    lo = start - skip
    ks = torch.cat([ks, cache[4][:, at % 64].double()[:, None]], 1)[:, lo:]
    vs = torch.cat([vs, vn[:, None]], 1)[:, lo:]
    w = torch.einsum("hn,hnd->hd", torch.softmax(torch.einsum("hd,hnd->hn", q, ks) * scale, -1), vs)
    # a rounding to bf16, probabilities of 11 bits, fp32 scores of 0.1 * 16 d at most off by 32 roundings
    tol = 2 ** -8 * w.abs() + (2 * scale * 16 * d * 32 * 2 ** -24 + 2 ** -11) * vs.abs().max()
    assert bool(((y.double().view(h, d) - w).abs() <= tol).all())


def test_codes_and_read_back_past_31_bits():
    """The third sequence's codes begin at byte 2^31, its rows of the read-back at value 2^31."""
    from them_bones_b200 import ops
    b, h, d, cap, n = 3, 4, 128, 1 << 21, 300
    at = cap - 320                                                    # a multiple of 64: what is put there can be compared with a small cache
    assert (2 * h * cap) * d >= 2 ** 31 and ((2 * cap + at) * h) * d > 2 ** 31 and at % 64 == 0
    torch.manual_seed(13)
    cache, small = ops.kv8_cache(b, cap, h, d, "cuda"), ops.kv8_cache(b, 320, h, d, "cuda")
    k, v = torch.randn(2, b, n, h, d, device="cuda").bfloat16()
    ops.kv8_append(cache, k, v, at)
    ops.kv8_append(small, k, v, 0)
    nb = at // 64
    assert torch.equal(cache.k[:, :, at:], small.k) and torch.equal(cache.v[:, :, nb:], small.v)
    assert torch.equal(cache.k_scale[:, :, nb:], small.k_scale) and torch.equal(cache.v_scale[:, :, nb:], small.v_scale)
    for i in range(b):
        assert not cache.k[i, :, :at].any() and not cache.v[i, :, :nb].any()
    rk, rv = ops.kv8_read(cache, at + n, cap)
    sk, sv = ops.kv8_read(small, n, 320)
    for far, near in ((rk, sk), (rv, sv)):
        assert torch.equal(far[:, at:], near)
        for i in range(b):
            assert not far[i, :at].any()
    del rk, rv, far
    cos, sin = (torch.rand(cap, d // 2, device="cuda") for _ in range(2))
    qkv = torch.randn(b, 3 * h * d, device="cuda").bfloat16()
    start = torch.tensor([at, at + 70, at + 1], dtype=torch.int32, device="cuda")
    y = ops.kv8_attention(qkv, cos, sin, cache, at + n, 0.1, start)
    for i in range(b):
        _close(y[i], qkv[i], cos, sin, at + n, [x[i] for x in cache], [x[i:i + 1] for x in small], at, int(start[i]), h, d)


def test_keys_and_rows_that_lie_far_apart():
    """Two sequences' keys, values and packed rows 2^31 values from one another."""
    from them_bones_b200 import ops
    from them_bones_b200.ref import functional as RF
    b, h, d, n = 2, 2, 64, 130
    torch.manual_seed(14)
    far = torch.empty((1 << 31) + (1 << 20), dtype=torch.bfloat16, device="cuda")
    k, v = torch.randn(2, b, n, h, d, device="cuda").bfloat16()
    qkv = torch.randn(b, 3 * h * d, device="cuda").bfloat16()
    fk, fv = (far.as_strided((b, n, h, d), (1 << 31, h * d, d, 1), o) for o in (0, 1 << 18))
    fq = far.as_strided((b, 3 * h * d), (1 << 31, 1), 1 << 19)
    for x, y in ((fk, k), (fv, v), (fq, qkv)):
        x.copy_(y)
    cos, sin = (x.cuda() for x in RF.rotary_tables(n + 1, d, 10000.0))
    got, want = (ops.kv8_cache(b, n + 1, h, d, "cuda") for _ in range(2))
    ops.kv8_append(got, fk, fv, 0)
    ops.kv8_append(want, k, v, 0)
    a, c = ops.kv8_attention(fq, cos, sin, got, n, 0.1), ops.kv8_attention(qkv, cos, sin, want, n, 0.1)
    assert torch.equal(a, c) and all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("shared", [True, False])
def test_a_position_past_2_to_the_25(shared, monkeypatch):
    """Codes past 2^32 bytes and rotary rows past 2^31 values of one sequence, by the form that shares long caches and by clusters."""
    from them_bones_b200 import ops
    h, d, n = 1, 128, 200
    at = 1 << 25
    cap = at + 256
    assert at * d >= 2 ** 32 and at * (d // 2) >= 2 ** 31
    if not shared:
        monkeypatch.setattr(ops._kv8, "LONG", 1 << 40)
    torch.manual_seed(15)
    cache, small = ops.kv8_cache(1, cap, h, d, "cuda"), ops.kv8_cache(1, 256, h, d, "cuda")
    k, v = torch.randn(2, 1, n, h, d, device="cuda").bfloat16()
    ops.kv8_append(cache, k, v, at)
    ops.kv8_append(small, k, v, 0)
    assert torch.equal(cache.k[:, :, at:], small.k) and torch.equal(cache.v[:, :, at // 64:], small.v)
    cos, sin = (torch.zeros(cap, d // 2, device="cuda") for _ in range(2))
    cos[at + n], sin[at + n] = torch.rand(2, d // 2, device="cuda")
    qkv = torch.randn(1, 3 * h * d, device="cuda").bfloat16()
    for start in (at, at + 63, at + 190):
        ds = torch.tensor([start], dtype=torch.int32, device="cuda")
        y = ops.kv8_attention(qkv, cos, sin, cache, at + n, 0.1, ds)
        _close(y[0], qkv[0], cos, sin, at + n, [x[0] for x in cache], small, at, start, h, d)
