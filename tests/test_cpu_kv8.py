"""The 8-bit key/value cache on the CPU: what it holds, its attention, its refusals."""
import pytest
import torch

from tests import kv8_oracle as O


def _fill(cache, k, v, pieces):
    from them_bones_b200 import ops
    at = 0
    for n in pieces:
        ops.kv8_append(cache, k[:, at:at + n], v[:, at:at + n], at)
        at += n
    return cache


@pytest.mark.parametrize("pieces", [[200], [1] * 200, [63, 1, 64, 65, 7], [10, 100, 90], [64, 128, 8], [199, 1]])
def test_the_pieces_leave_no_trace(pieces):
    from them_bones_b200 import ops
    torch.manual_seed(0)
    k, v = torch.randn(2, 2, 200, 3, 64).bfloat16()
    whole, parts = (_fill(ops.kv8_cache(2, 200, 3, 64), k, v, p) for p in ([200], pieces))
    for x, y in zip(whole[:4], parts[:4]):
        assert torch.equal(x, y)
    for x, y in zip(ops.kv8_read(whole, 200, 200), ops.kv8_read(parts, 200, 200)):
        assert torch.equal(x, y)


def test_codes_are_half_a_step_off_at_most():
    from them_bones_b200 import ops
    torch.manual_seed(1)
    k, v = torch.randn(2, 1, 130, 2, 128).bfloat16()
    c = _fill(ops.kv8_cache(1, 130, 2, 128), k, v, [130])
    for x, y, s in zip((k, v), ops.kv8_read(c, 130, 140), c[2:4]):
        assert y.shape[1] == 140 and not y[:, 130:].any() and torch.equal(y[:, 128:130], x[:, 128:])
        scale = s[0, :, :2].repeat_interleave(64, 1).T[None, :, :, None].double()
        off = (y[:, :128].double() - x[:, :128].double()).abs()
        # half a step of the codes, the rounding of x * (127 / most) (three fp32 roundings of a number up to 127) and bf16's of what is read
        assert bool((off <= scale * (0.5 + 127 * 3 * 2 ** -24) + 2 ** -8 * y[:, :128].double().abs()).all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_values_that_are_not_finite(bad):
    from them_bones_b200 import ops
    torch.manual_seed(2)
    k = torch.randn(1, 128, 2, 64).bfloat16()
    want = _fill(ops.kv8_cache(1, 128, 2, 64), k, k, [128])
    x = k.clone()
    i = int(k[0, :64, 1].float().abs().amin(1).argmin())               # a small value: the block's largest one stays
    j = int(k[0, i, 1].float().abs().argmin())
    x[0, i, 1, j] = bad
    got = _fill(ops.kv8_cache(1, 128, 2, 64), x, x, [128])
    for a, b in zip(ops.kv8_read(got, 128, 128), ops.kv8_read(want, 128, 128)):
        assert a[0, i, 1, j].isnan() and int(a.isnan().sum()) == 1
        a[0, i, 1, j] = b[0, i, 1, j]
        assert torch.equal(a, b)
    assert bool(got.k_scale.signbit()[0, 1, 0]) and int(got.k_scale.signbit().sum()) == 1


@pytest.mark.parametrize("value", [0.0, 1e-31, -3e-38, 3e38, 2.0 ** -100])
def test_blocks_of_one_value(value):
    from them_bones_b200 import ops
    k = torch.full((1, 64, 1, 64), value).bfloat16()
    c = _fill(ops.kv8_cache(1, 64, 1, 64), k, -k, [64])
    a, b = ops.kv8_read(c, 64, 64)
    want = k if abs(value) >= 2.0 ** -100 else torch.zeros_like(k)
    assert torch.equal(a, want) and torch.equal(b, -want)


@pytest.mark.parametrize("d,window", [(64, 0), (128, 0), (64, 128)])
def test_attention_from_the_first_token_on(d, window):
    from them_bones_b200 import ops
    from them_bones_b200.ref import functional as RF
    torch.manual_seed(3)
    b, h, n = 3, 2, 150
    cos, sin = RF.rotary_tables(192, d, 10000.0)
    qkv = torch.randn(b, n, 3 * h * d)
    cache = ops.kv8_cache(b, n, h, d)
    for p in range(n):
        pos = torch.tensor([p, p, -1], dtype=torch.int32)
        start = torch.tensor([0, max(0, p - 5), 0], dtype=torch.int32)
        before = [x.clone() for x in cache]
        y = ops.kv8_attention(qkv[:, p], cos, sin, cache, pos, 0.2, start, window).double().view(b, h, d)
        kept = cache.k_open[:, :, p % 64]
        want, most = O.attend(qkv[:, p], cos, sin, before, kept, pos.tolist(), 0.2, start, window)
        # fp32: scores of up to 0.2 * 2 * d off by d / 2 roundings, a few roundings of the sums
        assert bool(((y - want).abs().amax((1, 2)) <= (0.2 * 2 * d * d * 2 ** -24 + 2 ** -20) * most).all())
        assert not y[2].any() and all(torch.equal(x[2], w[2]) for x, w in zip(cache, before))
        for i in range(2):
            k = O.new_rows(qkv[i, p], cos, sin, p, h, d)[1]
            assert bool(((kept[i].double() - k).abs() <= (2 ** -8 + 2 ** -18) * k.abs() + 2 ** -20).all())


def test_a_query_that_sees_nothing_and_one_outside():
    from them_bones_b200 import ops
    from them_bones_b200.ref import functional as RF
    torch.manual_seed(4)
    cos, sin = RF.rotary_tables(100, 64, 10000.0)
    qkv, cache = torch.randn(4, 3 * 64), ops.kv8_cache(4, 128, 1, 64)
    pos = torch.tensor([5, 100, 128, 5], dtype=torch.int32)
    y = ops.kv8_attention(qkv, cos, sin, cache, pos, 1.0, torch.tensor([9, 0, 0, 5], dtype=torch.int32))
    assert not y[:3].any() and y[3].any()
    assert cache.k_open[0, 0, 5].any() and not cache.k_open[1:3].any()          # the blind query's key is kept all the same


def test_ragged_append_and_what_does_not_fit():
    from them_bones_b200 import ops
    torch.manual_seed(5)
    k, v = torch.randn(2, 6, 70, 1, 64).bfloat16()
    c = ops.kv8_cache(6, 128, 1, 64)
    pos, lens = (torch.tensor(x, dtype=torch.int32) for x in ([0, 0, -3, 100, 58, 0], [70, 0, 70, 70, 70, -2]))
    ops.kv8_append(c, k, v, pos, lens)
    a, _ = ops.kv8_read(c, torch.tensor([70, 0, 0, 0, 128, 0], dtype=torch.int32), 128)
    assert a[0, :70].any() and torch.equal(a[0, 64:70], k[0, 64:70]) and a[4, 64:].any() and not a[[1, 2, 3, 5]].any()
    assert not any(x[[1, 2, 3, 5]].any() for x in c)


def test_refusals():
    from them_bones_b200 import ops
    for args in ((1, 64, 2, 96), (0, 64, 2, 64), (1, 0, 2, 64), (1, 64, 0, 64), (1, 1 << 31, 1, 64), (70000, 64, 1, 64)):
        with pytest.raises(ValueError):
            ops.kv8_cache(*args, device="meta")
    c = ops.kv8_cache(2, 64, 2, 64)
    k = torch.randn(2, 5, 2, 64).bfloat16()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    bad = [(c, k[:1], k[:1], 0), (c, k, k[:, :4], 0), (c, k, k.float(), 0), (c, k.int(), k.int(), 0), (c, k, k, 60), (c, k, k, -1), (c, k, k, torch.tensor([0, 0])),
           (c, k, k, i32(0, 0, 0)), (c, k, k, 0, 6), (c, k, k, 0, -1), (c, k, k, i32(0), 6), (c, k, k, 0, torch.tensor([1.0])), (c, k[..., :32], k[..., :32], 0),
           (c._replace(k=c.k[:, :, :32]), k, k, 0), (c._replace(v=c.v.transpose(-1, -2)), k, k, 0), (c._replace(k_scale=c.k_scale.double()), k, k, 0),
           (c._replace(k_open=c.k_open.float()), k, k, 0)]
    for args in bad:
        with pytest.raises(ValueError):
            ops.kv8_append(*args)
    with pytest.raises(ValueError):
        ops.kv8_append(c, k.float().requires_grad_(), k.float(), 0)
    for args in ((c, 65, 64), (c, -1, 64), (c, 5, -1), (c, i32(1, 2, 3), 5)):
        with pytest.raises(ValueError):
            ops.kv8_read(*args)
    qkv, cos = torch.randn(2, 3 * 128), torch.ones(64, 32)
    for args in ((qkv[:1], cos, cos, c, 0, 1.0), (qkv[:, :-1], cos, cos, c, 0, 1.0), (qkv, cos[:, :16], cos[:, :16], c, 0, 1.0), (qkv, cos, cos[:3], c, 0, 1.0),
                 (qkv, cos, cos, c, 64, 1.0), (qkv, cos[:5], cos[:5], c, 5, 1.0), (qkv, cos, cos, c, -1, 1.0), (qkv, cos, cos, c, 0, 1.0, torch.zeros(2)),
                 (qkv, cos, cos, c, 0, 1.0, i32(0)), (qkv, cos, cos, c, 0, 1.0, None, 100), (qkv, cos, cos, c, 0, 1.0, None, -128)):
        with pytest.raises(ValueError):
            ops.kv8_attention(*args)
    with pytest.raises(ValueError):
        ops.kv8_attention(qkv.requires_grad_(), cos, cos, c, 0, 1.0)
    with torch.no_grad():
        ops.kv8_attention(qkv, cos, cos, c, 0, 1.0)
