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
    cos, sin = (x.to("cuda") for x in RF.rotary_tables(n + 1, d, 10000.0))
    cache = ops.kv8_cache(b, n + 1, h, d, "cuda")
    k, v = torch.randn(2, b, n, h, d, device="cuda").bfloat16()
    ops.kv8_append(cache, k, v, 0)
    before = [x.clone() for x in cache]
    qkv = torch.randn(b, 3, h, d, device="cuda").clamp(-4, 4)
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
    cos = torch.ones(64, 32, device="cuda")
    for part in (0, 1):
        cache = ops.kv8_cache(2, 64, 2, 64, "cuda")
        qkv = torch.randn(2, 3, 2, 64, device="cuda").bfloat16()
        qkv[1, part, 1, 5] = bad
        y = ops.kv8_attention(qkv.view(2, -1), cos, 0 * cos, cache, 0, 0.1).view(2, 2, 64)
        assert bool(y[0].isfinite().all()) and bool(y[1, 0].isfinite().all()) and bool(y[1, 1].isnan().all())


def _nearest_bf16(x):
    """fp64 to the nearest bf16 in one rounding: of the neighbours of what two roundings give, the nearest one."""
    b = x.float().bfloat16()
    near = [b] + [(b.view(torch.int16) + i).view(torch.bfloat16) for i in (-1, 1)]
    off = torch.stack([(n.double() - x).abs().nan_to_num(float("inf")) for n in near])
    return torch.stack(near).gather(0, off.argmin(0, keepdim=True))[0]


@pytest.mark.parametrize("d", [64, 128])
def test_the_new_key_is_rounded_once(d):
    """16 million keys' values: where fp32 lies between, one in 2^17 falls to the wrong side of the middle of two bf16 numbers."""
    from tests import kv8_oracle as O
    from them_bones_b200 import ops
    torch.manual_seed(9)
    b, h, n = 64, 16, 16 * 2 ** 20 // (64 * 16 * d)
    cache = ops.kv8_cache(b, 64, h, d, "cuda")
    cos, sin = torch.rand(2, 1, d // 2, device="cuda")
    for i in range(n):
        qkv = torch.randn(b, 3 * h * d, device="cuda").bfloat16()
        ops.kv8_attention(qkv, cos, sin, cache, 0, 0.1)
        want = O.new_rows(qkv.view(b, 3, h, d).transpose(0, 1).reshape(1, -1)[0], cos, sin, 0, b * h, d)[1].view(b, h, d)
        # a tie of two bf16 numbers to the last bits of fp64 is not met here
        assert torch.equal(cache.k_open[:, :, 0], _nearest_bf16(want)), i


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("places", [0, 5, 16, 17, 100, 1024])
def test_long_caches_take_no_more_room_than_there_is(places, d):
    """Parts of the result go to as many places as the call was given, whatever the SMs hold; behind them nothing is written."""
    from them_bones_b200 import ops
    from them_bones_b200.ops import _lib as L
    from them_bones_b200.ref import functional as RF
    torch.manual_seed(3)
    b, h, cap = 2, 3, 16384
    cos, sin = (x.cuda() for x in RF.rotary_tables(cap, d, 10000.0))
    qkv, pos = torch.randn(b, 3 * h * d, device="cuda").bfloat16(), torch.tensor([16000, 9000], dtype=torch.int32, device="cuda")
    cache = ops.kv8_cache(b, cap, h, d, "cuda")
    k, v = torch.randn(2, b, 16000, h, d, device="cuda").bfloat16()
    ops.kv8_append(cache, k, v, 0, pos)
    want = ops.kv8_attention(qkv, cos, sin, cache, pos, 0.1)
    y, room = torch.empty_like(want), torch.full((1024 * (d + 4),), 12345.0, device="cuda")
    c = cache
    L.call("bones_kv8_attention", qkv.data_ptr(), qkv.stride(0), cos.data_ptr(), sin.data_ptr(), cap, c.k.data_ptr(), c.v.data_ptr(), c.k_scale.data_ptr(), c.v_scale.data_ptr(),
           c.k_open.data_ptr(), c.v_open.data_ptr(), pos.data_ptr(), 1, 0, 0, y.data_ptr(), b, h, d, cap, 0.1, 0, 0, room.data_ptr(), places, L.raw_stream())
    assert bool((room[places * (d + 4):] == 12345.0).all())
    assert bool((room != 12345.0).any()) == (places >= 16)          # 8 * 6 heads in 3 of them; with fewer, clusters
    # other orders of the same sum: probabilities of 11 bits whose largest differs, and a rounding to bf16 of a result of size 1 at most
    assert float((y.float() - want.float()).abs().max()) <= 2 ** -8 + 2 ** -11 * 6


@pytest.mark.parametrize("d", [64, 128])
def test_a_key_that_is_not_finite_is_kept_as_the_formula_has_it(d):
    """Behind an infinite norm the finite values are zeros and the infinite ones have no number; a NaN leaves nothing."""
    from tests import kv8_oracle as O
    from them_bones_b200 import ops
    from them_bones_b200.ref import functional as RF
    torch.manual_seed(10)
    inf, nan = float("inf"), float("nan")
    cos, sin = (x.cuda() for x in RF.rotary_tables(64, d, 10000.0))
    qkv = torch.randn(4, 3, 2, d, device="cuda").bfloat16()
    qkv[0, 1, 0, 3], qkv[1, 1, 1, d - 1], qkv[2, 1, 0, 5], qkv[3, 1, 0, 7], qkv[3, 1, 1, 7] = inf, -inf, nan, inf, nan
    plain, kernel = (ops.kv8_cache(4, 64, 2, d, "cuda") for _ in range(2))
    ops.kv8_attention(qkv.view(4, -1), cos, sin, kernel, 63, 0.1)
    RF.kv8_attention(qkv.view(4, -1), cos, sin, plain, [63] * 4, 0.1)
    for i in range(4):
        want = O.new_rows(qkv[i].view(-1), cos, sin, 63, 2, d)[1]
        for c in (kernel, plain):
            got = c.k_open[i, :, 63].double()
            assert torch.equal(got.isnan(), want.isnan()) and not (got - want)[(want == 0) & ~want.isnan()].any()
            assert torch.equal(c.k[i, :, 63] == -128, want.isnan())
    assert int(kernel.k_open[0, 0, 63].isnan().sum()) == 2 and int(kernel.k_open[2, 0, 63].isnan().sum()) == d
