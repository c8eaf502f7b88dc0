"""The largest calls that the paged cache and the verification take, by the short way and the long one, and the first that neither takes."""
import pytest
import torch

from tests import paged_oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_wait_ran_out():
    yield
    from them_bones_b200.ops import _lib as L
    L.check_error_word()


def _one_token_each(b, h, longest):
    """A first token each of b sequences, in a page of its own: a query sees its own key alone, and its result is its value."""
    from them_bones_b200 import ops
    from them_bones_b200.ops import paged as P
    d, page = 64, 16
    g = torch.Generator(device="cuda").manual_seed(b + h)
    c = ops.paged_cache(b, h, d, page, "cuda")
    table = torch.randperm(b, device="cuda", generator=g).int()[:, None]
    starts, pos = torch.arange(b + 1, dtype=torch.int32, device="cuda"), torch.zeros(b, dtype=torch.int32, device="cuda")
    qkv = torch.randn(b, 3 * h * d, device="cuda", dtype=torch.bfloat16, generator=g)
    cos, sin = O.angles(16, d, "cuda")
    q = P.short_append(qkv, cos, sin, c, table, starts, pos)
    k = c.k.clone()
    again = P.append(P.check_append(qkv, cos, sin, c, table, starts, pos), qkv, cos, sin, c, table, starts, pos)
    assert q is not None and torch.equal(q, again) and torch.equal(k, c.k)
    y = P.short_attention(q, c, table, starts, pos, 0.1, None, 0, longest)
    args = (q, c, table, starts, pos, 0.1, None, 0, longest)
    again = P.attention(P.check_attention(*args), *args)
    v = qkv[:, 2 * h * d:].double()
    assert y is not None and torch.equal(y, again)
    # its one weight and the result are rounded to bf16
    assert bool(((y.double() - v).abs() <= (2 * O.HALF + 2.0 ** -15) * v.abs()).all())


@pytest.mark.parametrize("longest", [1, 17])
@pytest.mark.parametrize("b,h", [(65534, 1), (1, 65535), (3, 21845), (512, 3), (513, 3)])
def test_the_largest_numbers_of_sequences_and_heads(b, h, longest):
    _one_token_each(b, h, longest)


def test_one_more_is_refused_by_both_ways():
    from them_bones_b200 import ops
    from them_bones_b200.ops import paged as P
    d, page = 64, 16
    cos, sin = O.angles(16, d, "cuda")
    small = ops.paged_cache(2, 1, d, page, "cuda")
    one = dict(table=O.i32([[0]], "cuda"), starts=O.i32([0, 1], "cuda"), pos=O.i32([0], "cuda"))
    many = dict(table=torch.zeros(65535, 1, dtype=torch.int32, device="cuda"), starts=torch.zeros(65536, dtype=torch.int32, device="cuda"),
                pos=torch.zeros(65535, dtype=torch.int32, device="cuda"))
    long = dict(one, table=torch.zeros(1, (1 << 31) // 16 - 7, dtype=torch.int32, device="cuda"))
    heads = ops.PagedKV(*(torch.zeros(1, 65536, page, d, dtype=torch.bfloat16, device="cuda") for _ in range(2)))
    x = torch.zeros(1, 3 * d, dtype=torch.bfloat16, device="cuda")
    for c, at, n in ((small, many, 1), (small, long, 1), (heads, one, 1), (small, one, 1 << 26)):
        h = c.k.shape[1]
        qkv, q = (torch.zeros(1, w * h * d, dtype=torch.bfloat16, device="cuda").expand(n, w * h * d) for w in (3, 1))
        assert P.short_append(qkv, cos, sin, c, *at.values()) is None and P.short_attention(q, c, *at.values(), 0.1, None, 0, 1) is None
        with pytest.raises(ValueError):
            ops.paged_append(qkv, cos, sin, c, *at.values())
        with pytest.raises(ValueError):
            ops.paged_attention(q, c, *at.values(), 0.1)
    assert P.short_append(x, cos, sin, small, *one.values()) is not None


@pytest.mark.parametrize("t", [0.0, 1.0])
def test_the_largest_numbers_of_sequences_and_columns(t):
    from them_bones_b200 import ops
    from them_bones_b200.ops import verify as V
    n = 65535
    z = torch.zeros(n, 3, device="cuda")
    best = torch.arange(n, device="cuda") % 3
    z.scatter_(1, best[:, None], 200.0)
    ids, u = torch.zeros(n, dtype=torch.int64, device="cuda"), torch.rand(n, 2, device="cuda")
    starts = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    got = V.short(z, ids, starts, u, None, t, 3)
    want = V.native(z, ids, starts, u, None, t, 3)
    assert got is not None and torch.equal(got.token, best) and torch.equal(want.token, best) and not got.accepted.any()
    more = torch.zeros(n + 2, dtype=torch.int32, device="cuda")
    assert V.short(z, ids, more, u, None, t, 3) is None
    with pytest.raises(ValueError):
        ops.verify_drafts(z, ids, more, u, temperature=t)
    # 2^30 columns, a token and a draft, the last column the likely one
    wide = 1 << 30
    z = torch.zeros(2, wide + 8, dtype=torch.bfloat16, device="cuda")
    z[0, wide - 1], z[1, wide - 2], z[:, wide:] = 60.0, 60.0, 90.0
    ids, u, starts = torch.tensor([0, wide - 1], device="cuda"), torch.full((2, 2), 0.5, device="cuda"), O.i32([0, 2], "cuda")
    for out in (V.short(z, ids, starts, u, None, t, wide), V.native(z, ids, starts, u, None, t, wide)):
        assert (int(out.accepted), int(out.token)) == (1, wide - 2)
    assert V.short(z, ids, starts, u, None, t, wide + 1) is None
    with pytest.raises(ValueError):
        ops.verify_drafts(z, ids, starts, u, temperature=t, vocab=wide + 1)
