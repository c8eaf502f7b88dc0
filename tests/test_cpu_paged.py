"""The paged cache's statement against 64 bits, and the calls that are refused."""
import pytest
import torch

from tests import paged_oracle as O
from them_bones_b200 import ops

CASES = [  # heads, head_dim, page, new tokens, positions
    (2, 64, 16, [1], [0]), (1, 128, 64, [1, 1, 1], [0, 63, 64]), (3, 64, 32, [5, 0, 33, 1], [10, 3, 100, 127]), (2, 128, 128, [130, 40], [0, 200]),
    (2, 64, 16, [17, 16, 1], [15, 16, 300]), (1, 64, 64, [3, 4, 2], [-1, 7, 0])]


@pytest.mark.parametrize("h,d,page,lens,pos", CASES)
def test_append_is_the_formula(h, d, page, lens, pos):
    c, table, starts, at = O.world(len(lens), h, d, page, lens, pos)
    n = int(starts[-1])
    qkv = torch.randn(n + 3, 3 * h * d, generator=torch.Generator().manual_seed(2)).bfloat16()
    cos, sin = O.angles(512, d)
    (q, k, v), (qt, kt) = O.append(qkv[:n + 3], cos, sin, c, table, starts, at)
    got = ops.paged_append(qkv, cos, sin, c, table, starts, at)
    assert bool(((got.double() - q).abs() <= qt).all()) and bool(((c.k.double() - k).abs() <= kt).all()) and torch.equal(c.v.double(), v)


@pytest.mark.parametrize("window", [0, 128])
@pytest.mark.parametrize("h,d,page,lens,pos", CASES)
def test_attention_is_the_formula(h, d, page, lens, pos, window):
    c, table, starts, at = O.world(len(lens), h, d, page, lens, pos)
    n = int(starts[-1]) + 2
    q = O.queries(n, h, d)
    doc = O.i32([max(0, (7 * i) % 200 - 30) for i in range(n)])
    for ds in (None, doc):
        y, tol = O.attend(q, c, table, starts, at, 0.11, ds, window)
        got = ops.paged_attention(q, c, table, starts, at, 0.11, ds, window)
        assert bool(((got.double() - y).abs() <= tol).all())


def test_positions_without_a_page_are_not_stored_and_not_seen():
    c, table, starts, pos = O.world(2, 1, 64, 16, [40, 8], [0, 30])
    table[0, 1], table[1, 0] = -1, 99
    q = O.queries(48, 1, 64)
    before = [x.clone() for x in c]
    y, tol = O.attend(q, c, table, starts, pos, 0.1, None, 0)
    assert bool(((ops.paged_attention(q, c, table, starts, pos, 0.1).double() - y).abs() <= tol).all())
    ops.paged_append(torch.randn(48, 192).bfloat16(), *O.angles(64, 64), c, table, starts, pos)
    used = {int(x) for x in table.flatten() if 0 <= int(x) < c.k.shape[0]}
    for i in range(c.k.shape[0]):
        if i not in used:
            assert torch.equal(c.k[i], before[0][i]) and torch.equal(c.v[i], before[1][i])


def test_values_that_are_not_finite_reach_only_those_who_see_them():
    c, table, starts, pos = O.world(1, 1, 64, 16, [20], [10])
    q = O.queries(20, 1, 64)
    want = ops.paged_attention(q, c, table, starts, pos, 0.1)
    c.v[int(table[0, 1]), 0, 4, 3], c.v[int(table[0, 1]), 0, 4, 7] = float("inf"), float("nan")       # position 20
    got = ops.paged_attention(q, c, table, starts, pos, 0.1)
    seen = torch.arange(10, 30) >= 20
    assert torch.equal(got[~seen], want[~seen]) and bool(got[seen, 3].isinf().all()) and bool(got[seen, 7].isnan().all())
    rest = [i for i in range(64) if i not in (3, 7)]
    assert bool((got[:, rest].isfinite()).all())


def _ok():
    c, table, starts, pos = O.world(2, 2, 64, 16, [3, 4], [0, 5])
    cos, sin = O.angles(64, 64)
    return dict(qkv=torch.randn(7, 384).bfloat16(), cos=cos, sin=sin, cache=c, table=table, starts=starts, pos=pos)


@pytest.mark.parametrize("change", [
    dict(qkv=torch.zeros(7, 380).bfloat16()), dict(qkv=torch.zeros(384).bfloat16()), dict(qkv=torch.zeros(7, 384, dtype=torch.int32)),
    dict(qkv=torch.zeros(7, 384, requires_grad=True)), dict(cos=torch.zeros(64, 31)), dict(sin=torch.zeros(63, 32)), dict(table=torch.zeros(2, 1)),
    dict(table=torch.zeros(2, 1, dtype=torch.int64)), dict(table=torch.zeros(2, 0, dtype=torch.int32)), dict(table=torch.zeros(4, 2, dtype=torch.int32).T),
    dict(starts=torch.zeros(2, dtype=torch.int32)), dict(starts=torch.zeros(3, dtype=torch.int64)), dict(pos=torch.zeros(3, dtype=torch.int32)),
    dict(pos=torch.zeros(2)), dict(cache=ops.PagedKV(torch.zeros(3, 2, 16, 64).bfloat16(), torch.zeros(3, 2, 16, 64))),
    dict(cache=ops.PagedKV(torch.zeros(3, 2, 24, 64).bfloat16(), torch.zeros(3, 2, 24, 64).bfloat16())),
    dict(cache=ops.PagedKV(torch.zeros(3, 2, 16, 96).bfloat16(), torch.zeros(3, 2, 16, 96).bfloat16())),
    dict(cache=ops.PagedKV(torch.zeros(3, 16, 2, 64).bfloat16().transpose(1, 2), torch.zeros(3, 16, 2, 64).bfloat16().transpose(1, 2)))])
def test_calls_that_append_refuses(change):
    args = {**_ok(), **change}
    with pytest.raises(ValueError):
        ops.paged_append(**args)


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(7, 120).bfloat16()), dict(q=torch.zeros(7, 128)), dict(q=torch.zeros(7, 128).bfloat16().requires_grad_()), dict(window=100), dict(window=-128),
    dict(doc_start=torch.zeros(7, dtype=torch.int64)), dict(doc_start=torch.zeros(6, dtype=torch.int32)), dict(longest=-1), dict(scale=float("inf")),
    dict(scale=float("nan"))])
def test_calls_that_attention_refuses(change):
    a = _ok()
    args = {**dict(q=O.queries(7, 2, 64), cache=a["cache"], table=a["table"], starts=a["starts"], pos=a["pos"], scale=0.1), **change}
    with pytest.raises(ValueError):
        ops.paged_attention(**args)


@pytest.mark.parametrize("args", [(0, 2, 64), (3, 0, 64), (3, 2, 96), (3, 2, 64, 8), (3, 2, 64, 48), (1 << 25, 8, 64, 128)])
def test_caches_that_are_refused(args):
    with pytest.raises(ValueError):
        ops.paged_cache(*args)


def test_dual_tensors_are_refused():
    import torch.autograd.forward_ad as fa
    a = _ok()
    with fa.dual_level():
        a["qkv"] = fa.make_dual(torch.randn(7, 384), torch.randn(7, 384))
        with pytest.raises(ValueError):
            ops.paged_append(**a)


@pytest.mark.parametrize("what", ["cos", "sin", "k", "v"])
def test_tensors_that_ask_for_a_gradient_are_refused_wherever_they_come(what):
    a = _ok()
    if what in a:
        a[what].requires_grad_()
    else:
        getattr(a["cache"], what).requires_grad_()
    with pytest.raises(ValueError):
        ops.paged_append(**a)
    with torch.no_grad():
        ops.paged_append(**a)


def test_a_window_of_any_size():
    c, table, starts, pos = O.world(2, 1, 64, 16, [3, 40], [200, 300])
    q = O.queries(43, 1, 64)
    want = ops.paged_attention(q, c, table, starts, pos, 0.1)
    for window in (1 << 31, 1 << 45, 128 * ((1 << 32) + 1)):
        assert torch.equal(ops.paged_attention(q, c, table, starts, pos, 0.1, window=window), want)
