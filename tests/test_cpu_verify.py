"""The verification of drafts: the statement against 64 bits, the distribution it draws from, and the calls that are refused."""
import math

import pytest
import torch

from tests import paged_oracle as O
from them_bones_b200 import ops


def problem(lens, vocab, cols, dtype, model, seed=0, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    n = sum(lens)
    z = torch.randn(n, cols, generator=g) * spread
    near = z + 0.5 * torch.randn(n, cols, generator=g)
    starts = [0]
    for x in lens:
        starts.append(starts[-1] + x)
    ids = torch.randint(0, vocab, (n,), generator=g)
    take = torch.rand(n, generator=g) < 0.8
    ids[1:] = torch.where(take[1:], near[:-1, :vocab].argmax(1), ids[1:])
    return z.to(dtype), ids, O.i32(starts), torch.rand(n, 2, generator=g), near.to(dtype) if model else None


@pytest.mark.parametrize("t", [0.0, 0.5, 1.0, 2.0])
@pytest.mark.parametrize("lens,vocab,cols,dtype,model", [
    ([1], 1, 1, torch.float32, False), ([4], 50, 64, torch.float32, True), ([3, 0, 5, 1, 0], 100, 100, torch.bfloat16, True), ([40, 2], 33, 40, torch.float32, True),
    ([2, 8, 4], 257, 300, torch.bfloat16, False)])
def test_statement_is_the_definition(lens, vocab, cols, dtype, model, t):
    z, ids, starts, u, q = problem(lens, vocab, cols, dtype, model)
    want, near = O.verify(z, ids, starts, u, q, t, vocab)
    got = ops.verify_drafts(z, ids, starts, u if t else None, q, t, vocab)
    assert min(near) > 1e-12
    assert list(zip(got.accepted.tolist(), got.token.tolist())) == want
    assert got.accepted.dtype is torch.int32 and got.token.dtype is torch.int64


def test_tokens_follow_the_target_whatever_the_drafts():
    """Over the grid of both numbers, a draft drawn from q and its verification give every token as often as p says."""
    p, q = torch.tensor([0.5, 0.2, 0.2, 0.1], dtype=torch.float64), torch.tensor([0.1, 0.6, 0.2, 0.1], dtype=torch.float64)
    g = 50
    grid = (torch.arange(g) + 0.5) / g
    count = torch.zeros(4, dtype=torch.float64)
    z, d = p.log().float(), q.log().float()
    u = torch.cartesian_prod(grid, grid).float()
    for x in range(4):
        n = u.shape[0]
        ids = torch.zeros(2 * n, dtype=torch.int64)
        ids[1::2] = x
        uu = torch.zeros(2 * n, 2)
        uu[0::2] = u
        got = ops.verify_drafts(z.expand(2 * n, 4).contiguous(), ids, O.i32(list(range(0, 2 * n + 1, 2))), uu, d.expand(2 * n, 4).contiguous())
        first = torch.where(got.accepted > 0, torch.full_like(got.token, x), got.token)
        count += q[x] * torch.bincount(first, minlength=4).double() / n
    # a border of the grid's: one row of either side
    assert bool(((count - p).abs() <= 1.5 / g).all())


def test_rows_without_a_number():
    z, ids, starts, u, q = problem([3, 3, 3, 3], 20, 20, torch.float32, True)
    z[0, 3], z[3] = float("nan"), -math.inf
    z[7, 2] = math.inf
    q[9, 1] = float("nan")
    ids[7] = int(z[6].argmax())
    u[:, 0] = 0.0
    for t in (0.0, 1.0):
        got = ops.verify_drafts(z, ids, starts, u, q, t)
        assert got.accepted.tolist()[:3] == [0, 0, 1] and got.token.tolist()[:3] == [-1, -1, -1]
    got = ops.verify_drafts(z, ids, starts, u, q, 1.0)
    assert got.accepted.tolist()[3] == 0 and got.token.tolist()[3] >= 0


def test_masked_columns_and_drafts_outside():
    z = torch.full((2, 8), torch.finfo(torch.float32).min)
    z[:, 5] = 1.0
    u = torch.tensor([[0.5, 0.999], [0.5, 0.0]])
    for x, want in ((5, (1, 5)), (-1, (0, 5)), (8, (0, 5)), (3, (0, 5))):
        got = ops.verify_drafts(z, torch.tensor([0, x]), O.i32([0, 2]), u)
        assert (int(got.accepted), int(got.token)) == want


def test_equal_models_accept_every_draft():
    z, ids, starts, u, _ = problem([6, 6], 64, 64, torch.bfloat16, False)
    u[:, 0] = 1 - 2.0 ** -24
    got = ops.verify_drafts(z, ids, starts, u, z.clone(), 0.8)
    assert got.accepted.tolist() == [5, 5]


def _ok():
    z, ids, starts, u, q = problem([2, 3], 16, 16, torch.float32, True)
    return dict(logits=z, ids=ids, starts=starts, uniforms=u, draft_logits=q)


@pytest.mark.parametrize("change", [
    dict(logits=torch.zeros(5, dtype=torch.float32)), dict(logits=torch.zeros(5, 16, dtype=torch.int32)), dict(logits=torch.zeros(5, 16, requires_grad=True)),
    dict(ids=torch.zeros(4, dtype=torch.int64)), dict(ids=torch.zeros(5, dtype=torch.int32)), dict(starts=torch.zeros(1, dtype=torch.int32)),
    dict(starts=torch.zeros(3, dtype=torch.int64)), dict(uniforms=None), dict(uniforms=torch.zeros(5)), dict(uniforms=torch.zeros(5, 2, dtype=torch.float64)),
    dict(draft_logits=torch.zeros(5, 15)), dict(draft_logits=torch.zeros(5, 16).bfloat16()), dict(temperature=-1.0), dict(temperature=1e-9),
    dict(temperature=float("inf")), dict(temperature=1e7), dict(temperature=float("nan")), dict(vocab=0), dict(vocab=17)])
def test_calls_that_are_refused(change):
    with pytest.raises(ValueError):
        ops.verify_drafts(**{**_ok(), **change})
