"""Drafts outside the vocabulary: nobody drew them, so what falls with them is replaced by a token of the target's own law, with and without draft logits."""
import pytest
import torch

from tests import paged_oracle as O
from tests.test_cpu_verify import problem
from them_bones_b200 import ops


def outside(vocab, cols, dtype, model, seed=0):
    """A problem whose every third draft is outside, and the same one with a draft row in front of those that holds no number: by the definition both end alike."""
    z, ids, starts, u, q = problem([4, 2, 1, 7, 3, 5, 2, 6], vocab, cols, dtype, model, seed)
    u[:, 0] *= 0.3                                           # most of the others stand
    bad = [-1, vocab, cols, 1 << 40, -(1 << 40), (1 << 32) + 3]
    told = None if q is None else q.clone()
    for i, r in enumerate(range(1, ids.shape[0], 3)):
        if r in starts.tolist():
            continue
        ids[r] = bad[i % len(bad)]
        if told is not None:
            told[r - 1] = float("nan")
    return z, ids, starts, u, q, told


@pytest.mark.parametrize("t", [0.0, 0.6, 1.0])
@pytest.mark.parametrize("model", [False, True])
@pytest.mark.parametrize("vocab,cols,dtype", [(50, 64, torch.float32), (257, 257, torch.bfloat16), (5, 8, torch.float32)])
def test_the_token_is_the_target_s(vocab, cols, dtype, model, t):
    z, ids, starts, u, q, told = outside(vocab, cols, dtype, model)
    want, near = O.verify(z, ids, starts, u, told, t, vocab)
    assert min(near) > 1e-12 and any(a < e - s - 1 for (a, _), s, e in zip(want, starts.tolist(), starts.tolist()[1:]))
    got = ops.verify_drafts(z, ids, starts, u, q, t, vocab)
    assert list(zip(got.accepted.tolist(), got.token.tolist())) == want


def test_it_follows_the_target_whatever_the_draft_model():
    """Over a grid of numbers, the token is each one as often as p says, where p and q have nothing in common."""
    p, q = torch.tensor([0.5, 0.3, 0.15, 0.05]), torch.tensor([0.02, 0.18, 0.3, 0.5])
    n = 400
    u = torch.stack([torch.zeros(2 * n), (torch.arange(2 * n) // 2 + 0.5) / n], 1)
    ids = torch.zeros(2 * n, dtype=torch.int64)
    ids[1::2] = -1
    got = ops.verify_drafts(p.log().expand(2 * n, 4).contiguous(), ids, O.i32(list(range(0, 2 * n + 1, 2))), u, q.log().expand(2 * n, 4).contiguous())
    count = torch.bincount(got.token, minlength=4).double() / n
    assert not got.accepted.any() and bool(((count - p).abs() <= 1.5 / n).all())
