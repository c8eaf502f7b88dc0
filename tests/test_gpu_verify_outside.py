"""Drafts outside the vocabulary on the GPU: the token that follows is one of the target's law, with and without draft logits."""
import pytest
import torch

from tests import paged_oracle as O
from tests.test_cpu_verify_outside import outside

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [0.0, 0.6, 1.0])
@pytest.mark.parametrize("model", [False, True])
@pytest.mark.parametrize("vocab,cols,dtype", [(50, 64, torch.float32), (257, 257, torch.bfloat16), (5, 8, torch.float32), (9001, 9008, torch.bfloat16)])
def test_the_token_is_the_target_s(vocab, cols, dtype, model, t):
    from them_bones_b200 import ops
    z, ids, starts, u, q, told = outside(vocab, cols, dtype, model)
    want, near = O.verify(z, ids, starts, u, told, t, vocab)
    assert min(near) > 1e-12
    got = ops.verify_drafts(z.cuda(), ids.cuda(), starts.cuda(), u.cuda(), None if q is None else q.cuda(), t, vocab)
    assert list(zip(got.accepted.tolist(), got.token.tolist())) == want


def test_captured_with_drafts_that_come_and_go():
    """A fixed width filled up with -1: the captured call reads the drafts anew."""
    from them_bones_b200 import ops
    z, ids, starts, u, q, told = (None if x is None else x.cuda() for x in outside(1000, 1000, torch.float32, True, seed=3))
    good = torch.where((ids >= 0) & (ids < 1000), ids, torch.full_like(ids, 7))
    now = good.clone()
    ops.verify_drafts(z, now, starts, u, q, 1.0)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.verify_drafts(z, now, starts, u, q, 1.0)
    for drafts, draft_logits in ((ids, told), (good, q), (ids, told)):
        now.copy_(drafts)
        g.replay()
        want = ops.verify_drafts(z.cpu(), drafts.cpu(), starts.cpu(), u.cpu(), draft_logits.cpu(), 1.0)
        assert torch.equal(out.accepted.cpu(), want.accepted) and torch.equal(out.token.cpu(), want.token)
