"""The token behind a refused draft where the target and the draft model nearly agree: what is left of p beside q is a small part of either."""
import pytest
import torch

from tests import paged_oracle as O

pytestmark = pytest.mark.gpu

# Of itself, a weight of the law is off by 1.4e-13 at most (the remainder of its series) and a few roundings of 2^-53: 1.6e-13.  So p - q is off by 3.2e-13 of p at most, and a
# sum of such, column by column or in all, by 3.2e-13 of the whole p; of what is left, W, the borders move by twice that over W.
OFF = 2 * 3.2e-13


def _expected(z, q, x, u, t):
    """Of each row of ``z`` and ``q``, whose draft is ``x``: whether it stands, the token, and how near the decision is to a border (of the whole p)."""
    p, d = (torch.softmax((v.double() - v.double().amax(1, keepdim=True)) / t, 1) for v in (z, q))
    px, dx = (v.gather(1, x[:, None])[:, 0] for v in (p, d))
    stands = u[:, 0].double() * dx < px
    w = (p - d).clamp_min(0.0)
    left = w.sum(1)
    c = w.cumsum(1)
    need = u[:, 1:].double() * c[:, -1:]
    token = (c <= need).sum(1).clamp(max=z.shape[1] - 1)
    # columns without weight have no border
    near = torch.where(w > 0, (c - need).abs(), torch.ones_like(c)).amin(1)
    # the weight below the token: a number near 0 has its border in front of the first column
    return stands, token, left, torch.minimum(near, need[:, 0])


def _rows(n, vocab, kind, noise, dtype, seed):
    """Target's and draft's logits, and of each row the column that the draft model overrates most (of those that are not the rarest)."""
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(n, vocab, generator=g) * 2.0
    if kind == "all":                                   # the same model but for rounding, everywhere
        q = z + noise * torch.randn(n, vocab, generator=g)
    else:                                               # the same but for a few rare columns
        q = z.clone()
        z[:, :8] = -4.0 + torch.rand(n, 8, generator=g)
        q[:, :8] = z[:, :8] + noise * torch.tensor([1.0, -1.0, 0.5, -0.5, 0.25, -0.25, 1.0, -1.5])
    return z.to(dtype), q.to(dtype)


@pytest.mark.parametrize("vocab,kind,noise,t,dtype", [
    (1000, "all", 1e-7, 0.7, torch.float32), (8000, "all", 1e-7, 0.7, torch.float32), (8000, "all", 1e-6, 1.0, torch.float32), (50001, "all", 1e-4, 1.0, torch.float32),
    (1000, "all", 0.5, 1e6, torch.float32), (65536, "all", 0.5, 1e5, torch.bfloat16), (3000, "few", 1e-4, 1.0, torch.float32), (3000, "few", 1e-3, 1.0, torch.float32),
    (65536, "few", 0.1, 1.0, torch.float32), (65536, "few", 0.1, 0.6, torch.bfloat16), (8192, "few", 3.0, 1.0, torch.bfloat16), (4097, "all", 1e-2, 0.8, torch.float32)])
def test_small_residuals_are_the_definition(vocab, kind, noise, t, dtype):
    from them_bones_b200 import ops
    n = 300
    z, q = _rows(n, vocab, kind, noise, dtype, seed=vocab)
    z, q = z.cuda(), q.cuda()
    x = (torch.log_softmax(q.double() / t, 1) - torch.log_softmax(z.double() / t, 1)).argmax(1)
    u = torch.rand(n, 2, generator=torch.Generator().manual_seed(7)).cuda()
    u[:, 0] = 1 - 2.0 ** -24
    stands, want, left, near = _expected(z, q, x, u, t)
    ids = torch.zeros(2 * n, dtype=torch.int64, device="cuda")
    ids[1::2] = x
    two = lambda v: v.repeat_interleave(2, 0)  # noqa: E731
    starts = torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device="cuda")
    got = ops.verify_drafts(two(z), ids, starts, two(u), two(q), t)
    assert torch.equal(got.accepted.bool(), stands)
    sure = ~stands & (near > OFF) & (left > 2e-12)          # 1e-12 of p counts as nothing left
    assert int(sure.sum()) >= n // 4
    wrong = sure & (got.token != want)
    assert not bool(wrong.any()), (int(wrong.sum()), int(sure.sum()), float(left[wrong].min()), float(near[wrong].max()))
