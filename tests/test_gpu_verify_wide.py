"""Vocabularies so wide that sums in 32 bits say nothing of a draft near its border: decided in 64 bits all the same."""
import math

import pytest
import torch

from tests import paged_oracle as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("w,off", [(0.2, -3.1e-4), (0.2, 3.1e-4), (0.35, -3.1e-4), (0.35, 3.1e-4)])
def test_drafts_near_their_border(w, off):
    """2^25 times four columns of weights 1, w, w, w: a thread that adds 65536 such sums in fp32 ends 6e-4 of the whole too high (w = 0.2) or too low (0.35), and the draft's number
    lies between the border and where such sums put it, or as far on the other side."""
    from them_bones_b200 import ops
    quads, v = 1 << 25, 1 << 27
    low = torch.tensor(math.log(w), dtype=torch.float32)
    w = math.exp(float(low))
    z = torch.stack([torch.zeros(()), low, low, low]).cuda().repeat(2, quads)
    px, s = 1.0 / (quads * (1.0 + 3.0 * w)), 1.0 + 3.0 * w
    u = torch.tensor([[px * (1.0 + off), 0.1], [0.5, 0.1]])
    assert abs(float(u[0, 0]) / px - 1.0 - off) < 1e-7                                # a half step of fp32 is 6e-8
    x = 12345 * 4
    got = ops.verify_drafts(z, torch.tensor([0, x], device="cuda"), O.i32([0, 2], "cuda"), u.cuda())
    # the token of the last row: the quad and the place in it that 0.1 in fp32 says, 0.25 s from the next border of 5e7 in all
    quad, rest = divmod(float(u[1, 1]) * quads, 1.0)
    assert 0.1 < rest * s < 0.9
    assert (int(got.accepted), int(got.token) if off < 0 else -1) == ((1, 4 * int(quad)) if off < 0 else (0, -1))
