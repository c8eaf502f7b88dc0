"""The verification of drafts on the GPU against 64 bits, and the calls where it can go wrong."""
import pytest
import torch

from tests import paged_oracle as O
from tests.test_cpu_verify import problem

pytestmark = pytest.mark.gpu


def _cuda(z, ids, starts, u, q):
    return z.cuda(), ids.cuda(), starts.cuda(), u.cuda(), None if q is None else q.cuda()


def _check(z, ids, starts, u, q, t, vocab):
    """Against 64 bits; a decision closer to its border than the sums' roundings would say nothing (none of these is)."""
    from them_bones_b200 import ops
    want, near = O.verify(z, ids, starts, u, q, t, vocab)
    assert min(near) > 1e-12
    got = ops.verify_drafts(*_cuda(z, ids, starts, u, None)[:3], u.cuda() if t else None, None if q is None else q.cuda(), t, vocab)
    assert list(zip(got.accepted.tolist(), got.token.tolist())) == want


@pytest.mark.parametrize("t", [0.0, 0.3, 1.0, 3.0])
@pytest.mark.parametrize("lens,vocab,cols,dtype,model", [
    ([1], 1, 1, torch.float32, False), ([4], 50, 64, torch.float32, True), ([3, 0, 5, 1, 0], 100, 100, torch.bfloat16, True), ([40, 2, 70], 33, 40, torch.float32, True),
    ([2, 8, 4], 257, 300, torch.bfloat16, False), ([5, 5], 8191, 8192, torch.float32, True), ([3, 6], 8191, 8191, torch.bfloat16, True),
    ([2, 2], 16385, 16389, torch.bfloat16, False)])
def test_it_is_the_definition(lens, vocab, cols, dtype, model, t):
    _check(*problem(lens, vocab, cols, dtype, model), t, vocab)


@pytest.mark.parametrize("dtype,cols,model,t", [(torch.bfloat16, 65536, True, 1.0), (torch.float32, 65536, True, 0.7), (torch.bfloat16, 65531, False, 1.0),
                                                (torch.bfloat16, 65536, True, 0.0), (torch.float32, 50001, False, 1.3), (torch.float32, 200003, True, 1.0)])
def test_large_vocabularies_agree_with_the_statement(dtype, cols, model, t):
    """Some hundred draws: a border in 32 bits would miss one of them."""
    from them_bones_b200 import ops
    from them_bones_b200.ref import functional as RF
    z, ids, starts, u, q = _cuda(*problem([1 + i % 6 for i in range(200 if cols < 100000 else 60)], cols, cols, dtype, model, seed=5, spread=1.5))
    got = ops.verify_drafts(z, ids, starts, u if t else None, q, t)
    want = RF.verify_drafts(z, ids, starts, u, q, t, cols)
    assert torch.equal(got.accepted, want[0]) and torch.equal(got.token, want[1])
    assert 25 < int(got.accepted.sum()) < 500 or not t or not model          # without a model no draft is likely here
    again = ops.verify_drafts(z, ids, starts, u if t else None, q, t)
    assert torch.equal(got.accepted, again.accepted) and torch.equal(got.token, again.token)


def test_drafts_next_to_their_border():
    """Numbers one step of fp32 below and above p / q: decided as in 64 bits."""
    z, ids, starts, u, q = problem([2] * 64, 1000, 1000, torch.float32, True, seed=9)
    for i in range(64):
        r = 2 * i
        p, d = O.law(z[r].tolist(), 1.0), O.law(q[r].tolist(), 1.0)
        x = int(ids[r + 1])
        edge = torch.tensor(min(p[x] / d[x], 0.999))
        u[r, 0] = torch.nextafter(edge, torch.tensor(float(i % 2)))
    _check(z, ids, starts, u, q, 1.0, 1000)


def test_logits_far_from_zero_and_cold_temperatures():
    """Whole numbers of steps that the law's scale is cut into: large logits, and differences that are large multiples of the temperature."""
    for far, t in ((0.0, 1e-6), (1e4, 1.0), (-1e4, 0.01), (3e37, 1.0), (-3e38, 1e-6), (1e-3, 1e6), (2.0 ** 20, 0.5)):
        for dtype in (torch.float32, torch.bfloat16):
            z, ids, starts, u, q = problem([3, 2, 4], 700, 704, torch.float32, True, seed=3)
            z, q = (z + far).to(dtype), (q + far).to(dtype)
            ids[1], ids[4] = int(z[0, :700].float().argmax()), int(z[3, :700].float().argmax())
            _check(z, ids, starts, u, q, t, 700)
            _check(z, ids, starts, u, None, t, 700)


def test_the_ends_of_the_numbers():
    from them_bones_b200 import ops
    z = torch.full((3, 70000), -60.0)
    z[:, 4], z[:, 69000] = 0.0, 0.0
    z[2] = float("-inf")
    z[2, 69999] = -5.0
    u = torch.tensor([[0.0, 0.0], [0.0, 1 - 2.0 ** -24], [0.3, 1 - 2.0 ** -24]])
    got = ops.verify_drafts(z.cuda(), torch.zeros(3, dtype=torch.int64).cuda(), O.i32([0, 1, 2, 3], "cuda"), u.cuda())
    want, _ = O.verify(z, torch.zeros(3, dtype=torch.int64), O.i32([0, 1, 2, 3]), u, None, 1.0, 70000)
    assert got.token.tolist() == [t for _, t in want] and got.token.tolist()[0] == 0 and got.token.tolist()[2] == 69999


def test_rows_without_a_number():
    from them_bones_b200 import ops
    for dtype in (torch.float32, torch.bfloat16):
        z, ids, starts, u, q = problem([3, 3, 3, 3, 0], 20, 20, dtype, True)
        z[0, 3], z[3] = float("nan"), float("-inf")
        z[7, 2] = float("inf")
        q[9, 1], q[11] = float("nan"), float("nan")             # the second is nobody's
        ids[7] = int(z[6].float().argmax())
        u[:, 0] = 0.0
        for t in (0.0, 1.0):
            got = ops.verify_drafts(*_cuda(z, ids, starts, u, q), t)
            want = ops.verify_drafts(z, ids, starts, u, q, t)
            assert torch.equal(got.accepted.cpu(), want.accepted) and torch.equal(got.token.cpu(), want.token)
            assert got.token.tolist()[:3] == [-1, -1, -1] and got.token.tolist()[4] == -1 and got.accepted.tolist()[:3] == [0, 0, 1]


def test_masked_columns_and_drafts_outside():
    from them_bones_b200 import ops
    for dtype in (torch.float32, torch.bfloat16):
        for low in (float("-inf"), torch.finfo(dtype).min):
            z = torch.full((2, 300), low, dtype=dtype, device="cuda")
            z[:, 55] = 1.0
            u = torch.tensor([[0.5, 0.999], [0.5, 0.0]], device="cuda")
            for x, want in ((55, (1, 55)), (-1, (0, 55)), (300, (0, 55)), (1 << 40, (0, 55)), (3, (0, 55))):
                for t in (1.0, 0.0, 1e-6, 1e6):
                    got = ops.verify_drafts(z, torch.tensor([0, x], device="cuda"), O.i32([0, 2], "cuda"), u, temperature=t)
                    assert (int(got.accepted), int(got.token)) == want, (dtype, low, x, t)


def test_ties_go_to_the_lowest_index():
    from them_bones_b200 import ops
    z = torch.zeros(4, 9001, device="cuda")
    z[1, 8000], z[1, 77], z[2, 9000] = 2.0, 2.0, -1.0
    got = ops.verify_drafts(z, torch.tensor([5, 0, 77, 3], device="cuda"), O.i32([0, 3, 4], "cuda"), temperature=0.0)
    assert got.accepted.tolist() == [2, 0] and got.token.tolist() == [0, 0]


def test_rows_of_the_lowest_value_alone_and_lonely_numbers():
    from them_bones_b200 import ops
    for dtype in (torch.float32, torch.bfloat16):
        low = torch.finfo(dtype).min
        z = torch.full((4, 70001), float("-inf"), dtype=dtype)
        z[0] = low
        z[1, 69999], z[2, 3], z[2, 40000] = -2.0, 1.0, 1.5
        u = torch.full((4, 2), 0.5)
        for t in (0.0, 1.0):
            want = ops.verify_drafts(z, torch.zeros(4, dtype=torch.int64), O.i32([0, 1, 2, 3, 4]), u, temperature=t)
            got = ops.verify_drafts(z.cuda(), torch.zeros(4, dtype=torch.int64).cuda(), O.i32([0, 1, 2, 3, 4], "cuda"), u.cuda(), temperature=t)
            assert got.token.tolist() == want.token.tolist() and want.token.tolist()[1:] == [69999, 40000, -1] and (t or want.token[0] == 0)


def test_strided_and_unaligned_rows():
    from them_bones_b200 import ops
    z, ids, starts, u, q = _cuda(*problem([5, 4], 1000, 1000, torch.bfloat16, True))
    want = ops.verify_drafts(z, ids, starts, u, q)
    wide = torch.full((9, 1111), float("nan"), dtype=torch.bfloat16, device="cuda")
    for off in (0, 1, 7, 8):
        a, b = wide.clone(), wide.clone()
        a[:, off:off + 1000], b[:, 3:1003] = z, q
        got = ops.verify_drafts(a[:, off:], ids, starts, u, b[:, 3:], vocab=1000)
        assert torch.equal(got.accepted, want.accepted) and torch.equal(got.token, want.token)
    got = ops.verify_drafts(z.T.contiguous().T, ids, starts, u, q)
    assert torch.equal(got.token, want.token)


def test_equal_models_accept_every_draft():
    from them_bones_b200 import ops
    z, ids, starts, u, _ = _cuda(*problem([6, 6], 640, 640, torch.bfloat16, False))
    u[:, 0] = 1 - 2.0 ** -24
    assert ops.verify_drafts(z, ids, starts, u, z.clone(), 0.8).accepted.tolist() == [5, 5]


def test_captured_replayed_and_rows_behind():
    from them_bones_b200 import ops
    z, ids, starts, u, q = _cuda(*problem([4, 4, 4], 5000, 5000, torch.bfloat16, True))
    for t in (1.0, 0.0):
        ops.verify_drafts(z, ids, starts, u, q, t)
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = ops.verify_drafts(z, ids, starts, u, q, t)
            graphs.append((g, out))
        for s in ([0, 4, 8, 12], [0, 1, 1, 9], [2, 3, 12, 12], [0, 0, 0, 0]):
            starts.copy_(O.i32(s))
            want = ops.verify_drafts(z, ids, starts, u, q, t)
            ref = ops.verify_drafts(z.cpu(), ids.cpu(), starts.cpu(), u.cpu(), q.cpu(), t)
            assert torch.equal(want.accepted.cpu(), ref.accepted) and torch.equal(want.token.cpu(), ref.token)
            for g, out in graphs:
                out.token.fill_(-9)
                g.replay()
                assert torch.equal(out.accepted, want.accepted) and torch.equal(out.token, want.token)
        starts.copy_(O.i32([0, 4, 8, 12]))


def test_rows_past_31_bits():
    from them_bones_b200 import ops
    z = torch.zeros(35000, 65536, dtype=torch.bfloat16, device="cuda")            # 2.3e9 values
    z[34999, 65535], z[34998, 7], z[34997, 9] = 50.0, 50.0, 50.0
    ids = torch.zeros(35000, dtype=torch.int64, device="cuda")
    ids[34999], ids[34998] = 7, 9
    u = torch.full((35000, 2), 0.5, device="cuda")
    for t in (1.0, 0.0):
        got = ops.verify_drafts(z, ids, O.i32([34997, 35000], "cuda"), u, temperature=t)
        assert (int(got.accepted), int(got.token)) == (2, 65535)


def test_native_refusals():
    from them_bones_b200 import ops
    z = torch.zeros(2, 10, device="cuda")
    ids, starts, u = torch.zeros(2, dtype=torch.int64, device="cuda"), O.i32([0, 2], "cuda"), torch.zeros(2, 2, device="cuda")
    for bad in (dict(logits=z.half()), dict(logits=z.double()), dict(starts=starts.cpu()), dict(uniforms=u.cpu()), dict(ids=ids.cpu()), dict(draft_logits=z.cpu())):
        with pytest.raises(ValueError):
            ops.verify_drafts(**{**dict(logits=z, ids=ids, starts=starts, uniforms=u), **bad})


@pytest.mark.parametrize("t", [0.0, 0.7])
def test_calls_without_rows(t):
    from them_bones_b200 import ops
    for dtype in (torch.float32, torch.bfloat16):
        z = torch.zeros(0, 10, device="cuda", dtype=dtype)
        for q in (None, z):
            got = ops.verify_drafts(z, torch.zeros(0, dtype=torch.int64, device="cuda"), O.i32([0, 0, 0], "cuda"), torch.zeros(0, 2, device="cuda"), q, t)
            assert got.accepted.tolist() == [0, 0] and got.token.tolist() == [-1, -1]


def test_the_short_way_and_the_long_one_are_one_operator():
    from them_bones_b200 import ops
    from them_bones_b200.ops import verify as V
    for dtype, t in ((torch.float32, 0.7), (torch.bfloat16, 1.0), (torch.bfloat16, 0.0)):
        z, ids, starts, u, q = _cuda(*problem([3, 0, 5, 1], 900, 904, dtype, True))
        for draft in (q, None):
            a = (z, ids, starts, u, draft, t, 900)
            V.check(*a)
            got, want = V.short(*a), V.native(*a)
            assert got is not None and torch.equal(got.accepted, want.accepted) and torch.equal(got.token, want.token)
        one = ops.verify_drafts(z, ids, starts, u, q, 1, 900)                  # a whole number goes the long way
        assert torch.equal(one.token, ops.verify_drafts(z, ids, starts, u, q, 1.0, 900).token)
        a = [z, ids, starts, u, q, t, 900]
        for i, x in ((0, z.half()), (0, z[:, ::2]), (1, ids.int()), (1, ids[:-1]), (2, starts.long()), (2, starts[:1]), (4, q[:-1]), (4, q[:, :899]), (4, q.half()), (5, 1),
                     (5, float("nan")), (5, -1.0), (5, 1e-9), (6, 0), (6, 905), (6, True)):
            assert V.short(*a[:i], x, *a[i + 1:]) is None, (i, x)
        if t:
            for x in (None, u[:-1], u.double(), u.cpu()):
                assert V.short(*a[:3], x, *a[4:]) is None


def test_next_to_nothing_left_of_p_is_nothing():
    """p and q alike to 12 digits, and a draft that q would hardly ever give: the token is p's, not that of a rare column whose own weight is well above q's."""
    z = torch.tensor([[12.351143836975098, -0.10267984122037888, -0.30233708024024963, 4.481926441192627, -3.0466697216033936, 3.10713267326355, 0.4143826365470886]] * 2)
    q = torch.tensor([[12.44536018371582, -0.10847845673561096, -0.24057084321975708, 4.601906776428223, -2.91764235496521, 3.022629976272583, 0.4767337143421173]] * 2)
    for k in (0.01, 0.5, 0.77, 0.999):
        for rows, cols in ((z, 7), (torch.cat([z, z], 1), 14), (torch.nn.functional.pad(z, (0, 3000), value=-40.0), 3007)):
            if cols == 14 and k == 0.5:
                continue                                  # half of two equal halves is the border itself: no arithmetic says on which side
            draft = torch.cat([q, q], 1) if cols == 14 else torch.nn.functional.pad(q, (0, cols - 7), value=-40.0)
            u = torch.tensor([[0.9918550252914429, k], [0.5, 0.5]])
            _check(rows, torch.tensor([6, 4]), O.i32([0, 2]), u, draft, 0.3, cols)
