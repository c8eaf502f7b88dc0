"""The paged cache's kernels against 64 bits, and the calls where they can go wrong."""
import pytest
import torch

from tests import paged_oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_wait_ran_out():
    yield
    from them_bones_b200.ops import _lib as L
    L.check_error_word()


def _close(got, want, tol):
    far = ((got.double() - want).abs() - tol).max()
    assert bool(((got.double() - want).abs() <= tol).all()), f"{float(far)} beyond the tolerance"


CASES = [  # heads, head_dim, page, new tokens, positions
    (2, 64, 16, [1], [0]), (10, 128, 64, [1], [299]), (1, 128, 64, [1, 1, 1], [0, 63, 64]), (3, 64, 32, [5, 0, 33, 1], [10, 3, 100, 127]),
    (2, 128, 128, [130, 40], [0, 200]), (2, 64, 16, [17, 16, 1, 15], [15, 16, 300, 1]), (1, 64, 64, [3, 4, 2], [-1, 7, 0]),
    (5, 128, 16, [1] * 40, [37 * i for i in range(40)]), (9, 64, 64, [2, 9, 1, 16], [1500, 1023, 1024, 700]), (1, 128, 32, [300], [77]),
    (12, 128, 64, [0, 0, 1], [5, 0, 130])]


@pytest.mark.parametrize("h,d,page,lens,pos", CASES)
def test_append_is_the_formula(h, d, page, lens, pos):
    from them_bones_b200 import ops
    c, table, starts, at = O.world(len(lens), h, d, page, lens, pos, "cuda")
    n = int(starts[-1]) + 3
    qkv = torch.randn(n, 3 * h * d, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    cos, sin = O.angles(2048, d, "cuda")
    (q, k, v), (qt, kt) = O.append(qkv, cos, sin, c, table, starts, at)
    got = ops.paged_append(qkv, cos, sin, c, table, starts, at)
    _close(got, q, qt)
    _close(c.k, k, kt)
    assert torch.equal(c.v.double(), v)


@pytest.mark.parametrize("longest", [None, 1, 4096])
@pytest.mark.parametrize("window", [0, 128, 512])
@pytest.mark.parametrize("h,d,page,lens,pos", CASES)
def test_attention_is_the_formula(h, d, page, lens, pos, window, longest):
    from them_bones_b200 import ops
    c, table, starts, at = O.world(len(lens), h, d, page, lens, pos, "cuda")
    n = int(starts[-1]) + 2
    q = O.queries(n, h, d, "cuda")
    # starts in front of the sequence, on the way, and behind the token
    doc = O.i32([(0, 3, 64, 100, -7, 1 << 30)[(i // 3) % 6] for i in range(n)], "cuda")
    for ds in (None, doc):
        y, tol = O.attend(q, c, table, starts, at, d ** -0.5, ds, window)
        _close(ops.paged_attention(q, c, table, starts, at, d ** -0.5, ds, window, longest), y, tol)


@pytest.mark.parametrize("scale", [0.0, -0.1, 0.25])
@pytest.mark.parametrize("longest", [1, 4096])
def test_scales_of_either_sign(scale, longest):
    from them_bones_b200 import ops
    c, table, starts, at = O.world(2, 2, 128, 64, [20, 1], [100, 900], "cuda")
    q = O.queries(21, 2, 128, "cuda")
    y, tol = O.attend(q, c, table, starts, at, scale, None, 0)
    _close(ops.paged_attention(q, c, table, starts, at, scale, longest=longest), y, tol)


@pytest.mark.parametrize("h,d,page,lens,pos", [(10, 128, 128, [1, 1, 1, 1], [20000, 33333, 9000, 40]), (2, 64, 16, [5, 1, 16], [16384, 30000, 8200]),
                                               (1, 128, 64, [17], [60000]), (3, 64, 32, [1, 0, 2], [12000, 0, 3])])
@pytest.mark.parametrize("longest", [None, 4096])
def test_long_caches(h, d, page, lens, pos, longest):
    from them_bones_b200 import ops
    c, table, starts, at = O.world(len(lens), h, d, page, lens, pos, "cuda", room=5)
    n = int(starts[-1])
    q = O.queries(n, h, d, "cuda")
    doc = O.i32([0 if i % 2 else 5000 for i in range(n)], "cuda")
    for ds, window in ((None, 0), (doc, 0), (None, 16384)):
        y, tol = O.attend(q, c, table, starts, at, d ** -0.5, ds, window)
        got = ops.paged_attention(q, c, table, starts, at, d ** -0.5, ds, window, longest)
        _close(got, y, tol)
        assert torch.equal(got, ops.paged_attention(q, c, table, starts, at, d ** -0.5, ds, window, longest))


@pytest.mark.parametrize("longest", [1, 4096])
def test_positions_without_a_page_are_not_stored_and_not_seen(longest):
    from them_bones_b200 import ops
    c, table, starts, pos = O.world(3, 2, 64, 16, [40, 8, 150], [0, 30, 100], "cuda")
    table[0, 1], table[1, 0], table[2, 7], table[2, 0], table[0, 0] = -1, 99999, -1, 1 << 30, -1
    q = O.queries(198, 2, 64, "cuda")
    y, tol = O.attend(q, c, table, starts, pos, 0.1, None, 0)
    assert bool((y[:16] == 0).all())
    _close(ops.paged_attention(q, c, table, starts, pos, 0.1, longest=longest), y, tol)
    qkv, (cos, sin) = torch.randn(198, 384, device="cuda").bfloat16(), O.angles(300, 64, "cuda")
    (qq, k, v), (qt, kt) = O.append(qkv, cos, sin, c, table, starts, pos)
    _close(ops.paged_append(qkv, cos, sin, c, table, starts, pos), qq, qt)
    _close(c.k, k, kt)
    assert torch.equal(c.v.double(), v)


def test_what_lies_past_the_table_and_the_rotary_tables_is_left_out():
    from them_bones_b200 import ops
    c, table, starts, pos = O.world(2, 2, 64, 16, [20, 20], [0, 40], "cuda")
    table, pos = table[:, :3].contiguous(), O.i32([35, 2147483647], "cuda")               # 13 of the first fit; none of the second
    q = O.queries(40, 2, 64, "cuda")
    y, tol = O.attend(q, c, table, starts, pos, 0.1, None, 0)
    for longest in (1, 4096):
        got = ops.paged_attention(q, c, table, starts, pos, 0.1, longest=longest)
        _close(got, y, tol)
        assert bool((got[13:] == 0).all())
    qkv, (cos, sin) = torch.randn(40, 384, device="cuda").bfloat16(), O.angles(45, 64, "cuda")
    (qq, k, v), (qt, kt) = O.append(qkv, cos, sin, c, table, starts, pos)
    _close(ops.paged_append(qkv, cos, sin, c, table, starts, pos), qq, qt)
    _close(c.k, k, kt)
    assert torch.equal(c.v.double(), v) and bool((qq[10:] == 0).all())


@pytest.mark.parametrize("longest", [1, 4096])
@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("d", [64, 128])
def test_values_that_are_not_finite_reach_only_those_who_see_them(longest, page, d):
    from them_bones_b200 import ops
    c, table, starts, pos = O.world(3, 2, d, page, [150, 3, 20], [0, 299, 100], "cuda")
    q = O.queries(173, 2, d, "cuda")
    doc = O.i32([0] * 150 + [130] * 3 + [0] * 20, "cuda")
    want = ops.paged_attention(q, c, table, starts, pos, 0.1, doc, longest=longest)
    for i in range(3):                                          # behind every sequence's end: what a page held before
        end = int(pos[i] + starts[i + 1] - starts[i])
        if end % page:
            c.k[int(table[i, end // page]), :, end % page:] = float("nan")
            c.v[int(table[i, end // page]), :, end % page:] = float("inf")
    assert torch.equal(ops.paged_attention(q, c, table, starts, pos, 0.1, doc, longest=longest), want)
    put = lambda i, p, x, col: c.v[int(table[i, p // page]), :].select(1, p % page)[:, col].fill_(x)  # noqa: E731
    put(0, 70, float("inf"), 5)
    put(0, 140, float("nan"), 9)
    put(1, 129, float("-inf"), 11)                              # the document hides it
    put(1, 300, float("-inf"), 12)                              # the second of three new tokens
    c.k[int(table[2, 110 // page]), 0, 110 % page] = float("nan")        # a key: its readers' rows, in its head
    got = ops.paged_attention(q, c, table, starts, pos, 0.1, doc, longest=longest).view(173, 2, d)
    want = want.view(173, 2, d)
    row = torch.arange(150, device="cuda")
    assert torch.equal(got[:70], want[:70]) and bool((got[70:150, :, 5] == float("inf")).all()) and bool(got[140:150, :, 9].isnan().all())
    rest = [i for i in range(d) if i not in (5, 9)]
    assert torch.equal(got[:140][:, :, [i for i in range(d) if i != 5]], want[:140][:, :, [i for i in range(d) if i != 5]])
    assert bool(got[:150][:, :, rest].isfinite().all()) and row.numel() == 150
    assert torch.equal(got[150], want[150]) and bool((got[151:153, :, 12] == float("-inf")).all()) and bool(got[150:153, :, 11].isfinite().all())
    assert torch.equal(got[153:163], want[153:163]) and bool(got[163:, 0].isnan().all()) and torch.equal(got[163:, 1], want[163:, 1])


def test_norm_of_values_whose_squares_leave_fp32():
    from them_bones_b200 import ops
    c, table, starts, pos = O.world(1, 2, 128, 16, [6], [3], "cuda")
    cos, sin = O.angles(64, 128, "cuda")
    x = torch.randn(6, 3, 2, 128, device="cuda")
    x[0] *= 1e30
    x[1] *= 3e37
    x[2] *= 1e-30
    x[3, 0, 0] *= 1e25                                   # one head of the row
    x[4] = 0
    qkv = x.view(6, -1).bfloat16()
    (q, k, v), (qt, kt) = O.append(qkv, cos, sin, c, table, starts, pos)
    _close(ops.paged_append(qkv, cos, sin, c, table, starts, pos), q, qt + 1e-38)
    _close(c.k, k, kt + 1e-38)


def test_strided_rows_tables_and_unaligned_queries():
    from them_bones_b200 import ops
    h, d = 3, 64
    c, table, starts, pos = O.world(3, h, d, 32, [5, 1, 70], [60, 0, 10], "cuda")
    n = 76
    wide = torch.randn(n, 3 * h * d + 24, device="cuda").bfloat16()
    big = torch.full((3, table.shape[1] + 9), -5, dtype=torch.int32, device="cuda")
    big[:, 4:4 + table.shape[1]] = table
    cut = big[:, 4:4 + table.shape[1]]
    cos, sin = O.angles(128, d, "cuda")
    outs = []
    for qkv, t in ((wide[:, 8:8 + 3 * h * d], cut), (wide[:, 8:8 + 3 * h * d].contiguous(), table), (wide[:, 8:8 + 3 * h * d].contiguous()[:, :].clone(), cut)):
        outs.append((ops.paged_append(qkv, cos, sin, c, t, starts, pos), c.k.clone(), c.v.clone()))
    odd = torch.empty(n * 3 * h * d + 1, dtype=torch.bfloat16, device="cuda")[1:].view(n, -1).copy_(wide[:, 8:8 + 3 * h * d])          # on 2 bytes
    outs.append((ops.paged_append(odd, cos, sin, c, table, starts, pos), c.k.clone(), c.v.clone()))
    assert all(torch.equal(a, b) for o in outs[1:] for a, b in zip(o, outs[0]))
    q = outs[0][0]
    buf = torch.empty(n * h * d + 8, dtype=torch.bfloat16, device="cuda")
    ways = [q, torch.cat([q, q], 1)[:, :h * d], buf[1:1 + n * h * d].view(n, -1).copy_(q), q.repeat_interleave(2, 0)[::2]]
    for longest in (1, 4096):
        ys = [ops.paged_attention(x, c, t, starts, pos, 0.1, longest=longest) for x in ways for t in (table, cut)]
        assert all(torch.equal(y, ys[0]) for y in ys)


def test_shared_pages_and_the_same_page_twice():
    from them_bones_b200 import ops
    c, table, starts, pos = O.world(2, 2, 64, 16, [1, 30], [47, 90], "cuda")
    table[0, :3] = table[1, :3]
    table[1, 4] = table[1, 2]
    q = O.queries(31, 2, 64, "cuda")
    y, tol = O.attend(q, c, table, starts, pos, 0.1, None, 0)
    for longest in (1, 4096):
        _close(ops.paged_attention(q, c, table, starts, pos, 0.1, longest=longest), y, tol)


def test_rows_outside_all_pieces_are_zeros_and_empty_calls():
    from them_bones_b200 import ops
    c, table, starts, pos = O.world(2, 2, 64, 16, [3, 30], [0, 9], "cuda")
    late = starts + 4
    q = torch.full((45, 128), 1.0, device="cuda").bfloat16()
    for longest in (1, 4096):
        y = ops.paged_attention(q, c, table, late, pos, 0.1, longest=longest)
        assert bool((y[:4] == 0).all()) and bool((y[37:] == 0).all()) and bool((y[4:37] != 0).any(1).all())
        assert torch.equal(y[4:37], ops.paged_attention(q[:33], c, table, starts, pos, 0.1, longest=longest))
        # a piece that the rows cut off
        assert torch.equal(ops.paged_attention(q[:20], c, table, starts, pos, 0.1, longest=longest), y[4:24])
        assert ops.paged_attention(q[:0], c, table, starts * 0, pos, 0.1, longest=longest).shape == (0, 128)
    cos, sin = O.angles(64, 64, "cuda")
    before = c.k.clone()
    assert ops.paged_append(torch.zeros(0, 384, device="cuda").bfloat16(), cos, sin, c, table, starts * 0, pos).shape == (0, 128) and torch.equal(before, c.k)


def test_many_sequences_find_their_rows():
    from them_bones_b200 import ops
    lens = [(i * 7) % 4 for i in range(3000)]
    pos = [(i * 13) % 40 for i in range(3000)]
    c, table, starts, at = O.world(3000, 1, 64, 16, lens, pos, "cuda")
    n = int(starts[-1])
    qkv, (cos, sin) = torch.randn(n, 192, device="cuda").bfloat16(), O.angles(64, 64, "cuda")
    lot = ops.PagedKV(c.k.cpu(), c.v.cpu())
    want = ops.paged_append(qkv.cpu(), cos.cpu(), sin.cpu(), lot, table.cpu(), starts.cpu(), at.cpu())
    got = ops.paged_append(qkv, cos, sin, c, table, starts, at)
    assert torch.equal(c.v.cpu(), lot.v) and float((got.cpu().float() - want.float()).abs().max()) <= 2 ** -7 * 6     # one step of bf16 at values up to 6
    y = ops.paged_attention(O.queries(n, 1, 64, "cuda"), c, table, starts, at, 0.1)
    ref = ops.paged_attention(O.queries(n, 1, 64), ops.PagedKV(c.k.cpu(), c.v.cpu()), table.cpu(), starts.cpu(), at.cpu(), 0.1)
    assert float((y.cpu().float() - ref.float()).abs().max()) <= 3 * O.HALF * float(c.v.float().abs().max())


def test_captured_and_replayed_with_other_positions_and_on_another_stream():
    from them_bones_b200 import ops
    c, table, starts, pos = O.world(3, 2, 128, 64, [4, 4, 4], [700, 64, 300], "cuda")
    qkv, (cos, sin) = torch.randn(12, 768, device="cuda").bfloat16(), O.angles(1024, 128, "cuda")

    def step(longest):
        q = ops.paged_append(qkv, cos, sin, c, table, starts, pos)
        return ops.paged_attention(q, c, table, starts, pos, 0.08, longest=longest)

    for longest in (4, 4096):
        step(longest)
        graphs = []
        for _ in range(2):                                     # two graphs, replayed in turn and at once: they share no workspace
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = step(longest)
            graphs.append((g, out))
        for p, s in (([700, 64, 300], [0, 4, 8, 12]), ([5, 0, 1], [0, 1, 12, 12]), ([-1, 511, 2], [0, 4, 4, 9])):
            pos.copy_(O.i32(p))
            starts.copy_(O.i32(s))
            want = step(longest).clone()
            for g, out in graphs:
                out.fill_(7.0)
                g.replay()
                assert torch.equal(out, want)
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                got = step(longest)
            torch.cuda.current_stream().wait_stream(side)
            assert torch.equal(got, want)
        pos.copy_(O.i32([700, 64, 300]))
        starts.copy_(O.i32([0, 4, 8, 12]))


def test_pages_past_31_and_32_bits():
    from them_bones_b200 import ops
    c = ops.paged_cache(27000, 10, 128, 128, "cuda")            # 4.4e9 values each
    table = O.i32([[26999, 13106, 13107, 3], [26000, 1, 14000, 26998]], "cuda")
    for x in table.flatten().tolist():
        k = torch.randn(10, 128, 128, device="cuda")
        c.k[x] = k / k.square().mean(-1, keepdim=True).sqrt()
        c.v[x] = torch.randn(10, 128, 128, device="cuda")
    starts, pos = O.i32([0, 1, 41], "cuda"), O.i32([511, 460], "cuda")
    q = O.queries(41, 10, 128, "cuda")
    y, tol = _far(q, c, table, starts, pos, 0.08)
    for longest in (1, 4096):
        _close(ops.paged_attention(q, c, table, starts, pos, 0.08, longest=longest), y, tol)
    qkv, (cos, sin) = torch.randn(41, 3840, device="cuda").bfloat16(), O.angles(512, 128, "cuda")
    ops.paged_append(qkv, cos, sin, c, table, starts, pos)
    assert torch.equal(c.v[3, :, 127], qkv[0, 2560:].view(10, 128)) and torch.equal(c.v[26998, :, 115], qkv[40, 2560:].view(10, 128))
    assert torch.equal(c.v[26998, :, 76], qkv[1, 2560:].view(10, 128))
    del c
    torch.cuda.empty_cache()


def _far(q, c, table, starts, pos, scale):
    """The oracle on the pages in use alone."""
    ids = sorted(set(table.flatten().tolist()))
    from them_bones_b200 import ops
    small = ops.PagedKV(c.k[ids].clone(), c.v[ids].clone())
    return O.attend(q, small, O.i32([[ids.index(x) for x in row] for row in table.tolist()], "cuda"), starts, pos, scale, None, 0)


def test_the_same_bits_every_time():
    """Items of all kinds beside one another, often: what depended on which role came first would show."""
    from them_bones_b200 import ops
    lens, pos = [1, 300, 17, 128, 0, 5, 129, 64] * 4, [37 * i * (i % 5) for i in range(32)]
    c, table, starts, at = O.world(32, 5, 128, 16, lens, pos, "cuda")
    q = O.queries(sum(lens), 5, 128, "cuda")
    junk = torch.randint(-2 ** 31, 2 ** 31 - 1, (1 << 22,), dtype=torch.int32, device="cuda")
    want = {k: ops.paged_attention(q, c, table, starts, at, 0.1, longest=k) for k in (1, 4096)}
    y, tol = O.attend(q, c, table, starts, at, 0.1, None, 0)
    for k in (1, 4096):
        _close(want[k], y, tol)
    for i in range(300):
        junk += 1                                       # other kernels' leftovers in shared memory
        assert torch.equal(ops.paged_attention(q, c, table, starts, at, 0.1, longest=4096), want[4096])
        assert i % 10 or torch.equal(ops.paged_attention(q, c, table, starts, at, 0.1, longest=1), want[1])


def test_native_refusals():
    from them_bones_b200 import ops
    c, table, starts, pos = O.world(1, 1, 64, 16, [2], [0], "cuda")
    cos, sin = O.angles(16, 64, "cuda")
    with pytest.raises(ValueError):
        ops.paged_append(torch.zeros(2, 192, device="cuda"), cos, sin, c, table, starts, pos)
    with pytest.raises(ValueError):
        ops.paged_attention(O.queries(2, 1, 64, "cuda"), c, table, starts, pos, 0.6)
    with pytest.raises(ValueError):
        ops.paged_attention(O.queries(2, 1, 64, "cuda"), c, table.cpu(), starts, pos, 0.1)
    f = ops.paged_cache(3, 1, 64, 16, "cuda", torch.float32)
    with pytest.raises(ValueError):
        ops.paged_attention(torch.zeros(2, 64, device="cuda"), f, table, starts, pos, 0.1)


def test_a_run_of_pieces_is_the_training_attention():
    """A prompt in pieces of any length gives what ``ops.attention`` gives for all of it at once."""
    from them_bones_b200 import ops
    h, d, t = 4, 128, 700
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(1, t, 3 * h * d, generator=g).bfloat16().cuda()
    cos, sin = O.angles(t, d, "cuda")
    doc = O.i32([i // 211 * 211 for i in range(t)], "cuda")
    for window in (0, 256):
        want = ops.attention(qkv, cos, sin, h, d, d ** -0.5, doc.view(1, t), window)[0].float()
        c, m = ops.paged_cache(30, h, d, 32, "cuda"), 22
        table = torch.randperm(30, generator=g)[:m].int().view(1, m).cuda()
        p, out = 0, []
        for n in (1, 5, 16, 17, 100, 1, 200, 360):
            args = (c, table, O.i32([0, n], "cuda"), O.i32([p], "cuda"))
            q = ops.paged_append(qkv[0, p:p + n], cos, sin, *args)
            out.append(ops.paged_attention(q, *args, d ** -0.5, doc[p:p + n].contiguous(), window, longest=n))
            p += n
        # both round probabilities and results to bf16: 2^-8 of sums of |v| (up to 4 here at weights' sum 1) and of the result, each
        assert p == t and float((torch.cat(out).float() - want).abs().max()) <= 4 * O.HALF * 4


@pytest.mark.parametrize("longest", [1, 4096])
def test_windows_and_documents_beyond_all_positions(longest):
    """Windows whose tokens or tiles leave 32 bits hide nothing, and neither does a document that began far in front of its sequence."""
    from them_bones_b200 import ops
    c, table, starts, pos = O.world(3, 2, 64, 16, [3, 40, 1], [200, 300, 0], "cuda")
    q = O.queries(44, 2, 64, "cuda")
    want = ops.paged_attention(q, c, table, starts, pos, 0.1, longest=longest)
    for window in (1 << 31, 1 << 32, 128 * ((1 << 25) + 1), 1 << 37, 128 * ((1 << 32) + 1), 1 << 45):
        assert torch.equal(ops.paged_attention(q, c, table, starts, pos, 0.1, None, window, longest), want), window
    doc = O.i32([-2 ** 31, -2 ** 31 + 1, -1, 0] * 11, "cuda")
    assert torch.equal(ops.paged_attention(q, c, table, starts, pos, 0.1, doc, 0, longest), want)


@pytest.mark.parametrize("longest", [1, 4096])
@pytest.mark.parametrize("window", [0, 256])
def test_positions_next_to_the_last_of_32_bits(window, longest):
    """A table of 2^31 - 128 positions of which the last three pages are there: as three pages at the start."""
    from them_bones_b200 import ops
    m = (1 << 24) - 1
    c, near, starts, _ = O.world(1, 1, 64, 128, [20], [364], "cuda")
    table = torch.full((1, m), -1, dtype=torch.int32, device="cuda")
    table[0, -3:] = near[0, :3]
    off = (m - 3) * 128
    q = O.queries(20, 1, 64, "cuda")
    doc = O.i32([off + 10 * i for i in range(20)], "cuda")
    for at, ds in ((364, None), (300, doc)):
        y, tol = O.attend(q, c, near, starts, O.i32([at], "cuda"), 0.1, None if ds is None else ds - off, window)
        _close(ops.paged_attention(q, c, table, starts, O.i32([off + at], "cuda"), 0.1, ds, window, longest), y, tol)


def test_calls_whose_turns_leave_32_bits_go_by_the_larger_tiles():
    from them_bones_b200.ops import _lib as L
    room = lambda n, cap, tall: L.load().bones_paged_room(1, n, cap, 1, 64, 0, tall, 148)  # noqa: E731
    far = (1 << 31) - 128
    assert room(15, far, 0) == room(15, 4096, 0) != room(15, far, 1)
    assert room(1000, 1 << 20, 0) == room(1000, 4096, 0) and room(1000, far, 0) == room(1000, far, 1) != room(1000, 4096, 0)


def test_the_short_way_and_the_long_one_are_one_operator():
    """Calls that Python checks and launches give the bits of those that it does not; what the short way does not take it leaves alone."""
    from them_bones_b200 import ops
    from them_bones_b200.ops import paged as P
    for h, d, page, lens, pos in ((2, 64, 16, [5, 0, 33, 1], [10, 3, 100, 127]), (10, 128, 64, [1, 4], [299, 2000])):
        c, table, starts, at = O.world(len(lens), h, d, page, lens, pos, "cuda")
        n = int(starts[-1])
        qkv, (cos, sin) = torch.randn(n, 3 * h * d, device="cuda").bfloat16(), O.angles(4096, d, "cuda")
        a = (qkv, cos, sin, c, table, starts, at)
        q = P.short_append(*a)
        k = c.k.clone()
        assert q is not None and torch.equal(q, P.append(P.check_append(*a), *a)) and torch.equal(k, c.k)
        doc = O.i32([3] * n, "cuda")
        for ds in (None, doc):
            for window in (0, 128):
                for longest in (None, 1, 4096):
                    b = (q, c, table, starts, at, d ** -0.5, ds, window, longest)
                    y = P.short_attention(*b)
                    assert y is not None and torch.equal(y, P.attention(P.check_attention(*b), *b))
        assert torch.equal(ops.paged_attention(q, c, table, starts, at, 0), ops.paged_attention(q, c, table, starts, at, 0.0))          # a whole number
        before = c.k.clone()
        for bad in ((qkv.float(), *a[1:]), (qkv[:, 1:], *a[1:]), (qkv, cos.double(), *a[2:]), (*a[:3], ops.PagedKV(c.k, c.v[:-1]), *a[4:]), (*a[:4], table.long(), *a[5:]),
                    (*a[:5], starts[:-1], at), (*a[:6], at.cpu()), (torch.nn.Parameter(qkv), *a[1:])):
            assert P.short_append(*bad) is None
        for i, x in ((0, q.float()), (0, q[:, :-1]), (5, 33.0 / d), (5, float("nan")), (5, 1), (6, doc.long()), (6, doc[:-1]), (7, 100), (7, -128), (7, True), (8, -1),
                     (8, 1 << 80), (8, 1.0)):
            b = [q, c, table, starts, at, 0.1, None, 0, None]
            b[i] = x
            assert P.short_attention(*b) is None, (i, x)
        assert torch.equal(before, c.k)


def test_the_same_call_on_two_streams_at_once():
    from them_bones_b200 import ops
    worlds = [O.world(4, 2, 64, 16, [1, 40, 3, 200], [500, 30 + i, 0, 77], "cuda", seed=i) for i in range(2)]
    qs = [O.queries(244, 2, 64, "cuda").roll(i, 0) for i in range(2)]
    run = lambda i, k: ops.paged_attention(qs[i], *worlds[i], 0.1, longest=k)  # noqa: E731
    for k in (1, 4096):
        want = [run(i, k) for i in range(2)]
        torch.cuda.synchronize()
        streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
        for _ in range(40):
            for i, s in enumerate(streams):
                with torch.cuda.stream(s):
                    got[i].append(run(i, k))
        torch.cuda.synchronize()
        assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])
