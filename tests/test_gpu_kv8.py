"""The 8-bit cache's kernels: codes bit for bit against the statement, attention against 64 bits, and the calls where they can go wrong."""
import pytest
import torch

from tests import kv8_oracle as O

pytestmark = pytest.mark.gpu


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _ref(cache):
    from them_bones_b200 import ops
    return ops.KV8(*(x.clone() for x in cache))


def _same(a, b):
    """Equal bits (scales of blocks with a value that is not finite are -0.0 or negative; codes and tails are compared as integers)."""
    return all(torch.equal(x.view(torch.int16) if x.dtype == torch.bfloat16 else x.view(torch.int32) if x.dtype == torch.float32 else x,
                           y.view(torch.int16) if y.dtype == torch.bfloat16 else y.view(torch.int32) if y.dtype == torch.float32 else y) for x, y in zip(a, b))


def _random_cache(b, h, d, cap, seed=0):
    """Codes, scales and open tokens at random: every block distinct."""
    from them_bones_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = ops.kv8_cache(b, cap, h, d, "cuda")
    for x in c[:2]:
        x.copy_((torch.randn(x.shape, device="cuda", generator=g, dtype=torch.float16) * 40).clamp_(-127, 127).round_())
    for x in c[2:4]:
        x.copy_(0.02 + 0.02 * torch.rand(x.shape, device="cuda", generator=g))
    for x in c[4:]:
        x.copy_(torch.randn(x.shape, device="cuda", generator=g))
    return c


@pytest.mark.parametrize("b,h,d,cap,t,pos,lens", [
    (1, 1, 128, 64, 1, 0, None), (1, 3, 64, 128, 64, 64, None), (2, 2, 128, 320, 200, 100, None), (3, 2, 64, 256, 1, [63, 64, 255], None),
    (5, 2, 128, 512, 130, [0, 62, 64, 300, 382], [130, 2, 129, 130, 130]), (6, 1, 64, 256, 70, [10, 0, -1, 200, 186, 190], [54, 0, 70, 70, 70, 66]),
    (4, 3, 128, 1024, 1000, [1, 24, 0, 0], [1000, 1000, 999, 0]), (2, 1, 64, 128, 40, [120, 88], [8, 40])])
def test_append_leaves_the_statement_s_bits(b, h, d, cap, t, pos, lens):
    from them_bones_b200 import ops
    from them_bones_b200.ref import functional as RF
    torch.manual_seed(t)
    got = _random_cache(b, h, d, cap)
    want = _ref(got)
    k, v = torch.randn(2, b, t, h, d, device="cuda").bfloat16()
    k[0, 0, 0, :3] = torch.tensor([float("nan"), float("inf"), float("-inf")])
    p, n = (pos if isinstance(pos, int) else _i32(pos)), (None if lens is None else _i32(lens))
    ops.kv8_append(got, k, v, p, n)
    RF.kv8_append(want, k, v, ops._kv8.numbers(p, b), ops._kv8.numbers(t if n is None else n, b))
    assert _same(got, want)
    held = [max(0, q) + (t if lens is None else lens[i]) for i, q in enumerate([pos] * b if isinstance(pos, int) else pos)]
    held = [min(x, cap) for x in held]
    for length in (cap, 1, cap - 37):
        for x, y in zip(ops.kv8_read(got, _i32(held), length), RF.kv8_read(want, held, length)):
            assert x.shape == (b, length, h, d) and torch.equal(x.isnan(), y.isnan()) and torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0))


@pytest.mark.parametrize("form", ["packed", "transposed", "odd", "expanded"])
def test_append_reads_keys_and_values_where_they_lie(form):
    from them_bones_b200 import ops
    b, t, h, d = 2, 150, 3, 64
    torch.manual_seed(9)
    x = torch.randn(b, t, 3 * h * d + 1, device="cuda").bfloat16()
    if form == "packed":
        packed = x[..., :-1].contiguous()
        k, v = (packed[..., i * h * d:(i + 1) * h * d].view(b, t, h, d) for i in (1, 2))
    elif form == "transposed":
        k, v = (x[..., i:i + h * d].reshape(b, t, h, d).transpose(1, 2).contiguous().transpose(1, 2) for i in (0, 5))
    elif form == "odd":
        k, v = (x[..., i:i + h * d].unflatten(-1, (h, d)) for i in (1, h * d + 1))
    else:
        k, v = (x[:1, :, i:i + d].reshape(1, t, 1, d).expand(b, t, h, d) for i in (0, 64))
    got, want = ops.kv8_cache(b, 192, h, d, "cuda"), ops.kv8_cache(b, 192, h, d, "cuda")
    ops.kv8_append(got, k, v, 3)
    ops.kv8_append(want, k.contiguous(), v.contiguous(), 3)
    assert _same(got, want) and got.k.any()


def _attend_case(b, h, d, cap, pos, start, window, scale=0.09, seed=0, rows=None, shared=False):
    from them_bones_b200 import ops
    from them_bones_b200.ref import functional as RF
    torch.manual_seed(seed)
    cache = _random_cache(b, h, d, cap, seed)
    before = _ref(cache)
    cos, sin = (x.cuda() for x in RF.rotary_tables(rows or cap, d, 10000.0))
    qkv = torch.randn(b, 3 * h * d, device="cuda").bfloat16()
    at = pos if isinstance(pos, list) else [pos] * b
    p = pos if isinstance(pos, int) else _i32(pos[:1] if shared else pos)
    ds = None if start is None else _i32(start)
    y = ops.kv8_attention(qkv, cos, sin, cache, p, scale, ds, window).double().view(b, h, d)
    live = [q for q in range(b) if 0 <= at[q] < min(cap, rows or cap)]
    # what the step left behind: its own token, nothing else; full blocks as the append makes them
    want = _ref(before)
    new_k = torch.zeros(b, h, d, dtype=torch.bfloat16, device="cuda")
    for q in live:
        slot = at[q] % 64
        new_k[q] = cache.k_open[q, :, slot]
        k64, v64 = O.new_rows(qkv[q], cos, sin, at[q], h, d)[1:]
        # one rounding to bf16 behind a few of fp32
        assert bool(((new_k[q].double() - k64).abs() <= (2 ** -8 + 2 ** -18) * k64.abs() + 2 ** -20).all())
        want.k_open[q, :, slot], want.v_open[q, :, slot] = new_k[q], v64.bfloat16()
        if slot == 63:
            for src, codes, scales in ((want.k_open, want.k, want.k_scale), (want.v_open, want.v, want.v_scale)):
                c, s = RF.kv8_quantise(src[q])
                if codes is want.k:
                    codes[q, :, at[q] - 63:at[q] + 1] = c
                else:
                    codes[q, :, at[q] // 64] = c.transpose(-1, -2)
                scales[q, :, at[q] // 64] = s
    assert _same(cache, want)
    ref, most = O.attend(qkv, cos, sin, before, new_k, at, scale, ds, window)
    # the result's rounding to bf16; fp32 scores of size scale * |q| |k| <= scale * 16 d off by 32 roundings (a sum in parts of 32 at most),
    # which moves a probability by twice that; probabilities of 11 bits or more and their sums
    tol = 2 ** -8 * ref.abs() + (2 * scale * 16 * d * 32 * 2 ** -24 + 2 ** -11) * most[:, None, None]
    assert bool(((y - ref).abs() <= tol).all()), float(((y - ref).abs() - tol).max())
    return y


@pytest.mark.parametrize("b,h,d,cap,pos,start,window", [
    (1, 1, 128, 64, 0, None, 0), (1, 1, 64, 64, 0, None, 0), (2, 3, 128, 128, [63, 64], None, 0), (2, 3, 64, 128, [62, 127], None, 0),
    (1, 10, 128, 320, 299, None, 0), (7, 4, 64, 2048, [0, 1, 63, 64, 65, 1000, 2047], None, 0), (7, 2, 128, 2048, [0, 1, 63, 64, 65, 1000, 2047], None, 0),
    (5, 2, 128, 512, [300, 300, 300, 300, 300], [0, 1, 255, 256, 300], 0), (5, 2, 64, 512, [319, 319, 319, 319, 319], [0, 63, 64, 319, 318], 0),
    (6, 2, 128, 1024, [100, 127, 128, 500, 639, 1023], None, 128), (6, 2, 64, 1024, [100, 127, 128, 500, 639, 1023], [0, 100, 128, 499, 0, 600], 256),
    (1, 1, 128, 16384, 16000, None, 0), (2, 5, 128, 8192, [8191, 4000], [0, 3999], 0), (3, 3, 64, 8192, [8191, 6000, 10], None, 0),
    (64, 10, 128, 256, list(range(100, 164)), None, 0), (200, 3, 64, 128, [i % 128 for i in range(200)], [i % 64 for i in range(200)], 0)])
def test_attention(b, h, d, cap, pos, start, window):
    _attend_case(b, h, d, cap, pos, start, window)


@pytest.mark.parametrize("b,h,d,cap,pos,start,window", [
    (1, 2, 128, 32768, [32767], None, 0), (1, 10, 64, 32768, [40], None, 0), (1, 1, 128, 32832, [0], None, 0), (1, 3, 128, 65536, [65000], [64001], 0),
    (2, 3, 64, 16384, [16383, 16320], None, 0), (4, 3, 128, 16384, [5, 16383, 9000, 16384], [0, 16000, 9001, 0], 0), (6, 2, 64, 16384, [-1, -1, 63, 64, 16000, 1 << 30], None, 0),
    (32, 1, 128, 16384, [500 * i + 63 for i in range(32)], [i * i for i in range(32)], 0), (33, 1, 64, 16384, [500 * i for i in range(32)] + [16383], None, 0),
    (3, 10, 128, 40960, [40000, 39935, 127], None, 32768), (2, 2, 64, 32768, [30000, 200], [0, 100], 128), (16, 10, 64, 16384, [1000 * i + 300 for i in range(16)], None, 0),
    (17, 10, 64, 16384, [900 * i for i in range(17)], None, 0)])
def test_long_caches(b, h, d, cap, pos, start, window):
    """On both sides of where all heads and sequences share the CTAs in equal parts."""
    _attend_case(b, h, d, cap, pos, start, window)


def test_long_caches_one_position():
    _attend_case(1, 3, 128, 40000, 39990, None, 0)
    _attend_case(3, 2, 64, 20000 // 64 * 64, 19000, [0, 18999, 19000], 0)
    y = _attend_case(2, 2, 128, 16384, [-1, 16384], None, 0)
    assert not y.any()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_long_caches_values_that_are_not_finite(d, bad):
    """A key and a value of head 1 somewhere in the middle: who sees them has no number, others the bits they had without."""
    from them_bones_b200 import ops
    from them_bones_b200.ref import functional as RF
    torch.manual_seed(6)
    b, h, n = 4, 2, 16384
    k, v = torch.randn(2, b, 9000, h, d, device="cuda").bfloat16()
    cos, sin = (x.cuda() for x in RF.rotary_tables(n, d, 10000.0))
    qkv = torch.randn(b, 3 * h * d, device="cuda").bfloat16()
    at, start = _i32([8990, 8990, 8990, 70]), _i32([8000, 7000, 4097, 0])
    out = []
    for dirty in (False, True):
        if dirty:
            k[:, 7000, 1, 3], v[:, 4096, 1, 5] = bad, bad
        cache = ops.kv8_cache(b, n, h, d, "cuda")
        ops.kv8_append(cache, k, v, 0)
        out.append(ops.kv8_attention(qkv, cos, sin, cache, at, 0.1, start).view(b, h, d))
    clean, y = out
    assert torch.equal(y[:, 0], clean[:, 0]) and torch.equal(y[[0, 3]], clean[[0, 3]])
    assert bool(y[1:3, 1].isnan().all())
    cache.k[:, 1].view(b, n // 64, 64, d)[:, 7000 // 64, 7000 % 64] = 1           # the value alone
    cache.k_scale[:, 1, 7000 // 64] = 0.02
    y = ops.kv8_attention(qkv, cos, sin, cache, at, 0.1, _i32([4096] * 4)).view(b, h, d)
    assert bool(y[:3, 1, 5].isnan().all()) and bool(y[:3, 1, :5].isfinite().all()) and bool(y[:3, 1, 6:].isfinite().all())


def test_long_caches_captured_replayed_and_on_two_streams():
    """Each call's parts are its own: two graphs over two caches replayed side by side, and calls on two streams, give the bits of calls alone."""
    from them_bones_b200 import ops
    from them_bones_b200.ref import functional as RF
    torch.manual_seed(17)
    b, h, d, cap, n = 2, 4, 128, 32768, 40
    cos, sin = (x.cuda() for x in RF.rotary_tables(cap, d, 10000.0))
    qkv = torch.randn(n, b, 3 * h * d, device="cuda").bfloat16()
    at = _i32([[30000 + i, 20000 + 64 * i] for i in range(n)])
    start = _random_cache(b, h, d, cap, 5)
    caches = [_ref(start) for _ in range(4)]
    want = [ops.kv8_attention(qkv[i], cos, sin, caches[0], at[i].clone(), 0.1) for i in range(n)]
    graphs = []
    for c in caches[1:3]:
        pos, x = at[0].clone(), qkv[0].clone()
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            y = ops.kv8_attention(x, cos, sin, c, pos, 0.1)
        graphs.append((g, pos, x, y))
    streams, outs = [torch.cuda.Stream() for _ in range(3)], [[], [], []]
    torch.cuda.synchronize()
    for i in range(n):
        for (g, pos, x, y), s, out in zip(graphs, streams, outs):
            with torch.cuda.stream(s):
                x.copy_(qkv[i])
                pos.copy_(at[i])
                g.replay()
                out.append(y.clone())
        with torch.cuda.stream(streams[2]):
            outs[2].append(ops.kv8_attention(qkv[i], cos, sin, caches[3], at[i].clone(), 0.1))
    torch.cuda.synchronize()
    for out, c in zip(outs, caches[1:]):
        assert all(torch.equal(a, w) for a, w in zip(out, want)) and _same(c, caches[0])


@pytest.mark.parametrize("b,h,d,cap,pos,start", [(5, 2, 128, 256, 191, None), (130, 5, 64, 256, 191, None), (64, 10, 128, 320, 300, "some"), (90, 8, 128, 128, 63, None),
                                                  (500, 1, 64, 128, 5, None), (64, 9, 64, 1024, 990, "some"), (64, 9, 64, 2048, 1990, "some")])
def test_one_position_for_all(b, h, d, cap, pos, start):
    """Also as many sequences as the kernel has a form of its own for."""
    _attend_case(b, h, d, cap, [pos] * b, None if start is None else [i * pos // b for i in range(b)], 0, shared=True)


def test_sequences_outside_and_queries_that_see_nothing():
    y = _attend_case(6, 2, 128, 256, [-1, 256, 200, 100, 199, 63], [0, 0, 0, 101, 1 << 30, 64], 0, rows=200)
    assert not y.any()


@pytest.mark.parametrize("scale", [0.0, 1.0, 30.0])
def test_scales(scale):
    """Scores of a few thousand: all of the probability in one key, the others' exponentials 0."""
    if scale <= 1.0:
        _attend_case(2, 2, 128, 512, [500, 447], None, 0, scale=scale)
        return
    from them_bones_b200 import ops
    from them_bones_b200.ref import functional as RF
    torch.manual_seed(2)
    cache, h, d = _random_cache(1, 2, 128, 512, 3), 2, 128
    cos, sin = (x.cuda() for x in RF.rotary_tables(512, d, 10000.0))
    qkv = torch.randn(1, 3 * h * d, device="cuda").bfloat16()
    before = _ref(cache)
    y = ops.kv8_attention(qkv, cos, sin, cache, 500, scale).double().view(h, d)
    q, _, v = O.new_rows(qkv[0], cos, sin, 500, h, d)
    k_all, v_all = O.held(before, 0, 500)
    k_all, v_all = torch.cat([k_all, cache.k_open[0, :, 500 % 64].double()[:, None]], 1), torch.cat([v_all, v[:, None]], 1)
    s = torch.einsum("hd,hnd->hn", q, k_all) * scale
    top = s.topk(2, 1)
    for i in range(h):
        if float(top.values[i, 0] - top.values[i, 1]) > 20:
            w = v_all[i, top.indices[i, 0]]
            assert bool(((y[i] - w).abs() <= 2 ** -8 * w.abs() + 2 ** -11 * v_all.abs().max()).all())
    assert bool(y.isfinite().all())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bits", [10.5, 17.5, 25.5, 30.5])
def test_many_small_probabilities_beside_a_large_one(bits, d):
    """One key with a score `bits` above all others' and value 0, the others' value 1: the result is what the others weigh together."""
    from them_bones_b200 import ops
    b, h, n = 32, 10, 1990
    eye, none = torch.ones(n + 1, d // 2, device="cuda"), torch.zeros(n + 1, d // 2, device="cuda")           # a rotation by nothing
    k, v = torch.zeros(b, n, h, d, device="cuda", dtype=torch.bfloat16), torch.ones(b, n, h, d, device="cuda", dtype=torch.bfloat16)
    k[..., d // 2:] = 1
    peak = [(61 * i) % 1900 for i in range(b)]
    for i, p in enumerate(peak):
        k[i, p, :, :d // 2], k[i, p, :, d // 2:], v[i, p] = 1, 0, 0
    cache = ops.kv8_cache(b, n + 1, h, d, "cuda")
    ops.kv8_append(cache, k, v, 0)
    qkv = torch.zeros(b, 3, h, d, device="cuda", dtype=torch.bfloat16)
    qkv[:, 0, :, :d // 2], qkv[:, 1, :, d // 2:], qkv[:, 2] = 1, 1, 1
    top = d // 2 * 2 ** 0.5                                                                # the query's norm makes its ones sqrt(2); a query sees its own key as the others
    y = ops.kv8_attention(qkv.view(b, -1), eye, none, cache, n, bits * 0.6931471805599453 / top)
    w = n * 2.0 ** -bits
    # rounding to bf16 2^-8 at most; scores of 31 bits with 2^-20 of them 2^-15; probabilities by 2^-11 at most as fp16 (2^(15 - 30.5) is 362.04 of its smallest steps)
    assert float((y.double() / (w / (1 + w)) - 1).abs().max()) <= 2 ** -8 + 2 ** -11 + 2 ** -14


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_values_that_are_not_finite_reach_who_sees_them_only(d, bad):
    from them_bones_b200 import ops
    from them_bones_b200.ref import functional as RF
    torch.manual_seed(5)
    b, h, n = 4, 2, 200
    k, v = torch.randn(2, b, n, h, d, device="cuda").bfloat16()
    clean = ops.kv8_cache(b, n + 8, h, d, "cuda")
    ops.kv8_append(clean, k, v, 0)
    for x, rows in ((k, (0, 70, 198)), (v, (1, 71, 195))):                 # full blocks and the open one
        for r in rows:
            x[:, r, 1] = bad
    cache = ops.kv8_cache(b, n + 8, h, d, "cuda")
    ops.kv8_append(cache, k, v, 0)
    cos, sin = (x.cuda() for x in RF.rotary_tables(n + 8, d, 10000.0))
    qkv = torch.randn(b, 3 * h * d, device="cuda").bfloat16()
    start = _i32([72, 199, 71, 0])
    y, want = (ops.kv8_attention(qkv, cos, sin, c, n, 0.1, start).view(b, h, d) for c in (cache, clean))
    assert bool(y[:, 0].isfinite().all()) and bool(y[1].isfinite().all()) and torch.equal(y[1], want[1])
    for i in (2, 3):
        assert not y[i, 1].isfinite().all()
    # head 0 holds none of them, but its blocks' scales are its own
    assert torch.equal(y[:, 0], want[:, 0])
    for c in (cache, clean):                                                # behind the open block's: only full blocks are left to see
        c.k_open[:, :, :n % 64 + 1].zero_()
        c.v_open[:, :, :n % 64 + 1].zero_()
    y2 = ops.kv8_attention(qkv, cos, sin, cache, n, 0.1, _i32([72, 72, 72, 72])).view(b, h, d)
    assert bool(y2.isfinite().all())


def test_a_step_that_fills_a_block_of_values_that_are_not_finite():
    from them_bones_b200 import ops
    from them_bones_b200.ref import functional as RF
    cache = ops.kv8_cache(1, 128, 1, 64, "cuda")
    cache.k_open.normal_()
    cache.v_open.normal_()
    cache.v_open[0, 0, 5, 7] = float("nan")
    cos, sin = (x.cuda() for x in RF.rotary_tables(128, 64, 10000.0))
    qkv = torch.randn(1, 192, device="cuda").bfloat16()
    y = ops.kv8_attention(qkv, cos, sin, cache, 63, 0.1, _i32([6]))
    assert bool(y.isfinite().all()) and int(cache.v[0, 0, 0, 7, 5]) == -128 and bool(cache.v_scale.signbit()[0, 0, 0]) and not cache.k_scale.signbit().any()
    assert int((cache.v[0, 0, 0] == -128).sum()) == 1


@pytest.mark.parametrize("d", [64, 128])
def test_steps_and_one_run_leave_one_cache(d):
    """Token by token through the attention, or its keys and values appended in one run: the same codes."""
    from them_bones_b200 import ops
    from them_bones_b200.ref import functional as RF
    torch.manual_seed(6)
    b, h, n = 3, 2, 140
    cos, sin = (x.cuda() for x in RF.rotary_tables(n, d, 10000.0))
    qkv = torch.randn(n, b, 3 * h * d, device="cuda").bfloat16()
    steps, run = (ops.kv8_cache(b, n, h, d, "cuda") for _ in range(2))
    keys = []
    pos = torch.zeros(1, dtype=torch.int32, device="cuda")
    for i in range(n):
        ops.kv8_attention(qkv[i], cos, sin, steps, pos, 0.1)
        keys.append(steps.k_open[:, :, i % 64].clone())
        pos += 1
    ops.kv8_append(run, torch.stack(keys, 1), qkv[..., 2 * h * d:].transpose(0, 1).unflatten(-1, (h, d)), 0)
    assert _same(steps[:4], run[:4])
    for x, y in zip(ops.kv8_read(steps, n, n), ops.kv8_read(run, n, n)):
        assert torch.equal(x, y)


def test_captured_and_replayed():
    """A captured step reads its position, and two graphs over two caches do not share anything."""
    from them_bones_b200 import ops
    from them_bones_b200.ref import functional as RF
    torch.manual_seed(7)
    b, h, d, n = 2, 3, 128, 70
    cos, sin = (x.cuda() for x in RF.rotary_tables(128, d, 10000.0))
    qkv = torch.randn(n, b, 3 * h * d, device="cuda").bfloat16()
    eager = ops.kv8_cache(b, 128, h, d, "cuda")
    want = [ops.kv8_attention(qkv[i], cos, sin, eager, i, 0.1).clone() for i in range(n)]
    graphs = []
    for _ in range(2):
        cache, pos, x = ops.kv8_cache(b, 128, h, d, "cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"), qkv[0].clone()
        ops.kv8_attention(x, cos, sin, cache, pos, 0.1)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = ops.kv8_attention(x, cos, sin, cache, pos, 0.1)
            pos.add_(1)
        graphs.append((g, cache, x, y))
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    torch.cuda.synchronize()
    for i in range(n):
        for (g, _, x, y), s, out in zip(graphs, streams, outs):
            with torch.cuda.stream(s):
                x.copy_(qkv[i])
                g.replay()
                out.append(y.clone())
    torch.cuda.synchronize()
    for (_, cache, _, _), out in zip(graphs, outs):
        assert all(torch.equal(a, w) for a, w in zip(out, want)) and _same(cache, eager)


def test_on_another_stream_and_from_a_new_thread():
    import threading
    from them_bones_b200 import ops
    from them_bones_b200.ref import functional as RF
    torch.manual_seed(8)
    cos, sin = (x.cuda() for x in RF.rotary_tables(256, 64, 10000.0))
    qkv = torch.randn(3, 3 * 2 * 64, device="cuda").bfloat16()
    a, c, e = (_random_cache(3, 2, 64, 256, 4) for _ in range(3))
    want = ops.kv8_attention(qkv, cos, sin, a, 200, 0.1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.kv8_attention(qkv, cos, sin, c, 200, 0.1)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    torch.cuda.synchronize()
    box = []
    t = threading.Thread(target=lambda: box.append(ops.kv8_attention(qkv, cos, sin, e, 200, 0.1)))
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert torch.equal(box[0], want)


def test_the_same_bits_on_every_call():
    from them_bones_b200 import ops
    from them_bones_b200.ref import functional as RF
    torch.manual_seed(11)
    b, h, d, cap = 2, 5, 128, 8192
    cos, sin = (x.cuda() for x in RF.rotary_tables(cap, d, 10000.0))
    qkv = torch.randn(b, 3 * h * d, device="cuda").bfloat16()
    cache = _random_cache(b, h, d, cap, 1)
    first = ops.kv8_attention(qkv, cos, sin, cache, _i32([8190, 3000]), 0.1)
    for _ in range(20):
        assert torch.equal(ops.kv8_attention(qkv, cos, sin, cache, _i32([8190, 3000]), 0.1), first)


def test_rows_of_a_larger_tensor_and_other_table_types():
    from them_bones_b200 import ops
    from them_bones_b200.ref import functional as RF
    torch.manual_seed(12)
    h, d = 2, 64
    cos, sin = (x.cuda() for x in RF.rotary_tables(128, d, 10000.0))
    cos, sin = cos.bfloat16(), sin.bfloat16()
    big = torch.randn(6, 3 * h * d + 5, device="cuda").bfloat16()
    for view in (big[::2, :-5], big[:3, 1:-4], big[:3, 5:]):
        a, c = (_random_cache(3, h, d, 128, 4) for _ in range(2))
        got = ops.kv8_attention(view, cos, sin, a, 100, 0.1)
        want = ops.kv8_attention(view.clone(memory_format=torch.contiguous_format), cos.float(), sin.float(), c, 100, 0.1)
        assert torch.equal(got, want) and _same(a, c)


def test_offsets_past_32_bits():
    """2.2e9 bytes of key codes: the last sequence's last head lies past 2^31."""
    from them_bones_b200 import ops
    from them_bones_b200.ref import functional as RF
    b, h, d, cap = 2, 4, 128, 1 << 21
    torch.manual_seed(13)
    cache = ops.kv8_cache(b, cap, h, d, "cuda")
    assert cache.k.numel() > 1 << 30 and cache.k.numel() * 2 >= 1 << 32
    n, at = 300, cap - 310
    cos, sin = (torch.rand(cap, d // 2, device="cuda") for _ in range(2))
    k, v = torch.randn(2, b, n, h, d, device="cuda").bfloat16()
    ops.kv8_append(cache, k[:, :at % 64 and 64 - at % 64], v[:, :at % 64 and 64 - at % 64], at)
    cut = at % 64 and 64 - at % 64
    ops.kv8_append(cache, k[:, cut:], v[:, cut:], at + cut)
    qkv = torch.randn(b, 3 * h * d, device="cuda").bfloat16()
    start = _i32([at + cut, at + cut + 70])
    y = ops.kv8_attention(qkv, cos, sin, cache, at + n, 0.1, start).double().view(b, h, d)
    small = ops.kv8_cache(b, 512, h, d, "cuda")
    ops.kv8_append(small, k[:, cut:], v[:, cut:], 0)
    m = n - cut
    for i in range(b):
        q, _, vn = O.new_rows(qkv[i], cos, sin, at + n, h, d)
        ks, vs = O.held(small, i, m)
        lo = int(start[i]) - at - cut
        ks = torch.cat([ks, cache.k_open[i, :, (at + n) % 64].double()[:, None]], 1)[:, lo:]
        vs = torch.cat([vs, vn[:, None]], 1)[:, lo:]
        w = torch.einsum("hn,hnd->hd", torch.softmax(torch.einsum("hd,hnd->hn", q, ks) * 0.1, -1), vs)
        assert bool(((y[i] - w).abs() <= 2 ** -8 * w.abs() + 2 ** -9 * vs.abs().max()).all())
    del RF


def test_native_refusals():
    from them_bones_b200 import ops
    c = ops.kv8_cache(2, 64, 1, 64, "cuda")
    k = torch.randn(2, 5, 1, 64, device="cuda")
    with pytest.raises(ValueError):
        ops.kv8_append(c, k, k, 0)                       # fp32 keys
    with pytest.raises(ValueError):
        ops.kv8_append(c, k.bfloat16(), k.bfloat16(), torch.zeros(2, dtype=torch.int32))      # positions on the host
    cos = torch.ones(64, 32, device="cuda")
    with pytest.raises(ValueError):
        ops.kv8_attention(torch.randn(2, 192, device="cuda"), cos, cos, c, 0, 1.0)
    with pytest.raises(ValueError):
        ops.kv8_attention(torch.randn(2, 192, device="cuda").bfloat16(), cos.cpu(), cos.cpu(), c, 0, 1.0)
    assert not any(x.any() for x in c)


def test_the_statement_s_path_on_the_gpu():
    """The plain bodies run on the same cache and agree, within what the kernels' own tests allow."""
    from them_bones_b200 import ops
    from them_bones_b200.ref import functional as RF
    torch.manual_seed(14)
    b, h, d = 3, 2, 64
    cos, sin = (x.cuda() for x in RF.rotary_tables(256, d, 10000.0))
    qkv = torch.randn(b, 3 * h * d, device="cuda").bfloat16()
    k, v = torch.randn(2, b, 70, h, d, device="cuda").bfloat16()
    a, c = ops.kv8_cache(b, 256, h, d, "cuda"), ops.kv8_cache(b, 256, h, d, "cuda")
    ops.kv8_append(a, k, v, 0)
    y = ops.kv8_attention(qkv, cos, sin, a, 70, 0.1).float()
    ops.set_reference_path(True)
    try:
        ops.kv8_append(c, k, v, 0)
        w = ops.kv8_attention(qkv, cos, sin, c, 70, 0.1).float()
        r = ops.kv8_read(c, 71, 71)
    finally:
        ops.set_reference_path(False)
    # the new key may round to bf16 the other way in fp32; the rest is equal
    assert all(torch.equal(x, z) for x, z in zip(a[:4], c[:4])) and torch.equal(a.v_open, c.v_open)
    assert float((a.k_open.float() - c.k_open.float()).abs().max()) <= 2 ** -7 * 4 and float((y - w).abs().max()) <= 2 ** -7 * float(w.abs().max())
    assert torch.equal(ops.kv8_read(a, 70, 70)[0], r[0][:, :70])


def test_a_cache_as_a_plain_tuple():
    from them_bones_b200 import ops
    c = ops.kv8_cache(1, 64, 1, 64, "cuda")
    k = torch.randn(1, 3, 1, 64, device="cuda").bfloat16()
    ops.kv8_append(tuple(c), k, k, 0)
    assert torch.equal(ops.kv8_read(tuple(c), 3, 3)[0], k)
    with pytest.raises(ValueError):
        ops.kv8_append(tuple(c), k[:, :, :, :32], k[:, :, :, :32], 0)
