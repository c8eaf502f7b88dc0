"""Decoding from the paged cache on the GPU: the model's own logits say that each token is the one, whatever the route."""
import pytest
import torch

from tests.test_gpu_decode_kv8 import _model, _tokens

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_wait_ran_out():
    yield
    from them_bones_b200.ops import _lib as L
    L.check_error_word()


@pytest.mark.parametrize("kw", [{}, dict(attn_window=128, attn_long=(1,)), dict(value_embeds=1), dict(unet=True), dict(head_dim=64, n_head=4),
                                dict(moe_layers=(1,), moe_experts=8, moe_topk=2, moe_capacity=300, moe_hidden=256)])
def test_pieces_give_the_full_pass_s_logits(kw):
    from them_bones_b200.utils import paged as P
    model = _model(seq=640, **kw)
    lens = [1, 300, 77, 0, 513]
    toks = [_tokens(1, n + 20)[0] for n in lens]
    cache = P.PagedCache(model, [n + 20 for n in lens], page=16)
    for cut in (lens, [3, 1, 17, 16, 0], [1] * 5):
        held = cache.pos.tolist()
        ids = torch.cat([t[h:h + n] for t, h, n in zip(toks, held, cut)])
        starts = P._starts(cut, "cuda")
        x, doc = P.forward_pieces(model, ids, cache, starts, max(cut))
        from them_bones_b200 import ops
        z = ops.lmhead_logits(x, model.lm_head.weight, 1024, model.config.softcap)
        for i, (t, h, n) in enumerate(zip(toks, held, cut)):
            if n:
                with torch.no_grad():
                    want = model(t[None, :h + n])[0, h:]
                got = z[int(starts[i]):int(starts[i + 1])]
                # bf16 activations of two layers, row by row: what the decode step's logits are held to
                assert float(((got - want).norm(dim=1) / want.norm(dim=1)).max()) < 6e-2
                if doc is not None:
                    cache.doc_start[i] = doc[int(starts[i + 1]) - 1]
        cache.pos.add_(torch.tensor(cut, dtype=torch.int32, device="cuda"))


def _are_the_best(model, rows, prompts, n_new):
    """Each new token has the largest logit of the full pass behind its text, but for bf16 roundings of the activations (6e-2 of a row's norm, as above, is more
    than any of these differences; a wrong token is several units off in a model of untrained logits of size 1)."""
    for row, p in zip(rows, prompts):
        with torch.no_grad():
            z = model(row[None])[0, len(p) - 1:-1]
        taken = z.gather(1, row[len(p):, None])[:, 0]
        assert row.shape[0] == len(p) + n_new and torch.equal(row[:len(p)].cpu(), torch.as_tensor(p).cpu())
        assert float((z.amax(1) - taken).max()) < 0.1 * float(z.std()), float((z.amax(1) - taken).max())


@pytest.mark.parametrize("drafts,model_drafts", [(0, False), (1, False), (4, False), (3, True)])
def test_greedy_tokens_are_the_best(drafts, model_drafts):
    from them_bones_b200.utils import paged as P
    model = _model(seq=900)
    prompts = [_tokens(1, n)[0].tolist() for n in (1, 2, 64, 700, 130, 33)]
    rows = P.paged_decode(model, prompts, 40, drafts=drafts, draft=_model(n_layer=1, seq=900) if model_drafts else None)
    _are_the_best(model, rows, prompts, 40)


def test_long_prompts_and_the_native_step_agree():
    from them_bones_b200.utils import decode as D, paged as P
    model = _model(seq=900)
    prompts = _tokens(5, 600)
    out = P.paged_decode(model, prompts, 30)
    _are_the_best(model, out, prompts, 30)
    short = prompts[:, :50]
    a, b = P.paged_decode(model, short, 30), D.greedy_decode(model, short, 30)
    assert int((a == b).all(1).sum()) >= 3                    # a near tie that falls the other way ends the agreement of a row


def test_drawn_tokens_follow_the_model():
    """A prompt many times over, with the model's own drafts and without: the first token as often as its probability says."""
    from them_bones_b200.utils import paged as P
    model = _model(vocab_size=64)
    prompt, n, t = [0, 5, 9], 800, 0.7
    with torch.no_grad():
        law = torch.softmax(model(torch.tensor([prompt], device="cuda"))[0, -1].double() / t, -1).cpu()
    for kw in (dict(), dict(drafts=2), dict(drafts=2, draft=model)):
        rows = torch.stack(P.paged_decode(model, [prompt] * n, 3, temperature=t, seed=5, **kw))
        again = torch.stack(P.paged_decode(model, [prompt] * n, 3, temperature=t, seed=5, **kw))
        assert torch.equal(rows, again)
        count = torch.bincount(rows[:, 3].cpu(), minlength=64).double()
        # binomial counts: five standard deviations, and 3 % of a probability for the logits' bf16 roundings (2^-8 of values up to 5, over t)
        assert bool(((count - n * law).abs() <= 5 * (n * law * (1 - law)).sqrt() + 1 + 0.03 * n * law).all())


def test_on_another_stream_and_twice_over():
    from them_bones_b200.utils import paged as P
    model = _model()
    prompts = _tokens(3, 40)
    want = P.paged_decode(model, prompts, 20, drafts=3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = P.paged_decode(model, prompts, 20, drafts=3)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
