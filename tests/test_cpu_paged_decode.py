"""Decoding from the paged cache on the CPU: the tokens of the other routes, pieces, drafts and what is refused."""
import pytest
import torch

from tests.test_cpu_decode_kv8 import _model


@pytest.mark.parametrize("kw", [{}, dict(attn_window=128, attn_long=(1,)), dict(value_embeds=1), dict(unet=True), dict(moe_layers=(1,), moe_experts=4, moe_topk=2, moe_capacity=160, moe_hidden=64)])
def test_greedy_tokens_of_the_other_routes(kw):
    from them_bones_b200.utils import decode as D, paged as P
    model = _model(**kw)
    prompts = torch.randint(1, 97, (3, 41), generator=torch.Generator().manual_seed(1))
    prompts[1, 30] = prompts[2, 40] = 0
    want = D.greedy_decode(model, prompts, 20)
    for drafts in (0, 1, 4):
        assert torch.equal(P.paged_decode(model, prompts, 20, drafts=drafts, page=16), want), drafts


def test_prompts_of_any_lengths_in_pieces(monkeypatch):
    from them_bones_b200.utils import decode as D, paged as P
    monkeypatch.setattr(P, "PIECE", 17)
    model = _model()
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, 97, (n,), generator=g) for n in (1, 2, 50, 17, 90)]
    for drafts in (0, 3):
        got = P.paged_decode(model, [p.tolist() for p in prompts], 9, drafts=drafts, page=32)
        for p, row in zip(prompts, got):
            assert torch.equal(row, D.greedy_decode(model, p[None], 9)[0])


def test_a_draft_model_changes_nothing_but_the_steps(monkeypatch):
    from them_bones_b200 import ops
    from them_bones_b200.utils import paged as P
    model, small = _model(), _model(n_layer=1)
    prompts = torch.randint(1, 97, (3, 23), generator=torch.Generator().manual_seed(4))
    want, calls = P.paged_decode(model, prompts, 24), []
    real = ops.verify_drafts
    monkeypatch.setattr(ops, "verify_drafts", lambda *a, **k: calls.append(real(*a, **k)) or calls[-1])
    for draft, drafts in ((model, 3), (small, 3), (small, 1), (model, 7)):
        calls.clear()
        assert torch.equal(P.paged_decode(model, prompts, 24, drafts=drafts, draft=draft), want)
        if draft is model:                                          # its own drafts all stand: k passes of it and one of verification give k + 1 tokens
            assert len(calls) == (24 // (drafts + 1)) * (drafts + 1)
            own = [c.accepted for c in calls[drafts::drafts + 1]]
            assert all(bool((a == drafts).all()) for a in own)


@pytest.mark.parametrize("drafts,which", [(0, None), (2, None), (2, "small"), (3, "same")])
def test_drawn_tokens_follow_the_model(drafts, which):
    """The first two tokens behind one prompt, many times: as often as the model's own probabilities say."""
    from them_bones_b200.utils import paged as P
    model, small = _model(vocab_size=7, n_layer=1), _model(vocab_size=7, n_layer=1, n_embd=64, n_head=1)
    draft = {None: None, "small": small, "same": model}[which]
    n, t = 1500, 0.8
    prompt = [3, 5, 3, 5, 3]
    rows = P.paged_decode(model, [prompt] * n, 2, temperature=t, drafts=drafts, draft=draft, seed=11)
    got = torch.stack(rows)[:, 5:]
    with torch.no_grad():
        first = torch.softmax(model(torch.tensor([prompt]))[0, -1].double() / t, -1)
        second = torch.softmax(model(torch.tensor([prompt + [i] for i in range(7)]))[:, -1].double() / t, -1)
    law = (first[:, None] * second).flatten()
    count = torch.bincount(got[:, 0] * 7 + got[:, 1], minlength=49).double()
    # each of 49 counts is binomial: five standard deviations
    assert bool(((count - n * law).abs() <= 5 * (n * law * (1 - law)).sqrt() + 1).all())


def test_lookup_takes_the_last_occurrence():
    from them_bones_b200.utils.paged import lookup
    assert lookup([1, 2, 3, 9, 1, 2, 3], 2) == [9, 1] and lookup([1, 2, 3, 4, 2, 3, 5, 2, 3], 3) == [5, 2, 3]
    assert lookup([7, 8, 1, 8], 4) == [1, 8] and lookup([1, 2, 3], 2) == [] and lookup([5], 3) == []


def test_calls_that_are_refused():
    from them_bones_b200.utils import paged as P
    model = _model()
    ok = torch.randint(1, 97, (2, 10))
    for bad in (dict(prompts=[]), dict(prompts=[[1], []]), dict(n_new=151), dict(n_new=-1), dict(drafts=-1), dict(drafts=65), dict(temperature=-1.0), dict(draft=model),
                dict(drafts=2, draft=_model(vocab_size=50)), dict(drafts=2, draft=_model(sequence_len=80))):
        with pytest.raises(ValueError):
            P.paged_decode(model, **{**dict(prompts=ok, n_new=5), **bad})
    with pytest.raises(ValueError):
        P.paged_decode(_model(attn_layers=(1,)), ok, 3)
    assert torch.equal(P.paged_decode(model, ok, 0), ok)


def test_generate_offers_it():
    import inference
    model = _model()
    w = inference.ModelWrapper(model, {})
    prompts = torch.randint(1, 97, (2, 9))
    assert torch.equal(w.generate(prompts, 6, kv="paged", drafts=2), w.generate(prompts, 6))
    assert torch.equal(w.generate(prompts, 6, kv="paged", drafts=2, draft=w), w.generate(prompts, 6))
    for bad in (dict(kv="paged", logprobs=1), dict(temperature=1.0), dict(drafts=2)):
        with pytest.raises(ValueError):
            w.generate(prompts, 6, **bad)


def test_tokens_outside_the_vocabulary_are_refused():
    from them_bones_b200.utils import paged as P
    for bad in ([[1, 97]], [[-1, 3]], torch.tensor([[5, 1 << 40]])):
        with pytest.raises(ValueError):
            P.paged_decode(_model(), bad, 2)
