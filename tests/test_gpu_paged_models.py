"""The captured step of the paged decoding for each kind of model that it takes, and drafts behind refused document starts, on the GPU."""
import pytest
import torch

from tests.test_gpu_decode_kv8 import _model, _tokens
from tests.test_gpu_paged_decode import _are_the_best

pytestmark = pytest.mark.gpu

MODELS = [dict(attn_window=128, attn_long=(1,)), dict(value_embeds=1), dict(unet=True), dict(head_dim=64, n_head=4), dict(doc_mask=False),
          dict(moe_layers=(1,), moe_experts=8, moe_topk=2, moe_capacity=700, moe_hidden=256)]


@pytest.fixture(autouse=True)
def _no_wait_ran_out():
    yield
    from them_bones_b200.ops import _lib as L
    L.check_error_word()


@pytest.mark.parametrize("kw", MODELS)
@pytest.mark.parametrize("drafts,model_drafts", [(0, False), (4, False), (3, True), (20, False)])
def test_greedy_tokens_are_the_best(kw, drafts, model_drafts):
    """Steps of one token, of a few and of more than sixteen (the other kernel), each captured on its second call."""
    from them_bones_b200.utils import paged as P
    model = _model(seq=700, **kw)
    prompts = [_tokens(1, n)[0].tolist() for n in (1, 3, 64, 600, 130)]
    replayed = []
    run = P._Step.__call__
    with pytest.MonkeyPatch.context() as m:
        m.setattr(P._Step, "__call__", lambda self, gen: (run(self, gen), replayed.append(self.graph is not None))[0])
        rows = P.paged_decode(model, prompts, 24, drafts=drafts, draft=_model(n_layer=1, seq=700) if model_drafts else None)
    assert any(replayed)
    _are_the_best(model, rows, prompts, 24)


@pytest.mark.parametrize("kw", [{}, dict(attn_window=128, attn_long=(1,)), dict(value_embeds=1)])
def test_drawn_tokens_of_each_model_follow_it(kw):
    from them_bones_b200.utils import paged as P
    model, small = _model(vocab_size=64, **kw), _model(vocab_size=64, n_layer=1)
    prompt, n, t = [0, 5, 9], 800, 0.7
    with torch.no_grad():
        law = torch.softmax(model(torch.tensor([prompt], device="cuda"))[0, -1].double() / t, -1).cpu()
    for more in (dict(), dict(drafts=2), dict(drafts=2, draft=small)):
        rows = torch.stack(P.paged_decode(model, [prompt] * n, 3, temperature=t, seed=5, **more))
        count = torch.bincount(rows[:, 3].cpu(), minlength=64).double()
        # binomial counts: five standard deviations, and 3 % of a probability for the logits' bf16 roundings (2^-8 of values up to 5, over t)
        assert bool(((count - n * law).abs() <= 5 * (n * law * (1 - law)).sqrt() + 1 + 0.03 * n * law).all())


def test_drafts_behind_refused_document_starts():
    """What the draft model says at each draft is what its full pass over the text and the drafts before says."""
    from them_bones_b200.utils import paged as P
    model, small, k = _model(vocab_size=64), _model(vocab_size=64, n_layer=1), 4
    draw, forget, seen = P._ModelDrafts.draw, P._ModelDrafts.forget, dict(rows=0, refused=0)

    def looked_at(self, texts, done, gen):
        drafts = draw(self, texts, done, gen)
        self.last = drafts.tolist()
        live = [i for i, d in enumerate(done) if not d]
        for i in live[::7]:
            with torch.no_grad():
                want = small(torch.tensor([texts[i] + self.last[i]], device="cuda"))[0, len(texts[i]) - 1:-1]
            got = self.logits[i * (k + 1):i * (k + 1) + k]
            # bf16 activations of one layer, row by row, as test_pieces_give_the_full_pass_s_logits has of two
            assert float(((got - want).norm(dim=1) / want.norm(dim=1)).max()) < 6e-2, (i, len(texts[i]))
            seen["rows"] += k
        return drafts

    def counted(self, texts, accepted):
        seen["refused"] += sum(d[a:k - 1].count(0) for d, a in zip(self.last, accepted))
        return forget(self, texts, accepted)

    with pytest.MonkeyPatch.context() as m:
        m.setattr(P._ModelDrafts, "draw", looked_at)
        m.setattr(P._ModelDrafts, "forget", counted)
        prompts = [_tokens(1, n)[0].clamp(max=63).tolist() for n in [1, 7, 40, 100] * 16]
        P.paged_decode(model, prompts, 40, temperature=1.0, drafts=k, draft=small, seed=3)
    assert seen["rows"] > 200 and seen["refused"] > 3
