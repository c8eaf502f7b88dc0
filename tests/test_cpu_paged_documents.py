"""Drafts of a smaller model behind refused ones: what it says is what it says of the text alone, document starts among what was refused or not."""
import pytest
import torch

from tests.test_cpu_decode_kv8 import _model


@pytest.mark.parametrize("t,kw", [(1.0, {}), (0.0, {}), (1.0, dict(attn_window=128, attn_long=(1,))), (1.0, dict(doc_mask=False))])
def test_a_refused_document_start_is_taken_back(monkeypatch, t, kw):
    from them_bones_b200.utils import paged as P
    # unlike models of seven tokens: drafts often fall, and one in seven is a document start
    model, small = _model(vocab_size=7, **kw), _model(vocab_size=7, n_layer=1, n_embd=64, n_head=1, **({} if kw.get("doc_mask", True) else kw))
    k, refused, kept, checked = 4, 0, 0, 0
    draw, forget = P._ModelDrafts.draw, P._ModelDrafts.forget

    def looked_at(self, texts, done, gen):
        nonlocal checked
        drafts = draw(self, texts, done, gen)
        for i, text in enumerate(texts):
            if done[i]:
                continue
            for j in range(k):                                # the row in front of draft j: the text and the drafts before it
                row = torch.tensor([text + drafts[i, :j].tolist()])
                if row.shape[1] > small.config.sequence_len:
                    break
                with torch.no_grad():
                    want = small(row)[0, -1]
                # fp32 passes of other shapes: sums of up to 64 terms and 160 weights, a few thousand roundings of 2^-24 on values of size 1
                assert torch.allclose(self.logits[i * (k + 1) + j], want, rtol=1e-3, atol=1e-3), (i, j, len(text))
                checked += 1
        self.last = drafts.tolist()
        return drafts

    def counted(self, texts, accepted):
        nonlocal refused, kept
        for n, d, a in zip(texts, self.last, accepted):
            refused, kept = refused + d[a:k - 1].count(0), kept + d[:a].count(0)
        return forget(self, texts, accepted)

    monkeypatch.setattr(P._ModelDrafts, "draw", looked_at)
    monkeypatch.setattr(P._ModelDrafts, "forget", counted)
    prompts = [[0, 3, 5], [4], [1, 2, 0, 6, 5, 3, 3], [2, 0], [5] * 20, [1, 6, 6]]
    rows = P.paged_decode(model, prompts, 30, temperature=t, drafts=k, draft=small, seed=3)
    assert all(r.shape[0] == len(p) + 30 for r, p in zip(rows, prompts)) and checked > 100
    assert (refused and kept) or not t
