"""What the tokens of a prompt see of an 8-bit cache on the plain route."""
import pytest
import torch

from tests import kv8_oracle as O


def _model(**kw):
    from them_bones_b200.config import GPTConfig
    from them_bones_b200.models.gpt import GPT
    torch.manual_seed(3)
    model = GPT(GPTConfig(**{**dict(sequence_len=256, vocab_size=97, n_layer=1, n_head=2, n_embd=128, head_dim=64, doc_mask=False), **kw}))
    model.init_weights()
    for p in model.parameters():
        if p.dim() == 2:
            torch.nn.init.normal_(p, std=0.08)
    return model.eval()


@pytest.mark.parametrize("pieces", [[200], [1] * 130, [63, 1, 64, 65, 7], [64, 64, 72], [10, 150, 3], [130, 1, 1]])
def test_full_blocks_are_seen_from_their_codes_unrounded(pieces, monkeypatch):
    """Every query's keys and values: codes times scales with fp32's rounding alone, then its own block's tokens in bf16 as they came."""
    from them_bones_b200.utils import decode as D
    model, seen, attend = _model(), [], D._attend

    def look(q, k, v, scale, lo):
        seen.append((k.double().clone(), v.double().clone()))
        return attend(q, k, v, scale, lo)
    monkeypatch.setattr(D, "_attend", look)
    n = sum(pieces)
    toks, cache, at = torch.randint(1, 97, (2, n)), D.KVCache(model, 2, n, "int8"), 0
    for p in pieces:
        D._forward_cached(model, toks[:, at:at + p], cache)
        at += p
    assert len(seen) == n and cache.len == n
    kept = [O.held(cache.kv8[0], b, n // 64 * 64) for b in range(2)]
    for cur, (k, v) in enumerate(seen):
        first = cur // 64 * 64
        assert k.shape[1] == v.shape[1] == cur + 1
        for b in range(2):
            for x, y in zip((k, v), kept[b]):
                y = y[:, :first].transpose(0, 1)
                assert bool(((x[b, :first] - y).abs() <= 2.0 ** -24 * y.abs()).all())
        for x, last in ((k, seen[min(first + 63, n - 1)][0]), (v, seen[min(first + 63, n - 1)][1])):        # the same tokens for the whole block
            assert torch.equal(x[:, first:], last[:, first:cur + 1]) and torch.equal(x[:, first:], x[:, first:].bfloat16().double())
    if n % 64:
        for x, tail in zip(seen[-1], cache.kv8[0][4:]):
            assert torch.equal(x[:, n // 64 * 64:], tail[:, :, :n % 64].transpose(1, 2).double())
