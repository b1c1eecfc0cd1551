"""The prompt form of the small language model at the ends of its lengths."""
import pytest
import torch

from mogt_b200.selective_lm import SelectiveLM


def _embed_only():
    """No blocks: the logits are the head's of the embedding at the last token."""
    torch.manual_seed(0)
    m = SelectiveLM(11, 8, 0)
    ids = torch.randint(0, 11, (5, 6))
    head = lambda i, t: m._head(m.embedding(ids[i, t]))
    return m, ids, head


def test_lengths_are_clamped_like_the_operators():
    m, ids, head = _embed_only()
    logits, _ = m.prefill(ids, torch.tensor([0, 1, 6, 11, -3]))
    assert torch.allclose(logits[1], head(1, 0))
    assert torch.allclose(logits[2], head(2, 5)) and torch.allclose(logits[3], head(3, 5))
    # nothing has been read: no token is likelier than another
    assert bool((logits[0] == 0).all()) and bool((logits[4] == 0).all())


def test_prompts_without_tokens():
    m, ids, _ = _embed_only()
    for lengths in (None, torch.zeros(5, dtype=torch.int64)):
        logits, _ = m.prefill(ids[:, :0], lengths)
        assert logits.shape == (5, 11) and bool((logits == 0).all())


def test_int32_lengths_and_none():
    m, ids, head = _embed_only()
    a, _ = m.prefill(ids)
    b, _ = m.prefill(ids, torch.full((5,), 6, dtype=torch.int32))
    assert torch.equal(a, b) and torch.allclose(a[3], head(3, 5))


@pytest.mark.gpu
def test_a_prompt_of_no_tokens_then_tokens():
    """Starting from an empty prompt, single tokens give the training form's logits (fp32 bar of 1e-4)."""
    torch.manual_seed(1)
    m = SelectiveLM(31, 32, 2).cuda()
    ids = torch.randint(0, 31, (3, 6), device="cuda")
    with torch.no_grad():
        full = m(ids)
        logits, caches = m.prefill(ids, torch.tensor([0, 3, 99], device="cuda"))
        assert bool((logits[0] == 0).all())
        assert float((logits[1] - full[1, 2]).abs().max()) <= 1e-4 * float(full.abs().max())
        assert float((logits[2] - full[2, 5]).abs().max()) <= 1e-4 * float(full.abs().max())
        out = m.step(ids[:, 0], caches)
        assert float((out[0] - full[0, 0]).abs().max()) <= 1e-4 * float(full.abs().max())
        _, caches = m.prefill(ids[:, :0])
        for t in range(6):
            out = m.step(ids[:, t], caches)
            assert float((out - full[:, t]).abs().max()) <= 1e-4 * float(full.abs().max())
