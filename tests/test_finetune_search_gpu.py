"""What a beam search of the small model starts from."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_search_without_rounds_of_training():
    from t2fw_amd.finetune import finetune
    said = []
    history = finetune(rounds=0, batch=4, prompt=3, answer=5, vocab=40, width=64, layers=2, beams=3, selective=True, say=said.append)
    assert len(history) == len(said) == 1 and 0.0 <= history[0] <= 1.0 and "beam search of 3" in said[0]
    assert finetune(rounds=0, batch=4, vocab=40, width=64, layers=2, say=said.append) == [] and len(said) == 1


def test_the_search_follows_the_last_rounds_prompts():
    """the generator's draws are those of a training without a search"""
    from t2fw_amd.finetune import finetune
    options = dict(rounds=2, batch=4, prompt=3, answer=5, vocab=40, width=64, layers=2, say=lambda s: None)
    assert finetune(beams=2, **options)[:2] == finetune(**options)


def test_a_search_needs_a_prompt():
    from t2fw_amd.finetune import RecurrentLM
    model = RecurrentLM(vocab=40, width=64, layers=2).cuda()
    with pytest.raises(ValueError, match="at least one token"):
        model.beam_search(torch.zeros(2, 0, dtype=torch.int64, device="cuda"), 3, beams=2)
    tokens, scores = model.beam_search(torch.zeros(2, 1, dtype=torch.int64, device="cuda"), 3, beams=2)
    assert tokens.shape == (2, 2, 4) and bool(torch.isfinite(scores).all())
