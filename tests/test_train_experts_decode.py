"""The expert example's decoding: a prompt in one pass, then a token at a time."""

import pytest
import torch

from test_train_experts import example


def _whole(model, prompt, tokens):
    """Greedy tokens, each from the whole sequence before it."""
    ids = prompt[None]
    with torch.no_grad():
        for _ in range(tokens):
            ids = torch.cat((ids, model.head(model(ids)[:, -1]).argmax(-1, keepdim=True)), 1)
    return ids[0, len(prompt):]


def test_no_tokens():
    torch.manual_seed(0)
    got = example.decode(example.Model(vocab=40, hidden=16, inter=24), torch.tensor([3, 1, 4]), 0)
    assert got.shape == (0,) and got.dtype == torch.int64


@pytest.mark.parametrize("length", [1, 2, 37])
def test_the_tokens_are_those_of_the_whole_sequence(length):
    """In FP32, where a sum's order moves a logit far less than two of them are apart."""
    torch.manual_seed(length)
    model = example.Model(vocab=40, hidden=16, inter=24)
    prompt = torch.randint(0, 40, (length,))
    assert torch.equal(example.decode(model, prompt, 6), _whole(model, prompt, 6))


def test_a_prompt_is_one_pass_whatever_its_length(monkeypatch):
    torch.manual_seed(1)
    model, passes = example.Model(vocab=40, hidden=16, inter=24), []
    forward = example.ExpertBlock.forward
    monkeypatch.setattr(example.ExpertBlock, "forward", lambda self, x: (passes.append(x.shape[:-1]), forward(self, x))[1])
    example.decode(model, torch.randint(0, 40, (37,)), 5)
    assert len(passes) == 5 * len(model.blocks)
