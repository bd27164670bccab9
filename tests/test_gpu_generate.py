"""The example that runs the operators together: a prompt in one pass, in two passes over read-back keys, and token by token
over the cache lead to the same logits, within what the Q8 cache and fp16 leave; the same seed draws the same tokens."""

from pathlib import Path
import sys

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
import generate as example  # noqa: E402

pytestmark = pytest.mark.gpu

PROMPTS = [list(range(3, 40)), list(range(500, 511)), list(range(100, 162))]


@pytest.mark.parametrize("heads", [(8, 2, 64), (6, 1, 128)])
def test_prompt_in_one_pass_in_two_and_token_by_token(device, heads):
    q_heads, kv_heads, head_dim = heads

    def layer():
        return example.Layer(device, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim)

    whole = layer().prompts(PROMPTS, [0, 0, 0])
    split = layer()
    split.prompts([p[:8] for p in PROMPTS], [0, 0, 0])
    two = split.prompts([p[8:] for p in PROMPTS], [8, 8, 8])
    single = layer()
    short = [p[:11] for p in PROMPTS]
    for i in range(11):
        one = single.decode([p[i] for p in short], [i, i, i])
    cut = layer().prompts(short, [0, 0, 0])
    torch.cuda.synchronize()
    for got, want in ((two, whole), (one, cut)):
        got, want = got.double(), want.double()
        # The cache's error is at most 1/254 of a group's largest number, a few thousandths of the logits' size.
        assert ((got - want).norm(dim=1) <= 0.02 * want.norm(dim=1)).all(), (got - want).norm(dim=1) / want.norm(dim=1)


def test_generation_is_repeatable(device):
    runs = [example.generate(example.Layer(device), PROMPTS, 6, first=first, seed=3)[0] for first in (8, 8, None)]
    assert runs[0] == runs[1]
    for tokens in runs:
        assert all(len(own) == 6 and all(0 <= i < 1000 for i in own) for own in tokens)
