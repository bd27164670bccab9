"""The example that speculates through a layer of routed experts: the operators run together as they would be used."""

from pathlib import Path
import sys

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
import speculate as example  # noqa: E402

from test_gpu_verification import definition  # noqa: E402

pytestmark = pytest.mark.gpu

PROMPTS = [list(range(3, 40)), list(range(500, 511)), [7, 8]]


@pytest.mark.parametrize("drafts", [1, 4])
def test_tokens_are_what_the_rows_say(device, drafts):
    """Each pass's verdicts by the definition, from the rows that it saw; rows are distributions."""
    passes = []

    def watch(logits, target, proposal, drafted, u, tokens, accepted):
        for rows in (target, proposal):
            assert bool(((rows.double().sum(1) - 1).abs() < 1e-5).all())
        p, q = target.view(3, drafts + 1, -1).cpu().numpy(), proposal.view(3, drafts, -1).cpu().numpy()
        for b in range(3):
            want, count = definition(p[b], q[b], drafted[b].tolist(), drafts, u[b].double().cpu().numpy())
            assert (tokens[b].tolist(), int(accepted[b])) == (want, count)
        passes.append(int(accepted.sum()))

    runs = [example.speculate(example.ExpertLayer(device, pages=128), PROMPTS, 5, drafts, seed=4, watch=watch, temperature=4.0, top_k=50,
                              top_p=0.95) for _ in range(2)]
    assert runs[0] == runs[1] and sum(map(len, runs[0])) == 15 + sum(passes[:5])


def test_greedy_tokens_are_the_largest_logits(device):
    """At temperature 0 every emitted token is the largest logit of its row, whatever was drafted."""
    def watch(logits, target, proposal, drafted, u, tokens, accepted):
        best = logits.view(3, 4, -1).float().argmax(-1)
        for b in range(3):
            count = int(accepted[b])
            assert tokens[b, : count + 1].tolist() == best[b, : count + 1].tolist()
            assert tokens[b, count + 1:].tolist() == [-1] * (3 - count)

    example.speculate(example.ExpertLayer(device, pages=128), PROMPTS, 4, 3, watch=watch, temperature=0.0)
