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


@pytest.mark.parametrize("drafts", [1, 4])
def test_drafted_rows_are_those_of_single_tokens(device, drafts):
    """The rows of every pass's tokens that stood, over the cache that refused drafts were written to, against a fresh layer that
    decodes each sequence by itself and one token at a time. Attention is as large as the embedding, and the router's bias
    alone chooses the experts, so that no near scores part the two."""
    def layer(pages):
        got = example.ExpertLayer(device, pages=pages)
        columns = got.q_heads * got.head_dim
        got.o_proj = got.linear(torch.randn(got.hidden, columns, generator=torch.Generator().manual_seed(8)) * columns**-0.5)
        got.bias = 2.0 * torch.randperm(16, generator=torch.Generator().manual_seed(9)).float().to(device)
        return got

    passes = []

    class Watched:  # of decode_drafts: its tokens, its lengths and its rows
        def __init__(self, inner):
            self.inner = inner

        def __call__(self, ids, lengths):
            logits = self.inner(ids, lengths)
            passes.append(([list(row) for row in ids], list(lengths), logits.double().cpu()))
            return logits

    both, stood = layer(128), []
    both.decode_drafts = Watched(both.decode_drafts)
    emitted = example.speculate(both, PROMPTS, 5, drafts, seed=4, watch=lambda *of: stood.append(of[-1].tolist()), temperature=4.0,
                                top_k=50, top_p=0.95)
    assert any(count < drafts for row in stood for count in row)
    for b, (prompt, own) in enumerate(zip(PROMPTS, emitted)):
        sequence, alone = prompt + own[:-1], layer(16)
        rows = torch.cat([alone.decode([token], [at]) for at, token in enumerate(sequence)]).double().cpu()
        plain = alone.drafter_logits(sequence).double().cpu()
        torch.cuda.synchronize()
        for (ids, lengths, logits), counts in zip(passes, stood):
            first, count = lengths[b], counts[b] + 1
            assert ids[b][:count] == sequence[first: first + count]
            got, want = logits.view(3, drafts + 1, -1)[b, :count], rows[first: first + count]
            # The same codes are cached but where the projections' last bits move one by a step; a dozen roundings of 2^-11 beside it.
            assert bool(((got - want).norm(dim=1) <= 12 * 2.0**-11 * want.norm(dim=1)).all()), (got - want).norm(dim=1) / want.norm(dim=1)
            without = plain[first: first + count]
            assert bool(((without - want).norm(dim=1) >= 0.2 * want.norm(dim=1)).all())
