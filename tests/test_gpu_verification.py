"""Verification of drafts against the definition in 64 bits: the tokens are equal."""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def definition(p, q, drafted, count, u):
    """(tokens, accepted) of one sequence: p [drafts + 1, vocab], q [drafts, vocab] or None."""
    d, vocab = len(drafted), p.shape[1]
    p = np.where((p > 0) & np.isfinite(p), p, 0.0).astype(np.float64)
    tokens, at = [], 0
    count = min(max(count, 0), d)
    while at < count:
        token = int(drafted[at])
        if not 0 <= token < vocab:
            break
        chance = 1.0 if q is None else float(q[at, token])
        if not float(u[at]) * chance < p[at, token]:
            break
        tokens.append(token)
        at += 1
    rest = p[at]
    if at < count:
        if q is None:
            left = rest.copy()
            if 0 <= int(drafted[at]) < vocab:
                left[int(drafted[at])] = 0.0
        else:
            left = rest - q[at].astype(np.float64)
            left = np.where((left > 0) & (rest > 0), left, 0.0)
        if left.sum() > 0:
            rest = left
    some = np.flatnonzero(rest > 0)
    if not len(some):
        token = -1
    else:
        total = np.cumsum(rest)
        past = np.flatnonzero((rest > 0) & (total > float(u[d]) * total[-1]))
        token = int(past[0]) if len(past) else int(some[-1])
    return tokens + [token] + [-1] * (d - at), at


def check(backend, device, p, q, drafted, u, counts=None):
    n, d = drafted.shape
    vocab = p.shape[-1]
    print(f"case verification {n} x {d} of {vocab}, {'certain' if q is None else 'drawn'}", flush=True)
    plan = backend.prepare_verification(sequences=n, drafts=d, vocab=vocab, device=device)
    tokens = torch.full((n * (d + 1) + 16,), -9, dtype=torch.int64, device=device)
    accepted = torch.full((n + 16,), -9, dtype=torch.int32, device=device)
    workspace = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device=device)
    plan.run(p.float().view(n * (d + 1), vocab).to(device), drafted.to(device), u.float().to(device),
             proposal=None if q is None else q.float().view(n * d, vocab).to(device),
             counts=None if counts is None else torch.as_tensor(counts, dtype=torch.int32).to(device),
             tokens=tokens[8: 8 + n * (d + 1)].view(n, d + 1), accepted=accepted[8: 8 + n], workspace=workspace)
    torch.cuda.synchronize()
    for t, size in ((tokens, n * (d + 1)), (accepted, n)):
        assert bool((t[:8] == -9).all()) and bool((t[8 + size:] == -9).all())
    tokens, accepted = tokens[8: 8 + n * (d + 1)].view(n, d + 1).cpu().tolist(), accepted[8: 8 + n].cpu().tolist()
    for i in range(n):
        want, count = definition(p[i].float().numpy(), None if q is None else q[i].float().numpy(), drafted[i].numpy(),
                                 d if counts is None else int(counts[i]), u[i].float().double().numpy())
        assert (tokens[i], accepted[i]) == (want, count), i
    return tokens, accepted


def case(n, d, vocab, seed, noise=0.7, certain=False):
    gen = torch.Generator().manual_seed(seed)
    logits = 3 * torch.randn(n, d + 1, vocab, generator=gen)
    other = logits[:, :d] + noise * torch.randn(n, d, vocab, generator=gen)
    p = torch.softmax(logits, -1)
    p = torch.where(p < 1e-3 * p.amax(-1, keepdim=True), 0.0, p)
    p = p / p.sum(-1, keepdim=True)
    u = torch.rand(n, d + 1, generator=gen)
    if certain:
        return p, None, other.argmax(-1), u
    q = torch.softmax(other, -1)
    drafted = torch.multinomial(q.view(n * d, vocab), 1, generator=gen).view(n, d)
    return p, q, drafted, u


@pytest.mark.parametrize("certain", [False, True], ids=["drawn", "certain"])
@pytest.mark.parametrize("n,d,vocab", [(1, 1, 1), (3, 2, 2), (4, 3, 7), (9, 64, 5), (33, 7, 1000), (5, 4, 4095), (5, 4, 4097), (2, 3, 32003),
                                       (70, 2, 9001), (1, 4, 248320), (2, 5, 151937), (300, 1, 2100), (2100, 1, 300), (1, 1, 2**20)])
def test_random_drafts(backend, device, certain, n, d, vocab):
    for noise in (0.3, 1.5):
        p, q, drafted, u = case(n, d, vocab, n + vocab, noise, certain)
        check(backend, device, p, q, drafted, u)
    counts = torch.randint(-1, d + 2, (n,), generator=torch.Generator().manual_seed(1)).tolist()
    check(backend, device, p, q, drafted, u, counts)


def test_all_drafts_stand_and_none_does(backend, device):
    p, q, drafted, u = case(8, 5, 5001, 3)
    u[:, :5] = 0.0
    positive = p[:, :5].gather(2, drafted[..., None])[..., 0] > 0
    assert check(backend, device, p, q, drafted, u)[1] == positive.long().cumprod(1).sum(1).tolist()
    u[:, :5] = 1e30
    assert check(backend, device, p, q, drafted, u)[1] == [0] * 8
    assert check(backend, device, p, q, drafted, u, [0] * 8)[1] == [0] * 8


def test_borders_are_exact(backend, device):
    """Probabilities in units of 2^-12, whose sums are exact: a draft stands below the border and not at it, and the drawn
    token changes where the uniform is a running sum."""
    vocab, d = 4096 + 512, 1
    gen = torch.Generator().manual_seed(4)
    p = torch.zeros(64, 2, vocab)
    for i in range(64):
        at = torch.randperm(vocab, generator=gen)[:8]
        p[i, :, at] = torch.tensor([1024, 1024, 512, 512, 512, 256, 128, 128]) / 4096.0
    drafted = p[:, 0].argmax(-1, keepdim=True)
    q = torch.full((64, 1, vocab), 0.0)
    q.scatter_(2, drafted[:, None], 0.5)
    u = torch.zeros(64, 2)
    u[:, 0] = torch.tensor([0.5, 0.5 - 2.0**-25] * 32)  # p / q is 0.5 exactly
    u[:, 1] = torch.arange(64) / 64.0
    _, accepted = check(backend, device, p, q, drafted, u)
    assert accepted == [0, 1] * 32
    check(backend, device, p, None, drafted, u / 2)


def test_ends_of_the_uniforms(backend, device):
    for vocab in (50, 9001):
        p, q, drafted, u = case(6, 2, vocab, 5)
        for last in (0.0, 2.0**-30, 1 - 2.0**-24, 1.0, 2.0, -1.0, math.nan, math.inf):
            u[:, 2] = last
            check(backend, device, p, q, drafted, u)
        u[:, :2] = math.nan
        assert check(backend, device, p, q, drafted, u)[1] == [0] * 6


@pytest.mark.parametrize("vocab", [40, 9001])
def test_rows_that_leave_nothing(backend, device, vocab):
    """The drafter's row at or above the target's everywhere, empty rows, and values that are no probabilities."""
    p, q, drafted, u = case(10, 2, vocab, 6)
    u[:, :2] = 1e30
    q[0] = p[0, :2]
    q[1] = 1.0
    p[2] = 0.0
    p[3], p[4] = math.nan, -1.0
    p[5, 0, : vocab // 2] = math.inf
    q[6] = math.nan
    q[9] = -0.25
    p[7, 0] = 0.0
    p[7, 0, 17] = 1e-45
    drafted[8, 0], drafted[9, 0] = vocab, -3
    check(backend, device, p, q, drafted, u)
    check(backend, device, p, None, drafted, u)
    p[:, 0] = 0.0
    p.scatter_(2, drafted.clamp(0, vocab - 1)[..., None], 0.5)  # certain drafts hold the whole mass
    check(backend, device, p, None, drafted, u)


@pytest.mark.parametrize("n,d,vocab", [(2, 1, 16384), (3, 2, 16385), (2, 1, 32768), (2, 2, 32769), (5, 1, 40001), (256, 1, 17000), (257, 1, 17000),
                                       (300, 1, 5000), (300, 1, 16001), (300, 1, 100001), (1030, 1, 9001), (683, 1, 40001), (1100, 1, 8001),
                                       (256, 1, 270001)])
@pytest.mark.parametrize("certain", [False, True], ids=["drawn", "certain"])
def test_rows_in_one_part_and_in_several(backend, device, certain, n, d, vocab):
    """Both sides of the borders between a workgroup's registers, its second reading, and parts; the last of a row, too."""
    p, q, drafted, u = case(4, d, vocab, n + vocab, 0.7, certain)
    times = -(-n // 4)
    p, drafted, u = (t.repeat(times, *[1] * (t.dim() - 1))[:n].contiguous() for t in (p, drafted, u))
    q = None if q is None else q.repeat(times, 1, 1)[:n].contiguous()
    u[:, d] = torch.linspace(0, 1, n)
    u[: n // 2, :d] = 1e30  # refused
    check(backend, device, p, q, drafted, u)


def test_long_rows_that_leave_nothing(backend, device):
    """In parts: the drafter's row at or above the target's everywhere, or in all parts but one; empty rows."""
    vocab = 50001
    for certain in (False, True):
        p, q, drafted, u = case(7, 1, vocab, 9, 0.7, certain)
        u[:, 0] = 1e30
        p[4], p[5] = 0.0, math.nan
        if certain:
            p[0, 0] = p[1, 0] = 0.0
            p[0, 0, drafted[0, 0]] = 1.0
            p[1, 0, drafted[1, 0]], p[1, 0, vocab - 1 if drafted[1, 0] < 100 else 0] = 0.5, 0.25
        else:
            q[0], q[2], q[3] = p[0, :1], 1.0, math.nan
            q[1] = p[1, :1]
            q[1, 0, 30000:30010] = 0.0
            p[1, 0, 30005] = 0.125
        for last in (0.0, 0.5, 1.0):
            u[:, 1] = last
            check(backend, device, p, q, drafted, u)


def test_graph_of_rows_in_parts(backend, device):
    n, d, vocab = 3, 2, 40003
    plan = backend.prepare_verification(sequences=n, drafts=d, vocab=vocab, device=device)
    p, q, drafted, u = (t.to(device) for t in case(n, d, vocab, 1))
    p, q = p.view(n * (d + 1), vocab), q.view(n * d, vocab)
    tokens, accepted = torch.empty(n, d + 1, dtype=torch.int64, device=device), torch.empty(n, dtype=torch.int32, device=device)
    arguments = dict(proposal=q, tokens=tokens, accepted=accepted, workspace=torch.empty(plan.workspace_bytes, dtype=torch.uint8, device=device))
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        plan.run(p, drafted, u, **arguments)
    torch.cuda.current_stream(device).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.run(p, drafted, u, **arguments)
    for i in range(4):
        for t, new in zip((p, q, drafted, u), case(n, d, vocab, 20 + i)):
            t.copy_(new.view(t.shape))
        plan.run(p, drafted, u, **arguments)
        want = tokens.clone(), accepted.clone()
        tokens.zero_(), accepted.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(tokens, want[0]) and torch.equal(accepted, want[1])


def test_emitted_tokens_are_distributed_as_the_target(backend, device):
    """Drafts on a grid of the drafter's shares, uniforms on grids: the first token comes as often as its share says."""
    vocab, steps = 5, 64
    p = torch.tensor([0.4, 0.1, 0.25, 0.05, 0.2])
    q = torch.tensor([0.125, 0.25, 0.25, 0.25, 0.125])
    grid = (torch.arange(steps) + 0.5) / steps
    drafts = torch.searchsorted(q.cumsum(0), grid)
    n = steps**3
    if n > 65535:
        grid, drafts = grid[::2], drafts[::2]
        n = len(grid) ** 3
    d, a, b = (t.flatten() for t in torch.meshgrid(drafts.float(), grid, grid, indexing="ij"))
    tokens, _ = check(backend, device, p.expand(n, 2, vocab), q.expand(n, 1, vocab), d[:, None].long(), torch.stack([a, b], 1))
    first = torch.tensor([t[0] for t in tokens])
    for i in range(vocab):  # a grid of 32 points a side is off by a point at each border
        assert abs(float((first == i).double().mean()) - float(p[i])) <= 3 / len(grid)


def test_graph_and_side_stream(backend, device):
    for n, d, vocab in ((3, 4, 32003), (40, 2, 500)):
        plan = backend.prepare_verification(sequences=n, drafts=d, vocab=vocab, device=device)
        tensors = [t.to(device) for t in case(n, d, vocab, 1)]
        p, q, drafted, u = tensors
        p, q = p.view(n * (d + 1), vocab), q.view(n * d, vocab)
        tokens, accepted = torch.empty(n, d + 1, dtype=torch.int64, device=device), torch.empty(n, dtype=torch.int32, device=device)
        w = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device=device)
        arguments = dict(proposal=q, tokens=tokens, accepted=accepted, workspace=w)
        side = torch.cuda.Stream(device)
        side.wait_stream(torch.cuda.current_stream(device))
        with torch.cuda.stream(side):
            plan.run(p, drafted, u, **arguments)
        torch.cuda.current_stream(device).wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan.run(p, drafted, u, **arguments)
        for i in range(4):
            for t, new in zip((p, q, drafted, u), case(n, d, vocab, 20 + i)):
                t.copy_(new.view(t.shape))
            plan.run(p, drafted, u, **arguments)
            want = tokens.clone(), accepted.clone()
            tokens.zero_(), accepted.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(tokens, want[0]) and torch.equal(accepted, want[1])


def test_runs_that_share_no_workspace_overlap(backend, device):
    n, d, vocab = 5, 3, 60001
    plan = backend.prepare_verification(sequences=n, drafts=d, vocab=vocab, device=device)
    calls, want = [], []
    for i in range(2):
        p, q, drafted, u = (t.to(device) for t in case(n, d, vocab, 40 + i))
        out = torch.empty(n, d + 1, dtype=torch.int64, device=device), torch.empty(n, dtype=torch.int32, device=device)
        work = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device=device)
        calls.append(((p.view(n * (d + 1), vocab), drafted, u),
                      dict(proposal=q.view(n * d, vocab), tokens=out[0], accepted=out[1], workspace=work)))
        plan.run(*calls[i][0], **calls[i][1])
        want.append([t.clone() for t in out])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device) for _ in range(2)]
    for _ in range(20):
        for (inputs, outputs), stream in zip(calls, streams):
            with torch.cuda.stream(stream):
                plan.run(*inputs, **outputs)
    torch.cuda.synchronize()
    for (_, outputs), (tokens, accepted) in zip(calls, want):
        assert torch.equal(outputs["tokens"], tokens) and torch.equal(outputs["accepted"], accepted)


@pytest.mark.parametrize("vocab", [40, 50001])
def test_a_draft_without_a_probability_is_refused_whatever_its_proposal_and_uniform(backend, device, vocab):
    """Proposals and uniforms below 0 do not let a token of probability 0, or of none, stand, nor is it drawn."""
    n, inf, nan = 6, math.inf, math.nan
    p, q = torch.full((n, 2, vocab), 0.5 / vocab), torch.full((n, 1, vocab), 0.25 / vocab)
    drafted = torch.full((n, 1), 7)
    u = torch.full((n, 2), 0.5)
    p[:, 0, 7] = torch.tensor([0.0, -1.0, nan, inf, 0.0, 0.125])
    q[:, 0, 7] = torch.tensor([-0.25, -2.0, -0.25, -inf, 0.25, -0.25])
    u[4, 0] = -1.0
    plan = backend.prepare_verification(sequences=n, drafts=1, vocab=vocab, device=device)
    for proposal in (q, None):
        tokens, accepted = torch.empty(n, 2, dtype=torch.int64, device=device), torch.empty(n, dtype=torch.int32, device=device)
        uniforms = u if proposal is not None else torch.tensor([[-0.5, 0.5]] * n)
        plan.run(p.view(2 * n, vocab).to(device), drafted.to(device), uniforms.to(device),
                 proposal=None if proposal is None else q.view(n, vocab).to(device), tokens=tokens, accepted=accepted,
                 workspace=torch.empty(plan.workspace_bytes, dtype=torch.uint8, device=device))
        assert accepted.tolist() == [0, 0, 0, 0, 0, 1]
        assert all(token != 7 and 0 <= token < vocab and end == -1 for token, end in tokens[:5].tolist()) and tokens[5, 0] == 7


@pytest.mark.parametrize("certain", [False, True], ids=["drawn", "certain"])
@pytest.mark.parametrize("vocab", [500, 40001])
def test_what_lies_behind_the_last_token_has_no_effect(backend, device, certain, vocab):
    """Drafts past a sequence's count and rows past the drawn token's, of any bits."""
    n, d = 12, 5
    p, q, drafted, u = case(n, d, vocab, 31, 0.3, certain)
    counts = [i % (d + 1) for i in range(n)]
    tokens, accepted = check(backend, device, p, q, drafted, u, counts)
    assert any(a == c < d for a, c in zip(accepted, counts)) and any(a < c for a, c in zip(accepted, counts))
    for value, token in ((math.nan, 2**62), (math.inf, -2**63), (-1.0, vocab - 1)):
        for i in range(n):
            p[i, accepted[i] + 1:] = value
            u[i, counts[i]: d] = value
            drafted[i, counts[i]:] = token
            if q is not None:
                q[i, accepted[i] + 1:], q[i, counts[i]:] = value, value
        assert check(backend, device, p, q, drafted, u, counts) == (tokens, accepted)
