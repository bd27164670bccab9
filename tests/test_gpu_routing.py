"""Routing against the definition in 64 bits: experts equal and in order, weights to one rounding."""

from itertools import combinations
import math

import pytest
import torch

from venturi_amd.q4 import quantize_q4_rtn
from venturi_amd.moe import MoEGeometry, Q4ExpertBank

pytestmark = pytest.mark.gpu

FP16, BF16, FP32 = torch.float16, torch.bfloat16, torch.float32
NAMES = {FP16: "fp16", BF16: "bf16", FP32: "fp32"}


def definition(logits, bias, top_k, **settings):
    """(ids, weights) of one row, expert by expert."""
    return next(definitions(logits, bias, top_k, **settings))


def definitions(logits, bias, top_k, *, score="softmax", groups=1, kept_groups=1, group_rank="pairs", renormalize=True, scale=1.0):
    """The definition's (ids, weights), and with a bias those of groups that come as near as 64 bits tell sums apart: a score
    errs by 2^-53 of it for every expert in its sum, the exponentials, the division and the bias's addition, twice in a rank
    of two."""
    x = [float(v) for v in logits.double()]
    broken = any(math.isnan(v) for v in x) or (score == "softmax" and math.inf in x)
    if not broken:
        if score == "sigmoid":
            s = [1 / (1 + math.exp(-v)) if v > -700 else 0.0 for v in x]
        else:
            top = max(x)
            e = [0.0 if v == -math.inf else math.exp(v - top) for v in x]
            s = [v / sum(e) if sum(e) else 0.0 for v in e]
        c = [-math.inf if v == -math.inf else t + (0.0 if bias is None else float(bias[i])) for i, (v, t) in enumerate(zip(x, s))]
        broken = any(math.isnan(v) for v in c)
    if broken:
        yield [-1] * top_k, [math.nan] * top_k
        return
    size = len(x) // groups
    ranks = []
    for g in range(groups):
        best = sorted(c[g * size: (g + 1) * size], reverse=True)
        ranks.append(best[0] + best[1] if group_rank == "pairs" and size > 1 and best[1] > -math.inf else best[0])
    first = sorted(range(groups), key=lambda g: (-ranks[g], g))[:kept_groups]
    others = combinations(range(groups), kept_groups) if bias is not None and 1 < groups <= 8 else ()
    for kept in (first, *others):
        out = [ranks[g] for g in range(groups) if g not in kept]
        if out and min(ranks[g] for g in kept) < max(out) - (len(x) + 6) * 2.0**-52 * (1 + abs(max(out))):
            continue
        order = sorted((e for e in range(len(x)) if e // size in kept), key=lambda e: (-c[e], e))[:top_k]
        w = [s[e] for e in order]
        if renormalize:
            w = [v / sum(w) if sum(w) else 0.0 for v in w]
        yield order, [v * scale for v in w]


def check(backend, device, logits, bias=None, top_k=1, score_dtype=FP16, **settings):
    tokens, experts = logits.shape
    print(f"case routing {tokens} x {experts} top {top_k} {logits.dtype} {settings}", flush=True)
    plan = backend.prepare_routing(tokens=tokens, experts=experts, top_k=top_k, dtype=logits.dtype, device=device,
                                   score_dtype=score_dtype, **settings)
    ids = torch.full((tokens * top_k + 16,), -7, dtype=torch.int64, device=device)
    scores = torch.full((tokens * top_k + 16,), -7.0, dtype=score_dtype, device=device)
    inner = slice(8, 8 + tokens * top_k)
    plan.run(logits.to(device), None if bias is None else bias.to(device), indices=ids[inner].view(tokens, top_k),
             scores=scores[inner].view(tokens, top_k))
    torch.cuda.synchronize()
    for t in (ids, scores):
        assert bool((t[: inner.start] == -7).all()) and bool((t[inner.stop:] == -7).all())
    got, weights = ids[inner].view(tokens, top_k).cpu(), scores[inner].view(tokens, top_k).double().cpu()
    # One rounding to the scores' type and one to 32 bits before it; the smallest fp16 number's half below.
    step = torch.finfo(score_dtype).eps / 2 + 2.0**-24 + 2.0**-40
    least = {FP16: 2.0**-25, BF16: 2.0**-134, FP32: 2.0**-126}[score_dtype]
    for i in range(tokens):
        want, share = definition(logits[i], bias, top_k, **settings)
        if got[i].tolist() != want:
            near = (d for d in definitions(logits[i], bias, top_k, **settings) if d[0] == got[i].tolist())
            want, share = next(near, (want, share))
        assert got[i].tolist() == want, (i, got[i].tolist(), want)
        for a, b in zip(weights[i].tolist(), share):
            assert (math.isnan(a) and math.isnan(b)) or abs(a - b) <= step * abs(b) * 1.01 + least, (i, a, b)
    return got, weights


def random_logits(tokens, experts, dtype, seed, spread=1.5):
    return (torch.randn(tokens, experts, generator=torch.Generator().manual_seed(seed)) * spread).to(dtype)


def random_bias(experts, seed):
    return 0.05 * torch.randn(experts, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("dtype", [FP16, BF16, FP32], ids=NAMES.values())
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,top_k", [(1, 1), (2, 2), (7, 3), (8, 2), (16, 16), (60, 4), (64, 8), (65, 6), (100, 1), (128, 8),
                                           (129, 8), (160, 6), (256, 8), (300, 5), (384, 6), (512, 10), (513, 16), (1000, 9), (1024, 16)])
def test_scores(backend, device, dtype, score, experts, top_k):
    for tokens in (1, 6, 33):
        logits = random_logits(tokens, experts, dtype, experts + tokens)
        check(backend, device, logits, None, top_k, score=score)
        check(backend, device, logits, random_bias(experts, 1), top_k, score=score, scale=2.5, renormalize=tokens != 6)


@pytest.mark.parametrize("dtype", [FP16, BF16, FP32], ids=NAMES.values())
@pytest.mark.parametrize("experts,groups,kept,top_k", [(4, 4, 2, 2), (8, 2, 1, 4), (60, 4, 2, 6), (64, 8, 4, 8), (128, 8, 3, 8),
                                                       (160, 8, 3, 6), (256, 8, 4, 8), (256, 64, 5, 16), (512, 16, 4, 8), (1000, 10, 1, 16),
                                                       (1024, 64, 64, 16), (320, 64, 3, 9), (96, 3, 2, 5)])
def test_groups(backend, device, dtype, experts, groups, kept, top_k):
    for score in ("softmax", "sigmoid"):
        for rank in ("pairs", "max"):
            logits = random_logits(9, experts, dtype, experts)
            for bias in (None, random_bias(experts, 2)):
                check(backend, device, logits, bias, top_k, score=score, groups=groups, kept_groups=kept, group_rank=rank)


@pytest.mark.parametrize("score_dtype", [FP16, BF16, FP32], ids=NAMES.values())
def test_types_of_the_scores(backend, device, score_dtype):
    for dtype in NAMES:
        check(backend, device, random_logits(20, 128, dtype, 3), None, 8, score_dtype=score_dtype, score="sigmoid", renormalize=False)
        check(backend, device, random_logits(20, 128, dtype, 4, 8.0), None, 8, score_dtype=score_dtype, renormalize=False, scale=-3.0)


@pytest.mark.parametrize("dtype", [FP16, BF16, FP32], ids=NAMES.values())
@pytest.mark.parametrize("experts", [8, 64, 128, 256, 1000])
def test_equal_scores_go_by_index(backend, device, dtype, experts):
    gen = torch.Generator().manual_seed(5)
    logits = torch.randint(0, 3, (12, experts), generator=gen).to(dtype)
    logits[0] = 0.0
    logits[1, ::2] = -0.0
    logits[1, 1::2] = 0.0
    for score in ("softmax", "sigmoid"):
        check(backend, device, logits, None, 8, score=score)
        check(backend, device, logits, torch.zeros(experts), 8, score=score)
        check(backend, device, logits, None, 4, score=score, groups=4, kept_groups=2)
        check(backend, device, logits, (torch.arange(experts) % 2).float(), 4, score=score, groups=4, kept_groups=2)


def test_scores_that_differ_in_their_last_bits(backend, device):
    """The order of what 32 bits cannot tell apart: neighbouring logits and biases."""
    gen = torch.Generator().manual_seed(6)
    steps = torch.randint(0, 6, (40, 64), generator=gen, dtype=torch.int32)
    logits = (torch.full((40, 64), 9.0).view(torch.int32) + steps).view(FP32)
    for score in ("softmax", "sigmoid"):
        for top_k in (1, 8, 16):
            check(backend, device, logits, None, top_k, score=score)
            check(backend, device, logits, torch.zeros(64), top_k, score=score)
    wide = (torch.full((5, 700), -3.0).view(torch.int32) + torch.randint(0, 2000, (5, 700), generator=gen, dtype=torch.int32)).view(FP32)
    for top_k in (3, 16):
        check(backend, device, wide, random_bias(700, 5) * 1e-6, top_k, score="sigmoid")
        check(backend, device, wide, random_bias(700, 6) * 1e-7, top_k, score="softmax", renormalize=False)
    bias = (torch.full((64,), 0.001).view(torch.int32) + torch.randperm(64, generator=gen).int()).view(FP32)
    check(backend, device, torch.zeros(2, 64), bias, 8, score="sigmoid")
    check(backend, device, torch.zeros(2, 64), bias, 4, score="softmax", groups=8, kept_groups=2)
    check(backend, device, logits, bias, 8, score="softmax")


@pytest.mark.parametrize("experts", [64, 128, 252, 256, 512, 1008])
def test_near_scores_and_groups_of_a_bias(backend, device, experts):
    """What 32-bit scores cannot tell apart, sigmoid scores with biases on both sides of 4, and masked groups."""
    gen = torch.Generator().manual_seed(experts)
    steps = torch.randperm(experts, generator=gen).float()
    settings = dict(score="sigmoid", groups=4, kept_groups=2)
    for spacing in (2.0**-25, 2.0**-22, 2.0**-19):
        for rank in ("pairs", "max"):
            check(backend, device, torch.zeros(3, experts), 0.25 + spacing * steps, 8, group_rank=rank, **settings)
        check(backend, device, torch.zeros(3, experts), 0.25 + spacing * steps, 8, score="sigmoid")
    logits = torch.randn(9, experts, generator=gen)
    for scale in (1e-6, 0.1, 1.0, 3.0, 1e4):
        bias = scale * torch.randn(experts, generator=gen)
        check(backend, device, logits, bias, 8, **settings)
        check(backend, device, 30 * logits, bias, 8, **settings)
    bias[::3], bias[1::3] = 4.0, -4.0
    check(backend, device, logits, bias, 8, **settings)
    bias[3] = 4.0 + 2.0**-21
    check(backend, device, logits, bias, 8, **settings)
    logits[:, : 3 * experts // 4] = -math.inf  # fewer groups than are kept
    logits[4:, experts // 2:] = -math.inf
    logits[2, 5] = 1.0
    for bias in (0.1 * torch.randn(experts, generator=gen), 9.0 * torch.randn(experts, generator=gen)):
        for rank in ("pairs", "max"):
            check(backend, device, logits, bias, 8, group_rank=rank, **settings)
            check(backend, device, logits.half(), bias, 8, group_rank=rank, **settings)


@pytest.mark.parametrize("dtype", [FP16, BF16, FP32], ids=NAMES.values())
@pytest.mark.parametrize("experts", [16, 64, 160])
def test_masks_and_values_that_are_no_numbers(backend, device, dtype, experts):
    inf, nan = math.inf, math.nan
    logits = random_logits(14, experts, dtype, 7)
    logits[0] = -inf
    logits[1, 3:] = -inf
    logits[2, : experts - 2] = -inf
    logits[3, 5] = nan
    logits[4, experts - 1] = inf
    logits[5] = torch.finfo(dtype).min
    logits[6] = torch.finfo(dtype).max
    logits[7] = -90.0
    logits[8, ::2] = -inf
    logits[9, : experts // 2] = -inf
    logits[10, 0] = 300.0
    for score in ("softmax", "sigmoid"):
        for settings in ({}, dict(groups=4, kept_groups=2), dict(groups=2, kept_groups=1, group_rank="max"), dict(renormalize=False)):
            check(backend, device, logits, None, 4, score=score, **settings)
            check(backend, device, logits, random_bias(experts, 3), 4, score=score, **settings)
        bias = random_bias(experts, 4)
        bias[1], bias[2] = -inf, inf
        check(backend, device, logits, bias, 4, score=score)
        bias[7] = nan
        check(backend, device, logits, bias, 4, score=score)


def test_many_tokens(backend, device):
    """More tokens than a launch has workgroups at once, against the same rows routed few at a time."""
    logits = random_logits(70001, 128, BF16, 8).to(device)
    plan = backend.prepare_routing(tokens=70001, experts=128, top_k=8, dtype=BF16, device=device)
    ids, scores = torch.empty(70001, 8, dtype=torch.int64, device=device), torch.empty(70001, 8, dtype=FP16, device=device)
    plan.run(logits, indices=ids, scores=scores)
    x = logits.double()
    order = x.sort(dim=-1, descending=True, stable=True).indices[:, :8]
    assert torch.equal(ids, order)
    w = torch.softmax(x.gather(1, order), -1)
    assert float((scores.double() - w).abs().max()) <= 2.0**-11 + 2.0**-24


def test_graph_and_side_stream(backend, device):
    for tokens, settings in ((1, {}), (300, dict(score="sigmoid", groups=8, kept_groups=4))):
        plan = backend.prepare_routing(tokens=tokens, experts=128, top_k=8, dtype=FP32, device=device, **settings)
        logits, bias = torch.zeros(tokens, 128, device=device), random_bias(128, 9).to(device)
        ids, scores = torch.empty(tokens, 8, dtype=torch.int64, device=device), torch.empty(tokens, 8, dtype=FP16, device=device)
        side = torch.cuda.Stream(device)
        side.wait_stream(torch.cuda.current_stream(device))
        with torch.cuda.stream(side):
            plan.run(logits, bias, indices=ids, scores=scores)
        torch.cuda.current_stream(device).wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan.run(logits, bias, indices=ids, scores=scores)
        for i in range(4):
            logits.copy_(random_logits(tokens, 128, FP32, i))
            plan.run(logits, bias, indices=ids, scores=scores)
            want = ids.clone(), scores.clone()
            ids.zero_(), scores.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(ids, want[0]) and torch.equal(scores, want[1])


def test_routed_tokens_go_through_the_experts(backend, device):
    """Router logits to the experts' combined output: what the bank gives for the definition's ids and scores, and a NaN row
    for a token whose logits are no numbers."""
    geometry = MoEGeometry(hidden_size=64, num_experts=16, top_k=4, intermediate_size=48)
    gen = torch.Generator().manual_seed(11)
    experts = [(quantize_q4_rtn(torch.randn(96, 64, generator=gen) * 0.1), quantize_q4_rtn(torch.randn(64, 48, generator=gen) * 0.1))
               for _ in range(16)]
    bank = Q4ExpertBank.upload(backend, geometry, experts, device=device)
    tokens = 9
    plan = bank.prepare(tokens=tokens)
    x, logits = torch.randn(tokens, 64, generator=gen).half().to(device), random_logits(tokens, 16, FP16, 12)
    logits[4, 3] = math.nan
    router = backend.prepare_routing(tokens=tokens, experts=16, top_k=4, dtype=FP16, device=device, score="sigmoid", scale=2.0)
    ids, scores = torch.empty(tokens, 4, dtype=torch.int64, device=device), torch.empty(tokens, 4, dtype=FP16, device=device)
    router.run(logits.to(device), random_bias(16, 13).to(device), indices=ids, scores=scores)
    outs = []
    workspace = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device=device)
    by_hand = [definition(row, random_bias(16, 13), 4, score="sigmoid", scale=2.0) for row in logits]
    want_ids = torch.tensor([i for i, _ in by_hand], device=device)
    want_scores = torch.tensor([w for _, w in by_hand], dtype=torch.float64).float().half().to(device)
    for i, s in ((ids, scores), (want_ids, want_scores)):
        outs.append(torch.empty(tokens, 64, dtype=FP16, device=device))
        plan.run(x, i, s, out=outs[-1], workspace=workspace)
    assert bool(outs[0][4].isnan().all()) and torch.equal(outs[0].isnan(), outs[1].isnan())
    fine = [i for i in range(tokens) if i != 4]
    assert torch.equal(outs[0][fine], outs[1][fine])


@pytest.mark.parametrize("dtype", [FP16, BF16, FP32], ids=NAMES.values())
@pytest.mark.parametrize("experts", [16, 64, 160, 1024])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_masked_experts_come_after_those_with_a_bias_of_minus_infinity(backend, device, dtype, experts, score):
    """Experts and groups by (masked, c, index); a group of masked experts alone comes after all others."""
    inf, top_k = math.inf, 6
    logits = random_logits(5, experts, dtype, 21)
    logits[:, ::2] = -inf
    logits[1, : experts // 4] = -inf
    logits[2, 3:] = -inf
    logits[3, : experts - 3] = -inf
    logits[4] = -inf
    bias = torch.full((experts,), -inf)
    bias[5], bias[experts // 2 + 1], bias[0] = 0.25, inf, inf
    for groups, kept, rank in ((1, 1, "max"), (4, 2, "pairs"), (4, 2, "max"), (8, 6, "pairs")):
        size = experts // groups
        plan = backend.prepare_routing(tokens=5, experts=experts, top_k=top_k, dtype=dtype, device=device, score=score, groups=groups,
                                       kept_groups=kept, group_rank=rank, score_dtype=FP32, renormalize=False)
        ids = torch.empty(5, top_k, dtype=torch.int64, device=device)
        weights = torch.empty(5, top_k, device=device)
        plan.run(logits.to(device), bias.to(device), indices=ids, scores=weights)
        for x, got, shares in zip(logits.double(), ids.tolist(), weights.double().cpu()):
            s = torch.sigmoid(x) if score == "sigmoid" else torch.softmax(x, -1).nan_to_num(0.0)
            masked, c = (x == -inf).tolist(), (s + bias.double()).tolist()

            def group(g):
                there = sorted((c[e] for e in range(g * size, (g + 1) * size) if not masked[e]), reverse=True)[: 2 if rank == "pairs" else 1]
                return not there, -(inf if inf in there else sum(there)), g

            order = [g for g in sorted(range(groups), key=group)][:kept]
            order = sorted((e for e in range(experts) if e // size in order), key=lambda e: (masked[e], 0.0 if masked[e] else -c[e], e))
            assert got == order[:top_k], (groups, rank)
            want = torch.where(x == -inf, 0.0, s)[got]
            assert bool(((shares - want).abs() <= 2.0**-23 * want + 2.0**-126).all())


@pytest.mark.parametrize("bias", [None, 0.0], ids=["none", "zeros"])
def test_scores_below_2_to_the_minus_1000_count_as_0(backend, device, bias):
    """Shares of sigmoids down to logits of -693, and weights of 0 below; experts in order either way."""
    logits = -692.0 - torch.arange(16.0).flip(0) / 16  # the largest last, all above -693.1
    logits = torch.stack([logits, logits - 2, logits.clamp(min=-692.5)])
    logits[2, 9] = -1000.0
    offsets = None if bias is None else torch.full((16,), bias, device=device)
    plan = backend.prepare_routing(tokens=3, experts=16, top_k=8, dtype=FP32, device=device, score="sigmoid", score_dtype=FP32)
    ids, weights = torch.empty(3, 8, dtype=torch.int64, device=device), torch.empty(3, 8, device=device)
    plan.run(logits.to(device), offsets, indices=ids, scores=weights)
    weights = weights.double().cpu()
    for row in (0, 2):
        want = torch.softmax(logits[row].double()[ids[row].cpu()], 0)  # 1 / (1 + exp(-x)) is exp(x) here
        assert bool(((weights[row] - want).abs() <= 2.0**-23 * want).all())
    assert ids[0].tolist() == list(range(15, 7, -1)) and not bool(weights[1].any())
    assert ids[1].tolist() == (list(range(15, 7, -1)) if bias is None else list(range(8)))
