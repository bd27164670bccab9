"""Kept distributions against the definition in 64 bits, and against what sampling draws."""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

FP16, BF16 = torch.float16, torch.bfloat16
TYPES = pytest.mark.parametrize("dtype", [FP16, BF16], ids=["fp16", "bf16"])


def definition(x, t, k, p, least):
    """Probabilities of one row of float64 logits."""
    got = np.zeros(len(x))
    valid = np.flatnonzero(~np.isnan(x) & (x != -np.inf))
    if not len(valid):
        return got
    order = valid[np.argsort(-x[valid], kind="stable")]
    if not t > 0:
        got[order[0]] = 1.0
        return got
    limit = min(k, len(order)) if k > 0 else len(order)
    top = x[order[0]]
    with np.errstate(invalid="ignore"):  # inf - inf of an infinite maximum, replaced by 0
        w = np.exp((np.where(x[order] == top, 0.0, x[order] - top)) / min(t, 3.4028234e38))
    length = min(limit, int((w >= least).sum()))
    if not p >= 1:
        total = np.cumsum(w[:limit])
        length = min(length, int((total - w[:limit] < p * total[-1]).sum()))
    length = max(length, 1)
    got[order[:length]] = w[:length] / w[:length].sum()
    return got


def check(backend, device, logits, t=None, k=None, p=None, least=None):
    rows, vocab = logits.shape
    print(f"case distribution {rows} x {vocab} {logits.dtype}", flush=True)
    plan = backend.prepare_distribution(rows=rows, vocab=vocab, dtype=logits.dtype, device=device)
    base = torch.full((rows * vocab + 32,), -7.0, device=device)
    out = base[16: 16 + rows * vocab].view(rows, vocab)
    args = [None if a is None else torch.as_tensor(a).to(dtype).to(device)
            for a, dtype in ((t, torch.float32), (k, torch.int32), (p, torch.float32), (least, torch.float32))]
    workspace = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device=device)
    plan.run(logits.to(device), *args, probabilities=out, workspace=workspace)
    torch.cuda.synchronize()
    assert bool((base[:16] == -7).all()) and bool((base[16 + rows * vocab:] == -7).all())
    got = out.double().cpu().numpy()
    settings = [np.full(rows, d) if a is None else a.double().cpu().numpy() for a, d in zip(args, (1.0, 0, 1.0, 0.0))]
    x = logits.double().numpy()
    for i in range(rows):
        want = definition(x[i], float(settings[0][i]), int(settings[1][i]), float(settings[2][i]), float(settings[3][i]))
        assert np.array_equal(got[i] > 0, want.astype(np.float32) > 0) or float(want[(got[i] > 0) != (want > 0)].max()) < 1e-36, i
        # The exponential's one step (2^-23), and the roundings of its correction, of 1 / mass and of the product (2^-24 each).
        assert bool((np.abs(got[i] - want) <= 6 * 2.0**-24 * want + 1e-36).all()), (i, [float(s[i]) for s in settings])
    return out


def random_logits(rows, vocab, spread, dtype, seed):
    return (torch.randn(rows, vocab, generator=torch.Generator().manual_seed(seed)) * spread).to(dtype)


@TYPES
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 7), (2, 8), (9, 15), (7, 1000), (4, 1001), (3, 65535), (2, 65529), (2, 70001),
                                        (1, 151936), (2, 248320), (40, 32003), (300, 999)])
def test_settings(backend, device, dtype, rows, vocab):
    rng = np.random.default_rng(vocab)
    logits = random_logits(rows, vocab, 2.5, dtype, rows)
    check(backend, device, logits, rng.choice([0.0, 0.3, 0.8, 1.0, 1.7], rows), rng.choice([0, 1, 2, 20, 1000, vocab, vocab + 5, -3], rows),
          rng.choice([1.0, 0.95, 0.5, 1e-6, 0.0, 1.5], rows), rng.choice([0.0, 0.05, 0.5, 1.0], rows))
    check(backend, device, logits)


@TYPES
def test_each_setting_alone(backend, device, dtype):
    rows, vocab = 24, 5003
    logits = random_logits(rows, vocab, 3.0, dtype, 1)
    check(backend, device, logits, t=[0.5] * rows)
    check(backend, device, logits, k=list(range(rows)))
    check(backend, device, logits, p=[(i + 0.5) / rows for i in range(rows)])
    check(backend, device, logits, least=[i / rows for i in range(rows)])


@pytest.mark.parametrize("vocab", [5, 40000, 65536, 100003])
@pytest.mark.parametrize("value", [0.0, -65504.0, 3.0])
def test_equal_logits_are_cut_by_index(backend, device, vocab, value):
    logits = torch.full((4, vocab), value).half()
    check(backend, device, logits, p=[1.0, 0.9, 1.0, 1e-9], k=[0, 0, vocab // 2, 0])
    logits[:, ::3] = -0.0
    check(backend, device, logits, p=[1.0, 0.9, 1.0, 0.7], k=[0, 0, vocab // 2, 3])


@TYPES
def test_masked_logits(backend, device, dtype):
    lowest, inf, nan = torch.finfo(dtype).min, math.inf, math.nan
    logits = random_logits(10, 30001, 2.0, dtype, 7)
    logits[0, 5:] = -inf
    logits[1, 5:] = lowest
    logits[2, :29990] = -inf
    logits[3] = -inf
    logits[4] = nan
    logits[5, 1000:] = nan
    logits[6, 40] = logits[6, 7777] = inf
    logits[7] = lowest
    logits[8, ::2] = -inf
    logits[9, ::2] = -nan
    for t in (1.0, 0.0, 100.0, 3e38, inf, 1e-30, nan):
        out = check(backend, device, logits, t=[t] * 10, p=[0.9] * 10)
        assert not bool(out[3:5].any())


@pytest.mark.parametrize("rows,vocab", [(3, 5003), (3, 70001), (40, 60001)])
def test_temperatures_and_differences_beyond_32_bits(backend, device, rows, vocab):
    """Inverse temperatures above 3e38, and rows whose largest and smallest logits differ by more."""
    logits = random_logits(rows, vocab, 1.0, BF16, 11)
    far, small = logits.float().mul(1e38).clamp(-3e38, 3e38).to(BF16), logits.float().mul(1e-38).to(BF16)
    ties = logits.clamp(max=1.0)
    for t in (3e38, 3.4e38, 1e30, 1e-30, 1e-38, 1e-40, 1e-45):
        for x in (far, small, ties):
            check(backend, device, x, t=[t] * rows)
            check(backend, device, x, t=[t] * rows, p=[0.9, 1.0, 1.0] + [1.0] * (rows - 3), k=[0, 0, 9] + [0] * (rows - 3))


@TYPES
@pytest.mark.parametrize("rows", [2, 31, 32, 33])
@pytest.mark.parametrize("vocab", [57344, 57345, 57352, 65536 + 8, 147456 + 3])
def test_few_long_rows(backend, device, dtype, rows, vocab):
    logits = random_logits(rows, vocab, 2.5, dtype, vocab)
    check(backend, device, logits, k=[(0, 1, 50, 256, 257, 0)[i % 6] for i in range(rows)], p=[(1.0, 1.0, 0.9)[i % 3] for i in range(rows)])


@pytest.mark.parametrize("rows", [2, 40])
def test_masked_logits_of_long_rows(backend, device, rows):
    inf, nan, vocab = math.inf, math.nan, 70003
    for dtype, fill in ((FP16, -inf), (BF16, nan), (BF16, -inf), (FP16, inf)):
        for at in (0, 3, 8191, 8192, 70002):  # the only other logit
            logits = torch.full((rows, vocab), fill, dtype=dtype)
            logits[0, at] = -2.0
            check(backend, device, logits, k=[1] + [0] * (rows - 1))
            check(backend, device, logits)


def test_the_distribution_is_what_sampling_draws_from(backend, device):
    """The sampled token's probability, row by row, for random settings."""
    rows, vocab = 64, 9001
    logits = random_logits(rows, vocab, 2.5, BF16, 9).to(device)
    gen = torch.Generator().manual_seed(3)
    settings = [torch.rand(rows, generator=gen).to(device) + 0.3, torch.randint(0, 60, (rows,), generator=gen, dtype=torch.int32).to(device),
                torch.rand(rows, generator=gen).to(device), 0.1 * torch.rand(rows, generator=gen).to(device)]
    plan = backend.prepare_distribution(rows=rows, vocab=vocab, dtype=BF16, device=device)
    p = plan.run(logits, *settings, probabilities=torch.empty(rows, vocab, device=device),
                 workspace=torch.empty(plan.workspace_bytes, dtype=torch.uint8, device=device))
    sampling = backend.prepare_sampling(rows=rows, vocab=vocab, dtype=BF16, device=device)
    tokens, chances = torch.empty(rows, dtype=torch.int64, device=device), torch.empty(rows, device=device)
    for u in (0.0, 0.3, 0.99, 1.0):
        sampling.run(logits, torch.full((rows,), u, device=device), *settings, tokens=tokens, probabilities=chances)
        got = p.gather(1, tokens[:, None])[:, 0]
        assert bool(((got - chances).abs() <= 7 * 2.0**-24 * chances).all())


def test_graph_and_side_stream(backend, device):
    for rows, vocab in ((2, 70001), (300, 2000)):
        plan = backend.prepare_distribution(rows=rows, vocab=vocab, dtype=FP16, device=device)
        logits, k = torch.zeros(rows, vocab, dtype=FP16, device=device), torch.full((rows,), 50, dtype=torch.int32, device=device)
        p, w = torch.empty(rows, vocab, device=device), torch.empty(plan.workspace_bytes, dtype=torch.uint8, device=device)
        side = torch.cuda.Stream(device)
        side.wait_stream(torch.cuda.current_stream(device))
        with torch.cuda.stream(side):
            plan.run(logits, None, k, probabilities=p, workspace=w)
        torch.cuda.current_stream(device).wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan.run(logits, None, k, probabilities=p, workspace=w)
        for i in range(4):
            logits.copy_(random_logits(rows, vocab, 2.0, FP16, i))
            plan.run(logits, None, k, probabilities=p, workspace=w)
            want = p.clone()
            p.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(p, want)


def test_runs_that_share_no_workspace_overlap(backend, device):
    for rows, vocab in ((4, 70001), (64, 30001)):
        plan = backend.prepare_distribution(rows=rows, vocab=vocab, dtype=BF16, device=device)
        k = torch.tensor([0, 50, 400, 1] * (rows // 4), dtype=torch.int32, device=device)
        inputs = [random_logits(rows, vocab, 2.5, BF16, i).to(device) for i in range(2)]
        outs = [torch.empty(rows, vocab, device=device) for _ in range(2)]
        work = [torch.empty(plan.workspace_bytes, dtype=torch.uint8, device=device) for _ in range(2)]
        want = [plan.run(x, None, k, probabilities=torch.empty_like(outs[0]), workspace=work[0]).clone() for x in inputs]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(device) for _ in range(2)]
        for _ in range(10):
            for i, stream in enumerate(streams):
                with torch.cuda.stream(stream):
                    plan.run(inputs[i], None, k, probabilities=outs[i], workspace=work[i])
        torch.cuda.synchronize()
        for got, wanted in zip(outs, want):
            assert torch.equal(got, wanted)


@pytest.mark.parametrize("rows,vocab,exponent,apart", [(2, 151936, 7, 8192), (33, 57001, 8, 57001), (33, 70003, 9, 70003)])
def test_a_tail_that_holds_the_mass_and_is_no_multiple_of_the_largest_logits_last_bit(backend, device, rows, vocab, exponent, apart):
    """A difference of two logits that 32 bits do not hold: rounding it would move every weight of the tail, and so the mass, by
    6 to 9 x 2^-24. Else a weight errs by the exponential's step (2 x 2^-24) and its argument's rounding (0.2 x 2^-24), the mass by
    as much (the tail's sums are exact), and a probability by both and its own rounding: 5.4 x 2^-24, within check()'s 6."""
    far, near = 8.0625, 1.984375 * 2.0**-22
    for top, tail in ((far, near), (near, -far), (far, -near)):
        logits = torch.full((rows, vocab), tail, dtype=BF16)
        for i in range(rows):
            logits[i, 17 * i:: apart] = top
        check(backend, device, logits, t=[far / exponent] * rows)
