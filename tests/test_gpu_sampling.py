"""Sampling against the definition in 64 bits: tokens equal, probabilities to fp32 rounding."""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

FP16, BF16 = torch.float16, torch.bfloat16


def definition(x, u, t, k, p, least):
    """(token, probability) of one row of float64 logits."""
    valid = np.flatnonzero(~np.isnan(x) & (x != -np.inf))
    if not len(valid):
        return -1, 0.0
    order = valid[np.argsort(-x[valid], kind="stable")]
    if not t > 0:
        return int(order[0]), 1.0
    limit = min(k, len(order)) if k > 0 else len(order)
    top = x[order[0]]
    with np.errstate(invalid="ignore"):  # inf - inf of an infinite maximum, replaced by 0
        w = np.exp((np.where(x[order] == top, 0.0, x[order] - top)) / min(t, 3.4028234e38))
    length = min(limit, int((w >= least).sum()))
    if not p >= 1:
        total = np.cumsum(w[:limit])
        length = min(length, int((total - w[:limit] < p * total[-1]).sum()))
    length = max(length, 1)
    total = np.cumsum(w[:length])
    place = int((total <= u * total[-1]).sum())
    place = max(min(place, int((w[:length] > 0).sum()) - 1), 0)
    return int(order[place]), float(w[place] / total[-1])


def check(backend, device, logits, u, t=None, k=None, p=None, least=None):
    rows, vocab = logits.shape
    plan = backend.prepare_sampling(rows=rows, vocab=vocab, dtype=logits.dtype, device=device)
    tokens = torch.full((rows,), -7, dtype=torch.int64, device=device)
    chances = torch.full((rows,), -7.0, device=device)
    args = [None if a is None else torch.as_tensor(a).to(dtype).to(device)
            for a, dtype in ((t, torch.float32), (k, torch.int32), (p, torch.float32), (least, torch.float32))]
    plan.run(logits.to(device), torch.as_tensor(u).float().to(device), *args, tokens=tokens, probabilities=chances)
    torch.cuda.synchronize()
    tokens, chances = tokens.cpu().tolist(), chances.cpu().tolist()
    settings = [np.full(rows, d) if a is None else a.double().cpu().numpy() for a, d in zip(args, (1.0, 0, 1.0, 0.0))]
    x, u = logits.double().numpy(), torch.as_tensor(u).float().double().numpy()
    for i in range(rows):
        token, chance = definition(x[i], u[i], float(settings[0][i]), int(settings[1][i]), float(settings[2][i]), float(settings[3][i]))
        assert tokens[i] == token, (i, tokens[i], token, [s[i] for s in settings], u[i])
        assert abs(chances[i] - chance) <= 2.0**-24 * chance * 1.001 + 1e-12
    return tokens


def random_logits(rows, vocab, spread, dtype, seed):
    return (torch.randn(rows, vocab, generator=torch.Generator().manual_seed(seed)) * spread).to(dtype)


def uniforms(rows, seed):
    return torch.rand(rows, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("dtype", [FP16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 7), (2, 8), (7, 1000), (4, 1001), (3, 65535), (2, 65529), (2, 70001),
                                        (1, 151936), (2, 248320), (40, 32000), (300, 999)])
def test_settings(backend, device, dtype, rows, vocab):
    print(f"case sampling {rows} x {vocab} {dtype}", flush=True)
    rng = np.random.default_rng(vocab)
    logits = random_logits(rows, vocab, 2.5, dtype, rows)
    check(backend, device, logits, uniforms(rows, vocab), rng.choice([0.0, 0.3, 0.8, 1.0, 1.7], rows),
          rng.choice([0, 1, 2, 20, 1000, vocab, vocab + 5, -3], rows), rng.choice([1.0, 0.95, 0.5, 1e-6, 0.0, 1.5], rows),
          rng.choice([0.0, 0.05, 0.5, 1.0], rows))


@pytest.mark.parametrize("dtype", [FP16, BF16], ids=["fp16", "bf16"])
def test_defaults_and_each_setting_alone(backend, device, dtype):
    rows, vocab = 24, 5003
    logits, u = random_logits(rows, vocab, 3.0, dtype, 1), uniforms(rows, 2)
    check(backend, device, logits, u)
    check(backend, device, logits, u, t=[0.5] * rows)
    check(backend, device, logits, u, k=list(range(rows)))
    check(backend, device, logits, u, p=[(i + 0.5) / rows for i in range(rows)])
    check(backend, device, logits, u, least=[i / rows for i in range(rows)])


def test_ends_of_the_uniforms(backend, device):
    logits = random_logits(6, 3001, 2.0, FP16, 3)
    for u in (0.0, 2.0**-30, 1 - 2.0**-24, 1.0, 2.0, -1.0):
        check(backend, device, logits, [u] * 6, k=[0, 5, 0, 1, 0, 3001], p=[1.0, 1.0, 0.7, 0.7, 1.0, 0.2])


@pytest.mark.parametrize("vocab", [5, 40000, 65536, 100003, 248320])
@pytest.mark.parametrize("value", [0.0, -65504.0, 3.0])
def test_equal_logits(backend, device, vocab, value):
    """One class of every count, past the 16-bit counters; ties go by index."""
    logits = torch.full((3, vocab), value).half()
    tokens = check(backend, device, logits, [0.0, 0.5, 0.999], p=[1.0, 0.9, 1.0], k=[0, 0, vocab // 2])
    assert tokens[0] == 0


def test_few_values_many_times(backend, device):
    gen = torch.Generator().manual_seed(5)
    logits = torch.randint(0, 4, (6, 200003), generator=gen).half() - 2
    logits[:, 17] = -0.0
    check(backend, device, logits, uniforms(6, 6), t=[1.0, 0.3, 2.0, 1.0, 1.0, 5.0], k=[0, 60000, 100001, 3, 0, 0],
          p=[1.0, 0.9, 0.99, 0.5, 0.3, 1.0])


@pytest.mark.parametrize("dtype", [FP16, BF16], ids=["fp16", "bf16"])
def test_masked_logits(backend, device, dtype):
    lowest, inf, nan = torch.finfo(dtype).min, math.inf, math.nan
    logits = random_logits(9, 100000, 2.0, dtype, 7)
    logits[0, 5:] = -inf
    logits[1, 5:] = lowest
    logits[2, :99990] = -inf
    logits[3] = -inf
    logits[4] = nan
    logits[5, 1000:] = nan
    logits[6, 40] = logits[6, 77777] = inf
    logits[7] = lowest
    logits[8, ::2] = -inf
    for t in (1.0, 0.0, 100.0, 3e38, inf, 1e-30):
        tokens = check(backend, device, logits, uniforms(9, 8), t=[t] * 9, p=[0.9] * 9)
        assert tokens[3] == tokens[4] == -1


@pytest.mark.parametrize("dtype", [FP16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("vocab", [1000, 100001, 2**20])
def test_signs(backend, device, dtype, vocab):
    """The chosen class is looked for among the logits that may hold it: negative ones, zeros of either sign, NaN beside them."""
    logits = random_logits(8, vocab, 2.0, dtype, 11)
    logits[0] = -logits[0].abs() - 0.25
    logits[1] = -logits[1].abs()
    logits[1, ::3] = -0.0
    logits[2, : vocab // 2] = -logits[2, : vocab // 2].abs() - 5
    logits[2, vocab // 2:] = -logits[2, vocab // 2:].abs()
    logits[3, ::2] = -math.nan
    logits[3] = -logits[3].abs() - 1
    logits[4, ::2] = math.nan
    logits[5] = -0.0
    logits[5, vocab - 1] = 0.0
    logits[6, : vocab - 3] = -math.inf
    logits[7] = -logits[7].abs()
    logits[7, vocab - 2] = 1.0
    for k in (0, 1, 40):
        check(backend, device, logits, [0.999, 0.4, 0.8, 0.6, 0.9, 0.99, 0.5, 0.7], k=[k] * 8)


def test_settings_that_are_no_number(backend, device):
    logits = random_logits(4, 300, 2.0, FP16, 9)
    nan = math.nan
    check(backend, device, logits, [0.9] * 4, t=[nan, 1.0, 1.0, -2.0], p=[1.0, nan, 1.0, 1.0], least=[0.0, 0.0, nan, 2.0])
    check(backend, device, logits, [nan] * 4)


def test_many_draws_follow_the_weights(backend, device):
    """The uniforms of a fine grid: every token comes as often as its share says, to one."""
    rows, vocab = 4096, 11
    row = random_logits(1, vocab, 1.5, FP16, 10)
    tokens = check(backend, device, row.repeat(rows, 1), (torch.arange(rows) + 0.5) / rows)
    share = torch.softmax(row.double(), -1)[0]
    for i in range(vocab):
        assert abs(tokens.count(i) - rows * float(share[i])) <= 2


def test_graph_and_side_stream(backend, device):
    for rows, vocab in ((2, 70001), (300, 2000)):
        plan = backend.prepare_sampling(rows=rows, vocab=vocab, dtype=FP16, device=device)
        logits = torch.zeros(rows, vocab, dtype=FP16, device=device)
        u, k = torch.zeros(rows, device=device), torch.full((rows,), 50, dtype=torch.int32, device=device)
        tokens, chances = torch.empty(rows, dtype=torch.int64, device=device), torch.empty(rows, device=device)
        side = torch.cuda.Stream(device)
        side.wait_stream(torch.cuda.current_stream(device))
        with torch.cuda.stream(side):
            plan.run(logits, u, None, k, tokens=tokens, probabilities=chances)
        torch.cuda.current_stream(device).wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan.run(logits, u, None, k, tokens=tokens, probabilities=chances)
        for i in range(4):
            logits.copy_(random_logits(rows, vocab, 2.0, FP16, i))
            u.copy_(uniforms(rows, i))
            plan.run(logits, u, None, k, tokens=tokens, probabilities=chances)
            want = tokens.clone(), chances.clone()
            tokens.zero_(), chances.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(tokens, want[0]) and torch.equal(chances, want[1])


@pytest.mark.parametrize("dtype,value", [(FP16, 1.0), (FP16, 1.0009765625), (BF16, 1.0), (BF16, 1.0078125)],
                         ids=["fp16-even", "fp16-odd", "bf16-even", "bf16-odd"])
@pytest.mark.parametrize("vocab", [*range(106497, 106504), 106509, 106510, 155649])
def test_a_class_that_fills_the_last_segment_and_the_ragged_ends(backend, device, dtype, value, vocab):
    """Logits are counted 57344 and then 49152 at a time: a class one short of 16384 before the last segment that has all of
    that, and the row's ends as well, in rows of every alignment."""
    logits = torch.full((8, vocab), value).to(dtype)
    for i in range(8):
        head = -i * vocab % 8
        logits[i, head: head + (vocab - head) // 8 * 8 - 49152 - 16383] = 0.0
        logits[i, head + i] = value + 1  # the largest, once
    check(backend, device, logits, [0.999, 0.3, 0.7, 0.0, 0.9, 0.5, 0.99, 0.1], k=[0, 0, 2, 50000, 65537, 66000, 0, 70000],
          p=[1.0, 0.9, 1.0, 1.0, 1.0, 0.7, 0.99, 0.5])
