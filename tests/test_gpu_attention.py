"""Causal attention over packed sequences against the formula in 64 bits.

The kernel rounds weights to the model's type (half a step); the bound is attention_oracle.attention_bound."""

import pytest
import torch

from attention_oracle import attend, attention_bound, half_step

pytestmark = pytest.mark.gpu

FP16, BF16 = torch.float16, torch.bfloat16


def run(backend, device, q, k, v, qo, ko, hq, hk, d, dtype, scale=None):
    plan = backend.prepare_attention(tokens=len(q), keys=len(k), sequences=len(qo) - 1, q_heads=hq, kv_heads=hk, head_dim=d,
                                     dtype=dtype, device=device, scale=scale)
    out = torch.full((len(q), hq, d), 47.0, dtype=dtype, device=device)
    plan.run(q.to(device), k.to(device), v.to(device), torch.tensor(qo, dtype=torch.int32, device=device),
             torch.tensor(ko, dtype=torch.int32, device=device), out=out)
    torch.cuda.synchronize()
    return out.cpu()


def offsets(counts):
    return [0, *torch.tensor(counts).cumsum(0).tolist()]


def check(backend, device, queries, past, hq, hk, d, dtype, seed=0, scale=None, spread=1.0):
    print(f"case packed attention queries={queries} past={past} heads={hq}/{hk} d={d} {dtype} scale={scale}", flush=True)
    gen = torch.Generator().manual_seed(seed)
    qo, ko = offsets(queries), offsets([max(a + b, 0) for a, b in zip(queries, past)])
    q = (torch.randn(qo[-1], hq, d, generator=gen) * spread).to(dtype)
    k, v = (torch.randn(max(ko[-1], 1), hk, d, generator=gen).to(dtype) for _ in range(2))
    k[:, :, ::37] *= 3
    out = run(backend, device, q, k, v, qo, ko, hq, hk, d, dtype, scale)
    for b, t in enumerate(queries):
        part, mine = slice(qo[b], qo[b + 1]), slice(ko[b], ko[b + 1])
        n = ko[b + 1] - ko[b]
        seen = [n - (t - 1 - i) for i in range(t)]
        want, mean, size = attend(q[part], k[mine], v[mine], seen, scale)
        bound = attention_bound(want, mean, size, d, n, dtype, half_step(dtype))
        error = (out[part].double() - want).abs()
        assert (error <= bound).all(), (b, float((error / bound).max()))
        for i, count in enumerate(seen):
            if count <= 0:
                assert not out[qo[b] + i].any()


@pytest.mark.parametrize("dtype", [FP16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("hq,hk,d", [(48, 4, 128), (24, 2, 256), (32, 8, 128), (32, 4, 64), (16, 16, 128), (20, 4, 96), (7, 1, 32),
                                     (3, 3, 8), (6, 2, 72), (10, 2, 160), (4, 2, 224), (34, 2, 192)])
def test_heads(backend, device, dtype, hq, hk, d):
    check(backend, device, [77, 1, 130], [0, 40, 5], hq, hk, d, dtype, seed=hq + d)


@pytest.mark.parametrize("queries,past", [([1], [0]), ([2], [0]), ([5], [1500]), ([1, 1, 1], [0, 700, 64]), ([300], [0]),
                                          ([63, 64, 65], [0, 0, 0]), ([127, 128, 129], [1, 63, 64]), ([31, 0, 33], [0, 9, 0]),
                                          ([0, 0, 4], [3, 0, 0]), ([20, 7], [-13, -7]), ([513], [258]), ([1] * 70, [3] * 70)])
@pytest.mark.parametrize("hq,hk,d", [(12, 1, 128), (4, 4, 64), (24, 2, 256)])
def test_lengths(backend, device, queries, past, hq, hk, d):
    """Lengths around the tiles, sequences without queries or keys, and queries before the first key (past < 0)."""
    check(backend, device, queries, past, hq, hk, d, FP16, seed=len(queries))


@pytest.mark.parametrize("dtype", [FP16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("hk,d", [(1, 32), (1, 64), (1, 96), (1, 128), (1, 160), (1, 192), (1, 224), (1, 256), (2, 72)])
def test_few_rows_over_many_keys(backend, device, dtype, hk, d):
    """The keys of a block shared by several workgroups, some of which see none of a row's; sequences of other lengths."""
    check(backend, device, [5], [1500], hk, hk, d, dtype, seed=d)
    check(backend, device, [3, 1, 40], [1300, 0, 700], 3 * hk, hk, d, dtype, seed=d + 1)


@pytest.mark.parametrize("scale", [2.0**127, -(2.0**127)])
def test_largest_scales(backend, device, scale):
    check(backend, device, [33, 2], [0, 300], 4, 2, 64, BF16, seed=5, scale=scale, spread=2.0**-130)


def test_many_sequences(backend, device):
    queries = [(5 * i * i + i) % 23 for i in range(301)]
    check(backend, device, queries, [i % 4 for i in range(301)], 4, 2, 64, BF16, seed=4)


@pytest.mark.parametrize("dtype", [FP16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("spread,scale", [(30.0, None), (1.0, 0.0), (1.0, 0.7), (1.0, -0.2), (1e-3, None)])
def test_scale_and_peaked_weights(backend, device, dtype, spread, scale):
    check(backend, device, [150], [30], 8, 2, 64, dtype, seed=5, scale=scale, spread=spread)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_later_keys_that_hold_no_number_are_not_seen(backend, device, d):
    gen = torch.Generator().manual_seed(6)
    t, hq, hk, edge = 200, 4, 2, 101
    q, k, v = (torch.randn(t, h, d, generator=gen).half() for h in (hq, hk, hk))
    clean = run(backend, device, q, k, v, [0, t], [0, t], hq, hk, d, FP16)
    k[edge:], v[edge:] = float("nan"), float("inf")
    out = run(backend, device, q, k, v, [0, t], [0, t], hq, hk, d, FP16)
    assert torch.equal(out[:edge], clean[:edge])
    assert out[edge:].isnan().any(-1).all()
    # The next sequence's keys lie in the same tile.
    out = run(backend, device, q, k, v, [0, edge, t], [0, edge, t], hq, hk, d, FP16)
    assert torch.equal(out[:edge], clean[:edge])


def test_keys_of_minus_infinite_score(backend, device):
    """Scores of -inf weigh nothing; a row of nothing else is zero."""
    d = 64
    q = torch.ones(3, 1, d).half()
    k, v = torch.zeros(3, 1, d).half(), torch.ones(3, 1, d).half()
    k[:2, 0, 0] = -float("inf")
    out = run(backend, device, q, k, v, [0, 3], [0, 3], 1, 1, d, FP16)
    assert not out[:2].any() and torch.equal(out[2], v[2])


def test_offsets_that_do_not_cover_or_leave_the_rows(backend, device):
    gen = torch.Generator().manual_seed(7)
    q, k, v = (torch.randn(50, 2, 64, generator=gen).half() for _ in range(3))
    out = run(backend, device, q, k, v, [0, 20, 30], [0, 20, 30], 2, 2, 64, FP16)
    assert out[:30].any(-1).all() and not out[30:].any()
    # Past the tensors' ends: clamped, nothing outside is read.
    out = run(backend, device, q, k, v, [0, 20, 90], [0, 20, 10**6], 2, 2, 64, FP16)
    assert out.isfinite().all()
    out = run(backend, device, q, k, v, [0, 30, 20], [-5, 2**31 - 1, -2**31], 2, 2, 64, FP16)
    assert out.isfinite().all()


def test_same_bits_every_run_and_in_graphs(backend, device):
    gen = torch.Generator().manual_seed(8)
    q, k, v = (torch.randn(n, h, 128, generator=gen).to(device).bfloat16() for n, h in ((7, 12), (900, 2), (900, 2)))
    plan = backend.prepare_attention(tokens=7, keys=900, sequences=2, q_heads=12, kv_heads=2, head_dim=128, dtype=BF16,
                                     device=device)
    qo, ko = (torch.tensor(o, dtype=torch.int32, device=device) for o in ([0, 3, 7], [0, 800, 900]))
    out = torch.empty_like(q)
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        plan.run(q, k, v, qo, ko, out=out)
    torch.cuda.current_stream(device).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.run(q, k, v, qo, ko, out=out)
    for i in range(4):
        q.copy_(torch.randn(7, 12, 128, generator=gen))
        out.zero_()
        plan.run(q, k, v, qo, ko, out=out)
        want = out.clone()
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_cached_and_packed_attention_agree(backend, device):
    """One new token over the cache's read-back rows: the same within both bounds."""
    gen = torch.Generator().manual_seed(9)
    n, hq, hk, d = 333, 8, 2, 128
    cache = backend.create_kv_cache(pages=6, page_tokens=64, kv_heads=hk, head_dim=d, dtype=BF16, device=device)
    slots = torch.arange(n, device=device)
    x = torch.randn(n, 2 * hk * d, generator=gen).bfloat16().to(device)
    cache.prepare_write(tokens=n, q_heads=0, rotary=None).run(x, None, slots)
    k, v = (torch.empty(n, hk, d, dtype=BF16, device=device) for _ in range(2))
    cache.prepare_read(tokens=n).run(slots, keys=k, values=v)
    q = torch.randn(1, hq, d, generator=gen).bfloat16()
    packed = run(backend, device, q, k.cpu(), v.cpu(), [0, 1], [0, n], hq, hk, d, BF16)
    plan = cache.prepare_attention(sequences=1, q_heads=hq, query_tokens=1, max_pages=6)
    out = torch.empty(1, hq, d, dtype=BF16, device=device)
    plan.run(q.to(device), torch.arange(6, dtype=torch.int32, device=device)[None], torch.tensor([n], dtype=torch.int32, device=device),
             out=out, workspace=torch.empty(plan.workspace_bytes, dtype=torch.uint8, device=device))
    want, mean, size = attend(q, k.cpu(), v.cpu(), [n])
    step = half_step(BF16)
    bound = 2 * attention_bound(want, mean, size, d, n, BF16, step, step) + mean * 2 * step * size[..., None]
    assert ((packed.double() - out.cpu().double()).abs() <= bound).all()
