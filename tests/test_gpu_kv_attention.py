"""Attention over the paged Q8 cache against the formula in 64 bits on the cached values.

The kernel rounds weights and values to fp16 (half a step, 2^-11, each) whatever the model's type; the bound is
attention_oracle.attention_bound."""

import pytest
import torch

from attention_oracle import attend, attention_bound, q8_values

pytestmark = pytest.mark.gpu

FP16, BF16 = torch.float16, torch.bfloat16


def make(backend, device, lengths, hq, hk, d, dtype, page, t, seed, max_pages=None, spread=1.0, width=1.0):
    """A cache with shuffled pages; slots that no sequence owns hold NaN."""
    gen = torch.Generator().manual_seed(seed)
    need = [(n + page - 1) // page for n in lengths]
    pages = sum(need) + 2
    cache = backend.create_kv_cache(pages=pages, page_tokens=page, kv_heads=hk, head_dim=d, dtype=dtype, device=device)
    order = torch.randperm(pages, generator=gen).tolist()
    table = torch.full((len(lengths), max_pages or max(max(need), 1)), 2**30, dtype=torch.int32)
    x = (torch.randn(pages * page, 2 * hk, d, generator=gen) * width).to(dtype)
    x[:, :hk, ::37] *= 3
    owned = torch.zeros(pages * page, dtype=torch.bool)
    sequences = []
    for b, n in enumerate(lengths):
        mine, order = order[: need[b]], order[need[b]:]
        table[b, : need[b]] = torch.tensor(mine, dtype=torch.int32)
        at = torch.arange(n)
        slots = torch.tensor(mine, dtype=torch.int64)[at // page] * page + at % page if n else at
        owned[slots] = True
        sequences.append(slots)
    x[~owned] = float("nan")
    slots = torch.arange(pages * page, device=device)
    cache.prepare_write(tokens=pages * page, q_heads=0, rotary=None).run(x.reshape(pages * page, -1).to(device), None, slots)
    q = (torch.randn(len(lengths) * t, hq, d, generator=gen) * spread).to(dtype)
    return cache, q, table, sequences


def cached(cache, slots):
    page, at = slots // cache.page_tokens, slots % cache.page_tokens
    return [q8_values((c.cpu().permute(0, 2, 1, 3)[page, at].to(torch.int16) - 128)[..., : cache.head_dim],
                      s.cpu().permute(0, 3, 1, 2)[page, at])
            for c, s in ((cache.key_codes, cache.key_scales), (cache.value_codes, cache.value_scales))]


def run(cache, q, table, lengths, t, hq, device, scale=None, workspace_fill=255):
    plan = cache.prepare_attention(sequences=len(lengths), q_heads=hq, query_tokens=t, max_pages=table.shape[1], scale=scale)
    workspace = torch.full((plan.workspace_bytes,), workspace_fill, dtype=torch.uint8, device=device)
    out = torch.full_like(q, 47.0, device=device)
    plan.run(q.to(device), table.to(device), torch.tensor(lengths, dtype=torch.int32, device=device), out=out, workspace=workspace)
    torch.cuda.synchronize()
    return out.cpu()


def check(backend, device, lengths, hq, hk, d, dtype, page, t, seed=0, **more):
    print(f"case kv attention lengths={lengths} heads={hq}/{hk} d={d} {dtype} page={page} t={t} {more}", flush=True)
    scale = more.pop("scale", None)
    cache, q, table, sequences = make(backend, device, lengths, hq, hk, d, dtype, page, t, seed, **more)
    out = run(cache, q, table, lengths, t, hq, device, scale)
    for b, slots in enumerate(sequences):
        k, v = cached(cache, slots)
        seen = [len(slots) - (t - 1 - i) for i in range(t)]
        part = slice(b * t, (b + 1) * t)
        want, mean, size = attend(q[part], k, v, seen, scale)
        bound = attention_bound(want, mean, size, d, len(slots), dtype, 2.0**-11, 2.0**-11)
        error = (out[part].double() - want).abs()
        assert (error <= bound).all(), (b, float((error / bound).max()))
        for i, n in enumerate(seen):
            if n <= 0:
                assert not out[b * t + i].any()


@pytest.mark.parametrize("dtype", [FP16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("hq,hk,d", [(48, 4, 128), (24, 2, 256), (32, 8, 128), (32, 4, 64), (16, 16, 128), (20, 4, 96), (7, 1, 32),
                                     (3, 3, 8), (6, 2, 72), (10, 2, 160), (4, 2, 224), (34, 2, 192), (80, 2, 40)])
@pytest.mark.parametrize("t", [1, 5])
def test_heads_and_lengths(backend, device, dtype, hq, hk, d, t):
    check(backend, device, [1, 0, 64, 17, 257, 3], hq, hk, d, dtype, 32, t, seed=hq + d)


@pytest.mark.parametrize("dtype", [FP16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("hk,d", [(1, 32), (2, 64), (4, 96), (4, 128), (2, 160), (2, 192), (2, 224), (2, 256)])
@pytest.mark.parametrize("t", [12, 33])
def test_rows_of_two_and_four_tiles(backend, device, dtype, hk, d, t):
    check(backend, device, [300, 20, 41], 2 * hk, hk, d, dtype, 32, t, seed=d + t)


@pytest.mark.parametrize("hq,d", [(1, 64), (3, 128), (12, 256), (5, 96)])
def test_numbers_that_are_none_in_the_new_tokens(backend, device, hq, d):
    """The last new tokens' values and keys hold no number: the earlier ones do not see them. (Their bits may differ: the
    rows of a wave move their references together.)"""
    t, n = 4, 70
    cache, q, table, sequences = make(backend, device, [n], hq, 1, d, FP16, 16, t, seed=14)
    k, v = cached(cache, sequences[0])
    want, mean, size = attend(q, k, v, [n - 3, n - 2, n - 1, n])
    bound = attention_bound(want, mean, size, d, n, FP16, 2.0**-11, 2.0**-11)
    value, key = (int(sequences[0][n - i]) for i in (2, 1))
    cache.value_scales[value // 16, 0, 0, value % 16] = float("nan")
    cache.key_scales[key // 16, 0, 0, key % 16] = float("inf")
    out = run(cache, q, table, [n], t, hq, device)
    assert ((out[:2].double() - want[:2]).abs() <= bound[:2]).all()
    assert out[2, :, :32].isnan().all() and ((out[2, :, 32:].double() - want[2, :, 32:]).abs() <= bound[2, :, 32:]).all()
    assert out[3].isnan().any(-1).all()


@pytest.mark.parametrize("page", [16, 32, 48, 128, 1040])
@pytest.mark.parametrize("t", [1, 2, 9])
def test_pages(backend, device, page, t):
    check(backend, device, [page - 1, page, page + 1, 2 * page + 15, 5], 12, 2, 128, FP16, page, t, seed=page)


@pytest.mark.parametrize("lengths", [[2047], [2048], [2049], [5000, 1], [4095, 700, 1, 0, 33], [9001]])
def test_split_lengths(backend, device, lengths):
    check(backend, device, lengths, 8, 2, 64, FP16, 64, 1, seed=len(lengths))


def test_table_far_wider_than_the_sequences(backend, device):
    check(backend, device, [300, 5], 8, 2, 128, BF16, 32, 1, seed=3, max_pages=5000)


def test_many_sequences(backend, device):
    lengths = [(7 * i * i + 3 * i) % 190 for i in range(333)]
    check(backend, device, lengths, 4, 1, 64, FP16, 16, 1, seed=4)


def test_many_query_tokens(backend, device):
    check(backend, device, [70, 200], 6, 2, 64, FP16, 16, 67, seed=6)


@pytest.mark.parametrize("dtype,spread,width", [(FP16, 30.0, 1.0), (FP16, 1.0, 1e-4), (FP16, 1.0, 5000.0), (BF16, 1e-3, 1e4),
                                                (BF16, 1e-6, 3e5), (BF16, 1e30, 1e-3)])
def test_large_and_small_values(backend, device, dtype, spread, width):
    """Peaked and flat weights, values near both ends of the scales' range, queries outside fp16's."""
    check(backend, device, [500, 40], 8, 2, 128, dtype, 32, 1, seed=8, spread=spread, width=width,
          **({"scale": 1e-31} if spread == 1e30 else {}))


@pytest.mark.parametrize("scale", [0.0, 0.31, -0.2])
def test_scale(backend, device, scale):
    check(backend, device, [90], 4, 4, 64, FP16, 16, 2, seed=9, scale=scale)


@pytest.mark.parametrize("scale", [2.0**127, -(2.0**127)])
@pytest.mark.parametrize("d", [64, 256])
def test_largest_scales(backend, device, scale, d):
    check(backend, device, [90], 4, 4, d, BF16, 16, 2, seed=9, scale=scale, spread=2.0**-130)


def test_bad_pages_and_lengths_mark_their_sequence(backend, device):
    lengths = [40, 40, 40, 40, 40]
    cache, q, table, _ = make(backend, device, lengths, 4, 2, 64, FP16, 16, 2, seed=10)
    good = run(cache, q, table, lengths, 2, 4, device)
    table[1, 2], table[3, 0] = cache.pages, -1
    bad = run(cache, q, table, [40, 40, -1, 40, 49], 2, 4, device)
    assert bad[2:10].isnan().all()
    assert torch.equal(bad[:2], good[:2])
    table[4, 2] = 2**30  # past 32 keys: not reached
    fewer = run(cache, q, table, [40, 32, 0, 0, 32], 2, 4, device)
    assert fewer[:4].isfinite().all() and not fewer[4:8].any() and fewer[8:].isfinite().all()


def test_cached_numbers_that_are_none(backend, device):
    """A NaN in a seen value or key is the output's; in an unseen one it is not (make() puts them there)."""
    cache, q, table, sequences = make(backend, device, [30, 30], 2, 1, 64, FP16, 16, 1, seed=11)
    slot = int(sequences[0][12])
    cache.value_scales[slot // 16, 0, 1, slot % 16] = float("nan")
    out = run(cache, q, table, [30, 30], 1, 2, device)
    assert out[0, :, 32:].isnan().all() and out[0, :, :32].isfinite().all() and out[1].isfinite().all()


def test_cache_past_32_bit_offsets(backend, device):
    """4.3 G codes a side: the last pages' offsets do not fit 32 bits."""
    page, d = 256, 256
    pages = 2**32 // (page * d) + 3
    cache = backend.create_kv_cache(pages=pages, page_tokens=page, kv_heads=1, head_dim=d, dtype=FP16, device=device)
    gen = torch.Generator().manual_seed(12)
    n = 2 * page - 9
    mine = torch.tensor([pages - 1, pages - 3])
    at = torch.arange(n)
    slots = mine[at // page] * page + at % page
    x = torch.randn(n, 2, d, generator=gen).half()
    cache.prepare_write(tokens=n, q_heads=0, rotary=None).run(x.reshape(n, -1).to(device), None, slots.to(device))
    q = torch.randn(1, 4, d, generator=gen).half()
    out = run(cache, q, mine[None].int(), [n], 1, 4, device)
    keys, values = (torch.empty(n, 1, d, dtype=FP16, device=device) for _ in range(2))
    cache.prepare_read(tokens=n).run(slots.to(device), keys=keys, values=values)
    assert ((keys.cpu().double() - x[:, :1].double()).abs().amax() < 0.05)  # a step is max|x| / 127
    want, mean, size = attend(q, keys.cpu(), values.cpu(), [n])
    # The read-back rounds keys and values to fp16: half a step of each product of a score, and of a value.
    bound = attention_bound(want, mean, size, d, n, FP16, 2.0**-11, 2.0**-10) + mean * 2 * 2.0**-11 * size[..., None]
    assert ((out.double() - want).abs() <= bound).all()


def test_same_bits_every_run_and_in_graphs(backend, device):
    lengths = [3000, 1, 700, 64]
    cache, q, table, _ = make(backend, device, lengths, 12, 2, 128, BF16, 64, 2, seed=13)
    plan = cache.prepare_attention(sequences=4, q_heads=12, query_tokens=2, max_pages=table.shape[1])
    workspace = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device=device)
    qd, td, ld = q.to(device), table.to(device), torch.tensor(lengths, dtype=torch.int32, device=device)
    out = torch.empty_like(qd)
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        plan.run(qd, td, ld, out=out, workspace=workspace)
    torch.cuda.current_stream(device).wait_stream(side)
    first = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.run(qd, td, ld, out=out, workspace=workspace)
    for i in range(4):
        out.zero_()
        workspace.fill_(i)
        ld.copy_(torch.tensor([3000, 1, 700, 64] if i % 2 == 0 else [100, 2, 0, 5], dtype=torch.int32))
        plan.run(qd, td, ld, out=out, workspace=workspace)
        want = out.clone()
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        out, want = out.view(torch.int16), want.view(torch.int16)  # bits: the shorter lengths reach a slot that holds NaN
        assert torch.equal(out, want)
        assert torch.equal(want, first.view(torch.int16)) == (i % 2 == 0)
        out = out.view(BF16)


def rewrite(cache, slots, k, v, device):
    """Other rows [n, heads, d] in the cache's slots."""
    rows = torch.cat([k.flatten(1), v.flatten(1)], 1).to(cache.dtype).to(device)
    cache.prepare_write(tokens=len(slots), q_heads=0, rotary=None).run(rows, None, slots.to(device))
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [FP16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("hq,hk,d,t", [(1, 1, 32, 1), (2, 2, 64, 1), (6, 2, 96, 2), (8, 2, 128, 1), (8, 1, 128, 3), (5, 1, 160, 5),
                                       (7, 1, 224, 5), (12, 1, 256, 5), (2, 1, 256, 1)])
@pytest.mark.parametrize("bits", [14, 18, 20, 24, 31, 38])
def test_values_of_very_different_sizes(backend, device, dtype, hq, hk, d, t, bits):
    """Columns 2^bits smaller than others of their head, and keys 2^bits larger than others whose weights are nothing: every
    column's error goes by its own values. (A scale of 2^-24 has one bit; the cached values are what is compared with.)"""
    n = 205
    print(f"case kv values heads={hq}/{hk} d={d} {dtype} t={t} bits={bits}", flush=True)
    gen = torch.Generator().manual_seed(bits + d)
    top = 2.0**14  # the largest values' size: scales of 2^9
    for keys in (False, True):
        cache, q, table, sequences = make(backend, device, [n], hq, hk, d, dtype, 16, t, seed=bits)
        k, v = torch.randn(n, hk, d, generator=gen), torch.randn(n, hk, d, generator=gen).clamp(-3.9, 3.9)  # within fp16
        q[:] = q.abs() + 1
        if keys:  # large values at the first, middle and last common keys, whose scores lie below -200
            large = [0, 100, n - t]
            v *= top * 2.0**-bits
            v[large] *= 2.0**bits
            k[large] = -300.0
        else:  # columns by 16 and by 32: half a group of 32 is as small as the other half makes it
            v *= top
            for part in range(0, d, 32):
                v[:, :, part: part + 32] *= 2.0 ** -(bits if part // 32 % 2 == 0 else bits // 2)
            v[:, :, d - 16:] = torch.randn(n, hk, 16, generator=gen).clamp(-3.9, 3.9) * top
            v[3::7] = 0  # scales of 0 beside them
        rewrite(cache, sequences[0], k, v, device)
        out = run(cache, q, table, [n], t, hq, device)
        kc, vc = cached(cache, sequences[0])
        want, mean, size = attend(q, kc, vc, [n - (t - 1 - i) for i in range(t)])
        bound = attention_bound(want, mean, size, d, n, dtype, 2.0**-11, 2.0**-11)
        error = (out.double() - want).abs()
        assert (error <= bound).all(), (keys, float((error / bound).max()))


@pytest.mark.parametrize("d", [64, 128, 160, 256])
@pytest.mark.parametrize("dtype,spread,scale", [(BF16, 2.0**100, None), (BF16, 2.0**118, None), (BF16, 2.0**124, None), (BF16, 2.0**100, -1.0),
                                                (BF16, 2.0**124, 2.0**30), (FP16, 100.0, 2.0**110), (FP16, 1.0, -2.0**127)])
def test_scores_near_the_end_of_32_bits(backend, device, dtype, spread, scale, d):
    """Queries, or scales, so large that the largest score takes all of a row's weight: its value is the row's output."""
    n, t, hq = 70, 2, 3
    print(f"case kv scores d={d} {dtype} spread={spread} scale={scale}", flush=True)
    cache, q, table, sequences = make(backend, device, [n], hq, 1, d, dtype, 16, t, seed=d)
    q = (q.float().clamp(-4, 4) * spread).to(dtype)  # below 2^127
    q[1, 0] = 0  # equal weights
    out = run(cache, q, table, [n], t, hq, device, scale)
    kc, vc = cached(cache, sequences[0])
    factor = d ** -0.5 if scale is None else scale
    for i in range(t):
        seen = n - (t - 1 - i)
        for h in range(hq):
            products = kc[:seen, 0] * q[i, h].double()
            scores = products.sum(1) * factor
            if (i, h) == (1, 0):
                want, mean = vc[:seen, 0].mean(0), vc[:seen, 0].abs().mean(0)
            else:
                best, gap = int(scores.argmax()), scores.sort(descending=True)[0]
                # What 32-bit sums may be off, and what leaves the second weight nothing.
                assert gap[0] - gap[1] > 2 * (d + 6) * 2.0**-24 * float(products.abs().sum(1).max()) * abs(factor) + 100
                want, mean = vc[best, 0], vc[best, 0].abs()
            bound = attention_bound(want, mean, torch.zeros(()), d, n, dtype, 2.0**-11, 2.0**-11)
            error = (out[i, h].double() - want).abs()
            assert (error <= bound).all(), (i, h, float((error / bound).max()))


@pytest.mark.parametrize("side", ["key", "value"])
@pytest.mark.parametrize("d", [32, 64, 128, 192, 256])
@pytest.mark.parametrize("t", [1, 3])
def test_groups_whose_scale_overflows(backend, device, d, t, side):
    """Such a group reads back as NaN: so it is for the rows that see it, whatever the signs of their queries, and for no other."""
    n, hq = 75, 12
    print(f"case kv overflow d={d} t={t} {side}", flush=True)
    cache, q, table, sequences = make(backend, device, [n], hq, 1, d, BF16, 16, t, seed=d + t)
    gen = torch.Generator().manual_seed(d)
    k, v = torch.randn(n, 1, d, generator=gen), torch.randn(n, 1, d, generator=gen)
    q *= 2.0 ** -torch.randint(0, 20, q.shape, generator=gen)  # their sums are not exact in 32 bits
    last = n - 2 if t > 1 else 40  # not seen by the first of three new tokens
    (k if side == "key" else v)[last, 0, d - 1] = -1e38
    rewrite(cache, sequences[0], k, v, device)
    out = run(cache, q, table, [n], t, hq, device)
    for i in range(t):
        sees = last < n - (t - 1 - i)
        hit = out[i] if side == "key" else out[i, :, d - 32:]
        assert hit.isnan().all() if sees else hit.isfinite().all()
        if side == "value":
            assert out[i, :, : d - 32].isfinite().all()
