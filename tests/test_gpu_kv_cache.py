"""Rotary positions with the Q8 cache write, and the read-back, against the formulas in 64 bits.

Rotated rows: the angle's part of a turn is rounded to fp32 (2^-25 of a turn), sine and cosine to two units, products and
sum once each, so a row errs by less than 2^-20 of |x0| + |x1| before its own rounding. Cached bytes have to be the
rule's applied to the kernel's own K (and to V), read-back rows the rounded product of code and scale."""

import math

import pytest
import torch

from attention_oracle import half_step, q8_rule, q8_values, rotate
from venturi_amd import RotaryEmbedding

pytestmark = pytest.mark.gpu

SCALINGS = {
    "none": None,
    "linear": {"type": "linear", "factor": 4.0},
    "banded": {"type": "banded", "factor": 8.0, "low": 1.0, "high": 4.0, "original_context": 8192},
    "yarn": {"type": "yarn", "factor": 4.0, "original_context": 4096, "beta_fast": 32.0, "beta_slow": 1.0},
}


def rows(tokens, heads, d, dtype, seed):
    x = torch.randn(tokens, heads, d, generator=torch.Generator().manual_seed(seed))
    x[:, :, ::37] *= 3
    return x.to(dtype)


def planes(cache, slots):
    """Codes int8 and scales of the slots' K and V, on the CPU: [(codes [n, heads, d], scales [n, heads, groups])] * 2."""
    page, at = slots // cache.page_tokens, slots % cache.page_tokens
    got = []
    for codes, scales in ((cache.key_codes, cache.key_scales), (cache.value_codes, cache.value_scales)):
        c = codes.cpu().permute(0, 2, 1, 3)[page, at].to(torch.int16) - 128
        got.append((c.to(torch.int8), scales.cpu().permute(0, 3, 1, 2)[page, at]))
    return got


def check(backend, device, tokens, hq, hk, d, dtype, rotary, page_tokens, positions, seed=0, dense_k=True):
    print(f"case kv write tokens={tokens} heads={hq}/{hk} d={d} {dtype} rotary={rotary} page={page_tokens}", flush=True)
    gen = torch.Generator().manual_seed(seed)
    pages = (tokens + page_tokens - 1) // page_tokens + 2
    slots = torch.randperm(pages * page_tokens, generator=gen)[:tokens]
    x = rows(tokens, hq + 2 * hk, d, dtype, seed + 1)
    cache = backend.create_kv_cache(pages=pages, page_tokens=page_tokens, kv_heads=hk, head_dim=d, dtype=dtype, device=device)
    plan = cache.prepare_write(tokens=tokens, q_heads=hq, rotary=rotary)
    q = torch.empty(tokens, hq, d, dtype=dtype, device=device) if hq else None
    k = torch.empty(tokens, hk, d, dtype=dtype, device=device) if dense_k else None
    on = slots.to(device)
    plan.run(x.reshape(tokens, -1).to(device), positions.to(device), on, q=q, k=k)
    keys, values = (torch.empty(tokens, hk, d, dtype=dtype, device=device) for _ in range(2))
    cache.prepare_read(tokens=tokens).run(on, keys=keys, values=values)
    torch.cuda.synchronize()
    if rotary is None:
        want, size = x[:, : hq + hk].double(), torch.zeros(tokens, hq + hk, d)
    else:
        want, size = rotate(x[:, : hq + hk], positions, rotary.frequencies, rotary.factor, rotary.layout)
    bound = size * 2.0**-20 + want.abs() * half_step(dtype) * 1.001 + 2.0**-25
    if hq:
        assert ((q.cpu().double() - want[:, :hq]).abs() <= bound[:, :hq]).all()
    (kc, ks), (vc, vs) = planes(cache, slots)
    if dense_k:
        assert ((k.cpu().double() - want[:, hq:]).abs() <= bound[:, hq:]).all()
        codes, scales = q8_rule(k.cpu())
        assert torch.equal(ks, scales) and torch.equal(kc[..., :d], codes)
    codes, scales = q8_rule(x[:, hq + hk:])
    assert torch.equal(vs, scales) and torch.equal(vc[..., :d], codes)
    assert not kc[..., d:].any() and not vc[..., d:].any()
    for got, (c, s) in ((keys, (kc, ks)), (values, (vc, vs))):
        assert torch.equal(got.cpu(), q8_values(c[..., :d], s).to(dtype))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,hq,hk,d,r,page", [(1, 48, 4, 128, 128, 64), (61, 24, 2, 256, 64, 32), (7, 32, 4, 64, 32, 16),
                                                   (300, 20, 4, 96, 96, 128), (5, 3, 3, 72, 20, 16), (2, 1, 1, 8, 2, 16),
                                                   (33, 7, 7, 200, 46, 48)])
def test_write_and_read(backend, device, dtype, layout, tokens, hq, hk, d, r, page):
    positions = torch.arange(tokens) + 1000
    check(backend, device, tokens, hq, hk, d, dtype, RotaryEmbedding(d, rotary_dim=r, layout=layout, base=1e6), page, positions,
          seed=tokens)


@pytest.mark.parametrize("scaling", list(SCALINGS))
def test_scaled_rotation_at_far_positions(backend, device, scaling):
    positions = torch.tensor([0, 1, 4095, 4096, 131071, 10**6 + 3, 2**31 + 7, 2**40 + 11, -5])
    rotary = RotaryEmbedding(128, base=1e6, scaling=SCALINGS[scaling])
    check(backend, device, len(positions), 4, 2, 128, torch.float16, rotary, 16, positions, seed=9)


@pytest.mark.parametrize("hq,dense_k", [(0, False), (0, True), (5, False)])
def test_write_without_rotation_or_dense_keys(backend, device, hq, dense_k):
    check(backend, device, 19, hq, 5, 64, torch.bfloat16, None, 16, torch.zeros(19, dtype=torch.int64), seed=3, dense_k=dense_k)


def test_write_of_many_tokens(backend, device):
    check(backend, device, 1111, 6, 2, 128, torch.float16, RotaryEmbedding(128), 64, torch.arange(1111), seed=4)


def test_slots_outside_the_cache(backend, device):
    d, hk, page = 64, 2, 16
    cache = backend.create_kv_cache(pages=2, page_tokens=page, kv_heads=hk, head_dim=d, dtype=torch.float16, device=device)
    before = [t.clone() for t in cache.storage_tensors]
    slots = torch.tensor([-1, 32, 2**40, -2**40, 31], device=device)
    x = rows(5, 4 + 2 * hk, d, torch.float16, 5).reshape(5, -1).to(device)
    q = torch.full((5, 4, d), 7.0, dtype=torch.float16, device=device)
    cache.prepare_write(tokens=5, q_heads=4, rotary=None).run(x, None, slots, q=q)
    keys, values = (torch.empty(5, hk, d, dtype=torch.float16, device=device) for _ in range(2))
    cache.prepare_read(tokens=5).run(slots, keys=keys, values=values)
    torch.cuda.synchronize()
    assert torch.equal(q.flatten(1), x[:, : 4 * d])
    assert keys[:4].isnan().all() and values[:4].isnan().all() and not keys[4].isnan().any()
    for old, new in zip(before, cache.storage_tensors):  # nothing but token 15 of page 1 changed
        old, new = (t if t.dtype == torch.uint8 else t.transpose(2, 3) for t in (old, new))
        changed = (old != new).flatten(3).any(3).any(1).cpu()
        assert changed.nonzero().tolist() == [[1, 15]]


def test_rows_that_share_a_slot(backend, device):
    """Codes and scales of any of the rows stay there, and nothing else is touched."""
    d, hk, hq, tokens = 96, 2, 3, 300
    x = rows(tokens, hq + 2 * hk, d, torch.float16, 30)
    on = x.reshape(tokens, -1).to(device)
    cache = backend.create_kv_cache(pages=2, page_tokens=16, kv_heads=hk, head_dim=d, dtype=torch.float16, device=device)
    before = [t.clone() for t in cache.storage_tensors]
    q, k = torch.empty(tokens, hq, d, dtype=torch.float16, device=device), torch.empty(tokens, hk, d, dtype=torch.float16, device=device)
    slots = torch.full((tokens,), 21)
    cache.prepare_write(tokens=tokens, q_heads=hq, rotary=None).run(on, None, slots.to(device), q=q, k=k)
    torch.cuda.synchronize()
    assert torch.equal(q.cpu(), x[:, :hq]) and torch.equal(k.cpu(), x[:, hq: hq + hk])
    for (codes, scales), part in zip(planes(cache, slots[:1]), (x[:, hq: hq + hk], x[:, hq + hk:])):
        want, steps = q8_rule(part)
        assert (want.unflatten(2, (-1, 8)) == codes.unflatten(2, (-1, 8))).all(3).any(0).all()
        assert (steps == scales).any(0).all()
    for old, new in zip(before, cache.storage_tensors):
        old, new = (t if t.dtype == torch.uint8 else t.transpose(2, 3) for t in (old, new))
        assert (old != new).flatten(3).any(3).any(1).cpu().nonzero().tolist() == [[1, 5]]


@pytest.mark.parametrize("dtype,large", [(torch.float16, 65504.0), (torch.bfloat16, 1e38)], ids=["fp16", "bf16"])
def test_groups_that_hold_no_number(backend, device, dtype, large):
    d = 128
    x = rows(4, 2, d, dtype, 6)
    x[0, 0, 5], x[1, 1, 40], x[2, 0, 127], x[3, 1, 64] = math.inf, math.nan, -math.inf, large
    x[3, 0] = 0
    cache = backend.create_kv_cache(pages=1, page_tokens=16, kv_heads=1, head_dim=d, dtype=dtype, device=device)
    slots = torch.arange(4, device=device)
    cache.prepare_write(tokens=4, q_heads=0, rotary=None).run(x.reshape(4, -1).to(device), None, slots)
    keys, values = (torch.empty(4, 1, d, dtype=dtype, device=device) for _ in range(2))
    cache.prepare_read(tokens=4).run(slots, keys=keys, values=values)
    keys, values = keys.cpu()[:, 0], values.cpu()[:, 0]
    broken = torch.zeros(2, 4, 4, dtype=torch.bool)
    broken[0, 0, 0] = broken[1, 1, 1] = broken[0, 2, 3] = True
    broken[1, 3, 2] = dtype == torch.bfloat16  # the scale overflows fp16
    for got, mark in ((keys, broken[0]), (values, broken[1])):
        assert torch.equal(got.unflatten(1, (4, 32)).isnan().all(2), mark)
        assert torch.equal(got.unflatten(1, (4, 32)).isnan().any(2), mark)
    assert not keys[3].any()
    if dtype == torch.float16:
        assert values[3, 64] >= 65472  # 127 times the scale, at most half a step of the scale away


def test_read_of_one_side(backend, device):
    cache = backend.create_kv_cache(pages=1, page_tokens=16, kv_heads=2, head_dim=64, dtype=torch.float16, device=device)
    slots = torch.arange(16, device=device)
    x = rows(16, 4, 64, torch.float16, 8).reshape(16, -1).to(device)
    cache.prepare_write(tokens=16, q_heads=0, rotary=None).run(x, None, slots)
    both = [torch.empty(16, 2, 64, dtype=torch.float16, device=device) for _ in range(4)]
    plan = cache.prepare_read(tokens=16)
    plan.run(slots, keys=both[0], values=both[1])
    plan.run(slots, keys=both[2])
    plan.run(slots, values=both[3])
    assert torch.equal(both[0], both[2]) and torch.equal(both[1], both[3])


def test_graph_and_side_stream(backend, device):
    d, hk, hq, tokens = 128, 2, 4, 9
    cache = backend.create_kv_cache(pages=2, page_tokens=16, kv_heads=hk, head_dim=d, dtype=torch.float16, device=device)
    write = cache.prepare_write(tokens=tokens, q_heads=hq, rotary=RotaryEmbedding(d))
    read = cache.prepare_read(tokens=tokens)
    x = torch.empty(tokens, (hq + 2 * hk) * d, dtype=torch.float16, device=device)
    positions, slots = torch.zeros(tokens, dtype=torch.int64, device=device), torch.arange(tokens, device=device)
    q, keys, values = (torch.empty(tokens, h, d, dtype=torch.float16, device=device) for h in (hq, hk, hk))

    def step():
        write.run(x, positions, slots, q=q)
        read.run(slots, keys=keys, values=values)

    x.zero_()
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(device).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(3):
        x.copy_(rows(tokens, hq + 2 * hk, d, torch.float16, 20 + i).reshape(tokens, -1))
        positions.fill_(100 * i)
        step()
        want = [t.clone() for t in (q, keys, values)]
        for t in (q, keys, values):
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, (q, keys, values)))
