"""Rotary frequencies, and what the plans of the cache, of attention and of sampling refuse (no GPU): the checks of
`prepare` and `run` on CPU tensors with a backend that records its launches, and the C entry points' own."""

import math
from types import SimpleNamespace

import pytest
import torch

from venturi_amd import RotaryEmbedding, native
from venturi_amd.attention import PackedAttentionPlan
from venturi_amd.blocks import HipBackend
from venturi_amd.kv_cache import Q8KVCache
from venturi_amd.sampling import SamplingPlan

CPU = torch.device("cpu")
FP16, BF16 = torch.float16, torch.bfloat16


# -- rotary ------------------------------------------------------------------
def test_frequencies_without_scaling():
    r = RotaryEmbedding(128, rotary_dim=64, base=1e6)
    assert r.factor == 1.0 and r.rates.shape == (2, 32) and r.rates.dtype == torch.float64
    for i, f in enumerate(r.frequencies):
        assert f == pytest.approx(1e6 ** (-2 * i / 64), rel=1e-14)
        assert float(r.rates[0, i]) == pytest.approx(f / (2 * math.pi), rel=1e-15)
        assert abs(float(r.rates[1, i])) <= float(r.rates[0, i]) * 2.0**-53


def test_frequencies_with_scaling():
    plain = RotaryEmbedding(128, base=1e6).frequencies
    linear = RotaryEmbedding(128, base=1e6, scaling={"type": "linear", "factor": 4.0})
    assert linear.frequencies == tuple(f / 4 for f in plain) and linear.factor == 1.0
    banded = RotaryEmbedding(128, base=1e6, scaling={"type": "banded", "factor": 8.0, "low": 1.0, "high": 4.0,
                                                      "original_context": 8192})
    for f, g in zip(plain, banded.frequencies):
        turns = 8192 * f / (2 * math.pi)
        keep = min(max((turns - 1) / 3, 0), 1)
        assert g == pytest.approx(keep * f + (1 - keep) * f / 8, rel=1e-14)
    assert banded.frequencies[0] == plain[0] and banded.frequencies[-1] == plain[-1] / 8
    yarn = RotaryEmbedding(128, base=1e6, scaling={"type": "yarn", "factor": 4.0, "original_context": 32768, "beta_fast": 32.0,
                                                    "beta_slow": 1.0})
    assert yarn.factor == pytest.approx(0.1 * math.log(4) + 1)
    ends = [64 * math.log(32768 / (b * 2 * math.pi)) / math.log(1e6) for b in (32.0, 1.0)]
    for i, (f, g) in enumerate(zip(plain, yarn.frequencies)):
        ramp = min(max((i - math.floor(ends[0])) / (math.ceil(ends[1]) - math.floor(ends[0])), 0), 1)
        assert g == pytest.approx((1 - ramp) * f + ramp * f / 4, rel=1e-14)


@pytest.mark.parametrize("arguments", [
    dict(head_dim=0), dict(head_dim=64, rotary_dim=0), dict(head_dim=64, rotary_dim=66), dict(head_dim=64, rotary_dim=31),
    dict(head_dim=64, layout="pairs"), dict(head_dim=64, base=1.0), dict(head_dim=64, base=math.inf), dict(head_dim=64.0),
    dict(head_dim=64, scaling={"type": "other", "factor": 2.0}), dict(head_dim=64, scaling={"type": "linear"}),
    dict(head_dim=64, scaling={"type": "linear", "factor": 0.0}), dict(head_dim=64, scaling={"type": "linear", "factor": 2.0, "low": 1.0}),
    dict(head_dim=64, scaling={"type": "banded", "factor": 2.0, "low": 4.0, "high": 4.0, "original_context": 100}),
    dict(head_dim=64, scaling={"type": "yarn", "factor": 2.0, "original_context": 100, "beta_fast": 1.0, "beta_slow": 2.0})])
def test_rotary_refusals(arguments):
    with pytest.raises(ValueError):
        RotaryEmbedding(**arguments)


# -- plans over a backend that records ----------------------------------------
class Recorder:
    def __init__(self):
        self._native = native.load()
        self.launches = []

    def _call(self, entry, device, arguments):
        assert len(arguments) + 1 == len(entry.argtypes)
        for value, kind in zip(arguments, entry.argtypes):
            kind(value)
        self.launches.append(entry.__name__)

    def resolve_device(self, device):
        return CPU

    def validate_device(self, dtype, device):
        return CPU


@pytest.fixture
def backend(monkeypatch):
    """The plans' own code on the CPU: entering a device and waiting for its stream do nothing."""
    from contextlib import nullcontext

    monkeypatch.setattr(torch.cuda, "device", lambda device: nullcontext())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: SimpleNamespace(synchronize=lambda: None))
    return Recorder()


def cache(backend, **more):
    return Q8KVCache.create(backend, **{**dict(pages=4, page_tokens=16, kv_heads=2, head_dim=64, dtype=FP16, device=CPU), **more})


@pytest.mark.parametrize("more", [dict(pages=0), dict(page_tokens=8), dict(page_tokens=24), dict(page_tokens=8192), dict(kv_heads=0),
                                  dict(head_dim=60), dict(head_dim=264), dict(dtype=torch.float32), dict(pages=True)])
def test_cache_refusals(backend, more):
    with pytest.raises(ValueError):
        cache(backend, **more)


def test_cache_storage(backend):
    c = cache(backend, head_dim=72)
    assert c.slots == 64 and c.key_codes.shape == (4, 2, 16, 96) and c.value_scales.shape == (4, 2, 3, 16)
    assert c.storage_nbytes == 2 * 4 * 2 * 16 * (96 + 2 * 3)


def test_write_plan_refusals(backend):
    c = cache(backend)
    for arguments in (dict(tokens=0, q_heads=4, rotary=None), dict(tokens=3, q_heads=-1, rotary=None), dict(tokens=3, q_heads=2.0, rotary=None),
                      dict(tokens=3, q_heads=4, rotary=RotaryEmbedding(128))):
        with pytest.raises(ValueError):
            c.prepare_write(**arguments)
    with pytest.raises(TypeError):
        c.prepare_write(tokens=3, q_heads=4, rotary=64)
    plan = c.prepare_write(tokens=3, q_heads=4, rotary=RotaryEmbedding(64))
    rows, at = torch.zeros(3, 512, dtype=FP16), torch.zeros(3, dtype=torch.int64)
    q, k = torch.zeros(3, 4, 64, dtype=FP16), torch.zeros(3, 2, 64, dtype=FP16)
    plan.run(rows, at, at.clone(), q=q, k=k)
    assert backend.launches == ["venturi_kv_write_run"]
    buffer = torch.zeros(3 * 512 + 1, dtype=FP16)
    bad = [dict(rows=rows[:2]), dict(rows=rows.bfloat16()), dict(rows=buffer[1:].view(3, 512)), dict(rows=torch.zeros(512, 3, dtype=FP16).T),
           dict(positions=None), dict(positions=at.int()), dict(slots=at[:2]), dict(q=None), dict(q=rows.view(-1)[:768].view(3, 4, 64)),
           dict(q=q.transpose(0, 1)), dict(k=q.view(-1)[:384].view(3, 2, 64)), dict(k=k[:, :1])]
    for change in bad:
        arguments = {**dict(rows=rows, positions=at, slots=at.clone(), q=q, k=k), **change}
        with pytest.raises((ValueError, TypeError)):
            plan.run(arguments["rows"], arguments["positions"], arguments["slots"], q=arguments["q"], k=arguments["k"])
    with pytest.raises(ValueError, match="q is the output"):
        c.prepare_write(tokens=3, q_heads=0, rotary=None).run(torch.zeros(3, 256, dtype=FP16), None, at, q=q)
    assert len(backend.launches) == 1


def test_write_plans_of_one_embedding_share_its_upload(backend, monkeypatch):
    """Preparing again, as a batch does whenever its token count changes, copies nothing and waits for nothing."""
    c, rotary, waited = cache(backend), RotaryEmbedding(64), []
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: SimpleNamespace(synchronize=lambda: waited.append(device)))
    plans = [c.prepare_write(tokens=n, q_heads=4, rotary=rotary) for n in (1, 3, 3)]
    assert waited == [CPU] and all(p.storage_tensors[-1] is plans[0].storage_tensors[-1] for p in plans)
    c.prepare_write(tokens=1, q_heads=4, rotary=None)
    other = c.prepare_write(tokens=1, q_heads=4, rotary=RotaryEmbedding(64, base=1e6))
    assert waited == [CPU, CPU] and not torch.equal(other.storage_tensors[-1], plans[0].storage_tensors[-1])


def test_read_plan_refusals(backend):
    c = cache(backend)
    plan = c.prepare_read(tokens=5)
    slots, rows = torch.zeros(5, dtype=torch.int64), torch.zeros(5, 2, 64, dtype=FP16)
    plan.run(slots, keys=rows, values=rows.clone())
    for arguments in (dict(), dict(keys=rows, values=rows), dict(keys=rows[:4]), dict(values=rows.float())):
        with pytest.raises(ValueError):
            plan.run(slots, **arguments)
    with pytest.raises(ValueError):
        plan.run(slots.int(), keys=rows)
    assert len(backend.launches) == 1


def test_cached_attention_refusals(backend):
    c = cache(backend)
    base = dict(sequences=2, q_heads=4, query_tokens=3, max_pages=4)
    for change in (dict(sequences=0), dict(q_heads=3), dict(q_heads=0), dict(query_tokens=0), dict(max_pages=0),
                   dict(scale=math.inf), dict(scale="1"), dict(max_pages=2**31 - 1)):
        with pytest.raises(ValueError):
            c.prepare_attention(**{**base, **change})
    plan = c.prepare_attention(**base)
    q, out = torch.zeros(6, 4, 64, dtype=FP16), torch.zeros(6, 4, 64, dtype=FP16)
    table, lengths = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    store = torch.zeros(plan.workspace_bytes + 512, dtype=torch.uint8)
    store = store[(-store.data_ptr()) % 256:]
    workspace = store[: plan.workspace_bytes]
    plan.run(q, table, lengths, out=out, workspace=workspace)
    bad = [dict(q=q[:5]), dict(q=q.bfloat16()), dict(table=table.long()), dict(table=table[:, :3]), dict(lengths=lengths.long()),
           dict(out=q), dict(out=out.transpose(0, 1))]
    if plan.workspace_bytes:
        bad += [dict(workspace=None), dict(workspace=workspace[:-1]), dict(workspace=store[1: plan.workspace_bytes + 1])]
    for change in bad:
        a = {**dict(q=q, table=table, lengths=lengths, out=out, workspace=workspace), **change}
        with pytest.raises((ValueError, TypeError)):
            plan.run(a["q"], a["table"], a["lengths"], out=a["out"], workspace=a["workspace"])
    assert len(backend.launches) == 1


def test_packed_attention_refusals(backend):
    base = dict(tokens=6, keys=9, sequences=2, q_heads=4, kv_heads=2, head_dim=64, dtype=BF16, device=CPU)
    for change in (dict(tokens=0), dict(keys=0), dict(sequences=0), dict(q_heads=5), dict(head_dim=4), dict(head_dim=512),
                   dict(dtype=torch.float32), dict(scale=math.nan)):
        with pytest.raises(ValueError):
            PackedAttentionPlan.create(backend, **{**base, **change})
    plan = PackedAttentionPlan.create(backend, **base)
    q, out = torch.zeros(6, 4, 64, dtype=BF16), torch.zeros(6, 4, 64, dtype=BF16)
    k, v, offsets = torch.zeros(9, 2, 64, dtype=BF16), torch.zeros(9, 2, 64, dtype=BF16), torch.zeros(3, dtype=torch.int32)
    plan.run(q, k, v, offsets, offsets, out=out)
    for change in (dict(q=q[:5]), dict(k=k.half()), dict(v=v[:8]), dict(qo=offsets[:2]), dict(ko=offsets.long()), dict(out=q),
                   dict(out=out[:, :2])):
        a = {**dict(q=q, k=k, v=v, qo=offsets, ko=offsets, out=out), **change}
        with pytest.raises((ValueError, TypeError)):
            plan.run(a["q"], a["k"], a["v"], a["qo"], a["ko"], out=a["out"])
    assert len(backend.launches) == 1


def test_packed_workspace_is_free_before_the_first_run_and_held_until_the_last(backend, monkeypatch):
    """The plan's own memory, allocated on one stream and used on others: waited for once, recorded where it is used."""
    waited, recorded, stream = [], [], [7]
    fake = SimpleNamespace(synchronize=lambda: waited.append(stream[0]))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: fake)
    monkeypatch.setattr("venturi_amd.attention.stream_of", lambda device: stream[0], raising=False)
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda tensor, on: recorded.append((tensor.data_ptr(), on)))
    base = dict(q_heads=4, kv_heads=4, head_dim=64, dtype=FP16, device=CPU)
    without = PackedAttentionPlan.create(backend, tokens=64, keys=64, sequences=1, **base)
    assert not without.storage_tensors and not waited
    plan = PackedAttentionPlan.create(backend, tokens=2, keys=1024, sequences=1, **base)
    assert len(plan.storage_tensors) == 1 and waited == [7]
    rows, keys = torch.zeros(2, 4, 64, dtype=FP16), torch.zeros(1024, 4, 64, dtype=FP16)
    offsets = torch.zeros(2, dtype=torch.int32)
    for stream[0] in (7, 8):
        plan.run(rows, keys, keys, offsets, offsets, out=rows.clone())
    assert recorded == [(plan.storage_tensors[0].data_ptr(), fake)] and waited == [7]


def test_sampling_refusals(backend):
    for change in (dict(rows=0), dict(vocab=0), dict(vocab=2**20 + 1), dict(dtype=torch.float32)):
        with pytest.raises(ValueError):
            SamplingPlan.create(backend, **{**dict(rows=2, vocab=100, dtype=FP16, device=CPU), **change})
    plan = SamplingPlan.create(backend, rows=2, vocab=104, dtype=FP16, device=CPU)
    logits, u = torch.zeros(2, 104, dtype=FP16), torch.zeros(2)
    tokens, chances = torch.zeros(2, dtype=torch.int64), torch.zeros(2)
    plan.run(logits, u, tokens=tokens)
    plan.run(logits, u, u, tokens.int(), u, u, tokens=tokens, probabilities=chances)
    shifted = torch.zeros(209, dtype=FP16)[1:].view(2, 104)
    for change in (dict(logits=logits[:, :103]), dict(logits=shifted), dict(u=u.double()), dict(t=u.half()), dict(k=tokens), dict(p=u[:1]),
                   dict(m=chances.double()), dict(tokens=tokens.int()), dict(chances=u), dict(chances=chances.double())):
        a = {**dict(logits=logits, u=u, t=None, k=None, p=None, m=None, tokens=tokens, chances=chances), **change}
        with pytest.raises((ValueError, TypeError)):
            plan.run(a["logits"], a["u"], a["t"], a["k"], a["p"], a["m"], tokens=a["tokens"], probabilities=a["chances"])
    assert len(backend.launches) == 2


@pytest.mark.parametrize("scale", [1e39, -1e39, 2e38, pytest.param(10**400, id="10^400"), math.inf, math.nan, True, "1"])
def test_scales_out_of_range(backend, scale):
    with pytest.raises(ValueError, match="scale"):
        cache(backend).prepare_attention(sequences=2, q_heads=4, query_tokens=1, max_pages=4, scale=scale)
    with pytest.raises(ValueError, match="scale"):
        PackedAttentionPlan.create(backend, tokens=6, keys=9, sequences=2, q_heads=4, kv_heads=2, head_dim=64, dtype=BF16, device=CPU,
                                   scale=scale)
    if type(scale) is float:  # 1e39 is an infinity by the time an entry point has it
        for entry, good in (("venturi_kv_attention_run", ATTEND), ("venturi_packed_attention_run", PACKED)):
            assert getattr(native.load(), entry)(*{**good, "scale": scale}.values()) == -1 and "scale" in native.load().error()


@pytest.mark.parametrize("scale", [0, 2, -0.5, -(2.0**127)])
def test_scales_in_range(backend, scale):
    assert cache(backend).prepare_attention(sequences=2, q_heads=4, query_tokens=1, max_pages=4, scale=scale).scale == float(scale)


def test_capabilities():
    caps = object.__new__(HipBackend).capabilities
    for operation in ("kv_cache", "attention", "sampling"):
        for dtype in (FP16, BF16):
            assert caps.supports(operation, dtype=dtype, device="cuda:0")
        assert not caps.supports(operation, dtype=torch.float32, device="cuda:0")


# -- the C entry points ---------------------------------------------------------
A, B = 1 << 30, 1 << 36  # addresses that every alignment check accepts; nothing is launched
WRITE = dict(qkv=A, positions=A, slots=A, rates=A, q=B, k=B, kc=A, ks=A, vc=A, vs=A, tokens=1, q_heads=4, kv_heads=2, head_dim=64,
             rotary_dim=64, interleaved=0, factor=1.0, pages=2, page_tokens=16, dtype=0, stream=None)
READ = dict(kc=A, ks=A, vc=A, vs=A, slots=A, keys=B, values=B, tokens=1, kv_heads=2, head_dim=64, pages=2, page_tokens=16, dtype=0,
            stream=None)
ATTEND = dict(q=A, kc=A, ks=A, vc=A, vs=A, table=A, lengths=A, out=B, workspace=B, available=1 << 40, sequences=1, query_tokens=1,
              q_heads=4, kv_heads=2, head_dim=64, pages=2, page_tokens=16, max_pages=2, scale=1.0, dtype=0, stream=None)
PACKED = dict(q=A, k=A, v=A, qo=A, ko=A, out=B, workspace=B, available=1 << 40, tokens=1, keys=1, sequences=1, q_heads=4, kv_heads=2,
              head_dim=64, scale=1.0, dtype=0, stream=None)
SAMPLE = dict(logits=A, uniforms=A, t=None, k=None, p=None, m=None, tokens=B, chances=None, rows=1, vocab=10, dtype=0, stream=None)


@pytest.mark.parametrize("entry,good,changes", [
    ("venturi_kv_write_run", WRITE, [dict(qkv=None), dict(qkv=A + 2), dict(slots=None), dict(positions=None), dict(rates=None), dict(q=None),
                                     dict(q_heads=0), dict(kc=None), dict(vs=A + 8), dict(tokens=0), dict(head_dim=65), dict(head_dim=512),
                                     dict(rotary_dim=66), dict(rotary_dim=63), dict(kv_heads=0), dict(pages=0), dict(page_tokens=8),
                                     dict(dtype=2), dict(q_heads=1 << 30)]),
    ("venturi_kv_read_run", READ, [dict(keys=None, values=None), dict(slots=None), dict(keys=B + 2), dict(tokens=0), dict(dtype=2),
                                   dict(page_tokens=17)]),
    ("venturi_kv_attention_run", ATTEND, [dict(q=None), dict(q=A + 8), dict(out=None), dict(table=None), dict(lengths=None), dict(q_heads=3),
                                          dict(sequences=0), dict(query_tokens=0), dict(max_pages=1 << 28), dict(dtype=2), dict(kc=None),
                                          dict(head_dim=260)]),
    ("venturi_packed_attention_run", PACKED, [dict(q=None), dict(k=A + 2), dict(out=None), dict(qo=None), dict(tokens=0), dict(keys=0),
                                              dict(q_heads=5), dict(head_dim=12), dict(dtype=2)]),
    ("venturi_sample_run", SAMPLE, [dict(logits=None), dict(logits=A + 2), dict(uniforms=None), dict(tokens=None), dict(rows=0), dict(vocab=0),
                                    dict(vocab=(1 << 20) + 1), dict(dtype=2)])])
def test_entry_points_refuse_on_the_host(entry, good, changes):
    lib = native.load()
    for change in changes:
        assert getattr(lib, entry)(*{**good, **change}.values()) == -1, change
        assert lib.error()


def test_workspace_sizes_refuse_bad_geometry():
    lib = native.load()
    for entry, bad in (("venturi_kv_attention_bytes", (1, 1, 3, 2, 64, 2, 16)), ("venturi_packed_attention_bytes", (1, 1, 1, 4, 2, 300))):
        assert getattr(lib, entry)(*bad) == 0 and lib.error()
