"""What the plans of the residual norm, routing, distributions and verification refuse (no GPU): the checks of `prepare` and
`run` on CPU tensors with a backend that records its launches, and the C entry points' own; and which kernels they launch."""

from contextlib import nullcontext
import math
from types import SimpleNamespace

import pytest
import torch

from launches import LdsLimit, Launch, built, kernels, pointers, record
from venturi_amd import native, prepare_residual_rms
from venturi_amd.blocks import HipBackend, ResidentRMSNorm
from venturi_amd.routing import RoutingPlan
from venturi_amd.sampling import DistributionPlan
from venturi_amd.verification import VerificationPlan

CPU = torch.device("cpu")
FP16, BF16, FP32 = torch.float16, torch.bfloat16, torch.float32


class Recorder:
    def __init__(self):
        self._native, self.launches = native.load(), []

    def _call(self, entry, device, arguments):
        assert len(arguments) + 1 == len(entry.argtypes)
        for value, kind in zip(arguments, entry.argtypes):
            kind(value)
        self.launches.append(entry.__name__)

    def _check(self, status):
        self._native.check(status)

    def validate_device(self, dtype, device):
        return CPU


@pytest.fixture
def backend(monkeypatch):
    monkeypatch.setattr(torch.cuda, "device", lambda device: nullcontext())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: SimpleNamespace(synchronize=lambda: None))
    return Recorder()


def refused(run, good, changes):
    for change in changes:
        with pytest.raises((ValueError, TypeError)):
            run(**{**good, **change})


def aligned(count, dtype, align=256):
    """A tensor that starts at a multiple of `align` bytes."""
    size = torch.empty(0, dtype=dtype).element_size()
    store = torch.zeros(count + align // size, dtype=dtype)
    return store[(-store.data_ptr() % align) // size:][:count]


# -- residual norm ---------------------------------------------------------------
def norm_of(backend, features=96, dtype=FP16):
    return ResidentRMSNorm(backend, torch.ones(features), dtype, 1e-6)


def test_residual_norm_refusals(backend):
    norm = norm_of(backend)
    for change in (dict(tokens=0), dict(tokens=2.0), dict(a8_passes=3), dict(a8_passes=True), dict(a8_passes=-1)):
        with pytest.raises(ValueError):
            prepare_residual_rms(norm, **{**dict(tokens=3), **change})
    with pytest.raises(ValueError):
        prepare_residual_rms(torch.ones(96), tokens=3)
    for dtype in (BF16, FP32):
        with pytest.raises(ValueError):
            prepare_residual_rms(norm_of(backend, dtype=dtype), tokens=3, a8_passes=1)
    plan = prepare_residual_rms(norm, tokens=3, a8_passes=2)
    assert plan.workspace_bytes == 3 * 3 * 36 * 2 and plan.storage_tensors == norm.storage_tensors
    x, r, t, y = (torch.zeros(3, 96, dtype=FP16) for _ in range(4))
    w = aligned(plan.workspace_bytes, torch.uint8)
    good = dict(x=x, residual=r, total=t, out=y, workspace=w)
    plan.run(**good)
    plan.run(**{**good, "out": None})
    plan.run(**{**good, "total": x})
    plan.run(**{**good, "total": r})
    plan.run(**{**good, "residual": x, "total": x})
    assert backend.launches == ["venturi_residual_rms_run"] * 5
    buffer = torch.zeros(4 * 96, dtype=FP16)
    refused(plan.run, good, [
        dict(x=x[:2]), dict(x=x.bfloat16()), dict(residual=x.T.contiguous().T), dict(total=buffer[8:296].view(3, 96), x=buffer[:288].view(3, 96)),
        dict(out=x), dict(out=r), dict(out=t), dict(out=y.float()), dict(workspace=None), dict(workspace=w[:-1]),
        dict(workspace=x.view(torch.uint8).view(-1)[: plan.workspace_bytes]), dict(total=None),
        dict(x=torch.zeros(3, 96, dtype=FP16, requires_grad=True))])
    plain = prepare_residual_rms(norm, tokens=3)
    plain.run(x, r, total=t, out=y)
    refused(plain.run, dict(x=x, residual=r, total=t, out=y), [dict(out=None), dict(workspace=w)])
    assert len(backend.launches) == 6


# -- routing ---------------------------------------------------------------------
ROUTE = dict(tokens=3, experts=64, top_k=4, dtype=BF16, device=CPU)


@pytest.mark.parametrize("change", [
    dict(tokens=0), dict(experts=0), dict(experts=1025), dict(top_k=0), dict(top_k=17), dict(experts=3), dict(groups=5), dict(groups=0),
    dict(groups=128, experts=1024), dict(groups=4, kept_groups=5), dict(groups=32, kept_groups=1), dict(kept_groups=2), dict(score="relu"),
    dict(group_rank="sum"), dict(renormalize=1), dict(scale=math.inf), dict(scale=math.nan), dict(scale="1"), dict(scale=1e39),
    dict(dtype=torch.float64), dict(score_dtype=torch.int32), dict(scale=True)])
def test_routing_plan_refusals(backend, change):
    with pytest.raises(ValueError):
        RoutingPlan.create(backend, **{**ROUTE, **change})


def test_routing_refusals(backend):
    plan = RoutingPlan.create(backend, **ROUTE)
    x, b = torch.zeros(3, 64, dtype=BF16), torch.zeros(64)
    i, s = torch.zeros(3, 4, dtype=torch.int64), torch.zeros(3, 4, dtype=FP16)

    def run(logits, bias, indices, scores):
        plan.run(logits, bias, indices=indices, scores=scores)

    good = dict(logits=x, bias=None, indices=i, scores=s)
    run(**good)
    run(**{**good, "bias": b})
    refused(run, good, [dict(logits=x.half()), dict(logits=x[:2]), dict(bias=b.half()), dict(bias=b[:63]), dict(indices=i.int()),
                        dict(indices=i[:, :3]), dict(scores=s.float()), dict(scores=i.view(FP16)[:, :4]), dict(scores=None),
                        dict(scores=x.view(-1)[:12].view(3, 4).view(FP16))])
    assert backend.launches == ["venturi_route_run"] * 2


# -- distributions ---------------------------------------------------------------
def test_distribution_refusals(backend):
    base = dict(rows=2, vocab=104, dtype=FP16, device=CPU)
    for change in (dict(rows=0), dict(rows=65536), dict(vocab=0), dict(vocab=2**20 + 1), dict(dtype=FP32)):
        with pytest.raises(ValueError):
            DistributionPlan.create(backend, **{**base, **change})
    plan = DistributionPlan.create(backend, **base)
    logits, p, w = aligned(208, FP16).view(2, 104), torch.zeros(2, 104), aligned(plan.workspace_bytes, torch.uint8)
    t, k = torch.zeros(2), torch.zeros(2, dtype=torch.int32)

    def run(logits, t, k, m, p, w):
        plan.run(logits, t, k, None, m, probabilities=p, workspace=w)

    good = dict(logits=logits, t=None, k=None, m=None, p=p, w=w)
    run(**good)
    run(**{**good, "t": t, "k": k, "m": t})
    shifted = aligned(209, FP16)[1:].view(2, 104)
    refused(run, good, [dict(logits=logits[:, :103]), dict(logits=shifted), dict(t=t.half()), dict(k=k.long()), dict(m=t[:1]),
                        dict(p=p.double()), dict(p=p[:1]), dict(p=None), dict(w=None), dict(w=w[:-1]),
                        dict(w=aligned(plan.workspace_bytes + 16, torch.uint8)[16:]), dict(p=None, w=p.view(-1)[:16].view(torch.uint8))])
    assert backend.launches == ["venturi_distribution_run"] * 2


# -- verification ----------------------------------------------------------------
def test_verification_refusals(backend):
    base = dict(sequences=2, drafts=3, vocab=40000, device=CPU)
    for change in (dict(sequences=0), dict(sequences=65536), dict(drafts=0), dict(drafts=65), dict(vocab=0), dict(vocab=2**20 + 1),
                   dict(drafts=True)):
        with pytest.raises(ValueError):
            VerificationPlan.create(backend, **{**base, **change})
    plan = VerificationPlan.create(backend, **base)
    assert plan.workspace_bytes and not VerificationPlan.create(backend, **{**base, "vocab": 4000}).workspace_bytes
    good = dict(target=torch.zeros(8, 40000), drafted=torch.zeros(2, 3, dtype=torch.int64), uniforms=torch.zeros(2, 4),
                proposal=torch.zeros(6, 40000), counts=torch.zeros(2, dtype=torch.int32), tokens=torch.zeros(2, 4, dtype=torch.int64),
                accepted=torch.zeros(2, dtype=torch.int32), workspace=aligned(plan.workspace_bytes, torch.uint8))
    plan.run(**good)
    plan.run(**{**good, "proposal": None, "counts": None})
    refused(plan.run, good, [
        dict(target=good["target"][:7]), dict(target=good["target"].half()), dict(drafted=good["drafted"].int()),
        dict(drafted=good["drafted"][:, :2]), dict(uniforms=good["uniforms"][:, :3]), dict(uniforms=good["uniforms"].double()),
        dict(proposal=good["proposal"][:5]), dict(counts=good["drafted"][:, 0]), dict(tokens=good["drafted"]), dict(tokens=None),
        dict(accepted=good["counts"]), dict(accepted=good["accepted"].long()), dict(workspace=None), dict(workspace=good["workspace"][:-1]),
        dict(workspace=good["target"].view(-1)[: plan.workspace_bytes // 4].view(torch.uint8)),
        dict(accepted=good["tokens"].view(-1)[:1].view(torch.int32))])
    assert backend.launches == ["venturi_verify_run"] * 2


def test_capabilities():
    caps = object.__new__(HipBackend).capabilities
    assert caps.supports("distribution", dtype=BF16, device="cuda:0") and not caps.supports("distribution", dtype=FP32, device="cuda:0")
    assert caps.supports("verification", dtype=FP32, device="cuda:0") and not caps.supports("verification", dtype=FP16, device="cuda:0")
    for operation in ("routing", "residual_rmsnorm"):
        for dtype in (FP16, BF16, FP32):
            assert caps.supports(operation, dtype=dtype, device="cuda:0")


# -- the C entry points ------------------------------------------------------------
A, B, C, D, E, F = pointers(6)  # buffers far apart; nothing is launched
RMS = dict(x=A, residual=B, gamma=C, total=D, out=E, workspace=F, available=1 << 40, tokens=2, k=96, passes=1, dtype=0, epsilon=1e-6, stream=None)
ROUTED = dict(logits=A, bias=B, indices=C, scores=D, tokens=1, experts=64, top_k=4, groups=4, kept=2, sigmoid=0, pairs=1, renormalize=1,
              scale=1.0, dtype=0, score_dtype=0, stream=None)
KEPT = dict(logits=A, t=None, k=None, p=None, m=None, out=B, workspace=C, available=1 << 40, rows=1, vocab=10, dtype=0, stream=None)
VERIFY = dict(target=A, proposal=B, drafted=C, counts=None, uniforms=D, tokens=E, accepted=F, workspace=F + 4096, available=1 << 40, sequences=2,
              drafts=3, vocab=9000, stream=None)


@pytest.mark.parametrize("entry,good,changes", [
    ("venturi_residual_rms_run", RMS, [
        dict(x=None), dict(residual=None), dict(gamma=None), dict(total=None), dict(workspace=None), dict(available=100), dict(workspace=F + 8),
        dict(tokens=0), dict(k=0), dict(passes=3), dict(passes=-1), dict(dtype=1), dict(dtype=3), dict(epsilon=0.0), dict(epsilon=math.nan),
        dict(epsilon=math.inf), dict(x=A + 1), dict(gamma=C + 2), dict(total=A + 2), dict(out=A), dict(out=D), dict(workspace=A), dict(out=C),
        dict(workspace=E), dict(out=None, passes=0), dict(tokens=300000), dict(total=C, passes=0)]),
    ("venturi_route_run", ROUTED, [
        dict(logits=None), dict(indices=None), dict(scores=None), dict(logits=A + 1), dict(bias=B + 2), dict(indices=C + 4), dict(scores=D + 1),
        dict(tokens=0), dict(experts=0), dict(experts=1025), dict(top_k=0), dict(top_k=17), dict(groups=3), dict(groups=0), dict(kept=5),
        dict(kept=0), dict(groups=32, kept=1), dict(scale=math.inf), dict(dtype=3), dict(score_dtype=-1), dict(groups=128, experts=1024)]),
    ("venturi_distribution_run", KEPT, [
        dict(logits=None), dict(logits=A + 2), dict(out=None), dict(out=B + 2), dict(workspace=None), dict(available=31), dict(workspace=C + 128),
        dict(rows=0), dict(rows=65536), dict(vocab=0), dict(vocab=(1 << 20) + 1), dict(dtype=2)]),
    ("venturi_verify_run", VERIFY, [
        dict(target=None), dict(drafted=None), dict(uniforms=None), dict(tokens=None), dict(accepted=None), dict(target=A + 2),
        dict(drafted=C + 4), dict(workspace=None), dict(available=16), dict(workspace=F + 8), dict(sequences=0), dict(sequences=65536),
        dict(drafts=0), dict(drafts=65), dict(vocab=0), dict(vocab=(1 << 20) + 1)])])
def test_entry_points_refuse_on_the_host(entry, good, changes):
    lib = native.load()
    for change in changes:
        assert getattr(lib, entry)(*{**good, **change}.values()) == -1, change
        assert lib.error()


def test_workspace_sizes():
    lib = native.load()
    assert lib.venturi_distribution_bytes(96, 1000) == 96 * 32
    # Of up to 32 long rows also parts of 8192 logits and chunks of 128.
    assert [lib.venturi_distribution_bytes(*s) for s in ((5, 57344), (33, 81920), (32, 81920))] == [5 * 32, 33 * 32, 32 * (32 + 16 * 10 + 2 * 640)]
    for bad in ((0, 5), (65536, 5), (1, 0), (1, 2**20 + 1)):
        assert lib.venturi_distribution_bytes(*bad) == 0 and lib.error()
    for bad in ((0, 1, 5), (65536, 1, 5), (1, 0, 5), (1, 65, 5), (1, 1, 0), (1, 1, 2**20 + 1)):
        assert lib.venturi_verify_bytes(*bad) == 0 and lib.error()


# -- launches ------------------------------------------------------------------------
def rms(tokens, k, dtype, passes=0, shift=0):
    return "venturi_residual_rms_run", [A + shift, B, C, D, E, F if passes else None, 1 << 40, tokens, k, passes, dtype, 1e-6, None]


def route(tokens, experts, groups, bias, sigmoid, dtype, shift=0):
    return "venturi_route_run", [A + shift, B if bias else None, C, D, tokens, experts, min(2, experts), groups, groups, sigmoid, 1, 1, 1.0, dtype, 0,
                                 None]


def reached(calls):
    return {kernel for launched in kernels([(0, *call) for call in calls]) for kernel in launched}


def test_residual_norm_tests_reach_every_instance():
    shapes = [(1, 5120), (600, 5120), (600, 2048), (7, 5121), (600, 4100), (7, 33), (2, 64), (2050, 512), (2049, 1020), (2, 65544)]
    calls = [rms(t, k, dtype) for t, k in shapes for dtype in (0, 1, 2)] + [rms(300, 2051, dtype) for dtype in (0, 1, 2)]
    names = {name for kernel in ("residual_rms_any", "residual_rms_wave", "residual_rms_staged") for name in built(kernel)}
    assert names and names == reached(calls + [rms(2, 40000, 2)])


def test_routing_tests_reach_every_instance():
    sizes = [(64, 4), (128, 8), (256, 8), (512, 16), (1024, 64)]
    calls = [route(33, e - odd, 1 if odd else groups, bias, sigmoid, dtype) for e, groups in sizes for odd in (0, 1) for bias in (0, 1)
             for sigmoid in (0, 1) for dtype in (0, 1, 2)]
    calls += [route(6, e, 1, 0, 0, dtype) for e, _ in sizes for dtype in (0, 1, 2)]
    names = built("route_logits") | built("route_scores")
    assert names and names == reached(calls)


def test_distribution_raises_its_lds_limit_on_every_device():
    limits = {}
    logits, p, w = pointers(3)
    call = ("venturi_distribution_run", [logits, None, None, None, None, p, w, 1 << 40, 3, 1000, 1, None])
    for events in record([(device, *call) for device in (0, 1, 0, 70)]):
        launches = [e for e in events if isinstance(e, Launch)]
        limits.update({(e.kernel, e.device): e.bytes for e in events if isinstance(e, LdsLimit)})
        assert len(launches) == 2 and limits[launches[0].kernel, launches[0].device] >= launches[0].shared > 65536


@pytest.mark.parametrize("rows,vocab,kernels", [(3, 80000, 3), (32, 57345, 3), (3, 57344, 2), (33, 80000, 2), (3, 7, 2)])
def test_few_long_rows_are_looked_at_first(rows, vocab, kernels):
    logits, p, w = pointers(3)
    for dtype in (0, 1):
        events = record([(0, "venturi_distribution_run", [logits, None, None, None, None, p, w, 1 << 40, rows, vocab, dtype, None])])[0]
        launches = [e.kernel.split("<")[0] for e in events if isinstance(e, Launch)]
        assert launches == ["distribution_scan", "distribution_cut", "distribution"][3 - kernels:]


def test_launches_keep_their_threads_within_32_bits():
    """More rows than a launch takes go to several, which cover them all."""
    for call, rows in ((rms(20_000_000, 4096, 0), 20_000_000), (rms(30_000_001, 512, 1), 30_000_001), (rms(5_000_000, 70000, 2), 5_000_000),
                       (route(100_000_007, 64, 1, 0, 0, 1), 100_000_007), (route(50_000_000, 512, 64, 1, 1, 2), 50_000_000)):
        entry, arguments = call
        arguments = [(1 << 30) + (pointers(6).index(v) << 42) if v in pointers(6) else v for v in arguments]  # apart, whatever the size
        launches = [e for e in record([(0, entry, arguments)])[0] if isinstance(e, Launch)]
        assert len(launches) > 1 and all(e.blocks * e.threads < 2**32 for e in launches)
        per_row = {"residual_rms_wave": 64, "route_logits": 16, "route_scores": 64}.get(launches[0].kernel.split("<")[0], launches[0].threads)
        covered = sum(e.blocks * e.threads // per_row for e in launches)
        assert rows <= covered < rows + 256 * len(launches)


def test_verification_sums_rows_in_parts_where_they_are_long_and_few():
    counts = {(1, 4, 4000): 1, (1, 4, 32768): 1, (1, 4, 32769): 2, (256, 7, 32003): 1, (257, 7, 32003): 2, (300, 1, 16384): 1, (682, 1, 151936): 2,
              (683, 1, 151936): 1, (2048, 1, 151936): 1}
    for (n, d, v), count in counts.items():
        assert len(kernels([(0, "venturi_verify_run", verify(n, d, v)[1])])[0]) == count


def verify(n, d, vocab):
    return "venturi_verify_run", [*VERIFY.values()][:9] + [n, d, vocab, None]


def test_verification_tests_reach_every_instance():
    sizes = [(1, 1, 1), (1100, 1, 8001), (1030, 1, 9001), (300, 1, 5000), (300, 1, 16001), (300, 1, 100001), (2, 1, 16384), (2, 1, 32768),
             (256, 1, 270001), (5, 1, 40001)]
    names = built("verify_sum") | built("verify_take")
    assert names and names == reached([verify(*size) for size in sizes])


@pytest.mark.parametrize("entry,good,changes", [
    ("venturi_route_run", ROUTED, [
        dict(indices=A), dict(indices=A + 120), dict(indices=B + 248), dict(scores=A + 126), dict(scores=B), dict(scores=C + 24),
        dict(indices=D - 24), dict(indices=A + 248, dtype=2), dict(scores=C - 8, score_dtype=2)]),
    ("venturi_distribution_run", {**KEPT, "t": D, "k": D + 64, "p": E, "m": F}, [
        dict(out=A), dict(out=A + 16), dict(out=A - 36), dict(out=D - 36), dict(out=D + 64), dict(out=E), dict(out=F), dict(workspace=A),
        dict(workspace=D), dict(workspace=E), dict(workspace=F), dict(workspace=B), dict(out=C + 28)]),
    ("venturi_verify_run", VERIFY, [
        dict(tokens=A + 8 * 36000 - 8), dict(tokens=B), dict(tokens=C + 40), dict(tokens=D + 24), dict(accepted=A), dict(accepted=B + 215996),
        dict(accepted=C), dict(accepted=D + 28), dict(accepted=E + 60), dict(accepted=E - 4), dict(counts=E), dict(counts=F + 4)]),
    ("venturi_verify_run", {**VERIFY, "vocab": 40000}, [
        dict(workspace=A), dict(workspace=B), dict(workspace=C), dict(workspace=D), dict(workspace=E), dict(workspace=F), dict(tokens=F + 4096),
        dict(counts=F + 4096)])])
def test_entry_points_refuse_outputs_that_overlap(entry, good, changes):
    lib = native.load()
    for change in changes:
        assert getattr(lib, entry)(*{**good, **change}.values()) == -1, change
        assert "overlap" in lib.error(), (change, lib.error())


def test_operands_side_by_side_do_not_overlap():
    calls = [("venturi_route_run", {**ROUTED, "scores": A + 128, "indices": B + 256}),
             ("venturi_distribution_run", {**KEPT, "out": A + 20, "workspace": A + 256}),
             ("venturi_verify_run", {**VERIFY, "tokens": D + 32, "accepted": D + 96, "workspace": D + 96})]  # empty
    for entry, good in calls:
        assert record([(0, entry, list(good.values()))])[0]


def test_columns_whose_count_a_step_on_leaves_32_bits_are_refused():
    wide = {**RMS, "workspace": None, "passes": 0}
    for dtype in (0, 1, 2):
        for k in (2**31 - 1, 2**31 - 1024):
            assert native.load().venturi_residual_rms_run(*{**wide, "dtype": dtype, "k": k}.values()) == -1
            assert "columns" in native.load().error()
        assert kernels([(0, "venturi_residual_rms_run", list({**wide, "dtype": dtype, "k": 2**31 - 1025}.values()))])[0]
