"""The residual's addition with the norm after it: the bytes of the plans that it replaces, and the definition in 64 bits."""

import math

import pytest
import torch

from venturi_amd import prepare_residual_rms
from venturi_amd.operands import stream_of

pytestmark = pytest.mark.gpu

FP16, BF16, FP32 = torch.float16, torch.bfloat16, torch.float32


def rows(tokens, k, dtype, seed, device, shift=0):
    gen = torch.Generator().manual_seed(seed)
    x, r = torch.randn(tokens, k, generator=gen), 2 * torch.randn(tokens, k, generator=gen)
    r[:, ::101] *= 20
    made = []
    for t in (x, r):  # off the start of an allocation by `shift` elements
        made.append(torch.empty(tokens * k + shift, dtype=dtype, device=device)[shift:].view(tokens, k).copy_(t))
    return made


def norm_of(backend, device, k, dtype):
    gamma = 1 + 0.1 * torch.randn(k, generator=torch.Generator().manual_seed(k))
    return backend.upload_rmsnorm(gamma, dtype=dtype, device=device, epsilon=1e-6), gamma


def apart(backend, device, norm, x, r, passes):
    """The same by the plans for each step."""
    tokens, k = x.shape
    total, out, workspace = torch.empty_like(x), torch.empty_like(x), None
    backend.prepare_add(tokens=tokens, features=k, dtype=x.dtype, device=device).run(x, r, out=total)
    norm.prepare(tokens=tokens).run(total, out=out)
    if passes:
        lib = backend._native
        workspace = torch.empty(lib.venturi_q8_dp4a_bytes(tokens, k, passes), dtype=torch.uint8, device=device)
        backend._check(lib.venturi_q8_dp4a_quantize(out.data_ptr(), workspace.data_ptr(), workspace.numel(), tokens, k, passes,
                                                    stream_of(device)))
    return total, out, workspace


def guarded(shape, dtype, device, shift=0):
    """A buffer inside a larger one, and a check that nothing around it was written."""
    count = math.prod(shape)
    base = torch.full((count + 64,), 47, dtype=dtype, device=device)
    inner = slice(32 + shift, 32 + shift + count)

    def untouched():
        return bool((base[: inner.start] == 47).all()) and bool((base[inner.stop:] == 47).all())

    return base[inner].view(shape), untouched


def check(backend, device, x, r, norm, passes=0, shift=0, with_out=True):
    want_total, want_out, want_workspace = apart(backend, device, norm, x, r, passes)
    tokens, k = x.shape
    plan = prepare_residual_rms(norm, tokens=tokens, a8_passes=passes)
    total, a = guarded((tokens, k), x.dtype, device, shift)
    out, b = guarded((tokens, k), x.dtype, device, shift)
    workspace, c = guarded((plan.workspace_bytes,), torch.uint8, device) if passes else (None, lambda: True)
    plan.run(x, r, total=total, out=out if with_out else None, workspace=workspace)
    torch.cuda.synchronize()
    assert a() and b() and c()

    def same(u, v):
        return torch.equal(u.view(torch.uint8), v.view(torch.uint8))

    assert same(total, want_total)
    assert same(out, want_out) if with_out else bool((out == 47).all())
    assert not passes or same(workspace, want_workspace)
    return total, out


WIDTHS = [1, 3, 8, 31, 33, 64, 67, 100, 256, 257, 512, 1000, 1024, 1025, 2048, 2052, 4096, 4100, 5120, 6144, 8192, 8200, 8704, 12288, 17408]


@pytest.mark.parametrize("dtype", [FP16, BF16, FP32], ids=["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("k", WIDTHS)
def test_bytes_of_the_steps(backend, device, dtype, k):
    norm, gamma = norm_of(backend, device, k, dtype)
    for tokens in (1, 2, 7, 65, 600):
        print(f"case residual norm {dtype} {tokens} x {k}", flush=True)
        x, r = rows(tokens, k, dtype, tokens, device)
        total, out = check(backend, device, x, r, norm)
    # Half a step for the sum's one rounding (and 2^-24 for its 32-bit form); the norm's besides: 256 chains of k / 256 terms
    # and a tree of 8 levels, halved by the root, the division's, the root's and two products' roundings in 32 bits.
    half = torch.finfo(dtype).eps / 2
    exact = x.double() + r.double()
    assert bool(((total.double() - exact).abs() <= (half + 2.0**-24) * exact.abs() + 2.0**-25).all())
    h = total.double()
    ideal = h / (h.square().mean(-1, keepdim=True) + 1e-6).sqrt() * gamma.to(device).double()
    relative = half + ((k / 256 + 10) / 2 + 5) * 2.0**-24
    assert bool(((out.double() - ideal).abs() <= relative * 1.01 * ideal.abs() + 2.0**-25).all())


@pytest.mark.parametrize("passes", [1, 2])
@pytest.mark.parametrize("k", WIDTHS)
def test_bytes_of_the_int8_form(backend, device, passes, k):
    norm, _ = norm_of(backend, device, k, FP16)
    for tokens in (1, 5, 64, 600):
        print(f"case residual norm a8 {tokens} x {k} passes {passes}", flush=True)
        x, r = rows(tokens, k, FP16, tokens, device)
        check(backend, device, x, r, norm, passes, with_out=tokens != 5)


@pytest.mark.parametrize("dtype,tokens,k,shift,passes", [
    (FP16, 3, 5120, 1, 0), (FP16, 3, 5120, 4, 0), (FP16, 700, 2048, 2, 2), (BF16, 700, 4100, 4, 0), (FP32, 3, 1024, 1, 0),
    (FP16, 2, 30720, 0, 1), (FP16, 2, 30728, 0, 2), (BF16, 2, 65544, 0, 0), (FP32, 2, 15368, 0, 0), (FP32, 600, 4096, 0, 0),
    (FP16, 66000, 40, 0, 1), (BF16, 70000, 520, 0, 0), (FP16, 2050, 512, 0, 2), (FP16, 2049, 1020, 0, 1), (BF16, 300, 2051, 8, 0)])
def test_alignments_long_rows_and_many_rows(backend, device, dtype, tokens, k, shift, passes):
    print(f"case residual norm {dtype} {tokens} x {k} shift {shift} passes {passes}", flush=True)
    norm, _ = norm_of(backend, device, k, dtype)
    x, r = rows(tokens, k, dtype, 3, device, shift)
    check(backend, device, x, r, norm, passes, shift)


@pytest.mark.parametrize("tokens", [2, 900])
def test_in_place(backend, device, tokens):
    norm, _ = norm_of(backend, device, 2048, FP16)
    for passes in (0, 1):
        x, r = rows(tokens, 2048, FP16, 5, device)
        total, out, workspace = apart(backend, device, norm, x, r, passes)
        twice = apart(backend, device, norm, x, x, passes)
        plan = prepare_residual_rms(norm, tokens=tokens, a8_passes=passes)
        for first, second, place, want in ((x, r, 0, total), (x, r, 1, total), (x, x, 0, twice[0])):
            first, second = first.clone(), second.clone() if second is not first else None
            second = first if second is None else second
            got, codes = torch.empty_like(out), None if workspace is None else torch.empty_like(workspace)
            plan.run(first, second, total=(first, second)[place], out=got, workspace=codes)
            assert torch.equal((first, second)[place], want)
            assert torch.equal(got, twice[1] if want is twice[0] else out)


@pytest.mark.parametrize("k", [96, 2048, 5120, 5121])
def test_values_that_are_no_numbers(backend, device, k):
    """Infinities, NaN, overflowing sums and rows of zeros, in few and many rows."""
    norm, _ = norm_of(backend, device, k, FP16)
    for tokens in (6, 600):
        x, r = rows(tokens, k, FP16, 6, device)
        x[0, 5], x[1, 7], x[2, k - 1] = math.inf, math.nan, -math.inf
        r[2, k - 1] = math.inf
        x[3], r[3] = 60000.0, 60000.0
        x[4], r[4] = 0.0, -0.0
        for passes in (0, 1, 2):
            check(backend, device, x, r, norm, passes)


def test_graph_and_side_stream(backend, device):
    for tokens, passes in ((1, 0), (61, 2), (900, 1)):
        norm, _ = norm_of(backend, device, 5120, FP16)
        plan = prepare_residual_rms(norm, tokens=tokens, a8_passes=passes)
        x, r = rows(tokens, 5120, FP16, 7, device)
        out = torch.empty_like(x)
        workspace = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device=device) if passes else None
        side = torch.cuda.Stream(device)
        side.wait_stream(torch.cuda.current_stream(device))
        with torch.cuda.stream(side):
            plan.run(x, r, total=r, out=out, workspace=workspace)
        torch.cuda.current_stream(device).wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan.run(x, r, total=r, out=out, workspace=workspace)
        for i in range(4):
            start = rows(tokens, 5120, FP16, 10 + i, device)
            want = apart(backend, device, norm, *start, passes)
            x.copy_(start[0]), r.copy_(start[1]), out.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(r, want[0]) and torch.equal(out, want[1])
            assert not passes or torch.equal(workspace, want[2])
