"""64-bit oracles of the rotary write, the Q8 cache and causal attention, and the error bounds of their kernels."""

from fractions import Fraction
import math

import torch

GROUP = 32
TURN = 2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494459")


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def q8_rule(x):
    """Codes int8 [.., d] and scales fp16 [.., ceil(d / 32)] of rows, with the 32-bit arithmetic that the rule names."""
    d = x.shape[-1]
    groups = (d + GROUP - 1) // GROUP
    x = torch.nn.functional.pad(x.float(), (0, groups * GROUP - d)).unflatten(-1, (groups, GROUP))
    scales = (x.abs().amax(-1) / 127).half()
    s = scales.float()[..., None]
    codes = torch.where((s > 0) & s.isfinite(), torch.round(x / s).clamp(-127, 127), torch.zeros_like(x))
    return codes.to(torch.int8).flatten(-2)[..., :d], scales


def q8_values(codes, scales):
    """What codes and scales stand for, in 64 bits (their products are exact)."""
    return codes.double() * scales.double().repeat_interleave(GROUP, -1)[..., : codes.shape[-1]]


def rotate(x, positions, frequencies, factor, layout):
    """x [tokens, heads, d] in 64 bits; returns the rotated rows and the size that their error goes by. The angles'
    whole turns are taken off in exact arithmetic: in 64 bits the angle of position 2^40 is known to 1e-4 only."""
    x, r = x.double(), 2 * len(frequencies)
    rates = [Fraction(f) / TURN for f in frequencies]
    turns = [[float((p * rate + Fraction(1, 2)) % 1 - Fraction(1, 2)) for rate in rates] for p in positions.tolist()]
    angle = torch.tensor(turns, dtype=torch.float64)[:, None] * (2 * math.pi)
    c, s = factor * torch.cos(angle), factor * torch.sin(angle)
    a, b = (x[..., : r // 2], x[..., r // 2: r]) if layout == "half" else (x[..., 0:r:2], x[..., 1:r:2])
    y, size = torch.empty_like(x), x.abs().clone()
    y[..., r:] = x[..., r:]
    parts = (a * c - b * s, b * c + a * s)
    both = factor * (a.abs() + b.abs())
    if layout == "half":
        y[..., :r] = torch.cat(parts, -1)
        size[..., :r] = torch.cat([both, both], -1)
    else:
        y[..., :r] = torch.stack(parts, -1).flatten(-2)
        size[..., :r] = torch.stack([both, both], -1).flatten(-2)
    return y, size


def attend(q, k, v, seen, scale=None):
    """q [t, hq, d], k and v [n, hk, d]; query i sees the first seen[i] keys. Returns the 64-bit outputs, the mean of
    |v| under the same weights, and the largest sum_d |q_d k_d| * scale of every row."""
    t, hq, d = q.shape
    n, hk = k.shape[:2]
    scale = d ** -0.5 if scale is None else scale
    out, mean, size = (torch.zeros(t, hq, d, dtype=torch.float64) for _ in range(2)), None, torch.zeros(t, hq, dtype=torch.float64)
    out, mean = out
    q, k, v = q.double(), k.double(), v.double()
    hidden = torch.arange(n)[None] >= torch.as_tensor(seen)[:, None]
    for h in range(hq):
        kk, vv = k[:, h * hk // hq], v[:, h * hk // hq]
        scores = ((q[:, h] @ kk.T) * scale).masked_fill(hidden, -math.inf)
        weights = torch.softmax(scores, -1).nan_to_num(0.0) if n else scores
        out[:, h], mean[:, h] = weights @ vv, weights @ vv.abs()
        if n:
            size[:, h] = ((q[:, h].abs() @ kk.abs().T) * abs(scale)).masked_fill(hidden, 0.0).amax(-1)
    return out, mean, size


def attention_bound(out, mean, size, d, n, dtype, weight_step, value_step=0.0):
    """Largest error of an attention kernel with fp32 scores and sums.

    A score sums d products in fp32 (d + 2 roundings of a sum no larger than `size`, and the exponent's own 4), a
    weight moves by twice its score's error (its own and the largest's), weights and values are rounded by half a step
    each, their sum over n keys and the total round in fp32 (4 per key is never reached: n of them), and the output
    rounds once. Weights below 2^-20 may be rounded absolutely (fp16's subnormal numbers)."""
    scores = 2.0 * (d + 6) * 2.0**-24 * (size + 1.0)[..., None]
    relative = weight_step + value_step + scores + 2.0 * (n + 64) * 2.0**-24
    return mean * relative * 1.01 + out.abs() * half_step(dtype) * 1.01 + n * 2.0**-26 * mean + 2.0**-24
