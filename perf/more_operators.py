"""Performance cases of the operators of a speculative step through a mixture-of-experts layer: the residual's addition
with the norm after it, the routing of tokens to experts, the distribution that the sampling settings leave of a row of
logits, and the verification of drafted tokens against such rows.

A case is a dict of plain values with a ``kind``:

* ``norm``: total = x + residual, out = RMSNorm(total), and with ``a8_passes`` its int8 form for the A8 projections;
* ``route``: scores of every expert, top-k among the kept groups, renormalised weights;
* ``distribution``: per row, the probabilities that temperature, top-k, top-p and min-p leave;
* ``verify``: drafts of every sequence accepted or refused, and the token that follows them.

Sizes: hidden 5120 and 2048, 128 experts with 8 of them per token, and the vocabularies 151936 and 248320 are the
repository's; the others are generic.

``own`` False computes the plain form in elementary torch operations; True calls the package.
"""

import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
EPSILON = 1e-6
GROUP = 32  # columns of an int8 scale


def listed():
    return [
        # One user's token: launch and latency count.
        {"name": "norm_token", "kind": "norm", "tokens": 1, "hidden": 5120, "dtype": "fp16", "a8_passes": 0},
        # A decode batch whose projections take int8 activations, with the second pass for the first one's residuals.
        {"name": "norm_a8", "kind": "norm", "tokens": 61, "hidden": 5120, "dtype": "fp16", "a8_passes": 2},
        # A long prompt.
        {"name": "norm_prompt", "kind": "norm", "tokens": 8190, "hidden": 5120, "dtype": "bf16", "a8_passes": 0},
        # One token's experts.
        {"name": "route_token", "kind": "route", "tokens": 1, "experts": 128, "top_k": 8, "dtype": "fp16", "score": "softmax",
         "biased": False, "groups": 1, "kept_groups": 1, "scale": 1.0},
        # Prompts packed together, groups of experts on different nodes, a bias that balances their load.
        {"name": "route_groups", "kind": "route", "tokens": 4099, "experts": 256, "top_k": 8, "dtype": "fp32", "score": "sigmoid",
         "biased": True, "groups": 8, "kept_groups": 4, "scale": 2.5},
        # A large prefill batch.
        {"name": "route_prompt", "kind": "route", "tokens": 16384, "experts": 128, "top_k": 8, "dtype": "bf16",
         "score": "softmax", "biased": False, "groups": 1, "kept_groups": 1, "scale": 1.0},
        # One user's step: four drafted tokens and the one after them, the same settings in every row.
        {"name": "distribution_user", "kind": "distribution", "rows": 5, "vocab": 248320, "dtype": "fp16", "spread": 2.5,
         "settings": "one"},
        # A serving batch of drafts, everybody's own settings.
        {"name": "distribution_batch", "kind": "distribution", "rows": 96, "vocab": 151936, "dtype": "bf16", "spread": 3.0,
         "settings": "mixed"},
        # A drafter's rows by temperature alone, small vocabulary.
        {"name": "distribution_drafter", "kind": "distribution", "rows": 257, "vocab": 32003, "dtype": "fp16", "spread": 2.0,
         "settings": "temperature"},
        # One user's drafts, from a drafter that gives its probabilities.
        {"name": "verify_user", "kind": "verify", "sequences": 1, "drafts": 4, "vocab": 248320, "certain": False, "noise": 0.7},
        # A batch of drafts found in the prompt: certain ones, of differing number.
        {"name": "verify_certain", "kind": "verify", "sequences": 61, "drafts": 7, "vocab": 32003, "certain": True, "noise": 0.5},
        # A large batch with a drafter's probabilities.
        {"name": "verify_batch", "kind": "verify", "sequences": 128, "drafts": 3, "vocab": 151936, "certain": False, "noise": 1.0},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["norm", "route", "distribution", "verify"])
    if kind == "norm":
        hidden = rng.choice([5120, 2048, 6144, 8 * _log_int(rng, 64, 2176), _log_int(rng, 500, 9000)])
        dtype = rng.choice(["fp16", "bf16"])
        return {"kind": kind, "tokens": _log_int(rng, 1, min(16000, 40_000_000 // hidden)), "hidden": hidden, "dtype": dtype,
                "a8_passes": rng.choice([0, 1, 2]) if dtype == "fp16" else 0}
    if kind == "route":
        experts = rng.choice([8, 60, 64, 128, 128, 160, 256, 384, 512])
        groups = rng.choice([1, 1, 4]) if experts % 4 == 0 and experts >= 64 else 1
        return {"kind": kind, "tokens": _log_int(rng, 1, 2_000_000 // experts), "experts": experts,
                "top_k": rng.choice([1, 2, 4, 6, 8]), "dtype": rng.choice(["fp16", "bf16", "fp32"]),
                "score": rng.choice(["softmax", "sigmoid"]), "biased": rng.choice([False, True]), "groups": groups,
                "kept_groups": 2 if groups > 1 else 1, "scale": rng.choice([1.0, 2.5])}
    if kind == "distribution":
        vocab = _log_int(rng, 1000, 200_000)
        return {"kind": kind, "rows": _log_int(rng, 1, min(300, 14_000_000 // vocab)), "vocab": vocab,
                "dtype": rng.choice(["fp16", "bf16"]), "spread": rng.choice([1.0, 2.5, 4.0]),
                "settings": rng.choice(["one", "mixed", "temperature"])}
    vocab, drafts = _log_int(rng, 1000, 200_000), rng.choice([1, 2, 3, 5, 8])
    return {"kind": kind, "sequences": _log_int(rng, 1, min(128, 50_000_000 // (vocab * (drafts + 1)))), "drafts": drafts,
            "vocab": vocab, "certain": rng.choice([False, True]), "noise": rng.choice([0.3, 0.7, 1.5])}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _generators(seed):
    """Values on the GPU, settings and counts on the host."""
    return torch.Generator(device=DEVICE).manual_seed(int(seed)), np.random.default_rng(int(seed))


def _settings(case, rng):
    rows, kind = case["rows"], case["settings"]
    if kind == "one":
        got = {"temperature": [0.8] * rows, "top_k": [50] * rows, "top_p": [0.95] * rows, "min_p": [0.0] * rows}
    elif kind == "temperature":
        got = {"temperature": rng.choice([0.6, 0.8, 1.0], rows), "top_k": [0] * rows, "top_p": [1.0] * rows, "min_p": [0.0] * rows}
    else:
        got = {"temperature": rng.choice([0.6, 0.8, 1.0, 1.3, 0.0], rows, p=[0.25, 0.25, 0.25, 0.2, 0.05]),
               "top_k": rng.choice([0, 20, 50, 1000], rows), "top_p": rng.choice([1.0, 0.95, 0.8], rows),
               "min_p": rng.choice([0.0, 0.0, 0.05], rows)}
    types = {"temperature": torch.float32, "top_k": torch.int32, "top_p": torch.float32, "min_p": torch.float32}
    return {name: torch.as_tensor(np.asarray(v)).to(types[name]).to(DEVICE) for name, v in got.items()}


def _kept(logits):
    """Probabilities as truncated sampling leaves them: what is below a thousandth of a row's largest is gone."""
    p = torch.softmax(logits, -1)
    p = torch.where(p < 1e-3 * p.amax(-1, keepdim=True), 0.0, p)
    return p / p.sum(-1, keepdim=True)


def _inputs(case, seed):
    gen, rng = _generators(seed)
    kind = case["kind"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEVICE)

    if kind == "norm":
        tokens, hidden, dtype = case["tokens"], case["hidden"], DTYPES[case["dtype"]]
        residual = normal(tokens, hidden) * 2  # the stream: some channels are far larger than the rest
        residual[:, ::101] *= 20
        return {"x": normal(tokens, hidden).to(dtype), "residual": residual.to(dtype), "gamma": 1 + 0.1 * normal(hidden)}
    if kind == "route":
        got = {"logits": (normal(case["tokens"], case["experts"]) * 1.5).to(DTYPES[case["dtype"]])}
        got["bias"] = normal(case["experts"]) * 0.05 if case["biased"] else None
        return got
    if kind == "distribution":
        got = _settings(case, rng)
        got["logits"] = (normal(case["rows"], case["vocab"]) * case["spread"]).to(DTYPES[case["dtype"]])
        return got
    n, d, v = case["sequences"], case["drafts"], case["vocab"]
    logits = normal(n, d + 1, v) * 3
    proposal = logits[:, :d] + normal(n, d, v) * case["noise"]
    target = _kept(logits).view(n * (d + 1), v)
    del logits
    got = {"target": target, "uniforms": torch.rand(n, d + 1, generator=gen, device=DEVICE)}
    if case["certain"]:
        got["drafted"], got["proposal"] = proposal.argmax(-1), None
    else:
        q = _kept(proposal)
        mass = q.double().cumsum(-1)
        at = torch.rand(n, d, 1, generator=gen, device=DEVICE, dtype=torch.float64) * mass[..., -1:]
        got["drafted"] = torch.searchsorted(mass, at, right=True).clamp(max=v - 1)[..., 0]
        got["proposal"] = q.view(n * d, v)
    counts = np.full(n, d) if n == 1 else rng.integers(0, d + 1, n)
    got["counts"] = torch.as_tensor(counts, dtype=torch.int32, device=DEVICE)
    return got


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if own:  # the plans, and the buffers that a program keeps
        from venturi_amd import create_backend, prepare_residual_rms

        backend, kind = create_backend("hip"), case["kind"]

        def empty(*shape, dtype):
            return torch.empty(*shape, dtype=dtype, device=DEVICE)

        if kind == "norm":
            norm = backend.upload_rmsnorm(state["gamma"], dtype=DTYPES[case["dtype"]], device=DEVICE, epsilon=EPSILON)
            state["plan"] = prepare_residual_rms(norm, tokens=case["tokens"], a8_passes=case["a8_passes"])
            state["total"], state["out"] = torch.empty_like(state["x"]), torch.empty_like(state["x"])
            state["workspace"] = None
            if case["a8_passes"]:
                workspace = empty(state["plan"].workspace_bytes, dtype=torch.uint8)
                state["workspace"] = workspace
                shape = (case["a8_passes"], case["tokens"], (case["hidden"] + GROUP - 1) // GROUP)
                codes = math.prod(shape) * GROUP
                state["codes"] = workspace[:codes].view(torch.int8).view(*shape, GROUP)
                state["scales"] = workspace[codes:].view(torch.float32).view(*shape, 1)
        elif kind == "route":
            state["plan"] = backend.prepare_routing(
                tokens=case["tokens"], experts=case["experts"], top_k=case["top_k"], dtype=DTYPES[case["dtype"]], device=DEVICE,
                score=case["score"], groups=case["groups"], kept_groups=case["kept_groups"], scale=case["scale"])
            state["indices"] = empty(case["tokens"], case["top_k"], dtype=torch.int64)
            state["scores"] = empty(case["tokens"], case["top_k"], dtype=torch.float16)
        elif kind == "distribution":
            state["plan"] = backend.prepare_distribution(rows=case["rows"], vocab=case["vocab"], dtype=DTYPES[case["dtype"]],
                                                         device=DEVICE)
            state["workspace"] = empty(state["plan"].workspace_bytes, dtype=torch.uint8)
            state["probabilities"] = empty(case["rows"], case["vocab"], dtype=torch.float32)
        else:
            n, d = case["sequences"], case["drafts"]
            state["plan"] = backend.prepare_verification(sequences=n, drafts=d, vocab=case["vocab"], device=DEVICE)
            state["workspace"] = empty(state["plan"].workspace_bytes, dtype=torch.uint8)
            state["tokens"], state["accepted"] = empty(n, d + 1, dtype=torch.int64), empty(n, dtype=torch.int32)
    return state


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    kind = state["case"]["kind"]
    if not own:
        return {"norm": _norm, "route": _route, "distribution": _distribution, "verify": _verify}[kind](state)
    plan = state["plan"]
    if kind == "norm":
        plan.run(state["x"], state["residual"], total=state["total"], out=state["out"], workspace=state["workspace"])
        got = {"total": state["total"], "out": state["out"]}
        if state["workspace"] is not None:  # the values that the codes stand for, summed over the passes
            values = (state["codes"] * state["scales"]).sum(0).flatten(1)
            got["values"] = values[:, : state["case"]["hidden"]].to(state["x"].dtype)
        return got
    if kind == "route":
        plan.run(state["logits"], state["bias"], indices=state["indices"], scores=state["scores"])
        return {"indices": state["indices"], "scores": state["scores"]}
    if kind == "distribution":
        return plan.run(state["logits"], state["temperature"], state["top_k"], state["top_p"], state["min_p"],
                        probabilities=state["probabilities"], workspace=state["workspace"])
    plan.run(state["target"], state["drafted"], state["uniforms"], proposal=state["proposal"], counts=state["counts"],
             tokens=state["tokens"], accepted=state["accepted"], workspace=state["workspace"])
    return {"tokens": state["tokens"], "accepted": state["accepted"]}


def _norm(state):
    case, x, dtype = state["case"], state["x"], state["x"].dtype
    total = (x.float() + state["residual"].float()).to(dtype)
    h = total.float()
    out = (h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPSILON) * state["gamma"]).to(dtype)
    got = {"total": total, "out": out}
    if case["a8_passes"]:
        hidden = case["hidden"]
        left = torch.nn.functional.pad(out.float(), (0, -hidden % GROUP)).unflatten(-1, (-1, GROUP))
        first, values = _quantized(left)
        if case["a8_passes"] == 2:
            values = values + _quantized(first)[1]
        got["values"] = values.flatten(1)[:, :hidden].to(dtype)
    return got


def _quantized(x):
    """What is left of groups of columns after their int8 codes, and what the codes stand for."""
    most = x.abs().amax(-1, keepdim=True)
    inverse = torch.where(most > 0, 127 / most, torch.zeros_like(most))
    values = torch.round(x * inverse).clamp(-127, 127) * (most / 127)
    return x - values, values


def _route(state):
    case = state["case"]
    x, k, groups = state["logits"].double(), case["top_k"], case["groups"]
    if case["score"] == "softmax":
        e = torch.exp(x - x.amax(-1, keepdim=True))
        s = e / e.sum(-1, keepdim=True)
    else:
        s = 1 / (1 + torch.exp(-x))
    choice = s if state["bias"] is None else s + state["bias"].double()
    if groups > 1:
        parts = choice.unflatten(-1, (groups, -1))
        rank = parts.sort(dim=-1, descending=True).values[..., :2].sum(-1)
        best = rank.sort(dim=-1, descending=True, stable=True).indices[:, : case["kept_groups"]]
        kept = torch.zeros_like(rank, dtype=torch.bool).scatter(1, best, True)
        choice = torch.where(kept[..., None], parts, -torch.inf).flatten(1)
    indices = choice.sort(dim=-1, descending=True, stable=True).indices[:, :k]
    w = s.gather(1, indices)
    return {"indices": indices, "scores": (w / w.sum(-1, keepdim=True) * case["scale"]).half()}


def _distribution(state):
    x, order = state["logits"].double().sort(dim=-1, descending=True, stable=True)
    temperature, top_p, min_p = (state[name].double()[:, None] for name in ("temperature", "top_p", "min_p"))
    rank = torch.arange(x.shape[1], device=DEVICE)[None]
    greedy = temperature <= 0
    weights = torch.exp((x - x[:, :1]) / torch.where(greedy, torch.ones_like(temperature), temperature))
    limit = state["top_k"].long()[:, None]
    limit = torch.where(greedy, 1, torch.where(limit > 0, limit, x.shape[1]))
    weights = torch.where(rank < limit, weights, 0.0)
    before = weights.cumsum(-1) - weights
    kept = ((before < top_p * weights.sum(-1, keepdim=True)) | (top_p >= 1)) & (weights >= min_p)
    weights = torch.where(kept | (rank == 0), weights, 0.0)
    weights = weights / weights.sum(-1, keepdim=True)
    return torch.zeros_like(weights).scatter(1, order, weights).float()


def _verify(state):
    case = state["case"]
    n, d, v = case["sequences"], case["drafts"], case["vocab"]
    p, drafted, u = state["target"].view(n, d + 1, v), state["drafted"], state["uniforms"].double()
    q, counts = state["proposal"], state["counts"].long()
    at, rows = drafted[..., None], torch.arange(n, device=DEVICE)
    chance = p[:, :d].gather(2, at)[..., 0].double()
    offered = torch.ones_like(chance) if q is None else q.view(n, d, v).gather(2, at)[..., 0].double()
    fine = (u[:, :d] * offered < chance) & (torch.arange(d, device=DEVICE)[None] < counts[:, None])
    accepted = fine.long().cumprod(1).sum(1)
    refused, last = (accepted < counts)[:, None], accepted.clamp(max=d - 1)
    whole = p[rows, accepted].double()
    if q is None:
        rest = whole.scatter(1, drafted[rows, last][:, None], 0.0)
    else:
        rest = (whole - q.view(n, d, v)[rows, last].double()).clamp(min=0)
    rest = torch.where(refused & (rest.sum(-1, keepdim=True) > 0), rest, whole)
    mass = rest.cumsum(-1)
    token = (mass <= u[:, d:] * mass[:, -1:]).sum(-1)
    end = torch.where(rest > 0, torch.arange(v, device=DEVICE)[None], 0).amax(-1)
    token = torch.minimum(token, end)[:, None]
    place = torch.arange(d + 1, device=DEVICE)[None]
    padded = torch.nn.functional.pad(drafted, (0, 1))
    tokens = torch.where(place < accepted[:, None], padded, torch.where(place == accepted[:, None], token, -1))
    return {"tokens": tokens, "accepted": accepted.int()}


def work(case):
    kind = case["kind"]
    if kind == "norm":
        count = case["tokens"] * case["hidden"]
        return {"bytes": 8 * count + 4 * case["hidden"] + case["a8_passes"] * count * 36 / 32, "flops": 6 * count}
    if kind == "route":
        size = {"fp16": 2, "bf16": 2, "fp32": 4}[case["dtype"]]
        count = case["tokens"] * case["experts"]
        return {"bytes": size * count + 10 * case["tokens"] * case["top_k"], "flops": 4 * count}
    if kind == "distribution":
        count = case["rows"] * case["vocab"]
        return {"bytes": 6 * count, "flops": 4 * count}
    # The row that the last token comes from, and the drafter's where a draft was refused.
    count = case["sequences"] * case["vocab"] * (1 if case["certain"] else 2)
    return {"bytes": 4 * count + 32 * case["sequences"] * (case["drafts"] + 1), "flops": 2 * count}


# ---------------------------------------------------------------------------
# The same from the definitions, in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    kind = case["kind"]
    if kind == "verify":  # whole numbers alone
        return None
    state = _inputs(case, seed)
    if kind == "norm":
        return _exact_norm(case, state)
    if kind == "route":
        return _exact_route(case, state)
    return _exact_distribution(state)


def _exact_norm(case, state):
    total = torch.add(state["x"].double(), state["residual"].double())
    h = total.to(state["x"].dtype).double()  # the stream as it is stored
    size = torch.linalg.vector_norm(h, dim=-1, keepdim=True).square() / case["hidden"]
    out = h / (size + EPSILON).sqrt() * state["gamma"].double()
    got = {"total": total, "out": out}
    if case["a8_passes"]:
        parts = []
        for part in out.to(state["x"].dtype).double().split(GROUP, -1):
            values = torch.zeros_like(part)
            for _ in range(case["a8_passes"]):
                left = part - values
                step = left.abs().amax(-1, keepdim=True) / 127
                values = values + torch.where(step > 0, (left / step).round(), 0.0).nan_to_num(0.0) * step
            parts.append(values)
        got["values"] = torch.cat(parts, -1)
    return got


def _exact_route(case, state):
    scores = []
    for x in state["logits"].double().split(512):
        s = torch.softmax(x, -1) if case["score"] == "softmax" else torch.sigmoid(x)
        c = s if state["bias"] is None else s + state["bias"].double()
        at = torch.arange(c.shape[1], device=DEVICE)
        if case["groups"] > 1:
            size = c.shape[1] // case["groups"]
            sums = torch.stack([part.topk(min(2, size), -1).values.sum(-1) for part in c.split(size, -1)], -1)
            g = torch.arange(case["groups"], device=DEVICE)
            ahead = (sums[:, None, :] > sums[..., None]) | ((sums[:, None, :] == sums[..., None]) & (g[None] < g[:, None]))
            c = c.masked_fill((ahead.sum(-1) >= case["kept_groups"]).repeat_interleave(size, -1), -math.inf)
        # An expert's place is the number of experts ahead of it.
        place = ((c[:, None, :] > c[..., None]) | ((c[:, None, :] == c[..., None]) & (at[None] < at[:, None]))).sum(-1)
        chosen = torch.where(place < case["top_k"], s, 0.0)
        ordered = torch.zeros_like(s).scatter(1, place, chosen)[:, : case["top_k"]]
        scores.append(ordered * (case["scale"] / chosen.sum(-1, keepdim=True)))
    return {"indices": None, "scores": torch.cat(scores)}


def _exact_distribution(state):
    host = {name: v.double().cpu().numpy() for name, v in state.items()}
    got = np.zeros(host["logits"].shape)
    for i, x in enumerate(host["logits"]):
        t, k, p, least = (float(host[name][i]) for name in ("temperature", "top_k", "top_p", "min_p"))
        order = np.argsort(-x, kind="stable")
        if t <= 0:
            got[i, order[0]] = 1.0
            continue
        if k > 0:
            order = order[: int(k)]
        w = np.exp((x[order] - x[order[0]]) / t)
        if p < 1:
            cut = int(np.searchsorted(np.cumsum(w), p * w.sum(), side="left")) + 1
            order, w = order[:cut], w[:cut]
        count = max(1, int((w >= least).sum()))
        got[i, order[:count]] = w[:count] / w[:count].sum()
    return torch.as_tensor(got)
