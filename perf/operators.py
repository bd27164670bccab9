"""Performance cases of the operators around the projections: rotary positions with the Q8 cache,
attention over that cache, attention over packed prompts, and sampling from the vocabulary head's logits.

A case is a dict of plain values with a ``kind``:

* ``write``: a layer's QKV rows are rotated and their K and V quantized into cache slots, and those
  slots are read back (what a program does that goes on with a prompt in pieces);
* ``decode``: attention of ``query_tokens`` new tokens of every sequence over its pages;
* ``prompt``: causal attention over packed sequences, each after ``past`` keys of its own;
* ``sample``: one token per row of logits, with per-row temperature, top-k, top-p and min-p.

Head counts: 48 x 128 and 24 x 256 with 4 and 2 KV heads are the splits of the repository's
7168-row QKV and 6144-column o_proj projections; 32 with 8 is a common one.

``own`` False computes the plain form in elementary torch operations; True calls the package.
"""

import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
GROUP = 32


def listed():
    return [
        # One token of one sequence: launch and latency count.
        {"name": "write_step", "kind": "write", "tokens": 1, "q_heads": 48, "kv_heads": 4, "head_dim": 128, "dtype": "fp16",
         "layout": "half", "rotary_dim": 128, "scaling": "none", "first": 1000, "page_tokens": 64},
        # A decode batch, bf16, interleaved layout over a quarter of the head.
        {"name": "write_batch", "kind": "write", "tokens": 61, "q_heads": 24, "kv_heads": 2, "head_dim": 256, "dtype": "bf16",
         "layout": "interleaved", "rotary_dim": 64, "scaling": "none", "first": 20000, "page_tokens": 32},
        # A long prompt, positions past the trained range, frequencies scaled for it.
        {"name": "write_prompt", "kind": "write", "tokens": 8190, "q_heads": 32, "kv_heads": 8, "head_dim": 128,
         "dtype": "fp16", "layout": "half", "rotary_dim": 128, "scaling": "yarn", "first": 100000, "page_tokens": 64},
        # One user, about a thousand tokens in.
        {"name": "decode_one", "kind": "decode", "sequences": 1, "query_tokens": 1, "q_heads": 48, "kv_heads": 4,
         "head_dim": 128, "dtype": "fp16", "shortest": 1021, "longest": 1021, "page_tokens": 64},
        # A serving batch of ragged lengths, from a fresh chat to a long document.
        {"name": "decode_batch", "kind": "decode", "sequences": 64, "query_tokens": 1, "q_heads": 32, "kv_heads": 8,
         "head_dim": 128, "dtype": "fp16", "shortest": 1, "longest": 8190, "page_tokens": 64},
        # Drafted tokens checked together, wide heads.
        {"name": "decode_draft", "kind": "decode", "sequences": 16, "query_tokens": 5, "q_heads": 24, "kv_heads": 2,
         "head_dim": 256, "dtype": "bf16", "shortest": 700, "longest": 4100, "page_tokens": 32},
        # Few sequences with very long histories: the work has to be split over the length.
        {"name": "decode_long", "kind": "decode", "sequences": 4, "query_tokens": 1, "q_heads": 48, "kv_heads": 4,
         "head_dim": 128, "dtype": "bf16", "shortest": 90000, "longest": 131000, "page_tokens": 128},
        # A short chat prompt.
        {"name": "prompt_short", "kind": "prompt", "sequences": 1, "tokens": 77, "past": 0, "q_heads": 48, "kv_heads": 4,
         "head_dim": 128, "dtype": "fp16"},
        # Ragged prompts packed together, some of them continued after cached tokens; wide heads.
        {"name": "prompt_packed", "kind": "prompt", "sequences": 11, "tokens": 4096, "past": 2000, "q_heads": 24,
         "kv_heads": 2, "head_dim": 256, "dtype": "fp16"},
        # One long prompt.
        {"name": "prompt_long", "kind": "prompt", "sequences": 1, "tokens": 8192, "past": 0, "q_heads": 48, "kv_heads": 4,
         "head_dim": 128, "dtype": "bf16"},
        # One user's next token over the vocabulary of the head.
        {"name": "sample_one", "kind": "sample", "rows": 1, "vocab": 248320, "dtype": "fp16", "spread": 2.5},
        # A serving batch with everybody's own settings.
        {"name": "sample_batch", "kind": "sample", "rows": 256, "vocab": 151936, "dtype": "bf16", "spread": 3.0},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["write", "decode", "prompt", "sample"])
    q_heads, kv_heads, head_dim = rng.choice([(48, 4, 128), (24, 2, 256), (32, 8, 128), (32, 4, 64), (16, 16, 128), (20, 4, 96)])
    dtype = rng.choice(["fp16", "bf16"])
    if kind == "write":
        return {"kind": kind, "tokens": _log_int(rng, 1, 6000), "q_heads": q_heads, "kv_heads": kv_heads,
                "head_dim": head_dim, "dtype": dtype, "layout": rng.choice(["half", "interleaved"]),
                "rotary_dim": rng.choice([head_dim, head_dim // 2, 32]),
                "scaling": rng.choice(["none", "linear", "banded", "yarn"]), "first": _log_int(rng, 1, 200000),
                "page_tokens": rng.choice([32, 64, 128])}
    if kind == "decode":
        sequences = _log_int(rng, 1, 64)
        longest = _log_int(rng, 16, 200000 // sequences)
        return {"kind": kind, "sequences": sequences, "query_tokens": rng.choice([1, 1, 1, 2, 4]), "q_heads": q_heads,
                "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "shortest": rng.choice([1, longest // 2, longest]),
                "longest": longest, "page_tokens": rng.choice([32, 64, 128])}
    if kind == "prompt":
        tokens = _log_int(rng, 5, 5000)
        return {"kind": kind, "sequences": min(tokens, rng.choice([1, 1, 3, 9])), "tokens": tokens,
                "past": rng.choice([0, 0, _log_int(rng, 1, 1500)]), "q_heads": q_heads, "kv_heads": kv_heads,
                "head_dim": head_dim, "dtype": dtype}
    return {"kind": kind, "rows": _log_int(rng, 1, 200), "vocab": _log_int(rng, 1000, 160000), "dtype": dtype,
            "spread": rng.choice([1.0, 2.5, 4.0])}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
SCALINGS = {
    "none": None,
    "linear": {"type": "linear", "factor": 4.0},
    "banded": {"type": "banded", "factor": 8.0, "low": 1.0, "high": 4.0, "original_context": 8192},
    "yarn": {"type": "yarn", "factor": 4.0, "original_context": 32768, "beta_fast": 32.0, "beta_slow": 1.0},
}
BASE = 1e6


def _generators(seed):
    """Values on the GPU, plans (lengths, page orders, settings) on the host."""
    return torch.Generator(device=DEVICE).manual_seed(int(seed)), np.random.default_rng(int(seed))


def _lengths(case, rng):
    n = case["sequences"]
    lengths = np.exp(rng.uniform(math.log(case["shortest"]), math.log(case["longest"] + 1), n)).astype(np.int64)
    return np.clip(lengths, case["shortest"], case["longest"])


def _heads(gen, tokens, heads, dim, dtype, outliers):
    """Gaussian rows; keys have a few channels that are larger than the rest, as after real projections."""
    x = torch.randn(tokens, heads, dim, generator=gen, device=DEVICE)
    if outliers:
        x[:, :, ::37] *= 3.0
    return x.to(dtype)


def _inputs(case, seed):
    gen, rng = _generators(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    if kind == "sample":
        rows, vocab = case["rows"], case["vocab"]
        logits = (torch.randn(rows, vocab, generator=gen, device=DEVICE) * case["spread"]).to(dtype)
        settings = {
            "temperature": rng.choice([0.6, 0.8, 1.0, 1.3, 0.0], rows, p=[0.25, 0.25, 0.25, 0.2, 0.05]),
            "top_k": rng.choice([0, 20, 50, 1000], rows), "top_p": rng.choice([1.0, 0.95, 0.8], rows),
            "min_p": rng.choice([0.0, 0.0, 0.05], rows),
        }
        if rows == 1:
            settings = {"temperature": [0.8], "top_k": [50], "top_p": [0.95], "min_p": [0.0]}
        types = {"temperature": torch.float32, "top_k": torch.int32, "top_p": torch.float32, "min_p": torch.float32}
        got = {k: torch.as_tensor(np.asarray(v)).to(types[k]).to(DEVICE) for k, v in settings.items()}
        got["uniforms"] = torch.rand(rows, generator=gen, device=DEVICE)
        got["logits"] = logits
        return got
    hq, hk, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    if kind == "prompt":
        tokens, n = case["tokens"], case["sequences"]
        cuts = np.sort(rng.choice(np.arange(1, tokens), n - 1, replace=False)) if n > 1 else np.zeros(0, np.int64)
        q_offsets = np.concatenate([[0], cuts, [tokens]]).astype(np.int64)
        past = rng.integers(0, case["past"] + 1, n) if case["past"] else np.zeros(n, np.int64)
        k_offsets = np.concatenate([[0], np.cumsum(np.diff(q_offsets) + past)])
        keys = int(k_offsets[-1])
        return {"q": _heads(gen, tokens, hq, d, dtype, False), "k": _heads(gen, keys, hk, d, dtype, True),
                "v": _heads(gen, keys, hk, d, dtype, False),
                "q_offsets": torch.as_tensor(q_offsets, dtype=torch.int32, device=DEVICE),
                "k_offsets": torch.as_tensor(k_offsets, dtype=torch.int32, device=DEVICE)}
    page = case["page_tokens"]
    if kind == "write":
        tokens = case["tokens"]
        pages = (tokens + page - 1) // page + 3
        order = torch.as_tensor(rng.permutation(pages), device=DEVICE)
        at = torch.arange(tokens, device=DEVICE)
        qkv = torch.cat([_heads(gen, tokens, hq, d, dtype, False), _heads(gen, tokens, hk, d, dtype, True),
                         _heads(gen, tokens, hk, d, dtype, False)], 1).reshape(tokens, (hq + 2 * hk) * d)
        return {"qkv": qkv, "positions": case["first"] + at, "slots": order[at // page] * page + at % page, "pages": pages}
    lengths = _lengths(case, rng)
    need = (lengths + page - 1) // page
    pages = int(need.sum()) + 2
    order, table, begin = rng.permutation(pages), np.zeros((len(need), int(need.max())), np.int64), 0
    for b, count in enumerate(need):
        table[b, :count] = order[begin:begin + count]
        begin += count
    return {"q": _heads(gen, len(need) * case["query_tokens"], hq, d, dtype, False),
            "k": _heads(gen, pages * page, hk, d, dtype, True), "v": _heads(gen, pages * page, hk, d, dtype, False),
            "page_table": torch.as_tensor(table, dtype=torch.int32, device=DEVICE),
            "lengths": torch.as_tensor(lengths, dtype=torch.int32, device=DEVICE), "pages": pages}


def _quantize(x):
    """Codes [.., D] and scales [.., ceil(D / 32)] of the q8_g32_fp16 rule."""
    d = x.shape[-1]
    groups = (d + GROUP - 1) // GROUP
    x = torch.nn.functional.pad(x.float(), (0, groups * GROUP - d)).unflatten(-1, (groups, GROUP))
    scales = (x.abs().amax(-1) / 127).half()
    s = scales.float()[..., None]
    codes = torch.where(s > 0, torch.round(x / s), torch.zeros_like(x)).clamp(-127, 127)
    return codes.to(torch.int8).flatten(-2)[..., :d], scales


def _values(codes, scales):
    return codes.float() * scales.float().repeat_interleave(GROUP, -1)[..., : codes.shape[-1]]


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    if kind == "decode" and not own:  # the cached codes that the plain form reads
        state["k"], state["v"] = _quantize(state["k"]), _quantize(state["v"])
    if own:  # the plans, and the cache filled as a program fills it
        from venturi_amd import create_backend

        backend = create_backend("hip")
        where = {"dtype": dtype, "device": DEVICE}
        if kind == "sample":
            rows, vocab = state["logits"].shape
            state["plan"] = backend.prepare_sampling(rows=rows, vocab=vocab, **where)
            state["tokens"] = torch.empty(rows, dtype=torch.int64, device=DEVICE)
            state["probabilities"] = torch.empty(rows, dtype=torch.float32, device=DEVICE)
            return state
        hq, hk, d = case["q_heads"], case["kv_heads"], case["head_dim"]
        if kind == "prompt":
            state["plan"] = backend.prepare_attention(tokens=len(state["q"]), keys=len(state["k"]),
                                                      sequences=case["sequences"], q_heads=hq, kv_heads=hk, head_dim=d, **where)
            state["out"] = torch.empty_like(state["q"])
            return state
        cache = backend.create_kv_cache(pages=state["pages"], page_tokens=case["page_tokens"], kv_heads=hk, head_dim=d, **where)
        if kind == "write":
            from venturi_amd import RotaryEmbedding

            tokens = case["tokens"]
            rotary = RotaryEmbedding(d, rotary_dim=case["rotary_dim"], layout=case["layout"], base=BASE,
                                     scaling=SCALINGS[case["scaling"]])
            state["plan"] = cache.prepare_write(tokens=tokens, q_heads=hq, rotary=rotary)
            state["reader"] = cache.prepare_read(tokens=tokens)
            state["q"] = torch.empty(tokens, hq, d, **where)
            state["k"], state["keys"], state["values"] = (torch.empty(tokens, hk, d, **where) for _ in range(3))
            return state
        slots = torch.arange(len(state["k"]), device=DEVICE)
        rows = torch.cat([state.pop("k").flatten(1), state.pop("v").flatten(1)], 1)
        cache.prepare_write(tokens=len(slots), q_heads=0, rotary=None).run(rows, slots, slots)
        state["plan"] = cache.prepare_attention(sequences=case["sequences"], q_heads=hq, query_tokens=case["query_tokens"],
                                                max_pages=state["page_table"].shape[1])
        state["workspace"] = torch.empty(state["plan"].workspace_bytes, dtype=torch.uint8, device=DEVICE)
        state["out"] = torch.empty_like(state["q"])
    return state


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    kind = state["case"]["kind"]
    if own:
        if kind == "write":
            state["plan"].run(state["qkv"], state["positions"], state["slots"], q=state["q"], k=state["k"])
            state["reader"].run(state["slots"], keys=state["keys"], values=state["values"])
            return {name: state[name] for name in ("q", "k", "keys", "values")}
        if kind == "decode":
            return state["plan"].run(state["q"], state["page_table"], state["lengths"], out=state["out"],
                                     workspace=state["workspace"])
        if kind == "prompt":
            return state["plan"].run(state["q"], state["k"], state["v"], state["q_offsets"], state["k_offsets"],
                                     out=state["out"])
        state["plan"].run(state["logits"], state["uniforms"], state["temperature"], state["top_k"], state["top_p"],
                          state["min_p"], tokens=state["tokens"], probabilities=state["probabilities"])
        return {"tokens": state["tokens"], "probabilities": state["probabilities"]}
    return {"write": _write, "decode": _decode, "prompt": _prompt, "sample": _sample}[kind](state)


def _frequencies(rotary_dim, scaling):
    """Radians per position of every rotated pair (64 bits), and the factor on cos and sin."""
    f = BASE ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=DEVICE) / rotary_dim)
    if scaling is None:
        return f, 1.0
    s = scaling["factor"]
    if scaling["type"] == "linear":
        return f / s, 1.0
    turns = scaling["original_context"] * f / (2 * math.pi)
    if scaling["type"] == "banded":
        keep = ((turns - scaling["low"]) / (scaling["high"] - scaling["low"])).clamp(0, 1)
        return f * (keep + (1 - keep) / s), 1.0

    def pair(beta):
        return rotary_dim * math.log(scaling["original_context"] / (beta * 2 * math.pi)) / (2 * math.log(BASE))

    low = max(math.floor(pair(scaling["beta_fast"])), 0)
    high = min(math.ceil(pair(scaling["beta_slow"])), rotary_dim - 1)
    index = torch.arange(rotary_dim // 2, dtype=torch.float64, device=DEVICE)
    keep = 1 - ((index - low) / max(high - low, 0.001)).clamp(0, 1)
    return f * (keep + (1 - keep) / s), 0.1 * math.log(s) + 1


def _write(state):
    case = state["case"]
    hq, hk, d, r = case["q_heads"], case["kv_heads"], case["head_dim"], case["rotary_dim"]
    dtype = state["qkv"].dtype
    x = state["qkv"].float().view(-1, hq + 2 * hk, d)
    f, factor = _frequencies(r, SCALINGS[case["scaling"]])
    angle = state["positions"].double()[:, None] * f
    cos, sin = ((factor * t).float()[:, None, :] for t in (torch.cos(angle), torch.sin(angle)))
    rows, v = x[:, : hq + hk], x[:, hq + hk:].to(dtype)
    half = case["layout"] == "half"
    x0, x1 = (rows[..., : r // 2], rows[..., r // 2: r]) if half else (rows[..., 0:r:2], rows[..., 1:r:2])
    y0, y1 = x0 * cos - x1 * sin, x1 * cos + x0 * sin
    turned = torch.cat([y0, y1], -1) if half else torch.stack([y0, y1], -1).flatten(-2)
    rows = torch.cat([turned, rows[..., r:]], -1).to(dtype)
    k = rows[:, hq:]
    return {"q": rows[:, :hq], "k": k, "keys": _values(*_quantize(k)).to(dtype), "values": _values(*_quantize(v)).to(dtype)}


def _decode(state):
    case = state["case"]
    n, t, page = case["sequences"], case["query_tokens"], case["page_tokens"]
    hq, hk, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    lengths, table = state["lengths"].long(), state["page_table"].long()
    at = torch.arange(table.shape[1] * page, device=DEVICE)
    slots = table[:, at // page] * page + at % page
    k, v = (_values(c[slots], s[slots]).permute(0, 2, 1, 3) for c, s in (state["k"], state["v"]))  # [n, hk, keys, d]
    q = state["q"].float().view(n, t, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(n, hk, hq // hk * t, d)
    scores = torch.matmul(q, k.transpose(-1, -2)).view(n, hk, hq // hk, t, -1) / math.sqrt(d)
    seen = at[None, None] < lengths[:, None, None] - (t - 1 - torch.arange(t, device=DEVICE))[None, :, None]
    out = _weights(scores, seen[:, None, None]).view(n, hk, hq // hk * t, -1).matmul(v)
    return out.view(n, hk, hq // hk, t, d).permute(0, 3, 1, 2, 4).reshape(n * t, hq, d).to(state["q"].dtype)


def _weights(scores, seen):
    """Softmax over the seen keys in the scores' own memory; rows that see none are zero."""
    scores.masked_fill_(~seen, -torch.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top == -torch.inf, torch.zeros_like(top), top)).exp_()
    total = scores.sum(-1, keepdim=True)
    return scores.div_(torch.where(total > 0, total, torch.ones_like(total)))


def _prompt(state):
    case = state["case"]
    hq, hk, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    qo, ko = state["q_offsets"].long(), state["k_offsets"].long()
    at_q, at_k = torch.arange(len(state["q"]), device=DEVICE), torch.arange(len(state["k"]), device=DEVICE)
    seq_q, seq_k = torch.searchsorted(qo, at_q, right=True) - 1, torch.searchsorted(ko, at_k, right=True) - 1
    # A query's place counted from the end of its sequence is its key's place.
    seen = (seq_q[:, None] == seq_k[None]) & ((ko[seq_k + 1] - at_k)[None] >= (qo[seq_q + 1] - at_q)[:, None])
    q = state["q"].float().view(-1, hk, hq // hk, d).permute(1, 2, 0, 3).reshape(hk, -1, d)
    k, v = (state[name].float().permute(1, 0, 2).contiguous() for name in ("k", "v"))
    scores = torch.bmm(q, k.transpose(1, 2).contiguous()).div_(math.sqrt(d)).view(hk, hq // hk, len(at_q), len(at_k))
    out = torch.bmm(_weights(scores, seen).view(hk, -1, len(at_k)), v)
    return out.view(hk, hq // hk, -1, d).permute(2, 0, 1, 3).reshape(-1, hq, d).to(state["q"].dtype)


def _sample(state):
    x, order = state["logits"].double().sort(dim=-1, descending=True, stable=True)
    temperature, top_p, min_p, u = (state[name].double()[:, None] for name in ("temperature", "top_p", "min_p", "uniforms"))
    rank = torch.arange(x.shape[1], device=DEVICE)[None]
    greedy = temperature <= 0
    weights = torch.exp((x - x[:, :1]) / torch.where(greedy, torch.ones_like(temperature), temperature))
    limit = state["top_k"].long()[:, None]
    limit = torch.where(greedy, 1, torch.where(limit > 0, limit, x.shape[1]))
    weights = torch.where(rank < limit, weights, 0.0)
    before = weights.cumsum(-1) - weights
    kept = (rank < limit) & ((before < top_p * weights.sum(-1, keepdim=True)) | (top_p >= 1)) & (weights >= min_p)
    weights = torch.where(kept | (rank == 0), weights, 0.0)
    total = weights.cumsum(-1)
    place = (total <= u * total[:, -1:]).sum(-1, keepdim=True)
    place = torch.minimum(place, (weights > 0).sum(-1, keepdim=True) - 1)
    return {"tokens": order.gather(1, place)[:, 0], "probabilities": (weights.gather(1, place) / total[:, -1:])[:, 0].float()}


def work(case):
    kind = case["kind"]
    if kind == "sample":
        count = case["rows"] * case["vocab"]
        return {"bytes": 2 * count + 32 * case["rows"], "flops": 4 * count}
    hq, hk, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    cached = 2 * hk * (d + 2 * ((d + GROUP - 1) // GROUP))  # bytes of a token's K and V in the cache
    if kind == "write":
        rows = 2 * (hq + 2 * hk) * d + 2 * (hq + hk) * d + 16 + 2 * cached + 4 * hk * d
        return {"bytes": case["tokens"] * rows, "flops": case["tokens"] * (3 * (hq + hk) * case["rotary_dim"] + 8 * hk * d)}
    if kind == "decode":
        t, n = case["query_tokens"], case["sequences"]
        low, high = case["shortest"], case["longest"]  # the mean of lengths that are even over their logarithm
        total = n * (high if low == high else (high - low) / math.log(high / low))
        return {"bytes": total * cached + 4 * n * t * hq * d, "flops": 4 * total * t * hq * d}
    tokens, n, past = case["tokens"], case["sequences"], case["past"]
    pairs = tokens * (past / 2) + tokens * tokens / (n + 1 if n > 1 else 2)
    return {"bytes": 4 * tokens * hq * d + 4 * (tokens + n * past / 2) * hk * d, "flops": 4 * pairs * hq * d}


# ---------------------------------------------------------------------------
# The same from the definitions, in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    state = _inputs(case, seed)
    kind = case["kind"]
    if kind == "sample":
        return _exact_sample(state)
    hq, hk, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    if kind == "prompt":
        out = torch.zeros(len(state["q"]), hq, d, dtype=torch.float64, device=DEVICE)
        qo, ko = state["q_offsets"].tolist(), state["k_offsets"].tolist()
        for b in range(case["sequences"]):
            q, k, v = state["q"][qo[b]:qo[b + 1]], state["k"][ko[b]:ko[b + 1]], state["v"][ko[b]:ko[b + 1]]
            out[qo[b]:qo[b + 1]] = _exact_attention(q, k.double(), v.double())
        return out
    if kind == "decode":
        t, page = case["query_tokens"], case["page_tokens"]
        out = []
        for b, length in enumerate(state["lengths"].tolist()):
            at = torch.arange(length, device=DEVICE)
            slots = state["page_table"][b].long()[at // page] * page + at % page
            out.append(_exact_attention(state["q"][b * t:(b + 1) * t], _exact_cached(state["k"][slots]), _exact_cached(state["v"][slots])))
        return torch.cat(out)
    return _exact_write(case, state)


def _exact_attention(q, k, v):
    """[t, hq, d] over [n, hk, d] in 64 bits; query i of t sees the first n - (t - 1 - i) keys."""
    t, hq, d = q.shape
    n, hk = k.shape[:2]
    q = q.double()
    out = torch.zeros(t, hq, d, dtype=torch.float64, device=q.device)
    hidden = torch.ones(t, n, dtype=torch.bool, device=q.device).triu(n - t + 1)
    for h in range(hq):
        scores = (q[:, h] @ k[:, h * hk // hq].T) * d ** -0.5
        weights = torch.softmax(scores.masked_fill(hidden, -torch.inf), -1).nan_to_num(0.0)
        out[:, h] = weights @ v[:, h * hk // hq]
    return out


def _exact_cached(x):
    """What the cache holds of rows [n, heads, d]: by 32 columns, integers of at most 127 times an fp16 scale."""
    parts = []
    for part in x.double().split(GROUP, -1):
        scale = (part.abs().amax(-1, keepdim=True).float() / 127).half().double()
        parts.append(torch.where(scale > 0, (part / scale).round().clamp(-127, 127), 0.0) * scale)
    return torch.cat(parts, -1)


def _exact_write(case, state):
    hq, hk, d, r = case["q_heads"], case["kv_heads"], case["head_dim"], case["rotary_dim"]
    scaling, dtype = SCALINGS[case["scaling"]], state["qkv"].dtype
    rates, factor = [], 1.0
    for i in range(r // 2):
        f = BASE ** (-2 * i / r)
        if scaling is not None:
            s = scaling["factor"]
            if scaling["type"] == "linear":
                share = 0.0
            elif scaling["type"] == "banded":
                turns = scaling["original_context"] * f / (2 * math.pi)
                share = min(max((turns - scaling["low"]) / (scaling["high"] - scaling["low"]), 0.0), 1.0)
            else:
                ends = [r * math.log(scaling["original_context"] / (scaling[b] * 2 * math.pi)) / (2 * math.log(BASE))
                        for b in ("beta_fast", "beta_slow")]
                low, high = max(math.floor(ends[0]), 0), min(math.ceil(ends[1]), r - 1)
                share = 1 - min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
                factor = 0.1 * math.log(s) + 1
            f = share * f + (1 - share) * f / s
        rates.append(f)
    angle = torch.outer(state["positions"].double(), torch.tensor(rates, dtype=torch.float64, device=DEVICE))[:, None]
    turn = factor * torch.polar(torch.ones_like(angle), angle)
    rows = state["qkv"].double().view(-1, hq + 2 * hk, d)
    pairs = rows[:, : hq + hk, :r]
    if case["layout"] == "half":
        z = torch.complex(pairs[..., : r // 2].contiguous(), pairs[..., r // 2:].contiguous()) * turn
        turned = torch.cat([z.real, z.imag], -1)
    else:
        turned = torch.view_as_real(torch.view_as_complex(pairs.unflatten(-1, (-1, 2)).contiguous()) * turn).flatten(-2)
    turned = torch.cat([turned, rows[:, : hq + hk, r:]], -1)
    k = turned[:, hq:]
    return {"q": turned[:, :hq], "k": k, "keys": _exact_cached(k.to(dtype)), "values": _exact_cached(rows[:, hq + hk:])}


def _exact_sample(state):
    tokens, chances = [], []
    host = {name: v.double().cpu().numpy() for name, v in state.items()}
    for i, x in enumerate(host["logits"]):
        t, k, p, least, u = (float(host[name][i]) for name in ("temperature", "top_k", "top_p", "min_p", "uniforms"))
        order = np.argsort(-x, kind="stable")
        if t <= 0:
            tokens.append(int(order[0]))
            chances.append(1.0)
            continue
        if k > 0:
            order = order[: int(k)]
        w = np.exp((x[order] - x[order[0]]) / t)
        if p < 1:
            cut = int(np.searchsorted(np.cumsum(w), p * w.sum(), side="left")) + 1
            order, w = order[:cut], w[:cut]
        w = w[: max(1, int((w >= least).sum()))]
        total = np.cumsum(w)
        place = min(int(np.searchsorted(total, u * total[-1], side="right")), len(w) - 1)
        tokens.append(int(order[place]))
        chances.append(float(w[place] / total[-1]))
    return {"tokens": torch.tensor(tokens), "probabilities": torch.tensor(chances, dtype=torch.float64)}
