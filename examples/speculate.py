"""Generates tokens by speculation through one mixture-of-experts decoder layer.

The layer of generate.py with routed Q4 experts behind its attention: the residual's additions and norms in one launch each, a
router's logits turned into the experts' ids and scores. A drafter that looks at the last token alone (its embedding, the
norm and the head) proposes tokens; the layer runs over all drafts of every sequence at once, and the drafts that stand, with
the token after them, come from both models' distributions.

    python examples/speculate.py [--steps N] [--drafts D]
"""

import argparse

import torch

from generate import DTYPE, Layer
from venturi_amd import prepare_residual_rms
from venturi_amd.moe import MoEGeometry, Q4ExpertBank
from venturi_amd.q4 import quantize_q4_rtn


class ExpertLayer(Layer):
    def __init__(self, device, *, experts=16, top_k=4, inter=128, seed=0, **more):
        super().__init__(device, seed=seed, **more)
        gen = torch.Generator().manual_seed(seed + 1)
        self.geometry = MoEGeometry(hidden_size=self.hidden, num_experts=experts, top_k=top_k, intermediate_size=inter)

        def weight(rows, columns):
            return torch.randn(rows, columns, generator=gen) * columns**-0.5

        # What attention and experts add is small beside the embedding, so that the drafter is right now and then.
        small = self.hidden**-0.5
        self.o_proj = self.linear(small * weight(self.hidden, self.q_heads * self.head_dim))
        bank = [(quantize_q4_rtn(weight(2 * inter, self.hidden)), quantize_q4_rtn(small * weight(self.hidden, inter))) for _ in range(experts)]
        self.bank = Q4ExpertBank.upload(self.backend, self.geometry, bank, device=device)
        self.router = self.linear(weight(experts, self.hidden))
        self.bias = (0.05 * torch.randn(experts, generator=gen)).to(device)

    def linear(self, weight):
        return self.backend.upload_linear(self.backend.quantize_q8(weight.to(self.device)), dtype=DTYPE, device=self.device)

    def add_and_norm(self, x, residual):
        total, normed = torch.empty_like(x), torch.empty_like(x)
        prepare_residual_rms(self.norm, tokens=len(x)).run(x, residual, total=total, out=normed)
        return total, normed

    def output(self, x, attended):
        """Logits of the rows after o_proj, the experts and their residuals."""
        n, g = len(x), self.geometry
        out = self.o_proj.prepare(tokens=n).run(attended.view(n, -1), out=self.tensor(n, self.hidden))
        x, normed = self.add_and_norm(out, x)
        logits = self.router.prepare(tokens=n).run(normed, out=self.tensor(n, g.num_experts))
        routing = self.backend.prepare_routing(tokens=n, experts=g.num_experts, top_k=g.top_k, dtype=DTYPE, device=self.device,
                                               score="sigmoid", groups=4, kept_groups=2)
        ids, scores = routing.run(logits, self.bias, indices=self.tensor(n, g.top_k, dtype=torch.int64), scores=self.tensor(n, g.top_k))
        plan = self.bank.prepare(tokens=n)
        out = plan.run(normed, ids, scores, out=self.tensor(n, self.hidden), workspace=self.tensor(plan.workspace_bytes, dtype=torch.uint8))
        _, normed = self.add_and_norm(out, x)
        return self.head.prepare(tokens=n).run(normed, out=self.tensor(n, self.vocab))

    def decode_drafts(self, ids, lengths):
        """Logits [n * t, vocab] after each of the next t tokens (ids [n][t]) of every sequence, over the cache."""
        n, t = len(ids), len(ids[0])
        positions = [p + i for p in lengths for i in range(t)]
        slots = [s for b, p in enumerate(lengths) for s in self.slots(b, n, range(p, p + t))]
        x, qkv = self.project([i for row in ids for i in row])
        q, _, _ = self.write(qkv, positions, slots)
        width = (max(lengths) + t - 1) // self.page_tokens + 1
        plan = self.cache.prepare_attention(sequences=n, q_heads=self.q_heads, query_tokens=t, max_pages=width)
        table = self.integers([[b + n * i for i in range(width)] for b in range(n)], torch.int32)
        attended = plan.run(q, table, self.integers([p + t for p in lengths], torch.int32), out=torch.empty_like(q),
                            workspace=self.tensor(plan.workspace_bytes, dtype=torch.uint8))
        return self.output(x, attended)

    def drafter_logits(self, ids):
        x, _ = self.project(ids)
        normed = self.norm.prepare(tokens=len(ids)).run(x, out=torch.empty_like(x))
        return self.head.prepare(tokens=len(ids)).run(normed, out=self.tensor(len(ids), self.vocab))

    def distribution(self, logits, settings):
        plan = self.backend.prepare_distribution(rows=len(logits), vocab=self.vocab, dtype=DTYPE, device=self.device)
        return plan.run(logits, **settings, probabilities=self.tensor(*logits.shape, dtype=torch.float32),
                        workspace=self.tensor(plan.workspace_bytes, dtype=torch.uint8))

    def verify(self, target, drafted, uniforms, proposal):
        n, d = drafted.shape
        plan = self.backend.prepare_verification(sequences=n, drafts=d, vocab=self.vocab, device=self.device)
        tokens, accepted = self.tensor(n, d + 1, dtype=torch.int64), self.tensor(n, dtype=torch.int32)
        plan.run(target, drafted, uniforms, proposal=proposal, tokens=tokens, accepted=accepted,
                 workspace=self.tensor(plan.workspace_bytes, dtype=torch.uint8))
        return tokens, accepted


def speculate(layer, prompts, steps, drafts, *, seed=0, watch=None, **values):
    """`steps` passes of `drafts` drafts each; every sequence's new tokens. `watch` gets each pass's rows and verdicts."""
    n = len(prompts)
    gen = torch.Generator().manual_seed(seed)
    types = {"temperature": torch.float32, "top_k": torch.int32, "top_p": torch.float32, "min_p": torch.float32}

    def settings(rows):
        return {name: torch.full((rows,), value, dtype=types[name], device=layer.device) for name, value in values.items()}

    def uniforms(*shape):
        return torch.rand(*shape, generator=gen).to(layer.device)

    if len(prompts) and max(len(p) for p in prompts) > 1:
        layer.prompts([p[:-1] for p in prompts], [0] * n)
    lengths, last, emitted = [len(p) - 1 for p in prompts], [p[-1] for p in prompts], [[] for _ in prompts]
    for _ in range(steps):
        ids, rows = [[i] for i in last], []
        for _ in range(drafts):  # the drafter's own tokens, one after the other
            logits = layer.drafter_logits([row[-1] for row in ids])
            rows.append(layer.distribution(logits, settings(n)))
            for row, i in zip(ids, layer.sample(logits, uniforms(n), **settings(n))):
                row.append(i)
        drafted = layer.integers([row[1:] for row in ids])
        proposal = torch.stack(rows, 1).view(n * drafts, layer.vocab)
        logits = layer.decode_drafts(ids, lengths)
        target = layer.distribution(logits, settings(n * (drafts + 1)))
        u = uniforms(n, drafts + 1)
        tokens, accepted = layer.verify(target, drafted, u, proposal)
        if watch is not None:
            watch(logits, target, proposal, drafted, u, tokens, accepted)
        # Cached rows of refused drafts lie past the new length; the next pass writes over them.
        for own, row, count, at in zip(emitted, tokens.tolist(), accepted.tolist(), range(n)):
            own.extend(row[: count + 1])
            lengths[at] += count + 1
            last[at] = row[count]
    return emitted


if __name__ == "__main__":
    parser = argparse.ArgumentParser()
    parser.add_argument("--steps", type=int, default=8)
    parser.add_argument("--drafts", type=int, default=3)
    options = parser.parse_args()
    prompts = [list(range(3, 40)), list(range(500, 511)), list(range(100, 162))]
    room = 64 + options.steps * (options.drafts + 1)
    tokens = speculate(ExpertLayer("cuda:0", pages=room), prompts, options.steps, options.drafts, temperature=4.0, top_k=50, top_p=0.95)
    for prompt, own in zip(prompts, tokens):
        print(f"{len(prompt)} prompt tokens -> {own}", flush=True)
