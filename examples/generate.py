"""Generates tokens with one decoder layer, from the projections to the sampled token.

A random-weight layer (norm, Q8 QKV, rotary positions, attention, Q8 o_proj, residual) under a Q8 embedding and
vocabulary head. The prompts of a batch are packed: their first parts go through packed attention and into the Q8 cache,
their second parts through packed attention over the read-back keys and their own; then every step decodes one token per
sequence over the cache and samples it.

    python examples/generate.py [--steps N]
"""

import argparse
from pathlib import Path
import sys

import torch

ROOT = Path(__file__).resolve().parent.parent
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

from venturi_amd import Q8RowSplitWeight, RotaryEmbedding, create_backend  # noqa: E402

DTYPE = torch.float16


class Layer:
    def __init__(self, device, *, hidden=512, q_heads=8, kv_heads=2, head_dim=64, vocab=1000, pages=32, page_tokens=16, seed=0):
        self.backend, self.device = create_backend("hip"), torch.device(device)
        self.hidden, self.q_heads, self.kv_heads, self.head_dim, self.vocab = hidden, q_heads, kv_heads, head_dim, vocab
        gen = torch.Generator().manual_seed(seed)

        def linear(rows, columns):
            weight = Q8RowSplitWeight.from_dense(torch.randn(rows, columns, generator=gen) * columns**-0.5)
            return self.backend.upload_linear(weight, dtype=DTYPE, device=device)

        self.qkv = linear((q_heads + 2 * kv_heads) * head_dim, hidden)
        self.o_proj = linear(hidden, q_heads * head_dim)
        self.head = linear(vocab, hidden)  # also the embedding
        self.norm = self.backend.upload_rmsnorm(torch.ones(hidden), dtype=DTYPE, device=device, epsilon=1e-6)
        self.rotary = RotaryEmbedding(head_dim, base=1e4, scaling={"type": "linear", "factor": 2.0})
        self.cache = self.backend.create_kv_cache(pages=pages, page_tokens=page_tokens, kv_heads=kv_heads, head_dim=head_dim,
                                                  dtype=DTYPE, device=device)
        # Sequence b owns the pages b, b + n, b + 2n, ..: neighbours in a sequence are not neighbours in the cache.
        self.page_tokens, self.pages = page_tokens, pages

    def tensor(self, *shape, dtype=DTYPE):
        return torch.empty(*shape, dtype=dtype, device=self.device)

    def integers(self, values, dtype=torch.int64):
        return torch.tensor(values, dtype=dtype, device=self.device)

    def slots(self, sequence, sequences, positions):
        return [(sequence + p // self.page_tokens * sequences) * self.page_tokens + p % self.page_tokens for p in positions]

    def project(self, ids):
        """The tokens' residual rows and their QKV rows."""
        n = len(ids)
        x, normed = self.tensor(n, self.hidden), self.tensor(n, self.hidden)
        self.head.prepare_embedding(ids).run(out=x)
        self.norm.prepare(tokens=n).run(x, out=normed)
        return x, self.qkv.prepare(tokens=n).run(normed, out=self.tensor(n, self.qkv.out_features))

    def write(self, qkv, positions, slots):
        n = len(positions)
        q, k = self.tensor(n, self.q_heads, self.head_dim), self.tensor(n, self.kv_heads, self.head_dim)
        plan = self.cache.prepare_write(tokens=n, q_heads=self.q_heads, rotary=self.rotary)
        plan.run(qkv, self.integers(positions), self.integers(slots), q=q, k=k)
        return q, k, qkv[:, -self.kv_heads * self.head_dim:].contiguous().view(n, self.kv_heads, self.head_dim)

    def output(self, x, attended):
        """Logits of the rows after o_proj, the residual and the norm."""
        n = len(x)
        out, normed = self.tensor(n, self.hidden), self.tensor(n, self.hidden)
        self.o_proj.prepare(tokens=n).run(attended.view(n, -1), out=out)
        self.backend.prepare_add(tokens=n, features=self.hidden, dtype=DTYPE, device=self.device).run(x, out, out=out)
        self.norm.prepare(tokens=n).run(out, out=normed)
        return self.head.prepare(tokens=n).run(normed, out=self.tensor(n, self.vocab))

    def prompts(self, parts, past):
        """One packed pass over the next part of every prompt, after `past` cached tokens of each; the last rows' logits."""
        n = len(parts)
        ids = [i for part in parts for i in part]
        positions = [p + i for part, p in zip(parts, past) for i in range(len(part))]
        slots = [s for b, (part, p) in enumerate(zip(parts, past)) for s in self.slots(b, n, range(p, p + len(part)))]
        x, qkv = self.project(ids)
        q, k, v = self.write(qkv, positions, slots)
        if any(past):  # the cached keys and values in front of the new ones, sequence by sequence
            cached = [s for b, p in enumerate(past) for s in self.slots(b, n, range(p))]
            old_k, old_v = self.tensor(len(cached), *k.shape[1:]), self.tensor(len(cached), *k.shape[1:])
            self.cache.prepare_read(tokens=len(cached)).run(self.integers(cached), keys=old_k, values=old_v)
            sizes = [len(part) for part in parts]
            k, v = (torch.cat([piece for pair in zip(old.split(past), new.split(sizes)) for piece in pair])
                    for old, new in ((old_k, k), (old_v, v)))
        q_offsets, k_offsets = [0], [0]
        for part, p in zip(parts, past):
            q_offsets.append(q_offsets[-1] + len(part))
            k_offsets.append(k_offsets[-1] + len(part) + p)
        plan = self.backend.prepare_attention(tokens=len(ids), keys=len(k), sequences=n, q_heads=self.q_heads,
                                              kv_heads=self.kv_heads, head_dim=self.head_dim, dtype=DTYPE, device=self.device)
        attended = plan.run(q, k, v, self.integers(q_offsets, torch.int32), self.integers(k_offsets, torch.int32),
                            out=torch.empty_like(q))
        last = self.integers([o - 1 for o in q_offsets[1:]])
        return self.output(x[last].contiguous(), attended[last].contiguous())

    def decode(self, ids, lengths):
        """Logits after one more token of every sequence, over the cache."""
        n = len(ids)
        slots = [self.slots(b, n, [p])[0] for b, p in enumerate(lengths)]
        x, qkv = self.project(ids)
        q, _, _ = self.write(qkv, lengths, slots)
        width = max(lengths) // self.page_tokens + 1
        plan = self.cache.prepare_attention(sequences=n, q_heads=self.q_heads, query_tokens=1, max_pages=width)
        table = self.integers([[b + n * i for i in range(width)] for b in range(n)], torch.int32)
        attended = plan.run(q, table, self.integers([p + 1 for p in lengths], torch.int32), out=torch.empty_like(q),
                            workspace=self.tensor(plan.workspace_bytes, dtype=torch.uint8))
        return self.output(x, attended)

    def sample(self, logits, uniforms, **settings):
        tokens = self.tensor(len(logits), dtype=torch.int64)
        plan = self.backend.prepare_sampling(rows=len(logits), vocab=self.vocab, dtype=DTYPE, device=self.device)
        return plan.run(logits, uniforms, **settings, tokens=tokens).tolist()


def generate(layer, prompts, steps, *, first=None, seed=0, temperature=0.8, top_k=50, top_p=0.95):
    """`steps` tokens for every prompt. `first`: tokens of each prompt that go through in the first of two passes."""
    n = len(prompts)
    gen = torch.Generator().manual_seed(seed)
    settings = dict(temperature=torch.full((n,), temperature, device=layer.device),
                    top_k=torch.full((n,), top_k, dtype=torch.int32, device=layer.device),
                    top_p=torch.full((n,), top_p, device=layer.device))
    if first:
        layer.prompts([p[:first] for p in prompts], [0] * n)
        logits = layer.prompts([p[first:] for p in prompts], [first] * n)
    else:
        logits = layer.prompts(prompts, [0] * n)
    lengths, tokens = [len(p) for p in prompts], [[] for _ in prompts]
    for _ in range(steps):
        ids = layer.sample(logits, torch.rand(n, generator=gen).to(layer.device), **settings)
        for own, i in zip(tokens, ids):
            own.append(i)
        logits = layer.decode(ids, lengths)
        lengths = [length + 1 for length in lengths]
    return tokens, logits


if __name__ == "__main__":
    parser = argparse.ArgumentParser()
    parser.add_argument("--steps", type=int, default=16)
    steps = parser.parse_args().steps
    prompts = [list(range(3, 40)), list(range(500, 511)), list(range(100, 162))]
    tokens, _ = generate(Layer("cuda:0", pages=64 + steps), prompts, steps, first=8)
    for prompt, own in zip(prompts, tokens):
        print(f"{len(prompt)} prompt tokens -> {own}", flush=True)
