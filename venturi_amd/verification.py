"""Verification of drafted tokens against the target's probabilities, from given random numbers.

Draft i of a sequence stands while u_i * q_i(d_i) < p_i(d_i): p_i is the target's row behind the tokens before it, q_i the
drafter's, 1 for certain drafts (looked up, or a drafter's best). After the first refusal the next token is drawn from
max(p - q, 0) of that row (certain drafts: p without the draft), or from p where nothing is left; when all drafts stand, from p
of the row behind the last. Tokens so emitted are distributed as the target's own samples. The drawn token is the first, by
index, at which the running sum of the shares exceeds the uniform times their whole sum.

Rows need not add to 1; target probabilities that are no positive finite number count as 0 (such tokens are neither accepted
nor drawn), and a row of those alone gives token -1. A draft outside the vocabulary is refused, and one whose proposal is NaN.
Sums are 64-bit, in a fixed order: the result depends on the inputs alone. The rows come from
``HipBackend.prepare_distribution``. The reference decodes without drafts; this operator is an extension.
"""

from dataclasses import dataclass

import torch

from .kv_cache import settle
from .operands import address, apart, device_index, extents

MAX_DRAFTS, _MAX_VOCAB, _MAX_SEQUENCES = 64, 1 << 20, 65535


@dataclass(frozen=True)
class VerificationPlan:
    """``HipBackend.prepare_verification``. The workspace is the caller's: runs that share none may overlap."""

    _backend: object
    sequences: int
    drafts: int
    vocab: int
    device: torch.device
    workspace_bytes: int
    storage_tensors = ()

    def __post_init__(self):
        n, d, v = self.sequences, self.drafts, self.vocab
        settle(self, _entry=self._backend._native.venturi_verify_run, _index=device_index(self.device), _target=(n * (d + 1), v),
               _proposal=(n * d, v), _drafted=(n, d), _emitted=(n, d + 1), _row=(n,), _tail=(self.workspace_bytes, n, d, v))

    @classmethod
    def create(cls, backend, *, sequences, drafts, vocab, device):
        extents(sequences, drafts, vocab)
        if sequences > _MAX_SEQUENCES or drafts > MAX_DRAFTS or vocab > _MAX_VOCAB:
            raise ValueError(f"Verification takes at most {_MAX_SEQUENCES} sequences of {MAX_DRAFTS} drafts and a vocabulary of at "
                             f"most {_MAX_VOCAB}")
        target = backend.validate_device(torch.float32, device)
        return cls(backend, sequences, drafts, vocab, target, int(backend._native.venturi_verify_bytes(sequences, drafts, vocab)))

    def run(self, target, drafted, uniforms, *, proposal=None, counts=None, tokens, accepted, workspace=None):
        """``target`` fp32 [sequences * (drafts + 1), vocab], sequence after sequence; ``drafted`` int64 [sequences, drafts];
        ``uniforms`` fp32 [sequences, drafts + 1], the last of a sequence for its drawn token; ``proposal`` fp32
        [sequences * drafts, vocab], None for certain drafts; ``counts`` int32 [sequences], the drafts that a sequence has,
        None for all. Writes ``accepted`` int32 [sequences] and ``tokens`` int64 [sequences, drafts + 1]: the drafts that
        stand, the drawn token, and -1. Nothing behind a sequence's count, and no row behind the drawn token's, has an effect;
        the probabilities of the drafts there may be loaded all the same."""
        device, index, n, v = self.device, self._index, self.sequences, self.vocab
        d = self.drafts
        x = address(target, self._target, torch.float32, device, index, "target", 4)
        i = address(drafted, self._drafted, torch.int64, device, index, "drafted", 8)
        u = address(uniforms, self._emitted, torch.float32, device, index, "uniforms", 4)
        inputs = ((x, x + 4 * n * (d + 1) * v), (i, i + 8 * n * d), (u, u + 4 * n * (d + 1)))
        q = c = w = None
        if proposal is not None:
            q = address(proposal, self._proposal, torch.float32, device, index, "proposal", 4)
            inputs += ((q, q + 4 * n * d * v),)
        if counts is not None:
            c = address(counts, self._row, torch.int32, device, index, "counts", 4)
            inputs += ((c, c + 4 * n),)
        if self.workspace_bytes:
            w = address(workspace, (self.workspace_bytes,), torch.uint8, device, index, "workspace", 256)
            apart(w, self.workspace_bytes, *inputs)
            inputs += ((w, w + self.workspace_bytes),)
        t = address(tokens, self._emitted, torch.int64, device, index, "tokens", 8)
        apart(t, 8 * n * (d + 1), *inputs)
        a = address(accepted, self._row, torch.int32, device, index, "accepted", 4)
        apart(a, 4 * n, (t, t + 8 * n * (d + 1)), *inputs)
        self._backend._call(self._entry, device, (x, q, i, c, u, t, a, w, *self._tail))
        return tokens
