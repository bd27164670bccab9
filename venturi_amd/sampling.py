"""Sampling one token per row of logits from given random numbers.

A row's tokens are ordered by logit, largest first, equal logits by index. With weights w = exp((x - max) / temperature)
the kept tokens are the longest prefix of that order in which every token

* ranks below ``top_k`` (0: no limit),
* has less than ``top_p`` of the top-k tokens' whole mass before it (1 and above: no limit), and
* has w >= ``min_p``;

the first token is always kept. The sampled token is the one in whose share of the kept mass the uniform u of [0, 1)
falls, in that order; its probability is its share. A temperature of 0 (below, or NaN) takes the first token, with
probability 1. Logits of -inf and NaN are never taken; a row with no others gives token -1 with probability 0. The
reference samples on the host apart from its greedy kernel (ops_api.h:46-47); this operator is an extension.

The result depends on the inputs alone: counts are whole numbers, masses 64-bit sums in a fixed order.
"""

from dataclasses import dataclass, field

import torch

from .operands import DTYPE_CODES, admit, disjoint, extents

_SETTINGS = (("temperature", torch.float32), ("top_k", torch.int32), ("top_p", torch.float32), ("min_p", torch.float32))


@dataclass(frozen=True)
class SamplingPlan:
    """``HipBackend.prepare_sampling``. The plan owns its workspace, so runs of one plan must be ordered: one stream at a
    time."""

    _backend: object
    rows: int
    vocab: int
    dtype: torch.dtype
    device: torch.device
    _workspace: object = field(repr=False)
    workspace_bytes = 0  # nothing for the caller to provide

    @property
    def storage_tensors(self):
        return () if self._workspace is None else (self._workspace,)

    @classmethod
    def create(cls, backend, *, rows, vocab, dtype, device):
        extents(rows, vocab)
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("Sampling takes FP16/BF16 logits")
        target = backend.validate_device(dtype, device)
        lib = backend._native
        nbytes = lib.venturi_sample_bytes(rows, vocab)
        if nbytes == 0 and lib.venturi_blocks_error():
            raise ValueError(lib.error())
        workspace = None
        if nbytes:
            with torch.cuda.device(target):
                workspace = torch.empty(nbytes, dtype=torch.uint8, device=target)
        return cls(backend, rows, vocab, dtype, target, workspace)

    def run(self, logits, uniforms, temperature=None, top_k=None, top_p=None, min_p=None, *, tokens, probabilities=None):
        """``logits`` [rows, vocab], ``uniforms`` fp32 [rows]; per-row settings ``temperature``, ``top_p``, ``min_p`` fp32
        and ``top_k`` int32 [rows], each None for 1, no limit, no limit and no limit. Writes ``tokens`` int64 [rows] and,
        where given, ``probabilities`` fp32 [rows]."""
        rows = (self.rows,)
        admit(logits, (self.rows, self.vocab), self.dtype, self.device, "logits")
        admit(uniforms, rows, torch.float32, self.device, "uniforms")
        if logits.data_ptr() % 16:
            raise ValueError("logits require 16-byte alignment")
        inputs = [logits, uniforms]
        for (name, dtype), value in zip(_SETTINGS, (temperature, top_k, top_p, min_p)):
            if value is not None:
                admit(value, rows, dtype, self.device, name)
                inputs.append(value)
        inputs.extend(self.storage_tensors)
        admit(tokens, rows, torch.int64, self.device, "tokens")
        disjoint(tokens, inputs)
        if probabilities is not None:
            admit(probabilities, rows, torch.float32, self.device, "probabilities")
            disjoint(probabilities, inputs + [tokens])
        self._backend._launch("venturi_sample_run", self.device, logits, uniforms, temperature, top_k, top_p, min_p, tokens,
                              probabilities, self._workspace, 0 if self._workspace is None else self._workspace.numel(),
                              self.rows, self.vocab, DTYPE_CODES[self.dtype])
        return tokens
