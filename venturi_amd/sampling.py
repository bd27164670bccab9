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

from dataclasses import dataclass

import torch

from .kv_cache import settle
from .operands import DTYPE_CODES, address, apart, device_index, extents

_MAX_VOCAB = 1 << 20
_SETTINGS = (("temperature", torch.float32), ("top_k", torch.int32), ("top_p", torch.float32), ("min_p", torch.float32))


@dataclass(frozen=True)
class SamplingPlan:
    """``HipBackend.prepare_sampling``. It holds no memory: runs of one plan may overlap on several streams."""

    _backend: object
    rows: int
    vocab: int
    dtype: torch.dtype
    device: torch.device
    workspace_bytes = 0
    storage_tensors = ()

    def __post_init__(self):
        settle(self, _entry=self._backend._native.venturi_sample_run, _index=device_index(self.device), _logits=(self.rows, self.vocab),
               _row=(self.rows,), _tail=(self.rows, self.vocab, DTYPE_CODES[self.dtype]))

    @classmethod
    def create(cls, backend, *, rows, vocab, dtype, device):
        extents(rows, vocab)
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("Sampling takes FP16/BF16 logits")
        if vocab > _MAX_VOCAB:
            raise ValueError(f"Sampling takes a vocabulary of at most {_MAX_VOCAB}")
        return cls(backend, rows, vocab, dtype, backend.validate_device(dtype, device))

    def run(self, logits, uniforms, temperature=None, top_k=None, top_p=None, min_p=None, *, tokens, probabilities=None):
        """``logits`` [rows, vocab], ``uniforms`` fp32 [rows]; per-row settings ``temperature``, ``top_p``, ``min_p`` fp32
        and ``top_k`` int32 [rows], each None for 1, no limit, no limit and no limit. Writes ``tokens`` int64 [rows] and,
        where given, ``probabilities`` fp32 [rows]."""
        device, index, row, size = self.device, self._index, self._row, 4 * self.rows
        x = address(logits, self._logits, self.dtype, device, index, "logits")
        u = address(uniforms, row, torch.float32, device, index, "uniforms", 4)
        inputs = [(x, x + 2 * self.rows * self.vocab), (u, u + size)]
        settings = []
        for (name, dtype), value in zip(_SETTINGS, (temperature, top_k, top_p, min_p)):
            pointer = None
            if value is not None:
                pointer = address(value, row, dtype, device, index, name, 4)
                inputs.append((pointer, pointer + size))
            settings.append(pointer)
        t, p = address(tokens, row, torch.int64, device, index, "tokens", 8), None
        apart(t, 2 * size, *inputs)
        if probabilities is not None:
            p = address(probabilities, row, torch.float32, device, index, "probabilities", 4)
            apart(p, size, (t, t + 2 * size), *inputs)
        self._backend._call(self._entry, device, (x, u, *settings, t, p, *self._tail))
        return tokens
