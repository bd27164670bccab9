"""Routing of tokens to experts: from router logits to the expert ids and scores that ``RoutedExpertsPlan`` takes.

Scores s = softmax(logits) or 1 / (1 + exp(-logits)) over all experts. Experts are ordered by c = s + bias, largest first,
equal ones by index; with ``groups`` > 1 only those of the ``kept_groups`` best groups (consecutive experts of equal number),
ordered by the sum of their two largest c ("pairs"; a lone one that is not masked by itself) or by their largest ("max"), equal
ones by index. The first ``top_k`` are chosen. Their weights are s without the bias, divided by their sum with
``renormalize``, times ``scale``.

An expert whose logit is -inf is masked: it comes after all others, those with a bias of -inf among them, with weight 0,
whatever its bias, and so does a group of masked experts alone. A sum of +inf and -inf counts as +inf. Scores below 2^-1000
(sigmoids of logits under -693.1, and softmax scores that far under the largest) count as 0, and weights whose sum is 0 stay 0.
A token with a NaN among its logits or biased scores, or with +inf under softmax, gets ids -1 and NaN scores, which
the experts' plan turns into a NaN row. Scores are computed in 64 bits, so that the order is the definition's: experts go by
index where 64 bits do not tell them apart (without a bias, where their logits are equal).

The reference's routed experts take ids and scores (flash_next_moe.py:139-161); this operator is an extension.
"""

from dataclasses import dataclass

import torch

from .kv_cache import settle
from .operands import DTYPE_CODES, address, apart, device_index, extents

MAX_EXPERTS, MAX_TOP_K, MAX_GROUPS = 1024, 16, 64
SCORES, GROUP_RANKS = ("softmax", "sigmoid"), ("max", "pairs")


@dataclass(frozen=True)
class RoutingPlan:
    """``HipBackend.prepare_routing``. It holds no memory: runs of one plan may overlap on several streams."""

    _backend: object
    tokens: int
    experts: int
    top_k: int
    score: str
    groups: int
    kept_groups: int
    group_rank: str
    renormalize: bool
    scale: float
    dtype: torch.dtype
    score_dtype: torch.dtype
    device: torch.device
    workspace_bytes = 0
    storage_tensors = ()

    def __post_init__(self):
        size, score_size = (4 if t == torch.float32 else 2 for t in (self.dtype, self.score_dtype))
        settle(self, _entry=self._backend._native.venturi_route_run, _index=device_index(self.device),
               _logits=(self.tokens, self.experts), _bias=(self.experts,), _chosen=(self.tokens, self.top_k), _size=size,
               _score_size=score_size, _bytes=size * self.tokens * self.experts, _pairs=self.tokens * self.top_k,
               _tail=(self.tokens, self.experts, self.top_k, self.groups, self.kept_groups, SCORES.index(self.score),
                      GROUP_RANKS.index(self.group_rank), int(self.renormalize), self.scale, DTYPE_CODES[self.dtype],
                      DTYPE_CODES[self.score_dtype]))

    @classmethod
    def create(cls, backend, *, tokens, experts, top_k, dtype, device, score="softmax", groups=1, kept_groups=1, group_rank="pairs",
               renormalize=True, scale=1.0, score_dtype=torch.float16):
        extents(tokens, experts, top_k, groups, kept_groups)
        if score not in SCORES or group_rank not in GROUP_RANKS:
            raise ValueError(f"score is one of {SCORES}, group_rank one of {GROUP_RANKS}")
        if experts > MAX_EXPERTS or groups > MAX_GROUPS or experts % groups or kept_groups > groups:
            raise ValueError(f"routing takes at most {MAX_EXPERTS} experts in at most {MAX_GROUPS} groups of equal size")
        if top_k > MAX_TOP_K or top_k > experts // groups * kept_groups:
            raise ValueError(f"top_k must be at most {MAX_TOP_K} and the number of the kept groups' experts")
        if type(renormalize) is not bool:
            raise ValueError("renormalize must be a boolean")
        if type(scale) not in (int, float) or not abs(scale) <= torch.finfo(torch.float32).max:
            raise ValueError("scale must be a finite FP32 number")
        for t in (dtype, score_dtype):
            if t not in DTYPE_CODES:
                raise ValueError("Native blocks require FP16, BF16 or FP32")
        return cls(backend, tokens, experts, top_k, score, groups, kept_groups, group_rank, renormalize, float(scale), dtype,
                   score_dtype, backend.validate_device(dtype, device))

    def run(self, logits, bias=None, *, indices, scores):
        """``logits`` [tokens, experts], ``bias`` fp32 [experts] or None. Writes ``indices`` int64 and ``scores``
        [tokens, top_k], the chosen experts in order."""
        device, index = self.device, self._index
        x = address(logits, self._logits, self.dtype, device, index, "logits", self._size)
        inputs, b = ((x, x + self._bytes),), None
        if bias is not None:
            b = address(bias, self._bias, torch.float32, device, index, "bias", 4)
            inputs += ((b, b + 4 * self.experts),)
        i = address(indices, self._chosen, torch.int64, device, index, "indices", 8)
        apart(i, 8 * self._pairs, *inputs)
        s = address(scores, self._chosen, self.score_dtype, device, index, "scores", self._score_size)
        apart(s, self._score_size * self._pairs, (i, i + 8 * self._pairs), *inputs)
        self._backend._call(self._entry, device, (x, b, i, s, *self._tail))
        return indices, scores
