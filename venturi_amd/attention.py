"""Causal attention over packed prompts: sequences of different lengths side by side in one call.

Sequence b owns rows q_offsets[b] .. q_offsets[b + 1] of q and rows k_offsets[b] .. k_offsets[b + 1] of k and v. Its
queries are its last tokens: with n keys and t queries, query i sees the first n - (t - 1 - i) keys, so keys before the
queries' own (cached ones, read back) are seen by all of them. Head h of q reads KV head h * kv_heads // q_heads.
The reference's runtime calls its own attention kernel for one sequence (ops_api.h:13-15); packing, the past and the
prepared plan are this package's.
"""

from dataclasses import dataclass, field

import torch

from .kv_cache import head_geometry, settle, softmax_scale
from .operands import DTYPE_CODES, address, apart, device_index, extents, spans, stream_of


@dataclass(frozen=True)
class PackedAttentionPlan:
    """``HipBackend.prepare_attention``. The plan owns its workspace (partial sums of calls with few rows, split over
    their keys), so runs of one plan must be ordered: one stream at a time. Concurrent streams prepare a plan each, and a
    captured graph needs its plan for as long as it is replayed."""

    _backend: object
    tokens: int
    keys: int
    sequences: int
    q_heads: int
    kv_heads: int
    head_dim: int
    scale: float
    dtype: torch.dtype
    device: torch.device
    _workspace: object = field(repr=False)
    _stream: object = field(repr=False)  # of the workspace's allocation
    workspace_bytes = 0  # nothing for the caller to provide

    def __post_init__(self):
        w = self._workspace
        settle(self, _entry=self._backend._native.venturi_packed_attention_run, _index=device_index(self.device),
               _q=(self.tokens, self.q_heads, self.head_dim), _k=(self.keys, self.kv_heads, self.head_dim),
               _offsets=(self.sequences + 1,), _spans=spans(*self.storage_tensors),
               _tail=(None if w is None else w.data_ptr(), 0 if w is None else w.numel(), self.tokens, self.keys, self.sequences,
                      self.q_heads, self.kv_heads, self.head_dim, self.scale, DTYPE_CODES[self.dtype]))

    @property
    def storage_tensors(self):
        return () if self._workspace is None else (self._workspace,)

    @classmethod
    def create(cls, backend, *, tokens, keys, sequences, q_heads, kv_heads, head_dim, dtype, device, scale=None):
        extents(tokens, keys, sequences)
        head_geometry(q_heads, kv_heads, head_dim)
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("Packed attention takes FP16/BF16")
        factor = softmax_scale(scale, head_dim)
        target = backend.validate_device(dtype, device)
        lib = backend._native
        nbytes = lib.venturi_packed_attention_bytes(tokens, keys, sequences, q_heads, kv_heads, head_dim)
        if nbytes == 0 and lib.venturi_blocks_error():
            raise ValueError(lib.error())
        workspace = stream = None
        if nbytes:
            with torch.cuda.device(target):
                workspace, stream = torch.empty(nbytes, dtype=torch.uint8, device=target), stream_of(target)
                # Earlier work of this stream may still use the memory; the plan may run on another.
                torch.cuda.current_stream(target).synchronize()
        return cls(backend, tokens, keys, sequences, q_heads, kv_heads, head_dim, factor, dtype, target, workspace, stream)

    def run(self, q, k, v, q_offsets, k_offsets, *, out):
        """``q`` and ``out`` [tokens, q_heads, head_dim], ``k`` and ``v`` [keys, kv_heads, head_dim], offsets int32
        [sequences + 1] on the device, ascending from 0. Queries that see no key, and rows past the last offset, get
        zeros. Offsets are not checked on the host; the kernel reads no row outside q, k and v whatever they hold.
        """
        dtype, device, index = self.dtype, self.device, self._index
        x = address(q, self._q, dtype, device, index, "q")
        a = address(k, self._k, dtype, device, index, "k")
        b = address(v, self._k, dtype, device, index, "v")
        m = address(q_offsets, self._offsets, torch.int32, device, index, "q_offsets", 4)
        n = address(k_offsets, self._offsets, torch.int32, device, index, "k_offsets", 4)
        y = address(out, self._q, dtype, device, index, "out")
        size, rows, starts = 2 * self.tokens * self.q_heads * self.head_dim, 2 * self.keys * self.kv_heads * self.head_dim, 4 * self._offsets[0]
        apart(y, size, (x, x + size), (a, a + rows), (b, b + rows), (m, m + starts), (n, n + starts), *self._spans)
        self._backend._call(self._entry, device, (x, a, b, m, n, y, *self._tail))
        if self._workspace is not None and stream_of(device) != self._stream:
            # A plan that is dropped now leaves its workspace to this run until it is done.
            self._workspace.record_stream(torch.cuda.current_stream(device))
        return out
