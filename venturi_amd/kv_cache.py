"""Paged Q8 key/value cache: rows written with rotary positions, read back, and attended to.

A cache holds ``pages * page_tokens`` slots; slot s is token s % page_tokens of page s // page_tokens. A slot keeps K
and V of every KV head by the q8_g32_fp16 rule: per 32 columns scale = fp16(max|x| / 127) and
code = clamp(rint(x / scale), -127, 127) (0 where the scale is 0), of K as rounded to the cache's dtype. A group that
holds an infinity or a NaN, or whose scale overflows fp16, reads back as NaN. Planes (K and V each):

* codes uint8 [pages, kv_heads, page_tokens, padded head_dim]: code + 128; columns past head_dim hold 128;
* scales fp16 [pages, kv_heads, groups, page_tokens]: the keys' scales of one group side by side, as the attention
  kernel's lanes take them.

Plans follow the package's contract: ``prepare`` checks shapes and admits the device, ``run`` takes caller-owned
contiguous tensors and neither allocates nor synchronises, so it can be captured in a HIP graph. The reference has no
such cache (its runtime keeps K and V dense); these operators are extensions.
"""

from dataclasses import dataclass, field
import math

import torch

from .operands import DTYPE_CODES, admit, disjoint, extents
from .rotary import RotaryEmbedding

GROUP = 32
MAX_HEAD_DIM = 256


def head_geometry(q_heads, kv_heads, head_dim):
    """Checks head counts and size that the attention kernels take."""
    extents(q_heads, kv_heads, head_dim)
    if head_dim % 8 or head_dim > MAX_HEAD_DIM:
        raise ValueError(f"head_dim must be a multiple of 8 of at most {MAX_HEAD_DIM}")
    if q_heads % kv_heads:
        raise ValueError("q_heads must be a multiple of kv_heads")


def softmax_scale(scale, head_dim):
    """The factor on q k^T: 1 / sqrt(head_dim) unless given."""
    if scale is None:
        return 1.0 / math.sqrt(head_dim)
    if type(scale) in (int, float) and math.isfinite(scale):
        return float(scale)
    raise ValueError("attention scale must be a finite number")


def vector_aligned(*tensors):
    """The kernels move 16 bytes at a time."""
    for t in tensors:
        if t.data_ptr() % 16:
            raise ValueError("attention operands require 16-byte alignment")


@dataclass(frozen=True)
class Q8KVCache:
    """One layer's K and V on the device (``HipBackend.create_kv_cache``)."""

    _backend: object
    pages: int
    page_tokens: int
    kv_heads: int
    head_dim: int
    dtype: torch.dtype
    device: torch.device
    key_codes: torch.Tensor = field(repr=False)
    key_scales: torch.Tensor = field(repr=False)
    value_codes: torch.Tensor = field(repr=False)
    value_scales: torch.Tensor = field(repr=False)

    @classmethod
    def create(cls, backend, *, pages, page_tokens, kv_heads, head_dim, dtype, device):
        extents(pages, page_tokens)
        head_geometry(kv_heads, kv_heads, head_dim)
        if page_tokens % 16 or page_tokens > 4096:
            raise ValueError("page_tokens must be a multiple of 16 of at most 4096")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("The Q8 KV cache takes FP16/BF16 rows")
        target = backend.validate_device(dtype, device)
        groups = (head_dim + GROUP - 1) // GROUP
        with torch.cuda.device(target):
            codes = [torch.full((pages, kv_heads, page_tokens, groups * GROUP), 128, dtype=torch.uint8, device=target)
                     for _ in range(2)]
            scales = [torch.zeros(pages, kv_heads, groups, page_tokens, dtype=torch.float16, device=target) for _ in range(2)]
            torch.cuda.current_stream(target).synchronize()
        return cls(backend, pages, page_tokens, kv_heads, head_dim, dtype, target, codes[0], scales[0], codes[1], scales[1])

    @property
    def slots(self):
        return self.pages * self.page_tokens

    @property
    def storage_tensors(self):
        return (self.key_codes, self.key_scales, self.value_codes, self.value_scales)

    @property
    def storage_nbytes(self):
        return sum(t.nbytes for t in self.storage_tensors)

    def prepare_write(self, *, tokens, q_heads, rotary):
        """Plan of writing ``tokens`` projected rows [(q_heads + 2 kv_heads) * head_dim]: q heads, then K, then V.

        ``rotary`` (a RotaryEmbedding, or None) turns q and K. ``q_heads`` may be 0: rows of K and V alone.
        """
        extents(tokens)
        if type(q_heads) is not int or not 0 <= q_heads < 2**20:
            raise ValueError("q_heads must be a nonnegative integer")
        if rotary is not None and not isinstance(rotary, RotaryEmbedding):
            raise TypeError("rotary must be a RotaryEmbedding or None")
        if rotary is not None and rotary.head_dim != self.head_dim:
            raise ValueError("rotary and cache differ in head_dim")
        width = (q_heads + 2 * self.kv_heads) * self.head_dim
        extents(width)
        self._backend.resolve_device(self.device)
        rates = None
        if rotary is not None:
            with torch.cuda.device(self.device):
                rates = rotary.rates.to(self.device)
                torch.cuda.current_stream(self.device).synchronize()
        return KVWritePlan(self, tokens, q_heads, rotary, rates)

    def prepare_read(self, *, tokens):
        """Plan of reading ``tokens`` slots back as rows of the cache's dtype."""
        extents(tokens)
        self._backend.resolve_device(self.device)
        return KVReadPlan(self, tokens)

    def prepare_attention(self, *, sequences, q_heads, query_tokens, max_pages, scale=None):
        """Plan of attention of ``query_tokens`` new tokens of every sequence over its cached keys.

        ``max_pages`` is the width of the page table. The new tokens' own keys are in the cache: query i of t sees the
        first length - (t - 1 - i) keys.
        """
        extents(sequences, query_tokens, max_pages)
        head_geometry(q_heads, self.kv_heads, self.head_dim)
        factor = softmax_scale(scale, self.head_dim)
        self._backend.resolve_device(self.device)
        lib = self._backend._native
        nbytes = lib.venturi_kv_attention_bytes(sequences, query_tokens, q_heads, self.kv_heads, self.head_dim, max_pages,
                                                self.page_tokens)
        if nbytes == 0 and lib.venturi_blocks_error():
            raise ValueError(lib.error())
        return KVAttentionPlan(self, sequences, query_tokens, q_heads, max_pages, factor, int(nbytes))


@dataclass(frozen=True)
class KVWritePlan:
    cache: Q8KVCache
    tokens: int
    q_heads: int
    rotary: object
    _rates: object
    workspace_bytes = 0

    @property
    def storage_tensors(self):
        return self.cache.storage_tensors + (() if self._rates is None else (self._rates,))

    def run(self, rows, positions, slots, *, q=None, k=None):
        """Rotates and caches ``rows``; the rotated q heads go to ``q`` [tokens, q_heads, head_dim], and the rotated
        keys to ``k`` [tokens, kv_heads, head_dim] where one is given.

        ``positions`` (int64 [tokens]; unused without rotary, may then be None) and ``slots`` (int64 [tokens]) stay on
        the device. A row whose slot lies outside the cache (-1: padding) is not cached. Rows that share a slot leave
        one of theirs there, unspecified which.
        """
        c = self.cache
        admit(rows, (self.tokens, (self.q_heads + 2 * c.kv_heads) * c.head_dim), c.dtype, c.device, "rows")
        admit(slots, (self.tokens,), torch.int64, c.device, "slots")
        inputs = (rows, slots) + self.storage_tensors
        if self._rates is not None:
            admit(positions, (self.tokens,), torch.int64, c.device, "positions")
            inputs += (positions,)
        if (q is None) != (self.q_heads == 0):
            raise ValueError("q is the output of the plan's q heads: required with them, refused without")
        vector_aligned(rows)
        if q is not None:
            admit(q, (self.tokens, self.q_heads, c.head_dim), c.dtype, c.device, "q")
            vector_aligned(q)
            disjoint(q, inputs if k is None else inputs + (k,))
        if k is not None:
            admit(k, (self.tokens, c.kv_heads, c.head_dim), c.dtype, c.device, "k")
            vector_aligned(k)
            disjoint(k, inputs)
        r = self.rotary
        c._backend._launch("venturi_kv_write_run", c.device, rows, None if r is None else positions, slots, self._rates, q, k,
                           *c.storage_tensors, self.tokens, self.q_heads, c.kv_heads, c.head_dim,
                           0 if r is None else r.rotary_dim, int(r is not None and r.layout == "interleaved"),
                           1.0 if r is None else r.factor, c.pages, c.page_tokens, DTYPE_CODES[c.dtype])
        return q


@dataclass(frozen=True)
class KVReadPlan:
    cache: Q8KVCache
    tokens: int
    workspace_bytes = 0

    @property
    def storage_tensors(self):
        return self.cache.storage_tensors

    def run(self, slots, *, keys=None, values=None):
        """Writes the cached rows of ``slots`` (int64 [tokens]) to ``keys`` and ``values`` [tokens, kv_heads, head_dim]
        (either may be left out). A slot outside the cache reads as NaN."""
        c = self.cache
        admit(slots, (self.tokens,), torch.int64, c.device, "slots")
        inputs = (slots,) + c.storage_tensors
        if keys is None and values is None:
            raise ValueError("reading needs keys, values or both")
        for name, out in (("keys", keys), ("values", values)):
            if out is not None:
                admit(out, (self.tokens, c.kv_heads, c.head_dim), c.dtype, c.device, name)
                vector_aligned(out)
                disjoint(out, inputs)
        if keys is not None and values is not None:
            disjoint(keys, (values,))
        c._backend._launch("venturi_kv_read_run", c.device, *c.storage_tensors, slots, keys, values, self.tokens, c.kv_heads,
                           c.head_dim, c.pages, c.page_tokens, DTYPE_CODES[c.dtype])
        return keys, values


@dataclass(frozen=True)
class KVAttentionPlan:
    cache: Q8KVCache
    sequences: int
    query_tokens: int
    q_heads: int
    max_pages: int
    scale: float
    workspace_bytes: int

    @property
    def storage_tensors(self):
        return self.cache.storage_tensors

    def run(self, q, page_table, lengths, *, out, workspace=None):
        """out = softmax(scale q k^T) v over the pages ``page_table[b]`` (int32 [sequences, max_pages]) of every sequence.

        ``q`` and ``out`` are [sequences * query_tokens, q_heads, head_dim], sequence after sequence; ``lengths`` (int32
        [sequences]) counts the cached keys, the new tokens' own included. Both stay on the device: queries that see no
        key get zeros, and sequences whose length lies outside [0, max_pages * page_tokens], or that reach a page
        outside the cache, get NaN. Page table entries past a sequence's length are not read.
        """
        c = self.cache
        shape = (self.sequences * self.query_tokens, self.q_heads, c.head_dim)
        admit(q, shape, c.dtype, c.device, "q")
        admit(page_table, (self.sequences, self.max_pages), torch.int32, c.device, "page_table")
        admit(lengths, (self.sequences,), torch.int32, c.device, "lengths")
        admit(out, shape, c.dtype, c.device, "out")
        vector_aligned(q, out)
        inputs = (q, page_table, lengths) + c.storage_tensors
        if self.workspace_bytes:
            admit(workspace, (self.workspace_bytes,), torch.uint8, c.device, "workspace")
            if workspace.data_ptr() % 256:
                raise ValueError("attention workspace requires 256-byte alignment")
            disjoint(workspace, inputs)
            disjoint(out, inputs + (workspace,))
        else:
            disjoint(out, inputs)
        c._backend._launch("venturi_kv_attention_run", c.device, q, *c.storage_tensors, page_table, lengths, out,
                           workspace if self.workspace_bytes else None, self.workspace_bytes, self.sequences, self.query_tokens,
                           self.q_heads, c.kv_heads, c.head_dim, c.pages, c.page_tokens, self.max_pages, self.scale,
                           DTYPE_CODES[c.dtype])
        return out
