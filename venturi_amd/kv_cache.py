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

from .operands import DTYPE_CODES, address, apart, device_index, extents, spans
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
    """The factor on q k^T: 1 / sqrt(head_dim) unless given. Up to 2^127, so that log2 e times it is an FP32 number."""
    if scale is None:
        return 1.0 / math.sqrt(head_dim)
    if type(scale) in (int, float) and abs(scale) <= 2**127:
        return float(scale)
    raise ValueError("attention scale must be a number of at most 2^127")


def settle(plan, **values):
    """Sets what a frozen plan computes once."""
    for name, value in values.items():
        object.__setattr__(plan, name, value)


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
        return KVWritePlan(self, tokens, q_heads, rotary, None if rotary is None else rotary.rates_on(self.device))

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

    def __post_init__(self):
        c, r = self.cache, self.rotary
        settle(
            self, _entry=c._backend._native.venturi_kv_write_run, _index=device_index(c.device),
            _rows=(self.tokens, (self.q_heads + 2 * c.kv_heads) * c.head_dim), _at=(self.tokens,),
            _q=(self.tokens, self.q_heads, c.head_dim), _k=(self.tokens, c.kv_heads, c.head_dim),
            _spans=spans(*self.storage_tensors), _table=None if self._rates is None else self._rates.data_ptr(),
            _tail=(*(t.data_ptr() for t in c.storage_tensors), self.tokens, self.q_heads, c.kv_heads, c.head_dim,
                   0 if r is None else r.rotary_dim, int(r is not None and r.layout == "interleaved"),
                   1.0 if r is None else r.factor, c.pages, c.page_tokens, DTYPE_CODES[c.dtype]))

    @property
    def storage_tensors(self):
        return self.cache.storage_tensors + (() if self._rates is None else (self._rates,))

    def run(self, rows, positions, slots, *, q=None, k=None):
        """Rotates and caches ``rows``; the rotated q heads go to ``q`` [tokens, q_heads, head_dim], and the rotated
        keys to ``k`` [tokens, kv_heads, head_dim] where one is given.

        ``positions`` (int64 [tokens]; unused without rotary, may then be None) and ``slots`` (int64 [tokens]) stay on
        the device. A row whose slot lies outside the cache (-1: padding) is not cached. The slots inside it have to
        differ: rows that share one leave codes and scales of any of them there, not one row's whole. Other slots and
        ``q`` and ``k`` are not touched by that.
        """
        c, index, tokens = self.cache, self._index, self.tokens
        dtype, device = c.dtype, c.device
        if (q is None) != (self.q_heads == 0):
            raise ValueError("q is the output of the plan's q heads: required with them, refused without")
        x = address(rows, self._rows, dtype, device, index, "rows")
        s = address(slots, self._at, torch.int64, device, index, "slots", 8)
        inputs = ((x, x + 2 * tokens * self._rows[1]), (s, s + 8 * tokens)) + self._spans
        p = y = z = None
        if self._table is not None:
            p = address(positions, self._at, torch.int64, device, index, "positions", 8)
            inputs += ((p, p + 8 * tokens),)
        if k is not None:
            z, size = address(k, self._k, dtype, device, index, "k"), 2 * tokens * c.kv_heads * c.head_dim
            apart(z, size, *inputs)
            inputs += ((z, z + size),)
        if q is not None:
            y = address(q, self._q, dtype, device, index, "q")
            apart(y, 2 * tokens * self.q_heads * c.head_dim, *inputs)
        c._backend._call(self._entry, device, (x, p, s, self._table, y, z, *self._tail))
        return q


@dataclass(frozen=True)
class KVReadPlan:
    cache: Q8KVCache
    tokens: int
    workspace_bytes = 0

    def __post_init__(self):
        c = self.cache
        settle(self, _entry=c._backend._native.venturi_kv_read_run, _index=device_index(c.device), _at=(self.tokens,),
               _rows=(self.tokens, c.kv_heads, c.head_dim), _spans=spans(*c.storage_tensors),
               _planes=tuple(t.data_ptr() for t in c.storage_tensors),
               _tail=(self.tokens, c.kv_heads, c.head_dim, c.pages, c.page_tokens, DTYPE_CODES[c.dtype]))

    @property
    def storage_tensors(self):
        return self.cache.storage_tensors

    def run(self, slots, *, keys=None, values=None):
        """Writes the cached rows of ``slots`` (int64 [tokens]) to ``keys`` and ``values`` [tokens, kv_heads, head_dim]
        (either may be left out). A slot outside the cache reads as NaN."""
        if keys is None and values is None:
            raise ValueError("reading needs keys, values or both")
        c, index = self.cache, self._index
        s = address(slots, self._at, torch.int64, c.device, index, "slots", 8)
        inputs = ((s, s + 8 * self.tokens),) + self._spans
        size, k, v = 2 * self.tokens * c.kv_heads * c.head_dim, None, None
        if keys is not None:
            k = address(keys, self._rows, c.dtype, c.device, index, "keys")
            apart(k, size, *inputs)
            inputs += ((k, k + size),)
        if values is not None:
            v = address(values, self._rows, c.dtype, c.device, index, "values")
            apart(v, size, *inputs)
        c._backend._call(self._entry, c.device, (*self._planes, s, k, v, *self._tail))
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

    def __post_init__(self):
        c = self.cache
        settle(self, _entry=c._backend._native.venturi_kv_attention_run, _index=device_index(c.device),
               _rows=(self.sequences * self.query_tokens, self.q_heads, c.head_dim), _table=(self.sequences, self.max_pages),
               _lengths=(self.sequences,), _spans=spans(*c.storage_tensors),
               _planes=tuple(t.data_ptr() for t in c.storage_tensors),
               _tail=(self.workspace_bytes, self.sequences, self.query_tokens, self.q_heads, c.kv_heads, c.head_dim, c.pages,
                      c.page_tokens, self.max_pages, self.scale, DTYPE_CODES[c.dtype]))

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
        c, index = self.cache, self._index
        device = c.device
        x = address(q, self._rows, c.dtype, device, index, "q")
        t = address(page_table, self._table, torch.int32, device, index, "page_table", 4)
        n = address(lengths, self._lengths, torch.int32, device, index, "lengths", 4)
        y = address(out, self._rows, c.dtype, device, index, "out")
        size = 2 * self._rows[0] * self.q_heads * c.head_dim
        inputs = ((x, x + size), (t, t + 4 * self.sequences * self.max_pages), (n, n + 4 * self.sequences)) + self._spans
        w = None
        if self.workspace_bytes:
            w = address(workspace, (self.workspace_bytes,), torch.uint8, device, index, "workspace", 256)
            apart(w, self.workspace_bytes, *inputs)
            inputs += ((w, w + self.workspace_bytes),)
        apart(y, size, *inputs)
        c._backend._call(self._entry, device, (x, *self._planes, t, n, y, w, *self._tail))
        return out
