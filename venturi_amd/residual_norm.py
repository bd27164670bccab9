"""The residual's addition with the RMSNorm after it, in one launch.

``total = x + residual`` rounded to the rows' dtype, ``out`` its RMSNorm, and with ``a8_passes`` the norm's int8 form in the
workspace that ``PreparedQ8DP4A.project`` reads. The bytes are those of ``HipBackend.prepare_add``, the norm's own plan and
the A8 quantizer one after another. The reference runs them apart (blocks.py:574-581, 789-823); this plan is an extension.
"""

from dataclasses import dataclass

import torch

from .blocks import ResidentRMSNorm
from .kv_cache import settle
from .operands import DTYPE_CODES, address, apart, device_index, extents, spans


@dataclass(frozen=True)
class ResidualRMSPlan:
    """``prepare_residual_rms``. It holds no memory but the norm's: runs of one plan may overlap on several streams."""

    norm: ResidentRMSNorm
    tokens: int
    a8_passes: int
    workspace_bytes: int

    def __post_init__(self):
        n = self.norm
        size = 4 if n.dtype == torch.float32 else 2
        settle(self, _entry=n._backend._native.venturi_residual_rms_run, _index=device_index(n.device), _size=size,
               _rows=(self.tokens, n.features), _bytes=size * self.tokens * n.features, _spans=spans(*n.storage_tensors),
               _gamma=n._weight.data_ptr(),
               _tail=(self.workspace_bytes, self.tokens, n.features, self.a8_passes, DTYPE_CODES[n.dtype], n.epsilon))

    @property
    def storage_tensors(self):
        return self.norm.storage_tensors

    def run(self, x, residual, *, total, out=None, workspace=None):
        """``x``, ``residual``, ``total`` and ``out`` [tokens, features]. ``total`` may be ``x`` or ``residual`` itself;
        ``out`` may be left out where the plan writes the int8 form to ``workspace`` (uint8 [workspace_bytes])."""
        n, index, rows, size, align = self.norm, self._index, self._rows, self._bytes, self._size
        dtype, device = n.dtype, n.device
        a = address(x, rows, dtype, device, index, "x", align)
        b = address(residual, rows, dtype, device, index, "residual", align)
        t = address(total, rows, dtype, device, index, "total", align)
        apart(t, size, *((p, p + size) for p in (a, b) if p != t), *self._spans)
        used = ((a, a + size), (b, b + size), (t, t + size)) + self._spans
        y = w = None
        if out is not None:
            y = address(out, rows, dtype, device, index, "out", align)
            apart(y, size, *used)
            used += ((y, y + size),)
        elif not self.a8_passes:
            raise ValueError("out is required without the int8 form")
        if self.a8_passes:
            w = address(workspace, (self.workspace_bytes,), torch.uint8, device, index, "workspace", 16)
            apart(w, self.workspace_bytes, *used)
        elif workspace is not None:
            raise ValueError("a residual norm without the int8 form uses no workspace")
        n._backend._call(self._entry, device, (a, b, self._gamma, t, y, w, *self._tail))
        return out


def prepare_residual_rms(norm, *, tokens, a8_passes=0):
    """Plan of total = x + residual and its RMSNorm for ``tokens`` rows of a ResidentRMSNorm's dtype. ``a8_passes`` 1 or 2
    (with the second pass for the first one's residuals) adds the int8 form, of fp16 rows. A run takes up to 2^31 - 1025 features."""
    if not isinstance(norm, ResidentRMSNorm):
        raise ValueError("The residual norm requires a resident RMSNorm")
    if type(a8_passes) is not int or not 0 <= a8_passes <= 2:
        raise ValueError("a8_passes must be 0, 1 or 2")
    if a8_passes and norm.dtype != torch.float16:
        raise ValueError("RMS/A8 requires FP16 activations")
    extents(tokens, norm.features)
    norm._backend.validate_device(norm.dtype, norm.device)
    size = 0
    if a8_passes:
        size = norm._backend._native.venturi_q8_dp4a_bytes(tokens, norm.features, a8_passes)
        if not size:
            norm._backend._check(-1)
    return ResidualRMSPlan(norm, tokens, a8_passes, int(size))
