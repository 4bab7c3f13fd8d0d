"""Low-rank adapters of many requests beside a shared projection.

    y = x W^T + scale[i] * (x A[i]^T) B[i]^T        with each row's own adapter i

`Linear` computes x W^T once for all rows; `Adapters` adds every row's own part in one launch, whatever mixture of adapters
a batch holds. `Linear(weight, adapters=...)` does both in one call (see there). The reference has no adapters.
"""

from struct import Struct

import torch

from .. import _lib
from .._lib import DlmAdapters
from ..ops.paged_kv import _index_error

# The pointers that every call brings, which lie side by side in the descriptor.
_CALL, _CALL_AT = Struct("4Q"), DlmAdapters.x.offset
_MOST_PLANS = 4096


class Adapters:
    """The adapters of one projection: `a` [count, rank, K] and `b` [count, N, rank] BF16 contiguous, `scales` [count] FP32.
    Adapters of a lower rank are padded with zeros to the common one (a multiple of 8, at most 128)."""

    def __init__(self, a, b, scales):
        if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2]:
            raise ValueError(f"a {tuple(a.shape)}, b {tuple(b.shape)}: expected [count, rank, K] and [count, N, rank]")
        self.count, self.rank, self.k = a.shape
        self.n = b.shape[1]
        if self.rank % 8 or not 8 <= self.rank <= 128 or self.k % 8 or self.n % 8 or not self.k or not self.n or not self.count:
            raise ValueError(f"rank {self.rank}, K {self.k}, N {self.n}: expected multiples of 8, the rank at most 128")
        if a.dtype != torch.bfloat16 or b.dtype != torch.bfloat16 or not a.is_contiguous() or not b.is_contiguous():
            raise ValueError("a and b must be contiguous BF16 tensors")
        if scales.dtype != torch.float32 or scales.shape != (self.count,) or not scales.is_contiguous():
            raise ValueError(f"scales must be a contiguous FP32 [{self.count}] tensor")
        if not a.device == b.device == scales.device:
            raise ValueError("a, b and scales must be on one device")
        self.a, self.b, self.scales, self.device = a, b, scales, a.device
        self.status = torch.zeros(_lib.STATUS_WORDS, device=a.device, dtype=torch.int32)
        d = self._call = DlmAdapters()  # what every call starts from
        d.a, d.b, d.scales, d.status = a.data_ptr(), b.data_ptr(), scales.data_ptr(), self.status.data_ptr()
        d.n, d.k, d.rank, d.count, d.pdl = self.n, self.k, self.rank, self.count, 1
        self._plans = {}  # everything of a call's arguments but addresses -> its checked descriptor without these
        self._last = (None, None)  # the one used last, compared before the others are looked through
        _lib.lib()

    def check(self):
        """Raises IndexError for the first id past the last adapter since the last check (synchronises the stream)."""
        _index_error(self.status, "Adapters")

    def __call__(self, x, ids, base, out=None):
        """out = base + each row's own adapter applied to x. `x` [rows, K], `base` and `out` [rows, N] BF16 with contiguous
        rows (`out` may be `base`, but shares no elements with `x`; by default a new tensor), at most 256 rows; `ids` [rows] int32 in any order, negative for
        a row without adapter."""
        key = (x.shape, x.stride(), x.dtype, x.device, ids.shape, ids.stride(), ids.dtype, ids.device, base.shape, base.stride(),
               base.dtype, base.device, None if out is None else (out.shape, out.stride(), out.dtype, out.device))
        last, plan = self._last
        if key != last:
            plan = self._plans.get(key)
            if plan is None:
                plan = self._plan(x, ids, base, out)
                if len(self._plans) >= _MOST_PLANS:
                    self._plans.clear()
                self._plans[key] = plan
            self._last = key, plan
        if out is None:
            out = torch.empty_like(base, memory_format=torch.contiguous_format)
        d = DlmAdapters.from_buffer_copy(plan)
        _CALL.pack_into(d, _CALL_AT, x.data_ptr(), base.data_ptr(), out.data_ptr(), ids.data_ptr())
        code = _lib.launch("dlm_adapters_bf16", d, self.device)
        if code:
            _lib.check(code, f"adapters [{x.shape[0]}, {self.n}, {self.k}] of rank {self.rank}")
        return out

    def _plan(self, x, ids, base, out):
        """The checked descriptor of a call, without the addresses that it brings."""
        if x.dim() != 2 or x.shape[1] != self.k or base.shape != (x.shape[0], self.n):
            raise ValueError(f"Adapters [{self.n}, {self.k}]: x {tuple(x.shape)}, base {tuple(base.shape)}")
        if out is not None and out.shape != base.shape:
            raise ValueError(f"out {tuple(out.shape)}: expected {tuple(base.shape)}")
        m = x.shape[0]
        for t in (x, base) if out is None else (x, base, out):
            if t.dtype != torch.bfloat16 or t.stride(1) != 1 or t.device != self.device:
                raise ValueError(f"x, base and out must be BF16 with contiguous rows on {self.device}")
        if ids.dtype != torch.int32 or ids.shape != (m,) or not ids.is_contiguous() or ids.device != self.device:
            raise ValueError(f"ids must be a contiguous int32 [{m}] tensor on {self.device}")
        d = DlmAdapters.from_buffer_copy(self._call)
        d.m, d.ldx, d.ldb, d.ldo = m, x.stride(0), base.stride(0), self.n if out is None else out.stride(0)
        return d
