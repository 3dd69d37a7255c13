"""Low-rank adapters of many requests beside one shared projection (`nmoe_adapters_add`, include/nmoe.h).

    pool = AdapterPool(a, b, scales)            # the adapters of one projection
    y = x @ weight.t()                          # the projection, for all rows at once
    y = pool.add(x, y, ids, offsets, out=y)     # and what each sequence's adapter adds

a is [adapters, rank, inner], b [adapters, outer, rank] bf16 and scales [adapters] FP32; an adapter of a
lower rank is filled up with zeros.  `ids` [n] and `offsets` [n + 1] are int32 tensors on the device,
as the lists of a batch are in attention.py: entry i's rows take adapter ids[i], -1 none.  The
host reads neither, so a step can be recorded in a CUDA graph.  Calls run on the current stream and keep
nothing between them.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _check, _stream, load_library
from .attention import _require_list, _stream_of, _zeros

MAX_RANK = 128


class _Adapters(ctypes.Structure):
    _fields_ = [("adapters", ctypes.c_int32), ("rank", ctypes.c_int32), ("inner", ctypes.c_int32),
                ("outer", ctypes.c_int32), ("a", ctypes.c_void_p), ("b", ctypes.c_void_p),
                ("scales", ctypes.c_void_p)]


_library = None


def _lib() -> ctypes.CDLL:
    global _library
    if _library is None:
        lib = load_library()
        vp, i32, i64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64
        pool = ctypes.POINTER(_Adapters)
        lib.nmoe_adapters_workspace_bytes.restype = ctypes.c_size_t
        lib.nmoe_adapters_workspace_bytes.argtypes = [pool, i64, i32]
        lib.nmoe_adapters_add.argtypes = [pool, vp, vp, i64, vp, i64, vp, i64, i64, vp, vp, i32, vp,
                                          ctypes.c_size_t, vp]
        lib.nmoe_adapters_sync_status.argtypes = [vp, vp]
        _library = lib
    return _library


def _row_stride(t: torch.Tensor, name: str, rows: Optional[int], columns: int, device: torch.device) -> int:
    """Elements from row to row of a [rows, columns] bf16 tensor."""
    shape, stride = t.shape, t.stride()
    if t.dtype is not torch.bfloat16 or t.device != device or len(shape) != 2 or shape[1] != columns or \
            (rows is not None and shape[0] != rows):
        raise ValueError(f"{name} must be bfloat16 [{'rows' if rows is None else rows}, {columns}] on {device}")
    if shape[0] and (stride[1] != 1 or (shape[0] > 1 and (stride[0] < columns or stride[0] % 8)) or t.data_ptr() % 16):
        raise ValueError(f"{name}: rows begin on 16-byte boundaries, their elements lie side by side")
    return stride[0] if shape[0] > 1 else columns


class AdapterPool:
    """The adapters of one projection.  The tensors are the caller's: an adapter may be set or exchanged between
    calls."""

    def __init__(self, a: torch.Tensor, b: torch.Tensor, scales: Optional[torch.Tensor] = None):
        device = a.device
        _stream_of(device, "a")
        for t, name in ((a, "a"), (b, "b")):
            if t.dtype is not torch.bfloat16 or t.dim() != 3 or t.device != device or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous bfloat16 of three dimensions on {device}")
        self.adapters, self.rank, self.inner = a.shape
        self.outer = b.shape[1]
        if b.shape != (self.adapters, self.outer, self.rank) or self.adapters == 0:
            raise ValueError("a must be [adapters, rank, inner], b [adapters, outer, rank]")
        if self.rank % 8 or not 0 < self.rank <= MAX_RANK or self.inner % 8 or self.outer % 8 or not self.inner or \
                not self.outer:
            raise ValueError(f"rank (at most {MAX_RANK}), inner and outer must be multiples of 8")
        if scales is None:
            scales = torch.ones(self.adapters, dtype=torch.float32, device=device)
        if scales.dtype is not torch.float32 or scales.shape != (self.adapters,) or scales.device != device or \
                not scales.is_contiguous():
            raise ValueError(f"scales must be a contiguous vector of {self.adapters} float32 on {device}")
        self.a, self.b, self.scales, self.device = a, b, scales, device
        self._c = _Adapters(self.adapters, self.rank, self.inner, self.outer, a.data_ptr(), b.data_ptr(),
                            scales.data_ptr())
        self._ref = ctypes.byref(self._c)
        self.error = _zeros(1, torch.int32, device, "a pool's word")

    def add(self, x: torch.Tensor, y: torch.Tensor, ids: torch.Tensor, offsets: torch.Tensor,
            out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """y + scales[id] (x a[id]^T) b[id]^T for the rows of each entry; `out` may be y itself.  x is [rows, inner],
        y [rows, outer].  Sums are FP32 and the result is rounded once; rows of no entry are as `out` had
        them, undefined without it."""
        device = self.device
        stream = _stream_of(device, "the pool")
        x_stride = _row_stride(x, "x", None, self.inner, device)
        rows = x.shape[0]
        y_stride = _row_stride(y, "y", rows, self.outer, device)
        _require_list(ids, "ids", device)
        _require_list(offsets, "offsets", device)
        count = ids.shape[0]
        if offsets.shape[0] != count + 1:
            raise ValueError("offsets must have one entry more than ids")
        if rows and count == 0:
            raise ValueError("rows need an entry")
        if out is None:
            out = torch.empty((rows, self.outer), dtype=torch.bfloat16, device=device)
        out_stride = _row_stride(out, "out", rows, self.outer, device)
        library = _library or _lib()
        needed = library.nmoe_adapters_workspace_bytes(self._ref, rows, count) if rows else 0
        workspace = torch.empty(needed, dtype=torch.uint8, device=device)
        _check(library.nmoe_adapters_add(
            self._ref, stream, x.data_ptr(), x_stride, y.data_ptr(), y_stride, out.data_ptr(), out_stride, rows,
            ids.data_ptr(), offsets.data_ptr(), count, workspace.data_ptr(), needed, self.error.data_ptr()),
            "nmoe_adapters_add")
        return out

    def sync_status(self) -> int:
        """Waits for the current stream; what calls of `add` found wrong (an id that is no adapter's,
        offsets out of order), and clears it."""
        return _lib().nmoe_adapters_sync_status(self.error.data_ptr(), _stream())
