"""Base rows held in 4 bits on the GPU, and the products of a few queries with all of them.

Beside ``BruteforceSearch``: the same scan over every row, in 4.25 bits a value instead of 32 - a coarse score to pick
candidates by, or the scores themselves where that precision will do.  Everything runs on CUDA tensors and on torch's
current stream of their device (include/vdb_index.h, vdb_rows4_*)."""
from __future__ import annotations

import torch

from . import _lib
from ._lib import BF16, F16, F32, check

_U8, _F32 = torch.uint8, torch.float32
_codes = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}


def dtype_code(t, what: str) -> int:
    code = _codes.get(t.dtype)
    if code is None:
        raise ValueError(f"{what}: float32, float16 or bfloat16, got {t.dtype}")
    return code


def no_gradient() -> None:
    """For a tensor that requires one: refused where torch records operations, or the gradient would be lost without a word."""
    if torch.is_grad_enabled():
        raise ValueError("no gradient passes through this call: detach the tensor, or call under torch.no_grad()")


def on_device(index, call, *args) -> None:
    """Calls ``call(*args, stream)`` with device ``index`` current, on torch's current stream of it (as a number:
    torch.cuda.current_stream, which makes an object of it, costs the host 7 us a call)."""
    current = torch._C._cuda_getDevice()
    if current == index:
        status = call(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        torch.cuda.set_device(index)
        try:
            status = call(*args, torch._C._cuda_getCurrentRawStream(index))
        finally:
            torch.cuda.set_device(current)
    if status:
        check(status)


class Rows4:
    """``codes`` [n, ceil(dim / 32) * 16] uint8 and ``scales`` [n, ceil(dim / 32)] uint8, contiguous CUDA tensors in the
    layout that include/vdb_index.h describes: e2m1 codes, a power-of-two scale for every 32 columns of a row."""

    def __init__(self, codes, scales, dim: int):
        dim = int(dim)
        groups, index = (dim + 31) // 32, codes.get_device()
        if dim < 1:
            raise ValueError("dim must be positive")
        if codes.dtype is not _U8 or scales.dtype is not _U8 or not codes.is_cuda or scales.get_device() != index:
            raise ValueError("codes and scales: uint8 CUDA tensors on one device")
        shape = codes.shape
        if len(shape) != 2 or shape[1] != groups * 16 or scales.shape != (shape[0], groups):
            raise ValueError(f"expected codes [n, {groups * 16}] and scales [n, {groups}], got {tuple(shape)} and {tuple(scales.shape)}")
        if not (codes.is_contiguous() and scales.is_contiguous()):
            raise ValueError("codes and scales must be contiguous")
        self._l = _lib.lib()
        self.codes, self.scales, self.dim = codes, scales, dim
        self._n, self._index = shape[0], index

    @classmethod
    def pack(cls, rows) -> "Rows4":
        """Rounds rows [n, dim] (float32, float16 or bfloat16) to 4 bits."""
        if not rows.is_cuda or rows.dim() != 2:
            raise ValueError("rows: a CUDA tensor [n, dim]")
        t = dtype_code(rows, "rows")
        if rows.requires_grad:
            no_gradient()
        if rows.stride(1) != 1 or rows.stride(0) < 0:
            rows = rows.contiguous()
        n, dim = rows.shape
        groups = (dim + 31) // 32
        out = cls(torch.empty((n, groups * 16), dtype=torch.uint8, device=rows.device),
                  torch.empty((n, groups), dtype=torch.uint8, device=rows.device), dim)
        on_device(rows.get_device(), out._l.vdb_rows4_pack_device, rows.data_ptr(), t, n, dim, rows.stride(0), out.codes.data_ptr(), out.scales.data_ptr())
        return out

    def __len__(self) -> int:
        return self._n

    def unpack(self):
        """The values that the codes stand for, [n, dim] float32."""
        out = torch.empty((len(self), self.dim), dtype=torch.float32, device=self.codes.device)
        on_device(out.get_device(), self._l.vdb_rows4_unpack_device, self.codes.data_ptr(), self.scales.data_ptr(), len(self), self.dim, out.data_ptr())
        return out

    def products(self, queries, out=None):
        """Inner products of queries [nq, dim] (or [dim]) with every row: [nq, n] (or [n]) float32, into ``out`` if given.
        Has no gradient: queries that require one are refused where torch records operations."""
        index, n = self._index, self._n
        x = queries if queries.dim() == 2 else queries.unsqueeze(0)
        if queries.dim() not in (1, 2) or x.shape[1] != self.dim or x.get_device() != index:
            raise ValueError(f"expected queries [nq, {self.dim}] on {self.codes.device}, got {tuple(queries.shape)} on {queries.device}")
        t = dtype_code(x, "queries")
        if x.requires_grad or (out is not None and out.requires_grad):
            no_gradient()
        step, one = x.stride()
        if one != 1 or step < 0:
            x = x.contiguous()
            step = x.stride(0)
        nq = x.shape[0]
        if out is None:
            out = torch.empty((nq, n) if queries.dim() == 2 else (n,), dtype=_F32, device=x.device)
        elif out.dtype is not _F32 or out.get_device() != index or out.numel() != nq * n or not out.is_contiguous():
            raise ValueError(f"out: a contiguous float32 tensor of {nq} x {n} on {x.device}")
        on_device(index, self._l.vdb_rows4_products_device, self.codes.data_ptr(), self.scales.data_ptr(), n, self.dim, x.data_ptr(), t, nq, step, out.data_ptr())
        return out
