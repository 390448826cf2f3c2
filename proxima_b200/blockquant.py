"""Block quantiser: vectors as 8-bit floating codes (e4m3) with one power-of-two scale for
each block of 128 components, and the products of such rows on the tensor cores.

It stands beside ``ScalarQuantizer`` (ranges per component) and ``ProductQuantizer``
(codewords); the reference has no counterpart. A block scale needs no training and follows
each vector, so vectors of any distribution can be encoded as they arrive::

    bq = BlockQuantizer(768)
    base = bq.encode(vectors)                      # BlockCodes: 1 byte a component + 1 a block
    scores = bq.product(bq.encode(queries), base)  # (nq, n) dot products, f32 sums

``grouped_product`` pairs ragged groups of queries with ragged groups of rows: the queries
that probe an inverted list with the list's rows, a tenant's queries with the tenant's
rows, or the tokens of an expert with the expert's weights.

CUDA tensors in give CUDA tensors out, computed on the current stream without a wait; a
failure that only the device sees (bad offsets) is raised by a later call or by
``check()``. Host arrays in give NumPy arrays out. There is no CPU path.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import Any

import numpy as np

from . import _native as N
from .errors import Configuration, DimensionMismatch

BLOCK = 128
_DTYPES = {"float32": 0, "float16": 1, "bfloat16": 2}


def _is_cuda(x) -> bool:
    return hasattr(x, "is_cuda") and x.is_cuda


def _up(x: int, to: int) -> int:
    return -(-x // to) * to


def _dtype_code(dtype) -> int:
    name = str(dtype).split(".")[-1] if "torch" in str(dtype) else np.dtype(dtype).name
    if name not in _DTYPES:
        raise Configuration("dtype", 0, f"{name}: must be float32, float16 or bfloat16 (tensors only)")
    return _DTYPES[name]


@dataclass
class BlockCodes:
    """Encoded rows: ``codes`` (n, dim rounded up to 16) and ``scales`` (n, blocks rounded up
    to 4), both uint8, tensors or arrays. Row slices are views."""

    codes: Any
    scales: Any
    dim: int

    def __len__(self) -> int:
        return int(self.codes.shape[0])

    def __getitem__(self, rows: slice) -> "BlockCodes":
        if not isinstance(rows, slice):
            raise TypeError("rows are taken by slices")
        return BlockCodes(self.codes[rows], self.scales[rows], self.dim)

    @property
    def bytes_per_vector(self) -> int:
        return int(self.codes.shape[1] + self.scales.shape[1])


class BlockQuantizer:
    """Encodes, decodes and multiplies rows of ``dim`` components (``pxc_bq_*``)."""

    def __init__(self, dim: int, context=None):
        from .index import Context

        if not 1 <= int(dim) <= 1 << 20:
            raise Configuration("dim", dim, "must be between 1 and 1048576")
        self.dim = int(dim)
        self.blocks = -(-self.dim // BLOCK)
        self.ctx = context or Context.default()

    # -- arguments --
    def _stream(self, tensor) -> int:
        """The current stream of the tensor's device; 1 names the legacy default stream."""
        import torch

        if tensor.device.index != self.ctx.device:
            raise Configuration("device", tensor.device.index, f"the context is on device {self.ctx.device}")
        return torch.cuda.current_stream(tensor.device).cuda_stream or 1

    def _rows(self, c: BlockCodes, cuda: bool, name: str, device=None) -> N.PxcBqRows:
        if c.dim != self.dim:
            raise DimensionMismatch(self.dim, c.dim)
        out = []
        for a, unit, need in ((c.codes, 16, _up(self.dim, 16)), (c.scales, 4, _up(self.blocks, 4))):
            if _is_cuda(a) != cuda or (cuda and device is not None and a.device != device):
                raise Configuration(name, 0, "all operands on one device, or all on the host")
            if str(a.dtype).split(".")[-1] != "uint8" or a.ndim != 2 or a.shape[0] != len(c) or a.shape[1] < need:
                raise Configuration(name, 0, f"codes and scales are uint8, (n, >= {need}) here")
            row, step = (a.stride(0), a.stride(1)) if cuda else a.strides
            if step != 1 or (a.shape[0] > 1 and (row % unit or row < need)):
                raise Configuration(name, 0, f"rows are contiguous, their pitch a multiple of {unit}")
            out.append(row if a.shape[0] > 1 else need)
        return N.PxcBqRows(N.ptr(c.codes), N.ptr(c.scales), len(c), out[0], out[1])

    def _vectors(self, vectors):
        """(n, dim) with contiguous components, in one of the types."""
        if _is_cuda(vectors):
            v = vectors
        else:
            v = np.asarray(vectors)
            if v.dtype not in (np.float32, np.float16):
                v = v.astype(np.float32)
        if v.ndim == 1 and v.shape[0] % self.dim == 0:
            v = v.reshape(-1, self.dim)
        if v.ndim != 2 or v.shape[1] != self.dim:
            raise DimensionMismatch(self.dim, int(v.shape[-1]) if v.ndim else 0)
        return v

    # -- codes --
    def encode(self, vectors) -> BlockCodes:
        """Each row's codes and scales. Rows of a tensor may be strided. An infinity becomes the
        largest code of its block, 448 times the scale; a NaN stays one."""
        v = self._vectors(vectors)
        n, ld, sld = v.shape[0], _up(self.dim, 16), _up(self.blocks, 4)
        if _is_cuda(v):
            import torch

            code = _dtype_code(v.dtype)
            stream = self._stream(v)
            if (self.dim > 1 and v.stride(1) != 1) or (n > 1 and v.stride(0) < self.dim):
                v = v.contiguous()
            codes = torch.empty((n, ld), dtype=torch.uint8, device=v.device)
            scales = torch.empty((n, sld), dtype=torch.uint8, device=v.device)
            rows = N.PxcBqRows(codes.data_ptr(), scales.data_ptr(), n, ld, sld)
            N.call("pxc_bq_encode_device", self.ctx.handle, v.data_ptr(), code, v.stride(0) if n > 1 else self.dim,
                   self.dim, C.byref(rows), stream)
            return BlockCodes(codes, scales, self.dim)
        v = np.ascontiguousarray(v)
        codes, scales = np.zeros((n, ld), np.uint8), np.zeros((n, sld), np.uint8)
        rows = N.PxcBqRows(N.ptr(codes), N.ptr(scales), n, ld, sld)
        N.call("pxc_bq_encode", self.ctx.handle, N.ptr(v), _dtype_code(v.dtype), self.dim, self.dim, C.byref(rows))
        return BlockCodes(codes, scales, self.dim)

    def decode(self, codes: BlockCodes, dtype=None):
        """The vectors that the rows stand for, rounded once to ``dtype`` (float32)."""
        cuda = _is_cuda(codes.codes)
        rows = self._rows(codes, cuda, "codes")
        if cuda:
            import torch

            out = torch.empty((len(codes), self.dim), dtype=dtype or torch.float32, device=codes.codes.device)
            N.call("pxc_bq_decode_device", self.ctx.handle, C.byref(rows), self.dim, out.data_ptr(),
                   _dtype_code(out.dtype), self.dim, self._stream(out))
            return out
        out = np.zeros((len(codes), self.dim), dtype or np.float32)
        N.call("pxc_bq_decode", self.ctx.handle, C.byref(rows), self.dim, N.ptr(out), _dtype_code(out.dtype), self.dim)
        return out

    # -- products --
    def product(self, queries: BlockCodes, base: BlockCodes, dtype=None, out=None):
        """The dot product of every pair of rows, (nq, n): f32 sums, rounded once to ``dtype``
        (float32). ``out`` may be a tensor to write into, its rows strided."""
        cuda = _is_cuda(queries.codes)
        q, b = self._rows(queries, cuda, "queries"), self._rows(base, cuda, "base", queries.codes.device if cuda else None)
        shape = (len(queries), len(base))
        if cuda:
            import torch

            dev = queries.codes.device
            if out is None:
                out = torch.empty(shape, dtype=dtype or torch.float32, device=dev)
            elif (tuple(out.shape) != shape or out.device != dev or (dtype is not None and out.dtype != dtype)
                  or (shape[1] > 1 and out.stride(1) != 1) or (shape[0] > 1 and out.stride(0) < shape[1])):
                raise Configuration("out", 0, "must be (nq, n) on the operands' device, with contiguous rows")
            N.call("pxc_bq_product_device", self.ctx.handle, C.byref(q), C.byref(b), self.dim, out.data_ptr(),
                   _dtype_code(out.dtype), out.stride(0) if shape[0] > 1 else max(shape[1], 1), self._stream(out))
            return out
        if out is not None:
            raise Configuration("out", 0, "is for tensors")
        out = np.zeros(shape, dtype or np.float32)
        N.call("pxc_bq_product", self.ctx.handle, C.byref(q), C.byref(b), self.dim, N.ptr(out), _dtype_code(out.dtype),
               max(shape[1], 1))
        return out

    def grouped_product(self, queries: BlockCodes, query_offsets, base: BlockCodes, base_offsets=None,
                        out_size: int | None = None, dtype=None):
        """Each group's product: group g pairs ``queries[query_offsets[g]:query_offsets[g + 1]]`` with
        ``base[base_offsets[g]:base_offsets[g + 1]]``; either may be empty.

        Without ``base_offsets`` every group has len(base) / groups rows and the result is
        (nq, rows); rows of queries in no group are not written. With them the result is flat: the groups'
        matrices one after the other. ``out_size`` is its length (for tensors, reading the
        offsets back to find it waits for the device)."""
        cuda = _is_cuda(queries.codes)
        dev = queries.codes.device if cuda else None
        q, b = self._rows(queries, cuda, "queries"), self._rows(base, cuda, "base", dev)
        qo, bo = (self._offsets(o, cuda, dev) for o in (query_offsets, base_offsets))
        if qo is None or len(qo) < 2 or (bo is not None and len(bo) != len(qo)):
            raise Configuration("offsets", 0, "groups + 1 int64 values for the queries, and for the base where given")
        groups = len(qo) - 1
        if bo is None:
            if len(base) % groups:
                raise Configuration("base", len(base), "without base offsets the rows must be a multiple of the groups")
            shape = (len(queries), len(base) // groups)
        else:
            if out_size is None:
                out_size = int(((qo[1:] - qo[:-1]) * (bo[1:] - bo[:-1])).sum())
                if out_size < 0:
                    raise Configuration("offsets", 0, "offsets must rise")
            shape = (int(out_size),)
        size = int(np.prod(shape, dtype=np.int64))
        if cuda:
            import torch

            out = torch.empty(shape, dtype=dtype or torch.float32, device=dev)
            N.call("pxc_bq_grouped_product_device", self.ctx.handle, C.byref(q), qo.data_ptr(), C.byref(b), N.ptr(bo),
                   groups, self.dim, out.data_ptr(), _dtype_code(out.dtype), size, self._stream(out))
            return out
        out = np.zeros(shape, dtype or np.float32)
        N.call("pxc_bq_grouped_product", self.ctx.handle, C.byref(q), N.ptr(qo), C.byref(b), N.ptr(bo), groups, self.dim,
               N.ptr(out), _dtype_code(out.dtype), size)
        return out

    def _offsets(self, o, cuda: bool, dev):
        if o is None:
            return None
        if cuda:
            if not _is_cuda(o) or o.device != dev or str(o.dtype) != "torch.int64" or o.ndim != 1:
                raise Configuration("offsets", 0, "must be an int64 tensor on the operands' device")
            return o.contiguous()
        return np.ascontiguousarray(o, np.int64)

    def check(self) -> None:
        """Waits for the current stream and raises a failure that an earlier call left on the device."""
        import torch

        stream = torch.cuda.current_stream(self.ctx.device).cuda_stream or 1
        N.call("pxc_bq_check", self.ctx.handle, stream)
