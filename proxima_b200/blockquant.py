"""Block quantiser: vectors as 8-bit floating codes (e4m3) with one power-of-two scale for
each block of 128 components, and the products of such rows on the tensor cores.

It stands beside ``ScalarQuantizer`` (ranges per component) and ``ProductQuantizer``
(codewords); the reference has no counterpart. A block scale needs no training and follows
each vector, so vectors of any distribution can be encoded as they arrive::

    bq = BlockQuantizer(768)
    base = bq.encode(vectors)                      # BlockCodes: 1 byte a component + 1 a block (padded to 4 a row)
    scores = bq.product(bq.encode(queries), base)  # (nq, n) dot products, f32 sums

``grouped_product`` pairs ragged groups of queries with ragged groups of rows: the queries
that probe an inverted list with the list's rows, a tenant's queries with the tenant's
rows, or the tokens of an expert with the expert's weights.

CUDA tensors in give CUDA tensors out, computed on the current stream without a wait; a
failure that only the device sees (bad offsets) is raised by a later call of the same quantiser, or by its
``check()``, and by no other quantiser's: callers in several threads have one each. Of a quantiser that
is gone, any ``check()`` raises it. Host arrays in give NumPy arrays out. There is no CPU path.
"""
from __future__ import annotations

import ctypes as C
import itertools
from dataclasses import dataclass
from typing import Any

import numpy as np

from . import _native as N
from .errors import Configuration, DimensionMismatch

BLOCK = 128
_NAMES = {"float32": 0, "float16": 1, "bfloat16": 2}
_codes: dict = {}  # dtype -> its code, torch's types among them once torch is in use
_numbers = None  # the numbers under which quantisers make their calls


def _count():
    global _numbers
    if _numbers is None:
        _numbers = itertools.count(N.load().pxc_bq_callers(1 << 48))
    return _numbers


def _is_cuda(x) -> bool:
    return getattr(x, "is_cuda", False)


def _host_array(x, name: str):
    """Host rows as an array over the same memory."""
    if _is_cuda(x):
        raise Configuration(name, 0, "all operands on one device, or all on the host")
    if isinstance(x, np.ndarray):
        return x
    if str(getattr(x, "dtype", None)) != "torch.uint8":
        raise Configuration(name, 0, "codes and scales are uint8, one row per vector")
    return x.numpy()


def _host_vectors(x):
    if hasattr(x, "data_ptr"):
        x = x.detach()
        if str(x.dtype) == "torch.bfloat16":  # no such type in NumPy; every value is one in 32 bits
            x = x.float()
    return np.asarray(x)


def _dtype_code(dtype) -> int:
    code = _codes.get(dtype)
    if code is None:
        tensors = "torch" in str(dtype)
        name = str(dtype).split(".")[-1] if tensors else np.dtype(dtype).name
        if name not in _NAMES or not (tensors or np.dtype(dtype).isnative):
            raise Configuration("dtype", 0, f"{name}: must be float32, float16 or bfloat16 (tensors only)")
        code = _codes[dtype] = _NAMES[name]
    return code


class _Torch:
    """What the tensor paths take from torch, and their entry points, looked up once."""

    def __init__(self):
        import torch

        self.uint8, self.int64, self.float32, self.empty = torch.uint8, torch.int64, torch.float32, torch.empty
        self.current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda index: torch.cuda.current_stream(index).cuda_stream)
        self.encode, self.decode = N.bind("pxc_bq_encode_as"), N.bind("pxc_bq_decode_as")
        self.product, self.grouped = N.bind("pxc_bq_product_as"), N.bind("pxc_bq_grouped_product_as")


_torch_parts: _Torch | None = None


def _torch() -> _Torch:
    global _torch_parts
    if _torch_parts is None:
        _torch_parts = _Torch()
    return _torch_parts


@dataclass(slots=True)
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
        dim = int(dim)
        if not 1 <= dim <= 1 << 20:
            raise Configuration("dim", dim, "must be between 1 and 1048576")
        if context is None:
            from .index import Context

            context = Context.default()
        self.dim = dim
        self.ctx = context
        self.blocks = -(-dim // BLOCK)
        self._ld, self._sld = (dim + 15) & ~15, (self.blocks + 3) & ~3
        self._caller = next(_numbers or _count())
        try:  # quantisers of the context that are gone, until the native side is told
            self._gone = context._gone_callers
        except AttributeError:
            self._gone = context._gone_callers = []

    def __del__(self):
        try:
            self._gone.append(self._caller)
            if len(self._gone) >= 64:
                self._forget()
        except Exception:
            pass

    def _forget(self) -> None:
        gone = []
        try:
            while True:  # others may be at it too
                gone.append(self._gone.pop())
        except IndexError:
            pass
        N.call("pxc_bq_forget", self.ctx.handle, (C.c_uint64 * len(gone))(*gone), len(gone))

    def _host(self, name: str, *args) -> None:
        """A host form, which reports its own failure; what tensors' calls left is raised first."""
        N.call("pxc_bq_report_as", self.ctx.handle, self._caller)
        N.call(name, self.ctx.handle, *args)

    # -- arguments --
    def _stream(self, t: _Torch, tensor) -> int:
        """The current stream of the tensor's device; 1 names the legacy default stream."""
        index = tensor.get_device()
        if index != self.ctx.device:
            raise Configuration("device", index, f"the context is on device {self.ctx.device}")
        return t.current_stream(index) or 1

    def _rows(self, c: BlockCodes, cuda: bool, name: str) -> N.PxcBqRows:
        """The rows as the native calls take them: tensors on the context's device, or arrays."""
        if c.dim != self.dim:
            raise DimensionMismatch(self.dim, c.dim)
        codes, scales = c.codes, c.scales
        if not cuda:
            codes, scales = _host_array(codes, name), _host_array(scales, name)
        elif _is_cuda(codes) != cuda or _is_cuda(scales) != cuda:
            raise Configuration(name, 0, "all operands on one device, or all on the host")
        if codes.ndim != 2 or scales.ndim != 2:
            raise Configuration(name, 0, "codes and scales are uint8, one row per vector")
        if cuda:
            byte, where, p, s = (_torch_parts or _torch()).uint8, self.ctx.device, codes.data_ptr(), scales.data_ptr()
            (cr, cs), (sr, ss) = codes.stride(), scales.stride()
            if codes.get_device() != where or scales.get_device() != where:
                raise Configuration("device", codes.get_device(), f"the context is on device {where}")
        else:
            byte, p, s = np.uint8, N.ptr(codes), N.ptr(scales)
            (cr, cs), (sr, ss) = codes.strides, scales.strides
        if codes.dtype != byte or scales.dtype != byte:
            raise Configuration(name, 0, "codes and scales are uint8, one row per vector")
        (n, width), (rows, blocks) = codes.shape, scales.shape
        if rows != n or width < self._ld or blocks < self._sld:
            raise Configuration(name, n, f"codes are (n, >= {self._ld}) and scales (n, >= {self._sld}) here")
        if n <= 1:
            cr, sr = self._ld, self._sld
        if cs != 1 or ss != 1 or cr % 16 or sr % 4 or cr < self._ld or sr < self._sld:
            raise Configuration(name, n, "rows are contiguous, the codes' pitch a multiple of 16, the scales' of 4")
        return N.PxcBqRows(p, s, n, cr, sr)

    def _vectors(self, vectors):
        """(n, dim), an array in one of the types."""
        if _is_cuda(vectors):
            v = vectors
            if v.ndim == 2 and v.shape[1] == self.dim:
                return v
        else:
            v = _host_vectors(vectors)
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
        n, dim, ld, sld = len(v), self.dim, self._ld, self._sld
        if _is_cuda(v):
            t = _torch_parts or _torch()
            code = _codes.get(v.dtype)
            if code is None:
                code = _dtype_code(v.dtype)
            stream = self._stream(t, v)
            row, step = v.stride()
            if (step != 1 and dim > 1) or (row < dim and n > 1):
                v = v.contiguous()
                row = dim
            codes = t.empty(n, ld, dtype=t.uint8, device=v.device)
            scales = codes.new_empty(n, sld)
            rows = N.PxcBqRows(codes.data_ptr(), scales.data_ptr(), n, ld, sld)
            t.encode(self.ctx.handle, self._caller, v.data_ptr(), code, row if n > 1 else dim, dim, C.byref(rows),
                     stream)
            return BlockCodes(codes, scales, dim)
        v = np.ascontiguousarray(v)
        codes, scales = np.zeros((n, ld), np.uint8), np.zeros((n, sld), np.uint8)
        rows = N.PxcBqRows(N.ptr(codes), N.ptr(scales), n, ld, sld)
        self._host("pxc_bq_encode", N.ptr(v), _dtype_code(v.dtype), self.dim, self.dim, C.byref(rows))
        return BlockCodes(codes, scales, self.dim)

    def decode(self, codes: BlockCodes, dtype=None):
        """The vectors that the rows stand for, rounded once to ``dtype`` (float32)."""
        cuda = _is_cuda(codes.codes)
        rows = self._rows(codes, cuda, "codes")
        if cuda:
            t = _torch_parts or _torch()
            dtype = dtype or t.float32
            code = _codes.get(dtype)
            if code is None:
                code = _dtype_code(dtype)
            out = t.empty(rows.rows, self.dim, dtype=dtype, device=codes.codes.device)
            t.decode(self.ctx.handle, self._caller, C.byref(rows), self.dim, out.data_ptr(), code, self.dim,
                     self._stream(t, out))
            return out
        out = np.zeros((len(codes), self.dim), dtype or np.float32)
        self._host("pxc_bq_decode", C.byref(rows), self.dim, N.ptr(out), _dtype_code(out.dtype), self.dim)
        return out

    # -- products --
    def product(self, queries: BlockCodes, base: BlockCodes, dtype=None, out=None):
        """The dot product of every pair of rows, (nq, n): f32 sums of the tensor cores (errors of 1.1 to 1.8
        times those of plain f32 sums measured), rounded once to ``dtype`` (float32). ``out`` may be a
        tensor to write into, its rows strided."""
        cuda = _is_cuda(queries.codes)
        q, b = self._rows(queries, cuda, "queries"), self._rows(base, cuda, "base")
        shape = (q.rows, b.rows)
        if cuda:
            t, dev = _torch_parts or _torch(), queries.codes.device
            stride = shape[1] or 1
            if out is None:
                dtype = dtype or t.float32
                code = _codes.get(dtype)
                if code is None:
                    code = _dtype_code(dtype)
                out = t.empty(*shape, dtype=dtype, device=dev)
            else:
                if (tuple(out.shape) != shape or out.device != dev or (dtype is not None and out.dtype != dtype)
                        or (shape[1] > 1 and out.stride(1) != 1) or (shape[0] > 1 and out.stride(0) < shape[1])):
                    raise Configuration("out", 0, "must be (nq, n) on the operands' device, with contiguous rows")
                code = _dtype_code(out.dtype)
                stride = out.stride(0) if shape[0] > 1 else stride
            t.product(self.ctx.handle, self._caller, C.byref(q), C.byref(b), self.dim, out.data_ptr(), code,
                      stride, self._stream(t, out))
            return out
        if out is not None:
            raise Configuration("out", 0, "is for tensors")
        out = np.zeros(shape, dtype or np.float32)
        self._host("pxc_bq_product", C.byref(q), C.byref(b), self.dim, N.ptr(out), _dtype_code(out.dtype),
               max(shape[1], 1))
        return out

    def grouped_product(self, queries: BlockCodes, query_offsets, base: BlockCodes, base_offsets=None,
                        out_size: int | None = None, dtype=None):
        """Each group's product: group g pairs ``queries[query_offsets[g]:query_offsets[g + 1]]`` with
        ``base[base_offsets[g]:base_offsets[g + 1]]``; either may be empty.

        Without ``base_offsets`` every group has len(base) / groups rows and the result is
        (nq, rows); rows of queries in no group are not written (undefined in a tensor, 0 in an
        array). With them the result is flat: the groups' matrices one after the other. ``out_size`` is its
        length (for tensors, reading the offsets back to find it waits for the device)."""
        cuda = _is_cuda(queries.codes)
        dev = queries.codes.device if cuda else None
        q, b = self._rows(queries, cuda, "queries"), self._rows(base, cuda, "base")
        qo, bo = self._offsets(query_offsets, cuda, dev), self._offsets(base_offsets, cuda, dev)
        if qo is None or len(qo) < 2 or (bo is not None and len(bo) != len(qo)):
            raise Configuration("offsets", 0, "groups + 1 int64 values for the queries, and for the base where given")
        groups = len(qo) - 1
        if bo is None:
            if b.rows % groups:
                raise Configuration("base", b.rows, "without base offsets the rows must be a multiple of the groups")
            shape = (q.rows, b.rows // groups)
            size = shape[0] * shape[1]
        else:
            if out_size is None:
                out_size = int(((qo[1:] - qo[:-1]) * (bo[1:] - bo[:-1])).sum())
            if out_size < 0:
                raise Configuration("offsets", 0, "offsets must rise")
            size = int(out_size)
            shape = (size,)
        if cuda:
            t = _torch_parts or _torch()
            dtype = dtype or t.float32
            code = _codes.get(dtype)
            if code is None:
                code = _dtype_code(dtype)
            out = t.empty(*shape, dtype=dtype, device=dev)
            t.grouped(self.ctx.handle, self._caller, C.byref(q), qo.data_ptr(), C.byref(b), N.ptr(bo), groups,
                      self.dim, out.data_ptr(), code, size, self._stream(t, out))
            return out
        out = np.zeros(shape, dtype or np.float32)
        self._host("pxc_bq_grouped_product", C.byref(q), N.ptr(qo), C.byref(b), N.ptr(bo), groups, self.dim,
               N.ptr(out), _dtype_code(out.dtype), size)
        return out

    def _offsets(self, o, cuda: bool, dev):
        if o is None:
            return None
        if not cuda and _is_cuda(o):
            raise Configuration("offsets", 0, "all operands on one device, or all on the host")
        if cuda:
            if not _is_cuda(o) or o.device != dev or o.dtype != (_torch_parts or _torch()).int64 or o.ndim != 1:
                raise Configuration("offsets", 0, "must be an int64 tensor on the operands' device")
            return o.contiguous()
        o = np.asarray(o)
        if o.ndim != 1 or o.dtype.kind not in "iu":
            raise Configuration("offsets", 0, "must be one row of integers")
        return np.ascontiguousarray(o, np.int64)

    def check(self) -> None:
        """Waits for the current stream and raises a failure that an earlier call of this quantiser left on the
        device; or one of quantisers that are gone, or of C functions called without a caller's number on this stream."""
        if self._gone:
            self._forget()
        N.call("pxc_bq_check_as", self.ctx.handle, self._caller, _torch().current_stream(self.ctx.device) or 1)
