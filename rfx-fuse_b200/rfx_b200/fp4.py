"""Matrices in microscaled 4 bits on the device: quantisation, products, nearest rows.

    A = rfx_b200.fp4_quantize(x)              # x: CUDA tensor [rows, cols], float32/bfloat16/float16
    A.dequantize()                            # float32 [rows, cols]
    rfx_b200.fp4_product(A, B)                # A B^T, float32 [A.rows, B.rows]
    rfx_b200.fp4_topk(A, B, 50)               # (indices int32, values float32) [A.rows, 50]

Rows are e2m1 codes with one scale per block of columns: "nvfp4" (16 columns, e4m3 scales and one
power of two for the matrix; the closer of the two) or "mxfp4" (32 columns, power-of-two scales).
include/rfx_b200.h states the formats and the operators exactly.

Calls run on the current torch stream of the tensors' device, allocate from torch's caching
allocator, do not synchronise, and can be captured into a CUDA graph once they have run before.
Tensors made on another stream need the caller's event or ``wait_stream``, as with torch's own
operators, and a matrix that is dropped while another stream than its own still reads it needs
``record_stream``, as a tensor does.  There is no gradient: results never require one.
"""
from __future__ import annotations

import ctypes as C
import operator

from . import _abi as A

FORMATS = A.FP4_FORMATS
_BLOCK = {"mxfp4": 32, "nvfp4": 16}
MAX_ROWS, MAX_COLS = 2 ** 31 - 256, 16776960
TOPK_MAX_COLS = 256
TOPK_MAX_K = 64


# Bound on first use: torch, its dtypes' codes, the library.
_torch = None
_stream = None
_DTYPES = {}
_L = None


def _load():
    global _torch, _L, _stream
    if _L is None:
        import torch
        L = A.load_library()
        _DTYPES.update({torch.float32: 0, torch.bfloat16: 1, torch.float16: 2})
        # the current stream's handle without building a Stream object (3 us of a 14 us call)
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        _stream = raw or (lambda index: torch.cuda.current_stream(index).cuda_stream)
        _torch = torch
        _L = L
    return _L


def _dtype_code(dtype):
    code = _DTYPES.get(dtype)
    if code is None:
        raise TypeError(f"dtype must be float32, bfloat16 or float16, not {dtype}")
    return code


def _check_format(format):
    if format not in FORMATS:
        raise ValueError(f"format must be 'mxfp4' or 'nvfp4', not {format!r}")


def _check_shape(rows, cols):
    if rows > MAX_ROWS or not 1 <= cols <= MAX_COLS:
        raise ValueError(f"a matrix has at most {MAX_ROWS} rows and 1 to {MAX_COLS} columns, not {rows} x {cols}")


def _call(device, fn, *args):
    """fn(*args, stream) with the tensors' device current and its current stream."""
    cuda = _torch.cuda
    index = device.index
    before = cuda.current_device()
    if before == index:
        rc = fn(*args, _stream(index))
    else:
        cuda.set_device(index)
        try:
            rc = fn(*args, _stream(index))
        finally:
            cuda.set_device(before)
    if rc:
        A.check(rc)


class Fp4Matrix:
    """A [rows, cols] matrix in 4 bits on a CUDA device.  Made by ``fp4_quantize`` or
    ``from_parts``; its layout is the library's.  Treated as constant once made."""

    __slots__ = ("format", "shape", "device", "_c", "_p", "_pitch", "_tile_bytes", "_keep")

    def __init__(self, *_):
        raise TypeError("use fp4_quantize or Fp4Matrix.from_parts")

    @classmethod
    def _empty(cls, rows, cols, format, device):
        _check_shape(rows, cols)
        m = object.__new__(cls)
        # the layout of rfx_fp4_sizes
        padded = (cols + 63) // 64 * 64
        tiles = (rows + 127) // 128
        pitch = padded // 2
        tile_bytes = 512 * (padded // 64 if format == "nvfp4" else (padded + 127) // 128)
        codes = (rows * pitch + 255) & ~255
        scales = tiles * tile_bytes
        buf = _torch.empty(codes + scales + 256 + 4 * tiles, dtype=_torch.uint8, device=device)
        p = buf.data_ptr()
        m.format, m.shape, m.device = format, (rows, cols), buf.device
        m._pitch, m._tile_bytes, m._keep = pitch, tile_bytes, buf
        m._set(A.Fp4Struct(FORMATS[format], rows, cols, p, p + codes, p + codes + scales, p + codes + scales + 256))
        return m

    def _set(self, c):
        self._c = c
        self._p = C.addressof(c)

    @classmethod
    def from_parts(cls, codes, scales, scale=None, *, cols, format="nvfp4"):
        """From codes uint8 [rows, ceil(cols / 2)] (two a byte, even column in the low half),
        scale bytes uint8 [rows, ceil(cols / block)] (e8m0 for "mxfp4", unsigned e4m3 for
        "nvfp4") and the matrix scale: a positive number or one-element float32 tensor on the
        same device ("nvfp4" only; None: 1).  A tensor's value is not waited for: where it is not
        positive and finite, every value of the matrix is NaN."""
        L = _load()
        torch = _torch
        _check_format(format)
        cols = int(cols)
        if cols < 1:
            raise ValueError("cols must be at least 1")
        for name, t, width in (("codes", codes, (cols + 1) // 2), ("scales", scales, -(-cols // _BLOCK[format]))):
            if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.uint8:
                raise TypeError(f"{name} must be a CUDA uint8 tensor")
            if t.dim() != 2 or t.shape[1] != width:
                raise ValueError(f"{name} must be [rows, {width}], not {tuple(t.shape)}")
        if codes.shape[0] != scales.shape[0] or codes.device != scales.device:
            raise ValueError("codes and scales must have the same rows and device")
        if isinstance(scale, torch.Tensor):
            if scale.device != codes.device or scale.dtype != torch.float32 or scale.numel() != 1:
                raise ValueError("scale must be one float32 on the codes' device")
            if format == "mxfp4":
                raise ValueError("mxfp4 has no matrix scale")
            scale = scale.resolve_neg()
        elif scale is not None:
            scale = C.c_float(float(scale)).value  # as it is kept
            if not 0.0 < scale < float("inf"):
                raise ValueError("scale must be positive and finite in float32")
            if format == "mxfp4" and scale != 1.0:
                raise ValueError("mxfp4 has no matrix scale")
        m = cls._empty(codes.shape[0], cols, format, codes.device)
        codes, scales = codes.contiguous(), scales.contiguous()
        if scale is not None and not isinstance(scale, torch.Tensor):
            scale = None if scale == 1.0 else torch.full((1,), scale, dtype=torch.float32, device=m.device)
        _call(m.device, L.rfx_fp4_pack, codes.data_ptr(), scales.data_ptr(),
              None if scale is None else scale.data_ptr(), m._p)
        return m

    def parts(self):
        """(codes, scales, scale), the arguments of ``from_parts``."""
        torch = _torch
        rows, cols = self.shape
        codes = torch.empty((rows, (cols + 1) // 2), dtype=torch.uint8, device=self.device)
        scales = torch.empty((rows, -(-cols // _BLOCK[self.format])), dtype=torch.uint8, device=self.device)
        _call(self.device, _L.rfx_fp4_unpack, self._p, codes.data_ptr(), scales.data_ptr())
        if self.format == "mxfp4":
            return codes, scales, None
        at = self._c.scale_dev - self._keep.data_ptr()
        return codes, scales, self._keep[at:at + 4].view(_torch.float32).clone()

    def rows(self, begin, end):
        """Rows [begin, end) as a matrix that shares this one's memory; begin a multiple of 128."""
        n = self.shape[0]
        begin, end = operator.index(begin), operator.index(end)
        if not 0 <= begin <= end <= n:
            raise ValueError(f"rows [{begin}, {end}) are not in [0, {n}]")
        if begin % 128:
            raise ValueError("a view starts at a multiple of 128 rows")
        m = object.__new__(Fp4Matrix)
        m.format, m.shape, m.device = self.format, (end - begin, self.shape[1]), self.device
        m._pitch, m._tile_bytes, m._keep = self._pitch, self._tile_bytes, self._keep
        c = self._c
        m._set(A.Fp4Struct(c.format, end - begin, c.cols, c.codes_dev + begin * self._pitch,
                           c.scales_dev + begin // 128 * self._tile_bytes, c.scale_dev,
                           c.bounds_dev + begin // 128 * 4))
        return m

    def record_stream(self, stream):
        """Tell the allocator that ``stream`` uses this matrix's memory (views share it): it is not
        given out again before that stream's work so far is done."""
        self._keep.record_stream(stream)

    def dequantize(self, dtype=None, *, out=None):
        """The values [rows, cols], rounded once to ``dtype``: exact in float32 and bfloat16 for a
        quantised matrix (magnitudes from 2.9e38 on can read back as infinite; bfloat16 rounds some
        below 2^-128)."""
        if dtype is None:
            dtype = _torch.float32 if out is None else out.dtype
        code = _dtype_code(dtype)
        out = _out(out, self.shape, dtype, self.device)
        _call(self.device, _L.rfx_fp4_dequantize, self._p, 0, self.shape[0], out.data_ptr(), code, _row_stride(out))
        return out

    def __repr__(self):
        return f"Fp4Matrix({self.shape[0]} x {self.shape[1]}, {self.format}, {self.device})"


def _row_stride(t):
    return max(t.stride(0), t.shape[1]) if t.shape[0] > 1 else max(1, t.shape[1])


def _out(out, shape, dtype, device):
    if out is None:
        return _torch.empty(shape, dtype=dtype, device=device)
    if not isinstance(out, _torch.Tensor) or out.device != device or out.dtype != dtype or tuple(out.shape) != tuple(shape):
        raise ValueError(f"out must be a {dtype} tensor of shape {tuple(shape)} on {device}")
    if out.requires_grad or out.is_neg():
        raise ValueError("out must not require a gradient or be a negated view")
    if out.shape[1] > 1 and out.stride(1) != 1 or out.shape[0] > 1 and out.stride(0) < out.shape[1]:
        raise ValueError("out must have unit stride along its rows and rows that do not overlap")
    if not out.is_inference():  # a graph that saved it must not take it for unchanged
        _torch.autograd.graph.increment_version(out)
    return out


def _pair(a, b):
    if not isinstance(a, Fp4Matrix) or not isinstance(b, Fp4Matrix):
        raise TypeError("a and b must be Fp4Matrix")
    if a.format != b.format or a.shape[1] != b.shape[1] or a.device != b.device:
        raise ValueError(f"a and b must share format, columns and device: {a} and {b}")


def fp4_quantize(x, format="nvfp4"):
    """x [rows, cols] (CUDA float32, bfloat16 or float16, unit stride along its rows) in 4 bits."""
    L = _load()
    _check_format(format)
    if not isinstance(x, _torch.Tensor) or not x.is_cuda:
        raise TypeError("x must be a CUDA tensor")
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError("x must be [rows, cols] with at least one column")
    code = _dtype_code(x.dtype)
    rows, cols = x.shape
    s0, s1 = x.stride()
    if cols > 1 and s1 != 1 or rows > 1 and s0 < cols:
        raise ValueError("x must have unit stride along its rows and rows that do not overlap")
    if x.is_neg():
        x = x.resolve_neg()
        s0 = x.stride(0)
    m = Fp4Matrix._empty(rows, cols, format, x.device)
    _call(m.device, L.rfx_fp4_quantize, x.data_ptr(), code, s0 if rows > 1 else cols, m._p)
    return m


def fp4_product(a, b, dtype=None, *, out=None):
    """a b^T [a.rows, b.rows]: fp32 accumulation on the tensor cores, times the matrix scales in
    fp32, then rounded to ``dtype`` (float32 by default, bfloat16 or float16)."""
    _pair(a, b)
    if dtype is None:
        dtype = _torch.float32 if out is None else out.dtype
    code = _dtype_code(dtype)
    out = _out(out, (a.shape[0], b.shape[0]), dtype, a.device)
    _call(a.device, _L.rfx_fp4_product, a._p, b._p, out.data_ptr(), code, _row_stride(out))
    return out


def fp4_topk(queries, rows, k, *, self_offset=None):
    """The k rows with the largest product for every query: (indices int32, values float32)
    [queries, k], exact value descending, then index ascending; slots without a neighbour hold
    -1 and -inf.  self_offset: query i is row self_offset + i of ``rows`` and left out for it.
    k <= 64, at most 256 columns."""
    _pair(queries, rows)
    k = int(k)
    if not 1 <= k <= TOPK_MAX_K:
        raise ValueError(f"k must be in [1, {TOPK_MAX_K}]")
    if queries.shape[1] > TOPK_MAX_COLS:
        raise ValueError(f"fp4_topk takes at most {TOPK_MAX_COLS} columns")
    n = queries.shape[0]
    off = -1
    if self_offset is not None:
        off = int(self_offset)
        if off < 0 or off + n > rows.shape[0]:
            raise ValueError("self_offset must place the queries inside the rows")
    need = C.c_longlong()
    _call(queries.device, _workspace, queries._p, rows._p, k, C.byref(need))
    torch, device = _torch, queries.device
    idx = torch.empty((n, k), dtype=torch.int32, device=device)
    val = torch.empty((n, k), dtype=torch.float32, device=device)
    ws = torch.empty(need.value, dtype=torch.uint8, device=device)
    _call(device, _L.rfx_fp4_topk, queries._p, rows._p, k, off, idx.data_ptr(), val.data_ptr(), ws.data_ptr(),
          need.value)
    return idx, val


def _workspace(a, b, k, need, _stream):
    return _L.rfx_fp4_topk_workspace(a, b, k, need)


def fp4_status(device=None):
    """Wait for the device and raise RfxError if a kernel of fp4_product or fp4_topk on it, on any
    stream, reported a pipeline wait that timed out since the last call (its outputs are incomplete)."""
    _load()
    d = _torch.device("cuda" if device is None else (("cuda:%d" % device) if isinstance(device, int) else device))
    if d.index is None:
        d = _torch.device("cuda", _torch.cuda.current_device())
    _call(d, lambda _stream: _L.rfx_fp4_status())
