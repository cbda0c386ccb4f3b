"""4-bit microscaled matrices: quantisation, and products of two of them.

A matrix is held as 4-bit floats (e2m1) whose blocks of columns share an 8-bit
scale: value = q * s * g.

* ``nvfp4`` -- blocks of 16 columns, s in e4m3, one float32 g per matrix
* ``mxfp4`` -- blocks of 32 columns, s a power of two, g = 1

Unlike the LUT formats, whose products take 16-bit activations, both operands
of these products are 4-bit and the tensor cores multiply them as they are:
activations are quantised row by row (``quantize_fp4``, or fused with the
gate's SiLU: ``silu_mul_quantize_fp4``), weights once at load time
(``FP4Weight``).  ``fp4_matmul`` multiplies rows with one matrix
(``FP4Linear`` quantises and multiplies), ``fp4_grouped_matmul`` runs of rows
with one matrix per run, as the routed experts of a layer need it.

There is no counterpart in the reference (its products take 16-bit
activations: vllm_lut/quant_method.py:230-279).
"""
from __future__ import annotations

import ctypes as C
import functools
import struct
from dataclasses import dataclass
from typing import Optional, Sequence, Union

import torch

from . import _lib

_KIND = {"nvfp4": _lib.FP4_NV, "mxfp4": _lib.FP4_MX}
_BLOCK = {"nvfp4": 16, "mxfp4": 32}
_DT = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}
MIN_GLOBAL_SCALE, MAX_GLOBAL_SCALE = 2.0 ** -100, 2.0 ** 100
MAX_EXPERTS = 1024
MAX_ROWS = 1 << 22  # rows of one product

# looked up once; a torch without CUDA, which has neither, can still import the package
_current_device = getattr(torch._C, "_cuda_getDevice", None)
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)

Scale = Union[None, float, torch.Tensor]


@functools.lru_cache(maxsize=4096)
def _desc(kind: str, rows: int, cols: int) -> _lib.FP4Desc:
    """C description of a matrix (never written to: shared by the calls)."""
    if kind not in _KIND:
        raise ValueError(f"unknown 4-bit kind {kind!r}: 'nvfp4' or 'mxfp4'")
    return _lib.FP4Desc(_KIND[kind], 0, int(rows), int(cols))


@functools.lru_cache(maxsize=None)
def _function(what: str):
    return getattr(_lib.lib(), what)


def _launch(what: str, t: torch.Tensor, stream, *args) -> None:
    """The library's ``blut_<what>`` on t's device and the given (default: current) stream."""
    fn = _function(what)
    dev = t.get_device()
    if dev == _current_device():  # t is on the GPU, so CUDA is set up
        rc = fn(*args, _current_stream(dev) if stream is None else stream.cuda_stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _lib.stream_ptr(stream))
    if rc:
        _lib.check(rc, what[5:])


def _rows2d(x: torch.Tensor, what: str) -> tuple[torch.Tensor, int, int, int, int]:
    """x as a CUDA matrix with contiguous rows (any row pitch), copied only when its rows are not, with its dtype's
    code, rows, columns and row pitch."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor (no CPU path)")
    dt = _DT.get(x.dtype)
    if dt is None:
        raise ValueError(f"{what} must be float16, bfloat16 or float32, not {x.dtype}")
    shape = x.shape
    if len(shape) != 2 or shape[1] == 0:
        raise ValueError(f"{what} must be a matrix [rows, columns] with at least one column")
    rows, cols = shape
    if x.is_contiguous():
        return x, dt, rows, cols, cols
    if x.stride(1) != 1 or x.stride(0) < cols:  # transposed, expanded, overlapping
        return x.contiguous(), dt, rows, cols, cols
    return x, dt, rows, cols, x.stride(0)


def _pitch(x: torch.Tensor) -> int:
    """Elements between rows; a single row's stride says nothing."""
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _overlap(rows: int, a: int, a_pitch: int, a_width: int, b: int, b_pitch: int, b_width: int) -> bool:
    """Whether two matrices of as many rows may share a byte (address, bytes between rows, bytes of a row)."""
    if a + (rows - 1) * a_pitch + a_width <= b or b + (rows - 1) * b_pitch + b_width <= a:
        return False
    if a_pitch != b_pitch or rows == 1:
        return True
    d = (b - a) % a_pitch  # columns of one array side by side
    return d < a_width or d + b_width > a_pitch


def _scale_tensor(g: Scale, n: int, device: torch.device, what: str) -> torch.Tensor:
    """g as n float32 values on the device."""
    if isinstance(g, torch.Tensor):
        if g.numel() != n or g.dtype != torch.float32 or g.device != device:
            raise ValueError(f"{what} must be a float32 tensor of {n} value(s) on {device}")
        return g if n == 1 else g.reshape(n).contiguous()
    g = float(g)
    if not MIN_GLOBAL_SCALE <= g <= MAX_GLOBAL_SCALE:
        raise ValueError(f"{what} must be within 2^-100 .. 2^100, not {g}")
    return torch.full((n,), g, dtype=torch.float32, device=device)


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _bytes_view(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == torch.uint8 else t.view(torch.uint8)


def _data_bytes(kind: str, rows: int, cols: int) -> int:
    """A row takes 64 bytes of codes and 8 (nvfp4) or 4 of scales for 128 columns."""
    return rows * (72 if kind == "nvfp4" else 68) * ((cols + 127) // 128)


@functools.lru_cache(maxsize=4096)
def _tiled_bytes(kind: str, rows: int, cols: int) -> int:
    """Bytes of a matrix in the tiled layout."""
    n = int(_lib.lib().blut_fp4_tiled_bytes(C.byref(_desc(kind, rows, cols))))
    if n <= 0:
        raise ValueError(f"no 4-bit weight layout for [{rows}, {cols}]")
    return n


class _Operand:
    """What kernels read through: looked over before the first use after an attribute was assigned, since matrices and
    weights can be made and changed by hand, and a kernel would read past a short buffer, or on the host."""
    _ok = False

    def __setattr__(self, name, value):
        object.__setattr__(self, name, value)
        self.__dict__["_ok"] = False

    def __getstate__(self):  # a copy, or one loaded from a file onto another device, is looked over again
        return {k: v for k, v in self.__dict__.items() if k != "_ok"}

    def _look_over(self, t: torch.Tensor, need: int, n: int, what: str) -> None:
        """t holds the ``need`` bytes of codes and scales, global_scale (if there is one) n values beside it."""
        g = self.global_scale
        if t.dtype is not torch.uint8 or t.numel() < need or not t.is_contiguous():
            raise ValueError(f"{what} must be at least {need} contiguous bytes (uint8)")
        if g is not None and self.kind == "mxfp4":
            raise ValueError("mxfp4 has no global scale")
        if g is not None and (g.dtype is not torch.float32 or g.numel() != n or g.device != t.device or not g.is_contiguous()):
            raise ValueError(f"global_scale must be {n} float32 value(s) on the device of {what}")
        if not t.is_cuda:
            raise ValueError(f"{what} must be a CUDA tensor (no CPU path)")
        self.__dict__["_ok"] = True


@dataclass
class FP4Matrix(_Operand):
    """Rows in 4-bit form, as the quantisers write them (the FP4 layout of ``include/blut.h``): the codes, then the
    scales, in one buffer.  ``global_scale`` float32 [1] (nvfp4; kept as given, not copied) or None (1)."""
    kind: str
    rows: int
    cols: int
    data: torch.Tensor
    global_scale: Optional[torch.Tensor] = None

    @classmethod
    def empty(cls, kind: str, rows: int, cols: int, device, global_scale: Optional[torch.Tensor] = None) -> "FP4Matrix":
        _desc(kind, rows, cols)
        return cls(kind, rows, cols, torch.empty(_data_bytes(kind, rows, cols), dtype=torch.uint8, device=device),
                   global_scale)

    def _codes_bytes(self) -> int:
        return self.rows * 64 * ((self.cols + 127) // 128)

    @property
    def codes(self) -> torch.Tensor:
        """uint8 [Kp / 32, rows, 16], Kp = cols rounded up to 128: 32 columns of a row, the even one in the low half."""
        return self.data[:self._codes_bytes()].view((self.cols + 127) // 128 * 4, self.rows, 16)

    @property
    def scales(self) -> torch.Tensor:
        """uint8 [Kp / 64 (nvfp4) or Kp / 128 (mxfp4), rows, 4]: the scales of four consecutive blocks of a row."""
        return self.data[self._codes_bytes():].view(-1, self.rows, 4)

    def _ptrs(self) -> tuple[int, int]:
        """Addresses of the codes and the scales, which the kernels are about to write."""
        p = self.data.data_ptr()
        return p, p + self.rows * 64 * ((self.cols + 127) // 128)

    def _operand(self) -> tuple[int, int, int]:
        """Addresses of the codes, the scales and the global scale (0: none), which they are about to read."""
        if not self._ok:
            self._look_over(self.data, _data_bytes(self.kind, self.rows, self.cols), 1, "FP4Matrix.data")
        p, g = self.data.data_ptr(), self.global_scale
        return p, p + self.rows * 64 * ((self.cols + 127) // 128), 0 if g is None else g.data_ptr()

    @classmethod
    def from_checkpoint(cls, kind: str, codes: torch.Tensor, scales: torch.Tensor, cols: int,
                        global_scale: Scale = None, stream=None) -> "FP4Matrix":
        """From row-major bytes: codes [rows, nb * B / 2] (even column in the low half), scales [rows, nb]
        (e4m3 or e8m0 bytes), nb = ceil(cols / B), B = 16 (nvfp4) or 32 (mxfp4)."""
        return _import(kind, codes, scales, cols, global_scale, stream=stream)

    @_lib.stream_ordered
    def to_checkpoint(self, stream=None) -> tuple[torch.Tensor, torch.Tensor]:
        """Row-major (codes, scales), the arguments of ``from_checkpoint``."""
        b = _BLOCK[self.kind]
        nb = -(-self.cols // b)
        codes = torch.empty(self.rows, nb * b // 2, dtype=torch.uint8, device=self.data.device)
        scales = torch.empty(self.rows, nb, dtype=torch.uint8, device=self.data.device)
        if self.rows:
            d = _desc(self.kind, self.rows, self.cols)
            _launch("blut_fp4_export", codes, stream, C.byref(d), *self._operand()[:2], codes.data_ptr(), scales.data_ptr())
        return codes, scales


def _new_matrix(kind: str, rows: int, cols: int, x: torch.Tensor, g: Optional[torch.Tensor]) -> FP4Matrix:
    """One to be written on x's device, with a g that has been checked."""
    m = object.__new__(FP4Matrix)
    d = m.__dict__
    d["kind"], d["rows"], d["cols"], d["global_scale"], d["_ok"] = kind, rows, cols, g, True
    d["data"] = x.new_empty(_data_bytes(kind, rows, cols), dtype=torch.uint8)
    return m


@_lib.stream_ordered
def _import(kind, codes, scales, cols, global_scale, stream=None) -> FP4Matrix:
    codes, scales = _bytes_view(codes), _bytes_view(scales)
    rows, cols = codes.shape[0], int(cols)
    d = _desc(kind, rows, cols)
    nb = -(-cols // _BLOCK[kind])
    if cols < 1 or tuple(codes.shape) != (rows, nb * _BLOCK[kind] // 2) or tuple(scales.shape) != (rows, nb):
        raise ValueError(f"{kind} rows of {cols} columns are codes [rows, {nb * _BLOCK[kind] // 2}] and scales "
                         f"[rows, {nb}], not {tuple(codes.shape)} and {tuple(scales.shape)}")
    if not codes.is_cuda or scales.device != codes.device:
        raise ValueError("codes and scales must be CUDA tensors of one device")
    codes, scales = codes.contiguous(), scales.contiguous()
    g = _given_scale(kind, global_scale, codes.device)
    m = _new_matrix(kind, rows, cols, codes, g)
    if rows:
        _launch("blut_fp4_import", codes, stream, C.byref(d), codes.data_ptr(), scales.data_ptr(), *m._ptrs())
    return m


def _given_scale(kind: str, g: Scale, device, what: str = "global_scale") -> Optional[torch.Tensor]:
    """The matrix' own scale as the kernels take it: none for mxfp4, 1 where none is given for nvfp4."""
    if kind == "mxfp4":
        if g is not None:
            raise ValueError("mxfp4 has no global scale")
        return None
    return _scale_tensor(1.0 if g is None else g, 1, device, what)


@_lib.stream_ordered
def fp4_global_scale(x: torch.Tensor, silu_mul: bool = False, stream=None) -> torch.Tensor:
    """The nvfp4 scale g of x [rows, cols], float32 [1]: max|x| / 2688 over the finite values (at least 2^-100), with
    which the largest block's scale is 448, e4m3's last.  ``silu_mul``: of silu(gate) * up, x = [gate | up]."""
    x, dt, rows, width, ld = _rows2d(x, "x")
    return _global_scale(x, dt, rows, _gate_cols(width) if silu_mul else width, ld, silu_mul, stream)


def _global_scale(x, dt, rows, cols, ld, silu_mul, stream) -> torch.Tensor:
    buf = x.new_empty(4, dtype=torch.float32)
    if rows == 0:
        return buf.fill_(MIN_GLOBAL_SCALE)[:1]
    _launch("blut_fp4_global_scale", x, stream, x.data_ptr(), dt, rows, cols, ld, int(silu_mul), buf.data_ptr())
    return buf[:1]


def _gate_cols(width: int) -> int:
    if width % 2:
        raise ValueError(f"rows of gate and up have an even width, not {width}")
    return width // 2


@_lib.stream_ordered
def quantize_fp4(x: torch.Tensor, kind: str = "nvfp4", global_scale: Scale = None,
                 row_index: Optional[torch.Tensor] = None, stream=None) -> FP4Matrix:
    """x [rows, cols] (float16, bfloat16 or float32, any row pitch) in 4-bit form.

    nvfp4: s = e4m3(max|x| / (6 g)) per 16 columns; mxfp4: s = 2^(floor(log2 max|x|) - 2) per 32; q = e2m1(x / (s g)).
    Roundings go by the exact quotients (nearest, ties to even, saturating); a block with an infinity or a NaN gets
    the scale NaN.  ``global_scale`` (nvfp4): g as a float or a float32 [1] tensor, 2^-100 .. 2^100; None
    takes ``fp4_global_scale(x)``.  ``row_index`` int32 [n]: row i of the result is x[row_index[i]] (gathered in
    the same pass), a row of zeros where the index is outside x.
    """
    x, dt, rows, cols, ld = _rows2d(x, "x")
    n = rows
    if row_index is not None:
        if row_index.dim() != 1 or row_index.dtype != torch.int32 or row_index.device != x.device:
            raise ValueError("row_index must be an int32 vector on x's device")
        row_index = row_index.contiguous()
        n = row_index.shape[0]
    d = _desc(kind, n, cols)
    if global_scale is None and kind == "nvfp4":
        g = _global_scale(x, dt, rows, cols, ld, False, stream)
    else:
        g = _given_scale(kind, global_scale, x.device)
    m = _new_matrix(kind, n, cols, x, g)
    if n == 0:
        return m
    if rows == 0:  # every index is outside x
        m.data.zero_()
        return m
    _launch("blut_fp4_quantize", x, stream, C.byref(d), x.data_ptr(), dt, ld, _p(row_index), rows, _p(g), *m._ptrs())
    return m


@_lib.stream_ordered
def silu_mul_quantize_fp4(gate_up: torch.Tensor, kind: str = "nvfp4", global_scale: Scale = None,
                          stream=None) -> FP4Matrix:
    """silu(gate) * up in 4-bit form, gate_up = [gate | up] [rows, 2 cols] as the gate/up products write it; rounded
    once, from the exact product to its code.  Arguments as ``quantize_fp4``."""
    x, dt, rows, width, ld = _rows2d(gate_up, "gate_up")
    cols = _gate_cols(width)
    d = _desc(kind, rows, cols)
    if global_scale is None and kind == "nvfp4":
        g = _global_scale(x, dt, rows, cols, ld, True, stream)
    else:
        g = _given_scale(kind, global_scale, x.device)
    m = _new_matrix(kind, rows, cols, x, g)
    if rows == 0:
        return m
    _launch("blut_fp4_silu_mul_quantize", x, stream, C.byref(d), x.data_ptr(), dt, ld, _p(g), *m._ptrs())
    return m


@_lib.stream_ordered
def dequantize_fp4(q: FP4Matrix, dtype: torch.dtype = torch.bfloat16, stream=None) -> torch.Tensor:
    """The values q stands for, [rows, cols] in ``dtype`` (float32 products, rounded once to 16 bits)."""
    dt = _DT.get(dtype)
    if dt is None:
        raise ValueError(f"dtype must be float16, bfloat16 or float32, not {dtype}")
    out = q.data.new_empty((q.rows, q.cols), dtype=dtype)
    if q.rows == 0:
        return out
    codes, scales, g = q._operand()
    _launch("blut_fp4_dequantize", out, stream, C.byref(_desc(q.kind, q.rows, q.cols)), codes, scales, g, out.data_ptr(), dt, q.cols)
    return out


@dataclass
class FP4Weight(_Operand):
    """One weight matrix [rows, cols], or one per expert, in the products' tiled layout.

    ``experts`` None for a single matrix; ``global_scale`` float32 [max(experts, 1)] (nvfp4) or None.
    """
    kind: str
    rows: int
    cols: int
    experts: Optional[int]
    tiled: torch.Tensor
    stride: int
    global_scale: Optional[torch.Tensor] = None

    @classmethod
    def from_quantized(cls, mats: Union[FP4Matrix, Sequence[FP4Matrix]], stream=None) -> "FP4Weight":
        """Lay out one matrix, or a list of matrices of one kind and shape (the experts)."""
        return _pack(mats, stream=stream)

    @classmethod
    def from_checkpoint(cls, kind: str, codes: torch.Tensor, scales: torch.Tensor, cols: int,
                        global_scale: Scale = None, stream=None) -> "FP4Weight":
        """From row-major bytes (``FP4Matrix.from_checkpoint``), [rows, ...] or [experts, rows, ...] with one global
        scale per expert."""
        return _weight_from_checkpoint(kind, codes, scales, cols, global_scale, stream=stream)

    @classmethod
    def quantize(cls, w: torch.Tensor, kind: str = "nvfp4", stream=None) -> "FP4Weight":
        """From float weights [rows, cols] or [experts, rows, cols], each matrix with a global scale of its own."""
        return _weight_quantize(w, kind, stream=stream)

    def _fits(self) -> None:
        one, n = _tiled_bytes(self.kind, self.rows, self.cols), self.experts or 1
        if n > 1 and self.stride < one:
            raise ValueError(f"FP4Weight.stride must be at least {one}")
        self._look_over(self.tiled, one + (n - 1) * self.stride, n, "FP4Weight.tiled")

    def weight_bytes(self, experts: int = 1) -> int:
        """Bytes streamed for ``experts`` matrices."""
        return experts * self.stride


@_lib.stream_ordered
def _pack(mats, stream=None) -> FP4Weight:
    single = isinstance(mats, FP4Matrix)
    mats = [mats] if single else list(mats)
    if not mats or any((m.kind, m.rows, m.cols, m.data.device) != (mats[0].kind, mats[0].rows, mats[0].cols,
                                                                   mats[0].data.device) for m in mats):
        raise ValueError("FP4Weight needs matrices of one kind, shape and device")
    if len(mats) > MAX_EXPERTS:
        raise ValueError(f"at most {MAX_EXPERTS} experts")
    m0 = mats[0]
    d = _desc(m0.kind, m0.rows, m0.cols)
    stride = _tiled_bytes(m0.kind, m0.rows, m0.cols)
    parts = [m._operand()[:2] for m in mats]
    tiled = torch.empty(len(mats) * stride, dtype=torch.uint8, device=m0.data.device)
    for i, (codes, scales) in enumerate(parts):
        _launch("blut_fp4_pack_tiled", tiled, stream, C.byref(d), codes, scales, tiled.data_ptr() + i * stride)
    g = None
    if m0.kind == "nvfp4":  # (no scale: 1, as in the products)
        g = torch.cat([tiled.new_ones(1, dtype=torch.float32) if m.global_scale is None else m.global_scale.reshape(1) for m in mats])
    return FP4Weight(m0.kind, m0.rows, m0.cols, None if single else len(mats), tiled, stride, g)


@_lib.stream_ordered
def _weight_from_checkpoint(kind, codes, scales, cols, global_scale, stream=None) -> FP4Weight:
    if codes.dim() == 2:
        return _pack(_import(kind, codes, scales, cols, global_scale))
    if codes.dim() != 3 or scales.dim() != 3 or scales.shape[0] != codes.shape[0] or codes.shape[0] == 0:
        raise ValueError("expert codes and scales are [experts, rows, bytes]")
    n = codes.shape[0]
    g = [None] * n
    if kind == "nvfp4":
        g = list(_scale_tensor(1.0 if global_scale is None else global_scale, n, codes.device, "global_scale").split(1))
    elif global_scale is not None:
        raise ValueError("mxfp4 has no global scale")
    return _pack([_import(kind, codes[e], scales[e], cols, g[e]) for e in range(n)])


@_lib.stream_ordered
def _weight_quantize(w, kind, stream=None) -> FP4Weight:
    if w.dim() == 3:
        return _pack([quantize_fp4(w[e], kind) for e in range(w.shape[0])])
    return _pack(quantize_fp4(w, kind))


_MM = struct.Struct("iiqqPqPiiPPPPqPq")  # FP4MMArgs, packed at once: a field at a time takes 1.5 us more of a call


def _mm_args(w: FP4Weight, experts, offsets, out_dtype, x_codes, x_scales, x_scale, x_rows, y, y_ld) -> _lib.FP4MMArgs:
    """The products' arguments: addresses (0: none) of everything but the weight, which is taken as it is now."""
    g = w.global_scale
    if not w._ok:
        w._fits()
    return _lib.FP4MMArgs.from_buffer_copy(_MM.pack(
        _KIND[w.kind], 0, w.rows, w.cols, w.tiled.data_ptr(), w.stride, 0 if g is None else g.data_ptr(), experts, out_dtype,
        offsets, x_codes, x_scales, x_scale, x_rows, y, y_ld))


def _check_out(out: torch.Tensor, m: int, w: FP4Weight, out_dtype: Optional[torch.dtype]) -> None:
    if out.dtype not in _DT or (out_dtype is not None and out.dtype != out_dtype):
        raise ValueError("the output is float16, bfloat16 or float32 (and of out_dtype, where both are given)")
    if tuple(out.shape) != (m, w.rows) or out.get_device() != w.tiled.get_device():
        raise ValueError(f"out must be [{m}, {w.rows}] on {w.tiled.device}")
    if (w.rows > 1 and out.stride(1) != 1) or (m > 1 and out.stride(0) < w.rows):
        raise ValueError("out must have contiguous, separate rows")


def _product(x: FP4Matrix, w: FP4Weight, offsets, out, out_dtype, stream) -> torch.Tensor:
    if not isinstance(x, FP4Matrix) or not isinstance(w, FP4Weight):
        raise ValueError("4-bit products take an FP4Matrix and an FP4Weight")
    if x.kind != w.kind or x.cols != w.cols:
        raise ValueError(f"x is {x.kind} of {x.cols} columns, the weight {w.kind} of {w.cols}")
    if w.tiled.get_device() != x.data.get_device():
        raise ValueError(f"x is on {x.data.device}, the weight on {w.tiled.device}")
    if x.rows > MAX_ROWS:
        raise ValueError(f"at most {MAX_ROWS} rows in one product")
    if out is None:
        if out_dtype is not None and out_dtype not in _DT:
            raise ValueError("the output is float16, bfloat16 or float32")
        out = x.data.new_empty((x.rows, w.rows), dtype=out_dtype or torch.bfloat16)
    else:
        _check_out(out, x.rows, w, out_dtype)
    if x.rows == 0:
        return out
    experts, runs = (0, 0) if offsets is None else (w.experts, offsets.data_ptr())
    a = _mm_args(w, experts, runs, _DT[out.dtype], *x._operand(), x.rows, out.data_ptr(), _pitch(out))
    _launch("blut_fp4_matmul", out, stream, C.byref(a))
    return out


@_lib.stream_ordered
def fp4_matmul(x: FP4Matrix, w: FP4Weight, out: Optional[torch.Tensor] = None,
               out_dtype: Optional[torch.dtype] = None, stream=None) -> torch.Tensor:
    """y = x W^T, [x.rows, w.rows] in bfloat16 (``out_dtype``: or float16, float32); float32 sums."""
    if isinstance(w, FP4Weight) and w.experts is not None:
        raise ValueError("a stack of experts goes through fp4_grouped_matmul")
    return _product(x, w, None, out, out_dtype, stream)


@_lib.stream_ordered
def fp4_grouped_matmul(x: FP4Matrix, w: FP4Weight, offsets: torch.Tensor, out: Optional[torch.Tensor] = None,
                       out_dtype: Optional[torch.dtype] = None, stream=None) -> torch.Tensor:
    """y[t] = W_e x_t for offsets[e] <= t < offsets[e + 1].

    ``offsets`` int32 [experts + 1] on the device, not decreasing; it is read by the kernel, so nothing waits for
    the host and the call can be captured.  Runs may be empty or start anywhere.  Rows of ``out`` outside every run
    (before offsets[0], from offsets[-1]) are left as they were; without ``out`` they are undefined.
    """
    if not isinstance(w, FP4Weight) or not w.experts:
        raise ValueError("fp4_grouped_matmul takes a stack of experts")
    if not isinstance(offsets, torch.Tensor) or offsets.dtype != torch.int32 or tuple(offsets.shape) != (w.experts + 1,) \
            or offsets.device != w.tiled.device:
        raise ValueError(f"offsets must be an int32 vector of {w.experts + 1} on the weights' device")
    return _product(x, w, offsets.contiguous(), out, out_dtype, stream)


def fp4_check_status(device=None, stream=None) -> None:
    """Raise if a device-side wait of the products on ``device`` (default: current) timed out; synchronises."""
    with torch.cuda.device(device) if device is not None else torch.cuda.device(torch.cuda.current_device()):
        _lib.check(_lib.lib().blut_fp4_check_status(_lib.stream_ptr(stream)), "fp4 status")


@functools.lru_cache(maxsize=4096)
def _linear_ws(kind: str, rows: int, cols: int, m: int, given: bool) -> int:
    """Workspace bytes of a linear call on m rows, with or without a given scale of x."""
    need = int(_lib.lib().blut_fp4_linear_workspace_size(C.byref(_desc(kind, rows, cols)), m, int(given)))
    if need < 0:
        raise ValueError(f"at most {MAX_ROWS} rows in one product")
    return need


class FP4Linear:
    """y = x W^T with a 4-bit weight and activations quantised on the way in (``blut_fp4_linear``: the product's weight
    copies start beside the quantisation).

    ``act_scale`` (nvfp4): the activations' global scale, from calibration (float or float32 [1] tensor); None takes
    each call's own maximum (one more pass over x).  ``weight`` and ``act_scale`` can be assigned: each call takes them
    as they are.
    """

    def __init__(self, weight: FP4Weight, act_scale: Scale = None):
        self.weight = weight
        self.act_scale = act_scale

    @property
    def weight(self) -> FP4Weight:
        return self._weight

    @weight.setter
    def weight(self, weight: FP4Weight) -> None:
        if weight.experts is not None:
            raise ValueError("FP4Linear takes a single matrix")
        self._weight = weight

    @property
    def act_scale(self) -> Optional[torch.Tensor]:
        return self._act_scale

    @act_scale.setter
    def act_scale(self, g: Scale) -> None:
        w = self._weight
        self._act_scale = None if g is None else _given_scale(w.kind, g, w.tiled.device, "act_scale")

    @property
    def rows(self) -> int:
        return self._weight.rows

    @property
    def cols(self) -> int:
        return self._weight.cols

    @_lib.stream_ordered
    def forward(self, x: torch.Tensor, out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                stream=None) -> torch.Tensor:
        """x [..., cols] -> [..., rows] in x's dtype (or ``out_dtype``)."""
        w, g = self._weight, self._act_scale
        flat = x.dim() == 2
        if not flat and (x.dim() == 0 or x.shape[-1] != w.cols):
            raise ValueError(f"x must be [..., {w.cols}]")
        x2, dt, m, k, ld = _rows2d(x if flat else x.reshape(-1, w.cols), "x")
        if k != w.cols:
            raise ValueError(f"x must be [..., {w.cols}]")
        dev = x2.get_device()
        if dev != w.tiled.get_device():
            raise ValueError(f"x is on {x.device}, the weight on {w.tiled.device}")
        if g is not None and (w.kind == "mxfp4" or g.get_device() != dev):  # the weight was another one when it was given
            raise ValueError("act_scale: mxfp4 has no global scale" if w.kind == "mxfp4" else f"act_scale must be on {x.device}")
        if out is not None:
            if tuple(out.shape) != tuple(x.shape[:-1]) + (w.rows,):
                raise ValueError(f"out must be {list(x.shape[:-1]) + [w.rows]}")
            y = out if out.dim() == 2 else out.view(-1, w.rows)
            _check_out(y, m, w, out_dtype)
            if _overlap(m, x2.data_ptr(), ld * x2.element_size(), k * x2.element_size(),
                        y.data_ptr(), _pitch(y) * y.element_size(), w.rows * y.element_size()):
                # y is written while other parts of the product still read x
                x2, ld = x2.clone(memory_format=torch.contiguous_format), k
        else:
            if out_dtype is not None and out_dtype not in _DT:
                raise ValueError("the output is float16, bfloat16 or float32")
            y = x2.new_empty((m, w.rows), dtype=out_dtype) if out_dtype else x2.new_empty((m, w.rows))
        if m:
            need = _linear_ws(w.kind, w.rows, w.cols, m, g is not None)
            a = _mm_args(w, 0, 0, _DT[y.dtype], 0, 0, 0 if g is None else g.data_ptr(), m, y.data_ptr(),
                         w.rows if out is None else _pitch(y))
            ws = x2.new_empty(need, dtype=torch.uint8) if need else None
            _launch("blut_fp4_linear", x2, stream, C.byref(a), x2.data_ptr(), dt, ld, _p(ws), need)
        if out is not None:
            return out
        return y if flat else y.reshape(*x.shape[:-1], w.rows)

    __call__ = forward
