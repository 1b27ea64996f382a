"""Linear layers on 4-bit operands and the kernels that make them (csrc/lowbit.cu, fp4_gemm.cuh, lowbit_rows.cuh).

Formats: ``mxfp4`` — e2m1 values with a power of two per block of 32; ``nvfp4`` — e2m1 values with an e4m3 scale per block of 16 and an
fp32 factor per row; ``fp8`` (norm outputs only) — e4m3 values with an fp32 scale per block of 128, what the fp8 layers read.

``pack_weight`` quantises a matrix (or the matrices of all experts) once; ``quantize`` and ``rms_norm_quantize`` make the rows that ``linear`` and
``experts`` multiply with it.  A block that holds infinity or NaN becomes NaN as a whole (nvfp4: its row).  Every function has a PyTorch restatement
that runs on CPU tensors.
"""
from __future__ import annotations

import ctypes
import functools
import math
import struct

import torch
import torch.nn.functional as F

from . import _native as nv

c_int, c_long = ctypes.c_int, ctypes.c_long

FORMATS = {"mxfp4": 0, "nvfp4": 1, "fp8": 2}
BLOCK = {"mxfp4": 32, "nvfp4": 16, "fp8": 128}
MAX_COLS = 32768                      # a row stays in the registers of one block
ACT = {None: 0, "gelu_tanh": 1, "silu": 2}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def scale_words(fmt: str, cols: int) -> int:
    """Words of four scale bytes a row of a 4-bit format has."""
    return -(-cols // (4 * BLOCK[fmt]))


@functools.lru_cache(maxsize=4096)
def scale_shape(fmt: str, rows: int, cols: int) -> tuple[int, ...]:
    """Shape of the scales of a matrix [rows, cols]: 4-bit formats uint8 [rows / 128, words, 32, 4, 4], where the scale of row r and block b stands at
    [r // 128, b // 4, r % 32, r // 32 % 4, b % 4]; fp8 fp32 [rows, cols / 128]."""
    return (rows, cols // 128) if fmt == "fp8" else (-(-rows // 128), scale_words(fmt, cols), 32, 4, 4)


@functools.lru_cache(maxsize=4096)
def _parts(fmt: str, shape: tuple, gated: bool):
    """What codes of a shape stand for: experts, rows, columns, the scales' shape and type, the shape of the rows' factors."""
    if fmt not in FORMATS:
        raise ValueError(f"format {fmt!r}: one of {', '.join(FORMATS)}")
    if len(shape) not in (2, 3):
        raise ValueError("codes: contiguous uint8 [rows, cols] or [experts, rows, cols], scales contiguous")
    lead, rows, cols = tuple(shape[:-2]), shape[-2], shape[-1] * (1 if fmt == "fp8" else 2)
    step = 128 if fmt == "fp8" else 32
    if cols % step or cols == 0:
        raise ValueError(f"{fmt}: columns ({cols}) must be a multiple of {step}")
    if fmt == "fp8" and lead:
        raise ValueError("fp8: rows of one matrix only")
    if gated and rows % 16:
        raise ValueError(f"gated weight: rows ({rows}) must be a multiple of 16")
    return (lead[0] if lead else None, rows, cols, lead + scale_shape(fmt, rows, cols), torch.float32 if fmt == "fp8" else torch.uint8,
            lead + (rows,) if fmt == "nvfp4" else None)


class QuantRows:
    """Rows in a low-bit format, as the tensor cores read them: a batch's activations [R, K], a weight [N, K], or the weights of experts [E, N, K].

    ``codes`` uint8 [.., R, K / 2] (fp8: [R, K]), element 2 i in the low half of byte i; ``scales`` as ``scale_shape`` says, whose bytes for blocks past K
    (a row's last word) have to be zero: they are multiplied too, by codes of zero, and a NaN there would be one in the row's results; ``row_scale`` fp32
    [.., R] for nvfp4.  ``gated``: the rows of a SwiGLU weight, 8 gate rows, their 8 lift rows, the next 8 gate rows and so on."""

    __slots__ = ("fmt", "gated", "rows", "cols", "experts", "index", "_codes", "_scales", "_row", "_buf", "_ptr", "_seen")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, fmt: str, row_scale: torch.Tensor | None = None, gated: bool = False):
        index = codes.get_device()
        if codes.dtype is not torch.uint8 or not codes.is_contiguous() or not scales.is_contiguous():
            raise ValueError("codes: contiguous uint8 [rows, cols] or [experts, rows, cols], scales contiguous")
        experts, rows, cols, want, dtype, want_row = _parts(fmt, codes.shape, gated)
        if scales.shape != want or scales.dtype is not dtype or scales.get_device() != index:
            raise ValueError(f"{fmt} scales of {tuple(codes.shape)} codes: {want} expected on {codes.device}, got {scales.dtype} {tuple(scales.shape)} on {scales.device}")
        at, sat, rat = codes.data_ptr(), scales.data_ptr(), 0
        if want_row is not None:
            if row_scale is None or row_scale.dtype is not torch.float32 or row_scale.shape != want_row or not row_scale.is_contiguous() \
                    or row_scale.get_device() != index:
                raise ValueError(f"nvfp4 needs fp32 row scales {want_row} on {codes.device}")
            rat = row_scale.data_ptr()
        elif row_scale is not None:
            raise ValueError(f"{fmt} has no row scales")
        if index >= 0 and (at | sat) & 15:
            raise ValueError("codes and scales must begin on 16 bytes")
        self._ptr, self._codes, self._scales, self._row, self._buf = (at, sat, rat), codes, scales, row_scale, None
        self.fmt, self.gated, self.rows, self.cols, self.experts, self.index = fmt, gated, rows, cols, experts, index

    @classmethod
    def _empty(cls, fmt: str, rows: int, cols: int, index: int, experts: int | None = None, gated: bool = False) -> "QuantRows":
        """Rows that a kernel is to write, in one allocation; the three tensors are made when somebody asks for them."""
        q = cls.__new__(cls)
        q._codes = q._scales = q._row = None
        size, scales, row = _layout(fmt, rows, cols, experts or 1)
        q._buf = buf = torch.empty(size, dtype=torch.uint8, device=_device(index))
        q.fmt, q.gated, q.rows, q.cols, q.experts, q.index = fmt, gated, rows, cols, experts, index
        p = buf.data_ptr()
        q._ptr = (p, p + scales, p + row if fmt == "nvfp4" else 0)
        return q

    @classmethod
    def over(cls, buf: torch.Tensor, fmt: str, rows: int, cols: int, experts: int | None = None, gated: bool = False) -> "QuantRows":
        """Rows that lie in ``buf`` (what ``storage`` of such rows is), wherever that is at the time of a call: a module keeps a weight's bytes as a buffer, whose
        data may be moved off the GPU and back."""
        q = cls.__new__(cls)
        q._codes = q._scales = q._row = q._ptr = None
        q._seen = (0, 0, 0)
        q._buf, q.fmt, q.gated, q.rows, q.cols, q.experts, q.index = buf, fmt, gated, rows, cols, experts, buf.get_device()
        return q

    @property
    def _like(self) -> tuple:
        return self.fmt, self.rows, self.cols, self.experts, self.gated

    def storage(self) -> torch.Tensor:
        """Codes, scales and row factors as one uint8 tensor, each on 256 bytes."""
        if self._buf is None:
            size, *at = _layout(self.fmt, self.rows, self.cols, self.experts or 1)
            buf = torch.zeros(size, dtype=torch.uint8, device=self.device)
            for t, o in zip((self.codes, self.scales, self.row_scale), (0, *at)):
                if t is not None:
                    b = t.reshape(-1).view(torch.uint8)
                    buf[o:o + b.numel()] = b
            return buf
        return self._buf

    @property
    def _at(self) -> tuple[int, int, int]:
        """Where codes, scales and row factors lie."""
        if self._ptr is not None:
            return self._ptr
        p = self._buf.data_ptr()
        if p != self._seen[0] or not p:
            size, scales, row = _layout(self.fmt, self.rows, self.cols, self.experts or 1)
            if self._buf.numel() != size or p & 15 or self._buf.get_device() != self.index:
                raise RuntimeError(f"{self!r}: its weights are not in memory (asleep or offloaded), or not on 16 bytes")
            self._seen = (p, p + scales, p + row if self.fmt == "nvfp4" else 0)
        return self._seen

    def __reduce__(self):              # copies have addresses of their own
        if self._ptr is None:
            return QuantRows.over, (self._buf, *self._like)
        return QuantRows, (self.codes, self.scales, self.fmt, self.row_scale, self.gated)

    def _part(self, which: int) -> torch.Tensor:
        _, scales, row = _layout(self.fmt, self.rows, self.cols, self.experts or 1)
        lead = () if self.experts is None else (self.experts,)
        if which == 0:
            shape = (*lead, self.rows, self.cols if self.fmt == "fp8" else self.cols // 2)
            return self._buf[:math.prod(shape)].view(shape)
        if which == 1:
            shape = (*lead, *scale_shape(self.fmt, self.rows, self.cols))
            size = math.prod(shape) * (4 if self.fmt == "fp8" else 1)
            part = self._buf[scales:scales + size]
            return (part.view(torch.float32) if self.fmt == "fp8" else part).view(shape)
        return self._buf[row:row + 4 * self.rows * (self.experts or 1)].view(torch.float32).view(*lead, self.rows)

    @property
    def codes(self) -> torch.Tensor:
        return self._part(0) if self._codes is None else self._codes

    @property
    def scales(self) -> torch.Tensor:
        return self._part(1) if self._scales is None else self._scales

    @property
    def row_scale(self) -> torch.Tensor | None:
        return self._part(2) if self._row is None and self.fmt == "nvfp4" else self._row

    @property
    def shape(self) -> tuple[int, ...]:
        return (self.rows, self.cols) if self.experts is None else (self.experts, self.rows, self.cols)

    @property
    def device(self) -> torch.device:
        return (self._codes if self._buf is None else self._buf).device

    @property
    def is_cuda(self) -> bool:
        return self.index >= 0

    def as_rows(self) -> "QuantRows":
        """A gated weight's rows as those of an ordinary one."""
        return QuantRows.over(self.storage(), self.fmt, self.rows, self.cols, self.experts)

    def __repr__(self):
        return f"QuantRows({self.fmt}, {list(self.shape)}{', gated' if self.gated else ''}, {self.device})"


@functools.lru_cache(maxsize=4096)
def _layout(fmt: str, rows: int, cols: int, experts: int = 1) -> tuple[int, int, int]:
    """Bytes of one allocation for codes, scales and row factors, and where the scales and the factors begin (each on 256 bytes)."""
    if fmt == "fp8":
        n, m, r = rows * cols, rows * cols // 32, 0
    else:
        n, m, r = rows * cols // 2, -(-rows // 128) * scale_words(fmt, cols) * 512, 4 * rows if fmt == "nvfp4" else 0
    n, m, r = (-(-experts * v // 256) * 256 for v in (n, m, r))
    return n + m + r, n, n + m


@functools.lru_cache(maxsize=None)
def _device(index: int) -> torch.device:
    return torch.device("cuda", index)


@functools.lru_cache(maxsize=None)
def _status(index: int) -> int:
    return nv.status_word(_device(index)).data_ptr()


_current, _stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


# operands of an entry point as one block of 8-byte fields (csrc/lowbit.cu, csrc/moe.cu)
_BLOCKS = {"omni_lowbit_rows": "9qd8q", "omni_lowbit_dequantize": "10q", "omni_lowbit_linear": "26q", "omni_lowbit_experts": "35q", "omni_moe_plan_places": "15q"}


@functools.lru_cache(maxsize=None)
def _entry(name: str):
    """``call(*numbers)`` of an entry point; pointers that are absent are 0."""
    lib, pack = nv.lib("moe" if name == "omni_moe_plan_places" else "lowbit"), struct.Struct(_BLOCKS[name]).pack
    getattr(lib._cdll, name).argtypes = [ctypes.c_char_p]
    fn = getattr(lib, name)
    return lambda *fields: fn(pack(*fields))


_bounds = functools.lru_cache(maxsize=None)(nv.bounds_check_enabled)       # as it is when a library is loaded


@functools.lru_cache(maxsize=None)
def _combine():
    """``omni_moe_combine`` with plain Python numbers."""
    lib = nv.lib("moe")
    lib._cdll.omni_moe_combine.argtypes = [{"p": ctypes.c_void_p, "l": c_long, "i": c_int}[k] for k in "pppiiiplplp"]
    return lib.omni_moe_combine


def _rows16(t: torch.Tensor, name: str) -> torch.Tensor:
    """[rows, cols] bf16 whose rows begin on 16 bytes (a copy where they do not); a single row has the pitch ``cols``, whatever its stride says."""
    if t.dtype is not torch.bfloat16:
        raise ValueError(f"{name}: bf16 expected, got {t.dtype}")
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    (rows, cols), (ld, one) = t.shape, t.stride()
    if one != 1 or ld % 8 or t.data_ptr() % 16 or (rows > 1 and ld < cols):
        if rows == 1 and one == 1 and not t.data_ptr() % 16:
            return t.as_strided((1, cols), (cols, 1))
        t = t.clone(memory_format=torch.contiguous_format)       # (contiguous() keeps a single row where it is, pitch and all)
    return t


def _check_cols(fmt: str, cols: int) -> None:
    if fmt not in FORMATS:
        raise ValueError(f"format {fmt!r}: one of {', '.join(FORMATS)}")
    step = 128 if fmt == "fp8" else 32
    if cols % step or not 0 < cols <= MAX_COLS:
        raise ValueError(f"{fmt}: columns ({cols}) must be a multiple of {step} and at most {MAX_COLS}")


# ------------------------------------------------------------------ restatements in PyTorch
def _power(byte):
    byte = byte.to(torch.int32)
    return torch.where(byte == 255, torch.full((), float("nan")), torch.where(byte > 0, byte << 23, 1 << 22).view(torch.float32))


def _quantize_torch(x: torch.Tensor, fmt: str, gated: bool = False) -> QuantRows:
    """``x`` [.., R, K] bf16, exactly as the kernels round."""
    f = x.float()
    rows, cols = f.shape[-2:]
    b = f.unflatten(-1, (-1, BLOCK[fmt]))
    size = b.abs().amax(-1)
    if fmt == "fp8":
        size = size.clamp_min(1e-8)
        scale = size / torch.full_like(size, 448.0)            # a quotient of two tensors: one by a number is a product on a GPU
        q = (b / scale[..., None]).clamp(-448.0, 448.0)
        scale = torch.where(torch.isfinite(size), scale, float("nan"))
        return QuantRows(q.flatten(-2).to(torch.float8_e4m3fn).view(torch.uint8), scale.contiguous(), fmt)
    fine = torch.isfinite(size)
    size = torch.where(fine, size, 0.0)
    row = None
    if fmt == "mxfp4":
        byte = torch.where(size > 0, torch.frexp(size).exponent + 124, 0).clamp(0, 254)
        s, byte = _power(byte), torch.where(fine, byte, 255).to(torch.uint8)
    else:
        most = size.amax(-1, keepdim=True)
        row = torch.where(most > 0, _power((torch.frexp(most).exponent - 11).clamp(min=-126) + 127), 1.0)
        e4 = (size / row / torch.full_like(size, 6.0)).to(torch.float8_e4m3fn)
        s, b = e4.float(), b / row[..., None]
        byte = torch.where(fine, e4.view(torch.uint8), torch.full((), 0x7F, dtype=torch.uint8))
        row = torch.where(fine.all(-1), row[..., 0], float("nan")).contiguous()
    q = torch.where(s[..., None] > 0, b / s[..., None], 0.0).nan_to_num(0.0).flatten(-2)
    a = q.abs()
    code = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    code = code + q.signbit().to(torch.uint8) * 8
    words = scale_words(fmt, cols)
    full = torch.zeros(*byte.shape[:-2], -(-rows // 128) * 128, words * 4, dtype=torch.uint8, device=x.device)
    full[..., :rows, :byte.shape[-1]] = byte
    tiles = full.unflatten(-1, (words, 4)).unflatten(-3, (-1, 4, 32))                # [.., R/128, 4, 32, words, 4]
    n = tiles.dim()
    tiles = tiles.permute(*range(n - 5), n - 5, n - 2, n - 3, n - 4, n - 1).contiguous()
    return QuantRows((code[..., 0::2] + 16 * code[..., 1::2]).contiguous(), tiles, fmt, row, gated)


def _values_torch(q: QuantRows) -> torch.Tensor:
    if q.fmt == "fp8":
        return (q.codes.view(torch.float8_e4m3fn).float().unflatten(-1, (-1, 128)) * q.scales[..., None]).flatten(-2)
    code = torch.stack([q.codes & 15, q.codes >> 4], -1).flatten(-2).long()
    v = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=q.device)[code].unflatten(-1, (-1, BLOCK[q.fmt]))
    n = q.scales.dim()
    byte = q.scales.permute(*range(n - 5), n - 5, n - 2, n - 3, n - 4, n - 1).flatten(-2).flatten(-4, -2)[..., :q.rows, :q.cols // BLOCK[q.fmt]]
    s = _power(byte) if q.fmt == "mxfp4" else byte.contiguous().view(torch.float8_e4m3fn).float()
    v = (v * s[..., None]).flatten(-2)
    return v if q.row_scale is None else v * q.row_scale[..., None]


def _swiglu_torch(y):
    y = y.unflatten(-1, (-1, 2, 8))
    return F.silu(y[..., 0, :].flatten(-2)) * y[..., 1, :].flatten(-2)


# ------------------------------------------------------------------ quantisation
def _rows(x, fmt, experts=None, gated=False) -> QuantRows:
    index = x.get_device()
    if _current() != index:                       # kernels go to the current device's stream
        with torch.cuda.device(index):
            return _rows(x, fmt, experts, gated)
    rows, cols = x.shape
    per = rows // experts if experts else rows
    q = QuantRows._empty(fmt, per, cols, index, experts, gated)
    rc = _entry("omni_lowbit_rows")(x.data_ptr(), x.stride(0), rows, cols, per, FORMATS[fmt], 0, 0, 0, 0.0, 0, 0, 0, 0, *q._at, _stream(index))
    if rc:
        nv.check_rc(rc, "omni_lowbit_rows")
    return q


def quantize(x: torch.Tensor, fmt: str) -> QuantRows:
    """Rows [.., K] of bf16 (K a multiple of 32) as ``mxfp4`` or ``nvfp4`` rows [R, K]."""
    if fmt not in ("mxfp4", "nvfp4"):
        raise ValueError(f"quantize: format {fmt!r}, mxfp4 or nvfp4 expected")
    _check_cols(fmt, x.shape[-1])
    x2 = _rows16(x, "x")
    if not x.is_cuda:
        return _quantize_torch(x2, fmt)
    return _rows(x2, fmt)


def interleave_gated(w: torch.Tensor) -> torch.Tensor:
    """[.., gate rows | lift rows, K] in the row order of a gated weight."""
    f = w.shape[-2] // 2
    if w.shape[-2] % 16:
        raise ValueError(f"gated weight: {w.shape[-2]} rows, a multiple of 16 expected")
    return torch.stack([w[..., :f, :].unflatten(-2, (-1, 8)), w[..., f:, :].unflatten(-2, (-1, 8))], -3).flatten(-4, -2)


def pack_weight(w: torch.Tensor, fmt: str, gated: bool = False) -> QuantRows:
    """A weight [N, K] (or experts' [E, N, K]) of bf16 in a 4-bit format.  ``gated``: its rows are [gate | lift], and ``linear`` and ``experts`` give
    silu(gate) * lift."""
    if fmt not in ("mxfp4", "nvfp4"):
        raise ValueError(f"pack_weight: format {fmt!r}, mxfp4 or nvfp4 expected")
    if w.dim() not in (2, 3):
        raise ValueError(f"pack_weight: [N, K] or [E, N, K] expected, got {tuple(w.shape)}")
    _check_cols(fmt, w.shape[-1])
    if gated:
        w = interleave_gated(w)
    if not w.is_cuda:
        if w.dtype != torch.bfloat16:
            raise ValueError(f"w: bf16 expected, got {w.dtype}")
        return _quantize_torch(w, fmt, gated)
    return _rows(_rows16(w, "w"), fmt, w.shape[0] if w.dim() == 3 else None, gated)


def dequantize(q: QuantRows, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of ``q`` as bf16 or fp32 (4-bit formats quantised here: exactly in either, but for rows of less than 2^-110, whose smallest values are
    below what bf16 has)."""
    if dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"dequantize: bf16 or fp32, got {dtype}")
    if not q.is_cuda:
        return _values_torch(q).to(dtype)
    if _current() != q.index:
        with torch.cuda.device(q.index):
            return dequantize(q, dtype)
    out = torch.empty(q.shape, dtype=dtype, device=_device(q.index))
    codes, scales, row = q._at
    rc = _entry("omni_lowbit_dequantize")(codes, scales, row, q.rows * (q.experts or 1), q.cols, q.rows, FORMATS[q.fmt], int(dtype is torch.float32),
                                          out.data_ptr(), _stream(q.index))
    if rc:
        nv.check_rc(rc, "omni_lowbit_dequantize")
    return out


def rms_norm_quantize(x: torch.Tensor, weight: torch.Tensor, fmt: str, eps: float = 1e-6, residual: torch.Tensor | None = None,
                      total: torch.Tensor | None = None, normed: torch.Tensor | None = None) -> QuantRows:
    """The RMS norm of s = ``x`` (+ ``residual``), rows [.., K] of bf16, in a low-bit format: what the norm, a copy of its input and a quantiser of
    its output would take three passes for.

    ``total`` (may be ``residual`` or ``x``) receives s, ``normed`` the norm itself, both bf16 of ``x``'s shape; s and the norm are rounded to
    bf16 where a store of them would."""
    shape, index = x.shape, x.get_device()
    cols = shape[-1]
    _check_cols(fmt, cols)
    _check_operand("weight", weight, (cols,), index)
    if residual is not None:
        _check_operand("residual", residual, shape, index)
    if total is not None:
        _check_operand("total", total, shape, index)
    if normed is not None:
        _check_operand("normed", normed, shape, index)
    if index < 0:
        for name, t in (("total", total), ("normed", normed)):
            if t is not None and t.dim() == 2:
                _check_apart(name, t)
        s = _rows16(x, "x")
        if residual is not None:
            s = (s.float() + residual.reshape(s.shape).float()).to(x.dtype)
        f = s.float()
        y = (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + eps) * weight.float()).to(x.dtype)
        if total is not None:
            total.copy_(s.view(x.shape))
        if normed is not None:
            normed.copy_(y.view(x.shape))
        return _quantize_torch(y, fmt)

    if _current() != index:
        with torch.cuda.device(index):
            return rms_norm_quantize(x, weight, fmt, eps, residual, total, normed)
    x, weight = _rows16(x, "x"), _aligned(weight)
    rp = lr = tp = lt = np_ = ln = 0
    if residual is not None:
        residual = _rows16(residual, "residual")
        rp, lr = residual.data_ptr(), residual.stride(0)
    if total is not None:
        tp, lt = _out_rows(total, "total", cols)
    if normed is not None:
        np_, ln = _out_rows(normed, "normed", cols)
    rows = x.shape[0]
    q = QuantRows._empty(fmt, rows, cols, index)
    rc = _entry("omni_lowbit_rows")(x.data_ptr(), x.stride(0), rows, cols, rows, FORMATS[fmt], rp, lr, weight.data_ptr(), eps, tp, lt, np_, ln, *q._at, _stream(index))
    if rc:
        nv.check_rc(rc, "omni_lowbit_rows")
    return q


def _out_rows(t: torch.Tensor, name: str, cols: int) -> tuple[int, int]:
    """Where the rows of a result begin, and their pitch."""
    if t.dim() != 2:
        t = t.view(-1, cols)
    (ld, one), at = t.stride(), t.data_ptr()
    if t.shape[0] == 1:
        ld = cols
    if one != 1 or ld % 8 or at % 16:
        raise ValueError(f"{name}: rows must begin on 16 bytes")
    _check_apart(name, t)
    return at, ld


def _check_apart(name: str, t: torch.Tensor) -> None:
    """Rows that a kernel writes must not share memory (an expanded tensor's do).  Other layouts are copied into, which checks them."""
    if t.shape[0] > 1 and t.stride(1) == 1 and t.stride(0) < t.shape[1]:
        raise ValueError(f"{name}: rows overlap (pitch {t.stride(0)}, {t.shape[1]} columns)")


def _aligned(t: torch.Tensor) -> torch.Tensor:
    t = t if t.is_contiguous() else t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


# ------------------------------------------------------------------ products
def linear(x, w: QuantRows, bias: torch.Tensor | None = None, act: str | None = None, residual: torch.Tensor | None = None,
           gate: torch.Tensor | None = None, out: torch.Tensor | None = None, force_tile: int = 0, force_split: int = 0) -> torch.Tensor:
    """residual + gate * act(x @ w.T + bias) in bf16, as ``ops.gemm.linear`` does it; a gated ``w`` gives silu(gate) * lift, without the other operands.

    x: bf16 [.., K], quantised here in w's format, or ``QuantRows`` of that format.  bias [N], residual [.., N] (may be ``out``), gate [B, N] where the
    rows split evenly into B batches."""
    if not isinstance(w, QuantRows) or w.fmt == "fp8" or w.experts is not None:
        raise ValueError(f"w: a packed 4-bit matrix expected, got {w!r}")
    fmt, gated, N = w.fmt, w.gated, w.rows // 2 if w.gated else w.rows
    if act not in ACT:
        raise ValueError(f"act {act!r}: None, 'gelu_tanh' or 'silu'")
    if gated and not (bias is None and act is None and residual is None and gate is None):
        raise ValueError("a gated weight takes no bias, activation, gate or residual")
    if isinstance(x, QuantRows):
        if x.fmt != fmt or x.experts is not None or x.gated:
            raise ValueError(f"x is {x!r}, w {w!r}: rows of the same format expected")
        lead, q, M, cols, index = (x.rows,), x, x.rows, x.cols, x.index
    else:
        lead, q, cols, index = x.shape[:-1], None, x.shape[-1], x.get_device()
        M = lead[0] if len(lead) == 1 else math.prod(lead)
    if cols != w.cols or index != w.index:
        raise ValueError(f"x {list(x.shape)} on {x.device} does not fit w {w!r}")
    if bias is not None:
        _check_operand("bias", bias, (w.rows,), index)
    if residual is not None:
        _check_operand("residual", residual, (*lead, N), index)
    if out is not None:
        _check_operand("out", out, (*lead, N), index)
    if gate is not None and (gate.dim() != 2 or gate.shape[1] != N or gate.shape[0] == 0 or M % gate.shape[0] or gate.stride(1) != 1
                             or gate.dtype is not torch.bfloat16 or gate.get_device() != index):
        raise ValueError(f"gate: bf16 [B, {N}] with B dividing {M} rows expected, got {gate.dtype} {tuple(gate.shape)}")
    if index < 0:
        if out is not None and out.dim() == 2:
            _check_apart("out", out)
        y = _values_torch(q if q is not None else quantize(x, w.fmt)) @ _values_torch(w).t()
        if w.gated:
            y = _swiglu_torch(y)
        if bias is not None:
            y = y + bias.float()
        y = F.gelu(y, approximate="tanh") if act == "gelu_tanh" else F.silu(y) if act == "silu" else y
        if gate is not None:
            y = (y.view(gate.shape[0], -1, N) * gate.float()[:, None]).view(M, N)
        if residual is not None:
            y = y + residual.reshape(M, N).float()
        y = y.to(torch.bfloat16).view(*lead, N)
        return y if out is None else out.copy_(y)
    if _current() != index:
        with torch.cuda.device(index):
            return linear(x, w, bias, act, residual, gate, out, force_tile, force_split)
    raw = ldx = 0
    if q is None:
        _check_cols(fmt, cols)
        x = _rows16(x, "x")
        raw, ldx = x.data_ptr(), x.stride(0)
        q = QuantRows._empty(fmt, M, cols, index)
        nv.count_launches(1)
    if out is None:
        o2 = torch.empty(M, N, dtype=torch.bfloat16, device=_device(index))
        out = o2 if len(lead) == 1 else o2.view(*lead, N)
    else:
        try:
            o2 = out if out.dim() == 2 else out.view(M, N)
        except RuntimeError:                      # rows of several batches that no single pitch reaches
            return out.copy_(linear(x.view(*lead, cols) if raw else x, w, bias, act, residual, gate, None, force_tile, force_split))
        _check_apart("out", o2)
    ldo, yp = o2.stride(), o2.data_ptr()
    rp = bp = gp = lds = per = 0
    ldr = (0, 1)
    if residual is not None:
        r2 = residual if residual.dim() == 2 else residual.reshape(M, N)
        rp, ldr = r2.data_ptr(), r2.stride()
    if N > 1 and (ldo[1] != 1 or ldr[1] != 1):
        raise ValueError("out and residual: the last dimension must be contiguous")
    if bias is not None:
        bias = bias if bias.is_contiguous() else bias.contiguous()
        bp = bias.data_ptr()
    if gate is not None:
        gp, B = gate.data_ptr(), gate.shape[0]
        lds, per = gate.stride(0) if B > 1 else 0, max(1, M // B)
    rc = _entry("omni_lowbit_linear")(raw, ldx, *q._at, *w._at, yp, ldo[0], M, w.rows, cols, FORMATS[fmt], int(gated), bp, ACT[act], gp, lds, per, rp, ldr[0],
                                      force_tile, force_split, _status(index), _stream(index))
    if rc:
        nv.check_rc(rc, "omni_lowbit_linear")
    return out


def _check_operand(name: str, t: torch.Tensor, shape: tuple, index: int) -> None:
    if t.shape != shape or t.dtype is not torch.bfloat16 or t.get_device() != index:
        raise ValueError(f"{name}: bf16 {tuple(shape)} on {'cpu' if index < 0 else _device(index)} expected, got {t.dtype} {tuple(t.shape)} on {t.device}")


@functools.lru_cache(maxsize=1024)
def _expert_layout(fmt: str, pairs: int, max_tiles: int, scale_rows: int, D: int, Fd: int) -> tuple[int, list[int]]:
    """Bytes of the workspace of ``experts`` and where its parts begin: pairs' rows, three tables of tiles, the number of rows, places of pairs and rows, what lies between the
    products, the results; codes, scales and factors of the rows of either product."""
    at, end = [], 0
    for size in (4 * pairs, 4 * max_tiles, 4 * max_tiles, 4 * max_tiles, 4, 4 * pairs, 4 * pairs, 2 * pairs * Fd, 2 * pairs * D,
                 *(v for cols in (D, Fd) for v in (pairs * cols // 2, scale_rows * 4 * scale_words(fmt, cols), 4 * pairs))):
        at.append(end)
        end += -(-size // 256) * 256
    return end, at


def _tile_rows(pairs: int, experts: int) -> int:
    """The most rows of a tile.  128 experts, 2048 -> 768 -> 2048, nvfp4, us with 16, 128, 256: 8 pairs 19.1, 20.3, 22.6; 4 per expert 71, 74, 86; 16: 78, 84, 93; 32: 98, 92, 98;
    64: 148, 106, 114; 128: -, 140, 140; 154: -, 172, 147.  (64 takes as long as 128.)"""
    return 16 if pairs <= 16 * experts else 128 if pairs <= 128 * experts else 256


def experts(x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor, up: QuantRows, down: QuantRows, residual: torch.Tensor | None = None,
            out: torch.Tensor | None = None) -> torch.Tensor:
    """A mixture of experts on chosen experts: out[t] = residual[t] + sum_j weights[t, j] * down[e] (silu(gate) * lift), [gate | lift] = up[e] x[t],
    e = ids[t, j]; ids outside [0, E) add nothing.

    x bf16 [T, D]; ids int32 and weights fp32 [T, k]; up (gated) [E, 2 F, D] and down [E, D, F] of one 4-bit format.  Rows are quantised as they
    are gathered, what leaves ``up`` once more; an expert's result is a bf16 row, their sum is fp32."""
    if not isinstance(up, QuantRows) or up.experts is None or not isinstance(down, QuantRows) or down.experts is None:
        raise ValueError(f"up and down: the packed weights of experts expected, got {up!r} and {down!r}")
    D, Fd, E, fmt, index = up.cols, down.cols, up.experts, up.fmt, up.index
    if not up.gated or down.gated or fmt != down.fmt or E != down.experts or up.rows != 2 * Fd or D != down.rows or index != down.index:
        raise ValueError(f"up {up!r} and down {down!r} do not fit")
    chosen = ids.shape
    T, k = chosen if len(chosen) == 2 else (-1, 0)
    if k < 1 or ids.dtype is not torch.int32 or ids.get_device() != index:
        raise ValueError(f"ids: int32 [T, k] on {up.device} expected, got {ids.dtype} {tuple(chosen)} on {ids.device}")
    if weights.dtype is not torch.float32 or weights.shape != chosen or weights.get_device() != index:
        raise ValueError(f"weights: fp32 {tuple(chosen)} on {up.device} expected, got {weights.dtype} {tuple(weights.shape)} on {weights.device}")
    _check_operand("x", x, (T, D), index)
    if residual is not None:
        _check_operand("residual", residual, (T, D), index)
    if out is not None:
        _check_operand("out", out, (T, D), index)
        _check_apart("out", out)
    if E > 1024:
        raise ValueError(f"at most 1024 experts, got {E}")
    if index < 0:
        xv, y = _values_torch(_quantize_torch(x, fmt)), torch.zeros(T, D)
        for e in range(E):
            t, j = (ids == e).nonzero(as_tuple=True)
            if t.numel():
                one = lambda w: _values_torch(QuantRows(w.codes[e], w.scales[e], fmt, None if w.row_scale is None else w.row_scale[e]))
                h = _swiglu_torch(xv[t] @ one(up).t()).to(x.dtype)
                y.index_add_(0, t, (_values_torch(_quantize_torch(h, fmt)) @ one(down).t()).to(x.dtype).float() * weights[t, j][:, None])
        y = (y if residual is None else y + residual.float()).to(x.dtype)
        return y if out is None else out.copy_(y)
    if out is None:
        out = o2 = torch.empty(T, D, dtype=torch.bfloat16, device=_device(index))
    else:
        o2 = out if out.stride(1) == 1 and out.stride(0) % 8 == 0 and out.data_ptr() % 16 == 0 else torch.empty_like(out, memory_format=torch.contiguous_format)
    if T == 0:
        return out
    if _current() != index:
        with torch.cuda.device(index):
            return experts(x, ids, weights, up, down, residual, out)
    x2 = _rows16(x, "x")
    ids = ids if ids.is_contiguous() else ids.contiguous()
    weights = weights if weights.is_contiguous() else weights.contiguous()
    res = None if residual is None else _rows16(residual, "residual")
    pairs = T * k
    tile = _tile_rows(pairs, E)
    max_tiles, pitch = min(E, pairs) + pairs // tile, 256 if tile > 128 else 128
    scale_rows = max_tiles * pitch
    # one workspace: the plan, both products' rows, what is between them, the experts' results
    size, at = _expert_layout(fmt, pairs, max_tiles, scale_rows, D, Fd)
    work = torch.empty(size, dtype=torch.uint8, device=_device(index))
    base = work.data_ptr()
    row_of_pair, te, tr, tn, n_rows, of_pair, of_row, h, y, *ops = [base + v for v in at]
    if fmt != "nvfp4":
        ops[2] = ops[5] = 0
    status, stream = _status(index), _stream(index)
    if _bounds():
        nv.lib("moe").omni_moe_set_bounds(c_long(pairs), ctypes.c_void_p(status))
    rc = _entry("omni_moe_plan_places")(ids.data_ptr(), pairs, E, 0, E, tile, max_tiles, row_of_pair, te, tr, tn, n_rows, of_pair, pitch, stream)
    rc = rc or _entry("omni_lowbit_experts")(x2.data_ptr(), x2.stride(0), k, pairs, E, FORMATS[fmt], h, y, row_of_pair, of_pair, te, tr, tn, max_tiles, tile, n_rows, of_row, status,
                                             stream, *ops[:3], *up._at, up.rows, D, *ops[3:], *down._at, down.rows, Fd)
    rc = rc or _combine()(y, row_of_pair, weights.data_ptr(), T, k, D, 0 if res is None else res.data_ptr(), 0 if res is None else res.stride(0), o2.data_ptr(),
                          o2.stride(0), stream)
    if rc:
        nv.check_rc(rc, "experts")
    return out if o2 is out else out.copy_(o2)
