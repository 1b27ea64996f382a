"""Linear layers on 4-bit operands (csrc/gemm_fp4_sm100.cu) and the kernels that make them (csrc/lowbit.cu).

Formats: ``mxfp4`` — e2m1 values with a power of two per block of 32; ``nvfp4`` — e2m1 values with an e4m3 scale per block of 16 and an
fp32 factor per row; ``fp8`` (norm outputs only) — e4m3 values with an fp32 scale per block of 128, what the fp8 layers read.

``pack_weight`` quantises a matrix (or the matrices of all experts) once; ``quantize`` and ``rms_norm_quantize`` make the rows that ``linear`` and
``experts`` multiply with it.  A block that holds infinity or NaN becomes NaN as a whole (nvfp4: its row).  Every function has a PyTorch restatement
that runs on CPU tensors.
"""
from __future__ import annotations

import ctypes
import math

import torch
import torch.nn.functional as F

from . import _native as nv

c_int, c_long, c_float = ctypes.c_int, ctypes.c_long, ctypes.c_float

FORMATS = {"mxfp4": 0, "nvfp4": 1, "fp8": 2}
BLOCK = {"mxfp4": 32, "nvfp4": 16, "fp8": 128}
MAX_COLS = 32768                      # a row stays in the registers of one block
ACT = {None: 0, "gelu_tanh": 1, "silu": 2}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def scale_words(fmt: str, cols: int) -> int:
    """Words of four scale bytes a row of a 4-bit format has."""
    return -(-cols // (4 * BLOCK[fmt]))


def scale_shape(fmt: str, rows: int, cols: int) -> tuple[int, ...]:
    """Shape of the scales of a matrix [rows, cols]: 4-bit formats uint8 [rows / 128, words, 32, 4, 4], where the scale of row r and block b stands at
    [r // 128, b // 4, r % 32, r // 32 % 4, b % 4]; fp8 fp32 [rows, cols / 128]."""
    return (rows, cols // 128) if fmt == "fp8" else (-(-rows // 128), scale_words(fmt, cols), 32, 4, 4)


class QuantRows:
    """Rows in a low-bit format, as the tensor cores read them: a batch's activations [R, K], a weight [N, K], or the weights of experts [E, N, K].

    ``codes`` uint8 [.., R, K / 2] (fp8: [R, K]), element 2 i in the low half of byte i; ``scales`` as ``scale_shape`` says; ``row_scale`` fp32
    [.., R] for nvfp4.  ``gated``: the rows of a SwiGLU weight, 8 gate rows, their 8 lift rows, the next 8 gate rows and so on."""

    __slots__ = ("codes", "scales", "row_scale", "fmt", "gated", "rows", "cols", "experts")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, fmt: str, row_scale: torch.Tensor | None = None, gated: bool = False):
        if fmt not in FORMATS:
            raise ValueError(f"format {fmt!r}: one of {', '.join(FORMATS)}")
        if codes.dtype != torch.uint8 or codes.dim() not in (2, 3) or not codes.is_contiguous() or not scales.is_contiguous():
            raise ValueError("codes: contiguous uint8 [rows, cols] or [experts, rows, cols], scales contiguous")
        rows, cols = codes.shape[-2], codes.shape[-1] * (1 if fmt == "fp8" else 2)
        step = 128 if fmt == "fp8" else 32
        if cols % step or cols == 0:
            raise ValueError(f"{fmt}: columns ({cols}) must be a multiple of {step}")
        lead = codes.shape[:-2]
        if fmt == "fp8" and lead:
            raise ValueError("fp8: rows of one matrix only")
        want = lead + scale_shape(fmt, rows, cols)
        if tuple(scales.shape) != want or scales.dtype != (torch.float32 if fmt == "fp8" else torch.uint8) or scales.device != codes.device:
            raise ValueError(f"{fmt} scales of {tuple(codes.shape)} codes: {want} expected on {codes.device}, got {scales.dtype} {tuple(scales.shape)} on {scales.device}")
        if fmt == "nvfp4":
            if row_scale is None or row_scale.dtype != torch.float32 or tuple(row_scale.shape) != lead + (rows,) or not row_scale.is_contiguous() \
                    or row_scale.device != codes.device:
                raise ValueError(f"nvfp4 needs fp32 row scales {lead + (rows,)} on {codes.device}")
        elif row_scale is not None:
            raise ValueError(f"{fmt} has no row scales")
        if gated and rows % 16:
            raise ValueError(f"gated weight: rows ({rows}) must be a multiple of 16")
        self.codes, self.scales, self.row_scale, self.fmt, self.gated = codes, scales, row_scale, fmt, gated
        self.rows, self.cols, self.experts = rows, cols, lead[0] if lead else None

    @property
    def shape(self) -> tuple[int, ...]:
        return (*self.codes.shape[:-1], self.cols)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def out_features(self) -> int:
        return self.rows // 2 if self.gated else self.rows

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.codes, self.scales, self.row_scale) if t is not None)

    def __repr__(self):
        return f"QuantRows({self.fmt}, {list(self.shape)}{', gated' if self.gated else ''}, {self.device})"


class _on:
    """Makes a tensor's device the current one where it is not: kernels go to the current device's stream."""

    def __init__(self, t):
        self.idx = t.device.index

    def __enter__(self):
        self.prev = torch._C._cuda_getDevice()
        if self.prev != self.idx:
            torch._C._cuda_setDevice(self.idx)

    def __exit__(self, *exc):
        if self.prev != self.idx:
            torch._C._cuda_setDevice(self.prev)


def _rows16(t: torch.Tensor, name: str) -> torch.Tensor:
    """[rows, cols] bf16 whose rows begin on 16 bytes (a copy where they do not)."""
    if t.dtype != torch.bfloat16:
        raise ValueError(f"{name}: bf16 expected, got {t.dtype}")
    t = t if t.dim() == 2 else t.reshape(-1, t.shape[-1])
    if t.stride(1) != 1 or t.stride(0) % 8 or t.data_ptr() % 16 or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
    return t


def _check_cols(fmt: str, cols: int) -> None:
    if fmt not in FORMATS:
        raise ValueError(f"format {fmt!r}: one of {', '.join(FORMATS)}")
    step = 128 if fmt == "fp8" else 32
    if cols % step or not 0 < cols <= MAX_COLS:
        raise ValueError(f"{fmt}: columns ({cols}) must be a multiple of {step} and at most {MAX_COLS}")


def _empty(fmt: str, rows: int, cols: int, device, lead=()) -> tuple:
    codes = torch.empty(*lead, rows, cols if fmt == "fp8" else cols // 2, dtype=torch.uint8, device=device)
    scales = torch.empty(*lead, *scale_shape(fmt, rows, cols), dtype=torch.float32 if fmt == "fp8" else torch.uint8, device=device)
    return codes, scales, torch.empty(*lead, rows, dtype=torch.float32, device=device) if fmt == "nvfp4" else None


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
        scale = size.nan_to_num(0.0, float("inf")).clamp_min(1e-8) * torch.tensor(1.0 / 448.0, dtype=torch.float32)
        q = (b * (1.0 / scale)[..., None]).clamp(-448.0, 448.0)
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
def _rows(x, fmt, *, residual=None, gain=None, eps=0.0, total=None, normed=None, group=0, lead=()):
    rows, cols = x.shape
    codes, scales, row = _empty(fmt, rows if not lead else rows // lead[0], cols, x.device, lead)
    ld = lambda t: c_long(0 if t is None else t.stride(0))
    with _on(x):
        rc = nv.lib("lowbit").omni_lowbit_rows(
            nv.ptr(x), ld(x), c_long(rows), c_int(cols), c_long(group or rows), c_int(FORMATS[fmt]), nv.ptr(residual), ld(residual), nv.ptr(gain),
            c_float(eps), nv.ptr(total), ld(total), nv.ptr(normed), ld(normed), nv.ptr(codes), nv.ptr(scales), nv.ptr(row), nv.stream_ptr())
    nv.check_rc(rc, "omni_lowbit_rows")
    return codes, scales, row


def quantize(x: torch.Tensor, fmt: str) -> QuantRows:
    """Rows [.., K] of bf16 (K a multiple of 32) as ``mxfp4`` or ``nvfp4`` rows [R, K]."""
    if fmt not in ("mxfp4", "nvfp4"):
        raise ValueError(f"quantize: format {fmt!r}, mxfp4 or nvfp4 expected")
    _check_cols(fmt, x.shape[-1])
    x2 = _rows16(x, "x")
    if not x.is_cuda:
        return _quantize_torch(x2, fmt)
    codes, scales, row = _rows(x2, fmt)
    return QuantRows(codes, scales, fmt, row)


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
    lead = w.shape[:-2]
    if not w.is_cuda:
        if w.dtype != torch.bfloat16:
            raise ValueError(f"w: bf16 expected, got {w.dtype}")
        return _quantize_torch(w, fmt, gated)
    codes, scales, row = _rows(_rows16(w, "w"), fmt, group=w.shape[-2], lead=tuple(lead))
    return QuantRows(codes, scales, fmt, row, gated)


def dequantize(q: QuantRows, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of ``q`` as bf16 or fp32 (4-bit formats quantised here: exactly in either)."""
    if dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"dequantize: bf16 or fp32, got {dtype}")
    if not q.codes.is_cuda:
        return _values_torch(q).to(dtype)
    out = torch.empty(q.shape, dtype=dtype, device=q.device)
    with _on(out):
        rc = nv.lib("lowbit").omni_lowbit_dequantize(
            nv.ptr(q.codes), nv.ptr(q.scales), nv.ptr(q.row_scale), c_long(q.rows * (q.experts or 1)), c_int(q.cols), c_long(q.rows),
            c_int(FORMATS[q.fmt]), c_int(int(dtype == torch.float32)), nv.ptr(out), nv.stream_ptr())
    nv.check_rc(rc, "omni_lowbit_dequantize")
    return out


def rms_norm_quantize(x: torch.Tensor, weight: torch.Tensor, fmt: str, eps: float = 1e-6, residual: torch.Tensor | None = None,
                      total: torch.Tensor | None = None, normed: torch.Tensor | None = None) -> QuantRows:
    """The RMS norm of s = ``x`` (+ ``residual``), rows [.., K] of bf16, in a low-bit format: what the norm, a copy of its input and a quantiser of
    its output would take three passes for.

    ``total`` (may be ``residual`` or ``x``) receives s, ``normed`` the norm itself, both bf16 of ``x``'s shape; s and the norm are rounded to
    bf16 where a store of them would."""
    cols = x.shape[-1]
    _check_cols(fmt, cols)
    if weight.shape != (cols,) or weight.dtype != torch.bfloat16:
        raise ValueError(f"weight: bf16 [{cols}] expected, got {weight.dtype} {tuple(weight.shape)}")
    for name, t in (("residual", residual), ("total", total), ("normed", normed)):
        if t is not None and (t.shape != x.shape or t.dtype != torch.bfloat16 or t.device != x.device):
            raise ValueError(f"{name}: bf16 {tuple(x.shape)} on {x.device} expected, got {t.dtype} {tuple(t.shape)} on {t.device}")
    if weight.device != x.device:
        raise ValueError(f"weight is on {weight.device}, x on {x.device}")
    if not x.is_cuda:
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

    def out_rows(t, name):
        t2 = t.view(-1, cols)
        if t2.stride(1) != 1 or t2.stride(0) % 8 or t2.data_ptr() % 16:
            raise ValueError(f"{name}: rows must begin on 16 bytes")
        return t2

    x2 = _rows16(x, "x")
    codes, scales, row = _rows(x2, fmt, residual=None if residual is None else _rows16(residual, "residual"), gain=_aligned(weight), eps=eps,
                               total=None if total is None else out_rows(total, "total"),
                               normed=None if normed is None else out_rows(normed, "normed"))
    return QuantRows(codes, scales, fmt, row)


def _aligned(t: torch.Tensor) -> torch.Tensor:
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


# ------------------------------------------------------------------ products
def linear(x, w: QuantRows, bias: torch.Tensor | None = None, act: str | None = None, residual: torch.Tensor | None = None,
           gate: torch.Tensor | None = None, out: torch.Tensor | None = None, force_tile: int = 0, force_split: int = 0) -> torch.Tensor:
    """residual + gate * act(x @ w.T + bias) in bf16, as ``ops.gemm.linear`` does it; a gated ``w`` gives silu(gate) * lift, without the other operands.

    x: bf16 [.., K], quantised here in w's format, or ``QuantRows`` of that format.  bias [N], residual [.., N] (may be ``out``), gate [B, N] where the
    rows split evenly into B batches."""
    if not isinstance(w, QuantRows) or w.fmt not in ("mxfp4", "nvfp4") or w.experts is not None:
        raise ValueError(f"w: a packed 4-bit matrix expected, got {w!r}")
    if act not in ACT:
        raise ValueError(f"act {act!r}: None, 'gelu_tanh' or 'silu'")
    if w.gated and not (bias is None and act is None and residual is None and gate is None):
        raise ValueError("a gated weight takes no bias, activation, gate or residual")
    if isinstance(x, QuantRows):
        if x.fmt != w.fmt or x.experts is not None or x.gated:
            raise ValueError(f"x is {x!r}, w {w!r}: rows of the same format expected")
        lead, q = (x.rows,), x
    else:
        lead, q = tuple(x.shape[:-1]), None
    cols = x.shape[-1]
    if cols != w.cols or x.device != w.device:
        raise ValueError(f"x {list(x.shape)} on {x.device} does not fit w {w!r}")
    N, M = w.out_features, math.prod(lead)
    for name, t, shape in (("bias", bias, (w.rows,)), ("residual", residual, (*lead, N)), ("out", out, (*lead, N))):
        if t is not None and (tuple(t.shape) != shape or t.dtype != torch.bfloat16 or t.device != w.device):
            raise ValueError(f"{name}: bf16 {shape} on {w.device} expected, got {t.dtype} {tuple(t.shape)} on {t.device}")
    if gate is not None and (gate.dim() != 2 or gate.shape[1] != N or gate.shape[0] == 0 or M % gate.shape[0] or gate.stride(1) != 1
                             or gate.dtype != torch.bfloat16 or gate.device != w.device):
        raise ValueError(f"gate: bf16 [B, {N}] with B dividing {M} rows expected, got {gate.dtype} {tuple(gate.shape)}")
    if not w.codes.is_cuda:
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
    if q is None:
        q = quantize(x, w.fmt)
    if out is None:
        out = torch.empty(*lead, N, dtype=torch.bfloat16, device=w.device)
    o2 = out.view(M, N)
    r2 = None if residual is None else residual.reshape(M, N)
    if (M > 1 or N > 1) and (o2.stride(1) != 1 or (r2 is not None and r2.stride(1) != 1)):
        raise ValueError("out and residual: the last dimension must be contiguous")
    if bias is not None:
        bias = bias.contiguous()
    with _on(out):
        rc = nv.lib("gemm_fp4_sm100").omni_fp4_linear(
            nv.ptr(q.codes), nv.ptr(q.scales), nv.ptr(q.row_scale), nv.ptr(w.codes), nv.ptr(w.scales), nv.ptr(w.row_scale), nv.ptr(o2),
            c_long(o2.stride(0)), c_long(M), c_int(w.rows), c_int(cols), c_int(FORMATS[w.fmt]), c_int(int(w.gated)), nv.ptr(bias), c_int(ACT[act]),
            nv.ptr(gate), c_long(0 if gate is None or gate.shape[0] == 1 else gate.stride(0)), c_int(0 if gate is None else max(1, M // gate.shape[0])),
            nv.ptr(r2), c_long(0 if r2 is None else r2.stride(0)), c_int(force_tile), c_int(force_split), nv.ptr(nv.status_word(w.device)), nv.stream_ptr())
    nv.check_rc(rc, "omni_fp4_linear")
    return out


def _tile_rows(pairs: int, experts: int) -> int:
    return 64 if pairs <= 32 * experts else 128 if pairs <= 64 * experts else 256


def experts(x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor, up: QuantRows, down: QuantRows, residual: torch.Tensor | None = None,
            out: torch.Tensor | None = None) -> torch.Tensor:
    """A mixture of experts on chosen experts: out[t] = residual[t] + sum_j weights[t, j] * down[e] (silu(gate) * lift), [gate | lift] = up[e] x[t],
    e = ids[t, j]; ids outside [0, E) add nothing.

    x bf16 [T, D]; ids int32 and weights fp32 [T, k]; up (gated) [E, 2 F, D] and down [E, D, F] of one 4-bit format.  Rows are quantised as they
    are gathered, what leaves ``up`` once more; an expert's result is a bf16 row, their sum is fp32."""
    for name, w in (("up", up), ("down", down)):
        if not isinstance(w, QuantRows) or w.experts is None:
            raise ValueError(f"{name}: the packed weights of experts expected, got {w!r}")
    if not up.gated or down.gated or up.fmt != down.fmt or up.experts != down.experts or up.rows != 2 * down.cols or up.cols != down.rows \
            or up.device != down.device:
        raise ValueError(f"up {up!r} and down {down!r} do not fit")
    T, k = ids.shape if ids.dim() == 2 else (-1, 0)
    D, Fd, E, fmt = up.cols, down.cols, up.experts, up.fmt
    if tuple(x.shape) != (T, D) or x.dtype != torch.bfloat16 or x.device != up.device:
        raise ValueError(f"x: bf16 [{T}, {D}] on {up.device} expected, got {x.dtype} {tuple(x.shape)} on {x.device}")
    if ids.dtype != torch.int32 or k < 1 or ids.device != x.device:
        raise ValueError(f"ids: int32 [T, k] on {x.device} expected, got {ids.dtype} {tuple(ids.shape)} on {ids.device}")
    if weights.dtype != torch.float32 or weights.shape != ids.shape or weights.device != x.device:
        raise ValueError(f"weights: fp32 {tuple(ids.shape)} on {x.device} expected, got {weights.dtype} {tuple(weights.shape)} on {weights.device}")
    for name, t in (("residual", residual), ("out", out)):
        if t is not None and (t.shape != x.shape or t.dtype != x.dtype or t.device != x.device):
            raise ValueError(f"{name}: bf16 {tuple(x.shape)} on {x.device} expected, got {t.dtype} {tuple(t.shape)} on {t.device}")
    if E > 1024:
        raise ValueError(f"at most 1024 experts, got {E}")
    if not x.is_cuda:
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
        out = torch.empty(T, D, dtype=x.dtype, device=x.device)
    if T == 0:
        return out
    x2, ids, weights = _rows16(x, "x"), ids.contiguous(), weights.contiguous()
    res = None if residual is None else _rows16(residual, "residual")
    o2 = out if out.stride(1) == 1 and out.stride(0) % 8 == 0 and out.data_ptr() % 16 == 0 else torch.empty_like(out, memory_format=torch.contiguous_format)
    pairs = T * k
    tile = _tile_rows(pairs, E)
    max_tiles, pitch = min(E, pairs) + pairs // tile, 256 if tile > 128 else 128
    dev = x.device
    plan = torch.empty(pairs + 3 * max_tiles + 1, dtype=torch.int32, device=dev)
    row_of_pair, te, tr, tn, n_rows = plan.split([pairs, max_tiles, max_tiles, max_tiles, 1])

    def operand(cols):
        codes = torch.empty(pairs, cols // 2, dtype=torch.uint8, device=dev)
        scales = torch.empty(max_tiles * pitch // 128, scale_words(fmt, cols), 32, 4, 4, dtype=torch.uint8, device=dev)
        return codes, scales, torch.empty(pairs, dtype=torch.float32, device=dev) if fmt == "nvfp4" else None

    h = torch.empty(pairs, Fd, dtype=x.dtype, device=dev)
    y = torch.empty(pairs, D, dtype=x.dtype, device=dev)
    moe, low, g, fc = nv.lib("moe"), nv.lib("lowbit"), nv.lib("gemm_fp4_sm100"), c_int(FORMATS[fmt])
    with _on(x):
        st, status = nv.stream_ptr(), nv.ptr(nv.status_word(dev))
        if nv.bounds_check_enabled():
            moe.omni_moe_set_bounds(c_long(pairs), status)
        nv.check_rc(moe.omni_moe_plan_tiles(nv.ptr(ids), c_int(pairs), c_int(E), c_int(0), c_int(E), c_int(tile), c_int(max_tiles), nv.ptr(row_of_pair),
                                            nv.ptr(te), nv.ptr(tr), nv.ptr(tn), nv.ptr(n_rows), st), "omni_moe_plan_tiles")

        def product(src, per, pair_rows, w, dst):
            (codes, scales, row) = op = operand(w.cols)
            nv.check_rc(low.omni_lowbit_dispatch(nv.ptr(src), c_long(src.stride(0)), c_long(pairs), c_int(per), c_int(w.cols), fc, nv.ptr(pair_rows), nv.ptr(te),
                                                 nv.ptr(tr), nv.ptr(tn), c_int(max_tiles), c_int(pitch), nv.ptr(codes), nv.ptr(scales), nv.ptr(row), st),
                        "omni_lowbit_dispatch")
            nv.check_rc(g.omni_fp4_experts(nv.ptr(codes), nv.ptr(scales), nv.ptr(row), nv.ptr(w.codes), nv.ptr(w.scales), nv.ptr(w.row_scale), c_int(E),
                                           nv.ptr(dst), c_long(dst.stride(0)), c_long(pairs), c_int(w.rows), c_int(w.cols), fc, c_int(int(w.gated)),
                                           nv.ptr(te), nv.ptr(tr), nv.ptr(tn), c_int(max_tiles), c_int(tile), status, st), "omni_fp4_experts")
            return op

        product(x2, k, row_of_pair, up, h)
        product(h, 1, None, down, y)
        nv.check_rc(moe.omni_moe_combine(nv.ptr(y), nv.ptr(row_of_pair), nv.ptr(weights), c_int(T), c_int(k), c_int(D), nv.ptr(res),
                                         c_long(0 if res is None else res.stride(0)), nv.ptr(o2), c_long(o2.stride(0)), st), "omni_moe_combine")
    return out if o2 is out else out.copy_(o2)
