"""Linear layer whose forward is the tcgen05 GEMM with a fused epilogue.

The layer keeps the HF/diffusers parameter names (``weight`` [out, in], ``bias`` [out]) so
checkpoints load unchanged.  Optional LoRA deltas (``y += scale * (x A^T) B^T``, the
semantics of vllm_omni/diffusion/lora/layers/base_linear.py), fp8 block-scaled weights and 4-bit
weights attach to the same object.
"""
from __future__ import annotations

import math

import torch
from torch import nn
from torch.nn.modules.module import _has_any_global_hook

from ...ops import gemm


class QuantizedState:
    """Mix-in of modules with quantised weights: their bytes are buffers of the module, so that they move, copy and save with it (and keep their type in a
    cast of the module).  ``quantized_buffers`` names them; the attributes that layers use (``QuantRows``; codes and scales of fp8) share their memory."""

    def set_packed(self, name: str, q) -> None:
        """``self.<name>``: 4-bit weights (ops/lowbit.py ``QuantRows``)."""
        self.register_buffer(name + "_bytes", q.storage())
        setattr(self, name, q.over(getattr(self, name + "_bytes"), *q._like))

    def set_fp8(self, codes: torch.Tensor, scale: torch.Tensor) -> None:
        """``self.fp8``: block-scaled e4m3 codes (bytes on a GPU) and their fp32 scales."""
        self.register_buffer("fp8_codes", codes.view(torch.uint8))
        self.register_buffer("fp8_scale", scale)
        self._over_buffers()

    def quantized_buffers(self) -> list[str]:
        return [n for n in self._buffers if n in ("fp8_codes", "fp8_scale") or n.endswith("_bytes")]

    def _over_buffers(self) -> None:
        """The attributes anew, over what the buffers are now."""
        for n in self.quantized_buffers():
            if n.endswith("_bytes"):
                q = getattr(self, n.removesuffix("_bytes"))
                setattr(self, n.removesuffix("_bytes"), q.over(self._buffers[n], *q._like))
            elif n == "fp8_codes":
                c = self._buffers[n]
                self.fp8 = (c if c.is_cuda else c.view(torch.float8_e4m3fn), self.fp8_scale)

    def _apply(self, fn, recurse=True):
        fp32 = "fp8_scale" in self._buffers                # as whole numbers, which a cast to another floating-point type leaves alone
        if fp32:
            self._buffers["fp8_scale"] = self._buffers["fp8_scale"].view(torch.int32)
        try:
            super()._apply(fn, recurse)
        finally:
            if fp32:
                self._buffers["fp8_scale"] = self._buffers["fp8_scale"].view(torch.float32)
            self._over_buffers()
        return self

    def _load_from_state_dict(self, *args, **kw):
        super()._load_from_state_dict(*args, **kw)
        self._over_buffers()                               # (assign=True puts other tensors in their place)


def weight_tensors(module: nn.Module):
    """(name, tensor) of a module's weights: its parameters and the bytes of its quantised ones."""
    yield from module.named_parameters()
    for prefix, m in module.named_modules():
        if isinstance(m, QuantizedState):
            for n in m.quantized_buffers():
                yield (prefix + "." if prefix else "") + n, m._buffers[n]


class FusedLinear(QuantizedState, nn.Module):
    def __init__(self, in_features: int, out_features: int, bias: bool = True, dtype=torch.bfloat16,
                 device=None, init_std: float = 0.02):
        super().__init__()
        self.in_features, self.out_features = in_features, out_features
        self.weight = nn.Parameter(torch.empty(out_features, in_features, dtype=dtype, device=device),
                                   requires_grad=False)
        self.bias = nn.Parameter(torch.empty(out_features, dtype=dtype, device=device),
                                 requires_grad=False) if bias else None
        self.init_std = init_std
        self.lora = None      # set by the LoRA manager: list of (A [r, in], B [out, r], scale)
        self.fp8 = None       # set by the fp8 quantiser: (w_fp8, w_scale) block-scaled weights
        self.fp4 = None       # set by ``to_fp4``: packed 4-bit weights (ops/lowbit.py)
        self.reset_parameters()

    @torch.no_grad()
    def reset_parameters(self, generator=None):
        if self.weight.device.type == "meta":
            return
        self.weight.normal_(0.0, self.init_std, generator=generator)
        if self.bias is not None:
            self.bias.zero_()

    @property
    def quantized(self) -> bool:
        """The bf16 weight is gone: only the layer itself can compute its product."""
        return self.fp8 is not None or self.fp4 is not None

    @torch.no_grad()
    def to_fp4(self, fmt: str, gated: bool = False) -> None:
        """Replaces the weight by its ``mxfp4`` or ``nvfp4`` form.  ``gated``: its rows are [gate | lift], for layers that are used through ``swiglu``."""
        from ...ops import lowbit
        self.set_packed("fp4", lowbit.pack_weight(self.weight.data.to(torch.bfloat16), fmt, gated=gated))
        self.weight.data = torch.empty(0, dtype=self.weight.dtype, device=self.weight.device)

    def _forward_fp4(self, x, act, residual, gate, out, kw):
        """As the bf16 layer; rows that peers are to receive or send cannot be quantised on the way and are refused."""
        from ...ops import lowbit
        if any(kw.get(k) is not None for k in ("scatter", "row_scatter", "sync")):
            raise ValueError("4-bit weights: no fused exchange with peers (scatter, row_scatter, sync)")
        rows = x.view(-1, x.shape[-1]) if isinstance(x, torch.Tensor) and x.dim() != 2 and x.is_contiguous() else x
        lead = (x.rows,) if isinstance(x, lowbit.QuantRows) else tuple(x.shape[:-1])
        bf16 = isinstance(x, lowbit.QuantRows) or x.dtype == torch.bfloat16
        if not bf16:
            rows = rows.to(torch.bfloat16)             # the CPU's fp32 models: products of 4-bit operands are bf16
        N = self.out_features
        if residual is not None and residual.shape != (*lead, N):
            residual = residual.reshape(*lead, N)      # rows are what counts, as in the bf16 layer
        if out is not None and out.shape != (*lead, N) and out.numel() == math.prod(lead) * N:
            try:
                there = out.view(*lead, N)
            except RuntimeError:                       # no view of these strides: by a result of its own
                return out.copy_(self._forward_fp4(x, act, residual, gate, None, kw).reshape(out.shape))
            self._forward_fp4(x, act, residual, gate, there, kw)
            return out
        if act in lowbit.ACT and bf16 and not self.lora and not self.fp4.gated:
            return lowbit.linear(x, self.fp4, self.bias, act, residual=residual, gate=gate, out=out)
        w = self.fp4
        y = lowbit.linear(rows, w.as_rows() if w.gated else w)
        if w.gated:                                    # asked for as [gate | lift] rows
            y = y.unflatten(-1, (-1, 2, 8)).transpose(-3, -2).flatten(-3)
        y = y.reshape(*lead, N)
        if not bf16:
            y = y.to(x.dtype)
        if self.bias is not None:
            y = y + self.bias
        return _epilogue(self._adapted(y, x), act, residual, gate, out, kw.get("coef", (0.0, 0.0)))

    def _adapted(self, y, x):
        """y + the adapters' products of x (of the values of rows that a norm has quantised)."""
        if self.lora and not isinstance(x, torch.Tensor):
            from ...ops import lowbit
            x = lowbit.dequantize(x)
        for (A, B, scale) in self.lora or ():
            y = y + scale * gemm.linear(gemm.linear(x, A), B)
        return y

    def forward(self, x, act=None, residual=None, gate=None, out=None, **kw):
        if self.fp4 is not None:
            return self._forward_fp4(x, act, residual, gate, out, kw)
        if self.fp8 is not None:
            from ..quantization.fp8 import fp8_linear
            if not self.lora:
                return fp8_linear(x, self.fp8, self.bias, act=act, residual=residual, gate=gate, out=out, **kw)
            y = _epilogue(self._adapted(fp8_linear(x, self.fp8, self.bias), x), act, residual, gate, out, kw.get("coef", (0.0, 0.0)))
        elif self.lora:
            # the LoRA delta enters before the activation / gate, so apply the epilogue last
            y = self._adapted(gemm.linear(x, self.weight, self.bias), x)
            y = _epilogue(y, act, residual, gate, out, kw.get("coef", (0.0, 0.0)))
        else:
            y = gemm.linear(x, self.weight, self.bias, act=act, residual=residual, gate=gate, out=out, **kw)
        return y

    def swiglu(self, x):
        """silu(first half) * second half of the layer's outputs, which exist as such only where something else needs them: adapters, fp8 weights, a bias,
        hooks, a forward of one's own."""
        hooked = self._forward_hooks or self._forward_pre_hooks or self._backward_hooks or self._backward_pre_hooks or _has_any_global_hook()
        if self.fp8 is None and not self.lora and self.bias is None and not hooked and getattr(self.forward, "__func__", None) is FusedLinear.forward:
            if self.fp4 is None:
                return gemm.linear_swiglu(x, self.weight)
            if self.fp4.gated:
                from ...ops import lowbit
                rows = x if isinstance(x, lowbit.QuantRows) or x.dtype == torch.bfloat16 else x.to(torch.bfloat16)
                y = lowbit.linear(rows, self.fp4)
                return y if rows is x else y.to(x.dtype)
        from ...ops import fused
        return fused.silu_mul(self(x))

    def extra_repr(self):
        return f"in={self.in_features}, out={self.out_features}, bias={self.bias is not None}"


def _epilogue(y, act, residual, gate, out, coef=(0.0, 0.0)):
    import torch.nn.functional as F
    if act == "gelu_tanh":
        y = F.gelu(y.float(), approximate="tanh").to(y.dtype)
    elif act == "silu":
        y = F.silu(y)
    elif act == "relu2":
        y = F.relu(y).square()
    elif act == "xielu":
        y = gemm.xielu(y.float(), coef).to(y.dtype)
    if gate is not None:
        B = gate.shape[0]
        y = (y.reshape(B, -1, y.shape[-1]) * gate.unsqueeze(1)).reshape(y.shape)
    if residual is not None:
        y = y + residual
    if out is not None:
        out.copy_(y.reshape(out.shape))
        return out
    return y
