"""What quantised layers compute inside the models that hold them, with every operand they are given there."""
from __future__ import annotations

import pytest
import torch

from vllm_omni_b200.diffusion.layers.linear import FusedLinear
from vllm_omni_b200.ops import fused, moe
from vllm_omni_b200.ops import lowbit as L
from test_lowbit import close, want_linear
from test_lowbit_layers import decoder, prompt
from test_lowbit_state import image_transformer, quantised

BF = torch.bfloat16
FMT4 = ("mxfp4", "nvfp4")
gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]


@gpu
@pytest.mark.parametrize("batch", [1, 2])
@pytest.mark.parametrize("fmt", FMT4)
def test_layers_of_an_image_transformer(fmt, batch):
    """Products, biases, activations, gates, residuals and where results go, against 64 bits, for every quantised layer of both streams of a forward pass."""
    m = quantised(image_transformer(), fmt)
    for p in m.parameters():
        if p.dim() == 1 and p.numel():
            p.data.add_(0.1 * torch.randn_like(p))                           # biases that count
    calls, copied = {}, lambda v: v.clone() if isinstance(v, torch.Tensor) else v
    for name, lin in m.named_modules():
        if isinstance(lin, FusedLinear) and lin.fp4 is not None:
            lin.register_forward_pre_hook(lambda mod, args, kw, name=name: calls.__setitem__(name, [mod, copied(args[0]), {k: copied(v) for k, v in kw.items()}]),
                                          with_kwargs=True)
            lin.register_forward_hook(lambda mod, args, kw, out, name=name: calls[name].append((out.clone(), kw.get("out") is None or out is kw["out"])), with_kwargs=True)
    g = torch.Generator().manual_seed(2)
    m(torch.randn(batch, 64, 16, generator=g).to(BF).cuda(), torch.randn(batch, 6, 64, generator=g).to(BF).cuda(), torch.tensor([0.5], device="cuda").expand(batch),
      (1, 8, 8))
    assert {n.split(".", 2)[2] for n in calls} >= {f"{s}.{l}" for s in ("img", "txt") for l in ("to_qkv", "to_out", "mlp_up", "mlp_down")}
    seen = set()
    for name, (lin, x, kw, (out, placed)) in calls.items():
        rows = x.reshape(-1, x.shape[-1])
        res = kw.get("residual")
        close(out, want_linear(L.quantize(rows, fmt), lin.fp4, lin.bias, kw.get("act"), kw.get("gate"), None if res is None else res.reshape(-1, lin.out_features)))
        assert placed
        seen |= {k for k in ("act", "gate", "residual", "out") if kw.get(k) is not None}
    assert seen == {"act", "gate", "residual", "out"}


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fmt", FMT4)
def test_decoder_with_a_shared_expert_is_its_calls(fmt, device):
    m = decoder(True, device, shared=64)
    for l in m.layers:
        l.shared_expert_gate.data.normal_(0, 0.1)
    m.quantize(fmt)
    batch = prompt(21, device)
    got = m(batch)[0]
    cfg, eps = m.cfg, m.cfg.rms_norm_eps
    (H, Hkv), Dh = m.local_heads, cfg.head_dim
    norm = lambda t, gain: fused.norm_modulate(t, weight=gain, rms=True, eps=eps)
    mul = lambda lin, rows, **kw: L.linear(rows, lin.fp4, lin.bias, **kw)
    x, cos, sin = m.rows_and_rotation(batch)
    T = x.shape[0]
    for l in m.layers:
        qkv = mul(l.qkv_proj, L.rms_norm_quantize(x, l.input_layernorm, fmt, eps))
        fused.qk_norm_rope_(qkv.view(1, T, -1), H, Hkv, Dh, wq=l.q_norm, wk=l.k_norm, cos=cos, sin=sin, interleaved=False, eps=eps)
        x = mul(l.o_proj, m.attention_block(l, qkv, batch, None, None, torch.empty(T, H * Dh, dtype=x.dtype, device=x.device)), residual=x)
        xn = norm(x, l.post_attention_layernorm)
        g = torch.sigmoid(xn.float() @ l.shared_expert_gate.float().t())
        shared = mul(l.shared_down, fused.silu_mul(mul(l.shared_gate_up, xn))).float() * g
        ids, w = moe.route(l.router(xn), cfg.num_experts_per_tok, cfg.norm_topk_prob)
        x = L.experts(xn, ids, w, l.w13_fp4, l.w2_fp4, residual=x)
        x = x + shared.to(x.dtype)
    assert torch.equal(got, norm(x, m.norm))
