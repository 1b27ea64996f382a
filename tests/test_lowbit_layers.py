"""Low-bit weights where the framework uses them: ``FusedLinear``, image pipelines, the Qwen decoder and its engine stage."""
from __future__ import annotations

import types

import pytest
import torch

import lowbit_oracle as O
from vllm_omni_b200.diffusion.layers.linear import FusedLinear
from vllm_omni_b200.diffusion.quantization.fp8 import DiffusionFp8Config, fp8_linear, quantize_layer, quantize_pipeline, quantize_weight_blockwise
from vllm_omni_b200.models.qwen_decoder import DecoderConfig, ModelBatch, PrefillSeg, QwenDecoderModel
from vllm_omni_b200.ops import fused, moe
from vllm_omni_b200.ops import lowbit as L

BF = torch.bfloat16
FMT4 = ("mxfp4", "nvfp4")
U, STEP = 2.0 ** -8, 2.0 ** -23
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def layer(n_in, n_out, bias=True, device="cpu", dtype=BF, seed=0):
    torch.manual_seed(seed)
    m = FusedLinear(n_in, n_out, bias=bias, dtype=dtype, device=device)
    m.weight.data.normal_(0, n_in ** -0.5)
    if bias:
        m.bias.data.normal_()
    return m


def product(x, q):
    """(x's quantised rows times the packed weight, bound of an fp32 sum of it) in 64 bits."""
    a, w = torch.from_numpy(O.value_of(x.double().cpu().numpy(), q.fmt)), torch.from_numpy(O.values(q))
    return a @ w.t(), (a.abs() @ w.abs().t()) * (x.shape[-1] + 2) * STEP


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fmt", FMT4)
def test_fused_linear(fmt, device):
    m = layer(96, 48, device=device)
    m.to_fp4(fmt)
    assert m.quantized and m.weight.numel() == 0
    x = torch.randn(2, 5, 96, device=device).to(BF)
    y, d = product(x.view(10, 96), m.fp4)
    y = y + m.bias.double().cpu()
    assert ((m(x).double().cpu().view(10, 48) - y).abs() <= d + y.abs() * (U + STEP)).all()
    r = torch.randn(2, 5, 48, device=device).to(BF)
    want = m(x, act="silu", residual=r)
    out = torch.zeros(2, 9, 48, device=device, dtype=BF)                 # a slice that no single pitch reaches
    assert m(x, act="silu", residual=r, out=out[:, 2:7], out_rows_per_batch=5, out_batch_stride=9 * 48) is not None
    assert torch.equal(out[:, 2:7], want) and not out[:, :2].any() and not out[:, 7:].any()
    assert torch.equal(m(L.quantize(x, fmt)), m(x).view(10, 48))
    with pytest.raises(ValueError, match="peers"):
        m(x, scatter=(2, 8, [0, 0], 48))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fmt", FMT4)
def test_fused_linear_gated(fmt, device):
    m = layer(96, 64, bias=False, device=device)
    w = m.weight.data.clone()
    plain = layer(96, 64, bias=False, device=device)
    plain.weight.data.copy_(w)
    m.to_fp4(fmt, gated=True)
    plain.to_fp4(fmt)
    x = torch.randn(7, 96, device=device).to(BF)
    y, d = product(x, plain.fp4)
    g, lift, dg, dl = y[:, :32], y[:, 32:], d[:, :32], d[:, 32:]
    s = torch.nn.functional.silu(g)
    tol = 1.1 * dg * (lift.abs() + dl) + (s.abs() + 1.1 * dg) * dl + (s * lift).abs() * (U + 2.0 ** -16) + 1e-30
    assert ((m.swiglu(x).double().cpu() - s * lift).abs() <= tol).all()
    assert torch.equal(m(x), plain(x))                                   # both halves asked for: in the layer's own order
    seen = []
    m.register_forward_hook(lambda mod, a, out: seen.append(out.shape))
    hooked = m.swiglu(x)                                                 # by way of forward, whose output is rounded first
    assert seen == [(7, 64)]
    r = (g.abs() + dg) * U + dg, (lift.abs() + dl) * U + dl
    # (the two-launch SwiGLU takes tanh.approx, 2^-11 of its result)
    assert ((hooked.double().cpu() - s * lift).abs() <= 1.1 * r[0] * (lift.abs() + r[1]) + (s.abs() + 1.1 * r[0]) * r[1] + (s * lift).abs() * 2 * U + g.abs() * lift.abs() * 2.0 ** -11 + 1e-30).all()


@pytest.mark.parametrize("device", DEVICES)
def test_fused_linear_lora(device):
    m = layer(96, 48, device=device)
    x = torch.randn(6, 96, device=device).to(BF)
    A, B = torch.randn(4 * 2, 96, device=device).to(BF) / 10, torch.randn(48, 8, device=device).to(BF)
    m.to_fp4("nvfp4")
    base = m(x)
    m.lora = [(A, B, 0.5)]
    delta = 0.5 * (x.double() @ A.double().t()) @ B.double().t()
    err = (m(x).double() - base.double() - delta).abs()
    size = base.double().abs() + delta.abs() + 0.5 * (x.double().abs() @ A.double().abs().t()) @ B.double().abs().t()
    assert (err <= 8 * U * size + 1e-3).all()                            # eight bf16 roundings of sums no larger than that


def test_fused_linear_of_a_cpu_model_in_fp32():
    m = layer(64, 32, dtype=torch.float32)
    m.to_fp4("mxfp4")
    x = torch.randn(3, 64)
    y = m(x, act="gelu_tanh")
    assert y.dtype == torch.float32
    want = torch.nn.functional.gelu(L.linear(x.to(BF), m.fp4).float() + m.bias, approximate="tanh")
    assert torch.equal(y, want)


@pytest.mark.parametrize("device", DEVICES)
def test_fp8_rows_of_a_norm_feed_the_fp8_layer(device):
    torch.manual_seed(1)
    x, g = torch.randn(9, 256, device=device).to(BF), torch.randn(256, device=device).to(BF)
    w8, sw = quantize_weight_blockwise((torch.randn(128, 256, device=device) / 16).to(BF))
    state = (w8.view(torch.uint8) if device == "cuda" else w8, sw)
    normed = torch.empty_like(x)
    q = L.rms_norm_quantize(x, g, "fp8", normed=normed)
    a, b = fp8_linear(q, state), fp8_linear(normed, state)
    assert a.dtype == BF
    # the layer's own quantiser multiplies by a rounded reciprocal, the norm's restores ties: a code may be off by half a step of e4m3
    S = L.dequantize(q, torch.float32).abs() @ (w8.float().abs() * sw.repeat_interleave(128, 0).repeat_interleave(128, 1)).t()
    assert ((a.float() - b.float()).abs() <= 2 * U * b.float().abs() + S * 2.0 ** -4).all()
    with pytest.raises(ValueError, match="fp8 layer"):
        fp8_linear(L.quantize(x, "mxfp4"), state)


@pytest.mark.parametrize("fmt", FMT4)
def test_pipeline_cpu(fmt):
    from test_accel_features import _run, _tiny
    m = _tiny()
    ref = _run(m)
    n = quantize_pipeline(types.SimpleNamespace(transformer=m), types.SimpleNamespace(
        quantization=fmt, quantization_config=DiffusionFp8Config(min_features=128, ignored_layers=["*txt.mlp_*"])))
    blk = m.blocks[0]
    assert n > 0 and blk.img.to_qkv.fp4 is not None and blk.txt.mlp_up.fp4 is None and m.proj_out.fp4 is None
    out = _run(m)
    assert torch.isfinite(out).all() and not torch.equal(out, ref)
    par = types.SimpleNamespace(tensor_parallel_size=2)
    with pytest.raises(ValueError, match="parallelism"):
        quantize_pipeline(types.SimpleNamespace(transformer=_tiny()), types.SimpleNamespace(quantization=fmt, quantization_config=None, parallel_config=par))
    with pytest.raises(ValueError, match="unsupported"):
        quantize_pipeline(types.SimpleNamespace(transformer=_tiny()), types.SimpleNamespace(quantization="int3", quantization_config=None))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMT4)
def test_pipeline_on_a_gpu(fmt):
    """The tiny transformer in bf16 on the GPU: its layers give what the layers of a copy on the CPU give for the same rows."""
    from vllm_omni_b200.diffusion.models.qwen_image.transformer import QwenImageTransformer2DModel, QwenImageTransformerConfig
    cfg = QwenImageTransformerConfig(num_layers=2, attention_head_dim=128, num_attention_heads=2, joint_attention_dim=64, in_channels=16, out_channels=4,
                                     axes_dims_rope=(16, 56, 56))
    torch.manual_seed(0)
    m = QwenImageTransformer2DModel(cfg, dtype=BF, device="cuda")
    for p in m.parameters():
        if p.dim() > 1:
            p.data.normal_(0, 0.05)
    n = quantize_pipeline(types.SimpleNamespace(transformer=m), types.SimpleNamespace(quantization=fmt, quantization_config={"min_features": 128}))
    assert n >= 16
    seen = []
    for name, mod in m.named_modules():
        if isinstance(mod, FusedLinear) and mod.fp4 is not None:
            mod.register_forward_pre_hook(lambda mod, args, kw, name=name: seen.append((name, mod, args[0].clone())), with_kwargs=True)
    y = m(torch.randn(1, 64, 16, device="cuda").to(BF), torch.randn(1, 6, 64, device="cuda").to(BF), torch.tensor([0.5], device="cuda"), (1, 8, 8))
    assert torch.isfinite(y).all() and len(seen) >= n
    for name, mod, x in seen[:4]:
        rows = x.reshape(-1, x.shape[-1])
        want, d = product(rows, mod.fp4)
        got = L.linear(rows, mod.fp4).double().cpu()
        assert ((got - want).abs() <= d + want.abs() * U + 1e-30).all(), name


# ------------------------------------------------------------------ decoder
def decoder(moe_layers, device, dtype=BF, shared=0, width=128):
    cfg = DecoderConfig(vocab_size=512, hidden_size=width, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=64 if device == "cuda" else 32,
                        intermediate_size=256, num_experts=8 if moe_layers else 0, num_experts_per_tok=2, moe_intermediate_size=64,
                        shared_expert_intermediate_size=shared)
    torch.manual_seed(0)
    m = QwenDecoderModel(cfg, dtype=dtype, device=device)
    for p in m.parameters():
        if p.dim() == 1:
            p.data.normal_(1.0, 0.1)
    return m


def prompt(n, device):
    ids = torch.arange(n, device=device) * 37 % 512
    return ModelBatch(ids, torch.arange(n, device=device), torch.zeros(n, dtype=torch.int32, device=device), [PrefillSeg(0, n, 0, None)])


def by_hand(m, batch):
    """The quantised decoder's forward as the calls it should consist of."""
    cfg, fmt, eps = m.cfg, m.quantization, m.cfg.rms_norm_eps
    (H, Hkv), Dh = m.local_heads, cfg.head_dim
    x, cos, sin = m.rows_and_rotation(batch)
    T = x.shape[0]
    norm = lambda t, g: fused.norm_modulate(t, weight=g, rms=True, eps=eps)
    mul = lambda lin, rows, **kw: L.linear(rows, lin.fp4, lin.bias, **kw) if fmt != "fp8" else fp8_linear(rows, lin.fp8, lin.bias, **kw)
    for i, l in enumerate(m.layers):
        bf16_rows = fmt == "fp8" and cfg.num_experts and i > 0           # what the combining launch of bf16 experts leaves
        rows = norm(x, l.input_layernorm) if bf16_rows else L.rms_norm_quantize(x, l.input_layernorm, fmt, eps)
        qkv = mul(l.qkv_proj, rows)
        fused.qk_norm_rope_(qkv.view(1, T, -1), H, Hkv, Dh, wq=l.q_norm, wk=l.k_norm, cos=cos, sin=sin, interleaved=False, eps=eps)
        a = m.attention_block(l, qkv, batch, None, None, torch.empty(T, H * Dh, dtype=x.dtype, device=x.device))
        x = mul(l.o_proj, a, residual=x)
        if cfg.num_experts:
            xn = norm(x, l.post_attention_layernorm)
            logits = l.router(xn)
            if fmt == "fp8":
                x = moe.moe_forward(xn, logits, l.w13, l.w2, cfg.num_experts_per_tok, cfg.norm_topk_prob, residual=x)
            else:
                ids, w = moe.route(logits, cfg.num_experts_per_tok, cfg.norm_topk_prob)
                x = L.experts(xn, ids, w, l.w13_fp4, l.w2_fp4, residual=x)
        else:
            rows = L.rms_norm_quantize(x, l.post_attention_layernorm, fmt, eps)
            h = L.linear(rows, l.gate_up.fp4) if fmt != "fp8" else fused.silu_mul(mul(l.gate_up, rows))
            x = mul(l.down, h, residual=x)
    return norm(x, m.norm)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("moe_layers", [False, True])
@pytest.mark.parametrize("fmt", (*FMT4, "fp8"))
def test_decoder_is_its_calls(fmt, moe_layers, device):
    m = decoder(moe_layers, device)
    n = m.quantize(fmt)
    assert n == 2 * (2 if moe_layers and fmt == "fp8" else 4) and m.quantization == fmt
    batch = prompt(21, device)
    got, _ = m(batch)
    assert torch.isfinite(got).all() and torch.equal(got, by_hand(m, batch))
    assert torch.equal(m(batch)[0], got)
    with pytest.raises(ValueError, match="already"):
        m.quantize(fmt)


@pytest.mark.parametrize("device", DEVICES)
def test_decoder_with_a_shared_expert(device):
    m = decoder(True, device, shared=64)
    assert m.quantize("nvfp4") == 12
    assert torch.isfinite(m(prompt(9, device))[0]).all()


def test_decoder_in_fp32_on_the_cpu():
    for experts in (False, True):
        m = decoder(experts, "cpu", torch.float32)
        m.quantize("mxfp4")
        assert torch.isfinite(m(prompt(9, "cpu"))[0]).all()


def test_decoder_refusals():
    with pytest.raises(ValueError, match="unsupported"):
        decoder(False, "cpu").quantize("int4")
    with pytest.raises(ValueError, match="hidden_size \\(144\\)"):
        decoder(False, "cpu", width=144).quantize("mxfp4")
    m = decoder(True, "cpu")
    m.quantize("mxfp4")
    group = types.SimpleNamespace(world_size=2, rank_in_group=0)
    with pytest.raises(NotImplementedError):
        m.enable_tensor_parallel(group)
    with pytest.raises(NotImplementedError):
        m.enable_expert_parallel(group)
    m = decoder(False, "cpu")
    m.tp_group = group
    with pytest.raises(NotImplementedError):
        m.quantize("mxfp4")


def generate(**kw):
    from vllm_omni_b200.entrypoints.omni_llm import OmniLLM
    from vllm_omni_b200.inputs.data import SamplingParams
    llm = OmniLLM(None, model_arch="Qwen3ForCausalLM", model_overrides={"tiny": True, **kw.pop("overrides", {})}, load_format="dummy", num_gpu_blocks=64,
                  max_model_len=256, **kw)
    for i in range(3):
        llm.add_request(f"r{i}", {"prompt_token_ids": [(7 * i + j) % 250 for j in range(5 + 9 * i)]}, SamplingParams(temperature=0.0, max_tokens=6))
    done = {}
    while llm.has_unfinished_requests():
        for o in llm.step():
            if o.finished:
                done[o.request_id] = list(o.outputs[0].token_ids)
    return llm, done


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("overrides", [{}, {"moe": True}])
@pytest.mark.parametrize("fmt", FMT4)
def test_engine_stage(fmt, overrides, device):
    if device == "cuda":
        overrides = {**overrides, "head_dim": 128, "vocab_size": 264}
    kw = {} if device == "cuda" else {"device": "cpu"}
    llm, done = generate(quantization=fmt, overrides=dict(overrides), **kw)
    assert llm.model.decoder.quantization == fmt and len(done) == 3 and all(len(t) == 6 for t in done.values())
    _, again = generate(quantization=fmt, overrides=dict(overrides), **kw)
    assert again == done
    with pytest.raises(ValueError, match="unsupported"):
        generate(quantization="int4", **kw)


def test_stage_without_a_decoder_refuses():
    from vllm_omni_b200.entrypoints.omni_llm import OmniLLM
    with pytest.raises(NotImplementedError, match="quantised"):
        OmniLLM(None, model_arch="Tavulix", model_overrides={"tiny": True}, load_format="dummy", num_gpu_blocks=16, quantization="mxfp4", device="cpu")
