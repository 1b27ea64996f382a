"""Quantised weights as the state of their modules: copies, moves, casts, saved states, sleep and offloading."""
from __future__ import annotations

import copy
import types

import pytest
import torch
from torch import nn

from vllm_omni_b200.diffusion.layers.linear import FusedLinear, weight_tensors
from vllm_omni_b200.diffusion.quantization.fp8 import quantize_layer
from vllm_omni_b200.models.qwen_decoder import DecoderConfig, QwenDecoderModel
from vllm_omni_b200.ops import lowbit as L
from test_lowbit_layers import decoder, prompt
from test_model_zoo import GPU_CASES

BF = torch.bfloat16
FORMATS = ("fp8", "mxfp4", "nvfp4")
gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]


def layer(fmt, device="cpu", seed=0, n_in=256, n_out=128):
    g = torch.Generator().manual_seed(seed)
    m = FusedLinear(n_in, n_out, bias=True, device=device)
    m.weight.data.copy_(torch.randn(n_out, n_in, generator=g) / n_in ** 0.5)
    m.bias.data.copy_(torch.randn(n_out, generator=g))
    if fmt != "bf16":
        quantize_layer(m, fmt)
    return m


def rows(n=5, cols=256, device="cpu"):
    return torch.randn(n, cols, generator=torch.Generator().manual_seed(9)).to(BF).to(device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fmt", FORMATS)
def test_weights_are_the_module_s_state(fmt, device):
    m, x = layer(fmt, device), rows(device=device)
    y = m(x)
    size = sum(t.numel() * t.element_size() for _, t in weight_tensors(m))
    bits = {"fp8": 8, "mxfp4": 4.25, "nvfp4": 4.5}[fmt]
    assert size >= 128 * 256 * bits / 8 + 2 * 128                         # codes, scales and the bias
    other = copy.deepcopy(m)
    assert torch.equal(other(x), y)
    for _, t in weight_tensors(other):                                    # the copy's own memory
        if not t.is_floating_point() or t.dtype == torch.float8_e4m3fn:
            t.view(torch.uint8).zero_()
    assert torch.equal(m(x), y) and not torch.equal(other(x), y)
    fresh = layer(fmt, device, seed=5)
    fresh.load_state_dict(m.state_dict())
    assert torch.equal(fresh(x), y)
    fresh = layer(fmt, device, seed=5)
    fresh.load_state_dict({n: t.clone() for n, t in m.state_dict().items()}, assign=True)
    assert torch.equal(fresh(x), y)
    cast = copy.deepcopy(m).to(torch.float64).to(BF)                      # (the bias survives the way there and back)
    assert torch.equal(cast(x), y)


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_layers_move_between_devices(fmt):
    m, x = layer(fmt, "cuda", n_in=4096, n_out=4096), rows(cols=4096, device="cuda")
    y = m(x)
    before = torch.cuda.memory_allocated()
    m.to("cpu")
    assert before - torch.cuda.memory_allocated() >= 4096 * 4096 // 2
    on_cpu = m(x.cpu())
    assert ((on_cpu.float() - y.cpu().float()).abs() <= 0.05 * y.cpu().float().abs() + 0.05).all()        # the same weights, by the restatement
    m.to("cuda")
    assert torch.equal(m(x), y)


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_states_are_the_same_on_either_side(fmt):
    """A state saved on one side is loaded on the other byte by byte."""
    m, x = layer(fmt, "cuda"), rows(device="cuda")
    y = m(x)
    host = layer(fmt, "cpu", seed=5)
    host.load_state_dict({n: t.cpu() for n, t in m.state_dict().items()})
    back = layer(fmt, "cuda", seed=6)
    back.load_state_dict(host.state_dict())
    assert torch.equal(back(x), y)
    moved = copy.deepcopy(m).to("cpu")
    assert torch.equal(host(x.cpu()), moved(x.cpu()))


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_data_of_buffers_may_be_exchanged(fmt):
    """As sleep and offloading do it: a layer without its bytes refuses, and gives the same again with them back at another address."""
    m, x = layer(fmt, "cuda"), rows(device="cuda")
    y, kept = m(x), {n: t.data for n, t in weight_tensors(m)}
    for _, t in weight_tensors(m):
        t.data = torch.empty(0, dtype=t.dtype, device="cuda")
    with pytest.raises((RuntimeError, IndexError, ValueError)):
        m(x)
    for n, t in weight_tensors(m):
        t.data = kept[n].clone()
        kept[n].view(torch.uint8).fill_(1)
    assert torch.equal(m(x), y)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("experts", [False, True])
@pytest.mark.parametrize("fmt", FORMATS)
def test_copied_decoder(fmt, experts, device):
    m = decoder(experts, device)
    m.quantize(fmt)
    names = [n for n, _ in weight_tensors(m)]
    assert not experts or fmt == "fp8" or {"layers.0.w13_fp4_bytes", "layers.1.w2_fp4_bytes"} <= set(names)
    batch = prompt(9, device)
    want = m(batch)[0].clone()
    other = copy.deepcopy(m)
    for _, t in weight_tensors(m):
        t.view(torch.uint8).zero_()
    assert torch.equal(other(batch)[0], want)


@pytest.mark.parametrize("experts", [0, 4])
def test_decoder_is_quantised_as_a_whole_or_not_at_all(experts):
    """A width that no kernel takes is found before the first matrix is converted."""
    wide = dict(moe_intermediate_size=32800) if experts else dict(intermediate_size=32800)
    m = QwenDecoderModel(DecoderConfig(vocab_size=64, hidden_size=32, num_hidden_layers=1, num_attention_heads=1, num_key_value_heads=1, head_dim=32,
                                       num_experts=experts, num_experts_per_tok=2, **wide), dtype=BF, device="cpu")
    before = {n: t.clone() for n, t in weight_tensors(m)}
    with pytest.raises(ValueError, match="intermediate_size \\(32800\\)"):
        m.quantize("nvfp4")
    assert m.quantization is None and all(torch.equal(t, before[n]) for n, t in weight_tensors(m))


# ------------------------------------------------------------------ operands
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fmt", ("mxfp4", "nvfp4"))
def test_residual_and_out_of_another_shape(fmt, device):
    """Rows are what counts, as in the bf16 layer: [B, S, N] or [B S, N]."""
    m, x = layer(fmt, device), rows(6, 256, device).view(2, 3, 256)
    r = rows(6, 128, device)
    q = L.quantize(x, fmt)
    for act in (None, "relu2"):                                             # in the product's epilogue, and after it
        want = m(x, act=act, residual=r.view(2, 3, 128))
        assert want.shape == (2, 3, 128)
        for res in (r, r.view(1, 6, 128), r.view(3, 2, 128)):
            assert torch.equal(m(x, act=act, residual=res), want)
            assert torch.equal(m(q, act=act, residual=res), want.view(6, 128))
        for out in (torch.zeros_like(r), torch.zeros_like(r).view(1, 6, 128), torch.zeros(6, 136, dtype=BF, device=device)[:, :128],
                    torch.zeros(6, 1, 256, dtype=BF, device=device)[..., :128], torch.zeros(3, 4, 128, dtype=BF, device=device)[:, 1:3]):
            assert m(x, act=act, residual=r, out=out) is out and torch.equal(out.reshape(6, 128), want.view(6, 128))
            own = r.clone().view(out.shape)
            assert m(x, act=act, residual=own, out=own) is own and torch.equal(own.reshape(6, 128), want.view(6, 128))
    for bad in (dict(residual=r[:5]), dict(out=torch.zeros(5, 128, dtype=BF, device=device))):
        with pytest.raises((ValueError, RuntimeError)):
            m(x, **bad)


@gpu
@pytest.mark.parametrize("fmt", ("mxfp4", "nvfp4"))
@pytest.mark.parametrize("name", sorted(GPU_CASES))
def test_every_pipeline_on_a_gpu(name, fmt, monkeypatch):
    """All layers of all transformers that 4 bits can hold, in bf16 on the GPU, through two steps: no operand of theirs is refused."""
    from vllm_omni_b200.diffusion.quantization import fp8
    from vllm_omni_b200.entrypoints.omni_diffusion import OmniDiffusion
    from vllm_omni_b200.inputs import OmniDiffusionSamplingParams
    counted, convert = [], fp8.quantize_pipeline
    monkeypatch.setattr(fp8, "quantize_pipeline", lambda *a: counted.append(convert(*a)))
    tf, vae = GPU_CASES[name]
    o = OmniDiffusion(name, dtype="bfloat16", device="cuda", tf_model_config=tf, quantization=fmt, quantization_config={"min_features": 32},
                      vae_config=vae if vae is not None else dict(block_out_channels=(32, 32, 32, 32), layers_per_block=1, norm_num_groups=8))
    try:
        out = o.generate([{"prompt": "a small test", "negative_prompt": " "}],
                         OmniDiffusionSamplingParams(height=128, width=128, num_inference_steps=2, seed=0, num_frames=5, guidance_scale=3.0,
                                                     extra_args={"audio_seconds": 0.05}))[0]
        assert out.images or out.multimodal_output
        assert len(counted) == 1 and counted[0] > 0
    finally:
        o.close()


@gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_rows_and_weights_on_different_devices(fmt):
    """Refused before a kernel is given an address of the other side."""
    ones = torch.ones(256, dtype=BF)
    here, there = layer(fmt, "cuda"), layer(fmt, "cpu")
    x = rows()
    for m, v in ((there, x.cuda()), (there, L.rms_norm_quantize(x.cuda(), ones.cuda(), fmt)), (here, x), (here, L.rms_norm_quantize(x, ones, fmt))):
        with pytest.raises(ValueError, match=" on "):
            m(v)
    if fmt != "fp8":
        here._buffers["fp4_bytes"].data = here._buffers["fp4_bytes"].data.cpu()
        with pytest.raises(RuntimeError, match="not in memory"):
            here(x.cuda())


# ------------------------------------------------------------------ adapters
def adapters(device, n_in=256, n_out=128):
    g = torch.Generator().manual_seed(3)
    return [((torch.randn(8, n_in, generator=g) / 16).to(BF).to(device), torch.randn(n_out, 8, generator=g).to(BF).to(device), s) for s in (0.5, -0.25)]


def with_deltas(base, x, lora):
    """(base + the adapters' products, bound) in 64 bits: per adapter bf16 roundings of two products, of its scaling and of the sum."""
    y, size = base.double(), base.double().abs()
    for A, B, s in lora:
        y = y + s * (x.double() @ A.double().t()) @ B.double().t()
        size = size + abs(s) * (x.double().abs() @ A.double().abs().t()) @ B.double().abs().t()
    return y, 4 * len(lora) * 2.0 ** -8 * size + 1e-30


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fmt", ("mxfp4", "nvfp4"))
def test_adapters_of_a_layer_that_gets_quantised_rows(fmt, device):
    m, x = layer(fmt, device), rows(device=device)
    q = L.rms_norm_quantize(x, torch.ones(256, dtype=BF, device=device), fmt)
    base = m(q)
    m.lora = adapters(device)
    want, tol = with_deltas(base, L.dequantize(q), m.lora)
    assert ((m(q).double() - want).abs() <= tol).all()
    assert m.swiglu(q).shape == (5, 64)


@pytest.mark.parametrize("device", DEVICES)
def test_adapters_of_an_fp8_layer(device):
    """They take part, before the activation, for rows of bf16 and for rows that a norm has quantised."""
    m, x = layer("fp8", device), rows(device=device)
    q = L.rms_norm_quantize(x, torch.ones(256, dtype=BF, device=device), "fp8")
    plain, normed = m(x), m(q)
    m.lora = adapters(device)
    for got, base, v in ((m(x), plain, x), (m(q), normed, L.dequantize(q))):
        want, tol = with_deltas(base, v, m.lora)
        assert ((got.double() - want).abs() <= tol).all()
    assert torch.equal(m(x, act="silu"), torch.nn.functional.silu(m(x)))


# ------------------------------------------------------------------ sleep
class Denoiser(nn.Module):
    graph_safe_forward = True

    def __init__(self, fmt, device):
        super().__init__()
        self.blocks = nn.ModuleList(layer(fmt, device, seed, 1024, 1024) for seed in range(3))

    def forward(self, x):
        for b in self.blocks:
            x = b(x, act="silu")
        return x


class Pipe(nn.Module):
    def __init__(self, fmt, device="cpu"):
        super().__init__()
        self.transformer = Denoiser(fmt, device)


def worker_of(pipe, device):
    from vllm_omni_b200.diffusion.data import OmniDiffusionConfig
    from vllm_omni_b200.diffusion.worker import DiffusionWorker
    w = DiffusionWorker(0, 0, OmniDiffusionConfig(model="none", diffusion_load_format="dummy"))
    w.device, w.model_runner = torch.device(device), types.SimpleNamespace(pipeline=pipe)
    return w


def test_graphs_of_moving_weights_are_released():
    """On the CPU, with captures that are only names: a pipeline's graphed forwards and its captured loops."""
    from vllm_omni_b200.diffusion.graphed import GraphedForward, _Entry, release_graphs
    pipe = Pipe("bf16")
    f = pipe.transformer.forward = GraphedForward(pipe.transformer.forward)
    f.entries["a"], f.entries["b"] = _Entry(), _Entry()
    f.entries["a"].graph = "captured"
    pipe._loop_cache = {1: types.SimpleNamespace(graph="captured"), 2: types.SimpleNamespace(graph=None)}
    assert release_graphs(pipe) == 2 and not f.entries and not pipe._loop_cache
    assert release_graphs(pipe) == 0


@gpu
def test_sleep_after_a_capture():
    from vllm_omni_b200.diffusion.graphed import maybe_graph_transformer
    pipe, x = Pipe("bf16", "cuda"), rows(5, 1024, "cuda")
    want = pipe.transformer(x).clone()
    assert maybe_graph_transformer(pipe, types.SimpleNamespace(enforce_eager=False))
    w = worker_of(pipe, "cuda")
    for _ in range(2):
        for _ in range(4):
            assert torch.equal(pipe.transformer(x), want)
        assert pipe.transformer.forward.replays
        w.sleep(1)
        assert not pipe.transformer.forward.entries
        held = torch.full((3 * 1024 * 1024,), 7.0, dtype=BF, device="cuda")          # where the weights were
        w.wake_up()
        del held


@gpu
@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("fmt", FORMATS)
def test_sleep_moves_quantised_weights(fmt, captured):
    from vllm_omni_b200.diffusion.graphed import maybe_graph_transformer
    pipe, x = Pipe(fmt, "cuda"), rows(5, 1024, "cuda")
    want = pipe.transformer(x).clone()
    if captured:
        maybe_graph_transformer(pipe, types.SimpleNamespace(enforce_eager=False))
    w = worker_of(pipe, "cuda")
    for _ in range(2):
        for _ in range(3):
            assert torch.equal(pipe.transformer(x), want)
        before = torch.cuda.memory_allocated()
        freed = w.sleep(1)
        assert freed >= 3 * 1024 * 1024 // 2 and before - torch.cuda.memory_allocated() >= freed
        held = torch.full((8 * 1024 * 1024,), 0x55, dtype=torch.uint8, device="cuda")
        w.wake_up()
        del held


def test_weights_of_quantised_layers_are_not_loaded_again():
    for fmt in ("bf16", *FORMATS):
        pipe = Pipe(fmt)
        seen = []
        pipe.load_weights = lambda w: seen.append(dict(w))
        w = worker_of(pipe, "cpu")
        if fmt == "bf16":
            w.load_weights([("a", 1)])
            assert seen == [{"a": 1}]
        else:
            with pytest.raises(NotImplementedError, match="quantised"):
                w.load_weights([("a", 1)])
            assert not seen


# ------------------------------------------------------------------ offloading
def image_transformer():
    from vllm_omni_b200.diffusion.models.qwen_image.transformer import QwenImageTransformer2DModel, QwenImageTransformerConfig
    cfg = QwenImageTransformerConfig(num_layers=3, attention_head_dim=128, num_attention_heads=2, joint_attention_dim=64, in_channels=16, out_channels=4,
                                     axes_dims_rope=(16, 56, 56))
    torch.manual_seed(0)
    m = QwenImageTransformer2DModel(cfg, dtype=BF, device="cuda")
    for p in m.parameters():
        if p.dim() > 1:
            p.data.normal_(0, 0.05)
    return m


def quantised(m, fmt):
    from vllm_omni_b200.diffusion.quantization.fp8 import quantize_pipeline
    if fmt != "bf16":
        assert quantize_pipeline(types.SimpleNamespace(transformer=m), types.SimpleNamespace(quantization=fmt, quantization_config={"min_features": 128})) >= 24
    return m


@gpu
@pytest.mark.parametrize("fmt", ("bf16", *FORMATS))
def test_layerwise_offload(fmt):
    from vllm_omni_b200.diffusion.offloader import LayerWiseOffloadBackend
    args = (torch.randn(1, 64, 16, device="cuda").to(BF), torch.randn(1, 6, 64, device="cuda").to(BF), torch.tensor([0.5], device="cuda"), (1, 8, 8))
    m = quantised(image_transformer(), fmt)
    want = m(*args).clone()
    before = torch.cuda.memory_allocated()
    b = LayerWiseOffloadBackend(torch.device("cuda", 0))
    b.enable(types.SimpleNamespace(transformer=m))
    bits = {"bf16": 16, "fp8": 8, "mxfp4": 4.25, "nvfp4": 4.5}[fmt]
    block = 2 * (4 + 8) * 256 * 256 * bits / 8                               # both streams: qkv and out, MLP up and down
    assert before - torch.cuda.memory_allocated() >= 3 * block and all(h.numel() >= block for h in b.host)
    for _ in range(2):
        assert torch.equal(m(*args), want)
        assert not b.resident


@gpu
@pytest.mark.parametrize("fmt", ("bf16", *FORMATS))
def test_model_level_offload(fmt):
    from vllm_omni_b200.diffusion.offloader import ModelLevelOffloadBackend
    args = (torch.randn(1, 64, 16, device="cuda").to(BF), torch.randn(1, 6, 64, device="cuda").to(BF), torch.tensor([0.5], device="cuda"), (1, 8, 8))
    m = quantised(image_transformer(), fmt)
    want = m(*args).clone()
    b = ModelLevelOffloadBackend(torch.device("cuda", 0))
    b.enable(types.SimpleNamespace(transformer=m, text_encoder=nn.Linear(4, 4, device="cuda")))
    assert all(t.device.type == "cpu" for _, t in weight_tensors(m))
    for _ in range(2):
        b.use("transformer")
        assert torch.equal(m(*args), want)
        b.use("text_encoder")
        assert all(t.device.type == "cpu" for _, t in weight_tensors(m))


# ------------------------------------------------------------------ what a request for quantised weights reaches
def test_quantization_beside_a_stage_configuration(tmp_path, monkeypatch):
    """The stages of a configuration take it from there; asked for beside one it is refused (fp8: said not to have any effect), before a stage is started."""
    from vllm_omni_b200.entrypoints import stage_runtime
    path, said = tmp_path / "stages.yaml", []
    path.write_text("stage_args: []\n")
    monkeypatch.setattr(stage_runtime.logger, "warning", lambda text, *args: said.append(text % args))
    for fmt in ("mxfp4", "nvfp4"):
        with pytest.raises(ValueError, match="engine_args.quantization"):
            stage_runtime.build_stages(None, str(path), {"quantization": fmt})
    stage_runtime.build_stages(None, str(path), {"quantization": None})
    assert not said
    assert stage_runtime.build_stages(None, str(path), {"quantization": "fp8"})[0] == []
    assert len(said) == 1 and "engine_args.quantization" in said[0]
