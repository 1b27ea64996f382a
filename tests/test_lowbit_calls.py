"""Calls of the low-bit layers (ops/lowbit.py) that their documentation allows beside the ordinary ones, and results that have to be exact."""
from __future__ import annotations

import copy
import pickle
import subprocess
from pathlib import Path

import pytest
import torch

from vllm_omni_b200.ops import lowbit as L

BF = torch.bfloat16
FMT4 = ("mxfp4", "nvfp4")
gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]


def rows_of(rows, cols, seed=0, device="cpu"):
    return torch.randn(rows, cols, generator=torch.Generator().manual_seed(seed)).to(BF).to(device)


# ------------------------------------------------------------------ fp8 rows of a norm
def by_definition(normed):
    """(codes' values, scales) of bf16 rows on the CPU: s = fp32(max / 448), e4m3(fp32(x / s)), ties to even.  ``to`` rounds to nearest."""
    y = normed.float().cpu().unflatten(-1, (-1, 128))
    top = y.abs().amax(-1, keepdim=True).clamp(min=1e-8)
    scale = top / torch.full_like(top, 448.0)
    return (y / scale).to(torch.float8_e4m3fn).float(), scale


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows", [8, 2500])
def test_fp8_rows_are_the_definition_s(rows, device):
    x = rows_of(rows, 512, device=device) * torch.exp(2 * rows_of(rows, 1, 1, device).float()).to(BF)
    normed = torch.empty_like(x)
    q = L.rms_norm_quantize(x, 1 + rows_of(1, 512, 2, device)[0] / 4, "fp8", normed=normed)
    code, scale = by_definition(normed)
    assert torch.equal(q.scales.cpu(), scale[..., 0])
    assert torch.equal(q.codes.cpu().view(torch.float8_e4m3fn).float().unflatten(-1, (-1, 128)), code)
    for dtype in (torch.float32, BF):
        assert torch.equal(L.dequantize(q, dtype).cpu().unflatten(-1, (-1, 128)), (code * scale).to(dtype))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("top", [2.0, 2.0 ** -40, 2.0 ** 100, 2.0 ** 126])
def test_fp8_codes_of_every_pair_of_mantissas(top, device):
    """Every maximum of a binade beside every bf16 of it and of the fifteen below (then what an e4m3 code rounds to zero).  The norm of equal values is one,
    times the gain: a row of ones quantises the gain."""
    m = (1 + torch.arange(128) / 128) * top                               # 128 maxima
    y = ((1 + torch.arange(128) / 128) * 2.0 ** -torch.arange(16)[:, None]).flatten() * top          # 2048 values, 127 a block
    y = torch.cat([y, torch.zeros(-y.numel() % 127)]).view(1, -1, 127).expand(128, -1, -1)
    y = torch.where(y <= m[:, None, None], y, 0.0)
    gain = torch.cat([m[:, None, None].expand(*y.shape[:2], 1), y], -1).to(BF).flatten(1)             # [128, 17 blocks]
    x = torch.ones(1, gain.shape[1], dtype=BF, device=device)
    for g in gain:
        q = L.rms_norm_quantize(x, g.to(device), "fp8", eps=0.0)
        code, scale = by_definition(g[None])
        assert torch.equal(q.scales.cpu(), scale[..., 0])
        assert torch.equal(q.codes.cpu().view(torch.float8_e4m3fn).float().unflatten(-1, (-1, 128)), code)


@pytest.mark.parametrize("device", DEVICES)
def test_fp8_scales_of_every_maximum(device):
    """A block for every finite bf16 as its maximum."""
    top = torch.arange(0, 0x7F80, dtype=torch.int32).to(torch.int16).view(BF)
    gain = torch.zeros(-(-top.numel() // 64) * 64, 128, dtype=BF)         # 64 blocks a row of 8192
    gain[:top.numel(), 3] = top
    x = torch.ones(1, 8192, dtype=BF, device=device)
    for g in gain.view(-1, 8192):
        normed = torch.empty_like(x)
        q = L.rms_norm_quantize(x, g.to(device), "fp8", eps=0.0, normed=normed)
        assert torch.equal(normed.cpu().view(-1), g) and torch.equal(q.scales.cpu(), by_definition(normed)[1][..., 0])


def same(a, b):
    assert torch.equal(a.codes, b.codes) and torch.equal(L.dequantize(a), L.dequantize(b))


# ------------------------------------------------------------------ a single row, whose stride says nothing
def odd_row(cols, seed=0, device="cpu", at=0):
    """[1, cols] of a buffer whose pitch is no multiple of 8 elements."""
    return rows_of(4, cols + 4 + at, seed, device)[:1, at:at + cols]


@pytest.mark.parametrize("at", [0, 1, 3])
def test_single_row_has_its_own_pitch(at):
    x = odd_row(64, at=at)
    assert x.stride(0) % 8
    y = L._rows16(x, "x")
    assert y.stride() == (64, 1) and y.data_ptr() % 16 == 0 and torch.equal(x, y)
    if not at:
        assert y.data_ptr() == x.data_ptr()                              # in place where it begins on 16 bytes
        assert L._out_rows(x, "total", 64) == (x.data_ptr(), 64)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("at", [0, 1])
@pytest.mark.parametrize("fmt", FMT4)
def test_single_rows_of_an_odd_pitch(fmt, at, device):
    x, r, gain = odd_row(128, 1, device, at), odd_row(128, 2, device, at), rows_of(1, 128, 3, device)[0]
    xc, rc = x.clone(memory_format=torch.contiguous_format), r.clone(memory_format=torch.contiguous_format)
    same(L.quantize(x, fmt), L.quantize(xc, fmt))
    w = L.pack_weight(rows_of(48, 128, 4, device), fmt)
    assert torch.equal(L.linear(x, w), L.linear(xc, w))
    for f in L.FORMATS:
        total, normed = torch.empty_like(xc), torch.empty_like(xc)
        want = L.rms_norm_quantize(xc, gain, f, residual=rc, total=total, normed=normed)
        wide = torch.full((4, 132), 7.0, dtype=BF, device=device)
        n2 = torch.empty(2, 133, dtype=BF, device=device)[:1, :128]
        got = L.rms_norm_quantize(x, gain, f, residual=r, total=wide[:1, :128], normed=n2)
        same(got, want)
        assert torch.equal(wide[:1, :128], total) and torch.equal(n2, normed) and (wide[:, 128:] == 7).all() and (wide[1:] == 7).all()
    up, down = L.pack_weight(rows_of(3 * 64, 128, 5, device).view(3, 64, 128), fmt, gated=True), L.pack_weight(rows_of(3 * 128, 32, 6, device).view(3, 128, 32), fmt)
    ids, p = torch.tensor([[2, 0]], dtype=torch.int32, device=device), torch.tensor([[0.5, 0.25]], device=device)
    assert torch.equal(L.experts(x, ids, p, up, down, residual=r), L.experts(xc, ids, p, up, down, residual=rc))


# ------------------------------------------------------------------ results whose rows lie on one another
@pytest.mark.parametrize("device", DEVICES)
def test_rows_of_a_result_must_not_overlap(device):
    x, gain = rows_of(6, 64, device=device), rows_of(1, 64, 3, device)[0]
    w = L.pack_weight(rows_of(64, 64, 4, device), "nvfp4")
    up, down = L.pack_weight(rows_of(3 * 64, 64, 5, device).view(3, 64, 64), "nvfp4", gated=True), L.pack_weight(rows_of(3 * 64, 32, 6, device).view(3, 64, 32), "nvfp4")
    ids, p = torch.zeros(6, 1, dtype=torch.int32, device=device), torch.ones(6, 1, device=device)
    buf = torch.zeros(6 * 64, dtype=BF, device=device)
    for bad in (buf[:64].expand(6, 64), buf.as_strided((6, 64), (48, 1))):
        for call in (lambda: L.rms_norm_quantize(x, gain, "nvfp4", total=bad), lambda: L.rms_norm_quantize(x, gain, "nvfp4", normed=bad),
                     lambda: L.linear(x, w, out=bad), lambda: L.experts(x, ids, p, up, down, out=bad)):
            with pytest.raises(ValueError, match="overlap"):
                call()
    with pytest.raises((ValueError, RuntimeError)):
        L.linear(x.view(2, 3, 64), w, out=buf[:64].expand(2, 3, 64))
    turned = torch.zeros(64, 6, dtype=BF, device=device).t()               # columns side by side: copied into
    assert torch.equal(L.experts(x, ids, p, up, down, out=turned), L.experts(x, ids, p, up, down))
    one = buf.as_strided((1, 64), (0, 1))                                 # a single row: its stride does not count
    assert torch.equal(L.linear(x[:1], w, out=one), L.linear(x[:1], w))
    same(L.rms_norm_quantize(x, gain, "nvfp4", residual=gain.expand(6, 64)), L.rms_norm_quantize(x, gain, "nvfp4", residual=gain.repeat(6, 1)))      # read only: may


# ------------------------------------------------------------------ choice of experts
@pytest.mark.parametrize("device", DEVICES)
def test_route_of_views_and_its_refusals(device):
    from vllm_omni_b200.ops.moe import route
    z = rows_of(24, 40, device=device)                                     # [experts, tokens], and [tokens, experts] as a view of it
    ids, w = route(z.t(), 4)
    want, ww = route(z.t().contiguous(), 4)
    assert torch.equal(ids, want) and torch.equal(w, ww) and ids.shape == (40, 4)
    assert route(z[:0], 4)[0].shape == (0, 4)
    with pytest.raises(ValueError, match="T, E"):
        route(z[0], 4)
    if device == "cuda":
        with pytest.raises(ValueError, match="bf16"):
            route(z.float(), 4)


# ------------------------------------------------------------------ copies
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fmt", tuple(L.FORMATS))
def test_copies_have_addresses_of_their_own(fmt, device):
    """A copy outlives what it was made of: its kernels must not be given the original's addresses."""
    gain = rows_of(1, 256, 3, device)[0]
    q = L.rms_norm_quantize(rows_of(5, 256, device=device), gain, fmt)
    for other in (copy.deepcopy(q), pickle.loads(pickle.dumps(q)), copy.copy(q)):
        assert other._ptr == tuple(0 if t is None else t.data_ptr() for t in (other.codes, other.scales, other.row_scale))
        assert (other.fmt, other.shape, other.gated, other.index) == (q.fmt, q.shape, q.gated, q.index)
        same(other, q)
    assert copy.deepcopy(q)._ptr[0] != q._ptr[0]
    w = L.pack_weight(rows_of(3 * 32, 64, 4, device).view(3, 32, 64), "nvfp4", gated=True)
    other = copy.deepcopy(w)
    assert other.gated and other.shape == (3, 32, 64) and other._ptr[0] != w._ptr[0]
    same(other, w)


# ------------------------------------------------------------------ launches
CSRC = Path(__file__).resolve().parent.parent / "vllm_omni_b200" / "csrc"


def test_resident_pairs_are_kept_per_kernel_and_device(tmp_path):
    exe = tmp_path / "per_device"
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-o", str(exe), str(CSRC / "host_tests" / "per_device.cpp")], check=True)
    assert subprocess.run([str(exe)]).returncode == 0
