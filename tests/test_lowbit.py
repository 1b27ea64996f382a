"""Low-bit rows and their products (ops/lowbit.py): quantisation, the norm before it, dense and expert products.

Tolerances, with u = 2^-8 (half a step of bf16, relative): a product's fp32 sum of K terms is off by at most K steps of 2^-23 of the sum of
magnitudes S (an addition may cut instead of round), each further fp32 operation by 2^-23 of its result, and __expf by (2 + 1.173 |x|) 2^-23
(CUDA's bound), which is below 2^-17 for the |x| < 50 used here."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import lowbit_oracle as O
from vllm_omni_b200.ops import _native as nv
from vllm_omni_b200.ops import lowbit as L

BF = torch.bfloat16
U, STEP = 2.0 ** -8, 2.0 ** -23
FMT4 = ("mxfp4", "nvfp4")
gpu = pytest.mark.gpu


def rows_of(rows, cols, seed=0, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp(2 * torch.randn(rows, 1, generator=g))
    return x.to(BF).to(device)


def weight_of(*shape, seed=1, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) / shape[-1] ** 0.5).to(BF).to(device)


def hard_rows(cols, device="cpu"):
    """Zeros, ties, single values, the type's ends, infinities and NaN in one block each."""
    x = torch.zeros(16, cols)
    x[1] = torch.arange(cols) % 29 * 0.25 - 3.5                       # every tie of a scale of one
    x[2, -1] = 1e-30
    x[3] = torch.finfo(BF).max
    x[4] = torch.finfo(BF).tiny
    x[5] = 2.0 ** -130                                                # subnormal
    x[6, 0], x[6, 1] = float("inf"), 1.0
    x[7, cols // 2] = float("nan")
    x[8] = -0.0
    x[9] = torch.linspace(-6, 6, cols)
    x[10, :16] = 6.0
    x[10, 16:] = 6.0 / 1024                                           # nvfp4: scales at the small end of e4m3
    x[11] = 2.0 ** (torch.arange(cols) % 40 - 20).float()
    x[12] = 7.0                                                       # mxfp4: beyond the largest code
    x[13, 0] = 2688.0
    x[14, -1] = float("-inf")
    x[15] = torch.where(torch.arange(cols) % 2 == 0, 1.25, -2.5)
    return x.to(BF).to(device)


def same_as_oracle(q, x):
    code, byte, row = O.round4(x.float().cpu(), q.fmt)
    got, gbyte, grow = O.unpack(q)
    if row is not None:
        np.testing.assert_array_equal(grow, row)
        keep = ~np.isnan(row)                                         # what stands beside a factor of NaN does not count
        code, byte, got, gbyte = code[keep], byte[keep], got[keep], gbyte[keep]
    np.testing.assert_array_equal(gbyte, byte)
    fine = np.repeat(byte != (255 if q.fmt == "mxfp4" else 0x7F), O.BLOCK[q.fmt], 1)
    value = lambda c: O.CODES[c & 7] * np.where(c & 8, -1.0, 1.0)
    np.testing.assert_array_equal(value(got)[fine], value(code)[fine])
    blocks = q.cols // O.BLOCK[q.fmt]
    pad = q.scales.cpu().numpy().transpose(0, 3, 2, 1, 4).reshape(-1, q.scales.shape[1] * 4)[:q.rows, blocks:]
    assert not pad.any(), "scales of blocks past the last must be zero"


# ------------------------------------------------------------------ quantisation
@pytest.mark.parametrize("fmt", FMT4)
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 96), (130, 160), (257, 1056)])
def test_quantize_cpu(fmt, rows, cols):
    x = rows_of(rows, cols)
    q = L.quantize(x, fmt)
    same_as_oracle(q, x)
    np.testing.assert_array_equal(L.dequantize(q, torch.float32).double().numpy(), O.values(q))


@pytest.mark.parametrize("fmt", FMT4)
def test_quantize_hard_rows_cpu(fmt):
    x = hard_rows(192)
    same_as_oracle(L.quantize(x, fmt), x)


@gpu
@pytest.mark.parametrize("fmt", FMT4)
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 96), (130, 160), (1, 4096), (5, 12288), (297, 4128), (300, 64), (700, 2080), (2, 32768), (330, 16416)])
def test_quantize(fmt, rows, cols):
    x = rows_of(rows, cols, device="cuda")
    q = L.quantize(x, fmt)
    same_as_oracle(q, x)
    np.testing.assert_array_equal(L.dequantize(q, torch.float32).double().cpu().numpy(), O.values(q))
    assert torch.equal(L.dequantize(q).float(), L.dequantize(q, torch.float32))          # at most 6 bits: bf16 holds them


@gpu
@pytest.mark.parametrize("fmt", FMT4)
@pytest.mark.parametrize("cols", [64, 192, 1024])
def test_quantize_hard_rows(fmt, cols):
    x = hard_rows(cols, "cuda")
    same_as_oracle(L.quantize(x, fmt), x)
    many = x.repeat(40, 1)                                            # the form for many rows
    same_as_oracle(L.quantize(many, fmt), many)


@gpu
@pytest.mark.parametrize("fmt", FMT4)
def test_quantize_every_bf16_value(fmt):
    """Every finite bf16 beside each block maximum of one binade: all ties and all mantissas of scales."""
    v = torch.arange(0, 0x7F80, dtype=torch.int32).to(torch.int16).view(BF)
    v = v[(v >= 2.0 ** -6) & (v < 2.0 ** 4)]                          # ten binades, 1280 values
    top = torch.arange(128) / 128 + 1                                 # a maximum with each mantissa
    block = O.BLOCK[fmt]
    x = torch.zeros(128, -(-v.numel() // (block - 1)), block)
    x[..., 0] = (top * 16)[:, None]
    flat = torch.zeros(x.shape[1] * (block - 1))
    flat[:v.numel()] = v.float()
    x[..., 1:] = flat.view(x.shape[1], block - 1)
    x = x.flatten(1)
    x = torch.nn.functional.pad(x, (0, -x.shape[1] % 32)).to(BF).cuda()
    same_as_oracle(L.quantize(x, fmt), x)


@gpu
@pytest.mark.parametrize("fmt", FMT4)
def test_quantize_strided_rows(fmt):
    base = rows_of(40, 512, device="cuda")
    for x in (base[:, :256], base[::3], base[:, 8:264], base[:, 1:257], base.t()[:, :32], base.view(8, 5, 512)[:, 1:3]):
        same_as_oracle(L.quantize(x, fmt), x.reshape(-1, x.shape[-1]))


@gpu
@pytest.mark.parametrize("fmt", FMT4)
def test_quantize_beyond_32_bits(fmt):
    """More than 2^31 elements: the last rows as they would be by themselves."""
    x = torch.zeros(66000, 32768, dtype=BF, device="cuda")
    x[-3:] = rows_of(3, 32768, device="cuda")
    q, alone = L.quantize(x, fmt), L.quantize(x[-3:], fmt)
    assert torch.equal(q.codes[-3:], alone.codes)
    v = L.dequantize(q)
    assert torch.equal(v[-3:], L.dequantize(alone)) and not v[:-3].any()


@gpu
@pytest.mark.parametrize("fmt", FMT4)
def test_pack_weight_of_experts(fmt):
    w = weight_of(5, 48, 96, device="cuda")
    q, g = L.pack_weight(w, fmt), L.pack_weight(w, fmt, gated=True)
    both = L.interleave_gated(w)
    assert torch.equal(both[:, :8], w[:, :8]) and torch.equal(both[:, 8:16], w[:, 24:32]) and torch.equal(both[:, 16:24], w[:, 8:16])
    for e in range(5):
        for p, m in ((q, w), (g, both)):
            same_as_oracle(L.QuantRows(p.codes[e], p.scales[e], fmt, None if p.row_scale is None else p.row_scale[e]), m[e])
    np.testing.assert_array_equal(L.dequantize(q, torch.float32).double().cpu().numpy(), O.values(q))


# ------------------------------------------------------------------ norm
def check_norm(x, gain, fmt, residual, eps=1e-6):
    total, normed = torch.empty_like(x), torch.empty_like(x)
    q = L.rms_norm_quantize(x, gain, fmt, eps, residual=residual, total=total, normed=normed)
    s = x.double() if residual is None else (x.float() + residual.float()).to(BF).double()
    assert torch.equal(total.double(), s)
    s = s.reshape(-1, x.shape[-1])
    want = s / torch.sqrt(s.square().mean(-1, keepdim=True) + eps) * gain.double()
    # the sum of squares is off by up to K / (lanes) + 5 steps, by at most 64 here, its root by half of that; then four operations
    n2 = normed.reshape(s.shape).double()
    assert ((n2 - want).abs() <= (U + 40 * STEP) * want.abs() + 1e-38).all()
    if fmt == "fp8":
        scale = n2.reshape(n2.shape[0], -1, 128).abs().amax(-1).clamp_min(1e-8) / 448
        np.testing.assert_allclose(q.scales.double().cpu(), scale.cpu(), rtol=2 * STEP)
        v = L.dequantize(q, torch.float32).double().reshape(n2.shape[0], -1, 128)
        # half a step of e4m3 (2^-4) and three fp32 roundings; below its normal range (2^-6) half of 2^-9 of the scale
        err = (v - n2.view_as(v)).abs()
        assert (err <= (2.0 ** -4 + 4 * STEP) * n2.view_as(v).abs() + 2.0 ** -10 * (1 + 2.0 ** -20) * scale[..., None]).all()
    else:
        same_as_oracle(q, normed.reshape(s.shape))
    plain = L.rms_norm_quantize(x, gain, fmt, eps, residual=residual)
    assert torch.equal(plain.codes, q.codes) and (fmt == "fp8" or torch.equal(L.dequantize(plain), L.dequantize(q)))


@pytest.mark.parametrize("fmt", tuple(L.FORMATS))
@pytest.mark.parametrize("residual", [False, True])
def test_norm_cpu(fmt, residual):
    check_norm(rows_of(5, 256), weight_of(256) * 16, fmt, rows_of(5, 256, 3) if residual else None)


@gpu
@pytest.mark.parametrize("fmt", tuple(L.FORMATS))
@pytest.mark.parametrize("rows,cols,residual", [(1, 128, True), (1, 4096, True), (8, 4096, False), (300, 2048, True), (3, 32768, True), (700, 384, False),
                                                (299, 12288, True), (2, 5120, False)])
def test_norm(fmt, rows, cols, residual):
    check_norm(rows_of(rows, cols, device="cuda"), (weight_of(cols) * 16).cuda(), fmt, rows_of(rows, cols, 3, "cuda") if residual else None)


@gpu
@pytest.mark.parametrize("rows,cols", [(1500, 512), (1500, 768), (1300, 1024), (75777, 32), (2400, 256)])
def test_chunks_per_lane(rows, cols):
    """Many rows of one to four chunks per lane."""
    x = rows_of(rows, cols, device="cuda")
    for fmt in FMT4:
        same_as_oracle(L.quantize(x, fmt), x)
    for fmt in L.FORMATS:
        if cols % L.BLOCK[fmt] == 0:
            check_norm(x, (weight_of(cols) * 16).cuda(), fmt, rows_of(rows, cols, 3, "cuda"))


@gpu
@pytest.mark.parametrize("fmt", tuple(L.FORMATS))
@pytest.mark.parametrize("rows", [3, 400])
def test_norm_at_the_ends_of_bf16(fmt, rows):
    """Norms near the largest bf16 and near the smallest, by the gain; a zero gain; one channel that is nearly the whole row."""
    x = rows_of(rows, 256, device="cuda").clamp(-3, 3)
    x[1] = 0
    x[1, 17] = 1e10
    for g in (1e37, 1e-37, 0.0):
        check_norm(x, torch.full((256,), g, dtype=BF, device="cuda"), fmt, None)


@gpu
@pytest.mark.parametrize("fmt", tuple(L.FORMATS))
def test_norm_in_place_and_strided(fmt):
    gain = (weight_of(256) * 16).cuda()
    x, r = rows_of(40, 512, device="cuda"), rows_of(40, 512, 3, "cuda")
    for cut in (slice(0, 256), slice(8, 264), slice(1, 257)):
        want_total = torch.empty(40, 256, dtype=BF, device="cuda")
        want = L.rms_norm_quantize(x[:, cut].contiguous(), gain, fmt, residual=r[:, cut].contiguous(), total=want_total)
        r2, x2 = r.clone(), x.clone()
        if cut.start != 1:                                            # the sum in the residual's place, and in x's
            got = L.rms_norm_quantize(x2[:, cut], gain, fmt, residual=r2[:, cut], total=r2[:, cut])
            assert torch.equal(r2[:, cut], want_total) and torch.equal(got.codes, want.codes) and torch.equal(r2[:, cut.stop:], r[:, cut.stop:])
            L.rms_norm_quantize(x2[:, cut], gain, fmt, residual=r[:, cut], total=x2[:, cut])
            assert torch.equal(x2[:, cut], want_total)
        else:
            got = L.rms_norm_quantize(x2[:, cut], gain, fmt, residual=r2[:, cut])
            assert torch.equal(got.codes, want.codes)
            with pytest.raises(ValueError, match="16 bytes"):
                L.rms_norm_quantize(x2[:, cut], gain, fmt, total=r2[:, cut])
    zero = torch.zeros(2, 256, dtype=BF, device="cuda")
    assert not L.dequantize(L.rms_norm_quantize(zero, gain, fmt)).any()
    nan = rows_of(3, 256, device="cuda")
    nan[1, 100] = float("nan")
    v = L.dequantize(L.rms_norm_quantize(nan, gain, fmt))
    assert torch.isfinite(v[[0, 2]]).all() and v[1].isnan().all()


# ------------------------------------------------------------------ products
def want_linear(xq, wq, bias=None, act=None, gate=None, residual=None):
    """(values, tolerance) in 64 bits of what ``linear`` gives for quantised operands."""
    x, w = torch.from_numpy(O.values(xq)), torch.from_numpy(O.values(wq))
    M, K = x.shape
    y, d = x @ w.t(), (x.abs() @ w.abs().t()) * (K + 2) * STEP          # + the two factors
    c = lambda t: t.double().cpu()
    if wq.gated:
        y, d = (t.unflatten(-1, (-1, 2, 8)) for t in (y, d))
        g, lift, dg, dl = (t.flatten(-2) for t in (y[..., 0, :], y[..., 1, :], d[..., 0, :], d[..., 1, :]))
        s = torch.nn.functional.silu(g)
        y, d = s * lift, 1.1 * dg * (lift.abs() + dl) + (s.abs() + 1.1 * dg) * dl       # |silu'| < 1.1
        return y, d + y.abs() * (U + 2.0 ** -16) + 1e-38
    if bias is not None:
        y = y + c(bias)
        d = d + y.abs() * STEP
    if act is not None:
        y = torch.nn.functional.silu(y) if act == "silu" else torch.nn.functional.gelu(y, approximate="tanh")
        d = 1.2 * d + y.abs() * 2.0 ** -16 + 2.0 ** -22                  # both slopes are below 1.2; gelu's argument is off by a few steps, of at most 1
    if gate is not None:
        g = c(gate).repeat_interleave(M // gate.shape[0], 0)
        y, d = y * g, (d + y.abs() * STEP) * g.abs()
    if residual is not None:
        y = y + c(residual).reshape(y.shape)
        d = d + y.abs() * STEP
    return y, d + y.abs() * U + 1e-38


def close(got, want):
    y, tol = want
    got = got.double().cpu().reshape(y.shape)
    bad = ((got - y).abs() > tol) | got.isnan()
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: {got[bad][0]} for {y[bad][0]}, tolerance {tol[bad][0]}"
    if got.is_cuda or torch.cuda.is_available():
        nv.check_status()


@pytest.mark.parametrize("fmt", FMT4)
def test_linear_cpu(fmt):
    x, w = rows_of(6, 96), weight_of(40, 96)
    q, p = L.quantize(x, fmt), L.pack_weight(w, fmt)
    b, g, r = rows_of(1, 40, 5)[0], rows_of(3, 40, 6), rows_of(6, 40, 7)
    for act in (None, "silu", "gelu_tanh"):
        close(L.linear(x.view(2, 3, 96), p, b, act, residual=r.view(2, 3, 40), gate=g), want_linear(q, p, b, act, g, r))
    p = L.pack_weight(weight_of(48, 96), fmt, gated=True)
    close(L.linear(q, p), want_linear(q, p))


SHAPES = [(1, 128, 256), (1, 1, 32), (2, 7, 64), (3, 136, 96), (15, 1000, 288), (16, 128, 4128), (17, 256, 2048), (33, 1001, 1056), (64, 384, 512), (65, 264, 512),
          (100, 130, 2080), (128, 512, 1024), (129, 128, 352), (255, 300, 640), (256, 256, 256), (257, 640, 800), (513, 1032, 416)]


@gpu
@pytest.mark.parametrize("fmt", FMT4)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear(fmt, M, N, K):
    x, w = rows_of(M, K, device="cuda"), weight_of(N, K, device="cuda")
    q, p = L.quantize(x, fmt), L.pack_weight(w, fmt)
    want = want_linear(q, p)
    close(L.linear(x, p), want)
    kb = -(-K // 256)
    for tile, split in [(tile, s) for tile in (16, 64, 128) for s in (1, 2, 4)] + [(256, s) for s in (1, 2)]:
        if (tile <= 64 and M > tile) or split > kb:
            continue
        close(L.linear(q, p, force_tile=tile, force_split=split), want)


@gpu
@pytest.mark.parametrize("fmt", FMT4)
@pytest.mark.parametrize("M,N,K,tile,split", [(6, 136, 512, 16, 1), (6, 136, 512, 64, 1), (6, 1000, 512, 64, 2), (6, 77, 512, 0, 0), (130, 264, 512, 128, 1), (130, 264, 512, 128, 2), (260, 1000, 288, 256, 0),
                                              (260, 333, 288, 256, 0), (200, 333, 544, 256, 2), (260, 520, 1056, 256, 2), (4096, 256, 64, 0, 0)])
@pytest.mark.parametrize("act", [None, "silu", "gelu_tanh"])
def test_linear_epilogue(fmt, M, N, K, tile, split, act):
    x, w = rows_of(M, K, device="cuda"), weight_of(N, K, device="cuda")
    q, p = L.quantize(x, fmt), L.pack_weight(w, fmt)
    b, g, r = rows_of(1, N, 5, "cuda")[0], rows_of(2, N, 6, "cuda"), rows_of(M, N, 7, "cuda")
    kw = dict(force_tile=tile, force_split=split)
    close(L.linear(q, p, b, act, residual=r, gate=g, **kw), want_linear(q, p, b, act, g, r))
    close(L.linear(q, p, act=act, gate=g[:1], **kw), want_linear(q, p, None, act, g[:1]))
    # the sum in the residual's own place; rows of a wider buffer, on and off 16 bytes
    own = r.clone()
    assert L.linear(q, p, b, act, residual=own, out=own, **kw) is own
    close(own, want_linear(q, p, b, act, None, r))
    for cut in (8, 3):
        wide = torch.full((M, N + 24), 7.0, dtype=BF, device="cuda")
        L.linear(q, p, b, act, residual=r, out=wide[:, cut:cut + N], **kw)
        close(wide[:, cut:cut + N], want_linear(q, p, b, act, None, r))
        assert (wide[:, :cut] == 7).all() and (wide[:, cut + N:] == 7).all()


@gpu
@pytest.mark.parametrize("fmt", FMT4)
@pytest.mark.parametrize("M,N,K,tile,split", [(1, 136, 512, 16, 1), (16, 77, 1056, 16, 4), (40, 333, 512, 64, 2), (130, 264, 512, 128, 1), (200, 77, 544, 128, 2), (260, 1000, 288, 256, 0),
                                              (700, 333, 96, 256, 1), (200, 520, 1056, 256, 2)])
@pytest.mark.parametrize("act", [None, "silu", "gelu_tanh"])
def test_linear_bias_and_activation(fmt, M, N, K, tile, split, act):
    q, p = L.quantize(rows_of(M, K, device="cuda"), fmt), L.pack_weight(weight_of(N, K, device="cuda"), fmt)
    b, kw = rows_of(1, N, 5, "cuda")[0], dict(force_tile=tile, force_split=split)
    close(L.linear(q, p, b, act, **kw), want_linear(q, p, b, act))
    close(L.linear(q, p, None, act, **kw), want_linear(q, p, None, act))
    wide = torch.full((M, N + 5), 7.0, dtype=BF, device="cuda")
    L.linear(q, p, b, act, out=wide[:, 3:3 + N], **kw)
    close(wide[:, 3:3 + N], want_linear(q, p, b, act))
    assert (wide[:, :3] == 7).all() and (wide[:, 3 + N:] == 7).all()


@gpu
@pytest.mark.parametrize("fmt", FMT4)
@pytest.mark.parametrize("M,N,K,tile,split", [(1, 32, 64, 0, 0), (5, 272, 512, 16, 1), (5, 272, 512, 64, 1), (5, 272, 2080, 64, 4), (5, 272, 2080, 16, 2), (40, 4096, 512, 0, 0), (130, 528, 544, 128, 1), (100, 528, 1024, 128, 4),
                                              (300, 1040, 288, 256, 1), (300, 1040, 1056, 256, 2), (513, 512, 512, 256, 0)])
def test_linear_gated(fmt, M, N, K, tile, split):
    x, w = rows_of(M, K, device="cuda") / 4, weight_of(N, K, device="cuda")
    q, p = L.quantize(x, fmt), L.pack_weight(w, fmt, gated=True)
    want = want_linear(q, p)
    close(L.linear(q, p, force_tile=tile, force_split=split), want)
    wide = torch.full((M, N // 2 + 8), 7.0, dtype=BF, device="cuda")
    L.linear(q, p, out=wide[:, 3:3 + N // 2], force_tile=tile, force_split=split)
    close(wide[:, 3:3 + N // 2], want)
    assert (wide[:, :3] == 7).all() and (wide[:, 3 + N // 2:] == 7).all()


@gpu
@pytest.mark.parametrize("fmt", FMT4)
@pytest.mark.parametrize("tile,split,M", [(16, 1, 13), (16, 4, 13), (64, 1, 20), (64, 4, 20), (128, 1, 200), (256, 1, 300), (256, 2, 300)])
def test_linear_nan_rows_stay_alone(fmt, tile, split, M):
    """A row or a weight row of NaN makes its own results NaN and no others."""
    x, w = rows_of(M, 1024, device="cuda"), weight_of(200, 1024, device="cuda")
    x[M // 2, 500], x[M - 1, 3], w[17, 900] = float("nan"), float("inf"), float("nan")
    y = L.linear(L.quantize(x, fmt), L.pack_weight(w, fmt), force_tile=tile, force_split=split)
    bad = torch.zeros(M, 200, dtype=torch.bool, device="cuda")
    bad[M // 2] = bad[M - 1] = bad[:, 17] = True
    assert torch.equal(y.isnan(), bad)


@gpu
@pytest.mark.parametrize("fmt", FMT4)
def test_linear_beyond_32_bits(fmt):
    """More than 2^31 results: the last rows as they are by themselves."""
    x, w = rows_of(66000, 64, device="cuda"), L.pack_weight(weight_of(33000, 64, device="cuda"), fmt)
    r = torch.zeros(66000, 33000, dtype=BF, device="cuda")
    r[-2:] = 3.0
    y = L.linear(x, w, residual=r, out=r)
    close(y[-2:], want_linear(L.quantize(x[-2:], fmt), w, residual=torch.full((2, 33000), 3.0, dtype=BF)))
    close(y[:2], want_linear(L.quantize(x[:2], fmt), w))


@gpu
def test_linear_no_rows():
    w = L.pack_weight(weight_of(64, 64, device="cuda"), "nvfp4")
    assert L.linear(torch.empty(0, 64, dtype=BF, device="cuda"), w).shape == (0, 64)
    assert L.linear(torch.empty(2, 0, 64, dtype=BF, device="cuda"), w).shape == (2, 0, 64)
    assert L.dequantize(L.quantize(torch.empty(0, 64, dtype=BF, device="cuda"), "mxfp4")).shape == (0, 64)


# ------------------------------------------------------------------ experts
def want_experts(x, ids, weights, up, down, residual=None):
    """(values, tolerance) in 64 bits.  What leaves ``up`` is rounded to bf16 and to 4 bits, where an error of the sums may tip a code over: every
    element is quantised at both ends of its interval, under the scales of both ends of its block's maximum."""
    T, D = x.shape
    fmt, E = up.fmt, up.experts
    xv = torch.from_numpy(O.value_of(x.double().cpu().numpy(), fmt))
    uv, dv = O.values(up), O.values(down)
    ids, weights = ids.cpu().long(), weights.double().cpu()
    y, tol = torch.zeros(T, D, dtype=torch.float64), torch.zeros(T, D, dtype=torch.float64)
    for e in range(E):
        t, j = (ids == e).nonzero(as_tuple=True)
        if not t.numel():
            continue
        w = torch.from_numpy(uv[e])
        a, S = (v.unflatten(-1, (-1, 2, 8)) for v in (xv[t] @ w.t(), (xv[t].abs() @ w.abs().t()) * (D + 2) * STEP))
        g, lift, dg, dl = (v.flatten(-2) for v in (a[..., 0, :], a[..., 1, :], S[..., 0, :], S[..., 1, :]))
        s = torch.nn.functional.silu(g)
        h = s * lift
        dh = 1.1 * dg * (lift.abs() + dl) + (s.abs() + 1.1 * dg) * dl + h.abs() * 2.0 ** -16
        ends = [(h.abs() - dh).clamp(min=0).to(BF).double(), (h.abs() + dh).to(BF).double()]
        lo, hi = (quantised_under(ends[i], ends, fmt) for i in (0, 1))
        mid = torch.from_numpy(O.value_of(h.to(BF).double().numpy(), fmt))
        span = torch.maximum(hi[1] - mid.abs(), mid.abs() - lo[0]).clamp(min=0) * 1.0000001
        flip = (ends[0] == 0) & (ends[1] > 0)                              # the sign is open as well
        span = torch.where(flip, hi[1] + mid.abs(), span)
        w2 = torch.from_numpy(dv[e])
        r = mid @ w2.t()
        dr = span @ w2.abs().t() + ((mid.abs() + span) @ w2.abs().t()) * (w2.shape[1] + 2) * STEP
        p = weights[t, j][:, None]
        y.index_add_(0, t, r * p)
        tol.index_add_(0, t, (dr + (r.abs() + dr) * U) * p.abs() * 1.01)
    if residual is not None:
        y = y + residual.double().cpu()
    return y, tol + y.abs() * U + (ids.shape[1] + 1) * STEP * (tol + y.abs()) + 1e-30


def quantised_under(a, ends, fmt):
    """(least, most) of the magnitudes that ``a`` becomes under the scales of blocks whose maxima (and, for nvfp4, whose rows' maxima) are those of either end."""
    n = O.BLOCK[fmt]
    tops = [e.unflatten(-1, (-1, n)).amax(-1, keepdim=True) for e in ends]
    got = []
    for top in tops:
        for rowtop in (tops if fmt == "nvfp4" else tops[:1]):
            if fmt == "mxfp4":
                s = torch.exp2((torch.floor(torch.log2(top.clamp(min=2.0 ** -200))) - 2).clamp(-127, 127))
            else:
                m = rowtop.amax(-2, keepdim=True)
                row = torch.where(m > 0, torch.exp2((torch.floor(torch.log2(m.clamp(min=2.0 ** -200))) - 10).clamp(min=-126)), 1.0)
                s = torch.from_numpy(O.E4M3[O.nearest_even((top / row / 6).numpy(), O.E4M3)]) * row
            q = torch.where(s > 0, a.unflatten(-1, (-1, n)) / torch.where(s > 0, s, 1.0), 0.0)
            got.append((torch.from_numpy(O.CODES[O.nearest_even(q.numpy(), O.CODES)]) * s).flatten(-2))
    got = torch.stack(got)
    return got.amin(0), got.amax(0)


def routing(T, E, k, seed=0):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).to(torch.int32) if T else torch.empty(0, k, dtype=torch.int32)
    return ids, torch.rand(T, k, generator=g)


@pytest.mark.parametrize("fmt", FMT4)
def test_experts_cpu(fmt):
    x, up, down = rows_of(7, 64) / 4, L.pack_weight(weight_of(5, 64, 64), fmt, gated=True), L.pack_weight(weight_of(5, 64, 32, seed=2), fmt)
    ids, w = routing(7, 5, 2)
    r = rows_of(7, 64, 9)
    close(L.experts(x, ids, w, up, down, residual=r), want_experts(x, ids, w, up, down, r))


@gpu
@pytest.mark.parametrize("fmt", FMT4)
@pytest.mark.parametrize("T,E,k,D,F", [(1, 8, 2, 64, 32), (1, 128, 8, 2048, 768), (5, 60, 4, 288, 160), (64, 16, 8, 512, 96), (300, 4, 2, 256, 64), (200, 3, 3, 96, 224), (700, 2, 1, 64, 64),
                                       (90, 128, 8, 160, 32)])
def test_experts(fmt, T, E, k, D, F):
    x = rows_of(T, D, device="cuda") / 4
    up, down = L.pack_weight(weight_of(E, 2 * F, D, device="cuda"), fmt, gated=True), L.pack_weight(weight_of(E, D, F, seed=2, device="cuda"), fmt)
    ids, w = (t.cuda() for t in routing(T, E, k))
    r = rows_of(T, D, 9, "cuda")
    close(L.experts(x, ids, w, up, down), want_experts(x, ids, w, up, down))
    own = r.clone()
    assert L.experts(x, ids, w, up, down, residual=own, out=own) is own
    close(own, want_experts(x, ids, w, up, down, r))


@gpu
@pytest.mark.parametrize("fmt", FMT4)
def test_experts_uneven(fmt):
    """Experts without rows, one with all, the same expert twice for a token, ids of other ranks, and nothing chosen at all."""
    T, E, D, F = 150, 6, 128, 64
    x = rows_of(T, D, device="cuda") / 4
    up, down = L.pack_weight(weight_of(E, 2 * F, D, device="cuda"), fmt, gated=True), L.pack_weight(weight_of(E, D, F, seed=2, device="cuda"), fmt)
    w = torch.rand(T, 3, device="cuda")
    one = torch.full((T, 3), 4, dtype=torch.int32, device="cuda")
    mixed = torch.tensor([[5, 5, 0]], dtype=torch.int32, device="cuda").repeat(T, 1)
    mixed[::3, 1], mixed[::7, 2], mixed[1] = -1, E, -5
    for ids in (one, mixed):
        close(L.experts(x, ids, w, up, down), want_experts(x, ids, w, up, down))
    assert not L.experts(x, torch.full_like(one, -1), w, up, down).any()
    assert L.experts(x[:0], one[:0], w[:0], up, down).shape == (0, D)
    wide = torch.full((T, D + 9), 7.0, dtype=BF, device="cuda")
    L.experts(x, mixed, w, up, down, out=wide[:, 3:3 + D])
    close(wide[:, 3:3 + D], want_experts(x, mixed, w, up, down))
    assert (wide[:, :3] == 7).all() and (wide[:, 3 + D:] == 7).all()


@gpu
@pytest.mark.parametrize("fmt", FMT4)
def test_experts_few_rows_uneven(fmt):
    """Few rows per expert on the whole, but one expert with all of them; and as many as the smallest tile takes, one more, and one expert less."""
    E, D, F = 70, 160, 96
    up, down = L.pack_weight(weight_of(E, 2 * F, D, device="cuda"), fmt, gated=True), L.pack_weight(weight_of(E, D, F, seed=2, device="cuda"), fmt)
    for T, ids in ((100, torch.full((100, 2), 69)), (33, torch.arange(33)[:, None] // 16 * 3), (70 * 16 + 1, torch.arange(70 * 16 + 1)[:, None] % 70),
                   (70 * 16, torch.arange(70 * 16)[:, None] % 69)):
        x, w, ids = rows_of(T, D, device="cuda") / 4, torch.rand(T, ids.shape[1], device="cuda"), ids.int().cuda()
        close(L.experts(x, ids, w, up, down), want_experts(x, ids, w, up, down))


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("renorm", [False, True])
def test_route(device, renorm):
    from vllm_omni_b200.ops.moe import route
    z = (torch.randperm(40 * 60, generator=torch.Generator().manual_seed(1)).view(40, 60).float() / 256).to(BF).unique(dim=1)[:, :24]
    z = z.sort(-1).values[:, torch.randperm(24)].contiguous()
    ids, w = route(z.to(device), 5, renorm)
    p = torch.softmax(z.double(), -1)
    got = p.gather(1, ids.long().cpu())
    rest = p.scatter(1, ids.long().cpu(), 0).amax(-1, keepdim=True)
    assert ids.dtype == torch.int32 and (got >= rest).all() and (ids.sort(-1).values.diff(dim=-1) > 0).all()
    want = got / got.sum(-1, keepdim=True) if renorm else got
    np.testing.assert_allclose(w.double().cpu(), want, rtol=2.0 ** -16)           # 24 powers by __expf, their sum, a quotient
    for k in (0, 17, 25):
        with pytest.raises(ValueError, match="route"):
            route(z.to(device), k)


# ------------------------------------------------------------------ as they are used
def chain(x, gain, up, down):
    """The second half of a dense layer: norm, gate and lift, way back with the residual."""
    q = L.rms_norm_quantize(x, gain, up.fmt)
    return L.linear(L.linear(q, up), down, residual=x)


@gpu
@pytest.mark.parametrize("fmt", FMT4)
@pytest.mark.parametrize("rows", [1, 40, 300])
def test_chain(fmt, rows):
    D, F = 512, 640
    x, gain = rows_of(rows, D, device="cuda"), (1 + weight_of(D, seed=4)).cuda()
    up, down = L.pack_weight(weight_of(2 * F, D, device="cuda"), fmt, gated=True), L.pack_weight(weight_of(D, F, seed=2, device="cuda"), fmt)
    q = L.rms_norm_quantize(x, gain, fmt)
    h = L.linear(q, up)
    close(h, want_linear(q, up))
    y = L.linear(h, down, residual=x)
    close(y, want_linear(L.quantize(h, fmt), down, residual=x))
    assert torch.equal(chain(x, gain, up, down), y)                    # bit for bit: nothing depends on the order of anything


@gpu
@pytest.mark.parametrize("fmt", FMT4)
def test_captured_chains_and_experts(fmt):
    """Two graphs captured one after the other and replayed in turn, with other inputs in place, against eager calls."""
    D, F, E = 512, 640, 8
    gain = (1 + weight_of(D, seed=4)).cuda()
    up, down = L.pack_weight(weight_of(2 * F, D, device="cuda"), fmt, gated=True), L.pack_weight(weight_of(D, F, seed=2, device="cuda"), fmt)
    eu, ed = L.pack_weight(weight_of(E, 2 * F, D, device="cuda"), fmt, gated=True), L.pack_weight(weight_of(E, D, F, seed=2, device="cuda"), fmt)

    def step(x, ids, w):
        return L.experts(chain(x, gain, up, down), ids, w, eu, ed, residual=x)
    graphs = []
    for rows in (4, 90):
        x, (ids, w) = rows_of(rows, D, device="cuda"), (t.cuda() for t in routing(rows, E, 3))
        step(x, ids, w)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = step(x, ids, w)
        graphs.append((g, x, ids, w, y))
    for turn in range(3):
        for g, x, ids, w, y in graphs:
            x.copy_(rows_of(*x.shape, seed=20 + turn))
            ids.copy_(routing(*ids.shape[:1], E, 3, seed=30 + turn)[0])
            g.replay()
        torch.cuda.synchronize()
        for g, x, ids, w, y in graphs:
            assert torch.equal(y, step(x, ids, w))
    nv.check_status()


@gpu
def test_two_streams_at_once():
    D, F = 1024, 1536
    gain = (1 + weight_of(D, seed=4)).cuda()
    up, down = L.pack_weight(weight_of(2 * F, D, device="cuda"), "nvfp4", gated=True), L.pack_weight(weight_of(D, F, seed=2, device="cuda"), "nvfp4")
    xs = [rows_of(r, D, seed=r, device="cuda") for r in (3, 200)]
    want = [chain(x, gain, up, down) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(chain(xs[i], gain, up, down))
    torch.cuda.synchronize()
    for i, ys in enumerate(got):
        assert all(torch.equal(y, want[i]) for y in ys)
    nv.check_status()


# ------------------------------------------------------------------ refusals
def test_refusals():
    x, w = rows_of(4, 64), weight_of(32, 64)
    p = L.pack_weight(w, "nvfp4")
    for call, text in (
        (lambda: L.quantize(x, "fp8"), "format"), (lambda: L.quantize(x, "int4"), "format"), (lambda: L.quantize(x[:, :48], "mxfp4"), "multiple of 32"),
        (lambda: L.quantize(x.float(), "mxfp4"), "bf16"), (lambda: L.quantize(torch.zeros(1, 32800, dtype=BF), "mxfp4"), "at most"),
        (lambda: L.quantize(x[:, :0], "mxfp4"), "multiple of 32"),
        (lambda: L.pack_weight(w[0], "nvfp4"), "expected"), (lambda: L.pack_weight(w[:24], "nvfp4", gated=True), "multiple of 16"),
        (lambda: L.pack_weight(w.half(), "nvfp4"), "bf16"), (lambda: L.dequantize(p, torch.float16), "bf16 or fp32"),
        (lambda: L.rms_norm_quantize(x, w[0], "fp8"), "multiple of 128"), (lambda: L.rms_norm_quantize(x, w[0, :32], "mxfp4"), "weight"),
        (lambda: L.rms_norm_quantize(x, w[0], "mxfp4", residual=x[:2]), "residual"), (lambda: L.rms_norm_quantize(x, w[0], "mxfp4", total=x.float()), "total"),
        (lambda: L.rms_norm_quantize(x, w[0].float(), "mxfp4"), "weight"),
        (lambda: L.linear(x[:, :32], p), "does not fit"), (lambda: L.linear(x, w), "packed"), (lambda: L.linear(L.quantize(x, "mxfp4"), p), "same format"),
        (lambda: L.linear(x, p, act="relu"), "act"), (lambda: L.linear(x, p, bias=w[0]), "bias"), (lambda: L.linear(x, p, residual=x), "residual"),
        (lambda: L.linear(x, p, gate=w[:3, :32]), "gate"), (lambda: L.linear(x, p, out=torch.empty(4, 32)), "out"),
        (lambda: L.linear(x, L.pack_weight(w, "nvfp4", gated=True), act="silu"), "gated"),
        (lambda: L.QuantRows(p.codes, p.scales, "nvfp4"), "row scales"), (lambda: L.QuantRows(p.codes.repeat(1, 2), p.scales, "nvfp4", p.row_scale), "scales"),
        (lambda: L.QuantRows(p.codes, p.scales, "mxfp4", p.row_scale), "no row scales"),
        (lambda: L.QuantRows(p.codes, p.scales, "nvfp8"), "format"), (lambda: L.QuantRows(p.codes[:, :8], p.scales, "nvfp4"), "contiguous"),
        (lambda: L.QuantRows(p.codes.float(), p.scales, "nvfp4"), "uint8"),
    ):
        with pytest.raises(ValueError, match=text):
            call()
    up, down = L.pack_weight(weight_of(3, 64, 64), "nvfp4", gated=True), L.pack_weight(weight_of(3, 64, 32), "nvfp4")
    ids, wt = routing(4, 3, 2)
    for call, text in (
        (lambda: L.experts(x, ids.long(), wt, up, down), "int32"), (lambda: L.experts(x, ids, wt.half(), up, down), "fp32"),
        (lambda: L.experts(x[:3], ids, wt, up, down), "x:"), (lambda: L.experts(x, ids, wt, down, up), "do not fit"),
        (lambda: L.experts(x, ids, wt, up, p), "experts expected"), (lambda: L.experts(x, ids[:, 0], wt[:, 0], up, down), "x:|ids"),
        (lambda: L.experts(x, ids, wt, up, down, residual=x[:2]), "residual"),
        (lambda: L.experts(x, ids, wt, up, L.pack_weight(weight_of(3, 64, 32), "mxfp4")), "do not fit"),
    ):
        with pytest.raises(ValueError, match=text):
            call()


@gpu
def test_refusals_on_a_gpu():
    x, p = rows_of(4, 64, device="cuda"), L.pack_weight(weight_of(32, 64, device="cuda"), "nvfp4")
    with pytest.raises(ValueError, match="does not fit"):
        L.linear(x.cpu(), p)
    with pytest.raises(ValueError, match="contiguous"):
        L.linear(x, p, out=torch.empty(32, 4, dtype=BF, device="cuda").t())
    for bad in (dict(force_tile=32), dict(force_split=3), dict(force_split=8), dict(force_split=2)):        # one block of K only
        with pytest.raises(nv.NativeError):
            L.linear(x, p, **bad)
    with pytest.raises(nv.NativeError):
        L.linear(rows_of(65, 64, device="cuda"), p, force_tile=64)
