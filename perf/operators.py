"""Low-bit linear layers: quantisation of rows to 4-bit floats, RMS norm with a quantised output, products of 4-bit operands
(dense and grouped by expert), and an MLP block of them together.

A 4-bit operand [R, K] is ``codes`` uint8 [R, K / 2] (element 2 i in the low half of byte i; sign, 2 bits of exponent, 1 of mantissa)
and ``scales``, one byte per block of a row, laid out as the tensor cores read them: [R / 128, K / (4 blocks), 32, 4, 4], where
row r and block b stand at [r // 128, b // 4, r % 32, r // 32 % 4, b % 4].  ``mxfp4``: blocks of 32 and powers of two (byte - 127 is the
exponent); ``nvfp4``: blocks of 16, e4m3 scales and one fp32 scale per row.  Rows of a gated layer come as 8 gate rows, their 8 lift rows,
the next 8 gate rows and so on.

The plain forms work on the same operands in fp32; ``exact`` is the definition in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BF = torch.bfloat16
BLOCK = {"mxfp4": 32, "nvfp4": 16}
EPS = 1e-6
MOST_FLOPS = 2.0 * 8192 * 24576 * 4096          # the largest listed product


def listed():
    return [
        # one decoded token's attention output before the output projection: all latency
        dict(name="quantize_1", path="quantize", rows=1, cols=4096, fmt="nvfp4"),
        # a long prompt's MLP activations, an odd number of rows
        dict(name="quantize_8191", path="quantize", rows=8191, cols=12288, fmt="mxfp4"),
        # the norm before a projection in a decode step of eight conversations
        dict(name="norm_8", path="norm", rows=8, cols=4096, fmt="fp8", residual=True),
        # the same for the tokens of several prompts of one step
        dict(name="norm_12289", path="norm", rows=12289, cols=4096, fmt="fp8", residual=True),
        # gate and lift of a dense decoder's MLP for one token: weight traffic
        dict(name="linear_1", path="linear", rows=1, n=24576, k=4096, fmt="nvfp4", act="swiglu", bias=False, gate=0, residual=False),
        # the way back for a middling batch, with the residual
        dict(name="linear_33", path="linear", rows=33, n=4096, k=12288, fmt="mxfp4", act="", bias=False, gate=0, residual=True),
        # an image transformer's first MLP layer on the tokens of two images of odd sides
        dict(name="linear_2390", path="linear", rows=2390, n=8192, k=2048, fmt="mxfp4", act="gelu_tanh", bias=True, gate=0, residual=False),
        # gate and lift on a long prompt: the tensor cores
        dict(name="linear_8192", path="linear", rows=8192, n=24576, k=4096, fmt="nvfp4", act="swiglu", bias=False, gate=0, residual=False),
        # one token of a mixture of experts
        dict(name="experts_1", path="experts", tokens=1, experts=128, top=8, d=2048, f=768, fmt="nvfp4"),
        # 64 conversations: nearly every expert, few rows each
        dict(name="experts_64", path="experts", tokens=64, experts=128, top=8, d=2048, f=768, fmt="mxfp4"),
        # prompts beside conversations: many rows, as uneven as routers are
        dict(name="experts_2463", path="experts", tokens=2463, experts=128, top=8, d=2048, f=768, fmt="nvfp4"),
        # norm, gate and lift, way back with the residual: the second half of a dense layer, 200 rows
        dict(name="mlp_200", path="mlp", rows=200, d=4096, f=12288, fmt="nvfp4"),
    ]


def draw(rng):
    def spread(lo, hi, step=1):
        v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
        return min(hi, max(lo, round(v / step) * step))

    fmt, path = rng.choice(["mxfp4", "nvfp4"]), rng.choice(["quantize", "norm", "linear", "linear", "experts", "mlp"])
    if path == "quantize":
        rows, cols = spread(1, 8191), spread(64, 12288, 32)
        return dict(path=path, rows=rows, cols=cols, fmt=fmt)
    if path == "norm":
        return dict(path=path, rows=spread(1, 12289), cols=spread(128, 8192, 128), fmt="fp8", residual=rng.random() < 0.7)
    if path == "linear":
        act = rng.choice(["", "", "swiglu", "gelu_tanh", "silu"])
        n, k = spread(64, 24576, 16), spread(64, 12288, 32)
        rows = spread(1, max(1, min(8192, int(MOST_FLOPS / (2.0 * n * k)))))
        gate = 0 if act == "swiglu" else rng.choice([0, 0, 1])
        return dict(path=path, rows=rows, n=n, k=k, fmt=fmt, act=act, bias=act != "swiglu" and rng.random() < 0.5, gate=gate,
                    residual=act != "swiglu" and rng.random() < 0.5)
    if path == "experts":
        experts = rng.choice([8, 16, 60, 64, 128])
        return dict(path=path, tokens=spread(1, 2463), experts=experts, top=rng.randint(1, 8), d=spread(256, 4096, 32), f=spread(128, 1536, 32), fmt=fmt)
    return dict(path=path, rows=spread(1, 2048), d=spread(256, 4096, 32), f=spread(256, 12288, 32), fmt=fmt)


# ------------------------------------------------------------------ operands
def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) % (1 << 62))


def _activations(rows, cols, g):
    """Normal values, every row at a size of its own, a few channels that stand out: what a transformer's activations look like."""
    x = torch.randn(rows, cols, device=DEV, generator=g)
    x *= torch.exp(torch.randn(rows, 1, device=DEV, generator=g))
    x *= torch.where(torch.rand(cols, device=DEV, generator=g) < 0.005, 12.0, 1.0)
    return x.to(BF)


def _weight(shape, fmt, g, gated=False):
    """A checkpoint's matrix in 4 bits: (codes, scales, row scales)."""
    w = (torch.randn(*shape, device=DEV, generator=g) / math.sqrt(shape[-1])).to(BF)
    if gated:
        f = shape[-2] // 2
        w = torch.stack([w[..., :f, :].unflatten(-2, (-1, 8)), w[..., f:, :].unflatten(-2, (-1, 8))], -3).flatten(-4, -2)
    codes, scale, row = _round4(w, fmt)
    return dict(codes=_pack(codes), scales=_tiles(scale), row=row)


def _power(byte):
    """2 ** (byte - 127) in fp32, bytes 0 to 254, exactly (exp2 of a GPU is off by an ulp now and then, which moves ties)."""
    byte = byte.to(torch.int32)
    return torch.where(byte > 0, byte << 23, 1 << 22).view(torch.float32)


def _round4(x, fmt):
    """x [..., K] bf16 -> code per element, scale byte per block, row scale.  Quotients are those of two tensors: one by a Python number
    is a product with its rounded reciprocal on a GPU."""
    x = x.float()
    size = x.abs().unflatten(-1, (-1, BLOCK[fmt])).amax(-1)
    if fmt == "mxfp4":
        e = torch.frexp(size).exponent - 1                         # floor(log2)
        byte = torch.where(size > 0, e - 2 + 127, 0).clamp(0, 254)
        s, row = _power(byte), None
        scale = byte.to(torch.uint8)
    else:
        most = size.amax(-1, keepdim=True)
        row = torch.where(most > 0, _power((torch.frexp(most).exponent - 11).clamp(min=-126) + 127), 1.0)
        s8 = (size / row / torch.full_like(size, 6.0)).to(torch.float8_e4m3fn)
        s, scale, x = s8.float(), s8.view(torch.uint8), x / row
        row = row[..., 0]
    q = x.unflatten(-1, (-1, BLOCK[fmt])) / s.unsqueeze(-1)
    q = torch.where(s.unsqueeze(-1) > 0, q, 0.0).flatten(-2)
    a = q.abs()
    code = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)        # ties to even
    return code + (x.signbit() & (code > 0)).to(torch.uint8) * 8, scale, row


def _pack(code):
    return code[..., 0::2] + 16 * code[..., 1::2]


def _tiles(scale):
    r, b = scale.shape[-2:]
    full = torch.zeros(*scale.shape[:-2], -(-r // 128) * 128, -(-b // 4) * 4, dtype=torch.uint8, device=scale.device)
    full[..., :r, :b] = scale
    full = full.unflatten(-1, (-1, 4)).unflatten(-3, (-1, 4, 32))          # [..., R/128, 4, 32, B/4, 4]
    n = full.dim()
    return full.permute(*range(n - 5), n - 5, n - 2, n - 3, n - 4, n - 1).contiguous()


def _untile(tiles, r, b):
    n = tiles.dim()
    t = tiles.permute(*range(n - 5), n - 5, n - 2, n - 3, n - 4, n - 1)
    return t.flatten(-2).flatten(-4, -2)[..., :r, :b]


def prepare(case, seed):
    g, path = _generator(seed), case["path"]
    st = dict(case=case)
    if path == "quantize":
        st["x"] = _activations(case["rows"], case["cols"], g)
    elif path == "norm":
        st["x"] = _activations(case["rows"], case["cols"], g)
        st["gain"] = (1 + 0.2 * torch.randn(case["cols"], device=DEV, generator=g)).to(BF)
        st["residual"] = _activations(case["rows"], case["cols"], g) if case["residual"] else None
    elif path == "linear":
        m, n, k = case["rows"], case["n"], case["k"]
        st["x"] = _activations(m, k, g)
        st["w"] = _weight((n, k), case["fmt"], g, case["act"] == "swiglu")
        st["bias"] = torch.randn(n, device=DEV, generator=g).to(BF) if case["bias"] else None
        st["gate"] = torch.randn(case["gate"], n, device=DEV, generator=g).to(BF) if case["gate"] else None
        st["residual"] = torch.randn(m, n, device=DEV, generator=g).to(BF) if case["residual"] else None
    elif path == "experts":
        t, e, d, f = case["tokens"], case["experts"], case["d"], case["f"]
        st["x"] = _activations(t, d, g)
        score = torch.randn(t, e, device=DEV, generator=g) + torch.randn(e, device=DEV, generator=g)       # some experts are liked more
        val, ids = score.topk(case["top"], -1)
        st["ids"], st["weights"] = ids.to(torch.int32), torch.softmax(val, -1)
        st["most"] = int(torch.bincount(ids.flatten(), minlength=e).max())        # rows of the fullest expert
        st["up"] = _weight((e, 2 * f, d), case["fmt"], g, True)
        st["down"] = _weight((e, d, f), case["fmt"], g)
    else:
        r, d, f = case["rows"], case["d"], case["f"]
        st["x"] = _activations(r, d, g)
        st["gain"] = (1 + 0.2 * torch.randn(d, device=DEV, generator=g)).to(BF)
        st["up"] = _weight((2 * f, d), case["fmt"], g, True)
        st["down"] = _weight((d, f), case["fmt"], g)
    return st


# ------------------------------------------------------------------ plain forms
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _values(code, scale, row, fmt):
    """fp32 values of codes [..., K] with scale bytes [..., K / block]."""
    table = torch.tensor(VALUES + tuple(-v for v in VALUES), device=code.device)
    v = table[code.int()].unflatten(-1, (-1, BLOCK[fmt]))
    s = _power(scale) if fmt == "mxfp4" else scale.view(torch.float8_e4m3fn).float()
    v = (v * s.unsqueeze(-1)).flatten(-2)
    return v if row is None else v * row.unsqueeze(-1)


def _rows(x, fmt):
    return _values(*_round4(x, fmt), fmt)


def _matrix(w, fmt):
    code = torch.stack([w["codes"] & 15, w["codes"] >> 4], -1).flatten(-2)
    r, k = code.shape[-2:]
    return _values(code, _untile(w["scales"], r, k // BLOCK[fmt]).contiguous(), w["row"], fmt)


def _swiglu(y):
    y = y.unflatten(-1, (-1, 2, 8))
    gate, lift = y[..., 0, :].flatten(-2), y[..., 1, :].flatten(-2)
    return gate / (1 + torch.exp(-gate)) * lift


def _norm(s, gain):
    s = s.float()
    return (s * torch.rsqrt(s.square().mean(-1, keepdim=True) + EPS) * gain.float()).to(BF)


def _plain_linear(st, c):
    y = _rows(st["x"], c["fmt"]) @ _matrix(st["w"], c["fmt"]).t()
    if st["bias"] is not None:
        y = y + st["bias"].float()
    if c["act"] == "swiglu":
        y = _swiglu(y)
    elif c["act"] == "silu":
        y = y / (1 + torch.exp(-y))
    elif c["act"] == "gelu_tanh":
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    if st["gate"] is not None:
        y = y * st["gate"].float()
    if st["residual"] is not None:
        y = y + st["residual"].float()
    return y.to(BF)


def _by_expert(ids):
    """Where every pair's row stands in [experts, rows of the fullest]: its expert and its place among the expert's rows."""
    flat = ids.flatten().long()
    order = torch.argsort(flat, stable=True)
    sorted_ids = flat[order]
    first = torch.searchsorted(sorted_ids, sorted_ids)
    place = torch.empty_like(flat)
    place[order] = torch.arange(flat.numel(), device=flat.device) - first
    return flat, place


def _plain_experts(st, c):
    t, k, e, fmt = c["tokens"], c["top"], c["experts"], c["fmt"]
    token = torch.arange(t * k, device=DEV) // k
    up, down, most = st["up"], st["down"], st["most"]
    if t * k < e:                                                          # few pairs: only their experts' weights are looked at
        up, down = ({n: None if v is None else v[st["ids"].flatten().long()] for n, v in w.items()} for w in (up, down))
        e, most, expert, place = t * k, 1, torch.arange(t * k, device=DEV), torch.zeros(t * k, dtype=torch.long, device=DEV)
    else:
        expert, place = _by_expert(st["ids"])
    xs = torch.zeros(e, most, c["d"], device=DEV)
    xs[expert, place] = _rows(st["x"], fmt)[token]
    h = _swiglu(xs @ _matrix(up, fmt).transpose(1, 2)).to(BF)
    y = _rows(h, fmt) @ _matrix(down, fmt).transpose(1, 2)
    y = y[expert, place].to(BF).float().view(t, k, -1)                     # an expert's result is a bf16 row
    return (y * st["weights"].unsqueeze(-1)).sum(1).to(BF)


def _plain_mlp(st, c):
    n = _rows(_norm(st["x"], st["gain"]), c["fmt"])
    h = _swiglu(n @ _matrix(st["up"], c["fmt"]).t()).to(BF)
    return (_rows(h, c["fmt"]) @ _matrix(st["down"], c["fmt"]).t() + st["x"].float()).to(BF)


def _plain_norm(st):
    s = st["x"] if st["residual"] is None else (st["x"].float() + st["residual"].float()).to(BF)
    y = _norm(s, st["gain"]).float().unflatten(-1, (-1, 128))
    size = y.abs().amax(-1, keepdim=True).clamp(min=1e-8)
    scale = size / torch.full_like(size, 448.0)
    v = (y / scale).to(torch.float8_e4m3fn).float() * scale
    return [s, v.flatten(-2).to(BF)]


def run(st):
    c = st["case"]
    if own:
        return _own(st, c)
    if c["path"] == "quantize":
        return _rows(st["x"], c["fmt"]).to(BF)
    if c["path"] == "norm":
        return _plain_norm(st)
    if c["path"] == "linear":
        return _plain_linear(st, c)
    return _plain_experts(st, c) if c["path"] == "experts" else _plain_mlp(st, c)


def _own(st, c):
    from vllm_omni_b200.ops import lowbit

    def operand(w, gated=False):
        return lowbit.QuantRows(w["codes"], w["scales"], c["fmt"], row_scale=w["row"], gated=gated)

    if c["path"] == "quantize":
        return lowbit.dequantize(lowbit.quantize(st["x"], c["fmt"]))
    if c["path"] == "norm":
        total = None if st["residual"] is None else torch.empty_like(st["x"])
        q = lowbit.rms_norm_quantize(st["x"], st["gain"], c["fmt"], eps=EPS, residual=st["residual"], total=total)
        return [st["x"] if total is None else total, lowbit.dequantize(q)]
    if c["path"] == "linear":
        gated = c["act"] == "swiglu"
        return lowbit.linear(st["x"], operand(st["w"], gated), bias=st["bias"], act=None if gated else c["act"] or None, gate=st["gate"],
                             residual=st["residual"])
    if c["path"] == "experts":
        return lowbit.experts(st["x"], st["ids"], st["weights"], operand(st["up"], True), operand(st["down"]))
    n = lowbit.rms_norm_quantize(st["x"], st["gain"], c["fmt"], eps=EPS)
    h = lowbit.linear(n, operand(st["up"], True))
    return lowbit.linear(h, operand(st["down"]), residual=st["x"])


# ------------------------------------------------------------------ what a pass needs
def _bytes4(rows, k, fmt):
    return rows * k * (0.5 + 1.0 / BLOCK[fmt]) + (4 * rows if fmt == "nvfp4" else 0)


def work(case):
    c, path = case, case["path"]
    if path == "quantize":
        return {"bytes": 4.0 * c["rows"] * c["cols"], "flops": 3.0 * c["rows"] * c["cols"]}
    if path == "norm":
        return {"bytes": c["rows"] * c["cols"] * (8.0 if c["residual"] else 4.0) + 2 * c["cols"], "flops": 6.0 * c["rows"] * c["cols"]}
    if path == "linear":
        m, n, k = c["rows"], c["n"], c["k"]
        out = n // 2 if c["act"] == "swiglu" else n
        extra = (2 * n if c["bias"] else 0) + 2 * n * c["gate"] + (2 * m * n if c["residual"] else 0)
        return {"bytes": 2.0 * m * k + _bytes4(n, k, c["fmt"]) + 2.0 * m * out + extra, "flops": 2.0 * m * n * k}
    if path == "experts":
        t, k, e, d, f = (c[i] for i in ("tokens", "top", "experts", "d", "f"))
        used = e * (1 - (1 - 1.0 / e) ** (t * k)) if t > 1 else min(e, k)        # experts that got rows, were all liked the same
        return {"bytes": used * (_bytes4(2 * f, d, c["fmt"]) + _bytes4(d, f, c["fmt"])) + 4.0 * t * d + 8.0 * t * k, "flops": 6.0 * t * k * d * f}
    r, d, f = c["rows"], c["d"], c["f"]
    return {"bytes": 4.0 * r * d + 2 * d + _bytes4(2 * f, d, c["fmt"]) + _bytes4(d, f, c["fmt"]), "flops": 6.0 * r * d * f}


# ------------------------------------------------------------------ the definition in 64 bits
def _two_to(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _floor_log2(x):
    return torch.frexp(x).exponent.long() - 1


def _exact4(x, fmt):
    """Values nearest to x [..., K] among what the format holds, in 64 bits."""
    b = x.double().unflatten(-1, (-1, BLOCK[fmt]))
    size = b.abs().amax(-1, keepdim=True)
    tiny = size.clamp(min=2.0 ** -140)
    if fmt == "mxfp4":
        s = _two_to((_floor_log2(tiny) - 2).clamp(-127, 127))
    else:
        most = size.amax(-2, keepdim=True)
        row = torch.where(most > 0, _two_to((_floor_log2(most.clamp(min=2.0 ** -140)) - 10).clamp(min=-126)), 1.0)
        want = size / row / torch.full_like(size, 6)
        step = _two_to(_floor_log2(want.clamp(min=2.0 ** -6)) - 3)
        s = torch.round(want / step) * step * row
    z = torch.where(s > 0, b.abs() / torch.where(s > 0, s, 1.0), 0.0).clamp(max=6.0)
    step = torch.where(z < 2, 0.5, torch.where(z < 4, 1.0, 2.0))
    return (torch.copysign(torch.round(z / step) * step, b) * s).flatten(-2)


def _exact_matrix(w, fmt):
    lo, hi = w["codes"] % 16, torch.div(w["codes"], 16, rounding_mode="floor")
    code = torch.empty(*w["codes"].shape[:-1], 2 * w["codes"].shape[-1], dtype=torch.int64, device=w["codes"].device)
    code[..., 0::2], code[..., 1::2] = lo.long(), hi.long()
    r, k = code.shape[-2:]
    row, blk = torch.arange(r, device=code.device)[:, None], torch.arange(k // BLOCK[fmt], device=code.device)[None, :]
    byte = w["scales"][..., row // 128, blk // 4, row % 32, row // 32 % 4, blk % 4].long()
    if fmt == "mxfp4":
        s = _two_to(byte - 127)
    else:
        e, m = byte // 8, (byte % 8).double()
        s = torch.where(e > 0, (1 + m / 8) * _two_to(e - 7), m / 8 * 2.0 ** -6) * w["row"].double().unsqueeze(-1)
    e, m = code // 2 % 4, (code % 2).double()
    v = torch.where(e > 0, (1 + m / 2) * _two_to(e - 1), m / 2) * torch.where(code >= 8, -1.0, 1.0)
    return (v.unflatten(-1, (-1, BLOCK[fmt])) * s.unsqueeze(-1)).flatten(-2)


def _exact_gated(y):
    y = y.unflatten(-1, (-1, 2, 8))
    gate, lift = y[..., 0, :].flatten(-2), y[..., 1, :].flatten(-2)
    return gate * torch.sigmoid(gate) * lift


def _exact_norm(s, gain):
    s = s.double()
    return s * gain.double() / torch.sqrt(s.square().mean(-1, keepdim=True) + EPS)


def exact(case, seed):
    st, c = prepare(case, seed), case
    fmt, path = c["fmt"], c["path"]
    if path == "quantize":
        return _exact4(st["x"], fmt)
    if path == "norm":
        s = st["x"].double() if st["residual"] is None else st["x"].double() + st["residual"].double()
        y = _exact_norm(s.to(BF), st["gain"]).to(BF).double().unflatten(-1, (-1, 128))
        scale = y.abs().amax(-1, keepdim=True).clamp(min=1e-8) / torch.full((), 448.0, dtype=torch.float64, device=y.device)
        z = y / scale
        step = _two_to(_floor_log2(z.abs().clamp(min=2.0 ** -6)) - 3)
        return [s, (torch.round(z / step) * step * scale).flatten(-2)]
    if path == "linear":
        y = _exact4(st["x"], fmt) @ _exact_matrix(st["w"], fmt).t()
        if st["bias"] is not None:
            y = y + st["bias"].double()
        if c["act"] == "swiglu":
            y = _exact_gated(y)
        elif c["act"] == "silu":
            y = y * torch.sigmoid(y)
        elif c["act"] == "gelu_tanh":
            y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
        if st["gate"] is not None:
            y = y * st["gate"].double()
        return y if st["residual"] is None else y + st["residual"].double()
    if path == "mlp":
        n = _exact4(_exact_norm(st["x"], st["gain"]).to(BF), fmt)
        h = _exact_gated(n @ _exact_matrix(st["up"], fmt).t()).to(BF)
        return _exact4(h, fmt) @ _exact_matrix(st["down"], fmt).t() + st["x"].double()
    out = torch.zeros(c["tokens"], c["d"], dtype=torch.float64, device=DEV)
    x = _exact4(st["x"], fmt)
    for e in range(c["experts"]):
        token, choice = (st["ids"] == e).nonzero(as_tuple=True)
        if token.numel():
            up, down = ({n: None if v is None else v[e] for n, v in st[w].items()} for w in ("up", "down"))
            h = _exact_gated(x[token] @ _exact_matrix(up, fmt).t()).to(BF)
            y = (_exact4(h, fmt) @ _exact_matrix(down, fmt).t()).to(BF).double()
            out.index_add_(0, token, y * st["weights"][token, choice].double().unsqueeze(-1))
    return out
