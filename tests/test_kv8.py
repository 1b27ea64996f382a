"""The 8-bit key/value cache (ops/kv8.py): codes and scales bit for bit against a restatement of the definition in 64 bits, attention against 64 bits over pages whose
rows past a sequence's end hold NaN, and what is refused."""
import copy
import math

import pytest
import torch

from vllm_omni_b200.ops import _native as nv
from vllm_omni_b200.ops import kv8

BF, E4 = torch.bfloat16, torch.float8_e4m3fn


def bits(t):
    return t.view(torch.uint8) if t.dtype is E4 else t.view(torch.int16) if t.dtype is BF else t.view(torch.int32)


def same(a, b):
    return torch.equal(bits(a.cpu()), bits(b.cpu()))


# ---------------------------------------------------------------------------------------------------------------------- definition of a write
def nearest(x):
    """The e4m3 value next to x in 64 bits, ties to even; beyond 448 the largest; not a number stays one."""
    x = x.double()
    step = torch.exp2((torch.frexp(torch.where(x.isfinite(), x, 1.0)).exponent - 1).clamp(min=-6).double() - 3)
    return (torch.round(x.clamp(-448, 448) / step) * step).clamp(-448, 448)


def least(a):
    e = -120
    while 448.0 * 2.0 ** e < a:
        e += 1
    return e


def define_write(value, scale, x, slots):
    """value [pages, page, Hkv, D] and scale [pages, Hkv] in 64 bits, changed in place; rows of a page are one run."""
    page, n = value.shape[1], value.shape[0] * value.shape[1]
    by_page = {}
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < n:
            by_page.setdefault(s // page, []).append((t, s % page))
    for pg, rows in by_page.items():
        low = min(o for _, o in rows)
        for h in range(value.shape[2]):
            run = x[[t for t, _ in rows], h].double()
            fin = run[run.isfinite()].abs()
            e = least(float(fin.max()) if fin.numel() else 0.0)
            old = round(math.log2(float(scale[pg, h])))
            if low:
                e = max(e, old)
                if e > old:
                    value[pg, :low, h] = nearest(value[pg, :low, h] / 2.0 ** e) * 2.0 ** e
            scale[pg, h] = 2.0 ** e
            for i, (_, o) in enumerate(rows):
                value[pg, o, h] = nearest(run[i] / 2.0 ** e) * 2.0 ** e


def cache_of(pages, page, Hkv, D, dev, fill=None):
    c = kv8.Kv8Cache.empty(pages, page, Hkv, D, dev)
    if fill is not None:
        c.k.view(torch.uint8).fill_(fill)
        c.v.view(torch.uint8).fill_(fill)
    return c


def rows_for(T, Hkv, D, g, kind):
    x = torch.randn(T, Hkv, D, generator=g) * torch.exp(1.5 * torch.randn(T, Hkv, 1, generator=g))
    if kind == "wild":
        x = x * torch.exp2(torch.randint(-130, 120, (T, Hkv, 1), generator=g).float())
        x[torch.rand(T, Hkv, D, generator=g) < 0.03] = math.inf
        x[torch.rand(T, Hkv, D, generator=g) < 0.03] = -math.inf
        x[torch.rand(T, Hkv, D, generator=g) < 0.03] = math.nan
        x[torch.rand(T, Hkv, generator=g) < 0.1] = 0.0
        x[torch.rand(T, Hkv, generator=g) < 0.05] = 448.0
    return x.to(BF)


def steps_of(kind, page, g):
    """Slots of successive calls into a pool of 12 pages."""
    order = torch.randperm(12, generator=g)
    at = lambda pg, o: int(order[pg]) * page + o
    if kind == "prompts":                                             # two prompts, then their next tokens, one row skipped
        first = [at(i // page, i % page) for i in range(3 * page + 5)] + [at(5 + i // page, i % page) for i in range(page + 2)]
        return [first] + [[at(3, 5 + i), -1, at(6, 2 + i)] if 5 + i < page and 2 + i < page else [-1] for i in range(6)]
    if kind == "tokens":                                              # token by token over a page's end, three sequences
        return [[at(4 * s + i // page, i % page) for s in range(3)] for i in range(page + 3)]
    return [[at(0, o) for o in range(page)], [at(0, 0)], [at(0, o) for o in range(1, page)], [at(1, 3)], [at(1, 4), at(1, 5)]]     # a page starts over


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("kind", ["prompts", "tokens", "again"])
@pytest.mark.parametrize("values", ["normal", "wild"])
@pytest.mark.parametrize("page,Hkv,D", [(8, 1, 64), (16, 3, 128), (40, 2, 64), (128, 1, 128)])
def test_writes_are_the_definition(dev, kind, values, page, Hkv, D):
    g = torch.Generator().manual_seed(page + Hkv)
    c = cache_of(12, page, Hkv, D, dev)
    ref = {n: (torch.zeros(12, page, Hkv, D, dtype=torch.float64), torch.full((12, Hkv), 2.0 ** -120, dtype=torch.float64)) for n in "kv"}
    for step in steps_of(kind, page, g):
        slots = torch.tensor(step, dtype=torch.int32)
        k, v = (rows_for(len(step), Hkv, D, g, values) for _ in range(2))
        define_write(*ref["k"], k, slots)
        define_write(*ref["v"], v, slots)
        kv8.kv8_write(k.to(dev), v.to(dev), c, slots.to(dev))
    for codes, scale, (want, want_scale) in ((c.k, c.k_scale, ref["k"]), (c.v, c.v_scale, ref["v"])):
        assert torch.equal(scale.cpu().double(), want_scale)
        got = codes.cpu().float().double() * scale.cpu().double()[:, None, :, None]
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
    slots = torch.tensor([0, 12 * page - 1, -1, page, 3], dtype=torch.int32)
    for out, (want, _) in zip(kv8.kv8_read(c, slots.to(dev)), (ref["k"], ref["v"])):
        rows = want.view(-1, Hkv, D)[slots.clamp(min=0).long()]
        rows[2] = 0.0
        assert torch.equal(out.cpu().double().nan_to_num(), rows.nan_to_num()) and torch.equal(out.cpu().isnan(), rows.isnan())
    if dev == "cuda":
        assert nv.check_status(c.device) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 63, 64, 65, 1000, 5000])
@pytest.mark.parametrize("page,Hkv,D", [(8, 8, 128), (16, 2, 64), (64, 5, 128)])
def test_kernels_write_and_read_like_the_restatement(T, page, Hkv, D):
    """Many rows of sequences of odd lengths, packed beside other projections, some of them not written."""
    g = torch.Generator().manual_seed(T + page)
    slots, at = [], 0
    while len(slots) < T:
        n = int(torch.randint(1, 3 * page, (1,), generator=g))
        start = int(torch.randint(0, page, (1,), generator=g))
        slots += [at * page + start + i for i in range(n)]
        at += (start + n) // page + 1
    slots = torch.tensor(slots[:T], dtype=torch.int32)
    slots[torch.rand(T, generator=g) < 0.05] = -1
    if T == 1000:
        slots[100:131], slots[600:640] = -1, -1                        # within a page's rows, too
    pages = at + 1
    packed = rows_for(T, 3 * Hkv, D, g, "normal")
    a, b = cache_of(pages, page, Hkv, D, "cuda", fill=0x3c), cache_of(pages, page, Hkv, D, "cpu", fill=0x3c)
    start = torch.exp2(torch.randint(-9, 2, (pages, Hkv), generator=g).float())
    for c in (a, b):
        c.k_scale.copy_(start)
        c.v_scale.copy_(start)
    kv8.kv8_write(packed[:, Hkv:2 * Hkv], packed[:, 2 * Hkv:], b, slots)
    p = packed.cuda()
    kv8.kv8_write(p[:, Hkv:2 * Hkv], p[:, 2 * Hkv:], a, slots.cuda())
    assert same(a.k, b.k) and same(a.v, b.v) and torch.equal(a.k_scale.cpu(), b.k_scale) and torch.equal(a.v_scale.cpu(), b.v_scale)
    for x, y in zip(kv8.kv8_read(a, slots.cuda()), kv8.kv8_read(b, slots)):
        assert same(x, y)
    assert nv.check_status(a.device) == 0


@pytest.mark.gpu
def test_rows_that_are_not_aligned_are_copied():
    g = torch.Generator().manual_seed(1)
    x = rows_for(9, 2, 72, g, "normal").cuda()
    k, v = x[:, :, 3:67], x[:, :, 8:]                                  # neither begins on 16 bytes
    a, b = cache_of(3, 8, 2, 64, "cuda"), cache_of(3, 8, 2, 64, "cuda")
    slots = torch.arange(9, dtype=torch.int32, device="cuda")
    kv8.kv8_write(k, v, a, slots)
    kv8.kv8_write(k.contiguous(), v.contiguous(), b, slots)
    assert same(a.k, b.k) and same(a.v, b.v)
    q = x[:3, :, 5:69]
    tables, lens = torch.zeros(3, 1, dtype=torch.int32, device="cuda"), torch.full((3,), 8, dtype=torch.int32, device="cuda")
    assert same(kv8.kv8_decode(q, a, tables, lens), kv8.kv8_decode(q.contiguous(), a, tables, lens))


@pytest.mark.gpu
def test_slots_outside_the_cache_are_reported():
    c = cache_of(2, 16, 1, 64, "cuda")
    x = torch.ones(3, 1, 64, dtype=BF, device="cuda")
    kv8.kv8_write(x, x, c, torch.tensor([3, 32, 2 ** 31 - 1], dtype=torch.int32, device="cuda"))
    with pytest.raises(nv.NativeError):
        nv.check_status(c.device)
    k, _ = kv8.kv8_read(c, torch.tensor([3, 32], dtype=torch.int32, device="cuda"))
    assert bool((k[0] == 1).all()) and bool((k[1] == 0).all())
    with pytest.raises(nv.NativeError):
        nv.check_status(c.device)
    assert float(c.k.float().abs().sum()) == 448 * 64 * 0 + float(c.k.view(-1, 64)[3].float().sum())


@pytest.mark.gpu
def test_the_same_slot_twice_takes_the_later_row():
    for D in (64, 128):
        c, d = cache_of(2, 16, 1, D, "cuda"), cache_of(2, 16, 1, D, "cuda")
        x = torch.arange(1, 9, device="cuda").to(BF)[:, None, None].expand(8, 1, D)
        kv8.kv8_write(x, x, c, torch.tensor([0, 1, 1, 1, 2, 2, 0, 3], dtype=torch.int32, device="cuda"))
        y = torch.tensor([7, 4, 6, 8], device="cuda").to(BF)[:, None, None].expand(4, 1, D)
        kv8.kv8_write(y, y, d, torch.arange(4, dtype=torch.int32, device="cuda"))
        assert same(c.k, d.k) and same(c.v, d.v) and torch.equal(c.k_scale, d.k_scale)


# --------------------------------------------------------------------------------------------------------------------------------- attention
def filled(lens, page, Hkv, D, g, dev="cuda", kind="normal", extra=1):
    """A cache of sequences in pages of a random order; rows past the ends hold NaN, so do scales of pages that belong to nobody.  Keys and values in 64 bits."""
    per = [-(-n // page) for n in lens]
    total = sum(per) + extra
    order = torch.randperm(total, generator=g).to(torch.int32)
    c = cache_of(total, page, Hkv, D, dev, fill=0x7f)
    c.k_scale.fill_(math.nan)
    c.v_scale.fill_(math.nan)
    tables = torch.full((len(lens), max(1, max(per)) + 1), -5, dtype=torch.int32)
    at, ks, vs = 0, [], []
    for s, n in enumerate(lens):
        pages = order[at:at + per[s]]
        at += per[s]
        tables[s, :per[s]] = pages
        slots = torch.cat([torch.arange(page) + int(p) * page for p in pages])[:n].to(torch.int32) if n else torch.zeros(0, dtype=torch.int32)
        k, v = (rows_for(n, Hkv, D, g, kind) for _ in range(2))
        if kind == "levels":                                          # values of neighbouring pages are worlds apart
            v = (v.double() * 2.0 ** (40 * ((torch.arange(n) // page) % 3) - 40.0)[:, None, None]).to(BF)
        kv8.kv8_write(k.to(dev), v.to(dev), c, slots.to(dev))
        a, b = kv8.kv8_read(c, slots.to(dev))
        ks.append(a.double())
        vs.append(b.double())
    return c, tables.to(dev), ks, vs


def reference(q, k, v, scale):
    """One row of queries [H, D] over keys [n, Hkv, D] in 64 bits: (output, bound)."""
    if k.shape[0] == 0:
        return torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    G = q.shape[0] // k.shape[1]
    kk, vv = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    s = torch.einsum("hd,khd->hk", q.double(), kk) * scale
    w = torch.softmax(s, -1)
    ref = torch.einsum("hk,khd->hd", w, vv)
    # A weight in f16 is off by 2^-11 of itself, or 2^-39 of the largest where f16 is subnormal; scores in fp32: a sum of D products, D 2^-24 of their magnitudes, and q in f16
    # after division by a power of two: 2^-25 of its largest; both move a weight by their own size, and weight and normaliser by twice it.  ex2.approx: 2^-22.
    # The result is rounded to bf16 (2^-8 of it).
    ds = (torch.einsum("hd,khd->hk", q.double().abs(), kk.abs()) * (q.shape[1] * 2.0 ** -24) + q.double().abs().amax(-1, keepdim=True) * kk.abs().sum(-1).t() * 2.0 ** -25) * scale
    part = torch.einsum("hk,khd->hd", w * (2.0 ** -11 + 2.0 ** -21 + 2 * ds), vv.abs()) + torch.einsum("hk,khd->hd", w.amax(-1, keepdim=True) * 2.0 ** -39 + 0 * w, vv.abs())
    return ref, part * 1.01 + ref.abs() * (2.0 ** -8 + 2 * (w * ds).sum(-1, keepdim=True) + 2.0 ** -20) + 2.0 ** -133


HEADS = [(8, 1, 128), (32, 4, 128), (16, 8, 64), (12, 3, 128), (20, 10, 64), (16, 1, 128), (36, 3, 128), (5, 5, 64), (40, 1, 64), (34, 2, 128), (9, 1, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv,D", HEADS)
@pytest.mark.parametrize("page", [8, 16, 48, 128])
@pytest.mark.parametrize("lens", [[1], [7, 8, 0, 9, 31, 32, 33, 64, 65], [1000, 1, 333, 2047, 0] * 4])
def test_decode_against_64_bits(H, Hkv, D, page, lens):
    g = torch.Generator().manual_seed(H * 100 + page + len(lens))
    c, tables, ks, vs = filled(lens, page, Hkv, D, g)
    n = len(lens)
    q = torch.randn(n, H * D + 16, generator=g).to(BF).cuda()[:, :H * D].view(n, H, D)
    out = torch.full((n, H + 1, D), 9.0, dtype=BF, device="cuda")
    kv8.kv8_decode(q, c, tables, torch.tensor(lens, dtype=torch.int32, device="cuda"), out=out[:, :H])
    for s in range(n):
        ref, bound = reference(q[s], ks[s], vs[s], D ** -0.5)
        assert ((out[s, :H].double() - ref).abs() <= bound).all(), s
    assert bool((out[:, H] == 9).all()) and nv.check_status(c.device) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv,D", [(16, 4, 64), (32, 4, 128), (4, 4, 128), (12, 4, 64), (7, 1, 128), (32, 1, 64), (32, 2, 128)])
@pytest.mark.parametrize("seqs,per", [(3, 4), (9, 2), (1, 33), (20, 5)])
def test_rows_of_the_same_sequence(H, Hkv, D, seqs, per):
    """Proposed tokens: row i of a sequence sees one key more than row i - 1; rows of nobody lie between them."""
    g = torch.Generator().manual_seed(H + seqs * per)
    lens = [int(torch.randint(per, 900, (1,), generator=g)) for _ in range(seqs)]
    c, tables, ks, vs = filled(lens, 16, Hkv, D, g)
    row_seq, row_lens = [], []
    for s in range(seqs):
        row_seq += [s] * per + [-1] * (s % 2)
        row_lens += list(range(lens[s] - per + 1, lens[s] + 1)) + [0] * (s % 2)
    q = torch.randn(len(row_seq), H, D, generator=g).to(BF).cuda()
    out = kv8.kv8_decode(q, c, tables, torch.tensor(row_lens, dtype=torch.int32, device="cuda"), torch.tensor(row_seq, dtype=torch.int32, device="cuda"), scale=0.2)
    for r, (s, n) in enumerate(zip(row_seq, row_lens)):
        ref, bound = reference(q[r], ks[s][:n], vs[s][:n], 0.2)
        assert ((out[r].double() - ref).abs() <= bound).all(), r
    assert nv.check_status(c.device) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", [1.0, 2.0 ** 90, 2.0 ** -90])
def test_scales_worlds_apart(D, size):
    """Pages of values 2^40 apart, queries far from 1 in size (their keys the other way): the weights of small pages count where large ones have none."""
    g = torch.Generator().manual_seed(D)
    lens = [200, 77, 1500]
    c, tables, ks, vs = filled(lens, 16, 2, D, g, kind="levels")
    q = torch.randn(3, 8, D, generator=g).to(BF).cuda() * size
    c.k_scale.mul_(1 / size)
    out = kv8.kv8_decode(q, c, tables, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    for s in range(3):
        ref, bound = reference(q[s], ks[s] / size, vs[s], D ** -0.5)
        assert ((out[s].double() - ref).abs() <= bound).all(), s


@pytest.mark.gpu
def test_values_next_to_the_least_scale():
    """Values so small that their page has the least exponent, 2^-120, come out as they are."""
    c = cache_of(1, 16, 1, 64, "cuda")
    k = torch.zeros(5, 1, 64, dtype=BF, device="cuda")
    v = torch.full((5, 1, 64), 2.0 ** -125, dtype=BF, device="cuda")
    kv8.kv8_write(k, v, c, torch.arange(5, dtype=torch.int32, device="cuda"))
    out = kv8.kv8_decode(torch.ones(1, 1, 64, dtype=BF, device="cuda"), c, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([5], dtype=torch.int32, device="cuda"))
    assert torch.equal(out.double(), torch.full_like(out, 2.0 ** -125).double())


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[40], [3000, 40]])
def test_not_a_number_stays_in_its_rows(lens):
    g = torch.Generator().manual_seed(8)
    c, tables, ks, vs = filled(lens, 16, 2, 128, g)
    s = len(lens) - 1
    slot = int(tables[s, 1]) * 16 + 3
    c.v.view(torch.uint8).view(-1, 2, 128)[slot, 1, 5] = 0x7f             # head 1, channel 5
    q = torch.randn(len(lens), 4, 128, generator=g).to(BF).cuda()
    q[0, 0, 0] = math.nan if len(lens) > 1 else q[0, 0, 0]
    out = kv8.kv8_decode(q, c, tables, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    bad = out[s].isnan()
    assert bool(bad[2:, 5].all()) and not bool(bad[:2].any()) and int(bad.sum()) == 2
    if len(lens) > 1:
        assert bool(out[0, 0].isnan().all()) and not bool(out[0, 1:].isnan().any())


@pytest.mark.gpu
def test_pages_outside_the_cache_are_reported():
    g = torch.Generator().manual_seed(9)
    c, tables, ks, vs = filled([40, 50], 16, 1, 64, g)
    q, lens = torch.randn(2, 2, 64, generator=g).to(BF).cuda(), torch.tensor([40, 50], dtype=torch.int32, device="cuda")
    want = kv8.kv8_decode(q, c, tables, lens)
    tables[1, 2] = c.pages
    out = kv8.kv8_decode(q, c, tables, lens)
    assert same(out[0], want[0])
    with pytest.raises(nv.NativeError):
        nv.check_status(c.device)
    kv8.kv8_decode(q, c, tables, lens, torch.tensor([0, 2], dtype=torch.int32, device="cuda"))
    with pytest.raises(nv.NativeError):
        nv.check_status(c.device)
    long = kv8.kv8_decode(q[:1], c, tables[:1, :3], torch.tensor([4000], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert long.shape == q[:1].shape                                        # lengths count up to the table's columns


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv,n,length", [(32, 4, 64, 1800), (16, 1, 40, 700), (32, 8, 3, 2000)])
def test_neighbours_leave_a_sequence_alone(H, Hkv, n, length):
    D, page, width = 128, 16, 256
    g = torch.Generator().manual_seed(n)
    c = cache_of(2 * width, page, Hkv, D, "cuda")
    k, v = (rows_for(2 * width * page, Hkv, D, g, "normal").cuda() for _ in range(2))
    kv8.kv8_write(k, v, c, torch.arange(2 * width * page, dtype=torch.int32, device="cuda"))
    q = torch.randn(n, H, D, generator=g).to(BF).cuda()
    tables = torch.arange(width, 2 * width, dtype=torch.int32, device="cuda").repeat(n, 1)
    tables[0] -= width

    def first(others):
        return kv8.kv8_decode(q, c, tables, torch.tensor([length] + [others(i) for i in range(1, n)], dtype=torch.int32, device="cuda"))[0]
    want = first(lambda i: length)
    for others in (lambda i: 1, lambda i: 4096, lambda i: 1 + 997 * i % 4096, lambda i: 0):
        assert same(first(others), want)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Pages on both sides of 2^32 codes."""
    page, Hkv, D = 128, 8, 128
    pages = (1 << 32) // (page * Hkv * D) + 3
    codes = torch.zeros(2, pages, page, Hkv, D, dtype=torch.uint8, device="cuda").view(E4)
    c = kv8.Kv8Cache(codes[0], codes[1], *torch.full((2, pages, Hkv), 2.0 ** -120, device="cuda"))
    g = torch.Generator().manual_seed(2)
    tables = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device="cuda")
    slots = torch.cat([torch.arange(page) + p * page for p in tables[0].tolist()])[:300].to(torch.int32).cuda()
    k, v = (rows_for(300, Hkv, D, g, "normal").cuda() for _ in range(2))
    kv8.kv8_write(k, v, c, slots)
    a, b = kv8.kv8_read(c, slots)
    small = cache_of(3, page, Hkv, D, "cuda")
    kv8.kv8_write(k, v, small, torch.arange(300, dtype=torch.int32, device="cuda"))
    x, y = kv8.kv8_read(small, torch.arange(300, dtype=torch.int32, device="cuda"))
    assert same(a, x) and same(b, y)
    q, lens = torch.randn(1, 16, D, generator=g).to(BF).cuda(), torch.tensor([300], dtype=torch.int32, device="cuda")
    t3 = torch.arange(3, dtype=torch.int32, device="cuda")[None]
    assert same(kv8.kv8_decode(q, c, tables, lens), kv8.kv8_decode(q, small, t3, lens))
    rows = torch.randn(299, 16, D, generator=g).to(BF).cuda()
    assert same(kv8.kv8_prefill(rows, c, [(0, 299, 1, tables[0])]), kv8.kv8_prefill(rows, small, [(0, 299, 1, t3[0])]))


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("H,Hkv,D,page", [(8, 2, 128, 16), (4, 4, 64, 8), (7, 1, 128, 64), (6, 2, 64, 48)])
@pytest.mark.parametrize("segs", [[(0, 5, 0)], [(2, 1, 0), (3, 40, 70), (50, 33, 0), (83, 2, 300)], [(0, 300, 17), (300, 130, 0)], [(1, 1, 64), (4, 20, 1)]])
def test_portions_against_64_bits(dev, H, Hkv, D, page, segs):
    g = torch.Generator().manual_seed(H + page)
    c, tables, ks, vs = filled([n + ctx for _, n, ctx in segs], page, Hkv, D, g, dev)
    T = max(a + n for a, n, _ in segs) + 3
    q = torch.randn(T, H, D, generator=g).to(BF).to(dev)
    out = torch.full((T, H, D), 9.0, dtype=BF, device=dev)
    live = torch.zeros(T, dtype=torch.bool)
    per = [-(-(n + ctx) // page) for _, n, ctx in segs]
    kv8.kv8_prefill(q, c, [(a, n, ctx, tables[i, :per[i]].contiguous()) for i, (a, n, ctx) in enumerate(segs)], out=out)
    for i, (a, n, ctx) in enumerate(segs):
        live[a:a + n] = True
        for r in range(n):
            ref, bound = reference(q[a + r], ks[i][:ctx + r + 1], vs[i][:ctx + r + 1], D ** -0.5)
            G = H // Hkv
            w = torch.softmax(torch.einsum("hd,khd->hk", q[a + r].double(), ks[i][:ctx + r + 1].repeat_interleave(G, 1)) * D ** -0.5, -1)
            # Weights rounded to bf16 (2^-8 of each) in place of f16.  Keys that are hidden have scores of -inf, whose exponentials the tensor-core kernel takes from
            # a polynomial of an argument that is at least -126: each weighs up to 2^-126 (1 + 2^-13) over a normaliser of at least 1, which 1.01 * 2^-126 covers.
            bound = bound + torch.einsum("hk,khd->hd", w, vs[i][:ctx + r + 1].abs().repeat_interleave(G, 1)) * 2.0 ** -8
            bound = bound + vs[i].abs().sum(0).repeat_interleave(G, 0) * 1.01 * 2.0 ** -126
            assert ((out[a + r].double() - ref).abs() <= bound).all(), (i, r)
    assert bool((out[~live.to(dev)] == 9).all())


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv,D,page", [(4, 2, 128, 16), (3, 1, 64, 24)])
def test_more_portions_than_a_launch_takes(H, Hkv, D, page):
    segs, at = [], 1
    for i in range(35):
        n = (1, 7, 30, 65)[i % 4]
        segs.append((at, n, (0, 0, 131, 16)[(i * 5 + i // 4) % 4]))
        at += n + i % 2
    test_portions_against_64_bits("cuda", H, Hkv, D, page, segs[::-1])


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("H,Hkv,D", [(8, 2, 128), (4, 4, 64), (8, 1, 64), (16, 1, 128), (6, 3, 128)])
def test_what_is_not_a_number_is_its_own_rows(H, Hkv, D, dev):
    """Rows of a sequence that see different numbers of keys: a key or value that is not a number reaches those that see it, and leaves the others the same bits."""
    g = torch.Generator().manual_seed(H + D)
    n, per, page = 130, 5, 16
    q = torch.randn(2 * per, H, D, generator=g).to(BF).to(dev)
    lens = torch.tensor([n - per + 1 + i for i in range(per)] * 2, dtype=torch.int32, device=dev)
    seq = torch.arange(2, dtype=torch.int32, device=dev).repeat_interleave(per)
    tables = torch.arange(18, dtype=torch.int32, device=dev).view(2, 9)
    slots = torch.cat([torch.arange(n), torch.arange(n) + 144]).to(torch.int32).to(dev)
    k, v = (rows_for(2 * n, Hkv, D, g, "normal") for _ in range(2))
    for what in range(3):
        x, y = k.clone(), v.clone()
        if what == 1:
            y[n - 2, 0, D // 2 + 3] = math.nan                         # seen by the first sequence's last two rows
        elif what == 2:
            x[n - 1, Hkv - 1, 5] = math.nan                            # by its last one
            y[2 * n - 3, Hkv - 1, 1] = math.nan                        # by the second one's last three
        c = cache_of(18, page, Hkv, D, dev)
        kv8.kv8_write(x.to(dev), y.to(dev), c, slots)
        out = kv8.kv8_decode(q, c, tables, lens, row_seq=seq).view(2, per, Hkv, H // Hkv, D).cpu()
        if what == 0:
            want = out
            assert bool(out.isfinite().all())
            continue
        odd = torch.zeros_like(out, dtype=torch.bool)
        if what == 1:
            odd[0, -2:, 0, :, D // 2 + 3] = True
        else:
            odd[0, -1:, -1] = True
            odd[1, -3:, -1, :, 1] = True
        assert torch.equal(out.isnan(), odd)
        assert same(torch.where(odd, 0, out), torch.where(odd, 0, want))


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_a_cache_keeps_its_tensors_wherever_they_move(dev):
    g = torch.Generator().manual_seed(8)
    c = cache_of(3, 16, 2, 64, dev)
    k, v = (rows_for(20, 2, 64, g, "normal").to(dev) for _ in range(2))
    slots = torch.arange(20, dtype=torch.int32, device=dev)
    kv8.kv8_write(k, v, c, slots)
    want = kv8.kv8_read(c, slots)
    with pytest.raises(AttributeError):
        c.k = torch.zeros_like(c.k)
    twin = copy.deepcopy(c)
    kv8.kv8_write(-k, -v, twin, slots)
    assert all(same(a, b) for a, b in zip(kv8.kv8_read(c, slots), want))
    assert all(same(a, -b) for a, b in zip(kv8.kv8_read(twin, slots), want))
    old = [t.data for t in (c.k, c.v, c.k_scale, c.v_scale)]               # other memory behind the same tensors, the old filled with something else
    for t, o in zip((c.k, c.v, c.k_scale, c.v_scale), old):
        t.data = o.clone()
        o.view(torch.uint8).fill_(64)
    assert all(same(a, b) for a, b in zip(kv8.kv8_read(c, slots), want))
    with pytest.raises(ValueError):
        kv8.kv8_write(k[0, 0, 0], v, c, slots)


def test_portions_and_heads_that_are_refused():
    c, t = cache_of(2, 16, 1, 64, "cpu"), torch.arange(2, dtype=torch.int32)
    q = torch.zeros(8, 129, 64, dtype=BF)
    ok = q[:, :128]
    for bad in (lambda: kv8.kv8_prefill(ok, c, [(4, 4, 0, t), (0, 5, 0, t)]), lambda: kv8.kv8_prefill(ok, c, [(0, 8, 0, t), (2, 1, 0, t)]),
                lambda: kv8.kv8_prefill(q, c, [(0, 8, 0, t)]), lambda: kv8.kv8_decode(q, c, t[None], torch.ones(8, dtype=torch.int32), torch.zeros(8, dtype=torch.int32))):
        with pytest.raises(ValueError):
            bad()
    kv8.kv8_prefill(ok, c, [(4, 4, 0, t), (0, 4, 0, t), (2, 0, 0, t)])


@pytest.mark.gpu
def test_captured_and_on_another_stream():
    g = torch.Generator().manual_seed(3)
    lens = [500, 3, 70]
    c, tables, _, _ = filled(lens, 16, 2, 128, g)
    q, n = torch.randn(3, 8, 128, generator=g).to(BF).cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")
    slots = torch.tensor([int(tables[s, l // 16]) * 16 + l % 16 if l % 16 else -1 for s, l in enumerate(lens)], dtype=torch.int32, device="cuda")
    k, v = (rows_for(3, 2, 128, g, "normal").cuda() for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = kv8.kv8_decode(q, c, tables, n)
    torch.cuda.current_stream().wait_stream(side)
    out, more, back = torch.empty_like(q), torch.empty_like(q), torch.zeros(2, 3, 2, 128, dtype=BF, device="cuda")
    a, b = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()                  # two graphs that live together
    with torch.cuda.graph(a):
        kv8.kv8_decode(q, c, tables, n, out=out)
    with torch.cuda.graph(b):
        kv8.kv8_write(k, v, c, slots)
        kv8.kv8_read(c, slots, back[0], back[1])
        kv8.kv8_decode(q * 2, c, tables, n, out=more)
    for _ in range(2):
        a.replay()
        assert same(out, want)
        b.replay()
        a.replay()
        assert same(more, kv8.kv8_decode(q * 2, c, tables, n))
        assert all(same(x, y) for x, y in zip(back, kv8.kv8_read(c, slots)))
        want = kv8.kv8_decode(q, c, tables, n)
        assert same(out, want)


def test_refusals():
    c = cache_of(2, 16, 2, 64, "cpu")
    x, s, t, q = torch.zeros(3, 2, 64, dtype=BF), torch.zeros(3, dtype=torch.int32), torch.zeros(3, 1, dtype=torch.int32), torch.zeros(3, 4, 64, dtype=BF)
    u8 = torch.zeros(2, 16, 2, 64, dtype=torch.uint8)
    one = torch.ones(2, 2)
    for bad in (lambda: kv8.Kv8Cache(u8, u8, one, one), lambda: kv8.Kv8Cache(c.k, c.v[:1], one, one), lambda: kv8.Kv8Cache(c.k, c.v, one[0], one),
                lambda: kv8.Kv8Cache.empty(2, 12, 2, 64, "cpu"), lambda: kv8.Kv8Cache.empty(2, 16, 2, 80, "cpu"), lambda: kv8.Kv8Cache(c.k, c.v, one.double(), one.double()),
                lambda: kv8.kv8_write(x.float(), x, c, s), lambda: kv8.kv8_write(x[:, :1], x[:, :1], c, s), lambda: kv8.kv8_write(x, x[:2], c, s),
                lambda: kv8.kv8_write(x, x, c, s.long()), lambda: kv8.kv8_write(x, x, c, s[:2]), lambda: kv8.kv8_read(c, s.long()), lambda: kv8.kv8_read(c, s, x),
                lambda: kv8.kv8_read(c, s, x[:2], x[:2]), lambda: kv8.kv8_decode(q[:, :3], c, t, s), lambda: kv8.kv8_decode(q, c, t[:2], s),
                lambda: kv8.kv8_decode(q, c, t.long(), s), lambda: kv8.kv8_decode(q, c, t, s[:1]), lambda: kv8.kv8_decode(q, c, t, s, s[:1]),
                lambda: kv8.kv8_decode(q.float(), c, t, s), lambda: kv8.kv8_decode(q, c, t, s, out=q[:2]), lambda: kv8.kv8_prefill(q, c, [(0, 4, 0, t[0])]),
                lambda: kv8.kv8_prefill(q, c, [(0, 3, 14, t[0])]), lambda: kv8.kv8_prefill(q, c, [(0, 3, -1, t[0])]), lambda: kv8.kv8_prefill(q, c, [(0, 3, 0, t[0].long())])):
        with pytest.raises(ValueError):
            bad()
    kv8.kv8_write(x[:0], x[:0], c, s[:0])
    assert kv8.kv8_decode(q[:0], c, t[:0] if False else t, s[:0], s[:0]).shape == (0, 4, 64) and kv8.kv8_prefill(q, c, []).shape == q.shape


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv,D", [(16, 4, 64), (32, 4, 128), (4, 4, 128), (12, 4, 64), (8, 1, 128)])
@pytest.mark.parametrize("seqs,per,length", [(3, 4, 2000), (2, 16, 300), (20, 5, 900)])
def test_rows_of_a_sequence_leave_each_other_alone(H, Hkv, D, seqs, per, length):
    """Proposed tokens share products: queries and lengths of the others leave a row's bits as they are, whatever scale its neighbours' scores are of."""
    g = torch.Generator().manual_seed(seqs * per + D)
    c, tables, _, _ = filled([length] * seqs, 16, Hkv, D, g)
    n = seqs * per
    q = 0.1 * torch.randn(n, H, D, generator=g)                        # many keys count, and with them the roundings of their weights
    lens = torch.tensor([length - per + 1 + r % per for r in range(n)], dtype=torch.int32)
    seq = torch.arange(seqs, dtype=torch.int32, device="cuda").repeat_interleave(per)
    want = kv8.kv8_decode(q.to(BF).cuda(), c, tables, lens.cuda(), row_seq=seq)
    for turn in range(4):
        stays = torch.rand(n, generator=g) < 0.3
        other, short = q * torch.exp2(torch.randint(-2, 8, (n, 1, 1), generator=g).float()) + turn, torch.randint(0, length + 1, (n,), generator=g, dtype=torch.int32)
        x, m = torch.where(stays[:, None, None], q, other), torch.where(stays, lens, short if turn % 2 else lens)
        got = kv8.kv8_decode(x.to(BF).cuda(), c, tables, m.cuda(), row_seq=seq)
        assert same(got.cpu()[stays], want.cpu()[stays]), turn
    assert nv.check_status(c.device) == 0


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_rows_of_a_result_must_not_overlap(dev):
    c, t = cache_of(8, 16, 2, 64, dev), torch.arange(8, dtype=torch.int32, device=dev).view(4, 2)
    q, n = torch.zeros(4, 6, 64, dtype=BF, device=dev), torch.ones(4, dtype=torch.int32, device=dev)
    buf = torch.zeros(4 * 6 * 64, dtype=BF, device=dev)
    for bad in (buf[:384].view(6, 64).expand(4, 6, 64), buf[:256].view(4, 1, 64).expand(4, 6, 64), buf.as_strided((4, 6, 64), (320, 64, 1)), buf.as_strided((4, 6, 64), (64, 192, 1)),
                buf.as_strided((4, 6, 64), (384, 56, 1))):
        for call in (lambda: kv8.kv8_decode(q, c, t, n, out=bad), lambda: kv8.kv8_prefill(q, c, [(0, 4, 0, t[0])], out=bad)):
            with pytest.raises(ValueError, match="overlap"):
                call()
    heads_first = torch.zeros(6, 4, 64, dtype=BF, device=dev).transpose(0, 1)          # rows within heads: apart
    assert kv8.kv8_decode(q, c, t, n, out=heads_first) is heads_first


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_a_single_row_or_head_of_any_pitch_and_queries_that_are_the_same(dev):
    """A dimension of one entry has no pitch, and queries may be one row for all."""
    g = torch.Generator().manual_seed(9)
    c, t = cache_of(8, 16, 1, 64, dev), torch.arange(8, dtype=torch.int32, device=dev).view(1, 8)
    k, v = (rows_for(100, 1, 64, g, "normal").to(dev) for _ in range(2))
    kv8.kv8_write(k, v, c, torch.arange(100, dtype=torch.int32, device=dev))
    q = torch.randn(1, 3, 64, generator=g).to(BF).to(dev)
    n, seq = torch.tensor([100], dtype=torch.int32, device=dev), torch.zeros(5, dtype=torch.int32, device=dev)
    out = torch.zeros(500, dtype=BF, device=dev).as_strided((1, 3, 64), (3, 64, 1))
    assert same(kv8.kv8_decode(q, c, t, n, out=out), kv8.kv8_decode(q, c, t, n))
    assert same(kv8.kv8_prefill(q, c, [(0, 1, 99, t[0])], out=out), kv8.kv8_prefill(q, c, [(0, 1, 99, t[0])]))
    one = torch.randn(5, 1, 64, generator=g).to(BF).to(dev)
    out = torch.zeros(500, dtype=BF, device=dev).as_strided((5, 1, 64), (64, 11, 1))
    assert same(kv8.kv8_decode(one, c, t, n.repeat(5), seq, out=out), kv8.kv8_decode(one, c, t, n.repeat(5), seq))
    assert same(kv8.kv8_prefill(one, c, [(0, 5, 95, t[0])], out=out), kv8.kv8_prefill(one, c, [(0, 5, 95, t[0])]))
    wide = q.expand(5, 3, 64)
    assert same(kv8.kv8_decode(wide, c, t, n.repeat(5), seq), kv8.kv8_decode(wide.contiguous(), c, t, n.repeat(5), seq))
    assert same(kv8.kv8_prefill(wide, c, [(0, 5, 95, t[0])]), kv8.kv8_prefill(wide.contiguous(), c, [(0, 5, 95, t[0])]))


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv,D", [(48, 1, 64), (64, 1, 128), (200, 2, 64), (128, 1, 128), (128, 1, 64), (82, 2, 128)])
@pytest.mark.parametrize("page,lens", [(8, [1]), (16, [7, 0, 65]), (48, [1500, 1, 333])])
def test_large_groups_against_64_bits(H, Hkv, D, page, lens):
    g = torch.Generator().manual_seed(H + page)
    c, tables, ks, vs = filled(lens, page, Hkv, D, g)
    q = torch.randn(len(lens), H, D, generator=g).to(BF).cuda()
    out = kv8.kv8_decode(q, c, tables, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    for s in range(len(lens)):
        ref, bound = reference(q[s], ks[s], vs[s], D ** -0.5)
        assert ((out[s].double() - ref).abs() <= bound).all(), s
    assert nv.check_status(c.device) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv,D,seqs,per", [(4, 1, 64, 620, 1), (8, 1, 128, 560, 2)])
def test_many_rows_of_several_shares(H, Hkv, D, seqs, per):
    """More blocks of rows than have a list of their shares: those behind a row's end are empty."""
    g = torch.Generator().manual_seed(seqs)
    width, page = 512, 8
    lens = [int(torch.randint(0, 300, (1,), generator=g)) for _ in range(seqs)]
    lens[3], lens[seqs - 1], lens[200] = 4096, 3000, 0
    c, narrow, ks, vs = filled(lens, page, Hkv, D, g)
    tables = torch.full((seqs, width), -9, dtype=torch.int32, device="cuda")
    tables[:, :min(width, narrow.shape[1])] = narrow[:, :width]
    assert kv8._lib().omni_kv8_attn_shares(seqs * per, seqs, H, Hkv, D, per > 1, page, width * page) > 1
    q = torch.randn(seqs * per, H, D, generator=g).to(BF).cuda()
    n = torch.tensor(lens, dtype=torch.int32).repeat_interleave(per)
    n[per - 1::per] = (n[per - 1::per] - (per - 1)).clamp(min=0)       # the last of a sequence's rows sees less
    seq = torch.arange(seqs, dtype=torch.int32, device="cuda").repeat_interleave(per) if per > 1 else None
    out = kv8.kv8_decode(q, c, tables, n.cuda(), row_seq=seq)
    for r in range(seqs * per):
        ref, bound = reference(q[r], ks[r // per][:int(n[r])], vs[r // per][:int(n[r])], D ** -0.5)
        assert ((out[r].double() - ref).abs() <= bound).all(), r
    assert nv.check_status(c.device) == 0
