"""Sampling from given random numbers (ops/sampler.sample_given): the kernel against the definition in 64 bits, at ties, masks, borders of filters and vocabularies
of one to 262144 tokens.  Ids are equal; log probabilities are held to what a row's sum of weights in fp32 can be off by."""
import numpy as np
import pytest
import torch

from vllm_omni_b200.ops import sampler
from vllm_omni_b200.ops.sampler import sample_given

INF = float("inf")


def definition(x, u, t, k, p, m):
    """One row, written apart from the library's restatement: sets in place of sorted prefixes."""
    x = x.double()
    V = x.numel()
    ok = ~x.isnan()
    if not ok.any() or x[ok].max() == -INF:
        return -1, -INF, 0.0
    x = torch.where(ok, x, -INF)
    top = x.max()
    z = torch.where(x == top, 0.0, (x - top) / (t if t > 0 else 1.0)).nan_to_num(nan=-INF, neginf=-INF)
    w = torch.round(torch.exp(z) * 2 ** 44)
    log_all = torch.log(w.sum() / 2 ** 44)
    # The sum of weights e^z in fp32, pieces of 256 relative to their maxima and these to the row's: two exponentials (ex2.approx: 2^-22 each), 13 sums on the way (2^-24 each), and
    # arguments of a difference, a factor and a product (2^-24 each, of |z| in all).  Its logarithm is off by as much as it is off relative to itself.
    off = float((w * (2.0 ** -21 + 13 * 2.0 ** -24 + 3 * 2.0 ** -24 * z.abs().clamp(max=100))).sum() / w.sum())
    if not t > 0:
        return int((x == top).float().argmax()), float(-log_all), off
    rank = torch.empty(V, dtype=torch.long)
    rank[torch.from_numpy(np.lexsort((np.arange(V), -x.numpy())))] = torch.arange(V)
    keep = torch.ones(V, dtype=torch.bool)
    if 0 < k < V:
        keep &= rank < k
    keep &= torch.exp(z) >= min(m, 1.0)
    if p < 1:
        mass = torch.where(keep, w, 0.0)
        before = torch.zeros(V, dtype=torch.double)
        by = torch.argsort(rank)
        before[by] = torch.cumsum(mass[by], 0) - mass[by]
        keep &= (before < p * mass.sum()) | (rank == 0)
    mass = torch.cumsum(torch.where(keep, w, 0.0), 0)
    i = int((mass <= u * mass[-1]).sum())
    return i, float(z[i] - log_all), off


def close(got, want, off):
    # and the result's rounding (2^-24 of it), after a logarithm and a difference in 64 bits
    return got == want or abs(got - want) <= 2.0 ** -23 * abs(want) + 2.0 ** -40 + off


def rows_of(kind, V, B, g):
    x = 2.5 * torch.randn(B, V, generator=g)
    if kind == "ties":
        x = x.mul(2).round() / 2
    elif kind == "flat":
        x = torch.zeros(B, V)
    elif kind == "peaked":
        x = x * 0.01
        x[torch.arange(B), torch.randint(0, V, (B,), generator=g)] = 30.0
    elif kind == "masked":
        x[torch.rand(B, V, generator=g) < 0.9] = -INF
    elif kind == "odd":
        x[torch.rand(B, V, generator=g) < 0.3] = -INF
        x[torch.rand(B, V, generator=g) < 0.2] = float("nan")
        x[torch.rand(B, V, generator=g) < 0.1] = -0.0
        x[torch.rand(B, V, generator=g) < 0.1] = torch.finfo(torch.bfloat16).min
        x[0] = -INF
        if B > 1:
            x[1] = float("nan")
        if B > 2:
            x[2, V // 2] = INF
            x[2, V - 1] = INF
    return x


FILTERS = [(1.0, 0, 1.0, 0.0), (0.7, 50, 0.9, 0.0), (1.0, 1, 1.0, 0.0), (1.3, 0, 0.5, 0.0), (0.0, 5, 0.5, 0.1), (1.0, 0, 0.999, 0.02), (1.0, 7, 0.0, 0.0), (0.2, 1500, 0.97, 0.0),
           (1.0, 10 ** 6, 1.0, 1.0), (5.0, 3, 0.4, 0.5), (1.0, 0, 1e-9, 0.0), (100.0, 0, 0.9, 0.0), (1e-4, 20, 0.9, 0.0)]


def check(x, filters, dev, u, **kw):
    B = x.shape[0]
    t, k, p, m = (torch.tensor([f[i] for f in filters], dtype=torch.int32 if i == 1 else torch.float32) for i in range(4))
    ids, lp = sample_given(x.to(dev), u.to(dev), t.to(dev), k.to(dev), p.to(dev), m.to(dev), **kw)
    for r in range(B):
        i, want, off = definition(x[r].float().cpu(), float(u[r]), float(t[r]), int(k[r]), float(p[r]), float(m[r]))
        assert (int(ids[r]), close(float(lp[r]), want, off)) == (i, True), (r, filters[r], float(u[r]), int(ids[r]), i, float(lp[r]), want)


def cases(V, kind, dtype, seed, dev):
    g = torch.Generator().manual_seed(seed)
    B = len(FILTERS)
    x = rows_of(kind, V, B, g).to(dtype)
    u = torch.rand(B, generator=g)
    check(x, FILTERS, dev, u)
    check(x, FILTERS, dev, torch.tensor([0.0, 1 - 2.0 ** -24] * B)[:B])


@pytest.mark.parametrize("kind", ["normal", "ties", "flat", "peaked", "masked", "odd"])
@pytest.mark.parametrize("V", [1, 2, 37, 700])
def test_restatement(V, kind):
    cases(V, kind, torch.float32, V, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["normal", "ties", "flat", "peaked", "masked", "odd"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 2, 31, 513, 4608, 4609, 10007, 40000, 152064, 262144])
def test_kernel(V, kind, dtype):
    cases(V, kind, dtype, V + len(kind), "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["normal", "ties", "odd"])
@pytest.mark.parametrize("V", [3000, 40000, 152064])
def test_more_kept_by_top_k_than_there_are_pieces(V, kind):
    filters = [(1.0, 600, 0.9, 0.0), (0.7, 1000, 0.9, 0.01), (1.0, 2047, 0.99, 0.0), (1.3, 2048, 0.5, 0.001), (1.0, 2900, 0.9, 0.0), (0.9, 2950, 1.0, 0.0),
               (0.05, 1000, 0.999, 0.0)]
    g = torch.Generator().manual_seed(V)
    x = rows_of(kind, V, len(filters), g)
    for dtype in (torch.float32, torch.bfloat16):
        check(x.to(dtype), filters, "cuda", torch.rand(len(filters), generator=g))


@pytest.mark.gpu
def test_one_value_for_all_rows_and_pitches():
    g = torch.Generator().manual_seed(3)
    for odd in (0, 1, 3, 8):
        store = torch.randn(9, 5000 + odd, generator=g).cuda()
        x, u = store[:, :5000], torch.rand(9, generator=g).cuda()
        ids, lp = sample_given(x, u, 0.8, 40, 0.9, 0.01)
        full = lambda v, d: torch.full((9,), v, dtype=d, device="cuda")
        want = sample_given(x.contiguous(), u, full(0.8, torch.float32), full(40, torch.int32), full(0.9, torch.float32), full(0.01, torch.float32))
        assert torch.equal(ids, want[0])
        # A row's pieces of 256 begin on 16 bytes, so a pitch moves their borders and with them the order of its fp32 sum: either is within `off` of the definition, by what is
        # counted there.
        t, p, m = (float(torch.tensor(f)) for f in (0.8, 0.9, 0.01))
        for r in range(9):
            i, ref, off = definition(x[r].cpu(), float(u[r]), t, 40, p, m)
            assert int(ids[r]) == i and close(float(lp[r]), ref, off) and close(float(want[1][r]), ref, off)
        h = store.bfloat16()[:, odd // 2:5000]
        assert torch.equal(sample_given(h, u, 0.8, 40, 0.9, 0.01)[0], sample_given(h.contiguous(), u, 0.8, 40, 0.9, 0.01)[0])


@pytest.mark.gpu
def test_many_rows_have_the_same_bits_as_one():
    g = torch.Generator().manual_seed(4)
    x, u = (3 * torch.randn(300, 33000, generator=g)).bfloat16().cuda(), torch.rand(300, generator=g).cuda()
    ids, lp = sample_given(x, u, 0.9, 0, 0.95)
    for r in (0, 7, 150, 299):
        one = sample_given(x[r:r + 1], u[r:r + 1].clone(), 0.9, 0, 0.95)
        assert int(one[0]) == int(ids[r]) and float(one[1]) == float(lp[r])


@pytest.mark.gpu
def test_drawn_tokens_follow_the_distribution():
    """A grid of random numbers visits every kept token as often as its share says, to one cell."""
    g = torch.Generator().manual_seed(5)
    n, V = 4096, 50
    x = torch.randn(1, V, generator=g)
    u = (torch.arange(n) + 0.5) / n
    ids, _ = sample_given(x.cuda().expand(n, V), u.cuda(), 1.0, 10)
    p = torch.softmax(torch.where(x[0] >= x[0].topk(10).values[-1], x[0], -INF).double(), 0)
    seen = torch.bincount(ids.cpu().long(), minlength=V)
    assert ((seen - p * n).abs() <= 1.0 + 1e-6).all()


@pytest.mark.gpu
def test_captured_draws_take_new_numbers():
    g = torch.Generator().manual_seed(6)
    x, u = torch.randn(5, 20000, generator=g).cuda(), torch.zeros(5, device="cuda")
    out = (torch.zeros(5, dtype=torch.int32, device="cuda"), torch.zeros(5, device="cuda"))
    sample_given(x, u, 0.9, 100, 0.9, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sample_given(x, u, 0.9, 100, 0.9, out=out)
    for _ in range(3):
        x.copy_(torch.randn(5, 20000, generator=g))
        u.copy_(torch.rand(5, generator=g))
        graph.replay()
        want = sample_given(x, u, 0.9, 100, 0.9)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_refusals():
    x, u = torch.zeros(2, 8), torch.zeros(2)
    for bad in (lambda: sample_given(x.half(), u), lambda: sample_given(x[0], u), lambda: sample_given(x.t(), u), lambda: sample_given(x, u[:1]),
                lambda: sample_given(x, u.double()), lambda: sample_given(x, u, torch.ones(3)), lambda: sample_given(x, u, 1.0, torch.ones(2)),
                lambda: sample_given(x, u, 1.0, 0, torch.ones(2, dtype=torch.double)), lambda: sample_given(x[:, :0], u),
                lambda: sample_given(torch.zeros(1, sampler.MAX_VOCAB + 1), u[:1]), lambda: sample_given(x, u, out=(torch.zeros(2), torch.zeros(2)))):
        with pytest.raises(ValueError):
            bad()
    ids, lp = sample_given(x[:0], u[:0])
    assert ids.shape == (0,) and lp.shape == (0,)
