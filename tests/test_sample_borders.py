"""Top-p next to its border (ops/sampler.sample_given): the element that decides lies last in the vocabulary, and the random number is the largest below 1, so the
token says whether it stays.  Probabilities are the fp32 numbers around the border: steps of some 2^-24 of the mass."""
import numpy as np
import pytest
import torch

from vllm_omni_b200.ops.sampler import sample_given

LAST = 1 - 2.0 ** -24


def rows_of(kind, V, B, g):
    x = {"flat": 0.3, "normal": 1.0, "wide": 4.0, "steep": 12.0}[kind] * torch.randn(B, V, generator=g)
    x[torch.rand(B, V, generator=g) < 0.05] = -float("inf")
    return x


def borders(x, t, share):
    """For each row: its last element becomes the neighbour of the border at `share` of the mass; fp32 probabilities around that border, and what the definition keeps."""
    ps, ids, t = [], [], float(np.float32(t))                          # as the call takes it
    for r in range(x.shape[0]):
        row = x[r].double()
        order = np.lexsort((np.arange(row.numel()), -row.numpy()))
        z = np.exp((row.numpy() - row.max().item()) / t)[order]
        at = int((np.cumsum(z) < share * z.sum()).sum())
        x[r, -1] = x[r, order[max(at, 1)]]                             # ties with an earlier one: the last index is behind it
        row = x[r].double().numpy()
        order = np.lexsort((np.arange(row.size), -row))
        w = np.round(np.exp((row[order] - row.max()) / t) * 2.0 ** 44)
        before = np.cumsum(w) - w
        place = int((order == row.size - 1).nonzero()[0][0])
        middle = np.float32(before[place] / w.sum())
        for step in range(-3, 4):
            p = middle
            for _ in range(abs(step)):
                p = np.nextafter(p, np.float32(2.0 if step > 0 else -1.0))
            kept = (before < float(p) * w.sum()) | (np.arange(row.size) == 0)
            mass = np.zeros(row.size)
            mass[order[kept]] = w[kept]
            run = np.cumsum(mass)
            ps.append(float(p))
            ids.append(int((run <= LAST * run[-1]).sum()))
    return torch.tensor(ps, dtype=torch.float32), ids


def check(kind, V, B, dtype, t, share, odd, dev):
    g = torch.Generator().manual_seed(V + len(kind))
    x = rows_of(kind, V, B, g).to(dtype)
    p, want = borders(x, t, share)
    store = torch.zeros(B, V + odd, dtype=dtype, device=dev)
    store[:, :V] = x.to(dev)
    rows = torch.arange(B, device=dev).repeat_interleave(7)
    u = torch.full((7 * B,), LAST, device=dev)
    got = []
    for step in range(7):                                              # the same pitch for every draw
        got.append(sample_given(store[:, :V], u[:B], t, 0, p[step::7].to(dev).contiguous())[0].cpu())
    got = torch.stack(got, 1).flatten().tolist()
    assert rows.numel() == len(want)
    assert got == want
    assert 0 < sum(i == V - 1 for i in want) < len(want)               # some probabilities keep the element, some do not


@pytest.mark.parametrize("kind", ["flat", "normal", "wide", "steep"])
def test_restatement(kind):
    check(kind, 3000, 4, torch.float32, 1.0, 0.9, 0, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["flat", "normal", "wide", "steep"])
@pytest.mark.parametrize("V,t,share", [(40000, 1.0, 0.9), (152064, 1.3, 0.95), (10007, 0.5, 0.3)])
def test_kernel(kind, V, t, share):
    for odd in (0, 1, 3, 8):
        check(kind, V, 6, torch.float32, t, share, odd, "cuda")
    check(kind, V, 6, torch.bfloat16, t, share, 1, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("B", [1, 40, 300])
def test_kernel_with_more_and_fewer_blocks_a_row(B):
    check("normal", 33000, B, torch.float32, 1.0, 0.9, 1, "cuda")


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_numbers_are_what_a_tensor_of_them_is(dev):
    """A number counts as the fp32 or int32 that a row's value would be; what is no such integer is refused and does not wrap."""
    x, t = torch.tensor([[0.0, -1.0, -2.0, -3.0]], device=dev), 1.3
    z = np.exp(-np.arange(4) / float(np.float32(t)))
    share = np.float32(z[0] / z.sum())                                 # between the fp32 and the 64-bit temperature's border
    assert float(share) != np.exp(0) / np.exp(-np.arange(4) / t).sum()
    u = torch.tensor([LAST], device=dev)
    full = lambda v: torch.full((1,), v, device=dev)
    for p in (float(np.nextafter(share, np.float32(0))), float(share), float(np.nextafter(share, np.float32(1)))):
        ids, lp = sample_given(x, u, t, 0, p)
        want = sample_given(x, u, full(t), 0, full(p))
        assert int(ids[0]) == int(want[0][0]) and float(lp[0]) == float(want[1][0])
    a, b = float(np.float64(share) * (1 - 2.0 ** -40)), float(np.float64(share) * (1 + 2.0 ** -40))      # the same fp32 number
    assert int(sample_given(x, u, t, 0, a)[0]) == int(sample_given(x, u, t, 0, b)[0])
    for k in (2 ** 32 + 1, 2 ** 31, -2 ** 40, 1.5):
        with pytest.raises((ValueError, TypeError)):
            sample_given(x, u, 1.0, k)
    assert int(sample_given(x, u, 1.0, 2 ** 31 - 1)[0]) == 3 and int(sample_given(x, u, 1.0, 1)[0]) == 0


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("V", [5, 3000, 20000])
def test_parameters_that_are_not_numbers_cut_nothing(dev, V):
    g = torch.Generator().manual_seed(V)
    x, nan = torch.randn(3, V, generator=g).to(dev), float("nan")
    u = torch.tensor([0.0, 0.5, LAST], device=dev)
    for t, k, p, m, like in ((1.0, 0, nan, 0.0, (1.0, 0, 1.0, 0.0)), (1.0, 0, 1.0, nan, (1.0, 0, 1.0, 0.0)), (0.8, 3, 0.9, nan, (0.8, 3, 0.9, 0.0)), (0.8, 0, 0.9, nan, (0.8, 0, 0.9, 0.0)),
                             (nan, 3, 0.9, 0.1, (0.0, 3, 0.9, 0.1)), (0.8, 4, 0.9, -nan, (0.8, 4, 0.9, -1.0))):
        got, want = sample_given(x, u, t, k, p, m), sample_given(x, u, *like)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), (t, k, p, m)
    got, want = sample_given(x, torch.full((3,), nan, device=dev), 0.8, 50, 0.9), sample_given(x, torch.zeros(3, device=dev), 0.8, 50, 0.9)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("V,k", [(700, 0), (9000, 0), (9000, 600)])
@pytest.mark.parametrize("apart", [False, True])
def test_logits_further_apart_than_fp32_holds(dev, V, k, apart):
    """At a temperature of their size the lowest of all numbers still have mass: exp(-2) here, though their difference from the largest is no fp32 number."""
    x = torch.full((1, V), -3e38)
    x[0, :V // 50 if apart else V:1 if apart else 100] = 3e38          # beside one another, or one among many everywhere
    z = torch.where(x[0] > 0, 0.0, -2.0).double()
    w = torch.exp((x[0].double() - x[0].max().double()) / float(np.float32(3e38)))
    assert (w - torch.exp(z)).abs().max() < 1e-6
    for p in (0.3, 0.9):
        order = torch.sort(x[0], descending=True, stable=True).indices
        order = order[:k] if k else order
        n = torch.round(w * 2.0 ** 44)
        before = torch.cumsum(n[order], 0) - n[order]
        kept = torch.zeros(V, dtype=torch.bool)
        kept[order[before < float(np.float32(p)) * n[order].sum()]] = True
        mass = torch.cumsum(torch.where(kept, n, 0.0), 0)
        for u in (0.1, 0.77, LAST):
            u32 = torch.tensor([u], dtype=torch.float32)
            ids, lp = sample_given(x.to(dev), u32.to(dev), 3e38, k, p)
            i = int((mass <= float(u32) * mass[-1]).sum())
            assert int(ids[0]) == i
            assert abs(float(lp[0]) - float(torch.log(w[i] / w.sum()))) <= 2.0 ** -23 * 12 + 2.0 ** -20
