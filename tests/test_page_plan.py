"""Pages and slots of a step planned on the device (ops/page_plan.py): against a plain restatement that walks token by token, in place, captured, and what is
refused."""
import pytest
import torch

from vllm_omni_b200.ops import _native as nv
from vllm_omni_b200.ops import page_plan as PP

NAMES = ("q_start", "lens", "slots", "positions", "row_seq", "row_lens", "n_free")


def walk(free, n_free, tables, context, new, rows, page, num_blocks):
    """Token by token: every one takes the next row, and a page when it needs one."""
    free, tables = free[:n_free].tolist(), tables.tolist()
    q_start, lens, out = [0], [], []
    for s, (c, n) in enumerate(zip(context.tolist(), new.tolist())):
        have, held = -(-c // page), c
        stuck = False
        for i in range(n):
            if len(out) == rows:
                break
            pos = c + i
            if not stuck and pos // page >= have:
                if pos // page < len(tables[s]) and free:
                    tables[s][have] = free.pop()
                    have += 1
                else:
                    stuck = True
            if stuck:
                out.append((-1, pos, s, 0))
                continue
            held += 1
            p = tables[s][pos // page]
            out.append((p * page + pos % page, pos, s, pos + 1) if 0 <= p < num_blocks else (-1, pos, s, 0))
        q_start.append(len(out))
        lens.append(held)
    out += [(-1, 0, -1, 0)] * (rows - len(out))
    cols = [torch.tensor(c, dtype=torch.long) for c in zip(*out)] if rows else [torch.zeros(0, dtype=torch.long)] * 4
    return dict(q_start=torch.tensor(q_start), lens=torch.tensor(lens, dtype=torch.long), slots=cols[0], positions=cols[1], row_seq=cols[2], row_lens=cols[3],
                n_free=torch.tensor([len(free)])), torch.tensor(tables, dtype=torch.int32)


def setting(S, rows, page, most_context, most_new, free, seed, device="cpu", narrow=0, pitch=0):
    g = torch.Generator().manual_seed(seed)
    context = torch.randint(0, most_context + 1, (S,), generator=g, dtype=torch.int32)
    new = torch.randint(0, most_new + 1, (S,), generator=g, dtype=torch.int32)
    held = (context.long() + page - 1) // page
    W = max(1, -(-(most_context + most_new) // page) - narrow)
    W = max(W, int(held.max()) if S else 1)
    order = torch.randperm(int(held.sum()) + free + 3, generator=g).to(torch.int32)
    store = torch.full((S, W + pitch), -7, dtype=torch.int32)
    at = 0
    for s in range(S):
        store[s, :held[s]] = order[at:at + int(held[s])]
        at += int(held[s])
    stack = order[at:at + free + 3].clone()               # three entries above the height are not there
    store = store.to(device)
    return (PP.PagePool(stack.to(device), torch.tensor([free], dtype=torch.int32, device=device), page, order.numel()), store[:, :W], context.to(device),
            new.to(device), store)


SIZES = [(1, 1, 16, 40, 1, 3, 0), (1, 0, 16, 40, 5, 3, 0), (3, 40, 1, 9, 9, 30, 0), (7, 64, 8, 100, 9, 2, 0), (33, 700, 16, 300, 40, 1000, 0), (5, 3000, 128, 900, 600, 9, 0),
         (4, 2049, 48, 500, 512, 400, 6), (250, 2500, 16, 2000, 3, 60, 0), (6, 500, 32, 0, 90, 100, 0), (20, 64, 16, 50, 0, 4, 0), (9, 30, 16, 64, 20, 0, 0)]


@pytest.mark.parametrize("S,rows,page,most_context,most_new,free,narrow", SIZES)
@pytest.mark.parametrize("advance", [False, True])
def test_restatement_walks_like_tokens(S, rows, page, most_context, most_new, free, narrow, advance):
    pool, tables, context, new, _ = setting(S, rows, page, most_context, most_new, free, S + rows, narrow=narrow)
    want, want_tables = walk(pool.free, free, tables, context, new, rows, page, pool.num_blocks)
    before = context.clone()
    got = PP.plan_step(pool, tables, context, new, rows, advance=advance)
    for name in NAMES:
        assert torch.equal(getattr(got, name).long(), want[name].long()), name
    assert torch.equal(tables, want_tables)
    assert torch.equal(context.long(), want["lens"] if advance else before.long()) and int(pool.n_free) == (int(want["n_free"]) if advance else free)


@pytest.mark.gpu
@pytest.mark.parametrize("S,rows,page,most_context,most_new,free,narrow", SIZES + [(1024, 12000, 16, 3000, 20, 5000, 0), (4096, 9000, 16, 500, 4, 700, 0),
                                                                                  (2, 100000, 64, 3000, 60000, 2000, 0), (4095, 4096, 8, 30, 1, 4000, 0)])
@pytest.mark.parametrize("advance", [False, True])
def test_kernel_plans_like_the_restatement(S, rows, page, most_context, most_new, free, narrow, advance):
    pool, tables, context, new, store = setting(S, rows, page, most_context, most_new, free, S + rows, "cuda", narrow, pitch=3)
    want, want_tables = walk(pool.free.cpu(), free, tables.cpu(), context.cpu(), new.cpu(), rows, page, pool.num_blocks)
    before = context.clone()
    for _ in range(1 if advance else 2):                  # without `advance` the same call gives the same plan
        got = PP.plan_step(pool, tables, context, new, rows, advance=advance)
        for name in NAMES:
            assert torch.equal(getattr(got, name).cpu().long(), want[name].long()), name
        assert torch.equal(tables.cpu(), want_tables) and bool((store[:, tables.shape[1]:] == -7).all())
    assert torch.equal(context.cpu().long(), want["lens"] if advance else before.cpu().long())
    assert int(pool.n_free) == (int(want["n_free"]) if advance else free)
    assert nv.check_status(pool.device) == 0


@pytest.mark.gpu
def test_lengths_in_place_and_on_another_stream():
    pool, tables, context, new, _ = setting(300, 9000, 16, 500, 30, 2000, 5, "cuda")
    want, _ = walk(pool.free.cpu(), 2000, tables.cpu(), context.cpu(), new.cpu(), 9000, 16, pool.num_blocks)
    plan = PP.StepPlan.empty(300, 9000, "cuda")
    plan = PP.StepPlan(plan.q_start, context, plan.slots, plan.positions, plan.row_seq, plan.row_lens, pool.n_free)       # both its results and its operands
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        PP.plan_step(pool, tables, context, new, 9000, out=plan)
    torch.cuda.current_stream().wait_stream(side)
    for name in NAMES:
        assert torch.equal(getattr(plan, name).cpu().long(), want[name].long()), name


@pytest.mark.gpu
def test_pages_outside_the_pool_get_no_slot():
    pool, tables, context, new, _ = setting(4, 40, 16, 100, 8, 20, 2, "cuda")
    context.fill_(20)
    new.fill_(3)
    tables[:, 1] = torch.tensor([pool.num_blocks, -1, 0, 2 ** 31 - 1], dtype=torch.int32)
    got = PP.plan_step(pool, tables, context, new, 40, advance=False)
    assert got.slots[:12].tolist() == [-1] * 6 + [4, 5, 6] + [-1] * 3 and got.row_lens[:12].tolist() == [0] * 6 + [21, 22, 23] + [0] * 3
    with pytest.raises(nv.NativeError):
        nv.check_status(pool.device)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("lens", [[0], [5, 0, 33, 16, 17], [700] * 40 + [0, 1], [1] * 2000])
def test_pages_come_back(device, lens):
    page, S = 16, len(lens)
    per = [-(-n // page) for n in lens]
    W, total = max(1, max(per)), sum(per)
    pool = PP.PagePool.full(total + 4, page, device)
    tables, context = torch.zeros(S, W, dtype=torch.int32, device=device), torch.zeros(S, dtype=torch.int32, device=device)
    PP.plan_step(pool, tables, context, torch.tensor(lens, dtype=torch.int32, device=device), sum(lens))
    assert context.tolist() == lens and int(pool.n_free) == 4
    done = torch.tensor([i % 3 != 1 for i in range(S)], device=device)
    back = [p for s in range(S) if done[s] for p in tables[s, :per[s]].tolist()]
    PP.release_pages(pool, tables, context, done)
    assert context.tolist() == [0 if done[s] else lens[s] for s in range(S)]
    assert int(pool.n_free) == 4 + len(back) and pool.free[4:4 + len(back)].tolist() == back
    kept = [p for s in range(S) if not done[s] for p in tables[s, :per[s]].tolist()]
    assert sorted(kept + pool.free[:4 + len(back)].tolist()) == list(range(total + 4))


@pytest.mark.gpu
def test_more_pages_than_fit_come_back():
    pool = PP.PagePool.full(4, 16, "cuda")
    tables = torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2)
    lens = torch.tensor([32, 32], dtype=torch.int32, device="cuda")
    PP.release_pages(pool, tables, lens, torch.tensor([True, True], device="cuda"))
    assert int(pool.n_free) == 4 and pool.free.tolist() == [3, 2, 1, 0]
    with pytest.raises(nv.NativeError):
        nv.check_status(pool.device)


@pytest.mark.gpu
def test_captured_steps_take_pages():
    S, page = 5, 16
    pool = PP.PagePool.full(100, page, "cuda")
    tables, context = torch.zeros(S, 20, dtype=torch.int32, device="cuda"), torch.zeros(S, dtype=torch.int32, device="cuda")
    new, plan = torch.tensor([3, 0, 1, 7, 2], dtype=torch.int32, device="cuda"), PP.StepPlan.empty(S, 16, "cuda")
    PP.plan_step(pool, tables, context, new, 16, out=plan, advance=False)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        PP.plan_step(pool, tables, context, new, 16, out=plan)
    ref = PP.PagePool.full(100, page, "cpu")
    t, c = torch.zeros(S, 20, dtype=torch.int32), torch.zeros(S, dtype=torch.int32)
    for _ in range(9):
        g.replay()
        want = PP.plan_step(ref, t, c, new.cpu(), 16)
        for name in NAMES:
            assert torch.equal(getattr(plan, name).cpu(), getattr(want, name)), name
        used = [-(-int(n) // page) for n in c]
        assert all(torch.equal(tables[s, :used[s]].cpu(), t[s, :used[s]]) for s in range(S))


def test_refusals():
    pool = PP.PagePool.full(8, 16, "cpu")
    tables, ints = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for bad in (lambda: PP.PagePool(torch.zeros(4), torch.zeros(1, dtype=torch.int32), 16), lambda: PP.PagePool.full(1 << 28, 16, "meta"), lambda: PP.PagePool.full(4, 0, "cpu"),
                lambda: PP.plan_step(pool, tables, ints.long(), ints, 4), lambda: PP.plan_step(pool, tables, ints, ints[:1], 4), lambda: PP.plan_step(pool, tables.t(), ints, ints, 4),
                lambda: PP.plan_step(pool, tables[:1], ints, ints, 4), lambda: PP.plan_step(pool, tables, ints, ints, -1),
                lambda: PP.plan_step(pool, tables, ints, ints, 4, out=PP.StepPlan.empty(2, 5, "cpu")), lambda: PP.plan_step(pool, tables.float(), ints, ints, 4),
                lambda: PP.release_pages(pool, tables, ints, ints), lambda: PP.release_pages(pool, tables, ints, torch.zeros(3, dtype=torch.bool)),
                lambda: PP.plan_step(pool, torch.zeros(5000, 2, dtype=torch.int32), torch.zeros(5000, dtype=torch.int32), torch.zeros(5000, dtype=torch.int32), 4),
                lambda: PP.release_pages(PP.PagePool.full(2, 16, "cpu"), tables, torch.full((2,), 40, dtype=torch.int32), torch.ones(2, dtype=torch.bool))):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("S,W,bad", [(1, 1, [(0, 0, -1)]), (3, 4, [(0, 1, 99), (2, 3, -7)]), (60, 9, [(s, s % 9, 540 + s) for s in range(0, 60, 7)]),
                                     (2000, 2, [(s, 0, -2 ** 31) for s in range(1, 2000, 3)])])
def test_ids_outside_the_pool_do_not_come_back(device, S, W, bad):
    page = 8
    tables = torch.arange(S * W, dtype=torch.int32).view(S, W)
    for s, col, page_id in bad:
        tables[s, col] = page_id
    pool = PP.PagePool(torch.full((S * W + 5,), -3, dtype=torch.int32, device=device), torch.tensor([2], dtype=torch.int32, device=device), page, S * W)
    lens, done = torch.full((S,), W * page, dtype=torch.int32, device=device), torch.ones(S, dtype=torch.bool, device=device)
    with pytest.raises((ValueError, nv.NativeError)):
        PP.release_pages(pool, tables.to(device), lens, done)
        nv.check_status(pool.device)
    back = [p for p in tables.flatten().tolist() if 0 <= p < S * W]
    assert int(pool.n_free) == 2 + len(back) and pool.free[:2 + len(back)].tolist() == [-3, -3] + back
    assert not lens.any()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_sequences_whose_pages_do_not_fit_keep_them(device):
    lens = [17, 16, 0, 40, 5, 0]                          # pages of 8: 3, 2, none, 5 that do not fit, 1 behind them, none
    pool = PP.PagePool(torch.full((9,), -3, dtype=torch.int32, device=device), torch.tensor([1], dtype=torch.int32, device=device), 8, 100)
    tables, context = torch.arange(30, dtype=torch.int32, device=device).view(6, 5), torch.tensor(lens, dtype=torch.int32, device=device)
    with pytest.raises((ValueError, nv.NativeError)):
        PP.release_pages(pool, tables, context, torch.ones(6, dtype=torch.bool, device=device))
        nv.check_status(pool.device)
    assert context.tolist() == [0, 0, 0, 40, 5, 0]
    assert int(pool.n_free) == 6 and pool.free.tolist() == [-3, 0, 1, 2, 5, 6, -3, -3, -3]
