"""A decode loop that never asks the host: pages and slots planned, keys and values written in 8 bits, attention over them, the next token drawn, pages of finished
sequences given back, all in one captured graph."""
import pytest
import torch

from vllm_omni_b200.ops import _native as nv
from vllm_omni_b200.ops import kv8, page_plan as PP
from vllm_omni_b200.ops.sampler import sample_given

S, H, HKV, D, PAGE, V, LIMIT, WIDTH = 6, 8, 2, 64, 8, 500, 40, 6


class Loop:
    def __init__(self, dev, pages=S * WIDTH):
        g = torch.Generator().manual_seed(0)
        rows = H * D + 2 * HKV * D
        self.embed = torch.randn(V, rows, generator=g).to(torch.bfloat16).to(dev)
        self.head = (torch.randn(V, H * D, generator=g) / 8).to(torch.bfloat16).to(dev)
        self.limits = torch.tensor([LIMIT, 7, LIMIT - 5, 16, 1, 23], dtype=torch.int32, device=dev)
        self.numbers = torch.rand(200, S, generator=g).to(dev)
        self.cache = kv8.Kv8Cache.empty(pages, PAGE, HKV, D, dev)
        self.pool = PP.PagePool.full(pages, PAGE, dev)
        self.plan = PP.StepPlan.empty(S, S + 2, dev)                # two rows of padding
        z = lambda *s, dt=torch.int32: torch.zeros(*s, dtype=dt, device=dev)
        self.tables, self.context, self.new = z(S, WIDTH), z(S), torch.ones(S, dtype=torch.int32, device=dev)
        self.ids, self.logprob, self.u = z(S), z(S, dt=torch.float32), z(S, dt=torch.float32)
        self.x, self.out = z(S + 2, rows, dt=torch.bfloat16), z(S + 2, H, D, dt=torch.bfloat16)
        self.done = z(S, dt=torch.bool)

    def step(self):
        PP.release_pages(self.pool, self.tables, self.context, self.done)
        PP.plan_step(self.pool, self.tables, self.context, self.new, S + 2, out=self.plan)
        self.x[:S].copy_(self.embed[self.ids.long()])
        q, k, v = self.x.split([H * D, HKV * D, HKV * D], 1)
        kv8.kv8_write(k.view(-1, HKV, D), v.view(-1, HKV, D), self.cache, self.plan.slots)
        kv8.kv8_decode(q.view(-1, H, D), self.cache, self.tables, self.plan.row_lens, self.plan.row_seq, out=self.out)
        logits = self.out[:S].view(S, -1).float() @ self.head.float().t()
        sample_given(logits, self.u, 0.8, 50, 0.95, 0.01, out=(self.ids, self.logprob))
        torch.ge(self.context, self.limits, out=self.done)

    def run(self, n, step):
        seen = []
        for i in range(n):
            self.u.copy_(self.numbers[i])
            step()
            seen.append((self.ids.clone(), self.context.clone(), self.pool.n_free.clone(), self.plan.slots.clone(), self.out.clone()))
        return seen


def check(loop, seen, limits):
    context, live = [0] * S, [0] * S
    for ids, ctx, n_free, slots, out in seen:
        context = [1 if c >= n else c + 1 for c, n in zip(context, limits)]
        assert ctx.tolist() == context
        assert int(n_free) == loop.cache.pages - sum(-(-c // PAGE) for c in context)
        assert len(set(slots[:S].tolist())) == S and slots[S:].tolist() == [-1, -1] and int(slots[:S].min()) >= 0
        assert bool((ids >= 0).all()) and bool((out[S:] == 0).all()) and bool(out[:S].isfinite().all())
    held = [p for s in range(S) for p in loop.tables[s, :-(-context[s] // PAGE)].tolist()]
    assert sorted(held + loop.pool.free[:int(loop.pool.n_free)].tolist()) == list(range(loop.cache.pages))


def test_on_the_host():
    loop = Loop("cpu")
    check(loop, loop.run(60, loop.step), loop.limits.tolist())


@pytest.mark.gpu
def test_captured():
    eager = Loop("cuda")
    want = eager.run(100, eager.step)
    check(eager, want, eager.limits.tolist())
    loop = Loop("cuda")
    warm = Loop("cuda")
    warm.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loop.step()
    got = loop.run(100, graph.replay)
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    # the last step's attention against the restatement on the host, on the same pages
    host = kv8.Kv8Cache(loop.cache.k.cpu(), loop.cache.v.cpu(), loop.cache.k_scale.cpu(), loop.cache.v_scale.cpu())
    q = loop.x[:, :H * D].cpu().view(-1, H, D)
    ref = kv8.kv8_decode(q, host, loop.tables.cpu(), loop.plan.row_lens.cpu(), loop.plan.row_seq.cpu()).double()
    most = host.v.float().abs().amax() * host.v_scale.max()
    # either side rounds its result to bf16 (2^-8 of it); weights in f16, 2^-11 of each, over values of at most `most`, and as much again for fp32 scores
    assert ((loop.out.cpu().double() - ref).abs() <= ref.abs() * 2.0 ** -7 + most * 2.0 ** -10).all()
    assert nv.check_status(loop.pool.device) == 0


@pytest.mark.gpu
def test_too_few_pages():
    """Sequences that get no page stand still and go on once others have given theirs back."""
    loop = Loop("cuda", pages=9)
    seen = loop.run(200, loop.step)
    for ids, ctx, n_free, slots, out in seen:
        assert bool((ctx <= loop.limits).all()) and int(n_free) >= 0
    held = [p for s in range(S) for p in loop.tables[s, :-(-int(loop.context[s]) // PAGE)].tolist()]
    assert sorted(held + loop.pool.free[:int(loop.pool.n_free)].tolist()) == list(range(9))
    assert nv.check_status(loop.pool.device) == 0


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_sequences_wait_for_pages_and_go_on(dev):
    """Fewer pages than the sequences want: who gets none stands still, with no slot and its length as it was, and goes on when others have given theirs back.  They want 5, 1, 5,
    2, 1 and 3 pages, and sequences that all wait hold one less each, 11 in all: with 12 one of them has all it wants, ends and gives back."""
    loop = Loop(dev, pages=12)
    limits, before, waited, went_on = loop.limits.tolist(), [0] * S, set(), set()
    for i, (ids, ctx, n_free, slots, out) in enumerate(loop.run(200, loop.step)):
        ctx, slots = ctx.tolist(), slots.tolist()
        for s in range(S):
            context = 0 if before[s] >= limits[s] else before[s]       # those that were done began again
            assert ctx[s] == context + (slots[s] >= 0)
            if slots[s] < 0:
                assert context % PAGE == 0                             # only a new page can be missing
                if i < 150:                                            # the others have steps left to go on in
                    waited.add(s)
            elif s in waited:
                went_on.add(s)
        assert int(n_free) == 12 - sum(-(-c // PAGE) for c in ctx)
        before = ctx
    assert waited and went_on == waited
