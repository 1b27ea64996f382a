"""What a decode step does on the GPU between its projections: pages and slots planned from request lengths, keys and values written to
a cache of 8 bits, attention over that cache (decoded tokens and prompt portions), the next token drawn from given random numbers.

Plan.  A pool is a stack of free pages; sequence s has context[s] cached tokens in the pages of tables[s] and gets new[s] more, in rows of its own
of a batch with a fixed number of rows.  Pages are handed out in the order of the sequences; tokens that find no page, no column of the table
or no row are not taken (slot -1, no visible keys).

Cache.  A value is an e4m3 code times a power of two for each page and KV head, for keys and values apart: the least one by which the largest
finite value fits 448 (at least 2^-120).  A page whose first row is written starts over; else the scale only grows, and the rows before the
first written one are rounded again.  Infinities saturate.

Sampling.  Weights exp((x - max) / temperature) are whole multiples of 2^-44, so that sums have no order.  Of the order by logit (ties: the lower id first)
the first top_k stay, of these the ones of at least min_p of the largest, of these all before which less than top_p of their mass lies.
The token is the first kept id at which the running mass in the vocabulary's order passes u times the kept mass; its log probability is that of the
whole row at the temperature.  temperature 0: the largest.

The plain forms compute in fp32 or 64 bits with elementary operations; ``exact`` is the definition in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BF = torch.bfloat16
E4M3 = torch.float8_e4m3fn
MOST_KEYS = 64 * 4096 * 8 * 128            # keys x KV heads x channels of the largest listed cache
MOST_SCORES = 2039 * 32 * 16384            # scores of the largest listed prompt portion
LEAST = -120                               # smallest exponent of a page's scale


def listed():
    return [
        # one conversation's next token: all latency
        dict(name="plan_1", path="plan", seqs=1, rows=1, most_context=4000, most_new=1, page=16, short=False),
        # conversations beside prompts of one step, as many pages as are free: some prompts are cut
        dict(name="plan_12289", path="plan", seqs=250, rows=12289, most_context=8000, most_new=100, page=16, short=True),
        # tokens of seven conversations go to their pages, whose scales now and then grow; the pages are then handed over in bf16
        dict(name="write_7", path="write", seqs=7, new=1, most_context=300, kv=8, dim=128, page=16),
        # long prompts, an odd number of tokens each
        dict(name="write_16435", path="write", seqs=5, new=3287, most_context=700, kv=8, dim=128, page=64),
        # a short conversation's next token
        dict(name="decode_1", path="decode", seqs=1, per=1, most_keys=100, heads=32, kv=8, dim=128, page=16),
        # one very long document, pages of 64 tokens
        dict(name="decode_131071", path="decode", seqs=1, per=1, most_keys=131071, heads=64, kv=8, dim=128, page=64),
        # 64 conversations of uneven lengths
        dict(name="decode_64", path="decode", seqs=64, per=1, most_keys=4096, heads=32, kv=8, dim=128, page=16),
        # three proposed tokens behind the last one of each sequence, small heads
        dict(name="decode_23x4", path="decode", seqs=23, per=4, most_keys=2100, heads=16, kv=4, dim=64, page=32),
        # a follow-up question, heads of their own
        dict(name="prefill_131", path="prefill", rows=131, context=1000, heads=16, kv=16, dim=64, page=16),
        # a portion of a long prompt
        dict(name="prefill_2039", path="prefill", rows=2039, context=14345, heads=32, kv=8, dim=128, page=64),
        # one row of logits, all filters
        dict(name="sample_1", path="sample", rows=1, vocab=151936, bf16=False, odd=0, filters=True),
        # 256 rows in bf16, odd pitch, some rows greedy, some without filters
        dict(name="sample_256", path="sample", rows=256, vocab=152064, bf16=True, odd=1, filters=False),
    ]


def draw(rng):
    def spread(lo, hi, step=1):
        v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
        return min(hi, max(lo, round(v / step) * step))

    path = rng.choice(["plan", "write", "decode", "decode", "prefill", "sample", "sample"])
    page = rng.choice([8, 16, 32, 64, 128])
    if path == "plan":
        rows = spread(1, 12289)
        return dict(path=path, seqs=spread(1, min(rows, 1024)), rows=rows, most_context=spread(10, 8000), most_new=spread(1, 2000), page=page,
                    short=rng.random() < 0.3)
    if path == "write":
        new = spread(1, 16435)
        return dict(path=path, seqs=spread(1, max(1, 16435 // new)) if new > 64 else spread(1, 128), new=new, most_context=spread(10, 700), kv=rng.choice([1, 2, 4, 8]),
                    dim=rng.choice([64, 128]), page=page)
    if path == "decode":
        kv, group, dim = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16]), rng.choice([64, 128])
        keys = spread(1, 131071)
        per = rng.choice([1, 1, 1, 2, 4, 5])
        return dict(path=path, seqs=spread(1, max(1, min(256, MOST_KEYS // (keys * kv * dim * (2 if per > 1 else 1))))), per=per, most_keys=max(keys, per), heads=kv * group,
                    kv=kv, dim=dim, page=page)
    if path == "prefill":
        kv, group, dim = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 7]), rng.choice([64, 128])
        rows, context = spread(2, 2039), spread(1, 14345)
        kv = max(1, min(kv, MOST_SCORES // (rows * (rows + context) * group)))
        return dict(path=path, rows=rows, context=context if rng.random() < 0.9 else 0, heads=kv * group, kv=kv, dim=dim, page=page)
    vocab = spread(1000, 152064)
    return dict(path=path, rows=spread(1, 256), vocab=vocab, bf16=rng.random() < 0.5, odd=rng.choice([0, 1, 8]), filters=rng.random() < 0.5)


# ------------------------------------------------------------------ what a program has in hand
def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) % (1 << 62))


def _spread(lo, hi, n, g):
    """n lengths from lo to hi, evenly, in a random order."""
    v = torch.linspace(lo, hi, n, device=DEV).round().to(torch.int32) if n > 1 else torch.full((1,), (lo + hi) // 2, dtype=torch.int32, device=DEV)
    return v[torch.randperm(n, device=DEV, generator=g)]


def _kv_rows(rows, kv, dim, g):
    """Keys or values as projections leave them: heads at sizes of their own, some channels that stand out, a few loud tokens."""
    x = torch.randn(rows, kv, dim, device=DEV, generator=g)
    x *= torch.exp(0.5 * torch.randn(kv, 1, device=DEV, generator=g))
    x *= torch.where(torch.rand(kv, dim, device=DEV, generator=g) < 0.03, 8.0, 1.0)
    x *= torch.where(torch.rand(rows, 1, 1, device=DEV, generator=g) < 0.02, 5.0, 1.0)
    return x.to(BF)


def _page_lists(lens, page, g, spare=0):
    """Pages of sequences of `lens` tokens, in a random order of a pool: block tables int32 [S, W], pages in the pool."""
    per = (lens.long() + page - 1) // page
    width, total = max(1, int(per.max())), int(per.sum()) + spare
    order = torch.randperm(max(1, total), device=DEV, generator=g).to(torch.int32)
    first = torch.cumsum(per, 0) - per
    at = torch.arange(width, device=DEV)
    inside = at[None] < per[:, None]
    tables = torch.where(inside, order[(first[:, None] + at[None]).clamp(max=max(0, total - 1))], 0).to(torch.int32)
    return tables, max(1, total)


def _slots_of(tables, seq, pos, page):
    return (tables[seq, pos // page].long() * page + pos % page).to(torch.int32)


def _ragged(lens):
    """(sequence, position) of every token of sequences of `lens` tokens."""
    lens = lens.long()
    seq = torch.repeat_interleave(torch.arange(lens.numel(), device=DEV), lens)
    return seq, torch.arange(seq.numel(), device=DEV) - (torch.cumsum(lens, 0) - lens)[seq]


def _pool(pages, page, kv, dim):
    return dict(k=torch.zeros(pages, page, kv, dim, dtype=E4M3, device=DEV), v=torch.zeros(pages, page, kv, dim, dtype=E4M3, device=DEV),
                ks=torch.full((pages, kv), 2.0 ** LEAST, device=DEV), vs=torch.full((pages, kv), 2.0 ** LEAST, device=DEV))


def prepare(case, seed):
    g, path = _generator(seed), case["path"]
    st = dict(case=case)
    if path == "plan":
        n, page, rows = case["seqs"], case["page"], case["rows"]
        context, st["new"] = _spread(0, case["most_context"], n, g), _spread(1, case["most_new"], n, g)
        reach = context + st["new"]
        st["tables"], owned = _page_lists(context, page, g)
        wide = (case["most_context"] + case["most_new"]) // page + 1
        st["tables"] = torch.nn.functional.pad(st["tables"], (0, wide - st["tables"].shape[1])).contiguous()
        need = int(((reach + page - 1) // page - (context + page - 1) // page).sum())
        free = max(1, need // 2 if case["short"] else need + 5)
        st["free"] = (owned + torch.randperm(free, device=DEV, generator=g)).to(torch.int32)
        st["n_free"] = torch.tensor([free], dtype=torch.int32, device=DEV)
        st["context"], st["pages"] = context, owned + free
    elif path == "write":
        n, page, kv, dim = case["seqs"], case["page"], case["kv"], case["dim"]
        context = _spread(0, case["most_context"], n, g)
        lens = context + case["new"]
        tables, pages = _page_lists(lens, page, g)
        st.update(_pool(pages, page, kv, dim))
        seq, pos = _ragged(context)
        _write(st, _kv_rows(seq.numel(), kv, dim, g), _kv_rows(seq.numel(), kv, dim, g), _slots_of(tables, seq, pos, page))
        seq, pos = _ragged(torch.full_like(lens, case["new"]))
        st["slots"] = _slots_of(tables, seq, pos + context.long()[seq], page)
        st["new_k"], st["new_v"] = _kv_rows(seq.numel(), kv, dim, g), _kv_rows(seq.numel(), kv, dim, g)
        seq, pos = _ragged(lens)
        st["back"] = _slots_of(tables, seq, pos, page)
    elif path in ("decode", "prefill"):
        page, kv, dim = case["page"], case["kv"], case["dim"]
        if path == "decode":
            n, per, most = case["seqs"], case["per"], case["most_keys"]
            lens = _spread(max(per, int(0.6 * most)), most, n, g) if n > 1 else torch.full((1,), most, dtype=torch.int32, device=DEV)
        else:
            n, per = 1, case["rows"]
            lens = torch.tensor([case["rows"] + case["context"]], dtype=torch.int32, device=DEV)
        st["tables"], pages = _page_lists(lens, page, g)
        st.update(_pool(pages, page, kv, dim))
        seq, pos = _ragged(lens)
        _write(st, _kv_rows(seq.numel(), kv, dim, g), _kv_rows(seq.numel(), kv, dim, g), _slots_of(st["tables"], seq, pos, page))
        st["q"] = torch.randn(n * per, case["heads"], dim, device=DEV, generator=g).to(BF)
        st["per"] = per
        st["row_seq"] = torch.arange(n, device=DEV, dtype=torch.int32).repeat_interleave(per)
        st["row_lens"] = (lens.repeat_interleave(per) - per + 1 + torch.arange(per, device=DEV, dtype=torch.int32).repeat(n)).to(torch.int32)
    else:
        rows, vocab = case["rows"], case["vocab"]
        x = 2.5 * torch.randn(rows, vocab, device=DEV, generator=g)
        x += torch.where(torch.rand(rows, vocab, device=DEV, generator=g) < 8.0 / vocab, 7.0, 0.0)        # what a model thinks of next
        store = torch.empty(rows, vocab + case["odd"], dtype=BF if case["bf16"] else torch.float32, device=DEV)
        st["logits"] = store[:, :vocab]
        st["logits"].copy_(x)
        st["u"] = torch.rand(rows, device=DEV, generator=g)
        pick = lambda *v: torch.tensor(v, device=DEV)[torch.randint(0, len(v), (rows,), device=DEV, generator=g)]
        if case["filters"]:
            st["temperature"], st["top_k"] = pick(0.6, 0.7, 0.9), pick(20, 50, 200).to(torch.int32)
            st["top_p"], st["min_p"] = pick(0.8, 0.9, 0.95), pick(0.0, 0.01, 0.05)
        else:
            st["temperature"], st["top_k"] = pick(0.0, 0.7, 1.0, 1.3), pick(0, 0, 50).to(torch.int32)
            st["top_p"], st["min_p"] = pick(1.0, 0.9, 0.95), pick(0.0, 0.0, 0.02)
    return st


# ------------------------------------------------------------------ plain forms
def _plan(st):
    case, tables = st["case"], st["tables"]
    page, rows, width = case["page"], case["rows"], tables.shape[1]
    context, new, free = st["context"].long(), st["new"].long(), int(st["free"].numel())
    n_free = st["n_free"].long()
    ends = torch.cumsum(new, 0).clamp(max=rows)
    starts = torch.cat([torch.zeros_like(ends[:1]), ends])
    fit = ends - starts[:-1]
    mine = (context + page - 1) // page
    need = (((context + fit + page - 1) // page).clamp(max=width) - mine).clamp(min=0)
    base = torch.cumsum(need, 0) - need
    got = torch.minimum((n_free - base).clamp(min=0), need)
    column = torch.arange(width, device=DEV)[None]
    fresh = (column >= mine[:, None]) & (column < (mine + got)[:, None])
    at = (n_free - 1 - base)[:, None] - (column - mine[:, None])
    tables.copy_(torch.where(fresh, st["free"][at.clamp(0, free - 1)], tables))
    taken = torch.minimum(fit, (mine + got) * page - context).clamp(min=0)
    t = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(starts[1:], t, right=True)
    live = seq < new.numel()
    s = seq.clamp(max=new.numel() - 1)
    i = t - starts[s]
    pos = context[s] + i
    inside = live & (i < taken[s])
    slot = tables[s, (pos // page).clamp(max=width - 1)].long() * page + pos % page
    i32 = torch.int32
    return dict(q_start=starts.to(i32), lens=(context + taken).to(i32), slots=torch.where(inside, slot, -1).to(i32), positions=torch.where(live, pos, 0),
                row_seq=torch.where(live, s, -1).to(i32), row_lens=torch.where(inside, pos + 1, 0).to(i32),
                n_free=(n_free - torch.minimum(need.sum(), n_free)).to(i32), tables=tables)


def _exponent(size):
    """Least e with size <= 448 * 2^e, at least LEAST."""
    f, e = torch.frexp(size)                                  # size = f * 2^e, f in [1/2, 1)
    return torch.where(size > 0, e - 9 + (f > 0.875).to(e.dtype), LEAST).clamp(min=LEAST)


def _power(e):
    """2^e in fp32, exactly (exp2 of a GPU is off by an ulp now and then)."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _codes(x, e):
    return (x * _power(-e)).clamp(-448.0, 448.0).to(E4M3)


def _write_one(codes, scale, x, slots):
    pages, page, kv, dim = codes.shape
    slot = slots.long()
    at, offset = slot // page, slot % page
    x = x.float()
    size = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)                                                        # [T, kv]
    most = torch.zeros(pages, kv, device=DEV).scatter_reduce(0, at[:, None].expand(-1, kv), size, "amax")
    first = torch.full((pages,), page, device=DEV).scatter_reduce(0, at, offset, "amin")                          # lowest row written, `page`: none
    old = torch.frexp(scale).exponent - 1
    e = torch.where((first == 0)[:, None], _exponent(most), torch.maximum(old, _exponent(most)))
    e = torch.where((first == page)[:, None], old, e)
    again = (torch.arange(page, device=DEV)[None] < first[:, None]) & (first < page)[:, None]                     # rows before it
    again = again[:, :, None] & (e > old)[:, None]
    value = codes.float()
    codes.copy_(torch.where(again[..., None], (value * _power(old - e)[:, None, :, None]).to(E4M3).float(), value).to(E4M3))
    codes.view(torch.uint8).view(-1, kv, dim)[slot] = _codes(x, e[at][:, :, None]).view(torch.uint8)
    scale.copy_(_power(e))


def _write(st, k, v, slots):
    if slots.numel():
        _write_one(st["k"], st["ks"], k, slots)
        _write_one(st["v"], st["vs"], v, slots)


def _read(codes, scale, slots):
    slot = slots.long()
    return (codes.view(torch.uint8).view(-1, *codes.shape[2:])[slot].view(E4M3).float() * scale[slot // codes.shape[1]].unsqueeze(-1)).to(BF)


def _whole(codes, scale, tables):
    """fp32 values of every sequence's pages: [S, keys, kv, dim]."""
    t = tables.long()
    x = codes.view(torch.uint8)[t].view(E4M3).float() * scale[t][:, :, None, :, None]
    return x.flatten(1, 2)


def _attend(st):
    q, per = st["q"].float(), st["per"]
    k, v = _whole(st["k"], st["ks"], st["tables"]), _whole(st["v"], st["vs"], st["tables"])
    kv, dim = k.shape[2], k.shape[3]
    q = q.view(-1, per, kv, q.shape[1] // kv, dim) / math.sqrt(dim)
    s = torch.einsum("srhgd,slhd->shrgl", q, k)
    hidden = torch.arange(k.shape[1], device=DEV)[None, None] >= st["row_lens"].view(-1, per, 1)                  # [S, per, keys]
    s.masked_fill_(hidden[:, None, :, None], -math.inf)
    w = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.einsum("shrgl,slhd->srhgd", w, v) / w.sum(-1).permute(0, 2, 1, 3).unsqueeze(-1)
    return o.reshape(st["q"].shape).to(BF)


def _sample(st):
    x, u = st["logits"].float(), st["u"].double()
    rows, vocab = x.shape
    top = x.amax(-1, keepdim=True)
    t = st["temperature"].double()[:, None]
    z = (x.double() - top.double()) / torch.where(t > 0, t, 1.0)
    weight = torch.round(torch.exp(z) * 2.0 ** 44).long()
    whole = weight.sum(-1)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    place = torch.arange(vocab, device=DEV)[None]
    k = st["top_k"].long()[:, None]
    sorted_w = weight.gather(-1, order)
    keep = (place < torch.where(k > 0, k, vocab)) & (torch.exp(z.gather(-1, order)) >= st["min_p"].double()[:, None])
    sorted_w = torch.where(keep, sorted_w, 0)
    before = torch.cumsum(sorted_w, -1) - sorted_w
    p = st["top_p"].double()[:, None]
    keep &= (p >= 1) | (before.double() < p * sorted_w.sum(-1, keepdim=True).double()) | (place == 0)
    kept = torch.zeros_like(keep).scatter(-1, order, keep)
    mass = torch.cumsum(torch.where(kept, weight, 0), -1)
    want = u[:, None] * mass[:, -1:].double()
    ids = torch.where(t[:, 0] > 0, (mass.double() <= want).sum(-1).clamp(max=vocab - 1), order[:, 0])
    logprob = z.gather(-1, ids[:, None])[:, 0] - torch.log(whole.double() * 2.0 ** -44)
    return dict(ids=ids.to(torch.int32), logprob=logprob.float())


def run(st):
    path, case = st["case"]["path"], st["case"]
    if own:
        from vllm_omni_b200.ops import kv8, page_plan, sampler
        if path == "plan":
            if "plan" not in st:
                st["pool"] = page_plan.PagePool(st["free"], st["n_free"], case["page"], st["pages"])
                st["plan"] = page_plan.StepPlan.empty(case["seqs"], case["rows"], DEV)
            p = page_plan.plan_step(st["pool"], st["tables"], st["context"], st["new"], case["rows"], out=st["plan"], advance=False)
            return dict(q_start=p.q_start, lens=p.lens, slots=p.slots, positions=p.positions, row_seq=p.row_seq, row_lens=p.row_lens,
                        n_free=p.n_free, tables=st["tables"])
        if path == "sample":
            ids, logprob = sampler.sample_given(st["logits"], st["u"], st["temperature"], st["top_k"], st["top_p"], st["min_p"])
            return dict(ids=ids, logprob=logprob)
        if "cache" not in st:
            st["cache"] = kv8.Kv8Cache(st["k"], st["v"], st["ks"], st["vs"])
        if path == "write":
            kv8.kv8_write(st["new_k"], st["new_v"], st["cache"], st["slots"])
            k, v = kv8.kv8_read(st["cache"], st["back"])
            return dict(k=k, v=v, ks=st["ks"], vs=st["vs"])
        if path == "decode":
            return kv8.kv8_decode(st["q"], st["cache"], st["tables"], st["row_lens"], row_seq=st["row_seq"] if case["per"] > 1 else None)
        return kv8.kv8_prefill(st["q"], st["cache"], [(0, case["rows"], case["context"], st["tables"][0])])
    if path == "plan":
        return _plan(st)
    if path == "write":
        _write(st, st["new_k"], st["new_v"], st["slots"])
        return dict(k=_read(st["k"], st["ks"], st["back"]), v=_read(st["v"], st["vs"], st["back"]), ks=st["ks"], vs=st["vs"])
    return _sample(st) if path == "sample" else _attend(st)


def work(case):
    path = case["path"]
    if path == "plan":
        return dict(bytes=16.0 * case["seqs"] + 24.0 * case["rows"], flops=0.0)           # lengths, the plan's rows and the table entries they read
    if path == "write":
        rows = case["seqs"] * case["new"]
        held = rows + case["seqs"] * case["most_context"] / 2
        return dict(bytes=case["kv"] * case["dim"] * (6.0 * rows + 6.0 * held), flops=0.0)
    if path == "decode":
        keys = case["most_keys"] * (0.8 * case["seqs"] if case["seqs"] > 1 else 1)
        return dict(bytes=keys * case["kv"] * (2.0 * case["dim"] + 8.0 / case["page"]) + 4.0 * case["seqs"] * case["per"] * case["heads"] * case["dim"],
                    flops=4.0 * keys * case["per"] * case["heads"] * case["dim"])
    if path == "prefill":
        r, c = case["rows"], case["context"]
        return dict(bytes=2.0 * (r + c) * case["kv"] * case["dim"] + 4.0 * r * case["heads"] * case["dim"],
                    flops=4.0 * case["heads"] * case["dim"] * (r * c + r * (r + 1) / 2))
    return dict(bytes=float(case["rows"] * case["vocab"] * (2 if case["bf16"] else 4)), flops=8.0 * case["rows"] * case["vocab"])


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_plan(st):
    case = st["case"]
    page, rows = case["page"], case["rows"]
    context, new, tables, free = (st[k].tolist() for k in ("context", "new", "tables", "free"))
    starts, lens, out = [0], [], []
    for s, (c, n) in enumerate(zip(context, new)):
        n = min(n, rows - starts[-1])
        starts.append(starts[-1] + n)
        pages, taken = -(-c // page), 0
        while pages < min(len(tables[s]), -(-(c + n) // page)) and free:
            tables[s][pages] = free.pop()
            pages += 1
        for i in range(n):
            fits = c + i < pages * page
            taken += fits
            out.append((tables[s][(c + i) // page] * page + (c + i) % page if fits else -1, c + i, s, c + i + 1 if fits else 0))
        lens.append(c + taken)
    out += [(-1, 0, -1, 0)] * (rows - len(out))
    cols = [torch.tensor(v) for v in zip(*out)]
    return dict(q_start=torch.tensor(starts), lens=torch.tensor(lens), slots=cols[0], positions=cols[1], row_seq=cols[2], row_lens=cols[3],
                n_free=torch.tensor([len(free)]), tables=torch.tensor(tables))


def _nearest(x):
    """The e4m3 value next to x (in 64 bits, within +-448), ties to the even one."""
    step = torch.exp2((torch.frexp(x).exponent - 1).clamp(min=-6).double() - 3)
    return torch.round(x / step) * step


def _exact_write(st):
    case, page, got = st["case"], st["case"]["page"], {}
    slots, back = st["slots"].long(), st["back"].long()
    for codes, scale, new, name, sname in (("k", "ks", "new_k", "k", "ks"), ("v", "vs", "new_v", "v", "vs")):
        kv, dim = case["kv"], case["dim"]
        value = st[codes].float().double() * st[scale].double()[:, None, :, None]
        held, factor, x = value.view(-1, kv, dim), st[scale].double(), st[new].double()
        hit, turn = torch.unique(slots // page, return_inverse=True)
        for i in range(hit.numel()):
            mine = (turn == i).nonzero()[:, 0]
            p, low = int(hit[i]), int((slots[mine] % page).min())
            m, e = torch.frexp(x[mine].abs().amax((0, 2)) / 448.0)                   # m * 2^e, m in [1/2, 1); 0 has e = 0
            least = torch.ldexp(torch.ones_like(m), torch.where(m == 0, LEAST, torch.where(m > 0.5, e, e - 1)).clamp(min=LEAST))
            f = least if low == 0 else torch.maximum(least, factor[p])
            if low:
                grown = (f > factor[p])[:, None]
                value[p, :low] = torch.where(grown, _nearest(value[p, :low] / f[:, None]) * f[:, None], value[p, :low])
            factor[p] = f
            held[slots[mine]] = _nearest(x[mine] / f[:, None]) * f[:, None]
        got[name], got[sname] = held[back], factor
    return dict(k=got["k"], v=got["v"], ks=got["ks"], vs=got["vs"])


def _exact_attend(st):
    case, per, page = st["case"], st["per"], st["case"]["page"]
    kv, dim = case["kv"], case["dim"]
    q = st["q"].double().view(-1, per, kv, case["heads"] // kv, dim)
    lens, out = st["row_lens"].view(-1, per), []
    for s in range(q.shape[0]):
        pages = st["tables"][s].long()
        ks, vs = (st[c].float()[pages].double() * st[f][pages].double()[:, None, :, None] for c, f in (("k", "ks"), ("v", "vs")))
        ks, vs = ks.reshape(-1, kv, dim), vs.reshape(-1, kv, dim)
        o = []
        for h in range(kv):
            a = torch.matmul(q[s, :, h].reshape(-1, dim), ks[:, h].t()) / math.sqrt(dim)
            seen = torch.arange(ks.shape[0], device=DEV)[None] < lens[s].repeat_interleave(q.shape[3])[:, None]
            o.append(torch.matmul(torch.softmax(torch.where(seen, a, -math.inf), -1), vs[:, h]).view(per, -1, dim))
        out.append(torch.stack(o, 1).reshape(per, -1, dim))
    return torch.cat(out)


def _exact_sample(st):
    ids, logprobs = [], []
    for r in range(st["u"].numel()):
        x = st["logits"][r].double()
        t = float(st["temperature"][r])
        p = torch.softmax(x / (t if t > 0 else 1.0), -1)
        if t <= 0:
            i = int(torch.nonzero(x == x.max())[0])
        else:
            by = torch.argsort(x, descending=True, stable=True)
            if 0 < int(st["top_k"][r]) < by.numel():
                by = by[:int(st["top_k"][r])]
            by = by[p[by] >= p.max() * float(st["min_p"][r])]
            if float(st["top_p"][r]) < 1:
                run_mass = torch.cumsum(p[by], 0)
                by = by[(run_mass - p[by]) < float(st["top_p"][r]) * run_mass[-1]]
            by = torch.sort(by).values
            mass = torch.cumsum(p[by], 0)
            i = int(by[min(by.numel() - 1, int((mass <= float(st["u"][r]) * mass[-1]).sum()))])
        ids.append(i)
        logprobs.append(float(torch.log(p[i])))
    return dict(ids=torch.tensor(ids), logprob=torch.tensor(logprobs, dtype=torch.float64))


def exact(case, seed):
    st = prepare(case, seed)
    path = case["path"]
    if path == "plan":
        return _exact_plan(st)
    if path == "write":
        return _exact_write(st) if case["seqs"] * case["new"] < 20000 else None
    return _exact_sample(st) if path == "sample" else _exact_attend(st)
