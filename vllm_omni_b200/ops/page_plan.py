"""Pages and slots of a step planned on the device (csrc/page_plan.cu): what ``engine/kv_cache_manager.py`` decides on the host, from request lengths that
are on the GPU, so that a captured decode loop takes and returns pages without the host.

A ``PagePool`` is a stack of free pages.  ``plan_step`` hands them out in the order of the sequences and lists, for every row of the step's batch, the slot that
its keys and values go to, its position, its sequence and the keys it sees: the operands of ``kv8.kv8_write`` and ``kv8.kv8_decode`` (and of ``kv_cache.kv_write``
and ``paged_decode``).  ``release_pages`` puts the pages of finished sequences back.  The CPU paths restate the same semantics in PyTorch.

A page belongs to one sequence.  A page id outside the pool is reported, its rows get no slot, and it does not come back to the pool.
The GPU reports through the status word (``_native.check_status``); on the CPU ``release_pages`` raises when it is done."""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _native as nv

MAX_SEQS = 4096                       # csrc/page_plan.cu: a block scans them in its shared memory
_P, _I, _L = ctypes.c_void_p, ctypes.c_int, ctypes.c_long


@functools.lru_cache(maxsize=None)
def _lib():
    lib = nv.lib("page_plan")
    lib._cdll.omni_plan_step.argtypes = [_P] * 3 + [_L, _P, _P] + [_I] * 6 + [_P] * 11
    lib._cdll.omni_release_pages.argtypes = [_P] * 3 + [_L, _P, _P] + [_I] * 5 + [_P] * 2
    return lib


def _check_ints(name, t, shape, device):
    if t.dtype is not torch.int32 or t.shape != shape or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{name}: contiguous int32 {tuple(shape)} on {device} expected, got {t.dtype} {tuple(t.shape)} on {t.device}")


class PagePool:
    """Free pages: ``free`` int32 [N], of which the first ``n_free`` (int32 [1]) are a stack, its top last.  Page ids lie in [0, ``num_blocks``)."""

    def __init__(self, free: torch.Tensor, n_free: torch.Tensor, block_size: int, num_blocks: int | None = None):
        num_blocks = free.numel() if num_blocks is None else num_blocks
        _check_ints("free", free, (free.numel(),), free.device)
        _check_ints("n_free", n_free, (1,), free.device)
        if block_size < 1 or num_blocks < 1 or num_blocks * block_size > 0x7fffffff:
            raise ValueError(f"{num_blocks} pages of {block_size} tokens: at least one each, and fewer than 2^31 slots")
        self.free, self.n_free, self.block_size, self.num_blocks, self.device = free, n_free, int(block_size), int(num_blocks), free.device

    @classmethod
    def full(cls, num_blocks: int, block_size: int, device) -> "PagePool":
        """Every page free; page 0 is handed out first."""
        free = torch.arange(num_blocks - 1, -1, -1, dtype=torch.int32, device=device)
        return cls(free, torch.full((1,), num_blocks, dtype=torch.int32, device=device), block_size)


class StepPlan:
    """What ``plan_step`` writes: ``q_start`` int32 [S + 1] (rows of sequence s), ``lens`` int32 [S] (cached tokens after the step), per row ``slots`` int32
    (-1: none), ``positions`` int64, ``row_seq`` int32 (-1: no sequence), ``row_lens`` int32 (keys the row sees, 0: none), and ``n_free`` int32 [1]."""
    __slots__ = ("q_start", "lens", "slots", "positions", "row_seq", "row_lens", "n_free", "seqs", "rows", "device")

    def __init__(self, q_start, lens, slots, positions, row_seq, row_lens, n_free):
        self.seqs, self.rows, self.device = lens.numel(), slots.numel(), slots.device
        _check_ints("q_start", q_start, (self.seqs + 1,), self.device)
        for name, t, n in (("lens", lens, self.seqs), ("slots", slots, self.rows), ("row_seq", row_seq, self.rows), ("row_lens", row_lens, self.rows), ("n_free", n_free, 1)):
            _check_ints(name, t, (n,), self.device)
        if positions.dtype is not torch.int64 or positions.shape != (self.rows,) or not positions.is_contiguous() or positions.device != self.device:
            raise ValueError(f"positions: contiguous int64 [{self.rows}] on {self.device} expected")
        self.q_start, self.lens, self.slots, self.positions, self.row_seq, self.row_lens, self.n_free = q_start, lens, slots, positions, row_seq, row_lens, n_free

    @classmethod
    def empty(cls, seqs: int, rows: int, device) -> "StepPlan":
        up = lambda n: -(-n // 4) * 4                     # every part starts on 16 bytes
        sizes = (seqs + 1, seqs, rows, rows, rows, 1)
        buf, parts, at = torch.empty(sum(up(n) for n in sizes), dtype=torch.int32, device=device), [], 0
        for n in sizes:
            parts.append(buf[at:at + n])
            at += up(n)
        q_start, lens, slots, row_seq, row_lens, n_free = parts
        return cls(q_start, lens, slots, torch.empty(rows, dtype=torch.int64, device=device), row_seq, row_lens, n_free)


def _check_tables(tables, seqs, pool):
    if tables.dim() != 2 or tables.dtype is not torch.int32 or tables.shape[0] != seqs or tables.shape[1] < 1 or tables.stride(1) != 1 \
            or (seqs > 1 and tables.stride(0) < tables.shape[1]) or tables.device != pool.device:
        raise ValueError(f"tables: int32 [{seqs}, columns] with rows side by side on {pool.device} expected, got {tables.dtype} {tuple(tables.shape)}")
    if tables.shape[1] * pool.block_size > 0x7fffffff:
        raise ValueError("tables: fewer than 2^31 tokens a sequence")
    if seqs > MAX_SEQS:
        raise ValueError(f"{seqs} sequences: at most {MAX_SEQS}")


def plan_step(pool: PagePool, tables: torch.Tensor, context: torch.Tensor, new: torch.Tensor, rows: int, out: StepPlan | None = None,
              advance: bool = True) -> StepPlan:
    """Sequence s has ``context[s]`` cached tokens in the pages of ``tables[s]`` and gets ``new[s]`` more (both int32 [S]), which are the next rows of a batch of
    ``rows`` rows.  New entries of ``tables`` are written.  Tokens that find no page, no column or no row are not taken: their rows have slot -1.  Rows behind the
    last sequence have slot -1, position 0, sequence -1 and no keys.

    ``advance``: the pool's height and ``context`` become those after the step, in place.  Without it both stay, and the same call gives the same plan again."""
    S = context.numel()
    _check_ints("context", context, (S,), pool.device)
    _check_ints("new", new, (S,), pool.device)
    _check_tables(tables, S, pool)
    if rows < 0 or rows > 0x7fffffff:
        raise ValueError(f"rows {rows}: 0 to 2^31 - 1")
    if out is None:
        out = StepPlan.empty(S, rows, pool.device)
    elif out.seqs != S or out.rows != rows or out.device != pool.device:
        raise ValueError(f"out: a plan of {S} sequences and {rows} rows on {pool.device} expected, got {out.seqs} and {out.rows} on {out.device}")
    if pool.device.type != "cuda":
        return _plan_torch(pool, tables, context, new, rows, out, advance)
    if torch._C._cuda_getDevice() != pool.device.index:
        with torch.cuda.device(pool.device):
            return plan_step(pool, tables, context, new, rows, out, advance)
    c = context.data_ptr()
    n = pool.n_free.data_ptr()
    nv.check_rc(_lib().omni_plan_step(
        c, new.data_ptr(), tables.data_ptr(), tables.stride(0), pool.free.data_ptr(), n, S, tables.shape[1], pool.block_size, rows, pool.num_blocks,
        pool.free.numel(), out.q_start.data_ptr(), out.lens.data_ptr(), out.slots.data_ptr(), out.positions.data_ptr(), out.row_seq.data_ptr(),
        out.row_lens.data_ptr(), out.n_free.data_ptr(), c if advance else None, n if advance else None, nv.status_word(pool.device).data_ptr(), nv.stream_ptr()),
        "omni_plan_step")
    return out


def release_pages(pool: PagePool, tables: torch.Tensor, lens: torch.Tensor, done: torch.Tensor) -> None:
    """The pages that hold the ``lens[s]`` tokens (int32 [S]) of every sequence with ``done[s]`` (bool [S]) go back to the pool, and its length becomes 0.
    Where the pool has no room for all of a sequence's pages, that is reported; the sequence and those behind it keep their pages and their lengths."""
    S = lens.numel()
    _check_ints("lens", lens, (S,), pool.device)
    _check_tables(tables, S, pool)
    if done.dtype is not torch.bool or done.shape != (S,) or not done.is_contiguous() or done.device != pool.device:
        raise ValueError(f"done: contiguous bool [{S}] on {pool.device} expected, got {done.dtype} {tuple(done.shape)}")
    if pool.device.type != "cuda":
        height, cap = min(max(int(pool.n_free), 0), pool.free.numel()), pool.free.numel()
        back, bad, full = [], 0, False
        for s in (s for s in range(S) if done[s]):
            pages = tables[s, :min(tables.shape[1], -(-max(int(lens[s]), 0) // pool.block_size))].tolist()
            full |= len(back) + bad + len(pages) > cap - height
            if not full or not pages:
                lens[s] = 0
                good = [p for p in pages if 0 <= p < pool.num_blocks]
                back, bad = back + good, bad + len(pages) - len(good)
        pool.free[height:height + len(back)] = torch.tensor(back, dtype=torch.int32)
        pool.n_free.fill_(height + len(back))
        if full or bad:
            raise ValueError(f"pages of finished sequences: {bad} ids outside the pool's {pool.num_blocks}"
                             + (f", and more than there is room for ({cap - height})" if full else ""))
        return
    if torch._C._cuda_getDevice() != pool.device.index:
        with torch.cuda.device(pool.device):
            return release_pages(pool, tables, lens, done)
    nv.check_rc(_lib().omni_release_pages(lens.data_ptr(), done.data_ptr(), tables.data_ptr(), tables.stride(0), pool.free.data_ptr(), pool.n_free.data_ptr(), S,
                                          tables.shape[1], pool.block_size, pool.num_blocks, pool.free.numel(), nv.status_word(pool.device).data_ptr(), nv.stream_ptr()),
                "omni_release_pages")


def _plan_torch(pool, tables, context, new, rows, out, advance):
    page, W, height = pool.block_size, tables.shape[1], min(max(int(pool.n_free), 0), pool.free.numel())
    stack, left = pool.free.tolist(), height
    start, line = 0, []
    for s, (c, n) in enumerate(zip(context.tolist(), new.tolist())):
        c, n = min(max(c, 0), W * page), min(max(n, 0), rows - start)
        out.q_start[s] = start
        have = -(-c // page)
        while have < min(W, -(-(c + n) // page)) and left:
            left -= 1
            tables[s, have] = stack[left]
            have += 1
        took = max(0, min(n, have * page - c))
        for i in range(n):
            p = int(tables[s, (c + i) // page]) if i < took else -1
            ok = 0 <= p < pool.num_blocks
            line.append((p * page + (c + i) % page if ok else -1, c + i, s, c + i + 1 if ok else 0))
        out.lens[s] = c + took
        start += n
    out.q_start[len(out.lens)] = start
    line += [(-1, 0, -1, 0)] * (rows - start)
    for t, col in zip((out.slots, out.positions, out.row_seq, out.row_lens), zip(*line)):
        t.copy_(torch.tensor(col))
    out.n_free.fill_(left)
    if advance:
        context.copy_(out.lens)
        pool.n_free.fill_(left)
    return out
