"""A paged key/value cache of 8 bits (csrc/kv8.cu): the pages of ``kv_cache`` at half the bytes, with a scale for each page and KV head.

A value is an e4m3 code times a power of two.  ``kv8_write`` puts rows into their slots; a page whose first row is among those written starts over, with the least
exponent by which the largest finite magnitude fits 448 (at least -120); otherwise its exponent only grows, and the rows before the first written one are
rounded again.  Infinities saturate, NaN stays.  ``kv8_read`` gives rows back in bf16 (every value is exact in it), ``kv8_decode`` attends single rows to the
cache, ``kv8_prefill`` the portions of prompts.  The CPU paths restate the same semantics in PyTorch.

A page belongs to one sequence, is filled from its first row on, and its rows follow one another in a call (fewer than 128 rows that are not written may lie between
two of them).  Page ids and slots outside the cache are reported
through the status word (``_native.check_status``) and not followed."""
from __future__ import annotations

import ctypes
import functools
import math

import torch

from . import _native as nv

LEAST, MOST = -120, 120               # exponents of scales
HEAD_SIZES = (64, 128)
MAX_GROUP = 128                       # heads on one KV head
CODES = torch.float8_e4m3fn
_P, _I, _L, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_long, ctypes.c_float


@functools.lru_cache(maxsize=None)
def _lib():
    lib = nv.lib("kv8")
    c = lib._cdll
    c.omni_kv8_write.argtypes = [_P, _P, _P, _L, _L, _L, _L, _P, _I, _P]
    c.omni_kv8_read.argtypes = [_P, _I, _P, _P, _P, _I, _P, _P, _P]
    c.omni_kv8_attn_shares.argtypes = [_I] * 8
    c.omni_kv8_attn.argtypes = [_P, _P, _L, _L, _P, _L, _P, _P, _I, _I, _I, _I, _F, _I, _P, _P, _L, _L, _P]
    return lib


@functools.lru_cache(maxsize=None)
def _prefill_lib():
    lib = nv.lib("attention_sm100")
    lib._cdll.omni_attn_prefill_keys.argtypes = [_P, _L, _L, _P, _L, _L, _P, _L, _L, _P, _L, _L, _I, _I, _I, _I, _I, _P, _P, _P, _P, _F, _P, _P]
    return lib


@functools.lru_cache(maxsize=4096)
def _shares(R, S, H, Hkv, D, mapped, page, max_keys, device):
    return _lib().omni_kv8_attn_shares(R, S, H, Hkv, D, mapped, page, max_keys)


class _Fields(ctypes.Structure):      # Kv8Cache of csrc/kv8.cu
    _fields_ = [(n, _P) for n in ("k", "v", "k_scale", "v_scale", "status")] + [(n, _I) for n in ("pages", "page", "heads", "channels")]


class Kv8Cache:
    """``k``, ``v``: float8_e4m3fn [pages, page size, Hkv, D]; ``k_scale``, ``v_scale``: fp32 powers of two [pages, Hkv]."""
    __slots__ = ("k", "v", "k_scale", "v_scale", "pages", "block_size", "heads", "head_size", "device", "_fields", "_address")

    def __init__(self, k, v, k_scale, v_scale):
        if k.dim() != 4 or any(t.dtype is not CODES or t.shape != k.shape or not t.is_contiguous() or t.device != k.device for t in (k, v)):
            raise ValueError("k, v: contiguous float8_e4m3fn [pages, page size, KV heads, channels] on one device expected, got "
                             f"{k.dtype} {tuple(k.shape)} and {v.dtype} {tuple(v.shape)}")
        self.pages, self.block_size, self.heads, self.head_size = k.shape
        if self.head_size not in HEAD_SIZES:
            raise ValueError(f"head size {self.head_size}: one of {HEAD_SIZES}")
        if self.block_size < 8 or self.block_size % 8 or self.pages < 1 or self.heads < 1 or self.pages * self.block_size > 0x7fffffff:
            raise ValueError(f"{self.pages} pages of {self.block_size} tokens and {self.heads} heads: at least one each, pages of a multiple of 8 tokens, "
                             "fewer than 2^31 slots")
        if any(t.dtype is not torch.float32 or t.shape != (self.pages, self.heads) or not t.is_contiguous() or t.device != k.device for t in (k_scale, v_scale)):
            raise ValueError(f"scales: contiguous fp32 [{self.pages}, {self.heads}] on {k.device} expected")
        if k.is_cuda and (k.data_ptr() | v.data_ptr()) & 15:
            raise ValueError("k and v must begin on 16 bytes")
        self.k, self.v, self.k_scale, self.v_scale, self.device = k, v, k_scale, v_scale, k.device
        self._fields = _Fields(0, 0, 0, 0, nv.status_word(k.device).data_ptr() if k.is_cuda else 0, *k.shape)
        self._address = ctypes.addressof(self._fields)       # the last: nothing can be set from here on

    def __setattr__(self, name, value):
        if hasattr(self, "_address"):
            raise AttributeError(f"{name}: a cache keeps its tensors")
        object.__setattr__(self, name, value)

    def __reduce__(self):                                    # copies and pickles
        return Kv8Cache, (self.k, self.v, self.k_scale, self.v_scale)

    def _at(self) -> int:
        """Address of what the kernels take of it; the tensors' own addresses as they are now."""
        f = self._fields
        f.k, f.v, f.k_scale, f.v_scale = self.k.data_ptr(), self.v.data_ptr(), self.k_scale.data_ptr(), self.v_scale.data_ptr()
        return self._address

    @classmethod
    def empty(cls, pages: int, block_size: int, heads: int, head_size: int, device) -> "Kv8Cache":
        codes = torch.zeros(2, pages, block_size, heads, head_size, dtype=torch.uint8, device=device).view(CODES)
        scales = torch.full((2, pages, heads), 2.0 ** LEAST, device=device)
        return cls(codes[0], codes[1], scales[0], scales[1])


def _check_index(name, t, n, device):
    if t.dtype is not torch.int32 or t.shape != (n,) or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{name}: contiguous int32 [{n}] on {device} expected, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _check_rows(name, t, shape, device):
    if t.dtype is not torch.bfloat16 or t.shape != shape or t.device != device:
        raise ValueError(f"{name}: bf16 {tuple(shape)} on {device} expected, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _pitches(t):
    """(of rows, of heads, whether the kernels take the tensor where it is: channels side by side, everything on 16 bytes).  A single row or head has no pitch of its own."""
    (R, H, D), (a, b, c) = t.shape, t.stride()
    if H == 1:
        b = D
    if R <= 1:
        a = H * b
    return a, b, c == 1 and not (a | b) & 7 and not t.data_ptr() & 15


def _readable(t, H, D):
    """[rows, H, D] as the kernels take it, pitches of its rows and heads."""
    if not t.is_contiguous():
        a, b, fits = _pitches(t)
        if fits:
            return t, a, b
    elif not t.data_ptr() & 15:
        return t, H * D, D
    return torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t), H * D, D


def _elsewhere(device) -> bool:
    return torch._C._cuda_getDevice() != device.index


def _stream(device):
    return torch._C._cuda_getCurrentRawStream(device.index)


def kv8_write(k, v, cache: Kv8Cache, slots) -> None:
    """k, v: bf16 [T, Hkv, D]; slots int32 [T] (page * page size + row, below zero: not written).  A page's rows follow one another: a page that comes up again behind another one's
    rows, or behind 128 rows that are not written, would be scaled by two blocks at once, and is not looked for."""
    T = slots.numel()
    shape = (T, cache.heads, cache.head_size)
    _check_rows("k", k, shape, cache.device)
    _check_rows("v", v, shape, cache.device)
    _check_index("slots", slots, T, cache.device)
    if not k.is_cuda:
        _write_torch(cache.k, cache.k_scale, k, slots)
        _write_torch(cache.v, cache.v_scale, v, slots)
        return
    if _elsewhere(cache.device):
        with torch.cuda.device(cache.device):
            return kv8_write(k, v, cache, slots)
    k, kr, kh = _readable(k, cache.heads, cache.head_size)
    v, vr, vh = _readable(v, cache.heads, cache.head_size)
    nv.check_rc(_lib().omni_kv8_write(cache._at(), k.data_ptr(), v.data_ptr(), kr, kh, vr, vh, slots.data_ptr(), T, _stream(cache.device)), "omni_kv8_write")


def _out_pair(cache, rows, out_k, out_v):
    shape = (rows, cache.heads, cache.head_size)
    if (out_k is None) != (out_v is None):
        raise ValueError("out_k and out_v: both or neither")
    if out_k is None:
        return cache.k_scale.new_empty(shape, dtype=torch.bfloat16), cache.k_scale.new_empty(shape, dtype=torch.bfloat16)
    for name, t in (("out_k", out_k), ("out_v", out_v)):
        _check_rows(name, t, shape, cache.device)
        if not t.is_contiguous() or (t.is_cuda and t.data_ptr() & 15):
            raise ValueError(f"{name}: contiguous, from 16 bytes on")
    return out_k, out_v


def _read(cache, n, index, row0, rows, tables, k, v):
    nv.check_rc(_lib().omni_kv8_read(cache._at(), n, (_P * n)(*index), (_L * n)(*row0), (_L * n)(*rows), tables, k.data_ptr(), v.data_ptr(), _stream(cache.device)),
                "omni_kv8_read")


def kv8_read(cache: Kv8Cache, slots, out_k=None, out_v=None):
    """Rows of the cache in bf16: (k, v), each [T, Hkv, D], for ``slots`` int32 [T].  Slots below zero give zeros."""
    T = slots.numel()
    _check_index("slots", slots, T, cache.device)
    out_k, out_v = _out_pair(cache, T, out_k, out_v)
    if not slots.is_cuda:
        for out, codes, scale in ((out_k, cache.k, cache.k_scale), (out_v, cache.v, cache.v_scale)):
            out.copy_(_rows_torch(codes, scale, slots))
        return out_k, out_v
    if _elsewhere(cache.device):
        with torch.cuda.device(cache.device):
            return kv8_read(cache, slots, out_k, out_v)
    if T:
        _read(cache, 1, (slots.data_ptr(),), (0,), (T,), 0, out_k, out_v)
    return out_k, out_v


def _check_tables(tables, S, cache):
    if tables.dim() != 2 or tables.dtype is not torch.int32 or tables.shape[0] < 1 or tables.shape[1] < 1 or tables.stride(1) != 1 or tables.device != cache.device:
        raise ValueError(f"block_tables: int32 [sequences, columns] with rows side by side on {cache.device} expected, got {tables.dtype} {tuple(tables.shape)}")
    if tables.shape[1] * cache.block_size > 0x7fffffff:
        raise ValueError("block_tables: fewer than 2^31 tokens a sequence")
    if S is not None and tables.shape[0] != S:
        raise ValueError(f"block_tables of {tables.shape[0]} sequences for {S} rows: row_seq says which row is of which sequence")


def _check_apart(out):
    """Of the dimensions with more than one entry each step reaches over all that lies within it."""
    reach = 1
    for step, size in sorted((step, size) for step, size in zip(out.stride(), out.shape) if size > 1):
        if step < reach:
            raise ValueError(f"out: rows or heads overlap (strides {out.stride()} of {tuple(out.shape)})")
        reach += step * (size - 1)


def _check_queries(q, cache, out):
    if q.dim() != 3 or q.shape[1] < 1 or q.shape[1] % cache.heads:
        raise ValueError(f"q: [rows, heads, {cache.head_size}] with heads a multiple of {cache.heads} expected, got {tuple(q.shape)}")
    if q.shape[1] > MAX_GROUP * cache.heads:
        raise ValueError(f"{q.shape[1]} heads on {cache.heads} KV heads: at most {MAX_GROUP} to one")
    _check_rows("q", q, (q.shape[0], q.shape[1], cache.head_size), cache.device)
    if out is not None:
        _check_rows("out", out, q.shape, cache.device)
        if not out.is_contiguous():
            _check_apart(out)
        if out.is_cuda and not _pitches(out)[2]:
            raise ValueError("out: channels side by side, rows and heads on 16 bytes")


def kv8_decode(q, cache: Kv8Cache, block_tables, lens, row_seq=None, scale=None, out=None):
    """Attention of single rows: q bf16 [R, H, D]; row r sees the first ``lens[r]`` (int32 [R]) keys of sequence ``row_seq[r]`` (int32 [R]; without it sequence
    r), whose pages are ``block_tables[row_seq[r]]`` (int32 [S, columns]).  A row without keys gives zeros, whatever its sequence.  Several rows of a sequence (tokens
    that are proposed together) are best neighbours: they share what is read."""
    _check_queries(q, cache, out)
    R, H, D = q.shape
    _check_tables(block_tables, R if row_seq is None else None, cache)
    _check_index("lens", lens, R, cache.device)
    if row_seq is not None:
        _check_index("row_seq", row_seq, R, cache.device)
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if out is None:
        out = q.new_empty((R, H, D))
    if not q.is_cuda:
        for r in range(R):
            s = r if row_seq is None else int(row_seq[r])
            n = min(int(lens[r]), block_tables.shape[1] * cache.block_size) if 0 <= s < block_tables.shape[0] else 0
            out[r] = _attend_torch(q[r:r + 1], cache, block_tables[s] if n > 0 else None, max(n, 0), scale, 0)[0]
        return out
    if _elsewhere(cache.device):
        with torch.cuda.device(cache.device):
            return kv8_decode(q, cache, block_tables, lens, row_seq, scale, out)
    if R == 0:
        return out
    q, qr, qh = _readable(q, H, D)
    S, mapped, max_keys = block_tables.shape[0], row_seq is not None, block_tables.shape[1] * cache.block_size
    shares = _shares(R, S, H, cache.heads, D, mapped, cache.block_size, max_keys, cache.device.index)
    part = cache.k_scale.new_empty(R * H * shares * (D + 1)) if shares > 1 else None
    _, outr, outh = _readable(out, H, D)
    nv.check_rc(_lib().omni_kv8_attn(
        cache._at(), q.data_ptr(), qr, qh, block_tables.data_ptr(), block_tables.stride(0), lens.data_ptr(), row_seq.data_ptr() if mapped else None, R, S, H,
        max_keys, scale, shares, None if part is None else part.data_ptr(), out.data_ptr(), outr, outh, _stream(cache.device)), "omni_kv8_attn")
    if part is not None:
        nv.count_launches(1)
    return out


def kv8_prefill(q, cache: Kv8Cache, segs, scale=None, out=None):
    """Causal attention of the prompt portions of a step to the cache, into which their keys and values are written already.

    q bf16 [T, H, D]; ``segs``: (first row, rows, context, block table int32 [columns]) each, as in ``kv_cache.prefill_segments``: row i of a portion sees
    context + i + 1 keys.  Rows of no portion stay as they are in ``out``.  A value that is not a number may reach rows of its portion that do not see it, as in the
    attention to bf16 pages (not those of ``kv8_decode``)."""
    _check_queries(q, cache, out)
    T, H, D = q.shape
    segs = [s for s in segs if s[1] > 0]
    for first, rows, context, table in segs:
        if first < 0 or context < 0 or first + rows > T:
            raise ValueError(f"portion of rows {first} to {first + rows} with context {context}: {T} rows")
        if table.dim() != 1 or table.dtype is not torch.int32 or not table.is_contiguous() or table.device != cache.device:
            raise ValueError(f"block table: contiguous int32 [columns] on {cache.device} expected, got {table.dtype} {tuple(table.shape)}")
        if table.numel() * cache.block_size < context + rows:
            raise ValueError(f"block table of {table.numel()} pages of {cache.block_size}: {context + rows} tokens")
    if len(segs) > 1:
        order = sorted((s[0], s[1]) for s in segs)
        if any(a + n > b for (a, n), (b, _) in zip(order, order[1:])):
            raise ValueError("portions that share rows")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if out is None:
        out = q.new_empty((T, H, D))
    if not q.is_cuda:
        for first, rows, context, table in segs:
            out[first:first + rows] = _attend_torch(q[first:first + rows], cache, table, context + rows, scale, context)
        return out
    if _elsewhere(cache.device):
        with torch.cuda.device(cache.device):
            return kv8_prefill(q, cache, segs, scale, out)
    if not segs:
        return out
    if 0 in q.stride():                                      # one row or head for all: tensor maps want pitches
        q = q.contiguous()
    (q, qr, qh), (_, outr, outh), n = _readable(q, H, D), _readable(out, H, D), len(segs)
    total, row0 = 0, []
    for _, rows, context, _ in segs:
        row0.append(total)
        total += context + rows
    k, v = q.new_empty((2, total, cache.heads, D))
    _read(cache, n, [s[3].data_ptr() for s in segs], row0, [s[2] + s[1] for s in segs], 1, k, v)
    first, rows, context = ((_I * n)(*(s[i] for s in segs)) for i in range(3))
    rs = cache.heads * D
    nv.check_rc(_prefill_lib().omni_attn_prefill_keys(
        q.data_ptr(), qr, qh, k.data_ptr(), rs, D, v.data_ptr(), rs, D, out.data_ptr(), outr, outh, T, H, cache.heads, D, n,
        first, rows, context, (_L * n)(*row0), scale, cache._fields.status, _stream(cache.device)), "omni_attn_prefill_keys")
    nv.count_launches((n - 1) // 16)                         # of the pages, sixteen segments at a time
    if n > 8 or T > 248 * 256:                               # of the attention, eight segments and 256 blocks of 256 rows at a time
        nv.count_launches(sum(-(-sum(-(-s[1] // 256) for s in segs[i:i + 8]) // 256) for i in range(0, n, 8)) - 1)
    return out


# --------------------------------------------------------------------------- PyTorch restatements
def _exponent(size):
    f, e = torch.frexp(size)                              # size = f * 2^e, f in [1/2, 1): fits 448 = 7/8 * 2^9 times 2^(e - 9) or the next power
    return torch.where(size > 0, e - 9 + (f > 0.875), LEAST).clamp(min=LEAST)


def _write_torch(codes, scale, x, slots):
    page, T, n = codes.shape[1], x.shape[0], codes.shape[0] * codes.shape[1]
    rows, x, at = codes.view(-1, *codes.shape[2:]), x.float(), slots.tolist()
    t = 0
    while t < T:
        if not 0 <= at[t] < n:
            t += 1
            continue
        pg, mine, i = at[t] // page, [t], t + 1
        while i < T and i - mine[-1] <= 128:
            if 0 <= at[i] < n:
                if at[i] // page != pg:
                    break
                mine.append(i)
            i += 1
        low, run = min(at[i] for i in mine) - pg * page, x[mine]
        e = _exponent(torch.where(run.isfinite(), run.abs(), 0.0).amax((0, 2)))
        if low:
            old = (torch.frexp(scale[pg]).exponent - 1).clamp(LEAST, MOST)
            e = torch.maximum(e, old)
            before = torch.ldexp(codes[pg, :low].float(), (old - e)[None, :, None])
            codes[pg, :low] = torch.where((e > old)[None, :, None], before, codes[pg, :low].float()).to(CODES)
        scale[pg] = torch.ldexp(torch.ones_like(scale[pg]), e)
        for i in mine:
            rows[at[i]] = torch.ldexp(x[i], -e[:, None]).clamp(-448.0, 448.0).to(CODES)
        t = mine[-1] + 1


def _rows_torch(codes, scale, slots):
    ok = (slots >= 0) & (slots < codes.shape[0] * codes.shape[1])
    at = torch.where(ok, slots, 0).long()
    x = codes.view(-1, *codes.shape[2:]).view(torch.uint8)[at].view(CODES).float() * scale[at // codes.shape[1]].unsqueeze(-1)
    return torch.where(ok[:, None, None], x, 0.0)


def _attend_torch(q, cache, table, keys, scale, q_offset):
    """Rows of queries of one sequence; row i sees q_offset + i + 1 keys, a single row (q_offset 0) all of them."""
    if keys == 0:
        return torch.zeros_like(q)
    j = torch.arange(keys, device=q.device)
    slots = (table.long()[j // cache.block_size] * cache.block_size + j % cache.block_size).to(torch.int32)
    G = q.shape[1] // cache.heads
    k, v = (_rows_torch(c, s, slots).repeat_interleave(G, 1) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    s = torch.einsum("rhd,khd->hrk", q.float(), k) * scale
    if q.shape[0] > 1 or q_offset:
        s = s.masked_fill(j[None, None] > q_offset + torch.arange(q.shape[0], device=q.device)[None, :, None], -math.inf)
    return torch.einsum("hrk,khd->rhd", torch.softmax(s, -1), v).to(q.dtype)
