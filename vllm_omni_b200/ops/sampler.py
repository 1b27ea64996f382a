"""K16 — batched token sampling on the device (csrc/sampler.cu) with a PyTorch restatement
for CPU runs.  ``sample`` takes one ``RowParams`` per sequence.  ``sample_given`` (csrc/sample_given.cu) takes parameters and random numbers that are on the
device, and gives the token of its definition: ties go to the lowest id, and masses are sums of whole numbers, which have no order."""
from __future__ import annotations

import ctypes
import functools
import operator
from dataclasses import dataclass, field

import torch

from . import _native as nv


class _Row(ctypes.Structure):
    _fields_ = [("temperature", ctypes.c_float), ("top_p", ctypes.c_float), ("min_p", ctypes.c_float),
                ("top_k", ctypes.c_int), ("rep_penalty", ctypes.c_float), ("presence_penalty", ctypes.c_float),
                ("frequency_penalty", ctypes.c_float), ("seed", ctypes.c_ulonglong), ("step", ctypes.c_int),
                ("hist_off", ctypes.c_int), ("hist_len", ctypes.c_int), ("gen_off", ctypes.c_int),
                ("sup_off", ctypes.c_int), ("sup_len", ctypes.c_int), ("range_lo", ctypes.c_int),
                ("range_hi", ctypes.c_int)]


@dataclass
class RowParams:
    temperature: float = 1.0
    top_p: float = 1.0
    min_p: float = 0.0
    top_k: int = 0
    repetition_penalty: float = 1.0
    presence_penalty: float = 0.0
    frequency_penalty: float = 0.0
    seed: int = 0
    step: int = 0
    history: list = field(default_factory=list)      # prompt + generated token ids
    num_prompt_tokens: int = 0
    suppressed: list = field(default_factory=list)
    allowed_range: tuple | None = None                # (lo, hi) of admissible token ids


def _uniform(seed: int, step: int) -> float:
    def sm(x):
        x = (x + 0x9E3779B97F4A7C15) & 0xFFFFFFFFFFFFFFFF
        x = ((x ^ (x >> 30)) * 0xBF58476D1CE4E5B9) & 0xFFFFFFFFFFFFFFFF
        x = ((x ^ (x >> 27)) * 0x94D049BB133111EB) & 0xFFFFFFFFFFFFFFFF
        return x ^ (x >> 31)
    h = sm((seed & 0xFFFFFFFFFFFFFFFF) ^ sm(step))
    return ((h >> 40) + 0.5) / 16777216.0


def sample_reference(logits: torch.Tensor, rows: list[RowParams]):
    """Same pipeline in PyTorch: returns (ids int64 [B], logprobs [B])."""
    ids, lps = [], []
    for r, p in enumerate(rows):
        w = logits[r].float().clone()
        V = w.numel()
        if p.allowed_range is not None:
            lo, hi = p.allowed_range
            m = torch.ones(V, dtype=torch.bool)
            m[lo:hi] = False
            w[m] = float("-inf")
        for t in p.suppressed:
            if 0 <= t < V:
                w[t] = float("-inf")
        if p.repetition_penalty != 1.0 or p.presence_penalty or p.frequency_penalty:
            hist = torch.tensor(p.history, dtype=torch.long)
            if hist.numel():
                uniq = torch.unique(hist[(hist >= 0) & (hist < V)])
                x = w[uniq]
                if p.repetition_penalty != 1.0:
                    x = torch.where(x > 0, x / p.repetition_penalty, x * p.repetition_penalty)
                gen = hist[p.num_prompt_tokens:]
                cnt = torch.bincount(gen[(gen >= 0) & (gen < V)], minlength=V)[uniq].float()
                x = x - (cnt > 0).float() * p.presence_penalty - cnt * p.frequency_penalty
                w[uniq] = x
        if p.temperature <= 0:
            i = int(torch.argmax(w))
            ids.append(i)
            lps.append(float(torch.log_softmax(w, 0)[i]))
            continue
        w = w / p.temperature
        lp = torch.log_softmax(w, 0)
        mx = w.max()
        cut = torch.tensor(float("-inf"))
        if p.min_p > 0:
            cut = torch.maximum(cut, mx + torch.log(torch.tensor(p.min_p)))
        if 0 < p.top_k < V:
            cut = torch.maximum(cut, torch.topk(w, p.top_k).values[-1])
        keep = w >= cut
        if p.top_p < 1.0:
            pr = torch.where(keep, torch.exp(w - mx), torch.zeros(()))
            srt, order = torch.sort(pr, descending=True)
            cum = torch.cumsum(srt, 0)
            n = int((cum < p.top_p * pr.sum()).sum()) + 1       # mass of what survived min-p / top-k
            k2 = torch.zeros(V, dtype=torch.bool)
            k2[order[:n]] = True
            keep &= k2
        pr = torch.where(keep, torch.exp(w - mx), torch.zeros(()))
        u = _uniform(p.seed, p.step) * float(pr.sum())
        cum = torch.cumsum(pr, 0)
        i = int(torch.searchsorted(cum, torch.tensor(u), right=True).clamp(max=V - 1))
        while pr[i] == 0 and i > 0:
            i -= 1
        ids.append(i)
        lps.append(float(lp[i]))
    return torch.tensor(ids, dtype=torch.long), torch.tensor(lps)


_work: dict = {}


def pack_rows(rows: list[RowParams]) -> torch.Tensor:
    """Row parameters as the byte tensor the kernel reads (host memory).  Rows that use penalties or
    suppression lists are not supported here (their side tables vary in size): plain temperature /
    top-k / top-p / min-p / seed / step rows only, which is what a captured sampling step needs."""
    arr = (_Row * len(rows))()
    for r, p in enumerate(rows):
        a = arr[r]
        if p.repetition_penalty != 1.0 or p.presence_penalty or p.frequency_penalty or p.suppressed:
            raise ValueError("pack_rows: penalties and suppression lists need sample()")
        a.temperature, a.top_p, a.min_p, a.top_k = p.temperature, p.top_p, p.min_p, int(p.top_k or 0)
        a.rep_penalty, a.presence_penalty, a.frequency_penalty = 1.0, 0.0, 0.0
        a.seed, a.step = int(p.seed) & 0xFFFFFFFFFFFFFFFF, int(p.step)
        a.range_lo, a.range_hi = p.allowed_range if p.allowed_range is not None else (0, 0)
    return torch.frombuffer(bytearray(bytes(arr)), dtype=torch.uint8)


def row_bytes() -> int:
    return ctypes.sizeof(_Row)


def sample_packed(logits: torch.Tensor, rows_dev: torch.Tensor, out: torch.Tensor, work: torch.Tensor,
                  logprob: torch.Tensor | None = None) -> torch.Tensor:
    """Sampling on rows already packed on the device (``pack_rows(...).to(device)``): no host work and
    no allocation, so the call can be captured in a CUDA graph and the rows refreshed between replays.
    ``work``: fp32 [B, V] scratch; ``out``: int32 [B]."""
    B, V = logits.shape
    assert logits.is_cuda and logits.stride(1) == 1 and rows_dev.numel() >= B * row_bytes()
    rc = nv.lib("sampler").omni_sample(nv.ptr(logits), ctypes.c_int(1 if logits.dtype == torch.bfloat16 else 0),
                                       ctypes.c_long(logits.stride(0)), ctypes.c_int(V), ctypes.c_int(B), nv.ptr(rows_dev),
                                       nv.ptr(None), nv.ptr(None), nv.ptr(work), nv.ptr(None), nv.ptr(out),
                                       nv.ptr(logprob), nv.stream_ptr())
    nv.check_rc(rc, "omni_sample")
    return out


def sample(logits: torch.Tensor, rows: list[RowParams]):
    """logits [B, V] (fp32 or bf16).  Returns (ids int32 [B] on the logits' device, logprobs)."""
    if not logits.is_cuda:
        i, lp = sample_reference(logits, rows)
        return i.to(torch.int32), lp
    B, V = logits.shape
    assert logits.stride(1) == 1 and len(rows) == B
    arr = (_Row * B)()
    hist, sup = [], []
    need_cnt = False
    for r, p in enumerate(rows):
        a = arr[r]
        a.temperature, a.top_p, a.min_p, a.top_k = p.temperature, p.top_p, p.min_p, int(p.top_k or 0)
        a.rep_penalty, a.presence_penalty, a.frequency_penalty = p.repetition_penalty, p.presence_penalty, p.frequency_penalty
        a.seed, a.step = int(p.seed) & 0xFFFFFFFFFFFFFFFF, int(p.step)
        pen = p.repetition_penalty != 1.0 or p.presence_penalty != 0.0 or p.frequency_penalty != 0.0
        need_cnt |= pen
        a.hist_off, a.hist_len, a.gen_off = len(hist), (len(p.history) if pen else 0), p.num_prompt_tokens
        if pen:
            hist.extend(p.history)
        a.sup_off, a.sup_len = len(sup), len(p.suppressed)
        sup.extend(p.suppressed)
        a.range_lo, a.range_hi = p.allowed_range if p.allowed_range is not None else (0, 0)
    dev = logits.device
    rows_t = torch.frombuffer(bytearray(bytes(arr)), dtype=torch.uint8).to(dev)
    hist_t = torch.tensor(hist or [0], dtype=torch.int32, device=dev)
    sup_t = torch.tensor(sup or [0], dtype=torch.int32, device=dev)
    key = (dev.index, B, V)
    wk = _work.get(key)
    if wk is None:
        wk = [torch.empty(B, V, dtype=torch.float32, device=dev), None]
        _work[key] = wk
    if need_cnt and wk[1] is None:
        wk[1] = torch.empty(B, V, dtype=torch.int32, device=dev)
    out = torch.empty(B, dtype=torch.int32, device=dev)
    lp = torch.empty(B, dtype=torch.float32, device=dev)
    rc = nv.lib("sampler").omni_sample(nv.ptr(logits), ctypes.c_int(1 if logits.dtype == torch.bfloat16 else 0),
                                       ctypes.c_long(logits.stride(0)), ctypes.c_int(V), ctypes.c_int(B), nv.ptr(rows_t),
                                       nv.ptr(hist_t), nv.ptr(sup_t), nv.ptr(wk[0]), nv.ptr(wk[1] if need_cnt else None),
                                       nv.ptr(out), nv.ptr(lp), nv.stream_ptr())
    nv.check_rc(rc, "omni_sample")
    return out, lp


MAX_VOCAB = 262144                    # csrc/sample_given.cu: maxima and sums of a row's pieces of 256 lie in every block's shared memory


@functools.lru_cache(maxsize=None)
def _given_lib():
    P, I, L, F = ctypes.c_void_p, ctypes.c_int, ctypes.c_long, ctypes.c_float
    lib = nv.lib("sample_given")
    lib._cdll.omni_sample_given.argtypes = [P, I, L, I, I, P, P, F, P, I, P, F, P, F, P, P, P]
    return lib


def _per_row(name, v, B, dtype, device):
    """(address, value) of a parameter that is one number or a tensor of one per row."""
    if not isinstance(v, torch.Tensor):
        if dtype is torch.int32 and not -1 << 31 <= operator.index(v) < 1 << 31:
            raise ValueError(f"{name} {v}: an int32 expected")
        return None, v
    if v.dtype is not dtype or v.shape != (B,) or not v.is_contiguous() or v.device != device:
        raise ValueError(f"{name}: a number or contiguous {dtype} [{B}] on {device} expected, got {v.dtype} {tuple(v.shape)} on {v.device}")
    return v.data_ptr(), 0


def sample_given(logits: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out=None):
    """One token per row of ``logits`` [B, V] (bf16 or fp32) from the random numbers ``u`` (fp32 [B], in [0, 1)): (ids int32 [B], log probabilities fp32 [B]),
    into ``out``, such a pair, if given.  ``temperature``, ``top_p``, ``min_p`` (fp32 [B]) and ``top_k`` (int32 [B]) are numbers or one value per row.

    Weights are exp((x - max) / temperature) as multiples of 2^-44.  In the order by logit (ties: the lower id first) the first ``top_k`` stay (0: all), of these the
    ones of at least ``min_p`` of the largest, of these all before which less than ``top_p`` of their mass lies, and always the first.  The token is the
    first kept id at which the running mass in the order of the ids passes ``u`` times the kept mass.  Its log probability is that of the whole row at the temperature; the
    row's sum in it may be one in fp32, whose last bits depend on where the row begins against 16 bytes.
    Temperature 0 or below, or not a number: the largest logit, its log probability at temperature 1.  Cuts that are not numbers cut nothing.  Logits that are not numbers count as -inf; a row of nothing else
    gives id -1 and log probability -inf.  Does no host work and, with ``out``, no allocation: it can be captured."""
    if logits.dim() != 2 or logits.dtype not in (torch.bfloat16, torch.float32) or logits.stride(1) != 1:
        raise ValueError(f"logits: bf16 or fp32 [rows, vocabulary] with a row's values side by side expected, got {logits.dtype} {tuple(logits.shape)}")
    B, V = logits.shape
    if not 1 <= V <= MAX_VOCAB:
        raise ValueError(f"vocabulary of {V}: 1 to {MAX_VOCAB}")
    dev = logits.device
    if u.dtype is not torch.float32 or u.shape != (B,) or not u.is_contiguous() or u.device != dev:
        raise ValueError(f"u: contiguous fp32 [{B}] on {dev} expected, got {u.dtype} {tuple(u.shape)} on {u.device}")
    params = [_per_row("temperature", temperature, B, torch.float32, dev), _per_row("top_k", top_k, B, torch.int32, dev),
              _per_row("top_p", top_p, B, torch.float32, dev), _per_row("min_p", min_p, B, torch.float32, dev)]
    if out is None:
        ids, logprob = torch.empty(B, dtype=torch.int32, device=dev), torch.empty(B, dtype=torch.float32, device=dev)
    else:
        ids, logprob = out
        if any(t.dtype is not d or t.shape != (B,) or not t.is_contiguous() or t.device != dev for t, d in ((ids, torch.int32), (logprob, torch.float32))):
            raise ValueError(f"out: contiguous int32 [{B}] and fp32 [{B}] on {dev} expected")
    if not logits.is_cuda:
        for r in range(B):
            pick = [float(v[r]) if isinstance(v, torch.Tensor) else ctypes.c_float(v).value for v in (temperature, top_p, min_p)]     # numbers are fp32, too
            k = int(top_k[r]) if isinstance(top_k, torch.Tensor) else int(top_k)
            ids[r], logprob[r] = _given_row(logits[r].double(), float(u[r]), pick[0], k, *pick[1:])
        return ids, logprob
    if torch._C._cuda_getDevice() != dev.index:
        with torch.cuda.device(dev):
            return sample_given(logits, u, temperature, top_k, top_p, min_p, (ids, logprob))
    (t, tv), (k, kv), (p, pv), (m, mv) = params
    nv.check_rc(_given_lib().omni_sample_given(logits.data_ptr(), logits.dtype is torch.bfloat16, logits.stride(0), V, B, u.data_ptr(), t, tv, k, kv, p, pv, m, mv,
                                               ids.data_ptr(), logprob.data_ptr(), nv.stream_ptr()), "omni_sample_given")
    return ids, logprob


def _given_row(x, u, temperature, top_k, top_p, min_p):
    """The definition for one row in 64 bits."""
    x = torch.where(x.isnan(), -float("inf"), x)
    top = x.max()
    if top == -float("inf"):
        return -1, -float("inf")
    greedy = not temperature > 0
    z = torch.where(x == top, 0.0, (x - top) / (1.0 if greedy else temperature))
    z = torch.where(z.isnan(), -float("inf"), z)
    e = torch.exp(z)
    w = torch.round(e * 2.0 ** 44).long()
    log_all = torch.log(w.sum().double() * 2.0 ** -44)
    if greedy:
        i = int((x == top).nonzero()[0])
        return i, float(-log_all)
    order = torch.sort(x, descending=True, stable=True).indices
    if 0 < top_k < x.numel():
        order = order[:int(top_k)]
    order = order[e[order] >= (min(min_p, 1.0) if min_p > 0 else 0.0)]
    mass = torch.cumsum(w[order], 0)
    if top_p < 1:
        fits = (mass - w[order]).double() < top_p * mass[-1].double()
        order = order[:max(1, int(fits.sum()))]
    kept = torch.sort(order).values
    mass = torch.cumsum(w[kept], 0)
    i = int((mass.double() <= (u if u > 0 else 0.0) * mass[-1].double()).sum())
    if i == kept.numel():                                 # u = 1: the last one with mass
        i = int((w[kept] > 0).nonzero()[-1])
    return int(kept[i]), float(z[kept[i]] - log_all)
