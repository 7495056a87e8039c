"""Operators of a batched decoding step over an 8-bit paged K/V cache.

One step serves many requests at once, each with its own length:

* ``plan_step`` turns the request lengths into the step's row layout, assigns cache pages to
  the new tokens and lists what ``append_kv`` writes;
* ``append_kv`` quantises the step's keys and values into the cache, ``read_kv`` gives cached
  rows back as values;
* ``paged_attention`` attends the step's queries over the cache, causal inside a request;
* ``adjust_logits`` applies repetition / presence / frequency penalties, sparse biases and an
  allow-mask to the step's logits.

All lengths stay on the device, nothing here waits for the GPU, and every call runs on the
current stream (a captured CUDA graph replays them). As in :mod:`.functional`, CUDA tensors run
this library's sm_100a kernels and CPU tensors the same formulas in PyTorch.

Cache layout (:class:`PagedKV`): codes ``[pages, kv_heads, page_size, head_dim]`` in
``torch.float8_e4m3fn`` or ``torch.int8``, one fp32 scale per (page, kv head); value = code *
scale. Scales are powers of two in ``[2**-60, 2**60]``: the smallest one that fits the page's
largest finite magnitude into the codes' range (448 or 127), growing as larger values arrive on
the page. Infinities saturate; NaN stays NaN in e4m3 and becomes 0 in int8.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from ._ext import lib, status_word

PAGE_SIZES = (16, 32, 64, 128)
CODE_TYPES = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
MAX_REQUESTS = 4096           # requests of a step that the kernel of ``plan_step`` takes
MAX_BIAS = 1024               # biases of a row that the kernel of ``adjust_logits`` takes
_SCALE_EXP = 60


class PagedKV(NamedTuple):
    """Keys and values of one layer in 8 bits (see the module's text for the layout)."""

    k_pages: torch.Tensor
    v_pages: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    @staticmethod
    def create(num_pages: int, kv_heads: int, head_dim: int, *, page_size: int = 64,
               dtype: torch.dtype = torch.float8_e4m3fn, device="cuda") -> "PagedKV":
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
        if dtype not in CODE_TYPES:
            raise ValueError(f"cache codes are torch.float8_e4m3fn or torch.int8, not {dtype}")
        if min(num_pages, kv_heads, head_dim) < 1:
            raise ValueError("num_pages, kv_heads and head_dim must be >= 1")
        shape = (num_pages, kv_heads, page_size, head_dim)
        codes = [torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype)
                 for _ in range(2)]
        scales = [torch.ones(shape[:2], dtype=torch.float32, device=device) for _ in range(2)]
        return PagedKV(codes[0], codes[1], scales[0], scales[1])

    @property
    def page_size(self) -> int:
        return self.k_pages.shape[2]


class StepPlan(NamedTuple):
    """Row layout and cache pages of one step (int32 tensors).

    ``q_starts`` [B+1]: first row of each request; ``kv_lens`` [B]: keys after the step;
    ``positions`` / ``slots`` [num_tokens]: position in its request and cache slot
    (``page * page_size + offset``) of each row, 0 / -1 for rows past the last request;
    ``touched`` [U, 4]: (page, first row, first offset, rows) of every page that gets rows,
    (-1, 0, 0, 0) past the last; ``free_count`` [1]: free pages left; ``missing`` [1]: new
    pages that the free list could not give or a table has no column for (their rows have slot -1
    and are not cached; pages without a column stay in the free list).
    """

    q_starts: torch.Tensor
    kv_lens: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor
    touched: torch.Tensor
    free_count: torch.Tensor
    missing: torch.Tensor


def plan_step(context_lens: torch.Tensor, new_lens: torch.Tensor, tables: torch.Tensor,
              free_pages: torch.Tensor, free_count: torch.Tensor, *, page_size: int,
              num_tokens: int) -> StepPlan:
    """Plan a step: request ``b`` has ``context_lens[b]`` tokens cached and adds ``new_lens[b]``.

    ``tables`` [>= B, P] holds each request's pages; entries for the pages that the new tokens
    open are written here, taken from the end of ``free_pages[:free_count]`` in request order.
    ``num_tokens`` is the number of rows the step has (the sum of ``new_lens``, or more when the
    rest is padding; rows beyond it are dropped). ``free_count`` is not changed: the plan's own
    ``free_count`` is what is left. On CUDA a step has at most ``MAX_REQUESTS``.
    """
    if context_lens.is_cuda:
        return StepPlan._make(lib().plan_step(context_lens, new_lens, tables, free_pages,
                                              free_count, page_size, num_tokens))
    if page_size not in PAGE_SIZES:
        raise RuntimeError(f"page_size must be 16, 32, 64 or 128, got {page_size}")
    B, width = context_lens.numel(), tables.shape[1]
    if new_lens.numel() != B or tables.shape[0] < B:
        raise RuntimeError(f"new_lens and tables must hold {B} requests")
    room = min(num_tokens, num_tokens // page_size + 2 * B)
    positions, slots = [0] * num_tokens, [-1] * num_tokens
    touched, starts, kv = [], [0], []
    have = min(max(int(free_count), 0), free_pages.numel())
    taken = beyond = 0
    for b in range(B):
        ctx = max(int(context_lens[b]), 0)
        row = starts[-1]
        n = min(max(int(new_lens[b]), 0), num_tokens - row)
        old = -(-ctx // page_size)
        for lp in range(old, -(-(ctx + n) // page_size)):
            if lp >= width:
                beyond += 1
                continue
            tables[b, lp] = int(free_pages[have - 1 - taken]) if taken < have else -1
            taken += 1
        at = ctx
        while at < ctx + n:
            lp = at // page_size
            stop = min(ctx + n, (lp + 1) * page_size)
            page = int(tables[b, lp]) if lp < width else -1
            touched.append((page, row + at - ctx, at % page_size, stop - at))
            for i in range(at, stop):
                positions[row + i - ctx] = i
                if page >= 0:
                    slots[row + i - ctx] = page * page_size + i % page_size
            at = stop
        starts.append(row + n)
        kv.append(ctx + n)
    touched += [(-1, 0, 0, 0)] * (room - len(touched))

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=context_lens.device)

    return StepPlan(ints(starts), ints(kv), ints(positions), ints(slots),
                    ints(touched).reshape(room, 4), ints([max(have - taken, 0)]),
                    ints([max(taken - have, 0) + beyond]))


def _scale_exponent(amax: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Smallest e with ``amax <= qmax * 2**e``, in the range of scales."""
    m, e = torch.frexp(amax.double() / CODE_TYPES[dtype])
    e = torch.where(m == 0.5, e - 1, e).clamp(-_SCALE_EXP, _SCALE_EXP)
    return torch.where(amax == 0, -_SCALE_EXP, e)


def _encode(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    qmax = CODE_TYPES[dtype]
    if dtype == torch.int8:
        return x.nan_to_num(0.0, math.inf, -math.inf).clamp(-qmax, qmax).round().to(dtype)
    codes = x.clamp(-qmax, qmax).float().to(dtype)
    codes.view(torch.uint8)[x.isnan()] = 0x7F          # one NaN, without a sign
    return codes


def append_kv(cache: PagedKV, k: torch.Tensor, v: torch.Tensor, touched: torch.Tensor) -> None:
    """Write rows ``k`` / ``v`` [tokens, kv_heads, head_dim] into the pages that a plan's
    ``touched`` lists. A page whose scale grows has its older codes rescaled; a page written
    from offset 0 starts anew. ``touched`` lists a page once, as a plan does."""
    if cache.k_pages.is_cuda:
        lib().append_kv(*cache, k, v, touched)
        return
    for x, pages, scale in ((k, cache.k_pages, cache.k_scale), (v, cache.v_pages, cache.v_scale)):
        for page, row, off, n in touched.tolist():
            if page < 0 or page >= pages.shape[0] or n <= 0:
                continue
            new = x[row:row + n].double().transpose(0, 1)                   # [H, n, D]
            e = _scale_exponent(torch.where(new.isfinite(), new.abs(), 0.0).amax((1, 2)),
                                pages.dtype)
            now = torch.ldexp(torch.ones_like(e, dtype=torch.float64), e)
            if off:
                before = scale[page].double()
                now = torch.maximum(now, before)
                old = pages[page, :, :off].double() * (before / now)[:, None, None]
                pages[page, :, :off] = _encode(old, pages.dtype)
            pages[page, :, off:off + n] = _encode(new / now[:, None, None], pages.dtype)
            scale[page] = now.float()


def read_kv(cache: PagedKV, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Cached rows at ``slots`` (int32 [n]; a plan's numbering) as bf16 [n, kv_heads, head_dim]
    keys and values, exactly what the codes stand for; zeros for slot -1."""
    if cache.k_pages.is_cuda:
        k, v = lib().read_kv(*cache, slots)
        return k, v
    out = []
    idx = slots.long()
    total = cache.k_pages.shape[0] * cache.page_size
    live = (idx >= 0) & (idx < total)
    idx = idx.clamp(0, total - 1)
    page, off = idx // cache.page_size, idx % cache.page_size
    for pages, scale in ((cache.k_pages, cache.k_scale), (cache.v_pages, cache.v_scale)):
        x = pages.view(torch.uint8)[page, :, off].view(pages.dtype).float() * scale[page][:, :, None]
        out.append(torch.where(live[:, None, None], x, 0.0).to(torch.bfloat16))
    return out[0], out[1]


def paged_attention(q: torch.Tensor, cache: PagedKV, tables: torch.Tensor,
                    q_starts: torch.Tensor, kv_lens: torch.Tensor, *, max_new: int,
                    softmax_scale: float | None = None, lse: torch.Tensor | None = None
                    ) -> torch.Tensor:
    """Attention of rows ``q`` [tokens, heads, head_dim] over the cache: [tokens, heads, head_dim].

    Request ``b`` owns rows ``q_starts[b]:q_starts[b+1]``, the last of its ``kv_lens[b]`` cached
    positions; a row sees its own position and those before it. ``heads`` is a multiple of the
    cache's kv heads (grouped queries). ``max_new`` is an upper bound of the rows of one request
    (one that is too small costs speed only).
    Rows before ``q_starts[0]`` or past ``q_starts[B]`` and rows that see no key give 0; positions on a missing page
    (table entry -1, or past the table's columns) are not seen. NaN in a position reaches the rows that see it and no others.
    ``lse`` (fp32 [tokens, heads]) receives the base-2 log-sum-exp of the scaled scores, -inf for
    rows that see nothing. Value scales of one request's pages may differ by up to 2**100.

    On CUDA, more than 2**30 tiles of 32 keys by 16 rows in one call (prompts of more than 128
    heads per kv head) leave the output unwritten and a status for ``check_status``.
    """
    D = cache.k_pages.shape[3]
    scale = softmax_scale if softmax_scale is not None else 1.0 / math.sqrt(D)
    if q.is_cuda:
        return lib().paged_attention(q, *cache, tables, q_starts, kv_lens, max_new, scale, lse,
                                     status_word(q.device))
    T, heads, _ = q.shape
    kv_heads, ps = cache.k_pages.shape[1], cache.page_size
    if heads % kv_heads:
        raise RuntimeError(f"query heads ({heads}) must be a multiple of kv heads ({kv_heads})")
    out = torch.zeros_like(q, memory_format=torch.contiguous_format)
    if lse is not None:
        lse.fill_(-math.inf)
    starts = q_starts.tolist()
    cd = torch.float64 if q.dtype == torch.float64 else torch.float32
    for b, n in enumerate(kv_lens.tolist()):
        r0, r1 = starts[b], starts[b + 1]
        if r1 <= r0 or n <= 0:
            continue
        pos = n - (r1 - r0) + torch.arange(r1 - r0)
        n = min(n, tables.shape[1] * ps)                     # positions past the table have no page
        ids = tables[b, :-(-n // ps)].long()
        there = ((ids >= 0) & (ids < cache.k_pages.shape[0])).repeat_interleave(ps)[:n]
        ids = ids.clamp(0, cache.k_pages.shape[0] - 1)

        def dense(pages, sc):
            x = pages.view(torch.uint8)[ids].view(pages.dtype).to(cd) * sc[ids].to(cd)[..., None, None]
            x = x.transpose(1, 2).reshape(-1, kv_heads, D)[:n]                  # [n, H, D]
            x = torch.where(there[:, None, None], x, 0.0)
            return x.repeat_interleave(heads // kv_heads, 1).transpose(0, 1)

        s = (q[r0:r1].to(cd).transpose(0, 1) @ dense(cache.k_pages, cache.k_scale).transpose(1, 2)
             ) * scale
        seen = (torch.arange(n)[None] <= pos[:, None]) & there[None]
        s = s.masked_fill(~seen, -math.inf)
        z = torch.logsumexp(s, -1)
        p = torch.where(z[..., None] == -math.inf, 0.0, torch.exp(s - z[..., None]))
        v = dense(cache.v_pages, cache.v_scale)
        bad = v.isnan()                       # reaches the rows that see it and no others
        o = p @ torch.where(bad, 0.0, v)
        o = torch.where(seen.to(cd) @ bad.to(cd) > 0, math.nan, o)
        out[r0:r1] = o.transpose(0, 1).to(q.dtype)
        if lse is not None:
            lse[r0:r1] = (z / math.log(2.0)).transpose(0, 1).float()
    return out


def adjust_logits(logits: torch.Tensor, history: torch.Tensor, history_lens: torch.Tensor,
                  prompt_lens: torch.Tensor, *, repetition: torch.Tensor | None = None,
                  presence: torch.Tensor | None = None, frequency: torch.Tensor | None = None,
                  bias_ids: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                  allowed: torch.Tensor | None = None) -> torch.Tensor:
    """Next-token scores (fp32 [B, V]) from ``logits`` [B, V] and each request's rules.

    ``history`` [B, L] (int32) holds ``history_lens[b]`` tokens of request ``b``: its prompt
    (``prompt_lens[b]`` tokens), then what it has generated; ids outside the vocabulary count
    for nothing. In this order:

    * tokens that occur in the history: score / ``repetition[b]`` if positive, else times it;
    * tokens generated ``c > 0`` times: minus ``frequency[b] * c + presence[b]``;
    * ``bias[b, i]`` is added to token ``bias_ids[b, i]`` (int32; -1 = unused; repeated ids add;
      on CUDA at most ``MAX_BIAS`` a row);
    * tokens whose bit in ``allowed`` (int32 [B, ceil(V / 32)], bit ``v % 32`` of word
      ``v // 32``) is 0 become -inf, whatever their score.
    """
    if logits.is_cuda:
        return lib().adjust_logits(logits, history, history_lens, prompt_lens, repetition,
                                   presence, frequency, bias_ids, bias, allowed)
    B, V = logits.shape
    z = logits.to(torch.float64 if logits.dtype == torch.float64 else torch.float32).clone()
    if (bias_ids is None) != (bias is None):
        raise RuntimeError("bias_ids and bias come together")
    for b in range(B):
        h = history[b, :max(int(history_lens[b]), 0)].long()
        ok = (h >= 0) & (h < V)
        ids = h[ok].unique()
        if repetition is not None:
            r = repetition[b].to(z.dtype)
            z[b, ids] = torch.where(z[b, ids] > 0, z[b, ids] / r, z[b, ids] * r)
        made = h[max(int(prompt_lens[b]), 0):]
        ids, count = made[(made >= 0) & (made < V)].unique(return_counts=True)
        if frequency is not None:
            z[b, ids] -= frequency[b].to(z.dtype) * count
        if presence is not None:
            z[b, ids] -= presence[b].to(z.dtype)
        if bias is not None:
            ids = bias_ids[b].long()
            ok = (ids >= 0) & (ids < V)
            z[b].index_add_(0, ids[ok], bias[b, ok].to(z.dtype))
    if allowed is not None:
        bits = (allowed[:, :, None] >> torch.arange(32)) & 1
        z[bits.reshape(B, -1)[:, :V] == 0] = -math.inf
    return z
