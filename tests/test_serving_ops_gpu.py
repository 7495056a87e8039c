"""Batched-serving kernels (step plan, 8-bit paged K/V cache, attention over it, logit rules)
against plain 64-bit computations.

Tolerances: the cache write, read and plan are exact arithmetic (powers of two, integers), so
their results must be equal. Attention rounds its output once to bf16 (8 significant bits: half
an ulp is up to 2^-8 of the value) and each probability to f16 (2^-11 of it, with random signs:
under 2^-10 of the row's largest output in sum). Logits are a handful of fp32 operations: 4 ulp of the largest operand.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from nano_megatron_b200.ops import check_status, lib, serving  # noqa: E402

DEV = "cuda"
E4M3, INT8 = torch.float8_e4m3fn, torch.int8
QMAX = {E4M3: 448.0, INT8: 127.0}


def ints(v, dev=DEV):
    return torch.tensor(v, dtype=torch.int32, device=dev)


# ------------------------------------------------------------------------------ step plan
def _plan_inputs(contexts, news, page, width, pages, seed=0):
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=g).tolist()
    tables = torch.full((len(contexts) + 1, width), -1, dtype=torch.int32)
    at = 0
    for b, c in enumerate(contexts):
        for i in range(-(-c // page)):
            tables[b, i] = order[at]
            at += 1
    return tables, order[at:]


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("contexts,news,extra", [
    ([0], [1], 0),
    ([0, 15, 16, 17, 63, 64, 127, 128], [1] * 8, 0),
    ([5, 0, 130, 64], [0, 300, 1, 64], 7),            # a request that adds nothing, padding rows
    ([0] * 3, [0] * 3, 5),                            # nothing but padding
    (list(range(0, 900, 3)), [i % 5 for i in range(300)], 3),   # more requests than threads
])
def test_plan_matches_host(page, contexts, news, extra):
    tables, free = _plan_inputs(contexts, news, page, width=1100 // page + 2,
                                pages=sum(-(-(c + n) // page) for c, n in zip(contexts, news)) + 5)
    T = sum(news) + extra
    host_tables = tables.clone()
    want = serving.plan_step(ints(contexts, "cpu"), ints(news, "cpu"), host_tables,
                             ints(free, "cpu"), ints([len(free) - 2], "cpu"), page_size=page,
                             num_tokens=T)
    dev_tables = tables.to(DEV)
    got = serving.plan_step(ints(contexts), ints(news), dev_tables, ints(free),
                            ints([len(free) - 2]), page_size=page, num_tokens=T)
    for name, a, b in zip(got._fields, got, want):
        assert torch.equal(a.cpu(), b), name
    assert torch.equal(dev_tables.cpu(), host_tables)
    # the host form itself, from the definition
    pos = [c + i for c, n in zip(contexts, news) for i in range(n)]
    req = [b for b, n in enumerate(news) for _ in range(n)]
    assert want.positions.tolist() == pos + [0] * extra
    assert want.slots.tolist() == [int(host_tables[b, p // page]) * page + p % page
                                   for b, p in zip(req, pos)] + [-1] * extra
    assert int(want.missing) == 0


def test_plan_out_of_pages_and_out_of_table():
    tables = torch.full((2, 2), -1, dtype=torch.int32, device=DEV)
    p = serving.plan_step(ints([0, 0]), ints([40, 40]), tables, ints([7, 9, 3]), ints([2]),
                          page_size=16, num_tokens=80)
    # six pages wanted, two free; the table is two pages wide
    assert tables.tolist() == [[9, 7], [-1, -1]]
    assert p.missing.item() == 4 and p.free_count.item() == 0
    assert p.slots.tolist() == [9 * 16 + i for i in range(16)] + [7 * 16 + i for i in range(16)] + [-1] * 48
    # rows beyond num_tokens are dropped
    p = serving.plan_step(ints([0, 0]), ints([40, 40]), tables, ints(list(range(9))), ints([9]),
                          page_size=16, num_tokens=10)
    assert p.q_starts.tolist() == [0, 10, 10] and p.kv_lens.tolist() == [10, 0]


# ---------------------------------------------------------------------- cache write / read
def _cache(pages, heads, dim, page, dtype, dev=DEV, garbage=True):
    c = serving.PagedKV.create(pages, heads, dim, page_size=page, dtype=dtype, device=dev)
    if garbage:   # stale bytes: NaN in e4m3, large codes in int8
        for t in (c.k_pages, c.v_pages):
            t.view(torch.uint8).fill_(0x7F)
    return c


def _touched(contexts, news, page, seed=0):
    width = max(-(-(c + n) // page) for c, n in zip(contexts, news)) + 1
    total = sum(-(-(c + n) // page) for c, n in zip(contexts, news))
    tables, free = _plan_inputs(contexts, news, page, width, total + 3, seed)
    plan = serving.plan_step(ints(contexts, "cpu"), ints(news, "cpu"), tables, ints(free, "cpu"),
                             ints([len(free)], "cpu"), page_size=page, num_tokens=sum(news))
    return plan, tables, total + 3


def _rows(T, heads, dim, strided, seed=0, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(T, (2 * heads + 3) * dim, generator=g, device=DEV).mul_(scale).bfloat16()
    k, v = x[:, dim:(1 + heads) * dim], x[:, (2 + heads) * dim:(2 + 2 * heads) * dim]
    k, v = k.view(T, heads, dim), v.view(T, heads, dim)
    return (k, v) if strided else (k.contiguous(), v.contiguous())


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("strided", [False, True])
def test_append_and_read_match_64_bits(dtype, dim, page, strided):
    heads = 3
    contexts, news = [0, 5, page, 2 * page - 1, 7], [1, page + 3, 1, 2, 2 * page]
    plan0, _, pages = _touched([0] * 5, [max(c, 1) for c in contexts], page)
    gpu, cpu = _cache(pages + 40, heads, dim, page, dtype), _cache(pages + 40, heads, dim, page, dtype, "cpu")
    plan, tables, _ = _touched(contexts, news, page)
    # contexts first (small values), then the new rows (8 times as large: scales must grow)
    ctx_plan = serving.plan_step(ints([0] * 5, "cpu"), ints(contexts, "cpu"), tables.clone(),
                                 ints([0], "cpu"), ints([0], "cpu"), page_size=page,
                                 num_tokens=sum(contexts))
    entries, at = [], 0
    for b, c in enumerate(contexts):
        for lp in range(-(-c // page)):
            n = min(page, c - lp * page)
            entries.append((int(tables[b, lp]), at, 0, n))
            at += n
    assert ctx_plan.q_starts[-1] == at
    entries = torch.tensor(entries, dtype=torch.int32)
    for e, T, scale in ((entries, at, 0.2), (plan.touched, sum(news), 1.7)):
        k, v = _rows(T, heads, dim, strided, seed=T, scale=scale)
        serving.append_kv(gpu, k, v, e.to(DEV))
        serving.append_kv(cpu, k.cpu(), v.cpu(), e)
    for a, b in zip(gpu, cpu):
        assert torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8))
    slots = torch.cat([plan.slots, ints([-1, 0], "cpu")])
    for a, b in zip(serving.read_kv(gpu, slots.to(DEV)), serving.read_kv(cpu, slots)):
        assert a.dtype == torch.bfloat16 and torch.equal(a.cpu().nan_to_num(7.0), b.nan_to_num(7.0))
    # the new rows come back within half a step of their page's scale
    back = serving.read_kv(gpu, plan.slots.to(DEV))
    for x, y, s in ((k, back[0], gpu.k_scale), (v, back[1], gpu.v_scale)):
        step = s[(plan.slots // page).long().to(DEV)][:, :, None]
        err = (x.float() - y.float()).abs()
        bound = 0.5 * step if dtype == INT8 else torch.maximum(x.float().abs() * 2.0 ** -4, step * 2.0 ** -10)
        assert bool((err <= bound).all())


@pytest.mark.parametrize("dtype", [E4M3, INT8])
def test_append_special_values(dtype):
    """Zeros, infinities, NaN, magnitudes beyond the scales' range, a scale at a boundary."""
    heads, dim, page = 1, 64, 16
    qmax = QMAX[dtype]
    rows = torch.zeros(6, heads, dim)
    rows[1, 0, :3] = torch.tensor([math.inf, -math.inf, math.nan])
    rows[1, 0, 3] = 3.0
    rows[2, 0, 0] = qmax if dtype == INT8 else 448.0        # exactly fills scale 1
    rows[3, 0, 0] = qmax * 1.01                             # needs scale 2
    rows[4] = 1e-30
    rows[5, 0, 0] = 3e38
    x = rows.bfloat16()
    touched = ints([[i, i, 0, 1] for i in range(6)], "cpu")
    gpu, cpu = _cache(6, heads, dim, page, dtype), _cache(6, heads, dim, page, dtype, "cpu")
    serving.append_kv(gpu, x.to(DEV), x.to(DEV), touched.to(DEV))
    serving.append_kv(cpu, x, x, touched)
    for a, b in zip(gpu, cpu):
        assert torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8))
    s = gpu.k_scale[:, 0].tolist()
    # bf16 rounds 127 * 1.01 to 128 and 448 * 1.01 to 452
    assert s[0] == 2.0 ** -60 and s[2] == 1.0 and s[3] == 2.0 and s[4] == 2.0 ** -60 and s[5] == 2.0 ** 60
    back = serving.read_kv(gpu, ints([16 * i for i in range(6)]))[0].float().cpu()
    assert back[0].abs().max() == 0
    assert back[1, 0, 0] == qmax * s[1] and back[1, 0, 1] == -qmax * s[1] and back[1, 0, 3] == 3.0
    assert math.isnan(back[1, 0, 2]) == (dtype == E4M3)
    assert back[5, 0, 0] == qmax * 2.0 ** 60


def test_append_one_token_at_a_time_equals_at_once_e4m3():
    """Power-of-two scales: e4m3 codes do not depend on how the rows arrived, unless they
    underflow (values here stay well above)."""
    heads, dim, page = 2, 128, 32
    g = torch.Generator(device=DEV).manual_seed(3)
    x = (1.0 + torch.rand(page, heads, dim, generator=g, device=DEV)) * torch.linspace(
        0.5, 8.0, page, device=DEV)[:, None, None]
    x = x.bfloat16()
    one, many = _cache(1, heads, dim, page, E4M3), _cache(1, heads, dim, page, E4M3)
    serving.append_kv(one, x, x, ints([[0, 0, 0, page]]))
    for i in range(page):
        serving.append_kv(many, x[i:i + 1], x[i:i + 1], ints([[0, 0, i, 1]]))
    for a, b in zip(one, many):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_append_ignores_entries_out_of_range():
    c = _cache(2, 1, 64, 16, E4M3)
    before = [t.view(torch.uint8).clone() for t in c]
    x = torch.ones(4, 1, 64, device=DEV, dtype=torch.bfloat16)
    serving.append_kv(c, x, x, ints([[-1, 0, 0, 1], [2, 0, 0, 1], [0, 3, 0, 2], [0, 0, 15, 2],
                                     [1, -1, 0, 1], [1, 0, 0, 0], [1, 0, -1, 1]]))
    for a, b in zip(c, before):
        assert torch.equal(a.view(torch.uint8), b)


# -------------------------------------------------------------------------------- attention
def _filled(contexts, heads, dim, page, dtype, seed=0, level=1.0):
    """A cache with `contexts` tokens per request, everything else stale; tables; scales that
    differ from page to page by up to 2^12."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    used = [-(-c // page) for c in contexts]
    pages = sum(used) + 2
    cache = _cache(pages, heads, dim, page, dtype)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    tables = torch.full((len(contexts), max(used) + 1), 10 ** 6, dtype=torch.int32)
    at = 0
    for b, c in enumerate(contexts):
        if not c:
            continue
        entries = []
        for i in range(used[b]):
            tables[b, i] = order[at]
            entries.append((order[at], i * page, 0, min(page, c - i * page)))
            at += 1
        k = torch.randn(c, heads, dim, generator=g, device=DEV) * level
        v = torch.randn(c, heads, dim, generator=g, device=DEV)
        if level == 1.0:   # value levels by page
            e = torch.randint(-6, 7, (used[b],), generator=torch.Generator().manual_seed(b))
            v *= (2.0 ** e.float()).repeat_interleave(page)[:c, None, None].to(DEV)
        serving.append_kv(cache, k.bfloat16(), v.bfloat16(), ints(entries))
    return cache, tables.to(DEV)


def _oracle(q, cache, tables, starts, kv, scale):
    """Softmax attention in 64 bits from the cached values, one request and head at a time."""
    T, Hq, D = q.shape
    pages, H, ps, _ = cache.k_pages.shape
    out = torch.zeros(T, Hq, D, dtype=torch.float64, device=DEV)
    lse = torch.full((T, Hq), -math.inf, dtype=torch.float64, device=DEV)
    for b, n in enumerate(kv):
        ids = tables[b, :-(-n // ps)].long()
        there = ((ids >= 0) & (ids < pages)).repeat_interleave(ps)[:n]
        ids = ids.clamp(0, pages - 1)
        for r in range(starts[b], starts[b + 1]):
            seen = there & (torch.arange(n, device=DEV) <= n - (starts[b + 1] - r))
            if not seen.any():
                continue
            for h in range(H):
                k, v = ((p.view(torch.uint8)[ids, h].view(p.dtype).double()
                         * s[ids, h].double()[:, None, None]).reshape(-1, D)[:n][seen]
                        for p, s in ((cache.k_pages, cache.k_scale), (cache.v_pages, cache.v_scale)))
                j = slice(h * Hq // H, (h + 1) * Hq // H)
                z = q[r, j].double() @ k.T * scale
                lse[r, j] = torch.logsumexp(z, -1) / math.log(2.0)
                out[r, j] = torch.softmax(z, -1) @ v
    return out, lse


def _check(contexts, news, Hq, H, D, page, dtype, *, pad=0, seed=0, level=1.0, scale=None,
           strided=False, holes=()):
    cache, tables = _filled(contexts, H, D, page, dtype, seed, level)
    for b, i in holes:
        tables[b, i] = -1
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    T = starts[-1] + pad
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    q = torch.randn(T, Hq + (2 if strided else 0), D, generator=g, device=DEV).bfloat16()
    q = q[:, 1:1 + Hq] if strided else q
    lse = torch.full((T, Hq), 7.0, device=DEV)
    got = serving.paged_attention(q, cache, tables, ints(starts), ints(contexts),
                                  max_new=max(news), softmax_scale=scale, lse=lse)
    torch.cuda.synchronize()
    check_status(torch.device(DEV))
    want, want_lse = _oracle(q, cache, tables, starts, contexts, scale or D ** -0.5)
    top = want.abs().amax(-1, keepdim=True)
    assert got.dtype == torch.bfloat16
    assert bool(((got.double() - want).abs() <= top * (2.0 ** -8 + 2.0 ** -10)).all()), \
        ((got.double() - want).abs() / top.clamp(min=1e-30)).max().item()
    inf = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse), inf)
    # fp32 sums of exact products: 2^-18 of the largest score, or 2^-16 absolute
    assert bool(((lse.double() - want_lse)[~inf].abs() <= 2.0 ** -16 + want_lse[~inf].abs() * 2.0 ** -18).all())
    return got


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("Hq,H,D", [(16, 16, 64), (16, 4, 128), (6, 2, 64), (8, 1, 128), (20, 1, 64),
                                    (5, 5, 128)])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_decode_matches_64_bits(dtype, Hq, H, D, page):
    _check([1, 2, 15, 16, 17, 31, 32, 33, 100, 257, 640], [1] * 11, Hq, H, D, page, dtype)


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("n", [1, 31, 1000, 9000])
def test_decode_one_request(page, n):
    """One request is split over the whole GPU and put together again."""
    _check([n], [1], 4, 1, 128, page, E4M3)
    _check([n], [1], 2, 2, 64, page, INT8)


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("D,Hq,H,page", [(128, 32, 8, 64), (64, 16, 16, 16), (128, 64, 4, 128)])
def test_long_shares(dtype, D, Hq, H, page):
    """Enough keys that every block works through many tiles of several units."""
    _check([3000 - 61 * i for i in range(24)], [1] * 24, Hq, H, D, page, dtype)


@pytest.mark.parametrize("D,Hq,H", [(64, 4, 4), (128, 8, 2), (128, 3, 1), (64, 20, 1)])
@pytest.mark.parametrize("page", [16, 64])
def test_several_new_tokens_are_causal(D, Hq, H, page):
    """Continuations of every short length, prompts from nothing, requests that add nothing."""
    _check([5, 3, 77, 64, 130, 17, 65, 1, 40, 0], [5, 2, 4, 3, 0, 17, 33, 1, 7, 0], Hq, H, D, page,
           E4M3, pad=3)


@pytest.mark.parametrize("D,Hq,H", [(64, 16, 16), (128, 16, 4), (128, 32, 8), (64, 6, 2)])
@pytest.mark.parametrize("dtype", [E4M3, INT8])
def test_prompts(D, Hq, H, dtype):
    """Long runs of new tokens, from nothing and over a context, next to decoding requests."""
    _check([200, 391, 300, 129], [200, 130, 1, 128], Hq, H, D, 64, dtype, pad=1)
    _check([70, 513], [70, 257], Hq, H, D, 16, dtype)


def test_many_requests():
    n = 300
    contexts = [(i * 37) % 90 for i in range(n)]
    _check(contexts, [1 if c else 0 for c in contexts], 2, 1, 64, 16, E4M3)


def test_strides_scale_and_holes():
    _check([100, 50], [1, 1], 8, 2, 128, 16, E4M3, strided=True, scale=0.3)
    _check([100, 50], [3, 2], 8, 2, 64, 16, INT8, strided=True, scale=0.05)
    # a missing page in the middle, a request whose pages are all missing
    _check([100, 50, 40], [1, 2, 1], 8, 2, 128, 16, E4M3, holes=[(0, 2), (2, 0), (2, 1), (2, 2)])
    _check([200, 100], [1, 1], 8, 2, 64, 64, E4M3, holes=[(0, 1), (1, 0)])
    _check([200, 300], [150, 1], 8, 2, 64, 64, E4M3, holes=[(0, 1), (1, 0)])


def test_large_scores():
    """Scores of several hundred: the running maximum moves a lot between tiles."""
    _check([700, 90], [1, 3], 8, 2, 128, 64, E4M3, level=30.0)
    _check([300], [200], 8, 2, 128, 64, E4M3, level=30.0)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,n", [(2, 4), (6, 5), (2, 20), (4, 150), (2, 300)])
def test_nan_reaches_only_the_rows_that_see_it(D, Hq, n):
    """NaN keys and values among the new tokens: earlier rows are as without them; later rows are
    NaN (a NaN key) or NaN in the value's column."""
    ctx = 37
    cache, tables = _filled([ctx + n], 2, D, 16, E4M3)
    q = torch.randn(n, 2 * Hq, D, device=DEV).bfloat16()
    args = (tables, ints([0, n]), ints([ctx + n]))
    clean = serving.paged_attention(q, cache, *args, max_new=n)
    first = n // 2                       # row whose position holds the NaN value of head 0
    pos = ctx + first
    page, off = int(tables[0, pos // 16]), pos % 16
    cache.v_pages.view(torch.uint8)[page, 0, off, 5] = 0xFF
    later = ctx + n - 1                  # the last position's key of head 1
    cache.k_pages.view(torch.uint8)[int(tables[0, later // 16]), 1, later % 16, 3] = 0x7F
    got = serving.paged_attention(q, cache, *args, max_new=n)
    assert torch.equal(got[:first], clean[:first])
    assert bool(got[first:, :Hq, 5].isnan().all())
    others = [c for c in range(D) if c != 5]
    assert torch.equal(got[:, :Hq][..., others], clean[:, :Hq][..., others])
    assert torch.equal(got[:-1, Hq:], clean[:-1, Hq:]) and bool(got[-1, Hq:].isnan().all())


def test_row_offsets_past_the_keys_see_nothing():
    """kv_lens smaller than the rows (a caller's error): the first rows see no key and give 0."""
    cache, tables = _filled([20], 1, 64, 16, E4M3)
    q = torch.randn(30, 2, 64, device=DEV).bfloat16()
    lse = torch.empty(30, 2, device=DEV)
    o = serving.paged_attention(q, cache, tables, ints([0, 30]), ints([20]), max_new=30, lse=lse)
    assert o[:10].abs().max() == 0 and bool(torch.isinf(lse[:10]).all())
    assert o[10:].abs().amax((1, 2)).min() > 0


@pytest.mark.parametrize("D", [64, 128])
def test_rows_at_odd_addresses(D):
    """Rows that start at odd elements: the scalar loads of the cache write, a copied query."""
    T, H = 23, 2
    wide = torch.randn(T, 3 * H * D + 1, device=DEV).bfloat16()
    q, k, v = (wide[:, 1 + i * H * D:1 + (i + 1) * H * D].view(T, H, D) for i in range(3))
    assert k.data_ptr() % 16 and k.stride(0) % 8
    touched = ints([[1, 0, 0, 16], [0, 16, 0, 7]])
    odd, even = _cache(2, H, D, 16, E4M3), _cache(2, H, D, 16, E4M3)
    serving.append_kv(odd, k, v, touched)
    serving.append_kv(even, k.contiguous(), v.contiguous(), touched)
    for a, b in zip(odd, even):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    args = (odd, ints([[1, 0]]), ints([0, T]), ints([T]))
    assert torch.equal(serving.paged_attention(q, *args, max_new=T),
                       serving.paged_attention(q.contiguous(), *args, max_new=T))


def test_cache_beyond_4_gib():
    """Pages whose byte offsets pass 32 bits: write, read back, decode, prompt."""
    H, D, page, pages = 8, 128, 64, 70000                # 4.6 GB of codes each
    cache = serving.PagedKV.create(pages, H, D, page_size=page)
    small = serving.PagedKV.create(4, H, D, page_size=page)
    far = [pages - 1, 65536, pages - 2, 3]
    x = torch.randn(230, 2, H, D, device=DEV).bfloat16()
    rows = [(0, 64), (64, 64), (128, 64), (192, 38)]
    for c, ids in ((cache, far), (small, [0, 1, 2, 3])):
        serving.append_kv(c, x[:, 0], x[:, 1], ints([[p, r, 0, n] for p, (r, n) in zip(ids, rows)]))
    slots = [[p * page + i for p, (_, n) in zip(ids, rows) for i in range(n)]
             for ids in (far, [0, 1, 2, 3])]
    for a, b in zip(serving.read_kv(cache, ints(slots[0])), serving.read_kv(small, ints(slots[1]))):
        assert torch.equal(a, b)
    for n in (1, 200):
        q = torch.randn(n, 4 * H, D, device=DEV).bfloat16()
        a, b = (serving.paged_attention(q, c, ints([ids]), ints([0, n]), ints([230]), max_new=n)
                for c, ids in ((cache, far), (small, [0, 1, 2, 3])))
        assert torch.equal(a, b) and bool(a.isfinite().all())


def test_empty_calls():
    p = serving.plan_step(ints([]), ints([]), torch.zeros(0, 1, dtype=torch.int32, device=DEV),
                          ints([0]), ints([1]), page_size=16, num_tokens=3)
    assert p.q_starts.tolist() == [0] and p.slots.tolist() == [-1] * 3 and p.free_count.item() == 1
    cache, tables = _filled([20], 1, 64, 16, E4M3)
    q = torch.empty(0, 2, 64, device=DEV, dtype=torch.bfloat16)
    assert serving.paged_attention(q, cache, tables, ints([0, 0]), ints([20]), max_new=0).shape == (0, 2, 64)
    q = torch.ones(3, 2, 64, device=DEV, dtype=torch.bfloat16)
    o = serving.paged_attention(q, cache, tables[:0], ints([0]), ints([]), max_new=0)
    assert o.abs().max() == 0
    k, v = serving.read_kv(cache, ints([]))
    assert k.shape == v.shape == (0, 1, 64)
    serving.append_kv(cache, q[:, :1], q[:, :1], ints([]).view(0, 4))


def test_attention_repeats_bit_for_bit_and_in_graphs_and_streams():
    contexts = [900, 33, 2000, 450]
    cache, tables = _filled(contexts, 2, 128, 64, E4M3)
    q = torch.randn(4, 8, 128, device=DEV).bfloat16()
    starts, kv = ints([0, 1, 2, 3, 4]), ints(contexts)

    def call():
        return serving.paged_attention(q, cache, tables, starts, kv, max_new=1)

    want = call()
    for _ in range(5):
        assert torch.equal(call(), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        got = [call() for _ in range(3)]
    here = [call() for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got + here)
    with torch.cuda.graph(graph):
        out = call()
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)
    check_status(torch.device(DEV))


# ------------------------------------------------------------------------------- logit rules
def _logits_oracle(z, hist, lens, prompts, rep, pre, freq, ids, bias, allowed):
    z = z.double().cpu().clone()
    B, V = z.shape
    for b in range(B):
        h = [t for t in hist[b, :lens[b]].tolist()]
        made = [t for t in h[prompts[b]:]]
        for t in set(x for x in h if 0 <= x < V):
            if rep is not None:
                r = rep[b].double().item()
                z[b, t] = z[b, t] / r if z[b, t] > 0 else z[b, t] * r
        for t in set(x for x in made if 0 <= x < V):
            if freq is not None:
                z[b, t] -= freq[b].double().item() * made.count(t)
            if pre is not None:
                z[b, t] -= pre[b].double().item()
        if ids is not None:
            for t, x in zip(ids[b].tolist(), bias[b].double().tolist()):
                if 0 <= t < V:
                    z[b, t] += x
        if allowed is not None:
            for t in range(V):
                if not (allowed[b, t // 32].item() >> (t % 32)) & 1:
                    z[b, t] = -math.inf
    return z


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V,L,NB,mask,offset", [(1, 1, 1, True, 0), (31, 5, 0, True, 0), (33, 3, 2, False, 1),
                                                (1000, 300, 7, True, 0), (4096, 50, 40, True, 3),
                                                (4101, 700, 3, True, 1), (9000, 2000, 64, False, 0),
                                                (50257, 100, 5, True, 0)])
def test_logits_match_64_bits(dtype, V, L, NB, mask, offset):
    B = 3
    g = torch.Generator().manual_seed(V)
    wide = torch.randn(B, V + offset + 2, generator=g).mul(4).to(dtype).to(DEV)
    z = wide[:, offset:offset + V]                       # row stride and alignment of a slice
    hist = torch.randint(-2, min(V, 200) + 2, (B, L), generator=g).int()
    lens, prompts = [L, L // 2, 0], [L // 3, L, 0]
    rep, pre, freq = 1 + torch.rand(B, generator=g), torch.rand(B, generator=g), torch.rand(B, generator=g)
    ids = bias = allowed = None
    if NB:
        ids = torch.randint(-1, V + 1, (B, NB), generator=g).int()
        ids[:, -1] = ids[:, 0]                           # a repeated token: its values add
        bias = torch.randn(B, NB, generator=g)
        bias[0, 0] = 3.0
    if mask:
        allowed = torch.randint(-2 ** 31, 2 ** 31 - 1, (B, (V + 31) // 32), generator=g).int()
        allowed[2] = 0                                   # a row whose mask leaves nothing
    dev = [None if t is None else t.to(DEV) for t in (rep, pre, freq, ids, bias, allowed)]
    got = serving.adjust_logits(z, hist.to(DEV), ints(lens), ints(prompts), repetition=dev[0],
                                presence=dev[1], frequency=dev[2], bias_ids=dev[3], bias=dev[4],
                                allowed=dev[5]).cpu()
    want = _logits_oracle(z, hist, lens, prompts, rep, pre, freq, ids, bias, allowed)
    assert got.dtype == torch.float32 and torch.equal(torch.isinf(got), torch.isinf(want))
    ok = ~torch.isinf(want)
    big = max(16.0, float(freq.max()) * L)
    assert (got.double() - want)[ok].abs().max().item() <= 4 * big * 2.0 ** -23 if ok.any() else True


def test_logits_without_rules_and_special_values():
    z = torch.tensor([[1.0, -math.inf, math.inf, math.nan, torch.finfo(torch.bfloat16).min]],
                     device=DEV).bfloat16()
    hist, lens = ints([[0, 1, 2, 3, 4]]), ints([5])
    same = serving.adjust_logits(z, hist, lens, ints([0]))
    assert torch.equal(same.nan_to_num(5.0, 6.0, 7.0), z.float().nan_to_num(5.0, 6.0, 7.0))
    one = torch.ones(1, device=DEV)
    got = serving.adjust_logits(z, hist, lens, ints([0]), repetition=2 * one, presence=one,
                                allowed=ints([[0b01111]]))[0].tolist()
    assert got[0] == -0.5 and got[1] == -math.inf and got[2] == math.inf
    assert math.isnan(got[3]) and got[4] == -math.inf
    # masked NaN and infinity are -inf
    got = serving.adjust_logits(z, hist, lens, ints([0]), allowed=ints([[1]]))[0].tolist()
    assert got == [1.0] + [-math.inf] * 4
    assert serving.adjust_logits(z[:0], hist[:0], lens[:0], lens[:0]).shape == (0, 5)
    assert torch.equal(serving.adjust_logits(z[:, :1], hist[:, :0], ints([0]), ints([0])).cpu(),
                       torch.ones(1, 1))


# --------------------------------------------------------------------------------- refusals
def test_refusals():
    cache, tables = _filled([20], 2, 64, 16, E4M3)
    q = torch.zeros(1, 4, 64, device=DEV, dtype=torch.bfloat16)
    starts, kv = ints([0, 1]), ints([20])

    def attend(q=q, cache=cache, tables=tables, starts=starts, kv=kv, max_new=1, **kw):
        return serving.paged_attention(q, cache, tables, starts, kv, max_new=max_new, **kw)

    attend()
    bad = [dict(q=q.float()), dict(q=q[:, :3]), dict(q=torch.zeros(1, 4, 32, device=DEV).bfloat16()),
           dict(kv=kv.long()), dict(starts=ints([0, 1, 1])), dict(tables=tables.long()),
           dict(tables=tables[:0]), dict(tables=tables.cpu()), dict(max_new=-1),
           dict(cache=cache._replace(v_pages=cache.v_pages.view(INT8))),
           dict(cache=cache._replace(k_scale=cache.k_scale[:1])),
           dict(cache=cache._replace(k_scale=cache.k_scale.double())),
           dict(cache=cache._replace(k_pages=cache.k_pages.transpose(1, 2))),
           dict(lse=torch.empty(1, 3, device=DEV))]
    for kw in bad:
        with pytest.raises(RuntimeError):
            attend(**kw)
    with pytest.raises(RuntimeError, match="head_dim"):
        c = serving.PagedKV.create(2, 1, 32, page_size=16)
        serving.read_kv(c, ints([0]))
    x = torch.zeros(1, 2, 64, device=DEV, dtype=torch.bfloat16)
    for k, v, t in ((x.float(), x, ints([[0, 0, 0, 1]])), (x, x[:, :1], ints([[0, 0, 0, 1]])),
                    (x, x, ints([0, 0, 0, 1])), (x, x, torch.zeros(1, 4, device=DEV)),
                    (x.cpu(), x, ints([[0, 0, 0, 1]]))):
        with pytest.raises(RuntimeError):
            serving.append_kv(cache, k, v, t)
    with pytest.raises(RuntimeError):
        serving.read_kv(cache, torch.zeros(1, device=DEV))
    for kw in (dict(page_size=48), dict(num_tokens=-1), dict(fresh=ints([1, 1])), dict(fresh=ints([1]).long())):
        a = dict(fresh=ints([1]), page_size=16, num_tokens=1) | kw
        with pytest.raises(RuntimeError):
            serving.plan_step(ints([0]), a["fresh"], tables, ints([0]), ints([1]),
                              page_size=a["page_size"], num_tokens=a["num_tokens"])
    with pytest.raises(RuntimeError, match="4096"):
        n = 4097
        serving.plan_step(ints([0] * n), ints([0] * n), torch.zeros(n, 1, dtype=torch.int32, device=DEV),
                          ints([0]), ints([1]), page_size=16, num_tokens=0)
    z, h, n = torch.zeros(1, 40, device=DEV), ints([[1]]), ints([1])
    for kw in (dict(repetition=torch.ones(2, device=DEV)), dict(presence=torch.ones(1)),
               dict(frequency=torch.ones(1, device=DEV).double()), dict(bias_ids=ints([[1]])),
               dict(allowed=ints([[1]])), dict(bias_ids=ints([[1]]), bias=torch.ones(1, 2, device=DEV)),
               dict(bias_ids=torch.zeros(1, 1025, dtype=torch.int32, device=DEV),
                    bias=torch.zeros(1, 1025, device=DEV))):
        with pytest.raises(RuntimeError):
            serving.adjust_logits(z, h, n, n, **kw)
    with pytest.raises(RuntimeError):
        serving.adjust_logits(z.half(), h, n, n)
    for kw in (dict(page_size=8), dict(dtype=torch.float16), dict(num_pages=0)):
        a = dict(num_pages=1, page_size=16, dtype=E4M3) | kw
        with pytest.raises(ValueError):
            serving.PagedKV.create(a["num_pages"], 1, 64, page_size=a["page_size"], dtype=a["dtype"])


def test_kernels_are_this_librarys():
    cache, tables = _filled([20], 1, 64, 16, E4M3)
    q = torch.zeros(1, 1, 64, device=DEV, dtype=torch.bfloat16)
    before = lib().launch_count()
    serving.paged_attention(q, cache, tables, ints([0, 1]), ints([20]), max_new=1)
    assert lib().launch_count() > before
