"""Edges of the batched-serving kernels against plain 64-bit computations.

Tolerances as in ``test_serving_ops_gpu``: attention rounds its output once to bf16 (2^-8 of the
value) and each probability to f16 (under 2^-10 of the row's largest output in sum).
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from test_serving_ops_gpu import DEV, E4M3, INT8, _cache, _oracle, ints  # noqa: E402

from nano_megatron_b200.ops import check_status, serving  # noqa: E402

BOUND = 2.0 ** -8 + 2.0 ** -10


def _compare(q, cache, tables, starts, kv, max_new):
    lse = torch.empty(q.shape[:2], device=DEV)
    got = serving.paged_attention(q, cache, tables, ints(starts), ints(kv), max_new=max_new, lse=lse)
    torch.cuda.synchronize()
    check_status(torch.device(DEV))
    want, want_lse = _oracle(q, cache, tables, starts, kv, q.shape[2] ** -0.5)
    top = want.abs().amax(-1, keepdim=True)
    worst = ((got.double() - want).abs() / top.clamp(min=1e-300)).max().item()
    assert worst <= BOUND, worst
    inf = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse), inf)
    assert bool(((lse.double() - want_lse)[~inf].abs() <= 2.0 ** -16 + want_lse[~inf].abs() * 2.0 ** -18).all())


def _rows_and_cache(n, new, Hq, H, D, page, dtype, special):
    """One request of `n` keys, the last `new` of them new. Queries point along one direction, so
    that ``special(k, v, direction)`` can give single keys a chosen score; values are normal."""
    g = torch.Generator(device=DEV).manual_seed(n + new)
    u = torch.nn.functional.normalize(torch.randn(D, generator=g, device=DEV), dim=0)
    q = (4.0 * u + 0.1 * torch.randn(new, Hq, D, generator=g, device=DEV)).bfloat16()
    k = torch.randn(n, H, D, generator=g, device=DEV)
    k -= (k @ u)[..., None] * u                          # ordinary keys: scores near zero
    v = torch.randn(n, H, D, generator=g, device=DEV)
    special(k, v, u)
    pages = -(-n // page)
    cache = _cache(pages + 1, H, D, page, dtype)
    ids = torch.randperm(pages, generator=torch.Generator().manual_seed(n)).tolist()
    serving.append_kv(cache, k.bfloat16(), v.bfloat16(),
                      ints([[p, i * page, 0, min(page, n - i * page)] for i, p in enumerate(ids)]))
    return q, cache, ints([ids])


# (keys, new rows, query heads, kv heads): one row on one block and on many, a few rows, 16-row
# units, prompts in the other kernel
SHAPES = [(300, 1, 4, 2), (5000, 1, 4, 1), (200, 3, 2, 2), (150, 5, 8, 2), (400, 130, 4, 2)]


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 64)])
@pytest.mark.parametrize("n,new,Hq,H", SHAPES)
@pytest.mark.parametrize("power", [16, 20, 24, 30])
def test_value_outlier_of_low_weight(dtype, D, page, n, new, Hq, H, power):
    """One visible value of 2^power whose key has a score of about -90 (a weight under 1e-25): its page's
    scale is large, yet the other pages decide the result."""
    def special(k, v, u):
        k[7], v[7, :, 3] = -22.5 * D ** 0.5 * u, 2.0 ** power

    q, cache, tables = _rows_and_cache(n, new, Hq, H, D, page, dtype, special)
    _compare(q, cache, tables, [0, new], [n], new)


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 64)])
@pytest.mark.parametrize("n,new,Hq,H", [s for s in SHAPES if s[1] > 1])
@pytest.mark.parametrize("power", [16, 24, 30])
def test_value_outlier_hidden_by_causality(dtype, D, page, n, new, Hq, H, power):
    """The last position's value is 2^power: only the last row sees it, the others share its page's
    scale."""
    def special(k, v, u):
        v[-1, :, 3] = 2.0 ** power

    q, cache, tables = _rows_and_cache(n, new, Hq, H, D, page, dtype, special)
    _compare(q, cache, tables, [0, new], [n], new)


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 64)])
@pytest.mark.parametrize("n,new,Hq,H", SHAPES)
@pytest.mark.parametrize("bits", [12, 20, 30, 40, 60])
def test_key_that_takes_all_the_weight_but_has_no_value(dtype, D, page, n, new, Hq, H, bits):
    """A first key whose score is `bits` powers of two above the others and whose value is zero:
    the result is the others' sum, at 2^-bits of the largest probability."""
    def special(k, v, u):
        k[0], v[0] = bits * math.log(2.0) / 4.0 * D ** 0.5 * u, 0.0

    q, cache, tables = _rows_and_cache(n, new, Hq, H, D, page, dtype, special)
    _compare(q, cache, tables, [0, new], [n], new)


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 64)])
@pytest.mark.parametrize("n,new,Hq,H", SHAPES)
def test_values_of_zero(dtype, D, page, n, new, Hq, H):
    def special(k, v, u):
        v.zero_()

    q, cache, tables = _rows_and_cache(n, new, Hq, H, D, page, dtype, special)
    o = serving.paged_attention(q, cache, tables, ints([0, new]), ints([n]), max_new=new)
    assert o.abs().max() == 0


def test_generation_stops_at_a_kernels_status():
    """A kernel that gave up (here: its status word, set by hand) leaves its output unfinished:
    nothing is sampled from it."""
    from test_batch_generation_gpu import _model

    from nano_megatron_b200.inference import generate_batch
    from nano_megatron_b200.ops import status_word

    model, cfg = _model(DEV, torch.bfloat16, 4, 2)

    class Numbers:
        eos_token_id = 8191

        def encode(self, text, add_bos, add_eos):
            return [int(x) for x in text.split()]

        def decode(self, ids, skip_special_tokens):
            return " ".join(map(str, ids))

    from types import SimpleNamespace
    art = SimpleNamespace(tokenizer=Numbers(), model_config=cfg.model)
    word = status_word(torch.device(DEV))
    kw = dict(device=torch.device(DEV), max_new_tokens=2, temperature=0.0)
    try:
        word.fill_(0x201)
        with pytest.raises(RuntimeError, match="attention wait timed out"):
            generate_batch(art, model, ["1 2 3"], **kw)
    finally:
        word.zero_()
    assert len(generate_batch(art, model, ["1 2 3"], **kw)[0].generated_token_ids) == 2


def test_a_step_of_too_many_key_tiles_has_its_own_status():
    """Groups over 128 heads always take the decode kernel, which counts its key tiles in 31 bits."""
    from nano_megatron_b200.ops import status_word

    cache = serving.PagedKV.create(1, 1, 64, page_size=128)
    n, heads, keys = 16384, 130, 300 * 1024
    q = torch.zeros(n, heads, 64, device=DEV, dtype=torch.bfloat16)
    tables = torch.zeros(1, keys // 128, dtype=torch.int32, device=DEV)
    word = status_word(torch.device(DEV))
    try:
        serving.paged_attention(q, cache, tables, ints([0, n]), ints([keys]), max_new=n)
        with pytest.raises(RuntimeError, match="key tiles"):
            check_status(torch.device(DEV))
    finally:
        word.zero_()


def test_more_biases_than_the_kernel_takes_are_refused_before_the_first_step():
    from types import SimpleNamespace

    from test_batch_generation_gpu import _model

    from nano_megatron_b200.inference import LogitRules, generate_batch
    from nano_megatron_b200.ops import lib

    model, cfg = _model(DEV, torch.bfloat16, 4, 2)
    words = SimpleNamespace(eos_token_id=8191, encode=lambda t, add_bos, add_eos: [1, 2, 3],
                            decode=lambda ids, skip_special_tokens: "")
    art = SimpleNamespace(tokenizer=words, model_config=cfg.model)
    kw = dict(device=torch.device(DEV), max_new_tokens=2, temperature=0.0)
    before = lib().launch_count()
    with pytest.raises(ValueError, match=str(serving.MAX_BIAS)):
        generate_batch(art, model, ["a", "b"],
                       rules=[LogitRules(), LogitRules(bias={t: 0.5 for t in range(serving.MAX_BIAS + 1)})], **kw)
    assert lib().launch_count() == before
    most = LogitRules(bias={t: 100.0 for t in range(serving.MAX_BIAS)})
    assert max(generate_batch(art, model, ["a"], rules=most, **kw)[0].generated_token_ids) < serving.MAX_BIAS


def test_plan_keeps_the_pages_that_a_narrow_table_has_no_room_for():
    from test_batch_generation_edges import check_narrow_table_plans

    check_narrow_table_plans(DEV)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("most", [1, 3, 60])
def test_attention_sees_what_a_narrow_table_holds(D, most):
    """Lengths past a table's columns are missing pages, not shorter requests: a row's position stays."""
    from test_batch_generation_edges import lengths_beyond_the_table

    q, cache, narrow, wide, starts, lens, rows = lengths_beyond_the_table(DEV, D)
    pick = [i for i, r in enumerate(rows) if r <= most]
    q = torch.cat([q[starts[i]:starts[i + 1]] for i in pick])
    starts = [0]
    for i in pick:
        starts.append(starts[-1] + rows[i])
    got = serving.paged_attention(q, cache, narrow[pick], ints(starts), lens[pick].contiguous(), max_new=most)
    want, _ = _oracle(q, cache, wide[pick], starts, lens[pick].tolist(), D ** -0.5)
    top = want.abs().amax(-1, keepdim=True)
    assert float(top.min()) > 0
    assert bool(((got.double() - want).abs() <= top * BOUND).all())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("ctx", [0, 37, 3000])
@pytest.mark.parametrize("zero", [False, True])
def test_too_small_a_max_new_costs_speed_only(D, ctx, zero):
    """Several rows although `max_new` says one: NaN still reaches only the rows that see it."""
    from test_serving_ops_gpu import _filled

    n = 4
    cache, tables = _filled([ctx + n], 2, D, 16, E4M3)
    if zero:
        cache.v_pages.view(torch.uint8).zero_()
    page, off = int(tables[0, (ctx + 2) // 16]), (ctx + 2) % 16
    cache.v_pages.view(torch.uint8)[page, 0, off, 5] = 0xFF
    cache.k_pages.view(torch.uint8)[page, 1, off, 3] = 0x7F
    q = torch.randn(n, 8, D, device=DEV).bfloat16()
    got, want = (serving.paged_attention(q, cache, tables, ints([0, n]), ints([ctx + n]), max_new=m)
                 for m in (1, n))
    assert torch.equal(got.isnan(), want.isnan()) and not bool(got[:2].isnan().any())
    top = want.nan_to_num(0.0).double().abs().amax(-1, keepdim=True)
    assert bool(((got.double() - want.double()).nan_to_num(0.0).abs() <= 2 * BOUND * top).all())


@pytest.mark.parametrize("most", [2, 70])
def test_rows_before_the_first_request_are_zero(most):
    """A part of a plan: ``q_starts[1:]`` starts past row 0. Rows of nobody are 0, as on the CPU."""
    cache = serving.PagedKV.create(8, 2, 64, page_size=32, dtype=INT8)
    x = torch.randn(2 * most + 5, 3, 2, 64, device=DEV).bfloat16()
    k, v, q = x.unbind(1)
    tables = torch.full((3, 4), -1, dtype=torch.int32, device=DEV)
    plan = serving.plan_step(ints([0, 0, 0]), ints([3, 2, 2 * most]), tables, ints(list(range(8))), ints([8]),
                             page_size=32, num_tokens=2 * most + 5)
    serving.append_kv(cache, k, v, plan.touched)
    torch.full((64 << 20,), math.nan, device=DEV)        # what a new tensor would find in its memory
    lse = torch.zeros(2 * most + 5, 2, device=DEV)
    got = serving.paged_attention(q, cache, tables[1:], plan.q_starts[1:], plan.kv_lens[1:],
                                  max_new=2 * most, lse=lse)
    assert got[:3].abs().max() == 0 and bool((lse[:3] == -math.inf).all())
    want = serving.paged_attention(q, cache, tables, plan.q_starts, plan.kv_lens, max_new=2 * most)
    assert float(((got[3:] - want[3:]).abs().double() / want[3:].abs().amax(-1, keepdim=True)).max()) <= 2 * BOUND


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_weights_that_the_kernels_do_not_take_are_refused_at_once(dtype):
    from test_batch_generation_gpu import _model

    from nano_megatron_b200.inference import BatchDecoder

    model, _ = _model(DEV, dtype, 4, 2)
    with pytest.raises(ValueError, match="bfloat16"):
        BatchDecoder(model, max_requests=1, max_len=16)


def test_single_prompt_decoding_of_bf16_weights():
    """The single-prompt decoder next to the batch, on weights in bf16: 6 % of the scores' spread,
    as for the batch against fp32."""
    from test_batch_generation_gpu import _model

    from nano_megatron_b200.inference import BatchDecoder, KVCacheDecoder

    model, _ = _model(DEV, torch.bfloat16, 4, 2)
    cpu, _ = _model("cpu", torch.float32, 4, 2)
    cpu.load_state_dict({k: v.float().cpu() for k, v in model.state_dict().items()})
    ids = torch.randint(0, 8192, (120,), generator=torch.Generator().manual_seed(0)).tolist()
    single, batch = KVCacheDecoder(model, 130), BatchDecoder(model, max_requests=1, max_len=130)
    exact = KVCacheDecoder(cpu, 130)
    for part in (ids[:100], ids[100:]):
        want = exact.forward(part)
        spread = (want - want.mean()).norm()
        for got in (single.forward(part), batch.step({0: part})[0]):
            assert float((got.float().cpu() - want).norm()) <= 0.06 * float(spread)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_repetition_at_the_ends_of_its_range(dtype):
    """Scores of seen tokens: within 1.5 ulp of the quotient (one rounded reciprocal, one rounded
    product) and 0.5 of the product, whatever the repetition."""
    rep = torch.tensor([1.1, 1.3, 0.7, 3.0, 1e-39, 2.0 ** -126, 1e38, 3e38])
    B, V = len(rep), 1000
    z = torch.randn(B, V, generator=torch.Generator().manual_seed(0)).to(dtype)
    z[4:6] *= 1e-3                                       # quotients within fp32
    z[6:] *= 1e37
    hist = torch.arange(V).expand(B, V).int().to(DEV)
    got = serving.adjust_logits(z.to(DEV), hist, ints([V] * B), ints([V] * B), repetition=rep.to(DEV)).cpu()
    f, r = z.double(), rep[:, None].double()
    want = torch.where(f > 0, f / r, f * r)
    over = want.abs() >= 2.0 ** 128
    assert torch.equal(got.isinf(), over) and not bool(got.isnan().any())
    got, want = got.masked_fill(over, 0.0), want.masked_fill(over, 0.0)
    ulp = torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=2.0 ** -126))) - 23)
    assert bool(((got.double() - want).abs() <= torch.where(f > 0, 1.5, 0.5) * ulp).all())


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("D,Hq,H", [(64, 4, 4), (128, 8, 2)])
@pytest.mark.parametrize("most", [1, 6, 150])
def test_a_step_in_a_graph_follows_its_lengths(dtype, D, Hq, H, most):
    """Plan, cache write, read, attention and logit rules captured once and replayed with other
    lengths, rows and histories: as the same calls made one by one."""
    B, page, V, T = 5, 32, 3000, 5 * most
    g = torch.Generator().manual_seed(most)

    def make(seed):
        cache = _cache(200, H, D, page, dtype)
        tables = torch.full((B, 30), -1, dtype=torch.int32, device=DEV)
        order = torch.randperm(200, generator=torch.Generator().manual_seed(seed)).int().to(DEV)
        return cache, tables, order, ints([200])

    context, new = ints([0] * B), ints([0] * B)
    q, k, v = (torch.zeros(T, h, D, device=DEV, dtype=torch.bfloat16) for h in (Hq, H, H))
    logits, history = torch.zeros(B, V, device=DEV), torch.zeros(B, 700, dtype=torch.int32, device=DEV)
    prompts, rep = ints([3] * B), torch.full((B,), 1.2, device=DEV)

    def step(cache, tables, free, count):
        p = serving.plan_step(context, new, tables, free, count, page_size=page, num_tokens=T)
        serving.append_kv(cache, k, v, p.touched)
        o = serving.paged_attention(q, cache, tables, p.q_starts, p.kv_lens, max_new=most)
        z = serving.adjust_logits(logits, history, p.kv_lens, prompts, repetition=rep, presence=rep)
        return (o, z, *serving.read_kv(cache, p.slots), *p)

    graphed, eager = make(1), make(1)
    spare = make(2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*spare)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*graphed)
    lens = [0] * B
    for turn in range(4):
        adds = [int(torch.randint(1 if turn else 0, most + 1, (1,), generator=g)) for _ in range(B)]
        adds[turn % B] = most
        context.copy_(ints(lens))
        new.copy_(ints(adds))
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g))
        logits.copy_(torch.randn(B, V, generator=g))
        history.copy_(torch.randint(0, V, (B, 700), generator=g))
        graph.replay()
        want = step(*eager)
        for a, b in zip(out, want):
            assert torch.equal(a.nan_to_num(3.0) if a.is_floating_point() else a,
                               b.nan_to_num(3.0) if b.is_floating_point() else b)
        for a, b in zip((*graphed[0], graphed[1]), (*eager[0], eager[1])):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        for case in (graphed, eager):
            case[3].copy_(want[-2])                      # free_count
        lens = [a + b for a, b in zip(lens, adds)]
    check_status(torch.device(DEV))


@pytest.mark.parametrize("scale", [-0.3, 0.0, 1e-6])
@pytest.mark.parametrize("contexts,news", [([100, 37], [1, 1]), ([100, 37], [5, 3]), ([300, 200], [200, 90])])
@pytest.mark.parametrize("dtype", [E4M3, INT8])
def test_softmax_scales_of_zero_and_below(scale, contexts, news, dtype):
    from test_serving_ops_gpu import _filled

    cache, tables = _filled(contexts, 2, 64, 16, dtype)
    starts = [0, news[0], sum(news)]
    q = torch.randn(sum(news), 8, 64, device=DEV).bfloat16()
    got = serving.paged_attention(q, cache, tables, ints(starts), ints(contexts), max_new=max(news),
                                  softmax_scale=scale)
    want, _ = _oracle(q, cache, tables, starts, contexts, scale)
    top = want.abs().amax(-1, keepdim=True)
    assert bool(((got.double() - want).abs() <= top * BOUND).all())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G", [48, 65, 96, 128, 129, 200])
@pytest.mark.parametrize("new", [1, 3])
def test_wide_groups(D, G, new):
    """More heads of a group than a prompt's row tile halves, fills, and holds."""
    from test_serving_ops_gpu import _check

    _check([150, 33, 64], [new, 1, new], 2 * G, 2, D, 32, E4M3)


def test_more_requests_than_a_plan_takes_are_refused_at_once():
    from test_batch_generation_gpu import _model

    from nano_megatron_b200.inference import BatchDecoder

    model, _ = _model(DEV, torch.bfloat16, 4, 2)
    with pytest.raises(ValueError, match=str(serving.MAX_REQUESTS)):
        BatchDecoder(model, max_requests=serving.MAX_REQUESTS + 1, max_len=16, num_pages=1)
    dec = BatchDecoder(model, max_requests=serving.MAX_REQUESTS, max_len=16, page_size=16, num_pages=1)
    assert bool(dec.step({serving.MAX_REQUESTS - 1: [5]}).isfinite().all())


def test_rows_without_keys_and_too_small_a_max_new():
    """Rows that see nothing among several of a request, although `max_new` says one: 0, not NaN."""
    cache = serving.PagedKV.create(4, 1, 64, page_size=16)
    x = torch.randn(20, 2, 1, 64, device=DEV).bfloat16()
    serving.append_kv(cache, x[:, 0], x[:, 1], ints([[0, 0, 0, 16], [1, 16, 0, 4]]))
    q = torch.randn(6, 2, 64, device=DEV).bfloat16()
    for tables, lens, hidden in (([[0, 1]], [4], 2), ([[-1, 1]], [20], 1), ([[-1, -1]], [20], 6)):
        lse = torch.zeros(6, 2, device=DEV)
        got = serving.paged_attention(q, cache, ints(tables), ints([0, 6]), ints(lens), max_new=1, lse=lse)
        assert got[:hidden].abs().max() == 0 and bool((lse[:hidden] == -math.inf).all())
        want, _ = _oracle(q, cache, ints(tables), [0, 6], lens, 0.125)
        top = want.abs().amax(-1, keepdim=True)
        assert bool(((got.double() - want).abs() <= top * BOUND).all())


@pytest.mark.parametrize("rep", [2e-39, 2.0 ** 127])
@pytest.mark.parametrize("V", [700, 20001])
def test_all_rules_with_a_repetition_out_of_the_normal_range(rep, V):
    """The other rules around it: penalties, mask, biases, tokens that do not occur."""
    from test_serving_ops_gpu import _logits_oracle

    g = torch.Generator().manual_seed(V)
    z = torch.randn(2, V, generator=g) * (1e-2 if rep < 1 else 1.0)
    hist = torch.randint(0, V, (2, 300), generator=g).int()
    lens, prompts = [300, 100], [150, 0]
    rep, pre, freq = torch.full((2,), rep), torch.tensor([0.3, 0.1]), torch.tensor([0.0, 0.2])
    z = torch.where((torch.rand(2, V, generator=g) < 0.5) | (rep[:, None] < 1), z, z * 1e-30)
    z[z < 0] *= 1e-10                                     # products within fp32
    ids, bias = torch.randint(0, V, (2, 9), generator=g).int(), torch.randn(2, 9, generator=g)
    ids[:, :4] = hist[:, :4]
    allowed = torch.randint(-2 ** 31, 2 ** 31 - 1, (2, (V + 31) // 32), generator=g).int()
    got = serving.adjust_logits(z.to(DEV), hist.to(DEV), ints(lens), ints(prompts),
                                **{k: t.to(DEV) for k, t in dict(repetition=rep, presence=pre, frequency=freq,
                                                                 bias_ids=ids, bias=bias, allowed=allowed).items()}).cpu()
    want = _logits_oracle(z, hist, lens, prompts, rep, pre, freq, ids, bias, allowed)
    assert torch.equal(torch.isinf(got), torch.isinf(want))
    ok = ~torch.isinf(want)
    # a quotient or product, up to two penalties and a few biases: an ulp or so of the largest of them each
    err, size = (got.double() - want)[ok].abs(), want[ok].abs() + 16.0
    assert bool((err <= 4 * size * 2.0 ** -23).all())
