"""Edges of batched generation and of the serving operators' CPU forms."""

import math

import pytest
import torch
from test_batch_generation import CPU, PROMPTS, _artifact, _batch  # noqa: F401


def _state(dec):
    return (list(dec.lengths), dec.free, int(dec.free_count), dec.free_pages[:dec.free].tolist())


@pytest.mark.parametrize("bad", [-1, 10 ** 6, "vocab"])
def test_token_ids_outside_the_vocabulary_are_refused(tmp_path, bad):
    """Refused on the host, before anything of the step is planned or launched."""
    from nano_megatron_b200.inference import BatchDecoder

    _, model = _artifact(tmp_path)
    dec = BatchDecoder(model, max_requests=2, max_len=32, page_size=16)
    dec.step({0: [5, 6]})
    before, tables = _state(dec), dec.tables.clone()
    with pytest.raises(ValueError, match="vocabulary"):
        dec.step({0: [3], 1: [4, model.original_vocab_size if bad == "vocab" else bad, 7]})
    assert _state(dec) == before and torch.equal(dec.tables, tables)


def test_an_empty_allowed_set_is_refused():
    from nano_megatron_b200.inference import LogitRules

    for nothing in ((), [], set(), iter(())):
        with pytest.raises(ValueError, match="allowed"):
            LogitRules(allowed=nothing)


def test_allowed_may_be_any_iterable(tmp_path):
    """An iterator is not used up by the checks of its ids."""
    from nano_megatron_b200.inference import LogitRules

    art, model = _artifact(tmp_path)
    want = _batch(art, model, rules=LogitRules(allowed=[11, 12, 40]))
    got = _batch(art, model, rules=LogitRules(allowed=iter([11, 12, 40])))
    assert [r.generated_token_ids for r in got] == [r.generated_token_ids for r in want]
    assert {t for r in got for t in r.generated_token_ids} <= {11, 12, 40}


@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_rules_that_leave_no_token_stop_generation(tmp_path, temperature):
    from nano_megatron_b200.inference import LogitRules

    art, model = _artifact(tmp_path)
    rules = LogitRules(allowed=[7, 9], bias={7: -math.inf, 9: -math.inf})
    with pytest.raises(RuntimeError, match="no token"):
        _batch(art, model, rules=rules, temperature=temperature)


@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_biases_of_nan_or_infinity_are_refused(value):
    from nano_megatron_b200.inference import LogitRules

    with pytest.raises(ValueError, match="bias"):
        LogitRules(bias={3: 1.0, 4: value})
    assert LogitRules(bias={3: -math.inf}).bias == {3: -math.inf}


def narrow_table_plans(device):
    """Plans whose tables have no room for all new pages, with more free pages than needed."""
    from nano_megatron_b200.ops import serving

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=device)

    for contexts, news, width, missing in (([0], [40], 1, 2), ([16], [1], 1, 1), ([40, 3], [9, 60], 2, 3),
                                           ([5, 0, 31], [30, 100, 1], 3, 4), ([64], [5], 2, 1)):
        tables = torch.full((len(contexts), width), -1, dtype=torch.int32, device=device)
        pages = iter(range(100, 200))
        for b, c in enumerate(contexts):
            for lp in range(min(width, -(-c // 16))):
                tables[b, lp] = next(pages)
        held = int((tables >= 0).sum())
        p = serving.plan_step(ints(contexts), ints(news), tables, ints(list(range(20))), ints([20]),
                              page_size=16, num_tokens=sum(news))
        yield contexts, missing, held, tables.cpu(), p


def check_narrow_table_plans(device):
    for contexts, missing, held, tables, p in narrow_table_plans(device):
        # every page that left the free list is in a table
        assert int((tables >= 0).sum()) - held == 20 - int(p.free_count)
        assert int(p.missing) == missing, contexts
        starts, slots = p.q_starts.tolist(), p.slots.tolist()
        for b, c in enumerate(contexts):
            for row in range(starts[b], starts[b + 1]):
                pos = c + row - starts[b]
                page = int(tables[b, pos // 16]) if pos // 16 < tables.shape[1] else -1
                assert slots[row] == (page * 16 + pos % 16 if page >= 0 else -1)


def test_plan_keeps_the_pages_that_a_narrow_table_has_no_room_for():
    check_narrow_table_plans("cpu")


def lengths_beyond_the_table(device, D=64):
    """(q, cache, narrow tables, wide tables, starts, lens): requests longer than their tables'
    columns; the wide tables have the missing pages as -1."""
    from nano_megatron_b200.ops import serving

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=device)

    g = torch.Generator().manual_seed(1)
    cache = serving.PagedKV.create(12, 2, D, page_size=16, dtype=torch.int8, device=device)
    k, v = (torch.randn(192, 2, D, generator=g).bfloat16().to(device) for _ in range(2))
    serving.append_kv(cache, k, v, ints([[i, 16 * i, 0, 16] for i in range(12)]))
    narrow = ints([[0, 1, 2], [3, 4, 5], [6, 7, 8], [9, 10, 11]])
    wide = torch.cat([narrow, torch.full_like(narrow, -1)], 1)
    lens, rows = [70, 49, 50, 96], [40, 1, 3, 60]      # 48 positions have a page
    starts = [0, 40, 41, 44, 104]
    q = torch.randn(104, 4, D, generator=g).bfloat16().to(device)
    return q, cache, narrow, wide, ints(starts), ints(lens), rows


def test_attention_sees_what_a_narrow_table_holds():
    from nano_megatron_b200.ops import serving

    q, cache, narrow, wide, starts, lens, rows = lengths_beyond_the_table("cpu")
    got = [torch.empty(q.shape[:2]) for _ in range(2)]
    a, b = (serving.paged_attention(q, cache, t, starts, lens, max_new=max(rows), lse=z)
            for t, z in zip((narrow, wide), got))
    # (another width may add up in another order: fp32 sums of 64 products of scores up to 8)
    torch.testing.assert_close(a, b, rtol=2 ** -7, atol=2 ** -16)
    torch.testing.assert_close(*got, rtol=0, atol=2 ** -16)
    assert a.float().abs().amax((1, 2)).min() > 0


def test_a_step_that_fails_changes_nothing(tmp_path, monkeypatch):
    """An error in the middle of the layers: lengths and pages stay, and the step can be repeated."""
    from nano_megatron_b200.inference import BatchDecoder, batch

    _, model = _artifact(tmp_path)
    dec, other = (BatchDecoder(model, max_requests=2, max_len=64, page_size=16) for _ in range(2))
    first, second = {0: list(range(5, 20))}, {0: [7, 8, 9], 1: list(range(30, 55))}
    dec.step(first)
    other.step(first)
    before = _state(dec)
    plain, calls = batch.F.swiglu_act, []

    def failing(*a):
        calls.append(1)
        if len(calls) == 2:
            raise RuntimeError("out of memory")
        return plain(*a)

    monkeypatch.setattr(batch.F, "swiglu_act", failing)
    with pytest.raises(RuntimeError, match="out of memory"):
        dec.step(second)
    monkeypatch.setattr(batch.F, "swiglu_act", plain)
    assert _state(dec) == before
    assert torch.equal(dec.step(second), other.step(second))
    assert _state(dec) == _state(other)
    dec.release(0)
    dec.release(1)
    assert dec.free == int(dec.free_count) == dec.num_pages
    assert sorted(dec.free_pages.tolist()) == list(range(dec.num_pages))


@pytest.mark.parametrize("page_size", [0, -16])
def test_page_sizes_below_one_are_refused(tmp_path, page_size):
    art, model = _artifact(tmp_path)
    with pytest.raises(ValueError, match="page_size"):
        _batch(art, model, page_size=page_size)


def _cli(tmp_path, monkeypatch, *args):
    from nano_megatron_b200.cli import generate as gcli
    from nano_megatron_b200.inference import batch

    art, model = _artifact(tmp_path)
    monkeypatch.setattr(batch, "load_model_for_generation", lambda *a, **k: (art, model, CPU))
    gcli.main(["--model", "unused", "--max-new-tokens", "2", "--temperature", "0", *args])


def test_prompts_file_is_split_at_line_ends_only(tmp_path, monkeypatch, capsys):
    """Form feeds, separators and the like belong to a prompt: one result per line of the file."""
    import json

    lines = ["a\x0cb", "c d", "e\x1cf\x85g", "", "h"]
    (tmp_path / "p.txt").write_bytes("\r\n".join(lines).encode())
    _cli(tmp_path, monkeypatch, "--prompts-file", str(tmp_path / "p.txt"), "--json")
    out = [json.loads(x) for x in capsys.readouterr().out.split("\n") if x]
    assert [r["prompt"] for r in out] == lines
    (tmp_path / "p.txt").write_text("a\nb\n\n")
    _cli(tmp_path, monkeypatch, "--prompts-file", str(tmp_path / "p.txt"), "--json")
    assert [json.loads(x)["prompt"] for x in capsys.readouterr().out.split("\n") if x] == ["a", "b", ""]


@pytest.mark.parametrize("option", [["--repetition-penalty", "1.2"], ["--presence-penalty", "0.5"],
                                    ["--frequency-penalty", "0.5"], ["--cache-dtype", "int8"],
                                    ["--max-batch", "2"]])
def test_options_of_batches_are_refused_for_one_prompt(tmp_path, monkeypatch, capsys, option):
    with pytest.raises(SystemExit):
        _cli(tmp_path, monkeypatch, "--prompt", "x", *option)
    assert option[0] in capsys.readouterr().err


def test_recomputing_the_prefix_is_refused_for_batches(tmp_path, monkeypatch, capsys):
    (tmp_path / "p.txt").write_text("a\n")
    with pytest.raises(SystemExit):
        _cli(tmp_path, monkeypatch, "--prompts-file", str(tmp_path / "p.txt"), "--no-kv-cache")
    assert "--no-kv-cache" in capsys.readouterr().err
    _cli(tmp_path, monkeypatch, "--prompts-file", str(tmp_path / "p.txt"), "--kv-cache")


def test_options_of_batches_reach_them(tmp_path, monkeypatch):
    from nano_megatron_b200.cli import generate as gcli

    seen = {}
    monkeypatch.setattr(gcli, "generate_batch_from_artifact", lambda *a, **k: seen.update(k) or [])
    (tmp_path / "p.txt").write_text("a\n")
    args = ["--model", "unused", "--prompts-file", str(tmp_path / "p.txt")]
    gcli.main(args)
    assert (seen["max_batch"], seen["cache_dtype"], seen["rules"].empty) == (64, "e4m3", True)
    gcli.main(args + ["--max-batch", "3", "--cache-dtype", "int8", "--presence-penalty", "0.5"])
    assert (seen["max_batch"], seen["cache_dtype"], seen["rules"].presence) == (3, "int8", 0.5)


def test_a_text_is_not_a_list_of_prompts(tmp_path):
    art, model = _artifact(tmp_path)
    with pytest.raises(TypeError, match="prompts"):
        _batch(art, model, "once upon")
