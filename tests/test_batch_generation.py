"""Batched generation over the 8-bit paged cache (CPU forms of the serving operators)."""

import json
import math

import pytest
import torch

from nano_megatron_b200.ops import serving

E4M3, INT8 = torch.float8_e4m3fn, torch.int8


def _artifact(tmp_path, kv_heads=2):
    """A tiny random GPT with a tokenizer, as generation sees an artifact."""
    from types import SimpleNamespace

    from nano_megatron_b200.config import config_from_dict
    from nano_megatron_b200.inference.artifact import local_parallel
    from nano_megatron_b200.models.gpt.model import GPTModel
    from nano_megatron_b200.tokenizer import ByteBPETrainingConfig, ByteLevelBPETokenizer

    texts = ["once upon a time there was a little cat who liked to run in the sun. "] * 20
    tok = ByteLevelBPETokenizer.train(texts, ByteBPETrainingConfig(vocab_size=300))
    cfg = config_from_dict({
        "model": {"layers": 3, "hidden_size": 64, "ffn_hidden_size": 128, "heads": 4,
                  "kv_heads": kv_heads, "seq_length": 96, "vocab_size": tok.vocab_size},
        "precision": {"params": "float32", "compute": "float32"},
        "distributed": {"device": "cpu", "backend": "gloo"}})
    torch.manual_seed(3)
    model = GPTModel(cfg.model, parallel=local_parallel()).float().eval()
    with torch.no_grad():   # livelier than the initialisation: scores that differ
        for p in model.parameters():
            if p.dim() == 2:
                p.mul_(4.0)
    return SimpleNamespace(tokenizer=tok, model_config=cfg.model), model


PROMPTS = ["once upon", "a", "the little cat ran in the sun and", "there was a time", "cat cat cat"]
CPU = torch.device("cpu")


def _batch(art, model, prompts=PROMPTS, **kw):
    from nano_megatron_b200.inference import generate_batch

    kw = dict(device=CPU, max_new_tokens=20, temperature=0.0, page_size=16, cache_dtype="int8") | kw
    return generate_batch(art, model, prompts, **kw)


@pytest.mark.parametrize("dtype", [E4M3, INT8])
def test_scores_follow_the_single_decoder_on_the_same_cache(tmp_path, dtype):
    """Same tokens through the single-prompt decoder, attending to the values that the 8-bit
    cache stands for: only the order of fp32 sums differs (1e-4 of the scores' spread)."""
    from nano_megatron_b200.inference import BatchDecoder, KVCacheDecoder

    art, model = _artifact(tmp_path)
    ids = [art.tokenizer.encode(p, add_bos=True, add_eos=False) for p in PROMPTS[:3]]
    dec = BatchDecoder(model, max_requests=3, max_len=64, page_size=16, cache_dtype=dtype)
    singles = [KVCacheDecoder(model, 64) for _ in ids]

    def cached(slot, layer, n):
        at = torch.arange(n)
        slots = dec.tables[slot, at // 16] * 16 + at % 16
        return [t.float() for t in serving.read_kv(dec.caches[layer], slots.int())]

    for slot, single in enumerate(singles):
        plain, calls = single._attend, []

        def attend(q, kc, vc, t0, slot=slot, plain=plain, calls=calls):
            layer = len(calls) % len(dec.caches)
            calls.append(layer)
            return plain(q, *cached(slot, layer, kc.shape[0]), t0)

        single._attend = attend
    pending = {i: p for i, p in enumerate(ids)}
    for step in range(20):
        got = dec.step(pending)
        want = torch.stack([d.forward(pending[i]) for i, d in enumerate(singles)])
        assert (got - want).norm() <= 1e-4 * (want - want.mean(1, keepdim=True)).norm()
        pending = {i: [int(want[i].argmax())] for i in range(3)}
    assert dec.lengths == [d.length for d in singles]


def test_results_do_not_depend_on_the_batch(tmp_path):
    art, model = _artifact(tmp_path)
    for temp in (0.0, 0.9):
        together = _batch(art, model, temperature=temp, top_k=20, seed=5)
        alone = [_batch(art, model, [p], temperature=temp, top_k=20, seed=5)[0] for p in PROMPTS]
        queued = _batch(art, model, temperature=temp, top_k=20, seed=5, max_batch=2)
        tight = _batch(art, model, temperature=temp, top_k=20, seed=5, num_pages=4)
        for a, b, c, d, p in zip(together, alone, queued, tight, PROMPTS):
            assert a.generated_token_ids == b.generated_token_ids == c.generated_token_ids
            assert a.generated_token_ids == d.generated_token_ids
            assert a.prompt == p and a.text.startswith(p)


def test_pages_come_back_and_are_reused(tmp_path):
    from nano_megatron_b200.inference import BatchDecoder

    art, model = _artifact(tmp_path)
    dec = BatchDecoder(model, max_requests=3, max_len=48, num_pages=6, page_size=16)
    first = dec.step({1: list(range(5, 25))})
    dec.step({0: [3] * 33, 1: [7]})
    assert dec.free == 1 == int(dec.free_count) and dec.lengths == [33, 21, 0]
    with pytest.raises(RuntimeError, match="out of pages"):
        dec.step({2: [1] * 17})
    dec.release(0)
    assert dec.free == 4 == int(dec.free_count)
    assert sorted(dec.free_pages[:4].tolist() + dec.tables[1, :2].tolist()) == list(range(6))
    # the same tokens on recycled pages and another slot: the same scores
    again = dec.step({2: list(range(5, 25))})
    torch.testing.assert_close(again, first, rtol=1e-5, atol=1e-5)
    with pytest.raises(ValueError, match="48 positions"):
        dec.step({2: [1] * 29})
    for bad in ({}, {3: [1]}, {0: []}):
        with pytest.raises(ValueError):
            dec.step(bad)


def test_rules_reach_the_sampler(tmp_path):
    from nano_megatron_b200.inference import LogitRules

    art, model = _artifact(tmp_path)
    base = _batch(art, model)
    top = base[0].generated_token_ids[0]
    banned = _batch(art, model, rules=LogitRules(bias={top: -math.inf}))
    assert all(top not in r.generated_token_ids for r in banned)
    only = [11, 12, 40]
    mixed = _batch(art, model, rules=[LogitRules(allowed=only)] + [LogitRules()] * 4)
    assert set(mixed[0].generated_token_ids) <= set(only)
    assert [r.generated_token_ids for r in mixed[1:]] == [r.generated_token_ids for r in base[1:]]
    # a penalty larger than any score difference: no token twice
    distinct = _batch(art, model, rules=LogitRules(presence=1e6))
    assert all(len(set(r.generated_token_ids)) == len(r.generated_token_ids) for r in distinct)
    repeat = _batch(art, model, rules=LogitRules(frequency=-1e6))
    assert all(len(set(r.generated_token_ids)) == 1 for r in repeat)
    fresh = _batch(art, model, rules=LogitRules(repetition=1e6))
    assert [r.generated_token_ids for r in fresh] != [r.generated_token_ids for r in base]


def test_refusals(tmp_path):
    from nano_megatron_b200.inference import LogitRules

    art, model = _artifact(tmp_path)
    assert _batch(art, model, []) == []
    for kw in (dict(cache_dtype="fp4"), dict(max_batch=0), dict(page_size=10), dict(num_pages=1),
               dict(max_new_tokens=96), dict(rules=[LogitRules()]),
               dict(rules=LogitRules(bias={10 ** 6: 1.0})), dict(rules=LogitRules(allowed=[-1]))):
        with pytest.raises(ValueError):
            _batch(art, model, **kw)
    for kw in (dict(repetition=0.0), dict(presence=math.inf), dict(frequency=math.nan)):
        with pytest.raises(ValueError):
            LogitRules(**kw)
    with pytest.raises(TypeError):
        _batch(art, model, [3])


def test_cli_prompts_file(tmp_path, capsys, monkeypatch):
    from nano_megatron_b200.cli import generate as gcli
    from nano_megatron_b200.inference import batch

    art, model = _artifact(tmp_path)
    monkeypatch.setattr(batch, "load_model_for_generation", lambda *a, **k: (art, model, CPU))
    (tmp_path / "p.txt").write_text("once upon\na time\n")
    gcli.main(["--model", "unused", "--prompts-file", str(tmp_path / "p.txt"), "--max-new-tokens", "4",
               "--temperature", "0", "--json", "--repetition-penalty", "1.2", "--cache-dtype", "int8"])
    out = [json.loads(x) for x in capsys.readouterr().out.splitlines()]
    assert [r["prompt"] for r in out] == ["once upon", "a time"]
    assert all(1 <= len(r["generated_token_ids"]) <= 4 for r in out)
    with pytest.raises(SystemExit):
        gcli.main(["--model", "unused"])
    with pytest.raises(SystemExit):
        gcli.main(["--model", "unused", "--prompt", "x", "--prompts-file", "y"])


# ----------------------------------------------------------- the operators' CPU forms
def test_plan_append_read_attend_on_cpu():
    """One step of three requests, by hand: rows land where the plan says and attention is the
    softmax over what the cache stands for."""
    g = torch.Generator().manual_seed(0)
    cache = serving.PagedKV.create(6, 1, 8, page_size=16, dtype=INT8, device="cpu")
    tables = torch.full((3, 3), -1, dtype=torch.int32)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32)

    plan = serving.plan_step(ints([0, 0, 0]), ints([20, 0, 3]), tables, ints([5, 4, 3, 2, 1, 0]),
                             ints([6]), page_size=16, num_tokens=25)
    assert plan.q_starts.tolist() == [0, 20, 20, 23] and plan.kv_lens.tolist() == [20, 0, 3]
    assert tables.tolist() == [[0, 1, -1], [-1, -1, -1], [2, -1, -1]]
    assert plan.slots.tolist() == list(range(20)) + [32, 33, 34, -1, -1]
    assert plan.touched.tolist()[:3] == [[0, 0, 0, 16], [1, 16, 0, 4], [2, 20, 0, 3]]
    assert int(plan.free_count) == 3
    x = torch.randn(25, 2, 1, 8, generator=g)
    serving.append_kv(cache, x[:, 0], x[:, 1], plan.touched)
    k, v = serving.read_kv(cache, plan.slots)
    assert (k[:23].float() - x[:23, 0]).abs().max() <= x.abs().max() / 64 / 2 + 1e-6
    assert k[23:].abs().max() == 0
    q = torch.randn(25, 2, 8, generator=g)
    lse = torch.empty(25, 2)
    o = serving.paged_attention(q, cache, tables, plan.q_starts, plan.kv_lens, max_new=20, lse=lse)
    for r, (first, last) in {19: (0, 20), 4: (0, 5), 22: (20, 23), 20: (20, 21)}.items():
        s = q[r] @ k[first:last, 0].float().T / math.sqrt(8)
        torch.testing.assert_close(o[r], torch.softmax(s, -1) @ v[first:last, 0].float())
        torch.testing.assert_close(lse[r], torch.logsumexp(s, -1) / math.log(2))
    assert o[23:].abs().max() == 0 and bool(torch.isinf(lse[23:]).all())
