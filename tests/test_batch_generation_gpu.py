"""Batched generation on the GPU: the sm_100a serving kernels in a whole model."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(device, dtype, heads, kv_heads):
    from nano_megatron_b200.config import config_from_dict
    from nano_megatron_b200.inference.artifact import local_parallel
    from nano_megatron_b200.models.gpt.model import GPTModel

    cfg = config_from_dict({
        "model": {"layers": 3, "hidden_size": 512, "ffn_hidden_size": 1376, "heads": heads,
                  "kv_heads": kv_heads, "seq_length": 512, "vocab_size": 8192},
        "precision": {"params": "float32", "compute": "float32"},
        "distributed": {"device": "cpu", "backend": "gloo"}})
    torch.manual_seed(1)
    return GPTModel(cfg.model, parallel=local_parallel()).to(dtype=dtype, device=device).eval(), cfg


@pytest.mark.parametrize("heads,kv_heads", [(8, 8), (4, 2)])
@pytest.mark.parametrize("codes", [torch.float8_e4m3fn, torch.int8])
def test_scores_match_the_cpu_form(heads, kv_heads, codes):
    """Prompts of different lengths together, then single tokens. bf16 activations (2^-9 each,
    some thirty roundings in a row) against fp32: 6 % of the scores' spread."""
    from nano_megatron_b200.inference import BatchDecoder
    from nano_megatron_b200.ops import check_status, lib

    gpu, _ = _model("cuda", torch.bfloat16, heads, kv_heads)
    cpu, _ = _model("cpu", torch.float32, heads, kv_heads)
    cpu.load_state_dict({k: v.float().cpu() for k, v in gpu.state_dict().items()})
    decs = [BatchDecoder(m, max_requests=4, max_len=400, page_size=32, cache_dtype=codes)
            for m in (gpu, cpu)]
    g = torch.Generator().manual_seed(0)
    lens = [300, 1, 40, 129]
    pending = {i: torch.randint(0, 8192, (n,), generator=g).tolist() for i, n in enumerate(lens)}
    before = lib().launch_count()
    for _ in range(4):
        got, want = (d.step(pending) for d in decs)
        got = got.float().cpu()
        spread = (want - want.mean(1, keepdim=True)).norm(dim=1)
        assert bool(((got - want).norm(dim=1) <= 0.06 * spread).all())
        pending = {i: [int(t)] for i, t in enumerate(want.argmax(1))}
    assert lib().launch_count() > before
    check_status(torch.device("cuda"))


def test_generate_batch_runs_and_keeps_its_rules():
    from types import SimpleNamespace

    from nano_megatron_b200.inference import LogitRules, generate_batch

    model, cfg = _model("cuda", torch.bfloat16, 8, 4)

    class Words:        # a tokenizer of numbers
        eos_token_id = 8191

        def encode(self, text, add_bos, add_eos):
            return [int(x) for x in text.split()]

        def decode(self, ids, skip_special_tokens):
            return " ".join(map(str, ids))

    art = SimpleNamespace(tokenizer=Words(), model_config=cfg.model)
    prompts = [" ".join(str((7 * i + j) % 8000) for j in range(1 + 9 * i)) for i in range(9)]
    kw = dict(device=torch.device("cuda"), max_new_tokens=12, temperature=0.0)
    all_at_once = generate_batch(art, model, prompts, **kw)
    few = generate_batch(art, model, prompts, max_batch=3, **kw)
    assert [len(r.generated_token_ids) for r in all_at_once] == [12] * 9 == [
        len(r.generated_token_ids) for r in few]
    rules = LogitRules(presence=1e6, bias={5: 3.0}, allowed=range(100))
    for r in generate_batch(art, model, prompts, rules=rules, cache_dtype="int8", **kw):
        assert len(set(r.generated_token_ids)) == 12 and max(r.generated_token_ids) < 100
