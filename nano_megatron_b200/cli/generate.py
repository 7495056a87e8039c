"""Generate text on one device from an exported GPT artifact (``nano-megatron-generate``)."""

from __future__ import annotations

import argparse
import json
from collections.abc import Sequence
from pathlib import Path

from nano_megatron_b200.inference import (
    GenerationResult,
    LogitRules,
    generate_batch_from_artifact,
    generate_from_artifact,
)


def parser() -> argparse.ArgumentParser:
    p = argparse.ArgumentParser(description=__doc__)
    p.add_argument("--model", type=Path, required=True,
                   help="artifact directory written by nano-megatron-export")
    what = p.add_mutually_exclusive_group(required=True)
    what.add_argument("--prompt", help="text to continue")
    what.add_argument("--prompts-file", type=Path,
                      help="continue every line of this file, served as one batch over an 8-bit "
                           "paged K/V cache; prints one result per line, in order")
    p.add_argument("--device", default="auto",
                   help="'auto' uses CUDA when it is available; or cpu, cuda, cuda:N")
    p.add_argument("--dtype", choices=("auto", "float32", "bfloat16", "float16"),
                   default="auto",
                   help="'auto' = fp32 on CPU, the artifact's weight dtype on CUDA")
    p.add_argument("--max-new-tokens", type=int, default=128,
                   help="stop after this many sampled tokens (or at EOS)")
    p.add_argument("--temperature", type=float, default=0.8,
                   help="softmax temperature; 0 decodes greedily")
    p.add_argument("--top-p", type=float, default=0.95,
                   help="nucleus sampling mass (1 keeps the whole distribution)")
    p.add_argument("--top-k", type=int, default=0,
                   help="sample among the k most likely tokens only (0 = no limit)")
    p.add_argument("--seed", type=int, default=1234, help="sampling RNG seed")
    p.add_argument("--add-bos", action=argparse.BooleanOptionalAction, default=True,
                   help="start the prompt with the tokenizer's BOS id (on by default)")
    p.add_argument("--kv-cache", action=argparse.BooleanOptionalAction, default=True,
                   help="reuse cached keys/values between decode steps (on by default; "
                        "--no-kv-cache recomputes the whole prefix every step)")
    b = p.add_argument_group("batched generation (with --prompts-file only)")
    b.add_argument("--max-batch", type=int, help="prompts served at a time (default: 64)")
    b.add_argument("--cache-dtype", choices=("e4m3", "int8"),
                   help="8-bit format of the K/V cache (default: e4m3)")
    b.add_argument("--repetition-penalty", type=float,
                   help="divide positive scores of tokens seen before by this (default: 1 = off)")
    b.add_argument("--presence-penalty", type=float,
                   help="subtract this from tokens that were generated before (default: 0)")
    b.add_argument("--frequency-penalty", type=float,
                   help="subtract this once per earlier generation of a token (default: 0)")
    p.add_argument("--json", action="store_true",
                   help="print the whole result (prompt, completion, token ids, stop reason) "
                        "as one JSON object instead of the text")
    return p


def run_generate(model: Path, prompt: str, *, device: str = "auto", dtype: str = "auto",
                 max_new_tokens: int = 128, temperature: float = 0.8, top_p: float = 0.95,
                 top_k: int = 0, seed: int = 1234, add_bos: bool = True,
                 kv_cache: bool = True) -> GenerationResult:
    return generate_from_artifact(model, prompt, device=device, dtype=dtype,
                                  max_new_tokens=max_new_tokens, temperature=temperature,
                                  top_p=top_p, top_k=top_k, seed=seed, add_bos=add_bos,
                                  use_kv_cache=kv_cache)


# options of batched generation and their values when they are not given
_BATCH_DEFAULTS = {"max_batch": 64, "cache_dtype": "e4m3", "repetition_penalty": 1.0,
                   "presence_penalty": 0.0, "frequency_penalty": 0.0}


def _check_mode(p: argparse.ArgumentParser, a: argparse.Namespace) -> None:
    """Refuse options that the chosen mode would ignore; fill in the batch's defaults."""
    for name, default in _BATCH_DEFAULTS.items():
        if getattr(a, name) is None:
            setattr(a, name, default)
        elif a.prompts_file is None:
            p.error(f"--{name.replace('_', '-')} needs --prompts-file")
    if a.prompts_file is not None and not a.kv_cache:
        p.error("--no-kv-cache: a batch is always served from its paged cache")


def main(argv: Sequence[str] | None = None) -> None:
    p = parser()
    a = p.parse_args(argv)
    _check_mode(p, a)
    if a.prompts_file is not None:
        # (str.splitlines would also split at form feeds, line separators and others)
        with open(a.prompts_file, encoding="utf-8") as f:
            prompts = [line.removesuffix("\n") for line in f]
        for r in generate_batch_from_artifact(
                a.model, prompts, device=a.device, dtype=a.dtype,
                max_new_tokens=a.max_new_tokens, temperature=a.temperature, top_p=a.top_p,
                top_k=a.top_k, seed=a.seed, add_bos=a.add_bos, max_batch=a.max_batch,
                cache_dtype=a.cache_dtype,
                rules=LogitRules(repetition=a.repetition_penalty, presence=a.presence_penalty,
                                 frequency=a.frequency_penalty)):
            print(json.dumps(r.to_dict(), ensure_ascii=False, sort_keys=True) if a.json
                  else r.text.replace("\n", " "))
        return
    r = run_generate(a.model, a.prompt, device=a.device, dtype=a.dtype,
                     max_new_tokens=a.max_new_tokens, temperature=a.temperature, top_p=a.top_p,
                     top_k=a.top_k, seed=a.seed, add_bos=a.add_bos, kv_cache=a.kv_cache)
    print(json.dumps(r.to_dict(), ensure_ascii=False, sort_keys=True) if a.json else r.text)


if __name__ == "__main__":
    main()
