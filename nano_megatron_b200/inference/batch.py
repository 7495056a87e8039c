"""Batched generation from exported GPT artifacts over an 8-bit paged K/V cache.

:class:`BatchDecoder` serves several requests at once, each with its own length: a step takes
the new tokens of every active request (a whole prompt, or the token sampled last), plans the
rows and cache pages on the device, writes the new keys and values into the paged cache, attends
over it and returns one row of next-token scores per request. The operators are those of
:mod:`nano_megatron_b200.ops.serving`.

:func:`generate_batch` runs a list of prompts through it, admitting as many at a time as the
decoder has room for and handing the pages of finished requests to waiting ones. Sampling is
:func:`.generation.sample_next_token` with one generator per request, so a prompt's text does
not depend on what else is in the batch (up to the rounding of differently shaped products).
"""

from __future__ import annotations

import math
from collections.abc import Iterable, Sequence
from dataclasses import dataclass

import torch

from nano_megatron_b200.nn.rotary import rope_inv_freq
from nano_megatron_b200.ops import check_status, serving
from nano_megatron_b200.ops import functional as F

from .artifact import InferenceArtifact
from .generation import (
    GenerationResult,
    _check_args,
    fused_layer_weights,
    load_model_for_generation,
    sample_next_token,
)

CACHE_DTYPES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


@dataclass(frozen=True, slots=True)
class LogitRules:
    """What is done to the scores of a request before sampling (see ``adjust_logits``).

    ``repetition`` > 1 makes tokens of the prompt and the completion less likely,
    ``presence`` / ``frequency`` subtract a constant once / per occurrence in the completion,
    ``bias`` adds to single tokens (-inf bans one), ``allowed`` restricts sampling to a set of token ids (any
    iterable, kept as a tuple; at least one).
    """

    repetition: float = 1.0
    presence: float = 0.0
    frequency: float = 0.0
    bias: dict[int, float] | None = None
    allowed: Iterable[int] | None = None

    def __post_init__(self) -> None:
        if not (math.isfinite(self.repetition) and self.repetition > 0.0):
            raise ValueError("repetition must be finite and > 0")
        for name in ("presence", "frequency"):
            if not math.isfinite(getattr(self, name)):
                raise ValueError(f"{name} must be finite")
        for t, x in (self.bias or {}).items():
            if math.isnan(x) or x == math.inf:
                raise ValueError(f"bias of token {t} must be a number or -inf, not {x}")
        if self.allowed is not None:
            object.__setattr__(self, "allowed", tuple(self.allowed))
            if not self.allowed:
                raise ValueError("allowed is empty: no token could be sampled (None allows all)")

    @property
    def empty(self) -> bool:
        return (self.repetition == 1.0 and self.presence == 0.0 and self.frequency == 0.0
                and not self.bias and self.allowed is None)


class BatchDecoder:
    """Incremental decoder of up to ``max_requests`` requests over a ``GPTModel``'s weights.

    The cache holds ``num_pages`` pages of ``page_size`` tokens for all requests together; a
    request's pages are taken as it grows and returned by :meth:`release`. Lengths are known on
    the host as well, so running out of pages or positions is refused before a launch.
    """

    def __init__(self, model, *, max_requests: int, max_len: int, num_pages: int | None = None,
                 page_size: int = 64, cache_dtype: torch.dtype = torch.float8_e4m3fn) -> None:
        if max_requests < 1 or max_len < 1:
            raise ValueError("max_requests and max_len must be >= 1")
        if page_size not in serving.PAGE_SIZES:
            raise ValueError(f"page_size must be one of {serving.PAGE_SIZES}, got {page_size}")
        a0 = model.layers[0].attention
        self.model = model
        self.nh, self.nkv, self.d = a0.num_heads, a0.num_kv_heads, a0.head_dim
        self.eps = model.eps
        self.device = model.embedding.weight.device
        if self.device.type == "cuda" and self.d not in (64, 128):
            raise ValueError(f"batched generation on CUDA needs head_dim 64 or 128, not {self.d}")
        if self.device.type == "cuda" and model.embedding.weight.dtype != torch.bfloat16:
            raise ValueError("batched generation on CUDA needs bfloat16 weights, not "
                             f"{model.embedding.weight.dtype}")
        if self.device.type == "cuda" and max_requests > serving.MAX_REQUESTS:
            raise ValueError(f"at most {serving.MAX_REQUESTS} requests at a time on CUDA, "
                             f"got {max_requests}")
        self.max_requests, self.max_len, self.page_size = max_requests, max_len, page_size
        width = -(-max_len // page_size)
        self.num_pages = max_requests * width if num_pages is None else num_pages
        # in fp32 whatever the model's type (its own buffer is cast with the weights)
        self.inv_freq = rope_inv_freq(self.d, a0.rope_theta, device=self.device)
        self.weights = fused_layer_weights(model)
        self.caches = [serving.PagedKV.create(self.num_pages, self.nkv, self.d, page_size=page_size,
                                              dtype=cache_dtype, device=self.device)
                       for _ in self.weights]
        self.tables = torch.full((max_requests, width), -1, dtype=torch.int32, device=self.device)
        self.free_pages = torch.arange(self.num_pages - 1, -1, -1, dtype=torch.int32,
                                       device=self.device)
        self.free_count = torch.tensor([self.num_pages], dtype=torch.int32, device=self.device)
        self.free = self.num_pages                 # the host's copy of free_count
        self.lengths = [0] * max_requests

    def pages_for(self, length: int) -> int:
        return -(-length // self.page_size)

    @torch.inference_mode()
    def release(self, slot: int) -> None:
        """Forget request ``slot`` and return its pages."""
        n = self.pages_for(self.lengths[slot])
        self.free_pages[self.free:self.free + n] = self.tables[slot, :n]
        self.free_count = self.free_count + n
        self.free += n
        self.lengths[slot] = 0

    @staticmethod
    def _lin(x, w, b=None):
        y = F.linear(x, w)
        return y + b if b is not None else y

    @torch.inference_mode()
    def step(self, new_tokens: dict[int, Sequence[int]]) -> torch.Tensor:
        """Append ``new_tokens[slot]`` to each request named; returns the scores of the last
        token of each ([len(new_tokens), vocabulary], in the order of the slots' numbers).

        Does not wait for the GPU; on CUDA ``check_status`` says, once the scores are read, whether
        a kernel gave up and they are unfinished."""
        slots = sorted(new_tokens)
        if not slots:
            raise ValueError("a step needs at least one request")
        if slots[0] < 0 or slots[-1] >= self.max_requests:
            raise ValueError(f"request slots are 0..{self.max_requests - 1}")
        new = [0] * (slots[-1] + 1)
        need = 0
        for s in slots:
            n = new[s] = len(new_tokens[s])
            if n == 0:
                raise ValueError(f"request {s} adds no token")
            if self.lengths[s] + n > self.max_len:
                raise ValueError(f"the cache holds {self.max_len} positions of a request; "
                                 f"request {s} asks for {self.lengths[s] + n}")
            need += self.pages_for(self.lengths[s] + n) - self.pages_for(self.lengths[s])
        if need > self.free:
            raise RuntimeError(f"the cache is out of pages: {need} needed, {self.free} free")
        ids = [t for s in slots for t in new_tokens[s]]
        # (on CUDA a lookup outside the embedding would end the whole context)
        vocab = self.model.original_vocab_size
        if min(ids) < 0 or max(ids) >= vocab:
            raise ValueError(f"token ids are 0..{vocab - 1}, the model's vocabulary; got "
                             f"{min(ids) if min(ids) < 0 else max(ids)}")
        # one copy to the device: [token ids | context lengths | new lengths | last rows]
        ends, last = 0, []
        for s in slots:
            ends += new[s]
            last.append(ends - 1)
        B, T = len(new), len(ids)
        host = torch.tensor(ids + self.lengths[:B] + new + last, dtype=torch.int32)
        both = host.to(self.device)
        tokens, context, fresh, rows = both.split([T, B, B, len(slots)])
        plan = serving.plan_step(context, fresh, self.tables, self.free_pages, self.free_count,
                                 page_size=self.page_size, num_tokens=T)
        m = self.model
        h = m.embedding.weight.index_select(0, tokens)
        qc, kvc = self.nh * self.d, self.nkv * self.d
        most = max(new)
        for w, cache in zip(self.weights, self.caches):
            y, _ = F.rmsnorm(h, w["n1"], self.eps)
            qkv = self._lin(y, w["wqkv"], w["bqkv"])
            F.rope_(qkv, qc + kvc, self.d, plan.positions, self.inv_freq, inverse=False)
            serving.append_kv(cache, qkv[:, qc:qc + kvc].view(T, self.nkv, self.d),
                              qkv[:, qc + kvc:].view(T, self.nkv, self.d), plan.touched)
            a = serving.paged_attention(qkv[:, :qc].view(T, self.nh, self.d), cache, self.tables,
                                        plan.q_starts, plan.kv_lens, max_new=most)
            h = h + self._lin(a.view(T, qc), w["wo"], w["bo"])
            y, _ = F.rmsnorm(h, w["n2"], self.eps)
            gu = self._lin(y, w["wgu"], w["bgu"])
            h = h + self._lin(F.swiglu_act(gu, gu.shape[1] // 2), w["wd"], w["bd"])
        y, _ = F.rmsnorm(h.index_select(0, rows), m.final_norm.weight, self.eps)
        scores = F.linear(y, m.lm_head.weight)[:, :m.original_vocab_size]
        # only now, so that a step that raised can be repeated
        self.free_count = plan.free_count
        self.free -= need
        for s in slots:
            self.lengths[s] += new[s]
        return scores


class _Rules:
    """The rules of the decoder's requests as device tensors, one row per request slot."""

    def __init__(self, dec: BatchDecoder, rules: Sequence[LogitRules], vocab: int) -> None:
        n, dev = dec.max_requests, dec.device
        self.active = any(not r.empty for r in rules)
        if not self.active:
            return
        self.vocab = vocab
        most = max((len(r.bias or ()) for r in rules), default=0)
        self.history = torch.zeros(n, dec.max_len, dtype=torch.int32, device=dev)
        self.numbers = torch.zeros(3, n, device=dev)
        self.bias_ids = torch.full((n, most), -1, dtype=torch.int32, device=dev) if most else None
        self.bias = torch.zeros(n, most, device=dev) if most else None
        self.allowed = (torch.full((n, (vocab + 31) // 32), -1, dtype=torch.int32, device=dev)
                        if any(r.allowed is not None for r in rules) else None)
        self.prompts = [0] * n

    def admit(self, slot: int, prompt: Sequence[int], r: LogitRules) -> None:
        if not self.active:
            return
        dev = self.history.device
        self.prompts[slot] = len(prompt)
        self.history[slot, :len(prompt)] = torch.tensor(prompt, dtype=torch.int32).to(dev)
        self.numbers[:, slot] = torch.tensor([r.repetition, r.presence, r.frequency]).to(dev)
        if self.bias is not None:
            ids, values = list(r.bias or {}), list((r.bias or {}).values())
            self.bias_ids[slot] = -1
            if ids:
                self.bias_ids[slot, :len(ids)] = torch.tensor(ids, dtype=torch.int32).to(dev)
                self.bias[slot, :len(ids)] = torch.tensor(values, dtype=torch.float32).to(dev)
        if self.allowed is not None:
            bits = torch.full((self.allowed.shape[1] * 32,), r.allowed is None)
            if r.allowed is not None:
                bits[torch.tensor(list(r.allowed), dtype=torch.long)] = True
            words = (bits.view(-1, 32).long() << torch.arange(32)).sum(1)
            words = torch.where(words >= 2 ** 31, words - 2 ** 32, words)
            self.allowed[slot] = words.to(torch.int32).to(dev)

    def apply(self, logits: torch.Tensor, slots: Sequence[int], lengths: Sequence[int],
              last: Sequence[int]) -> torch.Tensor:
        """Scores of ``slots``; ``last``: the newest token of each (already part of it)."""
        if not self.active:
            return logits
        dev = logits.device
        both = torch.tensor([list(slots), [n - 1 for n in lengths], list(last), list(lengths),
                             [self.prompts[s] for s in slots]], dtype=torch.int32).to(dev)
        at, newest = both[0].long(), both[1].long()
        self.history[at, newest] = both[2]
        rep, pre, freq = self.numbers[:, at].contiguous()

        def pick(t):
            return None if t is None else t[at]

        return serving.adjust_logits(logits, self.history[at], both[3], both[4], repetition=rep,
                                     presence=pre, frequency=freq, bias_ids=pick(self.bias_ids),
                                     bias=pick(self.bias), allowed=pick(self.allowed))


def generate_batch(artifact: InferenceArtifact, model, prompts: Sequence[str], *,
                   device: torch.device, max_new_tokens: int = 128, temperature: float = 0.8,
                   top_p: float = 0.95, top_k: int = 0, seed: int = 1234, add_bos: bool = True,
                   rules: LogitRules | Sequence[LogitRules] = LogitRules(),
                   cache_dtype: str = "e4m3", page_size: int = 64, max_batch: int = 64,
                   num_pages: int | None = None) -> list[GenerationResult]:
    """Continue every prompt; results are in the prompts' order.

    ``rules`` is one set for all prompts or one per prompt. ``max_batch`` prompts are served at
    a time; ``num_pages`` bounds the cache (default: room for ``max_batch`` requests of the
    largest length needed): a waiting prompt is admitted when a slot and pages for its whole
    length are free.
    """
    if isinstance(prompts, str):
        raise TypeError("prompts must be a list of texts, not one text")
    prompts = list(prompts)
    for p in prompts:
        _check_args(p, max_new_tokens, temperature, top_p, top_k, seed, add_bos)
    if not prompts:
        return []
    if cache_dtype not in CACHE_DTYPES:
        raise ValueError(f"cache_dtype {cache_dtype!r}: use " + " or ".join(sorted(CACHE_DTYPES)))
    if max_batch < 1:
        raise ValueError("max_batch must be >= 1")
    rules = [rules] * len(prompts) if isinstance(rules, LogitRules) else list(rules)
    if len(rules) != len(prompts):
        raise ValueError(f"{len(prompts)} prompts, but {len(rules)} sets of rules")
    tok = artifact.tokenizer
    limit, vocab = artifact.model_config.seq_length, model.original_vocab_size
    ids = [tok.encode(p, add_bos=add_bos, add_eos=False) for p in prompts]
    for i, p in enumerate(ids):
        if not p:
            raise ValueError(f"prompt {i} encodes to zero tokens: give some text or add_bos=True")
        if len(p) + max_new_tokens > limit:
            raise ValueError(f"{len(p)} prompt tokens + {max_new_tokens} new tokens "
                             f"exceeds model sequence length {limit}")
        for t in list(rules[i].bias or ()) + list(rules[i].allowed or ()):
            if not 0 <= t < vocab:
                raise ValueError(f"token id {t} of the rules is outside the vocabulary ({vocab})")
        if model.embedding.weight.is_cuda and len(rules[i].bias or ()) > serving.MAX_BIAS:
            raise ValueError(f"at most {serving.MAX_BIAS} biases a prompt on CUDA, "
                             f"prompt {i} has {len(rules[i].bias)}")
    longest = max(len(p) for p in ids) + max_new_tokens
    dec = BatchDecoder(model, max_requests=min(max_batch, len(prompts)), max_len=longest,
                       num_pages=num_pages, page_size=page_size,
                       cache_dtype=CACHE_DTYPES[cache_dtype])
    if dec.pages_for(longest) > dec.num_pages:
        raise ValueError(f"{dec.num_pages} pages cannot hold one request of {longest} tokens")
    held = _Rules(dec, rules, vocab)
    waiting = list(range(len(prompts)))[::-1]
    serving_slots: dict[int, int] = {}             # slot -> prompt
    reserved = 0                                   # pages promised to the admitted requests
    new: list[list[int]] = [[] for _ in prompts]
    stop = ["length"] * len(prompts)
    gens = [torch.Generator(device="cpu").manual_seed(seed) for _ in prompts]
    pending: dict[int, list[int]] = {}

    def whole(i: int) -> int:
        return dec.pages_for(len(ids[i]) + max_new_tokens)

    with torch.inference_mode():
        while waiting or serving_slots:
            for slot in range(dec.max_requests):
                if waiting and slot not in serving_slots and \
                        reserved + whole(waiting[-1]) <= dec.num_pages:
                    i = waiting.pop()
                    serving_slots[slot] = i
                    reserved += whole(i)
                    pending[slot] = ids[i]
                    held.admit(slot, ids[i], rules[i])
            scores = dec.step(pending)
            slots = sorted(pending)
            scores = held.apply(scores, slots, [dec.lengths[s] for s in slots],
                                [pending[s][-1] for s in slots]).cpu()
            if dec.device.type == "cuda":
                check_status(dec.device)
            pending = {}
            for row, slot in zip(scores, slots):
                i = serving_slots[slot]
                nxt = sample_next_token(row, temperature=float(temperature), top_p=float(top_p),
                                        top_k=top_k, generator=gens[i])
                if not math.isfinite(float(row[nxt])):   # the largest, at temperature 0
                    raise RuntimeError(f"no token left to sample for prompt {i}: no score is finite")
                new[i].append(nxt)
                if nxt == tok.eos_token_id:
                    stop[i] = "eos"
                elif len(new[i]) < max_new_tokens:
                    pending[slot] = [nxt]
                    continue
                dec.release(slot)
                reserved -= whole(i)
                del serving_slots[slot]
    return [GenerationResult(prompt=p, text=tok.decode(a + n, skip_special_tokens=True),
                             completion=tok.decode(n, skip_special_tokens=True),
                             token_ids=tuple(a + n), generated_token_ids=tuple(n), stop_reason=s)
            for p, a, n, s in zip(prompts, ids, new, stop)]


def generate_batch_from_artifact(artifact_path, prompts: Sequence[str], *, device="auto",
                                 dtype: str = "auto", **options) -> list[GenerationResult]:
    """:func:`generate_batch` on an artifact directory."""
    artifact, model, dev = load_model_for_generation(artifact_path, device=device, dtype=dtype)
    return generate_batch(artifact, model, prompts, device=dev, **options)
