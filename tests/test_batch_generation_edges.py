"""Edges of batched generation and of the serving operators' CPU forms."""

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
