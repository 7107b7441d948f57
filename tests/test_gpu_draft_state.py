"""What decoders of drafted tokens and of log probabilities hold: rows, texts and records that belong together, whatever call comes first or fails."""

import pytest
import torch

from ajllm_amd import decoding
from tests.latent_models import config, random_weights
from tests.test_gpu_draft_decoder import VOCAB, _model, _prompt
from tests.test_gpu_latent import _build, _tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["graph", "fused", "shared", "dense"])
def test_log_probs_of_tokens_that_were_not_kept_are_refused(cuda, kind):
    """Tokens produced ahead of set_log_probs have no log probability to give; those of the next prompt have."""
    if kind == "dense":
        cfg = config(window=[9, 14, 30], positions=256)
        dec = decoding.DenseDecoder(_build(cfg, random_weights(cfg, 21), cuda, torch.bfloat16), 2, 80)
        prompt = torch.tensor([_tokens(cfg, 12, 40 + i) for i in range(2)], device=cuda)
    else:
        model, prompt = _model(cuda), _prompt(9, 2, 12)
        dec = (decoding.SharedPrefixDecoder(model, 2, 1, 16, 40) if kind == "shared"
               else (decoding.GraphDecoder if kind == "graph" else decoding.FusedDecoder)(model, 2, 64))
    dec.prefill(prompt)
    dec.generate(6)
    dec.set_log_probs(2)
    assert dec.log_probs(0).log_probs.shape == (2, 0)
    for many in (1, 6):
        with pytest.raises(ValueError, match="the first 6 tokens were produced ahead of set_log_probs"):
            dec.log_probs(many)
    dec.generate(10)
    with pytest.raises(ValueError, match="the first 6 tokens"):
        dec.log_probs(10)
    dec.set_log_probs()
    with pytest.raises(ValueError, match="the first 10 tokens"):
        dec.log_probs(10)
    dec.prefill(prompt)
    dec.generate(10)
    kept = dec.log_probs(10)
    assert bool((kept.log_probs < 0).all()) and bool((kept.ranks == 0).all()) and bool((kept.entropy > 0).all())


def test_draft_decoder_takes_its_caches_once(cuda):
    """Never more than its own caches and little beside them, while it is made as afterwards."""
    model = _model(cuda, context=4096)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before, reserved = torch.cuda.memory_allocated(), torch.cuda.memory_reserved()
    dec = decoding.DraftDecoder(model, 64, 4000, [-1, 0, 1])
    caches = dec.all_keys.nbytes + dec.all_values.nbytes
    assert caches == 2 * 2 * 64 * 2 * 4003 * 64 * 4                    # (layers, keys and values; 524 MB)
    assert torch.cuda.max_memory_allocated() - before < 1.2 * caches
    assert torch.cuda.memory_reserved() - reserved < 1.2 * caches
    assert [k.data_ptr() for k in dec.cache.keys] == [k.data_ptr() for k in dec.all_keys] and dec.cache.max_len == dec.cache.keys[0].shape[2] == len(dec.cache.slots)


@pytest.mark.parametrize("failures", [1, 2])
def test_a_pass_that_cannot_be_recorded_leaves_the_state_as_it_was(cuda, monkeypatch, failures):
    """Rows and tokens on the device are those of the texts when a graph could not be made (memory that is not there), and the passes behind it go on from them."""
    model, prompt = _model(cuda), _prompt(7, 2, 15)
    want = decoding.DraftDecoder(model, 2, 60, [-1])
    want.prefill(prompt)
    for _ in range(8):
        want.check([[], []])
    assert len(set(want.texts[0][-9:])) > 4                            # (a token left out would show)
    dec = decoding.DraftDecoder(model, 2, 60, [-1])
    dec.prefill(prompt)

    def no_memory():
        raise RuntimeError("no memory for a graph")

    with monkeypatch.context() as patch:
        patch.setattr(torch.cuda, "CUDAGraph", no_memory)
        failed = 0
        while failed < failures:
            try:
                dec.check([[], []])
            except RuntimeError:
                failed += 1
            assert [len(text) - 1 for text in dec.texts] == dec.rows.tolist() and [text[-1] for text in dec.texts] == dec.token[:, 0].tolist()
    while len(dec.texts[0]) < len(want.texts[0]):
        dec.check([[], []])
    assert dec.texts == want.texts


def test_guesses_of_another_shape_are_refused(cuda):
    dec = decoding.DraftDecoder(_model(cuda), 2, 40, [-1, 0, 0, 1])
    dec.prefill(_prompt(1, 2, 10))
    for bad in ([1, 2, 3, 4, 5, 6], [[1, 2], [3, 4], [5, 6]], [[[1, 2, 3], [4, 5, 6]]], torch.zeros(6, dtype=torch.long), torch.zeros(1, 2, 3, dtype=torch.long)):
        with pytest.raises(ValueError, match="guesses"):
            dec.check(bad)
    assert dec.rows.tolist() == [10, 10]
    assert all(len(new) >= 1 for new in dec.check(torch.full((2, 3), VOCAB - 1, device=cuda)))
