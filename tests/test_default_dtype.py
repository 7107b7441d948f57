"""Numbers that kernels read as fp32 are fp32 whatever torch's default dtype is."""

import contextlib
from types import SimpleNamespace

import pytest
import torch

from ajllm_amd import decoding, modeling, sampling
from tests import serve_plain

DEFAULTS = [torch.bfloat16, torch.float64]


@contextlib.contextmanager
def _default(dtype):
    before = torch.get_default_dtype()
    torch.set_default_dtype(dtype)
    try:
        yield
    finally:
        torch.set_default_dtype(before)


@pytest.mark.parametrize("dtype", DEFAULTS)
def test_numbers_become_fp32_rows(dtype):
    with _default(dtype):
        rows = sampling._of_rows("repetition", 1.25, 4, torch.device("cpu"))
    assert rows.dtype == torch.float32 and rows.tolist() == [1.25] * 4


def _stub(**more):
    """What the setters of a decoder look at, without a device."""
    return SimpleNamespace(batch=3, max_len=5, device=torch.device("cpu"), model=SimpleNamespace(vocab_size=11), _drop_graphs=lambda: None, **more)


@pytest.mark.parametrize("dtype", DEFAULTS)
def test_penalties_become_fp32_rows(dtype):
    stub = _stub()
    with _default(dtype):
        decoding.GraphDecoder.set_penalties(stub, repetition=1.25, frequency=0.5, presence=0.25, bias={4: 1.5})
    for name, value in (("repetition", [1.25] * 3), ("frequency", [0.5] * 3), ("presence", [0.25] * 3), ("bias", [[1.5]] * 3)):
        assert stub.adjustments[name].dtype == torch.float32 and stub.adjustments[name].tolist() == value, name


@pytest.mark.parametrize("dtype", DEFAULTS)
def test_random_numbers_of_a_draw_are_fp32(dtype):
    want, stub = _stub(), _stub()
    decoding.GraphDecoder.set_sampling(want, 0.8, seed=5)
    with _default(dtype):
        decoding.GraphDecoder.set_sampling(stub, 0.8, seed=5)
    assert stub.uniforms.dtype == torch.float32 and torch.equal(stub.uniforms, want.uniforms)


def _small_model(dtype=torch.float32):
    torch.manual_seed(0)
    with _default(torch.float32):
        return modeling.TransformerLM(vocab_size=101, context_length=64, d_model=64, num_layers=1, num_heads=2, d_ff=64).to(dtype)


def _decoded(model, cuda, **sampling_of):
    decoder = decoding.GraphDecoder(model, 3, 24)
    if sampling_of:
        decoder.set_sampling(**sampling_of)
    decoder.set_penalties(repetition=1.5, frequency=0.5, presence=0.25, bias={7: 1.5})
    decoder.prefill(torch.arange(12).view(3, 4))
    return decoder.generate(16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DEFAULTS)
def test_a_decoder_takes_penalties_under_any_default(cuda, dtype):
    model = _small_model().to(cuda)
    want = _decoded(model, cuda)
    with _default(dtype):
        assert torch.equal(_decoded(model, cuda), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DEFAULTS)
def test_a_decoder_draws_under_any_default(cuda, dtype):
    model = _small_model().to(cuda)
    want = _decoded(model, cuda, temperature=0.9, top_p=0.9, seed=4)
    with _default(dtype):
        assert torch.equal(_decoded(model, cuda, temperature=0.9, top_p=0.9, seed=4), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DEFAULTS)
def test_adjust_logits_takes_numbers_under_any_default(cuda, dtype):
    gen = torch.Generator().manual_seed(3)
    batch, vocab = 37, 1003
    logits = torch.randn((batch, vocab), generator=gen, dtype=torch.float32)
    tokens = torch.randint(0, 60, (batch, 41), generator=gen)
    numbers = dict(repetition=1.3, frequency=0.7, presence=-0.2)
    want, size = serve_plain.adjust_logits(logits, tokens, None, None, None, *numbers.values(), None, None, None, None)
    with _default(dtype):
        got = sampling.adjust_logits(logits.to(cuda), tokens=tokens.to(cuda), **numbers)
        rows = {k: torch.full((batch,), v, dtype=torch.float32, device=cuda) for k, v in numbers.items()}
        same = sampling.adjust_logits(logits.to(cuda), tokens=tokens.to(cuda), **rows)
    assert got.dtype == torch.float32 and torch.equal(got, same)
    # 4 roundings (quotient, count times frequency, sum with presence, difference) and the numbers' own to fp32: 5 steps of 2^-24 of what is added up
    assert bool(((got.double().cpu() - want).abs() <= 5 * 2.0 ** -24 * size).all())


@pytest.mark.parametrize("dtype", DEFAULTS)
def test_states_of_a_cache_are_fp32(dtype):
    with _default(dtype):
        cache = modeling.RingCache([4], [16], 2, 8, torch.device("cpu"), torch.bfloat16, states=[(4, 16, 4)])
    assert cache.states[0].dtype == torch.float32 and cache.rings[0].dtype == torch.bfloat16
