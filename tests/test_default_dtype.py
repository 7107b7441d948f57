"""Numbers that kernels read as fp32 are fp32 whatever torch's default dtype is."""

import contextlib

import pytest
import torch

from ajllm_amd import sampling
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
