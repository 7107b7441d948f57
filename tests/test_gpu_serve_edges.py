"""Ends of the ranges that the operators of decoding many continuations of one prompt (include/ajq_serve.h) take."""

import pytest
import torch

from ajllm_amd import attention, sampling
from tests import serve_plain

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
F32 = torch.float32


@pytest.mark.parametrize("hd", [128, 64, 32])
@pytest.mark.parametrize("in_type", [F32, BF16])
@pytest.mark.parametrize("tokens", [1, 3])
@pytest.mark.parametrize("size,epsilon", [(1e18, 1e-5), (1e19, 1e-5), (1e30, 1e-5), (2e37, 0.0), (1e-20, 0.0), (1e-37, 0.0), (1e-12, 0.0), (1e-30, 1e-38), (1.0, 1e38)])
def test_norm_rope_heads_whose_squares_pass_fp32(cuda, hd, in_type, tokens, size, epsilon):
    """Every second head of the given size, the others ordinary: roundings are those of any head (16 steps of 2^-24 of a pair's length: ``_near`` of the operators'
    tests), since a power of two takes none; a component of a length below 2^-126 may be off by fp32's smallest number."""
    gen = torch.Generator().manual_seed(hd + tokens)
    batch, heads, kv, max_len = 3, 4, 2, 8
    x = torch.randn((batch * tokens, heads + 2 * kv, hd), generator=gen).clamp(-10, 10)
    x[:, ::2] *= size
    qkv = x.view(batch * tokens, -1).to(in_type)
    angles = torch.arange(max_len, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    tables = angles.cos().float(), angles.sin().float()
    gains = 1 + 0.3 * torch.randn((2, hd), generator=gen)
    keys, values = torch.zeros((batch, kv, max_len, hd)), torch.zeros((batch, kv, max_len, hd))
    rows = torch.tensor([0, 2, 5])
    # (the epsilon that the kernel gets is an fp32 number)
    want = serve_plain.norm_rope(qkv, *tables, keys, values, rows, heads, tokens, *gains, float(torch.tensor(epsilon, dtype=F32)), None, None, 0)
    on = [t.to(cuda) for t in (qkv, *tables, keys, values, rows)]
    q = attention.norm_rope(*on, heads=heads, tokens=tokens, q_gain=gains[0].to(cuda), k_gain=gains[1].to(cuda), epsilon=epsilon)
    for got, exact, magnitude, what in ((q, want[0], want[3], "queries"), (on[3], want[1], want[4], "keys")):
        assert bool(torch.isfinite(got).all()), what
        assert bool(((got.double().cpu() - exact).abs() <= 16 * 2.0 ** -24 * magnitude + 2.0 ** -149).all()), what
    assert torch.equal(on[4].double().cpu(), want[2])


@pytest.mark.parametrize("type", [F32, BF16])
def test_adjust_logits_takes_lists_and_masks_that_rows_share(cuda, type):
    """Expanded lists and masks are the same as copies of them for every row, down to the bit."""
    gen = torch.Generator().manual_seed(9)
    batch, vocab = 5, 1500
    logits = (torch.randn((batch, vocab), generator=gen) * 4).to(type).to(cuda)
    prompt, tokens = (torch.randint(-3, 200, (1, n), generator=gen).to(cuda) for n in (90, 33))
    allowed = torch.randint(-2 ** 31, 2 ** 31, (1, 47), generator=gen).int().to(cuda)
    more = dict(lengths=torch.tensor([33, 0, 7, 20, 1], device=cuda), prompt_lengths=torch.tensor([60], device=cuda), repetition=1.5, frequency=0.25, presence=0.5)
    shared = dict(tokens=tokens.expand(batch, 33), prompt=prompt.expand(batch, 90), allowed=allowed.expand(batch, 47))
    assert all(t.stride(0) == 0 for t in shared.values())
    got = sampling.adjust_logits(logits, **shared, **more)
    assert torch.equal(got, sampling.adjust_logits(logits, **{k: t.contiguous() for k, t in shared.items()}, **more))
    want, size = serve_plain.adjust_logits(logits.cpu(), shared["tokens"].cpu(), more["lengths"].cpu(), shared["prompt"].cpu(), more["prompt_lengths"].cpu(), 1.5, 0.25, 0.5, None,
                                           None, shared["allowed"].cpu(), None)
    got = got.double().cpu()
    assert torch.equal(torch.isinf(got), torch.isinf(want))
    assert bool((torch.where(torch.isinf(want), 0.0, (got - want).abs()) <= 4 * 2.0 ** -24 * size).all())   # (four roundings, each 2^-24 of what is added up)
