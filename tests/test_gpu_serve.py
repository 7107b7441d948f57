"""The operators of decoding many continuations of one prompt (include/ajq_serve.h) against their definitions in 64 bits."""

import math

import pytest
import torch

from ajllm_amd import attention, sampling
from tests import serve_plain

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
F32 = torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _tables(positions, hd):
    angles = torch.arange(positions, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    return angles.cos().float(), angles.sin().float()


# ------------------------------------------------------------------ norm_rope
# In fp32: the factor of the norm has 8 products and 12 additions of positive terms (13 roundings on the longest way, halved by the root), the
# root's, the division's, the gain's and two for each term of a rotation, whose terms together are at most sqrt(2) of the pair's length.  Under
# 16 steps of 2^-24 of that length; a bf16 result is rounded once more, by 2^-8 of itself at most.
def _near(got, want, magnitude, what):
    bound = 16 * 2.0 ** -24 * magnitude + (2.0 ** -8 * want.abs() if got.dtype == BF16 else 0.0)
    off = (got.double().cpu() - want).abs()
    assert bool((off <= bound).all()), (what, float((off / bound.clamp(min=1e-300)).max()))


def _rotate(cuda, batch, tokens, heads, kv, hd, max_len, in_type, q_type, cache_type, seed, norm=True, ragged=True, ld=0, positions=True,
            offset=None, rows=None, counts=None, spread=0):
    gen = _gen(seed)
    width = (heads + 2 * kv) * hd
    qkv = (torch.randn((batch * tokens, width + ld), generator=gen) * 2).to(in_type)
    cosine, sine = _tables(max_len + 40, hd)
    whole = torch.randn((2, batch, kv, max_len + spread, hd), generator=gen).to(cache_type).to(cuda)
    keys, values = whole[0, :, :, :max_len], whole[1, :, :, :max_len]
    rows = torch.randint(0, max(1, max_len - tokens + 1), (batch,), generator=gen) if rows is None else torch.tensor(rows)
    at = rows + 31 if positions else None
    if counts is None and ragged:
        counts = torch.randint(0, tokens + 1, (batch,), generator=gen)
    elif counts is not None:
        counts = torch.tensor(counts)
    q_gain, k_gain = (1 + 0.3 * torch.randn(hd, generator=gen), 1 + 0.3 * torch.randn(hd, generator=gen)) if norm else (None, None)
    put = lambda t: None if t is None else t.to(cuda)  # noqa: E731
    before = whole.clone()
    want = serve_plain.norm_rope(qkv[:, :width], cosine, sine, keys, values, rows, heads, tokens, q_gain, k_gain, 1e-5, at, counts, offset or 0)
    q = attention.norm_rope(put(qkv)[:, :width], put(cosine), put(sine), keys, values, put(rows), heads=heads, tokens=tokens, q_gain=put(q_gain),
                            k_gain=put(k_gain), positions=put(at), counts=put(counts),
                            offset=None if offset is None else torch.tensor([offset], device=cuda), out_dtype=q_type)
    assert q.shape == (batch, heads, tokens, hd) and q.dtype == q_type
    _near(q, want[0], want[3], "queries")
    _near(keys, want[1], want[4], "keys")
    assert torch.equal(values.double().cpu(), want[2].to(cache_type).double())
    if spread:   # what lies between the heads is left as it was
        assert torch.equal(whole[:, :, :, max_len:], before[:, :, :, max_len:])


@pytest.mark.parametrize("hd", [128, 64, 32])
@pytest.mark.parametrize("in_type", [F32, BF16])
@pytest.mark.parametrize("q_type", [F32, BF16])
@pytest.mark.parametrize("cache_type", [F32, BF16])
def test_norm_rope_types_and_sizes(cuda, hd, in_type, q_type, cache_type):
    _rotate(cuda, 3, 5, 6, 2, hd, 11, in_type, q_type, cache_type, seed=hd)


@pytest.mark.parametrize("batch,tokens,heads,kv", [(1, 1, 1, 1), (7, 1, 16, 16), (2, 1, 32, 8), (5, 3, 12, 4), (1, 70, 5, 5), (300, 1, 8, 1)])
def test_norm_rope_heads_and_batches(cuda, batch, tokens, heads, kv):
    _rotate(cuda, batch, tokens, heads, kv, 64, tokens + 9, F32, BF16, BF16, seed=batch + tokens, ragged=tokens > 1)


def test_norm_rope_without_norm_positions_or_counts(cuda):
    _rotate(cuda, 4, 3, 8, 4, 128, 20, F32, F32, F32, seed=1, norm=False, ragged=False, positions=False)


def test_norm_rope_strides_and_offset(cuda):
    _rotate(cuda, 4, 3, 8, 4, 128, 20, F32, F32, BF16, seed=2, ld=12, offset=2, rows=[0, 3, 15, 1], spread=3)
    _rotate(cuda, 4, 1, 8, 4, 32, 20, BF16, BF16, F32, seed=3, ld=4, offset=1, spread=1)


def test_norm_rope_rows_outside_the_caches_are_not_written(cuda):
    # rows -2 .. 0, 6 .. 8, 8 .. 10 (behind the end) and far outside, where positions stay inside the tables as well
    _rotate(cuda, 4, 3, 4, 2, 64, 8, F32, F32, F32, seed=4, rows=[-2, 6, 8, 2 ** 40], ragged=False)
    _rotate(cuda, 4, 3, 4, 2, 64, 8, F32, F32, F32, seed=4, rows=[-2 ** 40, 6, 7, -1], counts=[3, 0, -4, 9])


def test_norm_rope_small_and_large_heads(cuda):
    """A head of zeros stays zero (the epsilon), one of 1e18 is normed without overflow of its squares' sum (128 * 1e36 < 3.4e38)."""
    keys, values = torch.zeros((1, 1, 4, 128), device=cuda), torch.zeros((1, 1, 4, 128), device=cuda)
    cosine, sine = (t.to(cuda) for t in _tables(4, 128))
    qkv = torch.cat((torch.zeros(1, 128), torch.full((1, 128), 1e18), torch.ones(1, 128)), dim=1).to(cuda)
    gain = torch.ones(128, device=cuda)
    q = attention.norm_rope(qkv, cosine, sine, keys, values, torch.zeros(1, dtype=torch.long, device=cuda), heads=1, q_gain=gain, k_gain=gain)
    assert torch.equal(q, torch.zeros_like(q))
    torch.testing.assert_close(keys[0, 0, 0], torch.ones(128, device=cuda), rtol=16 * 2.0 ** -24, atol=0)


def test_norm_rope_refuses(cuda):
    keys, values = torch.zeros((2, 2, 8, 64), device=cuda), torch.zeros((2, 2, 8, 64), device=cuda)
    cosine, sine = (t.to(cuda) for t in _tables(8, 64))
    qkv, rows = torch.zeros((2, 8 * 64), device=cuda), torch.zeros(2, dtype=torch.long, device=cuda)
    ok = dict(heads=4)
    attention.norm_rope(qkv, cosine, sine, keys, values, rows, **ok)
    bad = [
        ((qkv, cosine, sine, keys, values, rows), dict(heads=3)),
        ((qkv, cosine, sine, keys, values, rows), dict(heads=4, tokens=2)),
        ((qkv, cosine, sine, keys, values, rows.int()), ok),
        ((qkv, cosine, sine, keys, values, rows[:1]), ok),
        ((qkv, cosine, sine, keys, values, rows.cpu()), ok),
        ((qkv.half(), cosine, sine, keys, values, rows), ok),
        ((qkv, cosine.double(), sine, keys, values, rows), ok),
        ((qkv, cosine, sine[:4], keys, values, rows), ok),
        ((qkv, cosine, sine, keys.half(), values.half(), rows), ok),
        ((qkv, cosine, sine, keys, values.bfloat16(), rows), ok),
        ((qkv, cosine, sine, keys.transpose(1, 2).contiguous().transpose(1, 2), values, rows), ok),
        ((qkv, cosine, sine, keys[:1].expand(2, 2, 8, 64), values[:1].expand(2, 2, 8, 64), rows), ok),
        ((qkv, cosine, sine, keys, values, rows), dict(heads=4, q_gain=torch.ones(32, device=cuda))),
        ((qkv, cosine, sine, keys, values, rows), dict(heads=4, counts=rows[:1])),
        ((qkv, cosine, sine, keys, values, rows), dict(heads=4, offset=rows)),
        ((qkv, cosine, sine, keys, values, rows), dict(heads=4, out_dtype=torch.float16)),
        ((qkv.cpu(), cosine, sine, keys, values, rows), ok),
    ]
    for args, more in bad:
        with pytest.raises(ValueError, match="norm_rope"):
            attention.norm_rope(*args, **more)


# ------------------------------------------------------------------ shared_prefix_attention
# A weight is rounded to bf16 for the second product (2^-8 of it) and comes from a score whose factors have at least 16 bits; the sums are fp32.
# Together at most (2^-8 + 2^-10) of the weighted mean size of the values; the result is rounded by 2^-8 of itself.
def _attention_near(got, want, size):
    bound = (2.0 ** -8 + 2.0 ** -10) * size + 2.0 ** -8 * want.abs()
    off = (got.double().cpu() - want).abs()
    assert bool(torch.isfinite(got).all())
    assert bool((off <= bound).all()), float((off / bound.clamp(min=1e-300)).max())


def _share(cuda, groups, batch, tokens, heads, kv, hd, prefix, max_len, q_type, cache_type, seed, prefix_lengths=None, rows=None, counts=None,
           offset=None, garbage=True, scale=1.0, spread=0):
    gen = _gen(seed)
    randn = lambda *shape: torch.randn(shape, generator=gen)  # noqa: E731
    q = (randn(batch, heads, tokens, hd) * scale).to(q_type)
    pk, pv = (randn(groups, kv, prefix + spread, hd).to(cache_type)[:, :, :prefix] for _ in range(2))
    k, v = (randn(batch, kv, max_len + spread, hd).to(cache_type)[:, :, :max_len] for _ in range(2))
    prefix_lengths = torch.randint(0, prefix + 1, (groups,), generator=gen) if prefix_lengths is None else torch.tensor(prefix_lengths)
    rows = torch.randint(0, max(1, max_len - tokens + 1), (batch,), generator=gen) if rows is None else torch.tensor(rows)
    counts = None if counts is None else torch.tensor(counts)
    want, size = serve_plain.shared_prefix_attention(q, pk, pv, prefix_lengths, k, v, rows, counts, offset or 0)
    if garbage:   # rows that nobody sees may hold anything
        for g in range(groups):
            pk[g, :, max(0, int(prefix_lengths[g])):] = math.nan
            pv[g, :, max(0, int(prefix_lengths[g])):] = math.inf
        for b in range(batch):
            last = int(rows[b]) + (offset or 0) + (tokens if counts is None else min(max(int(counts[b]), 0), tokens))
            k[b, :, max(0, last):] = math.nan
            v[b, :, max(0, last):] = math.nan
    put = lambda t: None if t is None else t.to(cuda)  # noqa: E731

    def laid(t):   # (a copy to the device would lay the rows of a slice one head behind the other)
        if not spread:
            return t.to(cuda)
        room = torch.full((*t.shape[:2], t.shape[2] + spread, hd), math.nan, dtype=t.dtype, device=cuda)
        room[:, :, :t.shape[2]] = t.to(cuda)
        return room[:, :, :t.shape[2]]

    got = attention.shared_prefix_attention(put(q), laid(pk), laid(pv), put(prefix_lengths), laid(k), laid(v), put(rows), counts=put(counts),
                                            offset=None if offset is None else torch.tensor([offset], device=cuda))
    assert got.shape == (batch, tokens, heads * hd) and got.dtype == BF16
    _attention_near(got, want, size)
    return got


@pytest.mark.parametrize("hd", [128, 64, 32])
@pytest.mark.parametrize("q_type", [F32, BF16])
@pytest.mark.parametrize("cache_type", [F32, BF16])
@pytest.mark.parametrize("tokens", [1, 5])
def test_shared_attention_types_and_sizes(cuda, hd, q_type, cache_type, tokens):
    _share(cuda, 2, 6, tokens, 8, 2, hd, 75, 41, q_type, cache_type, seed=hd + tokens)


@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 1), (16, 16), (12, 4), (32, 4), (16, 1)])
@pytest.mark.parametrize("tokens", [1, 9])
def test_shared_attention_heads(cuda, heads, kv, tokens):
    _share(cuda, 1, 3, tokens, heads, kv, 64, 100, 33, BF16, BF16, seed=heads + tokens)


@pytest.mark.parametrize("prefix,max_len", [(1, 1), (1, 300), (31, 32), (32, 33), (33, 31), (64, 64), (65, 130), (500, 2), (1500, 700)])
@pytest.mark.parametrize("cache_type", [F32, BF16])
def test_shared_attention_lengths(cuda, prefix, max_len, cache_type):
    """Full and nearly full caches: blocks that end inside a tile, one short of it and one past it."""
    _share(cuda, 1, 4, 1, 8, 2, 128, prefix, max_len, BF16, cache_type, seed=prefix, prefix_lengths=[prefix],
           rows=[max_len - 1, 0, max_len // 2, max(0, max_len - 2)])


@pytest.mark.parametrize("tokens", [2, 16, 33, 64, 65, 150])
@pytest.mark.parametrize("cache_type", [F32, BF16])
def test_shared_attention_many_tokens(cuda, tokens, cache_type):
    _share(cuda, 1, 3, tokens, 8, 4, 64, 90, tokens + 70, BF16, cache_type, seed=tokens, rows=[0, 37, 70], counts=[tokens, tokens // 2, tokens - 1])


def test_shared_attention_many_sequences(cuda):
    _share(cuda, 1, 67, 1, 8, 2, 128, 300, 40, F32, BF16, seed=5)
    _share(cuda, 3, 66, 1, 8, 1, 32, 300, 40, BF16, F32, seed=6)


def test_shared_attention_rows_that_see_nothing(cuda):
    """No prefix and no row (zeros), no prefix, prefix alone, tokens that are not there, lengths outside the buffers."""
    got = _share(cuda, 3, 6, 1, 4, 2, 64, 20, 10, F32, BF16, seed=7, prefix_lengths=[0, -3, 20], rows=[-1, 4, -5, 0, -1, 9], garbage=False)
    assert torch.equal(got[0], torch.zeros_like(got[0])) and torch.equal(got[2], torch.zeros_like(got[2]))
    got = _share(cuda, 1, 4, 3, 4, 2, 64, 20, 10, F32, F32, seed=8, prefix_lengths=[0], rows=[-2, 0, 3, 7], counts=[3, 0, 2, -1])
    assert torch.equal(got[0, :1], torch.zeros_like(got[0, :1])) and torch.equal(got[1], torch.zeros_like(got[1]))
    _share(cuda, 1, 2, 1, 4, 2, 64, 20, 10, F32, BF16, seed=9, prefix_lengths=[2 ** 40], rows=[2 ** 40, -2 ** 40], garbage=False)


def test_shared_attention_offset_and_strides(cuda):
    _share(cuda, 2, 4, 1, 4, 2, 128, 50, 30, F32, BF16, seed=10, offset=7, rows=[0, 5, 22, -7], spread=3)
    _share(cuda, 2, 4, 4, 4, 2, 64, 50, 30, BF16, F32, seed=11, offset=3, rows=[0, 5, 22, -3], spread=5)


@pytest.mark.parametrize("cache_type", [F32, BF16])
def test_shared_attention_scores_far_apart(cuda, cache_type):
    """Scores of hundreds: maxima move between blocks, most weights vanish.  (An error of a score is one of its weight: 16 bits of a score of
    hundreds are no 2^-10 of a weight, so the queries are whole numbers that bf16 holds, products are exact and sums of a few thousand too.)"""
    gen = _gen(12)
    batch, heads, kv, hd, prefix, max_len = 3, 4, 2, 64, 400, 60
    whole = lambda *shape: torch.randint(-8, 9, shape, generator=gen).float()  # noqa: E731
    q, pk, k = whole(batch, heads, 1, hd) * 2, whole(1, kv, prefix, hd), whole(batch, kv, max_len, hd)
    pv, v = torch.randn((1, kv, prefix, hd), generator=gen).to(cache_type), torch.randn((batch, kv, max_len, hd), generator=gen).to(cache_type)
    rows, lengths = torch.tensor([59, 0, 30]), torch.tensor([prefix])
    want, size = serve_plain.shared_prefix_attention(q, pk, pv, lengths, k, v, rows, None, 0)
    got = attention.shared_prefix_attention(q.to(cuda), pk.to(cache_type).to(cuda), pv.to(cuda), lengths.to(cuda), k.to(cache_type).to(cuda), v.to(cuda),
                                            rows.to(cuda))
    _attention_near(got, want, size)


def _share_by_heads(cuda, groups, batch, tokens, heads, kv, hd, prefix, max_len, q_type, cache_type, seed):
    """Lengths, positions and counts at random, one sequence and one group full, one sequence without tokens; rows that nobody sees hold anything."""
    gen = torch.Generator(device=cuda).manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=gen, device=cuda)  # noqa: E731
    whole = lambda low, high, n: torch.randint(low, high + 1, (n,), generator=gen, device=cuda)  # noqa: E731
    q = randn(batch, heads, tokens, hd).to(q_type)
    pk, pv = (randn(groups, kv, prefix, hd).to(cache_type) for _ in range(2))
    k, v = (randn(batch, kv, max_len, hd).to(cache_type) for _ in range(2))
    lengths, rows, counts = whole(prefix // 2, prefix, groups), whole(0, max_len - tokens, batch), whole((tokens + 1) // 2, tokens, batch)
    lengths[-1], rows[0], counts[0] = prefix, max_len - tokens, tokens
    if batch > 2:
        counts[batch // 2] = 0
    if groups > 2:
        lengths[1] = 0
    want, size = serve_plain.shared_prefix_attention_by_heads(q, pk, pv, lengths, k, v, rows, counts)
    for g in range(groups):
        pk[g, :, int(lengths[g]):], pv[g, :, int(lengths[g]):] = math.nan, math.inf
    for b in range(batch):
        last = int(rows[b]) + int(counts[b])
        k[b, :, last:], v[b, :, last:] = math.inf, math.nan
        q[b, :, int(counts[b]):] = math.nan   # (a token that is not there: zeros, and nobody else's business)
    got = attention.shared_prefix_attention(q, pk, pv, lengths, k, v, rows, counts=counts)
    _attention_near(got, want.cpu(), size.cpu())


FEW = [   # (groups, batch, tokens, heads, kv, prefix, max_len): one and two tiles of queries a wave, for the prefix and for own rows; one launch and two
    (1, 2, 1, 8, 2, 900, 70), (1, 9, 1, 8, 2, 900, 70), (1, 2, 7, 8, 2, 900, 70), (3, 6, 1, 16, 4, 700, 600), (2, 4, 5, 4, 4, 1300, 9),
    (1, 2, 1, 8, 2, 100, 70), (1, 2, 7, 8, 2, 100, 70), (1, 2, 40, 6, 1, 1000, 300),
    (1, 66, 1, 12, 12, 900, 120), (3, 33, 3, 26, 26, 700, 250), (2, 50, 20, 8, 8, 840, 33),   # a wave for itself
    (1, 66, 1, 12, 12, 100, 200), (3, 33, 20, 13, 13, 30, 90), (2, 50, 40, 8, 8, 20, 44), (1, 130, 1, 16, 16, 1, 1), (1, 20, 1, 8, 2, 900, 70), (1, 3, 12, 8, 2, 900, 70),
    (5, 60, 3, 26, 26, 700, 40), (1, 24, 9, 10, 10, 300, 500),
]
MANY = [   # tiles of 64 and of 128 queries for the prefix, of 16 and of 32 for own rows
    (1, 40, 1, 8, 2, 900, 70), (3, 33, 1, 24, 2, 1000, 300), (1, 9, 7, 8, 2, 1500, 200), (1, 130, 1, 8, 2, 8200, 40), (2, 64, 9, 8, 2, 8500, 60), (1, 97, 1, 9, 9, 900, 256), (1, 130, 1, 8, 2, 14000, 40),
    (1, 70, 1, 12, 12, 11200, 40),
]
WALK = [   # several parts and one, most rows before or in the sequences' own, odd and even numbers of blocks
    (1, 2, 70, 4, 2, 500, 900), (2, 6, 33, 8, 2, 1000, 40), (1, 16, 64, 32, 8, 700, 300), (1, 16, 90, 32, 8, 1290, 200), (2, 32, 70, 8, 4, 130, 1000),
    (1, 32, 70, 8, 4, 64, 1000), (4, 32, 70, 8, 4, 700, 700), (1, 40, 150, 8, 8, 3, 777),
]


@pytest.mark.parametrize("hd", [128, 64, 32])
@pytest.mark.parametrize("q_type", [F32, BF16])
@pytest.mark.parametrize("cache_type,case", [(t, c) for c in FEW for t in (F32, BF16)] + [(BF16, c) for c in MANY + WALK])
def test_shared_attention_tiles_and_parts(cuda, hd, q_type, cache_type, case):
    groups, batch, tokens, heads, kv, prefix, max_len = case
    _share_by_heads(cuda, groups, batch, tokens, heads, kv, hd, prefix, max_len, q_type, cache_type, seed=hd + batch + tokens)


def test_shared_attention_offsets_past_32_bits(cuda):
    """A prefix of more than 2^31 elements a head, of which the last row alone weighs; caches more than 2^31 elements apart."""
    hd, rows = 32, 2 ** 31 // 32 + 100
    keys = torch.zeros((1, 1, rows, hd), dtype=BF16, device=cuda)
    values = torch.zeros_like(keys)
    keys[0, 0, -1] = 100.0
    values[0, 0, -1] = torch.arange(hd, device=cuda).to(BF16)
    own = torch.zeros((2, 1, 2, hd), dtype=BF16, device=cuda)
    q = torch.full((2, 2, 1, hd), 1.0, device=cuda)
    got = attention.shared_prefix_attention(q, keys, values, torch.tensor([rows], device=cuda), own, own, torch.tensor([0, 1], device=cuda))
    assert torch.equal(got.view(2, 2, hd)[1, 1].cpu(), torch.arange(hd).to(BF16))
    far = keys.view(-1).as_strided((2, 1, 4, hd), (2 ** 31, 0, hd, 1))
    far_values = values.view(-1).as_strided((2, 1, 4, hd), (2 ** 31, 0, hd, 1))
    values.zero_()
    far_values[1, 0, 2] = 3.0
    far[1, 0, 2] = 100.0
    got = attention.shared_prefix_attention(q, own[:1], own[:1], torch.tensor([1], device=cuda), far, far_values, torch.tensor([3, 3], device=cuda))
    assert torch.equal(got[1].cpu(), torch.full((1, 2 * hd), 3.0).to(BF16)) and torch.equal(got[0].cpu(), torch.zeros(1, 2 * hd).to(BF16))
    norm = attention.norm_rope(torch.ones((2, 3 * hd), device=cuda), *(t.to(cuda) for t in _tables(4, hd)), far, far_values,
                               torch.tensor([1, 3], device=cuda), heads=1, positions=torch.zeros(2, dtype=torch.long, device=cuda))
    assert norm.shape == (2, 1, 1, hd)
    assert torch.equal(far_values[:, 0].float().sum(-1).cpu(), torch.tensor([[0.0, 32, 0, 0], [0, 0, 96, 32]]))


def test_shared_attention_is_repeatable_and_takes_any_stream(cuda):
    gen = torch.Generator(device=cuda).manual_seed(13)
    randn = lambda *shape: torch.randn(shape, generator=gen, device=cuda)  # noqa: E731
    q, pk, pv, k, v = randn(9, 8, 1, 128), *(randn(1, 2, 900, 128).to(BF16) for _ in range(2)), *(randn(9, 2, 77, 128).to(BF16) for _ in range(2))
    lengths, rows = torch.tensor([900], device=cuda), torch.arange(9, device=cuda) * 9
    first = attention.shared_prefix_attention(q, pk, pv, lengths, k, v, rows)
    stream = torch.cuda.Stream(device=cuda)
    stream.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(stream):
        again = [attention.shared_prefix_attention(q, pk, pv, lengths, k, v, rows) for _ in range(3)]
    stream.synchronize()
    assert all(torch.equal(first, other) for other in again)


def test_shared_attention_refuses(cuda):
    q = torch.zeros((4, 4, 1, 64), device=cuda)
    p, c = torch.zeros((2, 2, 8, 64), device=cuda), torch.zeros((4, 2, 8, 64), device=cuda)
    n, rows = torch.zeros(2, dtype=torch.long, device=cuda), torch.zeros(4, dtype=torch.long, device=cuda)
    attention.shared_prefix_attention(q, p, p, n, c, c, rows)
    odd = torch.zeros((4, 2, 8 * 64 + 4), device=cuda)[:, :, :512].unflatten(2, (8, 64))
    bad = [
        (q.half(), p, p, n, c, c, rows), (q[:3], p, p, n, c[:3], c[:3], rows[:3]), (q, p, p, n, c, c, rows[:3]), (q, p, p, n[:1], c, c, rows),
        (q, p.bfloat16(), p.bfloat16(), n, c, c, rows), (q, p[:, :1], p[:, :1], n, c, c, rows), (q[..., :48], p[..., :48], p[..., :48], n, c[..., :48], c[..., :48], rows),
        (q, p, p.clone()[:, :, :4], n, c, c, rows), (q[:, :3], p, p, n, c, c, rows), (q, p, p, n, c, c, rows.cpu()), (q.cpu(), p, p, n, c, c, rows),
        (q, p, p, n, odd, odd, rows), (q[:0], p, p, n, c[:0], c[:0], rows[:0]), (q, p[:, :, :0], p[:, :, :0], n, c, c, rows),
    ]
    for args in bad:
        with pytest.raises(ValueError, match="shared_prefix_attention|ajqs_shared_attention"):
            attention.shared_prefix_attention(*args)


# ------------------------------------------------------------------ adjust_logits
# One rounding of the penalty's quotient or product, of its count times frequency, of their sum with presence, of each addition to the logit and to
# the sum of a token's biases: at most 4 + (biases of a token) steps of 2^-24 of what is added up.
def _adjusted(cuda, batch, vocab, seed, type=F32, history=True, given=True, biases=0, mask=None, padded=0, same_bias=False, in_place=False, numbers=False,
              lengths="rows", wild=False):
    gen = _gen(seed)
    logits = (torch.randn((batch, vocab + padded), generator=gen) * 4).to(type)[:, :vocab]
    args = dict.fromkeys(("tokens", "lengths", "prompt", "prompt_lengths", "repetition", "frequency", "presence", "bias_ids", "bias", "allowed",
                          "allowed_rows"))
    low, high = (-5, vocab + 5) if wild else (0, vocab)
    if history:
        args["tokens"] = torch.randint(low, min(high, 40), (batch, 57), generator=gen)
        args["lengths"] = {"rows": torch.randint(0, 58, (batch,), generator=gen), "one": torch.tensor([23]), "all": None}[lengths]
        if numbers:
            args["repetition"], args["frequency"], args["presence"] = 1.25, 0.5, 0.25
        else:
            args["repetition"] = 0.8 + torch.rand(batch, generator=gen)
            args["frequency"], args["presence"] = torch.rand(batch, generator=gen) - 0.3, torch.rand(batch, generator=gen) - 0.3
    if given:
        args["prompt"] = torch.randint(low, high, (batch, 91), generator=gen)
        args["prompt_lengths"] = torch.randint(0, 92, (batch,), generator=gen)
    if biases:
        args["bias_ids"] = torch.randint(low, high, (batch, biases), generator=gen)
        if same_bias:
            args["bias_ids"][:, ::2] = vocab - 1
        args["bias"] = torch.randn((batch, biases), generator=gen) * 5
    if mask:
        args["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (batch + 2, (vocab + 31) // 32), generator=gen).int()
        args["allowed"][0] = 0
        if mask == "states":
            args["allowed_rows"] = torch.randint(-2, batch + 4, (batch,), generator=gen)
    want, size = serve_plain.adjust_logits(logits, **args)
    on = {k: v.to(cuda) if isinstance(v, torch.Tensor) else v for k, v in args.items()}
    there = torch.full((batch, vocab + padded), math.nan, dtype=type, device=cuda)
    there[:, :vocab] = logits.to(cuda)
    got = sampling.adjust_logits(there[:, :vocab], out=there[:, :vocab] if in_place else None, **on)
    assert got.dtype == F32 and got.shape == (batch, vocab) and (in_place or got.stride(0) % 4 == 0)
    if in_place:
        assert got.data_ptr() == there.data_ptr() and bool(torch.isnan(there[:, vocab:]).all())
    else:
        assert torch.equal(there[:, :vocab].cpu(), logits)
    got = got.double().cpu()
    assert torch.equal(torch.isinf(got), torch.isinf(want))
    off = torch.where(torch.isinf(want), 0.0, (got - want).abs())
    assert bool((off <= (4 + biases) * 2.0 ** -24 * size).all()), float((off / size).max())


@pytest.mark.parametrize("vocab", [1, 3, 31, 32, 33, 1000, 8191, 8192, 8193, 32011])
@pytest.mark.parametrize("type", [F32, BF16])
def test_adjust_logits_vocabularies(cuda, vocab, type):
    _adjusted(cuda, 3, vocab, seed=vocab, type=type, biases=5, mask="rows", wild=True)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("history,given,biases,mask", [(True, False, 0, None), (False, True, 0, None), (False, False, 7, None), (False, False, 0, "rows"),
                                                       (False, False, 0, "states"), (True, True, 9, "states"), (False, False, 0, None)])
def test_adjust_logits_parts(cuda, in_place, history, given, biases, mask):
    _adjusted(cuda, 5, 2000, seed=biases, history=history, given=given, biases=biases, mask=mask, in_place=in_place)


@pytest.mark.parametrize("padded", [1, 2, 3, 4, 12])
@pytest.mark.parametrize("type", [F32, BF16])
def test_adjust_logits_strides(cuda, padded, type):
    _adjusted(cuda, 4, 1021, seed=padded, type=type, biases=3, mask="rows", padded=padded, in_place=type == F32 and padded != 4)


def test_adjust_logits_lengths_numbers_and_repeated_biases(cuda):
    _adjusted(cuda, 4, 500, seed=1, lengths="one", numbers=True)
    _adjusted(cuda, 4, 500, seed=2, lengths="all", numbers=True, wild=True)
    _adjusted(cuda, 1, 500, seed=3, lengths="one", biases=1)
    _adjusted(cuda, 2, 500, seed=4, biases=300, same_bias=True, wild=True)
    _adjusted(cuda, 2, 9000, seed=5, biases=1024, same_bias=True)


def test_adjust_logits_special_values(cuda):
    """Masked NaN and infinities are -inf; what is allowed stays what it is; a mask that leaves nothing leaves -inf."""
    logits = torch.tensor([[math.nan, math.inf, -math.inf, 1.0, -3.4e38, 0.0, -0.0, 2.0]], device=cuda).repeat(3, 1)
    allowed = torch.tensor([[0b10101010], [0b01111110], [0]], dtype=torch.int32, device=cuda)
    got = sampling.adjust_logits(logits, allowed=allowed).cpu()
    assert torch.equal(got[0], torch.tensor([-math.inf, math.inf, -math.inf, 1.0, -math.inf, 0.0, -math.inf, 2.0]))
    assert torch.equal(got[1], torch.tensor([-math.inf, math.inf, -math.inf, 1.0, -3.4e38, 0.0, -0.0, -math.inf]))
    assert torch.equal(got[2], torch.full((8,), -math.inf))
    got = sampling.adjust_logits(logits, tokens=torch.arange(8, device=cuda).repeat(3, 1), repetition=2.0).cpu()
    assert torch.equal(got[0, 1:], torch.tensor([math.inf, -math.inf, 0.5, -math.inf, 0.0, 0.0, 1.0])) and bool(torch.isnan(got[0, 0]))


def test_adjust_logits_a_long_history_of_one_token(cuda):
    """Counts of a hundred thousand are whole numbers."""
    logits = torch.zeros((2, 70), device=cuda)
    tokens = torch.full((2, 100003), 69, dtype=torch.long, device=cuda)
    got = sampling.adjust_logits(logits, tokens=tokens, lengths=torch.tensor([100003, 7], device=cuda), frequency=1.0)
    assert got[:, 69].tolist() == [-100003.0, -7.0] and float(got[:, :69].abs().max()) == 0


def test_adjust_logits_refuses(cuda):
    x = torch.zeros((2, 64), device=cuda)
    ids, f = torch.zeros((2, 3), dtype=torch.long, device=cuda), torch.zeros((2, 3), device=cuda)
    mask = torch.zeros((2, 2), dtype=torch.int32, device=cuda)
    big = torch.zeros((2, 1025), device=cuda)
    bad = [
        (x.half(), {}), (x[0], {}), (x.cpu(), {}), (x[:, :0], {}), (x.t(), {}), (x, dict(tokens=ids[:1])), (x, dict(tokens=ids.int())), (x, dict(lengths=ids[:, 0])),
        (x, dict(tokens=ids, lengths=ids.view(-1))), (x, dict(bias=f)), (x, dict(bias=f, bias_ids=ids[:, :2])), (x, dict(bias=big, bias_ids=big.long())),
        (x, dict(allowed=mask[:, :1])), (x, dict(allowed=mask[:1])), (x, dict(allowed=mask.long())), (x, dict(allowed_rows=ids[:, 0].contiguous())),
        (x, dict(out=x.bfloat16())), (x, dict(out=x[:1])), (x.bfloat16(), dict(out=x[:, :32])), (x, dict(repetition=f[:, 0])), (x, dict(prompt=ids.cpu())),
        (x, dict(out=x[:1].expand(2, 64))),
    ]
    for logits, more in bad:
        with pytest.raises(ValueError, match="adjust_logits"):
            sampling.adjust_logits(logits, **more)


# ------------------------------------------------------------------ the three together
def _step(state):
    """One decode step of a batch that shares a prefix, without its linears: rotation, attention, a head, adjusted logits, the choice."""
    s = state
    q = attention.norm_rope(s["qkv"], s["cosine"], s["sine"], s["keys"], s["values"], s["rows"], heads=8, q_gain=s["gain"], k_gain=s["gain"],
                            positions=s["positions"], offset=s["step"])
    out = attention.shared_prefix_attention(q, s["pk"], s["pv"], s["lengths"], s["keys"], s["values"], s["rows"], offset=s["step"])
    logits = (out[:, 0].float().unsqueeze(1) * s["head"]).sum(-1)
    sampling.adjust_logits(logits, tokens=s["out"], lengths=s["step"], repetition=s["penalty"], out=logits)
    token = logits.argmax(-1, keepdim=True)
    s["out"].scatter_(1, s["step"].expand(6, 1), token)
    s["qkv"].copy_(s["table"][token.view(-1)])
    s["step"].add_(1)
    return logits


def _fresh(cuda, seed):
    gen = torch.Generator(device=cuda).manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=gen, device=cuda)  # noqa: E731
    hd = 64
    cosine, sine = (t.to(cuda) for t in _tables(200, hd))
    rows = torch.tensor([0, 3, 1, 7, 0, 2], device=cuda)
    return dict(qkv=randn(6, 12 * hd), table=randn(50, 12 * hd), head=randn(50, 8 * hd), cosine=cosine, sine=sine, gain=1 + 0.1 * randn(hd),
                keys=randn(6, 2, 40, hd).to(BF16), values=randn(6, 2, 40, hd).to(BF16), pk=randn(2, 2, 100, hd).to(BF16), pv=randn(2, 2, 100, hd).to(BF16),
                lengths=torch.tensor([100, 61], device=cuda), rows=rows, positions=rows + 100, step=torch.zeros(1, dtype=torch.long, device=cuda),
                out=torch.zeros((6, 32), dtype=torch.long, device=cuda), penalty=torch.full((6,), 1.3, device=cuda))


def test_two_captured_steps_replay_as_eager_ones(cuda):
    """Two graphs with states of their own, replayed in turns with eager work between, against eager steps, every replay looked at."""
    eager = [_fresh(cuda, 1), _fresh(cuda, 2)]
    want = [[_step(s).clone() for _ in range(6)] for s in eager]
    states = [_fresh(cuda, 1), _fresh(cuda, 2)]
    graphs = []
    for s, w in zip(states, want):
        stream = torch.cuda.Stream(device=cuda)
        stream.wait_stream(torch.cuda.current_stream(cuda))
        with torch.cuda.stream(stream):
            assert torch.equal(_step(s), w[0])
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                logits = _step(s)
        torch.cuda.current_stream(cuda).wait_stream(stream)
        graphs.append((graph, logits))
    for i in range(1, 6):
        for (graph, logits), w in zip(graphs, want):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(logits, w[i]), i
            _step(_fresh(cuda, 3))
    for s, e in zip(states, eager):
        assert torch.equal(s["out"], e["out"]) and torch.equal(s["keys"], e["keys"])


def test_general_path_gives_the_same_bits(cuda, monkeypatch):
    """Without the extension module, under a mode that looks on, and where its functions leave a call to the lines behind them."""
    from ajllm_amd import _lib

    def everything():
        s = _fresh(cuda, 5)
        q = attention.norm_rope(s["qkv"], s["cosine"], s["sine"], s["keys"], s["values"], s["rows"], heads=8, k_gain=s["gain"], offset=s["step"],
                                out_dtype=BF16)
        out = attention.shared_prefix_attention(q, s["pk"], s["pv"], s["lengths"], s["keys"], s["values"], s["rows"])
        logits = sampling.adjust_logits(out.view(6, 512)[:, 1:], tokens=s["out"], lengths=s["step"], presence=s["penalty"])
        into = torch.zeros((6, 511), device=cuda)
        assert sampling.adjust_logits(out.view(6, 512)[:, 1:], out=into, bias_ids=s["out"], bias=torch.ones((6, 32), device=cuda)) is into
        return q, s["keys"], s["values"], out, logits, into

    def same(a, b):
        return all(torch.equal(x, y) for x, y in zip(a, b))

    fast = everything()
    strided = torch.zeros((6, 8, 2, 64), dtype=BF16, device=cuda)[:, :, :1]
    strided.copy_(fast[0])
    s = _fresh(cuda, 5)
    assert torch.equal(attention.shared_prefix_attention(strided, s["pk"], s["pv"], s["lengths"], fast[1], fast[2], s["rows"]), fast[3])
    with torch.overrides.BaseTorchFunctionMode():
        assert same(fast, everything())
    calls = []
    for name in ("norm_rope", "shared_prefix_attention", "adjust_logits"):
        monkeypatch.setitem(_lib._serve_native, name, lambda *a, name=name: calls.append(name))
    assert same(fast, everything()) and calls == ["norm_rope", "shared_prefix_attention", "adjust_logits", "adjust_logits"]
