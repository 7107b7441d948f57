"""shared_prefix_attention takes fp32 queries and rows with sixteen bits at least (include/ajq_serve.h), two bf16 numbers each on most of its paths: inputs whose upper
halves cancel, or are all alike, so that the lower ones alone make the result.

One kind of input carries the result in its lower halves, as 256 + d with 0 < d < 1 (upper half 256, lower half d to eight bits); the others are bf16 numbers.

* ``queries``: pairs of components 256 + d, 256 + d' against keys a, -a: a score is the sum of a (d - d').
* ``keys``: the same the other way round.
* ``values``: rows in pairs of one key (and so of one weight, to the last bit: a block holds both) with values 256 + d, -(256 + d')."""

import math

import pytest
import torch

from ajllm_amd import attention
from tests import serve_plain

BF16 = torch.bfloat16
F32 = torch.float32


def _bf16(x):
    return x.to(BF16).double()


def _inputs(kind, groups, batch, tokens, heads, kv, hd, prefix, max_len, seed):
    """(q, prefix keys, prefix values, lengths, keys, values, rows, counts) in float64, and what the values weigh where a pair's are taken together."""
    gen = torch.Generator().manual_seed(seed)
    uniform = lambda *shape: torch.rand(shape, generator=gen, dtype=torch.float64)  # noqa: E731
    randn = lambda *shape: torch.randn(shape, generator=gen, dtype=torch.float64)  # noqa: E731
    sign = lambda *shape: 2.0 * torch.randint(0, 2, shape, generator=gen).double() - 1  # noqa: E731
    pattern = sign(kv, hd // 2)                                           # of a key head's pairs, in its queries and its keys
    slope = sign(batch, kv, heads // kv, tokens) * (0.5 + 0.5 * uniform(batch, kv, heads // kv, tokens))
    size = 0.5 if hd == 128 else 1.0

    def pairs(x, low):   # of components: x, -x, or 256 + d, 256 + d' with d - d' = 0.9 x
        both = torch.stack((x, -x), dim=-1)
        return (256 + 0.5 + 0.45 * both if low else _bf16(size * both)).flatten(-2)

    q = pairs(slope[..., None] * pattern[None, :, None, None], kind == "queries").view(batch, heads, tokens, hd)

    def rows(n, count, paired):
        at = (2 * uniform(n, kv, (count + 1) // 2) - 1).repeat_interleave(2, dim=2)[:, :, :count]   # where a row's scores are
        keys = pairs(at[..., None] * pattern[None, :, None], kind == "keys")
        values = _bf16(at[..., None] * sign(n, kv, 1, hd) + 0.2 * randn(n, kv, count, hd))
        weigh = values.abs()
        if kind == "values":
            part = 0.4 * sign(n, kv, 1, hd) * (0.5 + 0.5 * uniform(n, kv, (count + 1) // 2, hd))
            both = torch.stack((256.5 + part, -(256.5 - part)), dim=3).flatten(2, 3)[:, :, :count]
            there = (torch.arange(count) < paired[:, None])[:, None, :, None]
            values = torch.where(there, both, values)
            weigh = torch.where(there, part.abs().repeat_interleave(2, dim=2)[:, :, :count], weigh)
        return keys.float().double(), values.float().double(), weigh

    even = lambda low, high, n: 2 * torch.randint(low // 2, high // 2 + 1, (n,), generator=gen)  # noqa: E731
    lengths, before = even(prefix // 2 + 1, prefix, groups), even(0, max_len - tokens, batch)
    counts = torch.randint((tokens + 1) // 2, tokens + 1, (batch,), generator=gen)
    pk, pv, pw = rows(groups, prefix, lengths)
    k, v, w = rows(batch, max_len, before)
    return (q.float().double(), pk, pv, lengths, k, v, before, counts), (pw, w)


def _bound(inputs, weigh, kind, device):
    """(exact result, largest error), float64.  With e the largest error of a score, weights are off by e^2e - 1; the other terms are a weight's rounding to bf16 and 2^-10 for
    its exponential and sum, as in the operators' other tests, the fp32 sums over the rows, the rounding of the values' lower halves, and the result's."""
    q, pk, pv, lengths, k, v, before, counts = inputs
    hd, n = q.shape[3], pk.shape[2] + k.shape[2]
    args = [t.to(device) for t in (lengths, before, counts)]
    on = lambda pv, v: serve_plain.shared_prefix_attention_by_heads(q.to(device), pk.to(device), pv.to(device), args[0], k.to(device), v.to(device), args[1], args[2])  # noqa: E731
    want, full = on(pv, v)
    together, _ = on(weigh[0], weigh[1])
    largest = max(float(pk.abs().sum(-1).max()), float(k.abs().sum(-1).max()))      # of a row's components together
    score = 2 * hd * 2.0 ** -24 * float(q.abs().max()) * largest                    # 2 hd additions of at most the sum of all terms' sizes
    if kind == "queries":
        score += 2.0 ** -9 * largest                                                # of each component's lower half, which is below 1
    if kind == "keys":
        score += 2.0 ** -9 * float(q.abs().sum(-1).max())
    score /= math.sqrt(hd)
    bound = (2.0 ** -8 + 2.0 ** -10) * together + math.expm1(2 * score) * (together + want.abs()) + n * 2.0 ** -24 * full + 2.0 ** -8 * want.abs()
    if kind == "values":
        bound = bound + 2.0 ** -9
    return want, bound


def _emulated(inputs, q_type, cache_type, drop):
    """The arithmetic of the two halves in float64, with or without (``drop``) the lower ones."""
    q, pk, pv, lengths, k, v, before, counts = inputs
    batch, heads, tokens, hd = q.shape
    kv, each = k.shape[1], batch // pk.shape[0]
    share = heads // kv

    def halves(x, type):
        hi = _bf16(x)
        return hi, torch.zeros_like(hi) if drop or type == BF16 else _bf16(x - hi)

    out = torch.zeros(batch, tokens, heads, hd, dtype=torch.float64)
    for b in range(batch):
        for h in range(kv):
            n = int(lengths[b // each])
            for t in range(int(counts[b])):
                own = int(before[b]) + t + 1
                kh, kl = halves(torch.cat((pk[b // each, h, :n], k[b, h, :own])), cache_type)
                vh, vl = halves(torch.cat((pv[b // each, h, :n], v[b, h, :own])), cache_type)
                qh, ql = halves(q[b, h * share:(h + 1) * share, t], q_type)
                s = (qh @ kh.t() + qh @ kl.t() + ql @ kh.t()) / math.sqrt(hd)
                w = torch.exp(s - s.amax(-1, keepdim=True))
                p = _bf16(w)
                out[b, t, h * share:(h + 1) * share] = (p @ vh + p @ vl) / w.sum(-1, keepdim=True)
    return _bf16(out.view(batch, tokens, heads * hd))


@pytest.mark.parametrize("kind", ["queries", "keys", "values"])
@pytest.mark.parametrize("hd", [128, 64, 32])
@pytest.mark.parametrize("shape", [(1, 2, 1, 8, 2), (2, 4, 3, 4, 4)])
def test_the_bound_tells_lower_halves_from_none(kind, hd, shape):
    """Without the lower halves the inputs miss the bound many times over, with them they keep it: what is asked of the kernels below can fail."""
    inputs, weigh = _inputs(kind, *shape, hd, 900, 70, seed=hd)
    want, bound = _bound(inputs, weigh, kind, "cpu")
    there = (torch.arange(shape[2]) < inputs[-1][:, None])[:, :, None]   # tokens that are there
    kept = (_emulated(inputs, F32, F32, drop=False) - want).abs()
    lost = (_emulated(inputs, F32, F32, drop=True) - want).abs()
    assert bool((kept <= bound).all()), float((kept / bound.clamp(min=1e-300)).max())
    missed = (lost > 2 * bound) & there
    assert float(missed.sum() / there.expand_as(missed).sum()) > 0.5


# (groups, batch, tokens, heads, kv, prefix, max_len)
F32_ROWS = [   # one launch, by workgroups and by waves; parts of tiles of 16, of 32 and 16, of 32, and by waves
    (1, 2, 1, 8, 2, 100, 70), (1, 66, 1, 12, 12, 100, 60), (1, 2, 1, 8, 2, 900, 70), (1, 9, 1, 8, 2, 900, 70), (1, 2, 40, 6, 1, 1000, 300), (1, 66, 1, 12, 12, 900, 120),
    (2, 50, 20, 8, 8, 840, 34),
]
BF16_ROWS = [  # one launch; tiles of 16, of 32; many, by 64 and by 128; the walk in parts and whole
    (1, 2, 1, 8, 2, 100, 70), (1, 2, 1, 8, 2, 900, 70), (1, 20, 1, 8, 2, 900, 70), (1, 40, 1, 8, 2, 900, 70), (1, 130, 1, 8, 2, 14000, 40), (1, 2, 70, 4, 2, 500, 900),
    (1, 32, 70, 8, 4, 64, 1000), (4, 32, 70, 8, 4, 700, 700),
]
CALLS = ([(kind, q_type, F32, shape) for shape in F32_ROWS for kind, q_type in (("queries", F32), ("keys", F32), ("keys", BF16), ("values", F32), ("values", BF16))]
         + [("queries", F32, BF16, shape) for shape in BF16_ROWS])


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [128, 64, 32])
@pytest.mark.parametrize("kind,q_type,cache_type,shape", CALLS)
def test_shared_attention_keeps_lower_halves(cuda, hd, kind, q_type, cache_type, shape):
    groups, batch, tokens, heads, kv, prefix, max_len = shape
    inputs, weigh = _inputs(kind, *shape[:5], hd, prefix, max_len, seed=hd + batch + tokens)
    want, bound = _bound(inputs, weigh, kind, cuda)
    q, pk, pv, lengths, k, v, before, counts = inputs
    q, pk, pv, k, v = q.to(q_type), pk.to(cache_type), pv.to(cache_type), k.to(cache_type), v.to(cache_type)
    for exact, given in zip((inputs[0], inputs[1], inputs[2], inputs[4], inputs[5]), (q, pk, pv, k, v)):
        assert torch.equal(exact, given.double())   # (nothing is lost on the way in)
    for g in range(groups):   # rows that nobody sees
        pk[g, :, int(lengths[g]):], pv[g, :, int(lengths[g]):] = math.nan, math.inf
    for b in range(batch):
        last = int(before[b]) + int(counts[b])
        k[b, :, last:], v[b, :, last:] = math.inf, math.nan
    on = [t.to(cuda) for t in (q, pk, pv, lengths, k, v, before)]
    got = attention.shared_prefix_attention(*on, counts=counts.to(cuda))
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound.clamp(min=1e-300)).max())
