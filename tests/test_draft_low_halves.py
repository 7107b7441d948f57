"""tree_attention takes fp32 queries and rows with sixteen bits at least (include/ajq_draft.h), two bf16 numbers each on most of its ways: the inputs of
test_serve_low_halves.py, whose upper halves cancel or are all alike, behind masks of trees, in every form that meets fp32 numbers."""

import math

import pytest
import torch

from ajllm_amd import attention
from tests import draft_plain
from tests.test_gpu_draft_forms import CALLS as FORMS
from tests.test_serve_low_halves import BF16, F32, _bf16, _inputs

CALLS = [(kind, *call) for call in FORMS for kind in (["values", "keys"] if not call[7] else []) + (["queries"] if not call[6] else [])]


def _case(kind, batch, nodes, heads, kv, hd, max_len):
    """(q, keys, values, rows, counts, masks) in float64, and what the values weigh where a pair's are taken together.  Rows come in pairs of one key: an even number is
    committed, and a token that sees one row of a pair of the tokens' own sees the other (``values``)."""
    fits, seed = max(max_len - nodes, 0), batch + 3 * nodes + hd + max_len
    (q, _, _, _, k, v, before, counts), (_, weigh) = _inputs(kind, 1, batch, nodes, heads, kv, hd, 2, max_len + nodes, seed)
    k, v, weigh = k[:, :, :max_len], v[:, :, :max_len], weigh[:, :, :max_len]
    before = before.clamp(max=fits // 2 * 2)
    before[0], counts[0] = fits // 2 * 2, nodes
    gen = torch.Generator().manual_seed(seed)
    at = torch.arange(nodes)
    masks = attention.tree_masks((at - 1 - torch.randint(0, 5, (batch, nodes), generator=gen)).clamp(min=0).masked_fill(at == 0, -1))[0]
    if kind == "values":
        even = masks & 0x55555555
        masks = even | even << 1
        part = 0.4 * (2.0 * torch.randint(0, 2, (batch, kv, 1, hd), generator=gen) - 1) * (0.5 + 0.5 * torch.rand((batch, kv, (max_len + 1) // 2, hd), generator=gen)).double()
        v = torch.stack((256.5 + part, -(256.5 - part)), dim=3).flatten(2, 3)[:, :, :max_len].float().double()
        weigh = part.abs().repeat_interleave(2, dim=2)[:, :, :max_len]
        for b in range(batch):   # (a row that has no other)
            alone = min(int(before[b] + counts[b]), max_len) // 2 * 2
            v[b, :, alone:], weigh[b, :, alone:] = 0.5, 0.5
    return (q, k, v, before, counts, masks), weigh


def _bound(case, weigh, kind, device):
    """(exact result, largest error), as test_serve_low_halves.py has it."""
    q, k, v, before, counts, masks = case
    hd, n = q.shape[3], k.shape[2]
    on = [t.to(device) for t in (q, k)]
    want, full = draft_plain.tree_attention(*on, v.to(device), before, masks, counts, 0)
    _, together = draft_plain.tree_attention(*on, weigh.to(device), before, masks, counts, 0)
    largest = float(k.abs().sum(-1).max())                                          # of a row's components together
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


def _emulated(case, q_type, cache_type, drop):
    """The two halves in 64 bits, with or without (``drop``) the lower ones."""
    q, k, v, before, counts, masks = case

    def taken(x, type):
        hi = _bf16(x)
        return hi if drop or type == BF16 else hi + _bf16(x - hi)

    return _bf16(draft_plain.tree_attention(taken(q, q_type), taken(k, cache_type), taken(v, cache_type), before, masks, counts, 0)[0])


@pytest.mark.parametrize("kind", ["queries", "keys", "values"])
@pytest.mark.parametrize("hd", [128, 64, 32])
@pytest.mark.parametrize("shape", [(2, 9, 8, 2, 300), (3, 40, 4, 2, 41), (2, 1, 4, 4, 700)])
def test_the_bound_tells_lower_halves_from_none(kind, hd, shape):
    """Without the lower halves most results miss the bound, with them all keep it: what is asked of the kernels below can fail."""
    batch, nodes, heads, kv, max_len = shape
    case, weigh = _case(kind, batch, nodes, heads, kv, hd, max_len)
    want, bound = _bound(case, weigh, kind, "cpu")
    there = (torch.arange(nodes) < case[4][:, None])[:, :, None]
    kept, lost = (_emulated(case, F32, F32, drop) - want for drop in (False, True))
    assert bool((kept.abs() <= bound).all()), float((kept.abs() / bound.clamp(min=1e-300)).max())
    missed = (lost.abs() > 2 * bound) & there
    assert float(missed.sum() / there.expand_as(missed).sum()) > 0.5


@pytest.mark.gpu
@pytest.mark.parametrize("kind,batch,nodes,heads,kv,hd,max_len,q_bf16,cache_bf16", CALLS)
def test_tree_attention_keeps_lower_halves(cuda, kind, batch, nodes, heads, kv, hd, max_len, q_bf16, cache_bf16):
    case, weigh = _case(kind, batch, nodes, heads, kv, hd, max_len)
    want, bound = _bound(case, weigh, kind, cuda)
    q, k, v, before, counts, masks = case
    given = [torch.empty(x.shape, dtype=BF16 if bf16 else F32).copy_(x) for x, bf16 in ((q, q_bf16), (k, cache_bf16), (v, cache_bf16))]
    for exact, x in zip((q, k, v), given):
        assert torch.equal(exact, x.double())   # (nothing is lost on the way in)
    for b in range(batch):
        last = min(int(before[b]) + int(counts[b]), max_len)
        given[1][b, :, last:], given[2][b, :, last:] = math.inf, math.nan
    on = [t.to(cuda) for t in (*given, before, masks)]
    got = attention.tree_attention(*on, counts=counts.to(cuda))
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound.clamp(min=1e-300)).max())
