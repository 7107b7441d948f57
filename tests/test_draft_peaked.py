"""Tree attention in all its forms on inputs that make single rows matter, however many there are.

Of normal scores a row of 100000 weighs 1 / 100000, and a result says nothing of it.  Here one committed row of every 32 (of more than 8192: 256 of them, spread evenly) and
the tokens' own rows have scores that lift them, together, above all others, each by a weight of its own, and a component has values from every sixteenth of them alone: a row
that is lost, or seen where it should not be, moves some component by percents.  The first test shows that on the CPU, with mistakes planted in the definition, for every
call that the second makes."""

import math

import pytest
import torch

from ajllm_amd import attention
from tests import draft_plain
from tests.test_gpu_draft_forms import CALLS

BF16 = torch.bfloat16
F32 = torch.float32
GROUPS, MOST = 16, 256


def _masks(gen, batch, nodes):
    """Trees; every third token does not see itself (of a single one, that of every second sequence)."""
    at = torch.arange(nodes)
    masks = attention.tree_masks((at - 1 - torch.randint(0, 5, (batch, nodes), generator=gen)).clamp(min=0).masked_fill(at == 0, -1))[0]
    blind = (at % 3 == 2).expand(batch, nodes) if nodes > 1 else (torch.arange(batch) % 2 == 0)[:, None]
    own = torch.where(at % 32 == 31, torch.tensor(-2 ** 31), 1 << (at % 32).clamp(max=30)).int()
    words = masks.gather(2, (at // 32)[None, :, None].expand(batch, nodes, 1))
    return masks.scatter(2, (at // 32)[None, :, None].expand(batch, nodes, 1), torch.where(blind[:, :, None], words & ~own[None, :, None], words))


def _inputs(gen, batch, nodes, heads, kv, hd, max_len, rows, counts, q_type, cache_type):
    """(q, keys, values) of the types, and for each sequence its planted committed rows."""
    share = heads // kv
    randn = lambda *shape: torch.randn(shape, generator=gen)  # noqa: E731
    u = 2.0 * torch.randint(0, 2, (kv, hd), generator=gen) - 1                                      # a key head's direction
    across = lambda x, u: x - (x * u).sum(-1, keepdim=True) / hd * u                                # noqa: E731
    q = (u[:, None, None] + across(randn(batch, kv, share, nodes, hd), u[:, None, None])).view(batch, heads, nodes, hd)
    keys, values = across(randn(batch, kv, max_len, hd), u[:, None]), 0.5 * randn(batch, kv, max_len, hd)
    planted = []
    for b in range(batch):
        last = min(rows[b] + counts[b], max_len)
        committed = min(rows[b], last)
        many = min(MOST, (committed + 31) // 32)
        edges = [committed * i // many for i in range(many + 1)] if many else []
        some = [low + int(torch.randint(0, high - low, (1,), generator=gen)) for low, high in zip(edges, edges[1:])]
        planted.append(some)
        at = torch.tensor(some + list(range(committed, last)), dtype=torch.long)
        if not len(at):
            continue
        seen = many + min(last - committed, 1 + nodes // 3)                                         # (about what a token sees of them)
        lift = math.log(max(1.0, 4 * (committed - many) / seen))
        keys[b, :, at] = 0.5 * keys[b, :, at] + lift / math.sqrt(hd) * u[:, None]
        of = (torch.arange(hd) % GROUPS == (torch.arange(len(at)) % GROUPS)[:, None])
        values[b, :, at] = torch.where(of, (1 + torch.rand((kv, len(at), hd), generator=gen)) * (2 * torch.randint(0, 2, (kv, len(at), hd), generator=gen) - 1), 0.0)
    return q.to(q_type), keys.to(cache_type), values.to(cache_type), planted


def _seen(table, rows, count, max_len, device):
    """[count, last]: which rows the tokens that are there see."""
    last = min(rows + count, max_len)
    node = torch.arange(last) - rows
    return torch.where(node < 0, True, table[:count][:, node.clamp(0, table.shape[1] - 1)]).to(device)


# A weight is off by its rounding to bf16 (2^-8), by 2^-10 for its exponential and the sums, and by what its score and the weights' sum are: with e the largest error of a score by
# e^2e - 1 of v - out.  A score's factors are bf16 numbers as they are, or two halves (off by 2^-16 of themselves, and 2^-16 for the product of two lower ones), its
# sum has 2 hd additions.  Values are two halves likewise, the result is rounded by 2^-8.
def _define(q, keys, values, seen):
    """(out, bound) of a key head's queries [share, count, hd] over rows [last, hd], in 64 bits."""
    share, count, hd = q.shape
    halves = (q.dtype == F32) + (keys.dtype == F32)
    x, k, v = q.double().reshape(-1, hd), keys.double(), values.double()
    seen = seen.repeat(share, 1)
    scores = (x @ k.t().contiguous() / math.sqrt(hd)).masked_fill(~seen, -math.inf)
    w = torch.softmax(scores, dim=-1).masked_fill(~seen.any(1, keepdim=True), 0.0)
    out, size = w @ v, w @ v.abs()
    sizes = (x.abs() @ k.abs().t().contiguous() / math.sqrt(hd)).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
    off = ((0, 1, 3)[halves] * 2.0 ** -16 + 2 * hd * 2.0 ** -24) * sizes
    bound = (2.0 ** -8 + 2.0 ** -10 + 2.0 ** -16) * size + torch.expm1(2 * off) * (size + out.abs()) + 2.0 ** -8 * out.abs()
    return out.view(share, count, hd), bound.view(share, count, hd)


def _seed(nodes, heads, hd, max_len, q_bf16, cache_bf16):
    return 7 * nodes + 11 * heads + 13 * hd + max_len + 2 * q_bf16 + cache_bf16


@pytest.mark.parametrize("batch,nodes,heads,kv,hd,max_len,q_bf16,cache_bf16", CALLS)
def test_mistakes_break_the_bound(batch, nodes, heads, kv, hd, max_len, q_bf16, cache_bf16):
    """Of each call a key head of its longest sequence: masks that are not looked at, one bit of a mask, a block of 32 rows, a 64th of the rows."""
    gen = torch.Generator().manual_seed(_seed(nodes, heads, hd, max_len, q_bf16, cache_bf16))
    rows, share = max(max_len - nodes, 0), heads // kv
    masks = _masks(gen, 1, nodes)
    q, keys, values, planted = _inputs(gen, 1, nodes, share, 1, hd, max_len, [rows], [nodes], BF16 if q_bf16 else F32, BF16 if cache_bf16 else F32)
    table = draft_plain.sees(masks, 1, nodes)[0]
    some = torch.arange(nodes)[-min(nodes, 16):]                                                    # (tokens: enough for what is to be shown)
    q = q[0][:, some]
    seen = _seen(table, rows, nodes, max_len, "cpu")[some]
    last = seen.shape[1]
    want, bound = _define(q, keys[0, 0, :last], values[0, 0, :last], seen)

    def rejected(what, wrong):
        off = (_define(q, keys[0, 0, :last], values[0, 0, :last], wrong)[0] - want).abs()
        assert float((off / bound.clamp(min=1e-300)).max()) > 1.5, what

    everything = seen.clone()
    everything[:, rows:] = True
    rejected("masks", everything)
    for t in (0, len(some) - 1):
        of = seen[t, rows:].nonzero()[:, 0]
        one = seen.clone()
        one[t, rows + (int(of[len(of) // 2]) if len(of) else 0)] ^= True
        rejected("a bit of a mask", one)
    places = planted[0] or list(range(min(last, 32)))
    for place in {places[0], places[len(places) // 2], places[-1]}:
        less = seen.clone()
        less[:, place & ~31:(place & ~31) + 32] = False
        rejected("a block", less)
    per = ((last + 63) // 64 + 31) & ~31
    for part in {0, (last - 1) // per // 2, (last - 1) // per}:
        less = seen.clone()
        less[:, part * per:(part + 1) * per] = False
        rejected("a part", less)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,nodes,heads,kv,hd,max_len,q_bf16,cache_bf16", CALLS)
def test_single_rows_matter(cuda, batch, nodes, heads, kv, hd, max_len, q_bf16, cache_bf16):
    gen = torch.Generator().manual_seed(_seed(nodes, heads, hd, max_len, q_bf16, cache_bf16))
    fits, share = max(max_len - nodes, 0), heads // kv
    rows = [fits] + torch.randint(0, fits + 1, (batch,), generator=gen).tolist()[1:]
    counts = [nodes] + torch.randint(0, nodes + 1, (batch,), generator=gen).tolist()[1:]
    masks = _masks(gen, batch, nodes)
    q, keys, values, _ = _inputs(gen, batch, nodes, heads, kv, hd, max_len, rows, counts, BF16 if q_bf16 else F32, BF16 if cache_bf16 else F32)
    for b in range(batch):   # (rows behind the tokens that are there)
        last = min(rows[b] + counts[b], max_len)
        keys[b, :, last:], values[b, :, last:] = math.inf, math.nan
    q, keys, values = q.to(cuda), keys.to(cuda), values.to(cuda)
    got = attention.tree_attention(q, keys, values, torch.tensor(rows, device=cuda), masks.to(cuda), counts=torch.tensor(counts, device=cuda)).view(batch, nodes, heads, hd)
    tables, worst = draft_plain.sees(masks, batch, nodes), []
    for b in range(batch):
        assert not bool(got[b, counts[b]:].any())
        if counts[b] == 0:
            continue
        seen = _seen(tables[b], rows[b], counts[b], max_len, cuda)
        for k in range(kv):
            of = slice(k * share, (k + 1) * share)
            want, bound = _define(q[b, of, :counts[b]], keys[b, k, :seen.shape[1]], values[b, k, :seen.shape[1]], seen)
            off = (got[b, :counts[b], of].transpose(0, 1).double() - want).abs()
            worst.append((off / bound.clamp(min=1e-300)).max())
    assert float(torch.stack(worst).max()) <= 1.0
