"""The operators of checking drafted tokens (include/ajq_draft.h) against their definitions in 64 bits."""

import math

import pytest
import torch

from ajllm_amd import attention, sampling
from tests import draft_plain

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
F32 = torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _tree(gen, nodes, batch=None, reach=5):
    """Random parents, each a few places ahead at most."""
    shape = (nodes,) if batch is None else (batch, nodes)
    at = torch.arange(nodes)
    return (at - 1 - torch.randint(0, reach, shape, generator=gen)).clamp(min=0).masked_fill(at == 0, -1)


# ------------------------------------------------------------------ tree_attention
# A weight is rounded to bf16 for the second product (2^-8 of it) and comes from a score whose factors have at least 16 bits; the sums are fp32.
# Together at most (2^-8 + 2^-10) of the weighted mean size of the values; the result is rounded by 2^-8 of itself.
def _attend(cuda, batch, nodes, heads, kv, hd, max_len, q_type, cache_type, seed, rows=None, counts=None, ragged=True, offset=None, masks=None,
            spread=0, scale=1.0, garbage=True, one_tree=False, mask_words=None):
    gen = _gen(seed)
    q = (scale * torch.randn((batch, heads, nodes, hd), generator=gen)).to(q_type).to(cuda)
    rows = torch.randint(0, max(1, max_len - nodes + 1), (batch,), generator=gen) if rows is None else torch.tensor(rows)
    whole = torch.randn((2, batch, kv, max_len + spread, hd), generator=gen).to(cache_type).to(cuda)
    keys, values = whole[0, :, :, :max_len], whole[1, :, :, :max_len]
    if counts is None and ragged:
        counts = torch.randint(0, nodes + 1, (batch,), generator=gen)
    elif counts is not None:
        counts = torch.tensor(counts)
    if masks is None:
        masks = attention.tree_masks(_tree(gen, nodes, None if one_tree else batch))[0]
    if mask_words:
        masks = torch.nn.functional.pad(masks, (0, mask_words - masks.shape[-1]), value=-1)   # (words beyond the tokens': never read as tokens)
    if garbage:   # rows behind what any token sees
        for b in range(batch):
            last = int(rows[b]) + (offset or 0) + (nodes if counts is None else min(max(int(counts[b]), 0), nodes))
            keys[b, :, max(last, 0):], values[b, :, max(last, 0):] = math.nan, math.inf
    want, size = draft_plain.tree_attention(q, keys, values, rows, masks, counts, offset or 0)
    put = lambda t: None if t is None else t.to(cuda)  # noqa: E731
    got = attention.tree_attention(q, keys, values, put(rows), put(masks), counts=put(counts), offset=None if offset is None else torch.tensor([offset], device=cuda))
    assert got.shape == want.shape and got.dtype == BF16
    off, bound = (got.double() - want).abs(), (2.0 ** -8 + 2.0 ** -10) * size + 2.0 ** -8 * want.abs()
    assert bool((off <= bound).all()), float((off / bound.clamp(min=1e-300)).max())


@pytest.mark.parametrize("nodes", [1, 2, 15, 16, 33, 64, 100])
@pytest.mark.parametrize("cache_type", [F32, BF16])
@pytest.mark.parametrize("q_type", [F32, BF16])
@pytest.mark.parametrize("hd", [128, 64, 32])
def test_tree_attention_types_and_sizes(cuda, hd, q_type, cache_type, nodes):
    _attend(cuda, 3, nodes, 8, 4, hd, 240, q_type, cache_type, seed=nodes)


@pytest.mark.parametrize("cache_type", [F32, BF16])
@pytest.mark.parametrize("nodes", [1, 9, 40])
@pytest.mark.parametrize("heads,kv", [(1, 1), (6, 2), (7, 1), (32, 8), (16, 16)])
def test_tree_attention_heads(cuda, heads, kv, nodes, cache_type):
    _attend(cuda, 2, nodes, heads, kv, 64, 150, F32, cache_type, seed=heads + nodes)


@pytest.mark.parametrize("cache_type", [F32, BF16])
@pytest.mark.parametrize("max_len", [1, 31, 32, 33, 64, 65, 500, 1031, 4100])
def test_tree_attention_lengths(cuda, max_len, cache_type):
    for nodes, share in ((1, 1), (7, 2), (32, 4)):
        if nodes <= max_len:
            _attend(cuda, 5, nodes, 2 * share, 2, 128, max_len, BF16, cache_type, seed=max_len, rows=[0, max_len - nodes, (max_len - nodes) // 2, 0, max_len - nodes])


@pytest.mark.parametrize("cache_type", [F32, BF16])
@pytest.mark.parametrize("nodes", [5, 31, 32, 33, 64, 70])
def test_tree_attention_every_place_of_the_tree_in_a_block(cuda, nodes, cache_type):
    """The drafted rows begin at every place of a block of 32 and of 64 rows."""
    rows = list(range(0, 66)) + [127, 128, 129, 191]
    _attend(cuda, len(rows), nodes, 4, 1, 32, 300, F32, cache_type, seed=nodes, rows=rows, ragged=False)


@pytest.mark.parametrize("cache_type", [F32, BF16])
@pytest.mark.parametrize("nodes", [6, 48])
def test_tree_attention_any_bits(cuda, nodes, cache_type):
    """Masks that are no trees: any bits, none at all, all of them; and what is there of the tokens cuts them."""
    gen = _gen(1)
    words = (nodes + 31) // 32
    masks = torch.randint(-2 ** 31, 2 ** 31, (6, nodes, words), generator=gen).int()
    masks[1], masks[2] = 0, -1
    _attend(cuda, 6, nodes, 4, 2, 64, 200, F32, cache_type, seed=nodes, masks=masks, rows=[100, 90, 0, 150, 3, 64], counts=[nodes, nodes, nodes - 1, nodes // 2, 1, 0])
    _attend(cuda, 6, nodes, 4, 2, 64, 200, F32, cache_type, seed=nodes, masks=masks[1], rows=[0, 90, 0, 150, 3, 64], counts=[nodes, nodes, nodes - 1, nodes // 2, 1, 0])


@pytest.mark.parametrize("cache_type", [F32, BF16])
def test_tree_attention_rows_outside_the_caches(cuda, cache_type):
    masks = torch.full((8, 9, 1), -1, dtype=torch.int32)
    for nodes_heads in (4, 32):
        _attend(cuda, 8, 9, nodes_heads, 1, 64, 40, F32, cache_type, seed=3, masks=masks, rows=[-2, -9, -100, 36, 40, 41, 2 ** 40, -2 ** 40], ragged=False, garbage=False)
        _attend(cuda, 8, 9, nodes_heads, 1, 64, 40, F32, cache_type, seed=4, masks=masks, rows=[0, 5, 31, 32, 40, 7, 8, 9], counts=[-1, 0, 2 ** 40, 9, 3, -2 ** 40, 4, 100],
                garbage=False)


@pytest.mark.parametrize("cache_type", [F32, BF16])
@pytest.mark.parametrize("nodes", [3, 35])
def test_tree_attention_strides_offset_and_one_tree(cuda, nodes, cache_type):
    _attend(cuda, 4, nodes, 8, 2, 128, 200, F32, cache_type, seed=5, spread=24, offset=17, rows=[0, 100, 148, 60])
    _attend(cuda, 4, nodes, 8, 2, 128, 200, BF16, cache_type, seed=6, one_tree=True, mask_words=5)
    _attend(cuda, 4, nodes, 8, 2, 128, 200, BF16, cache_type, seed=7, mask_words=4, offset=-3, rows=[3, 50, 160, 20])


@pytest.mark.parametrize("cache_type", [F32, BF16])
@pytest.mark.parametrize("batch,nodes,heads,kv,max_len", [(1, 8, 4, 4, 20000), (1, 64, 8, 2, 9000), (40, 4, 16, 16, 700), (2, 128, 16, 4, 3000), (3, 200, 4, 1, 2500), (70, 20, 8, 8, 300)])
def test_tree_attention_parts_and_tiles(cuda, batch, nodes, heads, kv, max_len, cache_type):
    _attend(cuda, batch, nodes, heads, kv, 128, max_len, BF16, cache_type, seed=nodes)
    _attend(cuda, batch, nodes, heads, kv, 64, max_len, F32, cache_type, seed=nodes + 1)


@pytest.mark.parametrize("cache_type", [F32, BF16])
@pytest.mark.parametrize("nodes,heads", [(3, 2), (40, 4), (90, 4)])
def test_tree_attention_parts_of_odd_sequences(cuda, nodes, heads, cache_type):
    """Rows in parts, dealt out to sequences that begin outside their caches, have no tokens, one row, or all of them; and one sequence alone."""
    rows = [-2, -2 ** 40, 6000 - 2, 6000, 2 ** 40, 0, 5000, 1]
    for counts in (None, [nodes, 2, nodes, 2, 1, 1, -5, 2 ** 40], [0] * 8, [0, 0, 0, 0, 0, 0, 0, 1]):
        _attend(cuda, 8, nodes, heads, 1, 64, 6000, F32, cache_type, seed=9, rows=rows, counts=counts, ragged=False, garbage=False)
    for alone in rows:
        _attend(cuda, 1, nodes, heads, 1, 128, 6000, BF16, cache_type, seed=10, rows=[alone], ragged=False, garbage=False)


@pytest.mark.parametrize("cache_type", [F32, BF16])
@pytest.mark.parametrize("nodes", [4, 40])
def test_tree_attention_scores_far_apart(cuda, nodes, cache_type):
    """Scores of hundreds: maxima move between blocks, most weights vanish.  (The queries are whole numbers that bf16 holds, and so are the keys: products are exact,
    and sums of a few thousand too.)"""
    gen = _gen(8)
    q = torch.randint(-60, 61, (3, 8, nodes, 64), generator=gen).float().to(cuda)
    keys = torch.randint(-8, 9, (3, 2, 400, 64), generator=gen).float()
    keys[1] *= torch.linspace(0, 1, 400).round()[:, None]
    values = torch.randn((3, 2, 400, 64), generator=gen)
    keys, values = keys.to(cache_type).to(cuda), values.to(cache_type).to(cuda)
    rows, masks = torch.tensor([300, 350, 0]), attention.tree_masks(_tree(gen, nodes, 3))[0]
    want, size = draft_plain.tree_attention(q, keys, values, rows, masks, None, 0)
    got = attention.tree_attention(q, keys, values, rows.to(cuda), masks.to(cuda))
    off, bound = (got.double() - want).abs(), (2.0 ** -8 + 2.0 ** -10) * size + 2.0 ** -8 * want.abs()
    assert bool((off <= bound).all()), float((off / bound.clamp(min=1e-300)).max())


def test_tree_attention_offsets_past_32_bits(cuda):
    """The second sequence's rows lie 2^31 elements behind the first's."""
    hd, far = 32, 2 ** 31
    if torch.cuda.mem_get_info()[0] < 12 * far:
        pytest.skip("not enough memory")
    gen = _gen(9)
    near = torch.randn((2, 2, 1, 64, hd), generator=gen).to(BF16)
    flat = [torch.empty(far + 64 * hd, dtype=BF16, device=cuda) for _ in range(2)]
    caches = [f.as_strided((2, 1, 64, hd), (far, 64 * hd, hd, 1)) for f in flat]
    for cache, x in zip(caches, near):
        cache.copy_(x)
    q = torch.randn((2, 4, 20, hd), generator=gen).to(BF16).to(cuda)
    rows, masks = torch.tensor([40, 44], device=cuda), attention.tree_masks(_tree(gen, 20))[0].to(cuda)
    got = attention.tree_attention(q, *caches, rows, masks)
    assert torch.equal(got, attention.tree_attention(q, *(x.to(cuda) for x in near), rows, masks))
    before = [x.clone() for x in near]
    index = torch.tensor([0, 3, 9], device=cuda)
    attention.keep_rows(*caches, rows, index)
    for cache, x in zip(caches, before):
        assert torch.equal(cache.cpu(), draft_plain.keep_rows(x[None], rows, index, None, 0)[0])


def test_tree_attention_is_a_chain_of_single_steps(cuda):
    """A tree that is a chain is what as many single steps are."""
    gen = _gen(10)
    q, keys, values = (torch.randn(s, generator=gen).to(cuda) for s in ((2, 4, 6, 64), (2, 2, 50, 64), (2, 2, 50, 64)))
    rows, one = torch.tensor([20, 44], device=cuda), torch.ones((1, 1), dtype=torch.int32, device=cuda)
    got = attention.tree_attention(q, keys, values, rows, attention.tree_masks(torch.arange(-1, 5))[0].to(cuda))
    for t in range(6):
        single = attention.tree_attention(q[:, :, t:t + 1], keys, values, rows + t, one)
        torch.testing.assert_close(got[:, t:t + 1].float(), single.float(), rtol=2.0 ** -7, atol=2.0 ** -7)


def test_tree_attention_is_repeatable_and_takes_any_stream(cuda):
    gen = _gen(11)
    q, keys, values = (torch.randn(s, generator=gen).to(BF16).to(cuda) for s in ((2, 16, 24, 128), (2, 4, 5000, 128), (2, 4, 5000, 128)))
    rows, masks = torch.tensor([4900, 2500], device=cuda), attention.tree_masks(_tree(gen, 24))[0].to(cuda)
    first = attention.tree_attention(q, keys, values, rows, masks)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        second = attention.tree_attention(q, keys, values, rows, masks)
    third = attention.tree_attention(q, keys, values, rows, masks)
    torch.cuda.synchronize()
    assert torch.equal(first, second) and torch.equal(first, third)


def test_tree_attention_refuses(cuda):
    q, cache, rows = torch.zeros(2, 4, 40, 64, device=cuda), torch.zeros(2, 2, 80, 64, device=cuda), torch.zeros(2, dtype=torch.long, device=cuda)
    masks = torch.zeros(2, 40, 2, dtype=torch.int32, device=cuda)
    call = attention.tree_attention
    for bad in (masks[:, :, :1], masks[:1], masks[:, :39], masks.long(), masks.cpu(), masks.transpose(0, 1), masks[0, 0], masks.mT.contiguous().mT):
        with pytest.raises(ValueError, match="masks int32"):
            call(q, cache, cache, rows, bad)
    for bad in (rows.int(), rows[:1], rows.cpu()):
        with pytest.raises(ValueError, match="rows must be"):
            call(q, cache, cache, bad, masks)
        with pytest.raises(ValueError, match="counts must be"):
            call(q, cache, cache, rows, masks, counts=bad)
    with pytest.raises(ValueError, match="offset must be"):
        call(q, cache, cache, rows, masks, offset=rows)
    with pytest.raises(ValueError, match="q \\[B, H, T, hd\\]"):
        call(q.half(), cache, cache, rows, masks)
    with pytest.raises(ValueError, match="caches"):
        call(q, cache, cache[:, :, :79], rows, masks)
    with pytest.raises(ValueError, match="caches \\[B, Hkv"):
        call(q[:1], cache, cache, rows, masks)
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        call(q, cache.half(), cache.half(), rows, masks)
    with pytest.raises(ValueError, match="one behind the other"):
        call(q, cache[:, :, ::2], cache[:, :, ::2], rows, masks)
    with pytest.raises(ValueError, match="unsupported shape"):
        call(q[:, :3], cache, cache, rows, masks)
    with pytest.raises(ValueError, match="unsupported shape"):
        call(q[:, :, :0], cache, cache, rows, masks[:, :0])


# ------------------------------------------------------------------ keep_rows
def _keep(cuda, layers, batch, kv, hd, max_len, dtype, rows, index, counts=None, offset=None, spread=0, five=True):
    gen = _gen(len(rows) + max_len)
    whole = torch.randn((2, layers, batch, kv, max_len + spread, hd), generator=gen).to(dtype)
    rows, index = torch.tensor(rows), torch.as_tensor(index)
    counts = None if counts is None else torch.tensor(counts)
    want = [draft_plain.keep_rows(x[:, :, :, :max_len], rows, index, counts, offset or 0) for x in whole]
    ours = whole.to(cuda)
    views = [x[:, :, :, :max_len] for x in ours]
    put = lambda t: None if t is None else t.to(cuda)  # noqa: E731
    attention.keep_rows(*(v if five else v[0] for v in views), put(rows), put(index), put(counts), offset=None if offset is None else torch.tensor([offset], device=cuda))
    for got, x, w in zip(ours.cpu(), whole, want):
        assert torch.equal(got[:, :, :, :max_len], w) and torch.equal(got[:, :, :, max_len:], x[:, :, :, max_len:])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("hd", [128, 64, 32])
@pytest.mark.parametrize("width", [1, 7, 16, 64, 65, 500])
def test_keep_rows_types_and_sizes(cuda, width, hd, dtype):
    gen = _gen(width)
    stay = torch.rand((3, 2 * width), generator=gen)
    index = torch.stack([s.sort().indices[:width].sort().values for s in stay])
    _keep(cuda, 2, 3, 4, hd, 2 * width + 20, dtype, [0, 20, 9], index, counts=[width, width // 2, width])
    _keep(cuda, 1, 3, 4, hd, 2 * width + 20, dtype, [0, 3, 1], index, offset=5, five=False)


def test_keep_rows_in_place_everything_and_nothing(cuda):
    _keep(cuda, 2, 3, 2, 64, 40, F32, [0, 5, 10], list(range(30)))                          # (nothing moves)
    _keep(cuda, 2, 3, 2, 64, 40, F32, [0, 5, 10], list(range(1, 30)), counts=[0, -5, 2 ** 40])
    _keep(cuda, 2, 1, 2, 64, 40, F32, [0], [[39]])
    _keep(cuda, 2, 1, 2, 64, 40, F32, [39], [[0]])


def test_keep_rows_lists_that_end_early(cuda):
    """Numbers that do not ascend, that are negative or outside the cache end a list; rows outside the caches have none."""
    lists = [[0, 2, 2, 5], [0, 3, 1, 7], [-1, 3, 4, 5], [2, -1, 3, 4], [4, 29, 30, 31], [0, 2, 4, 2 ** 40], [1, 2 ** 33 + 3, 5, 6], [0, 1, 2, -2 ** 40]]
    for dtype in (F32, BF16):
        _keep(cuda, 1, 8, 2, 64, 40, dtype, [10] * 8, lists)
        _keep(cuda, 1, 8, 2, 64, 40, dtype, [-1, 40, 39, 2 ** 40, -2 ** 40, 0, 37, 36], lists)
    # the same far into a long list
    index = torch.arange(1, 1201).repeat(3, 1)
    index[0, 700], index[1, 64], index[2, 1199] = 700, 0, 1500
    _keep(cuda, 1, 3, 2, 64, 1400, F32, [0, 0, 0], index)
    _keep(cuda, 1, 3, 2, 128, 1400, BF16, [0, 150, 230], index)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_keep_rows_long_lists(cuda, dtype):
    gen = _gen(20)
    for many, first in ((2000, 0), (4111, 33)):
        index = torch.rand((2, 5000), generator=gen).sort(1).indices[:, :many].sort(1).values
        _keep(cuda, 1, 2, 3, 128, 5100, dtype, [first, 0], index)
        _keep(cuda, 1, 2, 1, 32, 5100, dtype, [first, 0], index, counts=[many - 1, many // 2])


def test_keep_rows_strides(cuda):
    """Padded caches, keys and values interleaved, heads ahead of sequences."""
    _keep(cuda, 2, 2, 2, 64, 30, F32, [0, 5], [[0, 2, 9], [1, 3, 7]], spread=8)
    gen = _gen(21)
    both = torch.randn((3, 2, 2, 4, 30, 64), generator=gen)   # [layers, keys and values, B, Hkv, rows, hd]
    ours, index, rows = both.to(cuda), torch.tensor([1, 3, 7]), torch.tensor([0, 5])
    attention.keep_rows(ours[:, 0], ours[:, 1], rows.to(cuda), index.to(cuda))
    for i in range(2):
        assert torch.equal(ours[:, i].cpu(), draft_plain.keep_rows(both[:, i], rows, index, None, 0))
    heads_first = torch.randn((2, 4, 2, 30, 64), generator=gen).to(cuda)
    keys, values = (x.transpose(0, 1) for x in heads_first)
    want = [draft_plain.keep_rows(x.cpu()[None], rows, index, None, 0)[0] for x in (keys, values)]
    attention.keep_rows(keys, values, rows.to(cuda), index.to(cuda))
    assert torch.equal(keys.cpu(), want[0]) and torch.equal(values.cpu(), want[1])


def test_keep_rows_refuses(cuda):
    cache, rows, index = torch.zeros(2, 3, 4, 20, 64, device=cuda), torch.zeros(3, dtype=torch.long, device=cuda), torch.zeros(3, 5, dtype=torch.long, device=cuda)
    other = torch.zeros_like(cache)
    call = attention.keep_rows
    with pytest.raises(ValueError, match="overlap"):
        call(cache, cache, rows, index)
    with pytest.raises(ValueError, match="overlap"):
        call(cache[:1].expand(2, -1, -1, -1, -1), other[:1].expand(2, -1, -1, -1, -1), rows, index)
    with pytest.raises(ValueError, match="overlap"):
        call(cache[0, :, :, :10], cache[0, :, :, 5:15], rows, index)
    for bad in (index.int(), index[:2], index.cpu(), index[:, ::2], index[0, 0]):
        with pytest.raises(ValueError, match="index int64"):
            call(cache, other, rows, bad)
    for bad in (rows.int(), rows[:2], rows.cpu()):
        with pytest.raises(ValueError, match="rows must be"):
            call(cache, other, bad, index)
        with pytest.raises(ValueError, match="counts must be"):
            call(cache, other, rows, index, bad)
    with pytest.raises(ValueError, match="one shape"):
        call(cache, other[:1], rows, index)
    with pytest.raises(ValueError, match="caches"):
        call(cache[0], other, rows, index)
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        call(cache.half(), other.half(), rows, index)
    call(cache, other, rows, index[:, :0])   # nothing to do


# ------------------------------------------------------------------ token_log_probs
# A sum has at most 160 additions one behind the other (128 of a lane, the rest over lanes, waves and slices) of positive terms, each the hardware's 2^x (1 ulp) of d
# log2(e) with d = x - m rounded once: 2^-24 (2 + 2 |d|) of it.  So log s is off by 2^-24 (164 + 2 E|d| + 4 log s), u / s by 2^-24 (330 E|d| + 4 E d^2), a log probability by its own
# two roundings more.
STEP = 2.0 ** -24


def _score(cuda, logits, targets=None, top=0, seed=0):
    rows, vocab = logits.shape
    got = sampling.token_log_probs(logits.to(cuda) if not logits.is_cuda else logits, None if targets is None else targets.to(cuda), top=top)
    mine, ranks, entropy, top_log_probs, top_ids, spread = draft_plain.token_log_probs(logits, targets, top)
    of_s = 164 + 2 * spread["first"] + 4 * spread["log_total"]

    def near(x, want, slack, what):
        x = x.double().cpu()
        fine = torch.isfinite(want)
        assert torch.equal(x[~fine], want[~fine]), what
        off, bound = (x - want)[fine].abs(), STEP * slack.expand(want.shape)[fine]
        assert bool((off <= bound).all()), (what, float((off / bound).max()))

    assert got.entropy.dtype == F32 and got.entropy.shape == (rows,)
    near(got.entropy, entropy, of_s + 330 * spread["first"] + 4 * spread["second"] + 2 * entropy.abs(), "entropy")
    if targets is None:
        assert got.log_probs is None and got.ranks is None
    else:
        near(got.log_probs, mine, of_s + 4 * mine.abs().nan_to_num(posinf=0.0), "log probabilities")
        assert torch.equal(got.ranks.cpu(), ranks)
    if top == 0:
        assert got.top_log_probs is None and got.top_ids is None
    else:
        assert torch.equal(got.top_ids.cpu(), top_ids)
        near(got.top_log_probs, top_log_probs, of_s[:, None] + 4 * top_log_probs.abs().nan_to_num(posinf=0.0), "alternatives")
    return got


def _logits(rows, vocab, dtype, seed, scale=3.0):
    return (scale * torch.randn((rows, vocab), generator=_gen(seed))).to(dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 65, 255, 1000, 1023, 1024, 1025, 4095, 4099, 8192, 16385, 32000, 32011, 70001])
def test_log_probs_vocabularies(cuda, vocab, dtype):
    for rows, top in ((1, min(vocab, 5)), (7, min(vocab, 64)), (3, 0), (2, 1)):
        _score(cuda, _logits(rows, vocab, dtype, vocab + rows), torch.randint(0, vocab, (rows,), generator=_gen(rows)), top)
        _score(cuda, _logits(rows, vocab, dtype, vocab + rows), None, top)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", [(1, 300000), (5, 128256), (300, 5000), (1500, 777), (700, 33000)])
def test_log_probs_rows(cuda, rows, vocab, dtype):
    for top in (0, 1, 20):
        _score(cuda, _logits(rows, vocab, dtype, rows), torch.randint(0, vocab, (rows,), generator=_gen(rows)), top)


@pytest.mark.parametrize("top", [1, 2, 20, 63, 64])
@pytest.mark.parametrize("vocab", [64, 500, 4097, 33000])
def test_log_probs_order_of_equal_logits(cuda, vocab, top):
    """All equal, few values, ascending, descending, zeros of both signs, everything in one place, and the largest logits far apart."""
    gen = _gen(vocab)
    rows = [torch.zeros(vocab), torch.randint(0, 3, (vocab,), generator=gen).float(), torch.linspace(-20, 10, vocab), torch.linspace(10, -20, vocab),
            torch.where(torch.rand(vocab, generator=gen) < 0.5, 0.0, -0.0), torch.full((vocab,), -5.0), torch.full((vocab,), -math.inf), torch.randn(vocab, generator=gen)]
    rows[5][vocab // 2:vocab // 2 + 40] = 7.0
    rows[6][vocab // 3] = 1.0
    rows[7][::max(1, vocab // 100)] += 20.0
    logits = torch.stack(rows)
    for dtype in (F32, BF16):
        x = logits.to(dtype)
        targets = torch.randint(0, vocab, (8,), generator=gen)
        got = _score(cuda, x, targets, top)
        among = got.ranks < top
        assert torch.equal(got.top_ids.gather(1, got.ranks.clamp(max=top - 1)[:, None])[:, 0][among].cpu(), targets[among.cpu()])


def test_log_probs_rows_that_are_hard_to_order(cuda):
    """More tokens that may be among the first than there is room for: of a slice (whole groups of lanes above the border), of many slices (one of them far below the
    others, or with next to nothing in it)."""
    at = torch.arange(8192) // 4 % 128
    one = torch.where(at < 63, 2.0, torch.where(at == 63, 1.0, 0.0)) + torch.linspace(0, 0.5, 8192)
    _score(cuda, torch.stack((one, one.flip(0))), torch.tensor([5, 8000]), 64)
    _score(cuda, torch.cat((one, one))[None].bfloat16(), torch.tensor([9000]), 64)
    wide = torch.randn(5, 128256, generator=_gen(2))
    keep = torch.rand((5, 128256), generator=_gen(3)) < torch.tensor([0.0, 3e-4, 3e-3, 1e-2, 1e-5])[:, None]
    keep[3, 40000:90000] = False
    for top in (64, 20, 1):   # (a mask leaves a slice fewer tokens than that, or none)
        _score(cuda, wide.masked_fill(~keep, -math.inf), torch.tensor([7, 0, 128255, 50000, 3]), top)
        _score(cuda, wide.masked_fill(~keep, -math.inf).bfloat16(), None, top)
    for last in (8192, 6000, 1):
        many = torch.randn(1, 47 * 8192 + last, generator=_gen(last))
        many[:, 46 * 8192:] -= 100.0
        for top in (64, 63):
            _score(cuda, many, torch.tensor([46 * 8192 + 3]), top)
            _score(cuda, many.flip(1).contiguous(), torch.tensor([12]), top)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [70, 5000, 40000])
def test_log_probs_masked(cuda, vocab, dtype):
    """Rows that a mask leaves a few tokens of, one, none; the type's lowest value in its places instead of -inf."""
    x = _logits(6, vocab, dtype, vocab)
    keep = torch.rand((6, vocab), generator=_gen(1)) < torch.tensor([0.5, 0.01, 3 / vocab, 0.0, 0.0, 0.3])[:, None]
    keep[4, vocab - 1] = True
    targets = torch.tensor([0, vocab - 1, 5, 3, vocab - 1, 1])
    for top in (0, 4, 64):
        _score(cuda, x.masked_fill(~keep, -math.inf), targets, top)
        _score(cuda, x.masked_fill(~keep, torch.finfo(dtype).min), targets, top)


def test_log_probs_targets_outside(cuda):
    x = _logits(5, 1000, F32, 3)
    got = _score(cuda, x, torch.tensor([-1, 1000, 2 ** 40, -2 ** 63, 999]), 3)
    assert got.log_probs[:4].tolist() == [0.0] * 4 and got.ranks[:4].tolist() == [-1] * 4


@pytest.mark.parametrize("top", [0, 1, 30])
@pytest.mark.parametrize("vocab", [100, 3000, 50000])
def test_log_probs_without_numbers(cuda, vocab, top):
    """NaN and +inf: NaN for the row, ids and ranks inside the vocabulary; the rows beside it are as ever."""
    x = _logits(6, vocab, F32, 5)
    x[1, vocab // 2], x[3, 0], x[4, 1:40] = math.nan, math.inf, math.nan
    targets = torch.tensor([1, 2, 3, 0, 5, 6])
    got = sampling.token_log_probs(x.to(cuda), targets.to(cuda), top=top)
    want = draft_plain.token_log_probs(x[[0, 2, 5]], targets[[0, 2, 5]], top)
    bad, good = torch.tensor([1, 3, 4]), torch.tensor([0, 2, 5])
    assert bool(got.entropy.cpu()[bad].isnan().all()) and bool(got.log_probs.cpu()[bad].isnan().all())
    assert bool((got.ranks >= 0).all()) and bool((got.ranks < vocab).all())
    assert torch.equal(got.ranks.cpu()[good], want[1])
    torch.testing.assert_close(got.log_probs.cpu()[good].double(), want[0], rtol=0, atol=400 * STEP)
    if top:
        assert bool((got.top_ids >= 0).all()) and bool((got.top_ids < vocab).all())
        assert torch.equal(got.top_ids.cpu()[good], want[4])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_log_probs_strides_and_addresses(cuda, dtype):
    """Rows of a wider buffer that begin anywhere, one row for all, one column."""
    whole = _logits(6, 4200, dtype, 7).to(cuda)
    targets = torch.tensor([3, 0, 4000, 17, 1, 2])
    for first in (0, 1, 2, 3, 5):
        for width in (4097, 4096, 100):
            _score(cuda, whole[:, first:first + width], targets.clamp(max=width - 1), 20)
    _score(cuda, whole[:1].expand(6, -1), targets, 5)
    _score(cuda, whole[::2, :1], torch.zeros(3, dtype=torch.long), 1)


def test_log_probs_large_and_small_numbers(cuda):
    for scale in (1e-30, 1e30, 3e38, 1e-42):
        x = torch.linspace(-1, 1, 5000)[None].repeat(2, 1) * scale
        x[1] = x[1].flip(0)
        got = sampling.token_log_probs(x.to(cuda), torch.tensor([0, 0], device=cuda), top=3)
        want = draft_plain.token_log_probs(x, torch.tensor([0, 0]), 3)
        assert torch.equal(got.top_ids.cpu(), want[4]) and torch.equal(got.ranks.cpu(), want[1])
        torch.testing.assert_close(got.entropy.cpu().double(), want[2], rtol=2e-5, atol=2e-5)
        torch.testing.assert_close(got.top_log_probs.cpu().double(), want[3], rtol=1e-5, atol=2e-5)


def test_log_probs_refuses(cuda):
    x, targets = torch.zeros(4, 100, device=cuda), torch.zeros(4, dtype=torch.long, device=cuda)
    call = sampling.token_log_probs
    for bad in (x.half(), x[0], x.t(), x[:, ::2], x[:, :0]):
        with pytest.raises(ValueError, match="logits \\[R, V\\]"):
            call(bad, None)
    for bad in (targets.int(), targets[:3], targets.cpu(), targets[:, None], torch.zeros(8, dtype=torch.long, device=cuda)[::2]):
        with pytest.raises(ValueError, match="targets must be"):
            call(x, bad)
    for bad in (-1, 65, 101):
        with pytest.raises(ValueError, match="top must be"):
            call(x, top=bad)
    with pytest.raises(ValueError, match="top must be"):
        call(x[:, :10], top=11)
    empty = call(x[:0], targets[:0], top=3)
    assert empty.log_probs.shape == (0,) and empty.top_ids.shape == (0, 3)


# ------------------------------------------------------------------ follow_drafts
def _follow(cuda, tokens, parents, choices, counts=None):
    put = lambda t: None if t is None else t.to(cuda)  # noqa: E731
    got = sampling.follow_drafts(put(tokens), put(parents), put(choices), counts=put(counts))
    for x, want, what in zip(got, draft_plain.follow_drafts(tokens, parents, choices, counts), got._fields):
        assert torch.equal(x.cpu(), want), what
    return got


@pytest.mark.parametrize("batch,nodes", [(1, 1), (1, 16), (5, 2), (40, 33), (300, 64), (2, 255), (2, 257), (3, 1000), (1, 4096)])
def test_follow_drafts_sizes(cuda, batch, nodes):
    gen = _gen(nodes)
    tokens, choices = (torch.randint(0, 3, (batch, nodes), generator=gen) for _ in range(2))
    counts = torch.randint(0, nodes + 1, (batch,), generator=gen)
    _follow(cuda, tokens, _tree(gen, nodes, batch), choices)
    _follow(cuda, tokens, _tree(gen, nodes), choices, counts)
    chain = torch.arange(-1, nodes - 1)
    same = torch.zeros_like(tokens)
    assert _follow(cuda, same, chain, same).accepted.tolist() == [nodes] * batch
    _follow(cuda, same, chain, same, counts)


def test_follow_drafts_ties_padding_and_odd_parents(cuda):
    tokens = torch.tensor([[9, 5, 5, 7, 7, 5]])
    choices = torch.tensor([[5, 7, 7, 1, 2, 3]])
    _follow(cuda, tokens, torch.tensor([-1, 0, 0, 2, 1, 0]), choices)                                # (two children agree: the first, and its children)
    for bad in ([-1, -1, 0, 2, 1, 0], [0, 1, 0, 3, 2, 5], [-1, 2 ** 40, -2 ** 40, 0, 0, 0], [5, 4, 3, 2, 1, 0]):
        _follow(cuda, tokens, torch.tensor(bad), choices)
    wide = torch.randint(0, 3, (4, 50), generator=_gen(2))
    top_ids = torch.randint(0, 3, (200, 4), generator=_gen(3))
    _follow(cuda, wide, _tree(_gen(4), 50, 4), top_ids[:, :1].view(4, 50))                           # (every fourth number)
    _follow(cuda, wide[:, 3:40], _tree(_gen(4), 50, 4)[:, 13:], wide[:, 4:41], torch.tensor([-1, 0, 2 ** 40, 5]))
    _follow(cuda, wide[:1].expand(4, -1), _tree(_gen(4), 50)[None].expand(4, -1), wide)


def test_follow_drafts_refuses(cuda):
    tokens = torch.zeros(2, 6, dtype=torch.long, device=cuda)
    call = sampling.follow_drafts
    for bad in (tokens.int(), tokens[0], tokens[:, ::2]):
        with pytest.raises(ValueError, match="tokens int64"):
            call(bad, tokens[0], tokens)
    for bad in (tokens.int(), tokens[:1], tokens[0, :5], tokens.cpu(), torch.zeros(2, 12, dtype=torch.long, device=cuda)[:, ::2]):
        with pytest.raises(ValueError, match="parents int64"):
            call(tokens, bad, tokens)
    for bad in (tokens.int(), tokens[:1], tokens.cpu(), tokens[0]):
        with pytest.raises(ValueError, match="choices int64"):
            call(tokens, tokens, bad)
    with pytest.raises(ValueError, match="counts must be"):
        call(tokens, tokens, tokens, counts=torch.zeros(3, dtype=torch.long, device=cuda))
    with pytest.raises(ValueError, match="unsupported shape"):
        call(torch.zeros(1, 4097, dtype=torch.long, device=cuda), torch.zeros(4097, dtype=torch.long, device=cuda), torch.zeros(1, 4097, dtype=torch.long, device=cuda))
    many = tokens[:1, :1].expand(2 ** 32 + 5, 1)
    with pytest.raises(ValueError, match="2\\^31 trees"):
        call(many, tokens[0, :1], many)
    with pytest.raises(ValueError, match="dimensions below"):
        cache = torch.zeros(1, 1, 4, 64, device=cuda)
        attention.keep_rows(cache.expand(2 ** 32 + 5, 1, 1, 4, 64), cache.clone().expand(2 ** 32 + 5, 1, 1, 4, 64), tokens[0, :1], tokens[:1])
    assert call(tokens[:0], tokens[0], tokens[:0]).accepted.shape == (0,)
