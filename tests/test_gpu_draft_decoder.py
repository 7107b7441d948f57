"""Decoders on the operators of checking drafted tokens: trees of guesses checked in one pass, log probabilities kept beside tokens, texts scored, each against the model's
own code."""

import copy

import pytest
import torch

from ajllm_amd import attention, decoding, evaluation, modeling, quantize_model_, sampling
from tests import draft_plain
from tests.helpers import errors
from tests.latent_models import config, random_weights
from tests.test_gpu_latent import LOGIT_TOL, _build, _tokens

pytestmark = pytest.mark.gpu

VOCAB = 512
TREES = [[-1], [-1, 0, 1, 2, 3], [-1, 0, 0, 0, 1, 1, 2, 4], [-1] + [0] * 8 + [t // 2 for t in range(9, 40)]]


def _model(cuda, scheme="w8a16", head_norm=False, heads=4, kv_heads=2, context=256):
    torch.manual_seed(31)
    model = modeling.TransformerLM(vocab_size=VOCAB, context_length=context, d_model=256, num_layers=2, num_heads=heads, num_kv_heads=kv_heads,
                                   d_ff=640, head_norm=head_norm).eval()
    if head_norm:
        for layer in model.layers:
            torch.nn.init.uniform_(layer.attention.q_norm.weight, 0.5, 1.5)
            torch.nn.init.uniform_(layer.attention.k_norm.weight, 0.5, 1.5)
    return quantize_model_(copy.deepcopy(model).to(cuda), scheme)


def _prompt(seed, batch, length):
    return torch.randint(0, VOCAB, (batch, length), generator=torch.Generator().manual_seed(seed))


# What the logits of two ways through the layers may differ by, of a row's length (test_gpu_serve_decoders.py); no logit of a row by more than that.
LOGITS = 2e-2


def _own(model, ids):
    with torch.no_grad():
        return model(torch.tensor([ids], device=model.token_embeddings.weight.device))[0].float().cpu()


# ------------------------------------------------------------------ norm_rope's depths
@pytest.mark.parametrize("tokens", [1, 7])
@pytest.mark.parametrize("own", [False, True])
def test_norm_rope_depths(cuda, tokens, own):
    """A token's position goes by its depth, its row by its number: what one call a token at that position gives."""
    gen = torch.Generator().manual_seed(3)
    batch, heads, kv, hd, rows_of_cache = 3, 4, 2, 64, 40
    qkv = torch.randn((batch, tokens, (heads + 2 * kv) * hd), generator=gen).to(cuda)
    angles = torch.arange(60, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    cosine, sine = angles.cos().float().to(cuda), angles.sin().float().to(cuda)
    caches = [torch.randn((2, batch, kv, rows_of_cache, hd), generator=gen).to(cuda) for _ in range(1)] * 2
    mine, want = caches[0].clone(), caches[0].clone()
    rows = torch.tensor([0, 17, 30], device=cuda)
    depths = torch.randint(0, 6, (batch, tokens) if own else (tokens,), generator=gen).to(cuda)
    gain = 1 + 0.2 * torch.randn(hd, generator=gen).to(cuda)
    q = attention.norm_rope(qkv.view(batch * tokens, -1), cosine, sine, mine[0], mine[1], rows, heads=heads, tokens=tokens, q_gain=gain, k_gain=gain, depths=depths)
    for t in range(tokens):
        at = rows + (depths[:, t] if own else depths[t])
        single = attention.norm_rope(qkv[:, t], cosine, sine, want[0], want[1], rows + t, heads=heads, q_gain=gain, k_gain=gain, positions=at)
        assert torch.equal(q[:, :, t], single[:, :, 0])
    assert torch.equal(mine, want)
    plain = attention.norm_rope(qkv.view(batch * tokens, -1), cosine, sine, mine[0], mine[1], rows, heads=heads, tokens=tokens)
    assert torch.equal(plain, attention.norm_rope(qkv.view(batch * tokens, -1), cosine, sine, mine[0], mine[1], rows, heads=heads, tokens=tokens,
                                                  depths=torch.arange(tokens, device=cuda)))
    for bad in (depths.int(), depths.cpu(), torch.zeros(tokens + 1, dtype=torch.long, device=cuda), torch.zeros(2, tokens, dtype=torch.long, device=cuda)):
        with pytest.raises(ValueError, match="depths int64"):
            attention.norm_rope(qkv.view(batch * tokens, -1), cosine, sine, mine[0], mine[1], rows, heads=heads, tokens=tokens, depths=bad)


# ------------------------------------------------------------------ a pass over a tree
@pytest.mark.parametrize("kv_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("head_norm", [False, True])
@pytest.mark.parametrize("tree", range(len(TREES)))
def test_passes_are_the_models(cuda, tree, head_norm, kv_dtype):
    """Every node's logits are the model's behind the tokens that lead to it, every path the one that the choices take; right guesses are kept, wrong ones leave nothing."""
    parents, gen = TREES[tree], torch.Generator().manual_seed(tree)
    model = _model(cuda, head_norm=head_norm)
    dec = decoding.DraftDecoder(model, 3, 120, parents, kv_dtype)
    prompt = _prompt(5, 3, 20)
    dec.prefill(prompt)
    nodes = len(parents)
    for count in range(6):
        before = [list(text) for text in dec.texts]
        guesses = torch.randint(0, VOCAB, (3, nodes - 1), generator=gen)
        for b in range(3):   # along one branch, what the model says itself (sequence 2: in vain)
            path, text, t = [0], list(before[b]), 0
            while b < 2 and t in parents:
                t = max(i for i, up in enumerate(parents) if up == t)
                guesses[b, t - 1] = int(_own(model, text)[-1].argmax())
                text.append(int(guesses[b, t - 1]))
        going = [True, count != 3, count != 4]
        got = dec.check(guesses, going)
        logits, choices = dec.logits.float().cpu().view(3, nodes, VOCAB), dec.scored.top_ids.view(3, nodes).cpu()
        tokens = torch.cat((torch.tensor([[text[-1]] for text in before]), guesses), dim=1)
        assert torch.equal(choices, logits.argmax(-1))
        path, accepted, chosen = draft_plain.follow_drafts(tokens, torch.tensor(parents), choices, torch.tensor([nodes if on else 0 for on in going]))
        assert got == [row[:n].tolist() for row, n in zip(chosen, accepted)]
        assert dec.texts == [text + new for text, new in zip(before, got)]
        table, _ = draft_plain.ancestors(parents)
        for b in range(3):
            if not going[b]:
                assert got[b] == []
                continue
            for t in range(0, nodes, 1 if nodes < 10 else 7):
                leads = [int(tokens[b, u]) for u in range(1, nodes) if table[t, u]]
                assert errors(logits[b, t], _own(model, before[b] + leads)[-1])[1] <= LOGITS, (count, b, t)
    if nodes > 1:
        assert len(dec.texts[0]) > 20 + 1 + 6 + 3   # (the branch was right now and then: its rows were moved and read again)


@pytest.mark.parametrize("tree", [0, 2])
def test_generate_gives_the_greedy_tokens(cuda, tree):
    """Whatever is guessed the tokens are the model's first choices; repeating texts are guessed from themselves."""
    model = _model(cuda)
    dec = decoding.DraftDecoder(model, 2, 140, TREES[tree])
    prompt = torch.cat((_prompt(6, 2, 12), _prompt(6, 2, 12)), dim=1)
    dec.prefill(prompt)
    got = dec.generate(60)
    assert got.shape == (2, 60)
    for ids, new in zip(prompt.tolist(), got.tolist()):
        own = _own(model, ids + new)[len(ids) - 1:-1]
        behind = own.max(-1).values - own.gather(1, torch.tensor(new)[:, None])[:, 0]
        assert bool((behind <= 2 * LOGITS * own.norm(dim=-1)).all())   # (the first choice of logits that are off by LOGITS at most)
    again = decoding.DraftDecoder(model, 2, 140, TREES[tree])
    again.prefill(prompt)
    assert torch.equal(again.generate(10), got[:, :10])
    again.prefill(prompt)                                            # (a second prompt into the same caches and graph)
    assert torch.equal(again.generate(60, guess=lambda: [[0] * (len(TREES[tree]) - 1)] * 2), got)
    eos = int(got[0, 20])
    first = [row.index(eos) + 1 if eos in row else 60 for row in got.tolist()]
    again.prefill(prompt)
    assert torch.equal(again.generate(60, eos_token_id=eos), got[:, :max(first)])


def test_checks_end_with_the_cache(cuda):
    """Where a right path leads past the last position, what is behind it is not produced (no position there is the model's)."""
    model = _model(cuda, context=40)
    dec = decoding.DraftDecoder(model, 2, 40, [-1, 0, 1, 2, 3, 4])
    prompt = _prompt(14, 2, 36)
    dec.prefill(prompt)                                               # (37 tokens: four positions are left, 36 to 39)
    while min(map(len, dec.texts)) <= 40:                             # (what the passes say one by one: the model's first choices up to what logits are off by)
        dec.check([[0] * 5] * 2, [len(text) <= 40 for text in dec.texts])
    right = [list(text) for text in dec.texts]
    for text in right:
        own = _own(model, text[:40])[35:]
        behind = own.max(-1).values - own.gather(1, torch.tensor(text[36:])[:, None])[:, 0]
        assert len(text) == 41 and bool((behind <= 2 * LOGITS * own.norm(dim=-1)).all())
    dec.prefill(prompt)
    got = dec.check([text[37:] + [0] for text in right])
    assert [len(new) for new in got] == [4, 4] and dec.texts == right
    with pytest.raises(ValueError, match="too short"):
        dec.check([[0] * 5] * 2)
    assert dec.generate(4).tolist() == [text[36:40] for text in right]


def test_guesses_come_from_the_text(cuda):
    dec = decoding.DraftDecoder(_model(cuda), 1, 100, [-1, 0, 1, 0, 3])
    dec.prefill(torch.tensor([[1, 2, 3, 4, 1, 2, 5, 6, 1]]))
    dec.texts = [[1, 2, 3, 4, 1, 2, 5, 6, 1, 2]]
    assert dec.guess() == [[5, 6, 3, 4]]        # (behind 1 2: 5 6 the latest, 3 4 ahead of it)
    dec.texts = [[1, 2, 3, 4, 1, 2, 5, 6, 1, 2, 9]]
    assert dec.guess() == [[0, 0, 0, 0]]


def test_draft_decoder_refuses(cuda):
    model = _model(cuda)
    for bad in ([], [0], [-1, 1], [-1, 0, 2], [-1, -1]):
        with pytest.raises(ValueError, match="parents"):
            decoding.DraftDecoder(model, 1, 64, bad)
    dec = decoding.DraftDecoder(model, 2, 40, [-1, 0, 0])
    with pytest.raises(ValueError, match="prefill comes first"):
        dec.check([[1, 2], [3, 4]])
    dec.prefill(_prompt(1, 2, 30))
    for bad in ([[1], [2]], [[1, VOCAB], [2, 3]], [[1, -1], [2, 3]]):
        with pytest.raises(ValueError, match="guesses"):
            dec.check(bad)
    with pytest.raises(ValueError, match="truth values"):
        dec.check([[1, 2], [3, 4]], [True])
    with pytest.raises(ValueError, match="too short"):
        dec.generate(11)
    for call in (lambda: dec.set_sampling(1.0), lambda: dec.set_penalties(1.1), lambda: dec.set_log_probs()):
        with pytest.raises(ValueError, match="DraftDecoder"):
            call()
    assert dec.generate(10).shape == (2, 10)


# ------------------------------------------------------------------ log probabilities beside tokens, and of texts
@pytest.mark.parametrize("kind", ["graph", "fused", "shared"])
@pytest.mark.parametrize("temperature", [0.0, 0.9])
def test_decoders_keep_log_probs(cuda, kind, temperature):
    model = _model(cuda)
    prompt = _prompt(9, 4, 25)
    if kind == "shared":
        dec = decoding.SharedPrefixDecoder(model, 4, 1, 32, 40)
    else:
        dec = (decoding.GraphDecoder if kind == "graph" else decoding.FusedDecoder)(model, 4, 64)
    if temperature:
        dec.set_sampling(temperature, 0.9, seed=3)
    dec.set_penalties(bias={7: -50.0})
    dec.prefill(prompt)
    plain = dec.generate(20)
    dec.set_log_probs(5)
    dec.prefill(prompt)
    assert torch.equal(dec.generate(20), plain)                       # (keeping changes no token)
    kept = dec.log_probs(20)
    assert kept.log_probs.shape == (4, 20) and kept.top_ids.shape == (4, 20, 5)
    for b in range(4):
        own = _own(model, prompt[b].tolist() + plain[b].tolist())[24:-1].double()
        own[:, 7] -= 50.0
        want = torch.log_softmax(own, dim=-1)
        slack = 2 * LOGITS * own.norm(dim=-1)   # (the logit's, and the logarithm's of the sum)
        for mine, theirs in ((kept.log_probs[b][:, None], want.gather(1, plain[b].cpu()[:, None])), (kept.top_log_probs[b], want.gather(1, kept.top_ids[b].cpu()))):
            assert bool(((mine.double().cpu() - theirs).abs() <= slack[:, None]).all())
        # sum p log p: p is off by a factor of e^slack, log p by slack
        entropy, moved = -(want.exp() * want).sum(-1), slack.exp() - 1
        assert bool(((kept.entropy[b].double().cpu() - entropy).abs() <= moved * entropy + slack.exp() * slack).all())
    if not temperature:
        assert bool((kept.ranks == 0).all()) and torch.equal(kept.top_ids[:, :, 0], plain)
    assert bool((kept.ranks >= 0).all()) and bool((kept.top_log_probs[..., 1:] <= kept.top_log_probs[..., :-1]).all())
    dec.set_log_probs(None)
    with pytest.raises(ValueError, match="set_log_probs"):
        dec.log_probs(1)
    with pytest.raises(ValueError, match="alternatives"):
        dec.set_log_probs(65)
    dec.set_log_probs()
    dec.prefill(prompt)
    dec.generate(3)
    assert dec.log_probs(3).top_ids is None
    with pytest.raises(ValueError, match="4 of 3"):
        dec.log_probs(4)


def test_dense_decoder_keeps_log_probs(cuda):
    cfg = config(window=[9, 14, 30], positions=256)
    model = _build(cfg, random_weights(cfg, 21), cuda, torch.bfloat16)
    prompts = torch.tensor([_tokens(cfg, 37, 40 + i) for i in range(3)], device=cuda)
    dec = decoding.DenseDecoder(model, 3, 80)
    dec.prefill(prompts)
    plain = dec.generate(30)
    dec.set_log_probs(4)
    with pytest.raises(ValueError, match="31 of 30"):
        dec.log_probs(31)
    dec.prefill(prompts)
    assert torch.equal(dec.generate(30), plain)
    kept, cache = dec.log_probs(30), model.new_cache(3, 80)
    logits = model(prompts, cache, last_token_only=True)[:, -1]
    noise = 4 * LOGIT_TOL[torch.bfloat16]                             # (of a logit, test_gpu_latent.py; the logarithm of the sum moves by as much at most)
    for step in range(30):
        want = torch.log_softmax(logits.double(), dim=-1)
        for mine, theirs in ((kept.log_probs[:, step, None], want.gather(1, plain[:, step, None])), (kept.top_log_probs[:, step], want.gather(1, kept.top_ids[:, step]))):
            assert bool(((mine.double() - theirs).abs() <= 2 * noise).all()), step
        logits = model(plain[:, step:step + 1], cache)[:, -1]
    assert bool((kept.ranks == 0).all()) and torch.equal(kept.top_ids[:, :, 0], plain)
    for fresh in (decoding.DenseDecoder(model, 1, 40), decoding.GraphDecoder(_model(cuda), 1, 40)):
        fresh.set_log_probs()
        with pytest.raises(ValueError, match="1 of 0"):
            fresh.log_probs(1)


def test_scored_texts(cuda):
    model = _model(cuda)
    tokens = _prompt(11, 3, 50).to(cuda)
    scored = evaluation.score_tokens(model, tokens, alternatives=3)
    with torch.no_grad():
        logits = model(tokens[:, :-1])
    assert scored.log_probs.shape == (3, 49) and scored.top_ids.shape == (3, 49, 3)
    # (fp32 both: the mean of 147 numbers of some six nats, each off by the roundings of a sum of 512)
    assert abs(float(-scored.log_probs.mean()) - float(evaluation.cross_entropy(logits, tokens[:, 1:]))) < 1e-5
    assert torch.equal(scored.top_ids[..., 0], logits.argmax(-1))
    with pytest.raises(ValueError, match="tokens"):
        evaluation.score_tokens(model, tokens[:, :1])
    assert evaluation.score_tokens(model, tokens[:0], alternatives=3).top_ids.shape == (0, 49, 3)


# ------------------------------------------------------------------ the operators of a step in turn, captured
def test_two_captured_steps_replay_as_eager_ones(cuda):
    """Two graphs of a step's operators with states of their own, replayed in turns with eager work between, against eager steps, every replay looked at."""
    gen = torch.Generator().manual_seed(21)
    batch, nodes, heads, kv, hd, layers, vocab = 3, 12, 4, 2, 64, 2, 1000
    parents = torch.tensor([-1, 0, 0, 1, 1, 2, 3, 3, 5, 6, 8, 8], device=cuda)
    masks, depths = attention.tree_masks(parents)
    angles = torch.arange(400, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    cosine, sine = angles.cos().float().to(cuda), angles.sin().float().to(cuda)

    def state(seed):
        g = torch.Generator().manual_seed(seed)
        return dict(qkv=torch.randn((batch * nodes, (heads + 2 * kv) * hd), generator=g).to(cuda), logits=torch.randn((batch * nodes, vocab), generator=g).to(cuda),
                    tokens=torch.randint(0, 4, (batch, nodes), generator=g).to(cuda), rows=torch.tensor([5, 120, 250], device=cuda),
                    keys=torch.randn((layers, batch, kv, 380, hd), generator=g).to(cuda).bfloat16(), values=torch.randn((layers, batch, kv, 380, hd), generator=g).to(cuda).bfloat16(),
                    out=torch.zeros(batch, nodes, heads * hd, dtype=torch.bfloat16, device=cuda), probs=torch.zeros(batch * nodes, device=cuda))

    def step(s):
        for layer in range(layers):
            q = attention.norm_rope(s["qkv"], cosine, sine, s["keys"][layer], s["values"][layer], s["rows"], heads=heads, tokens=nodes, depths=depths)
            s["out"].copy_(attention.tree_attention(q, s["keys"][layer], s["values"][layer], s["rows"], masks))
        scored = sampling.token_log_probs(s["logits"], s["tokens"].view(-1), top=1)
        s["probs"].copy_(scored.log_probs)
        path, accepted, chosen = sampling.follow_drafts(s["tokens"], parents, scored.top_ids.view(batch, nodes) % 4)
        attention.keep_rows(s["keys"], s["values"], s["rows"], path, accepted)
        s["rows"].add_(accepted)
        s["qkv"].mul_(-0.9)
        s["logits"].copy_(s["logits"].roll(17, 1))
        s["tokens"].add_(1).remainder_(4)

    eager, captured = [state(1), state(2)], [state(1), state(2)]
    step(state(3))
    torch.cuda.synchronize()
    graphs = []
    for s in captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(s)
        graphs.append(graph)
    for turn in range(6):
        for want, got, graph in zip(eager, captured, graphs):
            graph.replay()
            step(want)
            attention.tree_attention(torch.randn((2, 8, 40, hd), generator=gen).to(cuda), *(x[0, :2] for x in (want["keys"], want["values"])), want["rows"][:2],
                                     torch.zeros((40, 2), dtype=torch.int32, device=cuda))   # (eager work between replays)
            torch.cuda.synchronize()
            for name in want:
                assert torch.equal(want[name], got[name]), (turn, name)


def test_general_path_gives_the_same_bits(cuda, monkeypatch):
    from ajllm_amd import _lib

    gen = torch.Generator().manual_seed(22)
    q, keys, values = (torch.randn(s, generator=gen).to(cuda) for s in ((2, 8, 9, 64), (2, 2, 90, 64), (2, 2, 90, 64)))
    rows, masks = torch.tensor([40, 70], device=cuda), attention.tree_masks(torch.arange(-1, 8))[0].to(cuda)
    counts, offset = torch.tensor([9, 4], device=cuda), torch.tensor([3], device=cuda)
    logits, targets = torch.randn((18, 5000), generator=gen).to(cuda), torch.randint(0, 5000, (18,), generator=gen).to(cuda)
    tokens, index = torch.randint(0, 3, (2, 9), generator=gen).to(cuda), torch.tensor([0, 2, 5], device=cuda)

    def everything():
        copies = keys.clone(), values.clone()
        attention.keep_rows(*copies, rows, index, counts, offset=offset)
        return (attention.tree_attention(q, keys, values, rows, masks, counts=counts, offset=offset), *copies, *sampling.token_log_probs(logits, targets, top=7),
                *sampling.follow_drafts(tokens, torch.arange(-1, 8, device=cuda), tokens.flip(1), counts=counts))

    short = everything()
    calls = []
    for name in ("tree_attention", "keep_rows", "token_log_probs", "follow_drafts"):
        monkeypatch.setitem(_lib._draft_native, name, lambda *a, name=name: calls.append(name))
    for got, want in zip(everything(), short):
        assert torch.equal(got, want)
    assert sorted(set(calls)) == ["follow_drafts", "keep_rows", "token_log_probs", "tree_attention"]
