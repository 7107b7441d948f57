"""Decoders on the operators of decoding many continuations of one prompt: shared prefixes, questions of different lengths, heads that are normed,
adjusted logits, each against the model's own code."""

import copy
import json

import pytest
import torch
from safetensors.torch import save_file

from ajllm_amd import checkpoint, decoding, modeling, quantize_model_
from tests.helpers import errors

pytestmark = pytest.mark.gpu

VOCAB = 512


def _model(cuda, scheme="w8a16", head_norm=False, heads=4, kv_heads=2, context=256):
    torch.manual_seed(31)
    model = modeling.TransformerLM(vocab_size=VOCAB, context_length=context, d_model=256, num_layers=2, num_heads=heads, num_kv_heads=kv_heads,
                                   d_ff=640, head_norm=head_norm).eval()
    if head_norm:
        for layer in model.layers:
            torch.nn.init.uniform_(layer.attention.q_norm.weight, 0.5, 1.5)
            torch.nn.init.uniform_(layer.attention.k_norm.weight, 0.5, 1.5)
    return quantize_model_(copy.deepcopy(model).to(cuda), scheme)


def _ids(seed, *lengths):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randint(0, VOCAB, (n,), generator=gen).tolist() for n in lengths]


# Both attentions round their result to bf16, flash arithmetic its weights too, and what the next product rounds moves with them: the bound on logits of two
# such runs that the decoders' tests have (test_gpu_model.py).
LOGITS = 2e-2


def _follow(model, dec, before, new):
    """Greedy tokens of ``dec``, step by step: its logits are the model's for the same tokens, its choice is its logits' maximum."""
    for count in range(1, new + 1):
        got = dec.generate(count).tolist()
        if count == 1:
            continue
        mine = dec.logits_full[:, :VOCAB].float().cpu()
        for b, ids in enumerate(before):
            with torch.no_grad():
                want = model(torch.tensor([ids + got[b][:-1]], device=dec.device))[0, -1].float().cpu()
            assert errors(mine[b], want)[1] <= LOGITS, (b, count)
            assert got[b][-1] == int(mine[b].argmax())
    return got


@pytest.mark.parametrize("kv_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("head_norm", [False, True])
@pytest.mark.parametrize("completions", [1, 3, 20])
def test_completions_of_shared_prompts(cuda, kv_dtype, head_norm, completions):
    model = _model(cuda, head_norm=head_norm)
    prompts = _ids(1, 33, 70)
    dec = decoding.SharedPrefixDecoder(model, 2, completions, 80, 40, kv_dtype)
    dec.prefill(prompts)
    if completions == 1:
        _follow(model, dec, prompts, 12)
        return
    got = dec.generate(12)
    assert all(torch.equal(got[b], got[b - b % completions]) for b in range(2 * completions))   # (greedy: all alike)
    one = decoding.SharedPrefixDecoder(model, 2, completions, 80, 40, kv_dtype)
    one.prefill(prompts)
    one.steps_per_graph = 1
    assert torch.equal(one.generate(12), got)
    one.prefill(_ids(2, 80, 1))   # the recorded step goes on with other prompts
    again = one.generate(5)
    fresh = decoding.SharedPrefixDecoder(model, 2, completions, 80, 40, kv_dtype)
    fresh.prefill(_ids(2, 80, 1))
    assert torch.equal(fresh.generate(5), again)


@pytest.mark.parametrize("kv_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("head_norm", [False, True])
def test_questions_behind_a_shared_text(cuda, kv_dtype, head_norm):
    model = _model(cuda, "w4a16_g128", head_norm)
    texts, questions = _ids(3, 50, 61), _ids(4, 1, 17, 40, 3)
    dec = decoding.SharedPrefixDecoder(model, 2, 2, 61, 64, kv_dtype)
    dec.prefill(texts, questions)
    _follow(model, dec, [texts[b // 2] + q for b, q in enumerate(questions)], 10)


def test_launches_of_a_step(cuda):
    model = _model(cuda)
    base = decoding.FusedDecoder(model, 4, 64)
    for prefix_len, dtype, launches in ((32, torch.bfloat16, 2), (160, torch.float32, 3)):   # (few rows: attention in one launch)
        dec = decoding.SharedPrefixDecoder(model, 1, 4, prefix_len, 40, dtype)
        assert dec.attention_launches == launches
        assert dec.launches_per_step() == base.launches_per_step() + 2 * (launches - base.attention_launches)
    assert decoding.FusedDecoder(_model(cuda, head_norm=True), 4, 64).launches_per_step() == base.launches_per_step() + 2


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("batch", [1, 6])
def test_normed_heads(cuda, fused, batch):
    """A model whose heads are normed: the all-kernel step and prompt against its own code."""
    model = _model(cuda, head_norm=True)
    prompt = torch.tensor(_ids(5, *[30] * batch))
    dec = decoding.FusedDecoder(model, batch, 64)
    dec.prefill(prompt, fused=fused)
    _follow(model, dec, prompt.tolist(), 10)


def test_normed_heads_are_configured_and_stored(cuda, tmp_path):
    from ajllm_amd import checkpoint

    config = {"d_model": 256, "num_layers": 1, "num_heads": 4, "context_length": 64, "d_ff": 640, "normalization": {"heads": True}}
    model = modeling.build_model(config, VOCAB)
    assert "layers.0.attention.q_norm.weight" in model.state_dict()
    torch.nn.init.uniform_(model.layers[0].attention.k_norm.weight, 0.5, 1.5)
    fast = quantize_model_(model.to(cuda), "w8a16")
    path = tmp_path / "q.safetensors"
    checkpoint.save_quantized(path, fast, "w8a16", checkpoint.model_config(fast))
    back, _ = checkpoint.load_quantized(path, cuda)
    tokens = torch.tensor(_ids(6, 20), device=cuda)
    assert torch.equal(back(tokens), fast(tokens))
    assert "q_norm" not in str(list(modeling.build_model({**config, "normalization": {}}, VOCAB).state_dict()))


def _decoders(cuda, batch):
    model = _model(cuda)
    prompt = torch.tensor(_ids(7, 20) * batch)

    def shared():
        dec = decoding.SharedPrefixDecoder(model, 1, batch, 20, 80)
        prefill = dec.prefill
        dec.prefill = lambda _: prefill(prompt[:1])
        return dec

    return prompt, [lambda: decoding.GraphDecoder(model, batch, 100), lambda: decoding.FusedDecoder(model, batch, 100), shared]


@pytest.mark.parametrize("batch", [1, 5])
def test_penalties_biases_and_masks_in_a_decoder(cuda, batch):
    prompt, decoders = _decoders(cuda, batch)
    words = (VOCAB + 31) // 32
    for make in decoders:
        dec = make()
        dec.set_penalties(frequency=1e4)                    # nothing is produced twice
        dec.prefill(prompt)
        got = dec.generate(60)
        assert all(len(set(row)) == 60 for row in got.tolist())
        few = make()
        few.steps_per_graph = 1
        few.set_penalties(frequency=1e4)
        few.prefill(prompt)
        few.generate(3)
        assert torch.equal(few.generate(60), got)
        dec.set_penalties(bias={7: 1e4, 11: 1e4 - 50}, presence=200.0)   # 7, then 11, then 7 and 11 are both 200 down: 7 again
        dec.prefill(prompt)
        assert dec.generate(4).tolist() == [[7, 11, 7, 7]] * batch
        dec.set_penalties(repetition=1e6)                   # nothing of the prompt either, while anything else has a positive logit
        dec.prefill(prompt)
        assert all(len(set(row) | set(ids)) == 40 + len(set(ids)) for row, ids in zip(dec.generate(40).tolist(), prompt.tolist()))
        allowed = torch.zeros((2, words), dtype=torch.int32, device=cuda)
        allowed[0, 3] = 0b1010                              # tokens 97 and 99
        allowed[1, 15] = -2 ** 31                           # token 511
        which = torch.zeros(batch, dtype=torch.long, device=cuda)
        dec.set_penalties(allowed=allowed, allowed_rows=which)
        dec.prefill(prompt)
        assert set(dec.generate(10).unique().tolist()) <= {97, 99}
        which.fill_(1)                                      # the program moves on in its grammar between calls
        assert dec.generate(14)[:, 10:].unique().tolist() == [511]
        allowed.zero_()                                     # nothing is allowed: the first token
        assert dec.generate(16)[:, 14:].unique().tolist() == [0]
        dec.set_penalties()
        dec.prefill(prompt)
        plain = make()
        plain.prefill(prompt)
        assert torch.equal(dec.generate(20), plain.generate(20))


def test_sampled_completions(cuda):
    """Sampling: completions of one prompt differ, equal seeds give equal ones, masks hold, a mask that leaves nothing gives the first token."""
    prompt, decoders = _decoders(cuda, 8)
    for make in decoders:
        runs = []
        for seed in (3, 3, 4):
            dec = make()
            dec.set_sampling(1.0, 0.95, seed=seed)
            dec.set_penalties(repetition=1.2, presence=0.5)
            dec.prefill(prompt)
            runs.append(dec.generate(30))
        assert torch.equal(runs[0], runs[1]) and not torch.equal(runs[0], runs[2])
        assert len({tuple(row) for row in runs[0].tolist()}) == 8
        allowed = torch.zeros((8, (VOCAB + 31) // 32), dtype=torch.int32, device=cuda)
        allowed[:, 2] = 0xF0
        dec.set_penalties(allowed=allowed)
        dec.prefill(prompt)
        assert set(dec.generate(12).unique().tolist()) <= {68, 69, 70, 71}
        allowed.zero_()
        assert dec.generate(14)[:, 12:].unique().tolist() == [0]


@pytest.mark.parametrize("top_p", [None, 0.9])
def test_sample_pick_of_a_row_that_allows_nothing(cuda, top_p):
    from ajllm_amd import _lib

    logits = torch.randn((3, 1000), generator=torch.Generator().manual_seed(1)).to(cuda)
    logits[1] = float("-inf")
    token, out, step = (torch.full((3, 1), 5, device=cuda) for _ in range(3))
    step.zero_()
    u = torch.full((1, 3), 0.7, device=cuda)
    _lib.check(_lib.load().ajq_sample_pick(logits.data_ptr(), 3, 1000, 1000, 1.0, top_p or 1.0, u.data_ptr(), 1, None, 0, None, token.data_ptr(),
                                           out.data_ptr(), 1, step.data_ptr(), None, None, None, torch.cuda.current_stream().cuda_stream), "sample_pick")
    assert token[1].item() == 0 and out[1].item() == 0 and 0 <= token[0].item() < 1000


def test_dense_decoder_with_penalties(cuda):
    """One of the dense models' decoders: nothing is produced twice, masks hold."""
    torch.manual_seed(2)
    mixer = {"heads": 4, "dim": 32, "rot_dim": 16, "vdim": 48, "kv_rank": 64, "scale": 0.15, "mask": {"size": 9}, "rot": {"base": 1000.0, "dims": 16}}
    model = modeling.build_model({"architecture": "Dorutar", "vocab": 97, "width": 80, "max_positions": 64, "norm": {"eps": 1e-5},
                                  "layers": [{"type": "latent_attention", "mixer": mixer, "mlp": {"kind": "dense", "ff": 96}}] * 2})
    model.to(cuda, torch.bfloat16).eval()
    prompt = torch.randint(0, 97, (3, 10), generator=torch.Generator().manual_seed(5))
    for seed in (None, 1):
        dec = decoding.DenseDecoder(model, 3, 60)
        if seed is not None:
            dec.set_sampling(1.0, 0.9, seed=seed)
        dec.set_penalties(frequency=1e4)
        dec.prefill(prompt)
        assert all(len(set(row)) == 40 for row in dec.generate(40).tolist())
        allowed = torch.zeros((3, 4), dtype=torch.int32, device=cuda)
        allowed[:, 3] = 1                                   # token 96, the last one
        dec.set_penalties(allowed=allowed)
        dec.prefill(prompt)
        assert dec.generate(8).unique().tolist() == [96]


def test_penalties_from_the_command_line(cuda, tmp_path, capsys):
    from ajllm_amd.__main__ import main as command

    torch.manual_seed(3)
    mixer = {"heads": 4, "dim": 32, "rot_dim": 16, "vdim": 48, "kv_rank": 64, "scale": 0.15, "mask": {"size": 9}, "rot": {"base": 1000.0, "dims": 16}}
    cfg = {"architecture": "Dorutar", "vocab": 97, "width": 80, "max_positions": 64, "norm": {"eps": 1e-5},
           "layers": [{"type": "latent_attention", "mixer": mixer, "mlp": {"kind": "dense", "ff": 96}}] * 2}
    (tmp_path / "config.json").write_text(json.dumps(cfg))
    model = modeling.build_model(cfg)
    names = model.checkpoint_names()
    save_file({names[k]: v.contiguous() for k, v in model.state_dict().items()}, str(tmp_path / "model.safetensors"))
    run = ["generate", "--model", str(tmp_path), "--tokens", "1,2,3,4", "--max-new-tokens", "40"]

    def tokens(*more):
        assert command(run + list(more)) == 0
        return [int(t) for t in capsys.readouterr().out.strip().splitlines()[-1].split(",")]

    model = checkpoint.load_model(tmp_path, cuda, torch.bfloat16)
    for more, penalties in (((), None), (("--presence-penalty", "1e4"), dict(presence=1e4)),
                            (("--repetition-penalty", "1.5", "--frequency-penalty", "0.5"), dict(repetition=1.5, frequency=0.5))):
        dec = decoding.DenseDecoder(model, 1, 44)
        if penalties:
            dec.set_penalties(**penalties)
        dec.prefill(torch.tensor([[1, 2, 3, 4]]))
        assert tokens(*more) == dec.generate(40)[0].tolist()
    assert len(set(tokens("--presence-penalty", "1e4"))) == 40
    with pytest.raises(SystemExit):
        command(run + ["--repetition-penalty", "0"])


def test_refusals(cuda):
    model = _model(cuda)
    for bad in (dict(prompts=0), dict(completions=0), dict(prefix_len=0), dict(max_len=250)):
        with pytest.raises(ValueError):
            decoding.SharedPrefixDecoder(**{**dict(model=model, prompts=1, completions=2, prefix_len=10, max_len=20), **bad})
    dec = decoding.SharedPrefixDecoder(model, 2, 2, 10, 20)
    for prompt, questions in ((_ids(1, 5), None), (_ids(1, 5, 11), None), (_ids(1, 5, 0), None), (_ids(1, 5, 5), _ids(2, 3, 3)), (_ids(1, 5, 5), _ids(2, 3, 3, 3, 20)),
                              (torch.zeros(5), None), ([[VOCAB], [1]], None), ([[1], [-1]], None), (_ids(1, 5, 5), [[1], [2], [3], [VOCAB]])):
        with pytest.raises(ValueError):
            dec.prefill(prompt, questions)
    dec.prefill(_ids(1, 5, 5), _ids(2, 3, 3, 3, 12))
    with pytest.raises(ValueError):
        dec.generate(9)
    with pytest.raises(ValueError):
        dec.set_penalties(repetition=0.0)
    with pytest.raises(ValueError):
        dec.set_penalties(bias={VOCAB: 1.0})
    with pytest.raises(ValueError):
        dec.set_penalties(allowed_rows=dec.rows)
