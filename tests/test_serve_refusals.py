"""What libajq_serve.so refuses and what it lets through, without a GPU: calls that nothing refuses are stopped by a later check, so that none is launched."""

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from ajllm_amd import _lib, sampling
from tests.test_serve_abi import LOGITS, NORM, SHARED, _filled, _refused, memory  # noqa: F401


@pytest.mark.parametrize("change", [dict(tokens_ld=0), dict(prompt_ld=0), dict(allowed_ld=0), dict(tokens_ld=0, prompt_ld=0, allowed_ld=0)])
def test_lists_and_masks_may_be_shared_by_all_rows(memory, change):  # noqa: F811
    args = _filled(_lib.AdjustLogitsArgs, memory, **{**LOGITS, "out": memory + 4, **change})   # (overlaps the logits: the last check)
    _refused(_lib.load_serve().ajqs_adjust_logits, args, -2, "out overlaps")


@pytest.mark.parametrize("change,message", [(dict(tokens_ld=-8), "tokens a row"), (dict(tokens_ld=1), "tokens a row"), (dict(prompt_ld=-1), "prompt tokens a row"),
                                            (dict(allowed_ld=-2), "words"), (dict(bias_ld=0), "biases a row")])
def test_other_strides_are_refused(memory, change, message):  # noqa: F811
    args = _filled(_lib.AdjustLogitsArgs, memory, **{**LOGITS, "out": memory + 1024, **change})
    _refused(_lib.load_serve().ajqs_adjust_logits, args, -2, message)


def test_launches_of_2_to_the_32_lanes_are_refused(memory):  # noqa: F811
    """A grid has fewer than 2^32 lanes in a dimension.  (One less is let through, to a later check.)"""
    lib = _lib.load_serve()
    many = 2 ** 24   # workgroups of 256 lanes
    for batch, tokens in ((many, 1), (2 ** 12, 2 ** 12), (3, many // 3 + 1)):
        _refused(lib.ajqs_norm_rope, _filled(_lib.NormRopeArgs, memory, **{**NORM, "batch": batch, "tokens": tokens, "values": memory + 2 ** 38}), -2, "tokens in a launch")
    _refused(lib.ajqs_norm_rope, _filled(_lib.NormRopeArgs, memory, **{**NORM, "batch": 1, "tokens": many - 1, "eps": -1.0, "values": memory + 2 ** 38}), -2, "epsilon")
    one = {**SHARED, "heads": 1, "kv_heads": 1, "groups": 1}
    # everything in one launch, four sequences a workgroup, or more tokens; parts, whose merge takes four queries a workgroup
    for change in (dict(batch=4 * many), dict(batch=4 * many, prefix_cap=4096), dict(batch=2, tokens=2 * many, prefix_cap=4096)):
        args = _filled(_lib.SharedAttentionArgs, memory, **{**one, **change})
        _refused(lib.ajqs_shared_attention, args, -2, "too many", memory, 1 << 62)
    for batch, vocab in ((2 ** 22, 16384), (2 ** 22, 3), (2 ** 19, 128256)):
        args = _filled(_lib.AdjustLogitsArgs, memory, **{**LOGITS, "out": memory + 4 * 2 ** 19, "batch": batch, "vocab": vocab, "ld": 2 ** 20, "out_ld": 2 ** 20, "allowed": None})
        _refused(lib.ajqs_adjust_logits, args, -2, f"{batch} rows of {vocab}")


@pytest.mark.filterwarnings("ignore:Accessing the data pointer")
@pytest.mark.parametrize("name", ["rows", "vocabulary", "tokens", "prompt", "biases", "masks"])
def test_adjust_logits_refuses_sizes_past_32_bits(name):
    """A size handed on as 32 bits of it would be another size: 2^32 + 5 tokens are not 5.  (Tensors without memory.)"""
    size = lambda this, other: 2 ** 32 + 5 if name == this else other  # noqa: E731
    with FakeTensorMode():
        whole = lambda *shape: torch.empty(shape, dtype=torch.long, device="cuda")  # noqa: E731
        batch, vocab = size("rows", 1), size("vocabulary", 64)
        args = dict(tokens=whole(batch, size("tokens", 3)), prompt=whole(batch, size("prompt", 3)), bias_ids=whole(batch, size("biases", 3)),
                    bias=torch.empty((batch, size("biases", 3)), dtype=torch.float32, device="cuda"),
                    allowed=torch.empty((size("masks", batch), (vocab + 31) // 32), dtype=torch.int32, device="cuda"))
        with pytest.raises(ValueError, match="2\\^31"):
            sampling.adjust_logits(torch.empty((batch, vocab), dtype=torch.float32, device="cuda"), **args)


@pytest.mark.parametrize("shape", [dict(prefix_cap=1024, max_len=512, prefix_group=131072, prefix_head=65536, cache_batch=65536, cache_head=32768),   # parts of either
                                   dict(prefix_cap=1024, max_len=16, tokens=40, cache_dtype=1, prefix_group=131072, prefix_head=65536)])             # a walk in parts
def test_workspaces_that_do_not_do_are_refused(memory, shape):  # noqa: F811
    lib = _lib.load_serve()
    args = _filled(_lib.SharedAttentionArgs, memory, **{**SHARED, **shape})
    need = lib.ajqs_shared_attention_workspace(ctypes.byref(args))
    assert need > 0 and need % (4 * 4 * args.tokens * (8 + 4 * 64)) == 0   # [parts, queries] of (maximum, sum) and 64 components, fp32
    for at, size, status, message in ((memory, need - 1, -6, "bytes needed"), (None, need, -6, "bytes needed"), (memory, 0, -6, "bytes needed"),
                                      (memory + 8, need, -3, "workspace must be")):
        _refused(lib.ajqs_shared_attention, args, status, message, at, size)
