"""What libajq_serve.so refuses and what it lets through, without a GPU: calls that nothing refuses are stopped by a later check, so that none is launched."""

import ctypes

import pytest

from ajllm_amd import _lib
from tests.test_serve_abi import LOGITS, _filled, _refused, memory  # noqa: F401


@pytest.mark.parametrize("change", [dict(tokens_ld=0), dict(prompt_ld=0), dict(allowed_ld=0), dict(tokens_ld=0, prompt_ld=0, allowed_ld=0)])
def test_lists_and_masks_may_be_shared_by_all_rows(memory, change):  # noqa: F811
    args = _filled(_lib.AdjustLogitsArgs, memory, **{**LOGITS, "out": memory + 4, **change})   # (overlaps the logits: the last check)
    _refused(_lib.load_serve().ajqs_adjust_logits, args, -2, "out overlaps")


@pytest.mark.parametrize("change,message", [(dict(tokens_ld=-8), "tokens a row"), (dict(tokens_ld=1), "tokens a row"), (dict(prompt_ld=-1), "prompt tokens a row"),
                                            (dict(allowed_ld=-2), "words"), (dict(bias_ld=0), "biases a row")])
def test_other_strides_are_refused(memory, change, message):  # noqa: F811
    args = _filled(_lib.AdjustLogitsArgs, memory, **{**LOGITS, "out": memory + 1024, **change})
    _refused(_lib.load_serve().ajqs_adjust_logits, args, -2, message)
