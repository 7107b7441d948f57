"""Workspaces of libajq_draft.so are what include/ajq_draft.h says of them."""

import ctypes

import pytest

from ajllm_amd import _lib


def _size(what, struct, at, **values):
    args = struct()
    for name, kind in struct._fields_:
        if kind is ctypes.c_void_p:
            setattr(args, name, at)
    for name, value in values.items():
        setattr(args, name, value)
    return getattr(_lib.load_draft(), what)(ctypes.byref(args))


@pytest.mark.parametrize("dtype,most", [(0, 32768), (1, 65536)])
@pytest.mark.parametrize("top", [0, 1, 64])
@pytest.mark.parametrize("rows", [1, 7, 5000])
def test_log_probs(rows, top, dtype, most):
    each = 16 // (4, 2)[dtype]   # logits of 16 bytes
    for vocab, ld, first in ((most, most, 0), (most + 1, most + each, 0), (most - each, most - 1, 4), (200000, 200000, 0), (200001, 200001, 4), (3 * most + 17, 4 * most, 0)):
        if vocab < top:
            continue
        size = _size("ajqt_log_probs_workspace", _lib.LogProbsArgs, 4096 + first, ld=ld, rows=rows, vocab=vocab, top=top, dtype=dtype)
        even = first == 0 and ld % each == 0
        if vocab <= (most if even else most - each):
            assert size == 0
            continue
        a_row, rest = divmod(size, rows)
        slices, left = divmod(a_row - 4, 16 + 8 * top)
        assert rest == 0 and left == 0 and vocab / most <= slices <= 2 + vocab / (most / 4 - each), (vocab, slices)


@pytest.mark.parametrize("batch,tokens,heads,kv,dim,max_len", [(1, 8, 16, 16, 128, 520), (8, 64, 32, 8, 128, 32832), (5, 3, 4, 1, 64, 4000), (1, 300, 5, 1, 32, 1500), (64, 2, 2, 2, 64, 100000)])
def test_tree_attention(batch, tokens, heads, kv, dim, max_len):
    for q_dtype in range(2):
        for cache_dtype in range(2):
            size = _size("ajqt_tree_attention_workspace", _lib.TreeAttentionArgs, 4096, cache_batch=kv * max_len * dim, cache_head=max_len * dim, batch=batch, tokens=tokens, heads=heads,
                         kv_heads=kv, dim=dim, max_len=max_len, q_dtype=q_dtype, cache_dtype=cache_dtype)
            if size:
                parts, left = divmod(size - 8 * batch, tokens * heads * (4 * dim + 8))
                assert left == 0 and batch < parts <= min(64 * batch, 1024 // kv)
