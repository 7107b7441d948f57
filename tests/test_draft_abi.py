"""libajq_draft.so without a GPU: it exports what its header declares, the ctypes structures have the header's layout, arguments are refused before any HIP
call; and the layout of a tree."""

import ctypes
import re
import subprocess
from pathlib import Path

import pytest
import torch

from ajllm_amd import _lib, attention, sampling
from tests import draft_plain

HEADER = Path(__file__).resolve().parents[1] / "include" / "ajq_draft.h"
STRUCTS = {"ajqt_tree_attention_args": _lib.TreeAttentionArgs, "ajqt_keep_rows_args": _lib.KeepRowsArgs, "ajqt_log_probs_args": _lib.LogProbsArgs,
           "ajqt_follow_drafts_args": _lib.FollowDraftsArgs}


def test_header_symbols_are_exported_and_bound():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    names = sorted(set(re.findall(r"\b(ajqt_[a-z0-9_]+)\s*\(", text)))
    lib = _lib.load_draft()
    assert names == sorted(_lib.DRAFT_SIGNATURES) and len(names) >= 7
    for name in names:
        assert hasattr(lib, name), f"{name} declared in ajq_draft.h but not exported by libajq_draft.so"


def test_structures_have_the_header_layout(tmp_path):
    lines = []
    for name, struct in STRUCTS.items():
        lines.append(f'  printf("{name} . %zu\\n", sizeof({name}));')
        lines += [f'  printf("{name} {field} %zu\\n", offsetof({name}, {field}));' for field, _ in struct._fields_]
    source = tmp_path / "layout.c"
    source.write_text("#include <stdio.h>\n#include \"%s\"\nint main(void) {\n%s\n  return 0;\n}\n" % (HEADER, "\n".join(lines)))
    subprocess.run(["gcc", str(source), "-o", str(tmp_path / "layout")], check=True)
    said = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout
    for line in said.splitlines():
        name, field, at = line.split()
        struct = STRUCTS[name]
        assert int(at) == (ctypes.sizeof(struct) if field == "." else getattr(struct, field).offset), line


def test_functions_need_a_gpu():
    whole = torch.zeros(2, 3, dtype=torch.long)
    cache = torch.zeros(2, 2, 8, 64)
    with pytest.raises(ValueError, match="tree_attention needs tensors on a ROCm device"):
        attention.tree_attention(torch.zeros(2, 4, 3, 64), cache, cache, whole[:, 0], torch.zeros(3, 1, dtype=torch.int32))
    with pytest.raises(ValueError, match="keep_rows needs tensors on a ROCm device"):
        attention.keep_rows(cache, cache.clone(), whole[:, 0], whole)
    with pytest.raises(ValueError, match="token_log_probs needs tensors on a ROCm device"):
        sampling.token_log_probs(torch.zeros(2, 100))
    with pytest.raises(ValueError, match="follow_drafts needs tensors on a ROCm device"):
        sampling.follow_drafts(whole, whole, whole)


@pytest.mark.parametrize("nodes", [1, 2, 31, 32, 33, 64, 65, 130])
def test_tree_masks(nodes):
    gen = torch.Generator().manual_seed(nodes)
    at = torch.arange(nodes)
    trees = [(at - 1 - torch.randint(0, 4, (nodes,), generator=gen)).clamp(min=0).masked_fill(at == 0, -1), at - 1, torch.zeros_like(at),
             torch.randint(-3, nodes + 3, (nodes,), generator=gen), torch.full_like(at, 2 ** 40), torch.full_like(at, -2 ** 63)]
    masks, depths = attention.tree_masks(torch.stack(trees))
    assert masks.dtype == torch.int32 and masks.shape == (len(trees), nodes, (nodes + 31) // 32) and depths.dtype == torch.int64
    table = draft_plain.sees(masks, len(trees), nodes)
    for i, tree in enumerate(trees):
        want, deep = draft_plain.ancestors(tree.tolist())
        assert torch.equal(table[i], want) and torch.equal(depths[i], deep)
        one, own = attention.tree_masks(tree)
        assert torch.equal(one, masks[i]) and torch.equal(own, depths[i])
    if nodes % 32:   # no bit behind the nodes
        assert int((masks[..., -1].long() & 0xFFFFFFFF).max()) < 2 ** (nodes % 32)


def test_tree_masks_refuses():
    for bad in (torch.zeros(3), torch.zeros(3, dtype=torch.int32), torch.zeros(1, 1, 3, dtype=torch.long), torch.zeros(0, dtype=torch.long),
                torch.zeros(2, 0, dtype=torch.long), torch.tensor(0)):
        with pytest.raises(ValueError, match="parents int64"):
            attention.tree_masks(bad)


@pytest.fixture()
def memory():
    buffer = ctypes.create_string_buffer(4096 + 16)   # host memory: only its address is inspected
    at = (ctypes.addressof(buffer) + 15) & ~15
    yield at
    del buffer


def _filled(struct, at, **values):
    args = struct()
    for name, kind in struct._fields_:
        if kind is ctypes.c_void_p:
            setattr(args, name, at)
    for name, value in values.items():
        setattr(args, name, value)
    return args


def _refused(call, args, status, message, *more):
    assert call(ctypes.byref(args), *more, None) == status
    assert message in _lib.load_draft().ajqt_last_error().decode()
    with pytest.raises(ValueError, match=message):
        _lib.check_draft(status, "call")


TREE = dict(cache_batch=2048, cache_head=1024, mask_batch=4, mask_token=1, batch=2, tokens=4, heads=4, kv_heads=2, dim=64, max_len=16)


def test_tree_attention_refuses(memory):
    lib = _lib.load_draft()
    call, more = lib.ajqt_tree_attention, (memory, 4096)
    assert call(None, None, 0, None) == -1 and lib.ajqt_tree_attention_workspace(None) == 0
    struct = _lib.TreeAttentionArgs
    for name in ("q", "keys", "values", "masks", "rows", "out"):
        _refused(call, _filled(struct, memory, **{**TREE, name: None}), -1, "null", *more)
        assert lib.ajqt_tree_attention_workspace(ctypes.byref(_filled(struct, memory, **{**TREE, name: None}))) == 0
    for change in (dict(batch=0), dict(tokens=0), dict(kv_heads=3), dict(kv_heads=0), dict(heads=-4), dict(max_len=0), dict(max_len=2 ** 30 + 1),
                   dict(tokens=2 ** 30 + 1)):
        _refused(call, _filled(struct, memory, **{**TREE, **change}), -2, "unsupported shape", *more)
    for change in (dict(batch=2 ** 20, tokens=2 ** 12), dict(batch=2 ** 30, tokens=2 ** 30)):
        _refused(call, _filled(struct, memory, **{**TREE, **change}), -2, "too many queries", *more)
    for change in (dict(dim=48), dict(dim=256)):
        _refused(call, _filled(struct, memory, **{**TREE, **change}), -4, "head size", *more)
    for change in (dict(q_dtype=2), dict(cache_dtype=-1)):
        _refused(call, _filled(struct, memory, **{**TREE, **change}), -4, "element type", *more)
    for change in (dict(mask_batch=-1), dict(mask_token=-1)):
        _refused(call, _filled(struct, memory, **{**TREE, **change}), -2, "mask stride", *more)
    for name in ("q", "out", "keys", "values"):
        _refused(call, _filled(struct, memory, **{**TREE, name: memory + 8}), -3, "aligned", *more)
    _refused(call, _filled(struct, memory, **{**TREE, "masks": memory + 2}), -3, "aligned", *more)
    for change in (dict(cache_head=1020), dict(cache_batch=2044)):
        _refused(call, _filled(struct, memory, **{**TREE, **change}), -3, "multiples of 8", *more)
    _refused(call, _filled(struct, memory, **{**TREE, "cache_head": -1024}), -2, "negative", *more)


def test_tree_attention_refuses_workspaces_and_large_launches(memory):
    lib = _lib.load_draft()
    args = _filled(_lib.TreeAttentionArgs, memory, **{**TREE, "batch": 1, "max_len": 20000, "cache_dtype": 1})   # (long and alone: in parts)
    size = lib.ajqt_tree_attention_workspace(ctypes.byref(args))
    assert size > 0
    call = lib.ajqt_tree_attention
    for room, given in ((None, 0), (None, size), (memory, 0), (memory, size - 1)):
        _refused(call, args, -6, "workspace of", room, given)
    _refused(call, args, -3, "16-byte aligned", memory + 8, size)
    _refused(call, _filled(_lib.TreeAttentionArgs, memory, **{**TREE, "batch": 2 ** 28, "tokens": 1, "heads": 1, "kv_heads": 1}), -2, "too many tiles", memory, 4096)


KEEP = dict(cache_layer=4096, cache_batch=2048, cache_head=1024, index_ld=5, layers=2, batch=2, kv_heads=2, dim=64, max_len=16, width=5)


def test_keep_rows_refuses(memory):
    call, struct = _lib.load_draft().ajqt_keep_rows, _lib.KeepRowsArgs
    far = {"values": memory + 2 ** 20}
    assert call(None, None) == -1
    for name in ("keys", "values", "rows", "index"):
        _refused(call, _filled(struct, memory, **{**KEEP, **far, name: None}), -1, "null")
    for change in (dict(layers=0), dict(batch=0), dict(kv_heads=0), dict(max_len=0), dict(width=0), dict(index_ld=-5), dict(index_ld=4), dict(max_len=2 ** 30 + 1)):
        _refused(call, _filled(struct, memory, **{**KEEP, **far, **change}), -2, "unsupported shape")
    _refused(call, _filled(struct, memory, **{**KEEP, **far, "dim": 48}), -4, "head size")
    _refused(call, _filled(struct, memory, **{**KEEP, **far, "dtype": 2}), -4, "element type")
    for change in (dict(cache_layer=4100), dict(cache_layer=-4096), dict(cache_head=1020), dict(cache_batch=2044), dict(keys=memory + 8), dict(values=memory + 8)):
        _refused(call, _filled(struct, memory, **{**KEEP, **far, **change}), -3, "8 elements")
    for change in (dict(cache_layer=2048), dict(cache_batch=1024), dict(cache_head=512), dict(cache_layer=0), dict(values=memory), dict(values=memory + 2048),
                   dict(keys=memory + 2 ** 20 + 4096 * 4 - 64)):
        _refused(call, _filled(struct, memory, **{**KEEP, **far, **change}), -2, "overlap")
    _refused(call, _filled(struct, memory, **{**KEEP, "layers": 2 ** 12, "batch": 2 ** 12, "cache_layer": 2 ** 26, "values": memory + 2 ** 50}), -2, "heads")


PROBS = dict(ld=100, rows=4, vocab=100, top=5)


def test_log_probs_refuses(memory):
    lib = _lib.load_draft()
    call, struct, more = lib.ajqt_log_probs, _lib.LogProbsArgs, (memory, 4096)
    assert call(None, None, 0, None) == -1 and lib.ajqt_log_probs_workspace(None) == 0
    for name in ("logits", "log_probs", "ranks", "top_log_probs", "top_ids"):
        _refused(call, _filled(struct, memory, **{**PROBS, name: None}), -1, "null", *more)
    for change in (dict(rows=0), dict(vocab=0), dict(ld=-1), dict(top=-1), dict(top=65), dict(vocab=4)):
        _refused(call, _filled(struct, memory, **{**PROBS, **change}), -2, "unsupported shape", *more)
    _refused(call, _filled(struct, memory, **{**PROBS, "dtype": 2}), -4, "element type", *more)
    for change in (dict(logits=memory + 2), dict(logits=memory + 1, dtype=1), dict(log_probs=memory + 2), dict(entropy=memory + 1), dict(top_log_probs=memory + 2)):
        _refused(call, _filled(struct, memory, **{**PROBS, **change}), -3, "aligned", *more)


def test_log_probs_refuses_workspaces_and_large_launches(memory):
    lib = _lib.load_draft()
    for dtype, top in ((0, 0), (0, 64), (1, 5)):
        args = _filled(_lib.LogProbsArgs, memory, **{**PROBS, "vocab": 200000, "ld": 200000, "top": top, "dtype": dtype})
        size = lib.ajqt_log_probs_workspace(ctypes.byref(args))
        assert size > 0
        for room, given in ((None, 0), (None, size), (memory, 0), (memory, size - 1)):
            _refused(lib.ajqt_log_probs, args, -6, "workspace of", room, given)
        _refused(lib.ajqt_log_probs, args, -3, "16-byte aligned", memory + 8, size)
    for change in (dict(rows=2 ** 24 + 1), dict(rows=2 ** 23, vocab=40000, ld=40000)):
        _refused(lib.ajqt_log_probs, _filled(_lib.LogProbsArgs, memory, **{**PROBS, **change}), -2, "rows", memory, 4096)


def test_follow_drafts_refuses(memory):
    call, struct = _lib.load_draft().ajqt_follow_drafts, _lib.FollowDraftsArgs
    base = dict(tokens_ld=6, parents_ld=6, choices_ld=6, choices_step=1, batch=2, nodes=6)
    assert call(None, None) == -1
    for name in ("tokens", "parents", "choices", "path", "accepted", "chosen"):
        _refused(call, _filled(struct, memory, **{**base, name: None}), -1, "null")
    for change in (dict(batch=0), dict(nodes=0), dict(nodes=4097), dict(tokens_ld=-1), dict(parents_ld=-1), dict(choices_ld=-1), dict(choices_step=-1),
                   dict(batch=2 ** 31 - 1)):
        _refused(call, _filled(struct, memory, **{**base, **change}), -2, "unsupported shape")


def test_norm_rope_at_refuses(memory):
    lib = _lib.load_serve()
    args = _filled(_lib.NormRopeArgs, memory, ld=512, cache_batch=2048, cache_head=1024, batch=2, tokens=1, heads=4, kv_heads=2, dim=64, max_len=16, table_rows=8, eps=1e-5,
                   values=memory + 2 ** 20)
    assert lib.ajqs_norm_rope_at(None, memory, 1, None) == -1
    assert lib.ajqs_norm_rope_at(ctypes.byref(args), memory, -1, None) == -2 and "stride of the depths" in lib.ajqs_last_error().decode()
