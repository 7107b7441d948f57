"""libajq_serve.so without a GPU: it exports what its header declares, the ctypes structures have the header's layout, and arguments are refused
before any HIP call."""

import ctypes
import re
import subprocess
from pathlib import Path

import pytest
import torch

from ajllm_amd import _lib, attention, sampling

HEADER = Path(__file__).resolve().parents[1] / "include" / "ajq_serve.h"
STRUCTS = {"ajqs_norm_rope_args": _lib.NormRopeArgs, "ajqs_shared_attention_args": _lib.SharedAttentionArgs,
           "ajqs_adjust_logits_args": _lib.AdjustLogitsArgs}


def test_header_symbols_are_exported_and_bound():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    names = sorted(set(re.findall(r"\b(ajqs_[a-z0-9_]+)\s*\(", text)))
    lib = _lib.load_serve()
    assert names == sorted(_lib.SERVE_SIGNATURES) and len(names) >= 5
    for name in names:
        assert hasattr(lib, name), f"{name} declared in ajq_serve.h but not exported by libajq_serve.so"


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
    q, cache, whole = torch.zeros(2, 4, 1, 64), torch.zeros(2, 2, 8, 64), torch.zeros(2, dtype=torch.long)
    with pytest.raises(ValueError, match="norm_rope needs tensors on a ROCm device"):
        attention.norm_rope(torch.zeros(2, 512), torch.zeros(8, 32), torch.zeros(8, 32), cache, cache.clone(), whole, heads=4)
    with pytest.raises(ValueError, match="shared_prefix_attention needs tensors on a ROCm device"):
        attention.shared_prefix_attention(q, cache, cache, whole, cache, cache, whole)
    with pytest.raises(ValueError, match="adjust_logits needs tensors on a ROCm device"):
        sampling.adjust_logits(torch.zeros(2, 100), repetition=1.5)


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
    assert message in _lib.load_serve().ajqs_last_error().decode()
    with pytest.raises(ValueError, match=message):
        _lib.check_serve(status, "call")


NORM = dict(ld=512, cache_batch=2048, cache_head=1024, batch=2, tokens=1, heads=4, kv_heads=2, dim=64, max_len=16, table_rows=8, eps=1e-5)


def test_norm_rope_refuses(memory):
    call = _lib.load_serve().ajqs_norm_rope
    assert call(None, None) == -1
    for name in ("qkv", "cosine", "sine", "rows", "keys", "values", "q"):
        _refused(call, _filled(_lib.NormRopeArgs, memory, **{**NORM, name: None}), -1, "null")
    for change in (dict(batch=0), dict(tokens=0), dict(kv_heads=3), dict(kv_heads=0), dict(heads=-4), dict(max_len=0), dict(table_rows=0),
                   dict(batch=2 ** 20, tokens=2 ** 12)):
        _refused(call, _filled(_lib.NormRopeArgs, memory, **{**NORM, **change}), -2, "unsupported shape")
    for change in (dict(ld=508), dict(ld=514), dict(ld=-512)):
        _refused(call, _filled(_lib.NormRopeArgs, memory, **{**NORM, **change}), -2, "rows of")
    for change in (dict(dim=48), dict(dim=256)):
        _refused(call, _filled(_lib.NormRopeArgs, memory, **{**NORM, **change}), -4, "head size")
    for change in (dict(in_dtype=2), dict(q_dtype=-1), dict(cache_dtype=3)):
        _refused(call, _filled(_lib.NormRopeArgs, memory, **{**NORM, **change}), -4, "element type")
    for name in ("qkv", "q", "cosine", "sine", "q_gain", "k_gain", "keys", "values"):
        _refused(call, _filled(_lib.NormRopeArgs, memory, **{**NORM, name: memory + 8}), -3, "aligned")
    for change in (dict(cache_head=1020), dict(cache_batch=2044)):
        _refused(call, _filled(_lib.NormRopeArgs, memory, **{**NORM, **change}), -3, "multiples of 8")
    for change in (dict(cache_head=512), dict(cache_batch=0)):
        _refused(call, _filled(_lib.NormRopeArgs, memory, **{**NORM, **change}), -2, "overlap")
    _refused(call, _filled(_lib.NormRopeArgs, memory, **{**NORM, "cache_head": -1024}), -2, "negative")
    for change in (dict(cache_head=1024, cache_batch=1024), dict(cache_head=2048, cache_batch=2048), dict(cache_head=1032, cache_batch=1024),
                   dict(batch=3, cache_head=4096, cache_batch=2048)):
        _refused(call, _filled(_lib.NormRopeArgs, memory, **{**NORM, **change}), -2, "cache heads that overlap")


def test_norm_rope_refuses_keys_and_values_that_overlap(memory):
    """Against the definition: no element of one's heads is one of the other's.  (Layouts that are in order are refused for their epsilon's sake:
    nothing is launched.)"""
    call = _lib.load_serve().ajqs_norm_rope
    heads = lambda at, b, h: {at + i * b + j * h + e for i in range(2) for j in range(2) for e in range(1024)}  # noqa: E731
    met = set()
    for d in (0, 8, 1016, 1024, 1032, 2048, 3064, 4096, 4104, 5120, 6144, 7160, 7168, 9000):
        for batch, head in ((2048, 1024), (4096, 2048), (1024, 2048), (8192, 1024), (1024, 8192), (2048, 4096)):
            meets = bool(heads(0, batch, head) & heads(d, batch, head))
            met.add(meets)
            args = _filled(_lib.NormRopeArgs, memory, **{**NORM, "values": memory + 4 * d, "cache_batch": batch, "cache_head": head})
            if meets:
                _refused(call, args, -2, "keys and values that overlap")
            else:
                args.eps = -1.0   # (the last check)
                _refused(call, args, -2, "epsilon")
    assert met == {False, True}


SHARED = dict(prefix_group=2048, prefix_head=1024, cache_batch=2048, cache_head=1024, groups=2, batch=4, tokens=1, heads=4, kv_heads=2, dim=64,
              prefix_cap=16, max_len=16)


def test_shared_attention_refuses(memory):
    lib = _lib.load_serve()
    call = lib.ajqs_shared_attention
    assert call(None, None, 0, None) == -1
    for name in ("q", "prefix_keys", "prefix_values", "keys", "values", "prefix_lengths", "rows", "out"):
        _refused(call, _filled(_lib.SharedAttentionArgs, memory, **{**SHARED, name: None}), -1, "null", memory, 1 << 30)
    for change in (dict(batch=0), dict(groups=0), dict(batch=5), dict(tokens=0), dict(kv_heads=3), dict(prefix_cap=0), dict(max_len=0), dict(heads=0)):
        args = _filled(_lib.SharedAttentionArgs, memory, **{**SHARED, **change})
        _refused(call, args, -2, "unsupported shape", memory, 1 << 30)
        assert lib.ajqs_shared_attention_workspace(ctypes.byref(args)) == 0
    _refused(call, _filled(_lib.SharedAttentionArgs, memory, **{**SHARED, "batch": 2 ** 20, "tokens": 2 ** 10}), -2, "too many queries", memory, 1 << 30)
    _refused(call, _filled(_lib.SharedAttentionArgs, memory, **{**SHARED, "dim": 96}), -4, "head size", memory, 1 << 30)
    for change in (dict(q_dtype=2), dict(cache_dtype=9)):
        _refused(call, _filled(_lib.SharedAttentionArgs, memory, **{**SHARED, **change}), -4, "element type", memory, 1 << 30)
    for name in ("q", "out", "prefix_keys", "prefix_values", "keys", "values"):
        _refused(call, _filled(_lib.SharedAttentionArgs, memory, **{**SHARED, name: memory + 4}), -3, "aligned", memory, 1 << 30)
    for change in (dict(prefix_head=1028), dict(cache_batch=3)):
        _refused(call, _filled(_lib.SharedAttentionArgs, memory, **{**SHARED, **change}), -3, "multiples of 8", memory, 1 << 30)
    need = lib.ajqs_shared_attention_workspace(ctypes.byref(_filled(_lib.SharedAttentionArgs, memory, **SHARED)))
    if need:
        _refused(call, _filled(_lib.SharedAttentionArgs, memory, **SHARED), -6, "bytes needed", memory, need - 1)
        _refused(call, _filled(_lib.SharedAttentionArgs, memory, **SHARED), -6, "bytes needed", None, need)
        _refused(call, _filled(_lib.SharedAttentionArgs, memory, **SHARED), -3, "workspace must be", memory + 8, need)


LOGITS = dict(ld=64, out_ld=64, tokens_ld=8, prompt_ld=8, bias_ld=4, allowed_ld=2, batch=2, vocab=64, max_tokens=8, max_prompt=8, biases=4, masks=2)


def test_adjust_logits_refuses(memory):
    call = _lib.load_serve().ajqs_adjust_logits
    good = {**LOGITS, "out": memory + 1024}
    assert call(None, None) == -1
    for name in ("logits", "out", "bias"):
        _refused(call, _filled(_lib.AdjustLogitsArgs, memory, **{**good, name: None}), -1, "null")
    for change in (dict(batch=0), dict(vocab=0), dict(ld=63), dict(out_ld=0)):
        _refused(call, _filled(_lib.AdjustLogitsArgs, memory, **{**good, **change}), -2, "unsupported shape")
    _refused(call, _filled(_lib.AdjustLogitsArgs, memory, **{**good, "dtype": 2}), -4, "element type")
    for change in (dict(dtype=1), dict(ld=68)):   # in place
        _refused(call, _filled(_lib.AdjustLogitsArgs, memory, **{**LOGITS, **change}), -4, "in place")
    for change, message in ((dict(max_tokens=9), "tokens a row"), (dict(max_tokens=2 ** 20, tokens_ld=2 ** 20), "tokens a row"), (dict(max_prompt=-1), "prompt"),
                            (dict(biases=1025, bias_ld=1025), "biases a row"), (dict(bias_ld=3), "biases a row"), (dict(allowed_ld=1), "words"), (dict(masks=0), "words"),
                            (dict(masks=1, allowed_rows=None), "masks for")):
        _refused(call, _filled(_lib.AdjustLogitsArgs, memory, **{**good, **change}), -2, message)
    for name, by in (("logits", 2), ("out", 1), ("allowed", 1)):
        _refused(call, _filled(_lib.AdjustLogitsArgs, memory, **{**good, name: memory + 512 + by}), -3, "aligned")


def test_adjust_logits_refuses_an_overlapping_out(memory):
    call = _lib.load_serve().ajqs_adjust_logits
    good = {**LOGITS, "ld": 128, "out_ld": 128, "batch": 2}
    for by in (4, 252, -4, -252, 512, 508, 516, 764):   # bytes; rows of 256 in a pitch of 512
        args = _filled(_lib.AdjustLogitsArgs, memory + 1024, **{**good, "out": memory + 1024 + by})
        _refused(call, args, -2, "out overlaps")
    for change in (dict(out=memory + 1024 + 256, out_ld=64), dict(out=memory + 1024 + 64, dtype=1, ld=256), dict(out=memory + 1024 + 64, batch=1)):
        _refused(call, _filled(_lib.AdjustLogitsArgs, memory + 1024, **{**good, **change}), -2, "out overlaps")
