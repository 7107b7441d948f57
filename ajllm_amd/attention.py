"""Host side of the library's causal prefill attention (``ajq_attn_prefill``), and of attention for sequences that share a prefix
(``norm_rope``, ``shared_prefix_attention``).

The first stands where the reference switches to its FlashAttention under ``use_flash_attention``
(src/ajllm/modeling/attention.py:106-117; its own kernels, flash_attention.py:44-108,194-298, need
CUDA/Triton).  Same contract as there: the arithmetic is flash attention's (bf16 products, fp32
online softmax), not bit-for-bit the eager fp32 one, so it is opt-in.
"""

from __future__ import annotations

import ctypes
from contextlib import nullcontext

import torch

from . import _lib

_HERE = nullcontext()
COPIED_WORK = 3.6e9   # half the FLOP below which ajq_attn_prefill_workspace says 0 (tests/test_modeling.py): short calls are not asked


def flash_prefill(q: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, start: int,
                  out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Causal attention of the ``T`` new positions ``start .. start + T - 1``.

    ``q`` fp32 ``[B, H, T, hd]`` (rotated; hd 128, 64 or 32); ``keys`` / ``values`` ``[B, Hkv, max_len, hd]`` fp32 or
    bf16 whose rows ``0 .. start + T - 1`` are filled (a KV cache, or the keys and values themselves
    with ``start == 0``).  Returns ``[B, T, H * hd]`` in ``out_dtype`` (fp32, or bf16 = its rounding)."""
    if not q.is_cuda:
        raise ValueError("flash_prefill needs tensors on a ROCm device (there is no CPU path)")
    batch, heads, seq, hd = q.shape
    kv_heads, max_len = keys.shape[1], keys.shape[2]
    if hd not in (128, 64, 32) or keys.shape != values.shape or keys.shape[0] != batch or keys.shape[3] != hd:
        raise ValueError("flash_prefill: q [B, H, T, hd] and caches [B, Hkv, max_len, hd] with hd 128, 64 or 32 expected")
    if keys.dtype not in (torch.float32, torch.bfloat16) or values.dtype != keys.dtype:
        raise ValueError("flash_prefill: the caches must be float32 or bfloat16")
    if not (keys.is_contiguous() and values.is_contiguous()):
        raise ValueError("flash_prefill: the caches must be contiguous")
    if out_dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("flash_prefill: out_dtype must be float32 or bfloat16")
    q = q.float().contiguous()
    out = torch.empty((batch, seq, heads * hd), dtype=out_dtype, device=q.device)
    flag = _lib.AJQ_KV_F32 if keys.dtype == torch.float32 else _lib.AJQ_KV_BF16
    # (entering and leaving a device that is the current one anyway: 1.1 of 12.2 us, what a small call takes)
    with _HERE if q.get_device() == torch.cuda.current_device() else torch.cuda.device(q.device):
        status = prefill_attention(q, keys, values, flag, batch, heads, kv_heads, seq, start, max_len, hd, out,
                                   _lib.AJQ_OUT_F32 if out_dtype == torch.float32 else _lib.AJQ_OUT_BF16,
                                   torch.cuda.current_stream().cuda_stream)
    _lib.check(status, "attn_prefill")
    return out


def prefill_attention(q: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, flag: int, batch: int, heads: int, kv_heads: int, seq: int,
                      start: int, max_len: int, hd: int, out: torch.Tensor, out_flag: int, stream: int) -> int:
    """``ajq_attn_prefill`` on the current device, with a bf16 copy of fp32 caches where that is faster; its status."""
    lib = _lib.load()
    if flag == _lib.AJQ_KV_F32 and batch * heads * seq * (2 * start + seq) * hd > COPIED_WORK:
        size = lib.ajq_attn_prefill_workspace(flag, batch, heads, kv_heads, seq, start, hd)
        try:
            room = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
        except torch.OutOfMemoryError:  # (the kernel that needs no copy)
            room = None
        if room is not None:
            return lib.ajq_attn_prefill_in(q.data_ptr(), keys.data_ptr(), values.data_ptr(), flag, batch, heads, kv_heads, seq, start, max_len,
                                           hd, out.data_ptr(), out_flag, room.data_ptr(), size, stream)
    return lib.ajq_attn_prefill(q.data_ptr(), keys.data_ptr(), values.data_ptr(), flag, batch, heads, kv_heads, seq, start, max_len, hd,
                                out.data_ptr(), out_flag, stream)


_TYPES = {torch.float32: _lib.AJQS_F32, torch.bfloat16: _lib.AJQS_BF16}


def _on(device: torch.device):
    return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _pointer(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _check_caches(what: str, keys: torch.Tensor, values: torch.Tensor, device: torch.device) -> None:
    if keys.dim() != 4 or keys.shape != values.shape or keys.stride() != values.stride() or keys.shape[3] not in (128, 64, 32):
        raise ValueError(f"{what}: caches [.., Hkv, rows, hd] of one shape and layout with hd 128, 64 or 32 expected")
    if keys.stride(3) != 1 or keys.stride(2) != keys.shape[3]:
        raise ValueError(f"{what}: the rows of a cache head must lie one behind the other")
    if keys.dtype not in _TYPES or values.dtype != keys.dtype:
        raise ValueError(f"{what}: the caches must be float32 or bfloat16")
    if keys.device != device or values.device != device:
        raise ValueError(f"{what}: all tensors must be on one device")


def _whole_numbers(what: str, name: str, t: torch.Tensor | None, count: int, device: torch.device) -> None:
    if t is not None and (t.dtype != torch.int64 or t.numel() != count or not t.is_contiguous() or t.device != device):
        raise ValueError(f"{what}: {name} must be {count} contiguous int64 on the device of the others")


def _floats(what: str, name: str, t: torch.Tensor | None, shape: tuple, device: torch.device) -> None:
    if t is not None and (t.dtype != torch.float32 or tuple(t.shape) != shape or not t.is_contiguous() or t.device != device):
        raise ValueError(f"{what}: {name} must be contiguous float32 {list(shape)} on the device of the others")


def norm_rope(qkv: torch.Tensor, cosine: torch.Tensor, sine: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, rows: torch.Tensor, *,
              heads: int, tokens: int = 1, q_gain: torch.Tensor | None = None, k_gain: torch.Tensor | None = None, epsilon: float = 1e-5,
              positions: torch.Tensor | None = None, counts: torch.Tensor | None = None, offset: torch.Tensor | None = None,
              out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Queries and keys of a projection's output, each head RMS-normed (``q_gain``, ``k_gain`` fp32 ``[hd]``; None: as it is) and rotated,
    keys and values written into the caches, in one launch: for sequences at positions of their own.

    ``qkv`` fp32 or bf16 ``[B * tokens, (heads + 2 Hkv) * hd]`` (query heads, key heads, value heads; rows may be further apart); ``cosine`` /
    ``sine`` fp32 ``[positions, hd / 2]``; ``keys`` / ``values`` ``[B, Hkv, max_len, hd]`` fp32 or bf16.  Token t of sequence b goes to row
    ``rows[b] + offset + t`` of its caches and turns by position ``positions[b] + offset + t`` (``positions`` None: the row); ``rows``,
    ``positions`` and ``counts`` int64 ``[B]``, ``offset`` one int64, all on the device.  Of the tokens of sequence b the first
    ``counts[b]`` are there (None: all); the others write no row, and zeros for queries.  A row outside the caches is not written, a
    position is held inside the tables; heads of the caches may not overlap.  Returns the queries ``[B, heads, tokens, hd]`` in ``out_dtype``,
    without a gradient, as all of these functions
    (RMSNorm.forward, src/ajllm/modeling/layers.py:70-74, on every head, then attention.py:36-60)."""
    what = "norm_rope"
    if not qkv.is_cuda:
        raise ValueError("norm_rope needs tensors on a ROCm device (there is no CPU path)")
    # tensors as the kernel takes them: one call of native code, which leaves everything else to the lines below it
    q = (_lib._serve_native.get(what) or _lib.serve_native(what))(
        qkv, cosine, sine, keys, values, rows, heads, tokens, q_gain, k_gain, epsilon, positions, counts, offset, out_dtype)
    if q is not None:
        return q
    device = qkv.device
    _check_caches(what, keys, values, device)
    batch, kv_heads, max_len, hd = keys.shape
    if qkv.dim() != 2 or tokens < 1 or qkv.shape[0] != batch * tokens or qkv.shape[1] != (heads + 2 * kv_heads) * hd or qkv.stride(1) != 1:
        raise ValueError("norm_rope: qkv [B * tokens, (heads + 2 Hkv) * hd] expected")
    if qkv.dtype not in _TYPES or out_dtype not in _TYPES:
        raise ValueError("norm_rope: qkv and out_dtype must be float32 or bfloat16")
    _floats(what, "cosine", cosine, (cosine.shape[0], hd // 2), device)
    _floats(what, "sine", sine, tuple(cosine.shape), device)
    _floats(what, "q_gain", q_gain, (hd,), device)
    _floats(what, "k_gain", k_gain, (hd,), device)
    _whole_numbers(what, "rows", rows, batch, device)
    _whole_numbers(what, "positions", positions, batch, device)
    _whole_numbers(what, "counts", counts, batch, device)
    _whole_numbers(what, "offset", offset, 1, device)
    q = torch.empty((batch, heads, tokens, hd), dtype=out_dtype, device=device)
    args = _lib.NormRopeArgs(
        qkv.data_ptr(), cosine.data_ptr(), sine.data_ptr(), _pointer(q_gain), _pointer(k_gain), rows.data_ptr(), _pointer(positions),
        _pointer(counts), _pointer(offset), keys.data_ptr(), values.data_ptr(), q.data_ptr(), qkv.stride(0), keys.stride(0), keys.stride(1),
        batch, tokens, heads, kv_heads, hd, max_len, cosine.shape[0], _TYPES[qkv.dtype], _TYPES[out_dtype], _TYPES[keys.dtype], epsilon)
    with _on(device):
        status = _lib.load_serve().ajqs_norm_rope(ctypes.byref(args), torch.cuda.current_stream().cuda_stream)
    _lib.check_serve(status, what)
    return q


def shared_prefix_launches(batch: int, heads: int, tokens: int, prefix_keys: torch.Tensor, keys: torch.Tensor, q_dtype: torch.dtype = torch.float32) -> int:
    """Kernel launches of ``shared_prefix_attention`` on such caches: two where what its workgroups make of a query is put together by a second."""
    at = keys.data_ptr()
    args = _lib.SharedAttentionArgs(at, at, at, at, at, at, at, None, None, at, prefix_keys.stride(0), prefix_keys.stride(1), keys.stride(0), keys.stride(1),
                                    prefix_keys.shape[0], batch, tokens, heads, keys.shape[1], keys.shape[3], prefix_keys.shape[2], keys.shape[2],
                                    _TYPES[q_dtype], _TYPES[keys.dtype])
    return 2 if _lib.load_serve().ajqs_shared_attention_workspace(ctypes.byref(args)) else 1


def shared_prefix_attention(q: torch.Tensor, prefix_keys: torch.Tensor, prefix_values: torch.Tensor, prefix_lengths: torch.Tensor,
                            keys: torch.Tensor, values: torch.Tensor, rows: torch.Tensor, *, counts: torch.Tensor | None = None,
                            offset: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of ``B`` sequences in groups that share a prefix, whose rows lie and are read once for the whole group.

    ``q`` fp32 or bf16 ``[B, H, T, hd]`` (rotated); ``prefix_keys`` / ``prefix_values`` ``[G, Hkv, capacity, hd]``, the first
    ``prefix_lengths[g]`` rows filled, for sequences ``g * B / G ..``; ``keys`` / ``values`` ``[B, Hkv, max_len, hd]`` with each sequence's own
    rows, the T new tokens' (``norm_rope`` writes them) included.  Token t of sequence b sees its group's prefix and its own rows up to ``rows[b]
    + offset + t``.  Caches fp32 or bf16; ``prefix_lengths`` int64 ``[G]``, ``rows`` and ``counts`` int64 ``[B]``, ``offset`` one int64, on
    the device, as in ``norm_rope``.  Returns bf16 ``[B, T, H * hd]`` (what the output projection takes); zeros for a token that is not there
    or sees nothing.  Rows that nobody sees may hold anything; values that a token of the sequence sees must be finite.  The launches are chosen by the
    capacities (``shared_prefix_launches``), not by the lengths: slices of the caches down to what can be filled are the faster.  Precision, and the memory that a call
    takes for itself: include/ajq_serve.h."""
    what = "shared_prefix_attention"
    if not q.is_cuda:
        raise ValueError("shared_prefix_attention needs tensors on a ROCm device (there is no CPU path)")
    out = (_lib._serve_native.get(what) or _lib.serve_native(what))(q, prefix_keys, prefix_values, prefix_lengths, keys, values, rows, counts, offset)
    if out is not None:
        return out
    device = q.device
    _check_caches(what, prefix_keys, prefix_values, device)
    _check_caches(what, keys, values, device)
    if q.dim() != 4 or q.dtype not in _TYPES:
        raise ValueError("shared_prefix_attention: q [B, H, T, hd] in float32 or bfloat16 expected")
    batch, heads, seq, hd = q.shape
    groups, kv_heads, capacity, _ = prefix_keys.shape
    if keys.shape[0] != batch or keys.shape[1] != kv_heads or keys.shape[3] != hd or prefix_keys.shape[3] != hd or keys.dtype != prefix_keys.dtype:
        raise ValueError("shared_prefix_attention: caches [B, Hkv, max_len, hd] and prefix caches [G, Hkv, capacity, hd] of one type expected")
    _whole_numbers(what, "prefix_lengths", prefix_lengths, groups, device)
    _whole_numbers(what, "rows", rows, batch, device)
    _whole_numbers(what, "counts", counts, batch, device)
    _whole_numbers(what, "offset", offset, 1, device)
    q = q.contiguous()
    out = torch.empty((batch, seq, heads * hd), dtype=torch.bfloat16, device=device)
    args = _lib.SharedAttentionArgs(
        q.data_ptr(), prefix_keys.data_ptr(), prefix_values.data_ptr(), keys.data_ptr(), values.data_ptr(), prefix_lengths.data_ptr(),
        rows.data_ptr(), _pointer(counts), _pointer(offset), out.data_ptr(), prefix_keys.stride(0), prefix_keys.stride(1), keys.stride(0),
        keys.stride(1), groups, batch, seq, heads, kv_heads, hd, capacity, keys.shape[2], _TYPES[q.dtype], _TYPES[keys.dtype])
    lib = _lib.load_serve()
    with _on(device):
        size = lib.ajqs_shared_attention_workspace(ctypes.byref(args))
        room = torch.empty(size, dtype=torch.uint8, device=device) if size else None
        status = lib.ajqs_shared_attention(ctypes.byref(args), _pointer(room), size, torch.cuda.current_stream().cuda_stream)
    _lib.check_serve(status, what)
    return out
