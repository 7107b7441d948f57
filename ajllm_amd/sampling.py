"""What a program does to logits ahead of the choice of a token: penalties for repeated tokens, biases, masks of allowed tokens
(``ajqs_adjust_logits``); what it reads off them: log probabilities, entropies, the most probable alternatives (``ajqt_log_probs``); and what the
choices behind drafted tokens come to (``ajqt_follow_drafts``).  The choice itself is ``decoding``'s (the reference's ``sample_next_token``,
src/ajllm/generation/sampling.py:8-22, has none of these)."""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib
from .attention import _TYPES, _on, _pointer

MOST_TOP = 64   # alternatives of token_log_probs


def _list(name: str, ids: torch.Tensor | None, lengths: torch.Tensor | None, batch: int, device: torch.device) -> tuple:
    """Pointers, row stride, width and stride of the counts of a row's token list."""
    if ids is None:
        if lengths is not None:
            raise ValueError(f"adjust_logits: lengths without {name}")
        return None, None, 0, 0, 0
    if ids.dim() != 2 or ids.shape[0] != batch or ids.dtype != torch.int64 or ids.device != device or (ids.shape[1] and ids.stride(1) != 1):
        raise ValueError(f"adjust_logits: {name} must be int64 [B, n] on the device of the logits")
    if lengths is not None and (lengths.dtype != torch.int64 or lengths.numel() not in (1, batch) or not lengths.is_contiguous()
                                or lengths.device != device):
        raise ValueError(f"adjust_logits: the lengths of {name} must be one int64, or one a row, on the device of the logits")
    if ids.shape[1] == 0:
        return None, None, 0, 0, 0
    return ids.data_ptr(), _pointer(lengths), _apart(ids), ids.shape[1], int(lengths is not None and lengths.numel() == batch and batch > 1)


def _apart(t: torch.Tensor) -> int:
    """Elements from a row to the next (of a single row: any number that holds it)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _of_rows(name: str, value: torch.Tensor | float | None, batch: int, device: torch.device) -> torch.Tensor | None:
    if value is None:
        return None
    if not isinstance(value, torch.Tensor):
        return torch.full((batch,), float(value), dtype=torch.float32, device=device)   # (the kernel reads fp32, whatever the default dtype)
    if value.dtype != torch.float32 or tuple(value.shape) != (batch,) or not value.is_contiguous() or value.device != device:
        raise ValueError(f"adjust_logits: {name} must be a number or contiguous float32 [B] on the device of the logits")
    return value


def adjust_logits(logits: torch.Tensor, *, tokens: torch.Tensor | None = None, lengths: torch.Tensor | None = None,
                  prompt: torch.Tensor | None = None, prompt_lengths: torch.Tensor | None = None,
                  repetition: torch.Tensor | float | None = None, frequency: torch.Tensor | float | None = None,
                  presence: torch.Tensor | float | None = None, bias_ids: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                  allowed: torch.Tensor | None = None, allowed_rows: torch.Tensor | None = None,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """fp32 ``[B, V]`` from ``logits`` ``[B, V]`` (fp32 or bf16), row by row, in this order:

    * a token that is in the row's ``prompt`` or ``tokens``: positive logits are divided by ``repetition``, others multiplied;
    * one that is n > 0 times among its ``tokens``: less ``frequency * n + presence``;
    * plus the row's ``bias`` (fp32 ``[B, n]``) at ``bias_ids`` (int64 ``[B, n]``, n up to 1024; an id given twice gets the sum);
    * ``-inf`` where the row's mask has a 0: bit ``v % 32`` of word ``v // 32`` of ``allowed`` (int32 ``[masks, >= V / 32]``).  Row b has mask
      ``allowed_rows[b]`` (int64 ``[B]``; a number outside ``[0, masks)``: none), or mask b without it.  A row whose mask leaves nothing is ``-inf``.

    ``tokens`` and ``prompt`` are int64 ``[B, n]``, of which the first ``lengths`` (``prompt_lengths``) count: int64 on the device, one a row or
    one for all (a decoder's step counter), None: all of them; lists and masks that all rows share may be expanded (a stride of 0).  Ids outside ``[0, V)`` are passed over.  ``repetition``, ``frequency`` and
    ``presence`` are numbers or fp32 ``[B]``.  ``out`` may be ``logits`` itself where they are fp32 (and overlaps them in no other way); without it the rows of the result begin
    on 16-byte boundaries, as ``ajq_sample_pick`` wants them (fp32 logits that nothing is to happen to are returned as they are)."""
    if not logits.is_cuda:
        raise ValueError("adjust_logits needs tensors on a ROCm device (there is no CPU path)")
    if (tokens is lengths is prompt is prompt_lengths is repetition is frequency is presence is bias_ids is bias is allowed is allowed_rows is out is None
            and logits.dtype == torch.float32 and logits.dim() == 2 and logits.stride(1) == 1 and 0 not in logits.shape):
        return logits   # (nothing to do)
    made = (_lib._serve_native.get("adjust_logits") or _lib.serve_native("adjust_logits"))(
        logits, tokens, lengths, prompt, prompt_lengths, repetition, frequency, presence, bias_ids, bias, allowed, allowed_rows, out)
    if made is not None:
        return made if out is None else out
    if logits.dim() != 2 or logits.dtype not in _TYPES or logits.stride(1) != 1 or 0 in logits.shape:
        raise ValueError("adjust_logits: logits [B, V] in float32 or bfloat16 expected")
    device = logits.device
    batch, vocab = logits.shape
    at, counts, ld, most, stride = _list("tokens", tokens, lengths, batch, device)
    before, prompt_counts, prompt_ld, most_before, prompt_stride = _list("prompt", prompt, prompt_lengths, batch, device)
    repetition = _of_rows("repetition", repetition, batch, device)
    frequency = _of_rows("frequency", frequency, batch, device)
    presence = _of_rows("presence", presence, batch, device)
    if (bias_ids is None) != (bias is None):
        raise ValueError("adjust_logits: bias_ids and bias go together")
    if bias is not None and (bias.dim() != 2 or bias.shape[0] != batch or bias_ids.shape != bias.shape or bias.dtype != torch.float32
                             or bias_ids.dtype != torch.int64 or not (bias.is_contiguous() and bias_ids.is_contiguous())
                             or bias.device != device or bias_ids.device != device):
        raise ValueError("adjust_logits: bias_ids int64 and bias float32, both contiguous [B, n] on the device of the logits, expected")
    if allowed is not None and (allowed.dim() != 2 or allowed.dtype != torch.int32 or allowed.stride(1) != 1 or allowed.device != device):
        raise ValueError("adjust_logits: allowed must be int32 [masks, words] on the device of the logits")
    if allowed_rows is not None and (allowed is None or allowed_rows.dtype != torch.int64 or tuple(allowed_rows.shape) != (batch,)
                                     or not allowed_rows.is_contiguous() or allowed_rows.device != device):
        raise ValueError("adjust_logits: allowed_rows must be contiguous int64 [B] on the device of the logits, beside masks")
    if max(batch, vocab, most, most_before, 0 if bias is None else bias.shape[1], 0 if allowed is None else allowed.shape[0]) >= 2 ** 31:
        raise ValueError("adjust_logits: fewer than 2^31 rows, tokens, listed tokens, biases and masks expected")
    if out is None:
        out = torch.empty((batch, vocab + -vocab % 4), dtype=torch.float32, device=device)[:, :vocab]
    elif out.shape != logits.shape or out.dtype != torch.float32 or out.stride(1) != 1 or out.device != device:
        raise ValueError("adjust_logits: out must be float32 [B, V] on the device of the logits")
    args = _lib.AdjustLogitsArgs(
        logits.data_ptr(), out.data_ptr(), at, counts, before, prompt_counts, _pointer(repetition), _pointer(frequency), _pointer(presence),
        _pointer(bias_ids), _pointer(bias), _pointer(allowed), _pointer(allowed_rows), _apart(logits), _apart(out), ld, prompt_ld,
        0 if bias is None else bias.shape[1], 0 if allowed is None else _apart(allowed), batch, vocab, most, most_before,
        0 if bias is None else bias.shape[1], 0 if allowed is None else allowed.shape[0], stride, prompt_stride, _TYPES[logits.dtype])
    if allowed is not None and allowed.shape[1] * 32 < vocab:
        raise ValueError("adjust_logits: a mask has a bit for every token")
    with _on(device):
        status = _lib.load_serve().ajqs_adjust_logits(ctypes.byref(args), torch.cuda.current_stream().cuda_stream)
    _lib.check_serve(status, "adjust_logits")
    return out


class TokenLogProbs(NamedTuple):
    """``token_log_probs``' results; None for what was not asked for."""

    log_probs: torch.Tensor | None       # fp32 [R]: of the targets
    ranks: torch.Tensor | None           # int64 [R]: how many tokens come ahead of the target (0: it is the most probable one)
    entropy: torch.Tensor                # fp32 [R]
    top_log_probs: torch.Tensor | None   # fp32 [R, top]: of the most probable tokens, the first one first
    top_ids: torch.Tensor | None         # int64 [R, top]


def token_log_probs(logits: torch.Tensor, targets: torch.Tensor | None = None, *, top: int = 0) -> TokenLogProbs:
    """Log probabilities of given tokens under ``softmax(logits)``, ranks, entropies (in nats) and the ``top`` most probable tokens, in one pass over the logits.

    ``logits`` ``[R, V]`` fp32 or bf16 (rows may be further apart), ``targets`` int64 ``[R]`` (None: neither log probabilities nor ranks; a target
    outside ``[0, V)`` asks for nothing: log probability 0, rank -1), ``top`` up to 64 and V.  Tokens of equal logits come in the order of their ids,
    for ranks as for the alternatives: ``top_ids[r, ranks[r]]`` is the target where it is among them, and ``top=1`` is the greedy choice.  A token that a mask has set to -inf has
    the log probability -inf and adds nothing to the entropy; a row of which nothing is left has -inf for every token, and an entropy of 0.  A row with NaN or +inf gives NaN,
    and ids and ranks that are some tokens'.  Without a gradient."""
    what = "token_log_probs"
    if not logits.is_cuda:
        raise ValueError("token_log_probs needs tensors on a ROCm device (there is no CPU path)")
    made = (_lib._draft_native.get(what) or _lib.draft_native(what))(logits, targets, top)
    if made is not None:
        return TokenLogProbs._make(made)
    device = logits.device
    if logits.dim() != 2 or logits.dtype not in _TYPES or logits.shape[1] == 0 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("token_log_probs: logits [R, V] in float32 or bfloat16 expected")
    rows, vocab = logits.shape
    if max(rows, vocab) >= 2 ** 31:
        raise ValueError("token_log_probs: fewer than 2^31 rows and tokens expected")
    if targets is not None and (targets.dtype != torch.int64 or tuple(targets.shape) != (rows,) or not targets.is_contiguous() or targets.device != device):
        raise ValueError("token_log_probs: targets must be contiguous int64 [R] on the device of the logits")
    if not 0 <= top <= min(MOST_TOP, vocab):
        raise ValueError(f"token_log_probs: top must be in [0, {min(MOST_TOP, vocab)}]")
    floats = lambda *shape: torch.empty(shape, dtype=torch.float32, device=device)  # noqa: E731
    whole = lambda *shape: torch.empty(shape, dtype=torch.int64, device=device)     # noqa: E731
    out = TokenLogProbs(floats(rows) if targets is not None else None, whole(rows) if targets is not None else None, floats(rows),
                        floats(rows, top) if top else None, whole(rows, top) if top else None)
    if rows == 0:
        return out
    args = _lib.LogProbsArgs(logits.data_ptr(), _pointer(targets), _pointer(out.log_probs), out.entropy.data_ptr(), _pointer(out.top_log_probs),
                             _pointer(out.ranks), _pointer(out.top_ids), _apart(logits), rows, vocab, top, _TYPES[logits.dtype])
    lib = _lib.load_draft()
    with _on(device):
        size = lib.ajqt_log_probs_workspace(ctypes.byref(args))
        room = torch.empty(size, dtype=torch.uint8, device=device) if size else None
        status = lib.ajqt_log_probs(ctypes.byref(args), _pointer(room), size, torch.cuda.current_stream().cuda_stream)
    _lib.check_draft(status, what)
    return out


class FollowedDrafts(NamedTuple):
    """``follow_drafts``' results."""

    path: torch.Tensor       # int64 [B, T]: the nodes that were right, from the root on, ascending; then -1
    accepted: torch.Tensor   # int64 [B]: how many there are (the root is one)
    chosen: torch.Tensor     # int64 [B, T]: the choices behind them, which is what the step has produced; then -1


def follow_drafts(tokens: torch.Tensor, parents: torch.Tensor, choices: torch.Tensor, *, counts: torch.Tensor | None = None) -> FollowedDrafts:
    """The drafts that are what the model chose: from the root of each tree on, to the first child that guesses the choice behind the node it hangs on.

    ``tokens`` int64 ``[B, T]``: node 0 is the root (its token is not looked at), node t guesses ``tokens[b, t]`` behind node ``parents[t]``; ``parents`` int64 ``[T]``
    or ``[B, T]`` as in ``tree_masks`` (a node whose parent is not in ``[0, t)`` is never reached); ``choices`` int64 ``[B, T]``, the model's choice behind each node,
    greedy or drawn (a view such as ``top_ids[:, :1].view(B, T)`` will do): what is accepted has the distribution that decoding a token at a time has.  The first ``counts[b]``
    nodes are there (None: all).  T up to 4096."""
    what = "follow_drafts"
    if not tokens.is_cuda:
        raise ValueError("follow_drafts needs tensors on a ROCm device (there is no CPU path)")
    made = (_lib._draft_native.get(what) or _lib.draft_native(what))(tokens, parents, choices, counts)
    if made is not None:
        return FollowedDrafts._make(made)
    device = tokens.device
    if tokens.dim() != 2 or tokens.dtype != torch.int64 or (tokens.shape[1] > 1 and tokens.stride(1) != 1):
        raise ValueError("follow_drafts: tokens int64 [B, T] expected")
    batch, nodes = tokens.shape
    if batch >= 2 ** 31:
        raise ValueError("follow_drafts: fewer than 2^31 trees expected")
    if parents.dtype != torch.int64 or tuple(parents.shape) not in ((nodes,), (batch, nodes)) or parents.device != device or (nodes > 1 and parents.stride(-1) != 1):
        raise ValueError("follow_drafts: parents int64 [T] or [B, T] on the device of the tokens expected")
    if choices.dtype != torch.int64 or choices.shape != tokens.shape or choices.device != device:
        raise ValueError("follow_drafts: choices int64 [B, T] on the device of the tokens expected")
    if counts is not None and (counts.dtype != torch.int64 or tuple(counts.shape) != (batch,) or not counts.is_contiguous() or counts.device != device):
        raise ValueError("follow_drafts: counts must be contiguous int64 [B] on the device of the tokens")
    whole = lambda *shape: torch.empty(shape, dtype=torch.int64, device=device)  # noqa: E731
    out = FollowedDrafts(whole(batch, nodes), whole(batch), whole(batch, nodes))
    if 0 in tokens.shape:
        return out._replace(accepted=out.accepted.zero_())
    args = _lib.FollowDraftsArgs(tokens.data_ptr(), parents.data_ptr(), choices.data_ptr(), _pointer(counts), *(t.data_ptr() for t in out), tokens.stride(0),
                                 parents.stride(0) if parents.dim() == 2 else 0, choices.stride(0), choices.stride(1), batch, nodes)
    with _on(device):
        status = _lib.load_draft().ajqt_follow_drafts(ctypes.byref(args), torch.cuda.current_stream().cuda_stream)
    _lib.check_draft(status, what)
    return out
