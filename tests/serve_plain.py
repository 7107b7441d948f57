"""The operators of decoding many continuations of one prompt from their definitions, in 64 bits, one row after the other."""

import math

import torch


def norm_rope(qkv, cosine, sine, keys, values, rows, heads, tokens, q_gain, k_gain, eps, positions, counts, offset):
    """(queries, keys, values, magnitude): float64 on the CPU; ``magnitude`` is the length of each query pair, in both places."""
    qkv, keys, values = qkv.double().cpu(), keys.double().cpu().clone(), values.double().cpu().clone()
    batch, kv, max_len, hd = keys.shape
    x = qkv.view(batch, tokens, heads + 2 * kv, hd)
    q = torch.zeros(batch, heads, tokens, hd, dtype=torch.float64)
    cosine, sine = cosine.double().cpu(), sine.double().cpu()
    magnitude_k = torch.zeros_like(keys)
    for b in range(batch):
        for t in range(tokens if counts is None else min(tokens, int(counts[b]))):
            row = int(rows[b]) + offset + t
            at = min(max((int(rows[b]) if positions is None else int(positions[b])) + offset + t, 0), cosine.shape[0] - 1)
            for head in range(heads + 2 * kv):
                y = x[b, t, head]
                gain = q_gain if head < heads else k_gain if head < heads + kv else None
                if gain is not None:
                    y = y / math.sqrt(float(y.square().mean()) + eps) * gain.double().cpu()
                if head < heads + kv:
                    e, o = y[::2], y[1::2]
                    y = torch.stack((e * cosine[at] - o * sine[at], e * sine[at] + o * cosine[at]), dim=-1).flatten()
                if head < heads:
                    q[b, head, t] = y
                elif 0 <= row < max_len:
                    (keys if head < heads + kv else values)[b, (head - heads) % kv, row] = y
                    if head < heads + kv:
                        magnitude_k[b, head - heads, row] = y.view(-1, 2).norm(dim=-1).repeat_interleave(2)
    magnitude_q = q.view(*q.shape[:-1], hd // 2, 2).norm(dim=-1).repeat_interleave(2, dim=-1)
    return q, keys, values, magnitude_q, magnitude_k


def shared_prefix_attention(q, prefix_keys, prefix_values, prefix_lengths, keys, values, rows, counts, offset):
    """(out, weight): float64; ``weight`` is the weighted mean of the values' sizes, what roundings of the weights act on."""
    q = q.double().cpu()
    batch, heads, tokens, hd = q.shape
    groups, kv, capacity, _ = prefix_keys.shape
    max_len, share, each = keys.shape[2], heads // kv, batch // groups
    out = torch.zeros(batch, tokens, heads, hd, dtype=torch.float64)
    size = torch.zeros_like(out)
    for b in range(batch):
        g = b // each
        before = min(max(int(prefix_lengths[g]), 0), capacity)
        for t in range(tokens if counts is None else min(tokens, int(counts[b]))):
            own = min(max(int(rows[b]) + offset + t + 1, 0), max_len)
            if before + own == 0:
                continue
            for k in range(kv):
                ks = torch.cat((prefix_keys[g, k, :before].cpu(), keys[b, k, :own].cpu())).double()
                vs = torch.cat((prefix_values[g, k, :before].cpu(), values[b, k, :own].cpu())).double()
                w = torch.softmax(q[b, k * share:(k + 1) * share, t] @ ks.t() / math.sqrt(hd), dim=-1)
                out[b, t, k * share:(k + 1) * share] = w @ vs
                size[b, t, k * share:(k + 1) * share] = w @ vs.abs()
    return out.view(batch, tokens, heads * hd), size.view(batch, tokens, heads * hd)


def adjust_logits(logits, tokens, lengths, prompt, prompt_lengths, repetition, frequency, presence, bias_ids, bias, allowed, allowed_rows):
    """(out, size): float64; ``size`` is the sum of the sizes of what is added up, what roundings act on."""
    x = logits.double().cpu().clone()
    batch, vocab = x.shape
    size = torch.zeros_like(x)

    def number(value, b, default):
        return default if value is None else float(value) if not isinstance(value, torch.Tensor) else float(value[b])

    def count(lengths, b, width):
        return width if lengths is None else min(max(int(lengths.view(-1)[b if lengths.numel() > 1 else 0]), 0), width)

    for b in range(batch):
        r, f, p = number(repetition, b, 1.0), number(frequency, b, 0.0), number(presence, b, 0.0)
        mine = [] if tokens is None else tokens[b, :count(lengths, b, tokens.shape[1])].tolist()
        given = [] if prompt is None else prompt[b, :count(prompt_lengths, b, prompt.shape[1])].tolist()
        for v in {i for i in mine + given if 0 <= i < vocab}:
            x[b, v] = x[b, v] / r if x[b, v] > 0 else x[b, v] * r
        size[b] = x[b].abs()
        for v in {i for i in mine if 0 <= i < vocab}:
            x[b, v] -= f * mine.count(v) + p
            size[b, v] += abs(f) * mine.count(v) + abs(p)
        if bias_ids is not None:
            for v, add in zip(bias_ids[b].tolist(), bias[b].tolist()):
                if 0 <= v < vocab:
                    x[b, v] += add
                    size[b, v] += abs(add)
        which = b if allowed_rows is None else int(allowed_rows[b])
        if allowed is not None and 0 <= which < allowed.shape[0]:
            words = allowed[which].tolist()
            for v in range(vocab):
                if not (words[v // 32] >> (v % 32)) & 1:
                    x[b, v] = -math.inf
    return x, size


def shared_prefix_attention_by_heads(q, prefix_keys, prefix_values, prefix_lengths, keys, values, rows, counts):
    """The same of larger calls: (out, weight), float64 on q's device, all queries of a sequence and a key head at once."""
    batch, heads, tokens, hd = q.shape
    groups, kv, capacity, _ = prefix_keys.shape
    max_len, share, each = keys.shape[2], heads // kv, batch // groups
    out = torch.zeros(batch, tokens, heads, hd, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    token = torch.arange(tokens, device=q.device)
    for b in range(batch):
        before = min(max(int(prefix_lengths[b // each]), 0), capacity)
        many = tokens if counts is None else min(max(int(counts[b]), 0), tokens)
        sees = (int(rows[b]) + token[:many] + 1).clamp(0, max_len)                       # own rows of each token
        if many == 0 or before + int(sees.max()) == 0:
            continue
        own = int(sees.max())
        hidden = torch.arange(before + own, device=q.device) >= before + sees[:, None]    # [many, rows]
        nothing = (before + sees == 0)[:, None, None]
        for k in range(kv):
            ks = torch.cat((prefix_keys[b // each, k, :before], keys[b, k, :own])).double()
            vs = torch.cat((prefix_values[b // each, k, :before], values[b, k, :own])).double()
            x = q[b, k * share:(k + 1) * share, :many].double().transpose(0, 1)           # [many, share, hd]
            score = (x.reshape(-1, hd) @ ks.t().contiguous()).view(many, share, -1) / math.sqrt(hd)
            w = torch.softmax(score.masked_fill(hidden[:, None, :], -math.inf), dim=-1).masked_fill(nothing, 0.0).view(many * share, -1)
            out[b, :many, k * share:(k + 1) * share] = (w @ vs).view(many, share, hd)
            size[b, :many, k * share:(k + 1) * share] = (w @ vs.abs()).view(many, share, hd)
    return out.view(batch, tokens, heads * hd), size.view(batch, tokens, heads * hd)
