"""The operators of checking drafted tokens from their definitions, in 64 bits."""

import math

import torch


def sees(masks, batch, nodes):
    """[B, T, T] truth values of mask words, on the CPU."""
    words = (masks if masks.dim() == 3 else masks.expand(batch, *masks.shape)).cpu().long()
    u = torch.arange(nodes)
    return (words[:, :, u // 32] >> (u % 32)) & 1 != 0


def ancestors(parents):
    """(sees, depths) of one tree: a list of parents, one walk upwards a node."""
    many = len(parents)
    table, depths = torch.zeros(many, many, dtype=torch.bool), torch.zeros(many, dtype=torch.long)
    for t in range(many):
        at = t
        while True:
            table[t, at] = True
            if at == 0 or not 0 <= parents[at] < at:
                break
            at = parents[at]
            depths[t] += 1
    return table, depths


def tree_attention(q, keys, values, rows, masks, counts, offset):
    """(out, size): float64 on q's device; ``size`` is the weighted mean of the values' sizes, what roundings of the weights act on."""
    batch, heads, nodes, hd = q.shape
    kv, max_len = keys.shape[1:3]
    share = heads // kv
    out = torch.zeros(batch, nodes, heads, hd, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    table = sees(masks, batch, nodes)
    for b in range(batch):
        before = int(rows[b]) + offset
        many = nodes if counts is None else min(max(int(counts[b]), 0), nodes)
        last = min(max(before + many, 0), max_len)
        if many == 0 or last == 0:
            continue
        node = torch.arange(last) - before
        seen = torch.where(node < 0, True, table[b, :many][:, node.clamp(0, nodes - 1)])          # [many, last]
        nothing = ~seen.any(1)
        seen, nothing = seen.to(q.device), nothing.to(q.device)
        for k in range(kv):
            ks, vs = keys[b, k, :last].double(), values[b, k, :last].double()
            never = ~seen.any(0)
            ks, vs = ks.masked_fill(never[:, None], 0.0), vs.masked_fill(never[:, None], 0.0)     # (rows that nobody sees may hold anything)
            x = q[b, k * share:(k + 1) * share, :many].double()
            score = (x.reshape(-1, hd) @ ks.t().contiguous()).view(share, many, -1) / math.sqrt(hd)
            w = torch.softmax(score.masked_fill(~seen, -math.inf), dim=-1).masked_fill(nothing[:, None], 0.0).view(share * many, -1)
            out[b, :many, k * share:(k + 1) * share] = (w @ vs).view(share, many, hd).transpose(0, 1)
            size[b, :many, k * share:(k + 1) * share] = (w @ vs.abs()).view(share, many, hd).transpose(0, 1)
    return out.view(batch, nodes, heads * hd), size.view(batch, nodes, heads * hd)


def keep_rows(cache, rows, index, counts, offset):
    """A copy of ``cache`` [layers, B, Hkv, max_len, hd] with the rows moved."""
    out = cache.clone()
    max_len = cache.shape[3]
    for b in range(cache.shape[1]):
        first, numbers = int(rows[b]) + offset, (index if index.dim() == 1 else index[b]).tolist()
        if not 0 <= first < max_len:
            continue
        last = -1
        for i, n in enumerate(numbers[:len(numbers) if counts is None else max(int(counts[b]), 0)]):
            if n <= last or first + n >= max_len:
                break
            out[:, b, :, first + i] = cache[:, b, :, first + n]
            last = n
    return out


def token_log_probs(logits, targets, top):
    """(log_probs, ranks, entropy, top_log_probs, top_ids, spread): float64 and int64 on the CPU, ``spread`` what roundings act on (of finite rows, and of rows
    that allow nothing)."""
    x = logits.double().cpu()
    rows, vocab = x.shape
    most = x.max(1, keepdim=True).values
    nothing = most == -math.inf
    far = x - most.masked_fill(nothing, 0.0)
    p = far.exp()
    total = p.sum(1, keepdim=True)
    log_p = torch.where(nothing, -math.inf, far - total.log())
    q = torch.where(nothing, 0.0, p / total)
    held = torch.where(q > 0, far, 0.0)
    entropy = torch.where(nothing, 0.0, -(q * log_p.masked_fill(q == 0, 0.0)).sum(1, keepdim=True))[:, 0]
    spread = dict(log_total=torch.where(nothing, 0.0, total.log())[:, 0], first=-(q * held).sum(1), second=(q * held * held).sum(1))
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    place = torch.empty_like(order).scatter_(1, order, torch.arange(vocab).expand(rows, vocab))
    mine = ranks = None
    if targets is not None:
        there = (targets >= 0) & (targets < vocab)
        at = targets.clamp(0, vocab - 1)[:, None]
        mine = torch.where(there, log_p.gather(1, at)[:, 0], 0.0)
        ranks = torch.where(there, place.gather(1, at)[:, 0], -1)
    ids = order[:, :top]
    return mine, ranks, entropy, log_p.gather(1, ids), ids, spread


def follow_drafts(tokens, parents, choices, counts):
    batch, nodes = tokens.shape
    path, chosen = torch.full((batch, nodes), -1), torch.full((batch, nodes), -1)
    accepted = torch.zeros(batch, dtype=torch.long)
    for b in range(batch):
        up = (parents if parents.dim() == 1 else parents[b]).tolist()
        many = nodes if counts is None else min(max(int(counts[b]), 0), nodes)
        at, steps = 0, []
        while at < many:
            steps.append(at)
            at = next((t for t in range(at + 1, many) if up[t] == at and tokens[b, t] == choices[b, at]), many)
        accepted[b] = len(steps)
        path[b, :len(steps)] = torch.tensor(steps, dtype=torch.long)
        chosen[b, :len(steps)] = choices[b, steps]
    return path, accepted, chosen
