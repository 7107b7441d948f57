"""What the speed of decoding many continuations of one prompt is measured on: three operators of one decode step (or of the pass over the
questions ahead of it), each reached as a user's program reaches it.

* ``rotate``   queries and keys of the projection output normed per head and rotated, keys and values into each sequence's cache, every
               sequence at a position of its own (``ajllm_amd.attention.norm_rope``).
* ``share``    attention of sequences whose common first part lies once in memory (``ajllm_amd.attention.shared_prefix_attention``).
* ``logits``   penalties for repeated tokens, biases and masks of allowed tokens (``ajllm_amd.sampling.adjust_logits``).

``run`` makes these calls where ``own`` is true and computes their plain form otherwise; ``exact`` is the definition in 64 bits.
"""

import math

import torch

own = False

DEVICE = "cuda"
EPS = 1e-5
THETA = 10000.0


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # eight completions of one prompt, one token of the 12-layer model (fp32 caches, the model's own type): the smallest call
        dict(name="rotate_token", kind="rotate", batch=8, seq=1, heads=16, kv_heads=16, dim=128, max_len=512, into="float32", q="float32"),
        # a batch at ragged positions, grouped heads, bf16 caches
        dict(name="rotate_batch", kind="rotate", batch=96, seq=1, heads=32, kv_heads=8, dim=128, max_len=1024, into="bfloat16", q="float32"),
        # questions of up to 333 tokens behind a common instruction, all at once
        dict(name="rotate_prompts", kind="rotate", batch=16, seq=333, heads=32, kv_heads=8, dim=128, max_len=512, into="bfloat16",
             q="bfloat16"),
        # a few completions of a short prompt, fp32 caches
        dict(name="share_few", kind="share", groups=1, batch=4, seq=1, heads=16, kv_heads=16, dim=128, prefix=512, max_len=256,
             cache="float32", q="float32"),
        # a batch of completions of one prompt, grouped heads
        dict(name="share_batch", kind="share", groups=1, batch=32, seq=1, heads=32, kv_heads=8, dim=128, prefix=2048, max_len=512,
             cache="bfloat16", q="float32"),
        # eight prompts of unequal lengths with eight completions each, the medium model's heads
        dict(name="share_groups", kind="share", groups=8, batch=64, seq=1, heads=12, kv_heads=12, dim=64, prefix=1500, max_len=300,
             cache="bfloat16", q="float32"),
        # questions of up to 100 tokens read behind a common instruction
        dict(name="share_questions", kind="share", groups=1, batch=16, seq=100, heads=32, kv_heads=8, dim=128, prefix=2048, max_len=160,
             cache="bfloat16", q="bfloat16"),
        # many completions behind a very long document
        dict(name="share_large", kind="share", groups=1, batch=128, seq=1, heads=32, kv_heads=8, dim=128, prefix=32768, max_len=1000,
             cache="bfloat16", q="bfloat16"),
        # one sequence, a small vocabulary: a launch is all there is
        dict(name="logits_one", kind="logits", batch=1, vocab=32000, prompt=512, tokens=200, biases=16, mask="none", type="float32"),
        # a batch under a grammar whose states have a mask each
        dict(name="logits_batch", kind="logits", batch=32, vocab=128256, prompt=2048, tokens=512, biases=16, mask="states", type="float32"),
        # an odd vocabulary and an odd batch, bf16 logits, masks only
        dict(name="logits_odd", kind="logits", batch=37, vocab=32011, prompt=0, tokens=0, biases=0, mask="rows", type="bfloat16"),
        # the largest batch, long histories
        dict(name="logits_large", kind="logits", batch=256, vocab=128256, prompt=8192, tokens=1024, biases=64, mask="rows", type="float32"),
    ]


# (query heads, key / value heads, head size) of this repository's models, and neighbours with other numbers of heads a key head
LAYOUTS = [(16, 16, 128), (32, 8, 128), (32, 32, 128), (16, 8, 128), (32, 4, 128), (12, 12, 64), (12, 6, 64), (12, 4, 64), (16, 16, 32),
           (16, 4, 32)]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _drawn(rng):
    kind = rng.choice(["rotate", "share", "share", "logits"])
    heads, kv_heads, dim = rng.choice(LAYOUTS)
    types = ["bfloat16", "float32"]
    if kind == "rotate":
        seq = rng.choice([1, 1, _log(rng, 2, 600)])
        return dict(kind=kind, batch=_log(rng, 1, 256 if seq == 1 else 32), seq=seq, heads=heads, kv_heads=kv_heads, dim=dim,
                    max_len=seq + _log(rng, 16, 1500), into=rng.choice(types), q=rng.choice(types))
    if kind == "share":
        seq = rng.choice([1, 1, 1, _log(rng, 2, 200)])
        groups = rng.choice([1, 1, rng.randrange(2, 9)])
        return dict(kind=kind, groups=groups, batch=groups * _log(rng, 1, (160 if seq == 1 else 24) / groups + 1), seq=seq, heads=heads,
                    kv_heads=kv_heads, dim=dim, prefix=_log(rng, 1, 32768 // groups), max_len=seq + _log(rng, 1, 1500),
                    cache=rng.choice(["bfloat16", "bfloat16", "float32"]), q=rng.choice(types))
    history = rng.random() < 0.8
    return dict(kind=kind, batch=_log(rng, 1, 256), vocab=rng.choice([32000, 128256, _log(rng, 1000, 160000)]),
                prompt=_log(rng, 1, 8192) if history else 0, tokens=_log(rng, 1, 2048) if history else 0, biases=rng.choice([0, 1, 16, 100]),
                mask=rng.choice(["none", "rows", "states"]), type=rng.choice(["float32", "float32", "bfloat16"]))


def draw(rng):
    def cost(case):
        w = work(case)
        return max(w["bytes"], w["flops"] / 50)

    most = max(cost(c) for c in listed()) / 2
    while True:
        case = _drawn(rng)
        if cost(case) <= most:
            return case


# ------------------------------------------------------------------ inputs
def _lengths(gen, count, low, high):
    """Whole numbers in [low, high], one of them the largest."""
    n = torch.randint(low, high + 1, (count,), generator=gen, device=DEVICE)
    n[int(torch.randint(0, count, (1,), generator=gen, device=DEVICE))] = high
    return n


def _angles(positions, dim):
    return torch.arange(positions, dtype=torch.float64, device=DEVICE)[:, None] * THETA ** (
        -torch.arange(0, dim, 2, dtype=torch.float64, device=DEVICE) / dim)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=gen, device=DEVICE)

    if case["kind"] == "rotate":
        b, t, h, g, d, m = (case[k] for k in ("batch", "seq", "heads", "kv_heads", "dim", "max_len"))
        into = getattr(torch, case["into"])
        counts = _lengths(gen, b, (t + 1) // 2, t)
        rows = _lengths(gen, b, 0, m - t)
        prefix = 700
        angles = _angles(prefix + m, d)
        return dict(kind="rotate", qkv=randn(b * t, (h + 2 * g) * d), cosine=angles.cos().float(), sine=angles.sin().float(),
                    keys=randn(b, g, m, d).to(into), values=randn(b, g, m, d).to(into), rows=rows, positions=rows + prefix,
                    counts=counts if t > 1 else None, heads=h, seq=t, q_gain=1 + 0.2 * randn(d), k_gain=1 + 0.2 * randn(d),
                    out=getattr(torch, case["q"]))
    if case["kind"] == "share":
        n, b, t, h, g, d, p, m = (case[k] for k in ("groups", "batch", "seq", "heads", "kv_heads", "dim", "prefix", "max_len"))
        cache = getattr(torch, case["cache"])
        lengths = _lengths(gen, n, (p + 1) // 2, p)
        return dict(kind="share", q=randn(b, h, t, d).to(getattr(torch, case["q"])), prefix_keys=randn(n, g, p, d).to(cache),
                    prefix_values=randn(n, g, p, d).to(cache), prefix_lengths=lengths, keys=randn(b, g, m, d).to(cache),
                    values=randn(b, g, m, d).to(cache), rows=_lengths(gen, b, 0, m - t),
                    counts=_lengths(gen, b, (t + 1) // 2, t) if t > 1 else None)
    b, v = case["batch"], case["vocab"]
    s = dict(kind="logits", logits=(3 * randn(b, v)).to(getattr(torch, case["type"])))
    uniform = lambda low, high: low + (high - low) * torch.rand(b, generator=gen, device=DEVICE)  # noqa: E731

    def text(length):
        """Tokens as a text has them: few of them make up most of it."""
        u = torch.rand((b, length), generator=gen, device=DEVICE)
        return (v ** u - 1).long().clamp_(0, v - 1), _lengths(gen, b, (length + 1) // 2, length)

    if case["tokens"]:
        s["prompt"], s["prompt_lengths"] = text(case["prompt"])
        s["tokens"], s["lengths"] = text(case["tokens"])
        s["repetition"], s["frequency"], s["presence"] = uniform(1.0, 1.5), uniform(0.0, 0.5), uniform(0.0, 0.5)
    if case["biases"]:
        first = torch.randint(0, v, (b, 1), generator=gen, device=DEVICE)
        s["bias_ids"] = (first + 7 * torch.arange(case["biases"], device=DEVICE)) % v   # (all of a row's are different)
        s["bias"] = 5 * randn(b, case["biases"])
    if case["mask"] != "none":
        states = b if case["mask"] == "rows" else 2 * b + 5
        s["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (states, (v + 31) // 32), generator=gen, device=DEVICE).int()
        if case["mask"] == "states":
            s["allowed_rows"] = torch.randint(-1, states, (b,), generator=gen, device=DEVICE)   # -1: a row without a mask
    return s


# ------------------------------------------------------------------ the plain forms
def _plain_rotate(s):
    qkv, keys, values, t = s["qkv"], s["keys"], s["values"], s["seq"]
    b, g, m, d = keys.shape
    x = qkv.float().view(b, t, -1, d)
    h = s["heads"]
    q, k, v = x[:, :, :h], x[:, :, h:h + g], x[:, :, h + g:]
    step = torch.arange(t, device=DEVICE)
    at = s["positions"][:, None] + step
    cosine, sine = s["cosine"][at][:, :, None], s["sine"][at][:, :, None]

    def turned(z, gain):
        z = z / torch.sqrt(torch.mean(z * z, dim=-1, keepdim=True) + EPS) * gain
        even, odd = z[..., ::2], z[..., 1::2]
        return torch.stack((even * cosine - odd * sine, even * sine + odd * cosine), dim=-1).flatten(-2)

    q, k = turned(q, s["q_gain"]), turned(k, s["k_gain"])
    there = torch.ones((b, t), dtype=torch.bool, device=DEVICE) if s["counts"] is None else step < s["counts"][:, None]
    q = torch.where(there[:, :, None, None], q, 0.0).transpose(1, 2).contiguous().to(s["out"])
    into = (s["rows"][:, None] + step)[:, None, :, None].expand(b, g, t, d)

    def put(cache, new):   # (a token that is not there writes back what its row holds)
        cache.scatter_(2, into, torch.where(there[:, None, :, None], new.transpose(1, 2).to(cache.dtype), cache.gather(2, into)))

    put(keys, k)
    put(values, v)
    return q, keys, values


def _plain_share(s):
    q, rows = s["q"].float(), s["rows"]
    b, h, t, d = q.shape
    n, g, p, _ = s["prefix_keys"].shape
    m, r, each = s["keys"].shape[2], h // g, b // n
    q = q.view(n, each, g, r * t, d).transpose(1, 2).contiguous()                                   # [n, g, each, r t, d]
    before = (q.view(n, g, each * r * t, d) @ s["prefix_keys"].float().transpose(-1, -2).contiguous()).view(n, g, each, r, t, p)
    mine = s["keys"].float().view(n, each, g, m, d).transpose(1, 2)
    behind = (q @ mine.transpose(-1, -2).contiguous()).view(n, g, each, r, t, m)
    step = torch.arange(t, device=DEVICE)
    there = torch.arange(p, device=DEVICE) < s["prefix_lengths"].view(n, 1, 1, 1, 1, 1)
    seen = torch.arange(m, device=DEVICE) <= (rows[:, None] + step).view(n, 1, each, 1, t, 1)
    scores = torch.cat((torch.where(there, before, -math.inf), torch.where(seen, behind, -math.inf)), dim=-1) / math.sqrt(d)
    weights = torch.exp(scores - torch.amax(scores, dim=-1, keepdim=True))
    total = torch.sum(weights, dim=-1, keepdim=True)
    out = (weights[..., :p].reshape(n, g, each * r * t, p) @ s["prefix_values"].float()).view(n, g, each, r, t, d)
    out = out + (weights[..., p:].reshape(n, g, each, r * t, m) @ s["values"].float().view(n, each, g, m, d).transpose(1, 2)).view(
        n, g, each, r, t, d)
    out = (out / total).permute(0, 2, 4, 1, 3, 5).reshape(b, t, h * d)
    if s["counts"] is not None:
        out = torch.where((step < s["counts"][:, None])[:, :, None], out, 0.0)
    return out.bfloat16()


def _plain_logits(s):
    x = s["logits"].float()
    b, v = x.shape
    if "tokens" in s:
        def counted(ids, lengths):
            there = torch.arange(ids.shape[1], device=DEVICE) < lengths[:, None]
            return torch.zeros((b, v), device=DEVICE).scatter_add_(1, ids, there.float())

        count, given = counted(s["tokens"], s["lengths"]), counted(s["prompt"], s["prompt_lengths"])
        r = s["repetition"][:, None]
        x = torch.where(count + given > 0, torch.where(x > 0, x / r, x * r), x)
        x = x - (s["frequency"][:, None] * count + torch.where(count > 0, s["presence"][:, None], 0.0))
    if "bias" in s:
        x = x.scatter_add(1, s["bias_ids"], s["bias"])
    if "allowed" in s:
        which = s.get("allowed_rows")
        words = s["allowed"] if which is None else torch.where(which[:, None] < 0, -1, s["allowed"][which.clamp(min=0)])
        bits = (words[:, :, None] >> torch.arange(32, dtype=torch.int32, device=DEVICE)) & 1
        x = torch.where(bits.view(b, -1)[:, :v] != 0, x, -math.inf)
    return x


def run(state):
    kind = state["kind"]
    if own:
        from ajllm_amd import attention, sampling

        s = state
        if kind == "rotate":
            q = attention.norm_rope(s["qkv"], s["cosine"], s["sine"], s["keys"], s["values"], s["rows"], heads=s["heads"],
                                    tokens=s["seq"], q_gain=s["q_gain"], k_gain=s["k_gain"], epsilon=EPS, positions=s["positions"],
                                    counts=s["counts"], out_dtype=s["out"])
            return q, s["keys"], s["values"]
        if kind == "share":
            return attention.shared_prefix_attention(s["q"], s["prefix_keys"], s["prefix_values"], s["prefix_lengths"], s["keys"],
                                                     s["values"], s["rows"], counts=s["counts"])
        return sampling.adjust_logits(**{k: x for k, x in s.items() if k != "kind"})
    return {"rotate": _plain_rotate, "share": _plain_share, "logits": _plain_logits}[kind](state)


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_rotate(s):
    keys, values, t, h = s["keys"].double(), s["values"].double(), s["seq"], s["heads"]
    b, g, m, d = keys.shape
    x = s["qkv"].double().view(b, t, h + 2 * g, d).cpu()
    turn = torch.complex(s["cosine"].double(), s["sine"].double()).cpu()
    x[:, :, :h + g] /= (x[:, :, :h + g].square().sum(-1, keepdim=True) / d + EPS).sqrt()
    x[:, :, :h] *= s["q_gain"].double().cpu()
    x[:, :, h:h + g] *= s["k_gain"].double().cpu()
    q = torch.zeros((b, h, t, d), dtype=torch.float64)
    keys, values = keys.cpu(), values.cpu()
    for i, (row, at) in enumerate(zip(s["rows"].tolist(), s["positions"].tolist())):
        many = t if s["counts"] is None else int(s["counts"][i])
        z = torch.view_as_complex(x[i, :many, :h + g].reshape(many, h + g, d // 2, 2)) * turn[at:at + many, None]
        z = torch.view_as_real(z).reshape(many, h + g, d).transpose(0, 1)
        q[i, :, :many] = z[:h]
        keys[i, :, row:row + many] = z[h:]
        values[i, :, row:row + many] = x[i, :many, h + g:].transpose(0, 1)
    return q, keys, values


def _exact_share(s):
    b, h, t, d = s["q"].shape
    n, g = s["prefix_keys"].shape[:2]
    r, each = h // g, b // n
    out = torch.zeros((b, t, h, d), dtype=torch.float64, device=DEVICE)
    longest = s["prefix_lengths"].tolist()
    rows = s["rows"].tolist()
    counts = [t] * b if s["counts"] is None else s["counts"].tolist()
    for k in range(g):
        for i in range(n):
            pk, pv = s["prefix_keys"][i, k, :longest[i]].double(), s["prefix_values"][i, k, :longest[i]].double()
            for j in range(i * each, (i + 1) * each):
                many = counts[j]
                last = rows[j] + many
                q = s["q"][j, k * r:(k + 1) * r, :many].double().reshape(r * many, d)
                dots = torch.cat((q @ pk.t().contiguous(), q @ s["keys"][j, k, :last].double().t().contiguous()), dim=1) / d ** 0.5
                future = torch.ones((many, last), dtype=torch.bool, device=DEVICE).triu_(rows[j] + 1).repeat(r, 1)
                dots[:, longest[i]:].masked_fill_(future, -math.inf)
                w = torch.softmax(dots, dim=1)
                o = w[:, :longest[i]] @ pv + w[:, longest[i]:] @ s["values"][j, k, :last].double()
                out[j, :many, k * r:(k + 1) * r] = o.view(r, many, d).transpose(0, 1)
    return out.view(b, t, h * d)


def _exact_logits(s):
    out = s["logits"].double()
    b, v = out.shape
    for i in range(b):
        x = out[i]
        if "tokens" in s:
            count = torch.bincount(s["tokens"][i, :int(s["lengths"][i])], minlength=v)
            given = torch.bincount(s["prompt"][i, :int(s["prompt_lengths"][i])], minlength=v)
            seen = ((count > 0) | (given > 0)).nonzero().view(-1)
            x[seen] *= torch.exp(-torch.sign(x[seen]) * torch.log(s["repetition"][i].double()))
            x -= s["frequency"][i].double() * count
            x[count > 0] -= s["presence"][i].double()
        if "bias" in s:
            x[s["bias_ids"][i]] += s["bias"][i].double()
        if "allowed" in s:
            which = i if "allowed_rows" not in s else int(s["allowed_rows"][i])
            if which >= 0:
                place = torch.arange(v, device=DEVICE)
                x[(s["allowed"][which].long()[place // 32] // 2 ** (place % 32)) % 2 == 0] = -math.inf
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotate": _exact_rotate, "share": _exact_share, "logits": _exact_logits}[case["kind"]](s)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = {"bfloat16": 2, "float32": 4}
    if case["kind"] == "rotate":
        b, h, g, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
        tokens = b * (case["seq"] if case["seq"] == 1 else 0.75 * case["seq"])       # (lengths are drawn from the upper half)
        read = tokens * ((h + 2 * g) * d * 4 + d * 4) + 2 * d * 4 + 8 * b
        write = b * case["seq"] * h * d * size[case["q"]] + tokens * 2 * g * d * size[case["into"]]
        return {"bytes": read + write, "flops": tokens * d * (8 * (h + g))}
    if case["kind"] == "share":
        n, b, t, h, g, d, m = (case[k] for k in ("groups", "batch", "seq", "heads", "kv_heads", "dim", "max_len"))
        prefix = case["prefix"] if n == 1 else 0.75 * case["prefix"] + 0.25 * case["prefix"] / n
        new = t if t == 1 else 0.75 * t
        mine = (m - t) / 2 + new
        rows = n * g * prefix + b * g * mine
        seen = prefix + (m - t) / 2 + (new + 1) / 2
        return {"bytes": rows * 2 * d * size[case["cache"]] + b * h * d * (new * size[case["q"]] + t * 2), "flops": 4 * b * h * new * d * seen}
    b, v = case["batch"], case["vocab"]
    ids = 0.75 * (case["prompt"] + case["tokens"]) * 8 + case["biases"] * 12 + (12 if case["tokens"] else 0)
    masks = (v / 8 if case["mask"] != "none" else 0) + (8 if case["mask"] == "states" else 0)
    return {"bytes": b * (v * (size[case["type"]] + 4) + ids + masks), "flops": 4 * b * v}
