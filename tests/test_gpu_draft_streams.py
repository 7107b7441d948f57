"""The operators of checking drafted tokens captured into graphs, on streams side by side and from threads: workspaces and results are a call's own."""

import threading

import pytest
import torch

from ajllm_amd import attention, sampling
from tests.test_gpu_draft import BF16, F32, _gen, _tree

pytestmark = pytest.mark.gpu


def _tree_call(cuda, batch, nodes, heads, kv, hd, max_len, q_type, cache_type):
    gen = _gen(nodes)
    q = torch.randn((batch, heads, nodes, hd), generator=gen).to(q_type).to(cuda)
    keys, values = (torch.randn((batch, kv, max_len, hd), generator=gen).to(cache_type).to(cuda) for _ in range(2))
    rows = torch.randint(0, max_len - nodes + 1, (batch,), generator=gen)
    rows[0] = max_len - nodes
    rows, masks = rows.to(cuda), attention.tree_masks(_tree(gen, nodes, batch))[0].to(cuda)
    return lambda: (attention.tree_attention(q, keys, values, rows, masks),)


def _calls(cuda):
    gen = _gen(5)
    logits, targets = torch.randn((3, 128256), generator=gen).to(cuda), torch.tensor([5, 128255, 70000], device=cuda)
    cache = torch.randn((2, 2, 2, 900, 64), generator=gen).to(cuda)
    index = torch.arange(0, 900, 3, device=cuda)
    tokens, parents = torch.randint(0, 2, (4, 300), generator=gen).to(cuda), _tree(gen, 300).to(cuda)

    rows = torch.tensor([0, 1], device=cuda)

    def keep(count):
        keys, values = cache.clone(), cache.flip(0).clone()
        attention.keep_rows(keys, values, rows, index[:count])
        return keys, values

    return [_tree_call(cuda, 1, 3, 2, 2, 64, 3000, F32, BF16),          # in parts, tiles of 16
            _tree_call(cuda, 1, 200, 4, 2, 128, 3000, BF16, BF16),      # in parts, waves on the same rows
            _tree_call(cuda, 8, 300, 4, 2, 128, 700, BF16, BF16),
            _tree_call(cuda, 2, 200, 32, 8, 32, 1500, F32, F32),        # fp32 rows laid down once, in parts
            _tree_call(cuda, 2, 9, 8, 8, 32, 200, F32, F32),
            lambda: tuple(sampling.token_log_probs(logits, targets, top=64)),
            lambda: tuple(sampling.token_log_probs(logits[:, :1000], top=3)[2:]),
            lambda: keep(300), lambda: keep(16),
            lambda: tuple(sampling.follow_drafts(tokens, parents, tokens.roll(1, 1)))]


def _same(got, want):
    return len(got) == len(want) and all(torch.equal(x, y) for x, y in zip(got, want))


def test_graphs_replay_as_eager_calls(cuda):
    calls = _calls(cuda)
    want = [call() for call in calls]
    torch.cuda.synchronize()
    graphs = []
    for call in calls + calls:   # (two graphs of each)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results = call()
        graphs.append((graph, results))
    for turn in range(4):
        for graph, results in graphs:
            for x in results:
                x.zero_()
        for graph, _ in graphs if turn % 2 else reversed(graphs):
            graph.replay()
        again = [call() for call in calls]   # (eager work behind them)
        torch.cuda.synchronize()
        for i, (_, results) in enumerate(graphs):
            assert _same(results, want[i % len(calls)]), (turn, i)
        for i, results in enumerate(again):
            assert _same(results, want[i]), (turn, i)


def test_streams_side_by_side(cuda):
    calls = _calls(cuda)
    want = [call() for call in calls]
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream() for _ in range(3)], []
    for turn in range(3):
        for k, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                order = list(range(len(calls)))[k:] + list(range(k))
                results.append((order, [calls[i]() for i in order]))
    torch.cuda.synchronize()
    for order, got in results:
        for i, x in zip(order, got):
            assert _same(x, want[i]), i


def test_threads(cuda):
    calls = _calls(cuda)
    want = [call() for call in calls]
    torch.cuda.synchronize()
    wrong = []

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for turn in range(5):
                for i in range(len(calls)):
                    i = (i + 3 * k) % len(calls)
                    got = calls[i]()
                    torch.cuda.current_stream().synchronize()
                    if not _same(got, want[i]):
                        wrong.append((k, turn, i))

    threads = [threading.Thread(target=work, args=(k,)) for k in range(3)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not wrong
