"""Which way tree attention goes (tree_plan.h) for the calls that test_gpu_draft_forms.py makes of every form: each goes the way that stands above it there, and no call of 200000
others goes a way that none of them does.  Compiled for the host alone."""

import random
import re
import subprocess
from pathlib import Path

import pytest

from tests import test_gpu_draft_forms as forms

ROOT = Path(__file__).resolve().parents[1]
PROGRAM = """
#include <stdio.h>
#include "%s"
int main() {
  ajqt_tree_attention_args a{};
  while (scanf("%%d %%d %%d %%d %%d %%d %%d %%d", &a.batch, &a.tokens, &a.heads, &a.kv_heads, &a.dim, &a.max_len, &a.q_dtype, &a.cache_dtype) == 8) {
    const TreePlan p = plan_tree(&a);
    printf("%%d %%d %%d %%d %%d %%d %%lld %%lld %%zu\\n", p.walk, p.rt, p.waves, p.alone, p.runs, p.tiles, p.blocks, p.queries, p.bytes);
  }
}
""" % (ROOT / "ajllm_amd" / "csrc" / "tree_plan.h")


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    at = tmp_path_factory.mktemp("plan")
    (at / "plan.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", str(at / "plan.cpp"), "-o", str(at / "plan")], check=True)

    def plans(calls):
        text = "".join(" ".join(map(str, call)) + "\n" for call in calls)
        lines = subprocess.run([str(at / "plan")], input=text, check=True, capture_output=True, text=True).stdout.splitlines()
        assert len(lines) == len(calls)
        return [tuple(map(int, line.split())) for line in lines]

    return plans


def _form(call, plan):
    walk, rt, waves, alone, runs = plan[:5]
    return (*call[4:5], *call[6:], walk, rt, waves, alone, runs > 0)


def test_calls_go_the_ways_above_them(plan):
    """The comments of the list name way, tiles, waves, and whether a second launch puts parts together."""
    said, heading = [], None
    for line in Path(forms.__file__).read_text().split("CALLS = [", 1)[1].split("\n]\n", 1)[0].splitlines():
        if line.strip().startswith("#"):
            heading = line.strip()[2:]
        else:
            said += [heading] * len(re.findall(r"\(\d[\d, ]+\)", line))
    assert len(said) == len(forms.CALLS)
    for call, heading, (walk, rt, waves, alone, runs, *_) in zip(forms.CALLS, said, plan(forms.CALLS)):
        if "each a wave's" in heading:
            assert alone and not walk and rt == 1 and not runs, (call, heading)
            continue
        tiles, wanted = re.match(r"(?:tiles of (\d+)|\d tiles of 16 a wave), (\d) waves", heading).groups()
        assert not alone and waves == int(wanted) and bool(runs) == ("in parts" in heading) and ("in parts" in heading) != ("in one launch" in heading), (call, heading)
        assert (walk, rt) == ((0, int(tiles) // 16) if tiles else (1, int(heading[0]))), (call, heading)
        assert ("laid down" in heading) == (walk == 1 and call[7] == 0), (call, heading)


def test_no_other_call_goes_another_way(plan):
    gen = random.Random(1)
    log = lambda low, high: round(low * (high / low) ** gen.random())  # noqa: E731
    calls = []
    for _ in range(200000):
        kv, share = gen.choice([1, 2, 3, 4, 8, 16, 32]), gen.choice([1, 2, 3, 4, 5, 8, 16, 32])
        calls.append((log(1, 600), log(1, 300), kv * share, kv, gen.choice([32, 64, 128]), log(1, 100000), gen.randrange(2), gen.randrange(2)))
    known = {_form(call, p) for call, p in zip(forms.CALLS, plan(forms.CALLS))}
    assert len(known) >= len(forms.CALLS) - 2
    for call, p in zip(calls, plan(calls)):
        assert _form(call, p) in known, (call, p)
        walk, rt, waves, alone, runs, tiles, blocks, queries, size = p
        batch, tokens, heads, kv, dim = call[:5]
        mine = tokens * (heads // kv)
        # every query in a tile, every tile in a workgroup; parts for batches that they can be dealt out to, and as many as the merge takes
        assert tiles == -(-mine // (16 * rt * (waves if walk else 1))) and queries == batch * heads * tokens
        assert blocks * (4 if alone else 1) >= (runs * kv if runs else batch * kv) * tiles
        assert runs == 0 or (batch < runs <= 64 * batch and batch <= 64)
        assert size == (runs * kv * mine * (8 + 4 * dim) + 8 * batch if runs else 0)
