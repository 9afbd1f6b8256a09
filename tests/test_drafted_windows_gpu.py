"""Steps of drafted trees in models of windowed layers that keep first positions, with softmax sinks, keys and values of different widths, heads that no
tile divides, and layers that read another one's cache: the logits of the trees' ways, from prompt to kept rows and beyond, captured and not."""

from __future__ import annotations

import copy

import pytest
import torch

import dolutar_configs as dc
import dolutar_plain as plain
import drafted_refs as refs
from mlx_omnia_b200.engine.engine import Engine, EngineArgs
from mlx_omnia_b200.engine.step import StepEntry
from mlx_omnia_b200.kernels import ops
from test_drafted import chosen_on

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"


def without_pairs(name):
    """The configuration with an embedding of tokens alone: the hashed pair's row goes by the token before, which is state of the request."""
    raw, weights = copy.deepcopy(dc.config(name)), dict(dc.tensors(name))
    del raw["embedding"]["bigram"], weights["bigram"]
    return raw, weights


def relative(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    return float((a - b).abs().max() / b.abs().max())


@pytest.mark.parametrize("name", list("PQRSO"))
def test_trees_have_the_logits_of_their_ways(name):
    raw, weights = without_pairs(name)
    page = 16 if name == "S" else 4
    engine = Engine.from_tensors(raw, weights, EngineArgs(dtype="float32", page_size=page, cache_tokens=2048, max_requests=4, device=DEVICE))
    assert engine.runner.drafted.why_not() is None
    vocab, prompts = engine.vocab_size, [dc.prompt(n, raw["vocab"], n) for n in (41, 3, 140)]
    requests = [engine.cache.open(str(i)) for i in range(3)]
    engine.runner.run([StepEntry(r, p[:-1]) for r, p in zip(requests, prompts)])
    for turn in range(6):
        trees = [refs.tree(n, 7 * turn + i, 3) for i, n in enumerate((9, 5, 2))]
        tokens = [[p[-1], *dc.prompt(len(t) - 1, raw["vocab"], 30 + 5 * turn + i)] for i, (p, t) in enumerate(zip(prompts, trees))]
        entries = [StepEntry(r, t, list(range(len(t))), p) for r, t, p in zip(requests, tokens, trees)]
        logits = engine.runner.run(entries).cpu()
        row, chosen = 0, []
        for p, mine, parents in zip(prompts, tokens, trees):
            picks = []
            for way in refs.ways(parents):
                expect = plain.forward(p[:-1] + [mine[j] for j in way], weights, raw)[-1]
                assert relative(logits[row], expect) < 2e-5
                picks.append(int(expect.argmax()))
                row += 1
            last = 0
            for _ in range(turn):  # the last child's way down
                children = [j for j, q in enumerate(parents) if q == last]
                if not children:
                    break
                picks[last] = mine[children[-1]]
                last = children[-1]
            chosen.append(picks)
        kept = engine.runner.keep(entries, chosen_on(DEVICE, [c for picks in chosen for c in picks]))
        for i, (mine, parents, picks, found) in enumerate(zip(tokens, trees, chosen, kept)):
            path = refs.accept(parents, mine, picks)
            assert found.tokens == [mine[j] for j in path[1:]] and found.next == picks[path[-1]]
            prompts[i] = prompts[i][:-1] + [mine[j] for j in path] + [found.next]
        engine.cache.check()
    got = engine.runner.run([StepEntry(r, [p[-1]], [0]) for r, p in zip(requests, prompts)]).cpu()
    for i, p in enumerate(prompts):
        assert relative(got[i], plain.forward(p, weights, raw)[-1]) < 2e-5
    assert vocab == raw["vocab"] and engine.runner.drafted_graphs.replays >= 1
    ops.raise_on_error(torch.device(DEVICE))
