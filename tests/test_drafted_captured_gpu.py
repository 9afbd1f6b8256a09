"""Steps of drafted trees from captured graphs: the logits of the trees' ways, whatever lengths and shapes a graph is replayed for, and the tokens of
generation without drafts."""

from __future__ import annotations

import random

import pytest
import torch

import drafted_refs as refs
import plain_impl
import tiny_configs
from mlx_omnia_b200 import GenerationOptions, min_p, repetition_penalty, sampler, temperature
from mlx_omnia_b200.engine.decode_graph import MIXED_MAX_GRAPHS
from mlx_omnia_b200.engine.generate import Generator
from mlx_omnia_b200.engine.step import StepEntry
from mlx_omnia_b200.kernels import ops
from test_drafted import chosen_on, engine_for

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"


@pytest.mark.parametrize("name", ["A", "B"])
def test_captured_trees_have_the_logits_of_their_ways(name):
    """Two or four requests, some of which bring a single token, 13 to 16 rows in all; what one request has is kept for the next step, and some leave."""
    engine, raw, weights = engine_for(name, DEVICE, cache_tokens=2048, page_size=16)
    vocab, rng = engine.vocab_size, random.Random(5)
    prompts = {str(i): tiny_configs.prompt(n, vocab, n) for i, n in enumerate((37, 6, 90, 1))}
    requests = {k: engine.cache.open(k) for k in prompts}
    held = [StepEntry(requests[k], p[:-1]) for k, p in prompts.items() if len(p) > 1]
    engine.runner.run(held)
    graphs, before = engine.runner.drafted_graphs, None
    for turn in range(14):
        names = rng.sample(sorted(prompts), 2 if turn % 3 == 2 else 4)
        sizes = [7, *(rng.choice([1, 3]) for _ in names[1:])]
        sizes[-1] = max(sizes[-1], 13 - sum(sizes[:-1]))
        trees = [refs.tree(n, 3 * turn + i, 3) for i, n in enumerate(sizes)]
        tokens = [[prompts[k][-1], *tiny_configs.prompt(n - 1, vocab, 9 * turn + n)] for k, n in zip(names, sizes)]
        entries = [StepEntry(requests[k], t, list(range(len(t))), p) for k, t, p in zip(names, tokens, trees)]
        result = engine.runner.run(entries)
        logits = result.cpu()
        if before is not None:  # a result is its caller's
            assert torch.equal(before[0], before[1].cpu())
        before = logits, result
        row, chosen = 0, []
        for k, t, parents in zip(names, tokens, trees):
            mine = []
            for way in refs.ways(parents):
                expect = plain_impl.forward(raw, weights, prompts[k][:-1] + [t[j] for j in way])[-1:]
                assert plain_impl.relative_diff(logits[row: row + 1], expect) < 2e-5
                mine.append(int(expect.argmax()))
                row += 1
            children = [j for j, q in enumerate(parents) if q == 0]
            if children:
                mine[0] = t[children[-1]]
            chosen.append(mine)
        kept = engine.runner.keep(entries, chosen_on(DEVICE, [c for mine in chosen for c in mine]))
        for k, t, parents, mine, found in zip(names, tokens, trees, chosen, kept):
            path = refs.accept(parents, t, mine)
            assert found.tokens == [t[j] for j in path[1:]] and found.next == mine[path[-1]]
            prompts[k] = prompts[k][:-1] + [t[j] for j in path] + [found.next]
        engine.cache.check()
    assert graphs.replays >= 4
    ops.raise_on_error(torch.device(DEVICE))


def test_generation_with_captured_steps_of_drafts():
    """Requests that come and go, a cache of another size in between, more shapes than graphs are kept for."""
    engine, _, _ = engine_for("B", DEVICE, cache_tokens=1024)
    options = [GenerationOptions(max_tokens=30, stop=()),
               GenerationOptions(max_tokens=30, stop=(), sampler=sampler(temperature(1.1), min_p(0.02), seed=9), penalty=repetition_penalty(1.2, context=7),
                                 frequency_penalty=0.3)]
    rng, replays, generator = random.Random(2), 0, None
    for turn in range(6):
        prompts = [tiny_configs.prompt(n, engine.vocab_size, 90 + n + turn) for n in (5, 1, 21)[: 1 + turn % 3]]
        which = [options[(turn + i) % 2] for i in range(len(prompts))]
        expect = [Generator(engine).generate([p], o)[0] for p, o in zip(prompts, which)]
        generator = Generator(engine, max_tokens_per_step=64)
        requests = [generator.add(p, o) for p, o in zip(prompts, which)]
        while not generator.scheduler.idle:
            drafts = {}
            for request, tokens in zip(requests, expect):
                at = len(request.generated)
                if at and request.status == "running":
                    ahead = tokens[at: at + rng.choice([2, 2, 2, 5])]
                    drafts[request.request_id] = ([*ahead[:-1], (ahead[-1] + 1) % engine.vocab_size] if ahead else [], None)
            generator.step_drafted(drafts)
        assert [r.generated for r in requests] == expect
        replays += engine.runner.drafted_graphs.replays
        assert len(engine.runner.drafted_graphs.captured) <= MIXED_MAX_GRAPHS
        if turn == 3:
            generator.resize_cache(1536)
            assert not engine.runner.drafted_graphs.captured
        engine.cache.check()
    assert replays > 20
    ops.raise_on_error(torch.device(DEVICE))


@pytest.mark.parametrize("held,sizes", [(300, [9]), (2030, [9]), (700, [3, 12, 1]), (60, [17])])
def test_a_step_has_the_same_logits_captured_or_not(held, sizes):
    """In bfloat16, bit for bit, at every coming: 9 tokens of 3 query heads are 27 rows of attention and 48 as they are rounded, on the two sides of the
    choice between its kernels."""
    engine, _, _ = engine_for("C", DEVICE, cache_tokens=8192, page_size=16, max_requests=8, dtype="bfloat16")
    vocab, graphs, found = engine.vocab_size, engine.runner.drafted_graphs, []
    bases = [engine.cache.open(f"base {i}") for i in range(len(sizes))]
    for i, base in enumerate(bases):
        engine.runner.run([StepEntry(base, tiny_configs.prompt(held + 5 * i, vocab, 7 + i))])
    for turn in range(6):
        entries = [StepEntry(engine.cache.fork(base, f"fork {i}"), tiny_configs.prompt(n, vocab, 40 + i), list(range(n)), refs.tree(n, i, 4))
                   for i, (base, n) in enumerate(zip(bases, sizes))]
        found.append(engine.runner.run(entries).clone())
        kept = engine.runner.keep(entries, chosen_on(DEVICE, [vocab - 1] * sum(sizes)))
        assert [k.next for k in kept] == [vocab - 1] * len(sizes)
        for i in range(len(sizes)):
            engine.cache.close(f"fork {i}")
    assert graphs.replays == 3 and len(graphs.captured) == 1
    assert all(torch.equal(x, found[0]) for x in found)
    engine.cache.check()
    ops.raise_on_error(torch.device(DEVICE))


def test_what_is_not_captured():
    engine, _, _ = engine_for("A", DEVICE, cache_tokens=2048)
    graphs, request, other = engine.runner.drafted_graphs, engine.cache.open("r"), engine.cache.open("o")
    for _ in range(5):  # more rows than are captured; a portion of a prompt beside drafts
        for entries in ([StepEntry(request, [1] * 200, list(range(200)), refs.chain(200)), StepEntry(other, [1] * 60, list(range(60)), refs.chain(60))],
                        [StepEntry(request, [1, 2], [0, 1], [-1, 0]), StepEntry(other, [1, 2], [1])]):
            engine.runner.run(entries)
            engine.runner.keep(entries, chosen_on(DEVICE, [7] * sum(len(e.want) for e in entries)))
    assert not graphs.captured and not graphs.replays
    engine.cache.check()
