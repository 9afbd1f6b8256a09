"""Steps of drafted trees and options on logits through the engine, with the kernels on a GPU and with plain implementations in their place on the
CPU: a tree's rows have the logits of their ways, what is kept leaves a request as if it had brought nothing else, generation with drafts has
the tokens of generation without, and what cannot be done is refused."""

from __future__ import annotations

import math
import random

import pytest
import torch

import drafted_refs as refs
import fokalorn_configs
import plain_impl
import tiny_configs
from mlx_omnia_b200 import GenerationOptions, min_p, repetition_penalty, sampler, temperature, top_k
from mlx_omnia_b200.cache import CacheError
from mlx_omnia_b200.engine.engine import Engine, EngineArgs
from mlx_omnia_b200.engine.generate import Generator, LanguageModel
from mlx_omnia_b200.engine.step import StepEntry
from mlx_omnia_b200.kernels import ops
from mlx_omnia_b200.parts.base import KVSpec, KVView, StepContext
from mlx_omnia_b200.sampling.batch import allowed_ids, text_of
from mlx_omnia_b200.sampling.options import SamplingParams


@pytest.fixture(params=["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)])
def device(request, monkeypatch):
    if request.param == "cpu":
        request.getfixturevalue("cpu_ops")
        refs.swap_in(monkeypatch, ops)
    return request.param


def engine_for(name, device, cache_tokens=512, page_size=4, max_requests=4, dtype="float32"):
    raw, weights = tiny_configs.config(name), tiny_configs.tensors(name)
    args = EngineArgs(dtype=dtype, page_size=page_size, cache_tokens=cache_tokens, max_requests=max_requests, device=device)
    return Engine.from_tensors(raw, weights, args), raw, weights


def chosen_on(device, tokens):
    return torch.tensor(tokens, dtype=torch.int32, device=device)


# -- the step --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("name", ["A", "B"])
def test_a_tree_has_the_logits_of_its_ways(device, name):
    """Beside a portion of a prompt; then what agrees is kept, and decoding goes on from there. (B has windows of 16 positions.)"""
    engine, raw, weights = engine_for(name, device)
    vocab = engine.vocab_size
    prompts = [tiny_configs.prompt(n, vocab, n) for n in (37, 6)]
    requests = [engine.cache.open(str(i)) for i in range(2)]
    engine.runner.run([StepEntry(r, p[:-1]) for r, p in zip(requests, prompts)])
    for turn in range(3):
        tokens, trees = [], []
        for i, p in enumerate(prompts):
            parents = refs.tree(9 + i, 10 * turn + i, 4)
            tokens.append([p[-1], *tiny_configs.prompt(len(parents) - 1, vocab, 50 + 7 * turn + i)])
            trees.append(parents)
        if turn == 1:
            tokens[1], trees[1] = tokens[1][:1], [-1]  # no drafts
        entries = [StepEntry(r, t, list(range(len(t))), p) for r, t, p in zip(requests, tokens, trees)]
        logits = engine.runner.run(entries).cpu()
        row, chosen = 0, []
        for i, p in enumerate(prompts):
            mine = []
            for way in refs.ways(trees[i]):
                expect = plain_impl.forward(raw, weights, p[:-1] + [tokens[i][j] for j in way])[-1:]
                assert plain_impl.relative_diff(logits[row: row + 1], expect) < 2e-5
                mine.append(int(expect.argmax()))
                row += 1
            # A choice that goes down the tree for some tokens: whatever the first child's is.
            path = [0]
            while len(path) < 2 + turn:
                child = next((j for j, q in enumerate(trees[i]) if q == path[-1] and j != path[-1] + 1), None)
                if child is None:
                    break
                mine[path[-1]] = tokens[i][child]
                path = path + [child]
            chosen.append(mine)
        expect = [refs.accept(trees[i], tokens[i], chosen[i]) for i in range(2)]
        with pytest.raises(ValueError, match="not kept yet"):
            engine.runner.run([StepEntry(requests[0], [1], [0])])
        with pytest.raises(CacheError, match="not kept yet"):
            engine.cache.fork(requests[0], "f")
        kept = engine.runner.keep(entries, chosen_on(device, chosen[0] + chosen[1]))
        for i, (path, k) in enumerate(zip(expect, kept)):
            assert k.tokens == [tokens[i][j] for j in path[1:]] and k.next == chosen[i][path[-1]]
            prompts[i] = prompts[i][:-1] + [tokens[i][j] for j in path] + [k.next]
            assert requests[i].tokens == len(prompts[i]) - 1
        engine.cache.check()
        got = engine.runner.run([StepEntry(r, [p[-1]], [0]) for r, p in zip(requests, prompts)]).cpu()
        for i, p in enumerate(prompts):
            expect = plain_impl.forward(raw, weights, p)[-1:]
            assert plain_impl.relative_diff(got[i: i + 1], expect) < 2e-5
            prompts[i] = p + [int(expect.argmax())]
    for i in range(2):
        engine.cache.close(str(i))
    engine.cache.check()
    if device != "cpu":
        ops.raise_on_error(torch.device(device))


def test_a_portion_of_a_prompt_beside_a_tree(device):
    engine, raw, weights = engine_for("B", device)
    a, b = (tiny_configs.prompt(n, engine.vocab_size, n) for n in (20, 41))
    ra, rb = engine.cache.open("a"), engine.cache.open("b")
    engine.runner.run([StepEntry(ra, a[:-1]), StepEntry(rb, b[:10])])
    parents = refs.tree(7, 3)
    tokens = [a[-1], *tiny_configs.prompt(6, engine.vocab_size, 8)]
    entries = [StepEntry(ra, tokens, list(range(7)), parents), StepEntry(rb, b[10:], [3, 30])]
    logits = engine.runner.run(entries).cpu()
    expect = plain_impl.forward(raw, weights, b)
    assert plain_impl.relative_diff(logits[7:], expect[[13, 40]]) < 2e-5
    for j, way in enumerate(refs.ways(parents)):
        assert plain_impl.relative_diff(logits[j: j + 1], plain_impl.forward(raw, weights, a[:-1] + [tokens[i] for i in way])[-1:]) < 2e-5
    assert rb.tokens == 41 and rb.drafted == 0
    kept = engine.runner.keep(entries, chosen_on(device, [7] * 9))
    assert kept[1] is None and ra.tokens == 19 + len(refs.accept(parents, tokens, [7] * 7))
    engine.cache.check()


def test_steps_of_trees_that_are_refused(device):
    engine, _, _ = engine_for("A", device)
    run, request = engine.runner.run, engine.cache.open("r")
    free = [g.pool.free for g in engine.cache.groups]
    for tokens, want, parents in (([], [], []), ([1] * 257, list(range(257)), refs.chain(257)), ([1, 2], [0, 1], [0, 0]), ([1, 2], [0, 1], [-1, 1]),
                                  ([1, 2], [0, 1], [-1]), ([1, 2], [0], [-1, 0]), ([1, 2], [0, 2], [-1, 0]), ([1, 2, 3], [0, 1, 2], [-1, -1, 0])):
        with pytest.raises(ValueError):
            run([StepEntry(request, tokens, want, parents)])
    with pytest.raises(ValueError, match="once"):
        run([StepEntry(request, [1], [0], [-1]), StepEntry(request, [1], [0], [-1])])
    with pytest.raises(ValueError, match="host"):
        run([StepEntry(request, [1], [0], [-1])], device_tokens=chosen_on(device, [1]))
    assert request.tokens == 0 and free == [g.pool.free for g in engine.cache.groups]
    entries = [StepEntry(request, [1, 2], [0, 1], [-1, 0])]
    with pytest.raises(ValueError, match="run last"):
        engine.runner.keep(entries, chosen_on(device, [1, 1]))
    run(entries)
    with pytest.raises(ValueError, match="every row"):
        engine.runner.keep(entries, chosen_on(device, [1]))
    with pytest.raises(ValueError, match="run last"):
        engine.runner.keep([StepEntry(request, [1, 2], [0, 1], [-1, 0])], chosen_on(device, [1, 1]))
    engine.cache.close("r")
    with pytest.raises(ValueError, match="ended"):
        engine.runner.keep(entries, chosen_on(device, [1, 1]))
    engine.cache.check()


def test_more_drafts_than_pages_take_nothing(device):
    engine, _, _ = engine_for("A", device, cache_tokens=16)
    request = engine.cache.open("r")
    engine.runner.run([StepEntry(request, list(range(1, 12)))])
    with pytest.raises(CacheError):
        engine.runner.run([StepEntry(request, [1] * 9, list(range(9)), refs.chain(9))])
    assert request.tokens == 11 and request.drafted == 0
    engine.cache.check()


def test_a_model_with_state_takes_no_trees():
    raw = fokalorn_configs.config("X")
    engine = Engine.from_tensors(raw, fokalorn_configs.tensors("X"), EngineArgs(dtype="float32", page_size=4, cache_tokens=64, max_requests=1, device="cpu"))
    with pytest.raises(ValueError, match="keys and values alone"):
        engine.runner.run([StepEntry(engine.cache.open("r"), [1], [0], [-1])])
    with pytest.raises(ValueError, match="keys and values alone"):
        Generator(engine).step_drafted({})


# -- generation ------------------------------------------------------------------------------------------------------
OPTIONS = {"greedy": {}, "no token twice": {"frequency_penalty": 30.0}, "sampled": {"sampler": sampler(temperature(0.9), top_k(40), seed=5)},
           "penalties": {"sampler": sampler(temperature(1.1), min_p(0.02), seed=9), "penalty": repetition_penalty(1.2, context=7), "frequency_penalty": 0.3,
                         "presence_penalty": 0.4},
           "bias and rule": {"bias": {3: 4.0, 8: -math.inf, 11: 2.5}, "frequency_penalty": 0.8,
                             "constraint": lambda made: None if len(made) % 3 else range(0, 500, 1 + len(made) % 2)},
           "repetition alone": {"penalty": repetition_penalty(1.4)}}


@pytest.mark.parametrize("name", ["A", "B"])
@pytest.mark.parametrize("which", list(OPTIONS))
def test_drafts_do_not_change_what_is_generated(device, name, which):
    """Drafts that are partly what comes, partly not, in trees; short ends, a stop token, and requests that come and go."""
    options = GenerationOptions(max_tokens=17, stop=(), **OPTIONS[which])
    engine, _, _ = engine_for(name, device)
    prompts = [tiny_configs.prompt(n, engine.vocab_size, 90 + n) for n in (5, 1, 21)]
    expect = [Generator(engine).generate([p], options)[0] for p in prompts]
    generator = Generator(engine, max_tokens_per_step=64)
    requests = [generator.add(p, options) for p in prompts]
    rng, steps = random.Random(3), 0
    while not generator.scheduler.idle:
        drafts = {}
        for request, tokens in zip(requests, expect):
            at = len(request.generated)
            if not at or request.status != "running":
                continue
            ahead, mine, parents = tokens[at: at + rng.randint(0, 5)], [], []
            last = -1
            for token in ahead:  # a wrong branch, then the right one, then sometimes a wrong end
                mine += [rng.randrange(engine.vocab_size), token]
                parents += [last, last]
                last = len(mine) - 1
            if rng.random() < 0.5:
                mine.append(rng.randrange(engine.vocab_size))
                parents.append(last)
            drafts[request.request_id] = (mine, parents)
        before = [list(r.generated) for r in requests]
        outputs = generator.step_drafted(drafts)
        steps += 1
        for r, old in zip(requests, before):
            assert [o.token for o in outputs if o.request is r and o.token is not None] == r.generated[len(old):]
    assert [r.generated for r in requests] == expect
    assert steps < 17 and not engine.cache.requests
    engine.cache.check()


def test_drafts_end_where_generation_does(device):
    engine, _, _ = engine_for("A", device)
    prompt, more = tiny_configs.prompt(9, engine.vocab_size, 4), {"frequency_penalty": 30.0}  # (no token comes twice)
    free = Generator(engine).generate([prompt], GenerationOptions(max_tokens=12, stop=(), **more))[0]
    at = next(i for i in range(3, 12) if free[i] not in free[:i])
    for limit, expect, reason in ((12, free[:at], "stop"), (at, free[:at], "length")):
        generator = Generator(engine)
        request = generator.add(prompt, GenerationOptions(max_tokens=limit, stop=(free[at],), **more))
        while not generator.scheduler.idle:
            done = len(request.generated)
            generator.step_drafted({request.request_id: (free[done: done + 9], None)})  # a chain of what comes
        assert request.generated == expect and request.finish_reason == reason
    engine.cache.check()


def test_drafts_are_left_aside_where_pages_are_short(device):
    engine, _, _ = engine_for("A", device, cache_tokens=24, max_requests=2)
    prompt = tiny_configs.prompt(9, engine.vocab_size, 4)
    expect = Generator(engine).generate([prompt], GenerationOptions(max_tokens=14, stop=()))[0]
    generator = Generator(engine)
    request = generator.add(prompt, GenerationOptions(max_tokens=14, stop=()))
    while not generator.scheduler.idle:
        at = len(request.generated)
        generator.step_drafted({request.request_id: (expect[at: at + 2] + [1] * 12, None)})
    assert request.generated == expect
    engine.cache.check()


def test_drafts_that_are_refused(device):
    engine, _, _ = engine_for("A", device)
    generator = Generator(engine)
    request = generator.add(tiny_configs.prompt(9, engine.vocab_size, 4), GenerationOptions(max_tokens=14, stop=()))
    generator.step_drafted({})
    for drafts in (([engine.vocab_size], None), ([-1], None), ([1, 2], [-1]), ([1, 2], [-1, 1]), ([1], [-2]), ([1] * 256, None)):
        with pytest.raises(ValueError, match="drafts"):
            generator.step_drafted({request.request_id: drafts})
    assert generator.step_drafted({request.request_id: ([1] * 255, None)}) and request.status == "running"
    generator.abort(request.request_id)


def test_a_rule_is_asked_only_about_what_it_let_come(device):
    """A rule that knows no other texts than its own, and nothing that may follow some of them."""
    engine, _, _ = engine_for("A", device)
    prompt, asked = tiny_configs.prompt(9, engine.vocab_size, 4), []

    def rule(made):
        asked.append(list(made))
        for i, token in enumerate(made):
            if token % 3 != i % 3:
                raise KeyError(token)
        return [] if made and made[-1] < 30 else {t for t in range(engine.vocab_size) if t % 3 == len(made) % 3}

    high = {t: -math.inf for t in range(30)}  # (nothing that ends is ever chosen)
    for stop_at in (None, 4):
        options = GenerationOptions(max_tokens=10, stop=(), bias=high, constraint=rule)
        expect = Generator(engine).generate([prompt], options)[0]
        if stop_at is not None:
            options = GenerationOptions(max_tokens=10, stop=(expect[stop_at],), bias=high, constraint=rule)
            expect = Generator(engine).generate([prompt], options)[0]
        asked.clear()
        generator, steps = Generator(engine), 0
        request = generator.add(prompt, options)
        while not generator.scheduler.idle:
            at = len(request.generated)
            ahead = expect[at: at + 3] + list(options.stop)
            mine, parents, last = [], [], -1
            for token in ahead:  # one that the rule does not let come and what goes on from it, one that nothing follows, the right one
                depth = at + len(parents) // 4
                mine += [token + 1, token, depth % 3, token]
                parents += [last, len(mine) - 4, last, last]
                last = len(mine) - 1
            generator.step_drafted({request.request_id: (mine, parents)})
            steps += 1
        assert request.generated == expect and steps < len(expect) and request.finish_reason == ("length" if stop_at is None else "stop")
        assert not any(t in options.stop for made in asked for t in made) and max(map(len, asked)) < 10
    engine.cache.check()


def test_refused_drafts_lose_nothing(device):
    """A step in flight is still to come, and the tokens are what they would have been."""
    engine, _, _ = engine_for("A", device)
    prompt = tiny_configs.prompt(9, engine.vocab_size, 4)
    expect = Generator(engine).generate([prompt], GenerationOptions(max_tokens=9, stop=()))[0]
    generator, got = Generator(engine), []
    request = generator.add(prompt, GenerationOptions(max_tokens=9, stop=()))
    for _ in range(3):
        got += generator.step()
    with pytest.raises(ValueError, match="drafts"):
        generator.step_drafted({request.request_id: ([1, 2], [0, 0])})
    while not generator.scheduler.idle:
        got += generator.step_drafted({request.request_id: ([1, 2], None)})
    assert [o.token for o in got if o.token is not None] == request.generated == expect
    engine.cache.check()


def test_what_waits_for_drafts_to_be_kept(device):
    engine, _, _ = engine_for("A", device)
    request = engine.cache.open("r")
    entries = [StepEntry(request, [1, 2], [0, 1], [-1, 0])]
    engine.runner.run(entries)
    with pytest.raises(ValueError, match="kept"):
        engine.runner.run([StepEntry(request, [1])])
    with pytest.raises(CacheError, match="kept"):
        engine.cache.resize(64)
    engine.cache.close("r")
    engine.cache.open("r")  # another request of that name
    with pytest.raises(ValueError, match="ended"):
        engine.runner.keep(entries, chosen_on(device, [1, 1]))
    engine.cache.check()


def test_a_rule_that_fails_ends_its_step(device):
    engine, _, _ = engine_for("A", device)
    prompt = tiny_configs.prompt(5, engine.vocab_size, 4)
    for rule in (lambda made: [] if made else None, lambda made: [engine.vocab_size] if made else None):
        generator = Generator(engine)
        with pytest.raises(ValueError, match="constraint"):
            generator.generate([prompt], GenerationOptions(max_tokens=3, stop=(), constraint=rule))
        generator = Generator(engine)
        request = generator.add(prompt, GenerationOptions(max_tokens=3, stop=(), constraint=rule))
        generator.step_drafted({})
        with pytest.raises(ValueError, match="constraint"):
            generator.step_drafted({request.request_id: ([1, 2], None)})
        assert request.status == "finished" and not engine.cache.requests
    engine.cache.check()


def test_a_step_that_fails_loses_no_output(device, monkeypatch):
    """Of the step in flight ahead of it, in which one request ended."""
    engine, _, _ = engine_for("A", device)
    prompts, options = [tiny_configs.prompt(n, engine.vocab_size, n) for n in (5, 7)], [GenerationOptions(max_tokens=n, stop=()) for n in (2, 9)]
    expect = [Generator(engine).generate([p], o)[0] for p, o in zip(prompts, options)]
    for failing in ("run", "keep"):
        generator = Generator(engine)
        generator.pipelined = False
        requests = [generator.add(p, o) for p, o in zip(prompts, options)]
        assert len(generator.step()) == 2
        generator._in_flight = generator._launch(generator.scheduler.plan())
        with monkeypatch.context() as patch:
            patch.setattr(engine.runner.drafted, failing, lambda *a, **k: (_ for _ in ()).throw(RuntimeError("no more")))
            with pytest.raises(RuntimeError, match="no more"):
                generator.step_drafted({requests[1].request_id: ([1, 2], None)})
        assert requests[1].status == "finished" and requests[1].finish_reason == "abort"
        outputs = generator.drain()
        assert [(o.request, o.token, o.finished) for o in outputs] == [(requests[0], expect[0][1], True), (requests[1], expect[1][1], False)]
        assert not generator.drain() and not generator.step() and not engine.cache.requests
    # ... and what is handed out by the next step.
    generator = Generator(engine)
    generator.pipelined = False
    first, second = (generator.add(p, o) for p, o in zip(prompts, options))
    generator.step()
    generator._in_flight = generator._launch(generator.scheduler.plan())
    with monkeypatch.context() as patch:
        patch.setattr(engine.runner.drafted, "run", lambda *a, **k: (_ for _ in ()).throw(RuntimeError("no more")))
        with pytest.raises(RuntimeError, match="no more"):
            generator.step_drafted({})
    third = generator.add(prompts[0], options[0])
    assert [(o.request, o.token) for o in generator.step()] == [(first, expect[0][1]), (second, expect[1][1]), (third, expect[0][0])]
    generator.run()
    engine.cache.check()


RULES = {"nothing": lambda made: [] if len(made) == 3 else None, "no token": lambda made: [10 ** 6] if len(made) == 3 else None,
         "an error": lambda made: {}["gone"] if len(made) == 3 else range(400), "no ids": lambda made: ["x"] if len(made) == 3 else None}


@pytest.mark.parametrize("which", list(RULES))
@pytest.mark.parametrize("drafted", [False, True])
def test_a_rule_that_fails_ends_its_own_request_alone(device, which, drafted):
    """The others have the tokens that they would have had, none of which is lost."""
    engine, _, _ = engine_for("A", device)
    prompts = [tiny_configs.prompt(n, engine.vocab_size, n) for n in (5, 9, 12)]
    options = [GenerationOptions(max_tokens=8, stop=(), sampler=sampler(temperature(0.8), seed=3), frequency_penalty=0.2),
               GenerationOptions(max_tokens=8, stop=(), constraint=RULES[which]), GenerationOptions(max_tokens=8, stop=())]
    expect = [Generator(engine).generate([p], o)[0] if o.constraint is None else None for p, o in zip(prompts, options)]
    generator, outputs, errors = Generator(engine), [], []
    requests = [generator.add(p, o) for p, o in zip(prompts, options)]
    while not generator.scheduler.idle or generator._in_flight is not None:
        drafts = {r.request_id: (e[len(r.generated): len(r.generated) + 2], None) for r, e in zip(requests, expect) if e is not None and r.generated}
        try:
            outputs += generator.step_drafted(drafts) if drafted else generator.step()
        except Exception as error:  # noqa: BLE001
            errors.append(error)
    outputs += generator.drain()
    assert [r.generated for r in requests[::2]] == expect[::2] and [r.finish_reason for r in requests] == ["length", "abort", "length"]
    assert errors == [requests[1].error] and len(requests[1].generated) == 3 and requests[0].error is None and requests[2].error is None
    for r in requests:
        mine = [o for o in outputs if o.request is r]
        assert [o.token for o in mine if o.token is not None] == r.generated
        assert [o.finished for o in mine] == [False] * (len(mine) - 1) + [True]
    assert not engine.cache.requests and not generator._seeds
    engine.cache.check()


def test_a_rule_that_fails_is_its_callers(device):
    """`generate` and streams beside a request whose rule fails go on; its own stream, and the call that it belongs to, raise the error."""
    engine, _, _ = engine_for("A", device)
    prompts = [tiny_configs.prompt(n, engine.vocab_size, n) for n in (5, 9, 12)]
    plain, wrong = GenerationOptions(max_tokens=6, stop=()), GenerationOptions(max_tokens=6, stop=(), constraint=RULES["an error"])
    expect = Generator(engine).generate(prompts[::2], plain)
    generator = Generator(engine)
    odd = generator.add(prompts[1], wrong)
    assert generator.generate(prompts[::2], plain) == expect
    assert isinstance(odd.error, KeyError) and odd.status == "finished"
    bystander = generator.add(prompts[2], plain)
    late = [r for r in generator.scheduler.waiting]
    with pytest.raises(KeyError):
        generator.generate(prompts[:2], wrong)
    assert late == [bystander] and bystander.status == "running" and generator.scheduler.running == [bystander] and not generator.scheduler.waiting
    generator.run()
    assert bystander.generated == expect[1]
    model = LanguageModel(engine)
    streams = [model.stream(prompts[0], plain), model.stream(prompts[1], wrong)]
    first, second = [next(streams[0]).token_id], []
    with pytest.raises(KeyError):
        while True:
            second.append(next(streams[1]).token_id)  # (takes the steps of both)
    with pytest.raises(StopIteration):
        while True:
            next(streams[0])
    assert model.generator.scheduler.idle and first == expect[0][:1]
    streams = [model.stream(prompts[1], wrong), model.stream(prompts[0], plain)]
    next(streams[0])
    assert [s.token_id for s in streams[1] if s.token_id >= 0] == expect[0]
    with pytest.raises(KeyError):
        list(streams[0])
    assert not engine.cache.requests
    engine.cache.check()


def test_a_rule_that_fails_at_a_draft_fails_when_it_comes(device):
    """A draft of a text that the rule fails at is left aside: the tokens and the end are those of steps without drafts."""
    engine, _, _ = engine_for("A", device)
    prompt = tiny_configs.prompt(9, engine.vocab_size, 4)
    free = Generator(engine).generate([prompt], GenerationOptions(max_tokens=8, stop=()))[0]
    never = next(t for t in range(engine.vocab_size) if t not in free)
    for rule in (lambda made: {}["gone"] if never in made else None, lambda made: [-1] if never in made else None):
        generator = Generator(engine)
        request = generator.add(prompt, GenerationOptions(max_tokens=8, stop=(), constraint=rule))
        while not generator.scheduler.idle:
            at = len(request.generated)
            ahead = free[at: at + 2]  # (as many as there are)
            generator.step_drafted({request.request_id: ([never, 5, *ahead], [-1, 0, -1, 2][: 2 + len(ahead)])} if at else {})
        assert request.generated == free and request.error is None
    engine.cache.check()


def test_options_on_logits_by_their_definition(device):
    """Greedy choices, redrawn from the plain implementation's logits."""
    engine, raw, weights = engine_for("B", device)
    prompt = tiny_configs.prompt(13, engine.vocab_size, 6)
    rule = lambda made: [t for t in range(engine.vocab_size) if t % 5 != len(made) % 5]  # noqa: E731
    options = GenerationOptions(max_tokens=12, stop=(), penalty=repetition_penalty(1.3, context=9), frequency_penalty=0.4, presence_penalty=-0.2,
                                bias={5: 3.0, 700: 1.0, 2: -math.inf}, constraint=rule)
    got = Generator(engine).generate([prompt], options)[0]
    for i, token in enumerate(got):
        z = plain_impl.forward(raw, weights, prompt + got[:i])[-1:]
        text = prompt + got[:i]
        z = refs.adjust(z, [text], [len(prompt)], [1.3], [0.4], [-0.2], [9], [[(5, 3.0), (700, 1.0), (2, -math.inf)]], [rule(got[:i])])[0]
        assert token != 2 and token in rule(got[:i]) and float(z.max() - z[token]) < 1e-3


def test_options_of_one_request_leave_the_others_alone(device):
    engine, _, _ = engine_for("A", device)
    prompts = [tiny_configs.prompt(n, engine.vocab_size, n) for n in (7, 12, 9)]
    plain, odd = GenerationOptions(max_tokens=10, stop=(), penalty=repetition_penalty(1.2)), GenerationOptions(max_tokens=10, stop=(), bias={4: 100.0})
    alone = [Generator(engine).generate([p], o)[0] for p, o in zip(prompts, (plain, odd, GenerationOptions(max_tokens=10, stop=())))]
    generator = Generator(engine)
    requests = [generator.add(p, o) for p, o in zip(prompts, (plain, odd, GenerationOptions(max_tokens=10, stop=())))]
    generator.run()
    assert [r.generated for r in requests] == alone and alone[1] == [4] * 10


# -- what needs no device --------------------------------------------------------------------------------------------
def test_options_that_are_refused():
    for wrong in ({"bias": {-1: 1.0}}, {"bias": {1: math.nan}}, {"bias": {1: math.inf}}, {"frequency_penalty": math.nan}, {"presence_penalty": math.inf}):
        with pytest.raises(ValueError):
            GenerationOptions(max_tokens=1, **wrong)
    assert GenerationOptions(max_tokens=1, bias={1: -math.inf}).params().adjusts
    assert GenerationOptions(max_tokens=1).params() is GenerationOptions(max_tokens=1).sampler


def test_options_that_the_sampler_brings(device):
    """They count as the generation's own do: checked, and kept beside these."""
    for wrong in ({"bias": ((-1, 1.0),)}, {"bias": ((1, math.nan),)}, {"bias": ((1, math.inf),)}, {"frequency_penalty": math.nan}, {"presence_penalty": -math.inf}):
        with pytest.raises(ValueError):
            SamplingParams(**wrong)
    own = SamplingParams(frequency_penalty=0.5, presence_penalty=0.25, bias=((4, 100.0),))
    made = GenerationOptions(max_tokens=1, sampler=own, presence_penalty=1.0).params()
    assert (made.frequency_penalty, made.presence_penalty, made.bias) == (0.5, 1.0, ((4, 100.0),))
    engine, _, _ = engine_for("A", device)
    generator, prompt = Generator(engine), tiny_configs.prompt(5, engine.vocab_size, 4)
    for options in ({"sampler": SamplingParams(bias=((engine.vocab_size, 1.0),))}, {"bias": {engine.vocab_size: 1.0}}):
        with pytest.raises(ValueError, match="outside the vocabulary"):
            generator.add(prompt, GenerationOptions(max_tokens=2, stop=(), **options))
    assert generator.scheduler.idle
    assert generator.generate([prompt], GenerationOptions(max_tokens=3, stop=(), sampler=SamplingParams(bias=((4, 100.0),)))) == [[4] * 3]


def test_a_repetition_penalty_that_sees_nothing(device):
    """A context of no tokens: beside other penalties and with drafts it does what it does by itself."""
    engine, _, _ = engine_for("A", device)
    prompt = tiny_configs.prompt(5, engine.vocab_size, 4)
    blind = SamplingParams(repetition_penalty=50.0, penalty_context=0)
    for more in ({}, {"frequency_penalty": 1e-3}):
        expect = Generator(engine).generate([prompt], GenerationOptions(max_tokens=8, stop=(), **more))[0]
        options = GenerationOptions(max_tokens=8, stop=(), sampler=blind, **more)
        assert Generator(engine).generate([prompt], options)[0] == expect
        generator = Generator(engine)
        request = generator.add(prompt, options)
        while not generator.scheduler.idle:
            at = len(request.generated)
            generator.step_drafted({request.request_id: (expect[at: at + 3], None)} if at else {})
        assert request.generated == expect


def test_the_text_that_penalties_go_by():
    prompt, made = list(range(100, 110)), [1, 2, 3]
    assert text_of(SamplingParams(), prompt, made).tokens == []
    text = text_of(SamplingParams(frequency_penalty=1.0), prompt, made)
    assert (text.tokens, text.prompt) == (made, 0)
    text = text_of(SamplingParams(repetition_penalty=1.2, penalty_context=5), prompt, made)
    assert (text.tokens, text.prompt) == ([108, 109, 1, 2, 3], 2)
    text = text_of(SamplingParams(repetition_penalty=1.2, penalty_context=2, presence_penalty=1.0), prompt, made)
    assert (text.tokens, text.prompt) == (made, 0)
    text = text_of(SamplingParams(repetition_penalty=1.2, penalty_context=2), prompt, made)
    assert (text.tokens, text.prompt) == ([2, 3], 0)
    text = text_of(SamplingParams(repetition_penalty=1.2, penalty_context=50), prompt, [])
    assert (text.tokens, text.prompt) == (prompt, 10)
    assert allowed_ids(SamplingParams(), []) is None
    with pytest.raises(ValueError):
        allowed_ids(SamplingParams(constraint=lambda made: []), [])


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype)


def test_tables_that_are_refused():
    good = {"held": ints([3]), "brought": ints([2]), "lists": [ops.PageLists(ints([1, 2]), ints([0], torch.int64), 2)], "page_size": 4, "tokens": 2}
    for wrong in ({"held": ints([3], torch.int64)}, {"held": ints([[3]])}, {"brought": ints([1, 2])}, {"held": ints([]), "brought": ints([])},
                  {"held": ints([1, 2, 3, 4])[::2], "brought": ints([1, 1])}, {"page_size": 0}, {"tokens": -1}, {"parents": ints([-1, 0])},
                  {"parents": ints([-1]), "most": 2}, {"most": 0}, {"most": 257}, {"lists": good["lists"] * 9},
                  {"lists": [ops.PageLists(ints([1], torch.int64), ints([0], torch.int64), 2)]}, {"lists": [ops.PageLists(ints([1]), ints([0]), 2)]},
                  {"lists": [ops.PageLists(ints([1]), ints([0, 1], torch.int64), 2)]}, {"lists": [ops.PageLists(ints([1]), ints([0], torch.int64), 0)]},
                  {"lists": [ops.PageLists(ints([1]), ints([0], torch.int64), 1, 0)]},
                  {"lists": [ops.PageLists(ints([1]), ints([0], torch.int64), 1, 2)], "most": 2}, {}):  # the last: on the CPU
        with pytest.raises(ops.KernelError):
            ops.step_tables(**good | wrong)


def test_attention_of_trees_that_is_refused():
    def step(**more):
        given = {"num_tokens": 2, "num_seqs": 1, "token_ids": ints([0, 0]), "positions": ints([3, 4]), "cu_seqlens": ints([0, 2]), "seq_lens": ints([5]),
                 "state_slots": ints([0]), "fresh": ints([0]), "logit_rows": ints([]), "q_lens": [2], "seq_lens_host": [5], "max_q_len": 2, "max_seq_len": 5,
                 "decode_only": False, "groups": {}, "tree": ops.StepTree(ints([[1], [3]]))}
        return StepContext(**given | more)

    spec = KVSpec.keys_and_values(2, 8)
    view = lambda **more: KVView(**{"pages": torch.zeros(3, 2, 2, 4, 8), "block_table": ints([[0, 1]]), "slot_mapping": ints([3, 4], torch.int64),  # noqa: E731
                                    "page_size": 4, "window": None, "spec": spec} | more)
    good = {"q": torch.zeros(2, 4, 8), "kv": view(), "step": step(), "scale": 0.3}
    for wrong in ({"step": step(tree=None)}, {"q": torch.zeros(2, 32)}, {"q": torch.zeros(4, 2, 8).transpose(0, 1)}, {"q": torch.zeros(2, 3, 8)},
                  {"q": torch.zeros(2, 4, 6)}, {"q": torch.zeros(2, 4, 8, dtype=torch.bfloat16)}, {"q": torch.zeros(2, 4, 8, dtype=torch.float16)},
                  {"step": step(tree=ops.StepTree(ints([[1]])))}, {"step": step(tree=ops.StepTree(ints([1, 3])))},
                  {"step": step(tree=ops.StepTree(ints([[1], [3]], torch.int64)))}, {"step": step(max_q_len=33)}, {"step": step(max_q_len=0)},
                  {"step": step(tree=ops.StepTree(torch.zeros(2, 9, dtype=torch.int32)))}, {"step": step(positions=ints([3]))},
                  {"step": step(cu_seqlens=ints([0]))}, {"step": step(seq_lens=ints([5, 5]))}, {"kv": view(block_table=ints([[0, 1], [1, 2]]))},
                  {"kv": view(spec=KVSpec(((2, 8), (2, 8)), stride=2))}, {"gate": torch.zeros(2, 32)[:, ::2]}, {"gate": torch.zeros(2, 31)},
                  {"gate": torch.zeros(2, 40), "gate_col": 9}, {"gate": torch.zeros(2, 40), "gate_col": -1}, {"gate": torch.zeros(3, 40)},
                  {"gate": torch.zeros(2, 40, dtype=torch.bfloat16)}, {"sink": torch.zeros(3)}, {"sink": torch.zeros(4, dtype=torch.bfloat16)},
                  {"window": 4, "keep_first": 1, "chunk": 4}, {"window": -2}, {"window": 4, "keep_first": -1}, {"chunk": -4}, {}):  # the last: on the CPU
        with pytest.raises(ops.KernelError):
            ops.tree_attention(**good | wrong)
    with pytest.raises(ops.KernelError, match="difference"):
        ops.paged_attention(good["q"], good["kv"], good["step"], 0.3, difference=ops.MapDifference(0.1, 1e-5, 1.0, 8))


def test_adjustments_that_are_refused():
    history = ops.TokenHistory(ints([1, 2, 3]), ints([0, 1], torch.int64), ints([1, 2]), ints([0, 0]))
    ones, logits = torch.ones(2), torch.zeros(2, 40)
    tree = ops.StepTree(ints([[1], [3]]))
    drafted = ops.DraftedRows(tree, ints([4, 5]), ints([0, 1, 2]), ints([0, 1]))
    good = {"logits": logits, "history": history, "repetition": ones}
    other = torch.zeros(4, 40)
    for wrong in ({"logits": logits.double()}, {"logits": logits[0]}, {"logits": torch.zeros(40, 2).t()}, {"logits": torch.zeros(1, 40).expand(2, 40)},
                  {"history": None}, {"repetition": torch.ones(3)}, {"repetition": ones.double()}, {"frequency": ints([1, 1])}, {"contexts": ones},
                  {"history": history._replace(tokens=ints([1], torch.int64))}, {"history": history._replace(starts=ints([0, 1]))},
                  {"history": history._replace(prompts=ints([0]))}, {"logits": torch.zeros(3, 40)}, {"requests": ints([0])},
                  {"requests": ints([0, 1], torch.int64)}, {"bias": ops.LogitBias(ints([1]), torch.ones(2), ints([0, 1, 1]))},
                  {"bias": ops.LogitBias(ints([1]), torch.ones(1), ints([0, 1]))}, {"masks": ops.TokenMasks(ints([[1]]), ints([0, 0]))},
                  {"masks": ops.TokenMasks(ints([[1, 1]]), ints([0]))}, {"masks": ops.TokenMasks(ints([1, 1]), ints([0, 0]))}, {"drafted": drafted},
                  {"drafted": drafted._replace(rows=ints([0])), "requests": ints([0, 1])}, {"drafted": drafted._replace(cu_seqlens=ints([0, 2])), "requests": ints([0, 1])},
                  {"drafted": drafted._replace(token_ids=ints([4])), "requests": ints([0, 1])}, {"out": torch.zeros(2, 41)}, {"out": torch.zeros(2, 40).double()},
                  {"logits": other[:2], "out": other[1:3]}, {"out": torch.zeros(40, 2).t()}, {"out": torch.zeros(1, 40).expand(2, 40)}, {}):  # the last: on the CPU
        with pytest.raises(ops.KernelError):
            ops.adjust_logits(**good | wrong)


def test_acceptance_that_is_refused():
    tree = ops.StepTree(ints([[1], [3]]))
    good = {"chosen": ints([4, 5]), "token_ids": ints([4, 5]), "tree": tree, "cu_seqlens": ints([0, 2])}
    for wrong in ({"chosen": ints([4])}, {"token_ids": ints([4, 5], torch.int64)}, {"tree": ops.StepTree(ints([1, 3]))}, {"cu_seqlens": ints([0])},
                  {"tree": ops.StepTree(torch.zeros(2, 9, dtype=torch.int32))}, {"tree": ops.StepTree(torch.zeros(2, 0, dtype=torch.int32))}, {}):
        with pytest.raises(ops.KernelError):
            ops.accept_drafts(**good | wrong)
    accepted = ops.Accepted(ints([[0, -1]]), ints([1]), ints([4]))
    keep = {"pages": torch.zeros(2, 3, 2, 1, 4, 8), "rows": ((1, 8), (1, 8)), "page_size": 4, "block_table": ints([[0, 1]]), "held": ints([3]), "accepted": accepted}
    for wrong in ({"rows": ((1, 8),)}, {"rows": ((1, 16), (0, 0))}, {"page_size": 3}, {"pages": torch.zeros(2, 3, 2, 1, 8, 4).transpose(4, 5)}, {"pages": torch.zeros(4)},
                  {"block_table": ints([0, 1])}, {"held": ints([3, 3])}, {"accepted": accepted._replace(kept=ints([1, 1]))},
                  {"accepted": accepted._replace(path=torch.zeros(1, 257, dtype=torch.int32))}, {"accepted": accepted._replace(path=ints([0, -1]))}, {}):
        with pytest.raises(ops.KernelError):
            ops.keep_rows(**keep | wrong)
