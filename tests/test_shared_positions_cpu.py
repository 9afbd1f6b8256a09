"""Requests that share their first positions, without a GPU: forks and resizing of the cache, what the
scheduler does with followers, the lists that the attention kernels read, and answers to one prompt."""

from __future__ import annotations

import dataclasses
import math
import random
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import plain_impl
import tiny_configs
from mlx_omnia_b200 import GenerationOptions, sampler, temperature
from mlx_omnia_b200.cache import CacheError, CacheManager, PagePool
from mlx_omnia_b200.engine.engine import Engine, EngineArgs
from mlx_omnia_b200.engine.generate import Generator, LanguageModel, common_start
from mlx_omnia_b200.engine.scheduler import Request, Scheduler
from mlx_omnia_b200.engine.step import StepEntry, shared_positions
from mlx_omnia_b200.kernels import ops
from mlx_omnia_b200.parts.base import KVSpec, KVView, StateSpec, StepContext
from mlx_omnia_b200.parts.model import CacheNeed

FULL, WINDOW = KVSpec.keys_and_values(2, 4, None), KVSpec.keys_and_values(2, 4, 10)
UNEQUAL, STRIDED = KVSpec(((2, 6), (2, 4))), KVSpec(((1, 3),), stride=3)


def manager(specs=(FULL, WINDOW), state=False, pages=24, page_size=4, max_requests=6, allocate=True):
    needs = [CacheNeed(spec, StateSpec((3,)) if state else None, None) for spec in specs]
    return CacheManager(needs, page_size=page_size, pages_per_group=pages, max_requests=max_requests, dtype=torch.float32, allocate=allocate)


def write(cache, request, count, mark):
    """What a step does to the cache: positions start .. start + count get rows that name `mark` and their position."""
    start = request.tokens
    cache.grow(request, count)
    for g, group in enumerate(cache.groups):
        for position in range(start, start + count):
            slot = cache.slot_of(request, g, position)
            page, row = divmod(slot, cache.page_size)
            at = 0
            flat = group.pages[:, page].flatten(1)
            for heads, width in group.spec.rows:
                flat[:, at: at + heads * cache.page_size * width].view(-1, heads, cache.page_size, width)[:, :, row] = 1000 * mark + position
                at += heads * cache.page_size * width
    for tensor, _ in cache.state_tensors():
        tensor[request.slot] = 1000 * mark + start + count
    request.fresh = False
    cache.release_behind_window(request)


def held(cache, request, group, position):
    group_, row = cache.groups[group], position // cache.groups[group].spec.stride
    page = request.tables[group][row // cache.page_size]
    assert page >= 0
    flat, found, at = group_.pages[:, page].flatten(1), set(), 0
    for heads, width in group_.spec.rows:
        size = heads * cache.page_size * width
        found |= set(flat[:, at: at + size].view(-1, heads, cache.page_size, width)[:, :, row % cache.page_size].flatten().tolist())
        at += size
    assert len(found) == 1
    return found.pop()


# -- the cache -----------------------------------------------------------------------------------------------------
def test_a_shared_page_is_free_after_its_last_reference():
    pool = PagePool(2)
    page = pool.take()
    pool.share(page)
    pool.give(page)
    assert pool.held() == [page] and pool.free == 1
    pool.give(page)
    assert pool.free == 2
    with pytest.raises(CacheError, match="twice"):
        pool.give(page)
    with pytest.raises(CacheError, match="cannot be shared"):
        pool.share(page)


@pytest.mark.parametrize("specs,state", [((FULL,), False), ((FULL, WINDOW), False), ((FULL, UNEQUAL), True), ((STRIDED, FULL), False)])
@pytest.mark.parametrize("positions", [1, 3, 4, 5, 8, 9, 15, 16])
def test_a_fork_holds_what_it_forked_and_neither_writes_to_the_other(specs, state, positions):
    cache = manager(specs, state)
    a = cache.open("a")
    write(cache, a, positions, 1)
    b = cache.fork(a, "b")
    cache.check()
    assert b.tokens == positions and not b.fresh
    for g, group in enumerate(cache.groups):
        whole = positions // group.spec.stride // cache.page_size
        assert b.tables[g][:whole] == a.tables[g][:whole]
        assert len(b.tables[g]) == len(a.tables[g]) and not set(b.tables[g][whole:]) & set(a.tables[g][whole:])
        assert b.table_array(g).tolist() == b.tables[g]
    write(cache, a, 7, 1)
    write(cache, b, 5, 2)
    cache.check()
    for g, group in enumerate(cache.groups):
        if group.spec.stride > 1:  # a row goes on until it is full, and then names its last position
            continue
        for request, mark in ((a, 1), (b, 2)):
            for position in range(max(group.spec.dead_below(request.tokens), 0), request.tokens):
                assert held(cache, request, g, position) == 1000 * (1 if position < positions else mark) + position
    for tensor, _ in cache.state_tensors():
        assert set(tensor[a.slot].tolist()) == {1000.0 + positions + 7} and set(tensor[b.slot].tolist()) == {2000.0 + positions + 5}
    cache.close("a")
    cache.check()
    cache.close("b")
    cache.check()
    assert all(g.pool.free == g.pool.count for g in cache.groups) and cache.slots.free == 6


def test_forks_behind_where_the_request_stands():
    cache = manager((FULL,))
    a = cache.open("a")
    write(cache, a, 11, 1)
    b = cache.fork(a, "b", 6)
    write(cache, b, 3, 2)
    cache.check()
    assert [held(cache, b, 0, p) for p in range(9)] == [1000 + p for p in range(6)] + [2000 + p for p in range(6, 9)]
    assert [held(cache, a, 0, p) for p in range(11)] == [1000 + p for p in range(11)]
    assert a.runs == b.runs and a.runs[0].positions == 6
    c = cache.fork(a, "c", 9)  # what a and c share is longer than what all three do
    assert [r.positions for r in c.runs] == [6, 9] == [r.positions for r in a.runs] and c.runs[0] is b.runs[0]
    d = cache.fork(a, "d", 9)
    assert d.runs == c.runs


@pytest.mark.parametrize("specs,state,tokens,positions,match", [
    ((FULL,), False, 5, 0, "between 1"), ((FULL,), False, 5, 6, "between 1"), ((FULL,), True, 5, 4, "the state of"),
    ((STRIDED,), False, 8, 7, "a stored row"), ((WINDOW,), False, 40, 20, "given back")])
def test_forks_that_cannot_be(specs, state, tokens, positions, match):
    cache = manager(specs, state)
    a = cache.open("a")
    write(cache, a, tokens, 1)
    with pytest.raises(CacheError, match=match):
        cache.fork(a, "b", positions)
    assert list(cache.requests) == ["a"]
    cache.check()


def test_a_fork_takes_nothing_when_pages_or_slots_are_short():
    cache = manager((FULL,), pages=3, max_requests=2)
    a = cache.open("a")
    write(cache, a, 9, 1)  # three pages, the last of one position
    with pytest.raises(CacheError, match="needs 1 pages"):
        cache.fork(a, "b")
    cache.fork(a, "b", 8)
    with pytest.raises(CacheError, match="no free request slot"):
        cache.fork(a, "c", 8)
    cache.check()


@pytest.mark.parametrize("fails", ["rows of the first group", "rows of the second group", "state"])
def test_a_fork_whose_copy_fails_leaves_nothing_behind(fails, monkeypatch):
    cache = manager((FULL, WINDOW), state=True)
    a = cache.open("a")
    write(cache, a, 7, 1)
    tables, calls, copy = [list(t) for t in a.tables], [], CacheManager._copy_rows

    def copy_rows(self, *args):
        calls.append(1)
        if len(calls) == (1 if fails == "rows of the first group" else 2):
            raise ops.KernelError("a copy failed")
        copy(self, *args)

    def state_tensors(self):
        raise ops.KernelError("a copy failed")

    with monkeypatch.context() as patch:
        if fails == "state":
            patch.setattr(CacheManager, "state_tensors", state_tensors)
        else:
            patch.setattr(CacheManager, "_copy_rows", copy_rows)
        with pytest.raises(ops.KernelError, match="a copy failed"):
            cache.fork(a, "b")
    assert list(cache.requests) == ["a"] and cache.slots.held() == [a.slot] and a.runs == [] and a.tables == tables
    cache.check()
    b = cache.fork(a, "b")  # the name, the slot and the pages are free
    assert [held(cache, b, g, p) for g in (0, 1) for p in range(7)] == 2 * [1000 + p for p in range(7)]
    cache.check()


@pytest.mark.parametrize("positions", [7, 6])
def test_a_fork_needs_the_page_that_it_goes_on_in(positions):
    cache = manager((FULL, WINDOW))
    a = cache.open("a")
    write(cache, a, 7, 1)
    cache.groups[1].pool.give(a.tables[1][1])
    a.tables[1][1] = a.arrays[1][1] = -1
    with pytest.raises(CacheError, match="given back"):
        cache.fork(a, "b", positions)
    assert list(cache.requests) == ["a"]
    cache.check()


def test_pages_are_not_copied_between_tensors_that_overlap(monkeypatch):
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    pages, row = torch.zeros(1, 8, 2 * 2 * 8 * 4), ((2, 8), (2, 8))
    for source, to in ((pages[:, :6], pages[:, 1:7]), (pages[:, 2:], pages[:, :3]), (pages[:, :5], pages[:, 4:])):
        with pytest.raises(ops.KernelError, match="overlap"):
            ops.copy_pages(source, row, 4, [(0, 1, 4)], to=to)
    layers = torch.zeros(24, 128)
    with pytest.raises(ops.KernelError, match="overlap"):  # page 8 of one layer is page 0 of the next
        ops.copy_pages(layers[:16].view(2, 8, 128), row, 4, [(0, 1, 4)], to=layers.view(2, 12, 128))
    with pytest.raises(ops.KernelError, match="another begins"):
        ops.copy_pages(pages[:, :5], row, 4, [(0, 1, 4), (1, 2, 4)], to=pages)
    # Nothing to move: neighbours and one tensor seen twice are taken.
    assert ops.copy_pages(pages[:, :4], row, 4, [], to=pages[:, 4:]).data_ptr() == pages[:, 4:].data_ptr()
    ops.copy_pages(pages, row, 4, [], to=pages[:, :5])


@pytest.mark.parametrize("specs", [(FULL, WINDOW), (UNEQUAL, FULL)])
@pytest.mark.parametrize("pages", [9, 60])
def test_resizing_keeps_what_is_held(specs, pages):
    cache = manager(specs)
    for i, name in enumerate("abcd"):
        write(cache, cache.open(name), 5 + i, i)
    b, d = cache.requests["b"], cache.requests["d"]
    cache.close("a")
    cache.close("c")
    e = cache.fork(b, "e")
    cache.resize(pages)
    cache.check()
    assert all(g.pool.count == pages and g.pages.shape[1] == pages for g in cache.groups)
    assert all(max(g.pool.held()) == len(g.pool.held()) - 1 for g in cache.groups)
    for g in range(len(cache.groups)):
        for request, mark in ((b, 1), (d, 3), (e, 1)):
            assert request.table_array(g).tolist() == request.tables[g]
            assert [held(cache, request, g, p) for p in range(request.tokens)] == [1000 * mark + p for p in range(request.tokens)]
    write(cache, e, 4, 5)
    cache.check()
    with pytest.raises(CacheError, match="does not take"):
        cache.resize(2)
    with pytest.raises(ValueError, match="at least one"):
        cache.resize(0)
    cache.check()


def failing_at(monkeypatch, count):
    """`torch.zeros` runs out of memory at its `count`th call from here on."""
    calls, zeros = [], torch.zeros

    def fake(*args, **options):
        calls.append(1)
        if len(calls) == count:
            raise torch.OutOfMemoryError("no memory")
        return zeros(*args, **options)

    monkeypatch.setattr(torch, "zeros", fake)


@pytest.mark.parametrize("specs", [(FULL, WINDOW), (UNEQUAL, FULL, STRIDED)])
def test_a_resize_that_runs_out_of_memory_changes_nothing(specs, monkeypatch):
    cache = manager(specs)
    a = cache.open("a")
    write(cache, a, 7, 1)
    write(cache, cache.fork(a, "b"), 2, 2)

    def everything():
        return ([(g.pool.count, g.pool.held(), g.pages.data_ptr(), g.pages.clone()) for g in cache.groups],
                [(r.tokens, [list(t) for t in r.tables], [x.tolist() for x in r.arrays]) for r in cache.requests.values()])

    before = everything()
    failing_at(monkeypatch, len(specs))
    with pytest.raises(torch.OutOfMemoryError):
        cache.resize(40)
    monkeypatch.undo()
    after = everything()
    assert after[1] == before[1] and [x[:3] for x in after[0]] == [x[:3] for x in before[0]]
    assert all(torch.equal(x[3], y[3]) for x, y in zip(after[0], before[0]))
    cache.check()


def test_block_tables_of_captured_mixed_steps_are_as_wide_as_a_resized_cache():
    from mlx_omnia_b200.engine.decode_graph import MixedGraphs

    cache = manager((FULL, STRIDED), pages=10, page_size=4)
    graphs = MixedGraphs(SimpleNamespace(cache=cache))
    assert graphs.widest == [10, 4]  # 40 positions
    cache.resize(50)
    assert graphs.widest == [50, 17]
    cache.resize(3)
    assert graphs.widest == [3, 1]


@pytest.mark.parametrize("seed", range(6))
def test_random_lives_lose_no_page(seed):
    rng = random.Random(seed)
    cache = manager((FULL, WINDOW) if seed % 2 else (FULL,), pages=40, max_requests=8)
    for i in range(300):
        names = list(cache.requests)
        act = rng.random()
        try:
            if act < 0.2 or not names:
                write(cache, cache.open(f"r{i}"), rng.randint(1, 12), i)
            elif act < 0.45:
                a = cache.requests[rng.choice(names)]
                cache.fork(a, f"r{i}", rng.randint(1, a.tokens))
            elif act < 0.75:
                write(cache, cache.requests[rng.choice(names)], rng.randint(1, 6), i)
            elif act < 0.95:
                cache.close(rng.choice(names))
            else:
                cache.resize(rng.randint(30, 60))
        except CacheError:
            pass
        for request in list(cache.requests.values()):
            if request.tokens == 0:
                cache.close(request.request_id)
        cache.check()


# -- the scheduler --------------------------------------------------------------------------------------------------
def run_step(scheduler, cache):
    plan = scheduler.plan()
    for e in plan.entries:
        cache.grow(e.request.cache, e.count)
        assert e.request.cache.tokens == e.start + e.count
        e.request.cache.fresh = False
        cache.release_behind_window(e.request.cache)
    outputs = scheduler.commit(plan, {e.request.request_id: 7 for e in plan.entries if e.samples})
    cache.check()
    return [(e.request.request_id, e.start, e.count, e.samples) for e in plan.entries], outputs


def scheduled(state=False, window=False, pages=32, budget=16, max_requests=6):
    cache = manager((FULL, WINDOW) if window else (FULL,), state, pages=pages, max_requests=max_requests, allocate=False)
    return Scheduler(cache, max_tokens_per_step=budget), cache


@pytest.mark.parametrize("state,window", [(False, False), (True, True)])
def test_followers_are_forked_where_their_leader_stands(state, window):
    scheduler, cache = scheduled(state, window)
    prompt = list(range(21))
    first = Request("a", prompt, 3)
    scheduler.add(first)
    for name in "bc":
        scheduler.add(Request(name, prompt, 3, leader=first, fork_at=20))
    assert run_step(scheduler, cache)[0] == [("a", 0, 16, False)]
    assert run_step(scheduler, cache)[0] == [("a", 16, 4, False)]  # cut where its followers fork
    assert run_step(scheduler, cache)[0] == [("a", 20, 1, True), ("b", 20, 1, True), ("c", 20, 1, True)]
    entries = [StepEntry(r.cache, [0]) for r in scheduler.running]
    assert shared_positions(entries) == ((20, (0, 1, 2)),)
    assert run_step(scheduler, cache)[0] == [("a", 21, 1, True), ("b", 21, 1, True), ("c", 21, 1, True)]
    run_step(scheduler, cache)
    assert scheduler.idle and all(g.pool.free == g.pool.count for g in cache.groups)


def test_followers_read_for_themselves_when_their_leader_has_gone():
    scheduler, cache = scheduled()
    prompt = list(range(9))
    first = Request("a", prompt, 3)
    scheduler.add(first)
    scheduler.add(Request("b", prompt, 3, leader=first, fork_at=8))
    scheduler.abort("a")
    assert run_step(scheduler, cache)[0] == [("b", 0, 9, True)]


def test_a_follower_is_forked_from_another_follower_when_the_leader_has_ended():
    scheduler, cache = scheduled(max_requests=2)
    prompt = list(range(9))
    first = Request("a", prompt, 1)
    scheduler.add(first)
    for name, most in (("b", 5), ("c", 3)):
        scheduler.add(Request(name, prompt, most, leader=first, fork_at=8))
    assert run_step(scheduler, cache)[0] == [("a", 0, 8, False)]
    assert run_step(scheduler, cache)[0] == [("a", 8, 1, True), ("b", 8, 1, True)]  # two slots: c waits, a ends
    assert run_step(scheduler, cache)[0] == [("b", 9, 1, True), ("c", 8, 1, True)]


def test_a_preempted_follower_comes_back_as_a_fork():
    scheduler, cache = scheduled(pages=4, budget=32)
    prompt = list(range(9))
    first = Request("a", prompt, 7)
    second = Request("b", prompt, 7, leader=first, fork_at=8)
    scheduler.add(first)
    scheduler.add(second)
    steps = []
    while not scheduler.idle:
        steps.append(run_step(scheduler, cache)[0])
        assert len(steps) < 60
    assert second.preemptions and len(first.generated) == len(second.generated) == 7
    assert all(g.pool.free == g.pool.count for g in cache.groups)


@pytest.mark.parametrize("prompt,at", [([0, 1, 2, 3], 4), ([0, 1, 2, 3], 0), ([0, 9, 2, 3], 3), ([5, 1, 2], 1)])
def test_requests_that_cannot_follow(prompt, at):
    scheduler, _ = scheduled()
    first = Request("a", [0, 1, 2, 3, 4], 3)
    scheduler.add(first)
    with pytest.raises(ValueError, match="begins with the same tokens"):
        scheduler.add(Request("b", prompt, 3, leader=first, fork_at=at))


def test_a_leader_that_stops_for_its_follower_is_not_starved():
    """Another request is admitted while the leader waits at the fork and takes every page; neither prompt fits beside the other."""
    scheduler, cache = scheduled(pages=8, budget=64)
    first = Request("a", list(range(24)), 2)
    scheduler.add(first)
    scheduler.add(Request("b", [99] * 30, 2))
    scheduler.add(Request("c", list(range(4)) + [50, 51], 2, leader=first, fork_at=4))
    assert run_step(scheduler, cache)[0] == [("a", 0, 4, False), ("b", 0, 28, False)]
    steps = 0
    while not scheduler.idle:
        run_step(scheduler, cache)
        steps += 1
        assert steps < 30
    assert all(g.pool.free == g.pool.count for g in cache.groups)


def test_a_request_follows_one_that_was_added_before():
    scheduler, _ = scheduled()
    with pytest.raises(ValueError, match="added before"):
        scheduler.add(Request("b", [1, 2, 3], 3, leader=Request("a", [1, 2, 3], 3), fork_at=2))


@pytest.mark.parametrize("seed", range(5))
def test_random_followers_under_pressure_all_end(seed):
    rng = random.Random(seed)
    scheduler, cache = scheduled(state=seed % 2 == 0, window=seed % 3 == 0, pages=10, budget=rng.randint(1, 20), max_requests=rng.randint(2, 5))
    firsts: list[Request] = []
    for i in range(14):
        if firsts and rng.random() < 0.7:
            leader = rng.choice(firsts)
            at = rng.randint(1, len(leader.prompt))
            prompt = leader.prompt[:at] + [99] * rng.randint(1, 4)
            scheduler.add(Request(f"r{i}", prompt, rng.randint(1, 5), leader=leader, fork_at=at))
        else:
            firsts.append(Request(f"r{i}", list(range(rng.randint(2, 15))), rng.randint(1, 6)))
            scheduler.add(firsts[-1])
    steps = 0
    while not scheduler.idle:
        run_step(scheduler, cache)
        steps += 1
        assert steps < 800
    assert all(g.pool.free == g.pool.count for g in cache.groups)


# -- which entries share what, and the kernels' list ----------------------------------------------------------------
def test_entries_go_with_the_longest_run_that_another_shares():
    cache = manager((FULL,), max_requests=6)
    a = cache.open("a")
    write(cache, a, 12, 1)
    b = cache.fork(a, "b", 6)
    c, d = cache.fork(a, "c", 10), cache.fork(b, "d", 5)
    other = cache.open("x")
    write(cache, other, 3, 2)
    entries = [StepEntry(r, [0]) for r in (d, a, other, b, c)]
    assert shared_positions(entries) == ((10, (1, 4)), (5, (0, 3)))
    assert shared_positions([entries[1], entries[3]]) == ((6, (0, 1)),)
    assert shared_positions([entries[2], entries[4]]) == ()


def step_of(lengths, shared, **more):
    return StepContext(num_tokens=len(lengths), num_seqs=len(lengths), token_ids=None, positions=None, cu_seqlens=None, seq_lens=None,
                       state_slots=None, fresh=None, logit_rows=None, q_lens=[1] * len(lengths), seq_lens_host=list(lengths), max_q_len=1,
                       max_seq_len=max(lengths), decode_only=True, groups={}, shared=shared, **more)


@pytest.mark.parametrize("group,nkv,block_rows,tile,places", [(2, 3, 256, 128, 148), (4, 8, 256, 128, 148), (1, 1, 32, 32, 592), (5, 2, 250, 128, 20),
                                                              (16, 1, 256, 128, 148)])
@pytest.mark.parametrize("seed", range(4))
def test_the_list_covers_every_row_and_position_once(group, nkv, block_rows, tile, places, seed):
    rng = random.Random(100 * seed + group)
    requests = list(range(rng.randint(4, 70)))
    rng.shuffle(requests)
    shared, at = [], 0
    for _ in range(rng.randint(1, 3)):
        count = rng.randint(1, max(1, len(requests) // 3))
        shared.append((rng.choice([1, 31, 32, 33, 127, 128, 129, 1000, 5000, 70001]), tuple(requests[at: at + count])))
        at += count
    shared = tuple(shared)
    lengths = [1] * len(requests)
    for positions, members in shared:
        for m in members:
            lengths[m] = positions + rng.randint(1, 50)
    step = step_of(lengths, shared)
    plan = ops.shared_plan(ops.shared_shape(shared), group, nkv, block_rows, tile, rng.randint(1, 5), places)
    flat = ops.shared_list(step, plan, group, nkv, block_rows, tile)
    n = len(lengths)
    assert flat.dtype == np.int32 and len(flat) == 2 * n + plan.members + 8 * plan.items
    starts, parts, members = flat[:n], flat[n: 2 * n], flat[2 * n: 2 * n + plan.members]
    seen: dict = {}
    for table_of, first, row0, rows, kvh, lo, hi, part in flat[2 * n + plan.members:].reshape(-1, 8).tolist():
        if rows < 1 or lo >= hi:
            continue
        assert lo % tile == 0 and 0 <= kvh < nkv and rows <= block_rows
        for row in range(row0, row0 + rows):
            request = int(members[first + row // group])
            pieces = seen.setdefault((request, kvh, row % group), {})
            assert part not in pieces
            pieces[part] = (lo, hi)
    for positions, which in shared:
        for m in which:
            assert starts[m] == positions
            for kvh in range(nkv):
                for head in range(group):
                    pieces = seen.pop((m, kvh, head))
                    assert sorted(pieces) == list(range(parts[m])) and parts[m] <= max(plan.parts)
                    cuts = [pieces[i] for i in range(parts[m])]
                    assert cuts[0][0] == 0 and cuts[-1][1] == positions
                    assert all(x[1] == y[0] for x, y in zip(cuts, cuts[1:])) and all(x[0] < x[1] for x in cuts)
    assert not seen
    alone = set(range(n)) - {m for _, which in shared for m in which}
    assert all(starts[m] == parts[m] == 0 for m in alone)


def test_a_captured_step_takes_groups_of_about_one_size():
    shared = ((2051, (0, 1, 2, 3, 4)), (300, (5, 6)))
    shape = ops.shared_shape(shared)
    assert shape == ops.shared_shape(((2100, (7, 8, 9, 1, 2, 3, 4)), (270, (0, 5))))
    plan = ops.shared_plan(shape, 2, 2, 256, 128, 2, 148)
    empty = ops.shared_list(step_of([1] * 10, (), shared_shape=shape), plan, 2, 2, 256, 128)
    assert not empty.any() and len(empty) == len(ops.shared_list(step_of([3000] * 10, shared, shared_shape=shape), plan, 2, 2, 256, 128))
    with pytest.raises(ops.KernelError, match="another shape"):
        ops.shared_list(step_of([9000] * 10, ((8000, (0, 1)),), shared_shape=shape), plan, 2, 2, 256, 128)


@pytest.mark.parametrize("shared,match", [(((0, (0, 1)),), "at least one position"), (((3, ()),), "at least one position"),
                                          (((3, (0, 1)), (2, (1, 2))), "each in one group"), (((3, (0, 0)),), "each in one group"),
                                          (((3, (0, 9)),), "of the step's requests"), (((3, (-1, 1)),), "of the step's requests"),
                                          (((8, (0, 1)),), "more positions than it shares")])
def test_groups_that_cannot_be(shared, match):
    with pytest.raises(ops.KernelError, match=match):
        ops.check_shared(step_of([9, 8, 7], shared))


def test_where_sharing_applies():
    def applies(shared, dtype=torch.bfloat16, window=None, decode_only=True, nkv=8, d=128, page=16, nq=16, spec=None):
        step = step_of([100000] * 80, shared)
        step.decode_only = decode_only
        pages = torch.empty(1, 2, nkv, page, d, dtype=dtype, device="meta")
        return ops.shared_applies(step, SimpleNamespace(pages=pages, spec=spec, page_size=page, window=window), nq)

    eight = (4096, tuple(range(8)))
    assert applies((eight,)) and not applies(()) and not applies((eight,), window=64) and not applies((eight,), decode_only=False)
    assert not applies(((200, (0, 1)),)) and applies(((200, (0, 1)),), dtype=torch.float32)
    assert applies((eight,), d=96) and applies((eight,), page=8) and applies((eight,), nq=8 * 17)
    assert not applies((eight,), d=96, nq=8 * 9) and not applies(((200, (0, 1)),), d=96)
    assert not applies((eight,), spec=KVSpec(((8, 128), (8, 128)), chunk=64))
    assert not applies((eight,), spec=KVSpec(((8, 128), (8, 128)), stride=2))


@pytest.mark.parametrize("groups,alone,pays", [
    ([(6200, [100, 100])], [6000 - 60 * i for i in range(60)], False), ([(1000, [200] * 8)], [3000 - 90 * i for i in range(8)], False),
    ([(4000, [200] * 8)], [3000] * 56, False), ([(512, [1 + 31 * i for i in range(64)])], [], False),
    ([(2051, [1 + 11 * i for i in range(64)])], [], True), ([(4096, [256] * 8)], [], True), ([(30000, [200] * 16)], [3000] * 16, True),
    ([(6200, [10, 10])], [], True)])
def test_sharing_is_weighed_against_what_requests_hold_of_their_own(groups, alone, pays):
    """Inside of a pass, where what a step's requests hold of their own would run by a list of equal pieces."""
    lengths, shared = [], []
    for positions, owns in groups:
        shared.append((positions, tuple(range(len(lengths), len(lengths) + len(owns)))))
        lengths += [positions + own for own in owns]
    lengths += alone
    step = step_of(lengths, tuple(shared))
    pages = torch.empty(1, 2, 8, 16, 128, dtype=torch.bfloat16, device="meta")
    kv = SimpleNamespace(pages=pages, spec=None, page_size=16, window=None)
    assert ops.shared_applies(step, kv, 16)
    ops.begin_pass(step)
    assert ops.shared_applies(step, kv, 16) == pays
    # A captured step of such numbers decides alike.
    batch = 1 << (len(lengths) - 1).bit_length()
    own = ops.own_bucket(max([own for _, owns in groups for own in owns] + alone), 16)
    captured = step_of([0] * batch, (), shared_shape=ops.shared_shape(shared), max_own=own)
    captured.seq_lens_host = []
    ops.begin_pass(captured)
    gain = ops.sharing_gain(ops.attention_layer(kv, 16), ops.shared_shape(shared), len(lengths), own)
    assert ops.shared_applies(captured, kv, 16) == pays == (gain >= 0)
    # Other types and widths have no list.
    pages = torch.empty(1, 2, 8, 16, 128, device="meta")
    assert ops.shared_applies(step, SimpleNamespace(pages=pages, spec=None, page_size=16, window=None), 16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_every_call_reads_the_lengths_and_the_list_of_its_own_step(dtype, monkeypatch):
    """Steps that share a workspace (`dataclasses.replace`) keep plans and scratch memory with it, and no tensor of one another's."""
    calls = []

    def function(library, name, argtypes, defines=None):
        def run(at, *rest):
            if not calls or calls[-1] is not at:
                calls.append(at)
            return 0

        return run

    monkeypatch.setattr(ops, "_function", function)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops, "sm_count", lambda device: 148)
    monkeypatch.setattr(ops, "error_word", lambda device: torch.zeros(1, dtype=torch.int32))
    monkeypatch.setattr(ops, "SHARED_LEAST_BYTES", 0)
    monkeypatch.setattr(ops, "_ints_to_device", lambda values, device: torch.as_tensor(values))

    def ints(values):
        return torch.tensor(values, dtype=torch.int32)

    step = step_of([300, 280, 290], ((256, (0, 1, 2)),))
    step.cu_seqlens, step.seq_lens = ints([0, 1, 2, 3]), ints([300, 280, 290])
    spec = KVSpec.keys_and_values(2, 64, None)
    kv = KVView(torch.zeros(64, 2, 2, 16, 64, dtype=dtype), ints([[0] * 20] * 4), torch.zeros(4, dtype=torch.int64), 16, None, spec=spec)

    def run(step):
        q = torch.zeros(step.num_seqs, 4, 64, dtype=dtype)
        ops.paged_attention(q, kv, step, 0.1)
        args = calls[-1]._obj
        assert (args.cu_seqlens, args.seq_lens) == (step.cu_seqlens.data_ptr(), step.seq_lens.data_ptr()) and args.requests == step.num_seqs
        held = next(call for call in step.workspace.values() if isinstance(call, ops._SharedCall) and call.args is args).held[0]
        assert args.plan == held.data_ptr()
        return held.tolist()

    first = run(step)
    other = dataclasses.replace(step, seq_lens=ints([299, 279, 289]), cu_seqlens=ints([0, 1, 2, 3]))
    assert other.workspace is step.workspace and run(other) == first and run(step) == first
    more = dataclasses.replace(step, num_seqs=4, num_tokens=4, cu_seqlens=ints([0, 1, 2, 3, 4]), seq_lens=ints([300, 280, 290, 5]))
    assert run(more)[:8] == [256, 256, 256, 0, *first[3:6], 0]
    # Lengths that the host does not know: what the step is laid out for follows from its bound.
    for longest in (300, 1200):
        run(dataclasses.replace(step, seq_lens_host=[], max_seq_len=longest))
        args = calls[-1]._obj
        assert args.max_chunks * args.chunk_keys >= longest


class Planned(Exception):
    pass


@pytest.mark.parametrize("positions,members,alone,windowed,pays", [(300, 4, 3, False, False), (4096, 8, 0, False, True), (4096, 8, 0, True, False),
                                                                   (40000, 2, 1, False, True)])
def test_a_captured_step_has_no_groups_where_no_layer_reads_them_once(positions, members, alone, windowed, pays, monkeypatch):
    """What a step is kept by is decided ahead of its capture: where no layer gains by groups, by what the same step without them is."""
    from mlx_omnia_b200.engine import decode_graph
    from mlx_omnia_b200.engine.decode_graph import DecodeGraphs

    monkeypatch.setattr(decode_graph, "CAPTURE_GAINS", 0)
    spec = KVSpec.keys_and_values(8, 128, None)
    cache = manager((spec,), pages=6000, page_size=16, max_requests=16, allocate=False)
    leader = cache.open("leader")
    cache.grow(leader, positions)
    requests = [leader] + [cache.fork(leader, f"f{i}") for i in range(members - 1)] + [cache.open(f"a{i}") for i in range(alone)]
    for request in requests[members:]:
        cache.grow(request, 50)
    runner = SimpleNamespace(cache=cache, attention_layers={ops.AttentionLayer(16, 8, 128, 128, torch.bfloat16, 16, not windowed): 1},
                             take_pages=lambda entries: [e.request.tokens for e in entries])
    graphs, keys = DecodeGraphs(runner), []

    def graph_for(*key):
        keys.append(key)
        raise Planned

    monkeypatch.setattr(graphs, "_graph_for", graph_for)
    entries = [StepEntry(r, [1], [0]) for r in requests]
    with pytest.raises(Planned):
        graphs.run(entries)
    batch, width = 1 << (len(requests) - 1).bit_length(), ops.width_bucket(-(-positions // 16))
    shape = ops.shared_shape(shared_positions(entries))
    assert keys == [(batch, width, shape, ops.own_bucket(51 if alone else 1, 16)) if pays else (batch, width)]


def test_a_shape_of_groups_is_captured_when_its_steps_are_worth_it(monkeypatch):
    from mlx_omnia_b200.engine.decode_graph import CAPTURE_GAINS, DecodeGraphs

    cache = manager((KVSpec.keys_and_values(8, 128, None),), pages=6000, page_size=16, max_requests=16, allocate=False)
    layer = ops.AttentionLayer(16, 8, 128, 128, torch.bfloat16, 16, True)
    graphs, keys = DecodeGraphs(SimpleNamespace(cache=cache, attention_layers={layer: 1}, take_pages=lambda entries: [e.request.tokens for e in entries])), []

    def graph_for(*key):
        keys.append(key)
        graphs.captured[key] = None
        raise Planned

    monkeypatch.setattr(graphs, "_graph_for", graph_for)

    def steps(entries, count):
        del keys[:]
        for _ in range(count):
            with pytest.raises(Planned):
                graphs.run(entries)
        return [len(key) > 2 for key in keys]

    leader = cache.open("leader")
    cache.grow(leader, 16000)
    entries = [StepEntry(r, [1], [0]) for r in [leader] + [cache.fork(leader, f"f{i}") for i in range(7)]]
    shape = ops.shared_shape(shared_positions(entries))
    gain = ops.sharing_gain(layer, shape, 8, ops.own_bucket(1, 16))
    first = math.ceil(CAPTURE_GAINS * ops.SHARED_LEAST_BYTES / gain)
    assert 10 < first < 100
    assert steps(entries, 3 * first) == [False] * (first - 1) + [True] * (2 * first + 1)
    # What the shape has gained since pays for the graph of the next bound of what requests hold of their own.
    for entry in entries:
        cache.grow(entry.request, 200)
    assert steps(entries, 2) == [True, True]
    # Another shape has an account of its own.
    assert steps(entries[:4], 2) == [False, False]
    graphs.gained |= {i: 1.0 for i in range(5000)}
    steps(entries, 1)
    assert len(graphs.gained) == 1


# -- answers ----------------------------------------------------------------------------------------------------------
def engine_for(name, cache_tokens=256, page_size=4, max_requests=4):
    raw, weights = tiny_configs.config(name), tiny_configs.tensors(name)
    args = EngineArgs(dtype="float32", page_size=page_size, cache_tokens=cache_tokens, max_requests=max_requests, device="cpu")
    return Engine.from_tensors(raw, weights, args), raw, weights


@pytest.mark.parametrize("prompts,start", [([[1, 2, 3], [1, 2, 4]], 2), ([[1, 2], [1, 2, 3], [1, 2, 3, 4]], 2), ([[5], [6]], 0), ([[], [1]], 0),
                                           ([[1, 1]], 2), ([], 0)])
def test_common_start(prompts, start):
    assert common_start(prompts) == start


@pytest.mark.parametrize("name", ["A", "B"])
@pytest.mark.parametrize("budget", [3, 64])
def test_greedy_answers_to_one_prompt_equal_plain(cpu_ops, name, budget):
    engine, raw, weights = engine_for(name)
    prompts = [tiny_configs.prompt(n, engine.vocab_size, 30 + n) for n in (1, 2, 17)]
    got = Generator(engine, max_tokens_per_step=budget).generate(prompts, GenerationOptions(max_tokens=6, stop=()), samples=3)
    assert got == [ids for p in prompts for ids in [plain_impl.greedy_generate(raw, weights, p, 6)] * 3]
    assert not engine.cache.requests
    engine.cache.check()


def test_prompts_that_begin_alike_equal_plain(cpu_ops):
    engine, raw, weights = engine_for("B", max_requests=8)
    start = tiny_configs.prompt(19, engine.vocab_size, 1)
    prompts = [start + tiny_configs.prompt(n, engine.vocab_size, n) for n in (1, 7, 3)] + [start]
    got = LanguageModel(engine).generate(prompts, GenerationOptions(max_tokens=5, stop=()), samples=2, share=True)
    assert got == [ids for p in prompts for ids in [plain_impl.greedy_generate(raw, weights, p, 5)] * 2]


def test_answers_draw_for_themselves_and_as_requests_of_their_own_would(cpu_ops):
    engine, _, _ = engine_for("A")
    prompt = tiny_configs.prompt(9, engine.vocab_size, 3)

    def options(seed):
        return GenerationOptions(max_tokens=8, sampler=sampler(temperature(1.5), seed=seed), stop=())

    got = Generator(engine).generate([prompt], options(5), samples=3)
    assert got == [Generator(engine).generate([prompt], options(5 + i))[0] for i in range(3)]
    assert len({tuple(ids) for ids in got}) == 3
    with pytest.raises(ValueError, match="samples"):
        Generator(engine).generate([prompt], options(5), samples=0)


def test_a_cache_resized_between_steps_changes_no_answer(cpu_ops):
    engine, raw, weights = engine_for("B")
    generator = Generator(engine)
    prompts = [tiny_configs.prompt(n, engine.vocab_size, 30 + n) for n in (5, 13)]
    requests = [generator.add(p, GenerationOptions(max_tokens=8, stop=())) for p in prompts]
    for tokens in (96, 44, 400):
        generator.step()
        generator.resize_cache(tokens)
        engine.cache.check()
    with pytest.raises(ValueError, match="may grow past"):
        generator.resize_cache(16)
    generator.run()
    assert [r.generated for r in requests] == [plain_impl.greedy_generate(raw, weights, p, 8) for p in prompts]


def test_captured_steps_are_gone_ahead_of_a_resize_that_fails(cpu_ops, monkeypatch):
    engine, raw, weights = engine_for("B")
    assert len(engine.cache.groups) > 1
    generator = Generator(engine)
    prompt = tiny_configs.prompt(13, engine.vocab_size, 43)
    request = generator.add(prompt, GenerationOptions(max_tokens=8, stop=()))
    generator.step()
    first, at_the_time = [g.pages.data_ptr() for g in engine.cache.groups], []
    monkeypatch.setattr(engine.runner, "forget_graphs", lambda: at_the_time.append([g.pages.data_ptr() for g in engine.cache.groups]))
    with monkeypatch.context() as patch:
        failing_at(patch, len(engine.cache.groups))
        with pytest.raises(torch.OutOfMemoryError):
            generator.resize_cache(96)
    assert at_the_time == [first] and engine.cache_tokens == 256 and generator.scheduler.capacity == engine.cache.capacity_tokens() == 256
    assert [g.pages.data_ptr() for g in engine.cache.groups] == first
    generator.resize_cache(96)
    assert at_the_time == [first, first] and generator.scheduler.capacity == 96
    generator.run()
    assert request.generated == plain_impl.greedy_generate(raw, weights, prompt, 8)
