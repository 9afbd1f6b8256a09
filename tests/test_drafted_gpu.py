"""A step's tables, attention of drafted trees, adjusted logits and accepted drafts on the GPU, against plain implementations in 64 bits."""

from __future__ import annotations

import dataclasses
import math
import random

import numpy as np
import pytest
import torch

import drafted_refs as refs
from mlx_omnia_b200.kernels import ops
from mlx_omnia_b200.parts.base import KVSpec, KVView, StepContext

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def no_errors():
    yield
    ops.raise_on_error(torch.device("cuda:0"))


@pytest.fixture(params=["few rows", "many rows"])
def way(request, monkeypatch):
    """Both kernels of the tensor cores, at every size that they take."""
    monkeypatch.setattr(ops, "TREE_MANY_ROWS", {"few rows": 1 << 30, "many rows": 0}[request.param])
    monkeypatch.setattr(ops, "TREE_MANY_KEYS", 1 << 30)


def ints(values, dtype=torch.int32):
    return torch.as_tensor(np.asarray(values), device="cuda").to(dtype)


def error_of(word):
    """The error word, taken (and zero again)."""
    bits = int(ops.error_word(torch.device("cuda:0")).item())
    ops.error_word(torch.device("cuda:0")).zero_()
    return bits & word


# -- tables ----------------------------------------------------------------------------------------------------------
def tables_of(held, brought, page, strides, tokens=None, trees=None, padding=0, seed=0, slack=2):
    """(step_tables' answer, the same by the definition)"""
    rng = random.Random(seed)
    n, tokens = len(held), tokens or max(sum(brought), 1)
    lists, plain = [], []
    for stride in strides:
        counts = [-(-(-(-(h + b) // stride)) // page) if h >= 0 else 0 for h, b in zip(held, brought)]
        pages, starts, flat = list(range(5 * sum(counts) + 5)), [], []
        rng.shuffle(pages)
        mine = []
        for c in counts:
            flat += [-7] * rng.randint(0, 2)  # lists need not touch
            starts.append(len(flat))
            mine.append(pages[:c])
            flat += pages[:c]
            del pages[:c]
        width = max([*counts, 1]) + slack
        lists.append(ops.PageLists(ints(flat + [-7]), ints(starts, torch.int64), width, stride))
        table = [m + [-1] * (width - len(m)) for m in mine]
        slots = []
        for h, b, m in zip(held, brought, mine):
            slots += [-1 if h < 0 else m[(h + j) // stride // page] * page + (h + j) // stride % page for j in range(b)]
        plain.append((table, slots + [-1] * (tokens - sum(brought))))
    parents = None if trees is None else ints([p for t in trees for p in t] + [-1] * (tokens - sum(brought)))
    most = None if trees is None else max([*brought, 1])
    made = ops.step_tables(ints(held), ints(brought), lists, page, tokens, parents=parents, most=most)
    positions, seen = [], []
    for r, (h, b) in enumerate(zip(held, brought)):
        for way in refs.ways(trees[r] if trees is not None else refs.chain(b)):
            positions.append(-1 if h < 0 else h + len(way) - 1)
            seen.append([] if h < 0 else way)
    rest = tokens - len(positions)
    expect = {"positions": positions + [-1] * rest, "cu_seqlens": np.cumsum([0] + brought).tolist(),
              "seq_lens": [0 if h < 0 else h + b for h, b in zip(held, brought)], "groups": plain,
              "words": refs.words(seen + [[]] * rest, -(-most // 32)).tolist() if most else None}
    return made, expect


def same_tables(made, expect):
    assert made.positions.tolist() == expect["positions"]
    assert made.cu_seqlens.tolist() == expect["cu_seqlens"]
    assert made.seq_lens.tolist() == expect["seq_lens"]
    for (table, slots), (plain_table, plain_slots) in zip(made.groups, expect["groups"], strict=True):
        assert table.tolist() == plain_table and slots.tolist() == plain_slots
    assert (made.tree is None) == (expect["words"] is None)
    if made.tree is not None:
        assert made.tree.ancestors.tolist() == expect["words"]


@pytest.mark.parametrize("held,brought,page,strides", [
    ([0], [1], 16, [1]), ([15, 16, 17], [1, 1, 1], 16, [1]), ([5, 0, 300], [700, 1, 33], 16, [1, 1]), ([3, 9], [0, 2], 1, [1]),
    ([40, -1, 7, -1], [3, 1, 1, 1], 8, [1]), ([31, 64, 65], [5, 6, 7], 16, [4, 1]), ([0, 0], [0, 0], 16, [1]), ([10] * 300, [1] * 300, 48, [1]),
    ([7], [9000], 16, [1, 2, 3]), ([12], [2], 7, [1] * 8), ([1], [1], 16, [])])
def test_tables(held, brought, page, strides):
    for tokens in (None, sum(brought) + 37):
        same_tables(*tables_of(held, brought, page, strides, tokens))


@pytest.mark.parametrize("sizes", [[1], [2], [31, 32, 33], [64] * 5, [256, 1, 255], [97, 0, 3], [5] * 200])
def test_tables_of_trees(sizes):
    held = [(37 * i) % 500 for i in range(len(sizes))]
    for kind in (refs.chain, lambda n: refs.tree(n, n), lambda n: [-1] * n, lambda n: ([-1] + [0] * (n - 1))[:n]):
        trees = [kind(n)[:n] for n in sizes]
        same_tables(*tables_of(held, sizes, 16, [1, 1], sum(sizes) + 3, trees=trees))
    made, expect = tables_of(held, sizes, 16, [1], trees=[refs.chain(n) for n in sizes])
    lists = [ops.PageLists(ints([0] * 40000), ints([0] * len(sizes), torch.int64), 60)]
    again = ops.step_tables(ints(held), ints(sizes), lists, 16, max(sum(sizes), 1), most=max(sizes))  # no parents: chains
    assert again.tree.ancestors.tolist() == expect["words"] and again.positions.tolist() == expect["positions"]


def test_tables_report_what_does_not_fit():
    lists = lambda pages, width: [ops.PageLists(ints(pages), ints([0], torch.int64), width)]  # noqa: E731
    made = ops.step_tables(ints([20]), ints([1]), lists([3, 4], 1), 16, 1)  # a table too narrow
    assert error_of(16) and made.groups[0][0].tolist() == [[-1]] and made.groups[0][1].tolist() == [-1]
    made = ops.step_tables(ints([20]), ints([1]), lists([3], 2), 16, 1)  # a list too short
    assert error_of(16) and made.groups[0][0].tolist() == [[-1, -1]]
    made = ops.step_tables(ints([20]), ints([1]), lists([3, -1], 2), 16, 1)  # the page was given back
    assert error_of(4) and made.groups[0][1].tolist() == [-1]
    made = ops.step_tables(ints([0]), ints([5]), lists([3], 1), 16, 3)  # more tokens than rows
    assert error_of(16) and made.positions.tolist() == [0, 1, 2] and made.cu_seqlens.tolist() == [0, 3]
    made = ops.step_tables(ints([0]), ints([3]), lists([3], 1), 16, 3, parents=ints([-1, 1, -2]), most=3)  # no earlier tokens
    assert error_of(16) and made.tree.ancestors.tolist() == [[1], [2], [4]]
    made = ops.step_tables(ints([0]), ints([40]), lists([1, 2, 3], 3), 16, 40, most=32)  # more than it was said
    assert error_of(16) and made.positions.tolist() == list(range(32)) + [-1] * 8


def test_tables_of_numbers_at_the_end_of_their_types():
    lists = lambda pages, width: [ops.PageLists(ints(pages), ints([0], torch.int64), width)]  # noqa: E731
    for trees in ({}, {"most": 2}):  # positions beyond 31 bits, by one and by two
        for held, brought in (([7, 2 ** 31 - 1, 3], [1, 1, 1]), ([7, 2 ** 31 - 2, 3], [1, 2, 1])):
            made = ops.step_tables(ints(held), ints(brought), [ops.PageLists(ints([3, 4]), ints([0, 1, 1], torch.int64), 1)], 16, sum(brought), **trees)
            n = brought[1]
            assert error_of(16) and made.positions.tolist() == [7] + [-1] * n + [3] and made.seq_lens.tolist() == [8, 0, 4]
            assert made.groups[0][0].tolist() == [[3], [-1], [4]] and made.groups[0][1].tolist() == [55] + [-1] * n + [67]
    made = ops.step_tables(ints([2 ** 31 - 2]), ints([1]), lists([3, 4], 2), 16, 1)  # the last position of 31 bits, in a table too narrow
    assert error_of(16) and made.seq_lens.tolist() == [2 ** 31 - 1] and made.groups[0][1].tolist() == [-1]
    made = ops.step_tables(ints([20]), ints([1]), [ops.PageLists(ints([3, 4]), ints([2 ** 63 - 1], torch.int64), 2)], 16, 1)  # a list that begins nowhere
    assert error_of(16) and made.groups[0][0].tolist() == [[-1, -1]] and made.groups[0][1].tolist() == [-1]


# -- attention -------------------------------------------------------------------------------------------------------
@dataclasses.dataclass
class Case:
    q: torch.Tensor
    rows: torch.Tensor  # the gate's columns behind as many of something else
    kv: KVView
    step: StepContext
    sink: torch.Tensor
    requests: list  # (first row, nodes, keys, values, positions, key positions, sees), on the host


def make(nq, nkv, d, dtype, page, requests, *, dv=None, seed=0, spread=1.0, masks=None, behind=0, window=None, keep=0):
    """`requests`: (positions held, parents). Pages in any order; whatever no request holds is NaN."""
    dv = dv or d
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    lengths = [held + len(parents) for held, parents in requests]
    width = max([-(-n // page) for n in lengths] + [1]) + 1
    tokens = sum(len(p) for _, p in requests)
    pages = list(range(sum(-(-n // page) for n in lengths) + 3))
    rng.shuffle(pages)
    spec = KVSpec(((nkv, d), (nkv, dv)), window, keep_first=keep)
    shape = (len(pages), 2, nkv, page, d) if d == dv else (len(pages), nkv * (d + dv) * page)
    store = torch.full(shape, math.nan, dtype=dtype, device="cuda")
    kv = KVView(store, None, ints([0] * tokens, torch.int64), page, window, spec=spec)
    k_row, v_row = kv.row(0), kv.row(1)
    table, held_of, first, seen = [], [], 0, []
    words = max(-(-max([len(p) for _, p in requests] + [1]) // 32), 1)
    for r, ((held, parents), n) in enumerate(zip(requests, lengths)):
        mine = [pages.pop() for _ in range(-(-n // page))]
        table.append(mine + [-1] * (width - len(mine)))
        k = torch.randn(n, nkv, d, generator=g, device="cuda").mul(spread).to(dtype)
        v = torch.randn(n, nkv, dv, generator=g, device="cuda").to(dtype)
        at = ints([mine[i // page] for i in range(n)], torch.int64), ints([i % page for i in range(n)], torch.int64)
        k_row[at[0], :, at[1]] = k
        v_row[at[0], :, at[1]] = v
        ways = refs.ways(parents) if masks is None or masks[r] is None else masks[r]
        depth = [len(w) - 1 for w in refs.ways(parents)]
        sees = torch.zeros(len(parents), len(parents), dtype=torch.bool)
        for i, w in enumerate(ways):
            sees[i, w] = True
        positions = torch.tensor([held + x for x in depth], dtype=torch.long)
        held_of.append((first, len(parents), k.cpu(), v.cpu(), positions, torch.cat([torch.arange(held), positions]), sees))
        seen += ways
        first += len(parents)
    q = torch.randn(tokens + behind, nq, d, generator=g, device="cuda").to(dtype)
    rows = torch.randn(tokens + behind, 2 * nq * dv, generator=g, device="cuda").to(dtype)
    kv = dataclasses.replace(kv, block_table=ints(table))
    counts = [len(p) for _, p in requests]
    step = StepContext(
        num_tokens=tokens + behind, num_seqs=len(requests), token_ids=ints([0] * (tokens + behind)),
        positions=ints([p for x in held_of for p in x[4].tolist()] + [-1] * behind), cu_seqlens=ints(np.cumsum([0] + counts)), seq_lens=ints(lengths),
        state_slots=ints([0]), fresh=ints([0]), logit_rows=ints([]), q_lens=counts, seq_lens_host=lengths, max_q_len=max(counts),
        max_seq_len=max(lengths), decode_only=False, groups={}, tree=ops.StepTree(ints(refs.words(seen + [[]] * behind, words))))
    return Case(q, rows, kv, step, torch.randn(nq, generator=g, device="cuda"), held_of)


def check(c, scale, gated=False, sink=False, window=0, keep=0, run=0, softcap=0.0, call=None, **options):
    tokens, nq, d = c.q.shape
    if call is None:
        call = lambda **more: ops.paged_attention(c.q, c.kv, c.step, scale, **more)  # noqa: E731
    dv = c.kv.row(1).shape[3]
    got = call(gate=c.rows if gated else None, gate_col=nq * dv, sink=c.sink if sink else None, softcap=softcap or None, chunk=run or None, **options)
    ops.raise_on_error(got.device)
    bf16 = c.q.dtype == BF16
    for first, nodes, k, v, positions, key_positions, sees in c.requests:
        if not nodes:
            continue
        q = c.q[first: first + nodes].cpu()
        out, size, largest = refs.attention(q, k, v, positions, key_positions, sees, scale, window, keep, run, softcap,
                                            c.sink.cpu() if sink else None)
        if gated:
            gate = torch.sigmoid(c.rows[first: first + nodes, nq * dv:].cpu().double()).view(nodes, nq, dv)
            out, size = out * gate, size * gate.abs()
        mine = got[first: first + nodes].cpu().double().view(nodes, nq, dv)
        # A score of d products in 32 bits is off by (d + 8) 2^-24 of the products' sizes added up, a weight by that and a sum of n terms twice,
        # exponentials and the tanh by some units of the last place of numbers up to 2^5 (their argument's rounding); in bfloat16 a weight is
        # rounded too (2^-8) and so is the result (2^-8 of itself).
        n = k.shape[0]
        score = (d + 8) * 2.0 ** -24 * largest + 2.0 ** -19
        bound = size * (2 * score + (n + 32) * 2.0 ** -23) + 1e-30
        if bf16:
            bound = bound + 2.0 ** -8 * (size + out.abs())
        assert torch.equal(torch.isfinite(mine), torch.isfinite(out))
        worst = ((mine - out).abs() / bound)[torch.isfinite(out)].max()
        assert worst <= 1, float(worst)
    return got


LAYOUTS = [(16, 8, 128, BF16, 16), (32, 8, 128, BF16, 16), (16, 4, 128, BF16, 32), (6, 2, 64, BF16, 16), (8, 1, 24, F32, 8), (4, 4, 128, F32, 16),
           (5, 1, 96, BF16, 8), (16, 1, 64, BF16, 48), (2, 2, 256, BF16, 16), (3, 1, 20, BF16, 5), (4, 2, 130, F32, 16), (2, 1, 512, F32, 4),
           (6, 3, 64, F32, 16), (2, 1, 200, F32, 16), (7, 1, 36, F32, 3)]


@pytest.mark.parametrize("layout", LAYOUTS, ids=str)
def test_attention_of_trees(layout, way):
    nq, nkv, d, dtype, page = layout
    c = make(nq, nkv, d, dtype, page, [(500, refs.tree(13, 1)), (0, refs.tree(5, 2)), (1, [-1]), (63, refs.chain(64)), (130, refs.tree(70, 3)),
                                       (16, refs.tree(16, 4))], seed=d)
    check(c, d ** -0.5)
    check(c, d ** -0.5, gated=True, sink=True)
    check(c, d ** -0.5, softcap=3.0)
    check(c, -0.3 * d ** -0.5, sink=True)


@pytest.mark.parametrize("layout", [LAYOUTS[0], LAYOUTS[3], LAYOUTS[4], LAYOUTS[8], LAYOUTS[9]], ids=str)
def test_a_scale_of_zero(layout, way):
    """All that a row sees weighs the same."""
    nq, nkv, d, dtype, page = layout
    c = make(nq, nkv, d, dtype, page, [(70, refs.tree(13, 1)), (0, refs.tree(5, 2)), (1, [-1])], seed=d)
    for scale in (0.0, -0.0, 1e-42):
        for options in ({}, {"sink": True}, {"softcap": 3.0}):
            check(c, scale, **options)
        check(c, scale, window=9, keep=2, call=lambda **more: ops.paged_attention(c.q, c.kv, c.step, scale, window=9, keep_first=2, **more))


WIDTHS = [(3, 1, 33, 33), (4, 2, 48, 32), (3, 3, 32, 80), (3, 1, 33, 17), (5, 1, 1, 7), (2, 1, 7, 300), (1, 1, 260, 129), (1, 1, 9, 511)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("layout", WIDTHS, ids=str)
def test_keys_and_values_of_any_widths(layout, dtype):
    """Keys and values that differ in width, odd widths: the kernel for any shape, its keys in one piece and in several (of an odd count too)."""
    nq, nkv, d, dv = layout
    for requests in ([(145, refs.tree(5, 1))], [(20, refs.tree(5, 2))], [(300, refs.chain(3)), (0, [-1]), (64, refs.tree(9, 3))], [(1000, [-1])]):
        c = make(nq, nkv, d, dtype, 16, requests, dv=dv, seed=d + dv)
        check(c, d ** -0.5)
        check(c, d ** -0.5, gated=True, sink=True, softcap=2.0)
        check_window(c, d, 150, keep=3, sink=True)


@pytest.mark.parametrize("layout", LAYOUTS[:6] + LAYOUTS[8:10], ids=str)
def test_attention_of_trees_under_windows(layout, way):
    nq, nkv, d, dtype, page = layout
    c = make(nq, nkv, d, dtype, page, [(500, refs.tree(33, 1)), (3, refs.chain(40)), (100, refs.tree(7, 2)), (36, refs.tree(9, 5))], seed=1)
    for window in (1, 5, 37, 400):
        check_window(c, d, window)
    check_window(c, d, 20, keep=4, sink=True)
    check_window(c, d, 1000, keep=40)
    check_run(c, d, 8)
    check_run(c, d, 100)


def check_window(c, d, window, keep=0, **more):
    call = lambda **options: ops.paged_attention(c.q, c.kv, c.step, d ** -0.5, window=window, keep_first=keep, **options)  # noqa: E731
    check(c, d ** -0.5, window=window, keep=keep, call=call, **more)


def check_run(c, d, run):
    check(c, d ** -0.5, run=run)


@pytest.mark.parametrize("held,nodes", [(1, 1), (64, 1), (4097, 17), (20000, 3), (3000, 256), (0, 256), (1, 200)])
def test_attention_of_trees_by_length(held, nodes, way):
    for layout in ((16, 8, 128, BF16, 16), (6, 2, 64, BF16, 16)) + (((8, 1, 24, F32, 8),) if held < 10000 else ()):
        nq, nkv, d, dtype, page = layout
        check(make(nq, nkv, d, dtype, page, [(held, refs.tree(nodes, held)), (held // 2, refs.tree(max(nodes // 3, 1), 9))], seed=nodes), d ** -0.5, gated=True)


@pytest.mark.parametrize("layout", LAYOUTS[:1] + LAYOUTS[3:5], ids=str)
def test_attention_of_any_masks(layout, way):
    """Rows that see nothing have zeros, rows may see later tokens, and none knows of what it does not see."""
    nq, nkv, d, dtype, page = layout
    c = make(nq, nkv, d, dtype, page, [(0, refs.chain(9)), (40, refs.chain(3)), (0, refs.chain(40))],
             masks=[[[], [0], [1, 2, 8], [], [4], [8], [0, 1, 2, 3], [7], []], [[2], [], [0, 1, 2]], [[39 - i] for i in range(39)] + [[]]])
    for options in ({}, {"sink": True}, {"gated": True}):
        got = check(c, d ** -0.5, **options)
        assert float(got[0].abs().max()) == 0 and float(got[3].abs().max()) == 0 and float(got[-1].abs().max()) == 0


@pytest.mark.parametrize("layout", LAYOUTS[:2] + LAYOUTS[3:5] + LAYOUTS[6:7], ids=str)
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_what_a_node_does_not_see_may_be_anything(layout, value, way):
    nq, nkv, d, dtype, page = layout
    c = make(nq, nkv, d, dtype, page, [(70, [-1, 0, 0, 1, 2, 2]), (200, refs.tree(40, 2))], seed=5)
    for r, (bad, held) in enumerate(((2, 70), (11, 200))):
        slot = held + bad
        at = int(c.kv.block_table[r, slot // page])
        for row, which in ((c.kv.row(0), 2), (c.kv.row(1), 3)):
            row[at, :, slot % page, d // 2] = value
            c.requests[r][which][slot, :, d // 2] = value
    got = check_some(c, d, {0: 2, 1: 11})
    assert torch.isfinite(got[:2]).all() and torch.isfinite(got[3]).all()
    if math.isnan(value):  # and what it does see reaches it
        assert torch.isnan(got[2]).all() and torch.isnan(got[4]).all()


def check_some(c, d, bad):
    """The rows that do not see token `bad` of their request are as ever."""
    got = ops.paged_attention(c.q, c.kv, c.step, d ** -0.5)
    for r, (first, nodes, k, v, positions, key_positions, sees) in enumerate(c.requests):
        fine = ~sees[:, bad[r]]
        k, v = k.nan_to_num(0, 0, 0), v.nan_to_num(0, 0, 0)
        out, size, _ = refs.attention(c.q[first: first + nodes].cpu(), k, v, positions, key_positions, sees, d ** -0.5)
        mine = got[first: first + nodes].cpu().double().view(out.shape)[fine]
        assert torch.isfinite(mine).all()
        assert ((mine - out[fine]).abs() <= 2.0 ** -7 * size[fine] + 1e-4).all()
    return got


def test_padding_and_rows_behind_the_last_request(way):
    """A request of no positions is there for the step's shape; rows behind the last request are not written."""
    for layout in LAYOUTS[:1] + LAYOUTS[4:5]:
        nq, nkv, d, dtype, page = layout
        c = make(nq, nkv, d, dtype, page, [(50, refs.tree(6, 1)), (7, [-1])], behind=3)
        c.step.seq_lens[1] = 0
        c.kv.block_table[1] = -1
        del c.requests[1]
        got = check(c, d ** -0.5)
        assert float(got[6].abs().max()) == 0


@pytest.mark.parametrize("layout", [LAYOUTS[0], LAYOUTS[4], LAYOUTS[9], LAYOUTS[7]], ids=str)
def test_requests_whose_rows_are_not_the_steps(layout, way):
    """Rows behind the step's last one, of a request that holds something and of one that is there for the shape only, and a list that goes back: reported,
    and the other requests' rows are as ever."""
    nq, nkv, d, dtype, page = layout
    c = make(nq, nkv, d, dtype, page, [(20, refs.tree(6, 1)), (7, refs.tree(4, 2))], seed=2)  # (a tile of keys each: no sum is split otherwise)
    expect = check(c, d ** -0.5)
    lengths, ends = c.step.seq_lens.clone(), c.step.cu_seqlens.clone()
    for held, cu in ((0, [0, 6, 13]), (11, [0, 6, 13]), (-1, [0, 6, 10 + 20]), (0, [0, 6, 2 ** 31 - 1]), (0, [0, 6, 5]), (11, [0, 6, 2]), (0, [0, 6, -4])):
        c.step.seq_lens.copy_(ints([26, held]))
        c.step.cu_seqlens.copy_(ints(cu))
        got = ops.paged_attention(c.q, c.kv, c.step, d ** -0.5)
        assert error_of(16) and torch.equal(got[:6], expect[:6])
        if cu[2] > 10:
            assert float(got[6:].abs().max()) == 0
    c.step.seq_lens.copy_(lengths)
    c.step.cu_seqlens.copy_(ends)
    assert torch.equal(check(c, d ** -0.5), expect)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_more_requests_times_heads_than_an_axis_of_a_grid_takes(dtype):
    """65,600 of them, for the kernel of any shape: more than 1,024 requests, with one piece of keys."""
    c = make(8, 8, 8, dtype, 4, [(i % 7, refs.chain(1 + i % 2)) for i in range(8200)], seed=1)
    c.requests = c.requests[::50] + c.requests[-3:]
    check(c, 8 ** -0.5, sink=True)


@pytest.mark.parametrize("d", [64, 128])
def test_blocks_of_many_items(d, way):
    """Blocks that work off eight items and more each, of few rows and of many in turn, again and again."""
    sizes = [(37 * i % 300, (5, 64, 1, 40, 33)[i % 5]) for i in range(300)]
    c = make(16, 4, d, BF16, 16, [(held, refs.tree(nodes, held)) for held, nodes in sizes], seed=d)
    expect = check(c, d ** -0.5)
    for _ in range(10):
        assert torch.equal(ops.paged_attention(c.q, c.kv, c.step, d ** -0.5), expect)


def test_a_captured_step_takes_the_lengths_of_its_replay(way):
    nq, nkv, d, dtype, page = LAYOUTS[0]
    big = make(nq, nkv, d, dtype, page, [(900, refs.tree(16, 1)), (300, refs.tree(16, 2))], seed=3)
    small = make(nq, nkv, d, dtype, page, [(200, refs.tree(16, 5)), (899, refs.tree(16, 7))], seed=4)
    step = dataclasses.replace(big.step, workspace={"private": True})
    kv = dataclasses.replace(big.kv, pages=torch.zeros(max(big.kv.pages.shape[0], small.kv.pages.shape[0]), *big.kv.pages.shape[1:], dtype=dtype, device="cuda"),
                             block_table=torch.full_like(big.kv.block_table, -1))
    q, moving = torch.empty_like(big.q), ("positions", "cu_seqlens", "seq_lens")

    def take(c):
        q.copy_(c.q)
        kv.pages[: c.kv.pages.shape[0]] = c.kv.pages
        kv.block_table.fill_(-1)
        kv.block_table[:, : c.kv.block_table.shape[1]] = c.kv.block_table
        held = {name: getattr(c.step, name).clone() for name in moving}
        for name in moving:
            getattr(step, name).copy_(held[name])
        step.tree.ancestors.copy_(c.step.tree.ancestors.clone())

    step.tree = ops.StepTree(step.tree.ancestors.clone())
    for name in moving:
        setattr(step, name, getattr(step, name).clone())
    take(big)
    ops.paged_attention(q, kv, step, d ** -0.5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.paged_attention(q, kv, step, d ** -0.5)
    for c in (small, big, small):
        take(c)
        graph.replay()
        check(c, d ** -0.5, call=lambda **_: out)


@pytest.mark.parametrize("layout", [LAYOUTS[0], (8, 1, 128, F32, 16), (4, 2, 130, F32, 16)], ids=str)
def test_lengths_beyond_the_plan(layout, way):
    """The kernel for any shape works by a plan for so many positions, the others by the lengths themselves; all by the most tokens."""
    nq, nkv, d, dtype, page = layout
    c = make(nq, nkv, d, dtype, page, [(900, refs.tree(40, 1))])
    c.step.max_seq_len = 300
    if d != 130:
        check(c, d ** -0.5)
    else:
        ops.paged_attention(c.q, c.kv, c.step, d ** -0.5)
        assert error_of(16)
    c.step.max_seq_len, c.step.max_q_len = 940, 3
    ops.paged_attention(c.q, c.kv, c.step, d ** -0.5)
    assert error_of(16)
    c.step.max_q_len, c.step.seq_lens[0] = 40, 10  # fewer positions than tokens
    ops.paged_attention(c.q, c.kv, c.step, d ** -0.5)
    assert error_of(16)
    c = make(nq, nkv, d, dtype, page, [(900, refs.tree(16, 1))])
    c.kv.block_table[0, 3] = 100000
    ops.paged_attention(c.q, c.kv, c.step, d ** -0.5)
    assert error_of(4)


# -- logits ----------------------------------------------------------------------------------------------------------
def bits_of(allowed, vocab, spare=0):
    return refs.words([sorted(a) for a in allowed], -(-vocab // 32) + spare)


def logits_case(rows, vocab, lengths, seed=0, biases=6, masked=0.5, gap=0):
    rng = random.Random(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    texts = [[rng.choice([rng.randrange(vocab), rng.randrange(min(vocab, 9)), vocab - 1]) for _ in range(n)] for n in lengths]
    prompts = [rng.randint(0, n) for n in lengths]
    values = [[float(np.float32(rng.uniform(*span))) for _ in lengths] for span in ((0.5, 2.0), (-0.5, 1.0), (-0.5, 1.0))]
    bias = [[(rng.choice([rng.randrange(vocab), 0]), float(np.float32(rng.gauss(0, 5)))) for _ in range(rng.randint(0, biases))] for _ in lengths]
    masks = [None if rng.random() > masked else {rng.randrange(vocab) for _ in range(rng.choice([0, 1, 30, vocab]))} for _ in range(rows)]
    logits = (torch.randn(rows, vocab + gap, generator=g, device="cuda") * 4)[:, :vocab]
    logits[0, 0], logits[0, vocab - 1] = 0.0, -math.inf
    return logits, texts, prompts, values, bias, masks


def call_adjust(logits, texts, prompts, values, bias, masks, use, requests=None, contexts=None, drafted=None, out=None):
    history = ops.TokenHistory(ints([v for t in texts for v in t] or np.zeros(0)), ints(np.cumsum([0] + [len(t) for t in texts])[:-1], torch.int64),
                               ints([len(t) for t in texts]), ints(prompts))
    floats = lambda v: torch.tensor(v, dtype=F32, device="cuda")  # noqa: E731
    some = [i for i, m in enumerate(masks) if m is not None]
    which = [some.index(i) if i in some else -1 for i in range(len(masks))]
    return ops.adjust_logits(
        logits, history=history if "p" in use else None, repetition=floats(values[0]) if "p" in use else None,
        frequency=floats(values[1]) if "p" in use else None, presence=floats(values[2]) if "p" in use else None,
        contexts=ints(contexts) if contexts is not None else None, requests=ints(requests) if requests is not None else None,
        bias=ops.LogitBias(ints([v for b in bias for v, _ in b] or np.zeros(0)), floats([x for b in bias for _, x in b]),
                           ints(np.cumsum([0] + [len(b) for b in bias]))) if "b" in use else None,
        masks=ops.TokenMasks(ints(bits_of([masks[i] for i in some], logits.shape[1], 1)) if some else ints(np.zeros((1, logits.shape[1] // 32 + 1))),
                             ints(which)) if "m" in use else None, drafted=drafted, out=out)


def close(got, expect, rows_of=lambda i: i, values=None, bias=None, texts=None):
    """Each of the up to 4 + (biases) roundings of a logit is off by 2^-24 of the largest number that it passes through."""
    got, expect = got.double().cpu(), expect.cpu()
    assert torch.equal(torch.isinf(got), torch.isinf(expect)) and not torch.isnan(got).any()
    fine = torch.isfinite(expect)
    assert ((got - expect).abs()[fine] <= 2.0 ** -24 * 12 * (expect.abs()[fine] + 150)).all()


@pytest.mark.parametrize("rows,vocab,lengths,gap", [
    (1, 777, [0], 0), (3, 1000, [1, 500, 30], 0), (2, 8192, [3000, 5], 8), (4, 8193, [20, 30, 0, 7], 3), (2, 32003, [700, 700], 0),
    (1, 151936, [4000], 0), (5, 16384, [9, 9, 9, 9, 9], 1), (1, 1, [3], 0), (2, 33, [40, 2], 0)])
@pytest.mark.parametrize("use", ["p", "b", "m", "pbm", "pb", "pm"])
def test_adjusted_logits(rows, vocab, lengths, gap, use):
    logits, texts, prompts, values, bias, masks = logits_case(rows, vocab, lengths, seed=rows * vocab, gap=gap)
    none = [1.0] * rows, [0.0] * rows, [0.0] * rows
    expect = refs.adjust(logits.cpu(), texts if "p" in use else [[]] * rows, prompts, *(values if "p" in use else none),
                         biases=bias if "b" in use else None, masks=masks if "m" in use else None)
    before = logits.clone()
    got = call_adjust(logits, texts, prompts, values, bias, masks, use)
    close(got, expect)
    assert torch.equal(logits, before)  # a new tensor
    other = torch.full((rows, vocab + 5), 7.0, device="cuda")[:, :vocab]
    assert call_adjust(logits, texts, prompts, values, bias, masks, use, out=other) is other
    assert torch.equal(other, got)
    assert call_adjust(logits, texts, prompts, values, bias, masks, use, out=logits) is logits  # in place
    assert torch.equal(logits, got)


@pytest.mark.parametrize("contexts", [None, [3, 0, 50, 1]])
def test_adjusted_rows_share_requests_and_contexts(contexts):
    vocab, requests = 5000, [2, 2, 0, 3, 1, 2, 2, 2, 2, 2, 2]
    logits, texts, prompts, values, bias, masks = logits_case(len(requests), vocab, [40, 7, 90, 3], seed=3)
    pick = lambda x: [x[r] for r in requests]  # noqa: E731
    expect = refs.adjust(logits.cpu(), pick(texts), pick(prompts), *map(pick, values), contexts=None if contexts is None else pick(contexts),
                         biases=pick(bias), masks=masks)
    close(call_adjust(logits, texts, prompts, values, bias, masks, "pbm", requests=requests, contexts=contexts), expect)


@pytest.mark.parametrize("contexts", [None, [3, 0, 20]])
@pytest.mark.parametrize("empty", [False, True])
def test_adjusted_rows_of_drafted_trees(contexts, empty):
    vocab, sizes = 9000, [5, 40, 1]
    trees = [refs.tree(n, n) for n in sizes]
    rng = random.Random(1)
    ids = [rng.choice([3, 5, rng.randrange(vocab)]) for _ in range(sum(sizes))]
    cu = np.cumsum([0] + sizes).tolist()
    rows = list(range(sum(sizes)))
    rng.shuffle(rows)
    rows = rows[:30]
    requests = [max(r for r in range(3) if cu[r] <= t) for t in rows]
    logits, texts, prompts, values, bias, masks = logits_case(len(rows), vocab, [0, 0, 0] if empty else [30, 100, 8], seed=4)
    ways = [[cu[r] + j for j in w] for r, tree in enumerate(trees) for w in refs.ways(tree)]
    pick = lambda x: [x[r] for r in requests]  # noqa: E731
    whole = [texts[r] + [ids[j] for j in ways[t]] for r, t in zip(requests, rows)]
    expect = refs.adjust(logits.cpu(), whole, pick(prompts), *map(pick, values), contexts=None if contexts is None else pick(contexts),
                         biases=pick(bias), masks=masks)
    words = refs.words([w for tree in trees for w in refs.ways(tree)], 2)
    drafted = ops.DraftedRows(ops.StepTree(ints(words)), ints(ids), ints(cu), ints(rows))
    for out in (None, logits):
        got = call_adjust(logits, texts, prompts, values, bias, masks, "pbm", requests=requests, contexts=contexts, drafted=drafted, out=out)
        close(got, expect)


def test_a_bias_named_many_times_adds_in_order():
    vocab = 20000
    logits = torch.zeros(1, vocab, device="cuda")
    rng = random.Random(0)
    entries = [(rng.choice([5, 7777, 19999, rng.randrange(vocab)]), float(np.float32(rng.gauss(0, 100)))) for _ in range(5000)]
    answers = {tuple(call_adjust(logits, [[]], [0], [[1.0], [0.0], [0.0]], [entries], [None], "b")[0].tolist()) for _ in range(3)}
    assert len(answers) == 1
    expect = np.zeros(vocab, dtype=np.float32)
    for v, b in entries:
        expect[v] = np.float32(expect[v] + np.float32(b))
    assert np.array_equal(np.asarray(answers.pop(), dtype=np.float32), expect)


@pytest.mark.parametrize("start,length", [(2 ** 63 - 1, 3), (2 ** 63 - 5, 2), (-1, 3), (-2 ** 63, 1), (8, 3), (0, 11), (11, 0), (0, -1)])
def test_texts_that_lie_nowhere(start, length):
    """Reported, and nothing is counted."""
    logits = torch.ones(1, 50, device="cuda")
    history = ops.TokenHistory(ints(list(range(10))), ints([start], torch.int64), ints([length]), ints([0]))
    got = ops.adjust_logits(logits, history=history, frequency=torch.ones(1, device="cuda"))
    assert error_of(16) and torch.equal(got, logits)


def test_masks_alone_go_by_no_requests():
    """Rows of requests of which nothing is given but masks: whose rows they are changes nothing."""
    logits = torch.randn(3, 70, device="cuda")
    masks = ops.TokenMasks(ints([[-1, 0, 63], [5, 0, 0]]), ints([0, -1, 1]))
    expect = ops.adjust_logits(logits, masks=masks)
    assert torch.equal(expect[1], logits[1]) and torch.isinf(expect[2]).sum() == 68 and torch.isinf(expect[0]).sum() == 32
    for requests in ([0, 0, 1], [9, 4, 100], [-1, 5, 2]):
        assert torch.equal(ops.adjust_logits(logits, masks=masks, requests=ints(requests)), expect)


def test_adjust_reports_bad_numbers():
    logits = torch.zeros(2, 100, device="cuda")
    run = lambda **more: call_adjust(logits, *({"texts": [[1], [2]], "prompts": [0, 0], "values": [[1.0] * 2] * 3, "bias": [[], []], "masks": [None] * 2} | more).values(), "pb")  # noqa: E731
    run(texts=[[1, 100], [2]])
    assert error_of(1)
    run(texts=[[1, -1], [2]])
    assert error_of(1)
    run(bias=[[(100, 1.0)], []])
    assert error_of(1)
    call_adjust(logits, [[1], [2]], [0, 0], [[1.0] * 2] * 3, [[], []], [None] * 2, "p", requests=[0, 2])
    assert error_of(16)


# -- accepted drafts -------------------------------------------------------------------------------------------------
def accept_case(trees, seed, vocab=4):
    rng = random.Random(seed)
    ids = [[rng.randrange(vocab) for _ in t] for t in trees]
    chosen = [[rng.randrange(vocab) for _ in t] for t in trees]
    return ids, chosen, [refs.accept(*x) for x in zip(trees, ids, chosen)]


def accept(trees, ids, chosen, words):
    sees = refs.words([w for t in trees for w in refs.ways(t)], words)
    return ops.accept_drafts(ints([x for t in chosen for x in t]), ints([x for t in ids for x in t]), ops.StepTree(ints(sees)),
                             ints(np.cumsum([0] + [len(t) for t in trees])))


@pytest.mark.parametrize("sizes", [[1], [2, 1], [8] * 20, [0, 5, 0], [33, 64, 256], [256] * 3, [31, 32, 3]])
@pytest.mark.parametrize("vocab", [1, 2, 4])
def test_accepted_drafts(sizes, vocab):
    for seed, kind in enumerate((refs.chain, lambda n: refs.tree(n, n + vocab), lambda n: refs.tree(n, 1, 3), lambda n: [-1] + [0] * (n - 1))):
        trees = [kind(n)[:n] for n in sizes]
        ids, chosen, paths = accept_case(trees, seed, vocab)
        words = -(-max(sizes) // 32)
        got = accept(trees, ids, chosen, words)
        assert got.kept.tolist() == [len(p) for p in paths]
        assert got.path.tolist() == [p + [-1] * (32 * words - len(p)) for p in paths]
        assert got.tokens.tolist() == [c[p[-1]] if p else -1 for c, p in zip(chosen, paths)]


@pytest.mark.parametrize("rows,page,dtype", [(((8, 128), (8, 128)), 16, BF16), (((1, 24), (1, 24)), 8, F32), (((2, 5), (2, 3)), 3, BF16),
                                             (((1, 576),), 16, BF16), (((3, 1), (3, 1)), 4, torch.uint8), (((2, 6), (1, 2), (1, 4)), 1, BF16)])
@pytest.mark.parametrize("sizes", [[1], [12, 40, 7], [256, 3], [0, 9]])
def test_kept_rows(rows, page, dtype, sizes):
    layers, held = 3, [11, 0, 37][: len(sizes)]
    trees = [refs.tree(n, n, 3)[:n] for n in sizes]
    ids, chosen, paths = accept_case(trees, 7, 2)
    elements = sum(h * w for h, w in rows) * page
    counts = [-(-(h + n) // page) for h, n in zip(held, sizes)]
    order = torch.randperm(sum(counts) + 2, generator=torch.Generator().manual_seed(1)).tolist()
    table, width = [], max(counts) + 1
    for c in counts:
        table.append([order.pop() for _ in range(c)])
    g = torch.Generator(device="cuda").manual_seed(2)
    pages = torch.randint(0, 100, (layers, sum(counts) + 2, elements), generator=g, device="cuda").to(dtype)
    expect = pages.cpu().clone()

    def place(r, at):  # views of the stored row of a position, by kind
        page_at, off, start = table[r][at // page], at % page, 0
        for h, w in rows:
            yield expect[:, page_at, start: start + h * w * page].view(layers, h, page, w)[:, :, off]
            start += h * w * page

    for r, path in enumerate(paths):
        for i, j in enumerate(path):
            for to, src in zip(place(r, held[r] + i), list(place(r, held[r] + j))):
                to.copy_(src.clone())
    accepted = accept(trees, ids, chosen, -(-max(sizes) // 32))
    got = ops.keep_rows(pages, rows, page, ints([t + [-1] * (width - len(t)) for t in table]), ints(held), accepted)
    assert got is pages and torch.equal(pages.cpu(), expect)
    again = pages.clone()
    ops.keep_rows(again, rows, page, ints([t + [-1] * (width - len(t)) for t in table]), ints([-1] * len(held)), accepted)  # nobody's
    assert torch.equal(again.cpu(), expect)


def test_kept_rows_report_bad_pages():
    pages = torch.zeros(1, 4, 2, 1, 4, 8, device="cuda")
    accepted = ops.Accepted(ints([[0, 2] + [-1] * 30]), ints([2]), ints([5]))
    for table in ([[0, -1]], [[0, 9]], [[0]]):
        ops.keep_rows(pages, ((1, 8), (1, 8)), 4, ints(table), ints([2]), accepted)
        assert error_of(4)
    for path in ([0, 0], [0, -1], [0, 40], [1, 1]):
        ops.keep_rows(pages, ((1, 8), (1, 8)), 4, ints([[0, 1]]), ints([2]), ops.Accepted(ints([path + [-1] * 30]), ints([2]), ints([5])))
        assert error_of(4)
