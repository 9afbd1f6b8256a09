"""The operators of a step of drafted tokens as a program would call them: captured together and replayed on other inputs, two captured steps in turn,
two streams at once, behind work of another stream, over memory beyond 2^31 elements, and with numbers that are none."""

from __future__ import annotations

import math
import random

import numpy as np
import pytest
import torch

import drafted_refs as refs
from mlx_omnia_b200.kernels import ops
from mlx_omnia_b200.parts.base import KVSpec, KVView, StepContext
from test_drafted_gpu import BF16, F32, check, check_window, ints, make, no_errors, way  # noqa: F401  (the fixtures too)

pytestmark = pytest.mark.gpu
PAGE, VOCAB, WORDS = 16, 9000, 1


class WholeStep:
    """A step of `n` requests that bring up to 20 drafted tokens each, from its tables to the rows that are kept, on buffers that stay."""

    def __init__(self, n, nq=4, nkv=2, d=64, dtype=BF16, longest=600):
        self.n, self.nq, self.d, self.rows, self.longest = n, nq, d, 20 * n, longest
        self.width = -(-longest // PAGE)
        self.held, self.brought, self.parents, self.ids = (torch.zeros(k, dtype=torch.int32, device="cuda") for k in (n, n, self.rows, self.rows))
        self.lists = ops.PageLists(torch.arange(n * self.width, dtype=torch.int32, device="cuda"),
                                   torch.arange(n, device="cuda") * self.width, self.width)
        self.spec = KVSpec.keys_and_values(nkv, d)
        self.pages = torch.zeros(2, n * self.width, 2, nkv, PAGE, d, dtype=dtype, device="cuda")  # of two layers
        self.q = torch.zeros(self.rows, nq, d, dtype=dtype, device="cuda")
        self.logits = torch.zeros(self.rows, VOCAB, device="cuda")
        self.history = ops.TokenHistory(torch.zeros(50 * n, dtype=torch.int32, device="cuda"), torch.arange(n, device="cuda") * 50,
                                        torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda"))
        self.penalty = torch.zeros(n, device="cuda")
        self.which, self.owner = torch.arange(self.rows, dtype=torch.int32, device="cuda"), torch.zeros(self.rows, dtype=torch.int32, device="cuda")

    def take(self, seed):
        rng, g = random.Random(seed), torch.Generator(device="cuda").manual_seed(seed)
        sizes = [rng.choice([1, 2, 17, 20]) for _ in range(self.n)]
        sizes[0] = 20
        rest = self.rows - sum(sizes)
        self.held.copy_(ints([rng.choice([0, 1, 300, self.longest - 20]) for _ in sizes]))
        self.brought.copy_(ints(sizes))
        self.parents.copy_(ints([p for k in sizes for p in refs.tree(k, seed)] + [-1] * rest))
        self.ids.copy_(torch.randint(0, 3, (self.rows,), generator=g, device="cuda"))
        self.owner.copy_(ints(np.repeat(np.arange(self.n), sizes).tolist() + [0] * rest))
        self.pages.copy_(torch.randn(self.pages.shape, generator=g, device="cuda"))
        self.q.copy_(torch.randn(self.q.shape, generator=g, device="cuda"))
        self.logits.copy_(torch.randn(self.logits.shape, generator=g, device="cuda"))
        self.logits[:, :3] += 20  # the choice lies among the drafts
        self.history.tokens.copy_(torch.randint(0, VOCAB, self.history.tokens.shape, generator=g, device="cuda"))
        self.history.lengths.copy_(ints([rng.randint(0, 50) for _ in sizes]))
        self.penalty.copy_(torch.rand(self.n, generator=g, device="cuda"))
        # (a row behind the last request's belongs to no tree: it is given the first row's)
        self.which.copy_(ints([*range(sum(sizes)), *([0] * rest)]))

    def run(self):
        made = ops.step_tables(self.held, self.brought, [self.lists], PAGE, self.rows, parents=self.parents, most=20)
        table, slots = made.groups[0]
        step = StepContext(num_tokens=self.rows, num_seqs=self.n, token_ids=self.ids, positions=made.positions, cu_seqlens=made.cu_seqlens,
                           seq_lens=made.seq_lens, state_slots=self.held, fresh=self.held, logit_rows=self.which, q_lens=[], seq_lens_host=[], max_q_len=20,
                           max_seq_len=self.longest, decode_only=False, groups={0: made.groups[0]}, tree=made.tree)
        out = ops.paged_attention(self.q, KVView(self.pages[1], table, slots, PAGE, None, spec=self.spec), step, self.d ** -0.5)
        adjusted = ops.adjust_logits(self.logits, history=self.history, frequency=self.penalty, presence=self.penalty, requests=self.owner,
                                     drafted=ops.DraftedRows(made.tree, self.ids, made.cu_seqlens, self.which))
        accepted = ops.accept_drafts(adjusted.argmax(1).int(), self.ids, made.tree, made.cu_seqlens)
        held = made.seq_lens - (made.cu_seqlens[1:] - made.cu_seqlens[:-1])
        ops.keep_rows(self.pages, self.spec.rows, PAGE, table, held, accepted)
        return out, made.positions, made.cu_seqlens, slots, table, adjusted, accepted.path, accepted.kept, accepted.tokens

    def answer(self, made):
        """What the step made, but for rows that no request has."""
        total = int(made[2][-1])
        return [made[0][:total], *made[1:], self.pages]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b, strict=True))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_two_captured_steps_in_turn(way, dtype):
    """Steps of two shapes, captured and replayed in turn on inputs that they were not captured with, have what the calls would have."""
    steps, graphs, outs = [WholeStep(n, dtype=dtype) for n in (3, 7)], [], []
    for s in steps:
        s.take(1)
        s.run()
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(s.run())
    kept = 0
    for seed in range(2, 6):
        expect = []
        for s in steps:
            s.take(seed)
            expect.append([x.clone() for x in s.answer(s.run())])
            kept += int(expect[-1][7].sum()) - s.n
        for s in steps:
            s.take(seed)
        for graph in graphs:
            graph.replay()
        for s, out, wanted in zip(steps, outs, expect):
            assert same(s.answer(out), wanted)
    assert kept > 10


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_two_streams_at_once(way, dtype):
    """Steps on two streams that run side by side, again and again, each behind work of its own."""
    steps, streams = [WholeStep(n, dtype=dtype, longest=3200) for n in (4, 5)], [torch.cuda.Stream(), torch.cuda.Stream()]
    expect = []
    for i, s in enumerate(steps):
        s.take(i)
        expect.append([x.clone() for x in s.answer(s.run())])
    busy = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    for _ in range(5):
        made = []
        for i, (s, stream) in enumerate(zip(steps, streams)):
            with torch.cuda.stream(stream):
                for _ in range(2):
                    busy @ busy
                s.take(i)
        for s, stream in zip(steps, streams):
            with torch.cuda.stream(stream):
                made.append(s.run())
        torch.cuda.synchronize()
        for s, got, wanted in zip(steps, made, expect):
            assert same(s.answer(got), wanted)


@pytest.mark.parametrize("layout", [(16, 8, 128, BF16, 16), (4, 4, 128, F32, 16), (2, 1, 200, F32, 16), (5, 1, 96, BF16, 8), (4, 2, 130, F32, 16)], ids=str)
def test_a_query_that_is_no_number_has_no_number(layout, way):
    """Long enough that many blocks have part in a row; the other rows are as ever."""
    nq, nkv, d, dtype, page = layout
    c = make(nq, nkv, d, dtype, page, [(5000, refs.tree(9, 1)), (40, refs.tree(5, 2))], seed=2)
    good = ops.paged_attention(c.q, c.kv, c.step, d ** -0.5).view(-1, nq, d)
    for value in (math.nan, math.inf):
        q = c.q.clone()
        q[3, nq - 1, 0], q[11, 0, d - 1] = value, value
        got = ops.paged_attention(q, c.kv, c.step, d ** -0.5).view(-1, nq, d)
        bad = torch.zeros(len(q), nq, dtype=torch.bool, device="cuda")
        bad[3, nq - 1] = bad[11, 0] = True
        assert torch.isnan(got[bad]).all() and torch.equal(got[~bad], good[~bad])


@pytest.mark.parametrize("layout", [(16, 8, 128, BF16, 16), (8, 2, 64, BF16, 16), (4, 4, 128, F32, 16), (4, 2, 130, F32, 16), (5, 1, 96, BF16, 8)], ids=str)
@pytest.mark.parametrize("n", [3, 64])
def test_a_key_that_is_no_number_reaches_all_who_see_it(layout, n, way):
    """Also where it is all that a row sees of a tile, whoever has that tile."""
    nq, nkv, d, dtype, page = layout
    rng = random.Random(n)
    c = make(nq, nkv, d, dtype, page, [(128 * rng.randint(1, 12), refs.chain(3) if r % 2 else [-1, -1, -1]) for r in range(n)], seed=n)
    for r, (first, nodes, k, *_) in enumerate(c.requests):
        held = len(k) - nodes
        c.kv.row(0)[int(c.kv.block_table[r, held // page]), :, held % page, 1] = math.nan  # the first node's
    got = ops.paged_attention(c.q, c.kv, c.step, d ** -0.5).view(n, 3, nq, d)
    assert torch.isnan(got[1::2]).all()  # a chain: all see it
    assert torch.isnan(got[0::2, 0]).all() and torch.isfinite(got[0::2, 1:]).all()


def test_pages_beyond_31_bits(way):
    """A pool of 5 GB: pages whose first element lies beyond 2^31, attended to and moved within."""
    nkv, d, pages = 8, 128, 72_000
    for dtype, count in ((BF16, pages), (F32, pages)):
        store = torch.empty(1, count, 2, nkv, PAGE, d, dtype=dtype, device="cuda")
        c = make(16, nkv, d, dtype, PAGE, [(100, refs.tree(12, 1)), (900, refs.tree(7, 3))], seed=1)
        far = count - c.kv.pages.shape[0]
        store[0, far:] = c.kv.pages
        table = torch.where(c.kv.block_table >= 0, c.kv.block_table + far, c.kv.block_table)
        got = ops.paged_attention(c.q, KVView(store[0], table, c.kv.slot_mapping, PAGE, None, spec=c.kv.spec), c.step, d ** -0.5)
        check(c, d ** -0.5, call=lambda **_: got)
        path = ints([[0, 2, 5] + [-1] * 29, [0, 1, 6] + [-1] * 29])
        accepted = ops.Accepted(path, ints([3, 3]), ints([0, 0]))
        ops.keep_rows(store, c.kv.spec.rows, PAGE, table, ints([100, 900]), accepted)
        ops.keep_rows(c.kv.pages[None], c.kv.spec.rows, PAGE, c.kv.block_table, ints([100, 900]), accepted)
        assert torch.equal(store[0, far:].view(torch.uint8), c.kv.pages.view(torch.uint8))
        del store


def test_logits_beyond_31_bits():
    """17,000 rows of 131,072 logits: 9 GB."""
    rows, vocab = 17_000, 131_072
    logits = torch.zeros(rows, vocab, device="cuda")
    ids = torch.arange(rows, dtype=torch.int32, device="cuda")
    bias = ops.LogitBias(ids, torch.full((rows,), 2.5, device="cuda"), torch.arange(rows + 1, dtype=torch.int32, device="cuda"))
    assert ops.adjust_logits(logits, bias=bias, out=logits) is logits
    assert float(logits.sum(dtype=torch.float64)) == 2.5 * rows and bool((logits.diagonal() == 2.5).all())
    masks = ops.TokenMasks(torch.ones(1, vocab // 32, dtype=torch.int32, device="cuda"), torch.where(ids >= rows - 2, 0, -1).int())
    ops.adjust_logits(logits, masks=masks, out=logits)
    assert bool(torch.isfinite(logits[: rows - 2]).all())
    assert torch.isfinite(logits[rows - 2:]).sum(1).tolist() == [vocab // 32] * 2


@pytest.mark.parametrize("layout", [(16, 8, 128, BF16, 16), (4, 4, 128, F32, 16), (4, 2, 130, F32, 16)], ids=str)
def test_windows_beyond_31_bits(layout, way):
    """As wide as a number can be said: all that is held, with or without kept positions."""
    nq, nkv, d, dtype, page = layout
    for window, keep in ((1 << 40, 0), ((1 << 31) - 1, 5), (1 << 31, 1 << 33)):
        check_window(make(nq, nkv, d, dtype, page, [(300, refs.tree(9, 1)), (1, [-1])], window=window, keep=keep), d, window, keep)
    with pytest.raises(ops.KernelError):
        ops.tree_attention(*(lambda c: (c.q, c.kv, c.step, 0.1))(make(nq, nkv, d, dtype, page, [(30, [-1])])), window=-2)


def test_the_most_requests_and_the_next():
    """1,024 requests go by equal shares, more by the kernel for any shape; tables of 65,534, and no more."""
    for n in (1024, 1025):
        c = make(2, 1, 64, BF16, 16, [(r % 5, [-1]) for r in range(n)], seed=n)
        check(c, 0.125)
    n = 65_534
    held = torch.arange(n, dtype=torch.int32, device="cuda") % 3
    lists = ops.PageLists(torch.arange(n, dtype=torch.int32, device="cuda"), torch.arange(n, device="cuda"), 1)
    made = ops.step_tables(held, torch.ones_like(held), [lists], 4, n + 3)
    assert torch.equal(made.positions[:n], held) and made.positions[n:].tolist() == [-1] * 3
    assert torch.equal(made.groups[0][1][:n], torch.arange(n, device="cuda") * 4 + held) and int(made.cu_seqlens[-1]) == n
    with pytest.raises(ops.KernelError):
        ops.step_tables(torch.zeros(n + 1, dtype=torch.int32, device="cuda"), torch.ones(n + 1, dtype=torch.int32, device="cuda"), [lists], 4, n + 3)


def test_one_token_brought_to_nothing_held():
    """The smallest step there is."""
    made = ops.step_tables(ints([0]), ints([1]), [], 16, 1, most=1)
    assert (made.positions.tolist(), made.cu_seqlens.tolist(), made.seq_lens.tolist(), made.tree.ancestors.tolist()) == ([0], [0, 1], [1], [[1]])
    none = ops.step_tables(ints([5]), ints([0]), [], 16, 0, most=1)
    assert none.positions.shape == (0,) and none.cu_seqlens.tolist() == [0, 0] and none.seq_lens.tolist() == [5]
    accepted = ops.accept_drafts(ints([4]), ints([9]), made.tree, made.cu_seqlens)
    assert (accepted.kept.tolist(), accepted.tokens.tolist(), accepted.path[0, :2].tolist()) == ([1], [4], [0, -1])
    assert ops.adjust_logits(torch.zeros(0, 5, device="cuda")).shape == (0, 5)
    c = make(2, 1, 64, BF16, 16, [(0, [-1])])
    check(c, 0.125)
