"""Attention over positions that requests share, copies of cache pages and of per-request state, and
answers that share a prompt, on the GPU, against plain 64-bit attention and plain copies."""

from __future__ import annotations

import dataclasses
import importlib
import math
import random

import pytest
import torch

import plain_impl
import tiny_configs
from mlx_omnia_b200 import GenerationOptions, load
from mlx_omnia_b200.cache import CacheManager
from mlx_omnia_b200.engine.engine import Engine, EngineArgs
from mlx_omnia_b200.engine.generate import Generator
from mlx_omnia_b200.kernels import ops
from mlx_omnia_b200.parts.base import KVSpec, KVView, StateSpec, StepContext
from mlx_omnia_b200.parts.model import CacheNeed
from trace_tools import write_folder

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def share_whatever_there_is(monkeypatch):
    monkeypatch.setattr(ops, "SHARED_LEAST_BYTES", 0)


@pytest.fixture(params=["tiles of the tensor-core kernel", "rows of the decode kernel", "by size"])
def way(request, monkeypatch):
    """Both kernels that take shared positions of bfloat16, at every size."""
    most = {"tiles of the tensor-core kernel": 0, "rows of the decode kernel": 1 << 60}.get(request.param)
    if most is not None:
        monkeypatch.setattr(ops, "ROWS_MOST_BYTES", most)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@dataclasses.dataclass
class Case:
    q: torch.Tensor
    rows: torch.Tensor  # the gate's columns behind as many of something else
    kv: KVView
    step: StepContext
    lengths: list
    ks: list  # [positions, nkv, d] of every request, in 64 bits
    vs: list
    sink: torch.Tensor


def make(nq, nkv, d, dtype, page, groups, *, dv=None, alone=(5,), padding=1, seed=0, spread=1.0):
    """`groups`: (shared positions, what each request holds beyond them); `alone`: lengths of requests that share nothing. Requests come
    in any order, pages in any; whatever no request holds is NaN."""
    dv = d if dv is None else dv
    rng = random.Random(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    requests = [(i, positions + own) for i, (positions, owns) in enumerate(groups) for own in owns] + [(None, n) for n in alone]
    order = list(range(len(requests)))
    rng.shuffle(order)
    requests = [requests[i] for i in order]
    lengths = [n for _, n in requests]
    width = max(-(-n // page) for n in lengths) + 1
    table, taken, first = [], 0, {}
    for of, n in requests:
        row = [-1] * width
        whole = groups[of][0] // page if of is not None else 0
        if of in first and of is not None:
            row[:whole] = first[of][:whole]
        else:
            row[:whole] = range(taken, taken + whole)
            taken += whole
            if of is not None:
                first[of] = row
        for i in range(whole, -(-n // page)):
            row[i] = taken
            taken += 1
        table.append(row)
    where = list(range(taken + 3))
    rng.shuffle(where)
    table = [[where[p] if p >= 0 else -1 for p in row] for row in table]
    ks_of = [torch.randn(positions, nkv, d, generator=g, device="cuda").to(dtype) for positions, _ in groups]
    vs_of = [torch.randn(positions, nkv, dv, generator=g, device="cuda").to(dtype) for positions, _ in groups]
    spec = KVSpec(((nkv, d), (nkv, dv)))
    elements = nkv * (d + dv) * page
    pages = torch.full((taken + 3, elements), float("nan"), device="cuda", dtype=dtype)
    k_view = pages[:, : nkv * d * page].view(-1, nkv, page, d)
    v_view = pages[:, nkv * d * page:].view(-1, nkv, page, dv)
    ks, vs = [], []
    for row, (of, n) in zip(table, requests):
        k = torch.randn(n, nkv, d, generator=g, device="cuda").to(dtype)
        v = torch.randn(n, nkv, dv, generator=g, device="cuda").to(dtype)
        if of is not None:
            k[: groups[of][0]], v[: groups[of][0]] = ks_of[of], vs_of[of]
        at = torch.arange(n, device="cuda")
        held = torch.tensor(row, device="cuda")[at // page]
        k_view[held, :, at % page], v_view[held, :, at % page] = k, v
        ks.append(k.double())
        vs.append(v.double())
    n = len(lengths) + padding
    q = (spread * torch.randn(n, nq, d, generator=g, device="cuda")).to(dtype)
    rows = torch.randn(n, 3 + nq * dv, generator=g, device="cuda").to(dtype)
    shared = tuple((positions, tuple(i for i, (of, _) in enumerate(requests) if of == j)) for j, (positions, _) in enumerate(groups))
    pad = [0] * padding
    step = StepContext(num_tokens=n, num_seqs=n, token_ids=ints([0] * n), positions=ints([x - 1 for x in lengths + pad]),
                       cu_seqlens=ints(list(range(n + 1))), seq_lens=ints(lengths + pad), state_slots=ints([0] * n), fresh=ints([0] * n),
                       logit_rows=ints([]), q_lens=[1] * n, seq_lens_host=lengths + pad, max_q_len=1, max_seq_len=max(lengths),
                       decode_only=True, groups={}, shared=shared)
    kv = KVView(pages if d != dv else pages.view(-1, 2, nkv, page, d), ints(table + [[-1] * width] * padding),
                torch.full((n,), -1, dtype=torch.int64, device="cuda"), page, None, spec=spec)
    return Case(q, rows, kv, step, lengths, ks, vs, torch.randn(nq, generator=g, device="cuda"))


def plain(case, scale, *, gate=False, sink=False, softcap=0.0, difference=None):
    """-> (answers, bounds on what they may be off by) of every request, in 64 bits.

    A float32 sum of products of d terms in any order is off by up to (d + 8) 2^-24 of the sum of their absolute values, and so is a score z (a cap
    adds what its float32 form is off by, 2^-20 of the cap); a weight e^z is then off by that much of itself and 2^-20 for the exponential, twice
    since the sum of the weights divides it. Weights and values are summed in tiles of 128 at most and joined over at most 400
    pieces: 600 * 2^-24. In bfloat16, whose eight bits round to the nearest by up to 2^-8 of a number, the weights are rounded ahead of the second product
    and the answer after it. All of it times sum p |v|."""
    nq, nkv = case.q.shape[1], case.ks[0].shape[1]
    group, half = nq // nkv, case.q.dtype == BF16
    answers, bounds = [], []
    for r, (k, v) in enumerate(zip(case.ks, case.vs)):
        q = case.q[r].double().view(nkv, group, -1)
        z = torch.einsum("kxd,pkd->kxp", q, k) * scale
        size = (torch.einsum("kxd,pkd->kxp", q.abs(), k.abs()) * abs(scale)).amax(2)
        if softcap:
            z = softcap * torch.tanh(z / softcap)
        every = torch.cat([z, case.sink.double().view(nkv, group, 1)], 2) if sink else z
        p = torch.softmax(every, 2)[..., : z.shape[2]]
        out = torch.einsum("kxp,pkd->kxd", p, v).reshape(nq, -1)
        most = torch.einsum("kxp,pkd->kxd", p, v.abs()).reshape(nq, -1)
        off = 2 * ((case.q.shape[2] + 8) * 2.0 ** -24 * size + softcap * 2.0 ** -20 + 2.0 ** -20) + 600 * 2.0 ** -24 + (2.0 ** -8 if half else 0.0)
        bound, rounding = off.reshape(nq, 1) * most, 2.0 ** -8 if half else 2.0 ** -24
        if difference is not None:
            dv = difference.dv
            pair = out.view(nq // 2, 2, -1)[..., :dv]
            a = pair[:, 0] - difference.lam * pair[:, 1]
            e = (bound.view(nq // 2, 2, -1)[..., :dv] * torch.tensor([1.0, abs(difference.lam)], dtype=torch.float64, device="cuda").view(1, 2, 1)).sum(1)
            rms = torch.sqrt(a.square().mean(1, keepdim=True) + difference.eps)
            out = a / rms * difference.factor
            bound = abs(difference.factor) * e / rms + out.abs() * torch.sqrt(e.square().mean(1, keepdim=True)) / rms
            bound = 1.01 * bound  # (second order)
        out, bound = out.reshape(-1), bound.reshape(-1)
        if gate:
            s = torch.sigmoid(case.rows[r, 3:].double())
            out, bound = out * s, bound * s
        answers.append(out)
        bounds.append(bound + (rounding + 2.0 ** -20) * out.abs() + 1e-30)
    return torch.stack(answers), torch.stack(bounds)


def check(case, scale=None, *, gate=False, sink=False, softcap=0.0, difference=None, run=None):
    scale = case.q.shape[2] ** -0.5 if scale is None else scale
    run = run or ops.paged_attention
    got = run(case.q, case.kv, case.step, scale, gate=case.rows if gate else None, gate_col=3, sink=case.sink if sink else None, softcap=softcap,
              **({} if difference is None else {"difference": difference}))
    ops.raise_on_error(case.q.device)
    expect, bound = plain(case, scale, gate=gate, sink=sink, softcap=softcap, difference=difference)
    off = (got[: len(case.lengths)].double() - expect).abs()
    assert torch.isfinite(got[: len(case.lengths)]).all()
    assert float((off / bound).max()) <= 1.0, float((off / bound).max())
    return got


LAYOUTS = {
    "16/8x128": (16, 8, 128, BF16, 16), "32/8x128": (32, 8, 128, BF16, 48), "6/2x64": (6, 2, 64, BF16, 32), "2/2x64": (2, 2, 64, BF16, 16),
    "32/2x128": (32, 2, 128, BF16, 16), "8/1x64": (8, 1, 64, BF16, 64), "8/4x64": (8, 4, 64, BF16, 16),
    "8/1x24 f32": (8, 1, 24, F32, 8), "4/2x128 f32": (4, 2, 128, F32, 16), "5/5x7 f32": (5, 5, 7, F32, 3), "34/1x64 f32": (34, 1, 64, F32, 16),
    "3/1x256 f32": (3, 1, 256, F32, 16), "2/1x512 f32": (2, 1, 512, F32, 4), "34/2x64": (34, 2, 64, BF16, 16),
    "16/8x128 p8": (16, 8, 128, BF16, 8), "8/8x96": (8, 8, 96, BF16, 16), "8/2x256": (8, 2, 256, BF16, 16), "6/2x24": (6, 2, 24, BF16, 5),
}
GROUPS = {
    "one position": [(1, [1, 1, 7])], "a page": [(16, [1, 2])], "inside a page": [(17, [3, 1, 40]), (30, [1, 1])],
    "a tile and its ends": [(127, [1, 5]), (128, [2, 2]), (129, [1, 130])], "many pieces": [(1111, [9, 1, 200, 77, 64])],
    "many requests": [(260, [1 + i % 37 for i in range(70)])], "one request": [(200, [5])],
}


@pytest.mark.parametrize("groups", GROUPS, ids=str)
@pytest.mark.parametrize("layout", LAYOUTS)
def test_attention(layout, groups, way):
    nq, nkv, d, dtype, page = LAYOUTS[layout]
    check(make(nq, nkv, d, dtype, page, GROUPS[groups], seed=len(layout)))


@pytest.mark.parametrize("options", [{"gate": True}, {"sink": True}, {"softcap": 3.0}, {"gate": True, "sink": True, "softcap": 30.0}], ids=str)
@pytest.mark.parametrize("layout", LAYOUTS)
def test_gates_sinks_and_caps(layout, options, way):
    nq, nkv, d, dtype, page = LAYOUTS[layout]
    check(make(nq, nkv, d, dtype, page, [(333, [1, 66, 20]), (64, [64, 1])], seed=3), **options)


@pytest.mark.parametrize("layout", ["16/8x128", "8/4x64", "8/1x64", "8/1x24 f32", "4/2x128 f32", "8/2x256"])
def test_the_difference_of_two_maps(layout, way):
    nq, nkv, d, dtype, page = LAYOUTS[layout]
    last = ops.MapDifference(0.7, 1e-5, 0.4, d - 4)
    check(make(nq, nkv, d, dtype, page, [(333, [1, 66, 20]), (64, [64, 1])], seed=3), difference=last)


@pytest.mark.parametrize("nq,nkv,d,dv,dtype", [(8, 2, 48, 32, F32), (4, 1, 33, 70, F32), (8, 2, 64, 32, BF16), (4, 4, 20, 128, BF16)])
def test_values_of_another_width(nq, nkv, d, dv, dtype):
    check(make(nq, nkv, d, dtype, 8, [(100, [1, 30, 9]), (31, [4, 4])], dv=dv), gate=True)


@pytest.mark.parametrize("layout", ["16/8x128", "32/8x128", "6/2x64", "32/2x128"])
@pytest.mark.parametrize("positions,members,own", [(9000, 3, 40), (2051, 64, 100), (5000, 150, 9), (20000, 33, 2)])
def test_long_positions_and_many_rows(layout, positions, members, own, way):
    nq, nkv, d, dtype, page = LAYOUTS[layout]
    check(make(nq, nkv, d, dtype, page, [(positions, [1 + (7 * i) % own for i in range(members)])], alone=(700, 1)), gate=True)


@pytest.mark.parametrize("layout", ["16/8x128", "6/2x64", "8/1x24 f32"])
def test_scores_far_apart(layout, way):
    """Weights that a single key takes, and maxima that move from tile to tile."""
    nq, nkv, d, dtype, page = LAYOUTS[layout]
    check(make(nq, nkv, d, dtype, page, [(1500, [1, 300]), (777, [50, 2, 9])], seed=5, spread=12.0), sink=True)


@pytest.mark.parametrize("layout", ["16/8x128", "6/2x64", "8/1x24 f32"])
@pytest.mark.parametrize("scale", [1e-4, 1.0, -0.1])
def test_scales(layout, scale, way):
    nq, nkv, d, dtype, page = LAYOUTS[layout]
    check(make(nq, nkv, d, dtype, page, [(300, [1, 90])], seed=6), scale)


@pytest.mark.parametrize("layout", ["16/8x128", "32/8x128", "6/2x64", "8/1x24 f32", "34/2x64"])
@pytest.mark.parametrize("cap", [0.5, 3.0])
def test_capped_scores_beyond_what_float32_holds(layout, cap, way):
    """Scores of +-2^128 and more are infinite in float32, and capped all the same: keys weigh e^c or e^-c by their sign.

    A weight is off by the exponential's and the cap's 2^-20 (see `plain`), their sum likewise; sums and joins 600 * 2^-24; in bfloat16 the weights' and
    the answer's rounding, 2^-8 each."""
    nq, nkv, d, dtype, page = LAYOUTS[layout]
    case = make(nq, nkv, d, dtype, page, [(700, [1, 30, 77])], seed=12)
    case.q = torch.full_like(case.q, 2.0 ** 64)
    # The same sign all over a position's key: the sign of its first dim.
    elements = nkv * d * page
    k_view = case.kv.pages.view(case.kv.pages.shape[0], -1)[:, :elements].view(-1, nkv, page, d)
    sign = torch.where(k_view[..., :1] < 0, -1.0, 1.0).to(dtype)
    k_view.copy_(torch.where(torch.isnan(k_view), k_view, sign * 2.0 ** 64))
    got = ops.paged_attention(case.q, case.kv, case.step, d ** -0.5, softcap=cap)
    ops.raise_on_error(case.q.device)
    half = dtype == BF16
    for r, (k, v) in enumerate(zip(case.ks, case.vs)):
        p = torch.softmax(torch.where(k[..., 0] < 0, -cap, cap).double(), 0)  # [positions, nkv]
        out, most = torch.einsum("pk,pkd->kd", p, v), torch.einsum("pk,pkd->kd", p, v.abs())
        off = 2 * (cap * 2.0 ** -20 + 2.0 ** -20) + 600 * 2.0 ** -24 + (2.0 ** -8 if half else 0.0)
        bound = off * most + ((2.0 ** -8 if half else 2.0 ** -24) + 2.0 ** -20) * out.abs() + 1e-30
        mine = got[r].double().view(nkv, nq // nkv, -1)
        assert float(((mine - out[:, None]).abs() / bound[:, None]).max()) <= 1.0


@pytest.mark.parametrize("layout", ["16/8x128", "2/2x64", "8/1x24 f32"])
def test_what_no_request_holds_does_not_matter(layout, way):
    """The pages' unused rows are NaN above; infinities and the lowest numbers there give the same bits."""
    nq, nkv, d, dtype, page = LAYOUTS[layout]
    case = make(nq, nkv, d, dtype, page, [(203, [1, 30, 77])], seed=7)
    got = check(case)
    unused = case.kv.pages.isnan()
    for value in (math.inf, -math.inf, torch.finfo(dtype).min):
        case.kv.pages[unused] = value
        assert torch.equal(ops.paged_attention(case.q, case.kv, case.step, d ** -0.5)[: len(case.lengths)], got[: len(case.lengths)])


@pytest.mark.parametrize("layout", ["16/8x128", "32/8x128", "34/1x64 f32"])
def test_the_same_call_gives_the_same_bits(layout, way):
    nq, nkv, d, dtype, page = LAYOUTS[layout]
    case = make(nq, nkv, d, dtype, page, [(4111, [1, 300, 12, 64, 5])], seed=8)
    n, first = len(case.lengths), None
    for _ in range(6):
        got = ops.paged_attention(case.q, case.kv, case.step, d ** -0.5)[:n]
        first = got if first is None else first
        assert torch.equal(got, first)


@pytest.mark.parametrize("layout", ["16/8x128", "8/1x24 f32"])
def test_pages_beyond_32_bits_of_elements(layout, way):
    """Pages whose elements are counted in more than 31 bits: the held pages are moved to the end of a tensor of that many."""
    nq, nkv, d, dtype, page = LAYOUTS[layout]
    case = make(nq, nkv, d, dtype, page, [(203, [1, 30, 77])], seed=9)
    small = case.kv.pages
    count = (1 << 32) // small[0].numel() + small.shape[0] + 5
    big = torch.empty(count, *small.shape[1:], dtype=dtype, device="cuda")
    big[count - small.shape[0]:] = small
    table = torch.where(case.kv.block_table >= 0, case.kv.block_table + (count - small.shape[0]), -1)
    case.kv = dataclasses.replace(case.kv, pages=big, block_table=table)
    check(case)


@pytest.mark.parametrize("layout", ["16/8x128", "4/2x128 f32"])
def test_on_another_stream(layout, way):
    nq, nkv, d, dtype, page = LAYOUTS[layout]
    case = make(nq, nkv, d, dtype, page, [(2000, [1, 300, 12])], seed=10)
    side = torch.cuda.Stream()

    def run(*args, **more):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            out = ops.paged_attention(*args, **more)
        torch.cuda.current_stream().wait_stream(side)
        return out

    got = check(case, run=run)
    case.step.workspace = None
    assert torch.equal(check(case)[: len(case.lengths)], got[: len(case.lengths)])


@pytest.mark.parametrize("layout", ["16/8x128", "32/8x128", "8/1x24 f32", "8/8x96"])
def test_a_captured_step_serves_other_groups(layout, way):
    nq, nkv, d, dtype, page = LAYOUTS[layout]
    cases = [make(nq, nkv, d, dtype, page, [(positions, [1 + (3 * i) % 50 for i in range(members)])], alone=(9,) * alone, padding=1, seed=seed)
             for seed, positions, members, alone in ((1, 1290, 7, 2), (2, 1400, 5, 4), (3, 1282, 8, 1))]
    shapes = {ops.shared_shape(c.step.shared) for c in cases}
    assert len(shapes) == 1 and len({c.step.num_seqs for c in cases}) == 1
    n, width = cases[0].step.num_seqs, max(c.kv.block_table.shape[1] for c in cases)
    pages = torch.zeros(max(c.kv.pages.shape[0] for c in cases), *cases[0].kv.pages.shape[1:], dtype=dtype, device="cuda")
    q, table, lengths = torch.zeros_like(cases[0].q), ints([[-1] * width] * n), ints([0] * n)
    step = dataclasses.replace(cases[0].step, seq_lens=lengths, seq_lens_host=[], shared=(), shared_shape=shapes.pop(), max_own=64,
                               max_seq_len=width * page, workspace={"private": True})
    kv = dataclasses.replace(cases[0].kv, pages=pages, block_table=table)
    ops.paged_attention(q, kv, step, d ** -0.5)  # nobody holds anything: the lists and the scratch memory are made
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.paged_attention(q, kv, step, d ** -0.5)
    for case in [*cases, cases[0]]:
        pages[: case.kv.pages.shape[0]] = case.kv.pages
        q.copy_(case.q)
        table.fill_(-1)
        table[:, : case.kv.block_table.shape[1]] = case.kv.block_table
        lengths.copy_(case.step.seq_lens)
        step.shared = case.step.shared
        ops.fill_step_lists(step)
        graph.replay()
        check(case, run=lambda *a, **k: out.clone())
        torch.cuda.synchronize()


@pytest.mark.parametrize("layout,positions,owns", [("16/8x128", 1000, [2000 - 7 * i for i in range(17)]), ("16/8x128", 1000, [1000 - 9 * i for i in range(9)]),
                                                   ("32/8x128", 9000, [900 - 3 * i for i in range(33)]), ("6/2x64", 1290, [1500 - i for i in range(19)]),
                                                   ("8/2x256", 2000, [1100 - 5 * i for i in range(9)]), ("8/1x24 f32", 700, [900 - 4 * i for i in range(11)])])
def test_a_captured_step_has_the_bits_of_one_that_is_not(layout, positions, owns, way):
    """Requests rounded up to a power of two, as the engine's captured steps are, and what they hold beyond the group to a bound."""
    nq, nkv, d, dtype, page = LAYOUTS[layout]
    case = make(nq, nkv, d, dtype, page, [(positions, owns)], alone=(), padding=0, seed=11)
    eager = check(case)
    n = len(owns)
    batch, width = 1 << (n - 1).bit_length(), ops.width_bucket(case.kv.block_table.shape[1])
    q, table = torch.zeros(batch, nq, d, dtype=dtype, device="cuda"), ints([[-1] * width] * batch)
    step = dataclasses.replace(case.step, num_tokens=batch, num_seqs=batch, cu_seqlens=ints(list(range(batch + 1))), seq_lens=ints([0] * batch),
                               seq_lens_host=[], shared=(), shared_shape=ops.shared_shape(case.step.shared), max_own=ops.own_bucket(max(owns), page),
                               max_seq_len=width * page, workspace={"private": True})
    kv = dataclasses.replace(case.kv, block_table=table)
    ops.paged_attention(q, kv, step, d ** -0.5)  # nobody holds anything: the lists and the scratch memory are made
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.paged_attention(q, kv, step, d ** -0.5)
    q[:n], table[:n, : case.kv.block_table.shape[1]], step.seq_lens[:n], step.shared = case.q, case.kv.block_table, case.step.seq_lens, case.step.shared
    ops.fill_step_lists(step)
    graph.replay()
    assert torch.equal(out[:n], eager)
    ops.raise_on_error(q.device)


def test_what_attention_over_shared_positions_refuses():
    case = make(16, 8, 128, BF16, 16, [(64, [1, 30]), (40, [2, 2])], alone=())

    def refuses(match, kv=case.kv, q=case.q, step=case.step, **more):
        with pytest.raises(ops.KernelError, match=match):
            ops.paged_attention(q, dataclasses.replace(kv), dataclasses.replace(step, workspace=None), 0.1, **more)

    refuses("each in one group", step=dataclasses.replace(case.step, shared=((8, (0, 1)), (8, (1, 2)))))
    refuses("more positions than it shares", step=dataclasses.replace(case.step, shared=((5000, (0, 1)),)))
    refuses("than a block table holds", step=dataclasses.replace(case.step, shared=((5000, (0, 1)),), seq_lens_host=[]))
    refuses("at least one position", step=dataclasses.replace(case.step, shared=((0, (0, 1)),)))
    refuses("contiguous", q=case.q.transpose(1, 2).contiguous().transpose(1, 2))
    refuses("of the cache's type", q=case.q.float())
    refuses("a token a request", q=case.q[1:])
    last = ops.MapDifference(0.5, 1e-5, 1.0, 128)
    refuses("no gate", difference=last, gate=case.rows)
    refuses("no more values", difference=dataclasses.replace(last, dv=129))
    projection = ops.Projection(*[case.rows if f.name == "rows" else 16 if f.name == "nq" else 8 if f.name == "nkv" else 128
                                  for f in dataclasses.fields(ops.Projection)])
    refuses("not projected rows", q=None, projection=projection)


def test_a_page_that_is_not_there_is_an_error():
    for layout in ("16/8x128", "8/1x24 f32"):
        nq, nkv, d, dtype, page = LAYOUTS[layout]
        case = make(nq, nkv, d, dtype, page, [(200, [1, 30])], alone=())
        case.kv.block_table[:, 1] = -1
        ops.paged_attention(case.q, case.kv, case.step, 0.1)
        with pytest.raises(ops.KernelError):
            ops.raise_on_error(case.q.device)


@pytest.mark.parametrize("layout", ["16/8x128", "8/1x24 f32", "8/8x96"])
def test_more_of_its_own_than_a_step_was_laid_out_for_is_an_error(layout, way):
    nq, nkv, d, dtype, page = LAYOUTS[layout]
    case = make(nq, nkv, d, dtype, page, [(200, [1, 1900])], alone=())
    case.step.max_own = 64
    ops.paged_attention(case.q, case.kv, case.step, 0.1)
    with pytest.raises(ops.KernelError):
        ops.raise_on_error(case.q.device)
    case.step.workspace, case.step.max_own = None, None
    check(case)


@pytest.mark.parametrize("layout", ["16/8x128", "8/1x24 f32"])
def test_lengths_that_the_host_does_not_know(layout, way):
    nq, nkv, d, dtype, page = LAYOUTS[layout]
    case = make(nq, nkv, d, dtype, page, [(200, [1, 1900, 30])])
    case.step.seq_lens_host = []
    check(case)


@pytest.mark.parametrize("layout", ["16/8x128", "32/8x128", "8/1x24 f32", "8/8x96", "34/2x64"])
@pytest.mark.parametrize("wrong", [200, 150, 1])
def test_lengths_no_longer_than_what_is_shared_are_an_error(layout, wrong, way):
    """Where the host knows the lengths it refuses these; where it does not, the kernels say so."""
    nq, nkv, d, dtype, page = LAYOUTS[layout]
    case = make(nq, nkv, d, dtype, page, [(200, [1, 190, 30])])
    lengths = case.step.seq_lens.clone()
    member = case.step.shared[0][1][1]
    case.step.seq_lens_host, case.step.seq_lens[member] = [], wrong
    ops.paged_attention(case.q, case.kv, case.step, 0.1)
    with pytest.raises(ops.KernelError):
        ops.raise_on_error(case.q.device)
    case.step.seq_lens.copy_(lengths)
    check(case)


@pytest.mark.parametrize("layout", ["16/8x128", "6/2x64"])
def test_queries_off_a_16_byte_boundary(layout, way):
    nq, nkv, d, dtype, page = LAYOUTS[layout]
    case = make(nq, nkv, d, dtype, page, [(200, [1, 190, 30])])
    held = torch.empty(case.q.numel() + 1, dtype=dtype, device="cuda")
    held[1:] = case.q.flatten()
    case.q = held[1:].view_as(case.q)
    check(case)


# -- copies -------------------------------------------------------------------------------------------------------------
def bits(shape, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    size = torch.empty(0, dtype=dtype).element_size()
    return torch.randint(0, 256, (*shape[:-1], shape[-1] * size), generator=g, device="cuda", dtype=torch.uint8).view(dtype)


def same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.parametrize("rows,page", [(((8, 128), (8, 128)), 16), (((2, 24), (2, 24)), 8), (((1, 7), (1, 7)), 5), (((2, 48), (2, 33)), 4), (((1, 576),), 16),
                                       (((3, 1), (1, 3)), 1)])
@pytest.mark.parametrize("dtype", [BF16, F32, torch.uint8])
@pytest.mark.parametrize("seed", range(3))
def test_copies_of_pages(rows, page, dtype, seed):
    rng = random.Random(seed)
    elements, layers, count = sum(h * w for h, w in rows) * page, rng.choice([1, 3, 28]), 700 if seed == 2 else 40
    pages, other = bits((layers, count, elements), dtype, seed), bits((layers, 330, elements), dtype, seed + 1)
    order = rng.sample(range(count), count)
    within = [(order[i], order[count // 2 + i], rng.randint(0, page)) for i in range(count // 2)]
    fork = [(order[0], to, rng.randint(1, page)) for to in order[1: count // 3]]
    across = [(order[i], to, rng.randint(0, page)) for i, to in enumerate(rng.sample(range(330), min(count, 300)))]
    for moves, to in ((within, None), (fork, None), (across, other), ([], None), ([(order[0], order[1], page)], None)):
        got, expect = pages.clone(), pages.clone()
        into = got if to is None else to.clone()
        target = expect if to is None else to.clone()
        for src, dst, n in moves:
            at = 0
            for heads, width in rows:
                block = slice(at, at + heads * page * width)
                target[:, dst, block].view(layers, heads, page, width)[:, :, :n] = pages[:, src, block].view(layers, heads, page, width)[:, :, :n]
                at += heads * page * width
        back = ops.copy_pages(got, rows, page, moves, to=None if to is None else into)
        assert back is into and same(into, target) and (to is None or same(got, pages))


def test_copies_of_pages_of_rows_apart():
    """A page as the cache has it for equal rows: [entries, pages, rows, heads, page size, width]."""
    pages = bits((3, 9, 2, 4, 16, 32), BF16)
    expect = pages.clone()
    expect[:, 5, :, :, :11], expect[:, 0] = expect[:, 2, :, :, :11], expect[:, 3]
    assert same(ops.copy_pages(pages, ((4, 32), (4, 32)), 16, [(2, 5, 11), (3, 0, 16)]), expect)


def test_what_copies_of_pages_refuse():
    rows, pages = ((2, 8), (2, 8)), torch.zeros(2, 6, 2 * 2 * 8 * 4, device="cuda")

    def refuses(match, moves, tensor=pages, rows=rows, page=4, to=None):
        with pytest.raises(ops.KernelError, match=match):
            ops.copy_pages(tensor, rows, page, moves, to=to)

    refuses("outside", [(6, 0, 1)])
    refuses("outside", [(0, 6, 1)])
    refuses("outside", [(-1, 0, 1)])
    refuses("outside", [(1 << 40, 0, 1)])
    refuses("the same place", [(0, 2, 1), (1, 2, 1)])
    refuses("another begins", [(0, 2, 1), (2, 3, 1)])
    refuses("another begins", [(1, 1, 4)])
    refuses("no more rows", [(0, 1, 5)])
    refuses("no more rows", [(0, 1, -1)])
    refuses("moves of", [(0, 1)])
    refuses("do not hold", [(0, 1, 1)], page=5)
    refuses("contiguous", [(0, 1, 1)], tensor=pages[:, ::2])
    refuses("the same layers", [(0, 1, 1)], to=torch.zeros(3, 6, 128, device="cuda"))
    refuses("the same layers", [(0, 1, 1)], to=torch.zeros(2, 6, 128, device="cuda", dtype=BF16))


@pytest.mark.parametrize("seed", range(4))
def test_copies_of_state(seed):
    rng = random.Random(seed)
    count = [5, 17, 65, 600][seed]
    shapes = [((16, 128, 128) if count < 100 else (7, 31), F32), ((5,), torch.int32), ((4, 3, 33), BF16), ((3,), torch.int8), ((1,), torch.int64), ((257,), BF16)]
    tensors = [bits((count + 1, *shape), dtype, i) for i, (shape, dtype) in enumerate(shapes)]
    order = rng.sample(range(count), count)
    for moves in ([(order[0], to) for to in order[1: count // 2 + 1]], [(order[i], order[count // 2 + i]) for i in range(count // 2)], []):
        expect = [t.clone() for t in tensors]
        for t in expect:
            for src, dst in moves:
                t[dst] = t[src]
        ops.copy_slots(tensors, moves)
        assert all(same(a, b) for a, b in zip(tensors, expect))


def test_what_copies_of_state_refuse():
    tensors = [torch.zeros(5, 3, device="cuda"), torch.zeros(6, 2, device="cuda")]
    for match, moves in (("outside", [(0, 5)]), ("outside", [(-1, 0)]), ("the same place", [(0, 2), (1, 2)]), ("another begins", [(0, 1), (1, 2)])):
        with pytest.raises(ops.KernelError, match=match):
            ops.copy_slots(tensors, moves)
    with pytest.raises(ops.KernelError, match="contiguous"):
        ops.copy_slots([torch.zeros(5, 4, device="cuda")[:, ::2]], [(0, 1)])


def test_copies_on_another_stream():
    pages, side = bits((4, 200, 8192), BF16), torch.cuda.Stream()
    expect = pages.clone()
    expect[:, 100:] = expect[:, :100]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        ops.copy_pages(pages, ((4, 64), (4, 64)), 16, [(i, 100 + i, 16) for i in range(100)])
    side.synchronize()
    assert same(pages, expect)


# -- the cache and the engine -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_fork_on_the_device(dtype):
    specs = (KVSpec.keys_and_values(2, 24, None), KVSpec(((2, 6), (2, 4))))
    needs = [CacheNeed(spec, StateSpec((3, 7)), None) for spec in specs for _ in range(3)]
    cache = CacheManager(needs, page_size=4, pages_per_group=20, max_requests=3, dtype=dtype, device="cuda")
    a = cache.open("a")
    cache.grow(a, 11)
    for group in cache.groups:
        group.pages.copy_(torch.randn(group.pages.shape, device="cuda"))
    for tensor, _ in cache.state_tensors():
        tensor.copy_(torch.randn(tensor.shape, device="cuda"))
    before = [g.pages.clone() for g in cache.groups]
    b = cache.fork(a, "b")
    for g, group in enumerate(cache.groups):
        assert b.tables[g][:2] == a.tables[g][:2] and b.tables[g][2] != a.tables[g][2]
        at, flat, old = 0, group.pages.flatten(2), before[g].flatten(2)
        for heads, width in group.spec.rows:
            block = slice(at, at + heads * 4 * width)
            new, held = (t[:, p, block].view(-1, heads, 4, width) for t, p in ((flat, b.tables[g][2]), (old, a.tables[g][2])))
            assert torch.equal(new[:, :, :3], held[:, :, :3])
            at += heads * 4 * width
    assert all(torch.equal(t[a.slot], t[b.slot]) for t, _ in cache.state_tensors())
    held = [[g.pages[:, p].clone() for p in a.tables[i]] for i, g in enumerate(cache.groups)]
    cache.resize(9)
    cache.check()
    assert all(torch.equal(g.pages[:, p], h) for i, g in enumerate(cache.groups) for p, h in zip(a.tables[i], held[i]))


@pytest.mark.parametrize("name,page,graphs", [("A", 4, True), ("B", 8, True), ("B", 8, False)])
def test_greedy_answers_that_share_equal_plain(tmp_path, name, page, graphs):
    raw, weights = write_folder(tmp_path / "m", name)
    vocab = raw["text_config"]["vocab_size"]
    model = load(tmp_path / "m", dtype="float32", page_size=page, cache_tokens=1024, max_requests=16, max_tokens_per_step=24)
    if not graphs:
        model.engine.runner.graphs = model.engine.runner.mixed_graphs = None
    start = tiny_configs.prompt(45, vocab, 1)
    prompts = [start + tiny_configs.prompt(n, vocab, n) for n in (1, 7, 3)] + [start[:-1]]
    expect = [plain_impl.greedy_generate(raw, weights, p, 12) for p in prompts]
    options = GenerationOptions(max_tokens=12, stop=())
    assert model.generate(prompts, options, samples=3) == [ids for ids in expect for _ in range(3)]
    assert model.generate(prompts, options, samples=2, share=True) == [ids for ids in expect for _ in range(2)]
    assert model.generate(prompts, options) == expect
    if graphs:
        assert any(len(key) > 2 for key in model.engine.runner.graphs.captured)
    assert not model.engine.cache.requests
    model.engine.cache.check()


def test_groups_that_no_layer_gains_by_cost_no_capture(tmp_path, monkeypatch):
    """Answers to several short prompts under the rule that a user has: every capture is one that a step without groups would make, and is kept."""
    monkeypatch.undo()
    assert ops.SHARED_LEAST_BYTES > 1 << 20
    write_folder(tmp_path / "m", "C")
    model = load(tmp_path / "m", page_size=16, cache_tokens=8192, max_requests=16, max_tokens_per_step=512)
    graphs, keys = model.engine.runner.graphs, []
    capture = graphs._capture
    monkeypatch.setattr(graphs, "_capture", lambda *key: keys.append(key) or capture(*key))
    prompts = [tiny_configs.prompt(60 + 50 * i, 777, i) for i in range(4)]
    assert len(model.generate(prompts, GenerationOptions(max_tokens=40, stop=()), samples=4)) == 16
    assert keys and all(len(key) == 2 for key in keys)
    assert len(keys) == len(set(keys)) == len(graphs.captured)


def test_answers_in_bfloat16_choose_what_is_nearly_best(tmp_path):
    raw, weights = write_folder(tmp_path / "m", "C")
    model = load(tmp_path / "m", page_size=16, cache_tokens=4096, max_requests=16, max_tokens_per_step=64)
    prompts = [tiny_configs.prompt(n, 777, 40 + n) for n in (5, 150, 290)]
    got = model.generate(prompts, GenerationOptions(max_tokens=10, stop=()), samples=4)
    assert any(len(key) > 2 for key in model.engine.runner.graphs.captured)
    for i, ids in enumerate(got):
        prompt = prompts[i // 4]
        logits = plain_impl.forward(raw, weights, prompt + ids)[len(prompt) - 1: -1]
        chosen = logits[torch.arange(len(ids)), torch.tensor(ids)]
        assert float((logits.max(dim=-1).values - chosen).max()) < 0.03 * float(logits.abs().max())


def test_a_running_engine_whose_cache_is_resized(tmp_path):
    raw, weights = write_folder(tmp_path / "m", "B")
    model = load(tmp_path / "m", dtype="float32", page_size=8, cache_tokens=512, max_requests=4, max_tokens_per_step=64)
    generator: Generator = model.generator
    generator.pipelined = False
    prompts = [tiny_configs.prompt(n, 1000, 30 + n) for n in (5, 33)]
    requests = [generator.add(p, GenerationOptions(max_tokens=12, stop=())) for p in prompts]
    for tokens in (256, 96, 2000):
        generator.step()
        generator.step()
        generator.resize_cache(tokens)
        model.engine.cache.check()
    generator.run()
    ops.raise_on_error(model.engine.runtime.device)
    assert [r.generated for r in requests] == [plain_impl.greedy_generate(raw, weights, p, 12) for p in prompts]


def test_a_pipelined_engine_is_drained_ahead_of_a_resize(tmp_path):
    raw, weights = write_folder(tmp_path / "m", "B")
    model = load(tmp_path / "m", dtype="float32", page_size=8, cache_tokens=512, max_requests=4, max_tokens_per_step=64)
    generator: Generator = model.generator
    assert generator.pipelined
    prompts = [tiny_configs.prompt(n, 1000, 30 + n) for n in (5, 33)]
    requests = [generator.add(p, GenerationOptions(max_tokens=12, stop=())) for p in prompts]
    in_flight = 0
    for tokens in (256, 96, 2000):
        generator.step()
        generator.step()
        if generator._in_flight is not None:
            in_flight += 1
            pages = [g.pages.data_ptr() for g in model.engine.cache.groups]
            with pytest.raises(ValueError, match="in flight"):
                generator.resize_cache(tokens)
            assert [g.pages.data_ptr() for g in model.engine.cache.groups] == pages
        held = sum(len(r.generated) for r in requests)
        assert sum(output.token is not None for output in generator.drain()) == sum(len(r.generated) for r in requests) - held
        generator.resize_cache(tokens)
        model.engine.cache.check()
    assert in_flight
    generator.run()
    ops.raise_on_error(model.engine.runtime.device)
    assert [r.generated for r in requests] == [plain_impl.greedy_generate(raw, weights, p, 12) for p in prompts]


def test_a_cache_that_has_grown_takes_longer_prompts_in_captured_mixed_steps(tmp_path):
    """A prompt longer than the first pools held is read in portions beside a decoding request, in steps of one shape."""
    raw, weights = write_folder(tmp_path / "m", "A")
    model = load(tmp_path / "m", dtype="float32", page_size=4, cache_tokens=128, max_requests=4, max_tokens_per_step=17)
    generator: Generator = model.generator
    generator.resize_cache(2048)
    vocab = raw["text_config"]["vocab_size"]
    prompts = [tiny_configs.prompt(n, vocab, 50 + n) for n in (9, 700)]
    requests = [generator.add(p, GenerationOptions(max_tokens=60, stop=())) for p in prompts]
    generator.run()
    ops.raise_on_error(model.engine.runtime.device)
    assert model.engine.runner.mixed_graphs.replays > 10
    for request, prompt in zip(requests, prompts):
        logits = plain_impl.forward(raw, weights, prompt + request.generated)[len(prompt) - 1: -1]
        chosen = logits[torch.arange(60), torch.tensor(request.generated)]
        assert float((logits.max(dim=-1).values - chosen).max()) <= 1e-4 * float(logits.abs().max())


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("family,name", [("bobarax", "K"), ("bobarax", "L"), ("dolutar", "P"), ("dolutar", "Q"), ("fokalorn", "X"), ("fokalorn", "Y"), ("gisudra", "G"),
                                         ("gisudra", "H"), ("narezen", "P"), ("narezen", "Q"), ("rinirax", "S"), ("rinirax", "T")])
def test_families_with_state_windows_and_latents(family, name, graphs):
    """Recurrent state is copied at the fork, windows and runs share what they still hold: greedy answers that share are those of requests
    of their own, in 32 bits."""
    configs = importlib.import_module(f"{family}_configs")
    raw = configs.config(name)
    engine = Engine.from_tensors(raw, configs.tensors(name), EngineArgs(dtype="float32", page_size=4, cache_tokens=1024, max_requests=8, cuda_graphs=graphs))
    generator = Generator(engine, max_tokens_per_step=16)
    start = configs.prompt(27, engine.vocab_size, 5)
    prompts = [start + configs.prompt(n, engine.vocab_size, n) for n in (1, 6)]
    options = GenerationOptions(max_tokens=9, stop=())
    alone = [generator.generate([p], options)[0] for p in prompts]
    assert generator.generate(prompts, options, samples=3) == [ids for ids in alone for _ in range(3)]
    assert generator.generate(prompts, options, samples=2, share=True) == [ids for ids in alone for _ in range(2)]
    assert not engine.cache.requests
    engine.cache.check()
