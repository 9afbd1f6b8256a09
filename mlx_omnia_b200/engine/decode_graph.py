"""Decode steps as replayed CUDA graphs.

A step in which every request brings one token launches some three hundred small
kernels; issued one by one from Python they cost more host time than the GPU needs to
run them. Such steps are therefore captured once per *bucket* (requests rounded up to
a power of two, block-table width rounded up to three significant bits; where requests share
positions, the rounded sizes of their groups and of what each holds beyond them) and replayed: the
host writes the step's metadata into one pinned buffer, one copy brings it to the
device buffer the captured kernels read, and the graph runs. Rows beyond the live
requests are padding: sequence length 0, cache slot -1, position -1, which every kernel
treats as "nothing to do", and the scratch state slot, which belongs to no request (so
a mixer with state of its own may read and write it freely). The metadata is laid out
and filled by the same `StepLayout` as an uncaptured step's.

At most `MAX_GRAPHS` captured graphs are kept; the one replayed longest ago is dropped
for a new bucket (each holds its own logits, activations and scratch buffers).

Mixed steps (`MixedGraphs`). A step of a few hundred tokens, portions of prompts beside
decoded tokens, launches some 230 kernels one by one from Python and is bound by the host
(16 us a launch) long before the GPU. In continuous batching such steps repeat in shape:
the same requests decode while a long prompt is read in portions of the token budget. So
a step whose shape (tokens per request, wanted rows per request, the bucket of the
longest decoding request, the width of the block tables: the next power of two above the
longest request's pages, so a prompt doubles before it leaves its graph; whether its
prompts all start at their first token, which kernels are chosen by) comes for the
third time is captured with exactly that shape, and replayed whenever it comes again. The
small lists that the attention kernels read (which block of query tokens runs where) are
given a place on the device before the capture and filled by the host before every replay
(`ops.fill_step_lists`). The capturing step runs uncaptured on the buffers the graph will
use (so every scratch buffer and list exists before the capture), and the capture that
follows runs nothing, so a mixer's state is never stepped twice; from its fourth coming on
the shape is replayed. (A capture costs about three steps' time. In a stream of 64 requests
of many lengths most shapes come once or twice: capturing at the second coming, with tables
as wide as the pool, made such a stream twice as slow as launching every step kernel by
kernel.)

Steps of groups. What a capture costs, a step that reads shared positions once gains back in ten
steps (64 requests of 65,536 positions) to thousands (four groups of four answers), and where several
groups come and go their sizes do so within a few dozen steps. So every shape of groups has an
account: each of its steps adds what it gains or would have gained, and its graph (one for every
bound of what requests hold beyond the groups) is captured when that amounts to a capture, which
is taken off. Until then the step runs as one without groups, which needs nothing of them and whose
results round otherwise (`ops.paged_attention`).

Steps of drafted trees (`DraftedGraphs`). Their tables are made on the device from the requests' lengths and lists of pages, by the first kernel of
the step, so one graph serves every step of as many requests, rows, drafts and pages, each rounded up; rows and requests beyond the step's belong to
requests that hold nothing. Such a step too is captured at its third coming, in the way of mixed steps; ahead of that it runs kernel by kernel in the
same rounded shape, since kernels are chosen and their work is cut by it.

The kernels and the model code are the same as in an uncaptured step; only the way
they are launched differs, so logits agree bit for bit with an eager step of the same
bucket, of groups or without. Capture is used only when every mixer of the model declares `graph_safe`
(no host-side loops over requests).

The reference compiles its one-token forward per (mode, batch, capacity) with
mx.compile and pads decode rows to buckets 1/2/4/8
(src/mlx_omnia/engine/core/decode.py:202-317, src/mlx_omnia/engine/batching.py:54,158-220);
CUDA graphs are this engine's counterpart.
"""

from __future__ import annotations

import contextlib
import gc
from dataclasses import dataclass, replace

import numpy as np
import torch

from mlx_omnia_b200.engine.step import DraftedLayout, StepLayout, shared_positions
from mlx_omnia_b200.kernels import ops
from mlx_omnia_b200.parts.base import StepContext, StepTree

MAX_GRAPHS = 24
CAPTURE_GAINS = 1152
"""What a capture of a step of groups costs, in `ops.SHARED_LEAST_BYTES` (24 MB) of a layer's reading. 28 layers, B200: 50 ms, of which the collector 38; after
long prompts, whose memory the allocator gives back ahead of a capture, up to a second; 126 ms on average over a stream of 2 x 16 answers to
prompts of 1,000 to 8,000 tokens. That is 4.5 ms a layer, in which it reads 28 GB."""


@contextlib.contextmanager
def capturing(graph: torch.cuda.CUDAGraph, **options):
    """`torch.cuda.graph` with the garbage collector out of the way. An object that owns a captured
    graph or CUDA memory and is kept alive by reference cycles only (an engine dropped a while ago)
    is freed whenever the collector next runs; if that is in the middle of a capture, freeing it is
    an operation the capturing stream does not permit, and the capture is lost. So what is dead is
    collected before the capture and nothing is collected during it."""
    gc.collect()
    enabled = gc.isenabled()
    gc.disable()
    try:
        with torch.cuda.graph(graph, **options):
            yield
    finally:
        if enabled:
            gc.enable()


def _bucket(n: int) -> int:
    b = 1
    while b < n:
        b *= 2
    return b


@dataclass
class _Captured:
    graph: torch.cuda.CUDAGraph
    step: StepContext
    layout: StepLayout | DraftedLayout
    host_tensor: torch.Tensor  # pinned int32 mirror of `device`
    device: torch.Tensor
    logits: torch.Tensor
    launches: int = 0  # this package's kernels inside the graph (counted at capture)
    copied: torch.cuda.Event | None = None  # the last host-to-device copy of the metadata


class DecodeGraphs:
    def __init__(self, runner) -> None:
        self.runner = runner
        self.captured: dict[tuple, _Captured] = {}  # in order of last use, oldest first
        self.gained: dict[tuple, float] = {}  # by groups' shape: what its steps gain or would have (`ops.sharing_gain`), less its captures
        self.replays = 0

    @staticmethod
    def supported(model) -> bool:
        return all(getattr(block.mixer, "graph_safe", False) for block in model.blocks)

    def _capture(self, batch: int, width: int, shape: tuple = (), own: int | None = None) -> _Captured:
        runner = self.runner
        device = runner.runtime.device
        layout = StepLayout(batch, batch, batch, [width] * len(runner.cache.groups))
        host_tensor = torch.zeros(layout.words, dtype=torch.int32).pin_memory()
        dev = torch.zeros(layout.words, dtype=torch.int32, device=device)
        # Kernels that need scratch memory keep it in the workspace, for as long as the graph lives.
        step = layout.context(dev, q_lens=[1] * batch, seq_lens_host=[], max_q_len=1,
                              max_seq_len=width * runner.cache.page_size, decode_only=True,
                              workspace={"private": True} | runner.ask_for_layers(), shared_shape=shape or None, max_own=own)
        # Padding everywhere, so the warm-up and the capture touch no page.
        layout.fill(host_tensor.numpy(), runner.cache, [], [], np.arange(batch, dtype=np.int32))
        dev.copy_(host_tensor)
        layers = runner.layer_contexts(step)
        side = torch.cuda.Stream(device=device)
        side.wait_stream(torch.cuda.current_stream(device))
        with torch.cuda.stream(side):
            runner.model.forward(step, layers)  # warm-up: loads kernels, sizes library workspaces
        runner.know_layers(step)
        torch.cuda.current_stream(device).wait_stream(side)
        torch.cuda.synchronize(device)
        graph = torch.cuda.CUDAGraph()
        before = ops.launches
        with capturing(graph):
            logits = runner.model.forward(step, layers)
        return _Captured(graph, step, layout, host_tensor, dev, logits, ops.launches - before)

    def _graph_for(self, *key) -> _Captured:
        """`key`: requests and table width, then (where requests share positions) the groups' shape and what a request holds beyond them."""
        captured = self.captured.pop(key, None)
        if captured is None:
            while len(self.captured) >= MAX_GRAPHS:
                oldest = next(iter(self.captured))
                torch.cuda.synchronize(self.runner.runtime.device)  # nothing of it is still running
                del self.captured[oldest]
            captured = self._capture(*key)
        self.captured[key] = captured  # most recently used last
        return captured

    def _affords(self, key: tuple, gain: float) -> bool:
        """Whether a step of groups runs as one: its graph is there, or the steps of this shape, this one among them, are worth its capture."""
        shape = key[2]
        if len(self.gained) > 4096:
            self.gained.clear()
        self.gained[shape] = self.gained.get(shape, 0.0) + gain
        if key in self.captured:
            return True
        if self.gained[shape] < CAPTURE_GAINS * ops.SHARED_LEAST_BYTES:
            return False
        self.gained[shape] -= CAPTURE_GAINS * ops.SHARED_LEAST_BYTES
        return True

    # -- one step ----------------------------------------------------------------------
    def run(self, entries, copy: bool = True, device_tokens: torch.Tensor | None = None) -> torch.Tensor:
        """Run a step whose entries all bring one token. -> logits [wanted, vocab].
        With `copy` False the result is the graph's own buffer, valid until the next step.
        `device_tokens` (int32 [entries], on the device) replace the entries' token ids."""
        runner = self.runner
        starts = runner.take_pages(entries)
        batch = _bucket(len(entries))
        width = ops.width_bucket(max(max((len(t) for t in e.request.tables), default=0) for e in entries))
        shared, beyond = shared_positions(entries), ()
        if shared:
            starts_of = {i: positions for positions, which in shared for i in which}
            own = ops.own_bucket(max(s + 1 - starts_of.get(i, 0) for i, s in enumerate(starts)), runner.cache.page_size)
            shape = ops.shared_shape(shared)
            gains = [(count, ops.sharing_gain(layer, shape, batch, own)) for layer, count in runner.attention_layers.items()]
            # A layer's, over all of the model's: those that read for each request, and those without attention, are captured too.
            gain = sum(count * g for count, g in gains if g >= 0) / len(runner.cache.needs)
            if any(g >= 0 for _, g in gains) and self._affords((batch, width, shape, own), gain):
                beyond = (shape, own)
            else:
                shared = ()  # the same step as without groups
        captured = self._graph_for(batch, width, *beyond)
        if captured.copied is not None:
            captured.copied.synchronize()  # the pinned buffer is free to be written again
        captured.layout.fill(captured.host_tensor.numpy(), runner.cache, entries, starts,
                             np.arange(batch, dtype=np.int32))
        captured.device.copy_(captured.host_tensor, non_blocking=True)
        if device_tokens is not None:
            captured.step.token_ids[: len(entries)].copy_(device_tokens[: len(entries)])
        if shared:
            captured.step.shared = shared
            ops.fill_step_lists(captured.step)
        if captured.copied is None:
            captured.copied = torch.cuda.Event()
        captured.copied.record()
        captured.graph.replay()
        self.replays += 1
        ops.launches += captured.launches  # the replay launches what the capture recorded
        wanted = [i for i, e in enumerate(entries) if e.want]
        if len(wanted) == len(entries):
            logits = captured.logits[: len(entries)]
        elif wanted:
            return captured.logits[torch.as_tensor(wanted, device=captured.logits.device)]
        else:
            return captured.logits[:0]
        # The graph owns its output buffer; the next replay overwrites it.
        return logits.clone() if copy else logits


MIXED_MAX_TOKENS = 4096
"""Steps of more tokens stay uncaptured (a captured step keeps buffers of its own for as long as its
graph lives). Steps of thousands of tokens are bound by the GPU, not by launching them, yet a replayed
graph still runs them faster: a kernel that follows a library product cannot start its preamble early,
and in a graph the gap between the two is shorter (a 2,048-token step: 7.71 -> 7.37 ms)."""
MIXED_MAX_REQUESTS = 16
"""Steps of more requests stay uncaptured: they are bound by the GPU (the decoding requests' attention
alone outlasts the launching of the step), and in a stream of many requests their shapes change
with every request that joins or leaves."""
MIXED_MAX_GRAPHS = 8
MIXED_CAPTURE_AT = 3
"""A shape is captured at this coming: a capture costs about three steps' time, and in a stream of
requests of many lengths most shapes come once or twice."""


class MixedGraphs:
    """Captured steps of mixed shape, keyed by that shape (see the head of the file)."""

    def __init__(self, runner) -> None:
        self.runner = runner
        self.seen: dict[tuple, int] = {}
        self.captured: dict[tuple, _Captured] = {}  # in order of last use, oldest first
        self.replays = 0

    @property
    def widest(self) -> list[int]:
        """No block table is wider than the longest request the pools can hold (as they are now: a cache is resized between steps)."""
        cache = self.runner.cache
        return [cache.pages_for(g, cache.capacity_tokens()) for g in range(len(cache.groups))]

    @staticmethod
    def supported(model) -> bool:
        return all(getattr(block.mixer, "graph_safe_mixed", False) for block in model.blocks)

    def key(self, entries) -> tuple | None:
        q_lens = tuple(len(e.tokens) for e in entries)
        if sum(q_lens) > MIXED_MAX_TOKENS or len(q_lens) > MIXED_MAX_REQUESTS or all(q == 1 for q in q_lens):
            return None
        page = self.runner.cache.page_size
        longest = max((e.request.tokens + 1 for e, q in zip(entries, q_lens) if q == 1), default=0)
        # Block tables are as wide as the next power of two above the longest request of the step: a
        # prompt that is read in portions doubles before it leaves its graph, and a step's tables
        # are at most twice what its requests need (tables as wide as the pool cost a step of 64
        # requests 2.4 MB of metadata to fill and to copy).
        pages = max(-(-(e.request.tokens + q) // page) for e, q in zip(entries, q_lens))
        # Whether every prompt of the step starts at its first token: kernels are chosen by it (a step's
        # launches are the captured ones for as long as its key is the same).
        fresh = all(e.request.tokens == 0 for e, q in zip(entries, q_lens) if q > 1)
        return (q_lens, tuple(len(e.want) for e in entries), ops.width_bucket(-(-longest // page)) if longest else 0,
                max(64, 1 << (pages - 1).bit_length()), fresh)

    def wants(self, entries) -> tuple | None:
        """The shape's key if this step should run from a graph: the shape has come before."""
        key = self.key(entries)
        if key is None:
            return None
        if key in self.captured:
            return key
        self.seen[key] = self.seen.get(key, 0) + 1
        if len(self.seen) > 4096:
            self.seen.clear()
        return key if self.seen[key] >= MIXED_CAPTURE_AT else None

    def run(self, key: tuple, entries, copy: bool = True) -> torch.Tensor:
        runner = self.runner
        for entry in entries:
            if not entry.tokens:
                raise ValueError(f"request {entry.request.request_id!r} brings no tokens to this step")
            if any(not 0 <= w < len(entry.tokens) for w in entry.want):
                raise ValueError(f"request {entry.request.request_id!r}: a wanted place lies outside its tokens")
        starts = runner.take_pages(entries)
        at, rows = 0, []
        for e in entries:
            rows += [at + w for w in e.want]
            at += len(e.tokens)
        captured = self.captured.pop(key, None)
        fresh = captured is None
        if fresh:
            while len(self.captured) >= MIXED_MAX_GRAPHS:
                torch.cuda.synchronize(runner.runtime.device)
                del self.captured[next(iter(self.captured))]
            layout = StepLayout(at, len(entries), len(rows), [min(key[3], widest) for widest in self.widest])
            host_tensor = torch.zeros(layout.words, dtype=torch.int32).pin_memory()
            dev = torch.zeros(layout.words, dtype=torch.int32, device=runner.runtime.device)
        else:
            layout, host_tensor, dev = captured.layout, captured.host_tensor, captured.device
            if captured.copied is not None:
                captured.copied.synchronize()  # the pinned buffers are free to be written again
        q_lens, held = layout.fill(host_tensor.numpy(), runner.cache, entries, starts, rows)
        dev.copy_(host_tensor, non_blocking=True)
        if fresh:
            # This step runs kernel by kernel on the graph's buffers; then the same launches are captured.
            step = layout.context(dev, q_lens=q_lens, seq_lens_host=held, max_q_len=max(q_lens), max_seq_len=max(held),
                                  decode_only=False, workspace={"private": True})
            layers = runner.layer_contexts(step)
            result = runner.model.forward(step, layers)
            torch.cuda.synchronize(runner.runtime.device)
            graph = torch.cuda.CUDAGraph()
            before = ops.launches
            with capturing(graph):
                logits = runner.model.forward(step, layers)
            launches = ops.launches - before
            ops.launches = before  # the capture launched nothing
            self.captured[key] = _Captured(graph, step, layout, host_tensor, dev, logits, launches)
            return result
        captured.step.seq_lens_host, captured.step.max_seq_len = held, max(held)
        self.captured[key] = captured  # most recently used last
        ops.fill_step_lists(captured.step)
        if captured.copied is None:
            captured.copied = torch.cuda.Event()
        captured.copied.record()
        captured.graph.replay()
        self.replays += 1
        ops.launches += captured.launches
        return captured.logits.clone() if copy else captured.logits


DRAFTED_MAX_TOKENS = 256
"""Steps of more drafted tokens stay uncaptured: their kernels outlast the launching (28 layers: 4.2 ms; 64 requests of 2,000 positions with four tokens
each take the GPU 7.8), and a graph keeps a row of logits for each."""


class DraftedGraphs:
    """Captured steps of drafted trees, keyed by their rounded shape (see the head of the file)."""

    def __init__(self, runner) -> None:
        self.runner = runner
        self.seen: dict[tuple, int] = {}
        self.captured: dict[tuple, _Captured] = {}  # in order of last use, oldest first
        self.replays = 0

    def shape(self, entries) -> tuple | None:
        """(requests, rows, drafts of a request, width of the tables), rounded, of a step that is captured when it comes often enough (None: never).
        (Their pages are taken.)"""
        brought = [len(e.tokens) for e in entries]
        if sum(brought) > DRAFTED_MAX_TOKENS or any(e.parents is None for e in entries):
            return None
        total = max(sum(brought), 8)
        step = 1 << (total.bit_length() - 2)  # rows by two significant bits: products of 16 rows and of 13 stream the same weights
        return (_bucket(len(entries)), -(-total // step) * step, _bucket(max(brought)),
                ops.width_bucket(max(len(t) for e in entries for t in e.request.tables)))

    def _comes_often(self, key: tuple) -> bool:
        if key in self.captured:
            return True
        self.seen[key] = self.seen.get(key, 0) + 1
        if len(self.seen) > 4096:
            self.seen.clear()
            return False
        return self.seen[key] >= MIXED_CAPTURE_AT

    def run(self, key: tuple, entries, starts: list[int], copy: bool = True) -> "tuple[torch.Tensor, StepContext]":
        """A step of this shape. -> logits of all the entries' tokens, and the step as these see it (of a captured step its tables are the graph's own:
        the next step overwrites them)"""
        runner, cache = self.runner, self.runner.cache
        requests, tokens, most, width = key
        often = self._comes_often(key)
        captured = self.captured.pop(key, None)
        fresh = captured is None
        if fresh:
            while often and len(self.captured) >= MIXED_MAX_GRAPHS:
                torch.cuda.synchronize(runner.runtime.device)
                del self.captured[next(iter(self.captured))]
            # Requests that hold nothing for the rows that no entry brings: fewer than `tokens` of them.
            layout = DraftedLayout(tokens, requests + -(-tokens // most), tokens, [width] * len(cache.groups), most)
            host_tensor = torch.zeros(layout.words, dtype=torch.int32, pin_memory=True)
            dev = torch.zeros(layout.words, dtype=torch.int32, device=runner.runtime.device)
        else:
            layout, host_tensor, dev = captured.layout, captured.host_tensor, captured.device
            if captured.copied is not None:
                captured.copied.synchronize()  # the pinned buffer is free to be written again
        layout.fill(host_tensor.numpy(), cache, entries, starts, np.arange(tokens, dtype=np.int32))
        dev.copy_(host_tensor, non_blocking=True)

        def forward(workspace: dict) -> "tuple[torch.Tensor, StepContext]":
            step = layout.context(dev, cache.page_size, width * cache.page_size, q_lens=[], seq_lens_host=[], workspace=workspace)
            return runner.model.forward(step, runner.layer_contexts(step)), step

        if not often:
            logits, step = forward(runner.ask_for_layers())
            runner.know_layers(step)
        elif fresh:
            # This step runs kernel by kernel on the graph's buffers; then the same launches are captured.
            workspace: dict = {"private": True}
            logits, step = forward(workspace)
            torch.cuda.synchronize(runner.runtime.device)
            graph = torch.cuda.CUDAGraph()
            before = ops.launches
            with capturing(graph):
                kept_logits, kept_step = forward(workspace)
            launches = ops.launches - before
            ops.launches = before  # the capture launched nothing
            self.captured[key] = _Captured(graph, kept_step, layout, host_tensor, dev, kept_logits, launches)
        else:
            self.captured[key] = captured  # most recently used last
            if captured.copied is None:
                captured.copied = torch.cuda.Event()
            captured.copied.record()
            captured.graph.replay()
            self.replays += 1
            ops.launches += captured.launches
            logits, step = captured.logits, captured.step
        n, total = len(entries), sum(len(e.tokens) for e in entries)
        mine = replace(step, num_tokens=total, num_seqs=n, token_ids=step.token_ids[:total], positions=step.positions[:total],
                       cu_seqlens=step.cu_seqlens[: n + 1], seq_lens=step.seq_lens[:n], logit_rows=step.logit_rows[:total],
                       groups={g: (table[:n], slots[:total]) for g, (table, slots) in step.groups.items()}, tree=StepTree(step.tree.ancestors[:total]))
        logits = logits[:total]
        return logits.clone() if copy and not fresh else logits, mine
