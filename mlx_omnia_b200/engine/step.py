"""The step function: one batch of (request, its next tokens) through the model.

A step takes entries `(request, tokens, want)`: the request's next tokens, any number
from one (a decoded token) to a whole prompt, cut anywhere, and the places among them
whose logits are wanted. All entries run as one flattened batch; only these tokens
are computed, everything earlier is read from the cache. It returns float32 logits
`[wanted, vocab]` in the order of the entries and of `want`.

The reference runs either one request's prompt block or a batch of single decode
tokens per forward, never both (src/mlx_omnia/server/runtime/rounds.py:159-202,
src/mlx_omnia/engine/batching.py:283-301,541-576); the mixed flattened batch is this
engine's own design.
"""

from __future__ import annotations

from collections import Counter
from dataclasses import dataclass, field

import numpy as np
import torch

from mlx_omnia_b200.cache.manager import CacheManager, RequestCache
from mlx_omnia_b200.kernels import ops
from mlx_omnia_b200.parts.base import KVView, LayerContext, Runtime, StepContext
from mlx_omnia_b200.parts.model import DecoderModel


@dataclass
class StepEntry:
    request: RequestCache
    tokens: list[int]
    want: list[int] = field(default_factory=list)  # indices into `tokens`
    parents: list[int] | None = None  # drafted tokens: for each the earlier one that it goes on from; -1 for the first, which is known


def shared_positions(entries: list[StepEntry]) -> tuple[tuple[int, tuple[int, ...]], ...]:
    """Which entries' requests share their first positions: (positions, entries) of each group of two or more, the largest first. A
    request that shares several runs of positions goes with the longest that another entry, not in a group yet, shares too."""
    members: dict = {}
    for i, entry in enumerate(entries):
        for run in entry.request.runs:
            members.setdefault(run, []).append(i)
    found, taken = [], set()
    for run in sorted(members, key=lambda run: -run.positions):
        which = tuple(i for i in members[run] if i not in taken)
        if len(which) > 1:
            found.append((run.positions, which))
            taken.update(which)
    return tuple(sorted(found, key=lambda group: (-group[0], -len(group[1]))))


class StepLayout:
    """Where each field of a step's metadata sits in one buffer of int32 words, so that one
    copy brings all of it to the device. A layout is made for `tokens` rows of the batch,
    `seqs` requests, `wanted` logit rows and a block-table width per group; a step with fewer
    requests than `seqs` pads the rest (each padding request brings one padding token). Both
    the eager step and the captured decode graphs lay their metadata out through this class
    and fill it with `fill`, so they cannot drift apart."""

    def __init__(self, tokens: int, seqs: int, wanted: int, widths: list[int]) -> None:
        self.tokens, self.seqs, self.wanted, self.widths = tokens, seqs, wanted, list(widths)
        self.fields: dict[str, tuple[int, int]] = {}
        at = 0
        # The int64 slot mappings come first, so they start on 8 bytes.
        for name, length in ([(f"slots{g}", 2 * tokens) for g in range(len(widths))] +
                             [("token_ids", tokens), ("positions", tokens), ("cu_seqlens", seqs + 1),
                              ("seq_lens", seqs), ("state_slots", seqs), ("fresh", seqs), ("logit_rows", wanted)] +
                             [(f"table{g}", seqs * w) for g, w in enumerate(widths)]):
            self.fields[name] = (at, length)
            at += length
        self.words = max(at, 1)

    def view(self, buffer, name: str):
        """The field `name` of `buffer` (a numpy array or a tensor of int32 words)."""
        at, length = self.fields[name]
        return buffer[at: at + length]

    def fill(self, host: np.ndarray, cache: CacheManager, entries: list[StepEntry], starts: list[int],
             wanted_rows) -> tuple[list[int], list[int]]:
        """Write the metadata of `entries` (whose requests held `starts[i]` positions before
        this step and have been grown since) into `host`; rows and requests beyond them become
        padding: position -1, sequence length 0, cache slot -1, the scratch state slot, block
        tables of -1. -> (tokens per entry, positions held after the step per entry)"""
        n, page = len(entries), cache.page_size
        q_lens = [len(e.tokens) for e in entries]
        total = sum(q_lens)
        if self.tokens - total != self.seqs - n or n > self.seqs:
            raise ValueError("a padded step brings one padding token per padding request")
        cu = np.arange(self.seqs + 1, dtype=np.int32) + (total - n)
        cu[0] = 0
        cu[1: n + 1] = np.cumsum(q_lens)
        self.view(host, "cu_seqlens")[:] = cu
        ids, positions = self.view(host, "token_ids"), self.view(host, "positions")
        ids[total:], positions[total:] = 0, -1
        for i, (e, s) in enumerate(zip(entries, starts)):
            ids[cu[i]: cu[i + 1]] = e.tokens
            positions[cu[i]: cu[i + 1]] = np.arange(s, s + q_lens[i], dtype=np.int32)
        held = [s + q for s, q in zip(starts, q_lens)]
        for name, values, pad in (("seq_lens", held, 0), ("state_slots", [e.request.slot for e in entries],
                                                           cache.scratch_slot),
                                  ("fresh", [int(e.request.fresh) for e in entries], 0)):
            field_ = self.view(host, name)
            field_[:n], field_[n:] = values, pad
        self.view(host, "logit_rows")[:] = wanted_rows
        for g, group in enumerate(cache.groups):
            table = self.view(host, f"table{g}").reshape(self.seqs, self.widths[g])
            table.fill(-1)
            slots = self.view(host, f"slots{g}").view(np.int64)
            slots[total:] = -1
            stride = group.spec.stride
            for i, e in enumerate(entries):
                t = e.request.table_array(g)
                table[i, : len(t)] = t
                row = positions[cu[i]: cu[i + 1]].astype(np.int64) // stride
                slots[cu[i]: cu[i + 1]] = t[row // page].astype(np.int64) * page + row % page
        return q_lens, held

    def context(self, device: torch.Tensor, **host_side) -> StepContext:
        """The step as the parts see it, its tensors being views of the `device` buffer."""
        groups = {g: (self.view(device, f"table{g}").view(self.seqs, w), self.view(device, f"slots{g}").view(torch.int64))
                  for g, w in enumerate(self.widths)}
        return StepContext(
            num_tokens=self.tokens, num_seqs=self.seqs, token_ids=self.view(device, "token_ids"),
            positions=self.view(device, "positions"), cu_seqlens=self.view(device, "cu_seqlens"),
            seq_lens=self.view(device, "seq_lens"), state_slots=self.view(device, "state_slots"),
            fresh=self.view(device, "fresh"), logit_rows=self.view(device, "logit_rows"), groups=groups, **host_side)


@dataclass(frozen=True)
class Kept:
    """What a request keeps of the tokens that it brought as drafts: the kept ones behind the first, and the token chosen behind the last of them."""

    tokens: list[int]
    next: int


class DraftedLayout:
    """Where what the host knows of a step of drafted trees lies in one buffer of int32 words: `tokens` rows of the batch, `seqs` requests, `wanted`
    rows of logits, lists of `widths` pages. The tables are made from it on the device (`ops.step_tables`), in an eager step and in a captured one."""

    def __init__(self, tokens: int, seqs: int, wanted: int, widths: list[int], most: int) -> None:
        self.tokens, self.seqs, self.widths, self.most = tokens, seqs, list(widths), most
        self.parts: dict[str, slice] = {}
        at = 0
        for name, size in ([(f"starts{g}", 2 * seqs) for g in range(len(widths))] +  # (8 bytes each)
                           [("held", seqs), ("brought", seqs), ("slots", seqs), ("fresh", seqs), ("parents", tokens), ("ids", tokens), ("rows", wanted)] +
                           [(f"pages{g}", seqs * w) for g, w in enumerate(widths)]):
            self.parts[name] = slice(at, at + size)
            at += size
        self.words = at

    def fill(self, host: np.ndarray, cache: CacheManager, entries: list[StepEntry], starts: list[int], rows) -> None:
        """Requests beyond `entries` are there for the step's shape: rows that no entry brings are theirs, and see nothing."""
        part = {name: host[where] for name, where in self.parts.items()}
        n, brought = len(entries), [len(e.tokens) for e in entries]
        total = sum(brought)
        spare = [max(0, min(self.most, self.tokens - total - i * self.most)) for i in range(self.seqs - n)]
        if max(brought) > self.most or total + sum(spare) != self.tokens:
            raise ValueError("a step of drafted trees has more rows than its requests bring")
        part["held"][:n], part["held"][n:] = starts, -1
        part["brought"][:n], part["brought"][n:] = brought, spare
        part["slots"][:n], part["slots"][n:] = [e.request.slot for e in entries], cache.scratch_slot
        part["fresh"][:n], part["fresh"][n:] = [int(e.request.fresh) for e in entries], 0
        part["parents"][:total] = [p for e in entries for p in (e.parents if e.parents is not None else range(-1, len(e.tokens) - 1))]
        part["ids"][:total] = [t for e in entries for t in e.tokens]
        part["parents"][total:], part["ids"][total:] = -1, 0
        part["rows"][:] = rows
        for g, width in enumerate(self.widths):
            part[f"starts{g}"].view(np.int64)[:] = np.arange(self.seqs, dtype=np.int64) * width
            table = part[f"pages{g}"].reshape(self.seqs, width)
            table.fill(-1)
            for i, e in enumerate(entries):
                mine = e.request.table_array(g)
                table[i, : len(mine)] = mine

    def context(self, device: torch.Tensor, page_size: int, max_seq_len: int, **more) -> StepContext:
        """The step, its tables made by a kernel from what the `device` buffer holds then."""
        part = {name: device[where] for name, where in self.parts.items()}
        lists = [ops.PageLists(part[f"pages{g}"], part[f"starts{g}"].view(torch.int64), width) for g, width in enumerate(self.widths)]
        made = ops.step_tables(part["held"], part["brought"], lists, page_size, self.tokens, parents=part["parents"], most=self.most)
        return StepContext(
            num_tokens=self.tokens, num_seqs=self.seqs, token_ids=part["ids"], positions=made.positions, cu_seqlens=made.cu_seqlens,
            seq_lens=made.seq_lens, state_slots=part["slots"], fresh=part["fresh"], logit_rows=part["rows"], max_q_len=self.most,
            max_seq_len=max_seq_len, decode_only=False, groups=dict(enumerate(made.groups)), tree=made.tree, **more)


class DraftedSteps:
    """Steps whose requests bring trees of drafted tokens. `run` reads all of them in one step; `keep` says which the model agrees with, moves
    their keys and values to where a request that had brought only these would have them, and takes the others' room back."""

    def __init__(self, runner: "StepRunner") -> None:
        self.runner = runner
        self.last: "tuple[list[StepEntry], StepContext, list[int]] | None" = None

    def why_not(self) -> str | None:
        """Why the model takes no drafted trees (None: it does). A tree's branches read the same positions and leave nothing behind but rows of the
        cache, which state that goes from token to token does not."""
        runner = self.runner
        if runner.cache.has_state or not all(getattr(block.mixer, "tree_safe", False) for block in runner.model.blocks):
            return "drafted trees take a model of attention over keys and values alone"
        if any(g.spec.stride != 1 for g in runner.cache.groups):
            return "drafted trees take caches with a row for every position"
        return None

    def run(self, entries: list[StepEntry], copy: bool = True) -> torch.Tensor:
        runner, cache, device = self.runner, self.runner.cache, self.runner.runtime.device
        why = self.why_not()
        if why is not None:
            raise ValueError(why)
        for e in entries:
            n, parents = len(e.tokens), e.parents
            if not 1 <= n <= ops.MOST_DRAFTED:
                raise ValueError(f"request {e.request.request_id!r} brings {n} tokens to a step of drafted trees, which takes 1 to {ops.MOST_DRAFTED}")
            if any(not 0 <= w < n for w in e.want):
                raise ValueError(f"request {e.request.request_id!r}: a wanted place lies outside its tokens")
            if parents is not None and (len(parents) != n or parents[0] != -1 or any(not 0 <= p < j for j, p in enumerate(parents) if j)):
                raise ValueError(f"request {e.request.request_id!r}: a drafted token goes on from an earlier one, the first from none")
            if parents is not None and e.want != list(range(n)):
                raise ValueError(f"request {e.request.request_id!r}: drafted tokens want all their logits")
        if len({id(e.request) for e in entries}) < len(entries):
            raise ValueError("a request comes once to a step")
        cache.reset_slots([e.request.slot for e in entries if e.request.fresh])
        starts = runner.take_pages(entries)
        graphs = runner.drafted_graphs
        key = graphs.shape(entries) if graphs is not None else None
        if key is not None:
            logits, step = graphs.run(key, entries, starts, copy)
        else:
            brought = [len(e.tokens) for e in entries]
            cu, held = np.cumsum([0, *brought]), [s + b for s, b in zip(starts, brought)]
            rows = [int(c) + w for c, e in zip(cu, entries) for w in e.want]
            widths = [max(len(e.request.tables[g]) for e in entries) for g in range(len(cache.groups))]
            layout = DraftedLayout(sum(brought), len(entries), len(rows), widths, max(brought))
            host_tensor = torch.empty(layout.words, dtype=torch.int32, pin_memory=device.type == "cuda")
            layout.fill(host_tensor.numpy(), cache, entries, starts, rows)
            packed = host_tensor.to(device, non_blocking=True) if device.type == "cuda" else host_tensor
            step = layout.context(packed, cache.page_size, max(held), q_lens=brought, seq_lens_host=held, workspace=runner.ask_for_layers())
            logits = runner.model.forward(step, runner.layer_contexts(step))
            runner.know_layers(step)
        for e in entries:
            e.request.fresh = False
            if e.parents is not None:
                e.request.drafted = len(e.tokens)
            else:
                cache.release_behind_window(e.request)
        self.last = (list(entries), step, starts)
        runner.steps_run += 1
        return logits

    def keep(self, entries: list[StepEntry], chosen: torch.Tensor) -> list[Kept | None]:
        """`chosen`: int32 on the device, the token that was chosen from every row of the logits of `entries`' step, the one just run. Every drafted
        token is kept whose way from the request's first is what was chosen; the requests hold these and no other from then on.
        -> for each entry what it keeps (None: it brought no drafts)"""
        if self.last is None or len(self.last[0]) != len(entries) or any(a is not b for a, b in zip(self.last[0], entries)):
            raise ValueError("keep() takes the entries of the step of drafted trees that was run last, once")
        cache, (_, step, starts) = self.runner.cache, self.last
        if any(e.parents is not None and (cache.requests.get(e.request.request_id) is not e.request or e.request.drafted != len(e.tokens)) for e in entries):
            raise ValueError("a request of the step has ended")
        if chosen.shape != step.logit_rows.shape:
            raise ValueError("a token is chosen from every row of the step's logits")
        picks = chosen
        if step.logit_rows.shape[0] != step.num_tokens:
            picks = torch.zeros(step.num_tokens, dtype=torch.int32, device=chosen.device)
            picks[step.logit_rows.long()] = chosen
        accepted = ops.accept_drafts(picks, step.token_ids, step.tree, step.cu_seqlens)
        held = step.seq_lens - (step.cu_seqlens[1:] - step.cu_seqlens[:-1])
        for g, group in enumerate(cache.groups):
            ops.keep_rows(group.pages, group.spec.rows, cache.page_size, step.groups[g][0], held, accepted)
        self.last = None
        path, kept, last = accepted.path.tolist(), accepted.kept.tolist(), accepted.tokens.tolist()
        found: list[Kept | None] = []
        for i, e in enumerate(entries):
            if e.parents is None:
                found.append(None)
                continue
            self.runner._shrink(e.request, len(e.tokens) - kept[i])
            e.request.drafted = 0
            cache.release_behind_window(e.request)
            found.append(Kept([e.tokens[j] for j in path[i][1: kept[i]]], last[i]))
        return found


class StepRunner:
    """Owns nothing but the glue: the model, the cache manager and the runtime."""

    def __init__(self, model: DecoderModel, cache: CacheManager, runtime: Runtime, cuda_graphs: bool = False) -> None:
        self.model, self.cache, self.runtime = model, cache, runtime
        self.steps_run = 0
        self.drafted = DraftedSteps(self)
        self.attention_layers: Counter = Counter()  # kinds (`ops.AttentionLayer`) that a step was seen to run, and how often
        self.cuda_graphs = cuda_graphs
        self.graphs = self.mixed_graphs = self.drafted_graphs = None
        self.forget_graphs()

    def forget_graphs(self) -> None:
        """Drop every captured step (they hold the addresses of the cache's tensors) and begin anew."""
        if not self.cuda_graphs or self.runtime.device.type != "cuda":
            return
        from mlx_omnia_b200.engine.decode_graph import DecodeGraphs, DraftedGraphs, MixedGraphs

        if self.graphs is not None:
            torch.cuda.synchronize(self.runtime.device)  # nothing of them is still running
        if DecodeGraphs.supported(self.model):
            self.graphs = DecodeGraphs(self)
            if MixedGraphs.supported(self.model):
                self.mixed_graphs = MixedGraphs(self)
                if self.drafted.why_not() is None:
                    self.drafted_graphs = DraftedGraphs(self)

    def ask_for_layers(self) -> dict:
        """A step's workspace, in which attention notes its layers until these are known. (Every step runs all of them, and requests share positions
        that a step has read, so they are known by the time that a captured step is asked whether it pays to read these once.)"""
        return {} if self.attention_layers else {"attention_layers": Counter()}

    def know_layers(self, step: StepContext) -> None:
        self.attention_layers = step.workspace.pop("attention_layers", self.attention_layers)

    # -- metadata ----------------------------------------------------------------------
    def take_pages(self, entries: list[StepEntry]) -> list[int]:
        """Grow every entry's request by its tokens, or none of them (the error is raised
        after what this step took has been given back). -> positions held before the step"""
        starts = [entry.request.tokens for entry in entries]
        grown: list[tuple[RequestCache, int]] = []
        try:
            for entry in entries:
                self.cache.grow(entry.request, len(entry.tokens))
                grown.append((entry.request, len(entry.tokens)))
        except Exception:
            for request, count in grown:
                self._shrink(request, count)
            raise
        return starts

    def build_context(self, entries: list[StepEntry]) -> StepContext:
        """Take the pages the entries' tokens need and lay the batch out."""
        cache = self.cache
        if not entries:
            raise ValueError("a step needs at least one entry")
        for entry in entries:
            if not entry.tokens:
                raise ValueError(f"request {entry.request.request_id!r} brings no tokens to this step")
            if any(not 0 <= w < len(entry.tokens) for w in entry.want):
                raise ValueError(f"request {entry.request.request_id!r}: a wanted place lies outside its tokens")
        starts = self.take_pages(entries)
        at, rows = 0, []
        for e in entries:
            rows += [at + w for w in e.want]
            at += len(e.tokens)
        widths = [max(max(len(e.request.tables[g]) for e in entries), 1) for g in range(len(cache.groups))]
        layout = StepLayout(at, len(entries), len(rows), widths)
        pinned = self.runtime.device.type == "cuda"
        host_tensor = torch.empty(layout.words, dtype=torch.int32, pin_memory=pinned)
        q_lens, held = layout.fill(host_tensor.numpy(), cache, entries, starts, rows)
        device = host_tensor.to(self.runtime.device, non_blocking=True) if pinned else host_tensor
        single = all(q == 1 for q in q_lens)
        return layout.context(device, q_lens=q_lens, seq_lens_host=held, max_q_len=max(q_lens),
                              max_seq_len=max(held), decode_only=single, shared=shared_positions(entries) if single else ())

    def _shrink(self, request: RequestCache, count: int) -> None:
        """Undo a `grow` of `count` tokens that no kernel has used."""
        request.tokens -= count
        for g, (group, table) in enumerate(zip(self.cache.groups, request.tables)):
            keep = self.cache.pages_for(g, request.tokens)
            while len(table) > keep:
                group.pool.give(table.pop())
                request.arrays[g][len(table)] = -1

    def layer_contexts(self, step: StepContext) -> list[LayerContext]:
        cache = self.cache
        step.model_state = cache.model_state or None
        contexts = []
        for entry, need in enumerate(cache.needs):
            kv = None
            if entry in cache.group_of_entry:
                g, _ = cache.group_of_entry[entry]
                table, slots = step.groups[g]
                kv = KVView(cache.entry_pages(entry), table, slots, cache.page_size, cache.groups[g].spec.window,
                            writes=need.reads is None, spec=cache.groups[g].spec)
            contexts.append(LayerContext(step, kv, cache.state.get(entry), entry,
                                         block_state=cache.block_state.get(entry)))
        return contexts

    # -- the step ----------------------------------------------------------------------
    def run(self, entries: list[StepEntry], copy: bool = True, device_tokens: torch.Tensor | None = None) -> torch.Tensor:
        """One step. Steps in which every request brings a single token are replayed
        from a captured CUDA graph when graphs are on; `copy=False` then returns the
        graph's own logits buffer, which the next step overwrites. `device_tokens`
        (int32 on the device, one per entry; graph steps only) are the step's tokens when
        the host does not know them yet. Entries with `parents` bring drafted tokens: the step
        is then one of drafted trees (`DraftedSteps`), and `keep` follows it."""
        for e in entries:
            if e.request.drafted:
                raise ValueError(f"request {e.request.request_id!r} holds drafted tokens that are not kept yet")
        if any(e.parents is not None for e in entries):
            if device_tokens is not None:
                raise ValueError("drafted tokens come from the host")
            return self.drafted.run(entries, copy)
        self.cache.reset_slots([e.request.slot for e in entries if e.request.fresh])
        if self.graphs is not None and entries and all(len(e.tokens) == 1 and e.want in ([], [0]) for e in entries):
            logits = self.graphs.run(entries, copy, device_tokens)
        else:
            if device_tokens is not None:
                raise ValueError("tokens that live on the device can only feed a captured single-token step")
            shape = self.mixed_graphs.wants(entries) if self.mixed_graphs is not None and entries else None
            if shape is not None:
                logits = self.mixed_graphs.run(shape, entries, copy)
            else:
                step = self.build_context(entries)
                step.workspace = self.ask_for_layers()
                logits = self.model.forward(step, self.layer_contexts(step))
                self.know_layers(step)
        for entry in entries:
            entry.request.fresh = False
            self.cache.release_behind_window(entry.request)
        self.steps_run += 1
        return logits

    def keep(self, entries: list[StepEntry], chosen: torch.Tensor) -> "list[Kept | None]":
        """What becomes of the drafted tokens of the step just run (see `DraftedSteps.keep`)."""
        return self.drafted.keep(entries, chosen)
