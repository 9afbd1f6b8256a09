"""Generation: the loop that plans a step, runs it, samples and commits; and the
`load(path)` -> `model.stream(prompt, GenerationOptions(...))` entry point.

The reference's entry point is `load` (src/mlx_omnia/engine/task.py:486-547) returning a
facade whose `stream(input, options)` yields segments with `.text`
(src/mlx_omnia/engine/model.py:201-202, src/mlx_omnia/engine/language.py:483-552), over a
continuous-batching loop of `begin_batch`/`step_batch`
(src/mlx_omnia/engine/batching.py:223-341,408-437). Here the loop is the scheduler's
plan -> the step function -> the sampling kernel -> commit, with one device-to-host
read of the chosen tokens per step.
"""

from __future__ import annotations

import dataclasses
import itertools
import secrets
from collections.abc import Collection, Iterator, Mapping, Sequence
from dataclasses import dataclass
from pathlib import Path

import numpy as np
import torch

from mlx_omnia_b200.engine.engine import DTYPES, Engine, EngineArgs
from mlx_omnia_b200.engine.meter import Meter
from mlx_omnia_b200.engine.scheduler import PlannedEntry, Request, Scheduler, StepOutput, StepPlan
from mlx_omnia_b200.engine.step import StepEntry
from mlx_omnia_b200.kernels import ops
from mlx_omnia_b200.sampling.batch import allowed_ids, id_array, sample_drafted, sample_rows, text_of
from mlx_omnia_b200.sampling.options import GenerationOptions
from mlx_omnia_b200.text.bpe import Detokenizer
from mlx_omnia_b200.text.defaults import GenerationDefaults


@dataclass(frozen=True)
class Segment:
    """One piece of a streamed answer."""

    text: str
    token_id: int


@dataclass(frozen=True)
class Text:
    """A text prompt, as the reference's `Text` input (src/mlx_omnia/engine/language.py:60-79)."""

    prompt: str | Sequence[int]


class TokenIdTokenizer:
    """Stands in when a model folder has no tokenizer: text is token ids in decimal,
    separated by spaces, both ways."""

    def encode(self, text: str) -> list[int]:
        try:
            return [int(piece) for piece in text.replace(",", " ").split()]
        except ValueError:
            raise ValueError("this model folder has no tokenizer.json; give the prompt as token ids "
                             "(integers separated by spaces) or as a list of ints") from None

    def decode(self, ids: Sequence[int]) -> str:
        return "".join(f"{i} " for i in ids)


@dataclass
class _Launched:
    """A step that is running on the GPU: its plan, the requests it samples for and their
    chosen tokens (still on the device)."""

    plan: StepPlan
    sampling: list[Request]
    chosen: torch.Tensor | None
    host_tokens: torch.Tensor | None = None  # pinned copy of `chosen`, on its way since the launch
    copied: "torch.cuda.Event | None" = None  # recorded behind that copy


def common_start(prompts: Sequence[Sequence[int]]) -> int:
    """How many first tokens all of the prompts have in common."""
    first, last = min(prompts, default=()), max(prompts, default=())  # whatever these two share, all between them do
    return next((i for i, (a, b) in enumerate(zip(first, last)) if a != b), min(len(first), len(last)))


class Generator:
    """Continuous batching over one `Engine`."""

    def __init__(self, engine: Engine, *, max_tokens_per_step: int = 2048, max_running: int | None = None,
                 stop: Sequence[int] | None = None) -> None:
        """`stop`: the ids that end a generation whose options name none (None: config.json's own)."""
        self.engine = engine
        self.default_stop = tuple(stop) if stop is not None else \
            tuple(engine.architecture.stop_tokens(engine.config))
        self.scheduler = Scheduler(engine.cache, max_tokens_per_step=max_tokens_per_step, max_running=max_running)
        self._ids = itertools.count()
        self._seeds: dict[str, int] = {}
        self._in_flight: _Launched | None = None
        self._held: list[StepOutput] = []  # committed, but not returned yet: a step that fails behind them leaves them to the next call
        self._failed: list[Request] = []  # ended by constraints of their own, which no call has raised yet
        self._token_slots: list[torch.Tensor] = []  # pinned buffers the chosen tokens come back in, used in turn
        self._token_slot = 0
        self.pipelined = True  # launch the next decode step before reading this one's tokens

    def add(self, prompt: Sequence[int], options: GenerationOptions, request_id: str | None = None, *,
            leader: Request | None = None, fork_at: int | None = None) -> Request:
        """Add a request. With a `leader`, a request whose prompt begins with the same `fork_at` tokens (None: as many as the two have in
        common; all but the last of this prompt at most), those are not read again but taken over from it, and steps of single tokens
        read their keys and values once for both."""
        prompt = [int(t) for t in prompt]
        vocab = self.engine.vocab_size
        if any(not 0 <= t < vocab for t in prompt):
            raise ValueError(f"a prompt token lies outside the vocabulary of {vocab}")
        params = options.params()
        if any(token >= vocab for token, _ in params.bias):
            raise ValueError(f"a bias names a token outside the vocabulary of {vocab}")
        budget = options.max_tokens
        if options.context_limit is not None:
            budget = min(budget, options.context_limit - len(prompt))
        stop = options.stop if options.stop is not None else self.default_stop
        request = Request(request_id or f"req-{next(self._ids)}", prompt, max(budget, 0), params, frozenset(stop))
        if leader is not None:
            request.fork_at = common_start([leader.prompt, prompt[:-1]]) if fork_at is None else int(fork_at)
            request.leader = leader if request.fork_at or fork_at is not None else None
        request.meter = options.meter if options.meter is not None else Meter()
        request.meter.begin(len(prompt))
        self.scheduler.add(request)
        self._seeds[request.request_id] = params.seed if params.seed is not None else secrets.randbits(63)
        return request

    def abort(self, request_id: str) -> None:
        self.scheduler.abort(request_id)
        self._seeds.pop(request_id, None)

    def drain(self) -> list[StepOutput]:
        """Commit the step that is still in flight, if any. -> its outputs, behind those of a call that failed"""
        self._land()
        return self._hand_out()

    def _land(self) -> None:
        launched, self._in_flight = self._in_flight, None
        if launched is not None:
            self._held += self._finalize(launched)

    def _hand_out(self) -> list[StepOutput]:
        outputs, self._held = self._held, []
        return outputs

    def _deliver(self) -> list[StepOutput]:
        """What a step returns. Where a request's constraint failed in it, that error is raised and the outputs, the request's end among them, are
        the next call's."""
        failed, self._failed = self._failed, []
        if failed:
            raise failed[0].error
        return self._hand_out()

    def _fail(self, request: Request, error: Exception) -> None:
        self.scheduler._finish(request, "abort")  # (frees what it holds)
        request.error = error
        self._seeds.pop(request.request_id, None)

    def _fail_alone(self, request: Request, error: Exception) -> None:
        """End a request by its own constraint's error: the step goes on for the others."""
        self._fail(request, error)
        self._held.append(StepOutput(request, None, True))
        self._failed.append(request)

    # -- one step -----------------------------------------------------------------------------
    # A decode step's tokens are chosen on the GPU and can feed the next step from there, so the
    # host need not wait for them before it launches that step: while the GPU runs step n + 1 the
    # host reads step n's tokens (one step late, as the reference does: src/mlx_omnia/engine/
    # batching.py:598-604), commits them and prepares step n + 2. A request that turns out to
    # have ended on a stop token has then computed one token too many, which is dropped.

    def _launch(self, plan: StepPlan, device_tokens: torch.Tensor | None = None) -> "_Launched":
        entries = []
        for planned in plan.entries:
            tokens = [0] * planned.count if device_tokens is not None else \
                planned.request.token_slice(planned.start, planned.count)
            entries.append(StepEntry(planned.request.cache, tokens, [planned.count - 1] if planned.samples else []))
        sampling = [p.request for p in plan.entries if p.samples]
        try:
            logits = self.engine.runner.run(entries, copy=False, device_tokens=device_tokens)
            chosen = self._choose(logits, sampling, 1 if device_tokens is not None else 0) if sampling else None
        except Exception as error:
            for planned in plan.entries:  # a failed step fails its requests
                if planned.request.error is None:
                    self._fail(planned.request, error)
            raise
        launched = _Launched(plan, sampling, chosen)
        if chosen is not None and chosen.is_cuda:
            # The tokens start for the host at once, behind this step only. Read with a blocking copy
            # when the host wants them, they would come behind everything launched since, the
            # next step included, and the host would prepare the step after that with the GPU idle.
            if not self._token_slots or self._token_slots[0].numel() < chosen.numel():
                self._token_slots = [torch.empty(max(64, chosen.numel()), dtype=torch.int32).pin_memory()
                                     for _ in range(4)]
            self._token_slot = (self._token_slot + 1) % len(self._token_slots)
            launched.host_tokens = self._token_slots[self._token_slot][: chosen.numel()]
            launched.host_tokens.copy_(chosen, non_blocking=True)
            launched.copied = torch.cuda.Event()
            launched.copied.record()
        return launched

    def _choose(self, logits: torch.Tensor, sampling: list[Request], ahead: int) -> torch.Tensor:
        """A token for every row of logits (`ahead`: draws already spent by a step that is not yet committed)."""
        histories = [r.token_slice(max(0, len(r.prompt) + len(r.generated) - r.sampling.penalty_context),
                                   r.sampling.penalty_context) if r.sampling.repetition_penalty != 1.0 else []
                     for r in sampling]
        adjusts = any(r.sampling.adjusts for r in sampling)
        params, seeds = [r.sampling for r in sampling], [self._seeds[r.request_id] for r in sampling]
        draws = [len(r.generated) + ahead for r in sampling]
        return sample_rows(logits, params, seeds, draws, histories, [text_of(r.sampling, r.prompt, r.generated) for r in sampling] if adjusts else None,
                           [self._allowed(r) for r in sampling] if adjusts else None)

    def _allowed(self, request: Request) -> np.ndarray | None:
        """What the request's constraint lets come next. A constraint that fails ends its request, which is given any token then and keeps none."""
        try:
            return id_array(allowed_ids(request.sampling, request.generated), self.engine.vocab_size)
        except Exception as error:
            self._fail_alone(request, error)
            return None

    def _finalize(self, launched: "_Launched") -> list[StepOutput]:
        """Read the launched step's tokens (this waits for it) and commit them."""
        plan = launched.plan
        if launched.copied is not None:
            launched.copied.synchronize()
            tokens = launched.host_tokens.tolist()
        else:
            tokens = launched.chosen.tolist() if launched.chosen is not None else []
        sampled = dict(zip((r.request_id for r in launched.sampling), tokens))
        # A request that ended (a stop token, an abort) after this step was launched is left out.
        live = [e for e in plan.entries if e.request.status == "running"]
        outputs = self.scheduler.commit(StepPlan(live, plan.preempted), sampled)
        for output in outputs:
            if output.token is not None:
                output.request.meter.token()
            if output.finished:
                self._seeds.pop(output.request.request_id, None)
        return outputs

    def _next_decode_plan(self, launched: "_Launched") -> StepPlan | None:
        """The plan of the step after `launched`, if it can be made before `launched`'s tokens
        are known: every entry decodes, nobody waits for admission, no request needs its own
        last token on the host (penalties, constraints), and the pages are there."""
        if self.engine.runner.graphs is None or self.scheduler.waiting or not self.pipelined:
            return None
        entries = launched.plan.entries
        if len(entries) != len(self.scheduler.running) or not all(e.count == 1 and e.samples for e in entries):
            return None
        following = []
        reserved = [0] * len(self.engine.cache.groups)
        for e in entries:
            r = e.request
            if r.status != "running" or r.sampling.needs_text:
                return None
            if len(r.generated) + 2 > r.max_tokens:  # it ends with the launched step's token: plan normally
                return None
            if self.scheduler._affordable(r, 1, reserved) < 1:  # (the launched step's page is already taken)
                return None
            self.scheduler._reserve(r, 1, reserved)
            following.append(PlannedEntry(r, e.start + 1, 1, True))
        return StepPlan(following, [])

    def step(self) -> list[StepOutput]:
        """Run one step (or, in steady decoding, launch the next one and) return what the oldest
        step in flight produced for each sampling request. (What a call that failed had committed comes first.) A request whose constraint
        fails ends, with the error as its `error`; the step goes on for the others and then raises it, and what it produced is the next call's to return."""
        self._advance()
        return self._deliver()

    def _advance(self) -> None:
        if self._in_flight is None:
            plan = self.scheduler.plan()
            if not plan.entries:
                return
            self._in_flight = self._launch(plan)
        launched = self._in_flight
        following = self._next_decode_plan(launched)
        if following is not None:
            self._in_flight = self._launch(following, device_tokens=launched.chosen)
        else:
            self._in_flight = None
        self._held += self._finalize(launched)

    def step_drafted(self, drafts: "Mapping[str, tuple[Sequence[int], Sequence[int] | None]]") -> list[StepOutput]:
        """Run one step in which decoding requests bring drafted tokens, and return what it produced: for a request one token as ever, and one
        more for every draft that it agrees with. The tokens are those of steps without drafts (drawn by the same numbers): a step of
        several rows rounds its sums otherwise than one of single tokens, so in bfloat16 an answer may part where two tokens are as good as equal.

        `drafts`: request id -> (tokens, parents): what may follow the request's latest token, as a tree: `parents[i]` is the earlier
        draft that token i goes on from, -1 the latest token itself; None: each goes on from the one ahead of it. Drafts are left aside where
        pages are short, where generation ends with them or ahead of them, where the request's constraint does not let them come, lets nothing follow or fails at them, in a step that
        reads prompts, and for requests that do not decode. ValueError, and nothing has happened, for drafts that are no such trees and for a
        model whose layers keep other than keys and values. What was committed ahead of a step that fails is the next call's (`step`, `step_drafted`,
        `drain`) to return. A constraint that fails ends its request, as in `step`."""
        runner = self.engine.runner
        why = runner.drafted.why_not()
        if why is not None:
            raise ValueError(why)
        vocab, trees = self.engine.vocab_size, {}
        for name, (tokens, parents) in drafts.items():
            tokens = [int(t) for t in tokens]
            parents = list(range(-1, len(tokens) - 1)) if parents is None else [int(p) for p in parents]
            if len(parents) != len(tokens) or any(not -1 <= p < i for i, p in enumerate(parents)) or any(not 0 <= t < vocab for t in tokens) or \
                    len(tokens) >= ops.MOST_DRAFTED:
                raise ValueError(f"request {name!r}: up to {ops.MOST_DRAFTED - 1} drafts of the vocabulary, each with an earlier parent or -1")
            trees[name] = tokens, parents
        self._land()
        plan = self.scheduler.plan()
        if not plan.entries:
            return self._hand_out()
        if any(e.count != 1 or not e.samples or not e.request.generated for e in plan.entries):
            self._held += self._finalize(self._launch(plan))
            return self._deliver()
        cache, entries, allowed = self.engine.cache, [], []
        reserved = [0] * len(cache.groups)
        for planned in plan.entries:
            self.scheduler._reserve(planned.request, 1, reserved)
        requests: list[Request] = []
        for planned in plan.entries:
            request = planned.request
            try:
                tokens, parents, lets = self._drafts_of(request, *trees.get(request.request_id, ((), ())))
            except Exception as error:
                self._fail_alone(request, error)
                continue
            held = request.cache.tokens
            mine = [cache.pages_for(g, held + len(tokens)) - cache.pages_for(g, held + 1) for g in range(len(cache.groups))]
            if any(r + m > g.pool.free for r, m, g in zip(reserved, mine, cache.groups)):
                tokens, parents, lets, mine = tokens[:1], parents[:1], lets[:1], [0] * len(mine)
            reserved = [r + m for r, m in zip(reserved, mine)]
            requests.append(request)
            entries.append(StepEntry(request.cache, tokens, list(range(len(tokens))), parents))
            allowed += lets
        if not entries:
            return self._deliver()
        try:
            logits = runner.run(entries, copy=False)
            owners, depths = [], []
            for r, entry in enumerate(entries):
                first = len(depths)
                for p in entry.parents:
                    owners.append(r)
                    depths.append(depths[first + p] + 1 if p >= 0 else 0)
            rows = list(range(len(depths)))
            params = [request.sampling for request in requests]
            # (A request's text ends ahead of the step's tokens, the first of which is its latest one.)
            texts = [text_of(p, request.prompt, request.generated[:-1]) for p, request in zip(params, requests)]
            chosen = sample_drafted(logits, runner.drafted.last[1], rows, owners, depths, params, [self._seeds[r.request_id] for r in requests],
                                    [len(r.generated) for r in requests], texts, allowed)
            kept = runner.keep(entries, chosen)
        except Exception as error:
            for request in requests:  # a failed step fails its requests
                self._fail(request, error)
            raise
        for request, mine in zip(requests, kept):
            for token in [*mine.tokens, mine.next]:
                some = self.scheduler.commit(StepPlan([PlannedEntry(request, request.computed, 1, True)], []), {request.request_id: token})
                for output in some:
                    if output.token is not None:
                        request.meter.token()
                self._held += some
                if request.status != "running":
                    self._seeds.pop(request.request_id, None)
                    break
        return self._deliver()

    def _drafts_of(self, request: Request, drafts: Sequence[int], above: Sequence[int]) -> "tuple[list[int], list[int], list[np.ndarray | None]]":
        """What a request brings to a step with these drafts: its latest token and the drafts that may come behind it, for each the one that it goes on
        from and what may follow it. What is left out: the request's last token and its stop tokens, which nothing is chosen behind; drafts that its
        constraint does not let come there (it is asked only about texts that it let come), lets nothing follow or fails at (should such a text
        come, it ends the request then); and what goes on from such."""
        vocab = self.engine.vocab_size
        lets = allowed_ids(request.sampling, request.generated)
        tokens, parents, rules, allowed = [request.generated[-1]], [-1], [lets], [id_array(lets, vocab)]
        ways: list[list[int]] = [[]]
        places = {-1: 0}  # of the drafts, those that stay: their place
        for i, (token, p) in enumerate(zip(drafts, above)):
            at = places.get(p)
            if at is None or len(request.generated) + len(ways[at]) + 1 >= request.max_tokens or token in request.stop:
                continue
            if rules[at] is not None and token not in rules[at]:
                continue
            way, lets = [*ways[at], token], None
            try:
                lets = allowed_ids(request.sampling, [*request.generated, *way])
                ids = id_array(lets, vocab)
            except Exception:
                continue
            places[i] = len(tokens)
            tokens.append(token)
            parents.append(at)
            rules.append(lets)
            allowed.append(ids)
            ways.append(way)
        return tokens, parents, allowed

    def resize_cache(self, tokens: int) -> None:
        """Give the page pools of a running engine room for `tokens` positions, more or fewer: what live requests hold is kept
        (CacheError where it would not fit, and nothing changed). A step in flight, which steady decoding leaves behind every `step()`, is a ValueError:
        `drain()` first, and read the outputs that it returns. Captured steps are made anew."""
        if self._in_flight is not None:
            raise ValueError("a step is in flight; drain() it and read its outputs first")
        engine = self.engine
        if any(r.max_tokens + len(r.prompt) > tokens for r in [*self.scheduler.running, *self.scheduler.waiting]):
            raise ValueError(f"a live request may grow past {tokens} tokens")
        engine.runner.forget_graphs()  # ahead of the change: none outlives the tensors it was captured on, and their memory is free for the new ones
        engine.cache.resize(-(-tokens // engine.cache.page_size))
        engine.cache_tokens, self.scheduler.capacity = tokens, engine.cache.capacity_tokens()

    def run(self) -> None:
        """Step until every request has finished."""
        while not self.scheduler.idle or self._in_flight is not None:
            self._idle(self.step())

    def _idle(self, outputs: list[StepOutput]) -> None:
        if not outputs and self._in_flight is None and not self.scheduler.running and self.scheduler.waiting:
            raise RuntimeError("the scheduler can admit nothing: the cache pool is too small")

    def advance_for(self, requests: Sequence[Request]) -> list[StepOutput]:
        """`step` for a caller that goes by its own requests: of constraints that failed, only theirs are raised."""
        self._advance()
        self._failed = [r for r in self._failed if any(r is mine for mine in requests)]
        return self._deliver()

    def generate(self, prompts: Sequence[Sequence[int]], options: GenerationOptions, *, samples: int = 1,
                 share: bool = False) -> list[list[int]]:
        """Generate for all prompts together; returns the generated ids per prompt.

        `samples`: answers to every prompt, one after the other in what is returned. The prompt is read once, and every answer
        goes on from there with draws of its own (the sampler's seed + i for answer i where a seed is given).
        `share`: tokens that all of the prompts begin with are read once for all of them. Either way the answers' steps read the keys and
        values of what they share once for all where that pays (on captured steps: when their graph is worth its capture, which depends on the steps
        before), and this rounds otherwise than reading them request by request: in bfloat16 an answer may part from the one that its prompt has by
        itself, or had in another call, where two tokens are as good as equal."""
        if samples < 1:
            raise ValueError("samples must be at least 1")
        prompts = [[int(t) for t in p] for p in prompts]
        start = common_start([p[:-1] for p in prompts]) if share and len(prompts) > 1 else 0
        requests: list[Request] = []
        for prompt in prompts:
            follows = {"leader": requests[0], "fork_at": start} if requests and start else {}
            first = self.add(prompt, options, **follows)
            requests.append(first)
            for i in range(1, samples):
                seed = options.sampler.seed
                draws = options if seed is None else \
                    dataclasses.replace(options, sampler=dataclasses.replace(options.sampler, seed=seed + i))
                requests.append(self.add(prompt, draws, leader=first))
        try:
            while not self.scheduler.idle or self._in_flight is not None:
                self._idle(self.advance_for(requests))
        except BaseException:
            for request in requests:  # the others are not left behind
                if request.status != "finished":
                    self.abort(request.request_id)
            raise
        ops.raise_on_error(self.engine.runtime.device)
        return [r.generated for r in requests]


class LanguageModel:
    """What `load` returns: a model that streams text (or token ids)."""

    def __init__(self, engine: Engine, tokenizer=None, defaults: GenerationDefaults | None = None,
                 **generator_args) -> None:
        self.engine = engine
        self.tokenizer = tokenizer or TokenIdTokenizer()
        self.defaults = defaults or GenerationDefaults(tuple(engine.architecture.stop_tokens(engine.config)))
        self.generator = Generator(engine, stop=self.defaults.stop, **generator_args)

    def _ids(self, prompt) -> list[int]:
        if isinstance(prompt, Text):
            prompt = prompt.prompt
        return list(self.tokenizer.encode(prompt)) if isinstance(prompt, str) else [int(t) for t in prompt]

    def stream(self, input, options: GenerationOptions) -> Iterator[Segment]:
        """Generate for one prompt, yielding each token as it is chosen. A segment's text is
        whole characters: bytes that do not yet end one wait for the token that completes them."""
        request = self.generator.add(self._ids(input), options)
        pieces = Detokenizer(self.tokenizer)
        try:
            while request.status != "finished":
                for output in self.generator.advance_for([request]):
                    if output.request is request and output.token is not None:
                        yield Segment(pieces.feed(output.token), output.token)
            if request.error is not None:  # (met in a step that another stream took)
                raise request.error
            rest = pieces.flush()
            if rest:
                yield Segment(rest, -1)
        finally:
            if request.status != "finished":
                self.generator.abort(request.request_id)

    def generate(self, inputs: Sequence, options: GenerationOptions, *, samples: int = 1, share: bool = False) -> list[list[int]]:
        """Generate for several prompts in one continuous batch; ids per prompt, `samples` answers to each one after the other. What the
        answers to a prompt (and with `share` all prompts) have in common is read and kept once: see `Generator.generate`."""
        return self.generator.generate([self._ids(p) for p in inputs], options, samples=samples, share=share)


def load(model: str | Path, *, dtype=None, quantize=None, page_size: int = 16, cache_tokens: int | None = None,
         max_requests: int = 64, max_tokens_per_step: int = 2048, device: str = "cuda:0") -> LanguageModel:
    """Load a model folder (config.json + safetensors, and tokenizer.json / generation_config.json
    where it has them).

    dtype: None or "bfloat16" keeps the checkpoint's bfloat16; "float32" runs everything
    in true 32-bit. `quantize` exists in the reference's signature; this engine has no
    quantised path and refuses it. The remaining arguments size the engine: tokens per
    cache page, tokens the page pool holds (None: sized from the device memory that is free
    once the weights are placed), live requests, tokens per step."""
    if quantize is not None:
        raise ValueError("quantised weights are not part of this engine")
    if isinstance(dtype, torch.dtype):
        dtype = {v: k for k, v in DTYPES.items()}[dtype]
    folder = Path(model)
    if not (folder / "config.json").exists():
        raise ValueError(f"{folder} is not a model folder (no config.json); hub downloads are not part of this engine")
    engine = Engine.from_folder(folder, EngineArgs(dtype=dtype or "bfloat16", page_size=page_size,
                                                   cache_tokens=cache_tokens, max_requests=max_requests, device=device))
    architecture = engine.architecture
    return LanguageModel(engine, tokenizer=architecture.tokenizer(folder),
                         defaults=architecture.defaults(folder, engine.config), max_tokens_per_step=max_tokens_per_step)
