"""One call of the sampling kernel for the rows of a step."""

from __future__ import annotations

from collections.abc import Collection, Sequence
from dataclasses import dataclass, replace

import numpy as np
import torch

from mlx_omnia_b200.kernels import ops
from mlx_omnia_b200.sampling.options import SamplingParams


@dataclass(frozen=True)
class Text:
    """What penalties and constraints go by: a request's tokens, how many of them were given to it."""

    tokens: Sequence[int]
    prompt: int


def text_of(params: SamplingParams, prompt: Sequence[int], generated: Sequence[int]) -> Text:
    """As much of a request's text as its penalties look at: what was generated where it is counted, and the last tokens in the repetition
    penalty's sight."""
    made = len(generated) if params.counts else 0
    seen = min(params.penalty_context, len(prompt) + len(generated)) if params.repetition_penalty != 1.0 else 0
    count = max(made, seen)
    old = max(count - len(generated), 0)
    tokens = [*prompt[len(prompt) - old:], *generated[len(generated) - (count - old):]]
    return Text(tokens, old)


def allowed_ids(params: SamplingParams, generated: Sequence[int]) -> "Collection[int] | None":
    """What a request's constraint lets come next (None: anything). ValueError where that is nothing."""
    if params.constraint is None:
        return None
    allowed = params.constraint(generated)
    if allowed is not None and not len(allowed):
        raise ValueError("a constraint allows no token")
    return allowed


def id_array(allowed: "Collection[int] | None", vocab: int) -> np.ndarray | None:
    """What a constraint lets come next as an array. ValueError for a token that there is not."""
    if allowed is None:
        return None
    ids = allowed if isinstance(allowed, np.ndarray) else np.asarray(list(allowed))
    ids = ids.astype(np.int64, copy=False)
    if ids.min() < 0 or ids.max() >= vocab:
        raise ValueError(f"a constraint allows a token outside the vocabulary of {vocab}")
    return ids


def _masks(allowed: "Sequence[Collection[int] | None]", vocab: int, device: torch.device) -> "ops.TokenMasks | None":
    """A mask of bits for every row that has one."""
    some = [i for i, a in enumerate(allowed) if a is not None]
    if not some:
        return None
    width = -(-vocab // 32)
    words = np.empty(len(allowed) + len(some) * width, dtype=np.int32)
    words[: len(allowed)] = -1
    for k, i in enumerate(some):
        ids = id_array(allowed[i], vocab)
        row = np.zeros(width * 32, dtype=bool)
        row[ids] = True
        words[i] = k
        words[len(allowed) + k * width: len(allowed) + (k + 1) * width] = np.packbits(row, bitorder="little").view(np.int32)
    packed = torch.from_numpy(words).to(device, non_blocking=True)
    return ops.TokenMasks(packed[len(allowed):].view(len(some), width), packed[: len(allowed)])


def adjust_rows(logits: torch.Tensor, params: Sequence[SamplingParams], texts: Sequence[Text], allowed: "Sequence[Collection[int] | None]",
                requests: Sequence[int] | None = None, drafted: "ops.DraftedRows | None" = None) -> None:
    """In place: every penalty, bias and constraint of the requests (`params`, `texts`) on their rows of logits (`allowed`: one a row;
    `requests`: the request of each row, where not row i is request i's)."""
    n = len(params)
    counting = any(p.counts or p.repetition_penalty != 1.0 for p in params)
    biases = [p.bias for p in params]
    entries, tokens = sum(len(b) for b in biases), sum(len(x.tokens) for x in texts) if counting else 0
    # One buffer and one copy: the texts' places (8 bytes each) first.
    parts = {"starts": 2 * n, "lengths": n, "prompts": n, "contexts": n, "repetition": n, "frequency": n, "presence": n, "bias_starts": n + 1,
             "requests": 0 if requests is None else len(requests), "bias_ids": entries, "bias_values": entries, "tokens": tokens}
    words, at, place = np.zeros(sum(parts.values()), dtype=np.int32), 0, {}
    for name, size in parts.items():
        place[name] = slice(at, at + size)
        at += size
    real = words.view(np.float32)
    if counting:
        lengths = [len(x.tokens) for x in texts]
        words[place["starts"]].view(np.int64)[:] = np.cumsum([0, *lengths])[:-1]
        words[place["lengths"]], words[place["prompts"]] = lengths, [x.prompt for x in texts]
        words[place["contexts"]] = [p.penalty_context if p.repetition_penalty != 1.0 else 0 for p in params]
        # (A context of 0 sees nothing, and is all of the text to the kernel.)
        real[place["repetition"]] = [p.repetition_penalty if p.penalty_context > 0 else 1.0 for p in params]
        real[place["frequency"]] = [p.frequency_penalty for p in params]
        real[place["presence"]] = [p.presence_penalty for p in params]
        words[place["tokens"]] = [t for x in texts for t in x.tokens]
    words[place["bias_starts"]] = np.cumsum([0, *(len(b) for b in biases)])
    words[place["bias_ids"]], real[place["bias_values"]] = [i for b in biases for i, _ in b], [v for b in biases for _, v in b]
    if requests is not None:
        words[place["requests"]] = requests
    packed = torch.from_numpy(words).to(logits.device, non_blocking=True)
    part = {name: packed[where] for name, where in place.items()}
    floats = {name: part[name].view(torch.float32) for name in ("repetition", "frequency", "presence", "bias_values")}
    ops.adjust_logits(
        logits, history=ops.TokenHistory(part["tokens"], part["starts"].view(torch.int64), part["lengths"], part["prompts"]) if counting else None,
        **({name: floats[name] for name in ("repetition", "frequency", "presence")} | {"contexts": part["contexts"]} if counting else {}),
        requests=None if requests is None else part["requests"],
        bias=ops.LogitBias(part["bias_ids"], floats["bias_values"], part["bias_starts"]) if entries else None,
        masks=_masks(allowed, logits.shape[1], logits.device), drafted=drafted if counting else None, out=logits)


def _adjusted(params: SamplingParams) -> SamplingParams:
    """What is left to do on adjusted logits. (No bias: new parameters check theirs, at every step.)"""
    return params if params.repetition_penalty == 1.0 else replace(params, repetition_penalty=1.0, bias=())


def sample_drafted(logits: torch.Tensor, step, rows: Sequence[int], requests: Sequence[int], depths: Sequence[int], params: Sequence[SamplingParams],
                   seeds: Sequence[int], draws: Sequence[int], texts: Sequence[Text], allowed: "Sequence[Collection[int] | None]") -> torch.Tensor:
    """Choose one token for every row of a step of drafted trees: `rows[i]` the step's row that logits row i belongs to, `requests[i]` its
    request, `depths[i]` how many tokens of the step are ahead of it on its way. `texts` end ahead of the step's tokens. Row i draws what its request
    would without drafts: its draw number is `draws` plus its depth."""
    if any(p.adjusts or p.repetition_penalty != 1.0 for p in params):
        at = torch.as_tensor(np.asarray(rows, dtype=np.int32)).to(logits.device, non_blocking=True)
        adjust_rows(logits, params, texts, allowed, requests, ops.DraftedRows(step.tree, step.token_ids, step.cu_seqlens, at))
    plain = [_adjusted(p) for p in params]
    return _choose(logits, [plain[r] for r in requests], [seeds[r] for r in requests], [draws[r] + d for r, d in zip(requests, depths)], [[]] * len(requests))


def sample_rows(logits: torch.Tensor, params: list[SamplingParams], seeds: list[int], draws: list[int],
                histories: list[list[int]], texts: Sequence[Text] | None = None,
                allowed: "Sequence[Collection[int] | None] | None" = None) -> torch.Tensor:
    """Choose one token per row of float32 `logits` [rows, vocab]. `seeds[i]` and
    `draws[i]` (how many tokens row i's request has drawn so far) fix the random stream;
    `histories[i]` are the request's latest tokens for the repetition penalty. Where a request's options say more about
    logits (`SamplingParams.adjusts`), `texts` and `allowed` are what they go by (`text_of`, `allowed_ids`), and the rows are modified.
    -> int32 [rows] on the device."""
    if any(p.adjusts for p in params):
        adjust_rows(logits, params, texts, allowed)
        params, histories = [_adjusted(p) for p in params], [[]] * len(params)
    return _choose(logits, params, seeds, draws, histories)


def _choose(logits: torch.Tensor, params: list[SamplingParams], seeds: list[int], draws: list[int], histories: list[list[int]]) -> torch.Tensor:
    if all(p.greedy and p.repetition_penalty == 1.0 for p in params):
        return ops.argmax(logits)
    rows = len(params)
    penalised = any(p.repetition_penalty != 1.0 for p in params)
    width = max(p.penalty_context for p in params) if penalised else 0
    # All rows' parameters in one buffer and one copy (`ops.sample` takes them one tensor each).
    words = np.empty((9 if penalised else 8) * rows + rows * width, dtype=np.int32)
    wide, real = words[: 4 * rows].view(np.int64), words.view(np.float32)
    wide[:rows] = [s & 0x7FFFFFFFFFFFFFFF for s in seeds]
    wide[rows:] = draws
    real[4 * rows: 5 * rows] = [p.temperature for p in params]
    words[5 * rows: 6 * rows] = [p.top_k for p in params]
    real[6 * rows: 7 * rows] = [p.top_p for p in params]
    real[7 * rows: 8 * rows] = [p.min_p for p in params]
    if penalised:
        real[8 * rows: 9 * rows] = [p.repetition_penalty for p in params]
        table = words[9 * rows:].reshape(rows, width)
        table.fill(-1)
        for i, (p, h) in enumerate(zip(params, histories)):
            recent = h[-p.penalty_context:] if p.repetition_penalty != 1.0 else []
            table[i, : len(recent)] = recent
    packed = torch.from_numpy(words).to(logits.device, non_blocking=True)
    whole, real = packed[: 4 * rows].view(torch.int64), packed.view(torch.float32)
    part = lambda t, i: t[i * rows: (i + 1) * rows]  # noqa: E731
    return ops.sample(logits, part(real, 4), part(packed, 5), part(real, 6), part(real, 7), part(whole, 0), part(whole, 1),
                      part(real, 8) if penalised else None, packed[9 * rows:].view(rows, width) if penalised else None)
