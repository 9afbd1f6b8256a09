"""Plain implementations, in 64 bits on the host, of what a step of drafted tokens asks for."""

from __future__ import annotations

import math
import random

import numpy as np
import torch


def tree(nodes: int, seed: int, reach: int = 7) -> list[int]:
    """Parents of a tree's nodes: each goes on from one of the last few."""
    rng = random.Random(seed)
    return [-1] + [rng.randint(max(0, j - reach), j - 1) for j in range(1, nodes)]


def chain(nodes: int) -> list[int]:
    return list(range(-1, nodes - 1))


def ways(parents: list[int]) -> list[list[int]]:
    """For every node the nodes on its way, itself the last."""
    found: list[list[int]] = []
    for j, p in enumerate(parents):
        found.append(([] if p < 0 else found[p]) + [j])
    return found


def words(seen: list[list[int]], count: int) -> np.ndarray:
    """Lists of numbers as rows of bits in `count` words."""
    bits = np.zeros((len(seen), 32 * count), dtype=bool)
    for row, which in zip(bits, seen):
        row[which] = True
    return np.packbits(bits, axis=1, bitorder="little").view(np.int32).reshape(len(seen), count)


def attention(q, keys, values, positions, key_positions, sees, scale, window=0, keep=0, run=0, softcap=0.0, sink=None):
    """One request in 64 bits: q [nodes, nq, d], keys [held + nodes, nkv, d], values [.., nkv, dv]; `sees` [nodes, nodes]. -> (out
    [nodes, nq, dv], the same sums over |v|, the largest sum of |q k| scale of a score)"""
    nodes, nq, _ = q.shape
    held = keys.shape[0] - nodes
    group = nq // keys.shape[1]
    q, keys, values = q.double(), keys.double().repeat_interleave(group, 1), values.double().repeat_interleave(group, 1)
    z = torch.einsum("ihd,khd->hik", q, keys) * scale
    size = float((torch.einsum("ihd,khd->hik", q.abs(), keys.abs().nan_to_num(0, 0, 0)) * abs(scale)).max()) if keys.shape[0] else 0.0
    if softcap:
        z = softcap * torch.tanh(z / softcap)
    i, k = positions[:, None], key_positions[None, :]
    seen = torch.ones(nodes, keys.shape[0], dtype=torch.bool)
    if window:
        seen &= (i - k < window) | (k < keep)
    if run:
        seen &= k >= i - i % run
    seen[:, held:] &= sees
    z = torch.where(seen, z, -math.inf)
    if sink is not None:
        z = torch.cat([z, sink.double().view(nq, 1, 1).expand(-1, nodes, 1)], dim=2)
    p = torch.softmax(z, dim=2)[..., : keys.shape[0]] if z.shape[2] else z
    p = torch.where(seen, p, 0.0)  # (a row that sees nothing)
    v = values.permute(1, 0, 2)
    # What a row does not see is not in its sums, whatever it holds.
    clean, dirty = v.nan_to_num(0.0, 0.0, 0.0), ~torch.isfinite(v)
    out = p @ clean
    for h, key in dirty.any(2).nonzero().tolist():
        out[h] += torch.where(p[h, :, key, None] != 0, p[h, :, key, None] * (v[h, key] - clean[h, key]), 0.0)
    return out.permute(1, 0, 2), (p @ clean.abs()).permute(1, 0, 2), size


def adjust(logits, texts, prompts, repetition=None, frequency=None, presence=None, contexts=None, biases=None, masks=None, vocab=None):
    """Rows in 64 bits: `texts[i]` row i's tokens, `prompts[i]` of them given; `biases[i]` pairs, `masks[i]` the allowed ids or None."""
    out = logits.double().clone()
    for i in range(out.shape[0]):
        text = texts[i]
        if repetition is not None:
            context = contexts[i] if contexts is not None else 0
            for v in set(text[max(len(text) - context, 0):] if context else text):
                z = float(out[i, v])
                out[i, v] = z / repetition[i] if z > 0 else z * repetition[i]
        made: dict[int, int] = {}
        for v in text[prompts[i]:]:
            made[v] = made.get(v, 0) + 1
        for v, n in made.items():
            out[i, v] -= (frequency[i] if frequency is not None else 0.0) * n + (presence[i] if presence is not None else 0.0)
        for v, b in (biases[i] if biases is not None else []):
            out[i, v] += b
        if masks is not None and masks[i] is not None:
            allowed = torch.zeros(out.shape[1], dtype=torch.bool)
            allowed[torch.as_tensor(sorted(masks[i]), dtype=torch.long)] = True
            out[i, ~allowed] = -math.inf
    return out


def accept(parents: list[int], ids: list[int], chosen: list[int]) -> list[int]:
    path = [0] if parents else []
    while path:
        child = next((j for j, p in enumerate(parents) if j and p == path[-1] and ids[j] == chosen[path[-1]]), None)
        if child is None:
            break
        path.append(child)
    return path
