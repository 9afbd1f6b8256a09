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


# -- the calls of `ops` on the host, in place of the kernels --------------------------------------------------------
def step_tables(held, brought, lists, page_size, tokens, parents=None, most=None):
    from mlx_omnia_b200.kernels import ops

    held, brought = held.tolist(), brought.tolist()
    cu = np.cumsum([0, *brought])
    ints = lambda v, t=torch.int32: torch.tensor(v, dtype=t)  # noqa: E731
    positions, seen = [], []
    for r, b in enumerate(brought):
        tree_of = chain(b) if parents is None else parents[cu[r]: cu[r] + b].tolist()
        for way in ways(tree_of):
            positions.append(held[r] + len(way) - 1)
            seen.append(way)
    groups = []
    for x in lists:
        pages, starts = x.pages.tolist(), x.starts.tolist()
        table, slots = [], []
        for r, (h, b) in enumerate(zip(held, brought)):
            count = -(-(-(-(h + b) // x.stride)) // page_size)
            mine = pages[starts[r]: starts[r] + count]
            table.append(mine + [-1] * (x.width - count))
            slots += [mine[(h + j) // x.stride // page_size] * page_size + (h + j) // x.stride % page_size for j in range(b)]
        groups.append((ints(table), ints(slots, torch.int64)))
    made = ops.StepTree(torch.from_numpy(words(seen, -(-most // 32)))) if most is not None else None
    return ops.StepTables(ints(positions), ints(cu.tolist()), ints([h + b for h, b in zip(held, brought)]), groups, made)


def tree_attention(q, kv, step, scale, gate=None, gate_col=0, sink=None, window=-1, keep_first=None, chunk=None, softcap=None):
    tokens, nq, d = q.shape
    window = (kv.window if window == -1 else window) or 0
    keep = kv.keep_first if keep_first is None else keep_first
    k_row, v_row = kv.row(0), kv.row(1)
    out = torch.zeros(tokens, nq, v_row.shape[3], dtype=torch.float64)
    cu = step.cu_seqlens.tolist()
    for r, (first, end) in enumerate(zip(cu, cu[1:])):
        n, length = end - first, int(step.seq_lens[r])
        at = torch.arange(length)
        pages = kv.block_table[r, at // kv.page_size].long().clamp(min=0)  # (what was given back no row sees)
        k, v = (x[pages, :, at % kv.page_size] for x in (k_row, v_row))
        bits = np.unpackbits(step.tree.ancestors[first:end].numpy().view(np.uint8), axis=1, bitorder="little")[:, :n]
        positions = step.positions[first:end].long()
        out[first:end] = attention(q[first:end], k, v, positions, torch.cat([torch.arange(length - n), positions]), torch.from_numpy(bits).bool(), scale,
                                   window, keep if window else 0, chunk or 0, softcap or 0.0, sink)[0]
    out = out.reshape(tokens, -1)
    if gate is not None:
        out = out * torch.sigmoid(gate[:, gate_col: gate_col + out.shape[1]].double())
    return out.to(q.dtype)


def accept_drafts(chosen, token_ids, tree_of, cu_seqlens):
    from mlx_omnia_b200.kernels import ops

    cu, most = cu_seqlens.tolist(), 32 * tree_of.ancestors.shape[1]
    paths, last = [], []
    for first, end in zip(cu, cu[1:]):
        bits = np.unpackbits(tree_of.ancestors[first:end].numpy().view(np.uint8), axis=1, bitorder="little")
        parents = [max(np.flatnonzero(row[:j]), default=-1) for j, row in enumerate(bits)]
        path = accept(parents, token_ids[first:end].tolist(), chosen[first:end].tolist())
        paths.append(path + [-1] * (most - len(path)))
        last.append(int(chosen[first + path[-1]]) if path else -1)
    kept = [sum(j >= 0 for j in p) for p in paths]
    return ops.Accepted(*(torch.tensor(x, dtype=torch.int32) for x in (paths, kept, last)))


def keep_rows(pages, rows, page_size, block_table, held, accepted):
    flat, at = pages.flatten(2), 0
    for heads, width in rows:
        size = heads * page_size * width
        block = flat[:, :, at: at + size].unflatten(2, (heads, page_size, width))
        for r, path in enumerate(accepted.path.tolist()):
            for i, j in enumerate(path[: int(accepted.kept[r])]):
                to, src = int(held[r]) + i, int(held[r]) + j
                block[:, block_table[r, to // page_size], :, to % page_size] = block[:, block_table[r, src // page_size], :, src % page_size].clone()
        at += size
    return pages


def adjust_logits(logits, *, history=None, repetition=None, frequency=None, presence=None, contexts=None, requests=None, bias=None, masks=None,
                  drafted=None, out=None):
    rows, vocab = logits.shape
    owner = list(range(rows)) if requests is None else requests.tolist()
    texts, prompts = [[]] * rows, [0] * rows
    if history is not None:
        whole = [history.tokens[s: s + n].tolist() for s, n in zip(history.starts.tolist(), history.lengths.tolist())]
        texts, prompts = [list(whole[r]) for r in owner], [int(history.prompts[r]) for r in owner]
        if drafted is not None:
            cu = drafted.cu_seqlens.tolist()
            for i, t in enumerate(drafted.rows.tolist()):
                bits = np.unpackbits(drafted.tree.ancestors[t].numpy().view(np.uint8), bitorder="little")
                texts[i] += [int(drafted.token_ids[cu[owner[i]] + m]) for m in np.flatnonzero(bits)]
    pick = lambda t: None if t is None else [t[r].item() for r in owner]  # noqa: E731
    biases = None
    if bias is not None:
        starts = bias.starts.tolist()
        biases = [list(zip(bias.ids[starts[r]: starts[r + 1]].tolist(), bias.values[starts[r]: starts[r + 1]].tolist())) for r in owner]
    allowed = None
    if masks is not None:
        bits = np.unpackbits(masks.words.numpy().view(np.uint8), axis=1, bitorder="little")[:, :vocab]
        allowed = [None if w < 0 else np.flatnonzero(bits[w]).tolist() for w in masks.rows.tolist()]
    made = adjust(logits, texts, prompts, pick(repetition), pick(frequency), pick(presence), pick(contexts), biases, allowed).float()
    if out is None:
        return made
    out.copy_(made)
    return out


def swap_in(monkeypatch, ops):
    """The calls above in place of the kernels'."""
    plain = ops.paged_attention

    def paged_attention(q, kv, step, scale, **more):
        if step.tree is None:
            return plain(q, kv, step, scale, **more)
        return tree_attention(q, kv, step, scale, **more)

    for name, call in (("step_tables", step_tables), ("accept_drafts", accept_drafts), ("keep_rows", keep_rows), ("adjust_logits", adjust_logits),
                       ("paged_attention", paged_attention)):
        monkeypatch.setattr(ops, name, call)
