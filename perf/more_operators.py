"""What a step that reads drafted tokens asks of the framework, as cases that can be timed and compared: the step's tables
(positions, slots, block tables, what each drafted token descends from), attention of trees of drafted tokens over a paged
cache, penalties, biases and masks on the logits of their rows, and what becomes of the drafts that the model agrees with.

A case is a dict of plain values; `prepare` makes its inputs from a seed, `run` is one pass: in plain torch operations
in 32 bits, or, where `own` is true, as the calls that a program makes of `mlx_omnia_b200.kernels.ops`.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

# Query heads, key/value heads, head size, element type: the layers of the benchmark's models of 1.7 and 8 billion
# parameters and of its sliding-window family, and of the tests' small models (one in 32 bits).
LAYOUTS = {"16/8x128": (16, 8, 128, "bfloat16"), "32/8x128": (32, 8, 128, "bfloat16"), "16/4x128": (16, 4, 128, "bfloat16"),
           "6/2x64": (6, 2, 64, "bfloat16"), "8/1x24 f32": (8, 1, 24, "float32"), "16/8x128 f32": (16, 8, 128, "float32")}

# What a page holds in every layer that keeps pages: layers, key/value heads, tokens a page, head size, element type.
POOLS = {"28 layers": (28, 8, 16, 128, "bfloat16"), "36 layers": (36, 8, 16, 128, "bfloat16"),
         "3 layers f32": (3, 1, 8, 24, "float32")}

VOCABS = [151936, 32003, 1000, 777]  # the benchmark's models', an odd one, the tests' small models'


def listed():
    tables = {"op": "tables", "page": 16, "groups": 1, "stride": 1}
    attention = {"op": "attention", "page": 16, "chain": False, "gated": True, "sink": False, "softcap": 0.0, "window": 0}
    logits = {"op": "logits", "vocab": 151936, "penalties": True, "biases": 0, "masks": 0.0, "nodes": 0}
    return [
        # Eight requests decode a token each: what a call costs at the least.
        tables | {"name": "tables, 8 decode", "requests": 8, "held": 4096, "brought": 1, "trees": False},
        # Sixty-four requests of long contexts bring a tree of 64 drafted tokens each, in a model with two kinds of cache.
        tables | {"name": "tables, 64 trees of 64", "requests": 64, "held": 32768, "brought": 64, "trees": True, "groups": 2},
        # One request in the middle of a short answer, and four tokens that a look-up proposes one after the other.
        attention | {"name": "a chain of 5, 500 held", "layout": "16/8x128", "requests": 1, "held": 500, "brought": 5, "chain": True},
        # Eight requests at the benchmark's context with a small tree each.
        attention | {"name": "8 trees of 16, 4096 held", "layout": "16/8x128", "requests": 8, "held": 4096, "brought": 16},
        # Thirty-two requests of 8,192 positions with wide trees: as many products as the cache has bytes.
        attention | {"name": "32 trees of 64, 8192 held", "layout": "32/8x128", "requests": 32, "held": 8192, "brought": 64},
        # The largest cache: four requests over documents as long as a long-context model takes.
        attention | {"name": "4 trees of 24, 131072 held", "layout": "32/8x128", "requests": 4, "held": 131072, "brought": 24},
        # The 32-bit path at the tests' odd head size: sinks, capped scores, a window, odd lengths.
        attention | {"name": "32-bit trees of 13", "layout": "8/1x24 f32", "requests": 12, "held": 1001, "brought": 13, "page": 8,
                     "gated": False, "sink": True, "softcap": 30.0, "window": 700},
        # One answer with penalties, a few hundred tokens long.
        logits | {"name": "a row's penalties", "rows": 1, "history": 300},
        # A full batch of answers to long prompts, with penalties and the biases that their callers gave.
        logits | {"name": "64 rows, penalties and biases", "rows": 64, "history": 6000, "biases": 40},
        # Trees under a grammar: every drafted token's row has a mask of its own and penalties along its path.
        logits | {"name": "16 trees of 32 under masks", "rows": 512, "history": 2000, "masks": 0.9, "nodes": 32},
        # One request keeps what the model agrees with of a dozen drafted tokens.
        {"op": "accept", "name": "keep of 12 drafted", "pool": "28 layers", "requests": 1, "brought": 12, "held": 245},
        # A full batch keeps what it agrees with of 64 drafted tokens each.
        {"op": "accept", "name": "keep of 64 trees of 64", "pool": "36 layers", "requests": 64, "brought": 64, "held": 300},
    ]


def _spread(rng, low, high):
    """A whole number between `low` and `high`, even over the logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.random()
    if kind < 0.2:
        trees = rng.random() < 0.6
        return {"op": "tables", "page": rng.choice([8, 16, 16, 32, 48]), "groups": rng.choice([1, 1, 2, 3]),
                "stride": 1 if trees else rng.choice([1, 1, 2, 4]), "requests": _spread(rng, 1, 64), "held": _spread(rng, 1, 32768),
                "brought": _spread(rng, 1, 64), "trees": trees}
    if kind < 0.35:
        pool = rng.choice(sorted(POOLS))
        return {"op": "accept", "pool": pool, "requests": _spread(rng, 1, 64), "brought": rng.randint(1, 64), "held": _spread(rng, 1, 300)}
    if kind < 0.6:
        nodes = rng.choice([0, 0, rng.randint(1, 64)])
        vocab = rng.choice([VOCABS[0], VOCABS[0], *VOCABS])
        case = {"op": "logits", "vocab": vocab, "penalties": rng.random() < 0.8, "biases": rng.choice([0, 0, rng.randint(1, 100)]),
                "masks": rng.choice([0.0, 0.0, 1.0, 0.5]), "nodes": nodes, "history": _spread(rng, 1, 8000),
                "rows": nodes * _spread(rng, 1, max(1, 400 // nodes)) if nodes else _spread(rng, 1, 400)}
        if not (case["penalties"] or case["biases"] or case["masks"]):
            case["penalties"] = True
        return case
    layout = rng.choice(["16/8x128", "16/8x128", "32/8x128", "32/8x128", "16/4x128", "6/2x64", "8/1x24 f32", "16/8x128 f32"])
    small = layout.endswith("f32")
    tops = [work(c) for c in listed() if c["op"] == "attention"]
    case = {"op": "attention", "layout": layout, "page": rng.choice([8, 16, 32] if small else [16, 16, 32, 48]),
            "chain": rng.random() < 0.25, "gated": rng.random() < 0.5, "sink": rng.random() < 0.25,
            "softcap": 30.0 if rng.random() < 0.15 else 0.0, "window": _spread(rng, 20, 4000) if rng.random() < 0.2 else 0,
            "requests": _spread(rng, 1, 16 if small else 48), "held": _spread(rng, 1, 3000 if small else 131072),
            "brought": _spread(rng, 1, 32 if small else 100)}
    while any(work(case)[k] > max(t[k] for t in tops) for k in ("bytes", "flops")):
        smaller = "held" if case["held"] > 2000 or case["requests"] == 1 else "requests"
        case[smaller] //= 2
    return case


# -- requests, trees and pages ---------------------------------------------------------------------------------------
def _lengths(case):
    """(positions that each request holds, tokens that each brings), the same for every seed."""
    rng = random.Random(f"{case['requests']} {case['held']} {case['brought']}")
    n = case["requests"]
    held = [rng.randint(case["held"] // 3, case["held"]) for _ in range(n)]
    brought = [rng.randint(1 + case["brought"] // 2, case["brought"]) if case["brought"] > 1 else 1 for _ in range(n)]
    at = rng.randrange(n)
    held[at], brought[at] = case["held"], case["brought"]
    return held, brought


def _trees(brought, seed, chain=False):
    """The parent of every drafted token within its request's, -1 for the first: each token goes on from one of the last few."""
    rng = random.Random(seed)
    return [[-1] + [j - 1 if chain else rng.randint(max(0, j - 6 if j < 12 else j - 16), j - 1) for j in range(1, n)] for n in brought]


def _pages(lengths, page, seed):
    """(a list of pages for each request of so many rows, in any order; pages in all)"""
    counts = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(counts), generator=torch.Generator().manual_seed(seed)).numpy().astype(np.int32)
    return np.split(order, np.cumsum(counts)[:-1]), int(sum(counts))


def _sees(trees):
    """For every drafted token which of its request's it descends from (itself too): rows of truth values, as wide as the widest tree."""
    most = max(len(t) for t in trees)
    sees = np.zeros((sum(len(t) for t in trees), most), dtype=bool)
    at = 0
    for tree in trees:
        for j, p in enumerate(tree):
            if p >= 0:
                sees[at + j] = sees[at + p]
            sees[at + j, j] = True
        at += len(tree)
    return sees


def _words(sees):
    """Truth values as bits of 32-bit words, the first the lowest."""
    padded = np.zeros((sees.shape[0], -(-sees.shape[1] // 32) * 32), dtype=bool)
    padded[:, : sees.shape[1]] = sees
    return np.packbits(padded, axis=1, bitorder="little").view(np.int32)


def _ints(values, dtype=torch.int32):
    return torch.as_tensor(np.asarray(values), device="cuda").to(dtype)


# -- tables ----------------------------------------------------------------------------------------------------------
def _tables_inputs(case, seed):
    held, brought = _lengths(case)
    page, stride = case["page"], case["stride"]
    trees = _trees(brought, seed)
    s = {"held": _ints(held), "brought": _ints(brought), "tokens": sum(brought), "most": max(brought),
         "parents": _ints([p for t in trees for p in t]) if case["trees"] else None, "lists": []}
    for g in range(case["groups"]):
        step = stride if g == 0 else 1
        lists, _ = _pages([-(-(h + b) // step) for h, b in zip(held, brought)], page, 7 * seed + g)
        starts = np.cumsum([0] + [len(x) for x in lists])[:-1]
        s["lists"].append((_ints(np.concatenate(lists)), _ints(starts, torch.int64), max(len(x) for x in lists), step))
    return s


def _tables_plain(s):
    case, held, brought, page = s["case"], s["held"].long(), s["brought"].long(), s["case"]["page"]
    device = held.device
    ends = torch.cumsum(brought, 0)
    cu = torch.cat([torch.zeros(1, dtype=torch.int64, device=device), ends])
    token = torch.arange(s["tokens"], device=device)
    request = (token[:, None] >= ends[None, :]).sum(1)
    node = token - cu[request]
    words = None
    depth = node
    if s["parents"] is not None:
        most = s["most"]
        bits = torch.arange(-(-most // 32) * 32, device=device)
        parent = s["parents"].long()
        sees = torch.zeros(held.shape[0], most, bits.shape[0], dtype=torch.bool, device=device)
        for j in range(most):  # a level after the other: a parent comes ahead of its children
            at = torch.minimum(cu[:-1] + j, ends - 1)
            up = parent[at]
            above = sees.gather(1, up.clamp(min=0)[:, None, None].expand(-1, 1, bits.shape[0]))[:, 0]
            sees[:, j] = (above & (up >= 0)[:, None]) | (bits == j)
        mine = sees[request, node]
        depth = mine.sum(1) - 1
        words = (mine.view(s["tokens"], -1, 32).long() << (bits % 32).view(1, -1, 32)).sum(2)
        words = torch.where(words >= 2 ** 31, words - 2 ** 32, words).int()
    out = {"positions": (held[request] + depth).int(), "cu_seqlens": cu.int(), "seq_lens": (held + brought).int(), "ancestors": words, "groups": []}
    for pages, starts, width, stride in s["lists"]:
        row = (held[request] + node) // stride
        slots = pages[starts[request] + row // page].long() * page + row % page
        count = ((held + brought + stride - 1) // stride + page - 1) // page
        column = torch.arange(width, device=device)[None]
        at = torch.minimum(starts[:, None] + column, torch.full_like(column, pages.shape[0] - 1))
        out["groups"].append((torch.where(column < count[:, None], pages[at].long(), -1).int(), slots))
    return out


def _tables_exact(case, seed):
    s = _tables_inputs(case, seed)
    held, brought, page = s["held"].tolist(), s["brought"].tolist(), case["page"]
    trees = _trees(brought, seed, chain=not case["trees"])
    sees = _sees(trees)
    positions = np.repeat(held, brought) + sees.sum(1) - 1
    out = {"positions": positions.astype(np.int32), "cu_seqlens": np.cumsum([0] + brought).astype(np.int32),
           "seq_lens": np.add(held, brought).astype(np.int32), "ancestors": _words(sees) if case["trees"] else None, "groups": []}
    for pages, starts, width, stride in s["lists"]:
        pages, starts = pages.tolist(), starts.tolist()
        table = np.full((len(held), width), -1, dtype=np.int32)
        slots = []
        for r, (h, b) in enumerate(zip(held, brought)):
            count = -(-(-(-(h + b) // stride)) // page)
            table[r, :count] = pages[starts[r]: starts[r] + count]
            for j in range(b):
                at, off = divmod((h + j) // stride, page)
                slots.append(pages[starts[r] + at] * page + off)
        out["groups"].append((table, np.asarray(slots, dtype=np.int64)))
    return out


# -- attention -------------------------------------------------------------------------------------------------------
def _attention_inputs(case, seed):
    nq, nkv, d, dtype = LAYOUTS[case["layout"]]
    dtype = getattr(torch, dtype)
    held, brought = _lengths(case)
    lists, count = _pages([h + b for h, b in zip(held, brought)], case["page"], seed)
    table = np.full((len(held), max(len(x) for x in lists)), -1, dtype=np.int64)
    for r, x in enumerate(lists):
        table[r, : len(x)] = x
    g = torch.Generator(device="cuda").manual_seed(seed)
    tokens = sum(brought)
    sees = _sees(_trees(brought, seed, case["chain"]))
    # Projected rows as a layer has them: the queries (normed, here beside them) and the gate's columns.
    return {"cache": torch.randn(count, 2, nkv, case["page"], d, generator=g, device="cuda", dtype=dtype),
            "q": torch.randn(tokens, nq, d, generator=g, device="cuda", dtype=dtype),
            "rows": torch.randn(tokens, 2 * nq * d, generator=g, device="cuda", dtype=dtype),
            "sink": torch.randn(nq, generator=g, device="cuda") if case["sink"] else None,
            "table": _ints(table), "held": held, "brought": brought, "sees": torch.from_numpy(sees).cuda(),
            "words": _ints(_words(sees)), "positions": _ints(np.repeat(held, brought) + sees.sum(1) - 1)}


def _attention_plain(s):
    """Requests side by side, each with as many held keys and drafted tokens as the largest has."""
    case, q, cache = s["case"], s["q"], s["cache"]
    nq, nkv, d, _ = LAYOUTS[case["layout"]]
    group, page = nq // nkv, case["page"]
    n, most, before, nodes, rows = len(s["held"]), max(s["brought"]), s["at_held"], s["at_nodes"], s["row_of"]
    table = s["table"].long()

    def stored(at):  # [requests, positions] -> keys and values [requests, nkv, positions, d]
        where = table.gather(1, at // page)
        return [cache[where, w, :, at % page].float().transpose(1, 2) for w in (0, 1)]

    x = (q.float() * d ** -0.5)[rows].view(n, most, nkv, group, d).permute(0, 2, 3, 1, 4).reshape(n, nkv, group * most, d)
    (kb, vb), (km, vm) = stored(before), stored(nodes)
    z = torch.cat([x @ kb.transpose(2, 3), x @ km.transpose(2, 3)], dim=3)
    if case["softcap"]:
        z = case["softcap"] * torch.tanh(z / case["softcap"])
    z = torch.where(s["visible"].repeat(1, group, 1)[:, None], z, -torch.inf)
    top = z.amax(3, keepdim=True)
    p = torch.exp(z - top)
    total = p.sum(3, keepdim=True)
    if case["sink"]:
        sink = s["sink"].view(1, nkv, group, 1, 1).expand(n, nkv, group, most, 1).reshape(n, nkv, group * most, 1)
        total = total + torch.exp(sink - top)
    p = p / total
    out = p[..., : kb.shape[2]] @ vb + p[..., kb.shape[2]:] @ vm
    out = out.view(n, nkv, group, most, d).permute(0, 3, 1, 2, 4).reshape(n * most, nq * d)[s["flat_of"]]
    if case["gated"]:
        out = out * torch.sigmoid(s["rows"][:, nq * d:].float())
    return out.to(q.dtype)


def _attention_exact(case, seed):
    s = _attention_inputs(case, seed)
    nq, nkv, d, _ = LAYOUTS[case["layout"]]
    answers, at = [], 0
    for r, (h, b) in enumerate(zip(s["held"], s["brought"])):
        where = torch.arange(h + b, device="cuda")
        kept = s["cache"][s["table"][r].long()[where // case["page"]], :, :, where % case["page"]]  # [h + b, 2, nkv, d]
        mine = s["positions"][at: at + b].long()
        key = torch.cat([torch.arange(h, device="cuda"), mine])
        seen = torch.cat([torch.ones(b, h, dtype=torch.bool, device="cuda"), s["sees"][at: at + b, :b]], dim=1)
        if case["window"]:
            seen &= mine[:, None] - key[None] < case["window"]
        for k in range(nkv):
            group = nq // nkv
            q = s["q"][at: at + b, k * group: (k + 1) * group].double()  # [b, group, d]
            z = torch.einsum("jgd,pd->jgp", q, kept[:, 0, k].double()) / math.sqrt(d)
            if case["softcap"]:
                z = case["softcap"] * torch.tanh(z / case["softcap"])
            z = z.masked_fill(~seen[:, None], -math.inf)
            if case["sink"]:
                z = torch.cat([z, s["sink"].double()[None, k * group: (k + 1) * group, None].expand(b, -1, -1)], dim=2)
            answers.append(torch.softmax(z, dim=2)[..., : h + b] @ kept[:, 1, k].double())
        answers[-nkv:] = [torch.cat(answers[-nkv:], dim=1).reshape(b, nq * d)]
        at += b
    out = torch.cat(answers)
    return out / (1 + torch.exp(-s["rows"][:, nq * d:].double())) if case["gated"] else out


def _step(s):
    """The step and the cache view that a model's layers are handed."""
    from mlx_omnia_b200.kernels import ops
    from mlx_omnia_b200.parts.base import KVSpec, KVView, StepContext

    case, held, brought = s["case"], s["held"], s["brought"]
    _, nkv, d, _ = LAYOUTS[case["layout"]]
    n, lengths = len(held), [h + b for h, b in zip(held, brought)]
    step = StepContext(
        num_tokens=sum(brought), num_seqs=n, token_ids=_ints([0] * sum(brought)), positions=s["positions"],
        cu_seqlens=_ints(np.cumsum([0] + brought)), seq_lens=_ints(lengths), state_slots=_ints([0] * n), fresh=_ints([0] * n),
        logit_rows=_ints([]), q_lens=brought, seq_lens_host=lengths, max_q_len=max(brought), max_seq_len=max(lengths),
        decode_only=False, groups={}, tree=ops.StepTree(s["words"]))
    spec = KVSpec.keys_and_values(nkv, d, case["window"] or None)
    return step, KVView(s["cache"], s["table"], torch.zeros(sum(brought), dtype=torch.int64, device="cuda"), case["page"],
                        case["window"] or None, spec=spec)


# -- logits ----------------------------------------------------------------------------------------------------------
def _logits_inputs(case, seed):
    rng = np.random.default_rng(seed)
    shape = random.Random(f"{case['rows']} {case['history']} {case['nodes']}")
    rows, vocab, nodes = case["rows"], case["vocab"], case["nodes"]
    n = rows // nodes if nodes else rows
    lengths = [shape.randint(case["history"] // 2, case["history"]) for _ in range(n)]
    prompts = [shape.randint(0, x) for x in lengths]
    # Tokens as answers have them: a few of them again and again.
    text = lambda count: np.minimum((rng.pareto(0.6, count) * 3).astype(np.float64), vocab - 1).astype(np.int32) * 7919 % vocab  # noqa: E731
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"logits": torch.randn(rows, vocab, generator=g, device="cuda") * 4, "tokens": _ints(text(sum(lengths))),
         "starts": _ints(np.cumsum([0] + lengths)[:-1], torch.int64), "lengths": _ints(lengths), "prompts": _ints(prompts),
         "requests": _ints(np.repeat(np.arange(n), nodes or 1)), "penalties": None, "bias": None, "masks": None, "drafted": None}
    if case["penalties"]:
        s["penalties"] = [torch.from_numpy(rng.uniform(*r, n).astype(np.float32)).cuda() for r in ((1.0, 1.5), (0.0, 1.0), (0.0, 1.0))]
    if case["biases"]:
        counts = [shape.randint(0, case["biases"]) for _ in range(n)]
        ids = [rng.choice(vocab, c, replace=False).astype(np.int32) for c in counts]
        s["bias"] = (_ints(np.concatenate(ids)), torch.from_numpy(rng.normal(0, 5, sum(counts)).astype(np.float32)).cuda(),
                     _ints(np.cumsum([0] + counts)))
    if case["masks"]:
        # A grammar allows a handful of tokens in most places and nearly all in others (the inside of a string).
        count = max(1, int(rows * case["masks"]))
        wide = rng.random(count) < 0.25
        allowed = torch.rand(count, -(-vocab // 32) * 32, generator=g, device="cuda") < \
            torch.from_numpy(np.where(wide, 0.97, 30 / vocab)).cuda()[:, None]
        allowed[torch.arange(count), torch.from_numpy(rng.integers(0, vocab, count)).cuda()] = True
        weights = 1 << torch.arange(32, device="cuda")
        words = (allowed.view(count, -1, 32).long() * weights).sum(2)
        which = np.full(rows, -1, dtype=np.int32)
        which[rng.permutation(rows)[:count]] = np.arange(count)
        s["masks"] = (torch.where(words >= 2 ** 31, words - 2 ** 32, words).int(), _ints(which))
    if nodes:
        trees = _trees([nodes] * n, seed)
        sees = _sees(trees)
        s["drafted"] = (_ints(_words(sees)), _ints(text(rows)), _ints(np.arange(n + 1) * nodes), _ints(np.arange(rows)))
        s["sees"] = torch.from_numpy(sees).cuda()
    return s


def _logits_plain(s):
    case, z = s["case"], s["logits"]
    rows, vocab = z.shape
    request = s["requests"].long()
    out = z.clone()
    if s["penalties"] is not None:
        n = s["lengths"].shape[0]
        ends = torch.cumsum(s["lengths"].long(), 0)
        token = torch.arange(s["tokens"].shape[0], device=z.device)
        of = torch.bucketize(token, ends, right=True)
        made = (token - s["starts"][of] >= s["prompts"][of]).float()
        flat = of * vocab + s["tokens"].long()
        seen = torch.zeros(n * vocab, device=z.device).index_add_(0, flat, torch.ones_like(made)).view(n, vocab)[request]
        times = torch.zeros(n * vocab, device=z.device).index_add_(0, flat, made).view(n, vocab)[request]
        if s["drafted"] is not None:
            nodes = case["nodes"]
            ids = s["drafted"][1].long().view(-1, nodes)[request]  # [rows, nodes]: the tokens of the row's tree
            on = s["sees"][:, :nodes].float()
            seen.scatter_add_(1, ids, on)
            times.scatter_add_(1, ids, on)
        repetition, frequency, presence = (p[request][:, None] for p in s["penalties"])
        out = torch.where(seen > 0, torch.where(out > 0, out / repetition, out * repetition), out)
        out = out - frequency * times - presence * (times > 0)
    if s["bias"] is not None:
        ids, values, starts = s["bias"]
        of = torch.bucketize(torch.arange(ids.shape[0], device=z.device), starts[1:].long(), right=True)
        dense = torch.zeros(starts.shape[0] - 1, vocab, device=z.device).index_put_((of, ids.long()), values, accumulate=True)
        out = out + dense[request]
    if s["masks"] is not None:
        words, which = s["masks"]
        bits = torch.arange(32, device=z.device, dtype=torch.int32)
        allowed = ((words[:, :, None] >> bits) & 1).view(words.shape[0], -1)[:, :vocab].bool()
        out = torch.where(allowed[which.long().clamp(min=0)] | (which < 0)[:, None], out, -torch.inf)
    return out


def _logits_exact(case, seed):
    s = _logits_inputs(case, seed)
    rows, vocab = s["logits"].shape
    out = s["logits"].double().cpu().numpy()
    request, starts, lengths, prompts = (s[k].tolist() for k in ("requests", "starts", "lengths", "prompts"))
    tokens = s["tokens"].cpu().numpy()
    penalties = None if s["penalties"] is None else [p.double().cpu().numpy() for p in s["penalties"]]
    bias = None if s["bias"] is None else [t.cpu().numpy() for t in s["bias"]]
    masks = None if s["masks"] is None else [t.cpu().numpy() for t in s["masks"]]
    for i in range(rows):
        r = request[i]
        if penalties is not None:
            text = tokens[starts[r]: starts[r] + lengths[r]]
            made = text[prompts[r]:]
            if s["drafted"] is not None:
                if i % case["nodes"] == 0:
                    drafted = s["drafted"][1][i: i + case["nodes"]].cpu().numpy()
                    sees = s["sees"][i: i + case["nodes"], : case["nodes"]].cpu().numpy()
                made = np.concatenate([made, drafted[sees[i % case["nodes"]]]])
                text = np.concatenate([text, made])
            seen = np.unique(text)
            x = out[i, seen]
            out[i, seen] = np.where(x > 0, x / penalties[0][r], x * penalties[0][r])
            ids, times = np.unique(made, return_counts=True)
            out[i, ids] -= penalties[1][r] * times + penalties[2][r]
        if bias is not None:
            span = slice(bias[2][r], bias[2][r + 1])
            np.add.at(out[i], bias[0][span], bias[1][span].astype(np.float64))
        if masks is not None and masks[1][i] >= 0:
            allowed = np.unpackbits(masks[0][masks[1][i]].view(np.uint8), bitorder="little")[:vocab]
            out[i, allowed == 0] = -np.inf
    return out


# -- accepted drafts -------------------------------------------------------------------------------------------------
def _paths(case):
    """Drafted trees and, for each, the tokens that the model agrees with, the same for every seed: a few of them, as with a good
    drafter, none of which moves to where another that is kept came from."""
    trees = _trees(_lengths(case)[1], f"{case['held']} {case['brought']}")
    paths = []
    for r, tree in enumerate(trees):
        path, which = [0], random.Random(f"{r} {case['brought']}")
        while which.random() < 0.8:
            children = [j for j, p in enumerate(tree) if p == path[-1]]
            if not children:
                break
            new = path + [which.choice(children)]
            if any(i != j and j < len(new) for i, j in enumerate(new)):
                break
            path = new
        paths.append(path)
    return trees, paths


def _accept_inputs(case, seed):
    """Drafted trees and what the model chose behind each token of them."""
    layers, nkv, page, d, dtype = POOLS[case["pool"]]
    held, brought = _lengths(case)
    rng = random.Random(seed)
    trees, paths = _paths(case)
    lists, count = _pages([h + b for h, b in zip(held, brought)], page, seed)
    table = np.full((len(held), max(len(x) for x in lists)), -1, dtype=np.int32)
    for r, x in enumerate(lists):
        table[r, : len(x)] = x
    ids, chosen = [], []
    for tree, path in zip(trees, paths):
        mine = [rng.randrange(1000) for _ in tree]
        picks = [1000 + rng.randrange(1000) for _ in tree]  # tokens that were not drafted
        for a, b in zip(path, path[1:]):
            picks[a] = mine[b]
            for j in range(b + 1, len(tree)):  # a later branch of the same token: the first is kept
                if tree[j] == a and j % 3 == 0:
                    mine[j] = mine[b]
            for j in range(b):  # and no earlier one
                if tree[j] == a and mine[j] == mine[b]:
                    mine[j] = 2500
        last = {mine[j] for j, p in enumerate(tree) if p == path[-1]}
        if picks[path[-1]] in last:
            picks[path[-1]] = 3000
        ids += mine
        chosen += picks
    g = torch.Generator(device="cuda").manual_seed(seed)
    sees = _sees(trees)
    return {"pages": torch.randn(layers, count, 2, nkv, page, d, generator=g, device="cuda", dtype=getattr(torch, dtype)),
            "table": _ints(table), "held": _ints(held), "ids": _ints(ids), "chosen": _ints(chosen), "words": _ints(_words(sees)),
            "cu": _ints(np.cumsum([0] + brought)), "parents": _ints([p for t in trees for p in t]), "paths": paths, "most": max(brought)}


def _accept_plain(s):
    _, _, page, _, _ = POOLS[s["case"]["pool"]]
    cu, ids, chosen, parents, most = s["cu"].long(), s["ids"].long(), s["chosen"].long(), s["parents"].long(), s["most"]
    n, device = cu.shape[0] - 1, cu.device
    column = torch.arange(most, device=device)[None]
    real = column < (cu[1:] - cu[:-1])[:, None]
    at = torch.minimum(cu[:-1, None] + column, cu[1:, None] - 1)
    ids, chosen, parents = ids[at], chosen[at], torch.where(real, parents[at], -2)
    now = torch.zeros(n, dtype=torch.int64, device=device)
    going = torch.ones(n, dtype=torch.bool, device=device)
    path = torch.full((n, -(-most // 32) * 32), -1, dtype=torch.int64, device=device)
    path[:, 0] = 0
    kept = torch.ones(n, dtype=torch.int64, device=device)
    for i in range(1, most):
        match = (parents == now[:, None]) & (ids == chosen.gather(1, now[:, None]))
        first = torch.where(match, column, most).amin(1)
        going = going & (first < most)
        now = torch.where(going, first, now)
        path[:, i] = torch.where(going, now, -1)
        kept = kept + going.long()
    # Every kept token's row of the cache to where a request that had brought only these would have it.
    place = torch.arange(path.shape[1], device=device)[None].expand_as(path)
    src = s["held"].long()[:, None] + torch.where(path >= 0, path, 0)
    dst = s["held"].long()[:, None] + torch.where(path >= 0, place, 0)
    table = s["table"].long()
    of, to = table.gather(1, src // page), table.gather(1, dst // page)
    s["pages"][:, to, :, :, dst % page] = s["pages"][:, of, :, :, src % page]
    return {"path": path.int(), "kept": kept.int(), "tokens": chosen.gather(1, now[:, None])[:, 0].int(), "pages": s["pages"]}


def _accept_exact(case, seed):
    s = _accept_inputs(case, seed)
    page = POOLS[case["pool"]][2]
    held, cu, table, chosen = s["held"].tolist(), s["cu"].tolist(), s["table"].tolist(), s["chosen"].tolist()
    path = np.full((len(held), -(-s["most"] // 32) * 32), -1, dtype=np.int32)
    pages = s["pages"].clone()
    for r, nodes in enumerate(s["paths"]):
        path[r, : len(nodes)] = nodes
        for i, j in enumerate(nodes):
            if i != j:
                a, b = held[r] + j, held[r] + i
                pages[:, table[r][b // page], :, :, b % page] = pages[:, table[r][a // page], :, :, a % page]
    return {"path": path, "kept": np.asarray([len(p) for p in s["paths"]], dtype=np.int32),
            "tokens": np.asarray([chosen[cu[r] + p[-1]] for r, p in enumerate(s["paths"])], dtype=np.int32), "pages": pages}


# -- what the tools call ---------------------------------------------------------------------------------------------
def prepare(case, seed):
    s = {"tables": _tables_inputs, "attention": _attention_inputs, "logits": _logits_inputs, "accept": _accept_inputs}[case["op"]](case, seed)
    s["case"] = case
    if case["op"] == "attention":
        held, brought = _ints(s["held"], torch.int64), _ints(s["brought"], torch.int64)
        most, cu = max(s["brought"]), torch.cumsum(brought, 0) - brought
        before, node = torch.arange(max(max(s["held"]), 1), device="cuda")[None], torch.arange(most, device="cuda")[None]
        s["at_held"], s["at_nodes"] = torch.minimum(before, (held[:, None] - 1).clamp(min=0)), torch.minimum(held[:, None] + node, (held + brought)[:, None] - 1)
        s["row_of"] = (cu[:, None] + torch.minimum(node, brought[:, None] - 1))
        real = node < brought[:, None]
        s["flat_of"] = real.reshape(-1).nonzero()[:, 0]
        mine = s["positions"].long()[s["row_of"]]  # [requests, most]
        seen = [(before < held[:, None])[:, None].expand(-1, most, -1), s["sees"][s["row_of"]][..., :most] & real[:, None]]
        if case["window"]:
            seen = [seen[0] & (mine[:, :, None] - before[:, None] < case["window"]), seen[1] & (mine[:, :, None] - mine[:, None] < case["window"])]
        s["visible"] = torch.cat(seen, dim=2)
        if own:
            s["step"], s["view"] = _step(s)
    return s


def run(state):
    s, case = state, state["case"]
    if not own:
        return {"tables": _tables_plain, "attention": _attention_plain, "logits": _logits_plain, "accept": _accept_plain}[case["op"]](s)
    from mlx_omnia_b200.kernels import ops

    if case["op"] == "tables":
        lists = [ops.PageLists(pages, starts, width, stride) for pages, starts, width, stride in s["lists"]]
        made = ops.step_tables(s["held"], s["brought"], lists, case["page"], s["tokens"], parents=s["parents"],
                               most=s["most"] if case["trees"] else None)
        return {"positions": made.positions, "cu_seqlens": made.cu_seqlens, "seq_lens": made.seq_lens,
                "ancestors": None if made.tree is None else made.tree.ancestors, "groups": made.groups}
    if case["op"] == "attention":
        nq, _, d, _ = LAYOUTS[case["layout"]]
        return ops.paged_attention(s["q"], s["view"], s["step"], d ** -0.5, gate=s["rows"] if case["gated"] else None, gate_col=nq * d,
                                   sink=s["sink"], softcap=case["softcap"] or None)
    if case["op"] == "logits":
        history = ops.TokenHistory(s["tokens"], s["starts"], s["lengths"], s["prompts"]) if s["penalties"] is not None else None
        repetition, frequency, presence = s["penalties"] or (None, None, None)
        drafted = None
        if s["drafted"] is not None:
            words, ids, cu, at = s["drafted"]
            drafted = ops.DraftedRows(ops.StepTree(words), ids, cu, at)
        return ops.adjust_logits(s["logits"], history=history, repetition=repetition, frequency=frequency, presence=presence,
                                 requests=s["requests"], bias=None if s["bias"] is None else ops.LogitBias(*s["bias"]),
                                 masks=None if s["masks"] is None else ops.TokenMasks(*s["masks"]), drafted=drafted)
    _, nkv, page, d, _ = POOLS[case["pool"]]
    accepted = ops.accept_drafts(s["chosen"], s["ids"], ops.StepTree(s["words"]), s["cu"])
    ops.keep_rows(s["pages"], ((nkv, d), (nkv, d)), page, s["table"], s["held"], accepted)
    return {"path": accepted.path, "kept": accepted.kept, "tokens": accepted.tokens, "pages": s["pages"]}


def work(case):
    if case["op"] == "logits":
        rows, vocab = case["rows"], case["vocab"]
        n = rows // case["nodes"] if case["nodes"] else rows
        return {"bytes": rows * vocab * 8 + (n * case["history"] * 3 if case["penalties"] else 0) + n * case["biases"] * 4 +
                int(rows * case["masks"]) * (vocab // 8) + (rows * (4 + case["nodes"] // 8) if case["nodes"] else 0),
                "flops": rows * vocab}
    held, brought = _lengths(case)
    tokens = sum(brought)
    if case["op"] == "tables":
        entries = sum(-(-(h + b) // case["page"]) for h, b in zip(held, brought))
        width = max(-(-(h + b) // case["page"]) for h, b in zip(held, brought))
        tree = tokens * (4 + -(-case["brought"] // 32) * 4) if case["trees"] else 0
        return {"bytes": len(held) * 16 + tokens * 4 + tree + case["groups"] * (entries * 4 + len(held) * (width * 4 + 8) + tokens * 8), "flops": 0}
    if case["op"] == "accept":
        layers, nkv, _, d, dtype = POOLS[case["pool"]]
        row = layers * 2 * nkv * d * getattr(torch, dtype).itemsize
        words = -(-case["brought"] // 32)
        moved = sum(i != j for path in _paths(case)[1] for i, j in enumerate(path))
        return {"bytes": tokens * (8 + words * 4) + len(held) * (words * 128 + 16) + moved * 2 * row, "flops": 0}
    nq, nkv, d, dtype = LAYOUTS[case["layout"]]
    item = getattr(torch, dtype).itemsize
    if case["window"]:
        held = [min(h, case["window"]) for h in held]
    return {"bytes": (sum(held) + tokens) * 2 * nkv * d * item + tokens * nq * d * item * (3 if case["gated"] else 2) + sum(held) // case["page"] * 4,
            "flops": sum(4 * nq * d * b * (h + 8) for h, b in zip(held, brought))}


def exact(case, seed):
    return {"tables": _tables_exact, "attention": _attention_exact, "logits": _logits_exact, "accept": _accept_exact}[case["op"]](case, seed)
