"""What decoding several requests over one shared prompt asks of the cache and of attention, as cases that can be
timed and compared: attention of single tokens whose requests share their first positions, the copies of pages that
a request's fork and a pool's resizing make, and the copies of per-request state that a fork makes.

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
# parameters and of its sliding-window family, and of two of the tests' small models (one in 32 bits).
LAYOUTS = {"16/8x128": (16, 8, 128, "bfloat16"), "32/8x128": (32, 8, 128, "bfloat16"), "16/4x128": (16, 4, 128, "bfloat16"),
           "6/2x64": (6, 2, 64, "bfloat16"), "8/1x24 f32": (8, 1, 24, "float32"), "16/8x128 f32": (16, 8, 128, "float32")}

# What a page holds in every layer that keeps pages: layers, key/value heads, tokens a page, head size, element type.
POOLS = {"28 layers": (28, 8, 16, 128, "bfloat16"), "36 layers": (36, 8, 16, 128, "bfloat16"),
         "3 layers f32": (3, 1, 8, 24, "float32")}

# The per-request state of recurrent layers: a list of (layers, elements a request): a linear attention's float32 states
# of 16 heads of 128 x 128; a state-space mixer's 64 heads of 64 x 128 with its convolution's last inputs; a gated
# recurrence's channels with its convolution's (odd in 16-byte units).
STATES = {"linear attention": ((4, 16 * 128 * 128),), "state space": ((4, 64 * 64 * 128), (4, 3 * 4352)),
          "channels": ((6, 2051), (6, 3 * 2051))}


def listed():
    attention = {"op": "attention", "page": 16, "groups": 1, "gated": True, "sink": False, "softcap": 0.0}
    return [
        # Two answers to one short question, the first tokens of them: what a call costs at the least.
        attention | {"name": "2 answers, 200 shared", "layout": "16/8x128", "members": 2, "prefix": 200, "suffix": 8},
        # Eight samples of one prompt at the benchmark's context.
        attention | {"name": "8 samples, 4096 shared", "layout": "16/8x128", "members": 8, "prefix": 4096, "suffix": 256},
        # Sixty-four samples of a middling prompt, well into their answers: what they do not share outweighs what they share.
        attention | {"name": "64 samples, 2051 shared", "layout": "16/8x128", "members": 64, "prefix": 2051, "suffix": 700},
        # Sixteen questions about one long document.
        attention | {"name": "16 questions, 32768 shared", "layout": "32/8x128", "members": 16, "prefix": 32768, "suffix": 500},
        # The largest: sixty-four questions about a document as long as a long-context model takes.
        attention | {"name": "64 questions, 65536 shared", "layout": "32/8x128", "members": 64, "prefix": 65536, "suffix": 1024},
        # Several prompts sampled at once by a model with sinks and capped scores, three query heads a key/value head, odd lengths.
        attention | {"name": "3 groups, sink and cap", "layout": "6/2x64", "members": 21, "prefix": 1537, "suffix": 333, "groups": 3,
                     "gated": False, "sink": True, "softcap": 30.0},
        # The 32-bit path, at the tests' odd head size.
        attention | {"name": "32-bit samples", "layout": "8/1x24 f32", "members": 12, "prefix": 1001, "suffix": 65, "page": 8},
        # A prompt of 4,107 tokens is forked seven ways: the eleven rows of its last page for each.
        {"op": "pages", "name": "fork seven ways", "pool": "28 layers", "pages": 600, "moves": 7, "rows": 11, "fork": True, "other": False},
        # Sixty-three ways, in the model of 8 billion parameters: the rows of the last page, 7.
        {"op": "pages", "name": "fork sixty-three ways", "pool": "36 layers", "pages": 400, "moves": 63, "rows": 7, "fork": True, "other": False},
        # A pool gives memory back: the pages that are held move into the smaller one.
        {"op": "pages", "name": "resize, 300 pages held", "pool": "36 layers", "pages": 400, "moves": 300, "rows": 16, "fork": False, "other": True},
        # Eight samples start from one prompt's recurrent state.
        {"op": "slots", "name": "state to 7 samples", "state": "linear attention", "slots": 16, "moves": 7, "fork": True},
        # Pairs of one slot to another for as many requests (a beam's survivors), large states and small ones.
        {"op": "slots", "name": "state of 24 beams", "state": "state space", "slots": 64, "moves": 24, "fork": False},
    ]


def _spread(rng, low, high):
    """A whole number between `low` and `high`, even over the logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.random()
    if kind < 0.2:
        pool = rng.choice(sorted(POOLS))
        pages = _spread(rng, 20, 400)
        fork = rng.random() < 0.6
        moves = _spread(rng, 1, min(63, pages // 2)) if fork else _spread(rng, 8, pages * 3 // 4)
        return {"op": "pages", "pool": pool, "pages": pages, "moves": moves, "rows": rng.randint(1, POOLS[pool][2]), "fork": fork,
                "other": not fork}
    if kind < 0.3:
        slots = _spread(rng, 4, 64)
        return {"op": "slots", "state": rng.choice(sorted(STATES)), "slots": slots, "moves": _spread(rng, 1, slots // 2),
                "fork": rng.random() < 0.5}
    layout = rng.choice(["16/8x128", "16/8x128", "32/8x128", "32/8x128", "16/4x128", "6/2x64", "8/1x24 f32", "16/8x128 f32"])
    small = layout.endswith("f32")
    top = work(listed()[4])
    case = {"op": "attention", "layout": layout, "page": rng.choice([8, 16, 32] if small else [16, 16, 32, 48]),
            "groups": rng.choice([1, 1, 2, 3]), "gated": rng.random() < 0.5, "sink": rng.random() < 0.25,
            "softcap": 30.0 if rng.random() < 0.15 else 0.0, "members": _spread(rng, 2, 16 if small else 96),
            "prefix": _spread(rng, 16, 3000 if small else 65536), "suffix": _spread(rng, 1, 300 if small else 1500)}
    while any(work(case)[k] > top[k] for k in top):
        case["prefix" if case["prefix"] > case["suffix"] else "members"] //= 2
    case["members"] = max(case["members"], 2)
    return case


# -- attention -----------------------------------------------------------------------------------------------------
def _lengths(case):
    """(positions each group shares, the positions of its own that each request holds, its current token's among them)."""
    rng = random.Random(f"{case['members']} {case['prefix']} {case['suffix']} {case['groups']}")
    prefixes = [max(1, case["prefix"] - g * (case["prefix"] // 3)) for g in range(case["groups"])]
    suffixes = [rng.randint(1 + case["suffix"] // 4, case["suffix"]) if case["suffix"] > 1 else 1
                for _ in range(case["groups"] * case["members"])]
    suffixes[rng.randrange(len(suffixes))] = case["suffix"]
    return prefixes, suffixes


def _tables(case, generator):
    """Block tables of requests that share their first pages: whole pages of the shared positions are the group's, the page
    that these end in is each request's own, as a fork leaves it. -> (tables on the host, pages in all)"""
    prefixes, suffixes = _lengths(case)
    page, members = case["page"], case["members"]
    lengths = [prefixes[r // members] + s for r, s in enumerate(suffixes)]
    table = np.full((len(lengths), max(-(-n // page) for n in lengths)), -1, dtype=np.int64)
    taken = 0
    for g, p in enumerate(prefixes):
        table[g * members: (g + 1) * members, : p // page] = np.arange(taken, taken + p // page)
        taken += p // page
    for r, n in enumerate(lengths):
        at, end = prefixes[r // members] // page, -(-n // page)
        table[r, at: end] = np.arange(taken, taken + end - at)
        taken += end - at
    order = torch.randperm(taken, generator=generator).numpy()
    return np.where(table >= 0, order[table], -1), taken


def _attention_inputs(case, seed):
    nq, nkv, d, dtype = LAYOUTS[case["layout"]]
    dtype = getattr(torch, dtype)
    prefixes, suffixes = _lengths(case)
    table, pages = _tables(case, torch.Generator().manual_seed(seed))
    g = torch.Generator(device="cuda").manual_seed(seed)
    requests, page, members = len(suffixes), case["page"], case["members"]
    cache = torch.randn(pages, 2, nkv, page, d, generator=g, device="cuda", dtype=dtype)
    for i, p in enumerate(prefixes):  # the rows that a fork copies into each request's own last page of the shared positions
        if p % page:
            own_pages = torch.from_numpy(table[i * members: (i + 1) * members, p // page]).cuda()
            cache[own_pages[1:], :, :, : p % page] = cache[own_pages[:1], :, :, : p % page]
    # Projected rows as a layer has them: the queries (normed, here beside them) and the gate's columns.
    q = torch.randn(requests, nq, d, generator=g, device="cuda", dtype=dtype)
    rows = torch.randn(requests, 2 * nq * d, generator=g, device="cuda", dtype=dtype)
    sink = torch.randn(nq, generator=g, device="cuda") if case["sink"] else None
    return {"q": q, "rows": rows, "cache": cache, "table": torch.from_numpy(table).to("cuda", torch.int32), "sink": sink,
            "lengths": [prefixes[r // members] + s for r, s in enumerate(suffixes)], "prefixes": prefixes}


def _attention_plain(s):
    case, q, cache = s["case"], s["q"], s["cache"]
    nq, nkv, d, _ = LAYOUTS[case["layout"]]
    groups, members, page = case["groups"], case["members"], case["page"]
    table, group = s["table"].long(), nq // nkv
    # Keys and values of the shared positions, a group's once [groups, positions, nkv, d]; of each request's own [requests, positions, nkv, d].
    shared, shared_seen = s["shared_at"], s["shared_seen"]
    mine, mine_seen = s["mine_at"], s["mine_seen"]
    first = table[::members].gather(1, shared // page)
    ks, vs = (cache[first, w, :, shared % page].float() for w in (0, 1))
    rest = table.gather(1, mine // page)
    km, vm = (cache[rest, w, :, mine % page].float() for w in (0, 1))
    x = q.float() * d ** -0.5
    zs = torch.einsum("gmkxd,gpkd->gmkxp", x.view(groups, members, nkv, group, d), ks).reshape(-1, nkv, group, shared.shape[1])
    zm = torch.einsum("rkxd,rpkd->rkxp", x.view(-1, nkv, group, d), km)
    z = torch.cat([zs, zm], dim=3)
    if case["softcap"]:
        z = case["softcap"] * torch.tanh(z / case["softcap"])
    seen = torch.cat([shared_seen.repeat_interleave(members, 0), mine_seen], dim=1)
    z = torch.where(seen[:, None, None, :], z, -torch.inf)
    top = z.amax(3, keepdim=True)
    p = torch.exp(z - top)
    total = p.sum(3, keepdim=True)
    if case["sink"]:
        total = total + torch.exp(s["sink"].view(1, nkv, group, 1) - top)
    p = p / total
    ps, pm = p[..., : shared.shape[1]], p[..., shared.shape[1]:]
    out = torch.einsum("gmkxp,gpkd->gmkxd", ps.reshape(groups, members, nkv, group, -1), vs).reshape(-1, nq * d)
    out = out + torch.einsum("rkxp,rpkd->rkxd", pm, vm).reshape(-1, nq * d)
    if case["gated"]:
        out = out * torch.sigmoid(s["rows"][:, nq * d:].float())
    return out.to(q.dtype)


def _attention_exact(case, seed):
    s = _attention_inputs(case, seed)
    nq, nkv, d, _ = LAYOUTS[case["layout"]]
    answers = []
    for r, n in enumerate(s["lengths"]):
        at = torch.arange(n, device="cuda")
        held = s["cache"][s["table"][r].long()[at // case["page"]], :, :, at % case["page"]]  # [n, 2, nkv, d]
        z = held[:, 0].double().permute(1, 0, 2) @ s["q"][r].double().view(nkv, nq // nkv, d).transpose(1, 2) / math.sqrt(d)
        if case["softcap"]:
            z = case["softcap"] * torch.tanh(z / case["softcap"])
        if case["sink"]:
            z = torch.cat([z, s["sink"].double().view(nkv, 1, -1)], dim=1)
        weight = torch.softmax(z, dim=1)[:, :n]
        answers.append((weight.transpose(1, 2) @ held[:, 1].double().permute(1, 0, 2)).reshape(-1))
    out = torch.stack(answers)
    return out / (1 + torch.exp(-s["rows"][:, nq * d:].double())) if case["gated"] else out


# -- copies --------------------------------------------------------------------------------------------------------
def _moves(case, most, seed):
    """Pairs (from, to) of different numbers below `most`: one place's contents to many others, or each its own."""
    order = torch.randperm(most, generator=torch.Generator().manual_seed(seed)).tolist()
    if case.get("other"):  # into another pool: the pages that are held, to its front
        return [(src, dst) for dst, src in enumerate(order[: case["moves"]])]
    if case["fork"]:
        return [(order[0], dst) for dst in order[1: case["moves"] + 1]]
    return list(zip(order[: case["moves"]], order[case["moves"]: 2 * case["moves"]]))


def _pages_inputs(case, seed):
    layers, nkv, page, d, dtype = POOLS[case["pool"]]
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = torch.randn(layers, case["pages"], 2, nkv, page, d, generator=g, device="cuda", dtype=getattr(torch, dtype))
    to = torch.zeros(layers, case["moves"], 2, nkv, page, d, device="cuda", dtype=pages.dtype) if case["other"] else pages
    return {"pages": pages, "to": to, "moves": [(a, b, case["rows"]) for a, b in _moves(case, case["pages"], seed)]}


def _slots_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = [torch.randn(case["slots"] + 1, size, generator=g, device="cuda") for layers, size in STATES[case["state"]]
             for _ in range(layers)]
    return {"state": state, "moves": _moves(case, case["slots"], seed)}


# -- what the tools call -------------------------------------------------------------------------------------------
def prepare(case, seed):
    if case["op"] == "pages":
        s = _pages_inputs(case, seed)
        s["index"] = [torch.tensor(column, device="cuda") for column in zip(*s["moves"])]
    elif case["op"] == "slots":
        s = _slots_inputs(case, seed)
        s["index"] = [torch.tensor(column, device="cuda") for column in zip(*s["moves"])]
    else:
        s = _attention_inputs(case, seed)
        prefixes, suffixes = _lengths(case)
        shared = torch.arange(max(prefixes), device="cuda")[None]
        ends = torch.tensor(prefixes, device="cuda")[:, None]
        s["shared_seen"], s["shared_at"] = shared < ends, torch.minimum(shared, ends - 1)
        starts = ends.repeat_interleave(case["members"], 0)
        lengths = torch.tensor(s["lengths"], device="cuda")[:, None]
        mine = starts + torch.arange(max(suffixes), device="cuda")[None]
        s["mine_seen"], s["mine_at"] = mine < lengths, torch.minimum(mine, lengths - 1)
        if own:
            s["step"], s["view"] = _step(case, s)
    s["case"] = case
    return s


def _step(case, s):
    """The step and the cache view that a model's layers are handed."""
    from mlx_omnia_b200.parts.base import KVSpec, KVView, StepContext

    nq, nkv, d, _ = LAYOUTS[case["layout"]]
    lengths, members = s["lengths"], case["members"]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    n = len(lengths)
    step = StepContext(
        num_tokens=n, num_seqs=n, token_ids=ints([0] * n), positions=ints([x - 1 for x in lengths]), cu_seqlens=ints(list(range(n + 1))),
        seq_lens=ints(lengths), state_slots=ints([0] * n), fresh=ints([0] * n), logit_rows=ints([]), q_lens=[1] * n,
        seq_lens_host=lengths, max_q_len=1, max_seq_len=max(lengths), decode_only=True, groups={},
        shared=tuple((p, tuple(range(g * members, (g + 1) * members))) for g, p in enumerate(s["prefixes"])))
    spec = KVSpec.keys_and_values(nkv, d)
    return step, KVView(s["cache"], s["table"], torch.zeros(n, dtype=torch.int64, device="cuda"), case["page"], None, spec=spec)


def run(state):
    s, case = state, state["case"]
    if own:
        from mlx_omnia_b200.kernels import ops

        if case["op"] == "pages":
            _, nkv, page, d, _ = POOLS[case["pool"]]
            return ops.copy_pages(s["pages"], ((nkv, d), (nkv, d)), page, s["moves"], to=s["to"])
        if case["op"] == "slots":
            ops.copy_slots(s["state"], s["moves"])
            return s["state"]
        nq, nkv, d, _ = LAYOUTS[case["layout"]]
        return ops.paged_attention(s["q"], s["view"], s["step"], d ** -0.5, gate=s["rows"] if case["gated"] else None, gate_col=nq * d,
                                   sink=s["sink"], softcap=case["softcap"] or None)
    if case["op"] == "attention":
        return _attention_plain(s)
    src, dst = s["index"][:2]
    if case["op"] == "slots":
        return [t.index_copy_(0, dst, t[src]) for t in s["state"]]
    s["to"][:, dst, :, :, : case["rows"]] = s["pages"][:, src, :, :, : case["rows"]]
    return s["to"]


def work(case):
    if case["op"] == "pages":
        layers, nkv, _, d, dtype = POOLS[case["pool"]]
        piece = layers * 2 * nkv * case["rows"] * d * getattr(torch, dtype).itemsize
        return {"bytes": piece * (case["moves"] + (1 if case["fork"] else case["moves"])), "flops": 0}
    if case["op"] == "slots":
        piece = sum(layers * size * 4 for layers, size in STATES[case["state"]])
        return {"bytes": piece * (case["moves"] + (1 if case["fork"] else case["moves"])), "flops": 0}
    nq, nkv, d, dtype = LAYOUTS[case["layout"]]
    prefixes, suffixes = _lengths(case)
    item, n = getattr(torch, dtype).itemsize, len(suffixes)
    seen = sum(prefixes) * case["members"] + sum(suffixes)
    held = sum(prefixes) + sum(suffixes)
    return {"bytes": held * 2 * nkv * d * item + n * nq * d * item * (3 if case["gated"] else 2) + held // case["page"] * 4,
            "flops": 4 * nq * d * seen}


def exact(case, seed):
    if case["op"] == "attention":
        return _attention_exact(case, seed)
    if case["op"] == "pages":
        s = _pages_inputs(case, seed)
        to = s["to"].double() if s["to"].numel() < 3e8 else s["to"].clone()
        for src, dst, rows in s["moves"]:
            to[:, dst, :, :, :rows] = s["pages"][:, src, :, :, :rows]
        return to
    s = _slots_inputs(case, seed)
    for t in s["state"]:
        for src, dst in s["moves"]:
            t[dst] = t[src]
    return s["state"]
