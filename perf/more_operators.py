"""Timed cases of a step over trees of drafted tokens: the model runs every token that a draft proposes for its
sequences at once, over the paged cache, and keeps the longest path that its own choices follow.

Kinds (key "kind"):
  norm       residual addition, RMS norm and int8 quantisation of a batch's rows (add_rmsnorm_quant): what stands
             between the int4 products
  plan       depths and ancestors of the trees' nodes from their parents (tree_plan), once a step
  append     head norm and rotation by depth of the nodes, their keys and values into the pages (paged_append_tree)
  attention  the nodes over the cache, each of its tree's ancestors and itself only (paged_attention_tree)
  accept     the path that the model's choices follow, its keys and values of all layers to consecutive places
             (pages_accept); the choices are given, or the largest logits

`own` chooses between the operators and their plain form in elementary torch operations.  Head shapes, widths and
the vocabulary are those of the Qwen3-4B configuration in the listed cases; lengths reach its
max_position_embeddings of 40960.  A tree's first node is the sequence's last token, whose keys are not in the
cache yet; `nodes` counts it.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

EPS = 1e-6
ROPE_THETA = 1000000.0
LAYERS = 36
VOCAB = 151936
NODES = 256                                     # of a tree, at most
WORDS = NODES // 32


# --------------------------------------------------------------------------- the cases
_SHAPE = dict(sequences=1, nodes=8, deep=5, page=64, kv_heads=8, groups=4, dim=128)


def _attention(**k) -> dict:
    return dict(_SHAPE, **dict(dict(kind="attention", window=0, sinks=0), **k))


def _append(**k) -> dict:
    return dict(_SHAPE, **dict(dict(kind="append"), **k))


def _accept(**k) -> dict:
    return dict(_SHAPE, **dict(dict(kind="accept", layers=LAYERS, vocab=VOCAB, page=16), **k))


def listed() -> list[dict]:
    return [
        # one chat's tree of 8 nodes between two projections
        dict(name="norm_8", kind="norm", rows=8, width=2560),
        # a prompt's pass of the batched prefill's size
        dict(name="norm_2048", kind="norm", rows=2048, width=2560),
        # the tree of one chat
        dict(name="plan_1", kind="plan", sequences=1, nodes=8, deep=5),
        # the trees of a server's 64 chats
        dict(name="plan_64", kind="plan", sequences=64, nodes=60, deep=9),
        # one chat 300 tokens in: the smallest call of a step
        _append(name="append_1", context=300, page=16),
        # 32 chats with trees of 60 nodes
        _append(name="append_32", sequences=32, context=2600, nodes=60, deep=9),
        # the same chat's attention
        _attention(name="tree_1", context=300, page=16),
        # a server's step: 32 chats of 2048 to 4096 tokens with trees of up to 16 nodes
        _attention(name="tree_32", sequences=32, context=4096, nodes=16, deep=6),
        # two long documents being asked about, trees of 64 nodes
        _attention(name="tree_long_2", sequences=2, context=40960, nodes=64, deep=9),
        # 20 long chats that see 1024 tokens and the first 4
        _attention(name="tree_window_20", sequences=20, context=16000, nodes=24, deep=7, window=1024, sinks=4),
        # one chat whose choices a sampler made
        _accept(name="accept_1", context=300, choose=False),
        # a server's greedy step: the logits of 32 chats' trees
        _accept(name="accept_32", sequences=32, context=100, nodes=16, deep=6, choose=True),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


HEADS = [(8, 4, 128), (8, 4, 128), (8, 2, 128), (4, 8, 128), (2, 3, 64), (8, 5, 64), (3, 1, 32), (2, 6, 16)]


def draw(rng) -> dict:
    kind = rng.choice(["norm", "plan", "append", "attention", "attention", "attention", "choices", "greedy"])
    if kind == "norm":
        width = rng.choice([_log_int(rng, 64, 10000), 64 * _log_int(rng, 1, 150)])
        return dict(kind="norm", rows=_log_int(rng, 1, min(4096, 5000000 // width)), width=width)
    kv, g, d = rng.choice(HEADS)
    shape = dict(kv_heads=kv, groups=g, dim=d, page=rng.choice([16, 32, 64, 128]), deep=_log_int(rng, 1, 20),
                 nodes=_log_int(rng, 1, NODES))
    most = max(1, 1900 // shape["nodes"])
    if kind == "plan":
        nodes = _log_int(rng, 12, NODES)
        return dict(kind="plan", sequences=_log_int(rng, 1, 3800 // nodes), nodes=nodes, deep=_log_int(rng, 3, 20))
    if kind == "append":
        return _append(sequences=_log_int(rng, 1, min(most, 64)), context=_log_int(rng, 1, 8000), **shape)
    if kind == "attention":
        context = _log_int(rng, 1, 40960)
        # (as many tokens, positions and scores as the listed ones at most)
        nodes = shape["nodes"]
        most = max(1, min(100, 100000 // context, 5000000 // ((context + nodes) * nodes), 8000 // nodes))
        window = rng.choice([0, 0, _log_int(rng, 1, 5000)])
        return _attention(sequences=_log_int(rng, 1, most), context=context, window=window,
                          sinks=rng.choice([0, 4, rng.randint(1, 70)]) if window else 0, **shape)
    shape |= dict(page=rng.choice([16, 32]), context=_log_int(rng, 1, 120), layers=rng.randint(4, 20),
                  choose=kind == "greedy")
    if kind == "choices":
        return _accept(sequences=_log_int(rng, 1, min(most, 32)), vocab=rng.randint(1000, VOCAB), **shape)
    shape["nodes"] = min(shape["nodes"], 64)
    vocab = _log_int(rng, 300, VOCAB)
    return _accept(sequences=_log_int(rng, 1, min(48, 70000000 // (vocab * shape["nodes"]) + 1)), vocab=vocab, **shape)


# --------------------------------------------------------------------------- sizes of a case
def _trees(case: dict, seed: int = 0):
    """Each sequence's parents (-1: the root, which comes first; others before their children) and lengths of the
    caches, the trees in them; trees from half of `nodes` to all of it, at most `deep` below the root."""
    shape = case["nodes"], case["sequences"], case["deep"]
    counts = np.random.default_rng(shape).integers((case["nodes"] + 1) // 2, case["nodes"] + 1, case["sequences"])
    counts[-1] = case["nodes"]
    rng = np.random.default_rng((*shape, seed))
    trees = []
    for n in counts.tolist():
        parents, depth = [-1], [0]
        for i in range(1, n):
            open_nodes = [j for j in range(i) if depth[j] < case["deep"]]
            j = open_nodes[int(rng.integers(0, len(open_nodes), 2).max())]     # (later ones more often)
            parents.append(j)
            depth.append(depth[j] + 1)
        trees.append(parents)
    if "context" not in case:
        return trees, None
    c = case["context"]
    bases = np.random.default_rng(c).integers(c // 2, c + 1, len(trees))
    bases[-1] = c
    return trees, [int(base) + len(t) for base, t in zip(bases, trees)]


def _depths(parents: list[int]) -> list[int]:
    depth = []
    for p in parents:
        depth.append(0 if p < 0 else depth[p] + 1)
    return depth


def _paths(case: dict):
    """The path of each tree that the model's choices follow: down from the root, to a random depth.  A pass moves
    its keys and values to other places than it takes any from, so that every pass over a state does the same."""
    rng = np.random.default_rng((case["nodes"], case["context"]))
    paths = []
    for parents in _trees(case)[0]:
        path = [0]
        while rng.random() < 0.8:
            children = [i for i, p in enumerate(parents) if p == path[-1]]
            if not children:
                break
            path.append(children[int(rng.integers(0, len(children)))])
        while any(v != i and v < len(path) for i, v in enumerate(path)):
            path.pop()
        paths.append(path)
    return paths


# --------------------------------------------------------------------------- inputs
def _normal(shape, gen, dtype=torch.float32) -> torch.Tensor:
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _pool(shape, gen) -> torch.Tensor:
    """N(0,1) fp16 pages, made a layer at a time."""
    out = torch.empty(shape, dtype=torch.float16, device="cuda")
    flat = out.view(shape[0], -1)
    for i in range(shape[0]):
        flat[i] = _normal(flat[i].shape, gen, torch.float16)
    return out


def _ints(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rng = np.random.default_rng(seed)
    kind = case["kind"]
    s = {"case": case}
    if kind == "norm":
        shape = case["rows"], case["width"]
        # a residual stream with a few large channels
        channels = torch.where(torch.rand(case["width"], generator=gen, device="cuda") < 0.01, 12.0, 1.0)
        return s | {"x": 2.0 * channels * _normal(shape, gen), "delta": 0.5 * _normal(shape, gen),
                    "gamma": 0.5 + torch.rand(case["width"], generator=gen, device="cuda"),
                    "sum": torch.empty(shape, device="cuda"), "q": torch.empty(shape, dtype=torch.int8, device="cuda"),
                    "stands_for": torch.empty(shape, dtype=torch.float16, device="cuda")}
    trees, lengths = _trees(case, seed if kind == "plan" else 0)
    counts = [len(t) for t in trees]
    starts = np.concatenate([[0], np.cumsum(counts)])
    tokens = int(starts[-1])
    s |= {"starts": _ints(starts), "parents": _ints(np.concatenate(trees)), "most": max(counts),
          "status": torch.zeros(1, dtype=torch.int32, device="cuda"),
          "deepest": max(max(_depths(t)) for t in trees)}
    s["seq"] = _ints(np.repeat(np.arange(len(trees)), counts)).long()
    if kind == "plan":
        return s | {"depths": torch.empty(tokens, dtype=torch.int32, device="cuda"),
                    "ancestors": torch.empty((tokens, WORDS), dtype=torch.int32, device="cuda")}
    # the step's plan of its trees, which every layer's calls take
    bits = np.zeros((tokens, NODES), dtype=np.uint8)
    for first, parents in zip(starts, trees):
        for i, p in enumerate(parents):
            bits[first + i] = bits[first + p] if p >= 0 else 0
            bits[first + i, i] = 1
    s["ancestors"] = torch.from_numpy(np.packbits(bits, axis=1, bitorder="little").view(np.int32)).cuda()
    s["depths"] = _ints(np.concatenate([_depths(t) for t in trees]))
    page, kv, d = case["page"], case["kv_heads"], case["dim"]
    heads = kv * case["groups"]
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + 5
    order = rng.permutation(pages)              # a sequence's pages lie anywhere
    table = np.full((len(need), max(need) + 2), -1, dtype=np.int32)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = order[at:at + n]
        at += n
    layers = (case["layers"],) if kind == "accept" else ()
    s |= {"table": _ints(table), "lengths": _ints(lengths), "keys": _pool((*layers, pages, kv, page, d), gen),
          "values": _pool((*layers, pages, kv, page, d), gen)}
    if kind == "accept":
        drafted, choices = [], []
        for parents, path in zip(trees, _paths(case)):
            ids = rng.choice(case["vocab"], 2 * len(parents), replace=False)     # the draft's, and others
            choice = ids[len(parents):].copy()
            for u, v in zip(path[:-1], path[1:]):
                choice[u] = ids[v]
            drafted.append(ids[:len(parents)])
            choices.append(choice)
        s |= {"drafted": _ints(np.concatenate(drafted)), "levels": s["deepest"] + 1, "logits": None}
        s["choices"] = _ints(np.concatenate(choices))
        if case["choose"]:
            s["logits"] = _normal((tokens, case["vocab"]), gen)
            s["logits"][torch.arange(tokens, device="cuda"), s["choices"].long()] += 9.0
            s["choices"] = None
        return s
    s["out"] = torch.empty((tokens, heads, d), device="cuda")
    if kind == "attention":
        s["query"] = _normal((tokens, heads, d), gen)
        return s
    s["qkv"] = 2.0 * _normal((tokens, (heads + 2 * kv) * d), gen)
    s["q_norm"], s["k_norm"] = (0.9 + 0.2 * torch.rand(d, generator=gen, device="cuda") for _ in range(2))
    inverse = ROPE_THETA ** (-np.arange(0, d, 2) / d)
    angles = np.arange(max(lengths) + 1)[:, None] * inverse[None, :]
    s["cos"], s["sin"] = (torch.from_numpy(f(angles).astype(np.float32)).cuda() for f in (np.cos, np.sin))
    return s


# --------------------------------------------------------------------------- one pass
def run(s: dict):
    case = s["case"]
    kind = case["kind"]
    if kind == "norm":
        if own:
            from harsh4b_amd.lightspark import add_rmsnorm_quant
            q, scale = add_rmsnorm_quant(s["x"], s["gamma"], EPS, delta=s["delta"], out=s["sum"], q=s["q"])
        else:
            q, scale = _plain_norm(s)
        # the int8 values times their scales: 127 steps, to which 16 bits do
        return s["sum"], torch.mul(q, scale[:, None], out=s["stands_for"])
    if kind == "plan":
        if own:
            from harsh4b_amd.tree import tree_plan
            tree = tree_plan(s["parents"], s["starts"], s["status"], depths=s["depths"], ancestors=s["ancestors"])
            return tree.depths, tree.ancestors
        return _plain_plan(s)
    if kind == "append":
        if own:
            from harsh4b_amd.tree import DraftTree, paged_append_tree
            tree = DraftTree(s["parents"], s["starts"], s["depths"], s["ancestors"])
            query = paged_append_tree(s["qkv"], s["q_norm"], s["k_norm"], s["cos"], s["sin"], EPS, s["keys"], s["values"],
                                      s["table"], s["lengths"], s["status"], tree, out=s["out"])
        else:
            query = _plain_append(s)
        return query, s["keys"], s["values"]
    if kind == "attention":
        if own:
            from harsh4b_amd.tree import DraftTree, paged_attention_tree
            tree = DraftTree(s["parents"], s["starts"], s["depths"], s["ancestors"])
            return paged_attention_tree(s["query"], s["keys"], s["values"], s["table"], s["lengths"], tree,
                                        window=case["window"], sinks=case["sinks"], out=s["out"])
        return _plain_attention(s)
    if own:
        from harsh4b_amd.tree import DraftTree, pages_accept
        tree = DraftTree(s["parents"], s["starts"], s["depths"], s["ancestors"])
        kept, path, after = pages_accept(s["keys"], s["values"], s["table"], s["lengths"], s["status"], tree,
                                         s["drafted"], choices=s["choices"], logits=s["logits"], levels=s["levels"])
    else:
        kept, path, after = _plain_accept(s)
    return s["keys"], s["values"], kept, path, after


# --------------------------------------------------------------------------- plain forms
def _plain_norm(s: dict):
    # (64 bits: many values lie next to a border of the int8 steps)
    x = torch.add(s["x"], s["delta"], out=s["sum"]).double()
    y = x / torch.sqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * s["gamma"]
    top = y.abs().amax(dim=-1).clamp_min(1e-5)
    return (y * (127.0 / top)[:, None]).round().clamp(-127.0, 127.0), top / 127.0


def _places(s: dict):
    """Of each node: its place in its tree, its sequence's first row and base (positions before the tree)."""
    starts = s["starts"].long()
    first = starts[:-1][s["seq"]]
    place = torch.arange(s["parents"].shape[0], device="cuda") - first
    base = s["lengths"].long() - (starts[1:] - starts[:-1]) if "lengths" in s else None
    return place, first, base


def _bits(s: dict) -> torch.Tensor:
    """Truth values [tokens, NODES]: the node's ancestors and itself."""
    words = s["ancestors"].long() & 0xFFFFFFFF
    return (words[:, :, None] >> torch.arange(32, device="cuda") & 1).bool().flatten(1)


def _plain_plan(s: dict):
    place, first, _ = _places(s)
    parents = s["parents"].long()
    depth = torch.zeros_like(parents)
    seen = torch.zeros((parents.shape[0], NODES), dtype=torch.bool, device="cuda")
    node = place
    row = torch.arange(parents.shape[0], device="cuda")
    for _ in range(s["deepest"] + 1):
        seen[row, node] = True
        up = parents[first + node]
        depth += up >= 0
        node = torch.where(up >= 0, up, node)
    words = (seen.view(-1, WORDS, 32).long() << torch.arange(32, device="cuda")).sum(dim=-1)
    return depth.int(), torch.where(words < 2 ** 31, words, words - 2 ** 32).int()


def _plain_append(s: dict) -> torch.Tensor:
    case = s["case"]
    kv, heads, d, page = case["kv_heads"], case["kv_heads"] * case["groups"], case["dim"], case["page"]
    place, _, base = _places(s)
    slot = base[s["seq"]] + place
    angle = base[s["seq"]] + s["depths"].long()
    x = s["qkv"].view(-1, heads + 2 * kv, d)
    cos, sin = s["cos"][angle][:, None, :], s["sin"][angle][:, None, :]

    def turned(a, weight):
        a = a / torch.sqrt((a * a).mean(dim=-1, keepdim=True) + EPS) * weight
        lo, hi = a[..., :d // 2], a[..., d // 2:]
        return torch.cat((lo * cos - hi * sin, hi * cos + lo * sin), dim=-1)

    where = s["table"][s["seq"], slot // page].long(), slice(None), slot % page
    s["keys"][where] = turned(x[:, heads:heads + kv], s["k_norm"]).half()
    s["values"][where] = x[:, heads + kv:].half()
    return turned(x[:, :heads], s["q_norm"])


def _plain_attention(s: dict) -> torch.Tensor:
    case, query = s["case"], s["query"]
    kv, g, d = case["kv_heads"], case["groups"], case["dim"]
    place, _, base = _places(s)
    rows, most, tokens = s["table"].shape[0], s["most"], query.shape[0]
    span = s["table"].shape[1] * case["page"]

    def history(pool):      # [rows, kv, positions, d]
        return pool[s["table"].clamp_min(0).long()].permute(0, 2, 1, 3, 4).reshape(rows, kv, span, d).float()

    token = (s["starts"].long()[:-1, None] + torch.arange(most, device="cuda")).clamp_max(tokens - 1)
    q = query[token].view(rows, most, kv, g, d).permute(0, 2, 3, 1, 4).reshape(rows, kv, g * most, d)
    scores = (q @ history(s["keys"]).transpose(-1, -2).contiguous()).view(rows, kv, g, most, span) / math.sqrt(d)
    # what a node sees of its tree, and the position that each place of the cache stands for
    j = torch.arange(span, device="cuda")[None, :]
    node = j - base[:, None]                                                              # [rows, positions]
    length = s["lengths"].long()[:, None]
    drafted = (node >= 0) & (j < length)
    depth = s["depths"].long()[token]                                                     # [rows, most]
    position = torch.where(drafted, base[:, None] + depth.gather(1, node.clamp(0, most - 1)), j)
    bits = _bits(s)[token].gather(2, node.clamp(0, NODES - 1)[:, None, :].expand(rows, most, span))
    seen = (node < 0)[:, None, :] | (drafted[:, None, :] & bits)
    if case["window"]:
        at = (base[:, None] + depth)[..., None]
        seen &= (position[:, None, :] > at - case["window"]) | (position < case["sinks"])[:, None, :]
    seen = seen[:, None, None]
    scores = scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(dim=-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    p = scores.sub_(top).exp_()
    o = p.view(rows, kv, g * most, span) @ history(s["values"])
    o = o.view(rows, kv, g, most, d) / p.sum(dim=-1, keepdim=True)
    return o.permute(0, 3, 1, 2, 4)[s["seq"], place].reshape(query.shape)


def _plain_accept(s: dict):
    place, _, base = _places(s)
    starts, parents = s["starts"].long(), s["parents"].long()
    rows, tokens, page = s["table"].shape[0], parents.shape[0], s["case"]["page"]
    choices = s["choices"].long() if s["logits"] is None else s["logits"].argmax(dim=-1)
    node, count = torch.zeros(rows, dtype=torch.long, device="cuda"), torch.ones(rows, dtype=torch.long, device="cuda")
    path = torch.full((tokens + 1,), -1, dtype=torch.long, device="cuda")       # (the last entry takes what is none)
    path[starts[:-1]] = 0
    for i in range(1, s["levels"]):
        choice = choices[starts[:-1] + node]
        fits = (parents == node[s["seq"]]) & (s["drafted"].long() == choice[s["seq"]])
        first = torch.full((rows,), NODES, dtype=torch.long, device="cuda")
        first.scatter_reduce_(0, s["seq"], torch.where(fits, place, NODES), "amin")
        go = (first < NODES) & (count == i)
        node = torch.where(go, first, node)
        path[torch.where(go, starts[:-1] + i, tokens)] = node
        count += go
    path = path[:tokens]
    # keys and values of the path's nodes to the places after the base
    moved = (path >= 0) & (path != place)
    source = torch.where(moved, base[s["seq"]] + path, 0)
    target = torch.where(moved, base[s["seq"]] + place, 0)
    for pool in (s["keys"], s["values"]):
        rows_of = pool[:, s["table"][s["seq"], source // page].long(), :, source % page]
        pool[:, s["table"][s["seq"], target // page].long(), :, target % page] = rows_of
        # (what is not moved: position 0 onto itself)
    return (base + count).int(), path.int(), choices[starts[:-1] + node].int()


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "norm":
        size = case["rows"] * case["width"]
        return {"bytes": 13 * size + 4 * case["width"] + 4 * case["rows"], "flops": 8 * size}
    trees, lengths = _trees(case)
    tokens = sum(len(t) for t in trees)
    if kind == "plan":
        return {"bytes": tokens * (4 + 4 + 4 * WORDS) + 4 * len(trees), "flops": tokens}
    kv, d = case["kv_heads"], case["dim"]
    heads = kv * case["groups"]
    if kind == "append":
        return {"bytes": tokens * (4 * (heads + 2 * kv) * d + 4 * heads * d + 4 * kv * d + 4 * d + 12),
                "flops": tokens * (heads + kv) * d * 8}
    if kind == "attention":
        pairs = read = 0
        for parents, length in zip(trees, lengths):
            base, depth = length - len(parents), _depths(parents)
            window, sinks = case["window"] or length + 1, case["sinks"]
            lowest = base
            for at in depth:
                low = max(0, base + at - window + 1)
                lowest = min(lowest, low)
                pairs += max(0, base - low) + min(low, sinks, base) + min(at + 1, window)
            read += base - lowest + min(lowest, sinks) + len(parents)
        return {"bytes": read * 4 * kv * d + tokens * (8 * heads * d + 4 * WORDS), "flops": 4 * d * heads * pairs}
    paths = _paths(case)
    moved = sum(v != i for path in paths for i, v in enumerate(path))
    rows = sum(len(path) for path in paths) if case["choose"] else 0
    return {"bytes": 4 * rows * case["vocab"] + 2 * moved * case["layers"] * 4 * kv * d + tokens * 16,
            "flops": tokens + rows * case["vocab"]}


# --------------------------------------------------------------------------- 64-bit results
def exact(case: dict, seed: int):
    kind = case["kind"]
    if kind == "plan":
        return None             # whole numbers: no rounding to measure
    s = prepare(case, seed)
    if kind == "norm":
        total = s["x"].double() + s["delta"].double()
        y = s["gamma"].double() * total * torch.rsqrt(total.pow(2).sum(-1, keepdim=True) / case["width"] + EPS)
        scale = y.abs().amax(-1, keepdim=True).clamp_min(1e-5) / 127
        return total, torch.round(y / scale) * scale
    return {"attention": _exact_attention, "append": _exact_append, "accept": _exact_accept}[kind](case, s)


def _exact_attention(case: dict, s: dict) -> torch.Tensor:
    trees, lengths = _trees(case)
    kv, g, d, page = case["kv_heads"], case["groups"], case["dim"], case["page"]
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device="cuda")
    token = 0
    for b, (parents, length) in enumerate(zip(trees, lengths)):
        n = len(parents)
        base, depth = length - n, _depths(parents)
        sees = np.zeros((n, length), dtype=bool)
        position = np.concatenate([np.arange(base), base + np.array(depth)])
        sees[:, :base] = True
        for i, p in enumerate(parents):
            if p >= 0:
                sees[i, base:] = sees[p, base:]
            sees[i, base + i] = True
        if case["window"]:
            far = position[base:, None] - position[None, :]
            sees &= (far < case["window"]) | (position < case["sinks"])[None, :]
        hidden = torch.from_numpy(~sees).cuda()
        ids = s["table"][b][:-(-length // page)].long()
        for h in range(kv):
            keys, values = (s[name][ids, h].reshape(-1, d)[:length].double() for name in ("keys", "values"))
            for head in range(h * g, (h + 1) * g):
                score = torch.mm(s["query"][token:token + n, head].double(), keys.t().contiguous()) * d ** -0.5
                out[token:token + n, head] = torch.mm(torch.softmax(score.masked_fill(hidden, -math.inf), dim=-1), values)
        token += n
    return out


def _exact_append(case: dict, s: dict):
    trees, lengths = _trees(case)
    kv, heads, d, page = case["kv_heads"], case["kv_heads"] * case["groups"], case["dim"], case["page"]
    x = s["qkv"].double().view(-1, heads + 2 * kv, d)
    keys, values = s["keys"].double(), s["values"].double()
    query = torch.empty((x.shape[0], heads, d), dtype=torch.float64, device="cuda")
    token = 0
    for b, (parents, length) in enumerate(zip(trees, lengths)):
        n = len(parents)
        angle = torch.tensor(_depths(parents), device="cuda") + length - n
        turn = torch.complex(s["cos"][angle].double(), s["sin"][angle].double())[:, None, :]
        part = x[token:token + n]

        def rotated(a, weight):
            a = a * torch.rsqrt(a.pow(2).sum(-1, keepdim=True) / d + EPS) * weight.double()
            z = torch.complex(a[..., :d // 2].contiguous(), a[..., d // 2:].contiguous()) * turn
            return torch.cat((z.real, z.imag), dim=-1)

        query[token:token + n] = rotated(part[:, :heads], s["q_norm"])
        at = torch.arange(length - n, length, device="cuda")
        ids = s["table"][b][at // page].long()
        keys[ids, :, at % page] = rotated(part[:, heads:heads + kv], s["k_norm"])
        values[ids, :, at % page] = part[:, heads + kv:]
        token += n
    return query, keys, values


def _exact_accept(case: dict, s: dict):
    """The rows of the paths that the choices were made for, in their places; whole numbers have no rounding."""
    trees, lengths = _trees(case)
    page, table = case["page"], s["table"].cpu().numpy()
    source, target = [], []
    for b, (parents, length, path) in enumerate(zip(trees, lengths, _paths(case))):
        base = length - len(parents)
        for i, v in enumerate(path):
            for place, node in ((source, v), (target, i)):
                place.append((int(table[b, (base + node) // page]), (base + node) % page))
    (a, i), (c, j) = (torch.tensor(x, device="cuda").t() for x in (source, target))
    pools = s["keys"].double(), s["values"].double()
    for pool in pools:
        pool[:, c, :, j] = pool[:, a, :, i]
    return (*pools, None, None, None)
