"""Timed cases of the paged KV cache's operators: the fp16 cache of many sequences in pages that they may
share, and what writes, reads and manages it.

Kinds (key "kind"):
  attention  grouped-query attention of a batch's new tokens over the pages (paged_attention): one token a
             sequence, a prompt's chunk, both together; with a sliding window and first tokens that stay visible
  append     head norm and rotation of a batch's new tokens, their keys and values into the pages (paged_append)
  fork       beams: forks of prompts released, made again and grown by a few tokens (pages_resize, pages_fork):
             the growth copies the partly filled page that the forks share
  compact    a cache with holes made dense (pages_compact)

`own` chooses between the operators and their plain form in elementary torch operations.  Head shapes are those
of the Qwen3-4B configuration in the listed cases; lengths reach its max_position_embeddings of 40960.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

EPS = 1e-6
ROPE_THETA = 1000000.0
LAYERS = 36


# --------------------------------------------------------------------------- the cases
def _attention(**k) -> dict:
    return dict(dict(kind="attention", sequences=1, chunks=0, new=1, page=64, window=0, sinks=0, kv_heads=8, groups=4,
                     dim=128), **k)


def _append(**k) -> dict:
    return dict(dict(kind="append", sequences=1, chunks=0, new=1, page=64, kv_heads=8, groups=4, dim=128), **k)


def listed() -> list[dict]:
    return [
        # one chat, 300 tokens in: the smallest call of a reply
        _attention(name="one_300", context=300, page=16),
        # a server's step: 32 chats of 2048 to 4096 tokens
        _attention(name="chats_32", sequences=32, context=4096),
        # three long documents being asked about
        _attention(name="long_3", sequences=3, context=40960),
        # a question's 501 tokens after 7000 of history
        _attention(name="question_501", chunks=1, new=501, context=7501, page=16),
        # a document's chunk of the batched prefill's size, 14336 tokens in
        _attention(name="chunk_2048", chunks=1, new=2048, context=16384),
        # a server's step that takes a prompt's chunk along with 24 replies
        _attention(name="mixed_25", sequences=25, chunks=1, new=250, context=3000, page=32),
        # replies of 16 long chats that see 1024 tokens and the first 4
        _attention(name="window_16", sequences=16, context=16000, window=1024, sinks=4),
        # a chunk of a long document under a window of odd length
        _attention(name="window_chunk_1500", chunks=1, new=1500, context=9000, window=1001, sinks=5, page=32),
        # one layer's rows of 32 replies
        _append(name="append_32", sequences=32, context=4096),
        # one layer's rows of a prompt
        _append(name="append_2000", chunks=1, new=2000, context=2600, page=16),
        # 8 prompts of about 700 tokens, 4 beams each, 5 tokens on
        dict(name="beams_32", kind="fork", prompts=8, beams=4, context=700, grow=5, page=16, layers=LAYERS, kv_heads=8,
             dim=128),
        # a cache of 384 pages, two of five in use
        dict(name="compact_384", kind="compact", pages=384, used=0.4, sequences=12, page=16, layers=LAYERS, kv_heads=8,
             dim=128),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


HEADS = [(8, 4, 128), (8, 4, 128), (8, 2, 128), (4, 8, 128), (2, 3, 64), (8, 5, 64), (3, 1, 32), (2, 6, 16)]


def draw(rng) -> dict:
    kind = rng.choice(["decode", "decode", "chunk", "chunk", "mixed", "append", "fork", "compact"])
    kv, g, d = rng.choice(HEADS)
    page = rng.choice([16, 32, 64, 128])
    shape = dict(kv_heads=kv, groups=g, dim=d, page=page)
    if kind in ("decode", "chunk", "mixed"):
        window = rng.choice([0, 0, _log_int(rng, 1, 5000)])
        seen = dict(shape, window=window, sinks=rng.choice([0, 4, rng.randint(1, 70)]) if window else 0)
        if kind == "decode":
            context = _log_int(rng, 1, 40960)
            return _attention(context=context, sequences=_log_int(rng, 1, min(64, 100000 // context + 1)), **seen)
        context = _log_int(rng, 2, 16384)
        new = _log_int(rng, 2, min(2048, context))
        if kind == "chunk":
            return _attention(context=context, chunks=1, new=new, **seen)
        context, new = min(context, 4096), min(new, 400, context)
        return _attention(context=context, sequences=rng.randint(2, 30), chunks=rng.randint(1, 2), new=new, **seen)
    if kind == "append":
        context = _log_int(rng, 2, 8000)
        if rng.random() < 0.5:
            return _append(context=context, sequences=_log_int(rng, 1, 64), **shape)
        return _append(context=context, chunks=1, new=_log_int(rng, 2, min(2048, context)), **shape)
    page = rng.choice([16, 32])
    if kind == "fork":
        return dict(kind="fork", prompts=rng.randint(1, 8), beams=rng.randint(2, 6), context=_log_int(rng, 8, 700),
                    grow=rng.randint(1, 40), page=page, layers=rng.randint(4, 20), kv_heads=kv, dim=d)
    return dict(kind="compact", pages=_log_int(rng, 16, 380), used=rng.choice([0.2, 0.5, 0.8]), sequences=rng.randint(1, 20),
                page=page, layers=rng.randint(4, 18), kv_heads=kv, dim=d)


# --------------------------------------------------------------------------- sizes of a case
def _batch(case: dict):
    """New tokens and lengths of each sequence: lengths from half of the context to all of it; the first
    `chunks` sequences bring `new` tokens, the others one."""
    c, n = case["context"], case["sequences"]
    lengths = np.random.default_rng(c).integers(max(1, c // 2), c + 1, n)
    lengths[-1] = c
    counts = np.ones(n, dtype=np.int64)
    counts[:case["chunks"]] = case["new"]
    lengths = np.maximum(lengths, counts)
    if case["chunks"]:
        lengths[0] = c
    return counts.tolist(), lengths.tolist()


def _fork_lengths(case: dict):
    """Tokens of each prompt, and of every row (prompts first, then their forks) after the growth."""
    rng = np.random.default_rng(case["context"])
    prompts = rng.integers(max(1, 3 * case["context"] // 4), case["context"] + 1, case["prompts"])
    rows = case["prompts"] * case["beams"]
    grown = prompts[np.arange(rows) % case["prompts"]] + rng.integers(1, case["grow"] + 1, rows)
    return prompts.tolist(), grown.tolist()


def _holes(case: dict):
    """How many sequences hold each page, and the table: `used` of the pages, scattered; some held twice."""
    rng = np.random.default_rng(case["pages"])
    live = np.sort(rng.permutation(case["pages"])[:max(1, int(case["used"] * case["pages"]))])
    rows = case["sequences"]
    entries = -(-len(live) // rows)
    table = np.full((rows + 1, entries + 1), -1, dtype=np.int32)
    order = rng.permutation(live)
    for r in range(rows):
        part = order[r * entries:(r + 1) * entries]
        table[r, :len(part)] = part
    table[rows] = table[0]                      # a fork of the first sequence
    refs = np.bincount(table[table >= 0], minlength=case["pages"]).astype(np.int32)
    return table, refs, live


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
    kind, page, kv, d = case["kind"], case["page"], case["kv_heads"], case["dim"]
    s = {"case": case}
    if kind in ("attention", "append"):
        counts, lengths = _batch(case)
        need = [-(-n // page) for n in lengths]
        pages = sum(need) + 5
        order = rng.permutation(pages)          # a sequence's pages lie anywhere
        table = np.full((len(need), max(need) + 2), -1, dtype=np.int32)
        at = 0
        for r, n in enumerate(need):
            table[r, :n] = order[at:at + n]
            at += n
        starts = np.concatenate([[0], np.cumsum(counts)])
        tokens, heads = int(starts[-1]), kv * case["groups"]
        s |= {"table": _ints(table), "lengths": _ints(lengths), "most": max(counts),
              "starts": None if max(counts) == 1 else _ints(starts),
              "keys": _pool((pages, kv, page, d), gen), "values": _pool((pages, kv, page, d), gen),
              "out": torch.empty((tokens, heads, d), device="cuda")}
        if kind == "attention":
            s["query"] = _normal((tokens, heads, d), gen)
        else:
            s["qkv"] = 2.0 * _normal((tokens, (heads + 2 * kv) * d), gen)
            s["q_norm"], s["k_norm"] = (0.9 + 0.2 * torch.rand(d, generator=gen, device="cuda") for _ in range(2))
            inverse = ROPE_THETA ** (-np.arange(0, d, 2) / d)
            angles = np.arange(max(lengths) + 1)[:, None] * inverse[None, :]
            s["cos"], s["sin"] = (torch.from_numpy(f(angles).astype(np.float32)).cuda() for f in (np.cos, np.sin))
            s["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        return s
    if kind == "fork":
        prompts, grown = _fork_lengths(case)
        rows = len(grown)
        need = [-(-n // page) for n in prompts]
        fresh = sum(-(-n // page) - prompts[r % len(prompts)] // page for r, n in enumerate(grown))
        pages = sum(need) + fresh + 3
        table = np.full((rows, max(-(-n // page) for n in grown) + 1), -1, dtype=np.int32)
        order = rng.permutation(pages)
        at = 0
        for r, n in enumerate(need):
            table[r, :n] = order[at:at + n]
            at += n
        refs = np.bincount(table[table >= 0], minlength=pages)
        s |= {"table": _ints(table), "lengths": _ints(prompts + [0] * (rows - len(prompts))), "refs": _ints(refs),
              "parents": _ints(np.arange(rows) % len(prompts)), "grown": _ints(grown),
              "released": _ints(prompts + [0] * (rows - len(prompts)))}
    else:
        table, refs, _ = _holes(case)
        pages = case["pages"]
        s |= {"table0": _ints(table), "refs0": _ints(refs), "live": torch.zeros(1, dtype=torch.int32, device="cuda")}
        s |= {"table": s["table0"].clone(), "refs": s["refs0"].clone()}
    s |= {"keys": _pool((case["layers"], pages, kv, page, d), gen), "values": _pool((case["layers"], pages, kv, page, d), gen),
          "status": torch.zeros(1, dtype=torch.int32, device="cuda")}
    return s


# --------------------------------------------------------------------------- one pass
def run(s: dict):
    case = s["case"]
    kind = case["kind"]
    if kind == "attention":
        if own:
            from harsh4b_amd.paged import paged_attention
            return paged_attention(s["query"], s["keys"], s["values"], s["table"], s["lengths"], starts=s["starts"],
                                   window=case["window"], sinks=case["sinks"], out=s["out"])
        return _plain_attention(s)
    if kind == "append":
        if own:
            from harsh4b_amd.paged import paged_append
            query = paged_append(s["qkv"], s["q_norm"], s["k_norm"], s["cos"], s["sin"], EPS, s["keys"], s["values"],
                                 s["table"], s["lengths"], s["status"], starts=s["starts"], out=s["out"])
        else:
            query = _plain_append(s)
        return query, s["keys"], s["values"]
    pools = s["keys"], s["values"]
    if kind == "fork":
        if own:
            from harsh4b_amd.paged import pages_fork, pages_resize
            book = s["table"], s["lengths"], s["refs"]
            pages_resize(*pools, *book, s["status"], s["released"])        # the last beams end
            pages_fork(*book, s["status"], s["parents"])
            pages_resize(*pools, *book, s["status"], s["grown"])
        else:
            _plain_resize(s, s["released"])
            _plain_fork(s)
            _plain_resize(s, s["grown"])
        return (*pools, s["table"], s["lengths"], s["refs"])
    s["table"].copy_(s["table0"])                                          # the holes come back
    s["refs"].copy_(s["refs0"])
    if own:
        from harsh4b_amd.paged import pages_compact
        pages_compact(*pools, s["table"], s["refs"], live=s["live"])
    else:
        _plain_compact(s)
    return (*pools, s["table"], s["refs"], s["live"])


# --------------------------------------------------------------------------- plain forms
def _places(s: dict):
    """Of each new token: its sequence, its place among the sequence's new tokens, its position."""
    tokens, rows = s["out"].shape[0], s["table"].shape[0]
    starts = s["starts"].long() if s["starts"] is not None else torch.arange(rows + 1, device="cuda")
    t = torch.arange(tokens, device="cuda")
    row = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    place = t - starts[row]
    count = starts[1:] - starts[:-1]
    return row, place, s["lengths"].long()[row] - count[row] + place, starts[:-1], count


def _plain_attention(s: dict) -> torch.Tensor:
    case, query = s["case"], s["query"]
    kv, g, d = case["kv_heads"], case["groups"], case["dim"]
    row, place, _, first, count = _places(s)
    rows, most = s["table"].shape[0], s["most"]
    span = s["table"].shape[1] * case["page"]

    def history(pool):      # [rows, kv, positions, d]
        return pool[s["table"].clamp_min(0).long()].permute(0, 2, 1, 3, 4).reshape(rows, kv, span, d).float()

    place_of = torch.arange(most, device="cuda")
    token = (first[:, None] + place_of[None, :]).clamp_max(query.shape[0] - 1)
    q = query[token].view(rows, most, kv, g, d).permute(0, 2, 3, 1, 4).reshape(rows, kv, g * most, d)
    scores = (q @ history(s["keys"]).transpose(-1, -2).contiguous()).view(rows, kv, g, most, span) / math.sqrt(d)
    at = (s["lengths"].long() - count)[:, None] + place_of[None, :]                       # [rows, most]
    j = torch.arange(span, device="cuda")
    seen = j <= at[..., None]
    if case["window"]:
        seen &= (j > at[..., None] - case["window"]) | (j < case["sinks"])
    seen &= (s["table"] >= 0).repeat_interleave(case["page"], dim=1)[:, None, :]
    seen = seen[:, None, None]
    scores = scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(dim=-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    p = scores.sub_(top).exp_()
    o = p.view(rows, kv, g * most, span) @ history(s["values"])
    o = o.view(rows, kv, g, most, d) / p.sum(dim=-1, keepdim=True)
    return o.permute(0, 3, 1, 2, 4)[row, place].reshape(query.shape)


def _plain_append(s: dict) -> torch.Tensor:
    case = s["case"]
    kv, heads, d, page = case["kv_heads"], case["kv_heads"] * case["groups"], case["dim"], case["page"]
    row, _, position, _, _ = _places(s)
    x = s["qkv"].view(-1, heads + 2 * kv, d)
    cos, sin = s["cos"][position][:, None, :], s["sin"][position][:, None, :]

    def turned(a, weight):
        a = a / torch.sqrt((a * a).mean(dim=-1, keepdim=True) + EPS) * weight
        lo, hi = a[..., :d // 2], a[..., d // 2:]
        return torch.cat((lo * cos - hi * sin, hi * cos + lo * sin), dim=-1)

    where = s["table"][row, position // page].long(), slice(None), position % page
    s["keys"][where] = turned(x[:, heads:heads + kv], s["k_norm"]).half()
    s["values"][where] = x[:, heads + kv:].half()
    return turned(x[:, :heads], s["q_norm"])


def _count_refs(s: dict) -> None:
    held = torch.where(s["table"] >= 0, s["table"], s["refs"].shape[0]).flatten().long()
    count = torch.zeros(s["refs"].shape[0] + 1, dtype=torch.int32, device="cuda")
    count.index_add_(0, held, torch.ones_like(held, dtype=torch.int32))
    s["refs"].copy_(count[:-1])


def _plain_fork(s: dict) -> None:
    parents = s["parents"].long()
    s["table"].copy_(s["table"][parents])
    s["lengths"].copy_(s["lengths"][parents])
    _count_refs(s)


def _plain_resize(s: dict, new: torch.Tensor) -> None:
    page, table, refs = s["case"]["page"], s["table"], s["refs"]
    rows, entries = table.shape
    r, e = torch.arange(rows, device="cuda"), torch.arange(entries, device="cuda")
    old = s["lengths"].long()
    growing = new > old
    # the partly filled page that a growing row writes to: kept by the first of the rows that grow in it where
    # all of its holders do, copied by the others
    last = (old // page).clamp_max(entries - 1)
    source = table[r, last].long()
    partial = growing & (old % page > 0) & (source >= 0)
    holds = torch.where(partial, source, refs.shape[0])
    same = holds[:, None] == holds[None, :]
    others = same.sum(dim=1)
    first = (same & (r[None, :] < r[:, None])).sum(dim=1) == 0
    copied = partial & (refs[source.clamp_min(0)] > 1) & ~(first & (others == refs[source.clamp_min(0)]))
    wanted = (e[None, :] * page < new[:, None]) & ((table < 0) & (e[None, :] * page >= old[:, None] - old[:, None] % page))
    wanted |= copied[:, None] & (e[None, :] == last[:, None])
    free = torch.nonzero(refs == 0).flatten()
    rank = wanted.flatten().long().cumsum(0).view(rows, entries) - 1
    fresh = free[rank.clamp(0, free.shape[0] - 1)].int()
    table.copy_(torch.where(wanted, fresh, torch.where(e[None, :] * page < new[:, None], table, -1)))
    c = torch.nonzero(copied).flatten()
    target, source = table[c, last[c]].long(), source[c]
    filled = (torch.arange(page, device="cuda")[None, :] < (old[c] % page)[:, None])[None, :, None, :, None]
    for pool in (s["keys"], s["values"]):
        pool[:, target] = torch.where(filled, pool[:, source], pool[:, target])
    s["lengths"].copy_(new)
    _count_refs(s)


def _plain_compact(s: dict) -> None:
    refs = s["refs"]
    page = torch.arange(refs.shape[0], device="cuda")
    live = (refs > 0).sum()
    source = torch.nonzero((refs > 0) & (page >= live)).flatten()
    target = torch.nonzero((refs == 0) & (page < live)).flatten()
    for pool in (s["keys"], s["values"]):
        pool[:, target] = pool[:, source]
    moved = page.clone()
    moved[source] = target
    s["table"].copy_(torch.where(s["table"] >= 0, moved[s["table"].clamp_min(0).long()].int(), s["table"]))
    _count_refs(s)
    s["live"].copy_(live)


# --------------------------------------------------------------------------- what a pass cannot do without
def _pairs(count: int, length: int, window: int, sinks: int):
    """(query, key) pairs that count, and the positions of the cache that any of the queries sees."""
    p = np.arange(length - count, length)
    low = np.maximum(0, p - window + 1) if window else np.zeros_like(p)
    pairs = p - low + 1 + np.minimum(low, sinks)
    return int(pairs.sum()), int(length - low[0] + min(low[0], sinks))


def work(case: dict) -> dict:
    kind, kv, d, page = case["kind"], case["kv_heads"], case["dim"], case["page"]
    if kind in ("attention", "append"):
        counts, lengths = _batch(case)
        tokens, heads = sum(counts), kv * case["groups"]
        if kind == "append":
            return {"bytes": tokens * (4 * (heads + 2 * kv) * d + 4 * heads * d + 4 * kv * d + 4 * d + 8),
                    "flops": tokens * (heads + kv) * d * 8}
        seen = [_pairs(n, length, case["window"], case["sinks"]) for n, length in zip(counts, lengths)]
        positions = sum(x[1] for x in seen)
        return {"bytes": positions * kv * d * 4 + positions // page * 4 + tokens * heads * d * 8,
                "flops": 4 * heads * d * sum(x[0] for x in seen)}
    row = case["layers"] * kv * d * 2 * 2                                # bytes of a position's keys and values
    if kind == "fork":
        prompts, grown = _fork_lengths(case)
        copied = sum(n % page for n in prompts) * (case["beams"] - 1)
        entries = sum(-(-n // page) for n in grown)
        return {"bytes": 2 * copied * row + 3 * 8 * entries, "flops": entries}
    _, _, live = _holes(case)
    return {"bytes": 2 * int((live >= len(live)).sum()) * page * row + 8 * len(live) + 8 * case["pages"],
            "flops": case["pages"]}


# --------------------------------------------------------------------------- 64-bit results
def _rows_of(pool, table_row, length: int):
    """One sequence's [positions, kv, d] in float64."""
    page = pool.shape[-2]
    ids = table_row[:-(-length // page)].long()
    return pool[ids].transpose(1, 2).reshape(-1, pool.shape[1], pool.shape[3])[:length].double()


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "attention":
        return _exact_attention(case, s)
    if kind == "append":
        return _exact_append(case, s)
    return None         # pages are copied and integers counted: no rounding to measure


def _exact_attention(case: dict, s: dict) -> torch.Tensor:
    counts, lengths = _batch(case)
    kv, g, d = case["kv_heads"], case["groups"], case["dim"]
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device="cuda")
    token = 0
    for b, (n, length) in enumerate(zip(counts, lengths)):
        keys, values = (_rows_of(s[name], s["table"][b], length) for name in ("keys", "values"))
        far = torch.arange(length - n, length, device="cuda")[:, None] - torch.arange(length, device="cuda")[None, :]
        hidden = far < 0
        if case["window"]:
            hidden |= (far >= case["window"]) & (torch.arange(length, device="cuda")[None, :] >= case["sinks"])
        for h in range(kv * g):
            q = s["query"][token:token + n, h].double()
            score = torch.mm(q, keys[:, h // g].t().contiguous()) * d ** -0.5
            weight = torch.softmax(score.masked_fill(hidden, -math.inf), dim=-1)
            out[token:token + n, h] = torch.mm(weight, values[:, h // g].contiguous())
        token += n
    return out


def _exact_append(case: dict, s: dict):
    counts, lengths = _batch(case)
    kv, heads, d, page = case["kv_heads"], case["kv_heads"] * case["groups"], case["dim"], case["page"]
    x = s["qkv"].double().view(-1, heads + 2 * kv, d)
    keys, values = s["keys"].double(), s["values"].double()
    query = torch.empty((x.shape[0], heads, d), dtype=torch.float64, device="cuda")
    token = 0
    for b, (n, length) in enumerate(zip(counts, lengths)):
        at = torch.arange(length - n, length, device="cuda")
        turn = torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, None, :]
        part = x[token:token + n]

        def rotated(a, weight):
            a = a * torch.rsqrt(a.pow(2).sum(-1, keepdim=True) / d + EPS) * weight.double()
            z = torch.complex(a[..., :d // 2].contiguous(), a[..., d // 2:].contiguous()) * turn
            return torch.cat((z.real, z.imag), dim=-1)

        query[token:token + n] = rotated(part[:, :heads], s["q_norm"])
        ids = s["table"][b][at // page].long()
        keys[ids, :, at % page] = rotated(part[:, heads:heads + kv], s["k_norm"])
        values[ids, :, at % page] = part[:, heads + kv:]
        token += n
    return query, keys, values
