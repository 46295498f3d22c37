"""The operators of steps that check drafted tokens, as cases that can be timed and checked.

A request that decodes with drafts brings a small tree of tokens to a step: node 0 is its newest certain
token, every other node a guess with a parent among the nodes before it.  Four operators deal with such trees:
`attend` is attention of all nodes over a paged cache (a node sees the rows before the step and, of the step's
own rows, those that its mask names: itself and its ancestors), `verify` walks from the root along the drafts that
the target model's probabilities accept and draws the token behind them, `keep` moves the accepted nodes' rows of
every layer's cache to the front of the step's rows, and `lookup` drafts: what followed the latest earlier
occurrences of a request's last few tokens, up to `branches` chains with different first tokens.
"""

from __future__ import annotations

import math
import random
from typing import Any, Optional

import numpy as np
import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
NEVER = -1e30  # a score that is masked
VOCAB = 151936  # the vocabulary of the dense presets


# ---------------------------------------------------------------------------
# the cases


def _attend(name: Optional[str], *, seqs: int, context: int, nodes: int, heads: int = 32, kv_heads: int = 8, dim: int = 128, page: int = 16,
            dtype: str = "bfloat16", ragged: bool = False, window: int = 0, sinks: bool = False, cap: float = 0.0, chain: bool = False) -> dict[str, Any]:
    """`seqs` requests of about `context` rows, the step's `nodes` among them; `ragged`: their lengths and trees differ in size."""
    c = {"op": "attend", "seqs": seqs, "context": context, "nodes": nodes, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
         "dtype": dtype, "ragged": ragged, "window": window, "sinks": sinks, "cap": cap, "chain": chain}
    return c if name is None else {"name": name, **c}


def _verify(name: Optional[str], *, seqs: int, nodes: int, vocab: int = VOCAB, dtype: str = "float32", chain: bool = False, probs: bool = False,
            ragged: bool = False, greedy: bool = False) -> dict[str, Any]:
    """Trees (or chains) of `nodes` nodes; `probs`: the drafts were drawn from given probabilities; `greedy`: every third request is greedy."""
    c = {"op": "verify", "seqs": seqs, "nodes": nodes, "vocab": vocab, "dtype": dtype, "chain": chain, "probs": probs, "ragged": ragged,
         "greedy": greedy}
    return c if name is None else {"name": name, **c}


def _keep(name: Optional[str], *, seqs: int, nodes: int, layers: int, context: int, kv_heads: int = 8, dim: int = 128, page: int = 16,
          dtype: str = "bfloat16") -> dict[str, Any]:
    c = {"op": "keep", "seqs": seqs, "nodes": nodes, "layers": layers, "context": context, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype}
    return c if name is None else {"name": name, **c}


def _lookup(name: Optional[str], *, seqs: int, length: int, depth: int, branches: int, longest: int = 4, shortest: int = 1) -> dict[str, Any]:
    """Requests of up to `length` tokens; suffixes of `shortest` to `longest` tokens are looked for."""
    c = {"op": "lookup", "seqs": seqs, "length": length, "depth": depth, "branches": branches, "longest": longest, "shortest": shortest}
    return c if name is None else {"name": name, **c}


def listed() -> list[dict[str, Any]]:
    return [
        # one user of the smallest preset with a handful of drafts: latency counts
        _attend("tree 1 at 500", seqs=1, context=517, nodes=6, heads=16),
        # a batch of chains, as a lookup in the request's own tokens gives them
        _attend("chains 32 at 4096", seqs=32, context=4096, nodes=5, ragged=True, chain=True),
        # the usual step of a server with trees
        _attend("trees 16 at 4096", seqs=16, context=4096, nodes=32, ragged=True),
        # large trees over long documents, five query heads per key head, pages of another size
        _attend("trees 4 at 30000", seqs=4, context=30000, nodes=61, heads=40, page=64),
        # a layer with a window and learned sinks in true float32, heads of 64
        _attend("trees window float32", seqs=12, context=3000, nodes=13, heads=64, dim=64, dtype="float32", ragged=True, window=1024, sinks=True),
        # a single request's chain
        _verify("verify chain 1", seqs=1, nodes=5, chain=True),
        # chains from a small draft model, whose probabilities count
        _verify("verify chains 32", seqs=32, nodes=6, chain=True, probs=True, ragged=True),
        # large trees of a batch
        _verify("verify trees 16 of 61", seqs=16, nodes=61, greedy=True),
        # one request of the smallest preset
        _keep("keep 1, 28 layers", seqs=1, nodes=6, layers=28, context=700),
        # a batch of a larger one
        _keep("keep 16, 36 layers", seqs=16, nodes=32, layers=36, context=90, page=64),
        # one request's tokens
        _lookup("lookup 1 at 700", seqs=1, length=700, depth=4, branches=1),
        # a batch of long documents, trees of four chains
        _lookup("lookup 64 at 30000", seqs=64, length=30000, depth=8, branches=4, longest=6),
    ]


def _spread(rng: random.Random, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng: random.Random) -> dict[str, Any]:
    most = {}
    for c in listed():
        for k, w in work(c).items():
            most[c["op"], k] = max(most.get((c["op"], k), 0), w)
    while True:  # one that costs no more than the largest of its kind
        c = _any(rng)
        if all(w <= most[c["op"], k] for k, w in work(c).items()):
            return c


def _any(rng: random.Random) -> dict[str, Any]:
    op = rng.choice(["attend", "attend", "attend", "verify", "verify", "keep", "lookup"])
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    if op == "attend":
        kv_heads = rng.choice([1, 2, 4, 8, 8])
        nodes, seqs = _spread(rng, 1, 64), _spread(rng, 1, 64)
        context = nodes + _spread(rng, 1, max(2, min(30000, 130000 // seqs)))
        window = _spread(rng, 16, 4096) if rng.random() < 0.25 else 0
        return _attend(None, seqs=seqs, context=context, nodes=nodes, heads=kv_heads * rng.choice([1, 2, 4, 4, 5, 7, 8, 16]), kv_heads=kv_heads,
                       dim=rng.choice([64, 128, 128, 128, 256]), page=rng.choice([16, 16, 32, 64, 128]), dtype=dtype, ragged=rng.random() < 0.6,
                       window=window, sinks=rng.random() < 0.25, cap=rng.choice([0.0, 0.0, 0.0, 30.0]), chain=rng.random() < 0.4)
    if op == "verify":
        return _verify(None, seqs=_spread(rng, 1, 64), nodes=_spread(rng, 1, 61), vocab=rng.choice([_spread(rng, 1000, 160000), VOCAB]),
                       dtype=rng.choice(["float32", "float32", "bfloat16"]), chain=rng.random() < 0.5, probs=rng.random() < 0.4,
                       ragged=rng.random() < 0.5, greedy=rng.random() < 0.4)
    if op == "keep":
        nodes = _spread(rng, 2, 64)
        return _keep(None, seqs=_spread(rng, 1, 24), nodes=nodes, layers=rng.randint(2, 40), context=nodes + _spread(rng, 1, 500), kv_heads=rng.choice([1, 2, 4, 8]),
                     dim=rng.choice([64, 128, 128, 256]), page=rng.choice([16, 16, 32, 64]), dtype=dtype)
    shortest = rng.choice([1, 1, 2])
    return _lookup(None, seqs=_spread(rng, 1, 128), length=_spread(rng, 2, 30000), depth=rng.randint(1, 10), branches=rng.randint(1, 6),
                   longest=rng.randint(shortest, 8), shortest=shortest)


def _sizes(case: dict[str, Any]) -> list[tuple[int, int]]:
    """(rows, nodes of this step) of every request; the same for every seed."""
    rng = random.Random("%d %d %d" % (case["seqs"], case.get("context", 0), case["nodes"]))
    out = []
    for _ in range(case["seqs"]):
        n, t = case.get("context", case["nodes"]), case["nodes"]
        if case.get("ragged"):
            n, t = max(1, round(n * rng.uniform(0.3, 1.0))), max(1, round(t * rng.uniform(0.3, 1.0)))
        out.append((max(n, t), t))
    return out


def _depth(nodes: int, chain: bool) -> int:
    """About how many drafts stand one behind the other in a tree of that many nodes."""
    return nodes - 1 if chain else min(nodes - 1, 2 + int(math.log2(max(1, nodes))))


def work(case: dict[str, Any]) -> dict[str, float]:
    if case["op"] == "attend":
        item, nq, nkv, d, w = DTYPES[case["dtype"]].itemsize, case["heads"], case["kv_heads"], case["dim"], case["window"]
        rows = pairs = tokens = 0
        for n, t in _sizes(case):
            seen = min(n - t, w) if w else n - t  # (about: deeper nodes see a little less of a window)
            inside = t * (t + 1) // 2 if case["chain"] else t * min(t, 1 + _depth(t, False))  # (about: a node and its ancestors)
            rows, pairs, tokens = rows + seen + t, pairs + t * seen + inside, tokens + t
        return {"bytes": 2 * rows * nkv * d * item + 2 * tokens * nq * d * item, "flops": 4.0 * pairs * nq * d}
    if case["op"] == "verify":
        # a row of logits for every node on the way, the root's among them: about 0.6 of the drafts are right (and where there are
        # probabilities of the drafter, the row of those at the node where a draft was refused)
        rows = sum(1 + sum(0.6**i for i in range(1, 1 + _depth(t, case["chain"]))) for _, t in _sizes(case))
        item = DTYPES[case["dtype"]].itemsize
        return {"bytes": rows * case["vocab"] * item + (case["seqs"] * case["vocab"] * 4 if case["probs"] else 0), "flops": 0}
    if case["op"] == "keep":
        moved = case["seqs"] * max(1, _depth(case["nodes"], False) // 2)
        return {"bytes": 4.0 * moved * case["layers"] * case["kv_heads"] * case["dim"] * DTYPES[case["dtype"]].itemsize, "flops": 0}
    return {"bytes": case["seqs"] * (case["length"] * 4.0 + 8 * (1 + case["depth"] * case["branches"])), "flops": 0}


# ---------------------------------------------------------------------------
# what a program has in hand


def _parents(rng: random.Random, nodes: int, chain: bool) -> list[int]:
    """A tree: every node hangs on one before it, the early ones (the likelier guesses) more often."""
    if chain:
        return list(range(-1, nodes - 1))
    return [-1] + [min(i - 1, int((i * rng.random() ** 1.3))) for i in range(1, nodes)]


def _ancestors(parents: list[int]) -> list[list[int]]:
    out: list[list[int]] = []
    for i, p in enumerate(parents):
        out.append((out[p] if p >= 0 else []) + [i])
    return out


def _words(nodes_seen: list[int], words: int) -> list[int]:
    out = [0] * words
    for i in nodes_seen:
        out[i // 64] |= 1 << (i % 64)
    return [w - (1 << 64) if w >= 1 << 63 else w for w in out]


def _pages(g, dev, rows: list[int], page: int):
    """A block table of pages in no order, and their number (a few belong to nobody)."""
    per = [-(-n // page) for n in rows]
    total = sum(per) + 3
    order = torch.randperm(total, generator=g, device=dev).int()
    table = torch.full((len(rows), max(per)), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, p in enumerate(per):
        table[b, :p] = order[at : at + p]
        at += p
    return table, total


def prepare(case: dict[str, Any], seed: int) -> dict[str, Any]:
    g = torch.Generator("cuda").manual_seed(seed)
    return {"attend": _prepare_attend, "verify": _prepare_verify, "keep": _prepare_keep, "lookup": _prepare_lookup}[case["op"]](
        case, g, torch.device("cuda"), random.Random(seed))


def _ints(dev, x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=dev)


def _prepare_attend(case, g, dev, rng):
    dtype = DTYPES[case["dtype"]]
    nq, nkv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    sizes = _sizes(case)
    rows, tokens = [n for n, _ in sizes], [t for _, t in sizes]
    table, total = _pages(g, dev, rows, page)
    width = torch.exp(0.5 * torch.randn((nkv, d), generator=g, device=dev))  # channels of keys differ in size
    k = torch.randn((total, page, nkv, d), generator=g, device=dev).mul_(width).to(dtype)
    v = torch.randn((total, page, nkv, d), generator=g, device=dev).to(dtype)
    words = -(-max(tokens) // 64)
    mask, positions, aimed = [], [], []
    for b, (n, t) in enumerate(sizes):
        seen = _ancestors(_parents(rng, t, case["chain"]))
        mask += [_words(s, words) for s in seen]
        positions += [n - t + len(s) - 1 for s in seen]
        j = (torch.rand((t,), generator=g, device=dev) * (n - t + 1)).long()  # every query looks for a row among those before it
        aimed.append(k.flatten(0, 1)[table[b, j // page].long() * page + j % page].float())
    T = sum(tokens)
    spread = width.repeat_interleave(nq // nkv, 0)
    q = 0.7 * torch.randn((T, nq, d), generator=g, device=dev) / spread + 0.4 * torch.cat(aimed).repeat_interleave(nq // nkv, 1) / spread**2
    return {"case": dict(case), "q": q.to(dtype).flatten(1), "k": k, "v": v, "table": table, "mask": _ints(dev, mask, torch.int64),
            "positions": _ints(dev, positions), "cu": _ints(dev, [sum(tokens[:b]) for b in range(len(tokens) + 1)]), "context_lens": _ints(dev, rows),
            "max_query": max(tokens), "max_context": max(rows),
            "head_sinks": torch.randn(nq, generator=g, device=dev) if case["sinks"] else None}


def _prepare_verify(case, g, dev, rng):
    V, dtype = case["vocab"], DTYPES[case["dtype"]]
    nodes = [t for _, t in _sizes(case)]
    T, B = sum(nodes), len(nodes)
    # a model's logits: a few candidates that hold most of the probability, and a long tail
    logits = torch.empty((T, V), device=dev, dtype=dtype)
    few = (torch.randint(0, V, (T, 1), generator=g, device=dev) + torch.arange(8, device=dev) * (V // 8)) % V  # eight different tokens
    top = math.log(V) + 1.1 + 2.5 - 0.9 * torch.arange(8, device=dev) + torch.randn((T, 8), generator=g, device=dev)
    for a in range(0, T, 64):
        x = 1.5 * torch.randn((min(64, T - a), V), generator=g, device=dev)
        logits[a : a + 64] = x.scatter_(1, few[a : a + 64], top[a : a + 64]).to(dtype)
    probs = None
    if case["probs"]:  # the drafter's: near the target's
        probs = torch.empty((T, V), device=dev)
        for a in range(0, T, 64):
            x = logits[a : a + 64].float()
            probs[a : a + 64] = torch.softmax(x + 0.6 * torch.randn(x.shape, generator=g, device=dev), -1)
    parents, at, parent_row = [], 0, []
    for t in nodes:
        p = _parents(rng, t, case["chain"])
        parents += p
        parent_row += [at + max(i, 0) for i in p]
        at += t
    parent_row = _ints(dev, parent_row, torch.int64)
    if probs is not None:
        race = torch.empty(T, dtype=torch.int64, device=dev)
        for a in range(0, T, 64):
            r = parent_row[a : a + 64]
            race[a : a + 64] = (probs[r] / torch.empty((len(r), V), device=dev).exponential_(generator=g)).argmax(-1)
        tokens = race
    else:  # the likeliest next token mostly, else one of the other candidates
        which = (torch.rand(T, generator=g, device=dev).pow(2.0) * 8).long()
        tokens = few[parent_row, which]
    temperatures = torch.tensor([0.0 if case["greedy"] and b % 3 == 1 else (0.7, 1.0, 1.2)[b % 3] for b in range(B)], device=dev)
    return {"case": dict(case), "logits": logits, "probs": probs, "tokens": tokens.int(), "parents": _ints(dev, parents),
            "cu": _ints(dev, [sum(nodes[:b]) for b in range(B + 1)]), "temperatures": temperatures,
            "uniforms": torch.rand(T, generator=g, device=dev),
            "keys": torch.randint(-(1 << 63), (1 << 63) - 1, (B,), generator=g, device=dev, dtype=torch.int64), "max_nodes": max(nodes)}


def _prepare_keep(case, g, dev, rng):
    dtype, nkv, d, page = DTYPES[case["dtype"]], case["kv_heads"], case["dim"], case["page"]
    sizes = _sizes(case)
    rows, tokens = [n for n, _ in sizes], [t for _, t in sizes]
    table, total = _pages(g, dev, rows, page)
    path = torch.full((len(sizes), max(tokens)), -1, dtype=torch.int32, device=dev)
    counts = []
    for b, t in enumerate(tokens):
        deepest = max(_ancestors(_parents(rng, t, False)), key=len)
        way = deepest[: rng.randint(1, len(deepest))]  # accepted up to some node
        path[b, : len(way)] = _ints(dev, way)
        counts.append(len(way) - 1)
    pools = torch.empty((2 * case["layers"], total, page, nkv, d), device=dev, dtype=dtype)
    for pool in pools:
        pool.copy_(torch.randn(pool.shape, generator=g, device=dev))
    s = {"case": dict(case), "pools": pools, "path": path, "counts": _ints(dev, counts), "table": table, "context_lens": _ints(dev, rows),
         "cu": _ints(dev, [sum(tokens[:b]) for b in range(len(tokens) + 1)])}
    if own:  # the layers' pools, named once for the life of the cache
        from tokensprint_b200 import ops

        s["handle"] = ops.RowPools(list(pools))
    return s


def _prepare_lookup(case, g, dev, rng):
    B, L = case["seqs"], case["length"]
    # text that comes back to itself: pieces copied from further up between new tokens
    history = torch.randint(0, 4000, (B, L), generator=g, device=dev, dtype=torch.int32)
    for _ in range(6):
        n = max(1, L // 9)
        if L > 2 * n:
            a, b = rng.randint(0, L - n), rng.randint(0, L - n)
            history[:, max(a, b) : max(a, b) + n] = history[:, min(a, b) : min(a, b) + n].clone()
    tail = min(case["longest"] + 2, L // 3)
    if tail:
        for _ in range(3):  # the last few tokens have been there before
            a = rng.randint(0, L - 2 * tail)
            history[:, a : a + tail] = history[:, L - tail :].clone()
    lengths = [max(1, L if b == 0 else round(L * rng.uniform(0.4, 1.0))) for b in range(B)]
    for b, n in enumerate(lengths):
        if n < L and tail and n > 3 * tail:
            history[b, n - tail : n] = history[b, L - tail :].clone()
    return {"case": dict(case), "history": history, "lengths": _ints(dev, lengths)}


# ---------------------------------------------------------------------------
# one pass


def run(s: dict[str, Any]) -> dict[str, Any]:
    op = s["case"]["op"]
    if own:
        return {"attend": _own_attend, "verify": _own_verify, "keep": _own_keep, "lookup": _own_lookup}[op](s)
    return {"attend": _plain_attend, "verify": _plain_verify, "keep": _plain_keep, "lookup": _plain_lookup}[op](s)


def _own_attend(s):
    from tokensprint_b200 import ops

    c, q = s["case"], s["q"]
    out = torch.empty_like(q)
    ops.attention_tree(q, s["k"], s["v"], out, s["mask"], s["cu"], s["context_lens"], s["table"], c["page"], c["seqs"], s["max_query"], s["max_context"],
                       c["heads"], c["kv_heads"], c["dim"], c["dim"] ** -0.5, window=c["window"], positions=s["positions"],
                       head_sinks=s["head_sinks"], softcap=c["cap"])
    return {"out": out}


def _own_verify(s):
    from tokensprint_b200 import ops

    c, dev = s["case"], s["logits"].device
    path, fresh = (torch.empty((c["seqs"], s["max_nodes"]), dtype=torch.int32, device=dev) for _ in range(2))
    counts = torch.empty(c["seqs"], dtype=torch.int32, device=dev)
    ops.verify_drafts(s["logits"], s["tokens"], s["parents"], s["cu"], s["temperatures"], s["uniforms"], s["keys"], path, fresh, counts, c["seqs"],
                      s["max_nodes"], draft_probs=s["probs"])
    return {"path": path, "tokens": fresh, "counts": counts}


def _own_keep(s):
    from tokensprint_b200 import ops

    ops.keep_drafted_rows(s["handle"], s["path"], s["counts"], s["cu"], s["context_lens"], s["table"], s["case"]["page"], s["case"]["seqs"])
    return {"pools": s["pools"]}


def _own_lookup(s):
    from tokensprint_b200 import ops

    c, dev = s["case"], s["history"].device
    tokens, parents = (torch.empty((c["seqs"], 1 + c["depth"] * c["branches"]), dtype=torch.int32, device=dev) for _ in range(2))
    counts = torch.empty(c["seqs"], dtype=torch.int32, device=dev)
    ops.lookup_drafts(s["history"], s["lengths"], tokens, parents, counts, c["seqs"], c["depth"], c["branches"], c["longest"], c["shortest"])
    return {"tokens": tokens, "parents": parents, "counts": counts}


def _plain_attend(s):
    c, q = s["case"], s["q"]
    nq, nkv, d, t_most = c["heads"], c["kv_heads"], c["dim"], s["max_query"]
    dev = q.device
    t = torch.arange(t_most, device=dev)
    count = (s["cu"][1:] - s["cu"][:-1])[:, None]
    there = t < count  # [B, t]
    token = (s["cu"][:-1, None] + t).clamp(max=q.shape[0] - 1).long()
    rows = s["table"].clamp(min=0).long()
    keys, values = (x[rows].flatten(1, 2).permute(0, 2, 1, 3).float() for x in (s["k"], s["v"]))  # [B, nkv, n, d]
    n = keys.shape[2]
    j = torch.arange(n, device=dev)
    first = s["context_lens"][:, None] - count  # rows before the step
    node = j - first  # [B, n], the node that lies in a row
    inside = (node >= 0) & (node < count)
    word = s["mask"][token]  # [B, t, words]
    which = node.clamp(0, 64 * word.shape[2] - 1)
    picked = torch.gather(word, 2, (which // 64)[:, None].expand(-1, t_most, -1).long())
    named = ((picked >> (which % 64)[:, None]) & 1) == 1
    seen = torch.where(inside[:, None], named, (node < 0)[:, None])
    if c["window"]:
        position = s["positions"][token]  # [B, t]
        of_node = torch.gather(position, 1, node.clamp(0, t_most - 1).long())
        of_row = torch.where(inside, of_node, j)
        seen = seen & (of_row[:, None] > position[..., None] - c["window"])
    seen = (seen & there[..., None])[:, None, None]  # [B, 1, 1, t, n]
    x = q.float().view(-1, nkv, nq // nkv, d)[token].permute(0, 2, 3, 1, 4)  # [B, nkv, G, t, d]
    scores = (x.flatten(2, 3) @ keys.transpose(-1, -2)).unflatten(2, (nq // nkv, -1)) * d**-0.5
    if c["cap"]:
        scores = c["cap"] * torch.tanh(scores / c["cap"])
    scores = torch.where(seen, scores, NEVER)
    top = scores.amax(-1, keepdim=True)
    if s["head_sinks"] is not None:
        sink = s["head_sinks"].view(1, nkv, -1, 1, 1)
        top = torch.maximum(top, sink)
    p = torch.exp(scores - top) * seen
    total = p.sum(-1, keepdim=True)
    if s["head_sinks"] is not None:
        total = total + torch.exp(sink - top)
    p = p / torch.where(total > 0, total, 1.0)
    out = (p.flatten(2, 3) @ values).unflatten(2, (nq // nkv, -1)).permute(0, 3, 1, 2, 4)
    return {"out": out[there].flatten(1).to(q.dtype)}


def _shift(z: torch.Tensor, n: int) -> torch.Tensor:
    """Bits moved down, zeros in front."""
    return (z >> n) & ((1 << (64 - n)) - 1)


def _signed(x: int) -> int:
    return x - (1 << 64) if x >= 1 << 63 else x


def _waits(keys: torch.Tensor, V: int) -> torch.Tensor:
    """Exponential waiting times [B, V] in 64 bits: E = -ln(1 - (c + 1/2) / 2^24), c 24 bits of a hash of (key, entry / 2), the upper ones of
    its 48 for even entries, the lower ones for odd."""
    pair = torch.arange((V + 1) // 2, device=keys.device)
    z = keys[:, None] ^ (pair * _signed(0xD1342543DE82EF95))
    z = (z ^ _shift(z, 32)) * _signed(0x94D049BB133111EB)
    z = z ^ _shift(z, 29)
    c = torch.stack((_shift(z, 40), _shift(z, 16) & 0xFFFFFF), -1).flatten(1)[:, :V]
    return -torch.log1p(-(c.double() + 0.5) / (1 << 24))


def _plain_verify(s):
    c, dev = s["case"], s["logits"].device
    B, V = c["seqs"], c["vocab"]
    first, count = s["cu"][:-1].long(), (s["cu"][1:] - s["cu"][:-1]).long()
    b = torch.arange(B, device=dev)
    greedy = s["temperatures"] <= 1e-10
    heat = torch.where(greedy, 1.0, s["temperatures"])[:, None].double()
    here = torch.zeros(B, dtype=torch.long, device=dev)
    accepted = torch.zeros(B, dtype=torch.long, device=dev)
    path = torch.full((B, s["max_nodes"]), -1, dtype=torch.int32, device=dev)
    path[:, 0] = 0
    fresh = torch.full((B, s["max_nodes"]), -1, dtype=torch.int32, device=dev)

    def target(node):  # the probabilities after a node, where borders lie: in 64 bits
        return torch.softmax(s["logits"][first + node].double() / heat, -1)

    def best(node):  # the largest logit, of equals the first
        x = s["logits"][first + node].float()
        return torch.where(x == x.amax(-1, keepdim=True), torch.arange(V, device=dev), V).amin(-1)

    left, choice = target(here), best(here)
    for i in range(1, s["max_nodes"]):  # a node's parent comes before it, and its children in their order
        at = (first + i).clamp(max=s["tokens"].numel() - 1)
        asked = (i < count) & (s["parents"][at] == here)
        x = s["tokens"][at].long()
        r = left[b, x]
        if s["probs"] is None:
            guess = torch.zeros_like(left)
            guess[b, x] = 1.0
        else:
            guess = s["probs"][first + here].double()
        yes = torch.where(greedy, x == choice, s["uniforms"][at].double() * guess[b, x] < r)
        taken, refused = asked & yes, asked & ~yes
        rest = (left - guess).clamp(min=0)
        total = rest.sum(-1, keepdim=True)
        left = torch.where(refused[:, None] & (total > 0), rest / torch.where(total > 0, total, 1.0), left)
        fresh[b, accepted] = torch.where(taken, x.int(), fresh[b, accepted])
        accepted = accepted + taken
        path[b, accepted] = torch.where(taken, i, path[b, accepted].long()).int()
        here = torch.where(taken, i, here)
        left = torch.where(taken[:, None], target(here), left)
        choice = torch.where(taken, best(here), choice)
    score = left / _waits(s["keys"], V)
    drawn = torch.where(score == score.amax(-1, keepdim=True), torch.arange(V, device=dev), V).amin(-1)
    fresh[b, accepted] = torch.where(greedy, choice, drawn).int()
    return {"path": path, "tokens": fresh, "counts": accepted.int()}


def _plain_keep(s):
    page = s["case"]["page"]
    t = s["cu"][1:] - s["cu"][:-1]
    first = (s["context_lens"] - t)[:, None]
    k = torch.arange(s["path"].shape[1], device=first.device)
    moved = (k >= 1) & (k <= s["counts"][:, None])

    def slots(row):
        row = row.clamp(min=0).long()
        return torch.gather(s["table"], 1, (row // page).clamp(max=s["table"].shape[1] - 1)).long() * page + row % page

    b = torch.arange(first.shape[0], device=first.device)[:, None].expand_as(moved)
    b, k = b[moved], k.expand_as(moved)[moved]
    source = slots(first + s["path"].clamp(min=0))[b, k]
    target = slots(first + torch.arange(s["path"].shape[1], device=first.device))[b, k]
    for pool in s["pools"]:
        flat = pool.flatten(0, 1)
        flat[target] = flat[source]
    return {"pools": s["pools"]}


def _plain_lookup(s):
    c, h = s["case"], s["history"]
    B, L = h.shape
    dev = h.device
    n = s["lengths"].long()[:, None]
    j = torch.arange(L, device=dev)
    row = torch.arange(B, device=dev)
    match = torch.zeros((B, L), dtype=torch.long, device=dev)
    still = (j < n - 1).expand(B, L)
    for m in range(1, c["longest"] + 1):
        want = torch.gather(h, 1, (n - m).clamp(min=0))
        earlier = torch.cat((torch.full((B, min(m - 1, L)), -1, dtype=h.dtype, device=dev), h[:, : max(0, L - m + 1)]), 1)  # the token m - 1 places before
        still = still & (j >= m - 1) & (n >= m) & (earlier == want)
        match = match + still
    rank = torch.where(match >= c["shortest"], match * (1 << 32) + j, -1)
    width = 1 + c["depth"] * c["branches"]
    tokens, parents = (torch.full((B, width), -1, dtype=torch.int32, device=dev) for _ in range(2))
    tokens[:, 0] = torch.gather(h, 1, n - 1)[:, 0]
    counts = torch.ones(B, dtype=torch.long, device=dev)
    following = torch.cat((h[:, 1:], torch.full((B, 1), -1, dtype=h.dtype, device=dev)), 1)
    for _ in range(c["branches"]):
        top, where = rank.max(1)
        found = top >= 0
        for k in range(c["depth"]):
            at = where + 1 + k
            there = found & (at < n[:, 0])
            place = counts.clamp(max=width - 1)
            tokens[row, place] = torch.where(there, h[row, at.clamp(max=L - 1)], tokens[row, place])
            parents[row, place] = torch.where(there, 0 if k == 0 else place - 1, parents[row, place].long()).int()
            counts = counts + there
        rank = torch.where(following == following[row, where][:, None], -1, rank)
    return {"tokens": tokens, "parents": parents, "counts": counts.int()}


# ---------------------------------------------------------------------------
# the same from the definition, in 64 bits


def exact(case: dict[str, Any], seed: int):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "verify": _exact_verify, "keep": _exact_keep, "lookup": _exact_lookup}[case["op"]](case, s)


def _exact_attend(case, s):
    nq, nkv, d, page, w = case["heads"], case["kv_heads"], case["dim"], case["page"], case["window"]
    q = s["q"].double().view(-1, nq, d)
    out, G, at = torch.empty_like(q), nq // nkv, 0
    for b, (n, t) in enumerate(_sizes(case)):
        pages = s["table"][b, : -(-n // page)].long()
        words = s["mask"][at : at + t].tolist()
        hidden = torch.tensor([[not (row[i // 64] >> (i % 64)) & 1 for i in range(t)] for row in words], device=q.device).view(t, t)
        hidden = torch.cat((torch.zeros((t, n - t), dtype=torch.bool, device=q.device), hidden), 1)
        if w:
            mine = s["positions"][at : at + t]
            of_row = torch.cat((torch.arange(n - t, device=q.device), mine))
            hidden = hidden | (mine[:, None] - of_row[None] >= w)
        for h in range(nkv):
            k, v = (x[pages, :, h].reshape(-1, d)[:n].double() for x in (s["k"], s["v"]))
            for i in range(h * G, h * G + G):
                z = q[at : at + t, i] @ k.T / math.sqrt(d)
                if case["cap"]:
                    z = case["cap"] * torch.tanh(z / case["cap"])
                z = z.masked_fill(hidden, -math.inf)
                if case["sinks"]:
                    z = torch.cat((z, s["head_sinks"][i].double().expand(t, 1)), 1)
                out[at : at + t, i] = torch.softmax(z, 1)[:, :n] @ v
        at += t
    return {"out": out.flatten(1)}


def _exact_verify(case, s):
    V = case["vocab"]
    ways, drawn = [], []
    cu, tokens, parents = s["cu"].tolist(), s["tokens"].tolist(), s["parents"].tolist()
    mask64 = (1 << 64) - 1
    for b in range(case["seqs"]):
        nodes, heat = range(cu[b], cu[b + 1]), float(s["temperatures"][b])
        way, out = [0], []
        while True:
            row = s["logits"][cu[b] + way[-1]].double()
            children = [t for t in nodes if t > cu[b] and parents[t] == way[-1]]
            onward = None
            if heat == 0:
                final = int((row == row.max()).nonzero()[0])
                onward = next((t for t in children if tokens[t] == final), None)
            else:
                p = torch.exp((row - row.max()) / heat)
                p /= p.sum()
                for t in children:
                    q = None if s["probs"] is None else s["probs"][cu[b] + way[-1]].double()
                    if float(s["uniforms"][t]) * (1.0 if q is None else float(q[tokens[t]])) < float(p[tokens[t]]):
                        onward = t
                        break
                    rest = p.clone()
                    if q is None:
                        rest[tokens[t]] = 0
                    else:
                        rest = torch.relu(p - q)
                    if float(rest.sum()) > 0:
                        p = rest / rest.sum()
            if onward is None:
                break
            way.append(onward - cu[b])
            out.append(tokens[onward])
        if heat > 0:
            z = np.uint64(int(s["keys"][b]) & mask64) ^ (np.arange((V + 1) // 2, dtype=np.uint64) * np.uint64(0xD1342543DE82EF95))
            z = (z ^ (z >> np.uint64(32))) * np.uint64(0x94D049BB133111EB)
            numbers = torch.from_numpy(((z ^ (z >> np.uint64(29))) >> np.uint64(16)).astype(np.int64))
            bits = torch.stack((numbers // (1 << 24), numbers % (1 << 24)), 1).flatten()[:V].to(p.device)
            gain = torch.log(p) - torch.log(-torch.log1p(-(2 * bits.double() + 1) / (1 << 25)))
            final = int((gain == gain.max()).nonzero()[0])
        ways.append(way)
        drawn.append(out + [final])

    def table(rows):
        return torch.tensor([r + [-1] * (s["max_nodes"] - len(r)) for r in rows], dtype=torch.int32, device=s["logits"].device)

    return {"path": table(ways), "tokens": table(drawn), "counts": torch.tensor([len(w) - 1 for w in ways], dtype=torch.int32, device=s["logits"].device)}


def _exact_keep(case, s):
    page, table, ways = case["page"], s["table"].tolist(), s["path"].tolist()
    pools = s["pools"].double()
    for b, (n, t) in enumerate(_sizes(case)):
        for k in range(1, int(s["counts"][b]) + 1):
            to, fro = n - t + k, n - t + ways[b][k]
            pools[:, table[b][to // page], to % page] = s["pools"][:, table[b][fro // page], fro % page].double()
    return {"pools": pools}


def _exact_lookup(case, s):
    width = 1 + case["depth"] * case["branches"]
    tokens, parents, counts = [], [], []
    for line, n in zip(s["history"].tolist(), s["lengths"].tolist()):
        line = line[:n]
        found: dict[int, list[int]] = {}
        for j in range(n - 1):
            m = 0
            while m < case["longest"] and m <= j and line[j - m] == line[n - 1 - m]:
                m += 1
            if m >= case["shortest"]:
                found.setdefault(m, []).append(j)
        starts: list[int] = []
        for m in sorted(found, reverse=True):
            for j in reversed(found[m]):
                if len(starts) < case["branches"] and all(line[j + 1] != line[i + 1] for i in starts):
                    starts.append(j)
        row, up = [line[-1]], [-1]
        for j in starts:
            for k, x in enumerate(line[j + 1 : j + 1 + case["depth"]]):
                up.append(0 if k == 0 else len(row) - 1)
                row.append(x)
        counts.append(len(row))
        tokens.append(row + [-1] * (width - len(row)))
        parents.append(up + [-1] * (width - len(up)))
    dev = s["history"].device
    return {"tokens": _ints(dev, tokens), "parents": _ints(dev, parents), "counts": _ints(dev, counts)}
