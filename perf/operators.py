"""The operators of the 4-bit cache, as cases that can be timed and checked.

Four operators work on one pool of pages: `store` writes rows of keys and values into it in 4 bits, `attend`
is causal attention over it (decoded tokens, and portions of prompts packed one behind the other), `weights`
is attention that also adds to every cached row the weight which the step's queries gave it, and `evict`
keeps of every head's rows those with the most weight and moves them to the front of the request's pages.

The pool is a uint8 tensor [pages, kv heads, page size / 16, 18 d].  The last dimension is the record of 16
tokens of one head: the codes of 16 key rows (d/2 bytes each, channel 2i in the low half of byte i), their
scales (d/16 bytes each), and the same of the values.  A value is (code - 8) times its group's scale; a group is
16 channels of a row, its scale a byte with 5 bits of exponent and 3 of mantissa (the upper bits of a positive half).
"""

from __future__ import annotations

import math
import random
from typing import Any, Optional

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
BLOCK = 16  # tokens of a record, and channels of a group
NEVER = -1e30  # a score that is masked


# ---------------------------------------------------------------------------
# the cases


def _case(name: Optional[str], op: str, *, seqs: int, context: int, query: int = 1, heads: int = 32, kv_heads: int = 8, dim: int = 128,
          page: int = 16, dtype: str = "bfloat16", ragged: bool = False, window: int = 0, sinks: bool = False, budget: int = 0,
          recent: int = 0, first: int = 0) -> dict[str, Any]:
    """`seqs` requests with about `context` cached rows (those of this step among them) that bring `query` tokens
    each; `ragged`: their lengths differ.  store: `seqs` times `query` tokens.  evict: `budget` rows stay, the
    first `first` and the last `recent` among them."""
    c = {"op": op, "seqs": seqs, "context": context, "query": query, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
         "dtype": dtype, "ragged": ragged, "window": window, "sinks": sinks, "budget": budget, "recent": recent, "first": first}
    return c if name is None else {"name": name, **c}


def listed() -> list[dict[str, Any]]:
    return [
        # the rows of a decode step of eight requests: launches count
        _case("store step of 8", "store", seqs=8, context=1024),
        # a full step of prompt tokens
        _case("store prompt 8192", "store", seqs=2, context=4096, query=4096, ragged=True),
        # one user of the smallest preset
        _case("decode 1 at 500", "attend", seqs=1, context=517, heads=16),
        # the usual serving step: many requests of different lengths
        _case("decode 32 at 4096", "attend", seqs=32, context=4096, ragged=True),
        # long documents, where a 4-bit cache is wanted most; pages of another size
        _case("decode 4 at 60000", "attend", seqs=4, context=60000, page=64),
        # a layer with a window and learned sinks, true float32, heads of 64
        _case("decode window float32", "attend", seqs=12, context=3000, heads=64, dim=64, dtype="float32", ragged=True, window=1024, sinks=True),
        # a whole prompt of a model with five query heads per key head
        _case("prompt 2048", "attend", seqs=1, context=2048, query=2048, heads=40),
        # portions of prompts of different lengths, packed, some with rows from earlier steps
        _case("portions 6 ragged", "attend", seqs=6, context=1500, query=301, ragged=True, page=64),
        # decode steps that keep track of the weights
        _case("weights decode 16", "weights", seqs=16, context=4096, ragged=True),
        # the last part of a prompt, after which the first eviction may follow
        _case("weights portion 512", "weights", seqs=1, context=2040, query=512, sinks=True),
        # one request over its budget
        _case("evict 1 to 512", "evict", seqs=1, context=700, budget=512, recent=64, first=4),
        # a batch at once, long caches cut by half
        _case("evict 16 to 4096", "evict", seqs=16, context=8190, budget=4096, recent=256, first=4, ragged=True, page=64),
    ]


def _spread(rng: random.Random, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng: random.Random) -> dict[str, Any]:
    most = [work(c) for c in listed()]
    while True:  # one that costs no more than the largest of its kind
        c = _any(rng)
        w = work(c)
        if all(w[k] <= max(m[k] for m in most) for k in w):
            return c


def _any(rng: random.Random) -> dict[str, Any]:
    op = rng.choice(["store", "attend", "attend", "prompt", "weights", "evict"])
    kv_heads = rng.choice([1, 2, 4, 8, 8])
    dim = rng.choice([64, 128, 128, 128, 256])
    heads = kv_heads * rng.choice([1, 2, 4, 4, 5, 7, 8, 16])
    shape: dict[str, Any] = {"heads": heads, "kv_heads": kv_heads, "dim": dim, "page": rng.choice([16, 16, 32, 64, 128]),
                             "dtype": rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"]), "ragged": rng.random() < 0.6}
    if op == "store":
        tokens = _spread(rng, 1, 8000)
        seqs = rng.randint(1, min(tokens, 16))
        return _case(None, op, seqs=seqs, context=tokens // seqs + rng.randint(0, 500), query=max(1, tokens // seqs), **shape)
    if op == "evict":
        seqs, context = _spread(rng, 1, 32), _spread(rng, 40, 8192)
        budget = rng.randint(context // 3, context - 1)
        recent = rng.randint(0, budget // 2)
        return _case(None, op, seqs=seqs, context=context, budget=budget, recent=recent, first=rng.randint(0, min(8, budget - recent)), **shape)
    if op == "prompt" or (op == "weights" and rng.random() < 0.4):
        seqs = _spread(rng, 1, 12)
        query = _spread(rng, 2, 2048 if seqs == 1 else 512)
        context = query + rng.choice([0, _spread(rng, 1, 2000)])
        return _case(None, "attend" if op == "prompt" else op, seqs=seqs, context=context, query=query, sinks=rng.random() < 0.3,
                     window=_spread(rng, 16, 1024) if rng.random() < 0.3 else 0, **shape)
    seqs = _spread(rng, 1, 128)
    context = _spread(rng, 1, min(60000, 240000 // seqs))
    return _case(None, op, seqs=seqs, context=context, query=rng.choice([1, 1, 1, min(context, 2), min(context, 5)]),
                 sinks=rng.random() < 0.3, window=_spread(rng, 16, 4096) if rng.random() < 0.3 else 0, **shape)


def _lengths(case: dict[str, Any]) -> list[tuple[int, int]]:
    """(cached rows, tokens of this step) of every request; the same for every seed."""
    rng = random.Random("%(seqs)d %(context)d %(query)d %(kv_heads)d" % case)
    out = []
    for _ in range(case["seqs"]):
        n, t = case["context"], case["query"]
        if case["ragged"]:
            n = max(1, round(n * rng.uniform(0.3, 1.0)))
            t = 1 if t == 1 else max(1, min(n, round(t * rng.uniform(0.3, 1.0))))
        out.append((max(n, t), t))
    return out


def _visible(case: dict[str, Any]) -> tuple[int, int]:
    """(rows that some query sees, pairs of a query and a row it sees), over all requests, for one head."""
    rows = pairs = 0
    w = case["window"]
    for n, t in _lengths(case):
        rows += n if not w else min(n, w + t - 1)
        if not w:
            pairs += t * (n - t) + t * (t + 1) // 2
        else:
            pairs += sum(min(w, n - t + i + 1) for i in range(t))
    return rows, pairs


def work(case: dict[str, Any]) -> dict[str, float]:
    item, nq, nkv, d = DTYPES[case["dtype"]].itemsize, case["heads"], case["kv_heads"], case["dim"]
    row = nkv * d * 9 / 8  # bytes of one cached row, keys and values
    tokens = sum(t for _, t in _lengths(case))
    if case["op"] == "store":
        return {"bytes": tokens * (2 * nkv * d * item + row + 2 * nkv * d * 2 + 4), "flops": 0}
    if case["op"] == "evict":
        rows = sum(n for n, _ in _lengths(case))
        kept = sum(min(n, case["budget"]) for n, _ in _lengths(case))
        return {"bytes": rows * nkv * 8 + kept * (2 * row + 2 * nkv * d * 2), "flops": 0}
    rows, pairs = _visible(case)
    bytes_ = rows * row + 2 * tokens * nq * d * item
    if case["op"] == "weights":
        bytes_ += rows * nkv * 8
    return {"bytes": bytes_, "flops": 4.0 * pairs * nq * d}


# ---------------------------------------------------------------------------
# rows in 4 bits, in elementary operations


def _scale_of(amax: torch.Tensor) -> torch.Tensor:
    """amax / 7 in 32 bits, rounded to three bits of mantissa (ties to even), subnormal below 2^-14, at most 8192."""
    t = amax / torch.full_like(amax, 7)  # (a number as divisor may become a product with its rounded inverse)
    exponent = torch.frexp(t)[1].int() - 1
    step = (exponent.clamp(min=-14) + 124 << 23).view(torch.float32)  # 2^(exponent - 3)
    return (torch.round(t / step) * step).clamp(max=8192.0)


def _quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [..., d] -> codes [..., d] (1 to 15, 8 is zero) and scales [..., d/16], both float32."""
    g = x.float().unflatten(-1, (-1, BLOCK))
    s = _scale_of(g.abs().amax(-1))
    c = torch.where(s[..., None] > 0, torch.round(g / torch.where(s > 0, s, 1.0)[..., None]), 0.0).clamp(-7, 7)
    return c.flatten(-2) + 8, s


def _bytes_of(x: torch.Tensor) -> torch.Tensor:
    """x [..., 16 tokens, d] -> the record's half [..., 9 d]: codes, then scales."""
    c, s = _quantise(x)
    c = c.to(torch.uint8).unflatten(-1, (-1, 2))
    c = c[..., 0] | (c[..., 1] << 4)
    s = (s.half().view(torch.int16) >> 7).to(torch.uint8)
    return torch.cat([c.flatten(-2), s.flatten(-2)], -1)


def _values_of(half: torch.Tensor, d: int) -> torch.Tensor:
    """A record's half [..., 9 d] -> float32 values [..., 16, d]."""
    c, s = half[..., : 8 * d].unflatten(-1, (BLOCK, d // 2)), half[..., 8 * d :].unflatten(-1, (BLOCK, d // BLOCK))
    c = torch.stack([c & 15, c >> 4], -1).flatten(-2).float() - 8
    s = (s.to(torch.int16) << 7).view(torch.float16).float()
    return (c.unflatten(-1, (-1, BLOCK)) * s[..., None]).flatten(-2)


def _rows_of(pool: torch.Tensor, table: torch.Tensor, d: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values [B, kv heads, rows, d] in float32 of the pages that `table` [B, pages] names."""
    r = pool[table.clamp(min=0).long()].transpose(1, 2).flatten(2, 3)  # [B, nkv, blocks, 18 d]
    return _values_of(r[..., : 9 * d], d).flatten(2, 3), _values_of(r[..., 9 * d :], d).flatten(2, 3)


# ---------------------------------------------------------------------------
# what a program has in hand


def prepare(case: dict[str, Any], seed: int) -> dict[str, Any]:
    g = torch.Generator("cuda").manual_seed(seed)
    dev, dtype = torch.device("cuda"), DTYPES[case["dtype"]]
    nq, nkv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    lens = _lengths(case)
    B, per = len(lens), [-(-n // page) for n, _ in lens]
    num_pages = sum(per) + 3  # a few pages belong to nobody
    order = torch.randperm(num_pages, generator=g, device=dev).int()
    table = torch.full((B, max(per)), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, p in enumerate(per):
        table[b, :p] = order[at : at + p]
        at += p
    pool = torch.zeros((num_pages, nkv, page // BLOCK, 18 * d), dtype=torch.uint8, device=dev)
    tokens = [t for _, t in lens]
    cu = torch.tensor([sum(tokens[:b]) for b in range(B + 1)], dtype=torch.int32, device=dev)
    T = sum(tokens)
    s = {"case": dict(case), "pool": pool, "table": table, "cu": cu, "tokens": T, "max_query": max(tokens),
         "context_lens": torch.tensor([n for n, _ in lens], dtype=torch.int32, device=dev), "max_context": max(n for n, _ in lens)}
    # channels of keys differ in size, as learned norms and projections make them
    width = torch.exp(0.5 * torch.randn((nkv, 1, d), generator=g, device=dev))

    def places(first: int, n: int, b: int) -> torch.Tensor:
        i = torch.arange(first, first + n, device=dev)
        return (table[b, i // page] * page + i % page).int()

    if case["op"] == "store":
        qkv = torch.randn((T, nq + 2 * nkv, d), generator=g, device=dev)
        qkv[:, nq : nq + nkv] *= width[:, 0]
        s["qkv"] = qkv.to(dtype)  # keys and values are read where the projection left them
        s["slots"] = torch.cat([places(n - t, t, b) for b, (n, t) in enumerate(lens)])
        return s
    aimed = []
    for b, (n, t) in enumerate(lens):
        rows = -(-n // page) * page
        k = torch.randn((nkv, rows, d), generator=g, device=dev) * width
        v = torch.randn((nkv, rows, d), generator=g, device=dev)
        halves = [_bytes_of(x.unflatten(1, (-1, BLOCK))) for x in (k, v)]  # [nkv, blocks, 9 d]
        pool[table[b, : per[b]].long()] = torch.cat(halves, -1).unflatten(1, (-1, page // BLOCK)).transpose(0, 1)
        # every query looks for a few rows among those before it
        i = (torch.rand((nkv, t), generator=g, device=dev) * (n - t + 1)).long()
        aimed.append(torch.gather(k, 1, i[..., None].expand(-1, -1, d)).transpose(0, 1))
    sums = torch.rand((num_pages, nkv, page), generator=g, device=dev)
    s["sums"] = sums * sums * sums * 4  # weight gathered so far: much on few rows
    if case["op"] == "evict":
        s["kept_slots"] = torch.full((B, case["budget"]), -1, dtype=torch.int32, device=dev)
        for b, (n, _) in enumerate(lens):
            keep = min(n, case["budget"])
            s["kept_slots"][b, :keep] = places(0, keep, b)
        return s
    look = torch.cat(aimed).repeat_interleave(nq // nkv, 1) / width.repeat_interleave(nq // nkv, 0)[:, 0] ** 2
    q = 0.7 * torch.randn((T, nq, d), generator=g, device=dev) / width.repeat_interleave(nq // nkv, 0)[:, 0] + 0.4 * look
    s["q"] = q.to(dtype).flatten(1)
    s["head_sinks"] = torch.randn(nq, generator=g, device=dev) if case["sinks"] else None
    return s


# ---------------------------------------------------------------------------
# one pass


def run(s: dict[str, Any]) -> dict[str, torch.Tensor]:
    op = s["case"]["op"]
    if own:
        return {"store": _own_store, "attend": _own_attend, "weights": _own_attend, "evict": _own_evict}[op](s)
    return {"store": _plain_store, "attend": _plain_attend, "weights": _plain_attend, "evict": _plain_evict}[op](s)


def _own_store(s):
    from tokensprint_b200 import ops

    c, T = s["case"], s["tokens"]
    nq, nkv, d = c["heads"], c["kv_heads"], c["dim"]
    ops.kv4_store(s["qkv"][:, nq : nq + nkv], s["qkv"][:, nq + nkv :], s["pool"], s["slots"])
    k, v = (torch.empty((T, nkv, d), device=s["pool"].device, dtype=torch.bfloat16) for _ in range(2))
    ops.kv4_load(s["pool"], s["slots"], k, v)
    return {"keys": k, "values": v}


def _own_attend(s):
    from tokensprint_b200 import ops

    c, q = s["case"], s["q"]
    out = torch.empty_like(q)
    sizes = (s["cu"], s["context_lens"], s["table"], c["seqs"], s["max_query"], s["max_context"], c["heads"], c["kv_heads"], c["dim"],
             c["dim"] ** -0.5)
    if c["op"] == "attend":
        ops.attention_kv4(q, s["pool"], out, *sizes, window=c["window"], head_sinks=s["head_sinks"])
        return {"out": out}
    lse = torch.empty((s["tokens"], c["heads"]), device=q.device, dtype=torch.float32)
    ops.attention_kv4(q, s["pool"], out, *sizes, window=c["window"], head_sinks=s["head_sinks"], lse=lse)
    ops.attention_kv4_weights(q, s["pool"], lse, s["sums"], *sizes, window=c["window"])
    return {"out": out, "sums": s["sums"]}


def _own_evict(s):
    from tokensprint_b200 import ops

    c = s["case"]
    lens = torch.empty_like(s["context_lens"])
    ops.kv4_evict(s["pool"], s["sums"], s["table"], s["context_lens"], lens, c["seqs"], s["max_context"], c["budget"], c["recent"], c["first"])
    k, v = (torch.empty((s["kept_slots"].numel(), c["kv_heads"], c["dim"]), device=lens.device, dtype=torch.bfloat16) for _ in range(2))
    ops.kv4_load(s["pool"], s["kept_slots"].view(-1), k, v)
    return {"keys": k, "values": v, "sums": s["sums"], "lens": lens}


def _record_rows(pool, slots, page):
    """Where the rows of flat `slots` lie: page, block of 16 tokens, token of the block."""
    slots = slots.long()
    return slots // page, slots % page // BLOCK, slots % BLOCK


def _plain_load(s, slots):
    c, pool, d = s["case"], s["pool"], s["case"]["dim"]
    p, blk, t = _record_rows(pool, slots.clamp(min=0), c["page"])
    r = pool[p, :, blk]  # [N, nkv, 18 d]
    i = torch.arange(r.shape[0], device=r.device)
    there = (slots >= 0).view(-1, 1, 1)
    return [torch.where(there, _values_of(r[..., o : o + 9 * d], d)[i, :, t], 0.0).to(torch.bfloat16) for o in (0, 9 * d)]


def _plain_store(s):
    c, pool = s["case"], s["pool"]
    nq, nkv, d = c["heads"], c["kv_heads"], c["dim"]
    p, blk, t = _record_rows(pool, s["slots"], c["page"])
    heads = torch.arange(nkv, device=pool.device).view(1, -1, 1)
    p, blk, t = p.view(-1, 1, 1), blk.view(-1, 1, 1), t.view(-1, 1, 1)

    def put(x, offset):
        codes, scales = _bytes_of(x[:, :, None]).split([d // 2, d // BLOCK], -1)
        pool[p, heads, blk, offset + t * (d // 2) + torch.arange(d // 2, device=pool.device)] = codes
        pool[p, heads, blk, offset + 8 * d + t * (d // BLOCK) + torch.arange(d // BLOCK, device=pool.device)] = scales

    put(s["qkv"][:, nq : nq + nkv], 0)
    put(s["qkv"][:, nq + nkv :], 9 * d)
    k, v = _plain_load(s, s["slots"])
    return {"keys": k, "values": v}


def _padded(s):
    """Where the packed tokens stand in [B, longest portion], and each one's number among its request's rows (-1: none)."""
    t = torch.arange(s["max_query"], device=s["cu"].device)
    count = (s["cu"][1:] - s["cu"][:-1])[:, None]
    there = t < count
    return there, (s["cu"][:-1, None] + t).clamp(max=s["tokens"] - 1).long(), s["context_lens"][:, None] - count + t


def _plain_attend(s):
    c, q = s["case"], s["q"]
    B, nq, nkv, d = c["seqs"], c["heads"], c["kv_heads"], c["dim"]
    there, token, number = _padded(s)
    keys, values = _rows_of(s["pool"], s["table"], d)  # [B, nkv, n, d]
    x = q.float().view(-1, nkv, nq // nkv, d)[token].permute(0, 2, 3, 1, 4)  # [B, nkv, G, t, d]
    scores = (x.flatten(2, 3) @ keys.transpose(-1, -2)).unflatten(2, (nq // nkv, -1)) * d**-0.5
    j = torch.arange(keys.shape[2], device=q.device)
    seen = there[..., None] & (j <= number[..., None])
    if c["window"]:
        seen &= j > number[..., None] - c["window"]
    seen = seen[:, None, None]  # [B, 1, 1, t, n]
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
    out = (p.flatten(2, 3) @ values).unflatten(2, (nq // nkv, -1)).permute(0, 3, 1, 2, 4)  # [B, t, nkv, G, d]
    out = out[there].flatten(1).to(q.dtype)
    if c["op"] == "attend":
        return {"out": out}
    w = p.sum((2, 3))  # [B, nkv, n]
    held = s["table"] >= 0
    s["sums"][s["table"][held].long()] += w.unflatten(2, (-1, c["page"])).transpose(1, 2)[held]
    return {"out": out, "sums": s["sums"]}


def _plain_evict(s):
    c, pool, table, lens = s["case"], s["pool"], s["table"], s["context_lens"]
    page, d, budget = c["page"], c["dim"], c["budget"]
    sums = s["sums"][table.clamp(min=0).long()].transpose(1, 2).flatten(2)  # [B, nkv, n]
    i = torch.arange(sums.shape[2], device=sums.device)
    n = lens[:, None, None]
    rank = torch.where((i < c["first"]) | (i >= n - c["recent"]), math.inf, sums)  # always kept
    rank = torch.where(i < n, rank, -math.inf)
    best = torch.sort(rank, dim=-1, descending=True, stable=True)[1][..., :budget]
    new = lens.clamp(max=budget)
    kept = torch.arange(best.shape[2], device=sums.device) < new[:, None, None]
    best = torch.sort(torch.where(kept, best, sums.shape[2]), -1)[0].clamp(max=sums.shape[2] - 1)  # in their order
    # a request within its budget keeps all, in order; rows behind the kept ones are left as they are
    r = pool[table.clamp(min=0).long()].transpose(1, 2).flatten(2, 3)  # [B, nkv, blocks, 18 d]
    parts = r.split([8 * d, d, 8 * d, d], -1)
    moved = []
    for x in parts:
        rows = x.unflatten(-1, (BLOCK, -1)).flatten(2, 3)  # [B, nkv, n, bytes]
        fresh = rows.clone()
        taken = torch.gather(rows, 2, best[..., None].expand(-1, -1, -1, rows.shape[-1]))
        fresh[:, :, : best.shape[2]] = torch.where(kept[..., None], taken, rows[:, :, : best.shape[2]])
        moved.append(fresh.unflatten(2, (-1, BLOCK)).flatten(3))
    held = table >= 0
    pool[table[held].long()] = torch.cat(moved, -1).unflatten(2, (-1, page // BLOCK)).transpose(1, 2)[held]
    fresh = torch.where(i < n, 0.0, sums)
    fresh[..., : best.shape[2]] = torch.where(kept, torch.gather(sums, 2, best), fresh[..., : best.shape[2]])
    s["sums"][table[held].long()] = fresh.unflatten(2, (-1, page)).transpose(1, 2)[held]
    k, v = _plain_load(s, s["kept_slots"].view(-1))
    return {"keys": k, "values": v, "sums": s["sums"], "lens": new}


# ---------------------------------------------------------------------------
# the same from the definition, in 64 bits


def _exact_rows(pool: torch.Tensor, pages: torch.Tensor, head: int, count: int, d: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values [count, d] of one head from its pages."""
    r = pool[pages.long(), head].reshape(-1, 18, d).long()
    out = []
    for o in (0, 9):
        code = r[:, o : o + 8].reshape(-1, d // 2)
        code = torch.stack((code % 16, code // 16), 2).reshape(-1, d // 16, 16)
        byte = r[:, o + 8].reshape(-1, d // 16, 1)
        e, m = byte // 8, byte % 8
        size = torch.where(e > 0, (8 + m).double() * 2.0 ** (e - 18).double(), m.double() * 2.0**-17)
        out.append(((code - 8) * size).reshape(-1, d)[:count])
    return out[0], out[1]


def _exact_held(x: torch.Tensor) -> torch.Tensor:
    """The values that rows [..., d] have in 4 bits."""
    x = x.double().reshape(*x.shape[:-1], -1, 16)
    want = x.abs().amax(-1, keepdim=True) / 7
    grid = torch.tensor([m * 2.0**-17 for m in range(8)] + [(8 + m) * 2.0 ** (e - 18) for e in range(1, 29) for m in range(8)], dtype=torch.float64,
                        device=x.device)
    grid = grid[grid <= 8192]
    up = torch.searchsorted(grid, want.reshape(-1)).clamp(max=len(grid) - 1)
    low, high, want = grid[(up - 1).clamp(min=0)], grid[up], want.reshape(-1)
    nearer_low = (want - low < high - want) | ((want - low == high - want) & ((up - 1) % 2 == 0))
    size = torch.where(nearer_low, low, high).reshape(*x.shape[:-1], 1)
    code = torch.round(x / size.clamp(min=2.0**-17)).clamp(-7, 7)
    return (code * size).flatten(-2)


def exact(case: dict[str, Any], seed: int):
    s = prepare(case, seed)
    nq, nkv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    lens = _lengths(case)
    dev = s["pool"].device
    if case["op"] == "store":
        return {"keys": _exact_held(s["qkv"][:, nq : nq + nkv]), "values": _exact_held(s["qkv"][:, nq + nkv :])}
    if case["op"] == "evict":
        sums = s["sums"].double()
        kept = [torch.zeros((len(lens), case["budget"], nkv, d), dtype=torch.float64, device=dev) for _ in range(2)]
        for b, (n, _) in enumerate(lens):
            pages = s["table"][b, : -(-n // page)].long()
            i = torch.arange(n, device=dev)
            for h in range(nkv):
                w = s["sums"][pages, h].reshape(-1)[:n].double()
                if n > case["budget"]:
                    middle = i[case["first"] : n - case["recent"]]
                    by_weight = sorted(zip((-w[middle]).tolist(), middle.tolist()))[: case["budget"] - case["first"] - case["recent"]]
                    i_kept = torch.tensor(sorted([*range(case["first"]), *range(n - case["recent"], n), *(j for _, j in by_weight)]), device=dev)
                else:
                    i_kept = i
                for x, rows in zip(kept, _exact_rows(s["pool"], pages, h, n, d)):
                    x[b, : len(i_kept), h] = rows[i_kept]
                fresh = torch.zeros(n, dtype=torch.float64, device=dev)
                fresh[: len(i_kept)] = w[i_kept]
                sums[pages[i // page], h, i % page] = fresh
        return {"keys": kept[0].flatten(0, 1), "values": kept[1].flatten(0, 1), "sums": sums, "lens": None}
    q = s["q"].double().view(-1, nq, d)
    out, sums, G = torch.empty_like(q), s["sums"].double(), nq // nkv
    at = 0
    for b, (n, t) in enumerate(lens):
        pages = s["table"][b, : -(-n // page)].long()
        number = torch.arange(n - t, n, device=dev)[:, None]
        j = torch.arange(n, device=dev)[None]
        hidden = j > number
        if case["window"]:
            hidden = hidden | (number - j >= case["window"])
        for h in range(nkv):
            k, v = _exact_rows(s["pool"], pages, h, n, d)
            for i in range(h * G, h * G + G):
                z = (q[at : at + t, i] @ k.T / math.sqrt(d)).masked_fill(hidden, -math.inf)
                if s["head_sinks"] is not None:
                    z = torch.cat((z, s["head_sinks"][i].double().expand(t, 1)), 1)
                p = torch.softmax(z, 1)[:, :n]
                out[at : at + t, i] = p @ v
                sums[pages[j[0] // page], h, j[0] % page] += p.sum(0)
        at += t
    return {"out": out.flatten(1)} if case["op"] == "attend" else {"out": out.flatten(1), "sums": sums}
