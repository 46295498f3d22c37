"""The 4-bit cache: store, load, attention, the weights of cached rows and eviction, against plain float64."""

import math
import random

import pytest
import torch

from tests.plain import kv4_plain as plain

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from tokensprint_b200 import ops

DEV = "cuda"


def rows_like(shape, gen, dtype=torch.float32):
    """Rows whose groups differ widely in size, some of them all zero."""
    x = torch.randn(shape, generator=gen) * torch.exp(1.5 * torch.randn((*shape[:-1], shape[-1] // 16, 1), generator=gen)).expand(
        *shape[:-1], shape[-1] // 16, 16).flatten(-2)
    x[torch.rand(shape[:-1], generator=gen) < 0.02] = 0
    return x.to(dtype)


def page_table(lens, page, gen, extra=3, base=0):
    per = [-(-n // page) for n, _ in lens]
    order = (torch.randperm(sum(per) + extra, generator=gen) + base).int()
    table = torch.full((len(lens), max([1, *per])), -1, dtype=torch.int32)
    at = 0
    for b, p in enumerate(per):
        table[b, :p] = order[at : at + p]
        at += p
    return table, sum(per) + extra + base


def filled(lens, nkv, d, page, gen, base=0, spoil=True):
    """A pool whose requests hold random rows; every byte that belongs to no row is 0xff (a scale that is no number)."""
    table, pages = page_table(lens, page, gen, base=base)
    pool = torch.full(ops.kv4_pool_shape(pages, page, nkv, d), 0xFF if spoil else 0, dtype=torch.uint8, device=DEV)
    keys, values = [], []
    for b, (n, _) in enumerate(lens):
        kept = [[], []]
        for h in range(nkv):
            m = -(-n // page) * page
            k, v = torch.randn((m, d), generator=gen), torch.randn((m, d), generator=gen)
            rec = plain.pack(k, v) if m else torch.zeros((0, 18 * d), dtype=torch.uint8)
            for i, x in enumerate(plain.unpack(rec, d)):
                kept[i].append(x[:n].to(DEV))
            if spoil and m > n:  # rows of the last page that were never stored
                for row in range(n, m):
                    r = rec[row // 16]
                    for o in (0, 9 * d):
                        r[o + row % 16 * (d // 2) : o + (row % 16 + 1) * (d // 2)] = 0xFF
                        r[o + 8 * d + row % 16 * (d // 16) : o + 8 * d + (row % 16 + 1) * (d // 16)] = 0xFF
            pool[table[b, : m // page].long().to(DEV), h] = rec.to(DEV).view(-1, page // 16, 18 * d)
        keys.append(torch.stack(kept[0]))
        values.append(torch.stack(kept[1]))
    return pool, table.to(DEV), keys, values


def batch(lens):
    cu = torch.tensor([sum(t for _, t in lens[:b]) for b in range(len(lens) + 1)], dtype=torch.int32, device=DEV)
    return cu, torch.tensor([n for n, _ in lens], dtype=torch.int32, device=DEV)


# ---------------------------------------------------------------------------
# rows in and out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nkv,d,page,tokens", [(8, 128, 16, 1), (1, 64, 16, 7), (3, 128, 48, 65), (2, 256, 128, 300), (8, 64, 32, 33)])
def test_store_writes_the_nearest_codes(nkv, d, page, tokens, dtype):
    """Codes and scales are those of the formula, bit by bit: every step of it is exact or correctly rounded."""
    gen = torch.Generator().manual_seed(tokens + d)
    pages = -(-tokens // page) + 2
    k, v = rows_like((tokens, nkv, d), gen, dtype), rows_like((tokens, nkv, d), gen, dtype)
    pool = torch.zeros(ops.kv4_pool_shape(pages, page, nkv, d), dtype=torch.uint8, device=DEV)
    slots = torch.randperm(pages * page, generator=gen)[:tokens].int()
    if tokens > 4:
        slots[3] = -1
    ops.kv4_store(k.to(DEV), v.to(DEV), pool, slots.to(DEV))
    want = torch.zeros_like(pool, device="cpu")
    for i, slot in enumerate(slots.tolist()):
        if slot < 0:
            continue
        for h in range(nkv):
            r = want[slot // page, h, slot % page // 16]
            for x, o in ((k[i, h], 0), (v[i, h], 9 * d)):
                code, byte = plain.quantise(x)
                t = slot % 16
                r[o + t * (d // 2) : o + (t + 1) * (d // 2)] = (code[0::2] + 16 * code[1::2]).to(torch.uint8)
                r[o + 8 * d + t * (d // 16) : o + 8 * d + (t + 1) * (d // 16)] = byte.to(torch.uint8)
    assert torch.equal(pool.cpu(), want)
    for out_dtype in (torch.float32, torch.bfloat16):  # the values are exact in both
        kk, vv = (torch.empty((tokens, nkv, d), device=DEV, dtype=out_dtype) for _ in range(2))
        ops.kv4_load(pool, slots.to(DEV), kk, vv)
        for x, got in ((k, kk), (v, vv)):
            held = plain.values_of(*plain.quantise(x))
            held[slots < 0] = 0
            assert torch.equal(got.cpu().double(), held)


def test_store_of_hard_values():
    """Zeros, the smallest and largest scales, ties of scale and code, infinities and NaN."""
    d = 64
    grid = plain.scale_grid()
    rows = [torch.zeros(d), torch.full((d,), 2.0**-17 * 3.4), torch.full((d,), 2.0**-22), torch.full((d,), 1e30), torch.full((d,), -57344.0)]
    ties = torch.zeros(d)
    ties[0], ties[1:8], ties[16], ties[32], ties[33] = 7.0, torch.arange(7) + 0.5, 7 * (9 + 0.5), 7 * (8 + 0.5) / 8, -3.3
    rows.append(ties)
    rows += [torch.linspace(-1, 1, d) * float(s) for s in grid[::9]]
    bad = torch.linspace(-2, 2, d)
    bad[3], bad[20], bad[40] = math.nan, math.inf, -math.inf
    rows += [bad, torch.full((d,), math.nan)]
    x = torch.stack(rows)[:, None]
    pool = torch.zeros(ops.kv4_pool_shape(len(rows) // 16 + 1, 16, 1, d), dtype=torch.uint8, device=DEV)
    slots = torch.arange(len(rows), dtype=torch.int32, device=DEV)
    ops.kv4_store(x.to(DEV), (-x).to(DEV), pool, slots)
    k, v = (torch.empty((len(rows), 1, d), device=DEV) for _ in range(2))
    ops.kv4_load(pool, slots, k, v)
    assert torch.isfinite(k).all() and torch.isfinite(v).all()
    assert torch.equal(k.cpu().double(), plain.values_of(*plain.quantise(x)))
    assert torch.equal(v.cpu().double(), plain.values_of(*plain.quantise(-x)))


def test_store_reads_strided_rows_and_clears_sums():
    gen = torch.Generator().manual_seed(5)
    T, nq, nkv, d, page = 9, 3, 2, 128, 32
    qkv = torch.randn((T, nq + 2 * nkv, d), generator=gen).to(torch.bfloat16).to(DEV)
    pool, dense = (torch.zeros(ops.kv4_pool_shape(2, page, nkv, d), dtype=torch.uint8, device=DEV) for _ in range(2))
    sums = torch.ones((2, nkv, page), device=DEV)
    slots = torch.tensor([40, 41, 3, -1, 63, 0, 17, 5, 999], dtype=torch.int32, device=DEV)  # (one outside the pool)
    ops.kv4_store(qkv[:, nq : nq + nkv], qkv[:, nq + nkv :], pool, slots, sums)
    ops.kv4_store(qkv[:, nq : nq + nkv].contiguous(), qkv[:, nq + nkv :].contiguous(), dense, slots)
    assert torch.equal(pool, dense)
    want = torch.ones((2, nkv, page))
    for s in slots.tolist():
        if 0 <= s < 2 * page:
            want[s // page, :, s % page] = 0
    assert torch.equal(sums.cpu(), want)


# ---------------------------------------------------------------------------
# attention and weights


def check_attention(lens, nq, nkv, d, page, dtype, window=0, sinks=False, seed=0, base=0, max_extra=0):
    """Bounds: scores are sums of D exact products in 32 bits (float32 queries: of three parts of 8 bits): off by at most
    2^-18 of scale sum |q||k|; a weight is off by 2^-10 at most (float32: 2^-20), in portions that run on tcgen05 by 2^-8 (it is
    rounded to bfloat16 there); the result is rounded to its type (2^-8, 2^-22)."""
    gen = torch.Generator().manual_seed(seed + 7919 * d + nq)
    pool, table, keys, values = filled(lens, nkv, d, page, gen, base=base)
    T = sum(t for _, t in lens)
    q = (torch.randn((T, nq, d), generator=gen) * torch.exp(torch.randn((T, nq, 1), generator=gen))).to(dtype).to(DEV)
    sink = torch.randn(nq, generator=gen).to(DEV) if sinks else None
    cu, context = batch(lens)
    scale = d**-0.5
    sizes = (cu, context, table, len(lens), max(t for _, t in lens) + max_extra, max(n for n, _ in lens) + max_extra, nq, nkv, d, scale)
    out = torch.full((T, nq * d), 7.0, dtype=dtype, device=DEV)
    lse = torch.full((T, nq), 7.0, device=DEV)
    sums = torch.rand((pool.shape[0], nkv, page), generator=gen).to(DEV)
    before = sums.clone()
    ops.attention_kv4(q.flatten(1), pool, out, *sizes, window=window, head_sinks=sink, lse=lse)
    ops.attention_kv4_weights(q.flatten(1), pool, lse, sums, *sizes, window=window)
    want, want_lse, weights, spread, reach = plain.attention(q.double(), keys, values, lens, window, sink.double() if sinks else None, scale)
    exact = dtype == torch.float32
    slack = 2.0**-18 * (reach + 1)
    got = out.double().view(T, nq, d)
    rounded = (max(t for _, t in lens) + max_extra) * (nq // nkv) > ops.ATTENTION_KV4_DIRECT_ROWS and d == 128  # on tcgen05
    bound = ((2.0**-20 if exact else 2.0**-8 if rounded else 2.0**-10) + 2 * slack[..., None]) * spread + (2.0**-22 if exact else 2.0**-8) * want.abs() + 1e-30
    assert torch.isfinite(got).all()
    assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse), empty) and (got[empty] == 0).all()
    close = (lse.double() - want_lse).abs() <= slack + 2.0**-20 * (1 + want_lse.abs())
    assert (close | empty).all()
    grown = (sums - before).double()
    for b, (n, _) in enumerate(lens):
        for j in range(0, n, 16):
            m = min(16, n - j)
            place = (table[b, j // page].long(), slice(None), slice(j % page, j % page + m))
            w = weights[b][:, j : j + m]
            limit = 4 * float(slack.max()) * w + 2.0**-20 * (w + before[place].double()) + 1e-12
            assert ((grown[place] - w).abs() <= limit).all()
    # nothing else of the sums changed
    held = torch.zeros_like(sums, dtype=torch.bool)
    for b, (n, _) in enumerate(lens):
        j = torch.arange(n, device=DEV)
        held[table[b, j // page].long(), :, j % page] = True
    assert torch.equal(sums[~held], before[~held])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq,nkv,d,page", [(16, 8, 128, 16), (4, 1, 128, 64), (5, 1, 128, 32), (7, 1, 64, 16), (16, 1, 64, 128), (2, 2, 256, 16),
                                           (12, 1, 256, 48), (24, 1, 128, 16)])
def test_decode_lengths(nq, nkv, d, page, dtype):
    lens = [(n, 1) for n in (1, 2, 15, 16, 17, 31, 64, 127, 128, 129, 300, 1025)]
    check_attention(lens, nq, nkv, d, page, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("window,sinks", [(0, True), (1, False), (16, True), (33, False), (200, True)])
def test_decode_windows_and_sinks(window, sinks, dtype):
    check_attention([(1, 1), (16, 1), (40, 1), (333, 1), (700, 2)], 8, 2, 128, 16, dtype, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens", [[(5, 5), (40, 3), (17, 17), (100, 1)], [(33, 2), (2, 2), (64, 19)], [(130, 130)], [(90, 30), (200, 64)]])
@pytest.mark.parametrize("nq,nkv,d", [(4, 1, 128), (5, 1, 64), (2, 2, 128), (3, 1, 256)])
def test_portions(lens, nq, nkv, d, dtype):
    check_attention(lens, nq, nkv, d, 16, dtype)


@pytest.mark.parametrize("window,sinks", [(1, True), (20, False), (64, True)])
def test_portions_with_windows(window, sinks):
    check_attention([(50, 50), (100, 37), (64, 1), (9, 4)], 6, 2, 128, 32, torch.bfloat16, window=window, sinks=sinks)
    check_attention([(50, 50), (100, 37)], 3, 1, 64, 16, torch.float32, window=window, sinks=sinks)


@pytest.mark.parametrize("sinks", [False, True])
def test_requests_without_tokens_or_rows(sinks):
    """Requests that bring nothing, that hold nothing, and queries that see nothing (more tokens than rows)."""
    check_attention([(0, 0), (20, 1), (0, 1), (7, 0), (3, 5), (0, 0), (64, 2)], 4, 2, 128, 16, torch.bfloat16, sinks=sinks)


def test_bounds_may_exceed_the_lengths():
    check_attention([(70, 1), (300, 1)], 8, 2, 128, 16, torch.bfloat16, max_extra=5000)
    check_attention([(70, 9), (300, 20)], 8, 2, 128, 16, torch.bfloat16, max_extra=300)


def test_long_portion_uses_the_same_numbers():
    check_attention([(700, 512), (300, 260)], 4, 2, 128, 64, torch.bfloat16)


@pytest.mark.parametrize("window,sinks", [(0, False), (0, True), (300, False), (130, True)])
def test_few_rows_over_many_keys(window, sinks):
    """Portions whose keys are cut into runs that are joined afterwards; some requests have fewer runs than others, one has no rows."""
    check_attention([(1700, 30), (260, 40), (0, 0), (1024, 1), (50, 50)], 4, 1, 128, 16, torch.bfloat16, window=window, sinks=sinks)
    check_attention([(900, 150)], 5, 1, 128, 16, torch.bfloat16, window=window, sinks=sinks)


@pytest.mark.parametrize("window", [0, 90])
@pytest.mark.parametrize("tokens,d,dtype", [(20, 128, torch.bfloat16), (50, 128, torch.bfloat16), (12, 128, torch.float32), (33, 64, torch.bfloat16),
                                            (9, 256, torch.bfloat16)])
def test_short_portions_over_many_keys(tokens, d, dtype, window):
    """Many requests with a few tokens each: weights are added up 16 or 32 rows at a time."""
    lens = [(1300, tokens), (700, 3), (tokens, tokens), (1290, 1), (1033, tokens - 1), (0, 0), (64, 5), (1100, 8)]
    check_attention(lens, 16, 8, d, 16, dtype, window=window)


@pytest.mark.parametrize("lens", [[(130, 130)], [(90, 30), (200, 64)], [(50, 50), (100, 37), (64, 1), (9, 4)]])
@pytest.mark.parametrize("window,sinks", [(0, False), (20, True)])
@pytest.mark.parametrize("nq,nkv", [(4, 1), (6, 2), (7, 1)])
def test_small_portions_on_tensor_memory(lens, nq, nkv, window, sinks, monkeypatch):
    """Portions of so little work that the kernel of decoded tokens takes them by itself, sent through the other one."""
    monkeypatch.setattr(ops, "_KV4_DIRECT_PIECES", 0)
    check_attention(lens, nq, nkv, 128, 16, torch.bfloat16, window=window, sinks=sinks)


@pytest.mark.parametrize("lens", [[(n, 1) for n in (600, 3, 1500, 77, 16, 2500, 900)], [(1000, 2)] * 3, [(40, 40), (1, 1), (900, 9)], [(5000, 1)]])
@pytest.mark.parametrize("nq,nkv,dtype", [(8, 2, torch.bfloat16), (16, 2, torch.bfloat16), (24, 2, torch.bfloat16), (8, 1, torch.float32)])
def test_shares_of_ranges(lens, nq, nkv, dtype):
    """Key ranges of one and of many lengths, cut into parts of their own."""
    check_attention(lens, nq, nkv, 128, 16, dtype)
    check_attention(lens, nq, nkv, 64, 16, dtype, window=300)


def test_portions_in_groups(monkeypatch):
    """Requests whose unpacked rows do not fit the workspace at once are taken in groups."""
    monkeypatch.setattr(ops, "ATTENTION_KV4_EXPAND_BYTES", 2 * 128 * 2 * 3 * 128 * 2 * 2)  # two requests of three pages
    check_attention([(300, 40), (129, 128), (17, 17), (384, 70), (200, 1)], 4, 2, 128, 16, torch.bfloat16, sinks=True)


@pytest.mark.parametrize("lens", [[(130, 130)], [(700, 512)], [(900, 40), (200, 200)]])
@pytest.mark.parametrize("sinks", [False, True])
def test_portions_without_denominators(lens, sinks):
    """Nobody asks for the denominators; the first rows see one key, whose zeros stay zeros whatever the masked keys hold.  (2^-13: room
    for exponentials from a cubic, which is not used here.)"""
    nq, nkv, d, page = 4, 1, 128, 16
    gen = torch.Generator().manual_seed(17)
    pool, table, keys, values = filled(lens, nkv, d, page, gen)
    T = sum(t for _, t in lens)
    q = torch.randn((T, nq, d), generator=gen).to(torch.bfloat16).to(DEV)
    sink = torch.randn(nq, generator=gen).to(DEV) if sinks else None
    cu, context = batch(lens)
    out = torch.empty((T, nq * d), dtype=torch.bfloat16, device=DEV)
    ops.attention_kv4(q.flatten(1), pool, out, cu, context, table, len(lens), max(t for _, t in lens), max(n for n, _ in lens), nq, nkv, d, d**-0.5,
                      head_sinks=sink)
    want, _, _, spread, reach = plain.attention(q.double(), keys, values, lens, 0, sink.double() if sinks else None, d**-0.5)
    bound = (2.0**-8 + 2.0**-13 + 2.0**-17 * (reach[..., None] + 1)) * spread + 2.0**-8 * want.abs()
    assert ((out.double().view(T, nq, d) - want).abs() <= bound).all()


def test_offsets_beyond_32_bits():
    """Pages whose records lie more than 4 GB into the pool."""
    page, nkv, d = 64, 2, 128
    base = (1 << 32) // (page * nkv * 18 * d // 16) + 5
    check_attention([(130, 1), (77, 3)], 8, nkv, d, page, torch.bfloat16, base=base)


def test_large_queries_and_nan():
    """A row is scaled before it becomes a half: large and tiny queries keep their precision; a NaN stays in its row."""
    gen = torch.Generator().manual_seed(3)
    lens, nq, nkv, d, page = [(100, 1)], 4, 1, 128, 16
    pool, table, keys, values = filled(lens, nkv, d, page, gen)
    q = torch.randn((1, nq, d), generator=gen)
    q[0, 0] *= 1e6
    q[0, 1] *= 1e-30
    q[0, 2, 5] = math.nan
    q = q.to(torch.bfloat16).to(DEV)
    cu, context = batch(lens)
    out = torch.empty((1, nq * d), dtype=torch.bfloat16, device=DEV)
    ops.attention_kv4(q.flatten(1), pool, out, cu, context, table, 1, 1, 100, nq, nkv, d, 1e-3)
    got = out.view(nq, d).double()
    assert torch.isnan(got[2]).all() and torch.isfinite(got[[0, 1, 3]]).all()
    for h in (0, 1, 3):
        p = torch.softmax(keys[0][0] @ q[0, h].double() * 1e-3, 0)
        assert (got[h] - p @ values[0][0]).abs().max() <= 2.0**-7


def test_streams_and_equal_bits():
    """The same bits twice, and on another stream."""
    gen = torch.Generator().manual_seed(11)
    lens, nq, nkv, d, page = [(900, 1), (37, 1), (2000, 1)], 16, 4, 128, 16
    pool, table, _, _ = filled(lens, nkv, d, page, gen)
    q = torch.randn((3, nq * d), generator=gen).to(torch.bfloat16).to(DEV)
    cu, context = batch(lens)

    def once():
        out, lse = torch.empty_like(q), torch.empty((3, nq), device=DEV)
        sums = torch.zeros((pool.shape[0], nkv, page), device=DEV)
        args = (cu, context, table, 3, 1, 2000, nq, nkv, d, 0.1)
        ops.attention_kv4(q, pool, out, *args, lse=lse)
        ops.attention_kv4_weights(q, pool, lse, sums, *args)
        return out, lse, sums

    first = once()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        second = once()
    side.synchronize()
    third = once()
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)
    assert abs(float(first[2].double().sum()) - 3 * nq) < 1e-3  # every softmax hands out a weight of one


# ---------------------------------------------------------------------------
# eviction


def check_evict(lens, nkv, d, page, budget, recent, first, weights=None, seed=0, repeat=1):
    gen = torch.Generator().manual_seed(seed + 31 * budget)
    pool, table, _, _ = filled([(n, 0) for n in lens], nkv, d, page, gen, spoil=False)
    sums = torch.rand((pool.shape[0], nkv, page), generator=gen).to(DEV) if weights is None else weights((pool.shape[0], nkv, page), gen).to(DEV)
    context = torch.tensor(lens, dtype=torch.int32, device=DEV)
    new = torch.full((len(lens),), -5, dtype=torch.int32, device=DEV)
    want_pool, want_sums = pool.cpu().clone(), sums.cpu().clone()
    ops.kv4_evict(pool, sums, table, context, new, len(lens), max(lens), budget, recent, first)
    assert new.tolist() == [min(n, budget) for n in lens]
    table = table.cpu()

    def row(p, r, h, x):
        """Views of a row's four pieces."""
        rec = p[int(table[r, x // page]), h, x % page // 16]
        t = x % 16
        return [rec[o : o + m] for o, m in ((t * (d // 2), d // 2), (8 * d + t * (d // 16), d // 16), (9 * d + t * (d // 2), d // 2),
                                            (17 * d + t * (d // 16), d // 16))]

    for b, n in enumerate(lens):
        for h in range(nkv):
            w = [float(want_sums[int(table[b, i // page]), h, i % page]) for i in range(n)]
            kept = plain.kept_rows(w, budget, recent, first)
            for to, src in enumerate(kept):  # forward only: what is read has not been overwritten
                for x, y in zip(row(want_pool, b, h, to), row(want_pool, b, h, src)):
                    x.copy_(y.clone())
            fresh = [w[i] for i in kept] + [0.0] * (n - len(kept))
            for i, x in enumerate(fresh):
                want_sums[int(table[b, i // page]), h, i % page] = x
    assert torch.equal(pool.cpu(), want_pool)
    assert torch.equal(sums.cpu().nan_to_num(nan=-1.0), want_sums.nan_to_num(nan=-1.0))


@pytest.mark.parametrize("nkv,d,page", [(2, 128, 16), (1, 64, 64), (3, 256, 32)])
@pytest.mark.parametrize("lens,budget,recent,first", [([1, 5, 300, 64], 64, 16, 4), ([257, 700, 256], 255, 0, 0), ([90, 91], 90, 45, 45),
                                                      ([40], 1, 0, 0), ([40], 1, 1, 0), ([1000, 513], 512, 100, 1)])
def test_evict(nkv, d, page, lens, budget, recent, first):
    check_evict(lens, nkv, d, page, budget, recent, first)


@pytest.mark.parametrize("kind", ["zeros", "few", "signs", "nan"])
def test_evict_ties_and_odd_weights(kind):
    def weights(shape, gen):
        if kind == "zeros":
            return torch.zeros(shape)
        if kind == "few":
            return torch.randint(0, 3, shape, generator=gen).float()
        if kind == "signs":
            return torch.randint(-2, 3, shape, generator=gen).float() * -0.0 + torch.randint(-2, 2, shape, generator=gen).float()
        w = torch.rand(shape, generator=gen)
        w[torch.rand(shape, generator=gen) < 0.05] = math.nan
        w[torch.rand(shape, generator=gen) < 0.05] = math.inf
        return w

    check_evict([600, 333, 129], 2, 128, 16, 128, 10, 3, weights)


def test_attention_after_eviction_is_that_over_the_kept_rows():
    gen = torch.Generator().manual_seed(2)
    lens, nq, nkv, d, page, budget = [(300, 1), (100, 1)], 8, 2, 128, 16, 128
    pool, table, keys, values = filled(lens, nkv, d, page, gen, spoil=False)
    sums = torch.rand((pool.shape[0], nkv, page), generator=gen).to(DEV)
    kept = [[plain.kept_rows([float(sums[table[b, i // page], h, i % page]) for i in range(n)], budget, 20, 4) for h in range(nkv)]
            for b, (n, _) in enumerate(lens)]
    cu, context = batch(lens)
    new = torch.empty_like(context)
    ops.kv4_evict(pool, sums, table, context, new, 2, 300, budget, 20, 4)
    q = torch.randn((2, nq, d), generator=gen).to(torch.bfloat16).to(DEV)
    out = torch.empty((2, nq * d), dtype=torch.bfloat16, device=DEV)
    ops.attention_kv4(q.flatten(1), pool, out, cu, new, table, 2, 1, budget, nq, nkv, d, 0.1)
    k = [torch.stack([keys[b][h][kept[b][h]] for h in range(nkv)]) for b in range(2)]
    v = [torch.stack([values[b][h][kept[b][h]] for h in range(nkv)]) for b in range(2)]
    want, _, _, spread, _ = plain.attention(q.double(), k, v, [(128, 1), (100, 1)], 0, None, 0.1)
    assert ((out.double().view(2, nq, d) - want).abs() <= 2.0**-9 * spread + 2.0**-8 * want.abs()).all()


# ---------------------------------------------------------------------------
# refusals


def test_refusals():
    with pytest.raises(ops.KernelError, match="heads of"):
        ops.kv4_pool_shape(4, 16, 2, 96)
    with pytest.raises(ops.KernelError, match="multiple of 16"):
        ops.kv4_pool_shape(4, 8, 2, 128)
    pool = torch.zeros(ops.kv4_pool_shape(4, 16, 2, 128), dtype=torch.uint8, device=DEV)
    slots = torch.zeros(3, dtype=torch.int32, device=DEV)
    k = torch.zeros((3, 2, 128), device=DEV)
    for bad_k, bad_v, bad_pool, bad_slots in (
        (k.half(), k.half(), pool, slots), (k, k.bfloat16(), pool, slots), (k[:, :1], k, pool, slots), (k, k, pool.int(), slots),
        (k, k, pool[:, :, :, :-18], slots), (k, k, pool, slots.long()), (k, k, pool, slots[:2]), (k.transpose(0, 1), k, pool, slots),
        (torch.zeros(3 * 258, device=DEV)[1:769].view(3, 2, 128), k, pool, slots), (k.cpu(), k, pool, slots),
    ):
        with pytest.raises(ops.KernelError):
            ops.kv4_store(bad_k, bad_v, bad_pool, bad_slots)
    with pytest.raises(ops.KernelError, match="sums"):
        ops.kv4_store(k, k, pool, slots, torch.zeros((4, 2, 8), device=DEV))
    with pytest.raises(ops.KernelError):
        ops.kv4_load(pool, slots, k, k[:2])
    q = torch.zeros((1, 4 * 128), device=DEV)
    cu, one = torch.tensor([0, 1], dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    table = torch.zeros((1, 1), dtype=torch.int32, device=DEV)
    good = [q, pool, q.clone(), cu, one, table, 1, 1, 1, 4, 2, 128, 1.0]

    def call(**changed):
        args = list(good)
        kw = {}
        for key, value in changed.items():
            if key.startswith("a"):
                args[int(key[1:])] = value
            else:
                kw[key] = value
        ops.attention_kv4(*args, **kw)

    call()
    for changed in ({"a0": q.half()}, {"a0": q[:, :-1]}, {"a1": pool.float()}, {"a2": q.bfloat16()}, {"a3": cu.long()}, {"a3": cu[:1]}, {"a5": table[0]},
                    {"a6": 2}, {"a9": 3}, {"a10": 4}, {"a11": 64}, {"a12": 0.0}, {"a12": -1.0}, {"window": -1}, {"head_sinks": torch.zeros(3, device=DEV)},
                    {"lse": torch.zeros((1, 4), device=DEV, dtype=torch.float64)}, {"a2": q.clone().expand(2, -1)}):
        with pytest.raises(ops.KernelError):
            call(**changed)
    with pytest.raises(ops.KernelError):
        ops.attention_kv4_weights(q, pool, torch.zeros((2, 4), device=DEV), torch.zeros((4, 2, 16), device=DEV), *good[3:])
    sums = torch.zeros((4, 2, 16), device=DEV)
    for budget, recent, first in ((0, 0, 0), (4, 3, 2), (4, -1, 0), (4, 0, -1)):
        with pytest.raises(ops.KernelError, match="budget"):
            ops.kv4_evict(pool, sums, table, one, one.clone(), 1, 1, budget, recent, first)
    with pytest.raises(ops.KernelError):
        ops.kv4_evict(pool, sums.double(), table, one, one.clone(), 1, 1, 4, 0, 0)


def test_empty_batches():
    """No rows, no tokens, no requests: nothing happens."""
    pool = torch.zeros(ops.kv4_pool_shape(2, 16, 1, 64), dtype=torch.uint8, device=DEV)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    k = torch.zeros((0, 1, 64), device=DEV)
    ops.kv4_store(k, k, pool, none)
    ops.kv4_load(pool, none, k, k.clone())
    q = torch.zeros((0, 64), device=DEV)
    cu, table = torch.zeros(1, dtype=torch.int32, device=DEV), torch.zeros((0, 1), dtype=torch.int32, device=DEV)
    ops.attention_kv4(q, pool, q.clone(), cu, none, table, 0, 0, 0, 1, 1, 64, 1.0)
    ops.kv4_evict(pool, torch.zeros((2, 1, 16), device=DEV), table, none, none.clone(), 0, 0, 4, 0)
    assert int(pool.sum()) == 0
