"""The 4-bit cache: what its operators' workspaces held before, and the ends of what their arguments may be."""

import pytest
import torch

from tests.plain import kv4_plain as plain
from tests.test_kv4_gpu import DEV, batch, check_attention, filled

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from tokensprint_b200 import ops


def spoil_workspaces(monkeypatch):
    """Every float tensor of torch.empty is NaN from its first entry to its last."""
    empty = torch.empty

    def spoiled(*args, **kw):
        t = empty(*args, **kw)
        return t.fill_(float("nan")) if t.is_floating_point() else t

    monkeypatch.setattr(torch, "empty", spoiled)


@pytest.mark.parametrize("runs", [True, False])
@pytest.mark.parametrize("oldest", [384, 385, 384 + 63, 384 + 64, 384 + 67, 384 + 127, 512])
@pytest.mark.parametrize("sinks", [False, True])
def test_windowed_portions_read_only_what_was_unpacked(monkeypatch, runs, oldest, sinks):
    """`oldest`, the first key that a query sees, lies anywhere in a page of 128 unpacked rows; the rows ahead of it have no weight, and
    nothing times what they hold may be anything but zero."""
    monkeypatch.setattr(ops, "_KV4_DIRECT_PIECES", 0)
    if not runs:
        monkeypatch.setattr(ops, "_KV4_MIN_RUN", 1 << 20)
    spoil_workspaces(monkeypatch)
    check_attention([(900, 150)], 5, 1, 128, 16, torch.bfloat16, window=900 - 150 + 1 - oldest, sinks=sinks)
    check_attention([(900, 150), (300, 17), (64, 64)], 4, 2, 128, 32, torch.bfloat16, window=900 - 150 + 1 - oldest, sinks=sinks)


@pytest.mark.parametrize("lens", [[(3, 400)], [(0, 300), (20, 100)], [(130, 700), (700, 200), (1, 1)], [(1700, 30), (40, 330), (0, 65), (129, 129)]])
@pytest.mark.parametrize("nq,nkv", [(4, 1), (6, 2)])
@pytest.mark.parametrize("window,sinks", [(0, False), (0, True), (70, True)])
def test_portions_with_more_tokens_than_rows(monkeypatch, lens, nq, nkv, window, sinks):
    """Queries ahead of the first cached row see nothing, whole tiles of them included: zeros, and the logarithm of nothing or of the sink."""
    monkeypatch.setattr(ops, "_KV4_DIRECT_PIECES", 0)
    spoil_workspaces(monkeypatch)
    check_attention(lens, nq, nkv, 128, 16, torch.bfloat16, window=window, sinks=sinks)
    ops.check_device_errors()


def test_eviction_refuses_lengths_that_overlap():
    """The new lengths in the place of the old ones, or of the block table: refused before anything is launched."""
    nkv, d, page = 2, 64, 16
    pool = torch.zeros(ops.kv4_pool_shape(8, page, nkv, d), dtype=torch.uint8, device=DEV)
    sums = torch.ones((8, nkv, page), device=DEV)
    words = torch.arange(16, dtype=torch.int32, device=DEV)
    table, lens = words[:8].view(2, 4), words[8:12]
    before = words.clone()
    for new in (lens, words[9:], words[7:9], words[:2], words[6:8]):
        with pytest.raises(ops.KernelError, match="overlap"):
            ops.kv4_evict(pool, sums, table, lens, new, 2, 9, 4, 1)
    assert torch.equal(words, before) and bool((sums == 1).all())
    new = words[10:12]  # next to the two lengths that the call reads
    ops.kv4_evict(pool, sums, table, lens, new, 2, 9, 4, 1)
    assert new.tolist() == [4, 4] and torch.equal(words[:10], before[:10])


@pytest.mark.parametrize("budget,recent,first", [(300, 20, 4), (1 << 20, 1 << 19, 5), (1 << 45, 0, 1 << 44)])
def test_a_budget_beyond_the_longest_request_takes_no_memory(budget, recent, first):
    gen = torch.Generator().manual_seed(6)
    lens, nkv, d, page = [300, 0, 7, 256], 2, 64, 16
    pool, table, _, _ = filled([(n, 0) for n in lens], nkv, d, page, gen)
    sums = torch.rand((pool.shape[0], nkv, page), generator=gen).to(DEV)
    context, new = torch.tensor(lens, dtype=torch.int32, device=DEV), torch.full((4,), -5, dtype=torch.int32, device=DEV)
    old_pool, old_sums = pool.clone(), sums.clone()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    ops.kv4_evict(pool, sums, table, context, new, 4, 300, budget, recent, first)
    assert torch.cuda.max_memory_allocated() - held < 1 << 16
    assert new.tolist() == lens and torch.equal(pool, old_pool) and torch.equal(sums, old_sums)


FORMS = [  # tokens of a request, head size, type: streamed, streamed in passes, keys in registers (twice), keys in tensor memory
    (1, 128, torch.bfloat16), (20, 64, torch.bfloat16), (200, 64, torch.bfloat16), (90, 128, torch.float32), (200, 128, torch.bfloat16)]


@pytest.mark.parametrize("tokens,d,dtype", FORMS)
def test_weights_leave_rows_that_nobody_sees_alone(tokens, d, dtype):
    """Pages ahead of the window have been given back (-1 in the block table, page 0 to the kernels): whoever has page 0 now loses nothing.
    Every request adds to every row of its own once, so the bits are those of a call in which the pages are still held."""
    gen = torch.Generator().manual_seed(21)
    nq, nkv, page, window = 16, 8, 16, 20
    lens = [(tokens, tokens)] + [(400 + 16 * b, tokens) for b in range(12)]
    pool, table, _, _ = filled(lens, nkv, d, page, gen, spoil=False)
    swap = table.clone()  # the request whose keys are all seen has page 0
    swap[table == 0], swap[table == table[0, 0]] = table[0, 0], 0
    table = swap
    given = table.clone()
    for b, (n, t) in enumerate(lens):
        given[b, : max(0, n - t - window + 1) // page] = -1
    assert int((given < 0).sum()) > int((table < 0).sum())
    T = sum(t for _, t in lens)
    q = torch.randn((T, nq * d), generator=gen).to(dtype).to(DEV)
    cu, context = batch(lens)
    lse = torch.full((T, nq), 3.0, device=DEV)
    sizes = (len(lens), tokens, max(n for n, _ in lens), nq, nkv, d, d**-0.5)
    want = torch.ones((pool.shape[0], nkv, page), device=DEV)
    ops.attention_kv4_weights(q, pool, lse, want, cu, context, table, *sizes, window=window)
    assert bool((want[0] != 1).all()) or tokens < page
    for _ in range(20):
        sums = torch.ones_like(want)
        ops.attention_kv4_weights(q, pool, lse, sums, cu, context, given, *sizes, window=window)
        assert torch.equal(sums, want)


@pytest.mark.parametrize("tokens,d,dtype", FORMS)
def test_weights_of_pages_that_requests_share(tokens, d, dtype):
    """Requests over the same pages: every one of them adds its weights.  The sums of 13 float32 numbers in any order are off by 13 * 2^-24; a request
    by itself may take another of the kernels, whose weights are off by 4 * 2^-18 (reach + 1) as in check_attention, with a reach below 15: 2^-12."""
    gen = torch.Generator().manual_seed(22)
    nq, nkv, page, n, B = 16, 8, 16, 400, 12
    pool, table, _, _ = filled([(n, tokens)], nkv, d, page, gen)
    q = torch.randn((B, tokens, nq * d), generator=gen).to(dtype).to(DEV)
    lse = torch.full((B * tokens, nq), 3.0, device=DEV)
    want = torch.ones((pool.shape[0], nkv, page), device=DEV, dtype=torch.float64)
    cu, context = batch([(n, tokens)])
    for b in range(B):
        one = torch.zeros(want.shape, device=DEV)
        ops.attention_kv4_weights(q[b], pool, lse[:tokens], one, cu, context, table, 1, tokens, n, nq, nkv, d, d**-0.5)
        want += one
    cu, context = batch([(n, tokens)] * B)
    for _ in range(20):
        sums = torch.ones(want.shape, device=DEV)
        ops.attention_kv4_weights(q.flatten(0, 1), pool, lse, sums, cu, context, table.expand(B, -1).contiguous(), B, tokens, n, nq, nkv, d, d**-0.5)
        assert ((sums - want).abs() <= 13 * 2.0**-24 * want + 2.0**-12 * (want - 1)).all()


@pytest.mark.parametrize("tokens,d,dtype", FORMS)
@pytest.mark.parametrize("window", [449, 450, 1 << 20, (1 << 31) - 1])
def test_windows_beyond_the_longest_request(tokens, d, dtype, window):
    """A window that no key falls out of is none, however large the number is (449 still hides a key from the last token)."""
    check_attention([(450, tokens), (tokens, tokens), (30, 1)], 8, 4, d, 16, dtype, window=window)
    check_attention([(450, tokens), (3, 9)], 4, 1, d, 16, dtype, window=window)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens", [1, 3, 100])
@pytest.mark.parametrize("pieces", [0, 600])
def test_sinks_of_minus_infinity_are_none(monkeypatch, dtype, tokens, pieces):
    """Heads without a sink beside heads with one; requests that see nothing: zeros, and the logarithm of nothing or of the sink."""
    monkeypatch.setattr(ops, "_KV4_DIRECT_PIECES", pieces)
    gen = torch.Generator().manual_seed(31)
    nq, nkv, d, page = 8, 2, 128, 16
    lens = [(0, tokens), (40, tokens), (tokens, tokens), (0, 1)]
    pool, table, keys, values = filled(lens, nkv, d, page, gen)
    T = sum(t for _, t in lens)
    q = torch.randn((T, nq * d), generator=gen).to(dtype).to(DEV)
    cu, context = batch(lens)
    sizes = (cu, context, table, len(lens), tokens, max(n for n, _ in lens), nq, nkv, d, d**-0.5)
    sink = torch.randn(nq, generator=gen).to(DEV)
    sink[::2] = -torch.inf
    out, lse = torch.empty_like(q), torch.empty((T, nq), device=DEV)
    ops.attention_kv4(q, pool, out, *sizes, head_sinks=sink, lse=lse)
    want, want_lse, _, spread, reach = plain.attention(q.double().view(T, nq, d), keys, values, lens, 0, sink.double(), d**-0.5)
    exact, slack = dtype == torch.float32, 2.0**-18 * (reach + 1)  # the bounds of check_attention
    bound = ((2.0**-20 if exact else 2.0**-8) + 2 * slack[..., None]) * spread + (2.0**-22 if exact else 2.0**-8) * want.abs() + 1e-30
    assert ((out.double().view(T, nq, d) - want).abs() <= bound).all()
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse), empty) and int(empty.sum()) >= tokens * nq // 2
    assert ((lse.double() - want_lse).abs() <= slack + 2.0**-20 * (1 + want_lse.abs()))[~empty].all()
