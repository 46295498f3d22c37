"""Steps with drafted tokens: attention over a tree, verification, the accepted rows, lookup, against plain float64."""

import math
import random

import pytest
import torch

from tests.plain import drafts_plain as plain

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from tokensprint_b200 import ops

DEV = "cuda"


def ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


def random_tree(rng, nodes, shape):
    if nodes == 0:
        return []
    if shape == "chain":
        return list(range(-1, nodes - 1))
    if shape == "star":
        return [-1] + [0] * (nodes - 1)
    return [-1] + [min(i - 1, int(i * rng.random() ** 1.3)) for i in range(1, nodes)]


# ---------------------------------------------------------------------------
# attention


def step(lens, nq, nkv, d, page, dtype, seed=0, shape="tree", seen=None, spoil=math.nan, page_gaps=3):
    """A batch with (rows, nodes) per request; what no request holds in the pools is `spoil`."""
    gen, rng = torch.Generator().manual_seed(seed), random.Random(seed)
    per = [-(-n // page) for n, _ in lens]
    total = sum(per) + page_gaps
    order = torch.randperm(total, generator=gen).int()
    table = torch.full((len(lens), max([1, *per])), -1, dtype=torch.int32)
    pools = [torch.full((total, page, nkv, d), spoil, dtype=dtype) for _ in range(2)]
    at, rows, trees, positions = 0, [], [], []
    for b, (n, t) in enumerate(lens):
        table[b, : per[b]] = order[at : at + per[b]]
        at += per[b]
        kv = []
        for i, pool in enumerate(pools):
            x = torch.randn((n, nkv, d), generator=gen).to(dtype)
            for j in range(n):
                pool[table[b, j // page], j % page] = x[j]
            kv.append(x.to(DEV))
        rows.append(kv)
        tree = plain.ancestors(random_tree(rng, t, shape)) if t else []
        trees.append(tree if seen is None else seen(b, t, tree))
        positions.append([n - t + len(a) - 1 for a in tree])
    T = sum(t for _, t in lens)
    words = max(1, -(-max(t for _, t in lens) // 64))
    mask = torch.cat([plain.mask_words(s, words) for s in trees if s] or [torch.zeros((0, words), dtype=torch.int64)])
    q = (1.5 * torch.randn((T, nq, d), generator=gen)).to(dtype)
    cu = [0]
    for _, t in lens:
        cu.append(cu[-1] + t)
    return {"q": q.flatten(1).to(DEV), "k": pools[0].to(DEV), "v": pools[1].to(DEV), "table": table.to(DEV), "mask": mask.to(DEV), "cu": ints(cu),
            "context": ints([n for n, _ in lens]), "rows": rows, "trees": trees, "positions": positions,
            "flat_positions": ints(sum(positions, [])), "lens": lens, "nq": nq, "nkv": nkv, "d": d, "page": page}


def attend(s, out=None, window=0, sinks=None, cap=0.0, scale=None, max_t=None, max_n=None):
    out = torch.full_like(s["q"], math.nan) if out is None else out
    ops.attention_tree(s["q"], s["k"], s["v"], out, s["mask"], s["cu"], s["context"], s["table"], s["page"], len(s["lens"]),
                       max_t or max(t for _, t in s["lens"]), max_n or max(n for n, _ in s["lens"]), s["nq"], s["nkv"], s["d"],
                       s["d"] ** -0.5 if scale is None else scale, window=window, positions=s["flat_positions"] if window else None, head_sinks=sinks, softcap=cap)
    return out


def check(s, out, window=0, sinks=None, cap=0.0, scale=None):
    """Bounds: bfloat16: the result's rounding (2^-8 of it), the weights' (2^-8 of every p |v|), 2^-20 for what is 32-bit.  float32: a score is off by (d + 6) 2^-24
    of the sum of its |products|; a weight by twice that (of scores below 40 in size, in units of log2 below 64: 2^-18 more per exponential's argument,
    and 2^-21 for exponentials and sums), the result by that of the sum of p |v|."""
    scale = s["d"] ** -0.5 if scale is None else scale
    at = 0
    for (n, t), (k, v), tree, pos in zip(s["lens"], s["rows"], s["trees"], s["positions"]):
        if t == 0:
            continue
        ref, spread, size = plain.attention(s["q"][at : at + t].view(t, s["nq"], -1), k, v, tree, pos, scale, window, sinks, cap)
        got = out[at : at + t].view(t, s["nq"], -1).double()
        if out.dtype == torch.bfloat16:
            # (a score in 32 bits as below; operands of the products are exact)
            bound = 2.0**-8 * (ref.abs() + spread) + (2 * (s["d"] + 6) * 2.0**-24 * size[..., None] + 2.0**-17) * spread + 1e-30
        else:
            bound = (2 * (s["d"] + 6) * 2.0**-24 * size[..., None] + 2.0**-18 + 2.0**-21) * spread + 1e-30
        assert torch.isfinite(got).all()
        worst = ((got - ref).abs() / bound).max()
        assert worst <= 1, f"request of {n} rows, {t} nodes: {float(worst):.2f} of the bound"
        at += t


BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lens,nq,nkv,d,page", [
    ([(1, 1)], 1, 1, 64, 16),
    ([(7, 7)], 4, 2, 128, 16),                                # nothing before the step
    ([(130, 3), (65, 1), (64, 9), (1, 1)], 16, 8, 128, 16),   # ends at and beside a block's
    ([(517, 6)], 16, 8, 128, 16),
    ([(700, 5), (20, 5), (333, 2)], 10, 2, 128, 64),          # five heads a group
    ([(200, 33), (90, 64)], 8, 1, 128, 32),
    ([(400, 65), (256, 256)], 4, 4, 64, 128),                 # two and four words of mask
    ([(150, 13), (80, 20)], 14, 2, 128, 8),                   # seven heads a group
    ([(90, 4), (33, 33)], 16, 1, 256, 16),
    ([(100, 5)], 6, 3, 96, 5),                                # a head and pages of other sizes
    ([(77, 8)], 2, 2, 24, 1),
    ([(300, 4), (0, 0), (41, 2)], 32, 8, 128, 16),            # a lane that belongs to nobody
    ([(260, 61), (515, 40)], 40, 8, 128, 64),
    ([(390, 50)], 64, 1, 64, 16),
])
def test_attention_of_trees(lens, nq, nkv, d, page, dtype):
    s = step(lens, nq, nkv, d, page, dtype, seed=len(lens) + d)
    check(s, attend(s))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lens,nq,nkv,d,page", [([(5000, 4)], 4, 1, 128, 16), ([(2500, 17), (120, 3), (1900, 30)], 8, 2, 64, 64)])
def test_attention_over_long_contexts(lens, nq, nkv, d, page, dtype):
    s = step(lens, nq, nkv, d, page, dtype, seed=3)
    check(s, attend(s))
    check(s, attend(s, max_n=16384))  # a captured step is planned for the longest


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape", ["chain", "star", "tree"])
@pytest.mark.parametrize("window", [1, 2, 5, 64, 100, 5000])
def test_windows_count_positions(shape, window, dtype):
    s = step([(300, 12), (9, 9), (129, 2)], 8, 4, 64 if dtype == F32 else 128, 16, dtype, seed=window, shape=shape)
    check(s, attend(s, window=window), window=window)


def test_a_window_over_pages_that_were_given_back():
    s = step([(400, 6), (200, 3)], 8, 4, 128, 16, BF16, seed=5)
    window = 50
    for b, (n, t) in enumerate(s["lens"]):
        first = n - t - window + 1  # the first row that the root sees
        for e in range(first // 16):
            s["k"][s["table"][b, e]] = math.nan
            s["v"][s["table"][b, e]] = math.nan
            s["table"][b, e] = -1
    check(s, attend(s, window=window), window=window)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_sinks_and_a_cap(d, dtype):
    s = step([(270, 5), (3, 3), (1000, 18)], 16, 4, d, 32, dtype, seed=d)
    sinks = 2 * torch.randn(16, generator=torch.Generator().manual_seed(1)).to(DEV)
    sinks[3] = -math.inf
    sinks[7] = 30.0
    check(s, attend(s, sinks=sinks), sinks=sinks)
    check(s, attend(s, sinks=sinks, cap=4.0), sinks=sinks, cap=4.0)
    check(s, attend(s, window=40, sinks=sinks, cap=7.5), window=40, sinks=sinks, cap=7.5)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("sink", [False, True])
def test_nodes_that_see_nothing_are_zeros(sink, dtype):
    def seen(b, t, tree):
        return [[] for _ in range(t)] if b == 0 else [a if i % 2 else [] for i, a in enumerate(tree)]

    s = step([(6, 6), (9, 9), (80, 5)], 8, 2, 128, 16, dtype, seed=2, seen=seen)
    sinks = torch.zeros(8, device=DEV) if sink else None
    out = attend(s, sinks=sinks)
    assert (out[:6] == 0).all() and (out[6:15:2] == 0).all()
    check(s, out, sinks=sinks)


def test_masks_need_not_be_trees():
    """Any bits: nodes behind the own one, none of the own."""
    def seen(b, t, tree):
        r = random.Random(b)
        return [[i for i in range(t) if r.random() < 0.5] for _ in range(t)]

    s = step([(100, 40), (70, 70), (300, 130)], 4, 2, 128, 16, BF16, seed=8, seen=seen)
    check(s, attend(s))


def test_rows_behind_the_last_request_stay():
    s = step([(60, 3), (30, 2)], 8, 2, 128, 16, BF16, seed=4)
    full = {**s, "q": torch.cat([s["q"], torch.full((7, s["q"].shape[1]), math.nan, device=DEV, dtype=BF16)]),
            "mask": torch.cat([s["mask"], torch.full((7, 1), -1, dtype=torch.int64, device=DEV)])}
    out = torch.full_like(full["q"], 7.0)
    attend(full, out=out)
    assert (out[5:] == 7.0).all()
    check(s, out[:5])
    again = torch.full_like(full["q"], 7.0)
    attend({**full, "lens": s["lens"] * 1}, out=again, max_n=5000, max_t=9)
    assert (again[5:] == 7.0).all()
    check(s, again[:5])


def test_lone_tokens_and_chains_are_what_decode_attention_gives():
    """A chain is a causal portion: the framework's own kernels for those, within the roundings of both."""
    s = step([(700, 4), (90, 4), (1500, 4)], 16, 4, 128, 16, BF16, seed=6, shape="chain", spoil=0.0)
    out, other = attend(s), torch.empty_like(s["q"])
    seq = ints([0] * 4 + [1] * 4 + [2] * 4)
    ops.attention_paged_mma(s["q"], s["k"], s["v"], other, s["cu"], s["context"], s["table"], seq, 16, 3, 4, 16, 4, 128, 128**-0.5)
    assert (out.float() - other.float()).abs().max() < 0.03
    check(s, other)


@pytest.mark.parametrize("d,dtype", [(128, BF16), (64, F32)])
def test_equal_inputs_give_equal_bits(d, dtype):
    s = step([(1900, 13), (300, 31), (7, 2)], 16, 4, d, 16, dtype, seed=9)
    first = attend(s)
    for _ in range(3):
        assert torch.equal(attend(s), first)


@pytest.mark.parametrize("d,dtype", [(128, BF16), (64, BF16), (256, BF16), (64, F32)])
def test_attention_captured_and_replayed_on_other_lengths(d, dtype):
    """One capture; the lengths, the masks and the queries change between replays; eager calls on another stream run between."""
    s = step([(1200, 9), (333, 9)], 8, 2, d, 16, dtype, seed=1)
    out = torch.zeros_like(s["q"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attend(s, out=out, max_n=4096)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        attend(s, out=out, max_n=4096)
    other = step([(800, 30)], 8, 2, d, 16, dtype, seed=11)
    for lens in ([(1200, 9), (333, 9)], [(1200, 9), (9, 9)], [(40, 9), (333, 9)]):
        context = [n for n, _ in lens]
        s["context"].copy_(ints(context))
        graph.replay()
        with torch.cuda.stream(side):
            eager = attend(other)
        torch.cuda.synchronize()
        check(other, eager)
        cut = {**s, "lens": lens, "rows": [(k[: n], v[: n]) for (k, v), n in zip(s["rows"], context)]}
        check(cut, out)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_many_requests(dtype):
    rng = random.Random(7)
    s = step([(n := rng.randrange(1, 300), rng.randrange(0, min(n, 9) + 1)) for _ in range(150)], 4, 2, 64, 16, dtype, seed=13)
    check(s, attend(s))


def test_attention_on_two_streams_at_once():
    steps = [step([(900, 20), (1400, 7)], 16, 4, 128, 16, BF16, seed=14), step([(2000, 33), (64, 3), (500, 1)], 16, 4, 128, 16, BF16, seed=15)]
    want = [attend(s) for s in steps]
    sides = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, side in enumerate(sides):
            with torch.cuda.stream(side):
                got[i].append(attend(steps[i]))
    torch.cuda.synchronize()
    for i, s in enumerate(steps):
        check(s, want[i])
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_caches_that_begin_beside_16_bytes_are_refused():
    s = step([(40, 3)], 4, 2, 64, 16, BF16)
    s["k"] = torch.empty(s["k"].numel() + 1, dtype=BF16, device=DEV)[1:].view(s["k"].shape)
    with pytest.raises(ops.KernelError, match="16 bytes"):
        attend(s)


@pytest.mark.parametrize("d", [64, 128])
def test_queries_that_begin_beside_16_bytes(d):
    s = step([(400, 9), (70, 2)], 8, 2, d, 16, BF16, seed=16)
    q = torch.empty(s["q"].numel() + 1, dtype=BF16, device=DEV)[1:].view(s["q"].shape)
    s["q"] = q.copy_(s["q"])
    check(s, attend(s))


# ---------------------------------------------------------------------------
# verification


def verification(nodes, V, seed, dtype=F32, shape="tree", probs=False, temps=(0.0, 0.7, 1.0), stride=0, same_logits=False):
    gen, rng = torch.Generator().manual_seed(seed), random.Random(seed)
    T, B = sum(nodes), len(nodes)
    logits = (2.5 * torch.randn((T, V), generator=gen)).to(dtype)
    q = torch.softmax(logits.float() + 0.7 * torch.randn((T, V), generator=gen), -1) if probs else None
    cu, parents, tokens = [0], [], []
    for t in nodes:
        tree = random_tree(rng, t, shape)
        for i, p in enumerate(tree):
            row = cu[-1] + max(p, 0)
            if probs:
                tokens.append(int(torch.multinomial(q[row], 1, generator=gen)))
            else:
                tokens.append(int(logits[row].float().topk(min(3, V)).indices[rng.randrange(min(3, V))]) if rng.random() < 0.9 else rng.randrange(V))
        parents += tree
        cu.append(cu[-1] + t)
    s = {"nodes": nodes, "logits": logits, "probs": q, "tokens": tokens, "parents": parents, "cu": cu, "temps": [temps[b % len(temps)] for b in range(B)],
         "uniforms": torch.rand(T, generator=gen), "keys": torch.randint(-(1 << 63), (1 << 63) - 1, (B,), generator=gen, dtype=torch.int64), "V": V, "stride": stride}
    return s


def run_verify(s, columns=0):
    V, wide = s["V"], s["V"] + s["stride"]
    T, B = len(s["tokens"]), len(s["nodes"])
    logits = torch.full((T, wide), 9.0, dtype=s["logits"].dtype, device=DEV)[:, :V]
    logits.copy_(s["logits"])
    probs = None
    if s["probs"] is not None:
        probs = torch.full((T, wide), 9.0, device=DEV)[:, :V]
        probs.copy_(s["probs"])
    columns = columns or max(s["nodes"])
    path, fresh = (torch.full((B, columns), 77, dtype=torch.int32, device=DEV) for _ in range(2))
    counts = torch.full((B,), 77, dtype=torch.int32, device=DEV)
    ops.verify_drafts(logits, ints(s["tokens"]), ints(s["parents"]), ints(s["cu"]), torch.tensor(s["temps"], device=DEV), s["uniforms"].to(DEV),
                      s["keys"].to(DEV), path, fresh, counts, B, max(s["nodes"]), draft_probs=probs)
    return path.tolist(), fresh.tolist(), counts.tolist()


def check_verify(s, got):
    """Whole numbers are equal where the nearest decision is further than 2^-16 from the other side: a probability is off by the rounding of the
    exponent's argument (|x - m| / T below 40: 40 x 2^-23), of the exponential and of a sum in pieces (below 2^-19 together), a race's quotient likewise."""
    paths, fresh, counts = got
    close = 0
    for b, t in enumerate(s["nodes"]):
        a = s["cu"][b]
        if t == 0:
            assert counts[b] == 0 and set(paths[b]) == {-1} and set(fresh[b]) == {-1}
            continue
        path, tokens, margin = plain.verify(s["logits"][a : a + t], s["tokens"][a : a + t], s["parents"][a : a + t], s["temps"][b],
                                            s["uniforms"][a : a + t], s["keys"][b], None if s["probs"] is None else s["probs"][a : a + t])
        if margin < 2.0**-16:
            close += 1
            continue
        width = len(paths[b])
        assert counts[b] == len(path) - 1
        assert paths[b] == path + [-1] * (width - len(path))
        assert fresh[b] == tokens + [-1] * (width - len(tokens))
    assert close <= 1 + len(s["nodes"]) // 20


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("shape", ["chain", "star", "tree"])
@pytest.mark.parametrize("nodes,V,dtype", [
    ([1], 1, F32), ([5], 2, F32), ([3, 1, 7], 37, F32), ([8] * 9, 1000, F32), ([4, 0, 12, 1], 4099, F32), ([6, 6, 6], 4096, BF16), ([2, 9], 33001, BF16),
    ([61, 5, 33], 777, F32), ([256, 3], 130, F32), ([5] * 40, 300, BF16),
])
def test_verification(nodes, V, dtype, shape, probs):
    s = verification(nodes, V, seed=V + len(nodes), dtype=dtype, shape=shape, probs=probs)
    check_verify(s, run_verify(s))


@pytest.mark.parametrize("stride", [1, 2, 64])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_verification_of_rows_that_lie_apart(stride, dtype):
    s = verification([7, 3, 4], 1027, seed=stride, dtype=dtype, probs=stride == 2, stride=stride)
    check_verify(s, run_verify(s, columns=11))


@pytest.mark.parametrize("V", [151936, 262145])
def test_verification_of_large_vocabularies(V):
    s = verification([5, 9, 1], V, seed=1, temps=(0.8, 0.0, 1.0))
    check_verify(s, run_verify(s))


def test_verification_on_two_streams_at_once():
    cases = [verification([9, 4, 1], 20011, seed=2, shape="chain", probs=True), verification([6] * 12, 5003, seed=3)]
    want = [run_verify(s) for s in cases]
    sides = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for s, side in zip(cases, sides):
            with torch.cuda.stream(side):
                got.append(run_verify(s))
        assert got == want


def test_verification_without_rows():
    """Requests without nodes accept nothing and draw nothing, and nodes behind the rows of logits are none."""
    path, fresh = (torch.full((2, 3), 77, dtype=torch.int32, device=DEV) for _ in range(2))
    counts = torch.full((2,), 77, dtype=torch.int32, device=DEV)
    for T, cu, nodes in ((0, [0, 0, 0], [0, 0]), (0, [0, 2, 3], [0, 0]), (2, [0, 0, 3], [0, 2]), (2, [5, 7, 9], [0, 0])):
        ops.verify_drafts(torch.zeros((T, 9), device=DEV), ints([0] * T), ints([-1] + [0] * (T - 1))[:T], ints(cu), torch.zeros(2, device=DEV), torch.zeros(T, device=DEV),
                          torch.zeros(2, dtype=torch.int64, device=DEV), path, fresh, counts, 2, 3)
        # (equal logits: the first entry is the largest, and the child's)
        assert counts.tolist() == [1 if n == 2 else 0 for n in nodes]
        assert path.tolist() == [[0, 1, -1] if n == 2 else [-1] * 3 for n in nodes] and fresh.tolist() == [[0, 0, -1] if n == 2 else [-1] * 3 for n in nodes]


@pytest.mark.parametrize("T", [1e-9, 1e30, 3e38, math.inf])
def test_temperatures_at_the_ends(T):
    """The smallest leave the largest entry, the largest every entry that is a number, alike (five sigma)."""
    B, V = 4000, 8
    logits = torch.tensor([1.0, -math.inf, 3.0, math.nan, -2.0, 2.0, -math.inf, 0.0], device=DEV).repeat(B, 1)
    path, fresh = (torch.empty((B, 1), dtype=torch.int32, device=DEV) for _ in range(2))
    counts = torch.empty(B, dtype=torch.int32, device=DEV)
    ops.verify_drafts(logits, ints([0] * B), ints([-1] * B), torch.arange(B + 1, device=DEV).int(), torch.full((B,), T, device=DEV), torch.zeros(B, device=DEV),
                      torch.arange(B, device=DEV) * 0x9E3779B97F4A7C1, path, fresh, counts, B, 1)
    seen = torch.bincount(fresh[:, 0].long(), minlength=V).tolist()
    if T < 1:
        assert seen[2] == B
    else:
        assert sum(seen[i] for i in (0, 2, 4, 5, 7)) == B and all(abs(seen[i] - B / 5) < 5 * (B * 0.16) ** 0.5 for i in (0, 2, 4, 5, 7))


def test_logits_that_are_no_numbers():
    """NaN and -inf have no probability, infinity is the largest number, a row without any number gives its first entry."""
    s = verification([4, 4, 4, 4, 4], 200, seed=5, shape="chain", temps=(1.0, 0.0))
    x = s["logits"]
    x[:, 50:] = -math.inf
    x[3, :25] = math.nan
    x[4:8, :] = math.nan
    x[8:12, 7] = math.inf
    x[12:16, :] = -math.inf
    s["tokens"][9] = s["tokens"][10] = 7
    s["tokens"][13] = 0
    check_verify(s, run_verify(s))


def test_tokens_and_parents_that_do_not_exist():
    s = verification([6, 6], 64, seed=3, temps=(0.0, 1.0))
    s["tokens"][1], s["tokens"][7] = 64, -1
    s["parents"][4], s["parents"][10] = 4, 5
    check_verify(s, run_verify(s))


def test_the_same_token_twice():
    s = verification([5, 5, 5, 5], 6, seed=4, shape="star", temps=(1.0,))
    s["tokens"] = [0, 3, 3, 3, 2] * 4
    s["logits"][:, 3] = -1.0
    check_verify(s, run_verify(s))


@pytest.mark.parametrize("probs,nodes", [(False, 2), (False, 4), (True, 2), (True, 4)])
def test_tokens_come_out_as_the_target_has_them(probs, nodes):
    """The first token of 60,000 requests with the same logits: its frequencies are the target's probabilities, whatever the drafts were (five sigma)."""
    B, V, T = 60000, 7, 0.9
    gen = torch.Generator(DEV).manual_seed(nodes)
    row = torch.tensor([0.3, 1.5, -1.0, 0.9, 0.0, 2.0, -3.0], device=DEV)
    q = torch.softmax(torch.tensor([1.0, 0.5, 0.5, 0.2, -1.0, 2.5, 0.0], device=DEV), -1)
    logits = row.expand(B * nodes, V).contiguous()
    drawn = torch.multinomial(q, B * nodes, replacement=True, generator=gen).int()
    guesses = ints([5, 5, 1, 3])[:nodes].repeat(B)
    path, fresh = (torch.empty((B, nodes), dtype=torch.int32, device=DEV) for _ in range(2))
    counts = torch.empty(B, dtype=torch.int32, device=DEV)
    ops.verify_drafts(logits, drawn if probs else guesses, ints([-1] + [0] * (nodes - 1)).repeat(B), torch.arange(0, B * nodes + 1, nodes, device=DEV).int(),
                      torch.full((B,), T, device=DEV), torch.rand(B * nodes, device=DEV, generator=gen),
                      torch.randint(-(1 << 63), (1 << 63) - 1, (B,), device=DEV, generator=gen, dtype=torch.int64), path, fresh, counts, B, nodes,
                      draft_probs=q.expand(B * nodes, V).contiguous() if probs else None)
    p = torch.softmax(row.double() / T, -1)
    seen = torch.bincount(fresh[:, 0].long(), minlength=V).double() / B
    assert ((seen - p).abs() < 5 * (p * (1 - p) / B).sqrt()).all()
    assert counts.float().mean() > 0.3


def test_verification_captured_with_padding():
    s = verification([6, 3, 5], 900, seed=12, temps=(0.9, 0.0))
    T, B, width = len(s["tokens"]), 3, 6
    dev = {"logits": s["logits"].to(DEV), "tokens": ints(s["tokens"]), "parents": ints(s["parents"]), "cu": ints(s["cu"] + [s["cu"][-1]]),
           "temps": torch.tensor(s["temps"] + [1.0], device=DEV), "uniforms": s["uniforms"].to(DEV), "keys": torch.cat([s["keys"], s["keys"][:1]]).to(DEV)}
    path, fresh = (torch.full((B + 1, width), 77, dtype=torch.int32, device=DEV) for _ in range(2))
    counts = torch.full((B + 1,), 77, dtype=torch.int32, device=DEV)

    def call():
        ops.verify_drafts(dev["logits"], dev["tokens"], dev["parents"], dev["cu"], dev["temps"], dev["uniforms"], dev["keys"], path, fresh, counts, B + 1, width)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call()
    for shift in (0, 1):
        fresh_logits = s["logits"].roll(shift, 0)
        dev["logits"].copy_(fresh_logits)
        graph.replay()
        torch.cuda.synchronize()
        check_verify({**s, "logits": fresh_logits, "nodes": s["nodes"] + [0], "cu": s["cu"] + [s["cu"][-1]]}, (path.tolist(), fresh.tolist(), counts.tolist()))


# ---------------------------------------------------------------------------
# accepted rows


@pytest.mark.parametrize("dtype,nkv,d", [(BF16, 8, 128), (F32, 2, 64), (BF16, 1, 6), (BF16, 3, 5), (BF16, 16, 256)])
@pytest.mark.parametrize("page", [1, 5, 16, 64])
def test_accepted_rows_move_to_the_front(page, dtype, nkv, d):
    gen, rng = torch.Generator().manual_seed(page), random.Random(page)
    lens = [(40, 9), (12, 12), (3, 1), (70, 64), (20, 6), (0, 0)]
    per = [-(-n // page) for n, _ in lens]
    order = torch.randperm(sum(per) + 2, generator=gen).int()
    table = torch.full((len(lens), max(per)), -1, dtype=torch.int32)
    at = 0
    for b, p in enumerate(per):
        table[b, :p] = order[at : at + p]
        at += p
    pools = [torch.randn((sum(per) + 2, page, nkv, d), generator=gen).to(dtype) for _ in range(6)]
    width, paths = 64, []
    for n, t in lens:
        way = max(plain.ancestors(random_tree(rng, t, "tree")), key=len) if t else [0]
        if t == 12:
            way = list(range(12))  # everything was accepted: nothing moves
        if t == 64:
            way = [0, 2, 3, 5, 8, 13, 21, 34, 55, 63]
        if t == 6:
            way = [0]
        paths.append(way)
    path = torch.tensor([w + [-1] * (width - len(w)) for w in paths], dtype=torch.int32)
    want = [p.clone() for p in pools]
    for b, (n, t) in enumerate(lens):
        for k, i in enumerate(paths[b]):
            if k:
                to, fro = n - t + k, n - t + i
                for x, old in zip(want, pools):
                    x[table[b, to // page], to % page] = old[table[b, fro // page], fro % page]
    cu = [0]
    for _, t in lens:
        cu.append(cu[-1] + t)
    dev = [p.to(DEV) for p in pools]
    ops.keep_drafted_rows(ops.RowPools(dev), path.to(DEV), ints([len(w) - 1 for w in paths]), ints(cu), ints([n for n, _ in lens]), table.to(DEV), page, len(lens))
    for x, y in zip(dev, want):
        assert torch.equal(x.cpu(), y)


def test_paths_and_pages_that_do_not_exist_move_nothing():
    pools = [torch.randn((4, 16, 2, 8), device=DEV) for _ in range(2)]
    before = [p.clone() for p in pools]
    rows = ops.RowPools(pools)
    path = ints([[0, 9, 2, 300], [0, 3, 4, 5], [0, 3, 4, 5]])
    # request 0: nodes that it has not; 1: its pages were given back; 2: a page beyond the pool
    table = ints([[0], [-1], [4]])
    ops.keep_drafted_rows(rows, path, ints([3, 3, 3]), ints([0, 6, 12, 18]), ints([10, 10, 10]), table, 16, 3)
    assert torch.equal(pools[1], before[1]) and torch.equal(pools[0], before[0])
    # more accepted than the path has columns, more nodes than rows: what exists moves
    ops.keep_drafted_rows(rows, ints([[0, 3]]), ints([9]), ints([0, 6]), ints([10]), ints([[0]]), 16, 1)
    want = before[0].clone()
    want[0, 5] = want[0, 7]
    assert torch.equal(pools[0], want)
    ops.keep_drafted_rows(rows, ints([[0, 3]]), ints([1]), ints([0, 6]), ints([2]), ints([[0]]), 16, 1)
    assert torch.equal(pools[0], want)


def test_pools_that_stand_twice_are_refused():
    """Two blocks would move the same rows."""
    whole = torch.zeros((6, 16, 2, 8), device=DEV)
    for pools in ([whole, whole], [whole[:4], whole[2:]], [whole[:2], whole[4:], whole[1:3]]):
        with pytest.raises(ops.KernelError, match="twice"):
            ops.RowPools(pools)
    ops.RowPools([whole[4:], whole[:2], whole[2:4]])


# ---------------------------------------------------------------------------
# lookup


@pytest.mark.parametrize("depth,branches,longest,shortest", [(4, 1, 4, 1), (1, 3, 2, 2), (8, 4, 6, 1), (10, 16, 16, 3), (64, 2, 1, 1)])
@pytest.mark.parametrize("L,kinds", [(1, 3), (2, 2), (9, 2), (100, 3), (700, 20), (5000, 50)])
def test_lookup(L, kinds, depth, branches, longest, shortest):
    gen = torch.Generator().manual_seed(L + branches)
    lengths = sorted({1, 2, min(3, L), L // 2, L - 1, L} - {0}) + [0]
    lengths = [n for n in lengths if n <= L]
    history = torch.randint(0, kinds, (len(lengths), L + 5), generator=gen, dtype=torch.int32)[:, :L]
    width = 1 + depth * branches
    tokens, parents = (torch.full((len(lengths), width), 77, dtype=torch.int32, device=DEV) for _ in range(2))
    counts = torch.full((len(lengths),), 77, dtype=torch.int32, device=DEV)
    wide = torch.full((len(lengths), L + 5), 1, dtype=torch.int32, device=DEV)[:, :L]
    wide.copy_(history)
    ops.lookup_drafts(wide, ints(lengths), tokens, parents, counts, len(lengths), depth, branches, longest, shortest)
    for b, n in enumerate(lengths):
        want_t, want_p = plain.lookup(history[b, :n].tolist(), depth, branches, longest, shortest)
        assert counts[b] == len(want_t)
        assert tokens[b].tolist() == want_t + [-1] * (width - len(want_t))
        assert parents[b].tolist() == want_p + [-1] * (width - len(want_p))


def test_lookup_of_one_token_over_and_over():
    history = torch.full((3, 40000), 5, dtype=torch.int32, device=DEV)
    history[1, ::2] = 6
    history[2, 39000] = 9
    tokens, parents = (torch.empty((3, 13), dtype=torch.int32, device=DEV) for _ in range(2))
    counts = torch.empty(3, dtype=torch.int32, device=DEV)
    lengths = [40000, 39999, 39001]
    ops.lookup_drafts(history, ints(lengths), tokens, parents, counts, 3, 4, 3, 8, 1)
    for b, n in enumerate(lengths):
        want_t, want_p = plain.lookup(history[b, :n].tolist(), 4, 3, 8, 1)
        assert counts[b] == len(want_t)
        assert tokens[b].tolist()[: len(want_t)] == want_t and parents[b].tolist()[: len(want_t)] == want_p


# ---------------------------------------------------------------------------
# together


def test_a_step_from_lookup_to_kept_rows():
    """Lookup, attention, verification and the accepted rows one behind the other, on what the one before left on the device."""
    gen = torch.Generator().manual_seed(0)
    B, depth, branches, V, nq, nkv, d, page, n0 = 3, 3, 2, 50, 8, 2, 128, 16, 90
    width = 1 + depth * branches
    history = torch.randint(0, 6, (B, n0), generator=gen, dtype=torch.int32)
    tokens, parents = (torch.empty((B, width), dtype=torch.int32, device=DEV) for _ in range(2))
    nodes = torch.empty(B, dtype=torch.int32, device=DEV)
    ops.lookup_drafts(history.to(DEV), ints([n0] * B), tokens, parents, nodes, B, depth, branches)
    count = nodes.tolist()
    assert all(1 + branches <= n <= width for n in count)
    packed = [(tokens[b, :n].tolist(), parents[b, :n].tolist()) for b, n in enumerate(count)]
    trees = [plain.ancestors(p) for _, p in packed]
    s = step([(n0 - 1 + n, n) for n in count], nq, nkv, d, page, BF16, seed=4, seen=lambda b, t, tree: trees[b])
    check(s, attend(s))
    cu = s["cu"].tolist()
    logits = 2 * torch.randn((cu[-1], V), generator=gen)
    second = [p.index(0, p.index(0) + 1) for _, p in packed]  # the second chain's nodes are likely, the first's are not
    for b, (x, p) in enumerate(packed):
        for i in range(second[b], count[b]):
            logits[cu[b] + p[i], x[i]] = 12.0 + b
    path, fresh = (torch.empty((B, width), dtype=torch.int32, device=DEV) for _ in range(2))
    counts = torch.empty(B, dtype=torch.int32, device=DEV)
    v = {"nodes": count, "cu": cu, "logits": logits, "tokens": sum((x for x, _ in packed), []), "parents": sum((p for _, p in packed), []),
         "temps": [0.0, 1.0, 0.5], "uniforms": torch.rand(cu[-1], generator=gen), "keys": torch.arange(B), "probs": None, "V": V}
    ops.verify_drafts(logits.to(DEV), ints(v["tokens"]), ints(v["parents"]), s["cu"], torch.tensor(v["temps"], device=DEV), v["uniforms"].to(DEV), v["keys"].to(DEV),
                      path, fresh, counts, B, width)
    check_verify(v, (path.tolist(), fresh.tolist(), counts.tolist()))
    assert all(p[1] == second[b] for b, p in enumerate(path.tolist()))
    old = s["k"].clone()
    ops.keep_drafted_rows(ops.RowPools([s["k"], s["v"]]), path, counts, s["cu"], s["context"], s["table"], page, B)
    table = s["table"].tolist()
    for b in range(B):
        for k in range(1, counts[b].item() + 1):
            to, fro = n0 - 1 + k, n0 - 1 + path[b, k].item()
            assert torch.equal(s["k"][table[b][to // page], to % page], old[table[b][fro // page], fro % page])
