"""ops.verify_drafts where few numbers decide: waiting times at their ends, what is left behind likely drafts that were refused."""

import math

import pytest
import torch

from tests.plain import drafts_plain as plain
from tokensprint_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
MASK64 = (1 << 64) - 1
MOST = (1 << 24) - 1


def key_with(pair, even, odd):
    """The key for which entries 2 pair and 2 pair + 1 get the 24 bits `even` and `odd`: the hash, walked backwards."""
    z = even << 40 | odd << 16
    z = z ^ (z >> 29) ^ (z >> 58)
    z = z * pow(0x94D049BB133111EB, -1, 1 << 64) & MASK64
    z ^= z >> 32
    z ^= pair * 0xD1342543DE82EF95 & MASK64
    return z - (1 << 64) if z >> 63 else z


def waiting(bits):
    return -math.log1p(-(bits + 0.5) / (1 << 24))


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def verify(logits, tokens, parents, uniforms, keys, nodes, temperature=1.0, probs=None):
    """Requests of `nodes` nodes each; returns counts and the tokens that came out."""
    B = len(keys)
    path, fresh = (torch.full((B, nodes), 77, dtype=torch.int32, device=DEV) for _ in range(2))
    counts = torch.full((B,), 77, dtype=torch.int32, device=DEV)
    ops.verify_drafts(logits.to(DEV), ints(tokens), ints(parents), torch.arange(0, B * nodes + 1, nodes, device=DEV).int(), torch.full((B,), temperature, device=DEV),
                      uniforms.to(DEV), torch.as_tensor(keys, dtype=torch.int64, device=DEV), path, fresh, counts, B, nodes, draft_probs=probs)
    return counts.tolist(), fresh.tolist()


# ---------------------------------------------------------------------------
# waiting times


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("entry", [0, 1, 37, 100, 129])
def test_the_longest_waiting_time_is_finite(entry, dtype):
    """The only entry with a probability is drawn, however long it waits."""
    key = key_with(entry // 2, MOST, MOST)
    assert float(plain.waiting_times(key, 130)[entry]) == waiting(MOST)
    logits = torch.full((2, 130), -math.inf, dtype=dtype)
    logits[:, entry] = 2.0
    logits[1, :] = torch.where(torch.arange(130) == entry, 200.0, 0.0).to(dtype)  # (others' weights: e^-198, none in float32)
    assert verify(logits, [5, 5], [-1, -1], torch.zeros(2), [key, key], 1)[1] == [[entry], [entry]]


def test_a_longest_waiting_time_behind_a_refusal():
    """The same where a refused child leaves one entry, with the drafter's probabilities and without."""
    logits = torch.full((2, 8), -math.inf)
    logits[:, 6], logits[:, 3] = 0.0, 0.0
    q = torch.zeros((2, 8), device=DEV)
    q[:, 3] = 1.0
    uniforms = torch.tensor([0.0, 0.75])
    for probs in (None, q):
        assert verify(logits, [0, 3], [-1, 0], uniforms, [key_with(3, MOST, 0)], 2, probs=probs) == ([0], [[6, -1]])


def test_long_waiting_times_are_exact():
    """Two entries whose quotients are 2^-12 apart: the logits' rounding (|x| < 24: 2^-19 of a weight), the exponential, the logarithm and the division are
    off by less than 2^-17 together."""
    rows, keys, want = [], [], []
    for a in (MOST, MOST - 1, MOST - 2, MOST - 5, MOST - 20, 1 << 23, (1 << 23) + 1, (1 << 23) - 1, 12345, 0):
        for b in (MOST, MOST - 1, MOST - 3, 1 << 23, (1 << 23) - 1, 777, 0):
            for side in (-1, 1):
                rows.append([math.log(waiting(a) / waiting(b)) + side * 2.0**-12, 0.0])
                keys.append(key_with(0, a, b))
                want.append([0 if side > 0 else 1])
    B = len(keys)
    assert verify(torch.tensor(rows), [0] * B, [-1] * B, torch.zeros(B), keys, 1)[1] == want


# ---------------------------------------------------------------------------
# what is left behind likely drafts that were refused

LAST = 1.0 - 2.0**-24  # the largest number that decides on a node


@pytest.mark.parametrize("temperature", [1.0, 0.25])
@pytest.mark.parametrize("V,top,second", [(2, 0, 1), (2, 1, 0), (9, 3, 7), (4099, 4098, 2500)])
@pytest.mark.parametrize("gap", [2.0, 5.0, 8.0, 11.98])
def test_a_child_with_all_that_is_left_is_accepted(gap, V, top, second, temperature):
    """Two tokens of which the likely one is refused (p <= 1 - 6.2e-6, asked with 1 - 2^-24): the other's probability is one then."""
    logits = torch.full((3, V), -math.inf)
    logits[0, top], logits[0, second] = gap * temperature, 0.0
    logits[1, top] = logits[2, second] = 1.0
    for tail in (1, 3):  # the last child, and one with children behind it (the same token, and one without a probability)
        extra = [top, (second + 1) % V][: tail - 1]
        rows = torch.cat([logits, logits[:1].expand(tail - 1, V)])
        n = 3 + len(extra)
        got = verify(rows, [0, top, second] + extra, [-1] + [0] * (n - 1), torch.full((n,), LAST), [11], n, temperature)
        assert got == ([1], [[second, second] + [-1] * (n - 2)])


def test_the_last_of_many_children_is_accepted():
    """Children that hold all the probability, the likeliest first, each asked with the largest number."""
    V, order = 40, [17, 0, 39, 5, 22]
    logits = torch.full((6, V), -math.inf)
    for i, x in enumerate(order):
        logits[0, x] = -2.5 * i * i  # 1, 0.08, 4.5e-5, 1.7e-10, 4e-18 of the largest
    logits[1:, 9] = 0.0
    p = torch.softmax(logits[0].double(), -1)[order]
    left = torch.flip(torch.cumsum(torch.flip(p, [0]), 0), [0])
    want = next(i for i in range(5) if LAST * float(left[i]) < float(p[i]))
    assert want == 3 and LAST - float(p[2] / left[2]) > 1e-6 and float(p[3] / left[3]) - LAST > 1e-8
    uniforms = torch.full((6,), LAST)
    uniforms[4] = 1 - 2.0**-18  # (the fourth has 1 - 2.2e-8 of what is left: asked with a number that float32 sums tell from it)
    assert verify(logits, [0] + order, [-1] + [0] * 5, uniforms, [4], 6) == ([1], [[5, 9, -1, -1, -1, -1]])


@pytest.mark.parametrize("V", [6, 5003, 151936])
@pytest.mark.parametrize("gap", [3.0, 7.0, 11.0, 14.0])
def test_what_is_left_keeps_its_precision(gap, V):
    """A second child asked 2^-14 beside its probability among what a refused one has left.  Off in the kernel: exponents' arguments (|x| 1.45 < 32: 2^-20 each),
    exponentials (2^-22), sums in pieces of a few dozen (2^-18 at the most)."""
    gen = torch.Generator().manual_seed(V)
    row = torch.randn(V, generator=gen)
    row = torch.where(torch.arange(V) < 6, row, row - 12)  # (few entries hold what the likely one leaves)
    row[3] = 0.0
    row[3] = float(torch.logsumexp(row.double(), 0)) + gap
    logits = row.expand(6, V).contiguous()
    p = torch.softmax(row.double(), -1)
    share = float(p[1] / (1 - p[3])) if gap < 5 else float(p[1] / torch.where(torch.arange(V) == 3, 0.0, p).sum())
    uniforms = torch.full((6,), LAST)
    uniforms[2], uniforms[5] = share * (1 + 2.0**-14), share * (1 - 2.0**-14)
    counts, fresh = verify(logits, [0, 3, 1, 0, 3, 1], [-1, 0, 0, -1, 0, 0], uniforms, [5, 5], 3)
    assert counts == [0, 1] and fresh[1][0] == 1
    assert fresh[0][0] not in (1, 3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B", [8, 15, 160])
def test_requests_whose_likely_drafts_are_refused(B, dtype):
    """Against the formulas in 64 bits: peaked rows, children from the likeliest down, numbers near one; batches that get many threads a request, and few."""
    gen, compared = torch.Generator().manual_seed(2), 0
    nodes, V = 5, 700
    logits = torch.randn((B * nodes, V), generator=gen)
    tokens, parents, uniforms = [], [], torch.ones(B * nodes)
    for b in range(B):
        at = b * nodes
        top = logits[at].topk(nodes - 1)
        for i in range(nodes - 1):
            logits[at, top.indices[i]] += (12 - 3 * i) * (b % 8) / 7
        tokens += [0] + top.indices.tolist()
        parents += [-1] + [0] * (nodes - 1)
        uniforms[at : at + nodes] -= 2.0 ** -(3 + 2 * (3 * b % 10) + torch.rand(nodes, generator=gen))
    uniforms.clamp_(max=LAST)
    keys = torch.randint(-(1 << 63), (1 << 63) - 1, (B,), generator=gen, dtype=torch.int64)
    logits = logits.to(dtype)
    counts, fresh = verify(logits, tokens, parents, uniforms, keys, nodes)
    refused = 0
    for b in range(B):
        r = slice(b * nodes, (b + 1) * nodes)
        path, out, margin = plain.verify(logits[r], tokens[r], parents[r], 1.0, uniforms[r], keys[b])
        refused += len(path) == 1 or path[1] > 1
        if margin < 2.0**-16:  # (what the sums and exponentials are off by, see test_drafts_gpu.check_verify)
            continue
        compared += 1
        assert counts[b] == len(path) - 1 and fresh[b] == out + [-1] * (nodes - len(out))
    assert compared > 0.8 * B and refused > 0.2 * B


def test_single_requests_are_compared():
    """One request a call, so that no other one stands in for it."""
    from tests.test_drafts_gpu import run_verify, verification

    for nodes, V, probs in ((1, 1, False), (5, 2, False), (5, 2, True), (9, 300, False), (9, 300, True), (33, 4099, True)):
        compared = 0
        for seed in range(12):
            s = verification([nodes], V, seed=seed, probs=probs, shape="tree", temps=(0.8,))
            path, out, margin = plain.verify(s["logits"], s["tokens"], s["parents"], 0.8, s["uniforms"], s["keys"][0], s["probs"])
            if margin >= 2.0**-16:
                compared += 1
                paths, fresh, counts = run_verify(s)
                assert counts == [len(path) - 1] and paths[0] == path + [-1] * (nodes - len(path)) and fresh[0] == out + [-1] * (nodes - len(out))
        assert compared >= 10


@pytest.mark.parametrize("probs", [False, True])
def test_tokens_behind_refusals_and_accepted_drafts_come_out_as_the_target_has_them(probs):
    """60,000 requests: the tokens at the root (a likely child and two others are asked there) and those behind an accepted child are distributed as the
    target has them (five sigma)."""
    B, V, nodes = 60000, 5, 5
    gen = torch.Generator(DEV).manual_seed(3)
    p = torch.tensor([[0.9, 0.06, 0.02, 0.015, 0.005], [0.02, 0.03, 0.05, 0.3, 0.6]], device=DEV, dtype=torch.float64)
    q = torch.tensor([[0.5, 0.2, 0.1, 0.1, 0.1], [0.1, 0.1, 0.1, 0.35, 0.35]], device=DEV)
    # root 0 with children 1, 2, 3, and 4 behind 1; every node but the root has the second row
    which = torch.tensor([0, 1, 1, 1, 1], device=DEV)
    logits = p.log().float()[which].repeat(B, 1)
    tokens = torch.tensor([0, 0, 1, 3, 4], device=DEV).int().repeat(B)
    if probs:
        tokens = tokens.view(B, nodes)
        for node, row in ((1, 0), (2, 0), (3, 0), (4, 1)):
            tokens[:, node] = torch.multinomial(q[row], B, replacement=True, generator=gen).int()
        tokens = tokens.view(-1)
    path, fresh = (torch.empty((B, nodes), dtype=torch.int32, device=DEV) for _ in range(2))
    counts = torch.empty(B, dtype=torch.int32, device=DEV)
    ops.verify_drafts(logits, tokens, ints([-1, 0, 0, 0, 1]).repeat(B), torch.arange(0, B * nodes + 1, nodes, device=DEV).int(), torch.ones(B, device=DEV),
                      torch.rand(B * nodes, device=DEV, generator=gen), torch.randint(-(1 << 63), (1 << 63) - 1, (B,), device=DEV, generator=gen, dtype=torch.int64),
                      path, fresh, counts, B, nodes, draft_probs=q[which].repeat(B, 1) if probs else None)
    for tokens, target in ((fresh[:, 0], p[0]), (fresh[counts >= 1, 1], p[1])):
        n = tokens.numel()
        seen = torch.bincount(tokens.long(), minlength=V).double() / n
        assert n > 20000 and ((seen - target).abs() < 5 * (target * (1 - target) / n).sqrt()).all()
