"""ops.verify_drafts where few numbers decide: waiting times at their ends."""

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
