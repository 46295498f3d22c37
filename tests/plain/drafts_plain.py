"""Steps with drafted tokens in plain float64, request by request, from the formulas."""

import math

import torch

MASK64 = (1 << 64) - 1


def ancestors(parents):
    """For every node itself and the nodes above it; parents[0] = -1."""
    out = []
    for i, p in enumerate(parents):
        out.append((out[p] if p >= 0 else []) + [i])
    return out


def mask_words(seen, words):
    """Lists of the nodes that every node sees -> int64 [len(seen), words]."""
    rows = []
    for nodes in seen:
        w = [0] * words
        for i in nodes:
            w[i // 64] |= 1 << (i % 64)
        rows.append([x - (1 << 64) if x >= 1 << 63 else x for x in w])
    return torch.tensor(rows, dtype=torch.int64).view(len(seen), words)


def attention(q, keys, values, seen, positions, scale, window=0, sinks=None, cap=0.0):
    """One request.  q [t, nq, d]; keys, values [n, nkv, d]; seen: per node the nodes it sees; positions per node.  Returns the outputs [t, nq, d], the
    weighted sums of |v| [t, nq, d] and per row (t, nq) the largest sum of |q k| scale (what errors are measured by), all float64."""
    t, nq, d = q.shape
    n, nkv = keys.shape[0], keys.shape[1]
    visible = torch.zeros((t, n), dtype=torch.bool, device=q.device)
    for i in range(t):
        for j in range(n):
            k = j - (n - t)
            if k < 0:
                visible[i, j] = window == 0 or j > positions[i] - window
            else:
                visible[i, j] = k in seen[i] and (window == 0 or positions[k] > positions[i] - window)
    q, keys, values = q.double(), keys.double(), values.double()
    out, spread, size = torch.zeros_like(q), torch.zeros_like(q), torch.zeros((t, nq), dtype=torch.float64, device=q.device)
    for h in range(nq):
        k, v = keys[:, h * nkv // nq], values[:, h * nkv // nq]
        s = scale * (q[:, h] @ k.T)
        if cap:
            s = cap * torch.tanh(s / cap)
        s = s.masked_fill(~visible, -math.inf)
        full = s if sinks is None else torch.cat((s, sinks[h].double().expand(t, 1)), 1)
        top = full.amax(1, keepdim=True)
        e = torch.where(full > -math.inf, torch.exp(full - torch.where(top > -math.inf, top, 0.0)), 0.0)
        total = e.sum(1, keepdim=True)
        p = (e / torch.where(total > 0, total, 1.0))[:, :n]
        held = torch.where(visible.any(0)[:, None], v, 0.0)  # (rows nobody sees count for nothing, whatever they hold)
        out[:, h], spread[:, h] = p @ held, p @ held.abs()
        if n:
            size[:, h] = (abs(scale) * (q[:, h].abs() @ torch.where(visible.any(0)[:, None], k, 0.0).abs().T)).amax(1)
    return out, spread, size


def waiting_times(key, vocab):
    """Exponential waiting times in float64: 24 bits per entry from a hash of (key, entry // 2)."""
    out = []
    for pair in range((vocab + 1) // 2):
        z = (key & MASK64) ^ (pair * 0xD1342543DE82EF95 & MASK64)
        z ^= z >> 32
        z = z * 0x94D049BB133111EB & MASK64
        z ^= z >> 29
        for bits in (z >> 40, (z >> 16) & 0xFFFFFF):
            out.append(-math.log1p(-(bits + 0.5) / (1 << 24)))
    return torch.tensor(out[:vocab], dtype=torch.float64)


def verify(logits, tokens, parents, temperature, uniforms, key, probs=None):
    """One request: logits [t, V]; returns (path, tokens, margin): how far, relative to what was compared, the nearest decision was from the other side."""
    V = logits.shape[1]
    x = logits.double().cpu()
    x = torch.where(torch.isnan(x), -math.inf, x).clamp(max=torch.finfo(torch.float32).max)
    here, path, out, margin = 0, [0], [], math.inf
    while True:
        row = x[here]
        children = [i for i in range(1, len(parents)) if parents[i] == here and 0 <= tokens[i] < V]
        top = float(row.max())
        if not temperature > 1e-10:
            final = int((row == top).nonzero()[0])
            onward = next((i for i in children if tokens[i] == final), None)
        else:
            r = torch.exp((row - top) / temperature) if top > -math.inf else torch.zeros(V, dtype=torch.float64)
            r = r / r.sum() if r.sum() > 0 else r
            onward = None
            for i in children:
                q = torch.zeros(V, dtype=torch.float64) if probs is None else probs[here].double().cpu()
                if probs is None:
                    q[tokens[i]] = 1.0
                left, right = float(uniforms[i]) * float(q[tokens[i]]), float(r[tokens[i]])
                margin = min(margin, abs(left - right) / max(left, right, 1e-30)) if right > 0 else margin
                if left < right:
                    onward = i
                    break
                rest = torch.clamp(r - q, min=0)
                if float(rest.sum()) > 0:
                    r = rest / rest.sum()
        if onward is None:
            break
        path.append(onward)
        out.append(int(tokens[onward]))
        here = onward
    if temperature > 1e-10:
        score = r / waiting_times(int(key), V)
        best = score.topk(min(2, V)).values
        if V > 1 and float(best[0]) > 0:
            margin = min(margin, float((best[0] - best[1]) / best[0]))
        final = int((score == score.max()).nonzero()[0])
    return path, out + [final], margin


def lookup(line, depth, branches, longest, shortest):
    """Tokens and parents of the tree that a request's tokens give."""
    if not line:
        return [], []
    n, found = len(line), []
    for j in range(n - 1):
        m = 0
        while m < longest and m <= j and line[j - m] == line[n - 1 - m]:
            m += 1
        if m >= shortest:
            found.append((m, j))
    tokens, parents, firsts = [line[-1]], [-1], set()
    for m, j in sorted(found, reverse=True):
        if len(firsts) == branches:
            break
        if line[j + 1] in firsts:
            continue
        firsts.add(line[j + 1])
        for k, x in enumerate(line[j + 1 : j + 1 + depth]):
            parents.append(0 if k == 0 else len(tokens) - 1)
            tokens.append(x)
    return tokens, parents
