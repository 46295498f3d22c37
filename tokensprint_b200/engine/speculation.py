"""Drafted tokens: proposed from a request's own tokens, checked by the model's next step.

A decoding request brings a small tree to a step: its newest token and, hanging on it, chains of guesses (ops.lookup_drafts: what
followed the earlier occurrences of its last few tokens).  The step runs all nodes at once; ops.verify_drafts walks down the guesses that the model's
probabilities accept and draws the token behind them, and the accepted nodes' rows of the cache move to where their positions are.  The tokens
that come out are distributed as those of plain decoding.  Which ones they are is, unlike there, no function of (seed, stream, position) alone: the numbers that decide
belong to the position where a step's tree begins, the token behind a prompt is drawn by the sampler, and where a tree begins and what it holds depends on portions, on
the budget and pages that drafts find, and on preemption.  With room for all of them, the batch does not matter.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Sequence as Seq

import numpy as np
import torch

from tokensprint_b200 import ops
from tokensprint_b200.engine.runner import ModelRunner
from tokensprint_b200.engine.sequence import Sequence
from tokensprint_b200.sampling.sampler import sample_key


@dataclass
class Tree:
    """A request's newest token and the guesses behind it; every node's parent comes before it."""

    tokens: list[int]
    parents: list[int]  # -1: the first

    def __len__(self) -> int:
        return len(self.tokens)

    def root(self) -> "Tree":
        return Tree(self.tokens[:1], [-1])

    def cut(self, depth: int) -> "Tree":
        """Without the nodes further than `depth` from the first."""
        place: dict[int, int] = {-1: -1}
        far: dict[int, int] = {-1: -1}
        out = Tree([], [])
        for i, (token, parent) in enumerate(zip(self.tokens, self.parents)):
            far[i] = far[parent] + 1
            if far[i] <= depth and parent in place:
                place[i] = len(out.tokens)
                out.tokens.append(token)
                out.parents.append(place[parent])
        return out


def _uniforms(key: int, count: int) -> np.ndarray:
    """`count` numbers in [0, 1) of 24 bits, a pure function of the key."""
    z = np.uint64(key & (1 << 64) - 1) + np.arange(1, count + 1, dtype=np.uint64) * np.uint64(0x9E3779B97F4A7C15)
    z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
    z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
    return ((z ^ (z >> np.uint64(31))) >> np.uint64(40)).astype(np.float32) * np.float32(2.0**-24)


class Speculator:
    @staticmethod
    def history_bytes(num_slots: int, max_model_len: int) -> int:
        """What it keeps on the device: every request's tokens."""
        return 4 * num_slots * max_model_len

    def __init__(self, runner: ModelRunner, depth: int, branches: int, suffix: int) -> None:
        for run in runner.model.spec.run_order:
            why = runner.model.blocks[run.layer].mixer.tree_refusal()
            if why is not None:
                raise ValueError(f"speculate: layer {run.layer}: {why}")
        if runner.kv4:
            raise ValueError("speculate needs cache_format 'model'")
        if depth > ops.LOOKUP_MAX_DEPTH or branches > ops.LOOKUP_MAX_BRANCHES or suffix > ops.LOOKUP_MAX_SUFFIX or 1 + depth * branches > ops.TREE_MAX_NODES:
            raise ValueError(f"speculate: at most {ops.LOOKUP_MAX_DEPTH} tokens a chain, {ops.LOOKUP_MAX_BRANCHES} chains, {ops.TREE_MAX_NODES} nodes and "
                             f"a suffix of {ops.LOOKUP_MAX_SUFFIX}, got {depth}, {branches}, {1 + depth * branches} and {suffix}")
        self.runner, self.depth, self.branches, self.suffix = runner, depth, branches, suffix
        self.device = runner.device
        self.length = runner.max_model_len
        self.history = torch.zeros((runner.num_slots, self.length), dtype=torch.int32, device=self.device)  # a row per state slot
        self._held: dict[int, tuple[int, int]] = {}  # slot -> (request, how many of its tokens the row holds)
        self.drafted = self.accepted = 0

    def propose(self, seqs: Seq[Sequence]) -> None:
        """Gives every sequence that decodes next (all its tokens but the newest cached) a tree."""
        seqs = [s for s in seqs if s.cache is not None and s.num_cached_tokens == len(s) - 1]
        if not seqs:
            return
        rows, places, tokens = [], [], []
        lengths = np.zeros(max(s.cache.slot for s in seqs) + 1, dtype=np.int32)
        for s in seqs:
            slot = s.cache.slot
            request, held = self._held.get(slot, (-1, 0))
            held = held if request == s.seq_id else 0
            fresh = s.token_ids[held:]
            rows += [slot] * len(fresh)
            places += range(held, len(s))
            tokens += fresh
            self._held[slot] = (s.seq_id, len(s))
            lengths[slot] = len(s)
        n, B, width = len(tokens), len(lengths), 1 + self.depth * self.branches
        packed = torch.from_numpy(np.concatenate([np.array(rows + places + tokens, dtype=np.int32), lengths])).pin_memory().to(self.device, non_blocking=True)
        self.history[packed[:n].long(), packed[n : 2 * n].long()] = packed[2 * n : 3 * n]
        out = torch.empty((2 * width + 1) * B, dtype=torch.int32, device=self.device)
        ops.lookup_drafts(self.history, packed[3 * n :], out[: width * B].view(B, width), out[width * B : 2 * width * B].view(B, width), out[2 * width * B :], B,
                          self.depth, self.branches, self.suffix)
        host = out.cpu().numpy()
        for s in seqs:
            slot = s.cache.slot
            count = int(host[2 * width * B + slot])
            tree = Tree(host[slot * width : slot * width + count].tolist(), host[(B + slot) * width : (B + slot) * width + count].tolist())
            # no further than the request may go: behind the accepted ones one more token comes in any case
            s.tree = tree.cut(max(0, min(self.depth, s.max_tokens - s.num_completion_tokens - 1, self.length - 1 - len(s))))

    def verify(self, logits: torch.Tensor, seqs: Seq[Sequence]) -> list[list[int]]:
        """The accepted drafts and the token behind them, for every sequence with a tree; logits [all nodes, V] of the step that ran them.  Moves
        the accepted rows; waits for the device."""
        sizes = [len(s.tree) for s in seqs]
        T, B, most = sum(sizes), len(seqs), max(sizes)
        cu = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
        uniforms = np.concatenate([_uniforms(sample_key(s.seed ^ 0x5DEECE66D, s.sample_stream, len(s)), n) for s, n in zip(seqs, sizes)])
        keys = np.array([sample_key(s.seed, s.sample_stream, len(s)) for s in seqs], dtype=np.int64)
        words = [keys.view(np.int32), np.array(sum((s.tree.tokens for s in seqs), []), dtype=np.int32), np.array(sum((s.tree.parents for s in seqs), []), dtype=np.int32),
                 cu, np.array([s.temperature for s in seqs], dtype=np.float32).view(np.int32), uniforms.view(np.int32)]
        packed = torch.from_numpy(np.concatenate(words)).pin_memory().to(self.device, non_blocking=True)
        key_words, tokens, parents, cu_dev, temps, u = packed.split([len(w) for w in words])
        out = torch.empty(B * (2 * most + 1), dtype=torch.int32, device=self.device)
        path, fresh, counts = out[: B * most].view(B, most), out[B * most : 2 * B * most].view(B, most), out[2 * B * most :]
        ops.verify_drafts(logits, tokens, parents, cu_dev, temps.view(torch.float32), u.view(torch.float32), key_words.view(torch.int64), path, fresh, counts, B, most)
        self.runner.keep_drafted(path, counts)
        host = out.cpu().numpy()
        taken = host[2 * B * most :]
        self.drafted += T - B
        self.accepted += int(taken.sum())
        return [host[(B + b) * most : (B + b) * most + int(taken[b]) + 1].tolist() for b in range(B)]
