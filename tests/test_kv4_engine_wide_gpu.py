"""The engine with its cache in 4 bits and heads of 128 in bfloat16: portions of prompts on tcgen05, sliding layers, budgets."""

import pytest
import torch

from tests.plain import qwen3_plain as plain
from tests.replay_helpers import make_folder, random_tokens
from tests.test_kv4_edges_gpu import spoil_workspaces
from tests.test_kv4_engine_gpu import TINY, make_runner, quantising, run_portions

pytestmark = pytest.mark.gpu

WIDE = {**TINY, "head_dim": 128, "num_attention_heads": 8, "max_position_embeddings": 1024}
SLIDING = {**WIDE, "use_sliding_window": True, "sliding_window": 130, "layer_types": ["full_attention", "sliding_attention", "sliding_attention"]}


def rounded(weights):
    return {k: v.bfloat16().float() for k, v in weights.items()}


@pytest.mark.parametrize("cfg", [WIDE, SLIDING], ids=["full", "sliding"])
@pytest.mark.parametrize("cuts", [[500], [200, 170, 130], [330, 1, 169]])
def test_portions_in_bfloat16(tmp_path, monkeypatch, cfg, cuts):
    """Against the plain model on the rounded weights whose rows are held in 4 bits.  The yardstick is the same plain model with every activation
    rounded to bfloat16 (some codes then fall to their neighbours): the engine, which rounds at about the same places, is within one and a half of
    its distance.  (Seen with plain models: a window of 150 instead of 130 keys alone changes as much as 1.6 of it.)  And whatever the
    workspaces held before, the bits are the same."""
    folder, weights = make_folder(tmp_path, cfg, 5, sharp=1.0)
    ids = random_tokens(cfg, 500, 9)
    runner = make_runner(folder, "bfloat16", num_pages=128, max_model_len=1024)
    got, rc = run_portions(runner, ids, cuts)
    runner.free(rc)
    with monkeypatch.context() as m:
        spoil_workspaces(m)
        again, rc = run_portions(runner, ids, cuts, "b")
    runner.free(rc)
    assert torch.isfinite(got).all() and torch.equal(got, again)
    quantising(monkeypatch)
    want = plain.forward_logits(rounded(weights), cfg, ids)
    yard = plain.forward_logits(rounded(weights), cfg, ids, rounding=plain.round_to_bfloat16)
    assert (got.cpu().double() - want).norm() < 1.5 * (yard - want).norm()
    assert runner.cache_manager.pages_in_use() == 0


def checked_engine(monkeypatch, folder, config, **kw):
    """An engine whose requests are looked at after every step: [rows that one was cut from], and no request may hold more than the
    budget and its slack."""
    from tokensprint_b200.cache.manager import CacheManager
    from tokensprint_b200.config.engine_config import Config
    from tokensprint_b200.engine.llm_engine import LLMEngine
    from tokensprint_b200.engine.runner import ModelRunner
    from tokensprint_b200.models.api import load_model

    cuts, shrink, step = [], CacheManager.shrink, ModelRunner.step

    def counting(self, rc, rows):
        cuts.append((rc.request, rc.num_tokens))
        shrink(self, rc, rows)

    def looking(self, entries, *args, **kw):
        logits = step(self, entries, *args, **kw)
        assert all(e.cache.num_tokens <= config["cache_budget"] + config["cache_slack"] for e in entries)
        self.cache_manager.check_invariants()
        return logits

    monkeypatch.setattr(CacheManager, "shrink", counting)
    monkeypatch.setattr(ModelRunner, "step", looking)
    model, _ = load_model(folder, device="cuda", dtype="bfloat16")
    return LLMEngine(model, Config(model=str(folder), max_model_len=1024, max_num_seqs=4, chunked_prefill=True, enforce_eager=False, cache_format="kv4",
                                   **config, **kw)), cuts


@pytest.mark.parametrize("overlap", [True, False])
def test_a_prompt_larger_than_the_pool_through_the_entry_point(tmp_path, monkeypatch, overlap):
    """Six pages of 16 rows, prompts of up to 700 tokens: cut after every portion, they run."""
    from tokensprint_b200.config.engine_config import SamplingParams

    folder, _ = make_folder(tmp_path, WIDE, 7)
    config = dict(cache_budget=48, cache_recent=16, cache_slack=16, num_kvcache_blocks=6, kvcache_block_size=16, max_num_batched_tokens=32)
    engine, cuts = checked_engine(monkeypatch, folder, config, overlap_steps=overlap)
    prompts = [random_tokens(WIDE, n, 60 + n) for n in (700, 20, 333)]
    out = engine.generate(prompts, SamplingParams(temperature=0.0, max_tokens=60, ignore_eos=True), use_tqdm=False)
    assert [len(o) for o in out] == [60] * 3
    # of n + 59 tokens that were stored at most 64 have a row at the end
    dropped = {}
    for request, rows in cuts:
        dropped[request] = dropped.get(request, 0) + rows - 48
    assert len(dropped) == 3 and all(gone >= n + 59 - 64 for gone, n in zip(sorted(dropped.values()), (20, 333, 700)))
    assert engine.model_runner.cache_manager.pages_in_use() == 0


def test_a_budget_with_portions_on_tensor_memory(tmp_path, monkeypatch):
    """What a step's queries give to the rows adds up to one a query and head; a cut keeps the rows with the largest sums; and with other
    contents of the workspaces every bit is the same.  (The weights' own bound, as in check_attention: 4 * 2^-18 (reach + 1), with rows
    of norm 11.3 a reach below 15: 2^-12.)"""
    from tests.plain import kv4_plain
    from tokensprint_b200 import ops

    folder, _ = make_folder(tmp_path, SLIDING | {"use_sliding_window": False, "layer_types": ["full_attention"] * 3}, 11)
    ids = random_tokens(WIDE, 900, 12)
    budget, recent, first, slack = 256, 32, 4, 64
    runner = make_runner(folder, "bfloat16", num_pages=128, max_model_len=1024, cache_budget=budget, cache_recent=recent, cache_first=first, cache_slack=slack)
    evict, seen = ops.kv4_evict, []

    def checked(pool, sums, table, lens, new, num_seqs, longest, *rest):
        rows = int(lens[0])
        pages = table[0].long().clamp(min=0)
        flat = sums[pages].transpose(0, 1).flatten(1)[:, :rows].cpu()
        evict(pool, sums, table, lens, new, num_seqs, longest, *rest)
        after = sums[pages].transpose(0, 1).flatten(1)[:, :rows].cpu()
        for w, x in zip(flat, after):
            kept = kv4_plain.kept_rows(w.tolist(), budget, recent, first)
            assert torch.equal(x[:budget], w[kept]) and bool((x[budget:] == 0).all())
        seen.append(rows)

    monkeypatch.setattr(ops, "kv4_evict", checked)
    cuts = [300, 250, 1, 63, 1, 100, 185]
    got, rc = run_portions(runner, ids, cuts[:1])
    for sums in runner.cache_tensors.sums:  # nothing is cut yet
        total = sums[torch.tensor(rc.tables[0], device=sums.device)].double().sum((0, 2))
        assert ((total - 300 * 4).abs() <= 2.0**-12 * 300 * 4).all() and seen == []
    runner.free(rc)
    got, rc = run_portions(runner, ids, cuts, "b")
    assert seen == [550] * 3 + [321] * 3 + [356] * 3 + [441] * 3 and rc.num_tokens == 256
    runner.free(rc)
    with monkeypatch.context() as m:
        spoil_workspaces(m)
        again, rc = run_portions(runner, ids, cuts, "c")
    assert torch.isfinite(got).all() and torch.equal(got, again)
