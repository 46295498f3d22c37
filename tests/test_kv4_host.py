"""The host side of the 4-bit cache: rows that a request gives up, options, sizes (no GPU)."""

import pytest

from tokensprint_b200 import ops
from tokensprint_b200.cache.manager import CacheError, CacheManager, GroupSpec
from tokensprint_b200.cache.tensors import page_bytes
from tokensprint_b200.config.engine_config import Config, SamplingParams
from tokensprint_b200.engine.scheduler import Scheduler
from tokensprint_b200.engine.sequence import Sequence
from tokensprint_b200.parts.base import CacheNeed


def test_a_shrunk_request_gives_pages_back_and_goes_on():
    cm = CacheManager([GroupSpec("full")], 16, [10], 4)
    rc = cm.admit("a")
    cm.extend(rc, 0, 100)
    assert len(rc.tables[0]) == 7
    kept = list(rc.tables[0][:3])
    cm.shrink(rc, 40)
    assert rc.num_tokens == 40 and rc.dropped == 60 and rc.tables[0] == kept
    assert cm.pages_in_use() == 3
    cm.check_invariants()
    # the token at position 100 has the row 40
    assert cm.can_extend(rc, 100, 101)
    cm.extend(rc, 100, 101)
    assert list(cm.slots_for(rc, 0, 100, 1)) == [kept[2] * 16 + 8]
    cm.extend(rc, 101, 120)
    assert rc.num_tokens == 60 and len(rc.tables[0]) == 4
    cm.shrink(rc, 48)
    assert rc.dropped == 72 and len(rc.tables[0]) == 3
    cm.check_invariants()
    cm.free(rc)
    assert cm.pages_in_use() == 0
    cm.check_invariants()


def test_shrinking_is_refused_where_it_has_no_meaning():
    cm = CacheManager([GroupSpec("full"), GroupSpec("window", 32)], 16, [10, 10], 4)
    rc = cm.admit("a")
    cm.extend(rc, 0, 20)
    with pytest.raises(CacheError, match="every group"):
        cm.shrink(rc, 10)
    cm = CacheManager([GroupSpec("full")], 16, [10], 4)
    rc = cm.admit("a")
    cm.extend(rc, 0, 20)
    for rows in (0, 21, -3):
        with pytest.raises(CacheError, match="cannot cut"):
            cm.shrink(rc, rows)
    cm.free(rc)
    with pytest.raises(CacheError, match="freed"):
        cm.shrink(rc, 5)


def test_sizes_of_the_pool():
    assert ops.kv4_pool_shape(7, 48, 2, 128) == (7, 2, 3, 18 * 128)
    need = CacheNeed(kind="full", kv_heads=8, head_dim=128)
    assert page_bytes([need], [0], 0, 16, 2, kv4=True) == 16 * 8 * 144
    assert page_bytes([need], [0], 0, 16, 2, kv4=True, weighed=True) == 16 * 8 * 148
    assert page_bytes([need], [0], 0, 16, 2) == 16 * 8 * 512
    for bad in ((4, 16, 2, 96), (4, 24, 2, 128), (4, 0, 2, 128)):
        with pytest.raises(ops.KernelError):
            ops.kv4_pool_shape(*bad)


def test_options(tmp_path):
    assert Config(model=str(tmp_path), cache_format="kv4", cache_budget=512).cache_recent == 64
    with pytest.raises(ValueError, match="cache_format"):
        Config(model=str(tmp_path), cache_format="int3")
    with pytest.raises(ValueError, match="cache_budget"):
        Config(model=str(tmp_path), cache_budget=512)
    with pytest.raises(ValueError, match="cache_budget"):
        Config(model=str(tmp_path), cache_format="kv4", cache_budget=-1)


def budgeted(tmp_path, budget, **kw):
    options = dict(num_kvcache_blocks=6, kvcache_block_size=16, max_num_batched_tokens=32, max_num_seqs=4, max_model_len=4096, chunked_prefill=True,
                   cache_format="kv4", cache_budget=budget, cache_recent=8, cache_slack=16)
    options.update(kw)
    config = Config(model=str(tmp_path), **options)
    cm = CacheManager([GroupSpec("full")], 16, [options["num_kvcache_blocks"]], options["max_num_seqs"])
    return Scheduler(config, cm), config


def test_a_budget_admits_prompts_longer_than_the_pool(tmp_path):
    """48 + 16 + 32 rows at most: six pages of 16 carry any prompt that comes in portions, alone and beside others."""
    s, config = budgeted(tmp_path, 48)
    seqs = [Sequence([1] * n, SamplingParams(max_tokens=40, ignore_eos=True)) for n in (700, 90, 333)]
    for x in seqs:
        s.add_sequence(x)
    most = steps = 0
    while not s.is_finished():
        step = s.schedule()
        need = [i for i, x in enumerate(step) if x.num_cached_tokens + x.num_new_tokens == len(x)]
        for x in step:  # what the runner does behind a step
            most = max(most, x.cache.num_tokens)
            if x.cache.num_tokens > config.cache_budget + config.cache_slack:
                s.cache_manager.shrink(x.cache, config.cache_budget)
        s.postprocess(step, [1] * len(need), need)
        s.cache_manager.check_invariants()
        steps += 1
        assert steps < 5000
    assert [x.num_completion_tokens for x in seqs] == [40] * 3 and most <= 96
    assert s.cache_manager.pages_in_use() == 0


def test_what_a_budget_does_not_admit(tmp_path):
    for kw in (dict(budget=0), dict(budget=49), dict(budget=48, num_kvcache_blocks=5), dict(budget=48, cache_slack=17)):
        if not kw["budget"]:
            kw["cache_format"] = "model"
        s, _ = budgeted(tmp_path, **kw)
        with pytest.raises(ValueError, match="never be scheduled"):
            s.add_sequence(Sequence([1] * 700, SamplingParams()))
    s, _ = budgeted(tmp_path, 48, chunked_prefill=False, max_num_batched_tokens=1024)  # the whole prompt at once needs all its pages
    with pytest.raises(ValueError, match="never be scheduled"):
        s.add_sequence(Sequence([1] * 700, SamplingParams()))
