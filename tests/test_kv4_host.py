"""The host side of the 4-bit cache: rows that a request gives up, options, sizes (no GPU)."""

import pytest

from tokensprint_b200 import ops
from tokensprint_b200.cache.manager import CacheError, CacheManager, GroupSpec
from tokensprint_b200.cache.tensors import page_bytes
from tokensprint_b200.config.engine_config import Config
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
