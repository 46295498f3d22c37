"""What the ops for drafted tokens refuse, before any launch (no GPU: tensors without memory stand in)."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from tokensprint_b200 import ops
from tokensprint_b200.ops import KernelError


@pytest.fixture(autouse=True)
def device_zero(monkeypatch):
    monkeypatch.setattr(ops, "_raw_device", lambda: 0)
    monkeypatch.setattr(ops, "_stream", lambda: 0)

    def launched(*a):
        raise AssertionError("launched")

    monkeypatch.setattr(ops, "_fn", lambda name: launched)
    monkeypatch.setattr(ops, "_attention_tree_fns", lambda d: (launched, launched))


I32, I64, F32, BF16 = torch.int32, torch.int64, torch.float32, torch.bfloat16


def fake(*shape, dtype=I32, device="cuda:0"):
    return torch.empty(shape, dtype=dtype, device=device)


def attend(**change):
    with FakeTensorMode():
        a = {"q": fake(6, 512, dtype=BF16), "k_cache": fake(9, 16, 2, 128, dtype=BF16), "v_cache": fake(9, 16, 2, 128, dtype=BF16), "out": fake(6, 512, dtype=BF16),
             "tree_mask": fake(6, 1, dtype=I64), "cu_seqlens_q": fake(3), "context_lens": fake(2), "block_table": fake(2, 4), "page_size": 16, "num_seqs": 2,
             "max_seqlen_q": 3, "max_context": 50, "num_heads": 4, "num_kv_heads": 2, "head_dim": 128, "scale": 0.1}
        for k, v in change.items():
            a[k] = v() if callable(v) else v
        ops.attention_tree(**a)


@pytest.mark.parametrize("change,why", [
    ({"q": lambda: fake(6, 512, dtype=torch.float16), "k_cache": lambda: fake(9, 16, 2, 128, dtype=torch.float16),
      "v_cache": lambda: fake(9, 16, 2, 128, dtype=torch.float16), "out": lambda: fake(6, 512, dtype=torch.float16)}, "float32 or bfloat16"),
    ({"k_cache": lambda: fake(9, 16, 2, 128, dtype=F32)}, "must be torch.bfloat16"),
    ({"q": lambda: fake(6, 512, dtype=BF16, device="cpu")}, "CUDA"),
    ({"q": lambda: fake(512, 6, dtype=BF16).t()}, "contiguous"),
    ({"q": lambda: fake(6, 512, dtype=BF16, device="cuda:1")}, "current device"),
    ({"num_heads": 3}, "no multiple"),
    ({"num_heads": 8}, "do not match"),
    ({"page_size": 8}, "caches must be"),
    ({"v_cache": lambda: fake(8, 16, 2, 128, dtype=BF16)}, "caches must be"),
    ({"max_seqlen_q": 0}, "1 to 256"),
    ({"max_seqlen_q": 257}, "1 to 256"),
    ({"max_seqlen_q": 65}, "tree_mask"),
    ({"tree_mask": lambda: fake(6, 1)}, "int64"),
    ({"tree_mask": lambda: fake(5, 1, dtype=I64)}, "tree_mask"),
    ({"block_table": lambda: fake(1, 4)}, "block_table"),
    ({"block_table": lambda: fake(2, 4, dtype=I64)}, "int32"),
    ({"cu_seqlens_q": lambda: fake(2)}, "shorter than the batch"),
    ({"context_lens": lambda: fake(1)}, "shorter than the batch"),
    ({"window": 5}, "positions"),
    ({"window": 5, "positions": lambda: fake(5)}, "positions"),
    ({"window": -1}, "negative"),
    ({"softcap": -1.0}, "negative"),
    ({"softcap": float("nan")}, "negative"),
    ({"softcap": float("inf")}, "finite"),
    ({"head_sinks": lambda: fake(5, dtype=F32)}, "one entry per query head"),
    ({"head_sinks": lambda: fake(4, dtype=BF16)}, "float32"),
])
def test_attention_refuses(change, why):
    with pytest.raises(KernelError, match=why):
        attend(**change)


def test_attention_of_nothing_launches_nothing():
    attend(num_seqs=0)


def test_head_sizes():
    assert [d for d in range(0, 300) if ops.attention_tree_supported(d)] == list(range(8, 257, 8))


def verify(**change):
    with FakeTensorMode():
        a = {"logits": fake(7, 90, dtype=F32), "tokens": fake(7), "parents": fake(7), "cu_seqlens": fake(3), "temperatures": fake(2, dtype=F32),
             "uniforms": fake(7, dtype=F32), "keys": fake(2, dtype=I64), "path": fake(2, 5), "next_tokens": fake(2, 5), "counts": fake(2), "num_seqs": 2, "max_nodes": 5}
        for k, v in change.items():
            a[k] = v() if callable(v) else v
        ops.verify_drafts(**a)


@pytest.mark.parametrize("change,why", [
    ({"logits": lambda: fake(7, 90, dtype=torch.float16)}, "float32 or bfloat16"),
    ({"logits": lambda: fake(7, 90, dtype=F32, device="cpu")}, "CUDA"),
    ({"logits": lambda: fake(90, 7, dtype=F32).t()}, "neighbouring"),
    ({"logits": lambda: fake(1, 90, dtype=F32).expand(7, 90)}, "overlap"),
    ({"logits": lambda: fake(7, 0, dtype=F32)}, "vocabulary"),
    ({"logits": lambda: fake(7, (1 << 20) + 1, dtype=BF16)}, "vocabulary"),
    ({"tokens": lambda: fake(6)}, "tokens needs 7"),
    ({"tokens": lambda: fake(7, dtype=I64)}, "int32"),
    ({"parents": lambda: fake(6)}, "parents needs 7"),
    ({"uniforms": lambda: fake(6, dtype=F32)}, "uniforms needs 7"),
    ({"cu_seqlens": lambda: fake(2)}, "cu_seqlens needs 3"),
    ({"temperatures": lambda: fake(1, dtype=F32)}, "temperatures needs 2"),
    ({"keys": lambda: fake(2)}, "int64"),
    ({"counts": lambda: fake(1)}, "counts needs 2"),
    ({"max_nodes": 6}, "path and next_tokens"),
    ({"max_nodes": 0}, "1 to 256"),
    ({"max_nodes": 257}, "1 to 256"),
    ({"next_tokens": lambda: fake(2, 6)}, "path and next_tokens"),
    ({"draft_probs": lambda: fake(7, 90, dtype=BF16)}, "draft_probs"),
    ({"draft_probs": lambda: fake(6, 90, dtype=F32)}, "draft_probs"),
    ({"keys": lambda: fake(2, dtype=I64, device="cuda:1")}, "current device"),
])
def test_verification_refuses(change, why):
    with pytest.raises(KernelError, match=why):
        verify(**change)


@pytest.mark.parametrize("pools,why", [
    (lambda: [], "at least one"),
    (lambda: [fake(4, 16, 2, 8, dtype=BF16), fake(4, 16, 2, 8, dtype=F32)], "must be"),
    (lambda: [fake(4, 16, 2, 8, dtype=BF16), fake(5, 16, 2, 8, dtype=BF16)], "one shape"),
    (lambda: [fake(4, 16, dtype=BF16)], "one shape"),
    (lambda: [fake(4, 16, 3, dtype=torch.uint8)], "even number"),
    (lambda: [fake(4, 16, 2, 8, dtype=BF16).transpose(1, 2)], "contiguous"),
])
def test_pools_of_rows_are_refused(pools, why):
    with FakeTensorMode(), pytest.raises(KernelError, match=why):
        ops.RowPools(pools())


def keep(**change):
    with FakeTensorMode():
        pools = object.__new__(ops.RowPools)
        pools.pools, pools.num_pages, pools.page_size, pools.row_bytes, pools.align, pools.addresses = [None], 4, 16, 32, 16, fake(1, dtype=I64)
        a = {"pools": pools, "path": fake(2, 5), "counts": fake(2), "cu_seqlens": fake(3), "context_lens": fake(2), "block_table": fake(2, 4), "page_size": 16, "num_seqs": 2}
        for k, v in change.items():
            a[k] = v() if callable(v) else v
        ops.keep_drafted_rows(**a)


@pytest.mark.parametrize("change,why", [
    ({"page_size": 32}, "pages of 32"),
    ({"path": lambda: fake(1, 5)}, "row per request"),
    ({"path": lambda: fake(2, 5, dtype=I64)}, "int32"),
    ({"block_table": lambda: fake(8)}, "row per request"),
    ({"counts": lambda: fake(1)}, "counts needs 2"),
    ({"cu_seqlens": lambda: fake(2)}, "cu_seqlens needs 3"),
    ({"context_lens": lambda: fake(1)}, "context_lens needs 2"),
    ({"counts": lambda: fake(2, device="cuda:1")}, "current device"),
])
def test_keeping_rows_refuses(change, why):
    with pytest.raises(KernelError, match=why):
        keep(**change)


def look(**change):
    with FakeTensorMode():
        a = {"history": fake(2, 90), "lengths": fake(2), "tokens": fake(2, 7), "parents": fake(2, 7), "counts": fake(2), "num_seqs": 2, "depth": 3, "branches": 2}
        for k, v in change.items():
            a[k] = v() if callable(v) else v
        ops.lookup_drafts(**a)


@pytest.mark.parametrize("change,why", [
    ({"history": lambda: fake(2, 90, dtype=I64)}, "int32 CUDA matrix"),
    ({"history": lambda: fake(1, 90)}, "row per request"),
    ({"history": lambda: fake(2, 0)}, "empty"),
    ({"history": lambda: fake(2, (1 << 30) + 1)}, "at most 1073741824 tokens"),
    ({"history": lambda: fake(1, 90).expand(2, 90)}, "overlap"),
    ({"depth": 0}, "depth 1"),
    ({"depth": 65}, "depth 1"),
    ({"branches": 17}, "branches 1"),
    ({"min_suffix": 0}, "min_suffix"),
    ({"min_suffix": 5}, "min_suffix"),
    ({"max_suffix": 17}, "max_suffix"),
    ({"depth": 4}, "must be"),
    ({"tokens": lambda: fake(1, 7)}, "must be"),
    ({"lengths": lambda: fake(1)}, "lengths needs 2"),
    ({"counts": lambda: fake(1)}, "counts needs 2"),
    ({"lengths": lambda: fake(2, device="cuda:1")}, "current device"),
])
def test_lookup_refuses(change, why):
    with pytest.raises(KernelError, match=why):
        look(**change)


# ---------------------------------------------------------------------------
# the engine's side


def test_a_tree_is_cut_to_a_depth():
    from tokensprint_b200.engine.speculation import Tree

    tree = Tree([9, 1, 2, 3, 4, 5, 6], [-1, 0, 1, 2, 0, 4, 1])
    assert tree.cut(9) == tree
    assert tree.cut(1) == Tree([9, 1, 4], [-1, 0, 0])
    assert tree.cut(2) == Tree([9, 1, 2, 4, 5, 6], [-1, 0, 1, 0, 3, 1])
    assert tree.cut(0) == tree.root() == Tree([9], [-1])


def test_places_of_drafts_that_were_not_accepted_go_back():
    from tokensprint_b200.cache.manager import CacheError, CacheManager, GroupSpec

    cm = CacheManager([GroupSpec("full"), GroupSpec("window", 32)], 16, [10, 10], 4)
    rc = cm.admit("a")
    cm.extend(rc, 0, 100)
    cm.extend(rc, 100, 130)
    kept = [t[:7] for t in rc.tables]
    cm.retract(rc, 103)
    assert rc.num_tokens == 103 and [len(t) for t in rc.tables] == [7, 7] and rc.tables == kept
    cm.check_invariants()
    cm.extend(rc, 103, 125)
    cm.check_invariants()
    for tokens in (126, -1):
        with pytest.raises(CacheError, match="cannot retract"):
            cm.retract(rc, tokens)
    cm.retract(rc, 125)
    cm.free(rc)
    cm.check_invariants()
    with pytest.raises(CacheError, match="freed"):
        cm.retract(rc, 5)


def test_options_that_do_not_go_together(tmp_path):
    from tokensprint_b200.config.engine_config import Config

    Config(model=str(tmp_path), speculate=4, speculate_branches=2)
    for bad in ({"speculate": -1}, {"speculate": 2, "speculate_branches": 0}, {"speculate": 2, "speculate_suffix": 0}, {"speculate": 2, "cache_format": "kv4"}):
        with pytest.raises(ValueError, match="speculate"):
            Config(model=str(tmp_path), **bad)


def test_layers_that_take_tokens_one_behind_the_other_say_so():
    from tokensprint_b200.parts.base import Mixer

    assert "one behind the other" in Mixer.tree_refusal(object.__new__(Mixer))
