"""Attention of a step that carries portions of prompts beside trees of drafted tokens, against plain float64."""

import pytest
import torch

from tests.plain import drafts_plain as plain
from tests.replay_helpers import make_folder
from tests.test_drafts_gpu import check
from tests.test_speculation_engine_gpu import NARROW, TINY, WINDOWED, engine

pytestmark = pytest.mark.gpu

PARENTS = [-1, 0, 1, 0, 3]


@pytest.mark.parametrize("portions", [[(0, 40), (0, 2)], [(60, 17), (0, 90), (5, 1)], [(33, 2), (100, 3)], [(140, 300)]], ids=["begin", "go on", "few rows", "long"])
@pytest.mark.parametrize("cfg,dtype,page,layer", [
    (TINY, "bfloat16", 16, 0), (WINDOWED, "bfloat16", 16, 1), (NARROW, "bfloat16", 16, 2), ({**TINY, "head_dim": 128}, "bfloat16", 16, 0),
    ({**TINY, "head_dim": 128}, "bfloat16", 12, 0), ({**TINY, "head_dim": 256}, "bfloat16", 16, 1), (TINY, "float32", 16, 0), (WINDOWED, "float32", 16, 1), (NARROW, "float32", 8, 0),
], ids=["64", "64 windowed", "24", "128", "128 pages of 12", "256", "64 float32", "64 windowed float32", "24 float32"])
def test_portions_beside_trees(tmp_path, cfg, dtype, page, layer, portions):
    """(bounds: see test_drafts_gpu.check; a portion is a chain whose every token sees those before it)"""
    from tokensprint_b200.engine.runner import StepEntry

    folder, _ = make_folder(tmp_path, cfg, 12)
    runner = engine(folder, dtype, kvcache_block_size=page, max_num_batched_tokens=512, max_model_len=512).model_runner
    mixer, cache, m = runner.model.blocks[layer].mixer, runner.layer_caches[layer], runner.cache_manager
    gen = torch.Generator("cuda").manual_seed(1)
    for pool in (cache.k_pages, cache.v_pages):
        pool.normal_(generator=gen)
    entries, lens, trees = [], [], []
    # trees first, and with them the portions of one token
    held = [(200, PARENTS), (37, PARENTS), (5, PARENTS)] + [(n, [-1]) for n, t in portions if t == 1] + [(n, list(range(-1, t - 1))) for n, t in portions if t > 1]
    for i, (before, parents) in enumerate(held):
        t = len(parents)
        rc = m.admit(i)
        m.extend(rc, 0, before)
        m.extend(rc, before, before + t)
        is_tree = i < 3 or t == 1
        entries.append(StepEntry(rc, [1] * t, before, range(t), parents=parents if is_tree else None))
        lens.append((before + t, t))
        trees.append(plain.ancestors(parents))
    step, _, _ = runner.build_context(entries)
    assert step.tree_seqs == sum(t == 1 for _, t in portions) + 3 and step.num_seqs == len(held)
    tables = step.groups[cache.group]
    nq, nkv, d = mixer.num_heads, mixer.num_kv_heads, mixer.head_dim
    T = sum(t for _, t in lens)
    q = (1.5 * torch.randn((T, nq * d), generator=gen, device="cuda")).to(cache.k_pages.dtype)
    out = torch.full_like(q, float("nan"))
    mixer._attend(q, out, step, cache, tables)
    rows = []
    for b, (n, _) in enumerate(lens):
        at = torch.arange(n, device="cuda")
        pages = tables.block_table[b].long()[at // page].clamp(min=0)  # (those given back lie outside the window)
        rows.append([pool[pages, at % page] for pool in (cache.k_pages, cache.v_pages)])
    check({"q": q, "rows": rows, "trees": trees, "positions": [[n - t + len(a) - 1 for a in tree] for (n, t), tree in zip(lens, trees)], "lens": lens, "nq": nq, "d": d},
          out, window=mixer.window, scale=mixer.scale)
