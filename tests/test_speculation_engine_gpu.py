"""The engine with drafted tokens: greedy tokens are those of plain decoding, whatever was guessed."""

import pytest
import torch

from tests.replay_helpers import make_folder, random_tokens

pytestmark = pytest.mark.gpu

TINY = {
    "architectures": ["Qwen3ForCausalLM"], "model_type": "qwen3", "num_hidden_layers": 3, "hidden_size": 96, "num_attention_heads": 4,
    "num_key_value_heads": 2, "head_dim": 64, "intermediate_size": 160, "vocab_size": 40, "rope_theta": 10000.0, "rms_norm_eps": 1e-6,
    "tie_word_embeddings": True, "max_position_embeddings": 512, "hidden_act": "silu", "attention_bias": False, "torch_dtype": "float32",
}
WINDOWED = {**TINY, "use_sliding_window": True, "sliding_window": 24, "layer_types": ["full_attention", "sliding_attention", "full_attention"]}
NARROW = {**TINY, "num_attention_heads": 6, "num_key_value_heads": 3, "head_dim": 24}


def engine(folder, dtype="float32", **options):
    from tokensprint_b200.config.engine_config import Config
    from tokensprint_b200.engine.llm_engine import LLMEngine
    from tokensprint_b200.models.api import load_model

    model, _ = load_model(folder, device="cuda", dtype=dtype)
    defaults = dict(max_num_batched_tokens=256, max_num_seqs=6, max_model_len=256, num_kvcache_blocks=120, dtype=dtype, eos=7)
    defaults.update(options)
    return LLMEngine(model, Config(model=str(folder), **defaults))


def prompts(cfg, seed=0):
    """Prompts that repeat themselves, so that their ends have been there before."""
    out = []
    for i, n in enumerate((5, 30, 61, 17, 90, 3, 44, 12)):
        piece = random_tokens(cfg, n, seed + i)
        out.append(piece + piece[: n // 2 + 1])
    return out


def run(e, ps, **sampling):
    from tokensprint_b200.config.engine_config import SamplingParams

    params = [SamplingParams(max_tokens=20 + 7 * i, ignore_eos=i % 2 == 0, seed=i, **sampling) for i in range(len(ps))]
    out = e.generate(ps, params, use_tqdm=False)
    e.model_runner.cache_manager.check_invariants()
    assert e.model_runner.cache_manager.pages_in_use() == 0
    return out


@pytest.mark.parametrize("cfg", [TINY, WINDOWED, NARROW], ids=["full", "windowed", "heads of 24"])
@pytest.mark.parametrize("depth,branches", [(1, 1), (4, 1), (3, 4), (9, 2)])
def test_greedy_tokens_are_those_of_plain_decoding(tmp_path, cfg, depth, branches):
    """Float32: the logits of a step differ from those of plain decoding in the order of sums only, far below the gaps between the largest ones."""
    folder, _ = make_folder(tmp_path, cfg, 5, sharp=2.0)
    want = run(engine(folder), prompts(cfg), temperature=0.0)
    e = engine(folder, speculate=depth, speculate_branches=branches)
    assert run(e, prompts(cfg), temperature=0.0) == want
    assert e.speculator.accepted > 0  # (a small model repeats itself)


def test_greedy_tokens_with_prompts_in_portions_and_few_pages(tmp_path):
    """Portions of prompts beside trees, drafts that find no pages, requests that lose their place."""
    folder, _ = make_folder(tmp_path, TINY, 6, sharp=2.0)
    want = run(engine(folder), prompts(TINY), temperature=0.0)
    e = engine(folder, speculate=4, speculate_branches=3, chunked_prefill=True, max_num_batched_tokens=40, num_kvcache_blocks=20, kvcache_block_size=16)
    assert run(e, prompts(TINY), temperature=0.0) == want
    assert e.scheduler.num_preemptions > 0


def test_a_request_ends_where_its_length_does(tmp_path):
    folder, _ = make_folder(tmp_path, TINY, 7, sharp=2.0)
    ps = [[3, 4] * 25]
    for limit in (52, 55, 64):
        want = run(engine(folder, max_model_len=limit), ps, temperature=0.0)
        assert run(engine(folder, max_model_len=limit, speculate=6, speculate_branches=2), ps, temperature=0.0) == want


def test_sampled_tokens_do_not_depend_on_the_batch(tmp_path):
    folder, _ = make_folder(tmp_path, TINY, 8, sharp=1.0)
    together = run(engine(folder, speculate=4, speculate_branches=2), prompts(TINY), temperature=1.0)
    again = run(engine(folder, speculate=4, speculate_branches=2, max_num_seqs=2), prompts(TINY), temperature=1.0)
    assert together == again
    assert all(0 <= t < TINY["vocab_size"] for out in together for t in out)


def test_bfloat16_steps_follow_the_largest_logits(tmp_path):
    """Each greedy token is, for a plain pass over the finished text, among the logits that bfloat16 cannot tell from the largest."""
    from tests.plain import qwen3_plain as plain

    cfg = {**TINY, "head_dim": 128}
    folder, weights = make_folder(tmp_path, cfg, 9, sharp=2.0)
    e = engine(folder, "bfloat16", speculate=5, speculate_branches=2, chunked_prefill=True, max_num_batched_tokens=64)
    ps = prompts(cfg)
    for p, out in zip(ps, run(e, ps, temperature=0.0)):
        logits = plain.forward_logits(weights, cfg, p + out)
        for i, t in enumerate(out):
            row = logits[len(p) + i - 1]
            assert row.max() - row[t] < 0.05 * (row.max() - row.min())


def test_models_that_cannot_are_refused(tmp_path):
    from tokensprint_b200.engine.speculation import Speculator

    folder, _ = make_folder(tmp_path, TINY, 5)
    with pytest.raises(ValueError, match="at most"):
        engine(folder, speculate=65)
    with pytest.raises(ValueError, match="nodes"):
        engine(folder, speculate=64, speculate_branches=4)
    runner = engine(folder).model_runner
    runner.model.blocks[1].mixer.chunk = 16  # a layer with blocks of positions
    with pytest.raises(ValueError, match="layer 1: attention over trees"):
        Speculator(runner, 4, 1, 4)
