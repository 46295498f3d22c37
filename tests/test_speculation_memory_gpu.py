"""Pages sized from free memory leave room for the steps that check drafts."""

import pytest
import torch

from tests.replay_helpers import make_folder, random_tokens

pytestmark = pytest.mark.gpu

CFG = {
    "architectures": ["Qwen3ForCausalLM"], "model_type": "qwen3", "num_hidden_layers": 2, "hidden_size": 96, "num_attention_heads": 4,
    "num_key_value_heads": 2, "head_dim": 64, "intermediate_size": 160, "vocab_size": 30000, "rope_theta": 10000.0, "rms_norm_eps": 1e-6,
    "tie_word_embeddings": True, "max_position_embeddings": 512, "hidden_act": "silu", "attention_bias": False, "torch_dtype": "float32",
}
SEQS, LENGTH, DEPTH, BRANCHES = 24, 256, 4, 3
ROWS = SEQS * (1 + DEPTH * BRANCHES)


def engine(folder, **options):
    from tokensprint_b200.config.engine_config import Config
    from tokensprint_b200.engine.llm_engine import LLMEngine
    from tokensprint_b200.models.api import load_model

    model, _ = load_model(folder, device="cuda", dtype="float32")
    return LLMEngine(model, Config(model=str(folder), dtype="float32", eos=7, max_num_batched_tokens=512, max_num_seqs=SEQS, max_model_len=LENGTH,
                                   gpu_memory_utilization=0.02, **options))


def test_sizing_counts_a_row_of_logits_for_every_node(tmp_path):
    from tokensprint_b200.engine.runner import StepEntry

    folder, _ = make_folder(tmp_path, CFG, 3)
    plain = engine(folder).model_runner.sizing
    runner = engine(folder, speculate=DEPTH, speculate_branches=BRANCHES).model_runner
    sized = runner.sizing
    logits = ROWS * CFG["vocab_size"] * 4
    assert sized["step_peak_bytes"] >= logits > 2 * plain["step_peak_bytes"]
    assert plain["reserved_bytes"] == 0 and sized["reserved_bytes"] == SEQS * LENGTH * 4  # (every request's tokens)
    assert sized["pages"] * sized["bytes_per_page"] <= sized["free_bytes"] * 0.02 - sized["step_peak_bytes"] - sized["reserved_bytes"] - sized["margin_bytes"]
    # a step in which every request brings a full tree takes no more than was measured (and its own small arrays)
    nodes = ROWS // SEQS
    parents = [-1] + [0 if i % DEPTH == 0 else i for i in range(nodes - 1)]
    entries = []
    for i in range(SEQS):
        cache = runner.cache_manager.admit(i)
        runner.cache_manager.extend(cache, 0, nodes)
        entries.append(StepEntry(cache, random_tokens(CFG, nodes, i), 0, range(nodes), parents=parents))
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = runner.step(entries)
    torch.cuda.synchronize()
    assert out.shape == (ROWS, CFG["vocab_size"])
    assert torch.cuda.max_memory_allocated() - before <= sized["step_peak_bytes"] + (4 << 20)
