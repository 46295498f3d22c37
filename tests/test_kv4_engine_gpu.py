"""The engine with its cache in 4 bits, and with a budget of rows, against the plain model."""

import pytest
import torch

from tests.plain import kv4_plain, qwen3_plain as plain
from tests.replay_helpers import make_folder, random_tokens

pytestmark = pytest.mark.gpu

TINY = {
    "architectures": ["Qwen3ForCausalLM"], "model_type": "qwen3", "num_hidden_layers": 3, "hidden_size": 96, "num_attention_heads": 4,
    "num_key_value_heads": 2, "head_dim": 64, "intermediate_size": 160, "vocab_size": 320, "rope_theta": 10000.0, "rms_norm_eps": 1e-6,
    "tie_word_embeddings": True, "max_position_embeddings": 512, "hidden_act": "silu", "attention_bias": False, "torch_dtype": "float32",
}
WINDOWED = {**TINY, "use_sliding_window": True, "sliding_window": 24, "layer_types": ["full_attention", "sliding_attention", "full_attention"]}


def held(x):
    """Rows [..., d] as a 4-bit cache gives them back (of their float32 values, as the engine has them)."""
    return kv4_plain.values_of(*kv4_plain.quantise(x.float().double()))


def quantising(monkeypatch):
    attention = plain.causal_attention
    monkeypatch.setattr(plain, "causal_attention", lambda q, k, v, **kw: attention(q, held(k), held(v), **kw))


def make_runner(folder, dtype="float32", **kw):
    from tokensprint_b200.engine.runner import ModelRunner
    from tokensprint_b200.models.api import load_model

    model, _ = load_model(folder, device="cuda", dtype=dtype)
    defaults = dict(page_size=16, num_pages=64, num_slots=8, max_num_batched_tokens=512, cache_format="kv4", max_model_len=512)
    defaults.update(kw)
    return ModelRunner(model, **defaults)


def run_portions(runner, ids, cuts, name="a"):
    """Logits of every token, the sequence given in portions."""
    from tokensprint_b200.engine.runner import StepEntry

    cm = runner.cache_manager
    rc = cm.admit(name)
    out, at = [], 0
    for n in cuts:
        cm.extend(rc, at, at + n)
        out.append(runner.step([StepEntry(rc, ids[at : at + n], at, list(range(n)))]).clone())
        at += n
    return torch.cat(out), rc


@pytest.mark.parametrize("cfg", [TINY, WINDOWED], ids=["full", "windowed"])
@pytest.mark.parametrize("cuts", [[90], [40, 1, 17, 1, 1, 30], [1] * 90])
def test_logits_are_those_of_the_model_with_quantised_rows(tmp_path, monkeypatch, cfg, cuts):
    """Float32 steps: what is left between the engine and the plain model whose keys and values are held in 4 bits is a few codes that
    fall on the other side of a half; it is far below what the 4 bits themselves change."""
    folder, weights = make_folder(tmp_path, cfg, 5, sharp=2.0)
    ids = random_tokens(cfg, 90, 9)
    exact = plain.forward_logits(weights, cfg, ids)
    quantising(monkeypatch)
    want = plain.forward_logits(weights, cfg, ids)
    runner = make_runner(folder, poison_freed_pages=True)
    got, rc = run_portions(runner, ids, cuts)
    changed = (want - exact).norm()
    assert (got.cpu().double() - want).norm() < 0.05 * changed
    runner.free(rc)
    runner.cache_manager.check_invariants()
    assert runner.cache_manager.pages_in_use() == 0


def test_bfloat16_decode_graphs_give_the_eager_logits(tmp_path):
    from tokensprint_b200.engine.runner import StepEntry

    folder, _ = make_folder(tmp_path, TINY, 6, sharp=2.0)
    prompts = [random_tokens(TINY, n, n) for n in (5, 33, 70)]
    logits = []
    for eager in (True, False):
        runner = make_runner(folder, "bfloat16", enforce_eager=eager)
        cm = runner.cache_manager
        rcs = []
        for i, p in enumerate(prompts):
            rc = cm.admit(i)
            cm.extend(rc, 0, len(p))
            rcs.append(rc)
        rows = [runner.step([StepEntry(rc, p, 0, [len(p) - 1]) for rc, p in zip(rcs, prompts)]).clone()]
        for k in range(20):
            for rc, p in zip(rcs, prompts):
                cm.extend(rc, len(p) + k, len(p) + k + 1)
            rows.append(runner.step([StepEntry(rc, [(7 * k + 3) % TINY["vocab_size"]], len(p) + k, [0]) for rc, p in zip(rcs, prompts)]).clone())
        assert eager or runner._graphs
        logits.append(torch.stack(rows))
    scale = logits[0].abs().max()
    # the same kernels on the same numbers; a batch padded to a graph's size may share key ranges out differently (sums in another order)
    assert (logits[0] - logits[1]).abs().max() < 2e-2 * scale


class WeighedPlain:
    """One sequence through the plain Qwen3 layers, token by token, with a 4-bit cache that is cut to a budget."""

    def __init__(self, weights, cfg, budget, recent, first, slack):
        self.w = {k: v.double() for k, v in weights.items()}
        self.cfg, self.budget, self.recent, self.first, self.slack = cfg, budget, recent, first, slack
        self.rows = [[([], [], []) for _ in range(cfg["num_key_value_heads"])] for _ in range(cfg["num_hidden_layers"])]  # keys, values, sums
        self.gaps = []  # how clearly every cut chose

    def step(self, ids, start):
        """Logits of the last of `ids` (positions from `start` on)."""
        c, w = self.cfg, self.w
        nq, nkv, d, eps = c["num_attention_heads"], c["num_key_value_heads"], c["head_dim"], c["rms_norm_eps"]
        h = plain.embedding(w["model.embed_tokens.weight"], ids)
        angles = plain.rope_angles(list(range(start, start + len(ids))), d, c["rope_theta"])
        for i in range(c["num_hidden_layers"]):
            p = f"model.layers.{i}."
            x = plain.rms_norm(h, w[p + "input_layernorm.weight"], eps)
            a = p + "self_attn."
            q, k, v = ((x @ w[a + n].T).view(len(ids), -1, d) for n in ("q_proj.weight", "k_proj.weight", "v_proj.weight"))
            q = plain.apply_rope(plain.rms_norm(q, w[a + "q_norm.weight"], eps), angles)
            k = held(plain.apply_rope(plain.rms_norm(k, w[a + "k_norm.weight"], eps), angles))
            v = held(v)
            out = torch.zeros_like(q)
            for g in range(nkv):
                keys, values, sums = self.rows[i][g]
                before = len(keys)
                keys += list(k[:, g])
                values += list(v[:, g])
                sums += [0.0] * len(ids)
                K, V = torch.stack(keys), torch.stack(values)
                for t in range(len(ids)):
                    n = before + t + 1
                    for head in range(g * nq // nkv, (g + 1) * nq // nkv):
                        prob = torch.softmax(K[:n] @ q[t, head] * d**-0.5, 0)
                        out[t, head] = prob @ V[:n]
                        for j in range(n):
                            sums[j] += float(prob[j])
            h = h + out.reshape(len(ids), -1) @ w[a + "o_proj.weight"].T
            h = h + plain.swiglu_ffn(plain.rms_norm(h, w[p + "post_attention_layernorm.weight"], eps), w, p + "mlp.")
        if len(self.rows[0][0][0]) > self.budget + self.slack:
            for layer in self.rows:
                for g, (keys, values, sums) in enumerate(layer):
                    kept = kv4_plain.kept_rows(sums, self.budget, self.recent, self.first)
                    middle = [j for j in range(self.first, len(sums) - self.recent)]
                    low = max(sums[j] for j in middle if j not in kept)
                    self.gaps.append(min(sums[j] for j in middle if j in kept) - low)
                    layer[g] = ([keys[j] for j in kept], [values[j] for j in kept], [sums[j] for j in kept])
        h = plain.rms_norm(h[-1:], w["model.norm.weight"], eps)
        return (h @ w["model.embed_tokens.weight"].T)[0]


@pytest.mark.parametrize("eager", [True, False])
def test_a_budget_keeps_the_rows_that_got_the_attention(tmp_path, eager):
    """A prompt in portions, then decoded tokens, cut again and again: rows, pages and logits are the plain cache's."""
    from tokensprint_b200.engine.runner import StepEntry

    folder, weights = make_folder(tmp_path, TINY, 8, sharp=2.0)
    budget, recent, first, slack = 32, 8, 2, 16
    runner = make_runner(folder, cache_budget=budget, cache_recent=recent, cache_first=first, cache_slack=slack, enforce_eager=eager, poison_freed_pages=True)
    oracle = WeighedPlain(weights, TINY, budget, recent, first, slack)
    ids = random_tokens(TINY, 110, 4)
    cm = runner.cache_manager
    rc = cm.admit("a")
    at = 0
    for n in [20, 13, 25] + [1] * 52:
        cm.extend(rc, at, at + n)
        got = runner.step([StepEntry(rc, ids[at : at + n], at, [n - 1])])[0].cpu().double()
        want = oracle.step(ids[at : at + n], at)
        at += n
        rows = len(oracle.rows[0][0][0])
        assert rc.num_tokens == rows and rc.dropped == at - rows and len(rc.tables[0]) == -(-rows // 16)
        cm.check_invariants()
        assert (got - want).abs().max() <= 2e-2 * want.abs().max(), at
    assert rc.dropped > 0 and min(oracle.gaps) > 0
    runner.free(rc)
    assert cm.pages_in_use() == 0


def test_generation_with_a_budget_through_the_entry_point(tmp_path):
    """Several requests of different lengths, graphs and overlapping steps; a budget that nobody reaches changes nothing."""
    from tokensprint_b200.config.engine_config import Config, SamplingParams
    from tokensprint_b200.engine.llm_engine import LLMEngine
    from tokensprint_b200.models.api import load_model

    folder, _ = make_folder(tmp_path, TINY, 7, sharp=2.0)
    prompts = [random_tokens(TINY, n, 60 + n) for n in (4, 50, 90, 130)]
    out = {}
    for budget in (0, 400, 48):
        model, _ = load_model(folder, device="cuda", dtype="bfloat16")
        engine = LLMEngine(model, Config(model=str(folder), max_model_len=512, num_kvcache_blocks=64, max_num_batched_tokens=64, max_num_seqs=4,
                                         chunked_prefill=True, enforce_eager=False, cache_format="kv4", cache_budget=budget, cache_recent=16, cache_slack=16))
        out[budget] = engine.generate(prompts, SamplingParams(temperature=0.0, max_tokens=80, ignore_eos=True), use_tqdm=False)
        assert [len(o) for o in out[budget]] == [80] * 4
        engine.model_runner.cache_manager.check_invariants()
        assert engine.model_runner.cache_manager.pages_in_use() == 0
    assert out[0] == out[400]
    assert out[48][0][:40] == out[0][0][:40]  # (4 + 40 rows: not cut yet)


def test_models_and_options_that_have_no_such_cache_are_refused(tmp_path):
    folder, _ = make_folder(tmp_path, {**TINY, "head_dim": 32}, 3)
    with pytest.raises(ValueError, match="heads of"):
        make_runner(folder)
    other = tmp_path / "b"
    other.mkdir()
    folder, _ = make_folder(other, TINY, 3)
    with pytest.raises(ValueError, match="multiple of 16"):
        make_runner(folder, page_size=8)
    with pytest.raises(ValueError, match="cannot hold"):
        make_runner(folder, cache_budget=32, cache_recent=40)
    with pytest.raises(ValueError, match="needs cache_format"):
        make_runner(folder, cache_format="model", cache_budget=32, cache_recent=4)
    third = tmp_path / "c"
    third.mkdir()
    folder, _ = make_folder(third, WINDOWED, 3)
    with pytest.raises(ValueError, match="keep all keys"):
        make_runner(folder, cache_budget=64, cache_recent=4)
