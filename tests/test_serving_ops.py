"""Serving operators without a GPU: rotary tables, refusals of CPU tensors."""

import math

import pytest
import torch

from pdattention_b200.ops import _ext
from pdattention_b200.ops.rotary import RotaryTable, rotary, rotary_cache, rotary_frequencies, rotary_table

needs_ext = pytest.mark.skipif(not _ext.available(), reason="extension not built")


def test_tables_hold_angles_of_far_positions():
    t = rotary_table(64, 131072, theta=500000.0, device="cpu")
    pos = 131071
    for i in (0, 1, 17, 31):
        angle = pos * 500000.0 ** (-2 * i / 64)  # python floats: 64 bits
        # the angle's own rounding in 64 bits (2^-53 * angle) and one rounding to fp32
        assert abs(float(t.cos[pos, i]) - math.cos(angle)) <= 2.0 ** -25 + 2.0 ** -51 * angle
        assert abs(float(t.sin[pos, i]) - math.sin(angle)) <= 2.0 ** -25 + 2.0 ** -51 * angle
    assert t.rotary_dim == 64 and not t.interleaved


def test_scaled_frequencies():
    base, one = rotary_frequencies(8, 10000.0)
    assert one == 1.0 and torch.allclose(base, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64))
    f, m = rotary_frequencies(8, 10000.0, {"type": "linear", "factor": 4.0})
    assert m == 1.0 and torch.allclose(f, base / 4)
    f, _ = rotary_frequencies(8, 10000.0, {"rope_type": "ntk", "factor": 4.0})
    assert f[0] == 1.0 and torch.allclose(f[-1], base[-1] / 4)  # the slowest pair stretches by the factor
    d = {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 100}
    assert torch.allclose(rotary_frequencies(8, 10000.0, d, 50)[0], base)  # not yet past the window
    f, _ = rotary_frequencies(8, 10000.0, d, 300)
    assert torch.allclose(f[-1], base[-1] / 5)  # 2 * 300 / 100 - 1
    llama = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
             "original_max_position_embeddings": 64}
    f, _ = rotary_frequencies(8, 10000.0, llama)
    turns = 64 * base / (2 * math.pi)  # 10.2, 1.02, 0.1, 0.01
    keep = (float(turns[1]) - 1) / 3
    assert torch.allclose(f, torch.stack([base[0], base[1] * keep + base[1] / 8 * (1 - keep), base[2] / 8, base[3] / 8]))
    yarn = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096}
    f, m = rotary_frequencies(128, 10000.0, yarn)
    full, _ = rotary_frequencies(128, 10000.0)
    assert m == pytest.approx(0.1 * math.log(4.0) + 1)
    assert torch.equal(f[:10], full[:10]) and torch.allclose(f[-10:], full[-10:] / 4)
    assert rotary_frequencies(128, 10000.0, {**yarn, "attention_factor": 1.5})[1] == 1.5
    t = rotary_table(128, 4, scaling=yarn, device="cpu")
    assert torch.allclose(t.cos[0], torch.full((64,), m, dtype=torch.float32))


@pytest.mark.parametrize("kw", [dict(rotary_dim=7), dict(rotary_dim=0), dict(scaling={"rope_type": "su"}),
                                dict(scaling={"rope_type": "linear", "factor": 0.5}),
                                dict(scaling={"rope_type": "linear", "factor": float("nan")}),
                                dict(scaling={"rope_type": "yarn", "factor": 2.0}),
                                dict(scaling={"rope_type": "llama3", "factor": 2.0, "low_freq_factor": 4.0,
                                              "high_freq_factor": 4.0, "original_max_position_embeddings": 64})])
def test_refused_tables(kw):
    with pytest.raises(ValueError):
        rotary_frequencies(**{**dict(rotary_dim=64), **kw})


@needs_ext
def test_cpu_tensors_are_refused():
    from pdattention_b200.inference.logits import LogitsRules, choose_tokens, process_logits
    from pdattention_b200.inference.shared_prefix import shared_prefix_attention

    t = rotary_table(64, 8, device="cpu")
    q = torch.zeros(3, 2, 64)
    pos = torch.zeros(3, dtype=torch.long)
    calls = [lambda: rotary(q, None, pos, t),
             lambda: rotary_cache(torch.zeros(3, 256), 2, 1, 64, pos, t, torch.zeros(4, 64), torch.zeros(4, 64),
                                  torch.zeros(3, dtype=torch.int32)),
             lambda: process_logits(torch.zeros(2, 10), LogitsRules()),
             lambda: choose_tokens(torch.zeros(2, 10), LogitsRules()),
             lambda: shared_prefix_attention(torch.zeros(1, 1, 64), torch.zeros(4, 64), torch.zeros(4, 64),
                                             torch.zeros(1, 4, 64), torch.zeros(1, 4, 64),
                                             torch.ones(1, dtype=torch.int32), 1, 1, 64)]
    for call in calls:
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()
    with pytest.raises(ValueError, match="append"):
        choose_tokens(torch.zeros(2, 10), LogitsRules(), append=True)
    assert isinstance(t, RotaryTable)


def test_history_appends_on_any_device():
    from pdattention_b200.inference.logits import TokenHistory

    h = TokenHistory.start(torch.tensor([[5, 6], [7, 0]]), torch.tensor([2, 1]), 1)
    h.append(torch.tensor([1, -1]))
    h.append(torch.tensor([9, 4]))  # row 0 is full
    assert h.ids.tolist() == [[5, 6, 1], [7, 4, 0]] and h.lengths.tolist() == [3, 2]
    assert h.prompt_lengths.tolist() == [2, 1]
    h.lengths[1] = -3  # a negative length: nothing yet
    h.append(torch.tensor([2, 8]))
    assert h.ids.tolist() == [[5, 6, 1], [8, 4, 0]] and h.lengths.tolist() == [3, 1]
    none = TokenHistory(torch.zeros((2, 0), dtype=torch.int32), torch.zeros(2, dtype=torch.int32))
    none.append(torch.tensor([1, 2]))
    assert none.lengths.tolist() == [0, 0]


@pytest.mark.parametrize("family,scaling", [
    ("llama", {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
               "original_max_position_embeddings": 32}),
    ("qwen2", {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32}),
    ("mistral", {"rope_type": "linear", "factor": 4.0})])
def test_scaled_positions_match_hugging_face(family, scaling):
    import transformers

    from pdattention_b200.hf.convert import config_from_hf, reference_from_hf
    from pdattention_b200.models.llama import PRALlamaReference, hf_config, tiny_llama

    cfg = tiny_llama(family=family, attention_bias=family == "qwen2", rope_scaling=scaling, max_position_embeddings=128)
    ours = PRALlamaReference(cfg).eval()
    ours.reset_parameters(seed=0, std=0.2)
    hcfg = hf_config(cfg)
    hcfg._attn_implementation = "eager"
    hf = {"llama": transformers.LlamaForCausalLM, "mistral": transformers.MistralForCausalLM,
          "qwen2": transformers.Qwen2ForCausalLM}[family](hcfg).eval()
    hf.load_state_dict(ours.state_dict(), strict=False)
    ids = torch.randint(0, cfg.vocab_size, (1, 100), generator=torch.Generator().manual_seed(1))
    with torch.no_grad():
        want = hf(ids).logits
    # the other side takes angles in 32 bits: 100 * 2^-23 on the last position's fastest pair, as much again from its
    # fp32 frequencies; scores of a few tens and two layers make of that at most some 1e-3 of logits near 1
    assert torch.allclose(ours(ids), want, atol=2e-3, rtol=1e-3)
    plain = PRALlamaReference(tiny_llama(family=family, attention_bias=family == "qwen2", max_position_embeddings=128)).eval()
    plain.load_state_dict(ours.state_dict())
    assert not torch.allclose(plain(ids), want, atol=2e-2, rtol=1e-2)  # the scaling matters here
    back = reference_from_hf(hf)
    assert back.cfg.rope_scaling["rope_type"] == scaling["rope_type"] and back.cfg.rope_theta == cfg.rope_theta
    assert torch.equal(back(ids), ours(ids))
    hcfg.rope_parameters = {"rope_type": "other", "factor": 2.0, "rope_theta": 1e4}
    with pytest.raises(ValueError, match="scaling"):
        config_from_hf(hcfg)
