"""Feed-forwards over 4-bit weights in the engine: a config.json key packs the checkpoint's matrices at load; the
plain model then runs on what the packed ones stand for."""
import json
import os

import pytest
import torch

import helpers
import plain_model as pm
from helpers import TOLERANCE

pytestmark = pytest.mark.gpu

CONFIGS = {
    "crucible": {
        "architectures": ["CrucibleGPT"], "vocab_size": 256, "n_layer": 2, "n_head": 4, "n_kv_head": 2, "n_embd": 64,
        "head_dim": 16, "intermediate_size": 192, "block_size": 512, "attention": "gqa", "pos_encoding": "rope",
        "activation": "swiglu", "norm": "rmsnorm", "norm_placement": "pre", "rope_theta": 10000.0, "rms_norm_eps": 1e-5,
        "tie_word_embeddings": True, "feed_forward_weight_group": 32},
    "llama": {
        "architectures": ["LlamaForCausalLM"], "vocab_size": 509, "num_hidden_layers": 2, "num_attention_heads": 4,
        "num_key_value_heads": 2, "hidden_size": 256, "head_dim": 64, "intermediate_size": 512,
        "max_position_embeddings": 512, "hidden_act": "silu", "rope_theta": 500000.0, "rms_norm_eps": 1e-6,
        "tie_word_embeddings": False, "feed_forward_weight_group": 128},
}


def _folder(tmp_path, name):
    from crucible_b200.weights import write_random_model
    out = os.path.join(str(tmp_path), name)
    write_random_model(CONFIGS[name], out, 3, std=helpers.TEST_STD)
    return out


def _plain(folder, name):
    """The plain model's config and weights, its feed-forwards' matrices packed and unpacked."""
    from crucible_b200.ops import quantized
    cfg, w = pm.read_folder(folder)
    group = CONFIGS[name]["feed_forward_weight_group"]
    for key in list(w):
        if any(part in key for part in ("gate_proj", "up_proj", "down_proj")):
            w[key] = quantized.Weights4.pack(w[key].float(), group).dense().to(w[key].dtype)
    return cfg, w


@pytest.mark.parametrize("name", sorted(CONFIGS))
def test_generation_in_32_bits_is_token_identical(tmp_path, name):
    from crucible_b200 import LLM, SamplingParams
    folder = _folder(tmp_path, name)
    vocab = CONFIGS[name]["vocab_size"]
    prompts = [helpers.random_tokens(vocab, n, 70 + i) for i, n in enumerate((1, 19, 60, 100))]
    cfg, w = _plain(folder, name)
    want = [pm.plain_generate(cfg, w, p, 12) for p in prompts]
    llm = LLM(folder, dtype="float32", max_batch=4, prefill_token_budget=48)
    assert llm.generate(prompts, SamplingParams(max_tokens=12)) == want
    assert llm.engine._graph_replays > 0 and not llm.engine._graph_failed
    eager = LLM(folder, dtype="float32", max_batch=4, prefill_token_budget=512, graph=False)
    assert eager.generate(prompts, SamplingParams(max_tokens=12)) == want


@pytest.mark.parametrize("name", sorted(CONFIGS))
def test_generation_in_bfloat16_follows_the_plain_model(tmp_path, name):
    from crucible_b200 import LLM, SamplingParams
    folder = _folder(tmp_path, name)
    vocab = CONFIGS[name]["vocab_size"]
    prompts = [helpers.random_tokens(vocab, n, 80 + i) for i, n in enumerate((5, 40, 90))]
    llm = LLM(folder, dtype="bfloat16", max_batch=4, prefill_token_budget=64)
    got = llm.generate(prompts, SamplingParams(max_tokens=16))
    cfg, w = _plain(folder, name)
    for prompt, out in zip(prompts, got):
        seq = list(prompt)
        for tok in out:
            logits = pm.plain_forward(cfg, w, seq)[-1]
            band = TOLERANCE["bfloat16"] * float(logits.abs().max())
            assert float(logits.max() - logits[tok]) <= 2 * band, "token outside the rounding band"
            seq.append(tok)


WIDE = {**CONFIGS["llama"], "num_hidden_layers": 2, "hidden_size": 1024, "num_attention_heads": 8, "num_key_value_heads": 4,
        "head_dim": 128, "intermediate_size": 8192, "max_position_embeddings": 1024, "feed_forward_weight_group": 64}


def test_a_wide_model_in_bfloat16_takes_prompts_by_every_form(tmp_path, monkeypatch):
    """Prompts of some hundred rows go through the tiles and the pairs inside a step, a few rows through the ring; in none of
    them does a product leave rows for a norm that does not read them."""
    from crucible_b200 import LLM, SamplingParams, ops
    from crucible_b200.ops import quantized
    from crucible_b200.weights import write_random_model
    monkeypatch.setitem(CONFIGS, "wide", WIDE)
    folder = write_random_model(WIDE, os.path.join(str(tmp_path), "wide"), 3, std=helpers.TEST_STD)
    forms, asked = set(), []
    form_of, emit_of = quantized.form_of, ops._norm_emit
    monkeypatch.setattr(quantized, "form_of", lambda *sizes: (forms.add(form_of(*sizes)[0]), form_of(*sizes))[1])

    def emit(ctx, rows, tensor_core):
        left = emit_of(ctx, rows, tensor_core)
        asked.append(left.norm if left is not None else None)
        return left
    monkeypatch.setattr(ops, "_norm_emit", emit)
    prompts = [helpers.random_tokens(WIDE["vocab_size"], n, 90 + i) for i, n in enumerate((40, 600))]
    cfg, w = _plain(folder, "wide")
    for prompt in prompts:
        # (a prompt of 600 whole, and in portions of 128 rows)
        for budget in (640, 128):
            llm = LLM(folder, dtype="bfloat16", max_batch=2, prefill_token_budget=budget)
            ahead = {id(layer.norms["feed_forward_norm"]) for layer in llm.engine.model.layers}
            asked.clear()
            out = llm.generate([prompt], SamplingParams(max_tokens=3))[0]
            assert not any(id(norm) in ahead for norm in asked)
            seq = list(prompt)
            for tok in out:
                logits = pm.plain_forward(cfg, w, seq)[-1]
                band = TOLERANCE["bfloat16"] * float(logits.abs().max())
                assert float(logits.max() - logits[tok]) <= 2 * band, "token outside the rounding band"
                seq.append(tok)
            del llm
    assert {"ring", "tiles", "pairs"} <= forms, forms
