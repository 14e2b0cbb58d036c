"""The engine with its cache in 4 bits: what it stores is the plain model's keys and values to half a step, and its
logits are the plain model's over what is stored."""
import os

import pytest
import torch

import cache4_cases as cc
import helpers
import plain_model as pm
from helpers import TOLERANCE

pytestmark = pytest.mark.gpu

CONFIGS = {
    "heads of 64": {
        "architectures": ["CrucibleGPT"], "vocab_size": 256, "n_layer": 3, "n_head": 6, "n_kv_head": 2, "n_embd": 128,
        "head_dim": 64, "intermediate_size": 192, "block_size": 1024, "attention": "gqa", "pos_encoding": "rope",
        "activation": "swiglu", "norm": "rmsnorm", "norm_placement": "pre", "rope_theta": 10000.0, "rms_norm_eps": 1e-5,
        "tie_word_embeddings": True},
    "heads of 128": {
        "architectures": ["LlamaForCausalLM"], "vocab_size": 509, "num_hidden_layers": 2, "num_attention_heads": 8,
        "num_key_value_heads": 2, "hidden_size": 256, "head_dim": 128, "intermediate_size": 512,
        "max_position_embeddings": 1024, "hidden_act": "silu", "rope_theta": 500000.0, "rms_norm_eps": 1e-6,
        "tie_word_embeddings": False},
}


def _folder(tmp_path, name):
    from crucible_b200.weights import write_random_model
    out = os.path.join(str(tmp_path), name.replace(" ", "_"))
    write_random_model(CONFIGS[name], out, 3, std=helpers.TEST_STD)
    return out


def _engine(folder, dtype, **more):
    from crucible_b200.engine.engine import Engine, EngineOptions
    return Engine(folder, EngineOptions(dtype=dtype, max_requests=4, **more))


def _stored(engine, request, layer):
    """(keys, values, their steps) [tokens, kv heads, ..] in float64 of what the engine holds of a request."""
    pages = engine.storages[0].pages(layer)
    held = engine.held_tokens(request)
    at = torch.arange(held)
    table = torch.tensor(engine.cache.block_table(request, 0))
    where, slot = table[torch.div(at, pages.page_tokens, rounding_mode="floor")], at % pages.page_tokens
    both = cc.values(pages.codes.cpu(), pages.scales.cpu())
    steps = pages.scales[..., 0].double().cpu().repeat_interleave(pages.group, dim=-1)
    return [both[i][where, :, slot] for i in (0, 1)], [steps[i][where, :, slot] for i in (0, 1)]


def _plain(cfg, w, tokens, engine, request, near, picked=None):
    """The plain model's logits over the stored keys and values, which are its own to half a step (and `near` of the
    largest, by which the engine's rows may be off before they are coded).  `picked`: {(layer, position): pages a kv head}."""
    cos, sin = pm.plain_rope_tables(cfg["head_dim"], len(tokens), cfg["theta"])
    x = pm.plain_embedding(w[pm.tensor_name(cfg, "embed")], tokens)
    t, hq, hkv, hd = len(tokens), cfg["heads"], cfg["kv_heads"], cfg["head_dim"]
    page = engine.options.page_tokens
    for layer in range(cfg["layers"]):
        name = lambda what: w[pm.tensor_name(cfg, what, layer)]  # noqa: E731
        n = pm.plain_rmsnorm(x, name("attn_norm"), cfg["eps"])
        q, k, v = ((n @ name(m).T).view(t, -1, hd) for m in ("q", "k", "v"))
        q, k = pm.plain_rope(q, cos, sin), pm.plain_rope(k, cos, sin)
        kept, steps = _stored(engine, request, layer)
        for mine, theirs, step in zip((k, v), kept, steps):
            # (half a step, what the rounding of the step cuts off the largest, and the pair's own rounding)
            assert ((mine - theirs).abs() <= step * (0.5 + 15 * 2.0 ** -8) + 2 * near * mine.abs().max()).all()
        k, v = kept
        out = torch.zeros_like(q)
        for h in range(hq):
            kv = h * hkv // hq
            scores = (q[:, h] @ k[:, kv].T) / hd ** 0.5
            key = torch.arange(t)
            hidden = key[None] > key[:, None]
            for i in range(t):
                pages = None if picked is None else picked.get((layer, i))
                if pages is not None:
                    hidden[i] |= ~torch.isin(key // page, pages[kv])
            out[:, h] = torch.softmax(scores.masked_fill(hidden, float("-inf")), dim=-1) @ v[:, kv]
        x = x + out.reshape(t, hq * hd) @ name("o").T
        n = pm.plain_rmsnorm(x, name("mlp_norm"), cfg["eps"])
        x = x + pm.plain_swiglu(n, name("gate"), name("up"), name("down"))
    x = pm.plain_rmsnorm(x, w[pm.tensor_name(cfg, "final_norm")], cfg["eps"])
    return x @ w[pm.tensor_name(cfg, "embed" if cfg["tie"] else "head")].T


@pytest.mark.parametrize("page_tokens", [16, 24])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name,group", [("heads of 64", 64), ("heads of 64", 32), ("heads of 128", 128), ("heads of 128", 32)])
def test_logits_over_a_cache_in_4_bits(tmp_path, name, group, dtype, page_tokens):
    """Prompts whole, in portions and beside decoded tokens, long and short."""
    from crucible_b200.engine.engine import StepEntry
    folder = _folder(tmp_path, name)
    cfg, w = pm.read_folder(folder)
    engine = _engine(folder, dtype, cache_group=group, page_tokens=page_tokens)
    tokens = {r: helpers.random_tokens(cfg["vocab"], n, 40 + i) for i, (r, n) in enumerate((("a", 150), ("b", 300), ("c", 9)))}
    fed = {r: 0 for r in tokens}
    got = {r: {} for r in tokens}
    for step in ([("a", 140)], [("a", 1), ("b", 250)], [("a", 1), ("c", 1), ("b", 40)], [("a", 1), ("c", 1), ("b", 1)],
                 [("a", 1), ("c", 1), ("b", 1)], [("a", 3), ("c", 2), ("b", 1)], [("a", 1), ("b", 1), ("c", 1)]):
        entries = [StepEntry(r, tokens[r][fed[r]:fed[r] + n], list(range(n))) for r, n in step]
        logits = engine.step(entries).clone().cpu().double()
        at = 0
        for r, n in step:
            for i in range(n):
                got[r][fed[r] + i] = logits[at + i]
            at += n
            fed[r] += n
    for r in tokens:
        near = 1e-5 if dtype == "float32" else 2e-2
        want = _plain(cfg, w, tokens[r][:fed[r]], engine, r, near)
        for i, row in got[r].items():
            assert float((row - want[i]).abs().max()) <= TOLERANCE[dtype] * float(want.abs().max()), (r, i)
    assert not engine._graph_failed


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_decoded_tokens_attend_to_the_pages_that_are_picked(tmp_path, dtype, monkeypatch):
    from crucible_b200.engine.engine import StepEntry
    from crucible_b200.ops import cache4
    name, count = "heads of 64", 5
    folder = _folder(tmp_path, name)
    cfg, w = pm.read_folder(folder)
    engine = _engine(folder, dtype, cache_group=64, attend_pages=count, graph=False)
    tokens = {r: helpers.random_tokens(cfg["vocab"], n, 50 + i) for i, (r, n) in enumerate((("a", 260), ("b", 200)))}
    seen, pick = [], cache4.pick_pages4

    def recorded(q, n_heads, batch, pages, picks, **more):
        pick(q, n_heads, batch, pages, picks, **more)
        assert picks.shape[0] == batch.lead
        seen.append((batch.positions[:batch.lead].tolist(), picks.clone().cpu()))
    monkeypatch.setattr(cache4, "pick_pages4", recorded)
    fed = {r: 0 for r in tokens}
    got, picked = {r: {} for r in tokens}, {r: {} for r in tokens}
    for step in ([("a", 250)], [("a", 1), ("b", 190)], [("a", 1), ("b", 1)], [("b", 1), ("a", 1)]):
        seen.clear()
        entries = [StepEntry(r, tokens[r][fed[r]:fed[r] + n], list(range(n))) for r, n in step]
        logits = engine.step(entries).clone().cpu().double()
        at = 0
        for r, n in step:
            for i in range(n):
                got[r][fed[r] + i] = logits[at + i]
            at += n
        lead = [r for r, n in step if n == 1]
        assert len(seen) == (cfg["layers"] if lead else 0)
        for layer, (positions, picks) in enumerate(seen):
            for i, r in enumerate(lead):
                assert positions[i] == fed[r]
                picked[r][layer, fed[r]] = picks[i]
        for r, n in step:
            fed[r] += n
    for r in tokens:
        assert any(len(p[0].unique()) == count for p in picked[r].values())
        want = _plain(cfg, w, tokens[r][:fed[r]], engine, r, 1e-5 if dtype == "float32" else 2e-2, picked[r])
        for i, row in got[r].items():
            assert float((row - want[i]).abs().max()) <= TOLERANCE[dtype] * float(want.abs().max()), (r, i)


def test_generation_replays_graphs_and_equals_eager_steps(tmp_path):
    from crucible_b200 import LLM, SamplingParams
    folder = _folder(tmp_path, "heads of 64")
    prompts = [helpers.random_tokens(256, n, 60 + i) for i, n in enumerate((1, 19, 300, 90))]
    for attend in (None, 4):
        outs = []
        for graph in (True, False):
            llm = LLM(folder, dtype="float32", max_batch=4, prefill_token_budget=128, graph=graph, cache_group=32, attend_pages=attend)
            outs.append(llm.generate(prompts, SamplingParams(max_tokens=24)))
            assert not llm.engine._graph_failed and (llm.engine._graph_replays > 0) == graph
            assert llm.engine._prompt_graph_replays == 0
            llm.engine.cache.check_invariants()
        assert outs[0] == outs[1]


def test_more_pages_than_there_are_is_all_of_them(tmp_path):
    from crucible_b200 import LLM, SamplingParams
    folder = _folder(tmp_path, "heads of 128")
    prompts = [helpers.random_tokens(509, n, 70 + i) for i, n in enumerate((5, 200))]
    outs = [LLM(folder, dtype="float32", max_batch=2, cache_group=64, attend_pages=attend).generate(
        prompts, SamplingParams(max_tokens=12)) for attend in (None, 64)]
    assert outs[0] == outs[1]


def test_what_the_engine_refuses(tmp_path):
    from crucible_b200.config.presets import SHAPES
    from crucible_b200.weights import write_random_model
    folder = _folder(tmp_path, "heads of 64")
    for options in (dict(cache_group=16), dict(cache_group=128), dict(cache_group=64, attend_pages=2),
                    dict(cache_group=64, attend_pages=8, page_tokens=24), dict(attend_pages=8)):
        with pytest.raises(ValueError, match="cache_group|attend_pages"):
            _engine(folder, "bfloat16", **options)
    small = write_random_model(SHAPES["tiny-a"], os.path.join(str(tmp_path), "small"), 0)
    with pytest.raises(ValueError, match="not 16 in groups of 32"):
        _engine(small, "bfloat16", cache_group=32)
    import vuvosun_cases
    other = vuvosun_cases.make_folder(tmp_path, sorted(vuvosun_cases.CASES)[0])
    with pytest.raises(ValueError, match="cache"):
        _engine(other, "bfloat16", cache_group=32)


def test_contexts_of_more_pages_than_are_picked_among(tmp_path):
    """Refused when the engine is made, not by a step of some later token; longer pages or shorter contexts are taken."""
    from crucible_b200.ops import cache4
    from crucible_b200.weights import write_random_model
    folder = os.path.join(str(tmp_path), "long")
    write_random_model(dict(CONFIGS["heads of 64"], n_layer=1, block_size=1_000_000), folder, 0)
    more = dict(cache_group=64, attend_pages=8, n_pages=100)
    with pytest.raises(ValueError, match="picks among"):
        _engine(folder, "bfloat16", **more)
    for options in (dict(page_tokens=32), dict(max_context=cache4.most_pages(3, 64) * 16)):
        from crucible_b200.engine.engine import StepEntry
        engine = _engine(folder, "bfloat16", **more, **options)
        engine.step([StepEntry("a", list(range(200)), [])])
        assert torch.isfinite(engine.step([StepEntry("a", [7], [0])])).all()
    with pytest.raises(ValueError, match="picks among"):
        _engine(folder, "bfloat16", **more, max_context=cache4.most_pages(3, 64) * 16 + 1)
