"""Which tokens attend to picked pages: what a request decodes, wherever its entry stands in the step, and nothing of a prompt,
however it is cut."""
import pytest
import torch

import helpers
import plain_model as pm
import test_cache4_engine_gpu as base
from helpers import TOLERANCE

pytestmark = pytest.mark.gpu
COUNT = 5


def _run(tmp_path, dtype, steps, monkeypatch, graph=False):
    """Runs steps of (request, tokens, whether they are a prompt's); checks every logit against the plain model, in which the
    decoded tokens, and these alone, attend to the pages that the engine picked."""
    from crucible_b200.engine.engine import StepEntry
    from crucible_b200.ops import cache4
    folder = base._folder(tmp_path, "heads of 64")
    cfg, w = pm.read_folder(folder)
    engine = base._engine(folder, dtype, cache_group=64, attend_pages=COUNT, graph=graph)
    seen, pick = [], cache4.pick_pages4

    def recorded(q, n_heads, batch, pages, picks, **more):
        pick(q, n_heads, batch, pages, picks, **more)
        seen.append((batch.positions[:picks.shape[0]].tolist(), batch.row_request[:picks.shape[0]].tolist(), picks.clone().cpu()))
    monkeypatch.setattr(cache4, "pick_pages4", recorded)
    tokens = {r: helpers.random_tokens(cfg["vocab"], 400, 80 + i) for i, r in enumerate("abc")}
    fed, got, picked = ({r: v() for r in tokens} for v in (int, dict, dict))
    for step in steps:
        seen.clear()
        entries = [StepEntry(r, tokens[r][fed[r]:fed[r] + n], list(range(n)), prompt=prompt) for r, n, prompt in step]
        logits = engine.step(entries).clone().cpu().double()
        decoded = [r for r, n, prompt in step if n == 1 and not prompt]
        assert len(seen) == (cfg["layers"] if decoded else 0)
        for layer, (positions, _, picks) in enumerate(seen):
            assert positions == [fed[r] for r in decoded]
            for i, r in enumerate(decoded):
                picked[r][layer, fed[r]] = picks[i]
        at = 0
        for r, n, _ in step:
            for i in range(n):
                got[r][fed[r] + i] = logits[at + i]
            at += n
            fed[r] += n
        assert at == logits.shape[0]
    for r in tokens:
        if not fed[r]:
            continue
        want = base._plain(cfg, w, tokens[r][:fed[r]], engine, r, 1e-5 if dtype == "float32" else 2e-2, picked[r])
        for i, row in got[r].items():
            assert float((row - want[i]).abs().max()) <= TOLERANCE[dtype] * float(want.abs().max()), (r, i)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_one_token_ahead_of_behind_and_between_longer_portions(tmp_path, dtype, monkeypatch):
    _run(tmp_path, dtype, [
        [("a", 200, True)],
        [("a", 1, True), ("b", 150, True)],                       # a prompt's, at the head
        [("b", 30, True), ("a", 1, True)],                        # ... and behind
        [("a", 1, False), ("b", 20, True)],                       # decoded, at the head
        [("b", 20, True), ("a", 1, False)],                       # ... and behind
        [("c", 40, True), ("a", 1, False), ("b", 1, True)],
        [("b", 1, True), ("a", 1, False), ("c", 1, True)],        # one token each, one of them decoded
        [("b", 1, False), ("c", 2, False), ("a", 1, False)],
        [("c", 1, True), ("b", 1, True)]], monkeypatch)


def test_choices_come_in_the_entries_order(tmp_path):
    """A step whose choice is part of it, decoded tokens behind portions; eager and captured, with ids that are on the device."""
    from crucible_b200.engine.engine import DEVICE_TOKEN, StepEntry
    folder = base._folder(tmp_path, "heads of 64")
    outs = []
    for turned in (False, True):
        engine = base._engine(folder, "float32", cache_group=64, attend_pages=COUNT)
        prompts = {r: helpers.random_tokens(256, n, 90 + i) for i, (r, n) in enumerate((("a", 180), ("b", 150), ("c", 31)))}
        got = []

        def step(entries):
            entries = entries[::-1] if turned else entries
            logits, ids = engine.step_choosing(entries)
            logits, ids = logits.clone().cpu(), ids.get()
            assert ids == logits.argmax(dim=-1).tolist()
            got.append(sorted(zip([e.request for e in entries], ids)))
        step([StepEntry("a", prompts["a"], [179], prompt=True)])
        step([StepEntry("a", [DEVICE_TOKEN], [0]), StepEntry("b", prompts["b"], [149], prompt=True)])
        for i in range(6):
            step([StepEntry("a", [DEVICE_TOKEN], [0]), StepEntry("b", [DEVICE_TOKEN], [0]), StepEntry("c", [prompts["c"][i]], [0], prompt=True)])
        engine.step([StepEntry("c", prompts["c"][6:], [], prompt=True), StepEntry("a", [0], [0])],
                    token_source=torch.tensor(prompts["c"][6:] + [17], dtype=torch.int32, device="cuda:0"))
        step([StepEntry("a", [3], [0]), StepEntry("b", [DEVICE_TOKEN], [0])])
        outs.append(got)
    assert outs[0] == outs[1]
