"""What a decode step and a prompt take with keys and values as they are, in 4 bits, and with picked pages beside that.

    python perf/decode_cache4.py [--dtype bfloat16] [--cases 1x2000,32x8000] [--layers 4]

Random weights of a Llama shape of width 4,096 (32 heads of 128 on 8, a feed-forward of 14,336), pages of 64 tokens, groups of 64,
16 pages picked.  For every batch x context the requests' contexts are run first; then 8 decode steps unmeasured and three runs of
32 (captured graphs, greedy, ids read two steps behind, as the scheduler does), each between two events; then a prompt of 2,000
tokens by itself, four times unmeasured and four times measured.  Prints the least milliseconds a step and a prompt."""
from __future__ import annotations

import argparse
import os
import random
import sys
import tempfile

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

FORMS = {"as is": {}, "4 bits": {"cache_group": 64}, "16 pages": {"cache_group": 64, "attend_pages": 16}}


def _ms(start, end, n):
    end.record()
    torch.cuda.synchronize()
    return start.elapsed_time(end) / n


def measure(folder, dtype, batch, context, more, vocab, seed=1):
    from crucible_b200.engine.engine import DEVICE_TOKEN, Engine, EngineOptions, StepEntry
    rng = random.Random(seed)
    engine = Engine(folder, EngineOptions(dtype=dtype, max_requests=batch, page_tokens=64, max_context=max(context, 2000) + 128, **more))
    for r in range(batch):
        tokens = [rng.randrange(vocab) for _ in range(context)]
        for at in range(0, context, 2048):
            engine.step([StepEntry(r, tokens[at:at + 2048], [], prompt=True)])
    engine.step_choosing([StepEntry(r, [rng.randrange(vocab)], [0]) for r in range(batch)])[1].get()
    entries = [StepEntry(r, [DEVICE_TOKEN], [0]) for r in range(batch)]
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    for _ in range(8):
        engine.step_choosing(entries)[1].get()
    step = prompt = float("inf")
    for _ in range(3):
        torch.cuda.synchronize()
        start.record()
        on_their_way = []
        for _ in range(32):
            on_their_way.append(engine.step_choosing(entries)[1])
            if len(on_their_way) > 2:
                on_their_way.pop(0).get()
        step = min(step, _ms(start, end, 32))
    for r in range(batch):
        engine.finish(r)
    tokens = [rng.randrange(vocab) for _ in range(2000)]
    for i in range(8):                             # (the first of them are captured, where steps of prompts are)
        torch.cuda.synchronize()
        start.record()
        engine.step([StepEntry("p", tokens, [len(tokens) - 1], prompt=True)])
        if i >= 4:
            prompt = min(prompt, _ms(start, end, 1))
        engine.finish("p")
    return step, prompt


def main():
    parser = argparse.ArgumentParser()
    parser.add_argument("--dtype", default="bfloat16", choices=["bfloat16", "float32"])
    parser.add_argument("--cases", default="1x2000,1x65000,8x8000,32x8000,64x2000")
    parser.add_argument("--layers", type=int, default=4)
    args = parser.parse_args()
    from crucible_b200.weights import write_random_model
    config = {"architectures": ["LlamaForCausalLM"], "vocab_size": 8192, "num_hidden_layers": args.layers, "num_attention_heads": 32,
              "num_key_value_heads": 8, "hidden_size": 4096, "head_dim": 128, "intermediate_size": 14336,
              "max_position_embeddings": 131072, "hidden_act": "silu", "rope_theta": 500000.0, "rms_norm_eps": 1e-6,
              "tie_word_embeddings": False}
    with tempfile.TemporaryDirectory() as folder:
        write_random_model(config, folder, 3, std=0.02)
        for case in args.cases.split(","):
            batch, context = map(int, case.split("x"))
            parts = []
            for name, more in FORMS.items():
                step, prompt = measure(folder, args.dtype, batch, context, more, config["vocab_size"])
                parts.append(f"{name} {step:.3f} (prompt {prompt:.2f})")
                torch.cuda.empty_cache()
            print(f"{args.dtype}, a batch of {batch} at {context}: " + ", ".join(parts), flush=True)


if __name__ == "__main__":
    main()
