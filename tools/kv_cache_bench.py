#!/usr/bin/env python
"""The engine with keys and values in the model's type and in 8 bits: time of a prompt pass and of a captured decoding step.  8B shape, bf16, random weights
and tokens; CUDA events, after a pass and steps that are not timed."""
import argparse
import json
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
import torch  # noqa: E402

import dgi_b200  # noqa: E402,F401
from bench import SHAPES, ShapeConfig  # noqa: E402
from dgi_b200.engine import PagedDecodeEngine  # noqa: E402
from dgi_b200.worker.distributed.model_shard import ModelShard  # noqa: E402


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--cases", default="64x1920,8x16000,1x1920", help="sequences x prompt tokens")
    ap.add_argument("--kinds", default="model,int8,e4m3")
    ap.add_argument("--steps", type=int, default=30)
    a = ap.parse_args()
    cfg = ShapeConfig(**SHAPES["8b"])
    shard = ModelShard.from_config(cfg, 0, cfg.num_hidden_layers, device="cuda:0", dtype=torch.bfloat16, seed=0)

    def timed(f):
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        torch.cuda.synchronize()
        begin.record()
        f()
        end.record()
        torch.cuda.synchronize()
        return begin.elapsed_time(end)

    for case in a.cases.split(","):
        B, P = map(int, case.split("x"))
        prompts = torch.randint(0, cfg.vocab_size, (B, P), generator=torch.Generator().manual_seed(1234))
        for kind in a.kinds.split(","):
            room = P + a.steps + 10
            eng = PagedDecodeEngine([shard], max_batch=B, max_seq_len=room, kv_cache_dtype=None if kind == "model" else kind)
            eng.allocate(B, room)
            eng.prefill(prompts)
            eng.allocate(B, room)
            first = []
            prompt_ms = timed(lambda: first.append(eng.prefill(prompts)))
            eng.ids_buf[:B, 0].copy_(first[0])
            for _ in range(6):      # the first one captures the step
                eng.decode_step_device()
            step_ms = timed(lambda: [eng.decode_step_device() for _ in range(a.steps)]) / a.steps
            print(json.dumps({"sequences": B, "prompt": P, "kv": kind, "prompt_ms": round(prompt_ms, 1), "step_ms": round(step_ms, 3)}), flush=True)
            eng.release()
            del eng
            torch.cuda.empty_cache()


if __name__ == "__main__":
    main()
