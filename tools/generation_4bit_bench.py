"""Decode step and prefill of the 7B stack in bf16, e4m3 and MXFP4 weights, the decode step on the bf16 and on the 4-bit KV cache (random weights; the step
is replayed from its graph).  Prints one line each, best of three repeats of the mean: python tools/generation_4bit_bench.py"""
import os
import sys
import time

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "handsonvlm-release_amd"))
from hvlm.config import HandsOnVLMConfig  # noqa: E402
from hvlm.llama import LlamaStack  # noqa: E402

FORMATS = (("bf16", {}), ("e4m3", dict(fp8=True)), ("mxfp4", dict(mxfp4=True)))


def ms(fn, n):
    for _ in range(3):
        fn()
    best = 1e9
    for _ in range(3):
        torch.cuda.synchronize()
        t = time.perf_counter()
        for _ in range(n):
            fn()
        torch.cuda.synchronize()
        best = min(best, (time.perf_counter() - t) / n * 1e3)
    return best


def main():
    cfg = HandsOnVLMConfig.vicuna_7b()
    st = LlamaStack(cfg, device="cuda:0", training=False)
    st.init_random(0)
    S = 880
    for B in (1, 32, 64):
        lens = torch.full((B,), S, dtype=torch.int32, device="cuda:0")
        x = torch.randn(B, cfg.hidden_size, device="cuda:0").bfloat16()
        for kv4 in (False, True):
            cache = st.new_cache(S + 16, batch=B, kv4=kv4)
            for c in cache:
                if kv4:
                    for t in c:
                        t.random_(100, 120)
                else:
                    c.normal_(0, 0.5)
            for name, kw in FORMATS:
                t = ms(lambda: st.decode_step_batched(x, lens, cache, **kw), 10)
                print(f"decode step, {B} samples, {S} cached tokens, {name} weights, {'4-bit' if kv4 else 'bf16'} cache: {t:.2f} ms", flush=True)
            del cache
    for B in (1, 16):
        x = torch.randn(B * 867, cfg.hidden_size, device="cuda:0").bfloat16()
        for name, kw in FORMATS:
            print(f"prefill, {B} x 867 rows, {name} weights: {ms(lambda: st.forward(x, B, 867, save=False, **kw), 3):.2f} ms", flush=True)


if __name__ == "__main__":
    main()
