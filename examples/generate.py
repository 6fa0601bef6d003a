"""Token-by-token answers of a decoder with a paged key-value cache.

    python examples/generate.py --model 70m --weights w4

Random weights (there are no checkpoints here), so the text means nothing: the example shows the calls and the rate.
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from mccl_b200.models import Generator, build_decoder  # noqa: E402


def main() -> None:
    p = argparse.ArgumentParser()
    p.add_argument("--model", default="70m")
    p.add_argument("--weights", default="bf16", choices=["bf16", "w4"])
    p.add_argument("--sequences", type=int, default=8)
    p.add_argument("--prompt", type=int, default=37)
    p.add_argument("--new", type=int, default=64)
    p.add_argument("--window", type=int, default=None)
    p.add_argument("--sinks", type=int, default=0)
    args = p.parse_args()
    dev = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    torch.manual_seed(0)
    model = build_decoder(args.model).to(dev)
    gen = Generator(model, max_sequences=args.sequences, weights=args.weights, window=args.window, sinks=args.sinks)
    prompt = torch.randint(0, model.cfg.vocab, (args.prompt,)).tolist()

    # one prompt, several continuations: the prompt's full pages are shared
    row, logits = gen.prefill(prompt)
    rows = [row] + gen.fork(row, args.sequences - 1)
    tokens = torch.softmax(logits.float(), -1).multinomial(args.sequences, replacement=True)
    gen.step(rows, tokens)   # captures the step
    if dev.type == "cuda":
        torch.cuda.synchronize()
    start = time.perf_counter()
    for _ in range(args.new):
        tokens = gen.step(rows, tokens).float().argmax(-1)
    if dev.type == "cuda":
        torch.cuda.synchronize()
    took = time.perf_counter() - start
    print(f"{args.model}, {args.weights} weights, {args.sequences} sequences: {took / args.new * 1e6:.0f} us per step, "
          f"{args.sequences * args.new / took:.0f} tokens/s; {gen.cache.free_pages} pages free")
    for r in rows[: args.sequences // 2]:
        gen.free(r)
    print(f"half the sequences gone: {gen.cache.free_pages} pages free, {gen.cache.compact()} in use after compaction")
    for r in rows[args.sequences // 2:]:
        gen.free(r)
    print("greedy:", gen.generate([prompt[:5]], 8)[0])


if __name__ == "__main__":
    main()
