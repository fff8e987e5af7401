"""A small serving loop over one attention layer: requests come and go on shared pages, prompts are answered
exactly, decode steps both exactly and from the compressed rows under the same block table.

    python examples/exact_step.py [--steps 24] [--prompts 300,41,700]

Prints, for every few steps, the pages in use and how far the compressed answer is from the exact one."""

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from smaq_b200 import ops  # noqa: E402
from smaq_b200.integration.exact import ExactPagedCache, RequestPool  # noqa: E402
from smaq_b200.integration.paged import PagedCompressedCache  # noqa: E402


def main(argv=None) -> list[float]:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--steps", type=int, default=24)
    ap.add_argument("--prompts", default="300,41,700")
    args = ap.parse_args(argv)
    prompts = [int(x) for x in args.prompts.split(",")]
    dev, Hq, Hkv, D, page = torch.device("cuda"), 28, 4, 128, 16
    R = len(prompts)
    blocks = sum(-(-(n + args.steps) // page) for n in prompts) + R
    pool = RequestPool(blocks, page, R, blocks, dev)
    exact = ExactPagedCache(blocks, page, Hkv, D, device=dev)
    compressed = PagedCompressedCache(blocks, page, Hkv, D, key_bits=4, capacity=64, device=dev)
    rope = ops.rope_table(max(prompts) + args.steps + 1, D, device=dev)
    weights = dict(q_weight=torch.ones(D, device=dev), k_weight=torch.ones(D, device=dev))
    gen = torch.Generator(device=dev).manual_seed(0)

    def projection(tokens):
        x = torch.randn(tokens, Hq + 2 * Hkv, D, generator=gen, device=dev).to(torch.bfloat16)
        return x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:]

    # the prompts, all in one ragged step
    lens = torch.tensor(prompts, dtype=torch.int32, device=dev)
    t = pool.step(lens, sum(prompts))
    q = exact.project(*projection(sum(prompts)), t, rope, compressed=compressed, **weights)
    exact.prefill(q, pool.block_table, t)
    compressed.note_prompts(pool.block_table, t.seq_lens, lens)
    gaps = []
    for step in range(args.steps):
        t = pool.step(torch.ones_like(lens), R)
        q = exact.project(*projection(R), t, rope, compressed=compressed, **weights)
        a = exact.decode(q, pool.block_table, t.seq_lens)
        b = compressed.decode(q, exact.kv, pool.block_table, t.seq_lens)
        gaps.append(float((a.float() - b.float()).norm() / a.float().norm()))
        if step % 8 == 0:
            print(f"step {step}: {blocks - int(pool.free_count)} of {blocks} pages, "
                  f"compressed against exact: relative L2 {gaps[-1]:.3f}")
    pool.step(torch.zeros_like(lens), 0, finished=torch.ones(R, dtype=torch.bool, device=dev))
    print(f"done: {int(pool.free_count)} of {blocks} pages free")
    return gaps


if __name__ == "__main__":
    main()
