"""Continuous batching with ragged prompts on a random model: prompts of different lengths are
admitted together, decoded greedily, and leave as they finish while new ones join.

    python examples/paged_serving.py [--layout BBBBBBBA] [--requests 32] [--steps 64]
"""

from __future__ import annotations

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from copy_on_write_sdm_b200.model import LanguageModel  # noqa: E402
from copy_on_write_sdm_b200.paged import PagedServing  # noqa: E402


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--layout", default="BBBBBBBA")
    ap.add_argument("--requests", type=int, default=32)
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--longest", type=int, default=512)
    args = ap.parse_args()

    torch.manual_seed(0)
    model = LanguageModel(vocab_size=4096, maximum_sequence_length=args.longest + args.steps, layout=args.layout, width=128,
                          heads=4, kv_heads=2, slots=256, reads=16, writes=4, activation_dtype=torch.float32)
    model.initialize_role_keyed(0)
    model = model.cuda().eval()
    serving = PagedServing(model, pages=args.requests * -(-(args.longest + args.steps) // 64))
    rng = torch.Generator().manual_seed(1)

    def prompts(count: int) -> list[torch.Tensor]:
        lengths = torch.randint(1, args.longest + 1, (count,), generator=rng).tolist()
        return [torch.randint(0, 4096, (n,), generator=rng) for n in lengths]

    named = args.requests
    next_ids = serving.admit(prompts(named), list(range(named))).argmax(-1)
    torch.cuda.synchronize()
    began, decoded = time.perf_counter(), 0
    for step in range(args.steps):
        next_ids = serving.decode(next_ids).argmax(-1)
        decoded += len(serving.requests)
        if step % 16 == 15:  # a quarter of the batch finishes, others join
            gone = serving.requests[::4]
            kept = [i for i, name in enumerate(serving.requests) if name not in set(gone)]
            serving.release(gone)
            logits = serving.admit(prompts(len(gone)), list(range(named, named + len(gone))))
            named += len(gone)
            next_ids = torch.cat((next_ids[kept], logits.argmax(-1)))
    torch.cuda.synchronize()
    seconds = time.perf_counter() - began
    serving.validate_invariants()
    print(f"{decoded} tokens in {seconds:.2f} s, {named} requests served, lengths now {min(serving.lengths)} to {max(serving.lengths)}, "
          f"{serving.free_pages} of {serving.cache.pages} K/V pages free")


if __name__ == "__main__":
    main()
