"""A serving loop over a paged cache whose pages the GPU hands out: a prompt in chunks, samples that fork from it, drafts
that are verified and partly dropped, and compaction at the end. Values are random; what is shown is the bookkeeping.

    python examples/chunk_step.py
"""

from __future__ import annotations

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "kernel-lab_b200"))

from kernel_lab import cuda_ops  # noqa: E402

HQ, HKV, DIM, PAGE, PAGES, WIDTH = 32, 8, 128, 16, 512, 64


def main() -> dict[str, int]:
    gen = torch.Generator(device="cuda").manual_seed(0)
    int32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    rand = lambda n, h: torch.randn(n, h, DIM, generator=gen, device="cuda").to(torch.bfloat16)  # noqa: E731
    pool = [torch.zeros(PAGES, PAGE, HKV, DIM, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    table, lens = torch.zeros(1, WIDTH, dtype=torch.int32, device="cuda"), int32([0])

    def step(table, lens, new, parents=None):
        """New tokens for every row: pages, append, attention; lengths grow by what was appended."""
        count = int32(new)
        table, lens, served = cuda_ops.paged_reserve(pool, table, lens, count, parents)
        assert bool(served.all()), "the pool is full"
        rows = sum(new)
        indptr = torch.nn.functional.pad(count.cumsum(0, dtype=torch.int32), (1, 0))
        cuda_ops.paged_kv_append(*pool, rand(rows, HKV), rand(rows, HKV), table, lens, indptr=indptr)
        lens = lens + count
        return table, lens, cuda_ops.paged_chunk_attention(rand(rows, HQ), *pool, table, lens, indptr)

    for chunk in (256, 256, 90):  # the prompt
        table, lens, out = step(table, lens, [chunk])
    table, lens, out = step(table, lens, [1, 1, 1, 1], int32([0, 0, 0, 0]))  # four samples: shared pages, own last ones
    forked = len(set(table[:, : -(-int(lens[0]) // PAGE)].flatten().tolist()))
    table, lens, out = step(table, lens, [5, 5, 5, 5])  # drafts, of which two, five, none and three are accepted
    lens = lens - int32([3, 0, 5, 2])
    table, lens, out = step(table, lens, [1, 1], int32([1, 3]))  # two samples end; their pages are free again
    table, used = cuda_ops.paged_compact(pool, table, lens)
    assert torch.isfinite(out).all() and cuda_ops.decode_status() == 0
    return {"tokens": int(lens.sum()), "pages after the fork": forked, "pages at the end": int(used)}


if __name__ == "__main__":
    print(main())
