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


def step(pool, q, k, v, table, lens, new, indptr, parents=None):
    """Pages, append and attention for every row's new tokens; no host synchronisation, so that it may be captured. A row that
    got no pages (or stands for no sequence) writes nothing, since its table names none for them, and keeps its length: its
    rows of the result are to be dropped, and its tokens to be tried again once pages are free."""
    sequences = lens.shape[0]
    table, lens, served = cuda_ops.paged_reserve(pool, table, lens, new, parents)
    if parents is not None:
        served = served & (parents >= 0) & (parents < sequences)
    cuda_ops.paged_kv_append(*pool, k, v, table, torch.where(served, lens, -1), indptr=indptr)
    lens = lens + torch.where(served, new, 0)
    return table, lens, served, cuda_ops.paged_chunk_attention(q, *pool, table, lens, indptr)


def main() -> dict[str, int]:
    gen = torch.Generator(device="cuda").manual_seed(0)
    int32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    rand = lambda n, h: torch.randn(n, h, DIM, generator=gen, device="cuda").to(torch.bfloat16)  # noqa: E731
    pool = [torch.zeros(PAGES, PAGE, HKV, DIM, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    table, lens = torch.zeros(1, WIDTH, dtype=torch.int32, device="cuda"), int32([0])

    def run(table, lens, new, parents=None):
        rows, count = sum(new), int32(new)
        indptr = torch.nn.functional.pad(count.cumsum(0, dtype=torch.int32), (1, 0))
        table, lens, _, out = step(pool, rand(rows, HQ), rand(rows, HKV), rand(rows, HKV), table, lens, count, indptr, parents)
        return table, lens, out

    for chunk in (256, 256, 90):  # the prompt
        table, lens, out = run(table, lens, [chunk])
    table, lens, out = run(table, lens, [1, 1, 1, 1], int32([0, 0, 0, 0]))  # four samples: shared pages, own last ones
    forked = len(set(table[:, : -(-int(lens[0]) // PAGE)].flatten().tolist()))
    table, lens, out = run(table, lens, [5, 5, 5, 5])  # drafts, of which two, five, none and three are accepted
    lens = lens - int32([3, 0, 5, 2])
    table, lens, out = run(table, lens, [1, 1], int32([1, 3]))  # two samples end; their pages are free again
    table, used = cuda_ops.paged_compact(pool, table, lens)
    assert torch.isfinite(out).all()
    assert cuda_ops.decode_status() == 0, "the pool was full"
    return {"tokens": int(lens.sum()), "pages after the fork": forked, "pages at the end": int(used)}


if __name__ == "__main__":
    print(main())
