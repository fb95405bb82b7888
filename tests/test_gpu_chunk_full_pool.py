"""The chunked step where the pool runs out: rows that got no pages write nothing, and the others go on."""

from __future__ import annotations

import importlib.util

import numpy as np
import pytest
import torch

from oracle import chunk
from tests.conftest import REPO
from tests.test_gpu_pages import int32

pytestmark = pytest.mark.gpu

HQ, HKV, DIM, PAGE, PAGES, WIDTH = 8, 2, 64, 16, 7, 6
# Sequence 0 has room in page 3, sequence 1's last page is partly filled, sequence 2's are full; no page is free.
TABLE = [[0, 3, 0, 0, 0, 0], [1, 2, 0, 0, 0, 0], [4, 5, 6, 0, 0, 0]]
LENS = [30, 20, 48]


def example():
    spec = importlib.util.spec_from_file_location("chunk_step", REPO / "examples" / "chunk_step.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("captured", [False, True])
def test_rows_without_pages_write_nothing(captured):
    from kernel_lab import cuda_ops

    step = example().step
    gen = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(torch.bfloat16)  # noqa: E731
    start = [rand(PAGES, PAGE, HKV, DIM) for _ in range(2)]
    pool = [t.clone() for t in start]
    table, lens = int32(TABLE), int32(LENS)
    # A token in its page; the writer that keeps the shared page; one that would need a copy of it; one that would need a
    # page; two empty rows.
    parents, new = int32([0, 1, 1, 2, -1, 7]), int32([1, 2, 2, 3, 2, 1])
    counts = new.tolist()
    indptr = np.cumsum([0, *counts]).astype(np.int32)
    rows = int(indptr[-1])
    q, k, v, ptr = rand(rows, HQ, DIM), rand(rows, HKV, DIM), rand(rows, HKV, DIM), int32(indptr)

    def run():
        return step(pool, q, k, v, table, lens, new, ptr, parents)

    cuda_ops.decode_status(clear=True)
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = run()
        graph.replay()
    else:
        got = run()
    torch.cuda.synchronize()
    assert cuda_ops.decode_status(clear=True) == 32
    got_table, got_lens, served, out = got
    assert served.tolist() == [True, True, False, False, False, False]
    assert got_lens.tolist() == [31, 22, 20, 48, 0, 0]
    want = [t.clone() for t in start]
    for w, fresh in zip(want, (k, v)):
        w[3, 14] = fresh[0]
        w[2, 4:6] = fresh[1:3]
    assert torch.equal(pool[0], want[0]) and torch.equal(pool[1], want[1])
    f64 = lambda t: t.double().cpu().numpy()  # noqa: E731
    ref, tol = chunk.attention(f64(q[:3]), f64(pool[0]), f64(pool[1]), got_table.cpu().numpy(), [31, 22], [0, 1, 3], DIM**-0.5, True, bits=8, p_bits=8)
    assert (np.abs(f64(out[:3]) - ref) <= tol).all()
    if captured:  # sequence 2 has ended, two rows only hold what the others copy: its three pages serve all
        for p, s in zip(pool, start):
            p.copy_(s)
        parents.copy_(int32([0, 1, 1, 0, -1, 1]))
        new.copy_(int32([1, 2, 2, 0, 2, 0]))
        ptr.copy_(int32([0, 1, 3, 5, 5, 7, 7]))
        graph.replay()
        torch.cuda.synchronize()
        assert cuda_ops.decode_status(clear=True) == 0
        assert served.tolist() == [True, True, True, True, False, True] and got_lens.tolist() == [31, 22, 22, 30, 0, 20]
        assert got_table[:, 1].tolist() == [4, 5, 6, 3, 0, 2]
        for p, s, fresh in zip(pool, start, (k, v)):
            for page, source, at, rows in ((4, 3, 14, slice(0, 1)), (5, 2, 4, slice(1, 3)), (6, 2, 4, slice(3, 5))):
                page_wanted = s[source].clone()
                page_wanted[at : at + rows.stop - rows.start] = fresh[rows]
                assert torch.equal(p[page], page_wanted)
            assert torch.equal(p[:4], s[:4])
