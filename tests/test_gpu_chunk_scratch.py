"""The scratch of the chunked step's calls: threads that share a stream, what a wait that ran out leaves behind."""

from __future__ import annotations

import gc
import threading
import time

import numpy as np
import pytest
import torch

from tests.test_gpu_chunk import Problem
from tests.test_gpu_pages import int32, tables

pytestmark = pytest.mark.gpu


class Pages:
    """Forks with copies on write, and compaction, of one pool: run again on the same table they do the same again."""

    def __init__(self, seed):
        rng = np.random.RandomState(seed)
        lens, self.pages, page = rng.randint(1, 300, 40), 3000, 16
        table = tables(lens, page, 64, self.pages, seed)
        self.pool = [torch.arange(self.pages, device="cuda", dtype=torch.int32)[:, None].repeat(1, 16).contiguous()]
        self.table, self.lens = int32(table), int32(lens)
        self.new, self.parents = int32(rng.randint(0, 60, 80)), int32(rng.randint(-1, 40, 80))
        self.out = [torch.zeros(80, 64, dtype=torch.int32, device="cuda"), torch.zeros(80, dtype=torch.int32, device="cuda"),
                    torch.zeros(80, dtype=torch.bool, device="cuda")]
        self.compacted, self.used = torch.zeros(40, 64, dtype=torch.int32, device="cuda"), torch.zeros((), dtype=torch.int32, device="cuda")

    def __call__(self):
        ops = torch.ops.kernel_lab
        ops.paged_reserve(*self.out, self.pool, self.table, self.lens, self.new, self.parents, 16)
        ops.paged_compact(self.compacted, self.used, self.pool, self.table, self.lens, 16)
        return [t.clone() for t in (*self.out, self.compacted, self.used)]


class Attention:
    """Rows that many CTAs share: pieces and counters in scratch."""

    def __init__(self, seed):
        p = Problem([(1, 6000), (4, 3000), (70, 700)], 8, 2, 128, 16, torch.bfloat16, seed=seed)
        ints = [torch.from_numpy(np.asarray(x, np.int32)).cuda() for x in (p.table, p.lens, p.indptr)]
        self.out = torch.zeros_like(p.q.cuda())
        self.args = [self.out, p.q.cuda(), p.device_cache("k"), p.device_cache("v"), *ints, 128**-0.5, True]

    def __call__(self):
        torch.ops.kernel_lab.paged_chunk_attention(*self.args)
        return [self.out.clone()]


def test_threads_share_a_stream():
    """Bookkeeping of several launches in some threads, attention that writes to the same scratch in others."""
    from kernel_lab import cuda_ops

    cuda_ops.decode_status(clear=True)
    calls = [Pages(1), Attention(2), Pages(3), Attention(4)]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    stream, wrong = torch.cuda.Stream(), []

    def work(call, expected):
        with torch.cuda.stream(stream):
            got = [call() for _ in range(100)]
            wrong.extend(1 for g in got if not all(torch.equal(a, b) for a, b in zip(g, expected)))

    threads = [threading.Thread(target=work, args=x) for x in zip(calls, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not wrong
    with torch.cuda.stream(stream):
        assert cuda_ops.decode_status(clear=True) == 0


def spoil(sync):
    """What a call leaves whose wait ran out: the status bit, and counters (page marks, for the bookkeeping) that are not zero."""
    words = sync[: sync.numel() // 4 * 4].view(torch.int32)
    words[64:] = 1
    words[0] = 4


@pytest.mark.parametrize("call", [Pages, Attention])
def test_clearing_a_timeout_makes_the_scratch_usable_again(call):
    """No wait runs out here: its traces are written by hand. Nothing runs on them before they are cleared."""
    from kernel_lab import _C, cuda_ops

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        cuda_ops.decode_status(clear=True)
        run = call(5)
        want = run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = run()
        graph.replay()
        stream.synchronize()
        buffers = _C.current_sync_buffers()
        for s in buffers:
            spoil(s)
        stream.synchronize()
        assert cuda_ops.decode_status() == 4  # reading alone changes nothing
        assert all(int(s[256]) == 1 for s in buffers)
        assert cuda_ops.decode_status(clear=True) == 4 and cuda_ops.decode_status() == 0
        assert not any(s.any() for s in buffers)
        for _ in range(2):
            assert all(torch.equal(a, b) for a, b in zip(run(), want))
            for t in got:
                t.zero_()
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert cuda_ops.decode_status(clear=True) == 0


def test_a_dead_graphs_timeout_is_cleared_before_its_scratch_is_used_again():
    from kernel_lab import _C, cuda_ops

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        cuda_ops.decode_status(clear=True)
        run = Attention(6)
        want = run()
        before = {s.data_ptr() for s in _C.current_sync_buffers()}
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            run()
        owned = [s for s in _C.current_sync_buffers() if s.data_ptr() not in before]
        assert len(owned) == 1
        spoil(owned[0])
        stream.synchronize()
        del graph
        gc.collect()
        time.sleep(0.05)
        assert cuda_ops.decode_status(clear=True) == 4
        assert not owned[0].any()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = run()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and cuda_ops.decode_status() == 0


def test_lengths_updated_in_place():
    """Where every row is its own parent the new lengths may take the old ones' place, those past the table clamped."""
    from kernel_lab import cuda_ops

    cuda_ops.decode_status(clear=True)
    table = int32([[4, 5] + [0] * 600, [7] * 602])
    pool = [torch.arange(40, device="cuda", dtype=torch.int32)[:, None].contiguous()]
    lens, out, served = int32([20, 602 * 16 + 5]), torch.zeros_like(table), torch.zeros(2, dtype=torch.bool, device="cuda")
    torch.ops.kernel_lab.paged_reserve(out, lens, served, pool, table, lens, int32([20, 0]), None, 16)
    assert cuda_ops.decode_status(clear=True) == 2
    assert lens.tolist() == [20, 602 * 16] and served.all() and out[0].tolist() == [4, 5, 0] + [0] * 599 and (out[1] == 7).all()
    with pytest.raises(RuntimeError):
        torch.ops.kernel_lab.paged_reserve(out, lens, served, pool, table, lens, int32([20, 0]), int32([1, 0]), 16)
