"""Calls captured into CUDA graphs: their scratch is the graph's own, whatever is captured, run eagerly or dropped
beside it."""

from __future__ import annotations

import gc
import threading
import time

import numpy as np
import pytest
import torch

from tests.test_gpu_block8 import Pool, make_q

pytestmark = pytest.mark.gpu

BAD_PAGE = 1


class Problem:
    """Selection, sparse and dense decode over a block-scaled pool, and decode over a bf16 pool: rows that many CTAs
    and selection blocks share, so that every kernel counts arrivals."""

    def __init__(self, lens, seed, num_selected=40, hq=16):
        from kernel_lab.kv_cache import random_paged_pool

        self.pool = Pool("e4m3", lens, 2, 128, 16, seed=seed)
        self.q = make_q(self.pool, hq, torch.bfloat16, seed)
        self.state, (self.table, self.lens) = self.pool.gpu(), self.pool.tables()
        self.bounds = torch.from_numpy(self.pool.bounds).cuda()
        self.num_selected = num_selected
        self.plain_q, self.plain = random_paged_pool(lens, hq, 2, 128, 16, dtype=torch.bfloat16, device="cuda", seed=seed)

    def __call__(self):
        from kernel_lab import cuda_ops

        chosen = cuda_ops.paged_block_select(self.q, self.state["k_cache"], self.state["k_scale"], self.bounds, self.table,
                                             self.lens, self.num_selected)
        step = {"block_table": self.table, "seq_lens": self.lens}
        kv = self.plain
        return [
            chosen,
            cuda_ops.paged_decode_attention_block8(self.q, **self.state, **step, selected=chosen),
            cuda_ops.paged_decode_attention_block8(self.q, **self.state, **step),
            cuda_ops.paged_decode_attention(self.plain_q, kv.k_cache, kv.v_cache, kv.block_table, kv.seq_lens),
        ]

    def capture(self, stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = self()
        return graph, got


def spoil(tensors):
    for t in tensors:
        t.fill_(-7)


def same(got, want):
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_graphs_of_one_stream_replay_in_any_order():
    """Neither stream nor graph has scratch before its capture; the second graph runs first."""
    a, b = Problem([6000, 5, 3000], 1), Problem([5000, 5000], 2)
    want_a, want_b = a(), b()
    stream = torch.cuda.Stream()
    (graph_a, got_a), (graph_b, got_b) = a.capture(stream), b.capture(stream)
    for order in ("ba", "ab", "bb", "aa"):
        spoil(got_a + got_b)
        for which in order:
            (graph_a if which == "a" else graph_b).replay()
        if "a" in order:
            same(got_a, want_a)
        if "b" in order:
            same(got_b, want_b)


def test_a_larger_call_after_the_capture_leaves_the_graph_its_memory():
    small, large = Problem([6000, 700], 3), Problem([3000, 50, 20, 100] * 12, 4, hq=32)  # more counters, larger states
    want, stream = small(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        small()  # the stream's own scratch
    stream.synchronize()
    graph, got = small.capture(stream)
    with torch.cuda.stream(stream):
        want_large = large()
        # What the stream's outgrown buffers would have become.
        others = [torch.full((n,), 7, dtype=torch.uint8, device="cuda") for n in [1 << 12, 1 << 16, 1 << 20, 3 << 20, 12 << 20] * 8]
        stream.synchronize()
        for _ in range(3):
            spoil(got)
            stream.synchronize()
            graph.replay()
            same(got, want)
            assert all(bool((t == 7).all()) for t in others)
        same(large(), want_large)


def test_a_capture_that_outgrows_its_first_scratch():
    small, large = Problem([2000, 700], 5), Problem([3000, 50, 20, 100] * 12, 6, hq=32)
    want = small() + large() + small()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        got = small() + large() + small()
    for _ in range(2):
        spoil(got)
        graph.replay()
        same(got, want)


def test_graphs_run_beside_each_other_and_beside_eager_calls():
    a, b, c = Problem([6000, 3000], 7), Problem([5000, 5000], 8), Problem([7000, 3], 9)
    want_a, want_b, want_c = a(), b(), c()
    stream, s1, s2 = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.Stream()
    (graph_a, got_a), (graph_b, got_b) = a.capture(stream), b.capture(stream)
    torch.cuda.synchronize()
    for _ in range(5):
        for _ in range(8):
            with torch.cuda.stream(s1):
                graph_a.replay()
            with torch.cuda.stream(s2):
                graph_b.replay()
            with torch.cuda.stream(stream):
                got_c = c()
        same(got_a, want_a)
        same(got_b, want_b)
        same(got_c, want_c)


def test_status_of_a_graphs_calls_is_read_and_kept():
    from kernel_lab import cuda_ops

    bad = Problem([64, 64], 10)
    bad.table[1, 2] = 1 << 20
    cuda_ops.decode_status(clear=True)
    graph, _ = bad.capture(torch.cuda.Stream())
    assert cuda_ops.decode_status() == 0
    graph.replay()
    assert cuda_ops.decode_status() == BAD_PAGE == cuda_ops.decode_status(clear=True)  # sticky until cleared
    assert cuda_ops.decode_status() == 0
    graph.replay()
    torch.cuda.synchronize()
    del graph
    gc.collect()
    time.sleep(0.2)
    assert cuda_ops.decode_status(clear=True) == BAD_PAGE
    assert cuda_ops.decode_status() == 0


def test_a_graphs_scratch_goes_with_it():
    problem = Problem([6000, 700], 11)
    stream = torch.cuda.Stream()
    problem()
    held = []
    for _ in range(12):
        graph, got = problem.capture(stream)
        graph.replay()
        torch.cuda.synchronize()
        del graph, got
        gc.collect()
        time.sleep(0.05)
        torch.cuda.empty_cache()
        held.append(torch.cuda.mem_get_info()[0])
    assert min(held[2:]) >= held[1] - (2 << 20)


def test_two_threads_grow_one_streams_scratch():
    """Each thread's calls need more than the ones before; both launch on one stream."""
    problems = [[Problem([500 * (k + 1), 9] * 6 * (k + 1), 20 + 10 * t + k, hq=16 if k < 2 else 32) for k in range(4)] for t in range(2)]
    want = [[p() for p in row] for row in problems]
    stream, got = torch.cuda.Stream(), [[], []]
    torch.cuda.synchronize()

    def work(t):
        with torch.cuda.stream(stream):
            for p in problems[t]:
                for _ in range(4):
                    got[t].append(p())

    threads = [threading.Thread(target=work, args=(t,)) for t in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for t in range(2):
        assert len(got[t]) == 16
        for i, outs in enumerate(got[t]):
            same(outs, want[t][i // 4])


def test_torch_compile_with_graphs():
    """Its captures allow no memory of their pool but the outputs'."""
    problem = Problem([6000, 700], 12)

    def step(q, plain_q, chosen):
        from kernel_lab import cuda_ops

        kv = problem.plain
        sparse = cuda_ops.paged_decode_attention_block8(q * 1, **problem.state, block_table=problem.table,
                                                        seq_lens=problem.lens, selected=chosen)
        return sparse * 1, cuda_ops.paged_decode_attention(plain_q * 1, kv.k_cache, kv.v_cache, kv.block_table, kv.seq_lens) * 1

    args = problem.q, problem.plain_q, problem()[0]
    want = step(*args)
    compiled = torch.compile(step, mode="reduce-overhead", fullgraph=True)
    for _ in range(4):
        torch.compiler.cudagraph_mark_step_begin()
        got = [t.clone() for t in compiled(*args)]
        same(got, want)


def test_a_captured_step_reads_what_each_replay_finds():
    """norm -> append -> selection -> decode, captured once and replayed with other activations and positions: outputs,
    caches, scales and bounds are the eager step's every time."""
    from kernel_lab import cuda_ops

    hq, hkv, dim, group = 16, 4, 128, 128
    pool = Pool("e4m3", [4000, 2500, 40], hkv, dim, 16, "hnd", seed=70)
    table, _ = pool.tables()
    width = (hq + 2 * hkv) * dim
    weight = torch.randn(width, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()

    def start():
        return {**pool.gpu(), "k_bounds": torch.from_numpy(pool.bounds).cuda(),
                "residual": torch.randn(3, width, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()}

    def step(s, x, position):
        codes, scales, residual = cuda_ops.fused_add_rms_norm_fp8(x, s["residual"], weight, 1e-5, group_size=group)
        s["residual"].copy_(residual)
        rows = (codes.float().unflatten(-1, (-1, group)) * scales[..., None]).to(torch.bfloat16).view(3, hq + 2 * hkv, dim)
        q, k, v = rows[:, :hq], rows[:, hq : hq + hkv], rows[:, hq + hkv :]
        cache = {name: s[name] for name in ("k_cache", "v_cache", "k_scale", "v_scale")}
        cuda_ops.paged_kv_append_block8(*cache.values(), k, v, table, position, k_bounds=s["k_bounds"])
        lens = position + 1
        chosen = cuda_ops.paged_block_select(q, s["k_cache"], s["k_scale"], s["k_bounds"], table, lens, 20)
        sparse = cuda_ops.paged_decode_attention_block8(q, **cache, block_table=table, seq_lens=lens, selected=chosen)
        return [codes.view(torch.uint8), scales, chosen, sparse,
                cuda_ops.paged_decode_attention_block8(q, **cache, block_table=table, seq_lens=lens)]

    xs = [torch.randn(3, width, generator=torch.Generator().manual_seed(10 + t)).to(torch.bfloat16).cuda() for t in range(5)]
    positions = [torch.tensor(p, dtype=torch.int32, device="cuda") for p in
                 ([3990, 2490, 0], [3991, 2491, 1], [3992, 30, 2], [100, 2492, 31], [3993, 0, 39])]
    step(start(), xs[0], positions[0])
    eager, captured = start(), start()
    x, position = xs[0].clone(), positions[0].clone()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        got = step(captured, x, position)
    for t in range(5):
        want = step(eager, xs[t], positions[t])
        x.copy_(xs[t])
        position.copy_(positions[t])
        graph.replay()
        same(got, want)
        for name in eager:
            a, b = (s[name].view(torch.uint8) if s[name].dtype == torch.float8_e4m3fn else s[name] for s in (captured, eager))
            assert torch.equal(a, b), name
