"""The chunked step under torch.compile: operators that write to lists of tensors and to their arguments."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_pages import int32

pytestmark = pytest.mark.gpu

HQ, HKV, DIM, PAGE, PAGES = 8, 2, 64, 16, 40


def inputs(seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(torch.bfloat16)  # noqa: E731
    pool = [rand(PAGES, PAGE, HKV, DIM) for _ in range(4)]
    table = int32([[7, 3, 9, 0, 0, 0], [12, 1, 0, 0, 0, 0]])
    return pool, rand(9, HQ, DIM), rand(9, HKV, DIM), rand(9, HKV, DIM), table, int32([45, 20]), int32([2, 4, 3]), int32([0, 2, 6, 9]), int32([0, 1, 1])


def step(pool, q, k, v, table, lens, new, indptr, parents):
    from kernel_lab import cuda_ops

    table, lens, served = cuda_ops.paged_reserve(pool, table, lens, new, parents)
    outs = []
    for layer in range(2):
        caches = pool[2 * layer], pool[2 * layer + 1]
        cuda_ops.paged_kv_append(*caches, k * (layer + 1), v, table, torch.where(served, lens, -1), indptr=indptr)
        outs.append(cuda_ops.paged_chunk_attention(q * 1, *caches, table, lens + new, indptr))
    lens = lens + new
    cuda_ops.paged_copy_pages(pool, table[:1, 0].contiguous(), torch.full_like(table[:1, 0], PAGES - 1))
    table, used = cuda_ops.paged_compact(pool, table, lens)
    return table * 1, lens, served, used + 0, *outs


@pytest.mark.parametrize("mode", ["default", "reduce-overhead"])
def test_a_compiled_step_is_the_eager_one(mode):
    compiled = torch.compile(step, mode=mode, fullgraph=True)
    for seed in (1, 2, 3, 4):
        a, b = inputs(seed), inputs(seed)
        want = step(*a)
        torch.compiler.cudagraph_mark_step_begin()
        got = [t.clone() for t in compiled(*b)]
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        assert all(torch.equal(x, y) for x, y in zip(b[0], a[0]))  # the pools
        assert not torch.equal(b[0][0], inputs(seed)[0][0])


def test_a_compiled_step_over_8_bit_caches():
    def step8(q, pool, scales, k, v, table, lens, indptr):
        from kernel_lab import cuda_ops

        cuda_ops.paged_kv_append_fp8(*pool, k * 1, v, *scales, table, lens, indptr=indptr)
        lens = lens + (indptr[1:] - indptr[:-1])
        return cuda_ops.paged_chunk_attention_fp8(q, *pool, *scales, table, lens, indptr) * 1

    def fresh():
        pool, q, k, v, table, lens, _, indptr, _ = inputs(5)
        codes = [(t * 10).to(torch.float8_e4m3fn) for t in pool[:2]]
        return q, codes, [torch.full((HKV,), 0.05, device="cuda") for _ in range(2)], k, v, table, lens, indptr[:3].contiguous()

    a, b = fresh(), fresh()
    want = step8(*a)
    got = torch.compile(step8, fullgraph=True)(*b)
    rows = slice(0, 6)
    assert torch.equal(got[rows], want[rows])
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a[1], b[1]))
