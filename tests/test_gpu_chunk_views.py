"""Queries that are views of any kind: the rows that the kernel cannot step over are copied first."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_pages import int32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("view", ["one row for all", "rows that overlap", "reversed heads", "every other element"])
@pytest.mark.parametrize("traced", [False, True])
def test_queries_of_any_strides(dtype, view, traced):
    from torch.utils._python_dispatch import TorchDispatchMode

    from kernel_lab import cuda_ops

    class Watched(TorchDispatchMode):  # past the direct calls
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    gen = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(dtype)  # noqa: E731
    k, v = rand(6, 16, 2, 64), rand(6, 16, 2, 64)
    if view == "one row for all":
        q = rand(1, 8, 64).expand(9, -1, -1)
    elif view == "rows that overlap":
        q = rand(17 * 64).as_strided((9, 8, 64), (64, 64, 1))
    elif view == "reversed heads":
        q = rand(9, 64, 8).transpose(1, 2)
    else:
        q = rand(9, 8, 128)[..., ::2]
    args = k, v, int32([[4, 0, 2], [1, 5, 3]]), int32([40, 33]), int32([0, 4, 9])
    want = cuda_ops.paged_chunk_attention(q.contiguous(), *args)
    if traced:
        with Watched():
            got = cuda_ops.paged_chunk_attention(q, *args)
    else:
        got = cuda_ops.paged_chunk_attention(q, *args)
    assert torch.equal(got, want)
