"""The chunked step over pools of more than 2^31 elements and 2^32 bytes: only the pages in use are ever written here."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import chunk
from tests.test_gpu_pages import int32

pytestmark = pytest.mark.gpu

PAGE, HKV, DIM = 16, 8, 128


def room(gigabytes):
    if torch.cuda.mem_get_info()[0] < gigabytes << 30:
        pytest.skip("not enough memory free")


def pools(pages, dtype, layout):
    if layout == "heads":
        return [torch.empty(pages, HKV, PAGE, DIM, dtype=dtype, device="cuda").permute(0, 2, 1, 3) for _ in range(2)]
    if layout == "interleaved":
        both = torch.empty(pages, 2, PAGE, HKV, DIM, dtype=dtype, device="cuda")
        return [both[:, 0], both[:, 1]]
    return [torch.empty(pages, PAGE, HKV, DIM, dtype=dtype, device="cuda") for _ in range(2)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("layout", ["tokens", "heads", "interleaved"])
def test_attention(dtype, layout):
    from kernel_lab import cuda_ops

    room(80)
    pages = 300_000  # 4.9e9 elements
    cache = pools(pages, dtype, layout)
    ids = [pages - 1, 5, 262_144, 131_071, pages - 7]
    gen = torch.Generator(device="cuda").manual_seed(1)
    for t in cache:
        for p in ids:
            x = torch.randn(PAGE, HKV, DIM, generator=gen, device="cuda")
            t[p] = (x * 40).round().clamp(-127, 127).to(dtype) if dtype.itemsize == 1 else x.to(dtype)
    qtype = torch.float16 if dtype.itemsize == 1 else dtype
    q = torch.randn(7, 16, DIM, generator=gen, device="cuda").to(qtype)
    table, lens, ptr = [[*ids]], [75], [0, 7]
    f64 = lambda t: t.double().cpu().numpy()  # noqa: E731
    small = [torch.stack([t[p].float() for p in ids]) for t in cache]
    bits = {torch.bfloat16: 8, torch.float32: 24}.get(dtype, 11)
    args = [int32(table), int32(lens), int32(ptr)]
    if dtype.itemsize == 1:
        scales = [torch.zeros(pages, HKV, device="cuda") for _ in range(2)]
        for s in scales:
            s[ids] = torch.rand(len(ids), HKV, generator=gen, device="cuda") / 40
        got = cuda_ops.paged_chunk_attention_block8(q, *cache, *scales, *args)
        extra = {"k_scale": f64(scales[0][ids]), "v_scale": f64(scales[1][ids])}
    else:
        got, extra = cuda_ops.paged_chunk_attention(q, *cache, *args), {}
    want, tol = chunk.attention(f64(q), f64(small[0]), f64(small[1]), np.arange(5)[None], lens, ptr, DIM**-0.5, True, bits=bits, p_bits=bits, **extra)
    assert (np.abs(f64(got) - want) <= tol).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_append_copy_reserve_and_compact(dtype):
    from kernel_lab import cuda_ops

    room(40)
    pages = 300_000
    cache = pools(pages, dtype, "tokens")
    top, other = pages - 1, pages - 3
    gen = torch.Generator(device="cuda").manual_seed(2)
    rows = [torch.randn(20, HKV, DIM, generator=gen, device="cuda").to(torch.bfloat16) for _ in range(2)]
    raw = lambda t: t.view(torch.uint8) if t.dtype.itemsize == 1 else t  # noqa: E731
    for t in cache:
        for p in (top, other, 0, 1, 150_000):
            raw(t)[p].zero_()
    table, at, ptr = int32([[top, other]]), int32([3]), int32([0, 20])
    if dtype is torch.bfloat16:
        cuda_ops.paged_kv_append(*cache, *rows, table, at, indptr=ptr)
        want = rows
    else:
        one = torch.ones(HKV, device="cuda")
        cuda_ops.paged_kv_append_fp8(*cache, *rows, one, one, table, at, indptr=ptr)
        want = [r.float().clamp(-448, 448).to(dtype) for r in rows]
    kept = []
    for t, w in zip(cache, want):
        both = torch.cat([raw(t)[top], raw(t)[other]])
        assert torch.equal(both[3:23], raw(w)) and not both[:3].any() and not both[23:].any()
        kept.append(both)
    cuda_ops.paged_copy_pages(cache, int32([top]), int32([150_000]))
    assert all(torch.equal(raw(t)[150_000], both[:PAGE]) for t, both in zip(cache, kept))
    # Two forks: a copy of the last page in the lowest free one.
    forks, lens, served = cuda_ops.paged_reserve(cache, table, at + 20, int32([1, 1]), int32([0, 0]))
    assert served.all() and forks.tolist() == [[top, other], [top, 0]] and lens.tolist() == [23, 23]
    assert all(torch.equal(raw(t)[0], both[PAGE:]) for t, both in zip(cache, kept))
    packed, used = cuda_ops.paged_compact(cache, forks, lens)
    assert int(used) == 3 and packed.tolist() == [[2, 1], [2, 0]]
    for t, both in zip(cache, kept):
        assert torch.equal(raw(t)[2], both[:PAGE]) and torch.equal(raw(t)[1], both[PAGE:]) and torch.equal(raw(t)[0], both[PAGE:])
