"""The pages of a cache: copied, reserved (growth, forks, copies on write), compacted. Everything is exact."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import chunk

pytestmark = pytest.mark.gpu


def int32(x):
    return torch.from_numpy(np.asarray(x, np.int32)).cuda()


def pools(pages, page, seed=0):
    """Tensors of many kinds: 16-, 8- and 32-bit, pages of an odd number of bytes, heads first, keys and values interleaved."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randint(-120, 120, s, generator=gen, device="cuda", dtype=torch.int32)  # noqa: E731
    both = rand(pages, 2, page, 2, 24).to(torch.bfloat16)
    return [
        rand(pages, page, 2, 64).to(torch.float16),
        rand(pages, 2, page, 80).to(torch.int8).permute(0, 2, 1, 3),
        rand(pages, 3).float(),
        both[:, 0],
        both[:, 1],
        rand(pages, page, 1, 5).to(torch.int8),
        rand(pages, 40000).to(torch.int8),
        rand(pages),
        rand(pages, 7).to(torch.int16),
    ]


def copies(tensors):
    return [t.clone() for t in tensors]


def moved(tensors, pairs):
    out = copies(tensors)
    for s, d in pairs:
        for o, t in zip(out, tensors):
            o[d] = t[s]
    return out


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("pairs", [1, 2, 37, 300])
def test_copy(pairs):
    from kernel_lab import cuda_ops

    t = pools(2 * pairs + 5, 8)
    order = np.random.RandomState(pairs).permutation(2 * pairs)
    src, dst = order[:pairs], order[pairs:]
    want = moved(t, zip(src.tolist(), dst.tolist()))
    cuda_ops.paged_copy_pages(t, int32(src), int32(dst))
    assert same(t, want)


def test_copy_skips_and_reports():
    from kernel_lab import cuda_ops

    t = pools(10, 8)
    want = moved(t, [(3, 4)])
    cuda_ops.decode_status(clear=True)
    cuda_ops.paged_copy_pages(t, int32([-1, 3, 2]), int32([5, 4, -7]))
    assert same(t, want) and cuda_ops.decode_status() == 0
    cuda_ops.paged_copy_pages(t, int32([10, 1]), int32([5, 2**31 - 1]))
    assert same(t, want) and cuda_ops.decode_status(clear=True) == 1
    cuda_ops.paged_copy_pages(t, int32([]), int32([]))


def test_copy_of_many_tensors():
    """More tensors than a launch takes."""
    from kernel_lab import cuda_ops

    t = [torch.full((6, 16), float(i), device="cuda") for i in range(150)]
    for i, x in enumerate(t):
        x[2] = i + 0.5
    cuda_ops.paged_copy_pages(t, int32([2]), int32([5]))
    assert all((x[5] == i + 0.5).all() and (x[0] == i).all() for i, x in enumerate(t))


def tables(lens, page, width, pages, seed, shared=()):
    """Rows of shuffled pages; shared: (row, other, tokens) lets `row` begin with the pages of `other`'s first tokens."""
    order = np.random.RandomState(seed).permutation(pages)
    table = np.random.RandomState(seed + 1).randint(0, pages, (len(lens), width)).astype(np.int32)  # past the pages: anything
    at = 0
    for b, n in enumerate(lens):
        k = -(-n // page)
        table[b, :k] = order[at : at + k]
        at += k
    for row, other, tokens in shared:
        k = -(-tokens // page)
        table[row, :k] = table[other, :k]
    return table


def check_reserve(lens, new, page, width, pages, parents=None, seed=0, shared=(), status=0):
    from kernel_lab import cuda_ops

    table = tables(lens, page, width, pages, seed, shared)
    t = pools(pages, page, seed)
    want_table, want_lens, want_served, pairs = chunk.reserve(table, lens, new, page, pages, parents)
    want = moved(t, pairs)
    cuda_ops.decode_status(clear=True)
    before = int32(table)
    got = cuda_ops.paged_reserve(t, before, int32(lens), int32(new), None if parents is None else int32(parents), page_size=page)
    assert cuda_ops.decode_status(clear=True) == status
    np.testing.assert_array_equal(got[2].cpu().numpy(), want_served)
    np.testing.assert_array_equal(got[1].cpu().numpy(), want_lens)
    np.testing.assert_array_equal(got[0].cpu().numpy(), want_table)
    assert same(t, want) and torch.equal(before, int32(table))
    return pairs


@pytest.mark.parametrize("page", [1, 3, 16])
@pytest.mark.parametrize("new", [[0, 1, 5, 16, 1, 40, 0, 1], [0] * 8, [1] * 8, [-3, 7, 2**20, 1, 1, 0, 2, 3]])
def test_reserve_growth(page, new):
    lens = [0, 16, 17, 31, 1, 0, 5, 48]
    width = 100
    status = 32 if 2**20 in new else 0
    check_reserve(lens, new, page, width, 400, status=status)


def test_reserve_runs_out():
    """Seven pages in use and needs of 31 + 6 + 0 + 1 + 0 (31 + 5 + 0 + 1 + 0): the row that they do not suffice for gets
    nothing, nor do those after it that need any."""
    check_reserve([20, 16, 32, 16, 7], [500, 90, 0, 16, 3], 16, 40, 8 + 37)
    check_reserve([20, 16, 32, 16, 7], [500, 80, 0, 16, 3], 16, 40, 8 + 37)
    check_reserve([20, 16, 32, 16, 7], [500, 90, 0, 16, 3], 16, 40, 7 + 37, status=32)
    check_reserve([20, 16, 32, 16, 7], [500, 90, 0, 16, 17], 16, 40, 7 + 36, status=32)
    check_reserve([20, 16, 32, 16, 7], [500, 90, 0, 16, 3], 16, 40, 7, status=32)
    check_reserve([16, 16], [1, 1], 16, 4, 3, status=32)
    check_reserve([16, 16], [1, 1], 16, 4, 4)
    check_reserve([16, 16], [0, 0], 16, 1, 2)


def test_reserve_forks_and_copies_on_write():
    lens = [20, 33, 16, 0, 7]
    # Three rows of sequence 0: its full page is shared, the partly filled one is the first row's, two copies.
    pairs = check_reserve(lens, [1] * 7, 16, 8, 60, parents=[0, 0, 1, 0, 2, 2, -1])
    assert len(pairs) == 2
    # A row that does not write keeps the page as it is: all writers copy.
    assert len(check_reserve(lens, [1, 0, 1, 1], 16, 8, 60, parents=[0, 0, 0, 0])) == 3
    # Nobody writes: nothing is copied.
    assert not check_reserve(lens, [0] * 4, 16, 8, 60, parents=[0, 0, 4, 4])
    # Dropped sequences' pages are given out again; parents out of range make empty rows.
    check_reserve(lens, [40, 40, 5], 16, 8, 12, parents=[4, 5, 2**31 - 1])
    # More rows than sequences, fewer, none.
    check_reserve(lens, [3] * 300, 16, 8, 900, parents=[i % 5 for i in range(300)])
    check_reserve(lens, [3], 16, 8, 30, parents=[3])


def test_reserve_shared_prefixes():
    """Rows that share pages without being forks of one call: a prefix held in full pages, one cut within a page."""
    lens = [64, 70, 40, 64, 41]
    shared = [(1, 0, 64), (2, 0, 40), (3, 0, 64), (4, 2, 41)]
    check_reserve(lens, [1, 1, 1, 0, 1], 16, 8, 60, shared=shared)
    check_reserve(lens, [0, 0, 1, 0, 0], 16, 8, 60, shared=shared)


def test_reserve_large_and_odd_pools():
    rng = np.random.RandomState(5)
    for pages, batch in [(1, 1), (5, 1), (4095, 40), (4097, 40), (33001, 700), (70001, 1500)]:
        lens = rng.randint(0, max(2, pages * 16 // batch // 2), batch)
        page, width = 16, int(lens.max()) // 16 + 6
        new = rng.randint(0, 50, batch)
        table = tables(lens, page, width, pages, 1)
        from kernel_lab import cuda_ops

        t = [torch.arange(pages, device="cuda", dtype=torch.int32)[:, None].repeat(1, 4).contiguous()]
        parents = rng.randint(-1, batch, batch) if pages > 5 else None
        want = chunk.reserve(table, lens, new, page, pages, None if parents is None else parents.tolist())
        got = cuda_ops.paged_reserve(t, int32(table), int32(lens), int32(new), None if parents is None else int32(parents), page_size=page)
        for g, w in zip(got, want):
            np.testing.assert_array_equal(g.cpu().numpy(), w)
        contents = np.arange(pages)
        for s, d in want[3]:
            contents[d] = s
        np.testing.assert_array_equal(t[0][:, 0].cpu().numpy(), contents)
        cuda_ops.decode_status(clear=True)


def check_compact(lens, page, width, pages, seed=0, shared=()):
    from kernel_lab import cuda_ops

    table = tables(lens, page, width, pages, seed, shared)
    t = pools(pages, page, seed)
    want_table, want_used, pairs = chunk.compact(table, lens, page, pages)
    want = moved(t, pairs)
    got, used = cuda_ops.paged_compact(t, int32(table), int32(lens), page_size=page)
    assert int(used) == want_used
    np.testing.assert_array_equal(got.cpu().numpy(), want_table)
    assert same(t, want)
    return pairs


@pytest.mark.parametrize("page", [1, 16])
def test_compact(page):
    assert check_compact([20, 33, 0, 16, 7], page, 40, 300)
    assert check_compact([64, 70, 40, 64, 41], 16, 8, 60, shared=[(1, 0, 64), (2, 0, 40), (3, 0, 64), (4, 2, 41)])
    check_compact([0, 0], page, 4, 10)
    check_compact([page * 3], page, 3, 3)  # a full pool
    check_compact([1], page, 1, 1)
    check_compact([1], page, 1, 2)


def test_compact_large_and_odd_pools():
    from kernel_lab import cuda_ops

    rng = np.random.RandomState(6)
    for pages, batch in [(4095, 40), (4097, 3), (33001, 700), (70001, 1500)]:
        lens = rng.randint(0, max(2, pages * 16 // batch), batch)
        table = tables(lens, 16, int(lens.max()) // 16 + 1, pages, 1)
        t = [torch.arange(pages, device="cuda", dtype=torch.int32)[:, None].repeat(1, 4).contiguous()]
        want_table, want_used, pairs = chunk.compact(table, lens, 16, pages)
        got, used = cuda_ops.paged_compact(t, int32(table), int32(lens), page_size=16)
        assert int(used) == want_used
        np.testing.assert_array_equal(got.cpu().numpy(), want_table)
        contents = np.arange(pages)
        for s, d in pairs:
            contents[d] = s
        np.testing.assert_array_equal(t[0][:, 0].cpu().numpy(), contents)


def test_entries_outside_the_pool_are_taken_over():
    from kernel_lab import cuda_ops

    table, lens = np.array([[5, -2, 7, 0], [99, 3, 0, 0]], np.int32), [40, 20]
    t = [torch.arange(10, device="cuda", dtype=torch.int32)[:, None].contiguous()]
    cuda_ops.decode_status(clear=True)
    got = cuda_ops.paged_reserve(t, int32(table), int32(lens), int32([20, 1]), page_size=16)
    assert cuda_ops.decode_status(clear=True) == 1
    assert got[0].tolist() == [[5, -2, 7, 0], [99, 3, 0, 0]]
    got, used = cuda_ops.paged_compact(t, int32(table), int32(lens), page_size=16)
    assert cuda_ops.decode_status(clear=True) == 1
    assert got.tolist() == [[1, -2, 2, 0], [99, 0, 0, 0]] and int(used) == 3


def test_lengths_past_the_table_are_clamped():
    from kernel_lab import cuda_ops

    t = [torch.arange(10, device="cuda", dtype=torch.int32)[:, None].contiguous()]
    cuda_ops.decode_status(clear=True)
    _, lens, served = cuda_ops.paged_reserve(t, int32([[4, 5]]), int32([100]), int32([0]), page_size=16)
    assert lens.tolist() == [32] and served.tolist() == [True] and cuda_ops.decode_status(clear=True) == 2


def test_a_captured_step_replays_with_other_inputs():
    """Reserve, append and attention in one graph, replayed as the sequences grow; another graph beside it."""
    from kernel_lab import cuda_ops

    hq, hkv, dim, page, batch = 8, 2, 64, 16, 3
    gen = torch.Generator(device="cuda").manual_seed(40)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(torch.bfloat16)  # noqa: E731
    pool = [torch.zeros(64, page, hkv, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    table, lens = torch.zeros(batch, 12, dtype=torch.int32, device="cuda"), int32([0, 0, 0])
    q, k, v, new = rand(6, hq, dim), rand(6, hkv, dim), rand(6, hkv, dim), int32([1, 2, 3])
    ptr = int32([0, 1, 3, 6])

    def step():
        got, _, served = cuda_ops.paged_reserve(pool, table, lens, new)
        table.copy_(got)
        cuda_ops.paged_kv_append(*pool, k, v, table, lens, indptr=ptr)
        lens.add_(new)
        return cuda_ops.paged_chunk_attention(q, *pool, table, lens, ptr), served

    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out, served = step()
        graphs.append((g, out, served))
    lens.zero_()
    history = [[] for _ in range(batch)]
    for i in range(40):
        for t in (q, k, v):
            t.copy_(rand(*t.shape))
        g, out, served = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        assert served.all()
        for b in range(batch):
            history[b].append((k[ptr[b] : ptr[b + 1]].clone(), v[ptr[b] : ptr[b + 1]].clone()))
    held = [n for b in range(batch) for n in table[b, : -(-int(lens[b]) // page)].tolist()]
    assert len(set(held)) == len(held) and max(held) < len(held)
    for b in range(batch):
        keys, values = (torch.cat([h[i] for h in history[b]]).double().repeat_interleave(hq // hkv, 1) for i in (0, 1))
        x = q[ptr[b] : ptr[b + 1]].double()
        s = torch.einsum("ihd,jhd->hij", x, keys) * dim**-0.5
        n, total = x.shape[0], keys.shape[0]
        s.masked_fill_(torch.arange(total, device="cuda") > total - n + torch.arange(n, device="cuda")[:, None], -np.inf)
        want = torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), values)
        # bf16: probabilities and outputs rounded, 2^-8 each of values of at most 4.
        assert (out[ptr[b] : ptr[b + 1]].double() - want).abs().max() <= 2 * 4 * 2.0**-8


def test_the_example_runs():
    """A prompt of 602 tokens in 38 pages; four samples, three with a copy of the last page; two go on, at 605 + 1 and 608 - 2 + 1."""
    import importlib.util

    from tests.conftest import REPO

    spec = importlib.util.spec_from_file_location("chunk_step", REPO / "examples" / "chunk_step.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    got = module.main()
    assert got["tokens"] == (602 + 1 + 5 + 1) + (602 + 1 + 3 + 1)
    # 37 full pages shared, the 38th each row's own, the 39th (tokens from 608 on) the first row's.
    assert got["pages after the fork"] == 37 + 4 and got["pages at the end"] == 37 + 2 + 1


def test_refusals():
    from kernel_lab import cuda_ops

    i = lambda *s, dtype=torch.int32: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    k = torch.zeros(10, 16, 2, 8, device="cuda")
    for caches in ([], [k, k[:9]], [k.cpu()], [k[:, ::2]], [k[:1].expand(10, -1, -1, -1)], [k[..., :7]], [torch.zeros((), device="cuda")]):
        with pytest.raises((RuntimeError, NotImplementedError)):
            cuda_ops.paged_copy_pages(caches, i(2), i(2))
    for src, dst in ((i(2), i(3)), (i(2, dtype=torch.int64), i(2, dtype=torch.int64)), (i(4)[::2], i(2)), (i(2).cpu(), i(2).cpu())):
        with pytest.raises((RuntimeError, NotImplementedError)):
            cuda_ops.paged_copy_pages([k], src, dst)
    for table, lens, new, parents in ((i(3, 4), i(3), i(2), None), (i(3, 4), i(4), i(3), None), (i(3, 4), i(3), i(3), i(2)), (i(3, 8)[:, ::2], i(3), i(3), None),
                                      (i(3, 4, dtype=torch.int64), i(3), i(3), None), (i(3, 4), i(3), i(3, dtype=torch.int64), None)):
        with pytest.raises(RuntimeError):
            cuda_ops.paged_reserve([k], table, lens, new, parents)
    for size in (0, -1):
        with pytest.raises(RuntimeError):
            cuda_ops.paged_reserve([k], i(3, 4), i(3), i(3), page_size=size)
        with pytest.raises(RuntimeError):
            cuda_ops.paged_compact([k], i(3, 4), i(3), page_size=size)
    with pytest.raises(RuntimeError):
        cuda_ops.paged_compact([k], i(3, 4), i(4))
    with pytest.raises(RuntimeError):  # the new table in the old one's place
        table = i(3, 4)
        torch.ops.kernel_lab.paged_compact(table, i(()), [k], table, i(3), 16)


def test_nothing_to_do():
    from kernel_lab import cuda_ops

    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    k = torch.ones(10, 16, 2, 8, device="cuda")
    table, lens, served = cuda_ops.paged_reserve([k], i(0, 4), i(0), i(0))
    assert table.shape == (0, 4) and lens.numel() == served.numel() == 0
    table, lens, served = cuda_ops.paged_reserve([k], i(2, 0), i(2), i(2))
    assert table.shape == (2, 0) and served.all()
    table, lens, served = cuda_ops.paged_reserve([k], i(0, 4), i(0), i(3) + 1, i(3))  # parents of no sequences
    assert (table == 0).all() and served.all()
    table, used = cuda_ops.paged_compact([k], i(0, 4), i(0))
    assert table.shape == (0, 4) and int(used) == 0
    cuda_ops.decode_status(clear=True)
