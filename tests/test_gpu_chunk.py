"""Chunks of new tokens over a paged cache: append and attention, against the 64-bit oracle. Tolerances come from the
oracle, by counting roundings."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import chunk

pytestmark = pytest.mark.gpu

BITS = {torch.float32: 24, torch.float16: 11, torch.bfloat16: 8}


class Problem:
    """A pool with NaN wherever nothing is to be read, and a batch of (new tokens, length)."""

    def __init__(self, shapes, hq, hkv, dim, page, dtype, kind="same", codes=torch.float8_e4m3fn, seed=0, lead=0, trail=0,
                 heads_first=False, spare=3, extra_width=0):
        gen = torch.Generator().manual_seed(seed)
        rand = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
        self.kind, self.dtype, self.dim, self.page = kind, dtype, dim, page
        self.new, self.lens = [n for n, _ in shapes], [n for _, n in shapes]
        needed = [-(-n // page) for n in self.lens]
        pages = sum(needed) + spare
        order = torch.randperm(pages, generator=gen).tolist()
        self.table = np.zeros((len(shapes), max(1, max(needed)) + extra_width), np.int32)
        self.table[:] = order[-1]  # padding names a poisoned page
        held = torch.zeros(pages, page, dtype=torch.bool)
        at = 0
        for b, n in enumerate(needed):
            self.table[b, :n] = order[at : at + n]
            at += n
            tok = np.arange(self.lens[b])
            held[self.table[b, tok // page], tok % page] = True
        self.cache, self.scale = {}, {}
        for name in "kv":
            x = rand(pages, page, hkv, dim)
            if kind == "same":
                x = x.to(dtype)
                x[~held] = float("nan")
            else:
                x = (x * 40).round().clamp(-127, 127).to(torch.int8) if codes is torch.int8 else (x * 60).clamp(-448, 448).to(codes)
                raw = x.view(torch.int8)
                raw[~held] = 127 if codes is torch.int8 else 0x7F  # 0x7f is e4m3's NaN
                shape = (pages, hkv) if kind == "block8" else (hkv,)
                self.scale[name] = torch.exp(0.5 * rand(*shape)) / 50
            self.cache[name] = x
        self.heads_first = heads_first
        self.indptr = (lead + np.cumsum([0, *self.new])).astype(np.int32)
        rows = int(self.indptr[-1]) + trail
        self.q = rand(rows, hq, dim).to(dtype)

    def device_cache(self, name):
        x = self.cache[name].cuda()
        if self.heads_first:
            return x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
        return x

    def run(self, q=None, causal=True, scale=None, out=None):
        from kernel_lab import cuda_ops

        q = self.q.cuda() if q is None else q
        table, lens, ptr = (torch.from_numpy(np.asarray(x, np.int32)).cuda() for x in (self.table, self.lens, self.indptr))
        args = [self.device_cache("k"), self.device_cache("v")]
        if self.kind != "same":
            args += [self.scale["k"].cuda(), self.scale["v"].cuda()]
        suffix = {"same": "", "e4m3": "_fp8", "block8": "_block8"}[self.kind]
        if out is not None:
            getattr(torch.ops.kernel_lab, "paged_chunk_attention" + suffix)(out, q, *args, table, lens, ptr,
                                                                         self.dim**-0.5 if scale is None else scale, causal)
            return out
        return getattr(cuda_ops, "paged_chunk_attention" + suffix)(q, *args, table, lens, ptr, scale=scale, causal=causal)

    def want(self, causal=True, scale=None):
        scale = self.dim**-0.5 if scale is None else scale
        f64 = lambda x: x.float().double().numpy()  # noqa: E731
        scales = {} if self.kind == "same" else {"k_scale": f64(self.scale["k"]), "v_scale": f64(self.scale["v"])}
        p_bits = BITS[self.dtype] if self.kind == "same" else 8
        return chunk.attention(f64(self.q), f64(self.cache["k"]), f64(self.cache["v"]), self.table, self.lens, self.indptr, scale,
                               causal, bits=BITS[self.dtype], p_bits=p_bits, **scales)

    def rows(self):
        return slice(int(self.indptr[0]), int(self.indptr[-1]))

    def check(self, got, causal=True, scale=None):
        want, tol = self.want(causal, scale)
        got = got.float().double().cpu().numpy()[self.rows()]
        want, tol = want[self.rows()], tol[self.rows()]
        assert np.isfinite(got).all()
        worst = np.unravel_index(np.argmax(np.abs(got - want) - tol), got.shape)
        assert (np.abs(got - want) <= tol).all(), f"{got[worst]} for {want[worst]}, tolerance {tol[worst]}, at {worst}"


# New tokens and lengths: none, one, the edges of pages and tiles, chunks longer than what the sequence holds.
EDGES = [(0, 40), (1, 1), (1, 128), (3, 129), (17, 127), (33, 300), (0, 0), (5, 0), (9, 4), (130, 130), (64, 257), (2, 16)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hq,hkv,dim", [(8, 2, 128), (8, 8, 64), (7, 1, 128), (10, 2, 96), (4, 2, 256), (6, 3, 80), (3, 1, 40), (5, 5, 17)])
@pytest.mark.parametrize("causal", [True, False])
def test_edges(dtype, hq, hkv, dim, causal):
    p = Problem(EDGES, hq, hkv, dim, 16, dtype, seed=1)
    p.check(p.run(causal=causal), causal)


@pytest.mark.parametrize("page", [1, 8, 16, 20, 64, 128, 256])
@pytest.mark.parametrize("dim", [64, 128])
def test_page_sizes(page, dim):
    p = Problem(EDGES, 8, 2, dim, page, torch.bfloat16, seed=2)
    p.check(p.run())


@pytest.mark.parametrize("hq,hkv", [(32, 1), (64, 1), (100, 1), (128, 1), (200, 1), (28, 4), (5, 1), (24, 2)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_groups(hq, hkv, dtype):
    p = Problem([(1, 300), (40, 40), (7, 513), (3, 3)], hq, hkv, 128, 16, dtype, seed=3)
    p.check(p.run())


@pytest.mark.parametrize("kind,codes", [("e4m3", torch.float8_e4m3fn), ("block8", torch.float8_e4m3fn), ("block8", torch.int8)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,dim,page,heads_first", [(8, 2, 128, 16, False), (8, 2, 128, 8, True), (4, 4, 64, 64, True),
                                                       (10, 2, 96, 32, False), (4, 2, 256, 16, True), (7, 1, 48, 24, False)])
@pytest.mark.parametrize("causal", [True, False])
def test_8bit_caches(kind, codes, dtype, hq, hkv, dim, page, heads_first, causal):
    p = Problem(EDGES, hq, hkv, dim, page, dtype, kind, codes, seed=4, heads_first=heads_first)
    p.check(p.run(causal=causal), causal)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_few_rows_over_long_contexts(dtype, dim):
    """The keys of a sequence are split over many CTAs and joined."""
    p = Problem([(1, 9000), (4, 5000), (2, 3)], 8, 2, dim, 16, dtype, seed=5)
    p.check(p.run())


@pytest.mark.parametrize("kind", ["same", "block8"])
def test_many_sequences(kind):
    rng = np.random.RandomState(6)
    shapes = [(int(n), int(n + c)) for n, c in zip(rng.randint(0, 4, 1500), rng.randint(0, 60, 1500))]
    p = Problem(shapes, 4, 2, 64, 16, torch.bfloat16, kind, seed=6)
    p.check(p.run())


def test_long_chunk():
    p = Problem([(1100, 1500), (513, 513)], 4, 1, 128, 16, torch.bfloat16, seed=7)
    p.check(p.run())


@pytest.mark.parametrize("scale", [0.5, 3.0, -0.7, 0.0])
def test_scales(scale):
    p = Problem(EDGES, 8, 2, 128, 16, torch.float16, seed=8)
    p.check(p.run(scale=scale), scale=scale)


@pytest.mark.parametrize("dim", [64, 128, 256, 40])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("kind,codes", [("same", None), ("block8", torch.float8_e4m3fn)])
def test_what_is_masked_does_not_count(dim, value, kind, codes):
    """The last token of a chunk holds no numbers: the tokens before it do not see it, it does."""
    if kind != "same" and (not np.isnan(value) or dim == 40):
        pytest.skip("e4m3 has NaN only")
    for n, length in [(9, 9), (40, 200), (140, 140), (70, 385)]:
        p = Problem([(n, length), (n, length)], 8, 2, dim, 16, torch.bfloat16, kind, codes or torch.float8_e4m3fn, seed=9)
        want, tol = p.want()
        last = length - 1
        for name in "kv":
            at = p.table[0, last // 16], last % 16
            if kind == "same":
                p.cache[name][at] = value
            else:
                p.cache[name].view(torch.int8)[at] = 0x7F
        got = p.run().float().double().cpu().numpy()
        seen = np.arange(len(got)) == n - 1
        assert np.isnan(got[seen]).all()
        assert np.isfinite(got[~seen]).all()
        assert (np.abs(got - want) <= tol)[~seen].all()


@pytest.mark.parametrize("dim", [64, 128])
def test_an_infinite_value_is_seen_by_those_after_it(dim):
    """An infinity in one element of V: infinite there from its token on, and nowhere else."""
    p = Problem([(150, 150)], 8, 2, dim, 16, torch.bfloat16, seed=10)
    want, tol = p.want()
    p.cache["v"][p.table[0, 100 // 16], 100 % 16, 1, 7] = float("inf")
    got = p.run().float().double().cpu().numpy()
    hit = np.zeros(got.shape, bool)
    hit[100:, 4:8, 7] = True
    assert np.isposinf(got[hit]).all()
    assert (np.abs(got - want) <= tol)[~hit].all()


@pytest.mark.parametrize("kind", ["same", "block8"])
@pytest.mark.parametrize("dim", [128, 40, 256])
def test_pages_outside_the_pool(kind, dim):
    from kernel_lab import cuda_ops

    dim = 48 if kind == "block8" and dim == 40 else dim
    p = Problem([(5, 100), (3, 300), (2, 20)], 4, 2, dim, 16, torch.bfloat16, kind, seed=11)
    cuda_ops.decode_status(clear=True)
    p.table[0, 2], p.table[1, 0], p.table[1, 9], p.table[2, :] = -1, 10**6, 2**31 - 1, -5
    got = p.run()
    assert cuda_ops.decode_status(clear=True) == 1
    p.check(got)


@pytest.mark.parametrize("dim", [128, 40])
def test_rows_of_no_sequence_stay(dim):
    p = Problem(EDGES, 8, 2, dim, 16, torch.bfloat16, seed=12, lead=5, trail=40)
    out = torch.full_like(p.q.cuda(), 7.0)
    p.run(out=out)
    assert (out[:5] == 7).all() and (out[int(p.indptr[-1]) :] == 7).all()
    p.check(out)


def test_lengths_past_the_table_are_clamped():
    from kernel_lab import cuda_ops

    p = Problem([(4, 64), (2, 30)], 4, 2, 128, 16, torch.bfloat16, seed=13)
    cuda_ops.decode_status(clear=True)
    want, tol = p.want()
    p.lens[0] = 1000
    got = p.run().float().double().cpu().numpy()
    assert cuda_ops.decode_status(clear=True) == 2
    assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("stride", ["fused", "odd"])
@pytest.mark.parametrize("dim", [128, 64, 80])
def test_strided_queries(stride, dim):
    p = Problem(EDGES, 8, 2, dim, 16, torch.bfloat16, seed=14)
    width = 8 * dim
    big = torch.zeros(p.q.shape[0], width + (2 * 2 * dim if stride == "fused" else 3), dtype=p.dtype, device="cuda")
    big[:, 3 if stride == "odd" else 0 :][:, :width] = p.q.cuda().view(-1, width)
    q = big[:, 3 if stride == "odd" else 0 :][:, :width].view(-1, 8, dim)
    p.check(p.run(q))
    flipped = p.q.cuda().transpose(0, 1).contiguous().transpose(0, 1)
    p.check(p.run(flipped))


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("page", [8, 16, 64])
@pytest.mark.parametrize("layout", ["heads", "interleaved", "padded", "fused"])
@pytest.mark.parametrize("hkv", [1, 2])
def test_caches_of_any_layout(dim, page, layout, hkv):
    """Pages head by head, keys beside values in one pool, pages and tokens with gaps, keys and values of a token side by side."""
    from kernel_lab import cuda_ops

    p = Problem(EDGES, 4 * hkv, hkv, dim, page, torch.bfloat16, seed=18)
    k, v = p.cache["k"].cuda(), p.cache["v"].cuda()
    if layout == "heads":
        k, v = (x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for x in (k, v))
    elif layout == "interleaved":
        both = torch.stack([k, v], dim=1)
        k, v = both[:, 0], both[:, 1]
    elif layout == "fused":
        both = torch.cat([k, v], dim=2)
        k, v = both[:, :, :hkv], both[:, :, hkv:]
    else:
        k, v = (torch.nn.functional.pad(x, (0, 8, 0, 1, 0, 3), value=float("nan"))[:, :page, :hkv, :dim] for x in (k, v))
    ints = [torch.from_numpy(np.asarray(x, np.int32)).cuda() for x in (p.table, p.lens, p.indptr)]
    p.check(cuda_ops.paged_chunk_attention(p.q.cuda(), k, v, *ints))


def test_a_pool_of_one_page():
    p = Problem([(5, 16)], 8, 2, 128, 16, torch.float16, seed=19, spare=0)
    p.check(p.run())


@pytest.mark.parametrize("kind", ["same", "block8"])
def test_captured_calls_replay_beside_one_another(kind):
    """Two graphs and eager calls, whose split blocks all meet in scratch, on three streams."""
    problems = [Problem([(1, 5000), (3, 900), (40, 64)], 8, 2, 128, 16, torch.bfloat16, kind, seed=s) for s in (20, 21)]
    from kernel_lab import cuda_ops

    name = "paged_chunk_attention" + {"same": "", "block8": "_block8"}[kind]
    calls = []
    for p in problems:
        args = [p.q.cuda(), p.device_cache("k"), p.device_cache("v")]
        args += [p.scale[n].cuda() for n in "kv"] if kind == "block8" else []
        args += [torch.from_numpy(np.asarray(x, np.int32)).cuda() for x in (p.table, p.lens, p.indptr)]
        calls.append(lambda args=args: getattr(cuda_ops, name)(*args))
    eager = [c() for c in calls]
    graphs = []
    for c in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = c()
        graphs.append((g, out))
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    extra = []
    for _ in range(20):
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            extra.append(calls[0]())
    torch.cuda.synchronize()
    for (_, out), want, p in zip(graphs, eager, problems):
        assert torch.equal(out, want)
        p.check(out)
    assert all(torch.equal(e, eager[0]) for e in extra)


def test_caches_at_odd_addresses():
    """Caches whose rows start on no 16 bytes."""
    from kernel_lab import cuda_ops

    p = Problem(EDGES, 8, 2, 128, 16, torch.float16, seed=15)
    views = []
    for name in "kv":
        c = p.cache[name]
        flat = torch.zeros(c.numel() + 1, dtype=c.dtype, device="cuda")
        flat[1:] = c.cuda().view(-1)
        views.append(flat[1:].view(c.shape))
    ints = [torch.from_numpy(np.asarray(x, np.int32)).cuda() for x in (p.table, p.lens, p.indptr)]
    p.check(cuda_ops.paged_chunk_attention(p.q.cuda(), *views, *ints))


def test_runs_are_bit_equal_and_other_streams_work():
    p = Problem([(1, 6000), (60, 700), (300, 300)], 8, 2, 128, 16, torch.bfloat16, seed=16)
    first = p.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = p.run()
    torch.cuda.synchronize()
    assert torch.equal(first, other) and torch.equal(first, p.run())
    p.check(first)


def test_decode_agrees_with_chunks_of_one_token():
    from kernel_lab import cuda_ops

    p = Problem([(1, n) for n in (1, 77, 128, 1000)], 32, 8, 128, 16, torch.bfloat16, seed=17)
    k, v = (torch.nan_to_num(p.device_cache(n)) for n in "kv")
    table, lens = torch.from_numpy(p.table).cuda(), torch.tensor(p.lens, dtype=torch.int32, device="cuda")
    a = cuda_ops.paged_decode_attention(p.q.cuda(), k, v, table, lens).double().cpu().numpy()
    want, tol = p.want()
    assert (np.abs(a - want) <= tol).all()
    p.check(p.run())


# ------------------------------------------------------------------ append


def append_reference(cache, rows, table, positions, indptr, page):
    for b, start in enumerate(positions):
        for i in range(int(indptr[b]), int(indptr[b + 1])):
            pos = int(start) + i - int(indptr[b])
            if start < 0 or pos // page >= table.shape[1] or not 0 <= table[b, pos // page] < cache.shape[0]:
                continue
            cache[table[b, pos // page], pos % page] = rows[i].view(cache.shape[2:])


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16", "e4m3"])
@pytest.mark.parametrize("hkv,dim,page", [(8, 128, 16), (2, 64, 8), (3, 80, 7), (1, 34, 16)])
@pytest.mark.parametrize("layout", ["contiguous", "fused", "odd"])
def test_append_chunks(kind, hkv, dim, page, layout):
    from kernel_lab import cuda_ops

    dtype = {"f32": torch.float32, "f16": torch.float16}.get(kind, torch.bfloat16)
    gen = torch.Generator().manual_seed(20)
    new, start = [0, 1, 5, 40, 0, 0, 33, 7, 3, 9], [3, 0, 14, 2, 0, 5, 100, -1, 6, 150]
    pages, width = 120, 23
    table = torch.randperm(pages, generator=gen)[: 10 * 10].view(10, 10).repeat(1, 3)[:, :width].to(torch.int32).numpy().copy()
    table[8, 0] = pages if kind != "e4m3" else -3
    indptr = (2 + np.cumsum([0, *new])).astype(np.int32)
    rows, cols = int(indptr[-1]) + 4, hkv * dim
    big = torch.randn(rows, 2 * cols + (1 if layout == "odd" else 0), generator=gen).to(dtype)
    big[3, 1], big[4, 2] = float("nan"), float("inf")
    gpu = big.cuda()
    lo = 1 if layout == "odd" else 0
    cut = lambda t, i: t[:, lo + i * cols : lo + (i + 1) * cols]  # noqa: E731
    k_new, v_new = cut(gpu, 0), cut(gpu, 1)
    if layout == "contiguous":
        k_new, v_new = k_new.contiguous(), v_new.contiguous().view(rows, hkv, dim)
        k_new = k_new.view(rows, hkv, dim)
    cache_type = torch.uint8 if kind == "e4m3" else dtype
    caches = [torch.randint(0, 255, (pages, page, hkv, dim), generator=gen).to(cache_type) for _ in range(2)]
    want = [c.clone() for c in caches]
    scales = [torch.rand(hkv, generator=gen) * 0.02 + 0.001 for _ in range(2)] if kind == "e4m3" else [None, None]
    as_type = (lambda c: c.view(torch.float8_e4m3fn)) if kind == "e4m3" else (lambda c: c)
    for i in range(2):
        ref = as_type(want[i])
        if kind == "e4m3":
            for b, s in enumerate(start):
                for r in range(int(indptr[b]), int(indptr[b + 1])):
                    pos = s + r - int(indptr[b])
                    if s < 0 or pos // page >= width or not 0 <= table[b, pos // page] < pages:
                        continue
                    x = cut(big, i)[r].view(hkv, dim).float() / scales[i][:, None]
                    x = torch.where(torch.isnan(x), x, x.clamp(-448, 448)).to(torch.float8_e4m3fn)
                    want[i][table[b, pos // page], pos % page] = x.view(torch.uint8)
        else:
            append_reference(ref, cut(big, i), table, start, indptr, page)
    got = [c.cuda() for c in caches]
    ints = [torch.from_numpy(np.asarray(x, np.int32)).cuda() for x in (table, start)]
    ptr = torch.from_numpy(indptr).cuda()
    cuda_ops.decode_status(clear=True)
    if kind == "e4m3":
        cuda_ops.paged_kv_append_fp8(*map(as_type, got), k_new, v_new, *(s.cuda() for s in scales), *ints, indptr=ptr)
    else:
        cuda_ops.paged_kv_append(*got, k_new, v_new, *ints, indptr=ptr)
    assert cuda_ops.decode_status(clear=True) == 1
    for g, w in zip(got, want):
        g, w = g.cpu(), w
        if kind == "e4m3":
            bad = (g != w) & ~((g & 0x7F == 0x7F) & (w & 0x7F == 0x7F))
            assert not bad.any()
        else:
            assert torch.equal(g.nan_to_num(nan=-77.0), w.nan_to_num(nan=-77.0))


@pytest.mark.parametrize("batch", [1, 31, 32, 33, 1023, 1025, 3000])
def test_append_finds_the_sequences_of_many(batch):
    from kernel_lab import cuda_ops

    rng = np.random.RandomState(batch)
    new = rng.randint(0, 4, batch)
    new[rng.rand(batch) < 0.3] = 0
    new[0] = 2
    indptr = np.cumsum([0, *new]).astype(np.int32)
    rows = int(indptr[-1])
    k = torch.arange(rows * 8, dtype=torch.float32, device="cuda").view(rows, 8)
    cache = torch.zeros(batch, 4, 1, 8, device="cuda")
    other = torch.zeros_like(cache)
    table = torch.arange(batch, dtype=torch.int32, device="cuda")[:, None].contiguous()
    cuda_ops.paged_kv_append(cache, other, k, -k, table, torch.zeros(batch, dtype=torch.int32, device="cuda"),
                             indptr=torch.from_numpy(indptr).cuda())
    want = torch.zeros(batch, 4, 8)
    for b in range(batch):
        want[b, : new[b]] = k[indptr[b] : indptr[b + 1]].cpu()
    assert torch.equal(cache.cpu().view(batch, 4, 8), want) and torch.equal(other, -cache)


# ------------------------------------------------------------------ the step, as it is used


@pytest.mark.parametrize("kind", ["same", "e4m3", "block8"])
def test_a_prompt_in_chunks_is_the_prompt_at_once(kind):
    """Reserve, append and attend chunk by chunk, beside a fork; one call over the whole prompt gives the same rows."""
    from kernel_lab import cuda_ops, kv_cache

    hq, hkv, dim, page, n = 8, 2, 128, 16, 200
    gen = torch.Generator(device="cuda").manual_seed(30)
    q, k, v = (torch.randn(n, h, dim, generator=gen, device="cuda").to(torch.bfloat16) for h in (hq, hkv, hkv))
    int32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731

    def caches():
        if kind == "block8":
            pool = kv_cache.block8_pool(40, page, hkv, dim, torch.int8)
            return [pool.k_cache, pool.v_cache], [pool.k_scale, pool.v_scale]
        dtype = torch.bfloat16 if kind == "same" else torch.float8_e4m3fn
        made = [torch.zeros(40, page, hkv, dim, dtype=torch.bfloat16, device="cuda").to(dtype) for _ in range(2)]
        return made, [] if kind == "same" else [torch.full((hkv,), 0.01, device="cuda") for _ in range(2)]

    def step(pool, scales, table, lens, rows):
        ptr = int32([0, len(rows)])
        if kind == "block8":
            cuda_ops.paged_kv_append_block8(*pool, *scales, k[rows], v[rows], table, lens, indptr=ptr)
            return cuda_ops.paged_chunk_attention_block8(q[rows], *pool, *scales, table, lens + len(rows), ptr)
        if kind == "e4m3":
            cuda_ops.paged_kv_append_fp8(*pool, k[rows], v[rows], *scales, table, lens, indptr=ptr)
            return cuda_ops.paged_chunk_attention_fp8(q[rows], *pool, *scales, table, lens + len(rows), ptr)
        cuda_ops.paged_kv_append(*pool, k[rows], v[rows], table, lens, indptr=ptr)
        return cuda_ops.paged_chunk_attention(q[rows], *pool, table, lens + len(rows), ptr)

    outs = []
    # Whole pages at a time, so that the block-scaled form rounds each page once in both runs.
    for sizes in ([n], [64, 112, 24]):
        pool, scales = caches()
        moved = pool + (scales if kind == "block8" else [])
        table, lens, at, got = torch.zeros(1, 20, dtype=torch.int32, device="cuda"), int32([0]), 0, []
        for size in sizes:
            table, lens, served = cuda_ops.paged_reserve(moved, table, lens, int32([size]))
            assert served.all()
            got.append(step(pool, scales, table, lens, range(at, at + size)))
            lens, at = lens + size, at + size
        outs.append(torch.cat(got).double())
        # Two samples go on from the prompt: a copy of its last page for one of them.
        table, lens, served = cuda_ops.paged_reserve(moved, table, lens, int32([1, 1]), parents=int32([0, 0]))
        assert served.all() and (table[0, :12] == table[1, :12]).all() and table[0, 12] != table[1, 12]
        before = pool[0].view(torch.uint8)[table[0, 12].long()]
        assert torch.equal(before[: n % page], pool[0].view(torch.uint8)[table[1, 12].long()][: n % page])
        # Only the second goes on; compaction moves what is left to the front.
        table, used = cuda_ops.paged_compact(moved, table[1:].contiguous(), lens[1:].contiguous())
        assert int(used) == 13 and sorted(table[0, :13].tolist()) == list(range(13))
        again = step(pool, scales, table, lens[1:] - 24, range(n - 24, n)) if kind == "same" else None
        if again is not None:
            assert torch.equal(again.double(), outs[-1][-24:]) or (again.double() - outs[-1][-24:]).abs().max() < 2.0**-6
    # Probabilities and outputs are rounded in both: 4 roundings of bf16 of values below 4.
    assert (outs[0] - outs[1]).abs().max() <= 4 * 4 * 2.0**-8


# ------------------------------------------------------------------ refusals


def test_attention_refusals():
    from kernel_lab import cuda_ops

    i = lambda *s, dtype=torch.int32: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    f = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    good = {"q": f(9, 8, 64), "k_cache": f(10, 16, 2, 64), "v_cache": f(10, 16, 2, 64), "block_table": i(3, 4), "seq_lens": i(3), "indptr": i(4)}
    cuda_ops.paged_chunk_attention(**good)
    k = good["k_cache"]
    for name, bad in [
        ("q", f(9, 8, 32)), ("q", f(9, 7, 64)), ("q", f(9, 512)[:, None, :64].half()), ("q", good["q"].cpu()), ("v_cache", f(10, 16, 4, 64)[:, :, ::2]),
        ("v_cache", f(10, 16, 1, 64)), ("k_cache", f(10, 16, 2, 128)[..., ::2]), ("block_table", i(3, 4, dtype=torch.int64)), ("block_table", i(2, 4)),
        ("block_table", i(3, 8)[:, ::2]), ("seq_lens", i(3, dtype=torch.int64)), ("seq_lens", i(6)[::2]), ("indptr", i(3)), ("indptr", i(4).cpu()),
        ("indptr", i(4, dtype=torch.int64)), ("indptr", i(8)[::2]),
    ]:
        with pytest.raises(RuntimeError):
            cuda_ops.paged_chunk_attention(**(good | {name: bad}))
    with pytest.raises(RuntimeError):  # head_dim above 256
        cuda_ops.paged_chunk_attention(f(9, 8, 320), f(10, 16, 2, 320), f(10, 16, 2, 320), i(3, 4), i(3), i(4))
    k8, s, ps = k.to(torch.float8_e4m3fn), f(2, dtype=torch.float32), f(10, 2, dtype=torch.float32)
    tables = good["block_table"], good["seq_lens"], good["indptr"]
    cuda_ops.paged_chunk_attention_fp8(good["q"], k8, k8, s, s, *tables)
    cuda_ops.paged_chunk_attention_block8(good["q"], k8, k8, ps, ps, *tables)
    for args in [(good["q"].float(), k8, k8, s, s), (good["q"], k, k, s, s), (good["q"], k8, k8, ps, ps), (good["q"], k8, k8, s, s.half())]:
        with pytest.raises(RuntimeError):
            cuda_ops.paged_chunk_attention_fp8(*args, *tables)
    for args in [(good["q"], k, k, ps, ps), (good["q"], k8, k8, s, s), (good["q"].float(), k8, k8, ps, ps)]:
        with pytest.raises(RuntimeError):
            cuda_ops.paged_chunk_attention_block8(*args, *tables)


def test_nothing_to_do():
    """No tokens, no sequences, a table without columns."""
    from kernel_lab import cuda_ops

    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    f = lambda *s: torch.ones(*s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    k = f(10, 16, 2, 64)
    assert cuda_ops.paged_chunk_attention(f(0, 8, 64), k, k, i(3, 4), i(3), i(4)).shape == (0, 8, 64)
    assert cuda_ops.paged_chunk_attention(f(5, 8, 64), k, k, i(0, 4), i(0), i(1)).shape == (5, 8, 64)
    ptr = torch.tensor([0, 2, 5], dtype=torch.int32, device="cuda")
    assert (cuda_ops.paged_chunk_attention(f(5, 8, 64), k, k, i(2, 0), i(2), ptr) == 0).all()
    cuda_ops.paged_kv_append(k, k.clone(), f(0, 2, 64), f(0, 2, 64), i(3, 4), i(3), indptr=i(4))


def test_append_refusals():
    from kernel_lab import cuda_ops

    i = lambda *s, dtype=torch.int32: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    f = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    good = [f(10, 16, 2, 64), f(10, 16, 2, 64), f(9, 2, 64), f(9, 2, 64), i(3, 4), i(3)]
    for at, bad in [(0, f(10, 16, 4, 64)[:, :, ::2]), (1, f(10, 16, 1, 64)), (2, f(9, 2, 32)), (3, f(9, 4, 64)[:, ::2]), (2, f(9, 2, 64, dtype=torch.half)),
                    (4, i(2, 4)), (5, i(3, dtype=torch.int64))]:
        args = [*good]
        args[at] = bad
        with pytest.raises(RuntimeError):
            cuda_ops.paged_kv_append(*args, indptr=i(4))
    for ptr in (i(3), i(4).cpu(), i(4, dtype=torch.int64)):
        with pytest.raises(RuntimeError):
            cuda_ops.paged_kv_append(*good, indptr=ptr)
