"""The block-scaled 8-bit cache: append, decode attention over all or selected pages, page selection.

Codes, scales, bounds and selections are defined element by element and compared exactly. Attention is
compared with 64 bits over the dequantised cache. Tolerance of an output element: the probabilities are
rounded to fp16 after a product with the value scale's ratio (2^-11 of sum p|v|, and 2^-14 more for the
roundings of ex2, that product and the sums), a score is off by some units of 2^-24 of the largest
(at most 2^-21 of it), products below fp16's normal range lose at most 2^-25 of the largest value for
each token (the sum of the probabilities is at least 1 in these units), the result is rounded to its type
(half an ulp).
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import block8

pytestmark = pytest.mark.gpu

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_ULP = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
CODE_DTYPE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


class Pool:
    """A pool whose pages hold arbitrary old codes, scales and bounds, on the GPU and in NumPy."""

    def __init__(self, kind, lens, heads, dim, page, layout="nhd", seed=0, spare=3):
        self.kind, self.page = kind, page
        rng = np.random.RandomState(seed)
        need = [-(-n // page) for n in lens]
        total = sum(need) + spare
        order = rng.permutation(total)
        self.table = np.zeros((len(lens), max(1, max(need, default=1))), np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at : at + n]
            at += n
        self.lens = np.array(lens, np.int32)
        self.k_scale, self.v_scale = (np.exp(rng.randn(total, heads)).astype(np.float32) / 64 for _ in range(2))
        x = rng.randn(2, total, page, heads, dim).astype(np.float32) * (100 if kind == "e4m3" else 40)
        self.k, self.v = block8.encode(x, kind)
        vals = np.nan_to_num(block8.decode_codes(self.k, kind), nan=0.0) / block8.BOUND_UNIT[kind]
        self.bounds = np.stack([np.floor(vals.min(axis=1)), np.ceil(vals.max(axis=1))], axis=2).astype(np.int8)
        self.layout = layout

    def code_tensor(self, codes):
        t = torch.from_numpy(codes.view(np.uint8).copy()).cuda()
        if self.layout == "hnd":  # pages hold one head after another
            t = t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
        elif self.layout == "padded":  # rows of a wider buffer
            wide = torch.zeros(*t.shape[:3], t.shape[3] + 16, dtype=torch.uint8, device="cuda")
            wide[..., : t.shape[3]] = t
            t = wide[..., : t.shape[3]]
        return t.view(CODE_DTYPE[self.kind])

    def gpu(self):
        return {
            "k_cache": self.code_tensor(self.k), "v_cache": self.code_tensor(self.v),
            "k_scale": torch.from_numpy(self.k_scale.copy()).cuda(), "v_scale": torch.from_numpy(self.v_scale.copy()).cuda(),
        }

    def tables(self):
        return torch.from_numpy(self.table.copy()).cuda(), torch.from_numpy(self.lens.copy()).cuda()


def as_numpy(t):
    return t.contiguous().view(torch.uint8).cpu().numpy() if t.dtype == torch.float8_e4m3fn else t.cpu().numpy()


def same_codes(got, want, kind):
    np.testing.assert_array_equal(block8.decode_codes(as_numpy(got), kind), block8.decode_codes(want, kind))


# ---------------------------------------------------------------- append


def run_append(pool, new, start, dtype, bounds=True, indptr=None, k_new=None, v_new=None, seed=0):
    """Appends on both sides and compares everything; returns the GPU's tensors."""
    from kernel_lab import cuda_ops

    heads, dim = pool.k.shape[2:]
    tokens = int(sum(new))
    g = torch.Generator().manual_seed(seed)
    if k_new is None:
        k_new, v_new = (torch.randn(tokens, heads, dim, generator=g).mul(s).to(dtype) for s in (3.0, 0.05))
    state = pool.gpu()
    kb = torch.from_numpy(pool.bounds.copy()).cuda() if bounds else None
    table, _ = pool.tables()
    positions = torch.tensor(start, dtype=torch.int32)
    ptr = None if indptr is None else torch.tensor(indptr, dtype=torch.int32).cuda()
    cuda_ops.decode_status(clear=True)
    cuda_ops.paged_kv_append_block8(
        *state.values(), k_new.cuda(), v_new.cuda(), table, positions.cuda(), indptr=ptr, k_bounds=kb
    )
    status = cuda_ops.decode_status(clear=True)
    block8.append(pool.kind, pool.k, pool.v, pool.k_scale, pool.v_scale, pool.bounds if bounds else None,
                  *(t.float().cpu().numpy().reshape(tokens, heads, dim) for t in (k_new, v_new)), pool.table, start, indptr)
    np.testing.assert_array_equal(state["k_scale"].cpu().numpy(), pool.k_scale)
    np.testing.assert_array_equal(state["v_scale"].cpu().numpy(), pool.v_scale)
    same_codes(state["k_cache"], pool.k, pool.kind)
    same_codes(state["v_cache"], pool.v, pool.kind)
    if bounds:
        np.testing.assert_array_equal(kb.cpu().numpy(), pool.bounds)
    return state, status


SHAPES = [(8, 128, 16), (1, 64, 8), (3, 96, 16), (2, 256, 32), (5, 40, 4), (2, 7, 1), (1, 1024, 3), (4, 128, 64), (2, 64, 100)]


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,dim,page", SHAPES)
@pytest.mark.parametrize("layout", ["nhd", "hnd"])
def test_append_one_token_each(kind, dtype, heads, dim, page, layout):
    start = [0, 1, page - 1, page, 2 * page + page // 2, 77]
    pool = Pool(kind, [s + 1 for s in start], heads, dim, page, layout, seed=1)
    assert run_append(pool, [1] * len(start), start, DTYPE[dtype])[1] == 0


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("heads,dim,page", SHAPES)
@pytest.mark.parametrize("bounds", [True, False])
def test_append_ragged_prompts(kind, heads, dim, page, bounds):
    """Sequences with no, one and many new tokens, starting in, at the end and at the start of a page."""
    new = [0, 1, 2 * page, 3 * page + 1, 0, page, 50, 0]
    start = [5, page - 1, 0, page // 2, 0, page, 3, 9]
    indptr = np.cumsum([0, *new]).tolist()
    pool = Pool(kind, [s + n for s, n in zip(start, new)], heads, dim, page, "nhd", seed=2)
    assert run_append(pool, new, start, torch.bfloat16, bounds, indptr)[1] == 0


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_append_padded_strides_and_odd_alignment(kind):
    """Rows of a wider buffer (16-byte strides) and new rows that start on odd elements."""
    pool = Pool(kind, [40, 17], 4, 64, 16, "padded", seed=3)
    run_append(pool, [20, 3], [20, 14], torch.float16, True, [0, 20, 23])
    pool = Pool(kind, [40, 17], 4, 64, 16, seed=3)
    wide = torch.randn(23, 2 * 256 + 3, device="cuda")
    run_append(pool, [20, 3], [20, 14], torch.float32, True, [0, 20, 23], wide[:, 1:257], wide[:, 258:514])


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_append_token_by_token_matches_the_oracle_and_covers_every_growth(kind):
    """Growing magnitudes: each token raises the scale, so the kept codes are rounded again each time."""
    pool = Pool(kind, [33], 2, 128, 16, seed=4)
    for t in range(33):
        rows = torch.randn(1, 2, 128, generator=torch.Generator().manual_seed(t)) * 1.7**t
        state, _ = run_append(pool, [1], [t], torch.float32, True, None, rows, -rows)
        pool.k, pool.v = as_numpy(state["k_cache"]).copy(), as_numpy(state["v_cache"]).copy()
    # Each code stays within its format's half step (int8: and half a step for each later growth).
    page = pool.table[0, 0]
    last = block8.decode_codes(pool.k[page, 15], kind) * pool.k_scale[page][:, None]
    want = torch.randn(1, 2, 128, generator=torch.Generator().manual_seed(15))[0].numpy() * np.float32(1.7**15)
    step = np.abs(want) * 2.0**-4 + pool.k_scale[page][:, None] * (2.0**-10 if kind == "e4m3" else 0.5)
    assert (np.abs(last - want) <= step * 1.001).all()


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_append_special_values(kind):
    """Zeros (scale 0), NaN, infinities, denormals and the largest floats, in fresh and in used pages."""
    big = 3.0e38
    rows = torch.zeros(6, 1, 64)
    rows[1, 0, :4] = torch.tensor([float("nan"), 1.0, -2.0, 0.5])
    rows[2, 0, :4] = torch.tensor([float("inf"), -float("inf"), 1.0, 448.0])
    rows[3, 0, :3] = torch.tensor([1e-42, -1e-40, 3e-45])
    rows[4, 0, :2] = torch.tensor([big, -big])
    rows[5, 0] = float("nan")
    for start in ([0] * 6, [3] * 6):
        pool = Pool(kind, [s + 1 for s in start], 1, 64, 16, seed=5)
        run_append(pool, [1] * 6, start, torch.float32, True, None, rows, rows.flip(0))


def test_append_powers_of_two_cover_the_largest_element():
    """e4m3: amax at, just below and just above 448 * 2^k."""
    vals = [448.0, np.nextafter(np.float32(448), np.float32(0)), np.nextafter(np.float32(448), np.float32(1e9)), 1.75, 1.0, 7.0, 3.5]
    pool = Pool("e4m3", [1] * len(vals), 1, 16, 8, seed=6)
    rows = torch.tensor(np.array(vals, np.float32))[:, None, None].repeat(1, 1, 16)
    run_append(pool, [1] * len(vals), [0] * len(vals), torch.float32, True, None, rows, -rows)
    scale = pool.k_scale[pool.table[:, 0], 0]
    assert scale.tolist() == [1.0, 1.0, 2.0, 2.0**-8, 2.0**-8, 2.0**-6, 2.0**-7]


def test_append_skips_and_flags():
    """Negative positions, positions past the table, page ids outside the pool: skipped, the last two flagged."""
    pool = Pool("int8", [16, 16, 16, 16], 2, 64, 16, seed=7)
    pool.table[2, 0], pool.table[3, 0] = 10_000, -5
    assert run_append(pool, [1] * 4, [-1, 16, 3, 4], torch.float16)[1] == 1
    pool = Pool("int8", [40, 40], 2, 64, 16, seed=7)
    assert run_append(pool, [20, 20], [-1, 36], torch.float16, True, [0, 20, 40])[1] == 1


def test_append_ignores_rows_of_no_sequence():
    """indptr that starts late or ends early leaves the other rows alone."""
    from kernel_lab import cuda_ops

    pool = Pool("e4m3", [16, 16], 2, 64, 16, seed=8)
    state, (table, _) = pool.gpu(), pool.tables()
    k_new = torch.randn(12, 2, 64)
    indptr = [2, 5, 9]
    cuda_ops.paged_kv_append_block8(*state.values(), k_new.cuda(), k_new.cuda(), table,
                                    torch.tensor([0, 3], dtype=torch.int32).cuda(),
                                    indptr=torch.tensor(indptr, dtype=torch.int32).cuda())
    x = k_new.numpy()
    block8.append("e4m3", pool.k, pool.v, pool.k_scale, pool.v_scale, None, x, x, pool.table, [0, 3], indptr)
    same_codes(state["k_cache"], pool.k, "e4m3")
    np.testing.assert_array_equal(state["v_scale"].cpu().numpy(), pool.v_scale)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("heads,dim,page,new", [(64, 64, 32, [2200, 900, 800]), (64, 8, 4, [500, 300, 250])])
def test_append_large_calls(kind, heads, dim, page, new):
    """Enough pages that a team takes several in turn: NaN and infinities inside, a page id outside the pool
    between good ones, sequences that begin within a page, rows of no sequence after the last."""
    start = [page // 2 + 1, 0, 3 * page]
    pool = Pool(kind, [s + n for s, n in zip(start, new)], heads, dim, page, seed=32)
    pool.table[0, 5] = 1 << 30
    g = torch.Generator().manual_seed(33)
    rows = [torch.randn(sum(new) + 9, heads, dim, generator=g).to(torch.bfloat16) for _ in range(2)]
    for at, value in [(3 * page, float("nan")), (7 * page + 1, float("inf")), (8 * page + 2, -float("inf"))]:
        rows[0][at, ::2, 1], rows[1][at, 1::3, 2] = value, value
    new_rows = [*new, 9]
    assert run_append(pool, new_rows, start, torch.bfloat16, True, np.cumsum([0, *new]).tolist(), *rows)[1] == 1


# ---------------------------------------------------------------- decode


def check_decode(pool, q, got, scale, selected=None):
    want, weight, score, value = block8.decode(pool.kind, q.float().cpu().numpy(), pool.k, pool.v, pool.k_scale,
                                               pool.v_scale, pool.table, pool.lens, scale, selected)
    bound = (2.0**-11 + 2.0**-14 + 2.0**-21 * score) * weight + HALF_ULP[q.dtype] * np.abs(want) + 2.0**-25 * value
    err = np.abs(got.float().cpu().numpy() - want)
    assert np.isfinite(err).all()
    assert (err <= bound).all(), float((err / np.maximum(bound, 1e-37)).max())


def make_q(pool, hq, dtype, seed=0):
    dim = pool.k.shape[3]
    return torch.randn(len(pool.lens), hq, dim, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


# (query heads, KV heads, head_dim, page): MHA, GQA of odd groups, MQA up to 128, padded widths.
HEADS = [(32, 8, 128, 16), (8, 8, 64, 16), (7, 1, 128, 8), (28, 4, 128, 32), (32, 1, 128, 16), (40, 2, 64, 64),
         (5, 5, 96, 16), (10, 2, 80, 48), (12, 3, 256, 16), (48, 1, 256, 8), (128, 1, 64, 16), (16, 1, 16, 16),
         (70, 1, 128, 16), (64, 1, 256, 16), (6, 2, 224, 8)]


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("hq,hkv,dim,page", HEADS)
def test_decode_heads(kind, hq, hkv, dim, page):
    from kernel_lab import cuda_ops

    pool = Pool(kind, [1, page - 1, page, page + 1, 0, 100, 333], hkv, dim, page, seed=10)
    for dtype in (torch.float16, torch.bfloat16):
        q = make_q(pool, hq, dtype)
        table, lens = pool.tables()
        cuda_ops.decode_status(clear=True)
        got = cuda_ops.paged_decode_attention_block8(q, **pool.gpu(), block_table=table, seq_lens=lens)
        assert cuda_ops.decode_status(clear=True) == 0
        assert (got[4] == 0).all()
        check_decode(pool, q, got, dim**-0.5)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("hq,hkv,dim,page", [(17, 1, 64, 16), (32, 1, 48, 8), (66, 2, 64, 16), (64, 1, 32, 32),
                                             (65, 1, 64, 8), (96, 3, 16, 16), (256, 2, 64, 16)])
def test_decode_many_heads_of_small_dim(kind, hq, hkv, dim, page):
    """Groups of 17 to 128 query heads for head_dim up to 64, short rows beside rows of several CTAs."""
    from kernel_lab import cuda_ops

    pool = Pool(kind, [3, 2100, 0, page, 5000, 1, 130], hkv, dim, page, "padded", seed=31)
    q = make_q(pool, hq, torch.bfloat16)
    table, lens = pool.tables()
    got = cuda_ops.paged_decode_attention_block8(q, **pool.gpu(), block_table=table, seq_lens=lens)
    assert (got[2] == 0).all()
    check_decode(pool, q, got, dim**-0.5)


@pytest.mark.parametrize("layout", ["nhd", "hnd", "padded"])
@pytest.mark.parametrize("lens", [[1], [15], [4096], [1025, 3, 700], [64] * 40, [2000, 1] * 8])
def test_decode_lengths_and_layouts(layout, lens):
    """From one token to rows that many CTAs share, ragged batches, each layout of the pool."""
    from kernel_lab import cuda_ops

    pool = Pool("e4m3", lens, 8, 128, 16, layout, seed=11)
    q = make_q(pool, 32, torch.bfloat16)
    table, seq = pool.tables()
    got = cuda_ops.paged_decode_attention_block8(q, **pool.gpu(), block_table=table, seq_lens=seq)
    check_decode(pool, q, got, 128**-0.5)
    again = cuda_ops.paged_decode_attention_block8(q, **pool.gpu(), block_table=table, seq_lens=seq)
    assert torch.equal(got, again)  # no order of arrival in the result


@pytest.mark.parametrize("hq,hkv,dim", [(32, 8, 128), (16, 1, 128), (32, 1, 64), (4, 2, 256), (24, 3, 128)])
def test_decode_more_sequences_than_cta_pieces(hq, hkv, dim):
    """Many short and some long rows: pieces that hold several rows, ends that cut rows."""
    from kernel_lab import cuda_ops

    rng = np.random.RandomState(0)
    pool = Pool("int8", [int(n) for n in rng.randint(0, 400, 150)] + [3000, 0, 2999], hkv, dim, 16, "hnd", seed=12)
    q = make_q(pool, hq, torch.float16)
    table, seq = pool.tables()
    got = cuda_ops.paged_decode_attention_block8(q, **pool.gpu(), block_table=table, seq_lens=seq, scale=0.3)
    check_decode(pool, q, got, 0.3)


def test_decode_never_reads_past_the_length():
    """NaN codes and scales in the tail of a page, in unused pages and in columns past the length."""
    from kernel_lab import cuda_ops

    pool = Pool("e4m3", [5, 33, 48], 2, 128, 16, seed=13)
    q = make_q(pool, 8, torch.float16)
    clean = block8.decode("e4m3", q.float().cpu().numpy(), pool.k, pool.v, pool.k_scale, pool.v_scale, pool.table,
                          pool.lens, 128**-0.5)[0]
    used = {int(p) for b, n in enumerate(pool.lens) for p in pool.table[b, : -(-n // 16)]}
    for p in set(range(len(pool.k))) - used:
        pool.k[p], pool.v[p], pool.k_scale[p], pool.v_scale[p] = 0x7F, 0xFF, np.nan, np.nan
    for b, n in enumerate(pool.lens):
        if n % 16:
            pool.k[pool.table[b, n // 16], n % 16 :] = 0x7F
            pool.v[pool.table[b, n // 16], n % 16 :] = 0x7F
    wide = np.full((3, 9), 1 << 30, np.int32)
    wide[:, : pool.table.shape[1]] = np.where(np.arange(pool.table.shape[1]) < -(-pool.lens[:, None] // 16), pool.table, 1 << 30)
    cuda_ops.decode_status(clear=True)
    got = cuda_ops.paged_decode_attention_block8(q, **pool.gpu(), block_table=torch.from_numpy(wide).cuda(),
                                                 seq_lens=torch.from_numpy(pool.lens).cuda())
    assert cuda_ops.decode_status(clear=True) == 0
    np.testing.assert_allclose(got.float().cpu().numpy(), clean, atol=2e-3 * np.abs(clean).max())


def test_decode_scales_of_any_size():
    """Pages whose scales differ by many powers of two, zero scales among them; large and tiny q."""
    from kernel_lab import cuda_ops

    pool = Pool("int8", [200, 64], 2, 64, 16, seed=14)
    pool.v_scale *= np.float32(2.0) ** np.random.RandomState(1).randint(-30, 30, pool.v_scale.shape).astype(np.float32)
    pool.v_scale[pool.table[0, 2]] = 0
    pool.k_scale[pool.table[0, 3]] = 0
    pool.v_scale[pool.table[1]] = 0  # a whole sequence of zero values
    table, seq = pool.tables()
    for size in (1.0, 2.0**-40, 2.0**60):
        q = (make_q(pool, 4, torch.bfloat16).float() * size).to(torch.bfloat16)
        got = cuda_ops.paged_decode_attention_block8(q, **pool.gpu(), block_table=table, seq_lens=seq, scale=0.05 / size)
        check_decode(pool, q, got, 0.05 / size)
        assert (got[1] == 0).all()


def test_decode_peaked_and_rising_scores():
    """Scores that rise along the sequence raise the running maximum again and again."""
    from kernel_lab import cuda_ops

    pool = Pool("int8", [640], 1, 64, 16, seed=15)
    ramp = np.linspace(-120, 120, 640).astype(np.int8)
    for t in range(640):
        pool.k[pool.table[0, t // 16], t % 16, 0, 0] = ramp[t]
    pool.k_scale[:] = 1.0
    q = torch.zeros(1, 8, 64, dtype=torch.float16, device="cuda")
    q[0, :, 0] = torch.tensor([1.0, -1.0, 0.1, 0.5, 2.0, -0.25, 0.0, 4.0])
    table, seq = pool.tables()
    got = cuda_ops.paged_decode_attention_block8(q, **pool.gpu(), block_table=table, seq_lens=seq, scale=1.0)
    check_decode(pool, q, got, 1.0)


def test_decode_bad_pages_and_long_lengths_are_flagged():
    from kernel_lab import cuda_ops

    pool = Pool("e4m3", [64, 64, 64], 2, 128, 16, seed=16)
    pool.table[1, 1], pool.table[1, 2] = -1, 10_000
    pool.lens[2] = 1000  # beyond the table's width
    q = make_q(pool, 8, torch.float16)
    table, seq = pool.tables()
    cuda_ops.decode_status(clear=True)
    got = cuda_ops.paged_decode_attention_block8(q, **pool.gpu(), block_table=table, seq_lens=seq)
    assert cuda_ops.decode_status(clear=True) == 3
    check_decode(pool, q, got, 128**-0.5)


# ---------------------------------------------------------------- selection and sparse decode


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("hq,hkv,dim,page", [(32, 8, 128, 16), (32, 1, 64, 16), (7, 1, 128, 8), (10, 2, 96, 32), (4, 2, 256, 16), (3, 3, 16, 5)])
def test_select_matches_the_oracle(kind, hq, hkv, dim, page):
    from kernel_lab import cuda_ops

    pool = Pool(kind, [0, 1, page, 7 * page, 7 * page + 1, 40 * page - 1, 130 * page + 3], hkv, dim, page, seed=20)
    table, seq = pool.tables()
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        q = make_q(pool, hq, dtype)
        for want, sink, recent in ((7, 1, 1), (8, 0, 0), (40, 3, 5), (4, 2, 2), (200, 1, 1)):
            state = pool.gpu()
            got = cuda_ops.paged_block_select(q, state["k_cache"], state["k_scale"], torch.from_numpy(pool.bounds).cuda(),
                                              table, seq, want, sink, recent)
            oracle = block8.select(kind, q.float().cpu().numpy(), pool.k_scale, pool.bounds, pool.table, pool.lens, page,
                                   want, sink, recent)
            np.testing.assert_array_equal(got.cpu().numpy(), oracle)


@pytest.mark.parametrize("pages", [300, 9000, 20000])
def test_select_long_rows_and_ties(pages):
    """Rows over several blocks and beyond the keys a block holds; bounds of few values, so that most
    scores tie, then all of them."""
    from kernel_lab import cuda_ops

    rng = np.random.RandomState(3)
    bounds = rng.randint(-2, 3, (pages, 1, 2, 16)).astype(np.int8)
    bounds.sort(axis=2)
    k_cache = torch.zeros(pages, 1, 1, 16, dtype=torch.int8, device="cuda")
    q = torch.from_numpy(rng.randint(-2, 3, (2, 2, 16)).astype(np.float32)).cuda()
    table = np.stack([rng.permutation(pages), rng.permutation(pages)]).astype(np.int32)
    lens = np.array([pages, pages - 7], np.int32)
    for scale in (rng.choice([0.5, 1.0], (pages, 1)).astype(np.float32), np.zeros((pages, 1), np.float32)):
        got = cuda_ops.paged_block_select(q, k_cache, torch.from_numpy(scale).cuda(), torch.from_numpy(bounds).cuda(),
                                          torch.from_numpy(table).cuda(), torch.from_numpy(lens).cuda(), 100)
        want = block8.select("int8", q.cpu().numpy(), scale, bounds, table, lens, 1, 100)
        np.testing.assert_array_equal(got.cpu().numpy(), want)


def test_select_special_queries_and_bad_pages():
    from kernel_lab import cuda_ops

    pool = Pool("int8", [640, 640, 640], 1, 64, 16, seed=21)
    pool.table[2, 5], pool.table[2, 6] = -1, 9999
    q = make_q(pool, 4, torch.float32)
    q[0, 0, 3], q[0, 1, 4], q[0, 2] = float("nan"), float("inf"), 0.0
    q[1] = 0.0
    state, (table, seq) = pool.gpu(), pool.tables()
    cuda_ops.decode_status(clear=True)
    got = cuda_ops.paged_block_select(q, state["k_cache"], state["k_scale"], torch.from_numpy(pool.bounds).cuda(), table, seq, 9)
    assert cuda_ops.decode_status(clear=True) == 1
    want = block8.select("int8", q.cpu().numpy(), pool.k_scale, pool.bounds, pool.table, pool.lens, 16, 9)
    np.testing.assert_array_equal(got.cpu().numpy(), want)
    assert got[1, 0].tolist() == [0, 1, 2, 3, 4, 5, 6, 7, 39]  # every score ties


def test_bounds_enclose_the_scores():
    """The score of a page is an upper bound of q . k over its keys, up to q's rounding to int8."""
    pool = Pool("e4m3", [160], 1, 64, 16, seed=22)
    q = np.random.RandomState(0).randn(64).astype(np.float32)
    sq = np.abs(q).max() / 127
    qi = np.clip(np.rint(q / sq), -127, 127)
    for p in pool.table[0]:
        keys = block8.decode_codes(pool.k[p, :, 0], "e4m3") * pool.k_scale[p, 0]
        lo, hi = pool.bounds[p, 0].astype(np.float64)
        bound = np.maximum(qi * lo, qi * hi).sum() * sq * 4 * pool.k_scale[p, 0]
        assert (keys @ (qi * sq)).max() <= bound * (1 + 1e-6) + 1e-6


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("hq,hkv,dim,page", [(32, 8, 128, 16), (7, 1, 128, 8), (32, 1, 64, 16), (10, 2, 96, 32), (4, 2, 256, 16)])
@pytest.mark.parametrize("layout", ["nhd", "hnd"])
def test_sparse_decode(kind, hq, hkv, dim, page, layout):
    """Selected pages only: lists from the selection, lists with holes, -1 everywhere (zeros)."""
    from kernel_lab import cuda_ops

    pool = Pool(kind, [0, 1, 3 * page + 1, 40 * page - 3, 130 * page + 1], hkv, dim, page, layout, seed=23)
    q = make_q(pool, hq, torch.bfloat16)
    table, seq = pool.tables()
    state = pool.gpu()
    bounds = torch.from_numpy(pool.bounds).cuda()
    for want in (2, 9, 33, 150):
        selected = cuda_ops.paged_block_select(q, state["k_cache"], state["k_scale"], bounds, table, seq, want)
        got = cuda_ops.paged_decode_attention_block8(q, **state, block_table=table, seq_lens=seq, selected=selected)
        check_decode(pool, q, got, dim**-0.5, selected.cpu().numpy())
    rng = np.random.RandomState(5)
    holes = np.stack([rng.permutation(160)[:40] for _ in range(5 * hkv)]).reshape(5, hkv, 40).astype(np.int32)
    holes[rng.rand(*holes.shape) < 0.3] = -1
    holes[3, 0] = -1
    got = cuda_ops.paged_decode_attention_block8(q, **state, block_table=table, seq_lens=seq, selected=torch.from_numpy(holes).cuda())
    check_decode(pool, q, got, dim**-0.5, holes)
    assert (got[3, : hq // hkv] == 0).all()


def test_selecting_every_page_is_the_whole_attention():
    from kernel_lab import cuda_ops

    pool = Pool("e4m3", [700, 1025], 8, 128, 16, seed=24)
    q = make_q(pool, 32, torch.float16)
    table, seq = pool.tables()
    state = pool.gpu()
    every = torch.arange(table.shape[1], dtype=torch.int32, device="cuda").expand(2, 8, -1).contiguous()
    whole = cuda_ops.paged_decode_attention_block8(q, **state, block_table=table, seq_lens=seq)
    got = cuda_ops.paged_decode_attention_block8(q, **state, block_table=table, seq_lens=seq, selected=every)
    torch.testing.assert_close(got, whole, atol=2e-3 * float(whole.abs().max()), rtol=2e-3)


# ---------------------------------------------------------------- boundary


def test_refusals():
    from kernel_lab import cuda_ops

    pool = Pool("e4m3", [64, 64], 2, 128, 16, seed=30)
    q = make_q(pool, 8, torch.float16)
    table, seq = pool.tables()
    state = pool.gpu()
    bounds = torch.from_numpy(pool.bounds).cuda()

    def decode(**change):
        args = {"q": q, **state, "block_table": table, "seq_lens": seq} | change
        return cuda_ops.paged_decode_attention_block8(**args)

    with pytest.raises(RuntimeError, match="fp16 or bf16"):
        decode(q=q.float())
    with pytest.raises(RuntimeError, match="float8_e4m3fn or int8"):
        decode(k_cache=state["k_cache"].half(), v_cache=state["v_cache"].half())
    with pytest.raises(RuntimeError, match="k_scale and v_scale"):
        decode(k_scale=state["k_scale"][:, :1].contiguous())
    with pytest.raises(RuntimeError, match="multiple of"):
        decode(q=q[:, :7].contiguous())
    with pytest.raises(RuntimeError, match="head_dim"):
        decode(q=q[..., :64].contiguous())
    with pytest.raises(RuntimeError, match="seq_lens"):
        decode(seq_lens=seq[:1])
    with pytest.raises(RuntimeError, match="selected"):
        decode(selected=torch.zeros(2, 1, 4, dtype=torch.int32, device="cuda"))
    for heads, dim, page in ((2, 72, 16), (2, 272, 16), (2, 64, 12)):  # unsupported widths and pages
        odd = Pool("int8", [8], heads, dim, page)
        t, n = odd.tables()
        with pytest.raises(RuntimeError, match="invalid argument"):
            cuda_ops.paged_decode_attention_block8(make_q(odd, 4, torch.float16), **odd.gpu(), block_table=t, seq_lens=n)
    with pytest.raises(RuntimeError, match="one new row per sequence"):
        cuda_ops.paged_kv_append_block8(*state.values(), q[:1, :2], q[:1, :2], table, seq)
    with pytest.raises(RuntimeError, match="indptr"):
        cuda_ops.paged_kv_append_block8(*state.values(), q[:, :2], q[:, :2], table, seq, indptr=seq)
    with pytest.raises(RuntimeError, match="contiguous rows"):
        cuda_ops.paged_kv_append_block8(*state.values(), q[:, :4:2], q[:, :4:2], table, seq)
    with pytest.raises(RuntimeError, match="k_bounds"):
        cuda_ops.paged_kv_append_block8(*state.values(), q[:, :2].contiguous(), q[:, :2].contiguous(), table, seq,
                                        k_bounds=bounds[:, :, :1].contiguous())
    with pytest.raises(RuntimeError, match="must fit"):
        cuda_ops.paged_block_select(q, state["k_cache"], state["k_scale"], bounds, table, seq, 1)
    with pytest.raises(RuntimeError, match="k_bounds"):
        cuda_ops.paged_block_select(q, state["k_cache"], state["k_scale"], bounds.float(), table, seq, 4)


def test_empty_batches():
    from kernel_lab import cuda_ops

    pool = Pool("int8", [16], 2, 64, 16)
    state = pool.gpu()
    none = torch.empty(0, 4, 64, dtype=torch.float16, device="cuda")
    table, seq = torch.empty(0, 3, dtype=torch.int32, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda")
    assert cuda_ops.paged_decode_attention_block8(none, **state, block_table=table, seq_lens=seq).shape == (0, 4, 64)
    cuda_ops.paged_kv_append_block8(*state.values(), none[:, :2], none[:, :2], table, seq)
    bounds = torch.from_numpy(pool.bounds).cuda()
    assert cuda_ops.paged_block_select(none, state["k_cache"], state["k_scale"], bounds, table, seq, 4).shape == (0, 2, 4)


def test_a_step_on_another_stream_and_in_a_graph():
    """norm -> append -> select -> decode, captured on a side stream; the replay reads what it appends."""
    from kernel_lab import cuda_ops

    pool = Pool("e4m3", [200, 70], 4, 128, 16, "hnd", seed=31)
    q = make_q(pool, 16, torch.bfloat16)
    k_new, v_new = make_q(pool, 4, torch.bfloat16, 1), make_q(pool, 4, torch.bfloat16, 2)
    table, seq = pool.tables()

    def step(state, bounds):
        cuda_ops.paged_kv_append_block8(*state.values(), k_new, v_new, table, seq - 1, k_bounds=bounds)
        chosen = cuda_ops.paged_block_select(q, state["k_cache"], state["k_scale"], bounds, table, seq, 6)
        return chosen, cuda_ops.paged_decode_attention_block8(q, **state, block_table=table, seq_lens=seq, selected=chosen)

    plain, bounds = pool.gpu(), torch.from_numpy(pool.bounds).cuda()
    want = step(plain, bounds)
    graph = torch.cuda.CUDAGraph()
    state, kb = pool.gpu(), torch.from_numpy(pool.bounds).cuda()
    warm = pool.gpu()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(warm, kb.clone())  # the stream's scratch
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            got = step(state, kb)
    side.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(kb, bounds)


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
def test_the_example_step_is_close_to_a_bf16_cache(dtype):
    """e4m3 keeps 3 fraction bits (an element is off by at most 2^-4 of itself, about 2^-5.2 in the mean
    square), int8 with a page's scale 1 / 254 of the page's largest: keys' and values' errors together
    stay below 0.08 and 0.04 of the output; every page selected reads as the whole."""
    import sys

    from tests.conftest import REPO

    sys.path.insert(0, str(REPO / "examples"))
    import block8_step

    whole, sparse = block8_step.run(hq=16, hkv=4, prompt=300, steps=3, pages=4, dtype=dtype)
    assert whole < (0.08 if dtype is torch.float8_e4m3fn else 0.04)
    assert whole < sparse < 2.0
    whole, sparse = block8_step.run(hq=16, hkv=4, prompt=100, steps=2, pages=64, dtype=dtype)
    assert abs(whole - sparse) < 0.01
