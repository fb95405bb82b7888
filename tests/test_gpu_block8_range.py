"""Block-scaled decode where the numbers spread widely: value scales and elements of q of unlike size.

Tolerance of an output element, from the definition's roundings: a token's weight p * v_scale is rounded to fp16
(2^-11 of itself, or 2^-25 of the head's largest weight where that is more), 2^-14 for ex2, the products and the
sums, 2^-21 of the largest |score| for the scores, and the result is rounded to its type. No term grows with a
value scale that carries no weight.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import block8
from tests.test_gpu_block8 import HALF_ULP, Pool

pytestmark = pytest.mark.gpu


def check(pool, q, got, scale, selected=None):
    batch, hq, dim = q.shape
    heads, page = pool.k.shape[2], pool.page
    group = hq // heads
    q64, got = q.double().cpu().numpy(), got.double().cpu().numpy()
    for b, n in enumerate(pool.lens):
        for h in range(heads):
            cols = np.arange(-(-n // page))
            if selected is not None:
                cols = selected[b, h][(selected[b, h] >= 0) & (selected[b, h] < len(cols))]
            at = pool.table[b, cols]
            there = (cols[:, None] * page + np.arange(page) < n).reshape(-1)
            k, v = (block8.decode_codes(c[at, :, h], pool.kind).astype(np.float64).reshape(-1, dim)[there] for c in (pool.k, pool.v))
            ks, vs = (np.repeat(t[at, h].astype(np.float64), page)[there] for t in (pool.k_scale, pool.v_scale))
            rows = slice(h * group, (h + 1) * group)
            s = q64[b, rows] @ (k * ks[:, None]).T * scale
            p = np.exp(s - s.max(axis=1, keepdims=True))
            p /= p.sum(axis=1, keepdims=True)
            want, size = (p * vs) @ v, (p * vs) @ np.abs(v)
            bound = (2.0**-11 + 2.0**-14 + 2.0**-21 * np.abs(s).max(axis=1, keepdims=True)) * size
            bound += 2.0**-25 * (p * vs).max(axis=1, keepdims=True) * np.abs(v).sum(axis=0) + HALF_ULP[q.dtype] * np.abs(want)
            err = np.abs(got[b, rows] - want)
            assert np.isfinite(err).all()
            assert (err <= bound).all(), (b, h, float((err / np.maximum(bound, 1e-300)).max()))


def spread_pool(kind, lens, heads, dim, page, far, at, seed):
    """One page of each sequence, the `at`-th part of the way along, with a value scale 2^far above the rest and keys
    that channel 0 tells from the others'."""
    pool = Pool(kind, lens, heads, dim, page, seed=seed)
    pool.k_scale[:] = 1.0
    pool.v_scale[:] = np.float32(2.0) ** np.random.RandomState(seed).randint(-6, -3, pool.v_scale.shape)
    small = np.random.RandomState(seed + 1).randint(-3, 4, pool.k.shape).astype(np.float32)
    small[..., 0] = 0
    for b, n in enumerate(lens):
        page_id = pool.table[b, int(at * (-(-n // page) - 1))]
        small[page_id, :, :, 0] = -60
        pool.v_scale[page_id] *= np.float32(2.0) ** far
    pool.k = block8.encode(small, kind)
    return pool


# Groups of 1, 8 and more, one and two tiles a step, query fragments in registers and in shared memory.
@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("hq,hkv,dim,page", [(4, 4, 128, 16), (32, 4, 128, 16), (32, 1, 128, 8), (40, 2, 64, 32), (8, 2, 256, 16), (14, 1, 64, 16)])
@pytest.mark.parametrize("far", [16, 26, 60])
@pytest.mark.parametrize("at", [0.0, 0.6, 1.0])
def test_a_large_value_scale_without_weight_takes_nothing(kind, hq, hkv, dim, page, far, at):
    """Even heads give the page of large values a weight of 2^-60 of the others', odd heads nearly all of it: a
    warp's heads want unlike references, and neither order of the pages matters."""
    from kernel_lab import cuda_ops

    pool = spread_pool(kind, [640, 33, 5000], hkv, dim, page, far, at, seed=40)
    rng = np.random.RandomState(41)
    q = rng.randn(3, hq, dim) / 8
    q[:, :, 0] = np.where(np.arange(hq) % 2, -1.0, 1.0)
    scale = float(np.log(2.0))
    table, seq = pool.tables()
    q = torch.from_numpy(q).to(torch.bfloat16).cuda()  # whose range holds the outputs
    got = cuda_ops.paged_decode_attention_block8(q, **pool.gpu(), block_table=table, seq_lens=seq, scale=scale)
    check(pool, q, got, scale)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_scales_that_rise_fall_and_vanish(kind):
    """Scales that double or halve page by page over 2^80, random ones over 2^60, and zeros among them."""
    from kernel_lab import cuda_ops

    rng = np.random.RandomState(42)
    pool = Pool(kind, [1280, 1280, 3000, 48], 2, 128, 16, seed=43)
    pool.k_scale /= 4
    steps = np.float32(2.0) ** np.linspace(-40, 40, 80).astype(int)
    pool.v_scale[pool.table[0]] = np.resize(steps, pool.table.shape[1])[:, None]
    pool.v_scale[pool.table[1]] = np.resize(steps[::-1], pool.table.shape[1])[:, None]
    pool.v_scale[pool.table[2]] = np.float32(2.0) ** rng.randint(-30, 30, (pool.table.shape[1], 2))
    pool.v_scale[pool.table[2, ::7]] = 0
    pool.v_scale[pool.table[3, :2]] = 0
    table, seq = pool.tables()
    for size in (0.02, 0.5):
        q = (size * torch.randn(4, 16, 128, generator=torch.Generator().manual_seed(1))).to(torch.bfloat16).cuda()
        got = cuda_ops.paged_decode_attention_block8(q, **pool.gpu(), block_table=table, seq_lens=seq, scale=0.05)
        check(pool, q, got, 0.05)


def test_selected_pages_of_unlike_scales():
    from kernel_lab import cuda_ops

    pool = spread_pool("e4m3", [640, 2000], 2, 128, 16, 26, 0.0, seed=44)
    q = torch.randn(2, 8, 128, generator=torch.Generator().manual_seed(2)) / 8
    q[:, :, 0] = 1.0
    q = q.to(torch.bfloat16).cuda()
    rng = np.random.RandomState(45)
    chosen = np.stack([np.concatenate([[0], 1 + rng.permutation(39)[:9]]) for _ in range(4)]).reshape(2, 2, 10).astype(np.int32)
    table, seq = pool.tables()
    got = cuda_ops.paged_decode_attention_block8(q, **pool.gpu(), block_table=table, seq_lens=seq, scale=float(np.log(2.0)),
                                                 selected=torch.from_numpy(chosen).cuda())
    check(pool, q, got, float(np.log(2.0)), chosen)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("hq,hkv,dim", [(8, 1, 64), (32, 1, 64), (16, 1, 128), (4, 1, 256)])
@pytest.mark.parametrize(
    "dtype,largest,small", [(torch.float16, 8.0, 1e-4), (torch.float16, 3e4, 2.0**-22), (torch.bfloat16, 1.0, 2.0**-20), (torch.bfloat16, 2.0**100, 2.0**70), (torch.bfloat16, 2.0**-110, 2.0**-130)]
)
def test_small_elements_of_q_beside_a_large_one(kind, hq, hkv, dim, dtype, largest, small):
    """The large element meets keys of zero, so the scores are the small ones': none of their bits may be lost."""
    from kernel_lab import cuda_ops

    pool = Pool(kind, [200, 31], hkv, dim, 16, seed=46)
    pool.k_scale[:] = 1.0
    x = block8.decode_codes(pool.k, kind).copy()
    x[..., 3] = 0
    pool.k = block8.encode(x, kind)
    q = small * (1 + np.random.RandomState(47).rand(2, hq, dim))
    q[..., 3] = largest
    q = torch.from_numpy(q).to(dtype).cuda()
    scale = 0.02 / small
    table, seq = pool.tables()
    got = cuda_ops.paged_decode_attention_block8(q, **pool.gpu(), block_table=table, seq_lens=seq, scale=scale)
    check(pool, q, got, scale)


@pytest.mark.parametrize("page", [16, 144, 4096])
def test_lengths_near_the_end_of_32_bits(page):
    """A table of nearly 2^31 tokens over three pages of the pool: the pages in use are counted without a sum that
    passes 31 bits, and the last one ends inside a tile."""
    from kernel_lab import cuda_ops

    pool = Pool("int8", [3 * page], 1, 16, page, seed=48)
    width = (2**31 - 1 - 64) // page
    table = torch.zeros(1, width, dtype=torch.int32, device="cuda")
    order = torch.from_numpy(pool.table[0].copy()).cuda()
    columns = torch.tensor([0, width // 2, width - 1], dtype=torch.int32, device="cuda")
    table[0, columns.long()] = order
    length = width * page - 5
    q = torch.randn(1, 4, 16, generator=torch.Generator().manual_seed(3)).to(torch.float16).cuda()
    got = cuda_ops.paged_decode_attention_block8(q, **pool.gpu(), block_table=table, scale=0.02, selected=columns.view(1, 1, 3),
                                                 seq_lens=torch.tensor([length], dtype=torch.int32, device="cuda"))
    pool.lens = np.array([3 * page - 5])
    check(pool, q, got, 0.02)
