"""The block-scaled cache with many sequences: the search among 128 and more, grids past 65535 windows, plans of
more sequences than a CTA has threads, prompts beside single tokens. Tolerances as in test_gpu_block8."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.test_gpu_block8 import Pool, check_decode, make_q, run_append

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("batch", [127, 128, 129, 300, 1025])
@pytest.mark.parametrize("most", [3, 40])
def test_append_ragged_rows_of_many_sequences(kind, batch, most):
    """Sequences of none to `most` tokens, runs of empty ones, some skipped, rows of no sequence at either end."""
    rng = np.random.RandomState(batch)
    new = rng.randint(0, most + 1, batch)
    new[rng.rand(batch) < 0.3] = 0
    new[5:40] = 0
    start = rng.randint(0, 40, batch)
    start[rng.rand(batch) < 0.1] = -1
    lens = [int(max(s, 0) + n) for s, n in zip(start, new)]
    pool = Pool(kind, lens, 1, 64, 16, seed=60)
    ptr = (3 + np.cumsum([0, *new])).tolist()
    rows = [torch.randn(ptr[-1] + 4, 1, 64, generator=torch.Generator().manual_seed(k)).to(torch.bfloat16) for k in (1, 2)]
    assert run_append(pool, [len(rows[0])], start.tolist(), torch.bfloat16, True, ptr, *rows)[1] == 0


@pytest.mark.parametrize("ragged", [False, True])
def test_append_past_the_second_dimension_of_a_grid(ragged):
    batch = 70_000
    pool = Pool("int8", [1] * batch, 1, 8, 1, seed=61, spare=0)
    indptr = list(range(batch + 1)) if ragged else None
    assert run_append(pool, [1] * batch, [0] * batch, torch.float16, True, indptr)[1] == 0


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("heads,dim,page", [(8, 128, 16), (2, 64, 64), (3, 96, 8)])
def test_append_a_prompt_beside_single_tokens(kind, heads, dim, page):
    """63 sequences of one token, in and at the ends of pages, around a chunk of 1000."""
    rng = np.random.RandomState(62)
    new = [1] * 31 + [1000] + [1] * 32
    start = rng.randint(0, 4 * page, 64)
    pool = Pool(kind, [int(s + n) for s, n in zip(start, new)], heads, dim, page, seed=63)
    assert run_append(pool, new, start.tolist(), torch.bfloat16, True, np.cumsum([0, *new]).tolist())[1] == 0


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("batch", [257, 700])
def test_decode_and_selection_of_many_sequences(kind, batch):
    """More sequences than a CTA's threads; empty ones, short ones, one that many CTAs share."""
    from kernel_lab import cuda_ops
    from oracle import block8

    rng = np.random.RandomState(64)
    lens = rng.randint(0, 90, batch)
    lens[rng.rand(batch) < 0.2] = 0
    lens[batch // 2] = 4000
    pool = Pool(kind, [int(n) for n in lens], 2, 64, 16, "hnd", seed=65)
    q = make_q(pool, 8, torch.float16)
    table, seq = pool.tables()
    state, bounds = pool.gpu(), torch.from_numpy(pool.bounds).cuda()
    check_decode(pool, q, cuda_ops.paged_decode_attention_block8(q, **state, block_table=table, seq_lens=seq), 64**-0.5)
    chosen = cuda_ops.paged_block_select(q, state["k_cache"], state["k_scale"], bounds, table, seq, 3)
    want = block8.select(kind, q.float().cpu().numpy(), pool.k_scale, pool.bounds, pool.table, pool.lens, 16, 3)
    np.testing.assert_array_equal(chosen.cpu().numpy(), want)
    got = cuda_ops.paged_decode_attention_block8(q, **state, block_table=table, seq_lens=seq, selected=chosen)
    check_decode(pool, q, got, 64**-0.5, want)
