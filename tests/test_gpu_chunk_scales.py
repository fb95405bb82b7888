"""Scales of 8-bit caches that are negative or no numbers, against the 64-bit oracle."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.test_gpu_chunk import EDGES, Problem

pytestmark = pytest.mark.gpu

E4M3, INT8 = torch.float8_e4m3fn, torch.int8
KINDS = [("e4m3", E4M3), ("block8", E4M3), ("block8", INT8)]


@pytest.mark.parametrize("kind,codes", KINDS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 8), (128, 64), (256, 16), (128, 20)])  # the last on the CUDA cores
@pytest.mark.parametrize("causal", [True, False])
def test_negative_scales(kind, codes, dtype, dim, page, causal):
    p = Problem(EDGES, 8, 2, dim, page, dtype, kind, codes, seed=50)
    for name, seed in (("k", 1), ("v", 2)):
        sign = torch.randint(0, 2, p.scale[name].shape, generator=torch.Generator().manual_seed(seed)) * 2 - 1
        p.scale[name] = p.scale[name] * sign
        assert (p.scale[name] < 0).any() or kind == "e4m3"
    p.scale["k"].view(-1)[0] = -0.01
    p.check(p.run(causal=causal), causal)


@pytest.mark.parametrize("kind,codes", KINDS[1:])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 16), (256, 16), (128, 8), (128, 20)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_page_whose_scale_is_no_number_counts_for_those_who_see_it(kind, codes, which, value, dim, page, dtype):
    """The last page of two sequences, which only the last tokens of their chunks see."""
    for n, length in [(page + 24, 8 * page), (140, 160 + page), (300, 300)]:
        p = Problem([(n, length), (n, length), (3, 5)], 8, 2, dim, page, dtype, kind, codes, seed=51)
        want, tol = p.want()
        first = (length - 1) // page * page  # the page's first token
        for b in range(2):
            p.scale[which][p.table[b, first // page]] = value
        p.scale[which][p.table[2, -1]] = value  # of no sequence
        got = p.run().float().double().cpu().numpy()
        position = np.concatenate([length - n + np.arange(n)] * 2 + [np.zeros(3)])
        before = position < first
        assert before.sum() > 20 and (~before).sum() > 0
        assert np.isfinite(got[before]).all() and (np.abs(got - want) <= tol)[before].all()
        if which == "v" or np.isnan(value):  # a score of minus infinity is one that does not count
            assert not np.isfinite(got[~before]).any()


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("dim", [64, 128, 256, 48])
def test_a_heads_scale_that_is_no_number_is_that_heads(which, dim):
    p = Problem(EDGES, 8, 2, dim, 16, torch.float16, "e4m3", seed=52)
    want, tol = p.want()
    p.scale[which][1] = float("nan")
    got = p.run().float().double().cpu().numpy()
    assert (np.abs(got - want) <= tol)[:, :4].all()
    row = 0
    for n, length in EDGES:
        for i in range(n):
            sees = length - n + i >= 0
            assert (np.isnan(got[row, 4:]).all() if sees else (got[row] == 0).all()), (row, n, length)
            row += 1
