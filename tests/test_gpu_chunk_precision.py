"""What fp16 callers get: a probability (over 8-bit caches one times its value scale) is off by at most 2^-11 of itself."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import chunk
from tests.test_gpu_chunk import EDGES, Problem

pytestmark = pytest.mark.gpu

E4M3, INT8 = torch.float8_e4m3fn, torch.int8
KINDS = [("e4m3", E4M3), ("block8", E4M3), ("block8", INT8)]


class Fp16(Problem):
    """The same tolerance over every cache: 11 significant bits of a probability."""

    def want(self, causal=True, scale=None):
        scale = self.dim**-0.5 if scale is None else scale
        f64 = lambda x: x.float().double().numpy()  # noqa: E731
        scales = {} if self.kind == "same" else {"k_scale": f64(self.scale["k"]), "v_scale": f64(self.scale["v"])}
        return chunk.attention(f64(self.q), f64(self.cache["k"]), f64(self.cache["v"]), self.table, self.lens, self.indptr, scale,
                               causal, bits=11, p_bits=11, **scales)


@pytest.mark.parametrize("kind,codes", KINDS)
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 8), (128, 64), (256, 16), (96, 32)])
@pytest.mark.parametrize("causal", [True, False])
def test_8_bit_caches(kind, codes, dim, page, causal):
    p = Fp16(EDGES, 8, 2, dim, page, torch.float16, kind, codes, seed=60)
    p.check(p.run(causal=causal), causal)


@pytest.mark.parametrize("kind,codes", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_contexts_that_many_ctas_share(kind, codes, dim):
    p = Fp16([(1, 9000), (4, 5000), (70, 800), (2, 3)], 8, 2, dim, 16, torch.float16, kind, codes, seed=61)
    p.check(p.run())


@pytest.mark.parametrize("kind", ["e4m3", "block8"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_what_is_masked_does_not_count(kind, dim):
    """The last token of a chunk holds NaN: the tokens before it do not see it, it does."""
    for n, length in [(9, 9), (40, 200), (140, 140), (70, 385)]:
        p = Fp16([(n, length), (n, length)], 8, 2, dim, 16, torch.float16, kind, E4M3, seed=65)
        want, tol = p.want()
        last = length - 1
        for name in "kv":
            p.cache[name].view(torch.int8)[p.table[0, last // 16], last % 16] = 0x7F
        got = p.run().float().double().cpu().numpy()
        seen = np.arange(len(got)) == n - 1
        assert np.isnan(got[seen]).all()
        assert (np.abs(got - want) <= tol)[~seen].all()


@pytest.mark.parametrize("kind", ["e4m3", "block8"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_pages_outside_the_pool(kind, dim):
    from kernel_lab import cuda_ops

    p = Fp16([(5, 100), (3, 300), (2, 20), (40, 700)], 4, 2, dim, 16, torch.float16, kind, E4M3, seed=66)
    cuda_ops.decode_status(clear=True)
    p.table[0, 2], p.table[1, 0], p.table[1, 9], p.table[2, :], p.table[3, 30] = -1, 10**6, 2**31 - 1, -5, -7
    got = p.run()
    assert cuda_ops.decode_status(clear=True) == 1
    p.check(got)


@pytest.mark.parametrize("codes", [E4M3, INT8])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_negative_and_unlike_scales(codes, dim):
    """Value scales of either sign that differ by up to 2^40, and are zero for some pages."""
    p = Fp16(EDGES, 8, 2, dim, 16, torch.float16, "block8", codes, seed=62)
    gen = torch.Generator().manual_seed(3)
    shape = p.scale["v"].shape
    power = torch.exp2(-torch.randint(0, 41, shape, generator=gen).float())
    sign = torch.randint(0, 2, shape, generator=gen) * 2 - 1
    p.scale["v"] = p.scale["v"] * power * sign
    p.scale["v"][::7] = 0.0
    p.check(p.run())


@pytest.mark.parametrize("codes", [E4M3, INT8])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("power", [12, 26, 60, 120])
@pytest.mark.parametrize("place", [0, 5, 39])
def test_a_page_of_large_values_and_no_weight_takes_no_bits(codes, dim, power, place):
    """One page's values are 2^power times the others', and its scores so low that its weights are below e^-300 of theirs."""
    p = Fp16([(5, 640), (200, 640)], 4, 2, dim, 16, torch.float16, "block8", codes, seed=63)
    p.q = (p.q.float() * 0.1 + 1.0).half()
    for b in range(2):
        page = p.table[b, place]
        low = torch.full((16, 2, dim), -100.0)
        p.cache["k"][page] = low.to(codes)
        p.scale["k"][page] = 1.0
        p.scale["v"][page] *= 2.0**power
    got = p.run().float().double().cpu().numpy()
    for b in range(2):
        p.table[b, place] = -1  # the oracle leaves it out: what is summed, and so the tolerance, is the others'
    want, tol = p.want()
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("kind,codes", [("same", None), *KINDS])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 130])
def test_a_long_tail_of_small_probabilities(kind, codes, dim, new):
    """One key has all but 2^-8 of the weight and values of zero; the others' weights are near 2^-22 of its own: the output is theirs.
    In fp16's subnormals beside a largest probability of 1 they would be off by up to an eighth of themselves."""
    length = 16000
    p = Fp16([(new, length)], 2, 1, dim, 16, torch.float16, kind, codes or E4M3, seed=64)
    p.q[:] = 1.0
    unit = 1.0 if kind == "same" else 0.25
    keys, values = torch.zeros(length, dim), torch.full((length, dim), 16.0)
    # Scores, by the scale of the call below: 0 for the first key, -22 ln 2 and a little around it for the others.
    keys[1:, 0] = -88.0
    keys[1:, 1] = torch.arange(length - 1) % 7
    values[0] = 0.0
    scale = 22 * np.log(2.0) / 88.0 / unit
    tok = np.arange(length)
    at = p.table[0, tok // 16], tok % 16
    for name, rows in (("k", keys), ("v", values)):
        p.cache[name][at] = rows[:, None].to(p.cache[name].dtype)
        if kind != "same":
            p.scale[name][:] = unit
    want, tol = p.want(scale=scale)
    assert (tol[:, :, 0] / want[:, :, 0]).max() < 2.0**-8
    many = 160  # so many sequences of the same pages that none is shared out over CTAs: pieces have maxima of their own
    p.q, p.table, p.lens = p.q.repeat(many, 1, 1), p.table.repeat(many, 0), [length] * many
    p.indptr = (np.arange(many + 1) * new).astype(np.int32)
    got = p.run(scale=scale).float().double().cpu().numpy().reshape(many, new, 2, dim)
    assert (np.abs(got - want) <= tol).all(), np.abs(got - want).max() / want.max()
