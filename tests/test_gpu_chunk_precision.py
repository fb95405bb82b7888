"""What fp16 callers get: a probability is off by at most 2^-11 of itself."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import chunk
from tests.test_gpu_chunk import Problem

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
