"""RMSNorm and fused add + RMSNorm with an e4m3 output, against the definition in 64 bits.

Tolerances. The kernel forms y = (r * rstd) * w in fp32: the sum of squares has at most 64 roundings
in a row (a thread's columns, the warp's tree, the block's warps), halved by the square root, and the
remaining operations a handful: y and the scale are within 64 * 2^-24 < 4e-6 of the 64-bit values. A code
is then the nearest e4m3 value to y / scale up to that: |code - y / scale| <= half the spacing of e4m3
there (2^-4 relative, 2^-10 below 2^-6) + 1e-5 of it.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import block8
from tests.conftest import make_rms_inputs, to_f32_numpy

pytestmark = pytest.mark.gpu

SCALE_RTOL = 4e-6


def check(x, w, eps, group, codes, scales):
    """x: the rows that are normalised."""
    y, want = block8.norm(to_f32_numpy(x), to_f32_numpy(w), eps, group)
    np.testing.assert_allclose(scales.cpu().numpy(), want, rtol=SCALE_RTOL, atol=0)
    group = group or x.shape[-1]
    each = np.repeat(want, group, axis=-1)[..., : x.shape[-1]]
    target = np.divide(y, each, out=np.zeros_like(y), where=each > 0)
    got = codes.float().cpu().numpy()
    assert np.isfinite(got).all()
    bound = np.maximum(np.abs(target) * 2.0**-4, 2.0**-10) + 1e-5 * np.abs(target)
    assert (np.abs(got - target) <= bound).all(), float((np.abs(got - target) - bound).max())


# Widths of the repository's tests and beyond: register rows, short last groups, odd widths, one column,
# rows wider than the registers.
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize(
    "shape", [(1, 64), (3, 100), (8, 4096), (2, 5, 8192), (3, 16384), (2, 40000), (5, 72), (7, 1), (4, 1000), (300, 520)]
)
@pytest.mark.parametrize("group", [0, 64, 128])
def test_rows_against_64_bits(shape, dtype, group):
    from kernel_lab import cuda_ops

    x, r, w = (t.cuda() for t in make_rms_inputs(shape, dtype, seed=3))
    codes, scales, new = cuda_ops.fused_add_rms_norm_fp8(x, r, w, 1e-5, group_size=group)
    assert torch.equal(new, (x.float() + r.float()).to(dtype))  # bit-exact
    groups = -(-shape[-1] // group) if group else 1
    assert codes.shape == x.shape and codes.dtype == torch.float8_e4m3fn and scales.shape == (*shape[:-1], groups)
    check(new, w, 1e-5, group, codes, scales)
    codes, scales = cuda_ops.rms_norm_fp8(x, w, 1e-5, group_size=group)
    check(x, w, 1e-5, group, codes, scales)


@pytest.mark.parametrize("group", [1, 3, 8, 16, 32, 48, 256, 512, 5000, 1 << 20])
def test_group_sizes(group):
    from kernel_lab import cuda_ops

    for dtype in (torch.float32, torch.bfloat16):
        x, _, w = (t.cuda() for t in make_rms_inputs((6, 1032), dtype, seed=4))
        codes, scales = cuda_ops.rms_norm_fp8(x, w, 1e-6, group_size=group)
        assert scales.shape == (6, -(-1032 // group))
        check(x, w, 1e-6, group, codes, scales)


def test_in_place_residual_strided_and_misaligned_rows():
    from kernel_lab import cuda_ops

    x, r, w = (t.cuda() for t in make_rms_inputs((16, 4096), torch.bfloat16))
    want = cuda_ops.fused_add_rms_norm_fp8(x, r, w, 1e-5, group_size=128)
    codes, scales, state = torch.empty_like(want[0]), torch.empty_like(want[1]), r.clone()
    torch.ops.kernel_lab.fused_add_rms_norm_fp8(codes, scales, state, x, state, w, 1e-5, 128)
    assert torch.equal(state, want[2]) and torch.equal(scales, want[1])
    assert torch.equal(codes.view(torch.uint8), want[0].view(torch.uint8))
    base = torch.randn(5, 300, device="cuda", dtype=torch.float16)
    for lo, hi in ((0, 256), (1, 257), (8, 208)):
        view, weight = base[:, lo:hi], torch.ones(hi - lo, device="cuda", dtype=torch.float16)
        check(view, weight, 1e-6, 64, *cuda_ops.rms_norm_fp8(view, weight, group_size=64))


def test_zero_nan_infinite_and_tiny_rows():
    """A row of zeros: scale 0, codes 0. NaN or infinity in a row: its NaN stay NaN, nothing else hangs on
    them (rstd is NaN or 0). A group whose largest y is below 2^-100: scale 0, codes 0."""
    from kernel_lab import cuda_ops

    for hidden in (256, 250):  # registers, fallback
        x = torch.randn(5, hidden, device="cuda")
        x[0] = 0
        x[1, 3] = float("nan")
        x[2, 7] = float("inf")
        w = torch.ones(hidden, device="cuda")
        tiny = torch.full((hidden,), 2.0**-110, device="cuda")
        for group in (0, 128):
            codes, scales = cuda_ops.rms_norm_fp8(x, w, group_size=group)
            v = codes.float()
            assert (v[0] == 0).all() and (scales[:3] == 0).all()
            assert v[1].isnan().all()
            assert v[2, 7].isnan() and (v[2].nan_to_num(0) == 0).all()
            check(x[3:], w, 1e-6, group, codes[3:], scales[3:])
            codes, scales = cuda_ops.rms_norm_fp8(x[3:], tiny, group_size=group)
            assert (scales == 0).all() and (codes.float() == 0).all()


def test_empty_input_and_refusals():
    from kernel_lab import cuda_ops

    w = torch.ones(32, device="cuda")
    codes, scales = cuda_ops.rms_norm_fp8(torch.empty(0, 32, device="cuda"), w)
    assert codes.shape == (0, 32) and scales.shape == (0, 1)
    x = torch.randn(2, 32, device="cuda")
    with pytest.raises(RuntimeError, match="weight size"):
        cuda_ops.rms_norm_fp8(x, torch.ones(16, device="cuda"))
    with pytest.raises(RuntimeError, match="group_size"):
        cuda_ops.rms_norm_fp8(x, w, group_size=-1)
    with pytest.raises(RuntimeError, match="residual"):
        cuda_ops.fused_add_rms_norm_fp8(x, torch.randn(2, 16, device="cuda"), w)
    with pytest.raises(RuntimeError, match="share a dtype"):
        cuda_ops.rms_norm_fp8(x, w.half())
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        cuda_ops.rms_norm_fp8(x.double(), w.double())
    with pytest.raises(RuntimeError, match="scales"):
        torch.ops.kernel_lab.rms_norm_fp8(codes.new_empty(2, 32), torch.empty(2, 2, device="cuda"), x, w, 1e-6, 0)


def test_runs_on_the_current_stream_and_in_a_graph():
    from kernel_lab import cuda_ops

    x, r, w = (t.cuda() for t in make_rms_inputs((64, 2048), torch.bfloat16))
    want = cuda_ops.fused_add_rms_norm_fp8(x, r, w, 1e-5, group_size=128)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        cuda_ops.fused_add_rms_norm_fp8(x, r, w, 1e-5, group_size=128)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        got = cuda_ops.fused_add_rms_norm_fp8(x, r, w, 1e-5, group_size=128)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
