"""The functions of kernel_lab.cuda_ops around the 8-bit cache under everything that watches operators through the
dispatcher: meta and fake tensors, tracing, dispatch modes, tensor subclasses, a profiler. On the CPU unless marked."""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.utils._python_dispatch import TorchDispatchMode

NAMES = ["rms_norm_fp8", "fused_add_rms_norm_fp8", "paged_kv_append_block8", "paged_block_select", "paged_decode_attention_block8"]


def step(device):
    """Every function once, on tensors of the device."""
    from kernel_lab import cuda_ops

    def empty(*shape, dtype=torch.bfloat16):
        return torch.zeros(*shape, dtype=torch.uint8, device=device).view(dtype) if dtype is torch.float8_e4m3fn else torch.zeros(*shape, dtype=dtype, device=device)

    f32, i32 = torch.float32, torch.int32
    x, w = empty(4, 256), empty(256)
    codes, scales = cuda_ops.rms_norm_fp8(x, w, group_size=100)
    codes2, scales2, residual = cuda_ops.fused_add_rms_norm_fp8(x, x, w)
    cache, scale, bounds = empty(4, 16, 2, 64, dtype=torch.float8_e4m3fn), empty(4, 2, dtype=f32), empty(4, 2, 2, 64, dtype=torch.int8)
    values, value_scale = cache.clone(), scale.clone()
    table, lens, new = empty(2, 2, dtype=i32), empty(2, dtype=i32), empty(2, 2, 64)
    table[1] += 2  # a page for each
    cuda_ops.paged_kv_append_block8(cache, values, scale, value_scale, new, new, table, lens, k_bounds=bounds)
    q = empty(2, 8, 64)
    chosen = cuda_ops.paged_block_select(q, cache, scale, bounds, table, lens, 2)
    out = cuda_ops.paged_decode_attention_block8(q, cache, values, scale, value_scale, table, lens, selected=chosen)
    assert codes.shape == codes2.shape == (4, 256) and codes.dtype == torch.float8_e4m3fn
    assert scales.shape == (4, 3) and scales2.shape == (4, 1) and residual.shape == x.shape
    assert chosen.shape == (2, 2, 2) and chosen.dtype == i32 and out.shape == q.shape and out.dtype == q.dtype
    return codes, scales, residual, chosen, out


def test_meta_tensors():
    assert all(t.is_meta for t in step("meta"))


@pytest.mark.parametrize("device", ["cuda", "meta"])
def test_fake_tensors(device):
    with FakeTensorMode():
        assert all(type(t).__name__ == "FakeTensor" and t.device.type == device for t in step(device))


def test_make_fx_traces_the_operators():
    from torch.fx.experimental.proxy_tensor import make_fx

    from kernel_lab import cuda_ops

    with FakeTensorMode():
        x, w = torch.empty(4, 64, device="cuda"), torch.empty(64, device="cuda")
    graph = make_fx(lambda x, w: cuda_ops.rms_norm_fp8(x, w), tracing_mode="fake")(x, w)
    assert any("rms_norm_fp8" in str(node.target) for node in graph.graph.nodes)


class Seen(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        if func.namespace == "kernel_lab":
            self.names.append(func._schema.name.split("::")[1])
        return func(*args, **(kwargs or {}))


def test_a_dispatch_mode_sees_the_operators_on_meta_tensors():
    with Seen() as mode:
        step("meta")
    assert mode.names == NAMES


def test_host_tensors_are_refused():
    with pytest.raises((RuntimeError, NotImplementedError), match="CPU|CUDA"):
        step("cpu")


@pytest.mark.gpu
def test_a_dispatch_mode_and_a_profiler_see_the_operators():
    step("cuda")
    with Seen() as mode:
        step("cuda")
    assert mode.names == NAMES
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as profile:
        step("cuda")
    assert {f"kernel_lab::{name}" for name in NAMES} <= {e.name for e in profile.events()}


@pytest.mark.gpu
def test_a_subclass_sees_the_operators():
    from kernel_lab import cuda_ops

    class Watched(torch.Tensor):
        names = []

        @classmethod
        def __torch_function__(cls, func, types, args=(), kwargs=None):
            cls.names.append(str(func))
            return super().__torch_function__(func, types, args, kwargs or {})

    x = torch.randn(4, 256, device="cuda").as_subclass(Watched)
    cuda_ops.rms_norm_fp8(x, torch.ones(256, device="cuda"))
    assert any("rms_norm_fp8" in name for name in Watched.names)


@pytest.mark.gpu
def test_the_direct_and_the_dispatched_call_agree():
    """The same results, also for a q that starts on no 16 bytes, and Parameters take the direct call."""
    from kernel_lab import cuda_ops
    from tests.test_gpu_block8 import Pool

    pool = Pool("e4m3", [40, 70], 2, 64, 16, seed=50)
    table, lens = pool.tables()
    state = pool.gpu()
    for shift in (0, 1, 8):
        q = torch.randn(2 * 8 * 64 + shift, device="cuda").to(torch.float16)[shift:].view(2, 8, 64)
        args = (q, *state.values(), table, lens)
        assert cuda_ops._direct(*args)
        direct = cuda_ops.paged_decode_attention_block8(*args)
        with Seen():
            assert not cuda_ops._direct(*args)
            assert torch.equal(cuda_ops.paged_decode_attention_block8(*args), direct)
    x, w = torch.randn(4, 256, device="cuda"), torch.nn.Parameter(torch.ones(256, device="cuda"))
    assert cuda_ops._direct(x, w, None) and not cuda_ops._direct(x, w.cpu())
