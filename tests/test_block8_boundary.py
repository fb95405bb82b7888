"""The boundary of the 8-bit serving step, checked without a GPU: the header's functions are exported and
bound, calls that need no device answer, the torch ops have Meta kernels; the oracle's own pieces."""

from __future__ import annotations

import ctypes
import re
import subprocess

import numpy as np
import pytest
import torch

from oracle import block8
from tests.conftest import REPO

HEADER = REPO / "include" / "kernel_lab_b200_block8.h"
INVALID = 1


def declared():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    return re.findall(r"^\s*(?:const\s+)?\w+\**\s+\**(kl_\w+)\s*\(", text, flags=re.M)


def test_library_exports_and_binds_the_header():
    from kernel_lab import capi

    lib = capi.load()
    assert set(declared()) == set(capi.BLOCK8_SIGNATURES)
    nm = subprocess.run(["nm", "-D", "--defined-only", str(capi.LIB_PATH)], capture_output=True, text=True, check=True)
    assert set(declared()) <= set(re.findall(r" T (kl_\w+)$", nm.stdout, flags=re.M))
    for name in declared():
        # As many parameters as the header declares.
        sig = re.search(name + r"\s*\((.*?)\);", re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S), flags=re.S)
        assert len(getattr(lib, name).argtypes) == sig.group(1).count(",") + 1, name


def test_header_compiles_as_c(tmp_path):
    src = tmp_path / "use.c"
    src.write_text('#include "kernel_lab_b200_block8.h"\nint main(void) { return KL_CODE_E4M3; }\n')
    subprocess.run(["gcc", "-Wall", "-Werror", f"-I{REPO / 'include'}", "-c", str(src), "-o", str(tmp_path / "use.o")], check=True)


def test_no_ops_and_refusals_without_a_device():
    from kernel_lab import capi

    lib = capi.load()
    norm = lambda rows, hidden=64, group=0, ptr=1, res=None: lib.kl_rms_norm_fp8(  # noqa: E731
        2, ptr, ptr, res, ptr, None, ptr, rows, hidden, 64, group, 1e-5, None)
    assert norm(0) == 0
    assert norm(-1) == norm(4, hidden=0) == norm(4, group=-1) == norm(4, ptr=None) == norm(4, res=1) == INVALID
    assert lib.kl_rms_norm_fp8(9, 1, 1, None, 1, None, 1, 4, 64, 64, 0, 1e-5, None) == INVALID

    def append(dtype=2, code=0, batch=4, tokens=4, heads=8, dim=128, page=16, stride=1024, indptr=None, ptr=1, width=4):
        return lib.kl_paged_kv_append_block8(dtype, code, ptr, ptr, ptr, ptr, None, ptr, ptr, ptr, ptr, indptr, batch, tokens,
                                             heads, dim, page, 16384, 1024, 128, 4, width, 10, stride, None, None)

    assert append(batch=0) == append(tokens=0, indptr=1) == 0
    for bad in ({"code": 2}, {"dtype": 5}, {"tokens": 5}, {"heads": 0}, {"dim": 1025}, {"page": 0}, {"stride": 1000},
                {"ptr": None}, {"width": 5}, {"batch": -1}, {"tokens": -1}):
        assert append(**bad) == INVALID, bad

    def decode(dtype=2, code=0, batch=4, hq=32, hkv=8, dim=128, page=16, token=1024, selected=None, n=0, q=16, bytes_=1 << 30):
        return lib.kl_paged_decode_block8(dtype, code, 16, q, 16, 16, 4, 4, 4, 4, selected, batch, hq, hkv, dim, page, 16384,
                                          token, 128, 4, 4, 10, n, 0.1, 16, bytes_, 16, bytes_, None)

    assert decode(batch=0) == 0
    for bad in ({"dtype": 0}, {"code": 2}, {"hq": 31}, {"hq": 8 * 129}, {"dim": 72}, {"dim": 272}, {"page": 12}, {"page": 0},
                {"token": 1000}, {"selected": 4}, {"n": 4}, {"q": 8}, {"bytes_": 16}, {"batch": -1}, {"dim": 256, "hq": 8 * 65}):
        assert decode(**bad) == INVALID, bad

    def select(dtype=2, code=0, batch=4, hq=32, hkv=8, dim=128, n=8, sink=1, recent=1, bounds=16, bytes_=1 << 20):
        return lib.kl_paged_block_select(dtype, code, 4, 4, bounds, 4, 4, 4, batch, hq, hkv, dim, 16, 4, 4, 10, n, sink, recent,
                                         4, bytes_, 4, bytes_, None)

    assert select(batch=0) == 0
    for bad in ({"dtype": 4}, {"code": 3}, {"hq": 31}, {"dim": 24}, {"dim": 272}, {"n": 0}, {"sink": 8}, {"sink": -1},
                {"bounds": 8}, {"bytes_": 16}, {"batch": 65536}):
        assert select(**bad) == INVALID, bad


def test_workspaces_grow_with_the_problem():
    from kernel_lab import capi

    lib = capi.load()
    part, sync = ctypes.c_size_t(1), ctypes.c_size_t(0)
    size = lambda *a: (lib.kl_paged_decode_block8_workspace_size(*a, ctypes.byref(part), ctypes.byref(sync)), part.value, sync.value)  # noqa: E731
    assert size(0, 32, 8, 128, 16, 4, 0) == (0, 0, 4)
    rc, p, s = size(64, 32, 8, 128, 16, 256, 0)
    assert rc == 0 and p > 0 and s == 4 * (1 + 64 * 8)
    assert size(64, 32, 8, 100, 16, 256, 0)[0] == INVALID
    assert size(64, 32, 1, 128, 16, 256, 0)[2] == 4 * (1 + 64 * 2)  # 32 query heads take two warps
    rc = lib.kl_paged_block_select_workspace_size(4, 8, 100, ctypes.byref(part), ctypes.byref(sync))
    assert (rc, part.value, sync.value) == (0, 4 * 8 * 100 * 4, 4 * 33)


def test_meta_kernels_trace_without_a_device():
    from kernel_lab import _C  # noqa: F401

    ops = torch.ops.kernel_lab
    e = lambda *shape, dtype=torch.bfloat16: torch.empty(*shape, dtype=dtype, device="meta")  # noqa: E731
    f32, i32 = torch.float32, torch.int32
    ops.rms_norm_fp8(e(4, 64, dtype=torch.float8_e4m3fn), e(4, 1, dtype=f32), e(4, 64), e(64), 1e-5, 0)
    ops.fused_add_rms_norm_fp8(e(4, 64, dtype=torch.float8_e4m3fn), e(4, 1, dtype=f32), e(4, 64), e(4, 64), e(4, 64), e(64), 1e-5, 0)
    cache, scale = e(4, 16, 2, 64, dtype=torch.int8), e(4, 2, dtype=f32)
    table, lens, new = e(2, 2, dtype=i32), e(2, dtype=i32), e(2, 2, 64)
    ops.paged_kv_append_block8(cache, cache, scale, scale, None, new, new, table, lens)
    ops.paged_kv_append_block8(cache, cache, scale, scale, e(4, 2, 2, 64, dtype=torch.int8), new, new, table, lens, lens)
    q = e(2, 8, 64)
    chosen = e(2, 2, 3, dtype=i32)
    ops.paged_block_select(chosen, q, cache, scale, e(4, 2, 2, 64, dtype=torch.int8), table, lens, 1, 1)
    ops.paged_decode_attention_block8(e(2, 8, 64), q, cache, cache, scale, scale, table, lens, 0.1)
    ops.paged_decode_attention_block8(e(2, 8, 64), q, cache, cache, scale, scale, table, lens, 0.1, chosen)


@pytest.mark.parametrize("amax,scale", [(448.0, 1.0), (448.5, 2.0), (7.0, 2.0**-6), (1e-45, 2.0**-126), (3e38, 2.0**120), (0.0, 0.0)])
def test_oracle_e4m3_scale(amax, scale):
    assert block8.scale_for(np.float32(amax), "e4m3") == scale


def test_oracle_append_then_decode_recovers_the_tokens():
    """A prompt appended in one piece and token by token dequantises to the tokens within the formats' steps."""
    rng = np.random.RandomState(0)
    x = rng.randn(2, 37, 2, 16).astype(np.float32)
    for kind, step in (("e4m3", 2.0**-4), ("int8", 2.0 / 127)):
        for pieces in ([37], [1] * 37):
            codes = np.zeros((2, 3, 16, 2, 16), np.uint8 if kind == "e4m3" else np.int8)
            scales = np.full((2, 3, 2), 9.0, np.float32)  # stale scales of an earlier use
            table = np.array([[2, 0, 1]], np.int32)
            at = 0
            for n in pieces:
                block8.append(kind, codes[0], codes[1], scales[0], scales[1], None, x[0, at : at + n], x[1, at : at + n],
                              table, [at], [0, n])
                at += n
            for t in range(2):
                got = block8.decode_codes(codes[t][table[0]], kind) * scales[t][table[0]][:, None, :, None]
                err = np.abs(got.reshape(-1, 2, 16)[:37] - x[t])
                assert err.max() <= step * np.abs(x[t]).max()


@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
def test_block8_pool_layouts(heads_first, dtype):
    from kernel_lab.kv_cache import block8_pool

    pool = block8_pool(5, 16, 3, 32, dtype, device="cpu", heads_first=heads_first)
    assert pool.k_cache.shape == (5, 16, 3, 32) and pool.k_cache.dtype == dtype
    assert pool.k_cache.stride() == ((1536, 32, 512, 1) if heads_first else (1536, 96, 32, 1))
    assert pool.k_scale.shape == (5, 3) and pool.k_bounds.shape == (5, 3, 2, 32)
    assert block8_pool(5, 16, 3, 32, dtype, device="cpu", bounds=False).k_bounds is None
    with pytest.raises(ValueError):
        block8_pool(5, 16, 3, 32, torch.float16, device="cpu")
