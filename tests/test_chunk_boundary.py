"""The boundary of the chunked step, checked without a GPU: the header's functions are exported and bound, calls that
need no device answer, bad arguments are refused, the torch ops have Meta kernels; the oracle's own pieces."""

from __future__ import annotations

import ctypes
import re
import subprocess

import numpy as np
import pytest
import torch

from oracle import chunk
from tests.conftest import REPO

HEADER = REPO / "include" / "kernel_lab_b200_chunk.h"
INVALID = 1


def text():
    return re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)


def declared():
    return re.findall(r"^\s*(?:const\s+)?\w+\**\s+\**(kl_\w+)\s*\(", text(), flags=re.M)


def test_library_exports_and_binds_the_header():
    from kernel_lab import capi

    lib = capi.load()
    assert set(declared()) == set(capi.CHUNK_SIGNATURES)
    nm = subprocess.run(["nm", "-D", "--defined-only", str(capi.LIB_PATH)], capture_output=True, text=True, check=True)
    assert set(declared()) <= set(re.findall(r" T (kl_\w+)$", nm.stdout, flags=re.M))
    for name in declared():
        sig = re.search(name + r"\s*\((.*?)\);", text(), flags=re.S)
        assert len(getattr(lib, name).argtypes) == sig.group(1).count(",") + 1, name


def test_header_compiles_as_c_and_its_struct_is_the_binding(tmp_path):
    from kernel_lab import capi

    src = tmp_path / "use.c"
    src.write_text('#include <stdio.h>\n#include "kernel_lab_b200_chunk.h"\nint main(void) { printf("%zu %zu %zu", '
                   "sizeof(kl_page_pools_t), offsetof(kl_page_pools_t, stride), offsetof(kl_page_pools_t, bytes)); return 0; }\n")
    exe = tmp_path / "use"
    subprocess.run(["gcc", "-Wall", "-Werror", f"-I{REPO / 'include'}", str(src), "-o", str(exe)], check=True)
    got = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout
    s = capi.PagePools
    assert got == f"{ctypes.sizeof(s)} {s.stride.offset} {s.bytes.offset}"


def pools(count=1, base=256, stride=64, size=64):
    from kernel_lab import capi

    n = max(count, 1)
    return capi.PagePools(count, (ctypes.c_void_p * n)(*[base] * n), (ctypes.c_int64 * n)(*[stride] * n),
                          (ctypes.c_int64 * n)(*[size] * n))


def test_no_ops_and_refusals_without_a_device():
    from kernel_lab import capi

    lib = capi.load()

    def append(dtype=2, batch=4, tokens=9, heads=8, dim=128, page=16, bt=4, width=4, pages=10, stride=1024, ptr=16):
        return lib.kl_paged_kv_append_chunks(dtype, ptr, ptr, ptr, ptr, ptr, ptr, ptr, batch, tokens, heads, dim, page, bt, width, pages,
                                             stride, None, None)

    def append8(dtype=2, batch=4, tokens=9, heads=8, dim=128, page=16, bt=4, width=4, pages=10, stride=1024, ptr=16, scale=16):
        return lib.kl_paged_kv_append_chunks_fp8(dtype, ptr, ptr, ptr, ptr, scale, scale, ptr, ptr, ptr, batch, tokens, heads, dim, page,
                                                 bt, width, pages, stride, None, None)

    for call in (append, append8):
        assert call(batch=0) == call(tokens=0) == 0
        for bad in ({"dtype": 5}, {"batch": -1}, {"tokens": -1}, {"heads": 0}, {"dim": 0}, {"page": 0}, {"bt": 3}, {"width": -1},
                    {"pages": -1}, {"stride": 1023}, {"ptr": None}, {"heads": 1 << 20, "stride": 1 << 40}):
            assert call(**bad) == INVALID, bad
    assert append8(dim=127) == append8(scale=None) == append8(ptr=17) == INVALID

    def attend(dtype=2, code=-1, batch=4, tokens=9, hq=32, hkv=8, dim=128, page=16, q_stride=4096, ps=16384, bt=4, width=4, pages=10,
               scales=None, sps=0, ptr=256, bytes_=1 << 30):
        return lib.kl_paged_chunk_attention(dtype, code, ptr, ptr, ptr, ptr, scales, scales, ptr, ptr, ptr, batch, tokens, hq, hkv, dim,
                                            page, q_stride, ps, 1024, 128, sps, bt, width, pages, 1, 0.1, ptr, bytes_, ptr, bytes_, None)

    assert attend(batch=0) == attend(tokens=0) == 0
    for bad in ({"dtype": 3}, {"code": 2}, {"code": 0}, {"code": 0, "dtype": 0, "scales": 4}, {"code": 1, "scales": 4, "sps": -1},
                {"batch": -1}, {"tokens": -1}, {"batch": 65536}, {"hq": 31}, {"hq": 0}, {"hkv": 0}, {"dim": 0}, {"dim": 257}, {"page": 0},
                {"q_stride": 4095}, {"ps": -1}, {"bt": 3}, {"pages": 0}, {"ptr": None}, {"bytes_": 16}, {"width": 1 << 28, "bt": 1 << 28}):
        assert attend(**bad) == INVALID, bad
    a, b = ctypes.c_size_t(), ctypes.c_size_t()
    assert lib.kl_paged_chunk_attention_workspace_size(2, -1, 9, 4, 32, 8, 128, ctypes.byref(a), ctypes.byref(b)) == 0 and b.value >= 256

    def copy(p=None, src=16, pairs=3, pages=10):
        return lib.kl_paged_copy_pages(ctypes.byref(pools()) if p is None else ctypes.byref(p), src, src, pairs, pages, None, None)

    assert copy(pairs=0) == copy(pairs=0, src=None) == 0
    for bad in ({"pairs": -1}, {"pages": -1}, {"src": None}, {"pairs": 1 << 31}, {"p": pools(-1)}, {"p": pools(base=None)},
                {"p": pools(stride=63)}, {"p": pools(size=-1)}):
        assert copy(**bad) == INVALID, bad
    assert lib.kl_paged_copy_pages(None, 16, 16, 3, 10, None, None) == INVALID
    size, sync = ctypes.c_size_t(), ctypes.c_size_t()
    out = ctypes.byref(size), ctypes.byref(sync)
    assert lib.kl_paged_reserve_workspace_size(1000, 64, *out) == 0 and size.value >= 4000 + 36 * 64 and sync.value >= 4256
    assert lib.kl_paged_reserve_workspace_size(-1, 64, *out) == lib.kl_paged_reserve_workspace_size(5, -1, *out) == INVALID
    assert lib.kl_paged_compact_workspace_size(-1, *out) == lib.kl_paged_compact_workspace_size(5, None, None) == INVALID

    def reserve(p=None, out=1 << 20, table=1 << 16, parents=None, batch=4, rows=4, width=4, page=16, bt=4, pages=10, bytes_=1 << 20, ptr=256, sync=256):
        return lib.kl_paged_reserve(ctypes.byref(pools() if p is None else p), out, ptr, ptr, table, ptr, ptr, parents, batch, rows, width,
                                    page, bt, pages, 256, bytes_, sync, bytes_, None)

    assert reserve(batch=0, rows=0) == 0
    for bad in ({"batch": -1, "rows": -1}, {"rows": 5}, {"page": 0}, {"bt": 3}, {"pages": -1}, {"bytes_": 64}, {"ptr": None}, {"out": None},
                {"table": None}, {"out": 1 << 16}, {"out": (1 << 16) + 60}, {"rows": (1 << 24) + 1, "parents": 16},
                {"width": 1 << 28, "bt": 1 << 28}, {"p": pools(stride=3)}, {"sync": None}, {"sync": 264}):
        assert reserve(**bad) == INVALID, bad

    def compact(p=None, out=1 << 20, used=16, table=1 << 16, batch=4, width=4, page=16, bt=4, pages=10, bytes_=1 << 20, lens=16, sync=256):
        return lib.kl_paged_compact(ctypes.byref(pools() if p is None else p), out, used, table, lens, batch, width, page, bt, pages, 256,
                                    bytes_, sync, bytes_, None)

    for bad in ({"batch": -1}, {"used": None}, {"out": 1 << 16}, {"table": None}, {"lens": None}, {"page": 0}, {"bytes_": 64}, {"bt": 1}, {"sync": None}):
        assert compact(**bad) == INVALID, bad


def test_meta_kernels():
    from kernel_lab import cuda_ops

    t = lambda *s, dtype=torch.bfloat16: torch.empty(*s, dtype=dtype, device="meta")  # noqa: E731
    i = lambda *s: t(*s, dtype=torch.int32)  # noqa: E731
    k = t(10, 16, 2, 64)
    out = cuda_ops.paged_chunk_attention(t(9, 8, 64), k, k, i(3, 4), i(3), i(4))
    assert out.shape == (9, 8, 64) and out.device.type == "meta"
    k8 = t(10, 16, 2, 64, dtype=torch.float8_e4m3fn)
    assert cuda_ops.paged_chunk_attention_fp8(t(9, 8, 64), k8, k8, t(2), t(2), i(3, 4), i(3), i(4)).shape == (9, 8, 64)
    assert cuda_ops.paged_chunk_attention_block8(t(9, 8, 64), k8, k8, t(10, 2), t(10, 2), i(3, 4), i(3), i(4)).shape == (9, 8, 64)
    cuda_ops.paged_kv_append(k, k, t(9, 2, 64), t(9, 2, 64), i(3, 4), i(3), indptr=i(4))
    cuda_ops.paged_kv_append_fp8(k8, k8, t(9, 2, 64), t(9, 2, 64), t(2), t(2), i(3, 4), i(3), indptr=i(4))
    cuda_ops.paged_copy_pages([k, k], i(3), i(3))
    table, lens, served = cuda_ops.paged_reserve([k], i(3, 4), i(3), i(5), i(5))
    assert table.shape == (5, 4) and lens.shape == served.shape == (5,) and served.dtype is torch.bool
    table, used = cuda_ops.paged_compact([k], i(3, 4), i(3))
    assert table.shape == (3, 4) and used.shape == ()


def test_fake_tensors_and_dispatch_modes_see_the_operators():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.utils._python_dispatch import TorchDispatchMode

    from kernel_lab import cuda_ops

    class Seen(TorchDispatchMode):
        names: list[str] = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.append(str(func))
            return func(*args, **(kwargs or {}))

    with FakeTensorMode():
        i = lambda *s: torch.empty(*s, dtype=torch.int32, device="cuda")  # noqa: E731
        k = torch.empty(10, 16, 2, 64, device="cuda")
        assert cuda_ops.paged_chunk_attention(torch.empty(9, 8, 64, device="cuda"), k, k, i(3, 4), i(3), i(4)).shape == (9, 8, 64)
        assert cuda_ops.paged_reserve([k], i(3, 4), i(3), i(3))[2].dtype is torch.bool
    meta = lambda *s: torch.empty(*s, dtype=torch.int32, device="meta")  # noqa: E731
    k = torch.empty(10, 16, 2, 64, device="meta")
    with Seen():
        cuda_ops.paged_compact([k, k], meta(3, 4), meta(3))
        cuda_ops.paged_copy_pages([k], meta(2), meta(2))
        cuda_ops.paged_kv_append(k, k, k[:, 0], k[:, 0], meta(3, 4), meta(3), indptr=meta(4))
    for name in ("paged_compact", "paged_copy_pages", "paged_kv_append_chunks"):
        assert any(name in n for n in Seen.names), name


def test_cpu_tensors_are_refused():
    from kernel_lab import cuda_ops

    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    k = torch.zeros(10, 16, 2, 64)
    with pytest.raises((RuntimeError, NotImplementedError)):
        cuda_ops.paged_chunk_attention(torch.zeros(9, 8, 64), k, k, i(3, 4), i(3), i(4))
    with pytest.raises((RuntimeError, NotImplementedError)):
        cuda_ops.paged_copy_pages([k], i(1), i(1))


def test_oracle_attention_by_hand():
    """Two tokens of one head: the first sees one key, the second both, with equal scores."""
    k = np.zeros((1, 4, 1, 2))
    v = np.arange(8, dtype=np.float64).reshape(1, 4, 1, 2)
    out, tol = chunk.attention(np.ones((2, 1, 2)), k, v, np.zeros((1, 1), int), [2], [0, 2], 1.0, True)
    np.testing.assert_allclose(out[:, 0], [[0, 1], [1, 2]])
    assert (tol > 0).all() and (tol < 1e-5).all()
    out, _ = chunk.attention(np.ones((2, 1, 2)), k, v, np.zeros((1, 1), int), [1], [0, 2], 1.0, True)
    np.testing.assert_allclose(out[:, 0], [[0, 0], [0, 1]])  # the first token has nothing to attend to


def test_oracle_reserve_by_hand():
    table = np.array([[5, 2, 0], [1, 0, 0]], np.int32)
    out, lens, served, moves = chunk.reserve(table, [6, 4], [3, 1], 4, 8)
    assert out.tolist() == [[5, 2, 0], [1, 3, 0]] and lens.tolist() == [6, 4] and served.all() and not moves
    # Forks of the first: its last page stays the first row's, the other gets a copy, and the dropped page 1 is free.
    out, lens, served, moves = chunk.reserve(table, [6, 4], [1, 1], 4, 8, parents=[0, 0])
    assert out.tolist() == [[5, 2, 0], [5, 0, 0]] and moves == [(2, 0)] and served.all()


def test_oracle_compact_by_hand():
    out, used, moves = chunk.compact(np.array([[5, 2, 7], [5, 0, 0]], np.int32), [6, 7], 4, 8)
    assert used == 3 and moves == [(5, 1)] and out.tolist() == [[1, 2, 0], [1, 0, 0]]
