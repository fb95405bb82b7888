"""Calls of the chunked step at the edge of what is accepted, refused before any launch: no GPU is needed."""

from __future__ import annotations

import ctypes

import pytest

INVALID = 1


def attend(dtype=2, tokens=9, batch=4, hq=32, hkv=8, dim=128, scales=None, code=-1, partials=1 << 20, sync=256):
    """kl_paged_chunk_attention of addresses that nothing reads: only calls that are refused."""
    from kernel_lab import capi

    lib = capi.load()
    a, b = ctypes.c_size_t(), ctypes.c_size_t()
    assert lib.kl_paged_chunk_attention_workspace_size(dtype, code, tokens, batch, hq, hkv, dim, ctypes.byref(a), ctypes.byref(b)) == 0
    return lib.kl_paged_chunk_attention(dtype, code, 256, 256, 256, 256, scales, scales, 256, 256, 256, batch, tokens, hq, hkv, dim, 16,
                                        hq * dim, 16 * hkv * dim, hkv * dim, dim, 0, 4, 4, 10, 1, 0.1, partials, a.value, sync, b.value, None)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("code,scales", [(-1, None), (0, 256), (1, 256)])
def test_pieces_are_stored_32_bytes_at_a_time(dim, code, scales):
    for at in (4, 8, 16, 48):
        assert attend(dim=dim, code=code, scales=scales, partials=(1 << 20) + at) == INVALID, at
    for at in (1, 2, 3):
        assert attend(dim=dim, code=code, scales=scales, sync=256 + at) == INVALID, at
        assert attend(dtype=0, sync=256 + at) == INVALID, at


def test_chunks_that_32_bit_rows_cannot_count():
    """A block has up to 256 tokens: one that ends past the last token is still counted in 32 bits."""
    for tokens in (2**31 - 256, 2**31 - 2, 2**31 - 1, 2**31, 2**40):
        assert attend(hq=1, hkv=1, dim=8, tokens=tokens) == INVALID, tokens
        assert attend(hq=1, hkv=1, dim=8, tokens=tokens, dtype=0) == INVALID, tokens


def reserve(out=1 << 20, lens_out=2 << 20, served=3 << 20, table=4 << 20, lens=5 << 20, new=6 << 20, parents=None):
    from kernel_lab import capi

    pools = capi.PagePools(0, None, None, None)
    return capi.load().kl_paged_reserve(ctypes.byref(pools), out, lens_out, served, table, lens, new, parents, 4, 4, 4, 16, 4, 10,
                                        8 << 20, 1 << 20, 9 << 20, 1 << 20, None)


def compact(out=1 << 20, used=2 << 20, table=4 << 20, lens=5 << 20):
    from kernel_lab import capi

    pools = capi.PagePools(0, None, None, None)
    return capi.load().kl_paged_compact(ctypes.byref(pools), out, used, table, lens, 4, 4, 16, 4, 10, 8 << 20, 1 << 20, 9 << 20, 1 << 20, None)


def test_outputs_of_the_bookkeeping_that_overlap_its_inputs():
    """Rows are read while others are written."""
    at, parents = 5 << 20, 7 << 20
    for bad in ({"lens_out": at, "parents": parents}, {"lens_out": at + 4}, {"lens_out": at - 12}, {"lens_out": 6 << 20}, {"lens_out": 6 << 20, "parents": parents},
                {"lens_out": parents, "parents": parents}, {"lens_out": (4 << 20) + 60}, {"served": at + 15}, {"served": 6 << 20}, {"served": (4 << 20) + 63},
                {"served": parents + 3, "parents": parents}, {"out": at - 60}, {"out": 6 << 20}, {"out": parents, "parents": parents}, {"out": 4 << 20},
                {"out": 2 << 20}, {"served": (1 << 20) + 8}, {"served": (2 << 20) + 8}):
        assert reserve(**bad) == INVALID, bad
    for bad in ({"out": at}, {"out": 4 << 20}, {"used": at + 12}, {"used": (4 << 20) + 8}, {"used": (1 << 20) + 60}):
        assert compact(**bad) == INVALID, bad
