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
