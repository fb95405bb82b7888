"""Python wrappers for the CUDA kernels (torch.ops.kernel_lab.*).

Same API as kernel-lab's ``kernel_lab/cuda_ops.py:11-61`` (``available``,
``why_unavailable``, ``rms_norm``, ``fused_add_rms_norm``, ``paged_decode_attention``),
plus ``num_splits`` on ``paged_decode_attention``, ``decode_status`` and the serving step around decode
(append, e4m3 and block-scaled 8-bit caches, page selection, e4m3 norms) and the chunked step (appends and attention
of chunks of new tokens, the pages that they need). There is no
fallback: if the extension is not built these functions raise RuntimeError.
"""

from __future__ import annotations

from collections.abc import Sequence

import torch

try:
    from kernel_lab import _C  # registers torch.ops.kernel_lab

    _LOADED = True
    _LOAD_ERROR = ""
except ImportError as exc:  # not built
    _LOADED = False
    _LOAD_ERROR = str(exc)


def available() -> bool:
    return _LOADED and torch.cuda.is_available()


def why_unavailable() -> str:
    if not _LOADED:
        return f"CUDA extension not built ({_LOAD_ERROR}); run `python kernel-lab_b200/build.py`"
    return "no CUDA device"


def _require() -> None:
    if not _LOADED:
        raise RuntimeError(f"kernel_lab: {why_unavailable()}")


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    _require()
    out = torch.empty_like(x, memory_format=torch.contiguous_format)
    torch.ops.kernel_lab.rms_norm(out, x, weight, eps)
    return out


def fused_add_rms_norm(
    x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6
) -> tuple[torch.Tensor, torch.Tensor]:
    """Functional form: returns (out, new_residual) and leaves ``residual`` untouched.
    Call torch.ops.kernel_lab.fused_add_rms_norm directly to update in place."""
    _require()
    out = torch.empty_like(x, memory_format=torch.contiguous_format)
    new_residual = residual.contiguous().clone()
    torch.ops.kernel_lab.fused_add_rms_norm(out, x, new_residual, weight, eps)
    return out, new_residual


def paged_decode_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    scale: float | None = None,
    num_splits: int | None = None,
) -> torch.Tensor:
    """Decode attention over a paged cache. ``num_splits=None`` uses the load-balanced
    planner; an integer forces that many KV splits per sequence (Triton semantics)."""
    _require()
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    out = torch.empty_like(q)
    if num_splits is None:
        torch.ops.kernel_lab.paged_decode_attention(out, q.contiguous(), k_cache, v_cache, block_table, seq_lens, scale)
    else:
        torch.ops.kernel_lab.paged_decode_attention_splits(
            out, q.contiguous(), k_cache, v_cache, block_table, seq_lens, scale, int(num_splits)
        )
    return out


def paged_kv_append(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_new: torch.Tensor,
    v_new: torch.Tensor,
    block_table: torch.Tensor,
    positions: torch.Tensor,
    indptr: torch.Tensor | None = None,
) -> None:
    """Write each sequence's new token's K/V rows ([batch, num_kv_heads, head_dim], rows may be a
    strided view) into its pages at token index ``positions[b]`` (in place; negative skips).
    With ``indptr`` (int32 [batch + 1]) sequence b's new tokens are the rows ``indptr[b]`` .. ``indptr[b + 1] - 1``
    and take the positions from ``positions[b]`` on. Caches are contiguous [num_pages, page_size, num_kv_heads, head_dim].
    Page ids outside the pool are skipped and reported by :func:`decode_status`."""
    _require()
    if indptr is not None:
        tensors = (k_cache, v_cache, k_new, v_new, block_table, positions, indptr)
        (_C if _direct(*tensors) else torch.ops.kernel_lab).paged_kv_append_chunks(*tensors)
        return
    torch.ops.kernel_lab.paged_kv_append(k_cache, v_cache, k_new, v_new, block_table, positions)


def paged_decode_attention_fp8(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    scale: float | None = None,
) -> torch.Tensor:
    """Decode attention over an e4m3 KV cache (torch.float8_e4m3fn) with per-KV-head float32
    scales: K = code * k_scale[h], V = code * v_scale[h]. q is fp16 or bf16."""
    _require()
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    out = torch.empty_like(q)
    torch.ops.kernel_lab.paged_decode_attention_fp8(
        out, q.contiguous(), k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, scale
    )
    return out


def paged_kv_append_fp8(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_new: torch.Tensor,
    v_new: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    block_table: torch.Tensor,
    positions: torch.Tensor,
    indptr: torch.Tensor | None = None,
) -> None:
    """paged_kv_append into an e4m3 cache: rows are quantised per KV head as
    e4m3(x / scale) (round to nearest-even, saturating to +-448)."""
    _require()
    if indptr is not None:
        tensors = (k_cache, v_cache, k_new, v_new, k_scale, v_scale, block_table, positions, indptr)
        (_C if _direct(*tensors) else torch.ops.kernel_lab).paged_kv_append_chunks_fp8(*tensors)
        return
    torch.ops.kernel_lab.paged_kv_append_fp8(k_cache, v_cache, k_new, v_new, k_scale, v_scale, block_table, positions)


def paged_decode_attention_cascade(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    prefix_block_table: torch.Tensor,
    prefix_lens: torch.Tensor,
    prefix_indptr: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    scale: float | None = None,
    k_scale: torch.Tensor | None = None,
    v_scale: torch.Tensor | None = None,
) -> torch.Tensor:
    """Shared-prefix (cascade) decode: the sequences of group p, ``prefix_indptr[p]`` up to
    ``prefix_indptr[p + 1]``, attend to the ``prefix_lens[p]`` tokens held in the pages of row p
    of ``prefix_block_table`` and then to their own ``seq_lens[b]`` tokens (``block_table`` row b).
    A prefix's pages are read once per block of its group's sequences, not once per sequence.
    With ``k_scale`` / ``v_scale`` the caches are e4m3 (torch.float8_e4m3fn)."""
    _require()
    out = torch.empty_like(q)
    torch.ops.kernel_lab.paged_decode_attention_cascade(
        out, q, k_cache, v_cache, prefix_block_table, prefix_lens, prefix_indptr, block_table, seq_lens,
        q.shape[-1] ** -0.5 if scale is None else scale, k_scale, v_scale,
    )
    return out


def _direct(*tensors: torch.Tensor | None) -> bool:
    """Whether a call may go past the dispatcher: real CUDA tensors, and nothing traces, transforms or watches it."""
    return not torch.compiler.is_compiling() and not torch.overrides.has_torch_function(tensors) and _C.direct(*tensors)


def rms_norm_fp8(
    x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, group_size: int = 0
) -> tuple[torch.Tensor, torch.Tensor]:
    """RMSNorm with an e4m3 output: (codes, scales), y = codes * scales. ``group_size`` columns share
    a scale (0: a whole row); codes are torch.float8_e4m3fn in x's shape, scales float32
    [..., ceil(hidden / group_size)]. A scale is its group's largest magnitude / 448."""
    _require()
    if _direct(x, weight):
        return _C.rms_norm_fp8(x, weight, eps, group_size)
    codes, scales = _fp8_outputs(x, group_size)
    torch.ops.kernel_lab.rms_norm_fp8(codes, scales, x, weight, eps, group_size)
    return codes, scales


def fused_add_rms_norm_fp8(
    x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, group_size: int = 0
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Functional form: (codes, scales, new_residual) of x + residual, ``residual`` left untouched.
    Call torch.ops.kernel_lab.fused_add_rms_norm_fp8 with residual_out = residual to update in place."""
    _require()
    if _direct(x, residual, weight):
        return _C.fused_add_rms_norm_fp8(x, residual, weight, eps, group_size)
    codes, scales = _fp8_outputs(x, group_size)
    new_residual = torch.empty_like(x, memory_format=torch.contiguous_format)
    torch.ops.kernel_lab.fused_add_rms_norm_fp8(
        codes, scales, new_residual, x, residual.contiguous(), weight, eps, group_size
    )
    return codes, scales, new_residual


def _fp8_outputs(x: torch.Tensor, group_size: int) -> tuple[torch.Tensor, torch.Tensor]:
    groups = 1 if group_size == 0 else -(-x.shape[-1] // group_size)
    codes = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    return codes, torch.empty((*x.shape[:-1], groups), dtype=torch.float32, device=x.device)


def paged_kv_append_block8(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    k_new: torch.Tensor,
    v_new: torch.Tensor,
    block_table: torch.Tensor,
    positions: torch.Tensor,
    indptr: torch.Tensor | None = None,
    k_bounds: torch.Tensor | None = None,
) -> None:
    """Append to an 8-bit cache (float8_e4m3fn or int8, [num_pages, page_size, num_kv_heads, head_dim],
    any order of pages, tokens and heads in memory) with a float32 scale for each page and KV head
    (in place). Sequence b's new rows ``indptr[b]`` .. ``indptr[b + 1] - 1`` (one row per sequence
    without ``indptr``) take the positions from ``positions[b]`` on (negative skips the sequence). A page's
    scale covers its largest element: it starts with the page's first token and grows when a later
    one needs it, the page's earlier codes being rounded again. ``k_bounds`` (int8 [num_pages,
    num_kv_heads, 2, head_dim]) keeps each touched page's per-channel key extremes for
    :func:`paged_block_select`. Two sequences must not append to one page. Page ids outside the pool
    are skipped and reported by :func:`decode_status`."""
    _require()
    tensors = (k_cache, v_cache, k_scale, v_scale, k_bounds, k_new, v_new, block_table, positions, indptr)
    append = _C.paged_kv_append_block8 if _direct(*tensors) else torch.ops.kernel_lab.paged_kv_append_block8
    append(*tensors)


def paged_decode_attention_block8(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    scale: float | None = None,
    selected: torch.Tensor | None = None,
) -> torch.Tensor:
    """Decode attention over an 8-bit cache with a scale for each page and KV head: K = code *
    k_scale[page, h], V = code * v_scale[page, h]. q is fp16 or bf16. With ``selected`` (int32 [batch,
    num_kv_heads, n], :func:`paged_block_select`) KV head h of sequence b reads only the pages in those
    columns of its block-table row (each at most once; -1 selects nothing)."""
    _require()
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    if _direct(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, selected):
        return _C.paged_decode_attention_block8(
            q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, scale, selected
        )
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    torch.ops.kernel_lab.paged_decode_attention_block8(
        out, q.contiguous(), k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, scale, selected
    )
    return out


def paged_block_select(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    k_scale: torch.Tensor,
    k_bounds: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    num_selected: int,
    sink_pages: int = 1,
    recent_pages: int = 1,
) -> torch.Tensor:
    """The pages a decode step should read: for each sequence and KV head the ``num_selected``
    block-table columns (int32 [batch, num_kv_heads, num_selected], ascending, then -1) whose key
    bounds allow the largest scores, the first ``sink_pages`` and the last ``recent_pages`` always among
    them. Scores are sums of whole numbers (q rounded to int8 per head), ties go to the lower column:
    the choice is the same on every run and rank."""
    _require()
    if _direct(q, k_cache, k_scale, k_bounds, block_table, seq_lens):
        return _C.paged_block_select(
            q, k_cache, k_scale, k_bounds, block_table, seq_lens, num_selected, sink_pages, recent_pages
        )
    selected = torch.empty((q.shape[0], k_cache.shape[2], num_selected), dtype=torch.int32, device=q.device)
    torch.ops.kernel_lab.paged_block_select(
        selected, q.contiguous(), k_cache, k_scale, k_bounds, block_table, seq_lens, sink_pages, recent_pages
    )
    return selected


def _rows_of_q(q: torch.Tensor) -> torch.Tensor:
    """q as rows of contiguous heads, any distance apart that keeps them from overlapping."""
    heads = q.stride(-1) == 1 and (q.stride(1) == q.shape[2] or q.shape[1] == 1)
    return q if heads and (q.stride(0) >= q.shape[1] * q.shape[2] or q.shape[0] <= 1) else q.contiguous()


def paged_chunk_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    indptr: torch.Tensor,
    scale: float | None = None,
    causal: bool = True,
) -> torch.Tensor:
    """Attention of chunks of new tokens over a paged cache (prompts, chunks of them, draft tokens, single
    tokens, in one call). q is [tokens, num_q_heads, head_dim] (rows may be a strided view); sequence b's new tokens are its
    rows ``indptr[b]`` .. ``indptr[b + 1] - 1`` (indptr: int32 [batch + 1]) and the last of the ``seq_lens[b]`` tokens in its
    pages: append them first (:func:`paged_kv_append`). A token attends to the tokens up to itself, without
    ``causal`` to all ``seq_lens[b]`` (cross attention over an encoder's states). What is masked does not count,
    whatever it holds; a token that has none to attend to gets zeros. The rows of the result that are no sequence's are
    undefined. Caches as in :func:`paged_decode_attention`, or views with any order of pages, tokens and heads in memory
    (those the 16-bit and e4m3 appends here cannot write: they take contiguous caches)."""
    _require()
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    tensors = (k_cache, v_cache, block_table, seq_lens, indptr)
    if _direct(q, *tensors):
        return _C.paged_chunk_attention(q, *tensors, scale, causal)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    torch.ops.kernel_lab.paged_chunk_attention(out, _rows_of_q(q), *tensors, scale, causal)
    return out


def paged_chunk_attention_fp8(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    indptr: torch.Tensor,
    scale: float | None = None,
    causal: bool = True,
) -> torch.Tensor:
    """:func:`paged_chunk_attention` over an e4m3 cache with per-KV-head float32 scales (as
    :func:`paged_decode_attention_fp8`). q is fp16 or bf16."""
    _require()
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    tensors = (k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, indptr)
    if _direct(q, *tensors):
        return _C.paged_chunk_attention_fp8(q, *tensors, scale, causal)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    torch.ops.kernel_lab.paged_chunk_attention_fp8(out, _rows_of_q(q), *tensors, scale, causal)
    return out


def paged_chunk_attention_block8(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    indptr: torch.Tensor,
    scale: float | None = None,
    causal: bool = True,
) -> torch.Tensor:
    """:func:`paged_chunk_attention` over an 8-bit cache with a scale for each page and KV head (as
    :func:`paged_decode_attention_block8`). q is fp16 or bf16."""
    _require()
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    tensors = (k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, indptr)
    if _direct(q, *tensors):
        return _C.paged_chunk_attention_block8(q, *tensors, scale, causal)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    torch.ops.kernel_lab.paged_chunk_attention_block8(out, _rows_of_q(q), *tensors, scale, causal)
    return out


def paged_copy_pages(caches: Sequence[torch.Tensor], src: torch.Tensor, dst: torch.Tensor) -> None:
    """Copy page ``src[i]`` to page ``dst[i]`` (int32 [n]; negative skips) in every tensor of ``caches``, in one launch for
    up to 64 of them: keys, values, scales and bounds of any number of layers, whose first dimension is the page
    and whose pages each fill one piece of memory. No page may be a destination twice, or both a source and a
    destination. Page ids outside the pool are skipped and reported by :func:`decode_status`."""
    _require()
    caches = list(caches)
    if _direct(*caches, src, dst):
        _C.paged_copy_pages(caches, src, dst)
    else:
        torch.ops.kernel_lab.paged_copy_pages(caches, src, dst)


def paged_reserve(
    caches: Sequence[torch.Tensor],
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    new_tokens: torch.Tensor,
    parents: torch.Tensor | None = None,
    page_size: int | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Pages for the tokens to come, on the device: (block_table, seq_lens, served), new tensors. Without ``parents`` the
    rows are the sequences; with it (int32 [rows]) row r is a fork of sequence ``parents[r]`` (negative: an empty row) and
    shares its pages, and sequences that no row names are dropped. A page is free if no row's first
    ceil(len / page_size) entries name it, so dropping or shortening a sequence frees its pages, and whatever is to keep
    pages (a stored prefix, say) has to be a row. In the order of the rows each takes the free pages with the
    lowest ids: a copy of its last page if ``new_tokens[r]`` > 0, that page is partly filled and others hold
    it too (copied in every tensor of ``caches``; of several that only write to it the lowest row keeps it), then pages
    for the ``new_tokens[r]`` tokens that are to be appended at ``seq_lens[r]``. ``served[r]`` is False, and the row
    gets nothing, where the table is too narrow or the free pages run out (then
    :func:`decode_status` has bit 32). Entries past a row's pages are 0, a page like any other: append for such a row at
    position -1 (``torch.where(served, seq_lens, -1)``) and let its length be, or it writes to pages of others. An empty row
    is served, whatever ``new_tokens`` says, and has no pages either; a parent past the last sequence makes one, without a
    status bit. The returned lengths do not count the new tokens. ``page_size`` is by default the second dimension of the
    first cache."""
    _require()
    caches = list(caches)
    page_size = caches[0].shape[1] if page_size is None else page_size
    if _direct(*caches, block_table, seq_lens, new_tokens, parents):
        return _C.paged_reserve(caches, block_table, seq_lens, new_tokens, parents, page_size)
    rows = (seq_lens if parents is None else parents).shape[0]
    table = torch.empty((rows, block_table.shape[1]), dtype=torch.int32, device=block_table.device)
    lens = torch.empty((rows,), dtype=torch.int32, device=block_table.device)
    served = torch.empty((rows,), dtype=torch.bool, device=block_table.device)
    torch.ops.kernel_lab.paged_reserve(
        table, lens, served, caches, block_table, seq_lens, new_tokens, parents, page_size
    )
    return table, lens, served


def paged_compact(
    caches: Sequence[torch.Tensor], block_table: torch.Tensor, seq_lens: torch.Tensor, page_size: int | None = None
) -> tuple[torch.Tensor, torch.Tensor]:
    """Move the pages in use to the lowest ids: (block_table, used), new tensors. ``used`` (int32 scalar) pages are
    named by the rows' first ceil(len / page_size) entries; those with ids of ``used`` and more go, in order, to the free
    ids below, in every tensor of ``caches``. Afterwards the pages from ``used`` on are free."""
    _require()
    caches = list(caches)
    page_size = caches[0].shape[1] if page_size is None else page_size
    if _direct(*caches, block_table, seq_lens):
        return _C.paged_compact(caches, block_table, seq_lens, page_size)
    table = torch.empty((seq_lens.shape[0], block_table.shape[1]), dtype=torch.int32, device=block_table.device)
    used = torch.empty((), dtype=torch.int32, device=block_table.device)
    torch.ops.kernel_lab.paged_compact(table, used, caches, block_table, seq_lens, page_size)
    return table, used


def decode_status(clear: bool = False) -> int:
    """KL_STATUS_* bits left by decode, append and selection calls on the current device and stream, and
    by those of CUDA graphs captured on the device (synchronises). After bit 4 (a wait inside a kernel ran out: the
    results of that call, and of later ones on its scratch, are invalid) ``clear`` also zeroes the scratch's counters,
    and calls work again; no graph that has the bit may run meanwhile."""
    _require()
    return int(_C.decode_status(clear))
