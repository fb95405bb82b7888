"""CPU oracle of the 8-bit serving step, from its definition (the comments of
``include/kernel_lab_b200_block8.h``): e4m3 norm, append to a block-scaled cache, page selection,
decode attention. Where the definition rounds to 32 bits the oracle does, element by element, so codes,
scales, bounds and selections are compared exactly; sums run in 64 bits. Test infrastructure only.

Caches are NumPy arrays [num_pages, page_size, num_kv_heads, head_dim] of codes (uint8 for e4m3, int8).
"""

from __future__ import annotations

import numpy as np

from oracle.oracle import e4m3_decode, e4m3_encode

QMAX = {"e4m3": 448.0, "int8": 127.0}
BOUND_UNIT = {"e4m3": 4, "int8": 1}
PER_127 = np.float32(1) / np.float32(127)
LEAST_SCALE = np.float32(2.0**-126)


def encode(x: np.ndarray, kind: str) -> np.ndarray:
    x = np.asarray(x, np.float32)
    if kind == "e4m3":
        return e4m3_encode(x)
    return np.clip(np.rint(np.where(np.isnan(x), 0, x)), -127, 127).astype(np.int8)


def decode_codes(codes: np.ndarray, kind: str) -> np.ndarray:
    return e4m3_decode(codes) if kind == "e4m3" else codes.astype(np.float32)


def scale_for(amax: np.float32, kind: str) -> np.float32:
    if not amax > 0:
        return np.float32(0)
    if kind == "int8":
        return max(np.float32(amax) * PER_127, LEAST_SCALE)
    k = -126
    while float(amax) > 448.0 * 2.0**k:
        k += 1
    return np.float32(2.0**k)


def reciprocal(scale) -> np.ndarray:
    scale = np.asarray(scale, np.float32)
    return np.where(scale >= LEAST_SCALE, np.float32(1) / np.where(scale >= LEAST_SCALE, scale, 1), 0).astype(np.float32)


def norm(x, weight, eps, group_size=0):
    """(y in 64 bits, scales in 64 bits) of rows x (already x + residual, rounded)."""
    x, w = np.asarray(x, np.float64), np.asarray(weight, np.float64)
    y = x / np.sqrt((x**2).mean(axis=-1, keepdims=True) + eps) * w
    group = group_size or x.shape[-1]
    cols = range(0, x.shape[-1], group)
    amax = np.stack([np.abs(y[..., a : a + group]).max(axis=-1) for a in cols], axis=-1)
    return y, np.where(amax >= 2.0**-100, amax / 448, 0)


def append(kind, k_cache, v_cache, k_scale, v_scale, k_bounds, k_new, v_new, table, positions, indptr=None):
    """In place; k_new and v_new are float32 [tokens, num_kv_heads, head_dim]."""
    page_size = k_cache.shape[1]
    ptr = list(range(len(positions) + 1)) if indptr is None else list(indptr)
    for b, start in enumerate(positions):
        if start < 0:
            continue
        at = ptr[b]
        while at < ptr[b + 1]:
            pos = start + at - ptr[b]
            col, s0 = divmod(pos, page_size)
            n = min(page_size - s0, ptr[b + 1] - at)
            page = table[b, col] if col < table.shape[1] else -1
            if 0 <= page < k_cache.shape[0]:
                for h in range(k_cache.shape[2]):
                    _put(kind, k_cache[page, :, h], k_scale[page], h, k_new[at : at + n, h], s0)
                    _put(kind, v_cache[page, :, h], v_scale[page], h, v_new[at : at + n, h], s0)
                    if k_bounds is not None:
                        v = np.nan_to_num(decode_codes(k_cache[page, : s0 + n, h], kind), nan=0.0) / BOUND_UNIT[kind]
                        k_bounds[page, h, 0] = np.floor(v.min(axis=0))
                        k_bounds[page, h, 1] = np.ceil(v.max(axis=0))
            at += n


def _put(kind, codes, scales, h, x, s0):
    x = np.asarray(x, np.float32)
    finite = np.abs(np.where(np.isfinite(x), x, 0))
    old = scales[h] if s0 > 0 else np.float32(0)
    new = max(old, scale_for(finite.max(), kind))
    if new > old and s0 > 0:
        codes[:s0] = encode(decode_codes(codes[:s0], kind) * (old / new), kind)
    with np.errstate(invalid="ignore", over="ignore"):
        codes[s0 : s0 + len(x)] = encode(x * reciprocal(new), kind)
    scales[h] = new


def select(kind, q, k_scale, k_bounds, table, seq_lens, page_size, num_selected, sink=1, recent=1):
    """q float32 [batch, heads, dim]; returns int32 [batch, kv heads, num_selected]."""
    batch, hq, _ = q.shape
    heads = k_scale.shape[1]
    group = hq // heads
    out = np.full((batch, heads, num_selected), -1, np.int32)
    for b, n in enumerate(seq_lens):
        count = -(-max(0, min(int(n), table.shape[1] * page_size)) // page_size)
        finite = np.where(np.isfinite(q[b]), np.abs(q[b]), 0)
        sq = (finite.max(axis=1) * PER_127).astype(np.float32)
        with np.errstate(invalid="ignore", over="ignore"):
            scaled = (q[b] * reciprocal(sq)[:, None]).astype(np.float32)
        qi = np.clip(np.rint(np.where(np.isnan(scaled), 0, scaled)), -127, 127).astype(np.int64)
        for h in range(heads):
            scores = np.empty(count, np.float32)
            for p in range(count):
                page = table[b, p]
                if not 0 <= page < k_scale.shape[0]:
                    scores[p] = -np.inf
                    continue
                lo, hi = k_bounds[page, h].astype(np.int64)
                rows = slice(h * group, (h + 1) * group)
                dots = np.maximum(qi[rows] * lo, qi[rows] * hi).sum(axis=1)
                best = (dots.astype(np.float32) * sq[rows]).max()
                scores[p] = best * (k_scale[page, h] * np.float32(BOUND_UNIT[kind]))
            scores[:sink] = np.inf
            scores[max(0, count - recent) :] = np.inf
            picked = np.sort(np.argsort(-scores, kind="stable")[:num_selected])
            out[b, h, : len(picked)] = picked
    return out


def decode(kind, q, k_cache, v_cache, k_scale, v_scale, table, seq_lens, scale, selected=None):
    """(out, weight, score, value): the attention in 64 bits; sum_t p_t |v_t| per element, the size that an
    error of the probabilities meets; each row's largest |score| and the sum of the largest magnitudes
    that its value scales allow, one per token. Rows with nothing to attend to are 0."""
    batch, hq, dim = q.shape
    pages, page_size, heads, _ = k_cache.shape
    group = hq // heads
    out, weight = np.zeros((batch, hq, dim)), np.zeros((batch, hq, dim))
    score, value = np.zeros((batch, hq, 1)), np.zeros((batch, hq, 1))
    for b, n in enumerate(seq_lens):
        n = max(0, min(int(n), table.shape[1] * page_size))
        count = -(-n // page_size)
        for h in range(heads):
            cols = range(count) if selected is None else [c for c in selected[b, h] if 0 <= c < count]
            cols = [c for c in cols if 0 <= table[b, c] < pages]
            if not cols:
                continue
            at = table[b, cols]
            pos = np.concatenate([np.arange(page_size) + c * page_size for c in cols])
            k = decode_codes(k_cache[at, :, h], kind).astype(np.float64) * k_scale[at, h, None, None]
            v = decode_codes(v_cache[at, :, h], kind).astype(np.float64) * v_scale[at, h, None, None]
            k, v = (t.reshape(-1, dim)[pos < n] for t in (k, v))
            rows = slice(h * group, (h + 1) * group)
            s = q[b, rows].astype(np.float64) @ k.T * scale
            p = np.exp(s - s.max(axis=1, keepdims=True))
            p /= p.sum(axis=1, keepdims=True)
            out[b, rows], weight[b, rows] = p @ v, p @ np.abs(v)
            score[b, rows] = np.abs(s).max(axis=1, keepdims=True)
            value[b, rows] = QMAX[kind] * np.abs(v_scale[at, h]).max() * len(v)
    return out, weight, score, value
