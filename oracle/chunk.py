"""The chunked step over a paged cache, in 64-bit NumPy: attention of chunks of new tokens with the error that a kernel
may have, and the pages' bookkeeping sequence by sequence."""

from __future__ import annotations

import numpy as np


def gather(cache, table, length):
    """[length, kv heads, dim] of one sequence from a [pages, page, kv heads, dim] cache."""
    page = cache.shape[1]
    tok = np.arange(length)
    return cache[table[tok // page], tok % page]


def attention(q, k_cache, v_cache, table, lens, indptr, scale, causal, k_scale=None, v_scale=None, bits=24, p_bits=24, num_pages=None):
    """(out, tol) of float64 inputs. Scales: [kv heads] or [pages, kv heads]. `bits`: the significand of the output
    type, `p_bits` that of a rounded probability. tol bounds the error: each probability rounded (2^-p_bits of it), the
    scores' fp32 sums (dim + 8 roundings of 2^-24 of the sum of magnitudes), the exponential (off by at most 3.0e-6 < 2^-18,
    beside a rounding to 8 bits 1.02e-4 < 2^-13: the largest relative errors of its polynomials) and the fp32 sums over the
    keys, the output rounded. Pages outside the pool count as masked."""
    rows, hq, dim = q.shape
    page, hkv = k_cache.shape[1:3]
    group = hq // hkv
    pages = k_cache.shape[0] if num_pages is None else num_pages
    out, tol = np.zeros((rows, hq, dim)), np.zeros((rows, hq, dim))
    for b, length in enumerate(lens):
        n = indptr[b + 1] - indptr[b]
        if n == 0 or length == 0:
            continue
        tok = np.arange(length)
        at = table[b, tok // page]
        fine = (at >= 0) & (at < pages)
        at = np.where(fine, at, 0)
        k, v = k_cache[at, tok % page], v_cache[at, tok % page]
        if k_scale is not None:
            ks, vs = (k_scale[None], v_scale[None]) if k_scale.ndim == 1 else (k_scale[at], v_scale[at])
            k, v = k * ks[..., None], v * vs[..., None]
        for i in range(n):
            seen = fine & ((tok <= length - n + i) if causal else True)
            if not seen.any():
                continue
            for g in range(hkv):
                kk, vv = k[seen, g], v[seen, g]
                x = q[indptr[b] + i, g * group : (g + 1) * group]
                with np.errstate(invalid="ignore"):
                    s = scale * (x @ kk.T)
                    size = abs(scale) * (np.abs(x) @ np.abs(kk).T)
                    p = np.exp(s - s.max(axis=1, keepdims=True))
                    p /= p.sum(axis=1, keepdims=True)
                    row = indptr[b] + i, slice(g * group, (g + 1) * group)
                    out[row] = p @ vv
                    spread = p @ np.abs(vv)
                    off = 2 * (dim + 8) * 2.0**-24 * size.max(axis=1, keepdims=True) + (2.0**-13 if p_bits == 8 else 0.0)
                    tol[row] = (spread * (2.0**-p_bits + off + 2.0**-18 + len(kk) * 2.0**-24) * 1.01 + np.abs(out[row]) * 2.0**-bits * 1.01
                                + 2.0**-25)
    return out, tol


def reserve(table, lens, new, page, num_pages, parents=None):
    """(table, lens, served, [(source, destination)]) sequence by sequence."""
    width = table.shape[1]
    parents = range(len(lens)) if parents is None else parents
    rows = [(table[p], int(lens[p])) if 0 <= p < len(lens) else (None, 0) for p in parents]
    new = [max(0, int(n)) if r[0] is not None else 0 for n, r in zip(new, rows)]
    have = [-(-n // page) for _, n in rows]
    holders = {}
    for r, (entries, n) in enumerate(rows):
        for c in range(have[r]):
            holders.setdefault(int(entries[c]), []).append((r, new[r] > 0 and n % page != 0 and c == have[r] - 1))
    free = [p for p in range(num_pages) if p not in holders]
    out, got_lens, served, moves, taken = np.zeros((len(rows), width), np.int32), [], [], [], 0
    for r, (entries, n) in enumerate(rows):
        out[r, : have[r]] = entries[: have[r]] if have[r] else 0
        got_lens.append(n)
        if n + new[r] > width * page:
            served.append(False)
            continue
        copy = False
        if new[r] > 0 and n % page != 0:
            mine = holders[int(entries[have[r] - 1])]
            copy = not (all(w for _, w in mine) and mine[0][0] == r)
        grown = -(-(n + new[r]) // page) - have[r]
        need = copy + grown
        served.append(need == 0 or taken + need <= len(free))
        if served[-1]:
            pages = free[taken : taken + need]
            if copy:
                moves.append((int(entries[have[r] - 1]), pages[0]))
                out[r, have[r] - 1] = pages[0]
            out[r, have[r] : have[r] + grown] = pages[copy:]
        taken += need
    return out, np.array(got_lens, np.int32), np.array(served), moves


def compact(table, lens, page, num_pages):
    """(table, used, [(source, destination)])."""
    have = [-(-int(n) // page) for n in lens]
    names = {int(p) for r, n in enumerate(have) for p in table[r, :n]}
    held, used = sorted(names), len(names)
    free = [p for p in range(used) if p not in names]
    moves = dict(zip([p for p in held if p >= used], free))
    out = np.zeros_like(table)
    for r, n in enumerate(have):
        out[r, :n] = [moves.get(int(p), int(p)) for p in table[r, :n]]
    return out, used, list(moves.items())
