"""Cases of the 8-bit serving step: RMSNorm with an e4m3 output, the append into a cache held in 8 bits
with a scale for each page and KV head, decode attention over that cache, and decode attention over the
pages that a cheap score selects.

``own = False`` computes each operator from elementary torch operations in 32 bits; ``own = True`` calls
``kernel_lab.cuda_ops``. Both take the state of ``prepare`` and return the same outputs.
"""

from __future__ import annotations

import math
import os
import random
import sys

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
QMAX = {"e4m3": 448.0, "int8": 127.0}
BOUND_UNIT = {"e4m3": 4.0, "int8": 1.0}
TINY = 2.0**-126


def listed():
    return [
        # A decode step's rows before the projections of a wide layer: one scale a row, latency counts.
        norm("norm_rows16", 16, 8192, "bf16", True, 0),
        # A prompt's rows with a scale for each 128 columns, the operand of a block-scaled product.
        norm("norm_prompt4096", 4096, 8192, "bf16", True, 128),
        # A width that no power of two divides, no residual, a short last group.
        norm("norm_odd", 1000, 5000, "f16", False, 128),
        # One new token for each of 64 sequences (Llama-3-8B heads).
        append("append_tokens64", "e4m3", "bf16", 64, 1, 1, 4096, 8, 128, 16, "nhd", True),
        # Prompts of ragged length written in one call.
        append("append_prompts", "e4m3", "bf16", 16, 300, 4096, 2000, 8, 128, 16, "nhd", True),
        # Chunks of prompts into int8 pages of 64 tokens, many heads of 64, no bounds.
        append("append_int8_chunks", "int8", "f16", 37, 1, 257, 1000, 32, 64, 64, "hnd", False),
        # The smallest decode call.
        decode("decode_b1_ctx512", "e4m3", "bf16", 1, 512, 512, 32, 8, 128, 16, "nhd"),
        # The headline geometry, batch 64 x 4096 tokens.
        decode("decode_b64_ctx4096", "e4m3", "bf16", 64, 4096, 4096, 32, 8, 128, 16, "nhd"),
        # Ragged lengths, one KV head for 32 query heads, int8 pages of 32 tokens.
        decode("decode_ragged_mqa", "int8", "f16", 128, 1, 16384, 32, 1, 128, 32, "nhd"),
        # Llama-3-70B heads at a serving batch.
        decode("decode_b128_ctx8192", "e4m3", "bf16", 128, 8192, 8192, 64, 8, 128, 16, "nhd"),
        # One long conversation, an eighth of its pages read.
        sparse("sparse_b1_ctx32768", "e4m3", "bf16", 1, 32768, 32768, 32, 8, 128, 16, "hnd", 256),
        # A ragged batch of long contexts, 128 pages of each read.
        sparse("sparse_b64_ragged", "e4m3", "bf16", 64, 1000, 16384, 32, 8, 128, 16, "hnd", 128),
    ]


def norm(name, rows, hidden, dtype, residual, group):
    return {"name": name, "op": "norm", "rows": rows, "hidden": hidden, "dtype": dtype, "residual": residual, "group": group}


def append(name, codes, dtype, batch, lo, hi, start, hkv, dim, page, layout, bounds):
    return {"name": name, "op": "append", "codes": codes, "dtype": dtype, "batch": batch, "new_min": lo, "new_max": hi,
            "start_max": start, "hkv": hkv, "dim": dim, "page": page, "layout": layout, "bounds": bounds}


def decode(name, codes, dtype, batch, lo, hi, hq, hkv, dim, page, layout):
    return {"name": name, "op": "decode", "codes": codes, "dtype": dtype, "batch": batch, "len_min": lo, "len_max": hi,
            "hq": hq, "hkv": hkv, "dim": dim, "page": page, "layout": layout}


def sparse(name, codes, dtype, batch, lo, hi, hq, hkv, dim, page, layout, pages):
    return decode(name, codes, dtype, batch, lo, hi, hq, hkv, dim, page, layout) | {"op": "sparse", "pages": pages}


def spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["norm", "append", "decode", "sparse"])
    dtype = rng.choice(["f16", "bf16"])
    if op == "norm":
        hidden = spread(rng, 512, 8192)
        hidden += 8 - hidden % 8 if rng.random() < 0.8 else 0
        case = norm("", spread(rng, 1, 4096), min(hidden, 8192), rng.choice(["f32", "f16", "bf16"]), rng.random() < 0.7,
                    rng.choice([0, 64, 128]))
    else:
        codes, layout = rng.choice(["e4m3", "int8"]), rng.choice(["nhd", "hnd"])
        page = rng.choice([8, 16, 16, 32, 64])
        hkv, dim, group = rng.choice([(8, 128, 4), (8, 128, 8), (1, 128, 32), (32, 64, 1), (4, 256, 2), (8, 128, 7), (2, 96, 5)])
        if op == "append":
            batch = spread(rng, 1, 64)
            most = spread(rng, 1, max(1, 24000 // batch))
            case = append("", codes, dtype, batch, rng.choice([1, most]), most, spread(rng, 1, 4096), hkv, dim, page,
                          layout, rng.random() < 0.6)
        else:
            # At most as many tokens of KV as 128 x 8192 of 8 heads of 128.
            batch = spread(rng, 1, 128)
            most = spread(rng, 1, min(32768, (128 * 8192 * 8 * 128 // 2) // (batch * hkv * dim)))
            lo = rng.choice([1, most])
            args = ("", codes, dtype, batch, lo, most, hkv * group, hkv, dim, page, layout)
            case = decode(*args) if op == "decode" else sparse(*args, spread(rng, 2, 256))
    del case["name"]
    return case


def whole_numbers(case, key, seed):
    """The case's lengths: uniform between its bounds, one at each bound; the same ones in another order for each seed."""
    lo, hi = case[key + "_min"], case[key + "_max"]
    r = random.Random(repr((lo, hi, case["batch"])))
    got = [r.randint(lo, hi) for _ in range(case["batch"])]
    got[0] = hi
    if case["batch"] > 1:
        got[-1] = lo
    random.Random(seed).shuffle(got)
    return got


def starts(case, seed):
    r = random.Random(repr((seed, "start")))
    return [r.randint(0, case["start_max"]) for _ in range(case["batch"])]


def pool_tables(needed, total, seed, device):
    """Shuffled pages of a pool of `total` for sequences that need so many each: (pages of the pool, block table)."""
    order = torch.from_numpy(np.random.RandomState(seed % 2**31).permutation(total).astype(np.int32))
    table = torch.zeros(len(needed), max(1, max(needed)), dtype=torch.int32)
    at = 0
    for b, n in enumerate(needed):
        table[b, :n] = order[at : at + n]
        at += n
    return total, table.to(device)


def empty_pool(case, total, dtype, device):
    """A pool [pages, page, kv heads, dim], stored in that order ("nhd") or head by head within a page ("hnd")."""
    p, h, d = case["page"], case["hkv"], case["dim"]
    if case["layout"] == "hnd":
        return torch.empty(total, h, p, d, dtype=dtype, device=device).permute(0, 2, 1, 3)
    return torch.empty(total, p, h, d, dtype=dtype, device=device)


def filled_pool(case, total, gen, device, drift):
    """Codes, scales and key bounds of a pool whose tokens are normal, with channels of unlike size and a drift of each page."""
    p, h, d = case["page"], case["hkv"], case["dim"]
    codes = empty_pool(case, total, CODES[case["codes"]], device)
    scale = torch.empty(total, h, device=device)
    bounds = torch.empty(total, h, 2, d, dtype=torch.int8, device=device)
    channel = torch.exp(0.5 * torch.randn(h, d, generator=gen, device=device))
    step = max(1, (1 << 26) // (p * h * d))
    for a in range(0, total, step):
        z = min(total, a + step)
        x = torch.randn(z - a, p, h, d, generator=gen, device=device)
        x += drift * torch.randn(z - a, 1, h, d, generator=gen, device=device)
        x *= channel
        s = scale_for(x.abs().amax(dim=(1, 3)), case["codes"])
        q = to_codes(x * inverse(s)[:, None, :, None], case["codes"])
        codes[a:z] = q
        scale[a:z] = s
        bounds[a:z] = bounds_of(q.float(), case["codes"])
    return codes, scale, bounds


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    if own:
        use_package()
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "norm":
        rows, hidden = case["rows"], case["hidden"]
        x = torch.randn(rows, hidden, generator=gen, device=device).to(dtype)
        r = (2 * torch.randn(rows, hidden, generator=gen, device=device)).to(dtype) if case["residual"] else None
        w = (1 + 0.1 * torch.randn(hidden, generator=gen, device=device)).to(dtype)
        return {"op": "norm", "x": x, "residual": r, "weight": w, "eps": 1e-5, "group": case["group"]}
    if case["op"] == "append":
        new, start = whole_numbers(case, "new", seed), starts(case, seed)
        room = sum(-(-(case["start_max"] + n) // case["page"]) for n in new) + 3
        total, table = pool_tables([-(-(s + n) // case["page"]) for s, n in zip(start, new)], room, seed, device)
        kc, ks, kb = filled_pool(case, total, gen, device, 0.0)
        vc, vs, _ = filled_pool(case, total, gen, device, 0.0)
        # New rows are views of a fused projection's output, as a layer has them.
        rows = sum(new)
        width = case["hkv"] * case["dim"]
        qkv = torch.randn(rows, 2 * width, generator=gen, device=device).mul_(1.5).to(dtype)
        indptr = None
        if case["new_max"] > 1:
            indptr = torch.tensor([0, *np.cumsum(new).tolist()], dtype=torch.int32, device=device)
        return {"op": "append", "codes": case["codes"], "k_cache": kc, "v_cache": vc, "k_scale": ks, "v_scale": vs,
                "k_bounds": kb if case["bounds"] else None, "k_new": qkv[:, :width], "v_new": qkv[:, width:],
                "block_table": table, "positions": torch.tensor(start, dtype=torch.int32, device=device), "indptr": indptr}
    lens = whole_numbers(case, "len", seed)
    needed = [-(-n // case["page"]) for n in lens]
    total, table = pool_tables(needed, sum(needed) + 3, seed, device)
    drift = 0.5 if case["op"] == "sparse" else 0.0
    kc, ks, kb = filled_pool(case, total, gen, device, drift)
    vc, vs, _ = filled_pool(case, total, gen, device, 0.0)
    q = torch.randn(case["batch"], case["hq"], case["dim"], generator=gen, device=device).to(dtype)
    state = {"op": case["op"], "codes": case["codes"], "q": q, "k_cache": kc, "v_cache": vc, "k_scale": ks, "v_scale": vs,
             "block_table": table, "seq_lens": torch.tensor(lens, dtype=torch.int32, device=device)}
    if case["op"] == "sparse":
        state |= {"k_bounds": kb, "pages": case["pages"]}
    return state


def use_package():
    path = os.path.join(os.getcwd(), "kernel-lab_b200")
    if path not in sys.path:
        sys.path.insert(0, path)


def run(state):
    return run_own(state) if own else run_plain(state)


def run_own(s):
    from kernel_lab import cuda_ops

    if s["op"] == "norm":
        if s["residual"] is None:
            codes, scales = cuda_ops.rms_norm_fp8(s["x"], s["weight"], s["eps"], group_size=s["group"])
            return {"codes": codes, "scales": scales}
        codes, scales, residual = cuda_ops.fused_add_rms_norm_fp8(s["x"], s["residual"], s["weight"], s["eps"], group_size=s["group"])
        return {"codes": codes, "scales": scales, "residual": residual}
    if s["op"] == "append":
        cuda_ops.paged_kv_append_block8(s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["k_new"], s["v_new"],
                                        s["block_table"], s["positions"], indptr=s["indptr"], k_bounds=s["k_bounds"])
        return updated(s)
    chosen = None
    if s["op"] == "sparse":
        chosen = cuda_ops.paged_block_select(s["q"], s["k_cache"], s["k_scale"], s["k_bounds"], s["block_table"],
                                             s["seq_lens"], s["pages"])
    out = cuda_ops.paged_decode_attention_block8(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"],
                                                 s["block_table"], s["seq_lens"], selected=chosen)
    return {"out": out} if chosen is None else {"out": out, "selected": chosen}


def updated(s):
    got = {name: s[name] for name in ("k_cache", "v_cache", "k_scale", "v_scale")}
    return got if s["k_bounds"] is None else got | {"k_bounds": s["k_bounds"]}


# ------------------------------------------------------------------ plain forms


def scale_for(amax, codes):
    """The scale that a block of this largest magnitude needs: amax / 127 for int8, for e4m3 the smallest power of two
    (at least 2^-126) that brings it to at most 448 = 0.875 * 2^9."""
    if codes == "int8":
        s = (amax / 127.0).clamp_min(TINY)
    else:
        f, e = torch.frexp(amax)
        k = torch.where(f <= 0.875, e - 9, e - 8).clamp_min(-126)
        s = ((k + 127) << 23).to(torch.int32).view(torch.float32)
    return torch.where(amax > 0, s, torch.zeros_like(s))


def inverse(scale):
    return torch.where(scale >= TINY, 1.0 / scale, torch.zeros_like(scale))


def to_codes(x, codes):
    if codes == "int8":
        return torch.nan_to_num(x, nan=0.0).round().clamp(-127, 127).to(torch.int8)
    return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)


def raw(t):
    """The codes as bytes: what indexing moves."""
    return t.view(torch.uint8) if t.dtype is torch.float8_e4m3fn else t


def values(t, codes):
    return (t.view(torch.float8_e4m3fn) if codes == "e4m3" else t).float()


def bounds_of(v, codes):
    """Per page, head and channel the least and largest value of [pages, tokens, heads, dim], in whole units, outward."""
    v = torch.nan_to_num(v, nan=0.0) / BOUND_UNIT[codes]
    return torch.stack([v.amin(dim=1).floor(), v.amax(dim=1).ceil()], dim=2).to(torch.int8)


def run_plain(s):
    return {"norm": plain_norm, "append": plain_append, "decode": plain_decode, "sparse": plain_sparse}[s["op"]](s)


def plain_norm(s):
    x, dtype = s["x"].float(), s["x"].dtype
    out = {}
    if s["residual"] is not None:
        out["residual"] = (x + s["residual"].float()).to(dtype)
        x = out["residual"].float()
    rows, hidden = x.shape
    y = x * (1.0 / torch.sqrt(x.square().mean(dim=-1, keepdim=True) + s["eps"])) * s["weight"].float()
    group = s["group"] or hidden
    groups = -(-hidden // group)
    y = torch.nn.functional.pad(y, (0, groups * group - hidden)).view(rows, groups, group)
    amax = torch.nan_to_num(y.abs(), nan=0.0, posinf=math.inf).amax(dim=-1)
    some = amax >= 2.0**-100
    inv = torch.where(some, 448.0 / amax, torch.zeros_like(amax))
    codes = to_codes(y * inv[..., None], "e4m3").view(rows, groups * group)[:, :hidden]
    return out | {"codes": codes.contiguous(), "scales": torch.where(some, amax / 448.0, torch.zeros_like(amax))}


def plain_append(s):
    table, start, codes = s["block_table"].long(), s["positions"].long(), s["codes"]
    pages, page, heads, dim = s["k_cache"].shape
    batch, rows = start.numel(), s["k_new"].shape[0]
    indptr = torch.arange(batch + 1, device=start.device) if s["indptr"] is None else s["indptr"].long()
    count = indptr[1:] - indptr[:-1]
    # The pages that the call touches, in order, in a list of fixed length; places past its end repeat the first.
    touched = torch.where(count > 0, (start + count - 1) // page - start // page + 1, 0)
    ends = touched.cumsum(0)
    u = torch.arange(rows // page + 2 * batch, device=start.device)
    u = torch.where(u < ends[-1], u, 0)
    b = torch.searchsorted(ends, u, right=True)
    col = start[b] // page + u - (ends - touched)[b]
    slot = torch.arange(page, device=start.device)
    pos = col[:, None] * page + slot
    token = indptr[b][:, None] + pos - start[b][:, None]
    kept = (pos < start[b][:, None])[..., None, None]
    fresh = ((pos >= start[b][:, None]) & (token < indptr[b + 1][:, None]))[..., None, None]
    at, token = table[b, col], token.clamp(0, rows - 1)
    for name in ("k", "v"):
        cache, scale = s[name + "_cache"], s[name + "_scale"]
        x = s[name + "_new"][token].float().view(*token.shape, heads, dim)
        old_codes = raw(cache)[at]
        amax = torch.where(fresh & torch.isfinite(x), x.abs(), 0.0).amax(dim=(1, 3))
        old = torch.where(kept[:, 0, 0], scale[at], 0.0)
        new = torch.maximum(old, scale_for(amax, codes))
        ratio = torch.where(new > old, old / new, 1.0)
        again = raw(to_codes(values(old_codes, codes) * ratio[:, None, :, None], codes))
        made = raw(to_codes(x * inverse(new)[:, None, :, None], codes))
        put = torch.where(fresh, made, torch.where(kept, again, old_codes))
        raw(cache)[at] = put
        scale[at] = new
        if name == "k" and s["k_bounds"] is not None:
            v = torch.nan_to_num(values(put, codes), nan=0.0) / BOUND_UNIT[codes]
            there = kept | fresh
            lo = torch.where(there, v, math.inf).amin(dim=1).floor()
            hi = torch.where(there, v, -math.inf).amax(dim=1).ceil()
            s["k_bounds"][at] = torch.stack([lo, hi], dim=2).to(torch.int8)
    return updated(s)


def plain_attention(s, chosen):
    """Decode attention over the pages `chosen` [batch, kv heads, n] of each sequence (-1: none)."""
    q, codes, lens = s["q"], s["codes"], s["seq_lens"].long()
    page, heads, dim = s["k_cache"].shape[1:]
    batch, hq, _ = q.shape
    n = chosen.shape[2]
    at = torch.gather(s["block_table"].long()[:, None, :].expand(-1, heads, -1), 2, chosen.clamp_min(0))
    h = torch.arange(heads, device=q.device)[None, :, None]
    pos = chosen[..., None] * page + torch.arange(page, device=q.device)
    there = ((chosen[..., None] >= 0) & (pos < lens[:, None, None, None])).view(batch, heads, 1, n * page)
    k = values(raw(s["k_cache"])[at, :, h], codes) * s["k_scale"][at, h][..., None, None]
    score = q.float().view(batch, heads, hq // heads, dim) @ k.view(batch, heads, n * page, dim).transpose(2, 3)
    del k
    score = torch.where(there, score * dim**-0.5, -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    p = torch.exp(score - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(dim=-1, keepdim=True)
    v = values(raw(s["v_cache"])[at, :, h], codes) * s["v_scale"][at, h][..., None, None]
    v = torch.where(there[:, :, 0, :, None], v.view(batch, heads, n * page, dim), 0.0)
    out = (p @ v) / torch.where(total > 0, total, 1.0)
    return out.view(batch, hq, dim).to(q.dtype)


def plain_decode(s):
    width = torch.arange(s["block_table"].shape[1], device=s["q"].device)
    return {"out": plain_attention(s, width.expand(s["q"].shape[0], s["k_cache"].shape[2], -1))}


def plain_sparse(s):
    q, codes, heads, page = s["q"].float(), s["codes"], s["k_cache"].shape[2], s["k_cache"].shape[1]
    batch, hq, dim = q.shape
    width, want = s["block_table"].shape[1], s["pages"]
    count = (s["seq_lens"].long() + page - 1) // page
    amax = torch.where(torch.isfinite(q), q.abs(), 0.0).amax(dim=-1, keepdim=True)
    sq = amax / 127.0
    qi = torch.nan_to_num(q * inverse(sq), nan=0.0).round().clamp(-127, 127).view(batch, heads, hq // heads, dim)
    at = s["block_table"].long()
    b = s["k_bounds"][at].float()  # [batch, pages, heads, 2, dim]; whole numbers, products and sums below 2^24: exact
    low, high = b[..., 0, :].permute(0, 2, 3, 1), b[..., 1, :].permute(0, 2, 3, 1)
    dots = qi.clamp_max(0.0) @ low + qi.clamp_min(0.0) @ high
    best = (dots * sq.view(batch, heads, -1, 1)).amax(dim=2)
    score = best * (s["k_scale"][at] * BOUND_UNIT[codes]).transpose(1, 2)
    col = torch.arange(width, device=q.device)
    always = (col < 1) | (col >= count[:, None] - 1)  # the first page and the last
    score = torch.where(always[:, None], math.inf, score)
    score = torch.where((col < count[:, None])[:, None], score, -math.inf)
    picked = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :want]
    picked = torch.where(picked < count[:, None, None], picked, width).sort(dim=-1).values
    picked = torch.nn.functional.pad(picked, (0, want - picked.shape[2]), value=width)
    chosen = torch.where(picked < width, picked, -1)
    return {"out": plain_attention(s, chosen), "selected": chosen.to(torch.int32)}


# ------------------------------------------------------------------ work


def work(case):
    if case["op"] == "norm":
        rows, hidden, e = case["rows"], case["hidden"], DTYPES[case["dtype"]].itemsize
        groups = -(-hidden // (case["group"] or hidden))
        n = rows * hidden
        return {"bytes": n * (e * (3 if case["residual"] else 1) + 1) + hidden * e + 4 * rows * groups, "flops": 8 * n}
    h, d, page = case["hkv"], case["dim"], case["page"]
    seed = 0
    if case["op"] == "append":
        new, start = whole_numbers(case, "new", seed), starts(case, seed)
        touched = sum((s + n - 1) // page - s // page + 1 for s, n in zip(start, new))
        kept = sum(s % page for s in start)
        rows = sum(new)
        # New rows in, their codes and the pages' scales out; bounds: the kept keys in, the bounds out.
        size = 2 * rows * h * d * (DTYPES[case["dtype"]].itemsize + 1) + touched * h * 8
        size += (kept * h * d + touched * h * 2 * d) if case["bounds"] else 0
        return {"bytes": size, "flops": 4 * rows * h * d}
    lens = whole_numbers(case, "len", seed)
    pages = [-(-n // page) for n in lens]
    size = 2 * case["batch"] * case["hq"] * d * 2
    if case["op"] == "decode":
        size += 2 * sum(lens) * h * d + sum(pages) * (8 * h + 4)
        return {"bytes": size, "flops": 4 * sum(lens) * case["hq"] * d}
    read = sum(min(n, case["pages"] * page) for n in lens)
    kept = sum(min(n, case["pages"]) for n in pages)
    size += sum(pages) * (h * (2 * d + 4) + 4)
    size += 2 * read * h * d + kept * h * 8 + case["batch"] * h * case["pages"] * 4
    return {"bytes": size, "flops": 4 * read * case["hq"] * d + 4 * sum(pages) * case["hq"] * d}


# ------------------------------------------------------------------ 64 bits


def e4m3_64(v):
    """64-bit numbers rounded to the nearest e4m3 value (ties to even), saturated."""
    exponent = torch.frexp(v).exponent.clamp_min(-5).double()  # |v| in [2^(e-1), 2^e); subnormal below 2^-6
    unit = torch.pow(2.0, exponent - 4)
    return (torch.round(v / unit) * unit).clamp(-448, 448)


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": exact_norm, "append": exact_append, "decode": exact_attention, "sparse": exact_sparse}[case["op"]](s)


def exact_norm(s):
    x, w = s["x"].double(), s["weight"].double()
    got = {}
    if s["residual"] is not None:
        x = (x + s["residual"].double()).float().to(s["x"].dtype).double()
        got["residual"] = x
    y = x * torch.rsqrt(x.square().mean(dim=1, keepdim=True) + s["eps"]) * w
    hidden = y.shape[1]
    group = s["group"] or hidden
    codes, scales = torch.empty_like(y), []
    for a in range(0, hidden, group):
        part = y[:, a : a + group]
        top = part.abs().amax(dim=1, keepdim=True)
        scales.append(top / 448)
        codes[:, a : a + group] = e4m3_64(part * (448 / top))
    return got | {"codes": codes, "scales": torch.cat(scales, dim=1)}


def exact_append(s):
    """Page by page. Whole numbers (int8 codes, bounds) have no 64-bit value of their own."""
    if s["codes"] == "int8":
        return {name: None for name in ("k_cache", "v_cache")} | exact_scales(s)
    start = s["positions"].tolist()
    ptr = list(range(len(start) + 1)) if s["indptr"] is None else s["indptr"].tolist()
    table, page = s["block_table"].cpu(), s["k_cache"].shape[1]
    got = {"k_bounds": None} if s["k_bounds"] is not None else {}
    for name in ("k", "v"):
        cache, scale = s[name + "_cache"].double(), s[name + "_scale"].double()
        new = s[name + "_new"].double().view(-1, *cache.shape[2:])
        for b, at in enumerate(start):
            done = 0
            while done < ptr[b + 1] - ptr[b]:
                pos = at + done
                p, slot = int(table[b, pos // page]), pos % page
                n = min(page - slot, ptr[b + 1] - ptr[b] - done)
                x = new[ptr[b] + done : ptr[b] + done + n]
                f, e = torch.frexp(x.abs().amax(dim=(0, 2)) / 448)
                need = torch.pow(2.0, (e - (f == 0.5).int()).double())
                if slot:
                    need = torch.maximum(need, scale[p])
                    cache[p, :slot] = e4m3_64(cache[p, :slot] * (scale[p] / need)[:, None])
                scale[p] = need
                cache[p, slot : slot + n] = e4m3_64(x / need[:, None])
                done += n
        got |= {name + "_cache": cache, name + "_scale": scale}
    return got


def exact_scales(s):
    start = s["positions"].tolist()
    ptr = list(range(len(start) + 1)) if s["indptr"] is None else s["indptr"].tolist()
    table, page = s["block_table"].cpu(), s["k_cache"].shape[1]
    got = {"k_bounds": None} if s["k_bounds"] is not None else {}
    for name in ("k", "v"):
        scale = s[name + "_scale"].double()
        new = s[name + "_new"].double().view(-1, *s["k_cache"].shape[2:])
        for b, at in enumerate(start):
            done = 0
            while done < ptr[b + 1] - ptr[b]:
                pos = at + done
                p, slot = int(table[b, pos // page]), pos % page
                n = min(page - slot, ptr[b + 1] - ptr[b] - done)
                need = new[ptr[b] + done : ptr[b] + done + n].abs().amax(dim=(0, 2)) / 127
                scale[p] = torch.maximum(need, scale[p]) if slot else need
                done += n
        got[name + "_scale"] = scale
    return got


def exact_attention(s, chosen=None):
    q, lens = s["q"].double(), s["seq_lens"].tolist()
    page, heads, dim = s["k_cache"].shape[1:]
    group = q.shape[1] // heads
    out = torch.zeros_like(q)
    codes = {name: (raw(s[name + "_cache"]), s[name + "_scale"].double()) for name in ("k", "v")}
    for b, n in enumerate(lens):
        for h in range(heads):
            cols = torch.arange(-(-n // page), device=q.device) if chosen is None else chosen[b][h]
            if not cols.numel():
                continue
            at = s["block_table"][b].long()[cols]
            there = (cols[:, None] * page + torch.arange(page, device=q.device) < n).view(-1)
            k, v = ((values(c[at, :, h], s["codes"]).double() * sc[at, h][:, None, None]).view(-1, dim)[there] for c, sc in codes.values())
            rows = slice(h * group, (h + 1) * group)
            out[b, rows] = torch.softmax(q[b, rows] @ k.T / math.sqrt(dim), dim=-1) @ v
    return {"out": out}


def exact_sparse(s):
    """The choice by whole numbers and the score's two roundings to 32 bits, which define it."""
    q = s["q"].cpu().double().numpy()
    lens, table = s["seq_lens"].tolist(), s["block_table"].cpu().numpy()
    page, heads, _ = s["k_cache"].shape[1:]
    group = q.shape[1] // heads
    unit = np.float32(BOUND_UNIT[s["codes"]])
    bounds, scale = s["k_bounds"].cpu().numpy(), s["k_scale"].cpu().numpy()
    chosen = []
    for b, n in enumerate(lens):
        count = -(-n // page)
        sq = (np.abs(q[b]).max(axis=1).astype(np.float32) / np.float32(127)).astype(np.float32)
        inv = (np.float32(1) / sq).astype(np.float32)
        qi = np.clip(np.rint(q[b].astype(np.float32) * inv[:, None]), -127, 127).astype(np.float64)
        at = table[b, :count]
        chosen.append([])
        for h in range(heads):
            rows = slice(h * group, (h + 1) * group)
            lo, hi = bounds[at, h, 0].astype(np.float64), bounds[at, h, 1].astype(np.float64)
            dots = np.minimum(qi[rows], 0) @ lo.T + np.maximum(qi[rows], 0) @ hi.T
            score = (dots.astype(np.float32) * sq[rows, None]).max(axis=0) * (scale[at, h] * unit)
            score[0] = score[-1] = np.inf
            best = np.sort(np.argsort(-score, kind="stable")[: s["pages"]])
            chosen[-1].append(torch.from_numpy(best).to(s["q"].device))
    return exact_attention(s, chosen) | {"selected": None}
