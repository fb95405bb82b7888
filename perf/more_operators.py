"""Cases of a chunked step over a paged cache: the append of chunks of new tokens, attention of those tokens over the
cache (in 32 and 16 bits, in e4m3 with a scale for each KV head, in 8 bits with a scale for each page and KV head), and
the pages themselves: copied, given to growing and forked sequences, and compacted.

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

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
FAR = 1 << 30


def listed():
    return [
        # Draft tokens of eight short conversations verified in one step: the smallest call, latency counts.
        attend("attend_verify", "same", "bf16", "bf16", 8, 4, 4, 1, 1024, 32, 8, 128, 16, True),
        # A prompt's tokens over itself, Llama-3-8B heads: the largest.
        attend("attend_prompt8192", "same", "bf16", "bf16", 1, 8192, 8192, 0, 0, 32, 8, 128, 16, True),
        # A continuous batch: single tokens beside chunks of prompts over contexts of any length, seven query heads a KV head.
        attend("attend_mixed", "same", "f16", "f16", 32, 1, 256, 0, 8000, 28, 4, 128, 32, True),
        # Chunks of eight long prompts over the block-scaled cache, Llama-3-70B heads, pages stored head by head.
        attend("attend_block8", "block8", "bf16", "e4m3", 8, 512, 512, 1000, 7680, 64, 8, 128, 16, True),
        # Chunks of a few tokens, rows of a fused projection (Llama-3-8B heads).
        append("append_drafts", "bf16", "bf16", 64, 1, 8, 4096, 8, 128, 16),
        # Prompts of ragged length into the e4m3 cache.
        append("append_prompts_e4m3", "bf16", "e4m3", 16, 300, 4096, 2000, 8, 128, 16),
        # The pages that a few sequences are about to write and share with others.
        copy("copy_few", 2, 12, 512, 16, 8, 128, "bf16"),
        # A stored prefix brought into a model's 24 layers.
        copy("copy_layers", 48, 250, 1000, 16, 8, 128, "bf16"),
        # A decode step: one more token for each of 256 sequences, a few of which need a page.
        reserve("reserve_step", 256, 0, 1, 1, 1, 8192, 514, 90000, 16, 2, 64),
        # Eight samples of each of 64 prompts begin: shared pages, a copy of each last one, room for a chunk.
        reserve("reserve_fork", 64, 512, 1, 40, 500, 3000, 256, 16000, 16, 8, 128),
        # A small pool after most sequences have ended.
        compact("compact_few", 16, 1, 500, 64, 3001, 16, 8, 128),
        # A large pool, two fifths of it in use.
        compact("compact_pool", 128, 100, 3000, 256, 25000, 16, 8, 128),
    ]


def attend(name, kind, dtype, codes, batch, lo, hi, ctx_lo, ctx_hi, hq, hkv, dim, page, causal):
    return {"name": name, "op": "attend", "kind": kind, "dtype": dtype, "codes": codes, "batch": batch, "new_min": lo, "new_max": hi,
            "ctx_min": ctx_lo, "ctx_max": ctx_hi, "hq": hq, "hkv": hkv, "dim": dim, "page": page, "causal": causal}


def append(name, dtype, codes, batch, lo, hi, start, hkv, dim, page):
    return {"name": name, "op": "append", "dtype": dtype, "codes": codes, "batch": batch, "new_min": lo, "new_max": hi,
            "ctx_min": 0, "ctx_max": start, "hkv": hkv, "dim": dim, "page": page}


def copy(name, tensors, pairs, pages, page, hkv, dim, dtype):
    return {"name": name, "op": "copy", "tensors": tensors, "pairs": pairs, "pages": pages, "page": page, "hkv": hkv, "dim": dim,
            "dtype": dtype}


def reserve(name, batch, forks, lo, hi, ctx_lo, ctx_hi, width, pages, page, hkv, dim):
    return {"name": name, "op": "reserve", "batch": batch, "forks": forks, "new_min": lo, "new_max": hi, "ctx_min": ctx_lo,
            "ctx_max": ctx_hi, "width": width, "pages": pages, "page": page, "hkv": hkv, "dim": dim, "dtype": "bf16"}


def compact(name, batch, ctx_lo, ctx_hi, width, pages, page, hkv, dim):
    return {"name": name, "op": "compact", "batch": batch, "ctx_min": ctx_lo, "ctx_max": ctx_hi, "width": width, "pages": pages,
            "page": page, "hkv": hkv, "dim": dim, "dtype": "bf16"}


def spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "append", "copy", "reserve", "compact"])
    dtype = rng.choice(["f16", "bf16"])
    page = rng.choice([8, 16, 16, 32, 64])
    if op == "attend":
        kind = rng.choice(["same", "same", "same", "e4m3", "block8"])
        hkv, dim, group = rng.choice([(8, 128, 4), (8, 128, 8), (1, 128, 32), (32, 64, 1), (4, 128, 7), (2, 96, 5), (4, 64, 6), (4, 256, 2)])
        codes = dtype if kind == "same" else "e4m3" if kind == "e4m3" else rng.choice(["e4m3", "int8"])
        seen = 180 * 10**9 // dim  # pairs of a query head and a key in all
        if kind == "same" and rng.random() < 0.15:
            dtype = codes = "f32"
            seen = 1 << 26
        batch = spread(rng, 1, 64)
        each = max(1, seen // (batch * hkv * group))
        new = spread(rng, 1, min(4096, math.isqrt(each)))
        ctx = spread(rng, 1, max(1, min(32768, each // new - new, (1 << 29) // (batch * hkv * dim) - new)))
        case = attend("", kind, dtype, codes, batch, rng.choice([1, new]), new, rng.choice([0, ctx]), ctx, hkv * group, hkv, dim,
                      page, rng.random() < 0.85)
    elif op == "append":
        hkv, dim = rng.choice([(8, 128), (1, 128), (32, 64), (4, 256), (2, 96), (3, 80)])
        batch = spread(rng, 1, 64)
        most = spread(rng, 1, max(1, 32000 // batch))
        codes = rng.choice([dtype, dtype, "e4m3"])
        case = append("", dtype, codes, batch, rng.choice([1, most]), most, spread(rng, 1, 4096), hkv, dim, page)
    elif op == "copy":
        hkv, dim = rng.choice([(8, 128), (1, 128), (32, 64), (3, 80)])
        pairs, tensors = spread(rng, 1, 400), rng.choice([1, 2, 2, 16, 48])
        case = copy("", tensors, pairs, 2 * pairs + spread(rng, 1, 200), page, hkv, dim, rng.choice(["f32", "bf16", "int8"]))
        while tensors * case["pages"] * page * hkv * dim * DTYPES[case["dtype"]].itemsize > 3 << 30:
            tensors = case["tensors"] = tensors // 2
    else:
        hkv, dim = rng.choice([(8, 128), (2, 64), (1, 128)])
        batch, longest = spread(rng, 1, 300), spread(rng, 16, 8192)
        longest = min(longest, max(16, (1 << 20) // batch))
        width = longest // page + spread(rng, 2, 64)
        # Enough pages, now and then too few for every sequence's growth.
        pages = batch * (longest // page + 1) + spread(rng, 1, 20000)
        while pages * page * hkv * dim * 2 > 2 << 30:
            hkv, dim, page = (1, dim, page) if hkv > 1 else (1, dim // 2, page)
        if op == "reserve":
            forks = rng.choice([0, spread(rng, 1, 300)])
            case = reserve("", batch, forks, rng.choice([0, 1]), rng.choice([1, page, 4 * page]), 1, longest, width, pages, page, hkv, dim)
        else:
            case = compact("", batch, 1, longest, width, pages, page, hkv, dim)
    del case["name"]
    return case


def whole_numbers(case, key, seed):
    """The case's lengths: uniform between its bounds, one at each bound; the same ones in another order for each seed."""
    lo, hi = case[key + "_min"], case[key + "_max"]
    r = random.Random(repr((key, lo, hi, case["batch"])))
    got = [r.randint(lo, hi) for _ in range(case["batch"])]
    got[0] = hi
    if case["batch"] > 1:
        got[-1] = lo
    random.Random(repr((key, seed))).shuffle(got)
    return got


def pages_of(tokens, page):
    return -(-tokens // page)


def tables(needed, total, width, seed):
    """A block table of shuffled pages of a pool of `total`, for sequences that need so many each."""
    order = torch.from_numpy(np.random.RandomState(seed % 2**31).permutation(total).astype(np.int32))
    table = torch.zeros(len(needed), max(1, width), dtype=torch.int32)
    at = 0
    for b, n in enumerate(needed):
        table[b, :n] = order[at : at + n]
        at += n
    return table.cuda()


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def ptr_of(counts):
    return ints([0, *np.cumsum(counts).tolist()])


def filled(shape, dtype, gen):
    """Normal values; 8-bit ones are codes over most of their range."""
    t = torch.empty(shape, dtype=dtype, device="cuda")
    rows = t.view(shape[0], -1)
    step = max(1, (1 << 26) // rows.shape[1])
    for a in range(0, shape[0], step):
        x = torch.randn(rows[a : a + step].shape, generator=gen, device="cuda")
        rows[a : a + step] = (x * 40).round().clamp(-127, 127) if dtype is torch.int8 else (x * 60).clamp(-448, 448) if dtype is torch.float8_e4m3fn else x
    return t


def bits(shape, dtype, gen):
    """A pool whose contents are only moved: any bytes."""
    size = math.prod(shape) * dtype.itemsize
    words = torch.randint(-(2**62), 2**62, (pages_of(size, 8),), generator=gen, device="cuda", dtype=torch.int64)
    return words.view(torch.uint8)[:size].view(dtype).view(shape)


def scales(shape, codes, gen):
    """Scales that bring the codes back to values of about one, a page's unlike another's."""
    size = torch.exp(0.3 * torch.randn(shape, generator=gen, device="cuda")) / (60 if codes == "e4m3" else 40)
    return torch.exp2(torch.log2(size).round()) if codes == "e4m3" and len(shape) > 1 else size


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if own:
        use_package()
    op, page, h, d = case["op"], case["page"], case["hkv"], case["dim"]
    dtype = DTYPES[case["dtype"]]
    if op == "copy":
        order = np.random.RandomState(seed % 2**31).permutation(case["pages"])
        caches = [bits((case["pages"], page, h, d), dtype, gen) for _ in range(case["tensors"])]
        n = case["pairs"]
        return {"op": op, "caches": caches, "src": ints(order[:n].tolist()), "dst": ints(order[n : 2 * n].tolist())}
    if op in ("reserve", "compact"):
        lens = whole_numbers(case, "ctx", seed)
        table = tables([pages_of(n, page) for n in lens], case["pages"], case["width"], seed)
        caches = [bits((case["pages"], page, h, d), dtype, gen) for _ in range(2)]
        s = {"op": op, "caches": caches, "block_table": table, "seq_lens": ints(lens)}
        if op == "compact":
            return s
        r = random.Random(repr((seed, "fork")))
        rows = case["forks"] or case["batch"]
        # Forks: every sequence in turn, so that the batch's samples of a prompt are spread over it; some rows stay empty.
        parents = [b % case["batch"] if r.random() < 0.98 else -1 for b in range(rows)] if case["forks"] else None
        new = [r.randint(case["new_min"], case["new_max"]) for _ in range(rows)]
        return s | {"new_tokens": ints(new), "parents": None if parents is None else ints(parents)}
    new, ctx = whole_numbers(case, "new", seed), whole_numbers(case, "ctx", seed)
    lens = [n + c for n, c in zip(new, ctx)]
    needed = [pages_of(n, page) for n in lens]
    total = sum(pages_of(n + case["ctx_max"], page) for n in new) + 3
    table = tables(needed, total, max(needed), seed)
    rows, codes = sum(new), case["codes"]
    s = {"op": op, "block_table": table, "indptr": ptr_of(new)}
    if op == "append":
        # New rows are views of a fused projection's output, as a layer has them.
        kv = (1.5 * torch.randn(rows, 2 * h * d, generator=gen, device="cuda")).to(dtype)
        s |= {"k_cache": filled((total, page, h, d), DTYPES[codes], gen), "v_cache": filled((total, page, h, d), DTYPES[codes], gen),
              "k_new": kv[:, : h * d], "v_new": kv[:, h * d :], "positions": ints(ctx)}
        return s | ({"k_scale": scales((h,), codes, gen), "v_scale": scales((h,), codes, gen)} if codes == "e4m3" else {"k_scale": None})
    s |= {"kind": case["kind"], "causal": case["causal"], "seq_lens": ints(lens), "new_max": case["new_max"]}
    qkv = torch.randn(rows, (case["hq"] + 2 * h) * d, generator=gen, device="cuda").to(dtype)
    s["q"] = qkv[:, : case["hq"] * d].view(rows, case["hq"], d)
    for name in ("k", "v"):
        if case["kind"] == "block8":  # stored head by head within a page
            s[name + "_cache"] = filled((total, h, page, d), DTYPES[codes], gen).permute(0, 2, 1, 3)
            s[name + "_scale"] = scales((total, h), codes, gen)
        else:
            s[name + "_cache"] = filled((total, page, h, d), DTYPES[codes], gen)
            s[name + "_scale"] = scales((h,), codes, gen) if case["kind"] == "e4m3" else None
    return s


def use_package():
    path = os.path.join(os.getcwd(), "kernel-lab_b200")
    if path not in sys.path:
        sys.path.insert(0, path)


def run(state):
    return run_own(state) if own else run_plain(state)


def run_own(s):
    from kernel_lab import cuda_ops

    if s["op"] == "attend":
        args = (s["block_table"], s["seq_lens"], s["indptr"])
        if s["kind"] == "same":
            out = cuda_ops.paged_chunk_attention(s["q"], s["k_cache"], s["v_cache"], *args, causal=s["causal"])
        else:
            call = cuda_ops.paged_chunk_attention_fp8 if s["kind"] == "e4m3" else cuda_ops.paged_chunk_attention_block8
            out = call(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], *args, causal=s["causal"])
        return {"out": out}
    if s["op"] == "append":
        if s["k_scale"] is None:
            cuda_ops.paged_kv_append(s["k_cache"], s["v_cache"], s["k_new"], s["v_new"], s["block_table"], s["positions"],
                                     indptr=s["indptr"])
        else:
            cuda_ops.paged_kv_append_fp8(s["k_cache"], s["v_cache"], s["k_new"], s["v_new"], s["k_scale"], s["v_scale"],
                                         s["block_table"], s["positions"], indptr=s["indptr"])
        return written(s)
    if s["op"] == "copy":
        cuda_ops.paged_copy_pages(s["caches"], s["src"], s["dst"])
        return {"caches": moved(s)}
    if s["op"] == "reserve":
        table, lens, served = cuda_ops.paged_reserve(s["caches"], s["block_table"], s["seq_lens"], s["new_tokens"], s["parents"])
        return {"block_table": table, "seq_lens": lens, "served": served, "caches": moved(s)}
    table, used = cuda_ops.paged_compact(s["caches"], s["block_table"], s["seq_lens"])
    return {"block_table": table, "used": used, "caches": moved(s)}


def written(s):
    """The pools after an append; where rows are stored as they are, the whole numbers that their bits are."""
    return {name: s[name] if s["k_scale"] is not None else raw(s[name]) for name in ("k_cache", "v_cache")}


def moved(s):
    """The pools as the whole numbers that their bits are: what is moved has to arrive as it was."""
    return [raw(c) for c in s["caches"]]


def raw(t):
    return t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.dtype.itemsize])


# ------------------------------------------------------------------ plain forms


def run_plain(s):
    return {"attend": plain_attend, "append": plain_append, "copy": plain_copy, "reserve": plain_reserve, "compact": plain_compact}[s["op"]](s)


def plain_attend(s):
    """The chunks padded to the longest; a query sees the keys up to its own position, the last query the last key."""
    q, lens, ptr, table = s["q"], s["seq_lens"].long(), s["indptr"].long(), s["block_table"].long()
    page, heads = s["k_cache"].shape[1:3]
    rows, hq, dim = q.shape
    new, most = ptr[1:] - ptr[:-1], s["new_max"]
    i = torch.arange(most, device=q.device)
    row = (ptr[:-1, None] + i).clamp_max(rows - 1)
    k, v = gathered(s, "k", table), gathered(s, "v", table)
    key = torch.arange(k.shape[2], device=q.device)
    there = key < lens[:, None]
    x = q[row].float().view(-1, most, heads, hq // heads, dim).permute(0, 2, 1, 3, 4).reshape(len(lens), heads, -1, dim)
    score = x @ k.transpose(2, 3)  # [batch, kv heads, queries x group, keys]
    del x, k
    last = (lens - new)[:, None] + i if s["causal"] else (lens - 1)[:, None].expand(-1, most)
    seen = (there[:, None] & (key <= last[..., None])).repeat_interleave(hq // heads, dim=1)[:, None]
    score = score.mul_(dim**-0.5).masked_fill_(~seen, -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    p = score.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()
    total = p.sum(dim=-1, keepdim=True)
    out = (p @ torch.where(there[:, None, :, None], v, 0.0)) / torch.where(total > 0, total, 1.0)
    out = out.view(len(lens), heads, most, hq // heads, dim).permute(0, 2, 1, 3, 4).reshape(len(lens), most, hq, dim).to(q.dtype)
    r = torch.arange(rows, device=q.device)
    b = torch.searchsorted(ptr[1:], r, right=True)
    return {"out": out[b, r - ptr[b]]}


def gathered(s, name, table):
    """Each sequence's keys or values in 32 bits: [batch, kv heads, tokens, dim]."""
    cache, scale = s[name + "_cache"], s[name + "_scale"]
    pages = (raw(cache) if cache.dtype is torch.float8_e4m3fn else cache)[table].view(cache.dtype).float()
    if scale is not None:
        pages = pages * (scale if scale.dim() == 1 else scale[table][:, :, None])[..., None]
    return pages.flatten(1, 2).transpose(1, 2).contiguous()


def plain_append(s):
    ptr, page = s["indptr"].long(), s["k_cache"].shape[1]
    r = torch.arange(s["k_new"].shape[0], device=ptr.device)
    b = torch.searchsorted(ptr[1:], r, right=True)
    pos = s["positions"].long()[b] + r - ptr[b]
    at = s["block_table"].long()[b, pos // page]
    for name in ("k", "v"):
        cache = s[name + "_cache"]
        x = s[name + "_new"].view(len(r), *cache.shape[2:])
        if s["k_scale"] is not None:
            x = (x.float() / s[name + "_scale"][:, None]).clamp(-448.0, 448.0).to(cache.dtype)
        raw(cache)[at, pos % page] = raw(x)
    return written(s)


def plain_copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    for cache in s["caches"]:
        raw(cache)[dst] = raw(cache)[src]
    return {"caches": moved(s)}


def plain_reserve(s):
    """A page is free that no sequence's tokens are in. Sequence by sequence, each takes the lowest free pages: first a copy
    of its last page, if it is about to write to it and another holds it too (the first of several that write keeps it),
    then pages for the tokens that its last page has no room for."""
    table, page, pages = s["block_table"].long(), s["caches"][0].shape[1], s["caches"][0].shape[0]
    lens, new, width = s["seq_lens"].long(), s["new_tokens"].long(), table.shape[1]
    if s["parents"] is not None:
        parents = s["parents"].long()
        table = table[parents.clamp_min(0)]
        lens = torch.where(parents >= 0, lens[parents.clamp_min(0)], 0)
        new = torch.where(parents >= 0, new, 0)
    batch = len(lens)
    row, col = torch.arange(batch, device=table.device), torch.arange(width, device=table.device)
    have = (lens + page - 1) // page
    live = col < have[:, None]
    writes = (new > 0) & (lens % page != 0)
    holder = torch.where(writes[:, None] & (col == have[:, None] - 1), row[:, None], -1)
    owner = torch.full((pages + 1,), FAR, device=table.device)
    owner.scatter_reduce_(0, torch.where(live, table, pages).flatten(), holder.flatten(), "amin")
    owner = owner[:pages]
    last = table.gather(1, (have - 1).clamp_min(0)[:, None])[:, 0]
    copied = writes & (owner[last] != row)
    fits = lens + new <= width * page
    grown = (lens + new + page - 1) // page - have
    need = torch.where(fits, copied + grown, 0)
    free = (owner == FAR).nonzero()[:, 0]
    ends = need.cumsum(0)
    served = fits & ((ends <= len(free)) | (need == 0))
    copied = copied & served
    begin = ends - need
    # Column c of a row gets its page number begin + copied + c - have; its last page's copy is number begin.
    number = begin[:, None] + copied[:, None] + col - have[:, None]
    fresh = served[:, None] & (col >= have[:, None]) & (col < (have + grown)[:, None])
    free = torch.cat([free, free.new_zeros(1)])
    got = free[torch.where(fresh, number, 0).clamp(0, len(free) - 1)]
    copy_at = copied[:, None] & (col == have[:, None] - 1)
    copy_to = free[begin.clamp_max(len(free) - 1)]
    out = torch.where(live, torch.where(copy_at, copy_to[:, None], table), torch.where(fresh, got, 0))
    src, dst = last[copied], copy_to[copied]
    for cache in s["caches"]:
        raw(cache)[dst] = raw(cache)[src]
    return {"block_table": out.to(torch.int32), "seq_lens": lens.to(torch.int32), "served": served, "caches": moved(s)}


def plain_compact(s):
    """The pages in use whose number is at least their count go, in order, to the free ones below it."""
    table, page, pages = s["block_table"].long(), s["caches"][0].shape[1], s["caches"][0].shape[0]
    have = (s["seq_lens"].long() + page - 1) // page
    live = torch.arange(table.shape[1], device=table.device) < have[:, None]
    used = torch.zeros(pages + 1, dtype=torch.bool, device=table.device)
    used[torch.where(live, table, pages)] = True
    used = used[:pages]
    count = used.sum()
    number = torch.arange(pages, device=table.device)
    src, dst = (used & (number >= count)).nonzero()[:, 0], (~used & (number < count)).nonzero()[:, 0]
    number[src] = dst
    for cache in s["caches"]:
        raw(cache)[dst] = raw(cache)[src]
    out = torch.where(live, number[torch.where(live, table, 0)], 0)
    return {"block_table": out.to(torch.int32), "used": count.to(torch.int32), "caches": moved(s)}


# ------------------------------------------------------------------ work


def work(case):
    page, h, d = case["page"], case["hkv"], case["dim"]
    e = DTYPES[case["dtype"]].itemsize
    if case["op"] == "copy":
        return {"bytes": 2 * case["tensors"] * case["pairs"] * page * h * d * e, "flops": 0}
    lens = whole_numbers(case, "ctx", 0)
    if case["op"] == "compact":
        used = sum(pages_of(n, page) for n in lens)
        moves = used * (case["pages"] - used) // case["pages"]  # of those in use, the share that lies above their count
        return {"bytes": 2 * 2 * moves * page * h * d * e + 8 * used + 4 * case["batch"], "flops": 0}
    if case["op"] == "reserve":
        rows = case["forks"] or case["batch"]
        held = sum(pages_of(lens[b % case["batch"]], page) for b in range(rows))
        copies = max(0, rows - case["batch"])
        return {"bytes": 2 * 2 * copies * page * h * d * e + 8 * held + 16 * rows, "flops": 0}
    new = whole_numbers(case, "new", 0)
    rows, c = sum(new), DTYPES[case["codes"]].itemsize
    if case["op"] == "append":
        return {"bytes": 2 * rows * h * d * (e + c) + 12 * case["batch"], "flops": 0}
    total = [n + x for n, x in zip(new, lens)]
    # Each sequence's keys and values once, queries and outputs; the products of the pairs that a query sees.
    pairs = sum(n * x + n * (n + 1) // 2 if case["causal"] else n * (n + x) for n, x in zip(new, lens))
    size = 2 * sum(total) * h * d * c + 2 * rows * case["hq"] * d * e + 12 * case["batch"]
    size += sum(pages_of(t, page) for t in total) * (4 + (8 * h if case["kind"] == "block8" else 0))
    return {"bytes": size, "flops": 4 * pairs * case["hq"] * d}


# ------------------------------------------------------------------ 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attend":
        return exact_attend(s)
    if case["op"] == "append":
        return exact_append(s)
    return None  # nothing is computed: pages, tables and counts are whole numbers


def exact_attend(s):
    """Sequence by sequence and head by head, in blocks of queries."""
    q, ptr, lens = s["q"], s["indptr"].tolist(), s["seq_lens"].tolist()
    page, heads, dim = s["k_cache"].shape[1:]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    group = q.shape[1] // heads
    for b, n in enumerate(lens):
        token = torch.arange(n, device=q.device)
        at = s["block_table"][b].long()[token // page]
        first, count = ptr[b], ptr[b + 1] - ptr[b]
        for h in range(heads):
            kv = []
            for name in ("k", "v"):
                cache, scale = s[name + "_cache"], s[name + "_scale"]
                x = (raw(cache) if cache.dtype.itemsize == 1 else cache)[at, token % page, h].view(cache.dtype).double()
                if scale is not None:
                    x = x * (scale[h] if scale.dim() == 1 else scale[at, h][:, None]).double()
                kv.append(x)
            for a in range(0, count, 1024):
                z = min(count, a + 1024)
                x = q[first + a : first + z, h * group : (h + 1) * group].double()
                score = torch.einsum("igd,jd->gij", x, kv[0]) / math.sqrt(dim)
                if s["causal"]:
                    place = n - count + torch.arange(a, z, device=q.device)
                    score.masked_fill_(token > place[:, None], -math.inf)
                w = torch.softmax(score, dim=-1)
                out[first + a : first + z, h * group : (h + 1) * group] = torch.einsum("gij,jd->igd", w, kv[1])
    return {"out": out}


def exact_append(s):
    if s["k_scale"] is None:
        return None
    got, ptr, start, page = {}, s["indptr"].tolist(), s["positions"].tolist(), s["k_cache"].shape[1]
    for name in ("k", "v"):
        cache = s[name + "_cache"].double()
        x = s[name + "_new"].double().view(-1, *cache.shape[2:]) / s[name + "_scale"].double()[:, None]
        unit = torch.pow(2.0, torch.frexp(x).exponent.clamp_min(-5).double() - 4)
        x = (torch.round(x / unit) * unit).clamp(-448, 448)
        for b, at in enumerate(start):
            n = ptr[b + 1] - ptr[b]
            pos = torch.arange(at, at + n, device=x.device)
            cache[s["block_table"][b].long()[pos // page], pos % page] = x[ptr[b] : ptr[b + 1]]
        got[name + "_cache"] = cache
    return got
