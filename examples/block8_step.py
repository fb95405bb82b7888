"""A decoder layer's attention half served over a cache held in 8 bits.

    python examples/block8_step.py [--heads 32/8] [--prompt 2000] [--steps 8] [--pages 32] [--int8]

Three prompts of unlike length are appended to a block-scaled cache (kernel_lab.cuda_ops), then every step
runs what a serving loop runs around its projections: the fused residual add + RMSNorm with an e4m3
output, the append of each sequence's new token, the selection of the pages to read, and decode
attention over those pages. Beside it the same steps run over a bf16 cache with the whole context, and the
difference is printed: what the 8 bits cost, and what reading a part of the pages costs. The weights are
random, so attention is spread thin and the second figure is an upper end.
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "kernel-lab_b200"))

from kernel_lab import cuda_ops, kv_cache  # noqa: E402

PAGE = 16


def run(hq=32, hkv=8, head_dim=128, prompt=2000, steps=8, pages=32, dtype=torch.float8_e4m3fn, seed=0):
    """Returns the relative differences from the bf16 cache: (8-bit cache, selected pages of it)."""
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(torch.bfloat16)

    hidden = hq * head_dim
    lens = [prompt, prompt // 2 + 1, max(1, prompt // 7)]
    batch = len(lens)
    w_qkv = rand(hidden, (hq + 2 * hkv) * head_dim, scale=hidden**-0.5)
    w_out = rand(hidden, hidden, scale=hidden**-0.5)
    w_norm = 1 + rand(hidden, scale=0.1)

    def project(codes, scales):
        """The projection of an e4m3 activation; a product that takes 8-bit operands would use them as they are."""
        x = (codes.float().unflatten(-1, (-1, 128)) * scales[..., None]).flatten(-2).to(torch.bfloat16)
        qkv = x @ w_qkv
        return qkv[:, :hidden], qkv[:, hidden : hidden + hkv * head_dim], qkv[:, hidden + hkv * head_dim :]

    # Every sequence's pages, shuffled over the pool.
    need = [kv_cache.pages_for(n + steps, PAGE) for n in lens]
    order = torch.randperm(sum(need), generator=torch.Generator().manual_seed(seed)).to(torch.int32).cuda()
    table = torch.zeros(batch, max(need), dtype=torch.int32, device="cuda")
    for b, n in enumerate(need):
        table[b, :n] = order[sum(need[:b]) :][:n]
    pool = kv_cache.block8_pool(sum(need), PAGE, hkv, head_dim, dtype, heads_first=True)
    plain = [torch.zeros(sum(need), PAGE, hkv, head_dim, dtype=torch.bfloat16, device="cuda") for _ in range(2)]

    # Prompts: one ragged append for all sequences.
    residual = rand(sum(lens), hidden)
    codes, scales, _ = cuda_ops.fused_add_rms_norm_fp8(rand(sum(lens), hidden), residual, w_norm, 1e-5, group_size=128)
    _, k, v = project(codes, scales)
    indptr = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    start = torch.zeros(batch, dtype=torch.int32, device="cuda")
    cuda_ops.paged_kv_append_block8(pool.k_cache, pool.v_cache, pool.k_scale, pool.v_scale, k, v, table, start,
                                    indptr=indptr, k_bounds=pool.k_bounds)
    for b, n in enumerate(lens):
        pos = torch.arange(n, device="cuda")
        for cache, new in zip(plain, (k, v)):
            cache[table[b].long()[pos // PAGE], pos % PAGE] = new[indptr[b] : indptr[b + 1]].view(n, hkv, head_dim)

    seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    residual, x = rand(batch, hidden), rand(batch, hidden)
    worst = [0.0, 0.0]
    for _ in range(steps):
        codes, scales, residual = cuda_ops.fused_add_rms_norm_fp8(x, residual, w_norm, 1e-5, group_size=128)
        q, k, v = project(codes, scales)
        q = q.reshape(batch, hq, head_dim)
        cuda_ops.paged_kv_append_block8(pool.k_cache, pool.v_cache, pool.k_scale, pool.v_scale, k, v, table, seq_lens,
                                        k_bounds=pool.k_bounds)
        cuda_ops.paged_kv_append(*plain, k.contiguous(), v.contiguous(), table, seq_lens)
        seq_lens = seq_lens + 1
        chosen = cuda_ops.paged_block_select(q, pool.k_cache, pool.k_scale, pool.k_bounds, table, seq_lens, pages)
        cache = (pool.k_cache, pool.v_cache, pool.k_scale, pool.v_scale, table, seq_lens)
        sparse = cuda_ops.paged_decode_attention_block8(q, *cache, selected=chosen)
        whole = cuda_ops.paged_decode_attention_block8(q, *cache)
        want = cuda_ops.paged_decode_attention(q, *plain, table, seq_lens)
        for i, got in enumerate((whole, sparse)):
            worst[i] = max(worst[i], float((got - want).float().norm() / want.float().norm()))
        x = whole.reshape(batch, hidden) @ w_out
    if cuda_ops.decode_status(clear=True):
        raise RuntimeError("a page id was outside the pool")
    return tuple(worst)


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--heads", default="32/8")
    ap.add_argument("--prompt", type=int, default=2000)
    ap.add_argument("--steps", type=int, default=8)
    ap.add_argument("--pages", type=int, default=32)
    ap.add_argument("--int8", action="store_true")
    args = ap.parse_args()
    hq, hkv = (int(n) for n in args.heads.split("/"))
    kind = torch.int8 if args.int8 else torch.float8_e4m3fn
    whole, sparse = run(hq, hkv, prompt=args.prompt, steps=args.steps, pages=args.pages, dtype=kind)
    print(f"{args.steps} steps over {kind}: relative difference from a bf16 cache {whole:.4f}, reading at most "
          f"{args.pages} pages of each sequence {sparse:.4f}")


if __name__ == "__main__":
    main()
