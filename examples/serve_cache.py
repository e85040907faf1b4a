"""Serving one attention layer from the 4-bit paged cache.

    python examples/serve_cache.py

A batch of prompts goes through the training operator (the exact α-entmax), its keys and
values into the cache; then tokens are decoded one by one over the cache, with all pages
and with a selection of them, and a chunk of further prompt tokens is attended at once.
Prints what the cache holds and how far its attention is from full-precision attention
over the same, unquantised keys and values.
"""
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "adaptive-splash-attention_b200"))
import splash_attention as sa  # noqa: E402


def full(q, k, v, length, alpha):
    """Attention of q [B, T, HQ, d] over k, v [B, n, H, d] in fp32, by the definition."""
    B, T, HQ, d = q.shape
    n, G = k.shape[1], HQ // k.shape[2]
    k, v = (x.float().repeat_interleave(G, 2).transpose(1, 2) for x in (k, v))
    s = q.float().transpose(1, 2) @ k.transpose(-1, -2) * d ** -0.5
    seen = torch.arange(n, device=q.device) <= (length[:, None] - T + torch.arange(T, device=q.device))[..., None]
    if alpha == 1.0:
        p = s.masked_fill(~seen[:, None], float("-inf")).softmax(-1)
    else:                                   # the root of sum (x - tau)_+^(1/(alpha-1)) = 1 by bisection
        x = ((alpha - 1) * s.clamp(-10, 10)).masked_fill(~seen[:, None], float("-inf"))
        hi = x.amax(-1, keepdim=True)
        lo = hi - 1
        for _ in range(40):
            mid = (lo + hi) / 2
            over = (x - mid).clamp(min=0).pow(1 / (alpha - 1)).sum(-1, keepdim=True) >= 1
            lo, hi = torch.where(over, mid, lo), torch.where(over, hi, mid)
        p = (x - lo).clamp(min=0).pow(1 / (alpha - 1))
        p = p / p.sum(-1, keepdim=True)
    return (p @ v).transpose(1, 2)


def main(B=2, prompt=1000, steps=8, heads=16, kv_heads=4, d=128, page=64, keep=8, alpha=1.5, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    total = prompt + steps + 96
    make = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    # keys in runs of 50 about a topic each; a query looks for the topic of a run before it
    topic = make(B, total // 50 + 1, kv_heads, d)
    run = torch.arange(total, device="cuda") // 50
    look = (torch.rand(B, total, generator=g, device="cuda") * (run + 1)).long()
    q = make(B, total, kv_heads, heads // kv_heads, d) + 0.8 * topic[torch.arange(B, device="cuda")[:, None], look].unsqueeze(3)
    q, k, v = q.flatten(2, 3).bfloat16(), (make(B, total, kv_heads, d) + 1.5 * topic[:, run]).bfloat16(), make(B, total, kv_heads, d).bfloat16()

    # a page of the pool to every `page` tokens, handed out in any order
    per = -(-total // page)
    cache = sa.new_cache(B * per, kv_heads, d, page)
    table = torch.randperm(B * per, generator=torch.Generator().manual_seed(seed)).view(B, per).int().cuda()

    # the prompt: the training operator computes its outputs, the cache keeps its keys and values
    rows = lambda x: x[:, :prompt].transpose(1, 2)  # noqa: E731
    at = torch.arange(prompt, dtype=torch.int32, device="cuda")
    prompt_out = sa.splash_attention(rows(q), rows(k).repeat_interleave(heads // kv_heads, 1),
                                     rows(v).repeat_interleave(heads // kv_heads, 1), at, at, alpha=alpha,
                                     tau_mode="exact", ref_tile_load=False).transpose(1, 2)
    zero = torch.zeros(B, dtype=torch.int32, device="cuda")
    sa.cache_write(k[:, :prompt], v[:, :prompt], cache, table, zero)
    lengths = zero + prompt
    err = {}

    def far(name, o, ref):
        err[name] = max(err.get(name, 0.0), float((o.float() - ref.float()).norm() / ref.float().norm()))

    # (the prompt's last queries, attended over the cache, are the training operator's outputs)
    far("prompt's last queries, cache against training operator",
        sa.cache_attention(q[:, prompt - 8: prompt], cache, table, lengths, alpha=alpha), prompt_out[:, -8:])
    for t in range(prompt, prompt + steps):
        one = slice(t, t + 1)
        sa.cache_write(k[:, one], v[:, one], cache, table, lengths)
        lengths = lengths + 1
        for a in (1.0, alpha):
            o = sa.cache_attention(q[:, one], cache, table, lengths, alpha=a)
            far("decoding, alpha %g" % a, o, full(q[:, one], k[:, : t + 1], v[:, : t + 1], lengths, a))
        pages = sa.select_pages(q[:, one], cache, table, lengths, keep)
        o = sa.cache_attention(q[:, one], cache, table, lengths, alpha=alpha, pages=pages)
        far("decoding, %d of %d pages, alpha %g" % (keep, -(-(t + 1) // page), alpha), o,
            full(q[:, one], k[:, : t + 1], v[:, : t + 1], lengths, alpha))
    more = slice(prompt + steps, total)
    sa.cache_write(k[:, more], v[:, more], cache, table, lengths)
    lengths = lengths + (total - prompt - steps)
    o = sa.cache_attention(q[:, more], cache, table, lengths)
    far("a chunk of %d tokens, softmax" % (total - prompt - steps), o, full(q[:, more], k, v, lengths, 1.0))
    back_k, back_v = sa.cache_read(cache, table, zero, total)
    far("keys read back", back_k, k)
    far("values read back", back_v, v)
    if sa.device_error():
        raise RuntimeError("the cache's kernels reported an error")
    held = cache.pool.numel() / (2 * B * per * page * kv_heads * d)
    print("%d tokens of %d key heads, %.2f bytes a number (bf16: 2)" % (B * total, kv_heads, held))
    for name, e in err.items():
        print("  %-58s relative error %.3f" % (name, e))
    return err


if __name__ == "__main__":
    main()
