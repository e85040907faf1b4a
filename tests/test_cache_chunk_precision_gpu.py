"""Chunks of prompts over the 4-bit cache where keys are far from zero.  The chunk kernel
holds a key as (c + n s) + (z - c), c = fp16(-7.5 s), the first part rounded to fp16: a
group's offset takes no bits from its codes, its own spread is rounded to 11 bits.  So
results are those of the keys as stored where offsets dwarf scales, and everywhere those
of the keys with that one rounding (`rounded`), within the bounds of 32-bit sums."""
import numpy as np
import pytest
import torch

import cache_f64 as F
from test_cache_gpu import check_attention, dev, fresh, num, sa
from test_cache_paths_gpu import widened
from test_cache_scores_gpu import LEVELS, asks, made

pytestmark = pytest.mark.gpu


def rounded(pool, d, P):
    """The keys as the chunk kernel has them, float64 [pages, H, P, d]."""
    y = np.empty(pool.shape[:2] + (P, d))
    at, g, ng = F.places(d, True), np.arange(d) // 32, d // 32
    for slot in range(P):
        row, par = F.row_at(d, P, slot, True)
        n = (pool[..., row + at] >> (4 * (np.arange(d) % 2)).astype(np.uint8)) & 15
        h = np.ascontiguousarray(pool[..., par: par + 4 * ng]).view(np.float16).astype(np.float64)
        s, z = h[..., g], h[..., ng + g]
        with np.errstate(over="ignore", invalid="ignore"):    # (pages nobody wrote hold anything)
            c = np.maximum((-7.5 * s).astype(np.float16).astype(np.float64), -F.F16_MAX)
            y[..., slot, :] = np.minimum((n * s + c).astype(np.float16).astype(np.float64), F.F16_MAX) + (z - c)
    return y


def sequences(k, v, table, lengths, P):
    out = []
    for b, n in enumerate(lengths):
        ids = table[b, : -(-n // P)]
        out.append(tuple(x[ids].transpose(1, 0, 2, 3).reshape(x.shape[1], -1, x.shape[3])[:, :n] for x in (k, v)))
    return out


@pytest.mark.parametrize("rows", [63, 64, 130])              # on both sides of the rule, and two tiles
@pytest.mark.parametrize("d,P", [(64, 32), (128, 64)])
@pytest.mark.parametrize("shift", ["all", "channels", "groups", "one"])
@pytest.mark.parametrize("tokens", [0, 32768])
def test_keys_far_from_zero(cuda, d, P, rows, shift, tokens):
    """Offsets of a group far above its scale, as a model's rotated or biased channels have them."""
    n, H = 500, 2
    g = torch.Generator().manual_seed(d + rows)
    K = torch.randn(1, n, H, d, generator=g)
    if shift == "all":
        K += 200.0
    elif shift == "channels":
        K += 200.0 * torch.sign(torch.randn(d, generator=g)).repeat_interleave(1)
    elif shift == "groups":
        K += 1000.0 * torch.linspace(-1, 1, d // 32).repeat_interleave(32)
    else:
        K[..., 5] -= 300.0
    V = torch.randn(1, n, H, d, generator=g)
    cache, table = fresh(1, [n], H, d, P)
    sa().cache_write(K.cuda(), V.cuda(), cache, dev(table), dev([0]))
    k, v = F.decode(cache.pool.cpu().numpy(), d, P)
    q = torch.randn(1, rows, H, d, generator=g).bfloat16().cuda()
    o = sa().cache_attention(q, cache, dev(widened(table, tokens // P)), dev([n]))
    if rows < 64 or shift in ("all", "groups"):
        check_attention(o, q, sequences(k, v, table, [n], P), [n], P, 1.0, d ** -0.5)
    if rows >= 64:
        check_attention(o, q, sequences(rounded(cache.pool.cpu().numpy(), d, P), v, table, [n], P), [n], P, 1.0, d ** -0.5)


@pytest.mark.parametrize("d", [64, 128])
def test_keys_over_all_of_the_range(cuda, d):
    """Groups from one end of fp16 to the other, beside ordinary ones; queries small enough for scores of some units."""
    n, H, P = 300, 1, 64
    g = torch.Generator().manual_seed(d)
    K = torch.randn(1, n, H, d, generator=g)
    K[..., :32] = 65504.0 * (2.0 * torch.rand(1, n, H, 32, generator=g) - 1.0)
    K[:, :, :, 0], K[:, :, :, 1] = 65504.0, -65504.0
    V = torch.randn(1, n, H, d, generator=g)
    cache, table = fresh(1, [n], H, d, P)
    sa().cache_write(K.cuda(), V.cuda(), cache, dev(table), dev([0]))
    k, v = F.decode(cache.pool.cpu().numpy(), d, P)
    ids = table[0, : -(-n // P)]
    seqs = [tuple(x[ids].transpose(1, 0, 2, 3).reshape(H, -1, d)[:, :n] for x in (k, v))]
    for rows in (3, 80):
        q = torch.randn(1, rows, H, d, generator=g)
        q[..., :32] *= 2.0 ** -15
        q = q.bfloat16().cuda()
        o = sa().cache_attention(q, cache, dev(table), dev([n]))
        check_attention(o, q, seqs, [n], P, 1.0, d ** -0.5)


@pytest.mark.parametrize("level", LEVELS)
@pytest.mark.parametrize("d,P", [(64, 16), (64, 128), (128, 64)])
@pytest.mark.parametrize("T,G,lengths,tokens", [
    (64, 1, [64, 64], 0),
    (40, 2, [300, 39], 0),
    (64, 3, [2000, 65], 0),
    (64, 1, [700, 64], 32768),
])
def test_scores_far_below(cuda, d, P, T, G, lengths, tokens, level):
    """Keys about +-2 in every channel: a group's offset lies opposite to half of its keys."""
    cache, table, seqs = made(lengths, 1, d, P, level, seed=6)
    q = asks(2, T, G, d, level)
    o = sa().cache_attention(q, cache, dev(widened(table, tokens // P)), dev(lengths))
    pool = cache.pool.cpu().numpy()
    seqs = sequences(rounded(pool, d, P), F.decode(pool, d, P)[1], table, lengths, P)
    check_attention(o, q, seqs, lengths, P, 1.0, d ** -0.5)
