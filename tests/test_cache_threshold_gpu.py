"""The alpha-entmax threshold over the 4-bit cache where it lies close below the largest
scores: many equal ones, scores at the clamp, exponents above 2.  Keys are constant over
a group of channels (scale 0), so that scores are exact and weights depend on the
threshold alone."""
import numpy as np
import pytest
import torch

import cache_f64 as F
from test_cache_gpu import dev, fresh, num, sa
from test_cache_paths_gpu import widened

pytestmark = pytest.mark.gpu
D = 32


def stored(z, P, seed, shift=1.0):
    """One sequence whose keys are z [n] in every channel; its values [n, D] as the cache holds them."""
    n = len(z)
    cache, table = fresh(1, [n], 1, D, P, seed=seed)
    g = torch.Generator().manual_seed(seed)
    K = torch.as_tensor(z, dtype=torch.float32)[None, :, None, None].expand(1, n, 1, D).cuda()
    V = (shift + torch.randn(1, n, 1, D, generator=g)).cuda()
    sa().cache_write(K, V, cache, dev(table), dev([0]))
    k, v = F.decode(cache.pool.cpu().numpy(), D, P)
    ids = table[0, : -(-n // P)]
    k, v = (x[ids, 0].reshape(-1, D)[:n] for x in (k, v))
    assert np.array_equal(k, np.repeat(np.asarray(z, np.float64)[:, None], D, 1))
    return cache, table, v


def weights(x, alpha, slack):
    """Weights of exact x = (alpha - 1) score in 64 bits, and what a threshold off by `slack` of its distance
    from the largest x moves them by, with a rounding to 11 bits (2^-11)."""
    y, ex = x - x.max(), 1.0 / (alpha - 1.0)
    lo, hi = -1.0, 0.0
    for _ in range(200):
        mid = 0.5 * (lo + hi)
        if (np.maximum(y - mid, 0.0) ** ex).sum() >= 1.0:
            lo = mid
        else:
            hi = mid
    u, e = y - lo, slack * abs(lo)
    p = np.maximum(u, 0.0) ** ex
    dp = np.maximum(u + e, 0.0) ** ex - np.maximum(u - e, 0.0) ** ex + p * 2.0 ** -11
    return p / p.sum(), dp / p.sum()


def check(o, v, x, alpha):
    """A step's sums of n terms of fp32 are within n/512 * 2^-23 of their size, logarithms and exponentials
    within 2^-20; the threshold's distance follows by alpha - 1 of that, and its solving stops within 2^-21: 2^-16
    covers them up to 40000 keys.  The output: its rounding to bf16, and 2^-10 of the values' mean size for the
    fp32 accumulation of up to 40000 products."""
    p, dp = weights(x, alpha, 2.0 ** -16)
    ref = p @ v
    bound = 2.0 ** -8 * np.abs(ref) + dp @ np.abs(v) + dp.sum() * np.abs(ref) + 2.0 ** -10 * (p @ np.abs(v))
    # not a bound that anything satisfies
    assert (bound < 0.25 * np.sqrt(np.mean(ref ** 2))).all()
    assert np.isfinite(o).all() and (np.abs(o - ref) <= bound).all(), float((np.abs(o - ref) / bound).max())


@pytest.mark.parametrize("tokens", [0, 131072])
@pytest.mark.parametrize("n", [1, 40, 1500, 20000])
@pytest.mark.parametrize("score", [-20.0, 0.3125, 7.5, 20.0])   # at the clamp, inside, and at the clamp
@pytest.mark.parametrize("alpha", [1.25, 1.5, 2.0, 2.5, 3.0])
def test_equal_keys_give_the_mean(cuda, alpha, score, n, tokens):
    cache, table, v = stored(np.full(n, score), 64, seed=n)
    q = torch.ones(1, 1, 3, D, device="cuda").bfloat16()
    o = num(sa().cache_attention(q, cache, dev(widened(table, tokens // 64)), dev([n]), sm_scale=1.0 / D, alpha=alpha))
    for row in o[0, 0]:
        check(row, v, np.full(n, (alpha - 1.0) * np.clip(score, -10.0, 10.0)), alpha)


@pytest.mark.parametrize("tokens", [0, 131072])
@pytest.mark.parametrize("n,best", [(60, 1), (3000, 5), (3000, 300), (20000, 2000)])
@pytest.mark.parametrize("alpha", [1.5, 2.0, 2.25, 2.5, 3.0])
def test_keys_just_below_the_largest(cuda, alpha, n, best, tokens):
    """`best` equal keys at 9.75, the others 2^-7 (the keys' grain there) and more below."""
    g = np.random.RandomState(n + best)
    z = 9.75 - g.randint(1, 64, n) * 2.0 ** -7
    z[g.permutation(n)[:best]] = 9.75
    cache, table, v = stored(z, 32, seed=best)
    q = torch.ones(1, 2, 2, D, device="cuda").bfloat16()
    o = num(sa().cache_attention(q, cache, dev(widened(table, tokens // 32)), dev([n]), sm_scale=1.0 / D, alpha=alpha))
    for t in range(2):
        for row in o[0, t]:
            check(row, v[: n - 1 + t], (alpha - 1.0) * z[: n - 1 + t], alpha)


@pytest.mark.parametrize("alpha", [2.0, 2.5, 3.0])
def test_clamped_scores_among_lower_ones(cuda, alpha):
    """Every third score beyond the clamp: they tie there, and share all weight."""
    n = 6000
    z = np.where(np.arange(n) % 3 == 0, 11.0 + np.arange(n) % 7, 4.0)
    cache, table, v = stored(z, 16, seed=3)
    q = torch.ones(1, 1, 9, D, device="cuda").bfloat16()
    lists = np.arange(n // 16, dtype=np.int32)[None, None, None]
    for pages in (None, dev(lists)):
        o = num(sa().cache_attention(q, cache, dev(table), dev([n]), sm_scale=1.0 / D, alpha=alpha, pages=pages))
        for row in o[0, 0]:
            check(row, v, (alpha - 1.0) * np.clip(z, -10.0, 10.0), alpha)


@pytest.mark.parametrize("tokens", [0, 131072])
@pytest.mark.parametrize("alpha", [1.5, 2.0, 2.125, 2.25, 2.5, 2.75, 3.0])
def test_keys_at_the_edge_of_the_support(cuda, alpha, tokens):
    """A few keys within a tenth of where support ends: above alpha 2 each enters it with infinite slope."""
    B, n, P = 96, 6, 16
    g = np.random.RandomState(int(8 * alpha))
    end = 1.0 / (alpha - 1.0)
    z = -np.round(end * (0.9 + 0.11 * g.rand(B, n)) * 2048.0) / 2048.0
    z[:, 0] = 0.0
    some = 1 + np.arange(B) % (n - 1)                         # keys that take part
    z = np.where(np.arange(n) <= some[:, None], z, -3.0 * end)
    z = z.astype(np.float16).astype(np.float64)
    cache, table = fresh(B, [n] * B, 1, D, P, seed=1)
    K = torch.as_tensor(z, dtype=torch.float32)[:, :, None, None].expand(B, n, 1, D).cuda()
    V = (1.0 + torch.randn(B, n, 1, D, generator=torch.Generator().manual_seed(1))).cuda()
    sa().cache_write(K, V, cache, dev(table), dev(np.zeros(B)))
    v = F.decode(cache.pool.cpu().numpy(), D, P)[1][table[:, 0], 0, :n]
    q = torch.ones(B, 1, 2, D, device="cuda").bfloat16()
    o = num(sa().cache_attention(q, cache, dev(widened(table, tokens // P)), dev([n] * B), sm_scale=1.0 / D, alpha=alpha))
    for b in range(B):
        for row in o[b, 0]:
            check(row, v[b], (alpha - 1.0) * z[b], alpha)
