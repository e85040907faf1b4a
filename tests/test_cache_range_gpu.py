"""The 4-bit cache at the ends of what its arguments can hold."""
import numpy as np
import pytest
import torch

import cache_f64 as F
from test_cache_gpu import check_attention, dev, filled, fresh, num, sa

pytestmark = pytest.mark.gpu
INVALID = 1


@pytest.mark.parametrize("d,T", [(32, 1), (64, 1), (96, 5), (128, 1), (64, 64), (128, 64)])
@pytest.mark.parametrize("q_scale", [1e33, 1e37])
def test_queries_near_the_largest_number(cuda, d, T, q_scale):
    """Softmax is the largest score's alone, whose value is the output (its rounding to bf16, and 2^-11 for
    values held in 11 bits); alpha-entmax clamps."""
    H, n, P = 2, 40 + T, 32
    cache, table, seqs = filled(1, [n], H, d, P, seed=d + T, k_scale=30.0)
    q = (torch.randn(1, T, 2 * H, d, generator=torch.Generator().manual_seed(5)) * q_scale).bfloat16().cuda()
    o = num(sa().cache_attention(q, cache, dev(table), dev([n])))
    assert np.isfinite(o).all()
    checked = 0
    for t in range(T):
        for h in range(2 * H):
            k, v = (x[h // 2][: n - T + t + 1] for x in seqs[0])
            s = k @ num(q).astype(np.float64)[0, t, h]
            best, second = np.sort(s)[-1], np.sort(s)[-2]
            if best - second < 2.0 ** -8 * np.abs(s).max():   # too near for 32 bits of sums to be certain of
                continue
            checked += 1
            ref = v[s.argmax()]
            assert (np.abs(o[0, t, h] - ref) <= (2.0 ** -8 + 2.0 ** -11) * np.abs(ref) + 2.0 ** -20 * np.abs(v).max()).all()
    assert checked > T
    if T <= 5:
        e = sa().cache_attention(q, cache, dev(table), dev([n]), alpha=1.5)
        check_attention(e, q, seqs, [n], P, 1.5, d ** -0.5)


def test_indices_past_32_bits(cuda):
    """Whole numbers that int32 does not hold are not other ones: a page is outside the pool, a length past the table."""
    H, d, P, n = 2, 64, 16, 100
    cache, table, seqs = filled(1, [n], H, d, P, seed=2)
    q = torch.randn(1, 1, 4, d, generator=torch.Generator().manual_seed(8)).bfloat16().cuda()
    tab = dev(table)
    sa().device_error()
    for far in (1 << 32, -(1 << 32), 1 << 40):
        away = tab.long()
        away[0, 1] += far
        o = sa().cache_attention(q, cache, away, dev([n]))
        assert sa().device_error() == INVALID
        check_attention(o, q, seqs, [n], P, 1.0, d ** -0.5, np.array([0, 2, 3, 4, 5, 6]).reshape(1, 1, 1, 6).repeat(H, 2))
    short = tab[:, :3].contiguous()
    o = sa().cache_attention(q, cache, short, torch.tensor([(1 << 32) + 5], device="cuda"))
    want = sa().cache_attention(q, cache, short, dev([48]))
    assert torch.equal(o, want)
    assert not sa().cache_attention(q, cache, short, torch.tensor([5 - (1 << 32)], device="cuda")).any()
    before = cache.pool.clone()
    x = torch.randn(1, 1, H, d).bfloat16().cuda()
    sa().device_error()
    sa().cache_write(x, x, cache, tab, torch.tensor([(1 << 32) + 3], device="cuda"))
    assert torch.equal(cache.pool, before) and sa().device_error() == INVALID
    lists = torch.tensor([0, 1 << 32], device="cuda").repeat(1, 1, H, 1)
    o = sa().cache_attention(q, cache, tab, dev([n]), pages=lists)
    check_attention(o, q, seqs, [n], P, 1.0, d ** -0.5, np.zeros((1, 1, H, 1), np.int32))


@pytest.mark.parametrize("d,P", [(32, 16), (64, 32), (96, 64), (128, 128)])
@pytest.mark.parametrize("rows", [1, 12, 64])
@pytest.mark.parametrize("bits", [8.3, 11.3, 13.7])
def test_small_weights_of_large_values(cuda, d, P, rows, bits):
    """A key whose values are 0, and one of 2^-bits of its weight with values up to 60000: the second's alone are the
    output.  Tolerance: the output's rounding (2^-8) and the weight's to 11 bits (2^-11 twice, for that and its
    product with the scale's rest), and scores off by 2^-20 of themselves (2^-16)."""
    n = rows + 1                                              # every row sees both keys; later ones are far below
    K = torch.zeros(1, n, 1, d)
    K[:, 0] = 1.0
    K[:, 2:] = -8.0
    V = torch.zeros(1, n, 1, d)
    V[:, 1] = 60000.0 * (2.0 * torch.rand(d, generator=torch.Generator().manual_seed(1)) - 1.0)
    V[0, 1, 0, ::32] = 60000.0
    V[0, 1, 0, 1::32] = -60000.0
    cache, table = fresh(1, [n], 1, d, P)
    sa().cache_write(K.cuda(), V.cuda(), cache, dev(table), dev([0]))
    v = F.decode(cache.pool.cpu().numpy(), d, P)[1][table[0, 0], 0, 1]
    q = torch.ones(1, rows, 1, d, device="cuda").bfloat16()
    o = num(sa().cache_attention(q, cache, dev(table), dev([n]), sm_scale=bits * float(np.log(2.0)) / d))
    want = v / (1.0 + 2.0 ** bits)
    tol = 2.0 ** -8 + 2.0 ** -10 + 2.0 ** -16
    assert (np.abs(o[0, :, 0] - want) <= tol * np.abs(want) + 2.0 ** -20 * 60000.0 * 2.0 ** -bits).all()
