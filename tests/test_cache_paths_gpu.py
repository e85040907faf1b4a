"""Attention over the 4-bit cache where its work is cut in each of its ways: an
item to a CTA, to a cluster of two, four and eight, to equal runs; eight rows at a
time and sixteen.  Which is taken goes by the table's width, so that a wide table
of short sequences reaches the ways of long ones."""
import numpy as np
import pytest
import torch

from test_cache_gpu import check_attention, dev, filled, sa

pytestmark = pytest.mark.gpu


def widened(table, pages):
    """The table with places that no sequence reaches."""
    wide = np.full((table.shape[0], max(pages, table.shape[1])), -1, np.int32)
    wide[:, : table.shape[1]] = table
    return wide


def check(B, T, G, H, d, P, lengths, pages, alpha, seed):
    cache, table, seqs = filled(B, lengths, H, d, P, seed=seed, k_scale=1.5)
    table = dev(widened(table, pages))
    q = torch.randn(B, T, H * G, d, generator=torch.Generator().manual_seed(seed)).bfloat16().cuda()
    o = sa().cache_attention(q, cache, table, dev(lengths), alpha=alpha)
    check_attention(o, q, seqs, lengths, P, alpha, d ** -0.5)
    again = sa().cache_attention(q, cache, table, dev(lengths), alpha=alpha)
    assert torch.equal(o, again)
    assert sa().device_error() == 0


@pytest.mark.parametrize("alpha", [1.0, 1.5])
@pytest.mark.parametrize("d,P", [(32, 16), (64, 64), (96, 32), (128, 128)])
@pytest.mark.parametrize("B,T,G,H,lengths,tokens", [
    (1, 1, 4, 2, [300], 320),                 # two CTAs an item
    (2, 1, 8, 1, [700, 31], 704),             # four
    (2, 2, 3, 2, [1500, 1], 1536),            # eight
    (3, 1, 1, 2, [2049, 0, 1000], 4096),      # eight, some of them without a tile
    (1, 3, 5, 1, [40], 8192),                 # eight, and more rows than eight
])
def test_clusters(cuda, d, P, B, T, G, H, lengths, tokens, alpha):
    check(B, T, G, H, d, P, lengths, tokens // P, alpha, seed=B + T + G)


@pytest.mark.parametrize("alpha", [1.0, 1.5])
@pytest.mark.parametrize("d,P", [(32, 16), (64, 64), (96, 32), (128, 128)])
@pytest.mark.parametrize("B,T,G,H,lengths", [
    (1, 1, 8, 1, [1]),
    (2, 1, 3, 2, [2500, 77]),
    (5, 2, 4, 3, [0, 900, 1, 33, 2000]),
])
def test_equal_runs(cuda, d, P, B, T, G, H, lengths, alpha):
    check(B, T, G, H, d, P, lengths, 65536 // P, alpha, seed=B + T + G)


@pytest.mark.parametrize("alpha", [1.0, 1.5, 1.25])
@pytest.mark.parametrize("d,P", [(32, 16), (64, 64), (96, 32), (128, 128)])
@pytest.mark.parametrize("B,T,G,H,lengths", [
    (3, 3, 3, 2, [1500, 0, 333]),             # nine rows: most of the second eight empty
    (2, 1, 16, 1, [1, 2100]),
    (2, 5, 7, 1, [2, 1111]),                  # three tiles of rows, the first tokens without a key
])
def test_sixteen_rows_at_a_time(cuda, d, P, B, T, G, H, lengths, alpha):
    rows = T * G
    tiles = -(-16 * 9 * 148 * 12 // (rows * B * H))
    check(B, T, G, H, d, P, lengths, tiles * 32 // P + 1, alpha, seed=B + T + G)


@pytest.mark.parametrize("alpha", [1.0, 1.5])
@pytest.mark.parametrize("B,H,pages,most", [
    (1100, 4, 8, 60),                         # a CTA an item
    (111, 2, 144, 700),                       # two
])
def test_sixteen_rows_of_many_items(cuda, B, H, pages, most, alpha):
    T, G, d, P = 2, 8, 32, 16
    lengths = [int(n) for n in np.random.RandomState(1).randint(0, most, B)]
    cache, table, seqs = filled(B, lengths, H, d, P, seed=1, k_scale=1.5)
    table = widened(table, pages)
    q = torch.randn(B, T, H * G, d, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    o = sa().cache_attention(q, cache, dev(table), dev(lengths), alpha=alpha)
    part = list(range(0, B, B // 20))
    check_attention(o[part], q[part], [seqs[b] for b in part], [lengths[b] for b in part], P, alpha, d ** -0.5)
    assert sa().device_error() == 0


@pytest.mark.parametrize("alpha", [1.25, 1.5, 2.0])
def test_support_found_from_the_largest(cuda, alpha):
    """Thousands of keys within reach of the largest, few of them with weight; more
    tiles than a list of maxima has places for."""
    lengths = [40000, 9000]
    check(2, 1, 2, 1, 64, 64, lengths, 0, alpha, seed=4)


@pytest.mark.parametrize("T,count,P", [(1, [1, 0, 1], 64), (5, [5, 2, 0], 16), (33, [33, 1, 20], 32), (300, [300, 299, 0], 128)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
def test_read_back(cuda, d, dtype, T, count, P):
    """What is read is what the record holds, zero behind the count."""
    lengths = [500, 333, 64]
    cache, table, seqs = filled(3, lengths, 3, d, P, seed=9)
    start = [min(7, lengths[b] - count[b]) for b in range(3)]
    K, V = sa().cache_read(cache, dev(table), dev(start), T, dev(count), dtype=dtype)
    for b in range(3):
        for got, want in zip((K, V), seqs[b]):
            want = torch.from_numpy(want[:, start[b]: start[b] + count[b]].transpose(1, 0, 2)).float().to(dtype)
            assert torch.equal(got[b, : count[b]].cpu(), want)
            assert not got[b, count[b]:].any()
    assert sa().device_error() == 0
