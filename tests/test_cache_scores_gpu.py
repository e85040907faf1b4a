"""Attention over the 4-bit cache where scores are far below zero: a row's weights
are relative to its largest score, wherever that lies.  What is compared: the 64-bit
form (test_cache_gpu.check_attention and its derived bounds), and, where a query sees
one key, that key's value: the output is its rounding to bf16 (8 bits: 2^-8 of it), with what a
weight's rounding to 11 bits may add (2^-11) and sums of fp32 lose against the
largest value of its group (2^-20)."""
import numpy as np
import pytest
import torch

import cache_f64 as F
from test_cache_gpu import check_attention, dev, fresh, num, sa
from test_cache_paths_gpu import widened

pytestmark = pytest.mark.gpu


def signs(d):
    """A direction of +-1, neither constant nor periodic in a group."""
    return torch.from_numpy(np.where(np.random.RandomState(d).rand(d) < 0.5, -1.0, 1.0)).float()


def made(lengths, H, d, P, level, seed=0, blocks=None):
    """A cache whose keys lie near 2 u, u of +-1, and so give scores near `level` with the
    queries of `asks`; blocks(b, n): the tokens whose keys are near 0 (scores near 0)."""
    B, T = len(lengths), max(max(lengths), 1)
    cache, table = fresh(B, lengths, H, d, P, seed=seed)
    g = torch.Generator().manual_seed(seed)
    K = 0.1 * torch.randn(B, T, H, d, generator=g)
    far = torch.ones(B, T)
    if blocks is not None:
        for b, n in enumerate(lengths):
            far[b, blocks(b, n)] = 0.0
    K = (K + 2.0 * far[:, :, None, None] * signs(d)).cuda()
    V = torch.randn(B, T, H, d, generator=g).cuda()
    sa().cache_write(K, V, cache, dev(table), dev(np.zeros(B)), dev(lengths))
    k, v = F.decode(cache.pool.cpu().numpy(), d, P)
    seqs = []
    for b, n in enumerate(lengths):
        ids = table[b, : -(-n // P)]
        seqs.append(tuple(x[ids].transpose(1, 0, 2, 3).reshape(H, -1, d)[:, :n] for x in (k, v)))
    return cache, table, seqs


def asks(B, T, HQ, d, level, seed=1):
    g = torch.Generator().manual_seed(seed)
    q = level * d ** 0.5 / (2 * d) * signs(d) * (1.0 + 0.02 * torch.randn(B, T, HQ, 1, generator=g))
    return q.bfloat16().cuda()


def check_one_key(o, v):
    """o, v [..., d]: the outputs of rows that see one key, and its value."""
    assert np.isfinite(o).all()
    top = np.abs(v).reshape(*v.shape[:-1], -1, 32).max(-1).repeat(32, -1)
    assert (np.abs(o - v) <= (2.0 ** -8 + 2.0 ** -11) * np.abs(v) + 2.0 ** -20 * top).all()


LEVELS = [-100.0, -1000.0, -10000.0]


# ---- a few query rows ------------------------------------------------------------
@pytest.mark.parametrize("level", LEVELS)
@pytest.mark.parametrize("d,P", [(32, 16), (64, 64), (96, 32), (128, 128)])
def test_one_key_far_below(cuda, d, P, level):
    H, G, lengths = 2, 3, [1, 1, 1]
    cache, table, seqs = made(lengths, H, d, P, level)
    for pages in (0, 4096 // P, 65536 // P):                  # a CTA an item, clusters, equal runs
        q = asks(3, 1, H * G, d, level)
        o = num(sa().cache_attention(q, cache, dev(widened(table, pages)), dev(lengths)))
        for b in range(3):
            check_one_key(o[b, 0].reshape(H, G, d), seqs[b][1][:, :1].repeat(G, 1))


@pytest.mark.parametrize("level", LEVELS)
@pytest.mark.parametrize("tokens", [0, 4096, 65536])
@pytest.mark.parametrize("d,P", [(32, 16), (64, 64), (96, 32), (128, 128)])
def test_all_scores_far_below(cuda, d, P, tokens, level):
    H, T, G, lengths = 2, 3, 4, [700, 33, 3]
    cache, table, seqs = made(lengths, H, d, P, level, seed=2)
    q = asks(3, T, H * G, d, level)
    o = sa().cache_attention(q, cache, dev(widened(table, tokens // P)), dev(lengths))
    check_attention(o, q, seqs, lengths, P, 1.0, d ** -0.5)
    assert sa().device_error() == 0


@pytest.mark.parametrize("level", LEVELS)
@pytest.mark.parametrize("tokens", [0, 4096, 65536])
@pytest.mark.parametrize("d,P", [(32, 16), (128, 64)])
def test_tiles_far_below_beside_others(cuda, d, P, tokens, level):
    """Whole 32-token tiles far below, among others near zero: whatever tile a warp meets first."""
    H, G, lengths = 1, 2, [1200, 640]
    pick = [np.random.RandomState(b).rand(64) < 0.3 for b in range(2)]
    cache, table, seqs = made(lengths, H, d, P, level, seed=3,
                              blocks=lambda b, n: np.nonzero(pick[b][np.arange(n) // 32])[0])
    q = asks(2, 1, H * G, d, level)
    o = sa().cache_attention(q, cache, dev(widened(table, tokens // P)), dev(lengths))
    check_attention(o, q, seqs, lengths, P, 1.0, d ** -0.5)


@pytest.mark.parametrize("level", LEVELS)
@pytest.mark.parametrize("d,P", [(32, 16), (64, 64), (96, 32), (128, 128)])
def test_sixteen_rows_far_below(cuda, d, P, level):
    B, T, G, H, lengths = 2, 3, 5, 1, [3, 1500]
    cache, table, seqs = made(lengths, H, d, P, level, seed=4)
    q = asks(B, T, H * G, d, level)
    tiles = -(-16 * 9 * 148 * 12 // (T * G * B * H))          # a table this wide takes rows by sixteens
    o = sa().cache_attention(q, cache, dev(widened(table, tiles * 32 // P + 1)), dev(lengths))
    check_attention(o, q, seqs, lengths, P, 1.0, d ** -0.5)


@pytest.mark.parametrize("level", LEVELS)
@pytest.mark.parametrize("d,P", [(32, 16), (64, 64), (96, 32), (128, 128)])
def test_listed_pages_far_below(cuda, d, P, level):
    """Among them a query whose own page holds a single key."""
    H, G, lengths = 2, 4, [5 * P + 1, P + 1, 1]
    cache, table, seqs = made(lengths, H, d, P, level, seed=5)
    q = asks(3, 1, H * G, d, level)
    lists = np.full((3, 1, H, 3), -1, np.int32)
    lists[0, 0, :] = [5, 1, 3]
    lists[1, 0, 0, 1], lists[1, 0, 1, 0] = 1, 0
    lists[2, 0, :, 2] = 0
    o = sa().cache_attention(q, cache, dev(table), dev(lengths), pages=dev(lists))
    check_attention(o, q, seqs, lengths, P, 1.0, d ** -0.5, lists)
    check_one_key(num(o)[1, 0, :G], seqs[1][1][0, P: P + 1].repeat(G, 0))


# ---- chunks of prompts -------------------------------------------------------------
@pytest.mark.parametrize("level", LEVELS)
@pytest.mark.parametrize("d,P", [(64, 16), (64, 128), (128, 64)])
@pytest.mark.parametrize("T,G,lengths,tokens", [
    (64, 1, [64, 64], 0),                    # a prompt: its first token sees one key
    (40, 2, [300, 39], 0),                   # and one that sees none before it
    (64, 3, [2000, 65], 0),
    (64, 1, [700, 64], 32768),               # cut into equal runs
])
def test_chunks_far_below(cuda, d, P, T, G, lengths, tokens, level):
    cache, table, seqs = made(lengths, 1, d, P, level, seed=6)
    q = asks(2, T, G, d, level)
    o = sa().cache_attention(q, cache, dev(widened(table, tokens // P)), dev(lengths))
    assert torch.isfinite(o).all() and not o[1, : max(0, T - lengths[1])].any()
    for b, n in enumerate(lengths):
        if 0 <= T - n < T:
            check_one_key(num(o)[b, T - n], seqs[b][1][0, :1].repeat(G, 0))
    assert sa().device_error() == 0


@pytest.mark.parametrize("level", LEVELS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("tokens", [0, 32768])
def test_chunks_whose_first_pages_cannot_be_read(cuda, d, tokens, level):
    """A row's first keys come with a later tile, its output already under way."""
    P, T, n = 64, 64, 900
    cache, table, seqs = made([n], 1, d, P, level, seed=7)
    bad = widened(table, tokens // P)
    bad[0, :3] = -1
    q = asks(1, T, 2, d, level)
    o = sa().cache_attention(q, cache, dev(bad), dev([n]))
    sa().device_error()
    seen = np.arange(3, -(-n // P), dtype=np.int32)
    check_attention(o, q, seqs, [n], P, 1.0, d ** -0.5, np.broadcast_to(seen, (1, T, 1, len(seen))))


@pytest.mark.parametrize("level", LEVELS)
@pytest.mark.parametrize("d", [64, 128])
def test_chunk_tiles_far_below_beside_others(cuda, d, level):
    pick = np.random.RandomState(0).rand(16) < 0.4
    cache, table, seqs = made([1800], 1, d, 64, level, seed=8,
                              blocks=lambda b, n: np.nonzero(pick[np.arange(n) // 128])[0])
    q = asks(1, 70, 1, d, level)
    for pages in (0, 512):
        o = sa().cache_attention(q, cache, dev(widened(table, pages)), dev([1800]))
        check_attention(o, q, seqs, [1800], 64, 1.0, d ** -0.5)
