"""The 4-bit paged cache on the GPU against its format and against 64-bit
arithmetic (tests/cache_f64.py): stored bytes and bounds bit for bit, selected
pages exactly, attention within bounds derived from its roundings."""
import numpy as np
import pytest
import torch

import cache_f64 as F

pytestmark = pytest.mark.gpu
INVALID = 1


def sa():
    import splash_attention
    return splash_attention


def dev(x, dtype=torch.int32):
    return torch.as_tensor(np.asarray(x), device="cuda").to(dtype)


def num(t):
    return t.detach().float().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def fresh(B, lengths, H, d, P, spare=3, seed=0, fill=255):
    """A cache whose bytes are all `fill`, and a table of shuffled pages."""
    need = [-(-n // P) for n in lengths]
    g = np.random.RandomState(seed)
    ids = g.permutation(sum(need) + spare)
    cache = sa().new_cache(len(ids), H, d, P)
    cache.pool.fill_(fill)
    cache.bounds.fill_(fill - 256 if fill > 127 else fill)
    table = np.full((B, max(max(need), 1) + 1), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at: at + n]
        at += n
    return cache, table


def filled(B, lengths, H, d, P, seed=0, k_scale=1.0, v_scale=1.0, v_shift=0.0, fill=255):
    """A cache that holds random tokens, and K, V float64 of each sequence."""
    cache, table = fresh(B, lengths, H, d, P, seed=seed, fill=fill)
    g = torch.Generator().manual_seed(seed)
    T = max(max(lengths), 1)
    K = (torch.randn(B, T, H, d, generator=g) * k_scale).bfloat16().cuda()
    V = (torch.randn(B, T, H, d, generator=g) * v_scale + v_shift).bfloat16().cuda()
    sa().cache_write(K, V, cache, dev(table), dev(np.zeros(B)), dev(lengths))
    k, v = F.decode(cache.pool.cpu().numpy(), d, P)
    seqs = []
    for b, n in enumerate(lengths):
        ids = table[b, : -(-n // P)]
        seqs.append(tuple(x[ids].transpose(1, 0, 2, 3).reshape(H, -1, d)[:, :n] for x in (k, v)))
    return cache, table, seqs


def check_attention(o, q, seqs, lengths, P, alpha, scale, lists=None):
    """o, q [B, T, HQ, d]; lists [B, T, H, keep] or None."""
    o, q = num(o).astype(np.float64), num(q).astype(np.float64)
    B, T, HQ, d = q.shape
    H = seqs[0][0].shape[0]
    worst = 0.0
    for b in range(B):
        for t in range(T):
            seen = max(0, lengths[b] - T + t + 1)
            for h in range(HQ):
                K, V = (x[h // (HQ // H)] for x in seqs[b])
                idx = np.arange(min(seen, K.shape[0]))
                if lists is not None:
                    mine = lists[b, t, h // (HQ // H)]
                    idx = idx[np.isin(idx // P, mine[mine >= 0])]
                ref, bound = F.attend(q[b, t, h], K[idx], V[idx], scale, alpha)
                err = np.abs(o[b, t, h] - ref)
                assert np.isfinite(o[b, t, h]).all(), (b, t, h)
                assert (err <= bound).all(), (b, t, h, float((err / np.maximum(bound, 1e-30)).max()))
                worst = max(worst, float((err / np.maximum(bound, 1e-30)).max(initial=0.0)))
    return worst


# ---- storing and reading back ----------------------------------------------------
@pytest.mark.parametrize("d,P,dtype,T,start,count", [
    (128, 64, torch.bfloat16, 1, (0, 63, 64, 200), None),
    (128, 16, torch.float32, 37, (0, 5, 16), (37, 11, 0)),
    (64, 32, torch.bfloat16, 70, (31, 0), (70, 1)),
    (96, 128, torch.float32, 130, (1,), None),
    (32, 16, torch.bfloat16, 17, (15, 3), (17, 2)),
])
def test_write_is_the_format(cuda, d, P, dtype, T, start, count):
    B, H = len(start), 3
    count = tuple(count or [T] * B)
    cache, table = fresh(B, [s + T for s in start], H, d, P, fill=0xA5)
    before, before_b = cache.pool.cpu().numpy().copy(), cache.bounds.cpu().numpy().copy()
    # pages whose first slot is not written keep their bounds: give them some
    before_b[:, :, :d], before_b[:, :, d: 2 * d] = 5, -7
    before_b[:, :, 2 * d: 2 * d + 4] = np.frombuffer(np.int32(-6).tobytes(), np.int8)
    cache.bounds.copy_(torch.from_numpy(before_b))
    g = torch.Generator().manual_seed(1)
    kv = torch.randn(B, T, H, 2, d, generator=g).to(dtype).cuda()
    K, V = kv[:, :, :, 0], kv[:, :, :, 1]                     # strided: one projection's halves
    sa().cache_write(K, V, cache, dev(table), dev(start), dev(count))
    want, want_b = before.copy(), before_b.copy()
    k, v = num(K), num(V)
    for b in range(B):
        top, low = {}, {}
        for t in range(count[b]):
            page, slot = divmod(start[b] + t, P)
            for h in range(H):
                F.encode_token(want, table[b, page], h, slot, d, P, k[b, t, h], v[b, t, h])
            top[page] = np.maximum(top.get(page, -np.inf), k[b, t])
            low[page] = np.minimum(low.get(page, np.inf), k[b, t])
        for page in top:
            rec = want_b[table[b, page]]
            if page * P < start[b]:
                top[page] = np.maximum(top[page], 5 * 2.0 ** -6)
                low[page] = np.minimum(low[page], -7 * 2.0 ** -6)
            up, lo, e = F.bounds_codes(top[page].astype(np.float64), low[page].astype(np.float64))
            rec[:, :d], rec[:, d: 2 * d] = up, lo
            rec[:, 2 * d: 2 * d + 4] = e[:, None].view(np.int8).reshape(H, 4)
    got, got_b = cache.pool.cpu().numpy(), cache.bounds.cpu().numpy()
    assert np.array_equal(got, want)
    assert np.array_equal(got_b[:, :, : 2 * d + 4], want_b[:, :, : 2 * d + 4])
    for out_dtype in (torch.float32, torch.bfloat16):
        rk, rv = sa().cache_read(cache, dev(table), dev(start), T, dev(count), dtype=out_dtype)
        assert rk.dtype == rv.dtype == out_dtype and rk.shape == (B, T, H, d)
        ek, ev = F.decode(want, d, P)
        for b in range(B):
            for t in range(T):
                page, slot = divmod(start[b] + t, P)
                for r, e in ((rk, ek), (rv, ev)):
                    ref = e[table[b, page], :, slot] if t < count[b] else np.zeros((H, d))
                    assert torch.equal(r[b, t].cpu(), torch.from_numpy(ref.astype(np.float32)).to(out_dtype))
    ids = np.unique(table[table >= 0])
    up, lo = sa().cache_bounds(cache, dev(ids))
    unit = np.exp2(got_b[ids][:, :, 2 * d: 2 * d + 4].copy().view(np.int32).astype(np.float32))
    assert np.array_equal(num(up), got_b[ids][:, :, :d] * unit)
    assert np.array_equal(num(lo), got_b[ids][:, :, d: 2 * d] * unit)
    assert sa().device_error() == 0


def test_one_by_one_equals_at_once(cuda):
    B, H, d, P, T = 2, 2, 64, 16, 45
    g = torch.Generator().manual_seed(2)
    K = torch.randn(B, T, H, d, generator=g)
    K[:, ::7] *= 30.0                                         # the bounds' unit grows as tokens come in
    K, V = K.cuda(), torch.randn(B, T, H, d, generator=g).cuda()
    one, table = fresh(B, [T, T], H, d, P, fill=0)
    all_, _ = fresh(B, [T, T], H, d, P, fill=0)
    sa().cache_write(K, V, all_, dev(table), dev([0, 0]))
    for t in range(T):
        sa().cache_write(K[:, t: t + 1], V[:, t: t + 1], one, dev(table), dev([t, t]))
    assert torch.equal(one.pool, all_.pool) and torch.equal(one.bounds, all_.bounds)
    up, lo = sa().cache_bounds(all_, dev(table[0, :2]))
    k = K[0, : 2 * P].reshape(2, P, H, d)
    assert (up >= k.amax(1)).all() and (lo <= k.amin(1)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_values_out_of_the_ordinary(cuda, dtype):
    d, P = 128, 16
    x = torch.randn(1, 8, 1, d)
    x[0, 0, 0, 3] = float("nan")
    x[0, 1, 0, 40] = float("inf")
    x[0, 1, 0, 70] = -float("inf")
    x[0, 2] = 0.0
    x[0, 3] = 7.25
    x[0, 4] *= 1e-8
    x[0, 5] *= 1e30
    x[0, 6] += 1000.0
    x = x.to(dtype).cuda()
    cache, table = fresh(1, [8], 1, d, P)
    sa().cache_write(x, x, cache, dev(table), dev([0]))
    k, v = sa().cache_read(cache, dev(table), dev([0]), 8, dtype=torch.float32)
    want = cache.pool.cpu().numpy().copy()
    for t in range(8):
        F.encode_token(want, table[0, 0], 0, t, d, P, num(x)[0, t, 0], num(x)[0, t, 0])
    ek, ev = F.decode(want, d, P)
    for got, e in ((k, ek), (v, ev)):
        np.testing.assert_array_equal(num(got)[0, :, 0], e[table[0, 0], 0, :8].astype(np.float32))
    assert torch.isnan(k[0, 0, 0, :32]).all() and torch.isfinite(k[0, 0, 0, 32:]).all()
    assert torch.isfinite(k[0, 1:]).all()
    up, lo = sa().cache_bounds(cache, dev(table[0, :1]))
    ref = torch.nan_to_num(x.float(), nan=0.0).clamp(-65504, 65504)[0, :, 0]
    assert (up[0, 0] >= ref.amax(0)).all() and (lo[0, 0] <= ref.amin(0)).all()


def test_places_outside_are_left_alone_and_reported(cuda):
    d, P, H = 64, 16, 2
    cache, table = fresh(2, [32, 32], H, d, P, fill=3)
    table = table[:, :2].copy()
    table[0, 1] = cache.pool.shape[0]                         # outside the pool
    table[1, 0] = -1
    before = cache.pool.clone()
    x = torch.randn(2, 40, H, d).bfloat16().cuda()
    sa().device_error()
    sa().cache_write(x, x, cache, dev(table), dev([0, -4]))   # and past the table's end, and before its start
    assert sa().device_error() == INVALID
    changed = (cache.pool != before).flatten(1).any(1).nonzero().flatten().tolist()
    assert sorted(changed) == sorted([int(table[0, 0]), int(table[1, 1])])
    k, v = sa().cache_read(cache, dev(table), dev([0, -4]), 40, dtype=torch.float32)
    assert sa().device_error() == INVALID
    assert (k[0, 16:] == 0).all() and (k[1, :20] == 0).all() and (k[1, 36:] == 0).all()
    assert (k[0, :16] != 0).any() and (k[1, 20:36] != 0).any()
    up, lo = sa().cache_bounds(cache, dev([int(table[0, 0]), -1, 10 ** 6]))
    assert sa().device_error() == INVALID and (up[1:] == 0).all() and (lo[1:] == 0).all()


# ---- attention -------------------------------------------------------------------
CASES = [
    # B, T, HQ, H, d, P, lengths
    (1, 1, 1, 1, 128, 64, [1]),
    (3, 1, 8, 2, 128, 64, [65, 17, 640]),
    (2, 1, 4, 4, 64, 16, [300, 16]),
    (2, 1, 40, 2, 96, 32, [129, 31]),
    (1, 1, 7, 1, 32, 128, [515]),
    (2, 3, 6, 2, 128, 16, [50, 3]),
    (2, 5, 8, 2, 64, 64, [4, 70]),            # the first sequence's first query sees nothing
    (3, 2, 2, 2, 128, 32, [0, 1, 33]),
    (1, 33, 12, 3, 128, 64, [100]),
    (1, 64, 4, 2, 64, 16, [64]),
    (1, 130, 8, 2, 128, 32, [333]),
    (1, 1, 16, 2, 128, 64, [4500]),
    (6, 1, 8, 8, 128, 64, [2000, 1, 700, 0, 64, 1333]),
]


@pytest.mark.parametrize("alpha", [1.0, 1.5])
@pytest.mark.parametrize("B,T,HQ,H,d,P,lengths", CASES)
def test_attention(cuda, B, T, HQ, H, d, P, lengths, alpha):
    cache, table, seqs = filled(B, lengths, H, d, P, seed=B + T + HQ, k_scale=1.5)
    q = torch.randn(B, T, HQ, d, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    o = sa().cache_attention(q, cache, dev(table), dev(lengths), alpha=alpha)
    assert o.dtype == torch.bfloat16 and o.shape == q.shape
    check_attention(o, q, seqs, lengths, P, alpha, d ** -0.5)
    assert sa().device_error() == 0


@pytest.mark.parametrize("alpha", [1.05, 1.25, 1.33, 2.0, 3.0])
def test_other_alphas(cuda, alpha):
    lengths = [700, 33]
    cache, table, seqs = filled(2, lengths, 2, 64, 32, seed=11, k_scale=2.0)
    q = torch.randn(2, 2, 6, 64, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    o = sa().cache_attention(q, cache, dev(table), dev(lengths), alpha=alpha)
    check_attention(o, q, seqs, lengths, 32, alpha, 64 ** -0.5)


@pytest.mark.parametrize("alpha", [1.0, 1.5])
@pytest.mark.parametrize("q_scale,k_scale,v_scale,v_shift,sm_scale", [
    (1.0, 1.0, 1e-6, 0.0, None),              # values near fp16's smallest steps
    (1.0, 1.0, 3000.0, 0.0, None),
    (1.0, 1.0, 1.0, 500.0, None),             # offsets far above the scales
    (1e-20, 1.0, 1.0, 0.0, 1e20),
    (1e20, 1.0, 1.0, 0.0, 1e-20),
    (40.0, 3.0, 1.0, 0.0, None),              # one key takes all
    (1.0, 1.0, 1.0, 0.0, -0.1),
    (1.0, 1.0, 1.0, 0.0, 0.0),
])
def test_magnitudes(cuda, alpha, q_scale, k_scale, v_scale, v_shift, sm_scale):
    lengths = [401, 90]
    cache, table, seqs = filled(2, lengths, 2, 128, 64, seed=3, k_scale=k_scale, v_scale=v_scale, v_shift=v_shift)
    q = (torch.randn(2, 1, 8, 128, generator=torch.Generator().manual_seed(5)) * q_scale).bfloat16().cuda()
    o = sa().cache_attention(q, cache, dev(table), dev(lengths), sm_scale=sm_scale, alpha=alpha)
    scale = 128 ** -0.5 if sm_scale is None else sm_scale
    check_attention(o, q, seqs, lengths, 64, alpha, scale)


@pytest.mark.parametrize("alpha", [1.0, 1.5])
def test_values_of_very_different_size_in_one_sequence(cuda, alpha):
    B, H, d, P, n = 1, 2, 128, 64, 640
    cache, table = fresh(B, [n], H, d, P)
    g = torch.Generator().manual_seed(9)
    K, V = (torch.randn(B, n, H, d, generator=g).cuda() for _ in range(2))
    V = V * torch.logspace(-5, 4, n).cuda()[None, :, None, None]
    sa().cache_write(K, V, cache, dev(table), dev([0]))
    k, v = F.decode(cache.pool.cpu().numpy(), d, P)
    seqs = [tuple(x[table[0, :10]].transpose(1, 0, 2, 3).reshape(H, -1, d) for x in (k, v))]
    q = torch.randn(B, 1, 8, d, generator=g).bfloat16().cuda()
    o = sa().cache_attention(q, cache, dev(table), dev([n]), alpha=alpha)
    check_attention(o, q, seqs, [n], P, alpha, d ** -0.5)


@pytest.mark.parametrize("alpha", [1.0, 1.5])
def test_nan_in_places_nobody_sees(cuda, alpha):
    """Pages of other sequences, slots past the end, and tokens after a query
    hold NaN: nothing of it shows.  A token that is seen shows in its group."""
    B, T, HQ, H, d, P = 1, 4, 4, 2, 128, 64
    lengths = [90]
    cache, table, seqs = filled(B, lengths, H, d, P, seed=4, fill=255)
    bad = torch.zeros(1, 2, H, d, device="cuda").bfloat16()
    bad[..., 5] = float("nan")
    bad[..., 69] = float("inf")
    sa().cache_write(bad, bad, cache, dev(table), dev([88]))  # the last two tokens; queries 0 and 1 stand before them
    q = torch.randn(B, T, HQ, d, generator=torch.Generator().manual_seed(6)).bfloat16().cuda()
    o = sa().cache_attention(q, cache, dev(table), dev(lengths), alpha=alpha)
    clean = [tuple(x[:, :88] for x in seqs[0])]
    check_attention(o[:, :2], q[:, :2], clean, [88], P, alpha, d ** -0.5)
    assert torch.isnan(o[:, 2:]).all()                        # NaN keys: NaN scores, a NaN row
    values = torch.zeros(1, 2, H, d, device="cuda").bfloat16()
    sa().cache_write(values, bad, cache, dev(table), dev([88]))
    if alpha != 1.0:
        q[:, 2:] = 0.0                                        # equal weights: a NaN of weight 0 need not show
    o = sa().cache_attention(q, cache, dev(table), dev(lengths), alpha=alpha)
    check_attention(o[:, :2], q[:, :2], clean, [88], P, alpha, d ** -0.5)
    assert torch.isnan(o[:, 2:, :, :32]).all() and torch.isfinite(o[:, 2:, :, 32:]).all()


def test_nan_query_is_its_own(cuda):
    lengths = [77, 20]
    cache, table, seqs = filled(2, lengths, 1, 64, 16, seed=4)
    q = torch.randn(2, 2, 8, 64, generator=torch.Generator().manual_seed(6)).bfloat16().cuda()
    q[0, 1, 3, 7] = float("nan")
    q[1, 0, 2, 9] = float("inf")
    for alpha in (1.0, 1.5):
        o = sa().cache_attention(q, cache, dev(table), dev(lengths), alpha=alpha)
        assert torch.isnan(o[0, 1, 3]).all() and torch.isnan(o[1, 0, 2]).all()
        o, clean = o.clone(), q.clone()
        for b, t, h in ((0, 1, 3), (1, 0, 2)):
            clean[b, t, h] = 0.0
            o[b, t, h] = sa().cache_attention(clean, cache, dev(table), dev(lengths), alpha=alpha)[b, t, h]
        check_attention(o, clean, seqs, lengths, 16, alpha, 64 ** -0.5)


@pytest.mark.parametrize("alpha", [1.0, 1.5])
@pytest.mark.parametrize("T,HQ,H,d,P", [(1, 8, 2, 128, 64), (3, 4, 2, 64, 16), (2, 20, 1, 96, 32)])
def test_listed_pages(cuda, alpha, T, HQ, H, d, P):
    lengths = [9 * P + 3, P - 1, 4 * P]
    B, keep = 3, 5
    cache, table, seqs = filled(B, lengths, H, d, P, seed=7, k_scale=1.5)
    g = np.random.RandomState(0)
    lists = np.full((B, T, H, keep), -1, np.int32)
    for b in range(B):
        for t in range(T):
            for h in range(H):
                n = -(-lengths[b] // P)
                some = g.permutation(n + 1)[: g.randint(0, min(keep, n + 1) + 1)]   # any order, a page past the end too
                lists[b, t, h, g.permutation(keep)[: len(some)]] = some
    lists[0, 0, 0] = -1                                       # a query without pages
    lists[1, 0, 0, 0] = 10 ** 6                               # past the table
    q = torch.randn(B, T, HQ, d, generator=torch.Generator().manual_seed(8)).bfloat16().cuda()
    o = sa().cache_attention(q, cache, dev(table), dev(lengths), alpha=alpha, pages=dev(lists))
    check_attention(o, q, seqs, lengths, P, alpha, d ** -0.5, lists)
    assert (o[0, 0, : HQ // H] == 0).all()


def test_unreadable_pages_are_not_seen_and_reported(cuda):
    lengths = [100]
    for alpha in (1.0, 1.5):
        cache, table, seqs = filled(1, lengths, 2, 64, 16, seed=2)
        bad = table.copy()
        bad[0, 1], bad[0, 4] = cache.pool.shape[0] + 5, -3
        keepers = np.array([0, 2, 3, 5, 6], np.int32)
        q = torch.randn(1, 1, 4, 64, generator=torch.Generator().manual_seed(8)).bfloat16().cuda()
        sa().device_error()
        o = sa().cache_attention(q, cache, dev(bad), dev(lengths), alpha=alpha)
        assert sa().device_error() == INVALID
        check_attention(o, q, seqs, lengths, 16, alpha, 64 ** -0.5, np.broadcast_to(keepers, (1, 1, 2, 5)))
        # a length past the table's end stops at it
        short = table[:, :3].copy()
        o = sa().cache_attention(q, cache, dev(short), dev([100]), alpha=alpha)
        sa().device_error()
        check_attention(o, q, [tuple(x[:, :48] for x in seqs[0])], [100], 16, alpha, 64 ** -0.5)


@pytest.mark.parametrize("alpha", [1.0, 1.5])
def test_strides_streams_graphs_and_repeats(cuda, alpha):
    B, T, HQ, H, d, P = 2, 2, 8, 2, 128, 64
    lengths = [1500, 321]
    cache, table, seqs = filled(B, lengths, H, d, P, seed=7)
    tab, n = dev(table), dev(lengths)
    wide = torch.randn(B, HQ, T, d + 8, generator=torch.Generator().manual_seed(8)).bfloat16().cuda()
    q = wide.permute(0, 2, 1, 3)[..., 4: 4 + d]               # strides of every dimension, rows off 16 bytes
    want = sa().cache_attention(q.contiguous(), cache, tab, n, alpha=alpha)
    check_attention(want, q, seqs, lengths, P, alpha, d ** -0.5)
    for _ in range(3):
        assert torch.equal(sa().cache_attention(q, cache, tab, n, alpha=alpha), want)
    wide_table = torch.full((B, 50), -1, dtype=torch.int64, device="cuda")
    wide_table[:, : table.shape[1]] = tab
    assert torch.equal(sa().cache_attention(q, cache, wide_table[:, : table.shape[1]], n.long(), alpha=alpha), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sa().cache_attention(q, cache, tab, n, alpha=alpha)
        pages = sa().select_pages(q, cache, tab, n, 4)
        some = sa().cache_attention(q, cache, tab, n, alpha=alpha, pages=pages)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    qs = q.clone()
    with torch.cuda.graph(graph):
        got2 = sa().cache_attention(qs, cache, tab, n, alpha=alpha)
        pages2 = sa().select_pages(qs, cache, tab, n, 4)
        some2 = sa().cache_attention(qs, cache, tab, n, alpha=alpha, pages=pages2)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got2, want) and torch.equal(pages2, pages) and torch.equal(some2, some)
    # the lengths live on the device: a captured call follows them
    n.fill_(200)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got2, sa().cache_attention(q, cache, tab, n, alpha=alpha))


def test_nothing_to_do(cuda):
    cache = sa().new_cache(2, 2, 64, 16)
    tab = dev(np.zeros((0, 3)))
    q = torch.zeros(0, 1, 4, 64, device="cuda").bfloat16()
    assert sa().cache_attention(q, cache, tab, dev(np.zeros(0))).shape == q.shape
    assert sa().select_pages(q, cache, tab, dev(np.zeros(0)), 3).shape == (0, 1, 2, 3)
    q = torch.zeros(2, 0, 4, 64, device="cuda").bfloat16()
    tab = dev(np.zeros((2, 3)))
    assert sa().cache_attention(q, cache, tab, dev([5, 5])).shape == q.shape
    sa().cache_write(q[:, :, :2], q[:, :, :2], cache, tab, dev([0, 0]))
    k, v = sa().cache_read(cache, tab, dev([0, 0]), 0)
    assert k.shape == v.shape == (2, 0, 2, 64)
    q = torch.randn(2, 3, 4, 64, device="cuda").bfloat16()
    none = torch.zeros(2, 0, dtype=torch.int32, device="cuda")       # sequences without a page
    assert (sa().cache_attention(q, cache, none, dev([0, 0])) == 0).all()
    assert (sa().cache_attention(q, cache, none, dev([0, 0]), alpha=1.5) == 0).all()
    assert (sa().select_pages(q, cache, none, dev([0, 0]), 2) == -1).all()
    up, lo = sa().cache_bounds(cache, dev(np.zeros(0)))
    assert up.shape == lo.shape == (0, 2, 64)


# ---- selecting pages -------------------------------------------------------------
@pytest.mark.parametrize("T,HQ,H,d,P,keep,lengths", [
    (1, 8, 2, 128, 64, 4, [1000, 64, 65, 0]),
    (3, 4, 4, 64, 16, 7, [500, 2]),
    (2, 12, 1, 96, 32, 1, [320, 97]),
    (1, 5, 1, 32, 16, 33, [4000]),
    (1, 32, 2, 128, 16, 64, [9000]),
    (2, 2, 2, 64, 128, 50, [700, 129]),
])
def test_select(cuda, T, HQ, H, d, P, keep, lengths):
    B = len(lengths)
    cache, table, _ = filled(B, lengths, H, d, P, seed=13)
    q = torch.randn(B, T, HQ, d, generator=torch.Generator().manual_seed(8)).bfloat16().cuda()
    q[0, 0, 0] = 0.0
    got = sa().select_pages(q, cache, dev(table), dev(lengths), keep)
    bounds, qn = cache.bounds.cpu().numpy(), num(q)
    for b in range(B):
        for t in range(T):
            want = F.select(qn[b], bounds, table[b], lengths[b], t, T, P, keep, HQ // H)
            assert np.array_equal(got[b, t].cpu().numpy(), want), (b, t)
    assert got.dtype == torch.int32 and sa().device_error() == 0


def test_select_ties_and_the_unordinary(cuda):
    H, d, P, n = 1, 64, 16, 40
    cache, table = fresh(1, [n * P], H, d, P)
    K = torch.randn(1, P, H, d).repeat(1, n, 1, 1).bfloat16().cuda()          # every page alike
    K[:, 25 * P: 26 * P] *= 2.0
    sa().cache_write(K, K, cache, dev(table), dev([0]))
    q = torch.randn(1, 1, 4, d).bfloat16().cuda()
    pages = sa().select_pages(q, cache, dev(table), dev([n * P]), 6).flatten().tolist()
    assert pages == [0, 1, 2, 3, 25, 39]                                      # ties to the earlier page
    q[0, 0, 1, 3] = float("nan")                                              # one head of the group: the others choose
    assert sa().select_pages(q, cache, dev(table), dev([n * P]), 6).flatten().tolist() == pages
    q[...] = float("nan")
    assert sa().select_pages(q, cache, dev(table), dev([n * P]), 6).flatten().tolist() == [0, 1, 2, 3, 4, 39]
    bad = table.copy()
    bad[0, 1] = 10 ** 6
    q = torch.randn(1, 1, 4, d).bfloat16().cuda()
    sa().device_error()
    assert sa().select_pages(q, cache, dev(bad), dev([n * P]), 6).flatten().tolist() == [0, 2, 3, 4, 25, 39]
    assert sa().device_error() == INVALID


def test_selecting_all_pages_is_full_attention(cuda):
    lengths = [700, 90]
    for alpha in (1.0, 1.5):
        cache, table, seqs = filled(2, lengths, 2, 128, 32, seed=3)
        q = torch.randn(2, 2, 8, 128, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
        pages = sa().select_pages(q, cache, dev(table), dev(lengths), 30)
        o = sa().cache_attention(q, cache, dev(table), dev(lengths), alpha=alpha, pages=pages)
        check_attention(o, q, seqs, lengths, 32, alpha, 128 ** -0.5)


# ---- refusals --------------------------------------------------------------------
def test_refusals(cuda):
    m = sa()
    cache = m.new_cache(4, 2, 64, 16)
    tab, n = dev(np.zeros((1, 2))), dev([5])
    q = torch.zeros(1, 1, 4, 64, device="cuda").bfloat16()
    kv = torch.zeros(1, 3, 2, 64, device="cuda").bfloat16()
    with pytest.raises(TypeError):
        m.cache_attention(q.float(), cache, tab, n)
    with pytest.raises(TypeError):
        m.cache_attention(q, cache, tab.float(), n)
    with pytest.raises(ValueError):
        m.cache_attention(q[:, :, :3], cache, tab, n)                # heads no multiple of the cache's
    with pytest.raises(ValueError):
        m.cache_attention(q[..., :32], cache, tab, n)                # another head_dim
    with pytest.raises(ValueError):
        m.cache_attention(q, cache, tab, dev([5, 5]))
    with pytest.raises(ValueError):
        m.cache_attention(q, cache, dev(np.zeros((2, 2))), n)
    for alpha in (0.5, 1.01, 3.5, float("nan")):
        with pytest.raises(ValueError):
            m.cache_attention(q, cache, tab, n, alpha=alpha)
    with pytest.raises(ValueError):
        m.cache_attention(q, cache, tab, n, pages=dev(np.zeros((1, 1, 4, 2))))
    with pytest.raises(ValueError):
        m.cache_attention(q, cache, tab, n, pages=dev(np.zeros((1, 1, 2, 0))))
    with pytest.raises(RuntimeError):
        m.cache_attention(q, cache, tab.cpu(), n)
    with pytest.raises(RuntimeError):
        m.cache_attention(q, cache, tab, n, sm_scale=float("inf"))
    with pytest.raises(ValueError):
        m.select_pages(q, cache, tab, n, 0)
    with pytest.raises(TypeError):
        m.cache_write(kv.half(), kv.half(), cache, tab, dev([0]))
    with pytest.raises(TypeError):
        m.cache_write(kv, kv.float(), cache, tab, dev([0]))
    with pytest.raises(ValueError):
        m.cache_write(kv, kv[:, :2], cache, tab, dev([0]))
    with pytest.raises(ValueError):
        m.cache_write(kv[:, :, :1], kv[:, :, :1], cache, tab, dev([0]))
    with pytest.raises(ValueError):
        m.cache_write(kv, kv, m.KVCache(cache.pool[:, :, :-16], cache.bounds), tab, dev([0]))
    with pytest.raises(TypeError):
        m.cache_read(cache, tab, dev([0]), 3, dtype=torch.float16)
    with pytest.raises(ValueError):
        m.cache_read(cache, tab, dev([0]), -1)


# ---- the paths that sizes choose ---------------------------------------------------
@pytest.mark.parametrize("alpha", [1.0, 1.5])
@pytest.mark.parametrize("T", [1, 3, 40])
@pytest.mark.parametrize("P", [16, 32, 64, 128])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
def test_every_head_dim_and_page_size(cuda, d, P, T, alpha):
    lengths = [T + 171, T]
    cache, table, seqs = filled(2, lengths, 2, d, P, seed=d + P + T, k_scale=1.5)
    q = torch.randn(2, T, 6, d, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    o = sa().cache_attention(q, cache, dev(table), dev(lengths), alpha=alpha)
    check_attention(o, q, seqs, lengths, P, alpha, d ** -0.5)


@pytest.mark.parametrize("alpha", [1.0, 1.5])
@pytest.mark.parametrize("T,HQ", [(1, 4), (2, 8)])
def test_many_sequences(cuda, T, HQ, alpha):
    """More sequences than a block of threads, their work cut into equal runs."""
    B, H, d, P = 330, 2, 32, 16
    g = np.random.RandomState(3)
    lengths = [int(x) for x in g.randint(0, 60, B)]
    lengths[7], lengths[300], lengths[329] = 1500, 900, 1100
    cache, table, seqs = filled(B, lengths, H, d, P, seed=1)
    q = torch.randn(B, T, HQ, d, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    o = sa().cache_attention(q, cache, dev(table), dev(lengths), alpha=alpha)
    check_attention(o, q, seqs, lengths, P, alpha, d ** -0.5)


@pytest.mark.parametrize("alpha,q_scale", [(1.5, 1e-3), (1.25, 0.1), (1.05, 1.0), (3.0, 1e-3)])
def test_wide_support(cuda, alpha, q_scale):
    """More support than a row's list holds."""
    lengths = [3000]
    cache, table, seqs = filled(1, lengths, 1, 64, 64, seed=6)
    q = (torch.randn(1, 1, 3, 64, generator=torch.Generator().manual_seed(5)) * q_scale).bfloat16().cuda()
    o = sa().cache_attention(q, cache, dev(table), dev(lengths), alpha=alpha)
    check_attention(o, q, seqs, lengths, 64, alpha, 64 ** -0.5)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("T,HQ,H,P,lengths", [
    (64, 1, 1, 64, [64, 200]),
    (40, 4, 2, 16, [1000, 25]),              # the second sequence's first queries see nothing
    (257, 3, 1, 128, [700, 257]),
    (130, 2, 2, 32, [130, 0]),
    (9, 64, 2, 64, [5000, 9]),
])
def test_chunks(cuda, d, T, HQ, H, P, lengths):
    cache, table, seqs = filled(2, lengths, H, d, P, seed=T, k_scale=1.2)
    wide = torch.randn(2, HQ, T, d + 8, generator=torch.Generator().manual_seed(8)).bfloat16().cuda()
    for q in (wide[..., :d].permute(0, 2, 1, 3).contiguous(), wide.permute(0, 2, 1, 3)[..., 4: 4 + d]):
        o = sa().cache_attention(q, cache, dev(table), dev(lengths))
        check_attention(o, q, seqs, lengths, P, 1.0, d ** -0.5)
    assert torch.equal(sa().cache_attention(q, cache, dev(table), dev(lengths)), o)
    assert sa().device_error() == 0


@pytest.mark.parametrize("d", [64, 128])
def test_chunk_nan_in_places_nobody_sees(cuda, d):
    T, HQ, H, P = 96, 2, 1, 64
    lengths = [300]
    cache, table, seqs = filled(1, lengths, H, d, P, seed=4, fill=255)
    bad = torch.zeros(1, 1, H, d, device="cuda").bfloat16()
    bad[..., 5] = float("nan")
    zeros = torch.zeros_like(bad)
    sa().cache_write(zeros, bad, cache, dev(table), dev([290]))        # query 86 stands there
    q = torch.randn(1, T, HQ, d, generator=torch.Generator().manual_seed(6)).bfloat16().cuda()
    q[0, 3, 1, 7] = float("nan")
    o = sa().cache_attention(q, cache, dev(table), dev(lengths))
    assert torch.isnan(o[0, 3, 1]).all()
    o, clean = o.clone(), q.clone()
    o[0, 3, 1], clean[0, 3, 1] = o[0, 3, 0], q[0, 3, 0]
    check_attention(o[:, :86], clean[:, :86], seqs, [290], P, 1.0, d ** -0.5)
    assert torch.isnan(o[0, 86:, :, :32]).all() and torch.isfinite(o[0, 86:, :, 32:]).all()
    sa().cache_write(bad, zeros, cache, dev(table), dev([290]))        # a NaN key: its rows' scores
    o = sa().cache_attention(clean, cache, dev(table), dev(lengths))
    check_attention(o[:, :86], clean[:, :86], seqs, [290], P, 1.0, d ** -0.5)
    assert torch.isnan(o[0, 86:]).all()


@pytest.mark.parametrize("v_scale,v_shift,k_scale,q_scale,sm_scale", [
    (1e-6, 0.0, 1.0, 1.0, None), (3000.0, 0.0, 1.0, 1.0, None), (1.0, 500.0, 1.0, 1.0, None),
    (1.0, 0.0, 3.0, 40.0, None), (1.0, 0.0, 1.0, 1e-20, 1e20), (1.0, 0.0, 1.0, 1.0, -0.1), (1.0, 0.0, 1.0, 1.0, 0.0),
])
def test_chunk_magnitudes(cuda, v_scale, v_shift, k_scale, q_scale, sm_scale):
    lengths = [401]
    cache, table, seqs = filled(1, lengths, 1, 128, 64, seed=3, k_scale=k_scale, v_scale=v_scale, v_shift=v_shift)
    q = (torch.randn(1, 70, 1, 128, generator=torch.Generator().manual_seed(5)) * q_scale).bfloat16().cuda()
    o = sa().cache_attention(q, cache, dev(table), dev(lengths), sm_scale=sm_scale)
    check_attention(o, q, seqs, lengths, 64, 1.0, 128 ** -0.5 if sm_scale is None else sm_scale)


def test_values_at_the_top_of_the_range(cuda):
    """A group over all of fp16's range: its largest value rounds past fp16."""
    P, d, n = 64, 64, 128
    V = torch.linspace(-65504, 65504, d).repeat(1, n, 1, 1).cuda()
    K = torch.randn(1, n, 1, d, generator=torch.Generator().manual_seed(1)).cuda()
    cache, table = fresh(1, [n], 1, d, P)
    sa().cache_write(K, V, cache, dev(table), dev([0]))
    _, v = F.decode(cache.pool.cpu().numpy(), d, P)
    v = v[table[0, 0], 0, 0]
    for T in (1, 80):
        q = torch.randn(1, T, 1, d, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
        o = num(sa().cache_attention(q, cache, dev(table), dev([n])))
        # every value is the same token's: the output is it, within fp16's and bf16's roundings
        assert np.isfinite(o).all() and (np.abs(o - v) <= 2.0 ** -7 * np.abs(v) + 1e-3).all()


def test_chunk_unreadable_pages(cuda):
    lengths = [200]
    cache, table, seqs = filled(1, lengths, 1, 64, 16, seed=2)
    bad = table.copy()
    bad[0, 1], bad[0, 4], bad[0, 12] = cache.pool.shape[0] + 5, -3, 1 << 30
    q = torch.randn(1, 64, 1, 64, generator=torch.Generator().manual_seed(8)).bfloat16().cuda()
    sa().device_error()
    o = sa().cache_attention(q, cache, dev(bad), dev(lengths))
    assert sa().device_error() == INVALID
    keepers = np.array([i for i in range(13) if i not in (1, 4, 12)], np.int32)
    check_attention(o, q, seqs, lengths, 16, 1.0, 64 ** -0.5, np.broadcast_to(keepers, (1, 64, 1, len(keepers))))
    short = table[:, :7].copy()
    o = sa().cache_attention(q, cache, dev(short), dev(lengths))
    assert sa().device_error() == 0                       # a length past the table's end is no error
    check_attention(o, q, [tuple(x[:, :112] for x in seqs[0])], lengths, 16, 1.0, 64 ** -0.5)


def test_more_pages_than_a_block_keeps(cuda):
    H, d, P, n = 1, 32, 16, 70000
    cache, table, _ = filled(1, [n], H, d, P, seed=13)
    q = torch.randn(1, 1, 2, d, generator=torch.Generator().manual_seed(8)).bfloat16().cuda()
    got = sa().select_pages(q, cache, dev(table), dev([n]), 40)
    want = F.select(num(q)[0], cache.bounds.cpu().numpy(), table[0], n, 0, 1, P, 40, 2)
    assert np.array_equal(got[0, 0].cpu().numpy(), want)


def test_pools_past_32_bits(cuda):
    """Records beyond 4 GiB of a pool."""
    H, d, P, n = 8, 128, 128, 300
    pages = 30000                                             # 20 KiB a record: 4.9 GB
    cache = sa().new_cache(pages, H, d, P)
    table = np.array([[pages - 1, 5, pages - 7, -1]], np.int32)
    g = torch.Generator().manual_seed(3)
    K, V = (torch.randn(1, n, H, d, generator=g).bfloat16().cuda() for _ in range(2))
    sa().cache_write(K, V, cache, dev(table), dev([0]))
    k, v = (num(x) for x in sa().cache_read(cache, dev(table), dev([0]), n, dtype=torch.float32))
    small = sa().KVCache(cache.pool[[pages - 1, 5, pages - 7]].contiguous(), cache.bounds[[pages - 1, 5, pages - 7]].contiguous())
    other = dev([[0, 1, 2, -1]])
    for a, b in zip(sa().cache_read(small, other, dev([0]), n, dtype=torch.float32), (k, v)):
        assert np.array_equal(num(a), b)
    for T in (1, 20):
        q = torch.randn(1, T, 32, d, generator=g).bfloat16().cuda()
        for alpha in (1.0, 1.5):
            assert torch.equal(sa().cache_attention(q, cache, dev(table), dev([n]), alpha=alpha),
                               sa().cache_attention(q, small, other, dev([n]), alpha=alpha))
        assert torch.equal(sa().select_pages(q, cache, dev(table), dev([n]), 2),
                           sa().select_pages(q, small, other, dev([n]), 2))
    assert k.any() and v.any() and sa().device_error() == 0


def test_select_refuses_too_many_heads(cuda):
    cache = sa().new_cache(2, 1, 32, 16)
    q = torch.zeros(1, 1, 257, 32, device="cuda").bfloat16()
    with pytest.raises(RuntimeError):
        sa().select_pages(q, cache, dev(np.zeros((1, 2))), dev([5]), 1)


def test_launches_are_counted_and_timed(cuda):
    from splash_attention import ops
    lengths = [300]
    cache, table, _ = filled(1, lengths, 2, 64, 16)
    q = torch.randn(1, 1, 4, 64).bfloat16().cuda()
    with ops.profile() as prof:
        sa().cache_attention(q, cache, dev(table), dev(lengths))
        sa().cache_attention(q, cache, dev(table), dev(lengths), alpha=1.5)
        sa().select_pages(q, cache, dev(table), dev(lengths), 2)
    assert {"cache_attention", "cache_entmax", "cache_select"} <= set(prof.result)
    assert all(ms > 0 and n > 0 for ms, n in prof.result.values())


def test_example(cuda):
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "serve_cache.py")
    spec = importlib.util.spec_from_file_location("serve_cache", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    err = m.main(prompt=400, steps=2)
    # a quantisation step is about range/15 of a group's 32 values: a uniform error of 1/sqrt(12)
    # of 4 sigma / 15, 0.08 of a value; attention averages values and sharpens scores
    assert err["keys read back"] < 0.1 and err["values read back"] < 0.1
    assert all(e < 0.6 for e in err.values()), err
