"""The 4-bit cache's operators under PyTorch's own checks of operators and under tracing."""
import numpy as np
import pytest
import torch

from test_cache_gpu import dev, filled, sa

pytestmark = pytest.mark.gpu


def parts():
    lengths = [40, 21]
    cache, table, _ = filled(2, lengths, 2, 64, 16, seed=1, fill=0)
    q = torch.randn(2, 2, 4, 64, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    kv = torch.randn(2, 2, 2, 64, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    return cache, dev(table), dev(lengths), q, kv


@pytest.mark.parametrize("what", ["write", "read", "bounds", "select", "attention", "entmax", "listed"])
def test_opcheck(cuda, what):
    ops = torch.ops.splash_attention
    (pool, bounds), table, lengths, q, kv = parts()
    pages = sa().select_pages(q, sa().KVCache(pool, bounds), table, lengths, 2)
    op, args = {
        "write": (ops.cache_write, (kv, kv, pool, bounds, table, lengths - 2, None)),
        "read": (ops.cache_read, (pool, bounds, table, lengths - 5, 5, None, False)),
        "bounds": (ops.cache_bounds, (bounds, dev([0, 2]))),
        "select": (ops.cache_select, (q, pool, bounds, table, lengths, 2)),
        "attention": (ops.cache_attention, (q, pool, bounds, table, lengths, None, 0.125, 1.0)),
        "entmax": (ops.cache_attention, (q, pool, bounds, table, lengths, None, 0.125, 1.5)),
        "listed": (ops.cache_attention, (q, pool, bounds, table, lengths, pages, 0.125, 1.0)),
    }[what]
    torch.library.opcheck(op.default, args)


def test_traced_steps_equal_eager_ones(cuda):
    """Writing, selecting and attending in one traced function: the write is kept, and kept in order."""
    cache, table, lengths, q, kv = parts()
    one, two = (sa().KVCache(cache.pool.clone(), cache.bounds.clone()) for _ in range(2))

    def step(pool, bounds, q, kv, lengths):
        c = sa().KVCache(pool, bounds)
        before = sa().cache_attention(q, c, table, lengths)
        sa().cache_write(kv, kv, c, table, lengths - 2)
        pages = sa().select_pages(q, c, table, lengths, 2)
        return before, sa().cache_attention(q, c, table, lengths, alpha=1.5, pages=pages)

    want = step(*one, q, kv, lengths)
    got = torch.compile(step, backend="aot_eager", fullgraph=True)(*two, q, kv, lengths)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert torch.equal(one.pool, two.pool) and torch.equal(one.bounds, two.bounds)
    assert not torch.equal(want[0], want[1]) and np.isfinite(want[1].float().cpu().numpy()).all()
