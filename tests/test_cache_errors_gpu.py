"""What the 4-bit cache's operators record is theirs: it neither makes the training
operators raise, nor is it lost to them, and the other way round."""
import numpy as np
import pytest
import torch

from test_cache_gpu import check_attention, dev, filled, sa

pytestmark = pytest.mark.gpu
INVALID, TIMEOUT = 1, 5


def step(n=256, d=64, **kw):
    """A training step: outputs and gradients."""
    g = torch.Generator("cuda").manual_seed(0)
    q, k, v = (torch.randn(1, 2, n, d, generator=g, device="cuda").bfloat16().requires_grad_() for _ in range(3))
    at = torch.arange(n, dtype=torch.int32, device="cuda")
    o = sa().splash_attention(q, k, v, at, at, **kw)
    o.float().square().sum().backward()
    return o.detach(), q.grad, k.grad, v.grad


def misuse(what):
    """A call that meets a place outside the table or the pool."""
    d, P = 64, 16
    cache, table, _ = filled(1, [40], 2, d, P, seed=1)
    tab, bad = dev(table), dev(np.where(table == table[0, 1], 10 ** 6, table))
    q = torch.randn(1, 1, 4, d).bfloat16().cuda()
    many = torch.randn(1, 64, 4, d).bfloat16().cuda()
    if what == "read":
        sa().cache_read(cache, tab, dev([0]), 200)
    elif what == "write":
        x = torch.randn(1, 3, 2, d).bfloat16().cuda()
        sa().cache_write(x, x, cache, tab, dev([4000]))
    elif what == "bounds":
        sa().cache_bounds(cache, dev([-7]))
    elif what == "select":
        sa().select_pages(q, cache, bad, dev([40]), 2)
    else:
        alpha = 1.5 if what == "entmax" else 1.0
        sa().cache_attention(many if what == "chunk" else q, cache, bad, dev([40]), alpha=alpha)


@pytest.mark.parametrize("mode", [{}, {"tau_mode": "exact", "ref_tile_load": False}])
@pytest.mark.parametrize("what", ["read", "write", "bounds", "select", "attention", "entmax", "chunk"])
def test_training_goes_on(cuda, what, mode):
    assert sa().device_error() == 0
    want = step(**mode)
    misuse(what)
    for _ in range(3):                                        # (an error would be raised a call later)
        for a, b in zip(step(**mode), want):
            assert torch.equal(a, b)
        torch.cuda.synchronize()
    assert sa().device_error() == INVALID                     # and is still there to be read
    assert sa().device_error() == 0


def test_both_are_reported(cuda):
    from splash_attention import ops
    assert sa().device_error() == 0
    misuse("read")
    ops.wait_probe(1000)
    assert [sa().device_error() for _ in range(3)] == [TIMEOUT, INVALID, 0]


def test_a_training_timeout_is_not_the_caches(cuda):
    from splash_attention import ops
    lengths = [3000, 90]
    cache, table, seqs = filled(2, lengths, 2, 128, 64, seed=3)
    for T, alpha in ((1, 1.0), (1, 1.5), (70, 1.0)):
        q = torch.randn(2, T, 4, 128, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
        ops.wait_probe(1000)
        o = sa().cache_attention(q, cache, dev(table), dev(lengths), alpha=alpha)
        assert [sa().device_error(), sa().device_error()] == [TIMEOUT, 0]
        check_attention(o, q, seqs, lengths, 64, alpha, 128 ** -0.5)


def test_a_wait_that_gives_up_is_reported(cuda):
    """The cache's kernels' bounded wait, on a barrier that nobody completes; training and the cache go on."""
    import ctypes
    from splash_attention import _lib as L
    assert sa().device_error() == 0
    want = step()
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert L.lib().asa_cache_wait_probe(0, stream) == INVALID
    assert L.lib().asa_cache_wait_probe(1000, stream) == 0
    for _ in range(3):
        for a, b in zip(step(), want):
            assert torch.equal(a, b)
        torch.cuda.synchronize()
    assert [sa().device_error(), sa().device_error()] == [TIMEOUT, 0]
    misuse("read")                                            # a time-out is not lost to what came before it
    assert L.lib().asa_cache_wait_probe(1, stream) == 0
    assert [sa().device_error(), sa().device_error()] == [TIMEOUT, 0]
    for T in (1, 70):
        cache, table, seqs = filled(1, [300], 2, 64, 16, seed=3)
        q = torch.randn(1, T, 4, 64, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
        o = sa().cache_attention(q, cache, dev(table), dev([300]))
        check_attention(o, q, seqs, [300], 16, 1.0, 64 ** -0.5)
    assert sa().device_error() == 0
