"""The 4-bit cache's operators as PyTorch's dispatcher has them: what they write to is
marked as written."""
import torch

import splash_attention  # noqa: F401  (registers the operators)


def tensors(device, B=2, T=3, H=2, d=64, P=16, pages=5):
    def make(*s, dtype=torch.bfloat16):
        return torch.empty(*s, dtype=dtype, device=device)
    kv = make(B, T, H, d)
    return kv, make(pages, H, P * d * 5 // 4, dtype=torch.uint8), make(pages, H, 2 * d + 16, dtype=torch.int8), \
        make(B, 2, dtype=torch.int32), make(B, dtype=torch.int32)


def test_a_write_counts_as_one():
    """Version counters tell autograd and compilers that a tensor has changed."""
    kv, pool, bounds, table, start = tensors("meta")
    others = (kv, table, start)
    for n in (1, 2):
        torch.ops.splash_attention.cache_write(kv, kv, pool, bounds, table, start, None)
        assert pool._version == bounds._version == n
        assert all(t._version == 0 for t in others)
    torch.ops.splash_attention.cache_read(pool, bounds, table, start, 3, None, True)
    torch.ops.splash_attention.cache_attention(kv, pool, bounds, table, start, None, 0.1, 1.0)
    assert pool._version == bounds._version == 2


def test_writes_in_inference_mode():
    with torch.inference_mode():
        kv, pool, bounds, table, start = tensors("meta")
        torch.ops.splash_attention.cache_write(kv, kv, pool, bounds, table, start, None)
    # a cache made there can be written to outside
    torch.ops.splash_attention.cache_write(tensors("meta")[0], kv, pool, bounds, table, start, None)


def test_saved_and_overwritten_is_noticed():
    """A graph that saved the cache refuses to go backward over a changed one."""
    kv, pool, bounds, table, start = tensors("meta")
    x = torch.ones(5, 2, 1, device="meta", requires_grad=True)
    y = (x * pool).sum()
    torch.ops.splash_attention.cache_write(kv, kv, pool, bounds, table, start, None)
    try:
        y.backward()
    except RuntimeError as e:
        assert "modified by an inplace operation" in str(e)
    else:
        raise AssertionError("the write was not noticed")
