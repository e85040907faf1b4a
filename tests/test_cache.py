"""The 4-bit paged cache without a GPU: the format's own arithmetic, the C ABI's
checks of arguments, the operators' schemas and shapes."""
import ctypes

import numpy as np
import pytest
import torch

import cache_f64 as F
import splash_attention as sa
from splash_attention import _lib as L


def params(**kw):
    p = L.CacheParams(B=2, T=1, heads=8, kv_heads=2, d=128, page_size=64, num_pages=10, table_width=4,
                      dtype=L.DTYPE_BF16, sm_scale=0.1, alpha=1.0)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def workspace(p, keep=0):
    a, s = ctypes.c_size_t(), ctypes.c_size_t()
    rc = L.lib().asa_cache_workspace_bytes(ctypes.byref(p), keep, ctypes.byref(a), ctypes.byref(s))
    return rc, a.value, s.value


@pytest.mark.parametrize("field,value,code", [
    ("B", -1, L.ASA_ERR_INVALID), ("T", -1, L.ASA_ERR_INVALID), ("heads", 7, L.ASA_ERR_INVALID),
    ("heads", 0, L.ASA_ERR_INVALID), ("kv_heads", 0, L.ASA_ERR_INVALID), ("d", 0, L.ASA_ERR_INVALID),
    ("d", 48, L.ASA_ERR_UNSUPPORTED), ("d", 160, L.ASA_ERR_UNSUPPORTED),
    ("page_size", 24, L.ASA_ERR_UNSUPPORTED), ("page_size", 0, L.ASA_ERR_INVALID),
    ("num_pages", -1, L.ASA_ERR_INVALID), ("table_width", -1, L.ASA_ERR_INVALID),
    ("table_width", 1 << 26, L.ASA_ERR_UNSUPPORTED), ("dtype", 5, L.ASA_ERR_INVALID),
    ("sm_scale", float("nan"), L.ASA_ERR_INVALID), ("alpha", 0.9, L.ASA_ERR_INVALID),
    ("alpha", 1.01, L.ASA_ERR_INVALID), ("alpha", 3.1, L.ASA_ERR_INVALID), ("alpha", float("inf"), L.ASA_ERR_INVALID),
])
def test_rejects_bad_params(field, value, code):
    assert workspace(params(**{field: value}))[0] == code


def test_workspaces():
    rc, a, s = workspace(params())
    assert rc == 0 and a % 16 == 0 and s % 16 == 0
    assert workspace(params(table_width=4096))[1] > 0 and workspace(params(table_width=4096))[2] > 0
    assert workspace(params(alpha=1.5), 3)[0] == 0
    assert workspace(params(), -1)[0] == L.ASA_ERR_INVALID


def test_null_pointers_are_refused():
    lib, p = L.lib(), params()
    st = (ctypes.c_int64 * 3)(1, 1, 1)
    assert lib.asa_cache_attention(ctypes.byref(p), None, st, None, None, None, None, 0, None, None, 0, None) == L.ASA_ERR_INVALID
    assert lib.asa_cache_select(ctypes.byref(p), None, st, None, None, None, 2, None, None, 0, None) == L.ASA_ERR_INVALID
    assert lib.asa_cache_write(ctypes.byref(p), None, None, st, st, None, None, None, None, None, None) == L.ASA_ERR_INVALID
    assert lib.asa_cache_read(ctypes.byref(p), None, None, None, None, None, None, None) == L.ASA_ERR_INVALID
    assert lib.asa_cache_bounds(ctypes.byref(p), None, None, 3, None, None, None) == L.ASA_ERR_INVALID
    assert lib.asa_cache_attention(None, None, st, None, None, None, None, 0, None, None, 0, None) == L.ASA_ERR_INVALID


@pytest.mark.parametrize("d", sa.cache.HEAD_DIMS)
@pytest.mark.parametrize("P", sa.cache.PAGE_SIZES)
def test_records(d, P):
    assert L.lib().asa_cache_record_bytes(d, P) == P * d * 5 // 4
    cache = sa.new_cache(3, 2, d, P, device="cpu")
    assert cache.pool.shape == (3, 2, P * d * 5 // 4) and cache.bounds.shape == (3, 2, 2 * d + 16)
    assert (cache.head_dim, cache.page_size, cache.kv_heads) == (d, P, 2)
    # every byte of a record belongs to one token's codes or scales
    used = np.zeros(P * d * 5 // 4, int)
    for key in (True, False):
        assert sorted(set(F.places(d, key))) == list(range(d // 2))
        for slot in range(P):
            row, par = F.row_at(d, P, slot, key)
            used[row: row + d // 2] += 1
            used[par: par + d // 8] += 1
    assert (used == 1).all()


@pytest.mark.parametrize("kw", [dict(head_dim=48), dict(head_dim=256), dict(page_size=8), dict(kv_heads=0), dict(num_pages=-1)])
def test_new_cache_refuses(kw):
    args = dict(num_pages=2, kv_heads=2, head_dim=64, page_size=16)
    with pytest.raises(ValueError):
        sa.new_cache(**{**args, **kw}, device="cpu")


def test_quantising_errs_by_half_a_step():
    g = np.random.RandomState(0)
    for scale, shift in ((1.0, 0.0), (1e-3, 0.0), (50.0, 10.0), (1.0, 300.0)):
        x = (g.randn(200, 128) * scale + shift).astype(np.float32)
        n, s, z = F.quantise(x)
        y = (z.astype(np.float64)[..., None] + n * s.astype(np.float64)[..., None]).reshape(x.shape)
        step = np.repeat(s.astype(np.float64), 32, -1)
        # half a step, and what rounding the offset and 15 scales to fp16 can cut off the ends
        assert (np.abs(y - x) <= 0.5 * step + np.abs(x).max() * 2.0 ** -10).all()


def test_bounds_do_not_depend_on_the_order():
    g = np.random.RandomState(1)
    x = g.randn(64, 32) * np.exp2(g.randint(-6, 7, (64, 1)))
    up, lo, e = F.bounds_codes(x.max(0), x.min(0))
    top, low = x[0], x[0]
    for row in x:
        u, l, ex = F.bounds_codes(np.maximum(top, row), np.minimum(low, row))
        top, low = u * np.exp2(float(ex)), l * np.exp2(float(ex))
    assert np.array_equal(u, up) and np.array_equal(l, lo) and ex == e
    assert (up * np.exp2(float(e)) >= x.max(0)).all() and (lo * np.exp2(float(e)) <= x.min(0)).all()


def test_entmax_weights_by_bisection_match_the_sorted_form():
    s = np.random.RandomState(2).randn(50) * 3
    x = np.sort(s / 2 - (s / 2).max())[::-1]
    n = np.arange(1, 51)
    mean = np.cumsum(x) / n
    tau = mean - np.sqrt(np.maximum((1 - (np.cumsum(x ** 2) - n * mean ** 2)) / n, 0))
    p = np.maximum(s / 2 - (s / 2).max() - tau[(tau <= x).sum() - 1], 0) ** 2
    assert np.abs(F.weights(s, 1.5)[0] - p).max() < 1e-12


def test_operator_shapes():
    ops = torch.ops.splash_attention
    meta = lambda *s, dtype=torch.bfloat16: torch.empty(*s, dtype=dtype, device="meta")  # noqa: E731
    i = lambda *s: meta(*s, dtype=torch.int32)  # noqa: E731
    q, pool, bounds = meta(2, 3, 8, 64), meta(5, 4, 16 * 80, dtype=torch.uint8), meta(5, 4, 144, dtype=torch.int8)
    assert ops.cache_attention(q, pool, bounds, i(2, 3), i(2), None, 0.1, 1.0).shape == q.shape
    assert ops.cache_select(q, pool, bounds, i(2, 3), i(2), 6).shape == (2, 3, 4, 6)
    k, v = ops.cache_read(pool, bounds, i(2, 3), i(2), 7, None, True)
    assert k.shape == v.shape == (2, 7, 4, 64) and k.dtype == torch.float32
    assert ops.cache_bounds(bounds, i(9))[0].shape == (9, 4, 64)
    assert "Tensor(a!) pool" in str(ops.cache_write.default._schema)
