"""The 4-bit paged cache by its documented format (include/asa.h), in numpy and
64 bits on the CPU: quantising, reading, bounds, page selection and attention."""
import numpy as np

F16_MAX = 65504.0
R15, R127 = np.float32(1.0) / np.float32(15.0), np.float32(1.0) / np.float32(127.0)


def quantise(x):
    """x fp32 [..., d] -> codes [..., d/32, 32] (0..15), scale and offset fp16 [..., d/32]."""
    x = np.asarray(x, np.float32)
    bad = np.isnan(x).reshape(*x.shape[:-1], -1, 32).any(-1)
    x = np.clip(np.nan_to_num(x, nan=0.0, posinf=np.inf, neginf=-np.inf), -F16_MAX, F16_MAX).astype(np.float32)
    x = x.reshape(*x.shape[:-1], -1, 32)
    z = x.min(-1).astype(np.float16)
    s = ((x.max(-1) - z.astype(np.float32)) * R15).astype(np.float16)
    sf = s.astype(np.float32)[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        n = np.where(sf > 0, np.clip(np.rint((x - z.astype(np.float32)[..., None]) / sf), 0, 15), 0)
    s, z = s.copy(), z.copy()
    s[bad] = z[bad] = np.float16(np.nan)
    return np.nan_to_num(n).astype(np.uint8), s, z


def places(d, key):
    """Of each channel its byte in a row of codes."""
    g, w = np.arange(d) // 32, np.arange(d) % 32
    return (w // 8) * 4 * (d // 32) + 4 * g + (w % 8) // 2 if key else (w // 4) * 2 * (d // 32) + 2 * g + (w % 4) // 2


def row_at(d, P, slot, key):
    """(offset of a slot's codes, offset of its scales) in a page's record."""
    block = 16 * (d // 2 + d // 8)
    base = (0 if key else P // 16 * block) + slot // 16 * block
    return base + slot % 16 * (d // 2), base + 8 * d + slot % 16 * (d // 8)


def decode(pool, d, P):
    """pool uint8 [pages, H, record] -> K, V float64 [pages, H, P, d]."""
    out = []
    for key in (True, False):
        y = np.empty(pool.shape[:2] + (P, d))
        at, g, ng = places(d, key), np.arange(d) // 32, d // 32
        for slot in range(P):
            row, par = row_at(d, P, slot, key)
            code = (pool[..., row + at] >> (4 * (np.arange(d) % 2)).astype(np.uint8)) & 15
            h = np.ascontiguousarray(pool[..., par: par + 4 * ng]).view(np.float16).astype(np.float64)
            y[..., slot, :] = h[..., ng + g] + code * h[..., g]
        out.append(y)
    return out


def encode_token(pool, page, h, slot, d, P, k, v):
    """Writes one token's fp32 k, v [d] into the pool."""
    for key, x in ((True, k), (False, v)):
        n, s, z = quantise(x)
        n = n.reshape(-1)
        row, par = row_at(d, P, slot, key)
        at = places(d, key)
        pool[page, h, row: row + d // 2] = 0
        for c in range(d):
            pool[page, h, row + at[c]] |= n[c] << (4 * (c % 2))
        pool[page, h, par: par + d // 8] = np.concatenate([s, z]).view(np.uint8)


def bounds_codes(top, low):
    """Bounds [..., d] -> upper and lower codes, exponent [...]."""
    m = np.maximum(np.abs(top), np.abs(low)).max(-1)
    f, e = np.frexp(m)
    e = np.where(m > 0, np.maximum(e - 7 + (f > 127 / 128), -126), -126).astype(np.int32)
    unit = np.exp2(e.astype(np.float64))[..., None]
    return np.ceil(top / unit).astype(np.int8), np.floor(low / unit).astype(np.int8), e


def select(q, bounds, table, length, t, T, P, keep, G):
    """The pages of one sequence's query t: int32 [H, keep].  q fp32 [T, HQ, d]."""
    d = q.shape[-1]
    H = q.shape[1] // G
    pos = min(length - T + t, len(table) * P - 1)
    n = pos // P + 1 if pos >= 0 else 0
    out = np.full((H, keep), -1, np.int32)
    for h in range(H):
        if n <= keep:
            out[h, :n] = np.arange(n)
            continue
        x = q[t, h * G: (h + 1) * G].astype(np.float32)
        unit = (np.abs(x).max(-1) * R127).astype(np.float32)
        with np.errstate(divide="ignore", invalid="ignore"):
            c = np.where(unit[:, None] > 0, np.rint(x / unit[:, None]), 0).astype(np.float64)
        rec = bounds[np.clip(table[: n - 1], 0, len(bounds) - 1), h]
        e = np.ascontiguousarray(rec[:, 2 * d: 2 * d + 4]).view(np.int32)[:, 0]
        up, lo = rec[:, :d].astype(np.float64), rec[:, d: 2 * d].astype(np.float64)
        whole = np.maximum(c[:, None] * up, c[:, None] * lo).sum(-1)                # [G, n-1]
        sc = ((whole * np.exp2(e.astype(np.float64))).astype(np.float32) * unit[:, None]).astype(np.float32)
        sc = np.where(np.isnan(sc), -np.inf, sc).max(0)
        sc = np.where((table[: n - 1] >= 0) & (table[: n - 1] < len(bounds)), sc, -np.inf)
        best = sorted(range(n - 1), key=lambda i: (-sc[i], i))[: keep - 1]
        out[h] = sorted(best + [n - 1])
    return out


def weights(s, alpha):
    """Weights of scores [n] float64 (seen keys only), normalised, and how far
    each may be off: a relative 2^-9 for one rounding to 8 bits or several to
    11, and what a score off by 2^-15 of the largest (2^-15 at least: 32-bit sums
    of 128 products) moves."""
    ds = 2.0 ** -15 * max(1.0, np.abs(s).max())
    if alpha == 1.0:
        p = np.exp(s - s.max())
        dp = p * (2.0 ** -9 + 2 * ds)
    else:
        x = (alpha - 1) * np.clip(s, -10, 10)
        ex = 1 / (alpha - 1)
        lo, hi = x.max() - 1, x.max()
        for _ in range(80):
            mid = 0.5 * (lo + hi)
            if (np.maximum(x - mid, 0) ** ex).sum() >= 1:
                lo = mid
            else:
                hi = mid
        u = x - lo
        p = np.maximum(u, 0) ** ex
        ds = 2 * (alpha - 1) * min(ds, 2.0 ** -15 * 10)
        dp = np.maximum(u + ds, 0) ** ex - np.maximum(u - ds, 0) ** ex + p * 2.0 ** -9
    return p / p.sum(), dp / p.sum()


def attend(q, K, V, scale, alpha):
    """One query row over its seen keys, float64: (o [d], bound [d]); the bound
    adds the output's rounding to bf16."""
    if len(K) == 0:
        return np.zeros(V.shape[1]), np.zeros(V.shape[1])
    p, dp = weights(K @ q * scale, alpha)
    o = p @ V
    return o, 2.0 ** -8 * np.abs(o) + dp @ np.abs(V) + dp.sum() * np.abs(o) + 1e-30
