"""The operators that serve a model from a 4-bit paged key/value cache: cases, plain forms and work.

Three operators: quantising keys and values into the cache's pages and reading them back (``kind`` "store"),
attention over the cache with softmax or alpha-entmax weights ("attend"), and attention over the pages that a
cheap score selects for each query ("select").

The cache is two tensors.  ``pool`` is uint8 [pages, kv heads, record]: a record holds a page's keys, then its
values, each as blocks of 16 tokens; a block holds 16 rows of d/2 bytes of codes, then 16 rows of 2 d/32 fp16
(the scales of the d/32 channel groups, then their offsets).  An element is ``offset + code * scale``, code in
0..15.  ``bounds`` is int8 [pages, kv heads, 2 d + 16]: upper codes, lower codes, one int32 exponent, padding.
``block_table`` [B, pages of a sequence] names the pages, -1 past the end.
"""
import math
import random

import torch

own = False

GROUP = 32
BLOCK = 16
F16_MAX = 65504.0
PAD = 16


# ---- the cache's layout, in elementary operations --------------------------------------------------------------
def _halves(pool, d):
    """Views of a pool's keys and values: codes [pages, H, P/16, 16, d/2] uint8 and (scale, offset) as
    [pages, H, P/16, 16, 2 d/32] fp16."""
    rec = pool.shape[-1] // 2
    block = BLOCK * (d // 2 + d // 8)
    out = []
    for part in (pool[..., :rec], pool[..., rec:]):
        part = part.unflatten(-1, (rec // block, block))
        codes = part[..., : BLOCK * d // 2].unflatten(-1, (BLOCK, d // 2))
        out.append((codes, part[..., BLOCK * d // 2:].unflatten(-1, (BLOCK, d // 8)).view(torch.float16)))
    return out


def _quantise(x):
    """float32 [..., d] -> codes uint8 [..., d/32, 32], scale and offset fp16 [..., d/32]."""
    x = x.clamp(-F16_MAX, F16_MAX).unflatten(-1, (-1, GROUP))
    z = x.amin(-1).half()
    s = ((x.amax(-1) - z.float()) / 15.0).half()
    step = s.float().unsqueeze(-1)
    n = torch.round((x - z.float().unsqueeze(-1)) / step).clamp(0.0, 15.0)
    return torch.where(step > 0, n, 0.0).to(torch.uint8), s, z


def _pack(n, width):
    """Codes [..., d/32, 32] as rows of d/2 bytes: the bytes of each run of ``width`` channels, run by run over the
    groups (``width`` 8 for keys, 4 for values), the even channel in the low four bits."""
    b = n[..., 0::2] | (n[..., 1::2] << 4)
    return b.unflatten(-1, (GROUP // width, width // 2)).transpose(-3, -2).flatten(-3)


def _unpack(rows, width):
    """The inverse of _pack: rows [..., d/2] -> codes [..., d/32, 32]."""
    b = rows.unflatten(-1, (GROUP // width, -1, width // 2)).transpose(-3, -2)
    return torch.stack((b & 15, b >> 4), -1).flatten(-3)


def _values(rows, params, width):
    """The values that rows of codes and their (scale, offset) stand for, float32 [..., d]."""
    s, z = params.float().unsqueeze(-1).chunk(2, -2)
    return (z + _unpack(rows, width).float() * s).flatten(-2)


def _power(e):
    """2^e in float32, e whole numbers in -126..127."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _exponent(m):
    f, e = torch.frexp(m)
    e = e - 7 + (f > 127.0 / 128.0).to(e.dtype)
    return torch.where(m > 0, e, -126).clamp(-126, 20)


def _bounds_record(hi, lo):
    """Bounds [..., H, d] as records [..., H, 2 d + 16] int8, rounded outward."""
    e = _exponent(torch.maximum(hi.abs(), lo.abs()).amax(-1))
    inv = _power(-e).unsqueeze(-1)
    tail = e.to(torch.int32).unsqueeze(-1).view(torch.int8)
    return torch.cat((torch.ceil(hi * inv).to(torch.int8), torch.floor(lo * inv).to(torch.int8), tail,
                      tail.new_zeros(*tail.shape[:-1], PAD - 4)), -1)


def _bounds_values(rec):
    d = (rec.shape[-1] - PAD) // 2
    e = rec[..., 2 * d: 2 * d + 4].contiguous().view(torch.int32)
    unit = _power(e.clamp(-126, 127))
    return rec[..., :d].float() * unit, rec[..., d: 2 * d].float() * unit


# ---- cases -----------------------------------------------------------------------------------------------------
def _store(B, T, kv_heads, d, page, behind, dtype, ragged):
    return {"kind": "store", "B": B, "T": T, "kv_heads": kv_heads, "d": d, "page": page, "behind": behind,
            "dtype": dtype, "ragged": ragged}


def _attend(B, T, heads, kv_heads, d, page, length, alpha, ragged):
    return {"kind": "attend", "B": B, "T": T, "heads": heads, "kv_heads": kv_heads, "d": d, "page": page,
            "length": length, "alpha": alpha, "ragged": ragged}


def _select(B, T, heads, kv_heads, d, page, length, keep, alpha, ragged):
    return dict(_attend(B, T, heads, kv_heads, d, page, length, alpha, ragged), kind="select", keep=keep)


def listed():
    return [
        # the new token of each of 64 running sequences, as every decoding step writes it
        dict(_store(64, 1, 8, 128, 64, 4096, "bf16", True), name="store_step"),
        # float32 prompts of several lengths behind an odd number of tokens, small pages and heads
        dict(_store(3, 1537, 4, 64, 16, 77, "f32", True), name="store_prompts_f32"),
        # two long documents, written at once
        dict(_store(2, 32768, 8, 128, 64, 0, "bf16", False), name="store_long"),
        # one user, one token, a short history, a key head to each head: latency
        dict(_attend(1, 1, 16, 16, 64, 64, 321, 1.0, False), name="attend_one"),
        # a server's decoding batch, sequences of very different lengths
        dict(_attend(48, 1, 32, 8, 128, 64, 8192, 1.0, True), name="attend_batch"),
        # two long contexts, few key heads
        dict(_attend(2, 1, 32, 4, 128, 64, 131072, 1.0, False), name="attend_long"),
        # a chunk of a prompt behind what is cached already
        dict(_attend(2, 192, 16, 4, 128, 32, 4096, 1.0, True), name="attend_chunk"),
        # decoding with the 1.5-entmax weights that the model was trained with
        dict(_attend(8, 1, 32, 8, 128, 64, 32768, 1.5, False), name="entmax_step"),
        # three guessed tokens checked at once, an odd number of sequences, small heads
        dict(_attend(5, 3, 12, 4, 64, 16, 1999, 1.5, True), name="entmax_guesses"),
        # one user, small pages, a few of them selected: latency
        dict(_select(1, 1, 16, 4, 64, 16, 4001, 24, 1.0, False), name="select_one"),
        # long contexts of a batch, a thirtieth of each read
        dict(_select(8, 1, 32, 8, 128, 64, 65536, 32, 1.0, True), name="select_long"),
        # four guessed tokens, each with pages of its own, entmax weights
        dict(_select(6, 4, 16, 4, 128, 32, 12000, 40, 1.5, True), name="select_guesses"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("store", "attend", "attend", "entmax", "select", "select"))
    d = rng.choice((32, 64, 96, 128, 128))
    page = rng.choice((16, 32, 64, 128))
    kv_heads = rng.choice((1, 2, 3, 4, 8))
    group = rng.choice((1, 2, 3, 4, 5, 8))
    ragged = rng.random() < 0.7
    if kind == "store":
        T = rng.choice((1, _log(rng, 2, 8), _log(rng, 16, 16384)))
        B = _log(rng, 1, max(1, min(128, 32768 // T)))
        return _store(B, T, kv_heads, d, page, _log(rng, 1, 4096) - 1, rng.choice(("bf16", "bf16", "f32")), ragged)
    T = rng.choice((1, 1, rng.randint(2, 8), _log(rng, 9, 160)) if kind != "select" else (1, 1, rng.randint(2, 6)))
    length = max(T, _log(rng, 16, 65536))
    most = 2 * 131072 * 4 // (2 * length * kv_heads)
    if T > 8:
        length = min(length, 8192)
        most = 1_500_000 * 8 // (T * length * kv_heads * group)
    elif kind != "attend":
        most = min(most, 8_000_000 // (T * length * kv_heads * group))
    B = _log(rng, 1, max(1, min(64, most)))
    alpha = 1.5 if kind == "entmax" or (kind == "select" and rng.random() < 0.4) else 1.0
    if kind == "select":
        keep = min(_log(rng, 2, 64), -(-length // page) + 2)
        return _select(B, T, kv_heads * group, kv_heads, d, page, length, keep, alpha, ragged)
    return _attend(B, T, kv_heads * group, kv_heads, d, page, length, alpha, ragged)


# ---- inputs ----------------------------------------------------------------------------------------------------
def _lengths(case, most, least):
    """The sequences' lengths, a property of the case: the first has the most tokens; ragged ones spread over the range."""
    r = random.Random(most * 7919 + least)
    if not case["ragged"]:
        return [most] * case["B"]
    return [most] + [_log(r, max(1, least), max(1, most)) if most else 0 for _ in range(case["B"] - 1)]


def _cache(case, lengths, seed, dev):
    """A filled cache: keys in runs of like ones (a centroid to every 64 tokens), values about zero, pages in
    random order, what lies past a sequence's end left over from others, spare pages full of NaN patterns."""
    g = torch.Generator(dev).manual_seed(seed * 1000003 + 17)
    H, d, P = case["kv_heads"], case["d"], case["page"]
    need = [-(-n // P) for n in lengths]
    wide, total = max(need), sum(need)
    pages = total + 3
    perm = torch.randperm(pages - 1, generator=g, device=dev).to(torch.int32)      # the last page stays free
    table = torch.full((case["B"], wide), -1, dtype=torch.int32)
    at = 0
    perm_cpu = perm.cpu()
    for b, n in enumerate(need):
        table[b, :n] = perm_cpu[at: at + n]
        at += n
    block = BLOCK * (d // 2 + d // 8)
    pool = torch.full((pages, H, 2 * (P // BLOCK) * block), 255, dtype=torch.uint8, device=dev)
    bounds = torch.full((pages, H, 2 * d + PAD), 127, dtype=torch.int8, device=dev)
    centres = torch.randn(64, H, d, generator=g, device=dev)
    halves = _halves(pool, d)
    step = max(1, (1 << 26) // (H * P * d))                                        # pages made at a time
    for lo in range(0, total, step):
        ids = perm[lo: lo + step].long()
        m = ids.numel()
        which = torch.randint(0, 64, (m,), generator=g, device=dev)
        k = torch.randn(m, P, H, d, generator=g, device=dev) + 1.5 * centres[which].unsqueeze(1)
        v = torch.randn(m, P, H, d, generator=g, device=dev)
        for (codes, params), x, width in zip(halves, (k, v), (8, 4)):
            n, s, z = _quantise(x.bfloat16().float().transpose(1, 2).unflatten(2, (-1, BLOCK)))
            codes[ids] = _pack(n, width)
            params[ids] = torch.cat((s, z), -1)
        bounds[ids] = _bounds_record(k.bfloat16().float().amax(1), k.bfloat16().float().amin(1))
    return pool, bounds, table.to(dev), centres, g


def prepare(case, seed):
    dev = torch.device("cuda")
    B, T, H, d, P = (case[n] for n in ("B", "T", "kv_heads", "d", "page"))
    state = {"case": dict(case)}
    if case["kind"] == "store":
        dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        start = _lengths(case, case["behind"], 1)
        count = _lengths(case, T, 1)
        pool, bounds, table, _, g = _cache(case, [s + T for s in start], seed, dev)
        # keys and values lie side by side, as one projection gives them
        kv = torch.randn(B, T, 2, H, d, generator=g, device=dev).mul_(1.5).to(dt)
        touched = [table[b, start[b] // P: (start[b] + max(1, count[b]) - 1) // P + 1] for b in range(B)]
        state.update(pool=pool, bounds=bounds, table=table, k=kv[:, :, 0], v=kv[:, :, 1],
                     start=torch.tensor(start, dtype=torch.int32, device=dev),
                     count=torch.tensor(count, dtype=torch.int32, device=dev), touched=torch.cat(touched))
        return state
    lengths = _lengths(case, case["length"], max(T, case["length"] // 64))
    pool, bounds, table, centres, g = _cache(case, lengths, seed, dev)
    # a query looks for one of the centroids
    look = torch.randint(0, 64, (B, T), generator=g, device=dev)
    q = torch.randn(B, T, H, case["heads"] // H, d, generator=g, device=dev) + 0.25 * centres[look].unsqueeze(3)
    state.update(pool=pool, bounds=bounds, table=table, q=q.flatten(2, 3).bfloat16(),
                 lengths=torch.tensor(lengths, dtype=torch.int32, device=dev))
    return state


# ---- the plain forms -------------------------------------------------------------------------------------------
def _store_plain(s):
    case = s["case"]
    P, T, d = case["page"], case["T"], case["d"]
    dev = s["k"].device
    free = s["pool"].shape[0] - 1
    start, count, table = s["start"].long(), s["count"].long(), s["table"].long()
    t = torch.arange(T, device=dev)
    pos = start[:, None] + t
    valid = t < count[:, None]
    page = torch.where(valid, table.gather(1, pos // P), free)                      # tokens that are not there go to the free page
    k32, v32 = s["k"].float(), s["v"].float()
    halves = _halves(s["pool"], d)
    outs = []
    (kc, kp), (vc, vp) = halves
    n, sc, z = _quantise(k32)
    kc[page, :, pos % P // BLOCK, pos % BLOCK] = _pack(n, 8)
    kp[page, :, pos % P // BLOCK, pos % BLOCK] = torch.cat((sc, z), -1)
    n, sc, z = _quantise(v32)
    vc[page, :, pos % P // BLOCK, pos % BLOCK] = _pack(n, 4)
    vp[page, :, pos % P // BLOCK, pos % BLOCK] = torch.cat((sc, z), -1)
    # bounds of the pages that were written to
    first = start // P
    wide = (T + P - 2) // P + 1
    j = torch.arange(wide, device=dev)
    tok = (first[:, None, None] + j[:, None]) * P + torch.arange(P, device=dev) - start[:, None, None]
    there = (tok >= 0) & (tok < count[:, None, None])                               # [B, wide, P]
    rows = k32.clamp(-F16_MAX, F16_MAX)[torch.arange(case["B"], device=dev)[:, None, None], tok.clamp(0, T - 1)]
    mask = there[..., None, None]
    hi = rows.masked_fill(~mask, -math.inf).amax(2)
    lo = rows.masked_fill(~mask, math.inf).amin(2)
    ids = torch.where(there.any(-1), table.gather(1, (first[:, None] + j).clamp(max=table.shape[1] - 1)), free)
    old_hi, old_lo = _bounds_values(s["bounds"][ids])
    keep = ~there[:, :, 0, None, None] & there.any(-1)[..., None, None]             # begun in an earlier call
    hi = torch.where(keep, torch.maximum(hi, old_hi), hi)
    lo = torch.where(keep, torch.minimum(lo, old_lo), lo)
    some = there.any(-1)[..., None, None]
    s["bounds"][ids] = _bounds_record(torch.where(some, hi, 0.0), torch.where(some, lo, 0.0))
    # reading it back
    gone = ~valid[..., None, None]
    outs.append(_values(kc[page, :, pos % P // BLOCK, pos % BLOCK], kp[page, :, pos % P // BLOCK, pos % BLOCK], 8))
    outs.append(_values(vc[page, :, pos % P // BLOCK, pos % BLOCK], vp[page, :, pos % P // BLOCK, pos % BLOCK], 4))
    out_dtype = s["k"].dtype
    bhi, blo = _bounds_values(s["bounds"][s["touched"].long()])
    return {"k": outs[0].masked_fill(gone, 0.0).to(out_dtype), "v": outs[1].masked_fill(gone, 0.0).to(out_dtype),
            "upper": bhi, "lower": blo}


def _weights(sc, seen, alpha):
    """Rows of weights over the last axis (not yet divided by their sum), and the sums."""
    if alpha == 1.0:
        sc = sc.masked_fill(~seen, -math.inf)
        top = sc.amax(-1, keepdim=True)
        p = torch.exp(sc - torch.where(top > -math.inf, top, 0.0))
    else:                                                                           # 1.5: the threshold in closed form
        x = (0.5 * sc.clamp(-10.0, 10.0)).masked_fill(~seen, -math.inf)
        top = x.amax(-1, keepdim=True)
        x = x - torch.where(top > -math.inf, top, 0.0)
        z = torch.sort(x, -1, descending=True).values.clamp(min=-4.0)
        n = torch.arange(1, z.shape[-1] + 1, device=z.device, dtype=torch.float32)
        mean = z.cumsum(-1) / n
        var = z.square().cumsum(-1) - n * mean.square()
        tau = mean - ((1.0 - var) / n).clamp(min=0.0).sqrt()
        size = ((tau <= z) & (z > -4.0)).sum(-1, keepdim=True).clamp(min=1)
        p = (x - tau.gather(-1, size - 1)).clamp(min=0.0).square()
    total = p.sum(-1, keepdim=True)
    return p, total


def _attend_plain(s):
    case = s["case"]
    B, T, H, d, P = (case[n] for n in ("B", "T", "kv_heads", "d", "page"))
    G = case["heads"] // H
    table = s["table"].clamp(min=0).long()
    (kc, kp), (vc, vp) = _halves(s["pool"], d)
    n = table.shape[1] * P
    k = _values(kc[table], kp[table], 8).permute(0, 2, 1, 3, 4, 5).reshape(B, H, n, d)
    v = _values(vc[table], vp[table], 4).permute(0, 2, 1, 3, 4, 5).reshape(B, H, n, d)
    q = s["q"].float().unflatten(2, (H, G)).permute(0, 2, 1, 3, 4).reshape(B, H, T * G, d)
    sc = (q @ k.transpose(-1, -2)) * d ** -0.5
    last = s["lengths"][:, None] - T + torch.arange(T, device=q.device)             # each query's own place
    at = torch.arange(n, device=q.device)
    seen = (at <= last[..., None]).repeat_interleave(G, 1).unsqueeze(1)
    v = torch.where((at < s["lengths"][:, None])[:, None, :, None], v, 0.0)
    p, total = _weights(sc, seen, case["alpha"])
    o = (p @ v) / torch.where(total > 0, total, 1.0)
    return o.reshape(B, H, T, G, d).permute(0, 2, 1, 3, 4).reshape(B, T, H * G, d).bfloat16()


def _select_plain(s):
    case = s["case"]
    B, T, H, d, P, k = (case[n] for n in ("B", "T", "kv_heads", "d", "page", "keep"))
    G = case["heads"] // H
    dev = s["q"].device
    table = s["table"].clamp(min=0).long()
    wide = table.shape[1]
    q = s["q"].float().unflatten(2, (H, G))                                         # [B, T, H, G, d]
    unit = q.abs().amax(-1, keepdim=True) / 127.0
    n = torch.where(unit > 0, torch.round(q / unit), 0.0)
    rec = s["bounds"][table]                                                        # [B, wide, H, .]
    e = rec[..., 2 * d: 2 * d + 4].contiguous().view(torch.int32)[..., 0]
    hi, lo = rec[..., :d].float().permute(0, 2, 3, 1), rec[..., d: 2 * d].float().permute(0, 2, 3, 1)
    n = n.permute(0, 2, 1, 3, 4).reshape(B, H, T * G, d)
    whole = n.clamp(min=0.0) @ hi + n.clamp(max=0.0) @ lo                           # whole numbers below 2^24
    score = (whole * _power(e.clamp(-126, 127)).permute(0, 2, 1).unsqueeze(2)).reshape(B, H, T, G, wide)
    score = (score * unit.permute(0, 2, 1, 3, 4)).amax(3).permute(0, 2, 1, 3)       # [B, T, H, wide]
    last = s["lengths"][:, None] - T + torch.arange(T, device=dev)                  # [B, T]
    mine = torch.where(last >= 0, last // P, -1)[..., None, None]
    at = torch.arange(wide, device=dev)
    score = torch.where(at == mine, math.inf, torch.where(at < mine, score, -math.inf))
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :k]
    order = torch.nn.functional.pad(order, (0, k - order.shape[-1]), value=wide)
    rank = torch.arange(k, device=dev)
    chosen = torch.where((rank < mine + 1) & (order < wide), order, wide).sort(-1).values
    pages = torch.where(chosen < wide, chosen, -1)                                  # [B, T, H, k]
    # attention over them alone
    at = pages.clamp(min=0)
    ids = table[torch.arange(B, device=dev)[:, None, None, None], at]
    head = torch.arange(H, device=dev)[None, None, :, None]
    (kc, kp), (vc, vp) = _halves(s["pool"], d)
    keys = _values(kc[ids, head], kp[ids, head], 8).reshape(B, T, H, k * P, d)
    vals = _values(vc[ids, head], vp[ids, head], 4).reshape(B, T, H, k * P, d)
    place = (at[..., None] * P + torch.arange(P, device=dev)).flatten(-2)
    seen = (pages >= 0).repeat_interleave(P, -1) & (place <= last[..., None, None])
    vals = torch.where(seen[..., None], vals, 0.0)
    sc = (q @ keys.transpose(-1, -2)) * d ** -0.5
    p, total = _weights(sc, seen.unsqueeze(3), case["alpha"])
    o = (p @ vals) / torch.where(total > 0, total, 1.0)
    return {"o": o.flatten(2, 3).bfloat16(), "pages": pages.to(torch.int32)}


# ---- one pass --------------------------------------------------------------------------------------------------
_module = None


def _framework():
    global _module
    if _module is None:
        import os
        import sys
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(root, "adaptive-splash-attention_b200"))
        import splash_attention
        _module = splash_attention
    return _module


def run(state):
    kind = state["case"]["kind"]
    if not own:
        return {"store": _store_plain, "attend": _attend_plain, "select": _select_plain}[kind](state)
    sa = _framework()
    case = state["case"]
    cache = sa.KVCache(state["pool"], state["bounds"])
    if kind == "store":
        sa.cache_write(state["k"], state["v"], cache, state["table"], state["start"], state["count"])
        k, v = sa.cache_read(cache, state["table"], state["start"], case["T"], state["count"],
                             dtype=state["k"].dtype)
        upper, lower = sa.cache_bounds(cache, state["touched"])
        return {"k": k, "v": v, "upper": upper, "lower": lower}
    if kind == "attend":
        return sa.cache_attention(state["q"], cache, state["table"], state["lengths"], alpha=case["alpha"])
    pages = sa.select_pages(state["q"], cache, state["table"], state["lengths"], case["keep"])
    o = sa.cache_attention(state["q"], cache, state["table"], state["lengths"], alpha=case["alpha"], pages=pages)
    return {"o": o, "pages": pages}


# ---- what a pass cannot do without -----------------------------------------------------------------------------
def work(case):
    B, T, H, d, P = (case[n] for n in ("B", "T", "kv_heads", "d", "page"))
    if case["kind"] == "store":
        size = 2 if case["dtype"] == "bf16" else 4
        start, count = _lengths(case, case["behind"], 1), _lengths(case, T, 1)
        tokens = sum(count)
        pages = sum((a + n - 1) // P - a // P + 1 for a, n in zip(start, count))
        # keys and values in, their records out and in again, values out; bounds out, in and out as values
        return {"bytes": tokens * H * (4 * d * size + 2.5 * d) + pages * H * (2 * (2 * d + 4) + 8 * d),
                "flops": 8.0 * tokens * H * d}
    heads = case["heads"]
    lengths = _lengths(case, case["length"], max(T, case["length"] // 64))
    ends = 4.0 * B * T * heads * d                                                  # queries in, outputs out
    part = 1.25 if case["alpha"] == 1.0 else 0.625                                  # entmax: of the values, the support's alone
    if case["kind"] == "attend":
        pairs = sum(T * n - T * (T - 1) // 2 for n in lengths)
        return {"bytes": sum(lengths) * (H * d * part + 4.0 / P) + ends, "flops": heads * pairs * 4.0 * d * part / 1.25}
    some = sum(min(n, case["keep"] * P) for n in lengths)
    pages = sum(-(-n // P) for n in lengths)
    # of the pages that the T queries of a sequence select, each is read once at least; they may all select the same
    return {"bytes": H * (pages * (2 * d + 4) + some * d * part) + pages * 4.0 + ends + 4.0 * B * T * H * case["keep"],
            "flops": T * heads * (4.0 * d * pages + some * 4.0 * d * part / 1.25)}


# ---- the definition, in 64 bits --------------------------------------------------------------------------------
def _read64(pool, ids, head, d, P, which):
    """The [pages * P, d] float64 values that pages ``ids`` of one kv head hold, looked up byte by byte."""
    ids = ids.long()
    rec = pool[ids, head].to(torch.int64)                                           # [m, record]
    half = rec.shape[1] // 2
    rec = rec[:, which * half: (which + 1) * half]
    token = torch.arange(P, device=pool.device)
    c = torch.arange(d, device=pool.device)
    g, w = c // 32, c % 32
    row = (w // 8) * (4 * (d // 32)) + g * 4 + (w % 8) // 2 if which == 0 else (w // 4) * (2 * (d // 32)) + g * 2 + (w % 4) // 2
    base = (token // 16) * (16 * (d // 2 + d // 8))
    code = (rec[:, (base + (token % 16) * (d // 2))[:, None] + row] >> (4 * (c % 2))) & 15
    par = (base + 8 * d + (token % 16) * (d // 8))[:, None]

    def half_at(off):
        return (rec[:, off] + 256 * rec[:, off + 1]).to(torch.int16).view(torch.float16).double()

    value = half_at(par + 2 * g + 2 * (d // 32)) + code * half_at(par + 2 * g)
    return value.reshape(-1, d)


def _rows64(sc, alpha):
    """Weights of rows of float64 scores by the definition: exp, or the root of the sum by bisection."""
    if alpha == 1.0:
        return torch.softmax(sc, -1)
    x = torch.where(sc == -math.inf, sc, (alpha - 1.0) * sc.clamp(-10.0, 10.0))
    hi = x.amax(-1, keepdim=True)
    lo = hi - 1.0
    for _ in range(60):
        mid = 0.5 * (lo + hi)
        over = (x - mid).clamp(min=0.0).pow(1.0 / (alpha - 1.0)).sum(-1, keepdim=True) >= 1.0
        lo, hi = torch.where(over, mid, lo), torch.where(over, hi, mid)
    p = (x - lo).clamp(min=0.0).pow(1.0 / (alpha - 1.0))
    return p / p.sum(-1, keepdim=True)


def _round64(x):
    """fp16 numbers of float64 ones, by way of float32 as the format says."""
    return x.float().half().double()


def _store64(s):
    case = s["case"]
    B, T, H, d, P = (case[n] for n in ("B", "T", "kv_heads", "d", "page"))
    out = {}
    start, count = s["start"].tolist(), s["count"].tolist()
    for name in ("k", "v"):
        x = s[name].double().reshape(B, T, H, d // 32, 32)
        z = _round64(x.min(-1, keepdim=True).values)
        step = _round64((x.max(-1, keepdim=True).values - z).float() / 15.0)
        code = ((x - z) / step).round().clamp(0, 15)
        code = torch.where(step > 0, code, torch.zeros_like(code))
        y = (z + code * step).reshape(B, T, H, d)
        for b in range(B):
            y[b, count[b]:] = 0.0
        out[name] = y
    old = s["bounds"].cpu()
    upper, lower = [], []
    for b in range(B):
        for j in range(start[b] // P, (start[b] + max(1, count[b]) - 1) // P + 1):
            lo, hi = max(j * P, start[b]), min((j + 1) * P, start[b] + count[b])
            x = s["k"][b, lo - start[b]: hi - start[b]].double().cpu()              # [m, H, d]
            top, low = x.max(0).values, x.min(0).values
            if lo > j * P:
                rec = old[int(s["table"][b, j])]
                was = rec[:, 2 * d: 2 * d + 4].contiguous().view(torch.int32).double()
                top = torch.maximum(top, rec[:, :d].double() * 2.0 ** was)
                low = torch.minimum(low, rec[:, d: 2 * d].double() * 2.0 ** was)
            m = torch.maximum(top.abs(), low.abs()).max(-1, keepdim=True).values
            unit = 2.0 ** torch.ceil(torch.log2(m / 127.0))
            upper.append(torch.ceil(top / unit) * unit)
            lower.append(torch.floor(low / unit) * unit)
    dev = s["k"].device
    out["upper"], out["lower"] = torch.stack(upper).to(dev), torch.stack(lower).to(dev)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "store":
        if case["B"] * case["T"] * case["kv_heads"] * case["d"] > 40_000_000 or case["B"] * case["T"] // case["page"] > 3000:
            return None
        return _store64(s)
    B, T, H, d, P = (case[n] for n in ("B", "T", "kv_heads", "d", "page"))
    G = case["heads"] // H
    lengths, table = s["lengths"].tolist(), s["table"]
    o = torch.zeros(B, T, H, G, d, dtype=torch.float64, device=table.device)
    if case["kind"] == "attend":
        for b in range(B):
            n = lengths[b]
            for h in range(H):
                ids = table[b, : -(-n // P)]
                k, v = (_read64(s["pool"], ids, h, d, P, w)[:n] for w in (0, 1))
                q = s["q"][b, :, h * G: (h + 1) * G].double()
                last = n - T + torch.arange(T, device=k.device)
                sc = (q @ k.T / math.sqrt(d)).masked_fill(torch.arange(n, device=k.device) > last[:, None, None], -math.inf)
                ok = last >= 0
                o[b, ok, h] = _rows64(sc[ok], case["alpha"]) @ v
        return o.flatten(2, 3)
    if B * T * H > 400:
        return None
    chosen = torch.full((B, T, H, case["keep"]), -1, dtype=torch.int32)
    for b in range(B):
        for h in range(H):
            rec = s["bounds"][table[b].clamp(min=0).long(), h]
            unit = 2.0 ** rec[:, 2 * d: 2 * d + 4].contiguous().view(torch.int32).double()
            hi, lo = rec[:, :d].double(), rec[:, d: 2 * d].double()
            for t in range(T):
                pos = lengths[b] - T + t
                if pos < 0:
                    continue
                q = s["q"][b, t, h * G: (h + 1) * G]
                grain = (q.float().abs().max(-1, keepdim=True).values / 127.0)
                n = (q.double() / grain.double()).round()
                per = (torch.maximum(n[:, None] * hi, n[:, None] * lo).sum(-1) * unit.T).float() * grain
                score = per.max(0).values[: pos // P + 1].tolist()
                score[-1] = math.inf
                best = sorted(sorted(range(len(score)), key=lambda i: (-score[i], i))[: case["keep"]])
                chosen[b, t, h, : len(best)] = torch.tensor(best, dtype=torch.int32)
                at = torch.tensor(best, device=table.device)
                k, v = (_read64(s["pool"], table[b, at], h, d, P, w) for w in (0, 1))
                place = (at[:, None] * P + torch.arange(P, device=at.device)).flatten()
                k, v = k[place <= pos], v[place <= pos]
                o[b, t, h] = _rows64(q.double() @ k.T / math.sqrt(d), case["alpha"]) @ v
    return {"o": o.flatten(2, 3), "pages": chosen.to(table.device)}
