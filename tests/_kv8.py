"""Plain float64 forms of the 8-bit KV cache operators, on the CPU, and inputs for their tests.

The numbers of a cache are made from bytes, so that the oracle and the kernels
see the same cache; the oracle reads them through torch's casts of the 8-bit
types, which the tests of the append pin bit by bit.
"""
import math

import torch

STORES = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
TOP = {torch.float8_e4m3fn: 8, torch.float8_e5m2: 15}      # largest number 1.75 * 2^TOP
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def scale_of(amax, store):
    """Byte of the least power of two 2^(byte - 127) with amax <= max * 2^(byte - 127)."""
    if amax == 0:
        return 0
    m, e = math.frexp(amax)
    return min(max(e - 1 - TOP[store] + (m > 0.875) + 127, 0), 254)


def bytes_of(x, byte, store):
    """x (float64) as bytes of an 8-bit type under scale ``byte``: one rounding (the
    scaled number is exact in fp32 within the type's range, and below it any
    rounding of it gives 0)."""
    y = (x.double() * 2.0 ** (127 - byte)).float()
    y = torch.where(torch.isfinite(x), y, torch.full_like(y, math.nan))
    return y.to(store).view(torch.uint8)


def cache_values(cache, scale):
    """The float64 numbers of a cache."""
    block = cache.shape[1] // scale.shape[1]
    e = scale.view(torch.uint8).double().repeat_interleave(block, dim=1)
    return cache.double() * torch.exp2(e - 127)[..., None]


def append(k, cache, scale, slots):
    """kvcache_append_8bit of one tensor on CPU copies: returns (cache, scale)."""
    store = cache.dtype
    cache, scale = cache.clone(), scale.clone()
    c, s = cache.view(torch.uint8), scale.view(torch.uint8)
    pages, page, heads, _ = cache.shape
    block = page // scale.shape[1]
    rows = slots.tolist()
    r = 0
    while r < len(rows):
        slot = rows[r]
        if not 0 <= slot < pages * page:
            r += 1
            continue
        n = 1
        while (r + n < len(rows) and rows[r + n] == slot + n and (slot + n) % block != 0):
            n += 1
        p, at, first = slot // page, slot % page, slot % block
        for h in range(heads):
            x = k[r:r + n, h].double()
            fine = x[torch.isfinite(x)]
            need = scale_of(float(fine.abs().max()) if fine.numel() else 0.0, store)
            old = min(int(s[p, at // block, h]), 254) if first else 0
            e = max(old, need)
            if e > old and first:
                held = cache[p, at - first:at, h].double() * 2.0 ** (old - e)
                c[p, at - first:at, h] = held.float().to(store).view(torch.uint8)
            c[p, at:at + n, h] = bytes_of(x, e, store)
            s[p, at // block, h] = e
        r += n
    return cache, scale


def same_bytes(a, b):
    """Equal bytes, any NaN equal to any other."""
    nan = torch.isnan(a.float()) & torch.isnan(b.float())
    return bool(((a.view(torch.uint8) == b.view(torch.uint8)) | nan).all())


def filled(pages, page, block, heads, dim, store, seed, spread=3):
    """A cache of random finite numbers, scales around 1, on the CPU."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(pages, page, heads, dim, generator=gen) * (40.0 if store == torch.float8_e4m3fn else 4000.0)
    s = torch.randint(127 - TOP[store] - spread, 127 - TOP[store] + 1 + spread // 2,
                      (pages, page // block, heads), generator=gen, dtype=torch.uint8)
    return x.clamp(-400, 400).to(store) if store == torch.float8_e4m3fn else x.to(store), s.view(torch.float8_e8m0fnu)


def attend(q, kc, ks, vc, vs, lens, table, cu=None, scale=None, causal=False, window=(-1, -1), softcap=0.0,
           alibi=None):
    """flash_attn_with_kvcache_8bit in float64 on the CPU: (out, bound) with
    ``bound`` what a kernel with 16-bit P and output and fp32 sums may be off by.

    One half step h of q's type for each P_j and for the output: h (sum_j p_j
    |v_j| + |out|).  fp32 scores: a product sum of D terms, a scale and the
    exponent's argument are off by at most (D + 8) 2^-24 (sum |q k| scale +
    |x|) and the exponential by 2^-22, relative to p, both in the sums over v
    and over p: twice that of sum_j p_j |v_j|.  fp16 also rounds v below its
    normal range, by 2^-25.
    """
    packed = cu is not None
    batch = len(lens)
    page = kc.shape[1]
    k_all, v_all = cache_values(kc, ks), cache_values(vc, vs)
    D, heads, hk = q.shape[-1], q.shape[-2], kc.shape[2]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64)
    bound = torch.zeros(q.shape, dtype=torch.float64)
    h = HALF_STEP[q.dtype]
    for b in range(batch):
        L = int(lens[b])
        rows = slice(int(cu[b]), int(cu[b + 1])) if packed else b
        qb = q[rows].double()
        n = qb.shape[0]
        if n == 0 or L == 0:
            continue
        j = torch.arange(L)
        pg = table[b].long()[j // page] if table is not None else torch.full_like(j, b)
        kb, vb = k_all[pg, j % page], v_all[pg, j % page]
        pos = torch.arange(n) + (L - n if causal else 0)
        gap = pos[:, None] - j[None]
        seen = torch.ones_like(gap, dtype=torch.bool)
        if causal:
            seen &= gap >= 0
        if window[0] >= 0:
            seen &= gap <= window[0]
        if window[1] >= 0:
            seen &= -gap <= window[1]
        for i in range(heads):
            x = qb[:, i] @ kb[:, i // (heads // hk)].T * scale
            size = qb[:, i].abs() @ kb[:, i // (heads // hk)].abs().T * abs(scale)
            if alibi is not None:
                x = x - alibi[b, i].double() * gap.abs()
                size = size + alibi[b, i].double().abs() * gap.abs()
            if softcap > 0:
                x = softcap * torch.tanh(x / softcap)
                size = size + 8 * softcap     # 1 - 2 / (e + 1) in fp32: steps of the size of 1
            x = x.masked_fill(~seen, -math.inf)
            top = x.max(dim=1, keepdim=True).values
            top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
            p = torch.exp(x - top)
            total = p.sum(dim=1, keepdim=True)
            p = torch.where(total > 0, p / total, torch.zeros_like(p))
            vh = vb[:, i // (heads // hk)]
            mean = p @ vh.abs()
            out[rows][:, i] = p @ vh
            far = torch.where(seen, size, torch.zeros_like(size)).max(dim=1, keepdim=True).values
            drift = (D + 8) * 2.0 ** -24 * 2 * far + 2.0 ** -21
            bound[rows][:, i] = (h * (1 + 2.0 ** -6) * (mean + (p @ vh).abs()) + 2 * drift * mean
                                 + (2.0 ** -24 if q.dtype == torch.float16 else 0.0))
    return out, bound


def slots_of(table, cached, added, free, page, rows, start=0):
    """paged_kvcache_slots in Python: (table, slots, positions, cu, seqlens, free_start)."""
    table = [list(t) for t in table]
    slots, pos, cu, lens, row, end, wanted = [-1] * rows, [0] * rows, [0], [], 0, start, start
    for b, (o, n) in enumerate(zip(cached, added)):
        have, upto = -(-o // page), -(-(o + n) // page)
        ok = upto <= len(table[b]) and row + n <= rows
        if ok:
            wanted += upto - have
            ok = upto == have or wanted <= len(free)
        if ok:
            table[b][have:upto] = free[wanted - (upto - have):wanted] if upto > have else []
            end = wanted
        for i in range(n):
            if row + i < rows:
                pos[row + i] = o + i
                if ok:
                    slots[row + i] = table[b][(o + i) // page] * page + (o + i) % page
        row += n
        cu.append(min(row, rows))
        lens.append(o + n if ok else o)
    return table, slots, pos, cu, lens, end
