"""The serving operators around a paged KV cache held in 8 bits, as a decode loop calls them.

* ``slots``   ``paged_kvcache_slots``: pages and slots of the next tokens of a batch of requests, from their lengths;
* ``append``  ``kvcache_append_8bit``: new K / V rows quantized into the cache, with a power-of-two scale per block of
  tokens and head;
* ``attend``  ``flash_attn_with_kvcache_8bit``: attention of the new queries over that cache.

``listed`` and ``draw`` give the cases (dicts of plain values), ``prepare`` builds what a program holds before the call,
``run`` is one pass (the plain form in elementary torch operations, or the framework's operators where ``own`` is true),
``exact`` the same outputs from the definition in 64 bits, ``work`` the bytes and flops a pass cannot do without.

A cached value is its 8-bit number times 2^(e - 127), ``e`` the byte of its block's scale.
"""
import math
import os
import random
import sys

import torch

own = False

_PKG = os.path.join(os.getcwd(), "flash-attn-triton_amd")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
KINDS = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
TOP_EXPONENT = {"e4m3": 9, "e5m2": 16}   # the largest number of the type is 0.875 * 2^this
DEV = "cuda"


# ----------------------------------------------------------------------------- the cases
def listed():
    return [
        # One decode step of a full batch: every request gets one more token. Latency decides.
        dict(name="slots_decode", kind="slots", B=64, page=64, cols=128, held=8000, new_hi=1, prompts=1.0, lens=0,
             short=False),
        # Continuous batching: most requests decode, some bring a prompt; small pages.
        dict(name="slots_mixed", kind="slots", B=200, page=16, cols=512, held=4000, new_hi=4001, prompts=0.05, lens=1,
             short=False),
        # Thousands of requests of short prompts, and too few free pages for the last of them.
        dict(name="slots_many", kind="slots", B=4096, page=256, cols=16, held=1500, new_hi=64, prompts=1.0, lens=2,
             short=True),
        # One decode step: a token of each of 64 sequences into the cache.
        dict(name="append_decode", kind="append", dtype="bf16", store="e4m3", B=64, Hk=8, D=128, page=256, block=64,
             held=2000, new_lo=1, new_hi=1, lens=3),
        # Prompts of uneven length, the first chunk of each sequence or a later one.
        dict(name="append_prompts", kind="append", dtype="bf16", store="e4m3", B=16, Hk=8, D=128, page=64, block=64,
             held=700, new_lo=300, new_hi=2000, lens=4),
        # A smaller model: 16-token pages with a scale each, wide-range numbers, odd chunks.
        dict(name="append_pages16", kind="append", dtype="fp16", store="e5m2", B=24, Hk=4, D=64, page=16, block=16,
             held=301, new_lo=1, new_hi=133, lens=5),
        # Smallest attention: two short sequences, one token each.
        dict(name="attend_small", kind="attend", dtype="bf16", store="e4m3", B=2, Sq=1, packed=False, Hq=8, Hk=8, D=64,
             page=64, block=64, lo=100, hi=300, lens=6, causal=True, window=-1, alibi=False),
        # One decode step of a full batch of a grouped-query decoder (the paged decode configuration, in 8 bits).
        dict(name="attend_decode", kind="attend", dtype="bf16", store="e4m3", B=64, Sq=1, packed=False, Hq=32, Hk=8,
             D=128, page=256, block=64, lo=512, hi=8192, lens=0, causal=True, window=-1, alibi=False),
        # One very long document and a single token: the key axis is all there is to split.
        dict(name="attend_long", kind="attend", dtype="fp16", store="e4m3", B=1, Sq=1, packed=False, Hq=32, Hk=8, D=128,
             page=256, block=128, lo=131001, hi=131001, lens=7, causal=True, window=-1, alibi=False),
        # A few draft tokens to verify, sliding window and ALiBi, head dim 64, a scale per 16 tokens.
        dict(name="attend_verify", kind="attend", dtype="fp16", store="e5m2", B=16, Sq=5, packed=False, Hq=16, Hk=4,
             D=64, page=16, block=16, lo=200, hi=4097, lens=8, causal=True, window=1024, alibi=True),
        # A chunk of a long prompt against the pages already cached.
        dict(name="attend_chunk", kind="attend", dtype="bf16", store="e4m3", B=4, Sq=512, packed=False, Hq=32, Hk=8,
             D=128, page=256, block=64, lo=512, hi=8192, lens=3, causal=True, window=-1, alibi=False),
        # Continuous batching: packed queries, most of them single tokens beside a few prompt chunks.
        dict(name="attend_mixed", kind="attend", dtype="bf16", store="e4m3", B=40, Sq=700, packed=True, Hq=16, Hk=4,
             D=128, page=64, block=32, lo=700, hi=4000, lens=9, causal=True, window=-1, alibi=False),
    ]


def _log(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    kind = rng.choice(["slots", "append", "attend", "attend"])
    if kind == "slots":
        page = rng.choice([16, 64, 128, 256])
        held, new_hi = _log(rng, 50, 8000), _log(rng, 1, 4000)
        return dict(kind=kind, B=_log(rng, 1, 4096), page=page, cols=-(-(held + new_hi) // page) + rng.randint(0, 20),
                    held=held, new_hi=new_hi, prompts=rng.choice([0.05, 0.3, 1.0]), lens=rng.randint(0, 999),
                    short=rng.random() < 0.3)
    page = rng.choice([16, 64, 128, 256])
    case = dict(kind=kind, dtype=rng.choice(["fp16", "bf16"]), store=rng.choice(["e4m3", "e4m3", "e5m2"]),
                page=page, block=rng.choice([b for b in (16, 32, 64, 128) if b <= page]), D=rng.choice([64, 128]),
                lens=rng.randint(0, 999))
    hq = rng.choice([4, 8, 16, 32])
    hk = rng.choice([h for h in (hq, hq // 2, hq // 4, hq // 8) if h >= 1])
    if kind == "append":
        new_hi = 1 if rng.random() < 0.4 else _log(rng, 2, 4000)
        return dict(case, B=_log(rng, 1, 64), Hk=hk, held=_log(rng, 1, 3000), new_lo=max(1, new_hi // 8), new_hi=new_hi)
    mode = rng.choice(["decode", "decode", "verify", "chunk", "mixed"])
    hi = _log(rng, 64, 130000 if mode == "decode" and rng.random() < 0.3 else 8192)
    sq = {"decode": 1, "verify": rng.randint(2, 8), "chunk": _log(rng, 16, 1024), "mixed": _log(rng, 16, 1024)}[mode]
    sq = min(sq, hi)
    features = rng.random() < 0.3
    most = max(1, min(64, 600000 // hi))
    return dict(case, B=_log(rng, 1, most) if mode != "chunk" else rng.randint(1, min(4, most)), Sq=sq,
                packed=mode == "mixed", Hq=hq, Hk=hk, lo=max(sq, hi // 16), hi=hi, causal=features or mode != "decode",
                window=_log(rng, 64, 2048) if features else -1, alibi=features)


def draw(rng):
    top = {}
    for c in listed():
        w = work(c)
        for k in w:
            top[c["kind"], k] = max(top.get((c["kind"], k), 0), w[k])
    while True:
        case = _draw(rng)
        w = work(case)
        if all(w[k] <= top[case["kind"], k] for k in w):
            return case


# ----------------------------------------------------------------------------- shared pieces
def _lengths(case):
    """(held, new) per request: what is cached before the call and how many tokens it adds (``slots``, ``append``), or
    (cached, queries) (``attend``)."""
    rng = random.Random(case["lens"])
    if case["kind"] == "slots":
        return ([rng.randint(0, case["held"]) for _ in range(case["B"])],
                [rng.randint(1, case["new_hi"]) if rng.random() < case["prompts"] else 1 for _ in range(case["B"])])
    if case["kind"] == "append":
        return ([rng.randint(0, case["held"]) for _ in range(case["B"])],
                [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["B"])])
    cached = [rng.randint(case["lo"], case["hi"]) for _ in range(case["B"])]
    if not case["packed"]:
        return cached, [case["Sq"]] * case["B"]
    # one request in eight brings a chunk (the first one the longest), the others one token
    return cached, [case["Sq"] if b == 0 else rng.randint(2, case["Sq"]) if b % 8 == 0 else 1 for b in range(case["B"])]


def _cu(lengths):
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return cu


def _int(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def _randn(gen, *shape):
    """Activations: normal, a few channels many times larger, the size varying from token to token."""
    x = torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float32)
    x *= torch.exp(torch.randn(shape[0], *([1] * (len(shape) - 1)), generator=gen, device=DEV) * 0.5)
    x[..., ::29] *= 6.0
    return x


def _slopes(heads):
    return (2.0 ** (-8.0 * (torch.arange(heads) + 1) / heads)).float().to(DEV)


def _pow2(e):
    """2^(e - 127) of the scale bytes, exactly, as fp32."""
    e = e.to(torch.int32)
    return torch.where(e == 0, torch.full_like(e, 0x00400000), e << 23).view(torch.float32)


def _scale_byte(amax, store):
    """The least e with amax <= (largest number of the type) * 2^(e - 127); 0 for zeros."""
    m, x = torch.frexp(amax)
    e = x - TOP_EXPONENT[store] + (m > 0.875).to(x.dtype) + 127
    return torch.where(amax > 0, e.clamp(0, 254), torch.zeros_like(e))


def _codes(x, e, store):
    """x (fp32) as the 8-bit numbers of blocks with scale bytes ``e``."""
    inv = _pow2(254 - e)   # 2^(127 - e)
    y = torch.where(torch.isfinite(x), x * inv, torch.full_like(x, float("nan")))
    return y.to(KINDS[store])


def _filled_cache(gen, case, pages):
    """A cache as a serving process holds it: every page full. Quantized page by page (whole blocks)."""
    page, block, hk, d, store = case["page"], case["block"], case["Hk"], case["D"], case["store"]
    cache = torch.empty(pages, page, hk, d, dtype=KINDS[store], device=DEV)
    scale = torch.empty(pages, page // block, hk, dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 27) // (page * hk * d))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        x = _randn(gen, n * page, hk, d).view(n, page // block, block, hk, d)
        e = _scale_byte(x.abs().amax(dim=(2, 4)), store)
        cache[p:p + n] = _codes(x, e[:, :, None, :, None], store).view(n, page, hk, d)
        scale[p:p + n] = e.to(torch.uint8)
    return cache, scale.view(torch.float8_e8m0fnu)


# ----------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    cached, new = _lengths(case)
    page = case["page"]
    state = dict(case)
    if case["kind"] == "slots":
        have = [-(-o // page) for o in cached]
        need = [-(-(o + n) // page) - h for o, n, h in zip(cached, new, have)]
        spare = sum(need) // 2 if case["short"] else sum(need) + 7
        total = sum(have) + spare + 5
        ids = torch.randperm(total, generator=gen, device=DEV).to(torch.int32)
        table = torch.full((case["B"], case["cols"]), -1, dtype=torch.int32, device=DEV)
        at = torch.arange(case["cols"], device=DEV)[None] < _int(have)[:, None]
        table[at] = ids[:sum(have)]
        state.update(table=table, cached=_int(cached), new=_int(new), free=ids[sum(have):], start=_int([5]),
                     rows=sum(new) + 13)
        return state
    if case["kind"] == "append":
        ends = [o + n for o, n in zip(cached, new)]
        counts = [-(-e // page) for e in ends]
        pages = sum(counts) + 3
        kc, ks = _filled_cache(gen, case, pages)
        vc, vs = _filled_cache(gen, case, pages)
        ids = torch.randperm(pages, generator=gen, device=DEV)
        first = _cu(counts)
        slots = []
        for b in range(case["B"]):
            pos = torch.arange(cached[b], ends[b], device=DEV)
            slots.append(ids[first[b] + pos // page] * page + pos % page)
        slots = torch.cat(slots)
        rows = slots.numel()
        dt = DTYPES[case["dtype"]]
        state.update(k=_randn(gen, rows, case["Hk"], case["D"]).to(dt), v=_randn(gen, rows, case["Hk"], case["D"]).to(dt),
                     k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, slots=slots)
        return state
    counts = [-(-o // page) for o in cached]
    pages = sum(counts) + 3
    kc, ks = _filled_cache(gen, case, pages)
    vc, vs = _filled_cache(gen, case, pages)
    table = torch.zeros((case["B"], max(counts) + 2), dtype=torch.int32, device=DEV)
    at = torch.arange(table.shape[1], device=DEV)[None] < _int(counts)[:, None]
    table[at] = torch.randperm(pages, generator=gen, device=DEV)[:sum(counts)].to(torch.int32)
    shape = (sum(new),) if case["packed"] else (case["B"], case["Sq"])
    q = torch.randn(*shape, case["Hq"], case["D"], generator=gen, device=DEV).to(DTYPES[case["dtype"]])
    state.update(q=q, k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, table=table, cached=_int(cached),
                 cu=_int(_cu(new)) if case["packed"] else None, max_q=max(new), max_k=max(cached),
                 slopes=_slopes(case["Hq"]) if case["alibi"] else None)
    return state


# ----------------------------------------------------------------------------- one pass
def run(state):
    if own:
        return _run_own(state)
    return {"slots": _plain_slots, "append": _plain_append, "attend": _plain_attend}[state["kind"]](state)


def _run_own(s):
    import flash_attn_triton as fa

    # The tables and slots come from paged_kvcache_slots, so the loop does not have each step's copy checked again
    # (validate=True reads device arrays back to the host).
    if s["kind"] == "slots":
        got = fa.paged_kvcache_slots(s["table"], s["cached"], s["new"], s["free"], s["page"], s["rows"],
                                     free_start=s["start"], validate=False)
        return {"slots": got[0], "positions": got[1], "cu": got[2], "seqlens": got[3], "free_start": got[4],
                "table": s["table"]}
    if s["kind"] == "append":
        fa.kvcache_append_8bit(s["k"], s["v"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["slots"],
                               validate=False)
        return {"k_cache": s["k_cache"], "v_cache": s["v_cache"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    return fa.flash_attn_with_kvcache_8bit(
        s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], cache_seqlens=s["cached"],
        block_table=s["table"], cu_seqlens_q=s["cu"], max_seqlen_q=s["max_q"] if s["packed"] else None,
        max_seqlen_k=s["max_k"], causal=s["causal"], window_size=(s["window"], -1), alibi_slopes=s["slopes"],
        validate=False)


def _plain_slots(s):
    """Requests in order: request b takes the free pages its new tokens need; one that does not fit its table row, or
    for which the free pages do not reach, gets no page and slots of -1, and keeps its length."""
    table, page, rows = s["table"], s["page"], s["rows"]
    old, new = s["cached"].long(), s["new"].long()
    cu = torch.cat([torch.zeros_like(new[:1]), torch.cumsum(new, 0)])
    have, end = (old + page - 1) // page, old + new
    fits = (end <= table.shape[1] * page) & (cu[1:] <= rows)
    need = torch.where(fits, (end + page - 1) // page - have, torch.zeros_like(have))
    upto = torch.cumsum(need, 0)
    left = s["free"].numel() - s["start"].long()
    served = fits & ((need == 0) | (upto <= left))
    start = s["start"].long()
    col = torch.arange(table.shape[1], device=table.device)[None]
    at = col - have[:, None]
    takes = served[:, None] & (at >= 0) & (at < need[:, None])
    which = (start + (upto - need)[:, None] + at).clamp(0, s["free"].numel() - 1)
    table.copy_(torch.where(takes, s["free"][which], table))
    r = torch.arange(rows, device=table.device)
    b = torch.searchsorted(cu[1:], r, right=True)
    inside = b < new.numel()
    b = b.clamp(max=new.numel() - 1)
    pos = torch.where(inside, old[b] + r - cu[b], torch.zeros_like(r))
    ok = inside & served[b]
    entry = table[b, (pos // page).clamp(max=table.shape[1] - 1)].long()
    slots = torch.where(ok & (entry >= 0), entry * page + pos % page, torch.full_like(r, -1))
    taken = torch.where(served, upto, torch.zeros_like(upto)).amax().reshape(1)
    return {"slots": slots, "positions": pos.int(), "cu": cu.clamp(max=rows).int(),
            "seqlens": torch.where(served, end, old).int(), "free_start": (start + taken).int(), "table": table}


def _plain_append(s):
    """Each block's scale grows to hold its new rows (a block begun by them starts anew), the rows that it holds already
    are rounded to the new scale, and the new ones quantized."""
    block, store, slots = s["block"], s["store"], s["slots"]
    for x, cache, scale in ((s["k"], s["k_cache"], s["k_scale"]), (s["v"], s["v_cache"], s["v_scale"])):
        hk, d = x.shape[1:]
        x = x.float()
        bytes_, codes = scale.view(torch.uint8).view(-1, hk), cache.view(torch.uint8).view(-1, hk, d)
        which = slots // block
        first = torch.full((bytes_.shape[0],), block, device=x.device).scatter_reduce(0, which, slots % block, "amin")
        amax = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(dim=2)
        most = torch.zeros(bytes_.shape, device=x.device).scatter_reduce(0, which[:, None].expand(-1, hk), amax, "amax")
        begins = slots[slots % block == first[which]]   # one row of each block
        g = begins // block
        old = torch.where((first[g] > 0)[:, None], bytes_[g].int(), torch.zeros_like(bytes_[g].int()))
        e = torch.maximum(old, _scale_byte(most[g], store))
        at = (g * block)[:, None] + torch.arange(block, device=x.device)[None]
        held = codes[at].view(KINDS[store]).float()
        moved = (held * _pow2((old + 127 - e).clamp(min=0))[:, None, :, None]).to(KINDS[store]).view(torch.uint8)
        keep = (torch.arange(block, device=x.device)[None] < first[g][:, None]) & (old < e).any(dim=1)[:, None]
        codes[at[keep]] = torch.where((old < e)[:, None, :, None], moved, codes[at])[keep]
        bytes_[g] = e.to(torch.uint8)
        codes[slots] = _codes(x, bytes_[which].int()[:, :, None], store).view(torch.uint8)
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _gather(cache, scale, table, s):
    """The keys or values of every sequence, padded to the longest: [B, max_k, Hk, D] fp32."""
    page, block = s["page"], s["block"]
    j = torch.arange(s["max_k"], device=table.device)
    p = table[:, j // page].long()
    codes = cache.view(torch.uint8)[p, j % page].view(KINDS[s["store"]])
    return codes.float() * _pow2(scale.view(torch.uint8)[p, j % page // block])[..., None]


def _plain_attend(s):
    q, hk = s["q"], s["Hk"]
    group, d = s["Hq"] // hk, s["D"]
    k = _gather(s["k_cache"], s["k_scale"], s["table"], s)
    v = _gather(s["v_cache"], s["v_scale"], s["table"], s)
    cached, sq, sk = s["cached"].long(), s["max_q"], s["max_k"]
    i, j = torch.arange(sq, device=q.device), torch.arange(sk, device=q.device)
    if s["packed"]:
        cu = s["cu"].long()
        count = cu[1:] - cu[:-1]
        qp = q[(cu[:-1, None] + i).clamp(max=q.shape[0] - 1)]
    else:
        count, qp = torch.full_like(cached, sq), q
    batch = qp.shape[0]
    qh = qp.float().view(batch, sq, hk, group, d).permute(0, 2, 3, 1, 4).reshape(batch, hk, group * sq, d)
    score = torch.matmul(qh, k.permute(0, 2, 3, 1)).view(batch, hk, group, sq, sk)
    score *= 1.0 / math.sqrt(d)
    at = i[None] + (cached - count)[:, None] if s["causal"] else i[None].expand(batch, -1)   # position of query i
    gap = at[:, :, None] - j[None, None]
    seen = (j[None] < cached[:, None])[:, None].expand(-1, sq, -1)
    if s["causal"]:
        seen = seen & (gap >= 0)
    if s["window"] >= 0:
        seen = seen & (gap <= s["window"])
    if s["slopes"] is not None:
        score -= s["slopes"].view(1, hk, group, 1, 1) * gap.abs().float()[:, None, None]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    score.sub_(torch.where(torch.isfinite(top), top, torch.zeros_like(top))).exp_()
    total = score.sum(dim=-1, keepdim=True)
    vis = torch.where(j[None, :, None, None] < cached[:, None, None, None], v, torch.zeros_like(v))
    out = torch.matmul(score.view(batch, hk, group * sq, sk), vis.permute(0, 2, 1, 3)).view(batch, hk, group, sq, d)
    out = out / torch.where(total > 0, total, torch.ones_like(total))
    out = out.permute(0, 3, 1, 2, 4).reshape(batch, sq, hk * group, d).to(q.dtype)
    if s["packed"]:
        r = torch.arange(q.shape[0], device=q.device)
        b = torch.searchsorted(cu[1:], r, right=True)
        out = out[b, r - cu[b]]
    return out


# ----------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"slots": _exact_slots, "append": _exact_append, "attend": _exact_attend}[case["kind"]](s)


def _exact_slots(s):
    table, old, new = (s[k].tolist() for k in ("table", "cached", "new"))
    free, page, at, row = s["free"].tolist(), s["page"], int(s["start"]), 0
    wanted = at
    slots, positions, lengths, cu = [-1] * s["rows"], [0] * s["rows"], [], [0]
    for b, (o, n) in enumerate(zip(old, new)):
        have, upto = -(-o // page), -(-(o + n) // page)
        ok = o + n <= s["cols"] * page and row + n <= s["rows"]
        if ok and upto > have:
            wanted += upto - have
            ok = wanted <= len(free)
            if ok:
                table[b][have:upto] = free[at:wanted]
                at = wanted
        for i in range(n):
            if row + i < s["rows"]:
                p = o + i
                positions[row + i] = p
                if ok and table[b][p // page] >= 0:
                    slots[row + i] = table[b][p // page] * page + p % page
        row += n
        cu.append(min(row, s["rows"]))
        lengths.append(o + n if ok else o)
    return {"slots": _int(slots, torch.int64), "positions": _int(positions), "cu": _int(cu), "seqlens": _int(lengths),
            "free_start": _int([at]), "table": _int(table)}


def _value64(cache, scale, block):
    """The numbers a cache stands for, in 64 bits."""
    e = scale.view(torch.uint8).double().repeat_interleave(block, dim=1)
    return cache.double() * torch.exp2(e - 127.0)[..., None]


def _exact_append(s):
    block, store = s["block"], s["store"]
    mantissa, low, top = {"e4m3": (3, -6, 448.0), "e5m2": (2, -14, 57344.0)}[store]

    def nearest(y):   # to the 8-bit numbers of the type, ties to even
        e = torch.frexp(y.abs())[1].double() - 1.0
        step = torch.exp2(torch.clamp(e, min=low) - mantissa)
        return torch.round(y / step) * step

    out = {}
    blocks = (s["slots"] // block).tolist()
    cuts = [i for i in range(len(blocks)) if i == 0 or blocks[i] != blocks[i - 1]] + [len(blocks)]
    lo, hi = torch.tensor(cuts[:-1], device=DEV), torch.tensor(cuts[1:], device=DEV)
    for name in ("k", "v"):
        x, cache, scale = s[name].double(), s[name + "_cache"].double(), s[name + "_scale"].view(torch.uint8).clone()
        flat, table = cache.view(-1, *x.shape[1:]), scale.view(-1, x.shape[1])
        # largest magnitude of each run, from a padded [runs, block] view of the new rows
        r = lo[:, None] + torch.arange(block, device=DEV)
        inside = r < hi[:, None]
        r = r.clamp(max=x.shape[0] - 1)
        most = torch.where(inside[..., None], x[r].abs().amax(dim=3), 0.0).amax(dim=1)
        want = torch.ceil(torch.log2(most / top)) + 127.0
        want = want + (most > top * torch.exp2(want - 127.0)).double() - (most <= top * torch.exp2(want - 128.0)).double()
        g, first = s["slots"][lo] // block, s["slots"][lo] % block
        old = table[g].double()
        e = torch.where((first > 0)[:, None], torch.maximum(old, want), want).clamp(0, 254)
        at = (g * block)[:, None] + torch.arange(block, device=DEV)
        held = torch.arange(block, device=DEV)[None] < first[:, None]
        moved = torch.where((e > old)[:, None, :, None], nearest(flat[at] * torch.exp2(old - e)[:, None, :, None]), flat[at])
        flat[at[held]] = moved[held]
        run_of = torch.repeat_interleave(torch.arange(lo.numel(), device=DEV), hi - lo)
        flat[s["slots"]] = nearest(x * torch.exp2(127.0 - e[run_of])[..., None])
        table[g] = e.to(torch.uint8)
        out[name + "_cache"], out[name + "_scale"] = cache, scale.view(torch.float8_e8m0fnu).double()
    return out


def _exact_attend(s):
    page, group = s["page"], s["Hq"] // s["Hk"]
    cached, cu = s["cached"].tolist(), s["cu"].tolist() if s["packed"] else None
    outs = []
    for b, length in enumerate(cached):
        q = (s["q"][cu[b]:cu[b + 1]] if s["packed"] else s["q"][b]).double()
        pages = s["table"][b, :-(-length // page)].long()
        k, v = (_value64(s[c][pages], s[e][pages], s["block"]).flatten(0, 1)[:length]
                for c, e in (("k_cache", "k_scale"), ("v_cache", "v_scale")))
        n = q.shape[0]
        at = torch.arange(n, device=DEV) + (length - n if s["causal"] else 0)
        gap = at[:, None] - torch.arange(length, device=DEV)[None]
        hidden = torch.zeros_like(gap, dtype=torch.bool)
        if s["causal"]:
            hidden |= gap < 0
        if s["window"] >= 0:
            hidden |= gap > s["window"]
        heads = []
        for h in range(s["Hq"]):
            score = q[:, h] @ k[:, h // group].T.contiguous() / math.sqrt(s["D"])
            if s["slopes"] is not None:
                score = score - s["slopes"][h].double() * gap.abs()
            p = torch.softmax(score.masked_fill(hidden, -math.inf), dim=1)
            heads.append(torch.nan_to_num(p) @ v[:, h // group].contiguous())
        outs.append(torch.stack(heads, dim=1))
    return torch.cat(outs) if s["packed"] else torch.stack(outs)


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    cached, new = _lengths(case)
    page, rows = case["page"], sum(new)
    if case["kind"] == "slots":
        # lengths in, lengths and offsets out, a table entry per page that new tokens fall on, its number from the list,
        # a slot (8 bytes) and a position (4) per token
        entries = sum(-(-(o + n) // page) - o // page for o, n in zip(cached, new))
        return {"bytes": 16 * case["B"] + 8 * entries + 12 * rows, "flops": 0}
    hk, d = case["Hk"], case["D"]
    if case["kind"] == "append":
        # both tensors: 2 bytes in and 1 out per value, a scale byte per block and head touched
        blocks = sum(-(-(o + n) // case["block"]) - o // case["block"] for o, n in zip(cached, new))
        return {"bytes": 2 * (3 * rows * hk * d + blocks * hk) + 8 * rows, "flops": 4 * rows * hk * d}
    pairs = keys = 0
    for length, n in zip(cached, new):
        low = length
        for i in ([0] if n == 1 else range(n)):
            at = length - n + i if case["causal"] else i
            end = min(length, at + 1) if case["causal"] else length
            begin = max(0, at - case["window"]) if case["window"] >= 0 else 0
            pairs += max(0, end - begin)
            low = min(low, begin)
        keys += length - low
    return {"bytes": 2 * keys * hk * d + 2 * keys * hk // case["block"] + 4 * rows * case["Hq"] * d,
            "flops": 4 * pairs * case["Hq"] * d}
