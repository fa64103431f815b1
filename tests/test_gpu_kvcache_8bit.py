"""The 8-bit KV cache operators against plain float64 forms (_kv8.py)."""
import math
import random

import pytest
import torch

import _kv8
from _kv8 import STORES

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _fa():
    import flash_attn_triton
    return flash_attn_triton


# ----------------------------------------------------------------------------- slots
def _slots_case(batch, page, held, new_hi, seed, spare=5, cols_more=2, zero_new=False, rows_more=3):
    rng = random.Random(seed)
    cached = [rng.choice([0, rng.randint(0, held), page * rng.randint(0, held // page + 1)]) for _ in range(batch)]
    added = [rng.randint(0 if zero_new else 1, new_hi) for _ in range(batch)]
    have = [-(-o // page) for o in cached]
    need = [-(-(o + n) // page) - h for o, n, h in zip(cached, added, have)]
    cols = max(h + x for h, x in zip(have, need)) + cols_more
    ids = list(range(sum(have) + max(sum(need) + spare, 1)))
    rng.shuffle(ids)
    it = iter(ids)
    table = [[next(it) for _ in range(h)] + [-7] * (cols - h) for h in have]
    return table, cached, added, list(it), sum(added) + rows_more


def _run_slots(table, cached, added, free, page, rows, start=None, ints=torch.int32, **kw):
    t = torch.tensor(table, dtype=torch.int32, device=DEV).reshape(len(table), len(table[0]) if table else 2)
    got = _fa().paged_kvcache_slots(
        t, torch.tensor(cached, dtype=ints, device=DEV), torch.tensor(added, dtype=ints, device=DEV),
        torch.tensor(free, dtype=torch.int32, device=DEV), page, rows,
        free_start=None if start is None else torch.tensor([start], dtype=torch.int32, device=DEV), **kw)
    return t, got


def _check_slots(table, cached, added, free, page, rows, start=None, **kw):
    t, got = _run_slots(table, cached, added, free, page, rows, start, **kw)
    want = _kv8.slots_of(table, cached, added, free, page, rows, start or 0)
    assert t.tolist() == want[0]
    assert got[0].dtype == torch.int64 and got[0].tolist() == want[1]
    assert got[1].tolist() == want[2]
    assert got[2].tolist() == want[3]
    assert got[3].tolist() == want[4]
    assert got[4].tolist() == [want[5]]


@pytest.mark.parametrize("batch", [1, 2, 63, 64, 65, 300])
@pytest.mark.parametrize("page", [1, 16, 48, 256])
def test_slots(batch, page):
    table, cached, added, free, rows = _slots_case(batch, page, 600, 40, batch + page)
    _check_slots(table, cached, added, free, page, rows)


@pytest.mark.parametrize("batch", [511, 512, 513, 1100, 2047, 2048, 2049, 5000])
def test_slots_of_many_requests(batch):
    table, cached, added, free, rows = _slots_case(batch, 16, 100, 9, batch, zero_new=True)
    _check_slots(table, cached, added, free, 16, rows, ints=torch.int64)


def test_slots_of_long_prompts():
    table, cached, added, free, rows = _slots_case(9, 64, 5000, 40000, 1)
    _check_slots(table, cached, added, free, 64, rows)


@pytest.mark.parametrize("batch", [7, 2500])
def test_slots_with_too_few_pages(batch):
    table, cached, added, free, rows = _slots_case(batch, 16, 200, 40, 3, zero_new=True)
    need = sum(-(-(o + n) // 16) - -(-o // 16) for o, n in zip(cached, added))
    for left in (0, 1, need // 2, need - 1):
        _check_slots(table, cached, added, free[:left] or [0][:left], 16, rows)
    _check_slots(table, cached, added, free, 16, rows, start=3)
    _check_slots(table, cached, added, free, 16, rows, start=len(free))
    _check_slots(table, cached, added, free, 16, rows, start=len(free) + 9)


def test_slots_refused_requests_are_not_overtaken():
    # request 1 needs 3 of 2 pages, request 2 none, request 3 one: the index passes the list, and stays there
    table = [[0, -1, -1, -1], [1, -1, -1, -1], [2, -1, -1, -1], [3, -1, -1, -1]]
    cached, added, free = [16, 16, 5, 16], [1, 48, 1, 0], [7, 8, 9]
    _check_slots(table, cached, added, free, 16, 60)
    t, got = _run_slots(table, cached, added, free, 16, 60)
    assert got[3].tolist() == [17, 16, 6, 16] and got[4].tolist() == [4]


def test_slots_without_tokens_or_requests():
    _check_slots([[1, 2], [3, 4]], [5, 0], [0, 0], [9], 16, 0)
    _check_slots([[1, 2], [3, 4]], [5, 0], [0, 0], [9], 16, 4)
    t, got = _run_slots([], [], [], [1, 2], 16, 3)
    assert [x.tolist() for x in got] == [[-1] * 3, [0] * 3, [0], [], [0]]


def test_slots_refuses_requests_that_do_not_fit_their_row():
    # request 1 passes its row of the table, request 3 the packed rows
    table = [[0, -1], [1, -1], [2, -1], [3, -1]]
    for rows in (60, 40, 36, 3):
        _check_slots(table, [10, 15, 16, 1], [4, 18, 16, 5], [20, 21, 22, 23], 16, rows, validate=False)


def test_slots_leave_what_they_do_not_own():
    table, cached, added, free, rows = _slots_case(5, 16, 100, 20, 8)
    wide = torch.full((5, len(table[0]) + 6), -3, dtype=torch.int32, device=DEV)
    view = wide[:, 2:2 + len(table[0])]
    view.copy_(torch.tensor(table, dtype=torch.int32))
    _fa().paged_kvcache_slots(view, torch.tensor(cached, device=DEV), torch.tensor(added, device=DEV),
                              torch.tensor(free, dtype=torch.int32, device=DEV), 16, rows)
    assert view.tolist() == _kv8.slots_of(table, cached, added, free, 16, rows)[0]
    assert bool((wide[:, :2] == -3).all()) and bool((wide[:, 2 + len(table[0]):] == -3).all())


def test_slots_refusals():
    with pytest.raises(ValueError, match="valid lengths"):
        _run_slots([[0, 1]], [-1], [1], [5], 16, 4)
    with pytest.raises(ValueError, match="non-negative"):
        _run_slots([[0, 1]], [1], [-1], [5], 16, 4)
    with pytest.raises(ValueError, match="do not fit in the block table"):
        _run_slots([[0, 1]], [20], [13], [5], 16, 40)
    with pytest.raises(ValueError, match="max_tokens must cover"):
        _run_slots([[0, 1]], [20], [5], [5], 16, 4)
    with pytest.raises(ValueError, match="free_start must be"):
        _run_slots([[0, 1]], [20], [5], [5], 16, 5, start=-1)


# ----------------------------------------------------------------------------- append
def _append(k, v, kc, ks, vc, vs, slots, **kw):
    dev = [t.to(DEV) for t in (k, v, kc, vc, ks, vs)]
    _fa().kvcache_append_8bit(*dev, slots.to(DEV), **kw)
    return [t.cpu() for t in dev[2:]]


def _check_append(k, v, kc, ks, vc, vs, slots, **kw):
    got = _append(k, v, kc, ks, vc, vs, slots, **kw)
    for x, c, s, gc, gs in ((k, kc, ks, got[0], got[2]), (v, vc, vs, got[1], got[3])):
        wc, ws = _kv8.append(x, c, s, slots)
        assert torch.equal(gs.view(torch.uint8), ws.view(torch.uint8))
        assert _kv8.same_bytes(gc, wc)


def _rows(n, heads, dim, dtype, seed, spread=3.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(n, heads, dim, generator=gen) * torch.exp(torch.randn(n, heads, 1, generator=gen) * spread)
    return x.clamp(-6e4, 6e4).to(dtype)


def _run_slots_list(runs):
    return torch.tensor([s + i for s, n in runs for i in range(n)], dtype=torch.int64)


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_append(dtype, store, dim):
    # runs that begin a block, begin inside one, fill one, cross blocks and pages; single tokens
    page, block, heads = 64, 32, 3
    kc, ks = _kv8.filled(9, page, block, heads, dim, STORES[store], 1)
    vc, vs = _kv8.filled(9, page, block, heads, dim, STORES[store], 2)
    slots = _run_slots_list([(2 * 64 + 5, 1), (3, 90), (5 * 64, 64), (7 * 64 + 33, 4), (4 * 64 + 31, 1), (6 * 64 + 17, 30)])
    k, v = (_rows(len(slots), heads, dim, dtype, s) for s in (3, 4))
    _check_append(k, v, kc, ks, vc, vs, slots)


@pytest.mark.parametrize("block,page", [(16, 16), (16, 48), (64, 64), (128, 256), (512, 512)])
@pytest.mark.parametrize("rows", [1, 700])
def test_append_blocks(block, page, rows):
    # 700 rows of 24 heads are more than the single-row windows serve
    heads, pages = 24 if rows > 1 else 2, 900 // page + 3
    kc, ks = _kv8.filled(pages, page, block, heads, 64, torch.float8_e4m3fn, 1)
    vc, vs = _kv8.filled(pages, page, block, heads, 64, torch.float8_e4m3fn, 2)
    slots = _run_slots_list([(page + 7, rows)])
    k, v = (_rows(rows, heads, 64, torch.bfloat16, s) for s in (3, 4))
    _check_append(k, v, kc, ks, vc, vs, slots)


def test_append_windows_of_many_runs():
    # many short runs within one window, runs across window ends, skipped rows between them
    page = block = 64
    rng = random.Random(0)
    runs, pages = [], 160
    for p in rng.sample(range(pages), 150):
        first = rng.randint(0, 60)
        runs.append((p * page + first, rng.randint(1, 64 - first)))
    slots = _run_slots_list(runs)
    keep = torch.rand(len(slots), generator=torch.Generator().manual_seed(1)) < 0.97
    slots = torch.where(keep, slots, torch.full_like(slots, -1))
    # (a skipped row splits its run: the part behind it would share the block)
    seen, out = set(), []
    for i, s in enumerate(slots.tolist()):
        cont = i and out[-1] >= 0 and s == out[-1] + 1 and s % block
        if s >= 0 and not cont and s // block in seen:
            s = -1
        if s >= 0:
            seen.add(s // block)
        out.append(s)
    slots = torch.tensor(out)
    for heads, n in ((2, 600), (8, len(slots))):
        kc, ks = _kv8.filled(pages, page, block, heads, 64, torch.float8_e4m3fn, 1)
        vc, vs = _kv8.filled(pages, page, block, heads, 64, torch.float8_e4m3fn, 2)
        k, v = (_rows(n, heads, 64, torch.float16, s) for s in (3, 4))
        _check_append(k, v, kc, ks, vc, vs, slots[:n])


@pytest.mark.parametrize("store", STORES)
def test_append_special_numbers(store):
    st = STORES[store]
    top = 1.75 * 2.0 ** _kv8.TOP[st]
    kinds = [0.0, -0.0, math.inf, -math.inf, math.nan, top, top * 2, top * 1.0000001, top * 1.5, 2.0 ** -126, 2.0 ** -149,
             1e-40, 3.4e38, 2.0 ** 127, 1.0, 1.0625, 1.1875, -1.0625, 2.0 ** -9, 2.0 ** -10, 2.0 ** -16, 2.0 ** -17]
    kc, ks = _kv8.filled(len(kinds) + 4, 16, 16, 1, 64, st, 1)
    vc, vs = _kv8.filled(len(kinds) + 4, 16, 16, 1, 64, st, 2)
    # one block each: the number beside smaller ones; then a whole block of it
    k = torch.zeros(2 * len(kinds), 1, 64)
    v = torch.zeros(2 * len(kinds), 1, 64)
    for i, x in enumerate(kinds):
        small = x if math.isfinite(x) else 3.0
        k[2 * i, 0] = torch.tensor([x] + [small * 2.0 ** -(j % 20) for j in range(63)])
        k[2 * i + 1, 0] = small * 0.3
        v[2 * i:2 * i + 2] = x
    slots = torch.tensor([s for i in range(len(kinds)) for s in (16 * i + (i % 3), 16 * i + (i % 3) + 1)])
    _check_append(k, v, kc, ks, vc, vs, slots)
    _check_append(k.bfloat16(), v.bfloat16(), kc, ks, vc, vs, slots)


def test_append_scale_only_grows_within_a_block():
    # a block written token by token holds what its final scale gives, and its
    # scale bounds every number by the type's largest
    for st in STORES.values():
        kc = torch.zeros(1, 32, 2, 64).to(st)
        ks = torch.full((1, 1, 2), 200, dtype=torch.uint8).view(torch.float8_e8m0fnu)   # left by an earlier owner
        k = _rows(32, 2, 64, torch.bfloat16, 5, spread=2.0)
        dev = [t.to(DEV) for t in (kc, kc, ks, ks)]
        for t in range(32):
            _fa().kvcache_append_8bit(k[t:t + 1].to(DEV), k[t:t + 1].to(DEV), *dev, torch.tensor([t], device=DEV),
                                      validate=False)
        want = [_kv8.scale_of(float(k[:, h].abs().max()), st) for h in range(2)]
        assert dev[2].cpu().view(torch.uint8).flatten().tolist() == want
        got = _kv8.cache_values(dev[0].cpu(), dev[2].cpu())[0]
        # one rounding to a number of 2 (3) fraction bits at first, and those
        # of numbers that became subnormal: 2^-9 or 2^-16 steps of the final scale, up to once per growth
        half = 2.0 ** -3 if st == torch.float8_e5m2 else 2.0 ** -4
        sub = (2.0 ** -16 if st == torch.float8_e5m2 else 2.0 ** -9) * torch.exp2(torch.tensor(want, dtype=torch.float64) - 127)
        assert bool(((got - k.double()).abs() <= half * k.double().abs() + sub[None, :, None]).all())


def test_append_strided_rows_and_head_major_cache():
    heads, dim, page, block = 4, 64, 32, 16
    qkv = torch.randn(50, 3, heads, dim, generator=torch.Generator().manual_seed(0)).half()
    kc, ks = _kv8.filled(4, page, block, heads, dim, torch.float8_e4m3fn, 1)
    vc, vs = _kv8.filled(4, page, block, heads, dim, torch.float8_e4m3fn, 2)
    slots = _run_slots_list([(32 + 3, 50)])
    want = [_kv8.append(qkv[:, i], c, s, slots) for i, c, s in ((1, kc, ks), (2, vc, vs))]
    pool = torch.zeros(2, 4, heads, page, dim, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    kd, vd = (x.transpose(1, 2) for x in pool)
    kd.view(torch.uint8).copy_(kc.view(torch.uint8))
    vd.view(torch.uint8).copy_(vc.view(torch.uint8))
    kss, vss = (s.view(torch.uint8).permute(2, 0, 1).contiguous().permute(1, 2, 0).to(DEV).view(torch.float8_e8m0fnu)
                for s in (ks, vs))
    qd = qkv.to(DEV)
    _fa().kvcache_append_8bit(qd[:, 1], qd[:, 2], kd, vd, kss, vss, slots.to(DEV))
    for (wc, ws), c, s in zip(want, (kd, vd), (kss, vss)):
        assert _kv8.same_bytes(c.cpu().contiguous(), wc)
        assert torch.equal(s.cpu().view(torch.uint8), ws.view(torch.uint8))


def test_append_skips_what_lies_outside():
    kc, ks = _kv8.filled(2, 16, 16, 1, 64, torch.float8_e4m3fn, 1)
    slots = torch.tensor([-1, 32, 5, 6, -1, 2 ** 40, -2 ** 50, 31, 32, 33])
    k = _rows(10, 1, 64, torch.bfloat16, 2)
    _check_append(k, k, kc, ks, kc, ks, slots, validate=False)


def test_append_of_no_rows():
    kc, ks = _kv8.filled(2, 16, 16, 1, 64, torch.float8_e4m3fn, 1)
    _check_append(torch.zeros(0, 1, 64).half(), torch.zeros(0, 1, 64).half(), kc, ks, kc, ks,
                  torch.zeros(0, dtype=torch.int64))


def test_append_refuses_targets_that_share_memory():
    kc, ks = (t.to(DEV) for t in _kv8.filled(2, 32, 16, 2, 64, torch.float8_e4m3fn, 1))
    vc, vs = kc.clone(), ks.clone()
    k, slots = torch.zeros(1, 2, 64, device=DEV).half(), torch.zeros(1, dtype=torch.int64, device=DEV)
    before = kc.cpu().view(torch.uint8).clone()
    for cache in ((kc, kc, ks, vs), (kc, vc, ks, ks)):
        with pytest.raises(ValueError, match="must not share"):
            _fa().kvcache_append_8bit(k, k, *cache, slots, validate=False)
    for cache in ((kc[:, :, :1].expand(-1, -1, 2, -1), vc, ks, vs), (kc, vc[:1].expand(2, -1, -1, -1), ks, vs),
                  (kc, vc, ks, vs[:, :1].expand(-1, 2, -1)), (kc, vc, ks.as_strided((2, 2, 2), (4, 1, 1)), vs)):
        with pytest.raises(ValueError, match="share memory"):
            _fa().kvcache_append_8bit(k, k, *cache, slots, validate=False)
    assert torch.equal(kc.cpu().view(torch.uint8), before)
    # K and V side by side in one allocation do not
    both = torch.stack([kc.view(torch.uint8)] * 2, dim=3).view(torch.float8_e4m3fn)
    _fa().kvcache_append_8bit(k, k, both[:, :, :, 0], both[:, :, :, 1], ks, vs, slots)
    assert not bool(both[0, 0].float().any()) and _kv8.same_bytes(both[0, 16:, :, 0].cpu(), kc[0, 16:].cpu())


def test_append_refusals():
    kc, ks = (t.to(DEV) for t in _kv8.filled(2, 32, 16, 1, 64, torch.float8_e4m3fn, 1))
    k = torch.zeros(4, 1, 64, device=DEV).half()

    def call(slots, k=k):
        _fa().kvcache_append_8bit(k, k, kc, kc.clone(), ks, ks.clone(), torch.tensor(slots, device=DEV))
    before = kc.cpu().view(torch.uint8).clone()
    for slots in ([0, 1, 2, 64], [0, 1, -2, 3]):
        with pytest.raises(ValueError, match="slot outside the cache"):
            call(slots)
    for slots in ([0, 1, 3, 4], [1, 0, 40, 41], [5, 5, 40, 41], [0, 16, 1, 17], [3, -1, 4, 5]):
        with pytest.raises(ValueError, match="two runs"):
            call(slots)
    assert torch.equal(kc.cpu().view(torch.uint8), before)
    call([15, 16, -1, -1])
    with pytest.raises(ValueError, match="no backward"):
        call([0, 1, 2, 3], k.clone().requires_grad_())


# ----------------------------------------------------------------------------- attention
def _table(lens, page, seed, pages_more=2, cols_more=1):
    counts = [-(-n // page) for n in lens]
    ids = torch.randperm(sum(counts) + pages_more, generator=torch.Generator().manual_seed(seed)).tolist()
    t = torch.zeros(len(lens), max(counts) + cols_more, dtype=torch.int32)
    at = 0
    for b, n in enumerate(counts):
        t[b, :n] = torch.tensor(ids[at:at + n])
        at += n
    return t, sum(counts) + pages_more


def _poison(kc, ks, vc, vs, lens, table, store):
    """NaN in every slot that no sequence holds, scales of blocks without any too."""
    page, block = kc.shape[1], kc.shape[1] // ks.shape[1]
    used = torch.zeros(kc.shape[:2], dtype=torch.bool)
    for b, n in enumerate(lens):
        for c in range(-(-n // page)):
            used[table[b, c], :min(page, n - c * page)] = True
    for c, s in ((kc, ks), (vc, vs)):
        c.view(torch.uint8)[~used] = 0x7f
        s.view(torch.uint8)[~used.view(kc.shape[0], -1, block).any(dim=2)] = 0xff


def _check_attend(lens, sq, heads, hk, dim, dtype, store, page=64, block=32, causal=True, seed=0, window=(-1, -1),
                  softcap=0.0, alibi=False, counts=None, q_scale=1.0, poison=True, max_k=None, cols_more=1, **kw):
    st = STORES[store]
    table, pages = _table(lens, page, seed, cols_more=cols_more)
    kc, ks = _kv8.filled(pages, page, block, hk, dim, st, seed + 1)
    vc, vs = _kv8.filled(pages, page, block, hk, dim, st, seed + 2)
    if poison:
        _poison(kc, ks, vc, vs, lens, table, st)
    gen = torch.Generator().manual_seed(seed + 3)
    cu = None
    if counts is not None:
        cu = torch.tensor([0] + counts).cumsum(0).int()
        q = torch.randn(int(cu[-1]), heads, dim, generator=gen) * q_scale
    else:
        q = torch.randn(len(lens), sq, heads, dim, generator=gen) * q_scale
    q = q.to(dtype)
    slopes = torch.rand(len(lens), heads, generator=gen) * 0.1 if alibi else None
    want, bound = _kv8.attend(q, kc, ks, vc, vs, lens, table, cu, kw.get("softmax_scale"), causal, window, softcap, slopes)
    out = _fa().flash_attn_with_kvcache_8bit(
        q.to(DEV), kc.to(DEV), vc.to(DEV), ks.to(DEV), vs.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV),
        table.to(DEV), cu_seqlens_q=None if cu is None else cu.to(DEV), max_seqlen_q=None if cu is None else max(counts),
        max_seqlen_k=max_k, causal=causal, window_size=window, softcap=softcap,
        alibi_slopes=None if slopes is None else slopes.to(DEV), **kw).cpu().double()
    over = (out - want).abs() - bound
    assert bool(torch.isfinite(out).all())
    assert float(over.max()) <= 0, f"beyond the bound by {float(over.max()):.3e}, bound {float(bound.max()):.3e}"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("cols_more", [1, 80])
def test_decode(dtype, store, dim, cols_more):
    # (a table of more than 4096 keys: the sequences share workgroups)
    _check_attend([1, 15, 16, 17, 31, 32, 33, 64, 65, 300, 777, 0, 40], 1, 8, 2, dim, dtype, store, cols_more=cols_more)


@pytest.mark.parametrize("heads,hk", [(1, 1), (7, 1), (32, 1), (40, 1), (12, 12), (16, 8), (33, 3)])
@pytest.mark.parametrize("cols_more", [1, 80])
def test_decode_heads(heads, hk, cols_more):
    _check_attend([200, 3, 130], 1, heads, hk, 64, torch.bfloat16, "e4m3", cols_more=cols_more)


@pytest.mark.parametrize("page,block", [(16, 16), (48, 16), (64, 64), (256, 64), (1024, 512)])
@pytest.mark.parametrize("dim", [64, 128])
def test_decode_pages(page, block, dim):
    _check_attend([5, 500, 1203], 1, 4, 2, dim, torch.bfloat16, "e4m3", page=page, block=block)


@pytest.mark.parametrize("max_k", [None, 20000])
def test_decode_long(max_k):
    # splits of one long sequence beside short ones, merged; and beside an empty one
    _check_attend([20000, 1, 0, 4095, 4097], 1, 8, 2, 128, torch.bfloat16, "e4m3", page=256, block=64, max_k=max_k)


@pytest.mark.parametrize("batch,packed", [(70, False), (255, False), (256, False), (2050, False), (2100, True)])
def test_decode_of_many_sequences(batch, packed):
    # more sequences than workgroups, and than one launch adds up; some without keys or queries
    rng = random.Random(batch)
    lens = [rng.choice([0, 1, rng.randint(2, 90), 600 if i % 97 == 0 else 33]) for i in range(batch)]
    counts = [rng.choice([0, 1, 2]) for _ in range(batch)] if packed else None
    _check_attend(lens, 1, 4, 2, 64, torch.bfloat16, "e4m3", counts=counts, cols_more=80)


def test_decode_with_long_stretches():
    # a workgroup takes more keys than its lanes hold pages of at a time; the pages repeat
    st = torch.float8_e4m3fn
    L, hk, page = 70001, 32, 64
    kc, ks = _kv8.filled(5, page, 16, hk, 64, st, 1)
    vc, vs = _kv8.filled(5, page, 16, hk, 64, st, 2)
    table = torch.randint(0, 5, (1, -(-L // page)), generator=torch.Generator().manual_seed(3), dtype=torch.int32)
    q = torch.randn(1, 1, hk, 64, generator=torch.Generator().manual_seed(4)).bfloat16()
    want, bound = _kv8.attend(q, kc, ks, vc, vs, [L], table)
    out = _fa().flash_attn_with_kvcache_8bit(q.to(DEV), kc.to(DEV), vc.to(DEV), ks.to(DEV), vs.to(DEV),
                                             torch.tensor([L], device=DEV), table.to(DEV)).cpu().double()
    assert bool(((out - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("sq", [3, 40])
def test_query_rows_are_apart(dtype, sq):
    # NaN and infinities in one query leave the others bit for bit as they were
    st = torch.float8_e4m3fn
    kc, ks = (t.to(DEV) for t in _kv8.filled(2, 256, 32, 2, 64, st, 1))
    q = torch.randn(2, sq, 4, 64, device=DEV).to(dtype)
    clean = _fa().flash_attn_with_kvcache_8bit(q, kc, kc, ks, ks)
    bad = q.clone()
    bad[0, 1, 2, 3], bad[1, 0, 0, 60] = math.nan, math.inf
    out = _fa().flash_attn_with_kvcache_8bit(bad, kc, kc, ks, ks)
    hit = torch.zeros(2, sq, 4, dtype=torch.bool, device=DEV)
    hit[0, 1, 2] = hit[1, 0, 0] = True
    assert bool(torch.isnan(out[hit]).all()) and torch.equal(out[~hit], clean[~hit])


def test_queries_of_any_size():
    # bf16 queries are split into 8-bit numbers by their row's largest: rows of very small and large numbers, of one
    # large number among small ones, of zeros
    st = torch.float8_e4m3fn
    lens = [300, 300]
    table, pages = _table(lens, 64, 0)
    kc, ks = _kv8.filled(pages, 64, 32, 2, 128, st, 1)
    vc, vs = _kv8.filled(pages, 64, 32, 2, 128, st, 2)
    q = torch.randn(2, 20, 4, 128, generator=torch.Generator().manual_seed(3))
    q[0, 0] = 0
    q[0, 1] *= 1e-30
    q[0, 2, :, 5] = 3e4
    q[0, 3, :, ::7] *= 2.0 ** -20
    q[0, 4] *= 1e3
    q = q.bfloat16()
    for sq in (1, 6, 20):
        want, bound = _kv8.attend(q[:, :sq], kc, ks, vc, vs, lens, table)
        out = _fa().flash_attn_with_kvcache_8bit(q[:, :sq].to(DEV), kc.to(DEV), vc.to(DEV), ks.to(DEV), vs.to(DEV),
                                                 torch.tensor(lens, device=DEV), table.to(DEV)).cpu().double()
        assert bool(((out - want).abs() <= bound).all())
    # a row with a number that is not finite is NaN, and it alone
    q[0, 5, 1, 7] = math.inf
    q[1, 2, 3, 100] = math.nan
    out = _fa().flash_attn_with_kvcache_8bit(q.to(DEV), kc.to(DEV), vc.to(DEV), ks.to(DEV), vs.to(DEV),
                                             torch.tensor(lens, device=DEV), table.to(DEV)).cpu()
    nan = torch.isnan(out).all(dim=-1)
    assert bool(nan[0, 5, 1]) and bool(nan[1, 2, 3]) and int(torch.isnan(out).any(dim=-1).sum()) == 2


@pytest.mark.parametrize("sq", [2, 3, 8, 33, 130])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim", [64, 128])
def test_chunks(sq, causal, dim):
    _check_attend([sq, sq + 1, 300, 517], sq, 4, 2, dim, torch.bfloat16, "e4m3", causal=causal)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_chunk_longer_than_the_cache(dim):
    # causal queries before the first key see none: zeros
    _check_attend([40, 3, 0, 70], 70, 4, 1, dim, torch.float16, "e5m2")


@pytest.mark.parametrize("window", [(0, -1), (5, -1), (100, -1), (40, 3), (-1, 2)])
@pytest.mark.parametrize("sq,causal", [(1, True), (6, True), (70, True), (70, False)])
def test_windows(window, sq, causal):
    for more in (1, 80):
        _check_attend([sq, 100, 611], sq, 4, 2, 64, torch.bfloat16, "e4m3", window=window, causal=causal, cols_more=more)


@pytest.mark.parametrize("kind", ["alibi", "softcap", "both", "window", "scale", "zero", "negative"])
@pytest.mark.parametrize("sq", [1, 40])
@pytest.mark.parametrize("dim", [64, 128])
def test_score_options(kind, sq, dim):
    more = {"alibi": dict(alibi=True), "softcap": dict(softcap=5.0), "both": dict(alibi=True, softcap=20.0),
            "window": dict(alibi=True, window=(50, 0)), "scale": dict(softmax_scale=0.3), "zero": dict(softmax_scale=0.0),
            "negative": dict(softmax_scale=-0.1)}[kind]
    _check_attend([sq, 129, 450], sq, 6, 3, dim, torch.float16, "e4m3", **more)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
def test_packed_queries(dtype, dim):
    _check_attend([300, 12, 700, 1, 64, 200], 0, 8, 2, dim, dtype, "e4m3", counts=[1, 12, 130, 1, 0, 33])
    _check_attend([3000, 12], 0, 8, 2, dim, dtype, "e4m3", counts=[1, 1])


@pytest.mark.parametrize("dim", [64, 128])
def test_large_scores(dim):
    # one key takes the whole weight, in every tile another running maximum
    _check_attend([900], 5, 4, 4, dim, torch.float16, "e4m3", q_scale=8.0)


def test_numbers_of_any_size():
    # a block's scale far from the next one's
    st = torch.float8_e4m3fn
    lens = [150]
    table, pages = _table(lens, 64, 0)
    kc, ks = _kv8.filled(pages, 64, 16, 2, 64, st, 1)
    vc, vs = _kv8.filled(pages, 64, 16, 2, 64, st, 2, spread=60)
    q = torch.randn(1, 1, 4, 64, generator=torch.Generator().manual_seed(3)).bfloat16()
    want, bound = _kv8.attend(q, kc, ks, vc, vs, lens, table)
    out = _fa().flash_attn_with_kvcache_8bit(q.to(DEV), kc.to(DEV), vc.to(DEV), ks.to(DEV), vs.to(DEV),
                                             torch.tensor(lens, device=DEV), table.to(DEV)).cpu().double()
    assert bool(((out - want).abs() <= bound).all())


def test_without_table_and_lengths():
    st = torch.float8_e4m3fn
    kc, ks = _kv8.filled(3, 96, 32, 2, 128, st, 1)
    vc, vs = _kv8.filled(3, 96, 32, 2, 128, st, 2)
    q = torch.randn(2, 4, 4, 128, generator=torch.Generator().manual_seed(3)).bfloat16()
    for lens in ([96, 96], [50, 0]):
        want, bound = _kv8.attend(q, kc, ks, vc, vs, lens, None, causal=True)
        args = [q.to(DEV), kc.to(DEV), vc.to(DEV), ks.to(DEV), vs.to(DEV)]
        out = _fa().flash_attn_with_kvcache_8bit(
            *args, cache_seqlens=None if lens[1] else torch.tensor(lens, device=DEV), causal=True).cpu().double()
        assert bool(((out - want).abs() <= bound).all())


def test_head_major_cache_and_strided_queries():
    st = torch.float8_e4m3fn
    lens = [100, 33]
    table, pages = _table(lens, 32, 0)
    kc, ks = _kv8.filled(pages, 32, 16, 2, 64, st, 1)
    vc, vs = _kv8.filled(pages, 32, 16, 2, 64, st, 2)
    qkv = torch.randn(2, 3, 3, 6, 64, generator=torch.Generator().manual_seed(3)).half()
    want, bound = _kv8.attend(qkv[:, :, 1], kc, ks, vc, vs, lens, table, causal=True)
    kd, vd = (c.transpose(1, 2).contiguous().to(DEV).transpose(1, 2) for c in (kc, vc))
    ksd, vsd = (s.view(torch.uint8).transpose(1, 2).contiguous().to(DEV).transpose(1, 2).view(torch.float8_e8m0fnu)
                for s in (ks, vs))
    wide = torch.zeros(2, table.shape[1] + 3, dtype=torch.int64, device=DEV)
    wide[:, :-3] = table.to(DEV)
    out = _fa().flash_attn_with_kvcache_8bit(qkv.to(DEV)[:, :, 1], kd, vd, ksd, vsd, torch.tensor(lens, device=DEV),
                                             wide, causal=True).cpu().double()
    assert bool(((out - want).abs() <= bound).all())


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("sq,window", [(6, (-1, -1)), (1, (20, -1)), (70, (-1, -1)), (70, (33, -1))])
def test_nan_reaches_only_rows_that_see_it(store, sq, window):
    st = STORES[store]
    lens = [203, 118]
    page = 64
    table, pages = _table(lens, page, 0)
    for dim in (64, 128):
        kc, ks = _kv8.filled(pages, page, 32, 2, dim, st, 1)
        vc, vs = _kv8.filled(pages, page, 32, 2, dim, st, 2)
        clean = vc.clone()
        spots = [(0, lens[0] - 1, 0, 5), (0, lens[0] - 3, 1, 7), (0, 160, 0, 40), (1, 117, 1, 63), (1, 50, 0, 2)]
        for b, j, h, d in spots:
            vc.view(torch.uint8)[table[b, j // page], j % page, h, d] = 0x7f if store == "e4m3" else 0x7e
        kc.view(torch.uint8)[table[0, (lens[0] - 2) // page], (lens[0] - 2) % page, 1, 3] = 0xff
        q = torch.randn(2, sq, 4, dim, generator=torch.Generator().manual_seed(3)).bfloat16()
        kclean = kc.clone()
        kclean.view(torch.uint8)[table[0, (lens[0] - 2) // page], (lens[0] - 2) % page, 1, 3] = 0
        want, bound = _kv8.attend(q, kclean, ks, clean, vs, lens, table, causal=True, window=window)
        out = _fa().flash_attn_with_kvcache_8bit(q.to(DEV), kc.to(DEV), vc.to(DEV), ks.to(DEV), vs.to(DEV),
                                                 torch.tensor(lens, device=DEV), table.to(DEV), causal=True,
                                                 window_size=window).cpu().double()
        bad = torch.zeros(out.shape, dtype=torch.bool)

        def sees(b, i, j):
            pos = i + lens[b] - sq
            return j <= pos and (window[0] < 0 or pos - j <= window[0])
        for i in range(sq):
            for b, j, h, d in spots:
                if sees(b, i, j):
                    bad[b, i, 2 * h:2 * h + 2, d] = True
            if sees(0, i, lens[0] - 2):
                bad[0, i, 2:4] = True
        assert torch.equal(torch.isnan(out), bad)
        assert bool(((out - want).abs() <= bound)[~bad].all())


def test_cache_beyond_32_bit_offsets():
    # 5 GiB of one tensor for K and V; the sequence lies in its last pages, the append too
    st = torch.float8_e4m3fn
    pages, page, hk, dim = 20480, 256, 8, 128
    big = torch.zeros(pages, page, hk, dim, dtype=torch.uint8, device=DEV).view(st)
    scale = torch.full((pages, 4, hk), 120, dtype=torch.uint8, device=DEV).view(torch.float8_e8m0fnu)
    kc, ks = _kv8.filled(3, page, 64, hk, dim, st, 1)
    big.view(torch.uint8)[-3:] = kc.view(torch.uint8).to(DEV)
    scale.view(torch.uint8)[-3:] = ks.view(torch.uint8).to(DEV)
    table = torch.tensor([[2, 0, 1]])
    q = torch.randn(1, 2, 16, dim, generator=torch.Generator().manual_seed(3)).bfloat16()
    for sq in (2, 40):
        q = torch.randn(1, sq, 16, dim, generator=torch.Generator().manual_seed(3)).bfloat16()
        want, bound = _kv8.attend(q, kc, ks, kc, ks, [700], table, causal=True)
        out = _fa().flash_attn_with_kvcache_8bit(q.to(DEV), big, big, scale, scale, torch.tensor([700], device=DEV),
                                                 (table + pages - 3).to(DEV), causal=True).cpu().double()
        assert bool(((out - want).abs() <= bound).all())
    other, oscale = big[-3:].clone(), scale.view(torch.uint8)[-3:].clone().view(torch.float8_e8m0fnu)
    k = _rows(300, hk, dim, torch.bfloat16, 4)
    first = page + 188
    slots = torch.arange(300) + first
    wc, ws = _kv8.append(k, kc, ks, slots)
    vbig, vscale = torch.zeros_like(big.view(torch.uint8)).view(st), scale.clone()
    _fa().kvcache_append_8bit(k.to(DEV), k.to(DEV), big, vbig, scale, vscale, slots.to(DEV) + (pages - 3) * page)
    assert _kv8.same_bytes(big[-3:].cpu(), wc) and torch.equal(scale[-3:].view(torch.uint8).cpu(), ws.view(torch.uint8))
    assert not bool(big.view(torch.uint8)[:16].any())


def test_no_visible_keys_at_all():
    st = torch.float8_e4m3fn
    kc, ks = (t.to(DEV) for t in _kv8.filled(3, 32, 16, 2, 64, st, 1))
    for sq in (1, 30):
        q = torch.randn(3, sq, 4, 64, device=DEV).half()
        zero = torch.zeros(3, dtype=torch.int32, device=DEV)
        for out in (_fa().flash_attn_with_kvcache_8bit(q, kc, kc, ks, ks, zero, max_seqlen_k=0),
                    _fa().flash_attn_with_kvcache_8bit(q, kc, kc, ks, ks, zero),
                    _fa().flash_attn_with_kvcache_8bit(q, kc[:0], kc[:0], ks[:0], ks[:0], None,
                                                       torch.zeros(3, 200, dtype=torch.int32, device=DEV), validate=False)):
            assert bool((out == 0).all())


def test_capture_without_a_warm_up():
    # the first call of its kind in the process is a captured one
    st = torch.float8_e5m2
    kc, ks = _kv8.filled(4, 48, 16, 3, 256, st, 1)
    q = torch.randn(1, 1, 6, 256, generator=torch.Generator().manual_seed(3)).half()
    want, bound = _kv8.attend(q, kc, ks, kc, ks, [150], torch.tensor([[3, 1, 0, 2]]), softcap=3.0)
    dev = [t.to(DEV) for t in (q, kc, ks)]
    lens, table = torch.tensor([150], dtype=torch.int32, device=DEV), torch.tensor([[3, 1, 0, 2]], dtype=torch.int32, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _fa().flash_attn_with_kvcache_8bit(dev[0], dev[1], dev[1], dev[2], dev[2], lens, table, softcap=3.0,
                                                 validate=False)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.empty(1 << 18, device=DEV).normal_()
        assert bool(((out.cpu().double() - want).abs() <= bound).all())


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("causal,window,softcap", [(True, (-1, -1), 0.0), (False, (-1, -1), 0.0), (True, (9001, -1), 0.0),
                                                   (True, (-1, -1), 9.0)])
def test_chunk_over_more_keys_than_lds_holds_pages_of(dim, causal, window, softcap):
    # 64 row blocks of 4 heads fill the GPU, so no block's keys are split, and one sequence has many
    _check_attend([20011, 16384, 8193] + [33 + i for i in range(61)], 33, 4, 4, dim, torch.bfloat16, "e4m3", causal=causal,
                  window=window, softcap=softcap)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("store", STORES)
def test_chunks_of_256_dims(dtype, store):
    _check_attend([70, 1, 300, 1517], 70, 6, 2, 256, dtype, store, page=48, block=16)
    _check_attend([70, 1, 300, 1517], 70, 6, 2, 256, dtype, store, page=48, block=16, causal=False, window=(40, 30))


@pytest.mark.parametrize("heads,hk", [(3, 1), (8, 2), (32, 8), (64, 16)])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lens", [[9001], [0, 5, 130, 7003], [700 * i + 1 for i in range(9)]])
def test_merging_few_and_many_pieces(heads, hk, dim, lens):
    # 512 pieces of a row to 2; rows of none and of one beside them
    for sq in (1, 2):
        _check_attend(lens, sq, heads, hk, dim, torch.bfloat16, "e4m3", seed=len(lens), cols_more=80, poison=False)


@pytest.mark.parametrize("heads,hk,sq", [(4, 1, 33), (4, 1, 300), (12, 3, 50)])
@pytest.mark.parametrize("lens", [[9001], [40, 5003, 0]])
def test_merging_the_splits_of_chunks(heads, hk, sq, lens):
    for dim in (64, 128, 256):
        _check_attend(lens, sq, heads, hk, dim, torch.float16, "e5m2", window=(3000, -1))


def test_nan_in_one_of_many_pieces():
    st = torch.float8_e4m3fn
    kc, ks = _kv8.filled(128, 64, 16, 1, 128, st, 1)
    vc, vs = kc.clone(), ks.clone()
    kc.view(torch.uint8)[77, 5] = 0x7f
    q = torch.randn(1, 1, 4, 128, generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV)
    table = torch.arange(128, dtype=torch.int32, device=DEV)[None]
    for n, bad in ((8192, True), (77 * 64 + 6, True), (77 * 64 + 5, False), (4000, False)):
        out = _fa().flash_attn_with_kvcache_8bit(q, kc.to(DEV), vc.to(DEV), ks.to(DEV), vs.to(DEV),
                                                 torch.tensor([n], device=DEV), table)
        assert bool(torch.isnan(out).all()) == bad and bool(torch.isnan(out).any()) == bad


def test_packed_chunks_of_many_sequences():
    # row blocks are counted in groups of 64 sequences; some have no queries, or no keys
    rng = random.Random(1)
    lens = [rng.choice([0, 1, 64, rng.randint(2, 400)]) for _ in range(200)]
    counts = [rng.choice([0, 0, 1, 7, rng.randint(2, 140)]) for _ in range(200)]
    _check_attend(lens, 1, 4, 2, 64, torch.bfloat16, "e4m3", counts=counts)


def test_attend_refusals():
    st = torch.float8_e4m3fn
    kc, ks = (t.to(DEV) for t in _kv8.filled(3, 32, 16, 2, 64, st, 1))
    q = torch.zeros(2, 1, 4, 64, device=DEV).half()
    lens = torch.tensor([5, 6], device=DEV)
    table = torch.tensor([[0, 1], [2, 0]], dtype=torch.int32, device=DEV)
    packed = torch.zeros(5, 4, 64, device=DEV).half()

    def call(q=q, lens=lens, table=table, **kw):
        return _fa().flash_attn_with_kvcache_8bit(q, kc, kc, ks, ks, lens, table, **kw)
    call()
    with pytest.raises(ValueError, match="invalid physical page"):
        call(table=table + 1)
    with pytest.raises(ValueError, match="invalid physical page"):
        call(table=table - 1)
    with pytest.raises(ValueError, match="valid lengths"):
        call(lens=lens + 60)
    with pytest.raises(ValueError, match="valid lengths"):
        call(lens=lens, max_seqlen_k=5)
    with pytest.raises(ValueError, match="valid lengths"):
        call(lens=lens - 6)
    cu = torch.tensor([0, 2, 5], dtype=torch.int32, device=DEV)
    call(q=packed, cu_seqlens_q=cu, max_seqlen_q=3)
    with pytest.raises(ValueError, match="start at zero"):
        call(q=packed, cu_seqlens_q=cu + 1, max_seqlen_q=3)
    with pytest.raises(ValueError, match="non-decreasing"):
        call(q=packed, cu_seqlens_q=torch.tensor([0, 4, 3], dtype=torch.int32, device=DEV), max_seqlen_q=4)
    with pytest.raises(ValueError, match="exceeds the packed queries"):
        call(q=packed[:4], cu_seqlens_q=cu, max_seqlen_q=3)
    with pytest.raises(ValueError, match="cover every packed sequence"):
        call(q=packed, cu_seqlens_q=cu, max_seqlen_q=2)
    with pytest.raises(ValueError, match="no backward"):
        call(q=q.clone().requires_grad_())


def test_device_arrays_out_of_range_stay_inside():
    """Unvalidated: clamped lengths, pages that read as zeros, sequences without queries."""
    st = torch.float8_e4m3fn
    kc, ks = _kv8.filled(3, 32, 16, 2, 64, st, 1)
    vc, vs = _kv8.filled(3, 32, 16, 2, 64, st, 2)
    q = torch.randn(3, 2, 4, 64, generator=torch.Generator().manual_seed(3)).half()
    dev = [t.to(DEV) for t in (kc, vc, ks, vs)]
    table = torch.tensor([[0, 1], [2, 0], [1, 2]], dtype=torch.int32)
    out = _fa().flash_attn_with_kvcache_8bit(q.to(DEV), *dev, torch.tensor([1000, -5, 40], device=DEV), table.to(DEV),
                                             causal=True, validate=False).cpu().double()
    want, bound = _kv8.attend(q, kc, ks, vc, vs, [64, 0, 40], table, causal=True)
    assert bool(((out - want).abs() <= bound).all())
    # a page outside the cache: its keys are zeros, with scores of 0
    bad = torch.tensor([[0, 99], [-1, 1], [1, 2]], dtype=torch.int32)
    kz, vz = torch.cat([kc, torch.zeros(1, 32, 2, 64).to(st)]), torch.cat([vc, torch.zeros(1, 32, 2, 64).to(st)])
    sz = [torch.cat([s.view(torch.uint8), torch.full((1, 2, 2), 127, dtype=torch.uint8)]).view(torch.float8_e8m0fnu)
          for s in (ks, vs)]
    out = _fa().flash_attn_with_kvcache_8bit(q.to(DEV), *dev, torch.tensor([64, 50, 40], device=DEV), bad.to(DEV),
                                             causal=True, validate=False).cpu().double()
    zero = torch.tensor([[0, 3], [3, 1], [1, 2]], dtype=torch.int32)
    want, bound = _kv8.attend(q, kz, sz[0], vz, sz[1], [64, 50, 40], zero, causal=True)
    assert bool(((out - want).abs() <= bound).all())
    # offsets outside q
    packed = q.flatten(0, 1)
    cu = torch.tensor([0, 2, 9000, 6], dtype=torch.int32)
    out = _fa().flash_attn_with_kvcache_8bit(packed.to(DEV), *dev, torch.tensor([64, 50, 40], device=DEV), table.to(DEV),
                                             cu_seqlens_q=cu.to(DEV), max_seqlen_q=4, causal=True, validate=False).cpu().double()
    want, bound = _kv8.attend(packed, kc, ks, vc, vs, [64], table, torch.tensor([0, 2]), causal=True)
    assert bool(((out - want).abs() <= bound).all()) and bool((out[2:] == 0).all())


def test_packed_rows_behind_the_last_sequence_are_zero():
    st = torch.float8_e4m3fn
    kc, ks = (t.to(DEV) for t in _kv8.filled(3, 32, 16, 2, 64, st, 1))
    q = torch.randn(9, 4, 64, device=DEV).half()
    cu = torch.tensor([0, 2, 5], dtype=torch.int32, device=DEV)
    torch.full((9, 4, 64), math.nan, device=DEV, dtype=torch.float16)   # what the allocator may hand out next
    out = _fa().flash_attn_with_kvcache_8bit(q, kc, kc, ks, ks, torch.tensor([5, 6], device=DEV), None, cu_seqlens_q=cu,
                                             max_seqlen_q=4, causal=True)
    assert bool((out[5:] == 0).all()) and bool((out[:5] != 0).any(dim=-1).all())


# ----------------------------------------------------------------------------- a run of them together
class _Server:
    """Requests served step by step on the three operators, beside what each has cached in float64."""

    def __init__(self, batch, page, block, heads, hk, dim, store, pages, cols, seed):
        self.gen = torch.Generator().manual_seed(seed)
        self.batch, self.page, self.block, self.heads, self.hk, self.dim, self.store = batch, page, block, heads, hk, dim, store
        shape, sshape = (pages, page, hk, dim), (pages, page // block, hk)
        self.cache = [torch.full(shape, 0x7f, dtype=torch.uint8, device=DEV).view(store) for _ in range(2)]
        self.scale = [torch.full(sshape, 0xff, dtype=torch.uint8, device=DEV).view(torch.float8_e8m0fnu) for _ in range(2)]
        self.table = torch.full((batch, cols), -1, dtype=torch.int32, device=DEV)
        self.free = torch.randperm(pages, generator=self.gen).int().to(DEV)
        self.start = torch.zeros(1, dtype=torch.int32, device=DEV)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=DEV)
        self.mirror = [(torch.zeros(1, cols * page, hk, dim, dtype=torch.uint8).view(store),
                        torch.zeros(1, cols * page // block, hk, dtype=torch.uint8).view(torch.float8_e8m0fnu))
                       for _ in range(2 * batch)]

    def rows(self, n, heads):
        x = torch.randn(n, heads, self.dim, generator=self.gen)
        return (x * torch.exp(torch.randn(n, 1, 1, generator=self.gen))).bfloat16()

    def step(self, q, k, v, new, rows, max_q, **kw):
        fa = _fa()
        slots, _, cu, lens, self.start = fa.paged_kvcache_slots(self.table, self.lens, new, self.free, self.page, rows,
                                                                free_start=self.start, **kw)
        fa.kvcache_append_8bit(k, v, *self.cache, *self.scale, slots, **kw)
        self.lens = lens
        return fa.flash_attn_with_kvcache_8bit(q, *self.cache, *self.scale, lens, self.table.clamp(min=0), cu_seqlens_q=cu,
                                               max_seqlen_q=max_q, causal=True, **kw)

    def expect(self, q, k, v, before, new):
        """The plain forms on a cache per request."""
        out, bound, at = [], [], 0
        for b, n in enumerate(new):
            for i, x in enumerate((k, v)):
                c, s = self.mirror[2 * b + i]
                self.mirror[2 * b + i] = _kv8.append(x[at:at + n], c, s, torch.arange(before[b], before[b] + n))
            (kc, ks), (vc, vs) = self.mirror[2 * b:2 * b + 2]
            o, e = _kv8.attend(q[at:at + n][None], kc, ks, vc, vs, [before[b] + n], None, causal=True)
            out.append(o[0])
            bound.append(e[0])
            at += n
        return torch.cat(out), torch.cat(bound)


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("validate", [True, False])
def test_steps_of_a_serving_loop(store, validate):
    s = _Server(5, 32, 16, 4, 2, 64, STORES[store], pages=40, cols=8, seed=1)
    before = [0] * 5
    for new in ([17, 1, 40, 0, 64], [1, 1, 1, 33, 1], [1] * 5, [3, 30, 1, 1, 2], [1] * 5):
        n = sum(new)
        q, k, v = s.rows(n, 4), s.rows(n, 2), s.rows(n, 2)
        pad = 6   # rows of a padded batch, behind the requests'
        qd, kd, vd = (torch.cat([x, torch.full((pad,) + x.shape[1:], math.nan, dtype=x.dtype)]).to(DEV) for x in (q, k, v))
        out = s.step(qd, kd, vd, torch.tensor(new, dtype=torch.int32, device=DEV), n + pad, 64, validate=validate)
        want, bound = s.expect(q, k, v, before, new)
        before = [a + b for a, b in zip(before, new)]
        assert s.lens.tolist() == before
        assert bool(((out[:n].cpu().double() - want).abs() <= bound).all())
        assert bool((out[n:] == 0).all())


def test_a_captured_decode_step():
    """One graph of a decode step, replayed with the lengths it wrote itself, beside other GPU work."""
    s = _Server(3, 16, 16, 4, 2, 128, torch.float8_e4m3fn, pages=30, cols=6, seed=2)
    new = torch.ones(3, dtype=torch.int32, device=DEV)
    first = [20, 5, 31]
    q, k, v = s.rows(56, 4), s.rows(56, 2), s.rows(56, 2)
    s.step(q.to(DEV), k.to(DEV), v.to(DEV), torch.tensor(first, dtype=torch.int32, device=DEV), 56, 31)
    s.expect(q, k, v, [0] * 3, first)
    lens, start = s.lens.clone(), s.start.clone()
    qd, kd, vd = (torch.zeros(3, h, 128, dtype=torch.bfloat16, device=DEV) for h in (4, 2, 2))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        state = [t.clone() for t in (s.table, lens, start, *(c.view(torch.uint8) for c in s.cache + s.scale))]
        s.step(qd, kd, vd, new, 3, 1, validate=False)   # warm-up, undone below
        s.table.copy_(state[0])
        for c, w in zip(s.cache + s.scale, state[3:]):
            c.view(torch.uint8).copy_(w)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    s.lens, s.start = lens, start
    with torch.cuda.graph(graph):
        out = s.step(qd, kd, vd, new, 3, 1, validate=False)
        lens.copy_(s.lens)
        start.copy_(s.start)
    before = list(first)
    for _ in range(7):
        q, k, v = s.rows(3, 4), s.rows(3, 2), s.rows(3, 2)
        qd.copy_(q), kd.copy_(k), vd.copy_(v)
        graph.replay()
        want, bound = s.expect(q, k, v, before, [1, 1, 1])
        before = [n + 1 for n in before]
        torch.empty(1 << 20, device=DEV).normal_()
        assert lens.tolist() == before
        assert bool(((out.cpu().double() - want).abs() <= bound).all())


def test_validation_is_refused_while_capturing():
    kc, ks = (t.to(DEV) for t in _kv8.filled(3, 32, 16, 2, 64, torch.float8_e4m3fn, 1))
    q = torch.zeros(3, 1, 4, 64, device=DEV).half()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        graph.capture_begin()
        try:
            with pytest.raises(RuntimeError, match="validate=False"):
                _fa().flash_attn_with_kvcache_8bit(q, kc, kc, ks, ks)
            with pytest.raises(RuntimeError, match="validate=False"):
                _fa().kvcache_append_8bit(q[:, 0, :2], q[:, 0, :2], kc, kc, ks, ks, torch.zeros(3, dtype=torch.int64, device=DEV))
        finally:
            graph.capture_end()


def test_calls_on_two_streams():
    """Each call has a workspace of its own."""
    st = torch.float8_e4m3fn
    calls = []
    for seed in (0, 10):
        lens = [3000, 1500]
        table, pages = _table(lens, 64, seed)
        kc, ks = _kv8.filled(pages, 64, 32, 2, 128, st, seed + 1)
        vc, vs = _kv8.filled(pages, 64, 32, 2, 128, st, seed + 2)
        q = torch.randn(2, 1, 8, 128, generator=torch.Generator().manual_seed(seed)).bfloat16()
        calls.append(([t.to(DEV) for t in (q, kc, vc, ks, vs, torch.tensor(lens), table)],
                      _kv8.attend(q, kc, ks, vc, vs, lens, table)))
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        for s, (args, _) in zip(streams, calls):
            with torch.cuda.stream(s):
                outs.append(_fa().flash_attn_with_kvcache_8bit(*args, validate=False))
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        want, bound = calls[i % 2][1]
        assert bool(((out.cpu().double() - want).abs() <= bound).all())


def test_results_do_not_change_from_call_to_call():
    st = torch.float8_e4m3fn
    lens = [5000, 77]
    table, pages = _table(lens, 64, 0)
    kc, ks = (t.to(DEV) for t in _kv8.filled(pages, 64, 32, 2, 128, st, 1))
    q = torch.randn(2, 1, 8, 128, device=DEV).bfloat16()
    outs = [_fa().flash_attn_with_kvcache_8bit(q, kc, kc, ks, ks, torch.tensor(lens, device=DEV), table.to(DEV),
                                               max_seqlen_k=5000) for _ in range(4)]
    assert all(torch.equal(o, outs[0]) for o in outs)
