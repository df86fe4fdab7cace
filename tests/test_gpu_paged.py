"""Serving from a paged cache, on the GPU: each operator against its restatement
(oracle/paged_oracle.py).  Whole numbers are equal; attention is within the bounds
of oracle/lm_oracle.py, which count the roundings a correct kernel makes."""

import math
import random

import pytest
import torch

import kotodama_amd
from kotodama_amd import paged
from oracle import paged_oracle as PO

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
BF, FP = torch.bfloat16, torch.float32


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device=DEV)


def _randn(g, *shape, dtype=BF, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def _within(name, got, want):
    value, bound = want
    assert got.shape == value.shape, name
    got = got.double()
    same = (got == value) | (got.isnan() & value.isnan())
    over = torch.where(same, 0.0, (got - value).abs() / bound.clamp_min(1e-300))
    worst = over.max().item() if over.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.3g} times its bound"


# ----------------------------------------------------------------- slots --


def _slots(table, held, new, free, count, page, tokens, dtype=torch.int32, native=True):
    t, f = _ints(table).reshape(len(held), len(table[0]) if table else 4), _ints(free)
    call = kotodama_amd.paged_slots if native else paged.paged_slots_op
    res = call(t, _ints(held, dtype), _ints(new, dtype), f, _ints([count]), page, tokens)
    want = PO.slots(table, held, new, free, count, page, tokens)
    for name, x, w in zip(("slots", "positions", "q_starts", "kv_lens", "free_count"), res, want):
        assert x.dtype == torch.int32
        assert x.tolist() == (w if isinstance(w, list) else [w]), name
    assert t.tolist() == want[-1], "block_table"
    assert f.tolist() == free, "free_pages"


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("b,tokens,pad,short", [(1, 1, 0, 0), (3, 40, 3, 0), (65, 300, 0, 5), (1024, 5000, 11, 0),
                                                (1025, 1025, 0, 100), (2500, 20000, 7, 300)])
def test_slots(b, tokens, pad, short, page):
    rng = random.Random(b + tokens)
    m = 8
    new = [0] * b
    for _ in range(tokens - pad):
        new[rng.randrange(b)] += 1
    held = [rng.choice((0, 1, page - 1, page, page + 1, rng.randrange(4 * page))) for _ in range(b)]
    table = [[rng.randrange(10**6) for _ in range(m)] for _ in range(b)]
    need = sum(max(0, -(-(h + n) // page) - (-(-h // page))) for h, n in zip(held, new))
    free = [rng.randrange(10**6) for _ in range(need + 5)]
    print(f"paged_slots b={b} tokens={tokens} page={page}", flush=True)
    _slots(table, held, new, free, max(0, need - short), page, tokens)


def test_slots_at_the_edges():
    t = [[5, 6, 7], [8, 9, 10]]
    _slots(t, [0, 0], [0, 0], [1, 2, 3], 3, 16, 0)  # nothing new
    _slots(t, [0, 0], [0, 0], [1, 2, 3], 3, 16, 5)  # padding alone
    _slots(t, [16, 31], [1, 2], [1, 2, 3], 0, 16, 3)  # no free pages: the second needs one, the first too
    _slots(t, [15, 16], [1, 1], [1, 2, 3], 1, 16, 2)  # one for two, but the first needs none
    _slots(t, [40, 0], [9, 1], [1, 2, 3], 3, 16, 10)  # over its row of the table; the next is served
    _slots(t, [0, 0], [4, 9], [1, 2, 3], 3, 16, 10)  # over the call's tokens
    _slots(t, [-1, 3], [2, 2], [1, 2, 3], 3, 16, 4)  # lengths that make no sense
    _slots(t, [0, 3], [-5, 2], [1, 2, 3], 3, 16, 4)
    _slots(t, [2**31 - 1, 3], [2, 2], [1, 2, 3], 3, 16, 4)
    _slots(t, [0, 0], [1, 1], [1, 2, 3], 99, 16, 2)  # a count over the list
    _slots(t, [0, 0], [1, 1], [1, 2, 3], -4, 16, 2)
    _slots(t, [0, 0], [1, 1], [], 0, 16, 2)
    _slots([], [], [], [1, 2], 2, 16, 3)
    _slots(t, [2**40, 0], [1, 1], [1, 2, 3], 3, 16, 2, torch.int64)
    _slots(t, [0, 7], [2**40, 1], [1, 2, 3], 3, 16, 2, torch.int64)
    _slots(t, [0, 7], [20, 30], [1, 2, 3], 3, 16, 60, torch.int64)
    _slots(t, [0, 7], [20, 30], [1, 2, 3], 3, 16, 60, native=False)


def test_slots_of_page_numbers_that_no_slot_can_name():
    # pages whose slots 32 bits do not hold, or negative ones: no slot
    t = _ints([[0, 0]])
    res = kotodama_amd.paged_slots(t, _ints([0]), _ints([20]), _ints([-7, 2**27]), _ints([2]), 16, 20)
    assert res.slots.tolist() == [-1] * 20 and t.tolist() == [[2**27, -7]]
    res = kotodama_amd.paged_slots(t, _ints([0]), _ints([1]), _ints([2**27 - 1]), _ints([1]), 16, 1)
    assert res.slots.tolist() == [(2**27 - 1) * 16]


def test_slots_again_gives_the_same():
    t, f, c = _ints([[9, 0, 0], [3, 0, 0]]), _ints([11, 12, 13, 14]), _ints([4])
    a = kotodama_amd.paged_slots(t, _ints([10, 3]), _ints([30, 1]), f, c, 16, 31)
    one = t.clone()
    b = kotodama_amd.paged_slots(t, _ints([10, 3]), _ints([30, 1]), f, c, 16, 31)
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and torch.equal(t, one)
    wide = _ints([[9, 0, 0, 77], [3, 0, 0, 77]])  # rows apart
    view = wide[:, :3]
    a = kotodama_amd.paged_slots(view, _ints([10, 3, 5])[:2], _ints([30, 9, 1])[::2], f, c, 16, 31)
    assert torch.equal(view, one) and wide[:, 3].tolist() == [77, 77] and torch.equal(a.slots, b.slots)


@pytest.mark.parametrize("b,m", [(1, 1), (3, 5), (300, 40), (1500, 64)])
def test_release(b, m):
    rng = random.Random(b)
    page = 16
    held = [rng.randrange(m * page + 1) for _ in range(b)]
    kept = [rng.choice((0, h, rng.randint(0, h))) for h in held]
    if b > 2:
        held[0], kept[0] = -3, 1
        held[1], kept[1] = 5, 50
        kept[2] = -7
    table = [[rng.randrange(10**6) for _ in range(m)] for _ in range(b)]
    total = sum(max(0, -(-h // page) - (-(-max(0, min(k, h)) // page))) for h, k in zip(held, kept) if h >= 0)
    for room in (total + 3, max(0, total - 2)):
        free = [rng.randrange(10**6) for _ in range(4 + room)]
        want = PO.release(table, held, kept, free, 4, page)
        t, f = _ints(table), _ints(free)
        for dtype in (torch.int32, torch.int64):
            got = kotodama_amd.paged_release(t, _ints(held, dtype), _ints(kept, dtype), f, _ints([4]), page)
            assert got.tolist() == [want[0]] and f.tolist() == want[1]
        assert t.tolist() == table


def test_pages_given_back_are_taken_again():
    t, f = _ints([[0] * 4, [0] * 4]), _ints([7, 6, 5, 4, 3, 2, 1, 0])
    a = kotodama_amd.paged_slots(t, _ints([0, 0]), _ints([40, 20]), f, _ints([8]), 16, 60)
    before = t.clone()
    count = kotodama_amd.paged_release(t, a.kv_lens, _ints([17, 20]), f, a.free_count, 16)
    assert a.free_count.tolist() == [3] and count.tolist() == [4]
    b = kotodama_amd.paged_slots(t, _ints([17, 20]), _ints([23, 0]), f, count, 16, 23)
    assert torch.equal(t, before) and b.free_count.tolist() == [3] and torch.equal(b.slots, a.slots[17:40])


# ----------------------------------------------------------------- write --


def _caches(g, pages, hk, page, d, dtype, layout="pages"):
    if layout == "pages":
        return _randn(g, pages, hk, page, d, dtype=dtype), _randn(g, pages, hk, page, d, dtype=dtype)
    if layout == "tokens":  # (pages, page_size, Hk, D) memory, keys and values side by side
        both = _randn(g, pages, page, 2, hk, d, dtype=dtype)
        return both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    both = _randn(g, hk, pages, page, d + 8, dtype=dtype)  # heads outside, rows apart
    other = _randn(g, pages, hk, page, d, dtype=dtype)
    return both.transpose(0, 1)[..., :d], other


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
@pytest.mark.parametrize("layout", ["pages", "tokens", "apart"])
@pytest.mark.parametrize("n,hk,page,d", [(0, 1, 16, 8), (1, 1, 16, 8), (7, 3, 32, 72), (301, 8, 64, 128),
                                         (3000, 2, 16, 64)])
def test_write(n, hk, page, d, layout, dtype):
    g = _gen(n + d)
    pages = n // page + 3
    kc, vc = _caches(g, pages, hk, page, d, dtype, layout)
    k = _randn(g, n, hk, d, dtype=dtype)
    v = _randn(g, hk, n, d, dtype=dtype).transpose(0, 1)
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:n].int()
    if n > 3:
        slots[1], slots[2], slots[3] = -1, pages * page, -(2**31)
    want = []
    for c, x in ((kc, k), (vc, v)):
        w = c.clone()
        for i, s in enumerate(slots.tolist()):
            if 0 <= s < pages * page:
                w[s // page, :, s % page] = x[i]
        want.append(w)
    print(f"paged_write n={n} hk={hk} page={page} d={d} {layout} {dtype}", flush=True)
    version = kc._version
    assert kotodama_amd.paged_write(k, v, kc, vc, slots) is None
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1]) and kc._version > version
    kc.zero_(), vc.zero_()
    kotodama_amd.paged_write(k, v, kc, vc, slots.long())
    paged.paged_write_op(k, v, kc, vc, slots)
    live = [s for s in slots.tolist() if 0 <= s < pages * page]
    for s in live[:50]:
        assert torch.equal(kc[s // page, :, s % page], want[0][s // page, :, s % page])


def test_write_of_unaligned_rows():
    g = _gen(5)
    kc, vc = _caches(g, 4, 2, 16, 64, BF)
    k = _randn(g, 9, 2, 67)[..., 3:]  # rows that no 16-byte piece fits: copied
    v = _randn(g, 9 * 128 + 1)[1:].view(9, 2, 64)
    slots = torch.arange(20, 29, device=DEV)
    kotodama_amd.paged_write(k, v, kc, vc, slots)
    assert torch.equal(kc[1, :, 4:13], k.transpose(0, 1)) and torch.equal(vc[1, :, 4:13], v.transpose(0, 1))


def test_write_refuses_caches_whose_rows_lie_on_one_another():
    x = torch.zeros(5, 2, 64, dtype=BF, device=DEV)
    cache = torch.zeros(3, 2, 16, 64, dtype=BF, device=DEV)
    for over in (cache[:1].expand(3, -1, -1, -1), cache[:, :1].expand(-1, 2, -1, -1),
                 cache[:, :, :1].expand(-1, -1, 16, -1)):
        for kc, vc in ((over, cache), (cache, over)):
            with pytest.raises(ValueError, match="on one another"):
                kotodama_amd.paged_write(x, x, kc, vc, torch.arange(5, device=DEV))
    one = cache[:1].as_strided((1, 2, 16, 64), (0, 1024, 64, 1))  # one page: no other lies on it
    kotodama_amd.paged_write(x + 1, x + 2, one, cache[1:2], torch.arange(5, device=DEV))
    assert (cache[0, :, :5] == 1).all() and (cache[1, :, :5] == 2).all()


# ------------------------------------------------------------- attention --


def _batch(seed, new, lens, h, hk, page, d, dtype, pad=0, layout="pages", index=torch.int32, extra=3, slack=2):
    """Packed queries, caches whose unused rows hold NaN and infinity, and their table."""
    g = _gen(seed)
    m = max([-(-n // page) for n in lens] + [1]) + slack
    pages = sum(-(-n // page) for n in lens) + extra
    kc, vc = _caches(g, pages, hk, page, d, dtype, layout)
    order = torch.randperm(pages, generator=g, device=DEV).tolist()
    # entries behind the length are not read
    table = torch.full((len(lens), m), -(2**31), dtype=torch.int32, device=DEV)
    used = torch.zeros(pages, page, dtype=torch.bool, device=DEV)
    for b, n in enumerate(lens):
        mine = [order.pop() for _ in range(-(-n // page))]
        table[b, :len(mine)] = _ints(mine)
        for i, p in enumerate(mine):
            used[p, :max(0, min(page, n - i * page))] = True
    kc.masked_fill_(~used[:, None, :, None], math.nan)
    vc.masked_fill_(~used[:, None, :, None], math.inf)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = _randn(g, starts[-1] + pad, h, d, dtype=dtype, scale=1.5)
    return q, kc, vc, table, _ints(lens, index), starts


def _attention(seed, new, lens, h, hk, page, d, dtype, pad=0, layout="pages", index=torch.int32, single=False,
               scale=None):
    print(f"paged_attention new={new if len(new) < 20 else len(new)} lens={lens if len(lens) < 20 else max(lens)} "
          f"h={h}/{hk} page={page} d={d} {dtype} pad={pad} {layout}", flush=True)
    q, kc, vc, table, kv_lens, starts = _batch(seed, new, lens, h, hk, page, d, dtype, pad, layout, index)
    q_starts = None if single else _ints(starts, index)
    out, lse = kotodama_amd.paged_attention(q, kc, vc, table, kv_lens, q_starts, scale=scale, want_lse=True)
    # a sequence whose new tokens are more than its keys: the first see none
    want, want_lse = PO.attention(q, kc, vc, table, lens, starts, scale)
    _within("out", out, want)
    _within("lse", lse, want_lse)
    again = kotodama_amd.paged_attention(q, kc, vc, table, kv_lens, q_starts, scale=scale)
    assert torch.equal(again, out)
    return out


DTYPES = pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])


@DTYPES
@pytest.mark.parametrize("new,lens,h,hk,page,d,pad", [
    ([1], [1], 1, 1, 16, 8, 0),
    ([1, 1, 1], [33, 1, 0], 4, 2, 16, 128, 0),
    ([3, 0, 1, 5], [3, 20, 130, 64], 2, 1, 32, 64, 4),
    ([17, 1, 64], [17, 129, 200], 6, 2, 16, 80, 1),
    ([129], [129], 3, 3, 64, 72, 0),
    ([40, 7, 1], [300, 7, 128], 8, 2, 128, 96, 130),
    ([2, 5], [1, 3], 4, 4, 16, 32, 0),  # fewer keys than new tokens
    ([4, 4], [0, 4], 5, 1, 16, 40, 3),  # a refused sequence
    ([33], [4096], 1, 1, 4096, 64, 0),  # one page
    ([8, 8, 8], [1000, 77, 513], 24, 8, 32, 128, 8),
    ([1] * 70, [1 + 13 * i for i in range(70)], 2, 2, 16, 64, 0),
    ([1, 2] * 150, [2 + i % 40 for i in range(300)], 2, 1, 16, 16, 5),  # more sequences than a workgroup's threads
])
def test_attention(dtype, new, lens, h, hk, page, d, pad):
    _attention(len(new) + d, new, lens, h, hk, page, d, dtype, pad)


@DTYPES
@pytest.mark.parametrize("lens,h,hk,d", [([5000], 8, 1, 128), ([70000], 1, 1, 64), ([3000, 1, 0, 129, 2500], 4, 2, 80),
                                         ([1] * 300 + [9000] + [7] * 40, 2, 2, 64)])
def test_single_tokens_over_a_split_cache(dtype, lens, h, hk, d):
    _attention(d, [1] * len(lens), lens, h, hk, 16, d, dtype, single=True)


@DTYPES
@pytest.mark.parametrize("new,lens,h,hk,page,d,pad", [
    ([2050, 1, 1, 9], [2050, 700, 1, 3000], 32, 8, 64, 128, 3),  # chunks of 128 rows a tile beside single tokens
    ([700, 0, 1400, 8], [900, 0, 1400, 8], 16, 16, 16, 64, 200),
    ([3000], [9000], 8, 8, 32, 72, 0),  # few tiles, long: split
    ([1300, 700, 30], [1300, 700, 30], 32, 8, 64, 64, 0),  # all tiles at once, none split
    ([1040], [16000], 32, 8, 64, 64, 0),  # halves
])
def test_many_rows(dtype, new, lens, h, hk, page, d, pad):
    _attention(sum(new), new, lens, h, hk, page, d, dtype, pad)


@DTYPES
def test_many_rows_of_many_sequences(dtype):
    # more sequences than a workgroup's threads, the long ones in the second stretch of them, and split
    new = [1] * 280 + [2100] + [3] * 40
    lens = [1 + 7 * i for i in range(280)] + [6000] + [3 + 100 * i for i in range(40)]
    _attention(17, new, lens, 32, 8, 64, 64, dtype, 5)


def test_starts_that_fall():
    # rows named many times over: whatever they then hold, nothing leads out of the call
    for n, h, hk in ((4, 4, 2), (2100, 32, 8)):
        lens = [700 + i for i in range(40)] + [700] * 260
        q, kc, vc, table, kv_lens, _ = _batch(19, [0] * 300, lens, h, hk, 64, 64, BF, pad=n + 9)
        print(f"paged_attention, falling starts: {n} tokens", flush=True)
        starts = [0] + [n, 0] * 150
        out = kotodama_amd.paged_attention(q, kc, vc, table, kv_lens, _ints(starts))
        assert out[0].isfinite().all()
        want = kotodama_amd.paged_attention(q, kc, vc, table, kv_lens, _ints([0] * 301))
        assert not want.any()  # the next call finds nothing of it


@DTYPES
@pytest.mark.parametrize("layout", ["tokens", "apart"])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_layouts(dtype, layout, index):
    _attention(3, [5, 1, 40], [64, 300, 40], 4, 2, 16, 64, dtype, 2, layout, index, scale=0.07)


def test_strided_queries_and_tables():
    q, kc, vc, table, lens, starts = _batch(9, [5, 1, 40], [64, 300, 40], 4, 2, 16, 64, BF)
    want = kotodama_amd.paged_attention(q, kc, vc, table, lens, _ints(starts))
    views = [q.transpose(0, 1).contiguous().transpose(0, 1), torch.cat((q, q), 2)[..., :64],
             torch.nn.functional.pad(q, (3, 0))[..., 3:]]  # heads outside; rows apart; no 16-byte pieces
    wide = torch.cat((table, table), 1)
    for v in views:
        for t, n, s in ((table, lens, _ints(starts)), (wide[:, :table.shape[1]], lens.repeat_interleave(2)[::2],
                                                       _ints([x for s in starts for x in (s, -1)])[::2])):
            assert torch.equal(kotodama_amd.paged_attention(v, kc, vc, t, n, s), want)
    out, _ = paged.paged_attention_op(q, kc, vc, table, lens, _ints(starts), 1 / 8)
    assert torch.equal(out, want)


@DTYPES
@pytest.mark.parametrize("new,lens,h,bad", [([5, 3, 1], [64, 300, 40], 4, 1), ([1, 1], [9000, 70], 2, 0),
                                            ([1500, 1500, 1], [1600, 1500, 40], 16, 0)])
def test_pages_outside_the_cache(dtype, new, lens, h, bad):
    hk, page, d = 2, 16, 64
    q, kc, vc, table, kv_lens, starts = _batch(11, new, lens, h, hk, page, d, dtype, pad=2)
    want = kotodama_amd.paged_attention(q, kc, vc, table, kv_lens, _ints(starts))
    for value in (-1, kc.shape[0], 2**31 - 1):
        t = table.clone()
        t[bad, 0] = value  # every row of the sequence sees it
        print(f"page {value} of sequence {bad}: new={new} lens={lens} {dtype}", flush=True)
        out, lse = kotodama_amd.paged_attention(q, kc, vc, t, kv_lens, _ints(starts), want_lse=True)
        mine = slice(starts[bad], starts[bad + 1])
        assert out[mine].isnan().all() and lse[mine].isnan().all()
        out[mine] = want[mine]
        assert torch.equal(out, want)  # no other sequence


def test_lengths_are_taken_into_what_there_is():
    q, kc, vc, table, kv_lens, starts = _batch(13, [2, 3], [32, 48], 2, 2, 16, 64, BF, slack=0)
    kc, vc = kc.nan_to_num(), vc.nan_to_num(posinf=1.0)
    table = table.clamp(min=0)
    full = kotodama_amd.paged_attention(q, kc, vc, table, _ints([48, 48]), _ints(starts))
    for lens in ([48, 1000], [2**31 - 1, 48]):
        assert torch.equal(kotodama_amd.paged_attention(q, kc, vc, table, _ints(lens), _ints(starts)), full)
    none = kotodama_amd.paged_attention(q, kc, vc, table, _ints([-5, 0]), _ints(starts))
    assert not none.any()
    # starts that lead out of the tokens
    a = kotodama_amd.paged_attention(q, kc, vc, table, _ints([48, 48]), _ints([0, 2, 900]))
    assert torch.equal(a, full)
    a = kotodama_amd.paged_attention(q, kc, vc, table, _ints([48, 48]), _ints([-3, 2, 5]))
    assert torch.equal(a, full)
    # falling starts name row 1 twice, the first sequence's and behind the last: row 0 is the first's alone
    a = kotodama_amd.paged_attention(q, kc, vc, table, _ints([48, 48]), _ints([0, 2, 1]))
    assert torch.equal(a[:1], full[:1])


def test_empty_calls():
    g = _gen(1)
    kc, vc = _caches(g, 3, 2, 16, 64, BF)
    q = _randn(g, 4, 2, 64)
    assert kotodama_amd.paged_attention(q[:0], kc, vc, _ints([[0]]), _ints([5]), _ints([0, 0])).shape == (0, 2, 64)
    table = torch.zeros((0, 4), dtype=torch.int32, device=DEV)
    out, lse = kotodama_amd.paged_attention(q, kc, vc, table, _ints([]), _ints([0]), want_lse=True)
    assert not out.any() and (lse == -math.inf).all()  # padding alone
    out = kotodama_amd.paged_attention(q, kc, vc, torch.zeros((1, 0), dtype=torch.int32, device=DEV), _ints([9]),
                                       _ints([0, 4]))
    assert not out.any()
    out = kotodama_amd.paged_attention(q, kc[:0], vc[:0], _ints([[0]]), _ints([9]), _ints([0, 4]))
    assert not out.any()


def test_a_cache_over_4_gib():
    # offsets past 32 bits, in bytes and in elements: the last pages of a 9 GiB cache
    pages, hk, page, d = 70000, 8, 64, 128
    kc = torch.empty((pages, hk, page, d), dtype=BF, device=DEV)
    vc = torch.empty_like(kc)
    assert kc.numel() > 2**32
    g = _gen(3)
    k, v = _randn(g, 100, hk, d), _randn(g, 100, hk, d)
    table = _ints([[pages - 1, 35000]])
    slots = torch.cat((torch.arange(64, device=DEV) + (pages - 1) * page, torch.arange(36, device=DEV) + 35000 * page))
    kotodama_amd.paged_write(k, v, kc, vc, slots)
    assert torch.equal(kc[pages - 1], k[:64].transpose(0, 1)) and torch.equal(vc[35000, :, :36], v[64:].transpose(0, 1))
    q = _randn(g, 3, 16, d)
    out = kotodama_amd.paged_attention(q, kc, vc, table, _ints([100]), _ints([0, 3]))
    want, _ = PO.attention(q, kc[[pages - 1, 35000]], vc[[pages - 1, 35000]], _ints([[0, 1]]), [100], [0, 3])
    _within("out", out, want)


# ---------------------------------------------------------------- verify --


def _verify(logits, ids, starts, u, q=None, temperature=1.0):
    want = PO.verify(logits, ids, starts, u, q, temperature)
    tokens, counts = kotodama_amd.verify_drafts(logits, ids, _ints(starts), u, q, temperature)
    assert tokens.dtype == ids.dtype and counts.dtype == torch.int32
    assert counts.tolist() == want[1]
    assert tokens.tolist() == want[0]
    return tokens, counts


def _drafts(g, new, v, dtype=BF, spread=2.0, near=0.7, probs=True, pad=0):
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    n = starts[-1] + pad
    logits = _randn(g, n, v, dtype=dtype, scale=spread)
    q = torch.softmax(logits.float() + near * torch.randn((n, v), generator=g, device=DEV), -1).to(dtype)
    pick = torch.multinomial(q.float() + 1e-9, 1, generator=g)[:, 0] if n else torch.zeros(0, device=DEV).long()
    ids = torch.cat((pick[:1], pick[:-1]))
    u = torch.rand((n, 2), generator=g, device=DEV)
    return logits, ids, starts, u, q if probs else None


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp32"])
@pytest.mark.parametrize("temperature", [0.0, 0.5, 1.0])
@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("new,v,pad", [([1], 1, 0), ([3], 7, 0), ([1, 0, 4, 2], 8, 3), ([5] * 9, 511, 0),
                                       ([2, 9, 1], 513, 1), ([20, 1, 40], 1000, 0), ([4, 3], 4097, 2),
                                       ([5, 1, 6], 49152, 0), ([3, 2], 130001, 1)])
def test_verify(new, v, pad, probs, temperature, dtype):
    g = _gen(v + len(new))
    logits, ids, starts, u, q = _drafts(g, new, v, dtype, probs=probs, pad=pad)
    print(f"verify_drafts new={new} vocab={v} probs={probs} t={temperature} {dtype}", flush=True)
    _verify(logits, ids, starts, u, q, temperature)


def test_verify_at_the_edges():
    g = _gen(21)
    v = 700
    logits, ids, starts, u, q = _drafts(g, [4, 4, 4, 4, 1], v, FP)
    u[0], u[5], u[16] = 0.0, 1 - 2**-24, 0.0
    _verify(logits, ids, starts, u, q)
    _verify(logits, ids.int(), starts, u, q)
    # drafts no row names
    bad = ids.clone()
    bad[2], bad[5], bad[9] = v, -1, 2**40
    _verify(logits, bad, starts, u, q)
    _verify(logits, bad, starts, u, None)
    _verify(logits, bad, starts, u, None, 0.0)
    # logits of minus infinity (a constrained vocabulary), the draft's own among them
    cut = logits.clone()
    cut[:, 5:650] = -math.inf
    _verify(cut, ids, starts, u, q)
    _verify(cut, ids, starts, u, None, 0.0)
    # a draft of probability zero, and one that the draft model held impossible
    z = q.clone()
    z[0, ids[1]] = 0
    _verify(logits, ids, starts, u, z)
    # the same distribution on both sides: nothing is left over of p - q
    p = torch.softmax(logits.double(), -1).float()
    one = torch.zeros_like(logits).masked_fill(torch.arange(v, device=DEV) != 3, -math.inf)
    q1 = (torch.arange(v, device=DEV) == 3).float().expand_as(logits).contiguous()
    same = torch.full_like(ids, 4)
    _verify(one, same, starts, u, q1)  # the draft 4 falls; of p - q nothing is left, so p's own token
    _verify(logits, ids, starts, u, p)
    # rows without a distribution
    for value in (math.nan, math.inf):
        odd = logits.clone()
        odd[1, 600] = value
        odd[4, 0] = value
        odd[15, 3] = value
        for t in (1.0, 0.0):
            _verify(odd, ids, starts, u, q, t)
    none = logits.clone()
    none[6] = -math.inf
    none[16] = -math.inf
    _verify(none, ids, starts, u, q)
    _verify(none, ids, starts, u, q, 0.0)


def test_verify_refuses_temperatures_before_rounding_them():
    logits, ids, starts, u, probs = _drafts(_gen(23), [3, 2], 50)
    for t in (1e-300, 1e-7, 9e-7, -1e-300, 2e38, 1e300, math.inf, math.nan):
        with pytest.raises(ValueError, match="temperature"):
            kotodama_amd.verify_drafts(logits, ids, _ints(starts), u, probs, t)
    _verify(logits, ids, starts, u, probs, 2.0**-19)


def test_verify_takes_the_lowest_of_equal_logits():
    g = _gen(5)
    logits = torch.randint(0, 3, (6, 9000), generator=g, device=DEV).to(BF)
    ids = torch.zeros(6, dtype=torch.int64, device=DEV)
    tops = [int((r == r.max()).nonzero()[0]) for r in logits.float().cpu()]
    ids[1], ids[2], ids[4] = tops[0], tops[1], tops[3] + 1
    u = torch.zeros((6, 2), device=DEV)
    tokens, counts = _verify(logits, ids, [0, 3, 6], u, None, 0.0)
    assert tokens.tolist() == [tops[0], tops[1], tops[2], tops[3], -1, -1] and counts.tolist() == [3, 1]


@pytest.mark.parametrize("probs", [True, False])
def test_verify_next_to_the_border(probs):
    # numbers one step of fp32 on either side of where a draft just stays
    g = _gen(31)
    v, n = 5000, 40
    logits, ids, starts, u, q = _drafts(g, [2] * n, v, FP, probs=probs)
    p = torch.softmax(logits.double(), -1)
    rows = torch.arange(0, 2 * n, 2, device=DEV)
    d = ids[rows + 1]
    ratio = p[rows, d] / (q[rows, d].double() if probs else 1.0)
    edge = ratio.clamp(max=1 - 2**-24).float()
    for step in (-1, 0, 1):
        near = edge if step == 0 else torch.nextafter(edge, torch.full_like(edge, float(step)))
        u[rows, 0] = near.clamp(0, 1 - 2**-24)
        _verify(logits, ids, starts, u, q)


def test_verify_of_strided_rows():
    g = _gen(41)
    logits, ids, starts, u, q = _drafts(g, [3, 5, 1], 1001, BF)
    want = kotodama_amd.verify_drafts(logits, ids, _ints(starts), u, q)
    wide, wq = torch.zeros((9, 1016), dtype=BF, device=DEV), torch.zeros((9, 1003), dtype=FP, device=DEV)
    wide[:, :1001], wq[:, 2:] = logits, q.float()
    columns = logits.t().contiguous().t()
    for x, y in ((wide[:, :1001], q), (logits, wq[:, 2:]), (columns, q), (wide[:, :1001], wq[:, 2:])):
        for i in (ids, ids.repeat_interleave(2)[::2]):
            got = kotodama_amd.verify_drafts(x, i, _ints(starts).long(), u, y)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    got = paged.verify_drafts_op(logits, ids, _ints(starts), u, q, 1.0)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_sampled_tokens_follow_the_target():
    # drafts and their replacements together are distributed as the target: 40000 sequences of one draft,
    # each token's count within 6 standard deviations
    g = _gen(51)
    n, v = 40000, 12
    row = torch.randn(v, generator=g, device=DEV)
    p = torch.softmax(row.double(), -1)
    q = torch.softmax(row + torch.randn(v, generator=g, device=DEV), -1)
    logits = row.expand(2 * n, v).contiguous()
    drafts = torch.multinomial(q, n, replacement=True, generator=g)
    ids = torch.stack((torch.zeros_like(drafts), drafts), 1).flatten()
    u = torch.rand((2 * n, 2), generator=g, device=DEV)
    tokens, counts = kotodama_amd.verify_drafts(logits, ids, torch.arange(0, 2 * n + 1, 2, device=DEV), u,
                                                q.expand(2 * n, v).contiguous())
    first = torch.bincount(tokens[::2], minlength=v).double()
    assert ((first - n * p).abs() <= 6 * (n * p * (1 - p)).sqrt()).all()
    stay = counts == 2
    second = torch.bincount(tokens[1::2][stay], minlength=v).double()
    m = int(stay.sum())
    assert ((second - m * p).abs() <= 6 * (m * p * (1 - p)).sqrt()).all()


# --------------------------------------------------------- run together --


def test_a_captured_step_is_the_eager_one():
    # slots, write, attention and release in one graph, replayed over growing sequences beside an eager copy
    b, h, hk, page, d, pages = 5, 4, 2, 16, 64, 60
    g = _gen(61)
    caches = [kotodama_amd.PagedCache(1, pages, page, hk, d, b, 8 * page, BF, DEV) for _ in range(2)]
    caches[1].kv.copy_(caches[0].kv.zero_())
    n = 40
    new, drop = torch.zeros(b, dtype=torch.int32, device=DEV), torch.zeros(b, dtype=torch.int32, device=DEV)
    q, k, v = (_randn(g, n, x, d) for x in (h, hk, hk))

    def step(cache):
        with torch.no_grad():
            s = cache.extend(new, n)
            layer = cache.layers(s)[0]
            kotodama_amd.paged_write(k, v, layer.k, layer.v, s.slots)
            out = kotodama_amd.paged_attention(q, layer.k, layer.v, cache.block_table, s.kv_lens, s.q_starts)
            cache.keep(cache.lens - drop)
        return out, s

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(caches[0])  # nothing new: loads the kernels
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, s = step(caches[0])
    rng = random.Random(3)
    for i in range(8):
        new.copy_(_ints([rng.randint(0, 8) if i else 8 for _ in range(b)]))
        drop.copy_(_ints([rng.randint(0, 3) if i else 0 for _ in range(b)]).minimum(new))
        for x in (q, k, v):
            x.copy_(_randn(g, *x.shape))
        graph.replay()
        torch.cuda.synchronize()
        want, ws = step(caches[1])
        torch.cuda.synchronize()
        assert torch.equal(got, want), i
        assert all(torch.equal(x, y) for x, y in zip(s, ws))
        for name in ("lens", "free_count", "free_pages", "block_table", "kv"):
            assert torch.equal(getattr(caches[0], name), getattr(caches[1], name)), (i, name)


def test_another_stream():
    q, kc, vc, table, lens, starts = _batch(71, [1] * 40, [3000 + i for i in range(40)], 8, 2, 16, 128, BF)
    want = kotodama_amd.paged_attention(q, kc, vc, table, lens)
    g = _gen(72)
    logits, ids, vs, u, probs = _drafts(g, [4] * 20, 20000)
    tokens, counts = kotodama_amd.verify_drafts(logits, ids, _ints(vs), u, probs)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for s in streams:  # two calls at once, each with a workspace of its own
            with torch.cuda.stream(s):
                got.append((kotodama_amd.paged_attention(q, kc, vc, table, lens),
                            *kotodama_amd.verify_drafts(logits, ids, _ints(vs), u, probs)))
    torch.cuda.synchronize()
    for o, t, c in got:
        assert torch.equal(o, want) and torch.equal(t, tokens) and torch.equal(c, counts)


def test_two_graphs_at_once():
    # split attention and verification, each graph with a workspace of its own, replayed on two streams together
    q, kc, vc, table, lens, starts = _batch(73, [2] * 30, [2000 + 50 * i for i in range(30)], 8, 2, 16, 64, BF)
    g = _gen(74)
    logits, ids, vs, u, probs = _drafts(g, [5] * 30, 9001)
    s, v = _ints(starts), _ints(vs)
    sides = [(q.clone(), logits.clone(), u.clone()) for _ in range(2)]

    def call(x):
        return (*kotodama_amd.paged_attention(x[0], kc, vc, table, lens, s, want_lse=True),
                *kotodama_amd.verify_drafts(x[1], ids, v, x[2], probs))

    want = call(sides[0])
    torch.cuda.synchronize()
    graphs, results, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for x in sides:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(call(x))
        graphs.append(graph)
    for i in range(4):
        for x in sides:
            for t in x:
                t.copy_(torch.rand(t.shape, generator=g, device=DEV) if t.shape[-1] == 2 else
                        _randn(g, *t.shape, dtype=t.dtype))
        want = [call(x) for x in sides]
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(results, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b)), i


def test_under_inference_mode():
    with torch.inference_mode():
        cache = kotodama_amd.PagedCache(1, 9, 16, 2, 64, 2, 64, BF, DEV)
        g = _gen(75)
        q, k, v = (_randn(g, 40, h, 64) for h in (4, 2, 2))
        for native in (True, False):
            step = cache.extend(_ints([20, 17]), 40)
            layer = cache.layers(step)[0]
            if native:
                kotodama_amd.paged_write(k, v, layer.k, layer.v, step.slots)
                out = kotodama_amd.paged_attention(q, layer.k, layer.v, cache.block_table, step.kv_lens, step.q_starts)
            else:
                paged._paged_write_impl(k, v, layer.k, layer.v, step.slots)
                again, _ = paged._paged_attention_impl(q, layer.k, layer.v, cache.block_table, step.kv_lens,
                                                       step.q_starts, 1 / 8)
                assert torch.equal(out, again)
            assert step.kv_lens.tolist() == [20, 17]
            cache.keep(_ints([0, 0]))
    want, bound = PO.attention(q, layer.k, layer.v, cache.block_table, [20, 17], [0, 20, 37])[0]
    assert ((out.double() - want).abs() <= bound).all()


def test_compiled_calls():
    q, kc, vc, table, lens, starts = _batch(81, [3, 2], [40, 70], 4, 2, 16, 64, BF)
    g = _gen(82)
    logits, ids, vs, u, probs = _drafts(g, [3, 2], 500)
    held, free, count, s = _ints([37, 68]), torch.arange(9, dtype=torch.int32, device=DEV), _ints([9]), _ints(starts)

    def step(q, table):
        st = kotodama_amd.paged_slots(table, held, _ints5, free, count, 16, 5)
        kotodama_amd.paged_write(q[:, :2], q[:, 2:], kc, vc, torch.full_like(st.slots, -1))
        back = kotodama_amd.paged_release(table, st.kv_lens, held, free_out, st.free_count, 16)
        return (kotodama_amd.paged_attention(q, kc, vc, table, lens, s) * 1.0, st.slots + 0, back,
                *kotodama_amd.verify_drafts(logits, ids, _ints(vs), u, probs))

    _ints5 = _ints([3, 2])
    free_out = torch.zeros(12, dtype=torch.int32, device=DEV)
    t = table.clone()
    want = step(q, t)
    t2 = table.clone()
    got = torch.compile(step, backend="aot_eager")(q, t2)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert torch.equal(t, t2)


@pytest.mark.parametrize("op", ["slots", "release", "write", "attention", "verify"])
def test_ops_are_registered_soundly(op):
    q, kc, vc, table, lens, starts = _batch(91, [3, 2], [40, 70], 4, 2, 16, 64, BF)
    g = _gen(92)
    logits, ids, vs, u, probs = _drafts(g, [3, 2], 500)
    free, count = torch.arange(9, dtype=torch.int32, device=DEV), _ints([5])
    fn, args = {
        "slots": (paged.paged_slots_op, (table, _ints([37, 68]), _ints([3, 2]), free, count, 16, 5)),
        "release": (paged.paged_release_op, (table.clamp(min=0), lens, _ints([3, 2]), free, count, 16)),
        "write": (paged.paged_write_op, (q[:, :2], q[:, 2:], kc, vc, torch.arange(5, device=DEV))),
        "attention": (paged.paged_attention_op, (q, kc.nan_to_num(), vc.nan_to_num(), table, lens, _ints(starts),
                                                 0.125)),
        "verify": (paged.verify_drafts_op, (logits, ids, _ints(vs), u, probs, 1.0)),
    }[op]
    torch.library.opcheck(fn, args, test_utils=("test_schema", "test_faketensor"))
