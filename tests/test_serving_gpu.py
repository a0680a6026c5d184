"""Block tables on the GPU, pages in 4 bits with their attention, and log probabilities, against plain implementations in
64 bits; their refusals; a run of them together, captured and replayed."""

from __future__ import annotations

import random

import pytest
import torch
from plain import serving_plain as plain

from lockstep_amd.ops import Fp4Pages, KernelError, kernels

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}        # half a step, relative


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# -- tables ---------------------------------------------------------------------------------------------------------
def run_tables(lengths, news, table, page, free, cursor, room):
    n = len(lengths)
    out = {"slots": i32([7] * room), "tok_seq": i32([7] * room), "tok_pos": i32([7] * room), "offsets": i32([7] * (n + 1)),
           "new_lengths": i32([7] * n), "progress": i32([7, 7])}
    t = torch.tensor(table, dtype=torch.int32, device=DEV).reshape(n, -1 if n else 1)
    kernels().step_tables(i32(lengths), i32(news), t, page, i32(free), i32([cursor]), out["slots"], out["tok_seq"],
                          out["tok_pos"], out["offsets"], out["new_lengths"], out["progress"])
    found = {k: v.tolist() for k, v in out.items()}
    found["table"] = t.tolist()
    return found


def check_tables(lengths, news, table, page, free, cursor, room):
    found = run_tables(lengths, news, table, page, free, cursor, room)
    want = plain.step_tables(lengths, news, [list(r) for r in table], page, free, cursor, room)
    for key in want:
        assert found[key] == want[key], key


@pytest.mark.parametrize("requests,longest,new,page,spare,short_rows", [
    (1, 0, 1, 16, 0, 0), (1, 16, 1, 16, 0, 0), (1, 15, 1, 16, 0, 0), (64, 300, 1, 16, 5, 0), (7, 100, 65, 8, 0, 0),
    (255, 40, 9, 32, 3, 0), (257, 40, 9, 4, 0, 0), (1100, 20, 7, 8, 0, 0), (3, 1000, 5000, 128, 0, 0), (40, 90, 30, 8, -9, 0),
    (40, 90, 30, 8, 0, 55), (40, 90, 30, 8, -30, 100), (513, 10, 3, 4, -100, 400)])
def test_tables(requests, longest, new, page, spare, short_rows):
    rng = random.Random(requests * 31 + new)
    lengths = [rng.randint(0, longest) for _ in range(requests)]
    news = [rng.choice((0, 1, new, rng.randint(0, new))) for _ in range(requests)]
    columns = -(-(longest + new) // page)
    ids = list(range(requests * columns))
    rng.shuffle(ids)
    table = [[-1] * columns for _ in range(requests)]
    for row, length in zip(table, lengths):
        for c in range(-(-length // page)):
            row[c] = ids.pop()
    need = sum(-(-(h + n) // page) - -(-h // page) for h, n in zip(lengths, news))
    cursor = rng.choice((0, 3))
    free = [rng.randrange(1 << 20) for _ in range(max(0, cursor + need + spare))]
    room = max(0, sum(news) + (5 if not short_rows else -short_rows))
    check_tables(lengths, news, table, page, free, cursor, room)


def test_tables_of_odd_requests():
    # negative numbers, more than the row holds, a released page in the row, a negative page in the list, no free list
    check_tables([-1, 3, 60, 8, 2, 2147483647], [2, -4, 10, 2, 0, 5], [[1] * 8, [2] * 8, [3] * 8, [4, 5] + [-1] * 6, [-1] * 8, [6] * 8], 8,
                 [-3, 11], 0, 30)
    check_tables([8, 20], [1, 3], [[5, -1, -1, -1], [6, 7, -1, -1]], 8, [], 0, 9)
    check_tables([8, 20], [1, 3], [[5, -1, -1, -1], [6, 7, -1, -1]], 8, [1, 2], -1, 9)
    check_tables([8, 20], [0, 0], [[5, -1, -1, -1], [6, 7, 1, -1]], 8, [1, 2], 5, 0)


def test_tables_refusals():
    k = kernels()
    base = dict(lengths=i32([1, 2]), news=i32([1, 1]), table=torch.zeros((2, 3), dtype=torch.int32, device=DEV), page_size=8,
                free_pages=i32([1, 2]), cursor=i32([0]), slots=i32([0] * 4), tok_seq=i32([0] * 4), tok_pos=i32([0] * 4),
                offsets=i32([0] * 3), new_lengths=i32([0] * 2), progress=i32([0] * 2))
    k.step_tables(**base)
    both = i32([0] * 8)
    for change in (dict(news=i32([1])), dict(page_size=12), dict(page_size=2), dict(cursor=i32([0, 1])), dict(tok_pos=i32([0] * 3)),
                   dict(offsets=i32([0, 0])), dict(progress=i32([0])), dict(lengths=i32([1, 2]).long()),
                   dict(table=torch.zeros((3, 3), dtype=torch.int32, device=DEV)), dict(table=torch.zeros((2, 6), dtype=torch.int32, device=DEV)[:, ::2]),
                   dict(new_lengths=base["lengths"]), dict(slots=both[:4], tok_seq=both[2:6])):
        with pytest.raises(KernelError):
            k.step_tables(**{**base, **change})
    many = 8193
    with pytest.raises(KernelError, match="at most"):
        k.step_tables(**{**base, "lengths": i32([0] * many), "news": i32([0] * many), "table": torch.zeros((many, 1), dtype=torch.int32, device=DEV),
                         "offsets": i32([0] * (many + 1)), "new_lengths": i32([0] * many)})
    torch.cuda.synchronize()


def test_tables_of_the_most_requests():
    n = 8192
    check_tables([i % 9 for i in range(n)], [1 + i % 2 for i in range(n)], [[i, -1, -1] for i in range(n)], 8, list(range(n, 2 * n)), 0, 2 * n)


# -- pages in 4 bits --------------------------------------------------------------------------------------------------
def random_rows(g, tokens, heads, d, dtype):
    x = torch.randn((tokens, heads * d), generator=g) * torch.exp(torch.randn((tokens, heads * d), generator=g))
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,heads,d,page", [(1, 1, 32, 4), (3, 2, 64, 8), (37, 3, 96, 16), (70, 1, 128, 64), (9, 2, 256, 128), (130, 5, 160, 8)])
def test_write_and_read(tokens, heads, d, page, dtype):
    g = torch.Generator().manual_seed(tokens * d)
    k, v = (random_rows(g, tokens, heads, d, dtype) for _ in range(2))
    # values on the borders between two levels, small and large magnitudes, zeros
    borders = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -0.75, -2.5, -5.0, 7.9, 0.0, -0.0, 0.2499])
    k[0, :16] = borders.to(dtype)
    k[0, 16:32] = 0
    v[0, :32] = 0
    v[tokens - 1, d - 32:d] = (v[tokens - 1, d - 32:d].float() * 2.0 ** 100).to(dtype)
    v[tokens // 2, :32] = (v[tokens // 2, :32].float() * 2.0 ** -118).to(dtype)
    pages = tokens // page + 3
    pool = Fp4Pages.empty(pages, heads, page, d, device=DEV)
    for t in pool:
        t.random_(0, 255)           # (no 255: groups of zeros and ones in between)
    before = [t.clone() for t in pool]
    order = torch.randperm(pages * page, generator=g)[:tokens]
    slots = order.to(torch.int32).to(DEV)
    wide = torch.full((tokens, heads * d + 8), 3.0, dtype=dtype)      # rows that are parts of wider ones, not aligned to 16 bytes
    wide[:, 1:heads * d + 1] = k
    kernels().fp4_write(wide.to(DEV)[:, 1:heads * d + 1], v.to(DEV), slots, pool)
    keys, values = plain.values_of_pages(pool)
    flat = [x.transpose(1, 2).reshape(pages * page, heads * d) for x in (keys, values)]
    assert torch.equal(flat[0][order], plain.held(k))
    assert torch.equal(flat[1][order], plain.held(v))
    # nothing else has changed
    old = [x.transpose(1, 2).reshape(pages * page, heads * d) for x in plain.values_of_pages(before)]
    rest = torch.ones(pages * page, dtype=torch.bool)
    rest[order] = False
    assert all(torch.equal(a[rest], b[rest]) for a, b in zip(flat, old))
    # and back, exact in both types
    for out_dtype in (torch.float32, torch.bfloat16):
        rows = torch.full((tokens, heads * d + 24), 5.0, dtype=out_dtype, device=DEV)
        other = torch.full((tokens, heads * d), 5.0, dtype=out_dtype, device=DEV)
        kernels().fp4_read(pool, slots, rows[:, 3:heads * d + 3], other)
        assert torch.equal(rows[:, 3:heads * d + 3].cpu().double(), plain.held(k))
        assert torch.equal(other.cpu().double(), plain.held(v))
        assert bool((rows[:, :3] == 5).all()) and bool((rows[:, heads * d + 3:] == 5).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_slots_that_are_none_and_groups_that_are_not_finite(dtype):
    heads, d, page, pages = 2, 64, 8, 3
    g = torch.Generator().manual_seed(5)
    k, v = (random_rows(g, 6, heads, d, dtype) for _ in range(2))
    k[1, 70], v[1, 3], v[2, 40] = float("nan"), float("inf"), float("-inf")
    pool = Fp4Pages.empty(pages, heads, page, d, device=DEV)
    slots = i32([0, 23, 9, -1, 24, 2147483647])
    kernels().fp4_write(k.to(DEV), v.to(DEV), slots, pool)
    keys, values = plain.values_of_pages(pool)
    flat = [x.transpose(1, 2).reshape(pages * page, heads * d) for x in (keys, values)]
    for row, slot in ((0, 0), (1, 23), (2, 9)):
        for x, got in ((k, flat[0]), (v, flat[1])):
            assert torch.equal(torch.nan_to_num(got[slot], nan=77.0), torch.nan_to_num(plain.held(x[row]), nan=77.0))
    untouched = [s for s in range(24) if s not in (0, 23, 9)]
    assert not flat[0][untouched].any() and not flat[1][untouched].any()
    back = torch.full((6, heads * d), 5.0, dtype=dtype, device=DEV)
    other = back.clone()
    kernels().fp4_read(pool, slots, back, other)
    assert torch.isnan(back[1, 64:96]).all() and torch.isnan(other[2, 32:64]).all()
    assert bool((back[3:] == 5).all()) and bool((other[3:] == 5).all())


def test_numbers_below_the_smallest_scale():
    x = torch.zeros((1, 32))
    x[0, :6] = torch.tensor([2.0 ** -126, 1.5 * 2.0 ** -127, 2.0 ** -127, 2.0 ** -128, -(2.0 ** -126), 3 * 2.0 ** -149])
    pool = Fp4Pages.empty(1, 1, 4, 32, device=DEV)
    kernels().fp4_write(x.to(DEV), x.to(DEV), i32([1]), pool)
    assert torch.equal(plain.values_of_pages(pool)[0][0, 0, 1], plain.held(x[0]))


def test_page_refusals():
    k = kernels()
    pool = Fp4Pages.empty(2, 2, 16, 64, device=DEV)
    x = torch.zeros((3, 128), device=DEV)
    s = i32([0, 1, 2])
    k.fp4_write(x, x, s, pool)
    for args in ((x[:, :64], x, s, pool), (x, x.bfloat16(), s, pool), (x, x[:2], s, pool), (x, x, s[:2], pool), (x, x, s.long(), pool),
                 (x.half(), x.half(), s, pool), (x.t(), x, s, pool), (x, x, s, pool._replace(k_scales=pool.k_scales[:1])),
                 (x, x, s, pool._replace(v_codes=pool.v_codes.float())), (x, x, s, pool._replace(v_codes=pool.v_codes.transpose(2, 3)))):
        with pytest.raises(KernelError):
            k.fp4_write(*args)
    one = torch.zeros((1, 128), device=DEV)
    with pytest.raises(KernelError, match="overlap"):
        k.fp4_read(pool, s, one.expand(3, 128), x)
    with pytest.raises(KernelError, match="overlap"):
        k.fp4_read(pool, s, x, x)
    torch.cuda.synchronize()


# -- attention ----------------------------------------------------------------------------------------------------------
def make_cache(g, lengths, heads, d, page, extra_columns=0, spare_pages=3):
    """Pages of random keys and values; what no request holds reads as NaN."""
    need = [-(-max(n, 0) // page) for n in lengths]
    pages = sum(need) + spare_pages
    pool = Fp4Pages.empty(pages, heads, page, d, device=DEV)
    for t in pool:
        t.fill_(255)
    ids = torch.randperm(pages, generator=g).tolist()
    columns = max(max(need, default=0), 1) + extra_columns
    table, slots = [], []
    for n, c in zip(lengths, need):
        row = [ids.pop() for _ in range(c)]
        slots += [row[p // page] * page + p % page for p in range(max(n, 0))]
        table.append(row + [-1] * (columns - c))
    if slots:
        spread = torch.exp(0.3 * torch.randn(heads * d, generator=g))
        k, v = ((torch.randn((len(slots), heads * d), generator=g) * spread).to(DEV) for _ in range(2))
        kernels().fp4_write(k, v, i32(slots), pool)
    return pool, table


def run_attention(q, heads, kv_heads, d, pool, table, offsets, lengths, window, scale=None, most=None, longest=None):
    n = [b - a for a, b in zip(offsets, offsets[1:])]
    out = torch.full_like(q, 9.0)
    kernels().fp4_attention(q, heads, kv_heads, d, pool, torch.tensor(table, dtype=torch.int32, device=DEV), i32(offsets), i32(lengths),
                            max(n) if most is None else most, max(max(lengths), 0) if longest is None else longest, out,
                            d ** -0.5 if scale is None else scale, window=window)
    return out


def check_attention(out, q, heads, kv_heads, d, pool, table, offsets, lengths, page, window, scale=None):
    keys, values = plain.values_of_pages(pool)
    want, spread, reach = plain.attention(q, heads, kv_heads, d, keys, values, table, offsets, lengths, page,
                                          d ** -0.5 if scale is None else scale, window)
    rows = offsets[-1]
    got = out[:rows, :heads * d].double().cpu()
    want, spread, reach = want[:rows], spread[:rows], reach[:rows]
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    # A score is a sum of d products, in 32 bits: off by (d + 4) 2^-24 of the sum of their magnitudes at most, which moves a
    # weight by that factor, and twice the output's spread (weights and their sum); a hardware exponential is within 2^-21.
    # Weights and outputs are rounded to the type (weights in float32: three terms, exact); sums of n terms in 32 bits are
    # off by n 2^-24 of their magnitudes, n at most the length, the folds included.
    u = U[q.dtype]
    weights = u if q.dtype == torch.bfloat16 else 0.0
    sums = (max(lengths) + 64) * 2.0 ** -24
    bound = 2 * spread * ((d + 4) * 2.0 ** -24 * reach + 2.0 ** -21) + spread * (weights + 2 * sums) + u * want.abs() + 1e-30
    wrong = (got - want).abs() > bound
    assert not bool(wrong.any()), ((got - want).abs() / bound).nan_to_num().max()
    return got, want


SHAPES = [
    # lengths, new tokens of each, query heads, kv heads, d, page, window
    ([1], [1], 1, 1, 32, 4, 0),
    ([5, 1, 33], [1, 1, 1], 4, 2, 64, 8, 0),
    ([532, 17, 256, 257], [1, 1, 1, 1], 8, 4, 128, 16, 0),
    ([700, 0, 31, 32], [1, 1, 1, 1], 6, 2, 96, 8, 0),
    ([300, 1000], [2, 3], 4, 1, 128, 64, 0),
    ([90, 40], [1, 1], 16, 1, 256, 32, 0),
    ([513], [1], 3, 3, 160, 128, 0),
    ([400, 90], [1, 1], 2, 1, 224, 16, 77),
    ([40], [40], 2, 2, 32, 4, 0),
    ([100, 70], [61, 70], 4, 2, 64, 16, 0),
    ([130, 260], [129, 131], 3, 1, 128, 16, 0),
    ([200, 30], [100, 30], 2, 2, 256, 32, 0),
    ([150], [77], 4, 4, 96, 8, 0),
    ([260, 64], [70, 64], 4, 2, 128, 16, 33),
    ([333], [50], 2, 1, 64, 8, 1),
    # prompts beside decoded tokens, requests that bring nothing, splits of a short portion of a long context
    ([150, 500, 20, 90, 0], [60, 1, 0, 2, 0], 8, 2, 128, 16, 0),
    ([2100], [20], 4, 4, 64, 32, 0),
    ([1500, 700], [40, 1], 2, 2, 128, 16, 400),
    ([70], [70], 40, 1, 32, 16, 0),
    ([30, 9], [1, 1], 40, 2, 64, 16, 0),
    # many rows in several splits: their sums lie by request, not by row
    ([2300], [2048], 4, 1, 32, 16, 0),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention(shape, dtype):
    lengths, news, heads, kv_heads, d, page, window = SHAPES[shape]
    g = torch.Generator().manual_seed(shape)
    pool, table = make_cache(g, lengths, kv_heads, d, page, extra_columns=shape % 3)
    offsets = [0]
    for n in news:
        offsets.append(offsets[-1] + n)
    wide = (2.0 * torch.randn((offsets[-1] + 2, heads * d + 24), generator=g)).to(dtype).to(DEV)
    q = wide[:, 8:]
    out = run_attention(q, heads, kv_heads, d, pool, table, offsets, lengths, window)
    check_attention(out, q[:, :heads * d], heads, kv_heads, d, pool, table, offsets, lengths, page, window)
    assert bool((out[offsets[-1]:] == 9).all()) and bool((out[:, heads * d:] == 9).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [32, 96, 128, 256])
def test_rows_off_every_boundary(d, dtype):
    """Queries and outputs at odd elements of rows of odd length: one split, several, single tokens, prompts."""
    g = torch.Generator().manual_seed(17)
    lengths, news = [9, 1700, 40, 1300], [1, 1, 33, 60]
    pool, table = make_cache(g, lengths, 2, d, 16)
    offsets = [0, 1, 2, 35, 95]
    wide = torch.randn((95, 4 * d + 7), generator=g).to(dtype).to(DEV)
    q = wide[:, 3:4 * d + 3]
    rows = torch.full((95, 4 * d + 9), 9.0, dtype=dtype, device=DEV)
    out = rows[:, 5:4 * d + 5]
    for first, last in ((0, 4), (0, 2), (2, 4)):
        rows.fill_(9.0)
        lo, hi = offsets[first], offsets[last]
        kernels().fp4_attention(q[lo:hi], 4, 2, d, pool, torch.tensor(table[first:last], dtype=torch.int32, device=DEV),
                                i32([o - lo for o in offsets[first:last + 1]]), i32(lengths[first:last]), max(news[first:last]),
                                max(lengths[first:last]), out[lo:hi], d ** -0.5)
        check_attention(out[lo:hi], q[lo:hi], 4, 2, d, pool, table[first:last], [o - lo for o in offsets[first:last + 1]],
                        lengths[first:last], 16, 0)
        assert bool((rows[:, :5] == 9).all()) and bool((rows[:, 4 * d + 5:] == 9).all())
        assert bool((rows[:lo] == 9).all()) and bool((rows[hi:] == 9).all())


def test_attention_of_one_key_is_its_value():
    g = torch.Generator().manual_seed(3)
    pool, table = make_cache(g, [1], 1, 64, 8)
    q = torch.randn((1, 64), generator=g).to(DEV)
    out = run_attention(q, 1, 1, 64, pool, table, [0, 1], [1], 0)
    assert torch.equal(out.cpu().double(), plain.values_of_pages(pool)[1][table[0][0], 0, 0][None])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("news", [[1, 2], [40, 33]])
def test_pages_that_are_not_there(news, dtype):
    heads, kv_heads, d, page, lengths = 4, 2, 64, 8, [200, 90]
    g = torch.Generator().manual_seed(11)
    pool, table = make_cache(g, lengths, kv_heads, d, page)
    table[0][0], table[0][7], table[0][11] = -1, pool.k_codes.shape[0], 2 ** 31 - 1
    table[1] = [-5] * len(table[1])                    # nothing left
    offsets = [0, news[0], sum(news)]
    q = torch.randn((sum(news), heads * d), generator=g).to(dtype).to(DEV)
    out = run_attention(q, heads, kv_heads, d, pool, table, offsets, lengths, 0)
    check_attention(out, q, heads, kv_heads, d, pool, table, offsets, lengths, page, 0)
    assert not out[news[0]:].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [32, 64, 128, 96])
def test_groups_that_are_not_finite_reach_the_rows_that_see_them(d, dtype):
    heads, kv_heads, page, lengths, news = 4, 2, 16, [70, 300], [30, 1]
    g = torch.Generator().manual_seed(d)
    pool, table = make_cache(g, lengths, kv_heads, d, page)
    # a key at position 50 and a value at position 60 of request 0 (seen by some of its rows), a value at position 290 of request 1
    pool.k_scales[table[0][3], 0, 2, 0] = 255
    pool.v_scales[table[0][3], 1, 3, d // 32 - 1, 0] = 255
    pool.v_scales[table[1][18], 0, 0, 0, 2] = 255
    offsets = [0, 30, 31]
    q = torch.randn((31, heads * d), generator=g).to(dtype).to(DEV)
    for window in (0, 10):
        out = run_attention(q, heads, kv_heads, d, pool, table, offsets, lengths, window)
        got, _ = check_attention(out, q, heads, kv_heads, d, pool, table, offsets, lengths, page, window)
        assert bool(torch.isnan(got).any()) and bool(torch.isfinite(got[:10]).all())


@pytest.mark.parametrize("news", [1, 40])
def test_queries_that_are_not_finite_stay_in_their_rows(news):
    g = torch.Generator().manual_seed(2)
    pool, table = make_cache(g, [90, 90], 2, 64, 16)
    q = torch.randn((2 * news, 4 * 64), generator=g)
    q[0, 70] = float("nan")
    out = run_attention(q.to(DEV), 4, 2, 64, pool, table, [0, news, 2 * news], [90, 90], 0).cpu()
    assert torch.isnan(out[0, 64:128]).all()
    out[0, 64:128] = 0
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_request_has_the_same_bits_beside_others(dtype):
    heads, kv_heads, d, page = 8, 2, 128, 16
    lengths, news = [700, 3000, 90, 5000], [1, 1, 40, 1]
    g = torch.Generator().manual_seed(4)
    pool, table = make_cache(g, lengths, kv_heads, d, page)
    offsets = [0, 1, 2, 42, 43]
    q = torch.randn((43, heads * d), generator=g).to(dtype).to(DEV)
    together = run_attention(q, heads, kv_heads, d, pool, table, offsets, lengths, 0)
    for i in range(4):
        part = q[offsets[i]:offsets[i + 1]]
        alone = run_attention(part, heads, kv_heads, d, pool, [table[i]], [0, news[i]], [lengths[i]], 0)
        assert torch.equal(alone, together[offsets[i]:offsets[i + 1]]), i
        again = run_attention(part, heads, kv_heads, d, pool, [table[i]], [0, news[i]], [lengths[i]], 0, most=news[i], longest=len(table[i]) * page)
        assert torch.equal(again, alone), i


def test_offsets_and_lengths_that_do_not_fit():
    g = torch.Generator().manual_seed(6)
    pool, table = make_cache(g, [40, 40, 40], 1, 32, 8)
    q = torch.randn((6, 32), generator=g).to(DEV)
    # requests 0 and 2 end beyond the rows or before they begin: their rows stay; request 1 says more keys than its table has
    out = run_attention(q, 1, 1, 32, pool, table, [4, 1, 3, 90], [40, 1000, 40], 0, most=6, longest=40)
    assert bool((out[0] == 9).all()) and bool((out[3:] == 9).all())
    check_attention(out[1:3], q[1:3], 1, 1, 32, pool, [table[1]], [0, 2], [40], 8, 0)
    # a length below the rows: those before the first key see nothing
    out = run_attention(q[:5], 1, 1, 32, pool, table[:1], [0, 5], [2], 0)
    assert not out[:3].any() and bool(out[3:].any())


@pytest.mark.parametrize("news", [1, 40])
def test_queries_beyond_the_largest_bfloat16(news):
    """The largest float32 numbers round to an infinity in bfloat16; with keys as small as they get the scores are ordinary."""
    g = torch.Generator().manual_seed(21)
    length, page, d = 50, 16, 32
    pool, table = make_cache(g, [length], 1, d, page)
    pool.k_scales[pool.k_scales < 255] = 2                  # keys of at most 6 times 2^-125
    q = torch.randn((news, 2 * d), generator=g)
    q[:, 3], q[:, 7], q[:, d + 1] = torch.finfo(torch.float32).max, -3.395e38, 3.4e38
    q = q.to(DEV)
    out = run_attention(q, 2, 1, d, pool, table, [0, news], [length], 0, scale=0.25)
    got, _ = check_attention(out, q, 2, 1, d, pool, table, [0, news], [length], page, 0, scale=0.25)
    assert bool(torch.isfinite(got).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads", [4, 64])
def test_more_rows_or_keys_than_stated(heads, dtype):
    """A request of more rows than stated is left out, also where the fold of splits would find its rows; a greater length counts as
    the greatest one."""
    g = torch.Generator().manual_seed(14)
    lengths, news = [2000, 900, 1300, 5000], [1, 40, 2, 1]
    pool, table = make_cache(g, lengths, 2, 64, 16)
    offsets = [0, 1, 41, 43, 44]
    q = torch.randn((44, heads * 64), generator=g).to(dtype).to(DEV)
    for most in (1, 2):
        out = run_attention(q, heads, 2, 64, pool, table, offsets, lengths, 0, most=most, longest=2100)
        left = [i for i, n in enumerate(news) if n > most]
        for i in left:
            assert bool((out[offsets[i]:offsets[i + 1]] == 9).all()), i
        for i in set(range(4)) - set(left):
            check_attention(out[offsets[i]:offsets[i + 1]], q[offsets[i]:offsets[i + 1]], heads, 2, 64, pool, [table[i]], [0, news[i]],
                            [min(lengths[i], 2100)], 16, 0)
    out = run_attention(q, heads, 2, 64, pool, table, offsets, lengths, 0, most=40, longest=950)
    check_attention(out, q, heads, 2, 64, pool, table, offsets, [min(n, 950) for n in lengths], 16, 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("window", [0, 1000])
def test_many_portions_behind_long_contexts(dtype, window):
    """Splits' sums of requests of every size lie beside one another: portions of a few tokens, decoded tokens, requests that bring
    nothing or more than stated, each with the bits that it has alone."""
    heads, kv_heads, d, page = 8, 2, 64, 16
    lengths = [2500, 1900, 1300, 2900, 3000, 700, 1100, 2600, 1700, 2200]
    news = [33, 1, 5, 0, 9, 90, 1, 33, 2, 17]
    g = torch.Generator().manual_seed(40)
    pool, table = make_cache(g, lengths, kv_heads, d, page)
    offsets = [0]
    for n in news:
        offsets.append(offsets[-1] + n)
    q = torch.randn((offsets[-1] + 3, heads * d), generator=g).to(dtype).to(DEV)
    out = run_attention(q, heads, kv_heads, d, pool, table, offsets, lengths, window, most=33)
    left = news.index(90)                   # more rows than stated: left out
    assert bool((out[offsets[left]:offsets[left + 1]] == 9).all()) and bool((out[offsets[-1]:] == 9).all())
    whole = run_attention(q, heads, kv_heads, d, pool, table, offsets, lengths, window)
    check_attention(whole, q, heads, kv_heads, d, pool, table, offsets, lengths, page, window)
    whole[offsets[left]:offsets[left + 1]] = 9
    assert torch.equal(out, whole)
    for i, n in enumerate(news):
        if n and i != left:
            rows = slice(offsets[i], offsets[i + 1])
            assert torch.equal(run_attention(q[rows], heads, kv_heads, d, pool, [table[i]], [0, n], [lengths[i]], window), out[rows]), i


@pytest.mark.parametrize("news", [1, 30])
def test_windows_as_wide_as_the_context(news):
    g = torch.Generator().manual_seed(10)
    pool, table = make_cache(g, [300, 90], 2, 64, 16)
    q = torch.randn((2 * news, 4 * 64), generator=g).to(DEV)
    args = (q, 4, 2, 64, pool, table, [0, news, 2 * news], [300, 90])
    whole = run_attention(*args, 0)
    for window in (300, 301, 2 ** 31 - 1, 2 ** 40):
        assert torch.equal(run_attention(*args, window), whole)
    check_attention(run_attention(*args, 299), q, 4, 2, 64, pool, table, [0, news, 2 * news], [300, 90], 16, 299)


def test_rows_of_no_request_do_not_hide_a_decoded_token():
    """As many rows as if every request brought the most: the last ones belong to none."""
    g = torch.Generator().manual_seed(9)
    pool, table = make_cache(g, [50, 70], 2, 64, 16)
    q = torch.randn((80, 4 * 64), generator=g).to(DEV)
    out = run_attention(q, 4, 2, 64, pool, table, [0, 40, 41], [50, 70], 0, most=40)
    check_attention(out, q, 4, 2, 64, pool, table, [0, 40, 41], [50, 70], 16, 0)
    assert bool((out[41:] == 9).all())


def test_pages_beyond_32_bits():
    heads, d, page = 8, 128, 16
    pages = 2 ** 32 // (heads * page * d // 2) + 40             # codes of more than 4 GiB
    pool = Fp4Pages(*(torch.empty(s, dtype=torch.uint8, device=DEV) for s in Fp4Pages.shapes(pages, heads, page, d)))
    ids = [pages - 1, 3, pages - 7, 0, pages // 2]
    g = torch.Generator().manual_seed(8)
    n = 5 * page - 3
    k, v = (torch.randn((n, heads * d), generator=g).to(DEV) for _ in range(2))
    slots = [ids[p // page] * page + p % page for p in range(n)]
    kernels().fp4_write(k, v, i32(slots), pool)
    q = torch.randn((1, heads * d), generator=g).to(DEV)
    out = run_attention(q, heads, heads, d, pool, [ids], [0, 1], [n], 0)
    few = Fp4Pages(*(t[torch.tensor(ids, device=DEV)].contiguous() for t in pool))
    check_attention(out, q, heads, heads, d, few, [[0, 1, 2, 3, 4]], [0, 1], [n], page, 0)


def test_attention_refusals():
    k = kernels()
    pool = Fp4Pages.empty(4, 2, 16, 64, device=DEV)
    base = dict(q=torch.zeros((3, 256), device=DEV), nq=4, nkv=2, d=64, pages=pool, table=torch.zeros((2, 2), dtype=torch.int32, device=DEV),
                offsets=i32([0, 1, 3]), lengths=i32([5, 7]), max_tokens=2, max_length=7, out=torch.zeros((3, 256), device=DEV), scale=0.1)
    k.fp4_attention(**base)
    for change in (dict(nq=5), dict(nkv=1), dict(d=32), dict(q=base["q"].half()), dict(out=base["out"].bfloat16()), dict(q=base["q"][:, :128]),
                   dict(out=base["out"][:2]), dict(offsets=i32([0, 3])), dict(lengths=i32([5])), dict(max_length=33), dict(window=-1),
                   dict(table=base["table"].long()), dict(table=base["table"][0]), dict(out=base["out"][:1].expand(3, 256)), dict(max_tokens=-1),
                   dict(scale=float("nan")), dict(scale=float("inf")), dict(out=base["q"])):
        with pytest.raises(KernelError):
            k.fp4_attention(**{**base, **change})
    torch.cuda.synchronize()


@pytest.fixture(params=["module", "python"])
def route(request):
    """Calls through the extension module, and through Python's checks alone."""
    k = kernels()
    k.serving, k.fp4_attention_lib(64)
    module = k._calls
    assert module is not None
    if request.param == "python":
        k._calls = None
    yield request.param
    k._calls = module


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_refuses_outputs_in_its_operands(route, dtype):
    k = kernels()
    g = torch.Generator().manual_seed(30)
    pool, table = make_cache(g, [20, 30], 2, 64, 16)
    rows = torch.randn((6, 600), generator=g).to(dtype).to(DEV)
    call = lambda q, out, **change: k.fp4_attention(**{**dict(  # noqa: E731
        q=q, nq=4, nkv=2, d=64, pages=pool, table=torch.tensor(table, dtype=torch.int32, device=DEV), offsets=i32([0, 1, 3]),
        lengths=i32([20, 30]), max_tokens=2, max_length=30, out=out, scale=0.125), **change})
    before = rows.clone()
    for q, out in ((rows[:3], rows[:3]), (rows[:3], rows[1:4]), (rows[1:4], rows[:3]), (rows[:3], rows[2:5]), (rows[:3], rows[:3, 1:]),
                   (rows[:3], rows[:3, 255:]), (rows[:3, 255:], rows[:3]), (rows[:3], rows[:5:2]), (rows[:3, 300:], rows[1:4, 45:])):
        with pytest.raises(KernelError, match="overlap"):
            call(q, out)
    ints = torch.zeros(3 * 256, dtype=torch.float32, device=DEV)
    room = ints.view(torch.int32)
    if dtype is torch.float32:
        room[:3] = i32([0, 1, 3])
        for change in (dict(offsets=room[:3]), dict(lengths=room[766:]), dict(table=room[100:104].view(2, 2))):
            with pytest.raises(KernelError, match="overlap"):
                call(rows[:3], ints.view(3, 256), **change)
    torch.cuda.synchronize()
    assert torch.equal(rows, before)
    # columns side by side, rows behind one another: taken
    want = torch.empty((3, 256), dtype=dtype, device=DEV)
    call(rows[:3], want)
    for q, out in ((rows[:3], rows[:3, 256:512]), (rows[:3], rows[3:]), (rows[:3], rows[2:5, 256:]), (rows[:3], rows[:3, 344:])):
        rows.copy_(before)
        call(q, out)
        assert torch.equal(out[:, :256], want) and torch.equal(rows[:3, :256], before[:3, :256])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_reading_refuses_rows_in_its_operands(route, dtype):
    k = kernels()
    g = torch.Generator().manual_seed(31)
    pool, table = make_cache(g, [20], 2, 64, 16)
    slots = i32([table[0][0] * 16 + 1, table[0][0] * 16 + 7, table[0][1] * 16 + 2])
    rows = torch.full((6, 400), 5.0, dtype=dtype, device=DEV)
    for keys, values in ((rows[:3, :128], rows[:3, :128]), (rows[:3, :128], rows[1:4, :128]), (rows[:3, :128], rows[:3, 127:255]),
                         (rows[:3, 100:228], rows[:3, :128]), (rows[:3, :128], rows[:5:2, :128]), (rows[:3, 272:], rows[1:4, :128].as_strided((3, 128), (400, 1), 399))):
        with pytest.raises(KernelError, match="overlap"):
            k.fp4_read(pool, slots, keys, values)
    bytes_of = [t.view(-1)[:3 * 256 * rows.element_size()] for t in (pool.k_codes, pool.v_codes)]
    for held in bytes_of:
        inside = held[:3 * 128 * rows.element_size()].view(dtype).view(3, 128)
        for pair in ((inside, rows[:3, :128]), (rows[:3, :128], inside)):
            with pytest.raises(KernelError, match="overlap"):
                k.fp4_read(pool, slots, *pair)
    if dtype is torch.float32:
        own = torch.zeros((3, 128), device=DEV)
        own.view(torch.int32).view(-1)[5:8] = slots
        with pytest.raises(KernelError, match="overlap"):
            k.fp4_read(pool, own.view(torch.int32).view(-1)[5:8], own, rows[:3, :128])
    torch.cuda.synchronize()
    assert bool((rows == 5).all())
    want = [torch.empty((3, 128), dtype=dtype, device=DEV) for _ in range(2)]
    k.fp4_read(pool, slots, *want)
    for keys, values in ((rows[:3, :128], rows[:3, 128:256]), (rows[:3, 272:], rows[:3, :128]), (rows[:3, :128], rows[3:, :128]),
                         (rows[:3, :128], rows[2:5, 200:328])):
        rows.fill_(5.0)
        k.fp4_read(pool, slots, keys, values)
        assert torch.equal(keys, want[0]) and torch.equal(values, want[1])


def test_writing_refuses_operands_in_the_pages(route):
    k = kernels()
    pool = Fp4Pages.empty(4, 2, 16, 64, device=DEV)
    x, slots = torch.ones((3, 128), device=DEV), i32([0, 1, 2])
    inside = pool.v_codes.view(-1)[64:64 + 3 * 512].view(torch.float32).view(3, 128)
    scales = pool.k_scales.view(-1)[16:28].view(torch.int32)
    shifted = torch.zeros(2 * pool.k_scales.numel(), dtype=torch.uint8, device=DEV)
    half = pool.k_scales.numel()
    for args in ((inside, x, slots, pool), (x, inside, slots, pool), (x, x, scales, pool),
                 (x, x, slots, pool._replace(v_codes=pool.k_codes.view(pool.v_codes.shape))),
                 (x, x, slots, pool._replace(v_scales=pool.k_scales.view(pool.v_scales.shape))),
                 (x, x, slots, pool._replace(k_scales=shifted[:half].view(pool.k_scales.shape),
                                             v_scales=shifted[half - 16:2 * half - 16].view(pool.v_scales.shape)))):
        with pytest.raises(KernelError, match="overlap"):
            k.fp4_write(*args)
    torch.cuda.synchronize()
    assert not any(bool(t.any()) for t in pool)
    # pages that lie behind one another in one allocation, and one tensor as keys and values: taken
    whole = torch.zeros(sum(t.numel() for t in pool), dtype=torch.uint8, device=DEV)
    parts, at = [], 0
    for t in pool:
        parts.append(whole[at:at + t.numel()].view(t.shape))
        at += t.numel()
    k.fp4_write(x, x, slots, Fp4Pages(*parts))
    keys, values = torch.zeros_like(x), torch.zeros_like(x)
    k.fp4_read(Fp4Pages(*parts), slots, keys, values)
    assert torch.equal(keys, x) and torch.equal(values, x)


def test_logprobs_refuse_outputs_in_their_operands(route):
    k = kernels()
    f, i = (lambda *s: torch.full(s, 9.0, device=DEV)), (lambda *s: torch.full(s, 9, dtype=torch.int32, device=DEV))
    logits = torch.randn((6, 50), generator=torch.Generator().manual_seed(32)).to(DEV)
    before = logits.clone()
    base = dict(logits=logits, tokens=i32([1, 2, 3, 4, 5, 6]), logprob=f(6), entropy=f(6), rank=i(6), top_ids=i(6, 4), top_logprobs=f(6, 4))
    both, ints = f(11), i(24 + 6)
    for change in (dict(entropy=base["logprob"]), dict(logprob=both[:6], entropy=both[5:]), dict(rank=base["tokens"]),
                   dict(rank=base["logprob"].view(torch.int32)), dict(top_ids=base["top_logprobs"].view(torch.int32)),
                   dict(rank=ints[:6], top_ids=ints[5:29].view(6, 4)), dict(logprob=logits.view(-1)[100:106]),
                   dict(top_logprobs=logits.view(-1)[276:].view(6, 4)), dict(tokens=ints[23:29], top_ids=ints[:24].view(6, 4))):
        with pytest.raises(KernelError, match="overlap"):
            k.token_logprobs(**{**base, **change})
    torch.cuda.synchronize()
    assert torch.equal(logits, before) and bool((both == 9).all()) and bool((ints == 9).all())
    k.token_logprobs(**base)
    one = f(12)
    near = dict(logprob=one[:6], entropy=one[6:], rank=ints[:6], top_ids=ints[6:].view(6, 4))       # behind one another: taken
    k.token_logprobs(**{**base, **near})
    assert all(torch.equal(x, base[name]) for name, x in near.items())


def test_no_memory_of_a_call_in_noted_launches():
    """Launches that are noted to be made again would use a call's memory after its end; those without any may be noted."""
    k = kernels()
    pool = Fp4Pages.empty(100, 2, 16, 64, device=DEV)
    table = torch.zeros((1, 100), dtype=torch.int32, device=DEV)
    q, out = torch.zeros((1, 256), device=DEV), torch.zeros((1, 256), device=DEV)
    f, i = (lambda *s: torch.zeros(s, device=DEV)), (lambda *s: torch.zeros(s, dtype=torch.int32, device=DEV))
    try:
        k.tape = []
        k.fp4_attention(q, 4, 2, 64, pool, table, i32([0, 1]), i32([40]), 1, 40, out, 0.1)
        k.token_logprobs(f(2, 400), i(2), f(2), f(2), i(2), i(2, 1), f(2, 1))
        assert len(k.tape) == 2
        with pytest.raises(KernelError, match="repeatable"):
            k.fp4_attention(q, 4, 2, 64, pool, table, i32([0, 1]), i32([1600]), 1, 1600, out, 0.1)
        with pytest.raises(KernelError, match="repeatable"):
            k.token_logprobs(f(2, 60000), i(2), f(2), f(2), i(2), i(2, 1), f(2, 1))
        assert len(k.tape) == 2
    finally:
        k.tape = None
    torch.cuda.synchronize()


# -- log probabilities ----------------------------------------------------------------------------------------------------
def run_logprobs(logits, tokens, top):
    n = logits.shape[0]
    f = lambda *s: torch.full(s, 9.0, device=DEV)  # noqa: E731
    i = lambda *s: torch.full(s, 9, dtype=torch.int32, device=DEV)  # noqa: E731
    out = {"logprob": f(n), "entropy": f(n), "rank": i(n), "top_ids": i(n, top), "top_logprobs": f(n, top)}
    kernels().token_logprobs(logits, i32(tokens), out["logprob"], out["entropy"], out["rank"], out["top_ids"], out["top_logprobs"])
    return out


def check_logprobs(logits, tokens, top):
    got = {k: v.cpu() for k, v in run_logprobs(logits, tokens, top).items()}
    want = plain.token_logprobs(logits, tokens, top)
    assert got["rank"].tolist() == want["rank"]
    assert got["top_ids"].tolist() == want["top_ids"]
    # The sum of the weights: at most 160 additions one after the other for these rows (32 of a lane's piece, a stream's
    # pieces, the lanes, the streams), each off by 2^-24, and weights within 2^-21; a logarithm's ulp; two subtractions.
    # The entropy has the same sums over terms of up to log S + H.
    sums = 160 * 2.0 ** -24 + 2.0 ** -21
    scale = want["log_sum"].abs()
    for name, bound in (("logprob", sums + 4 * 2.0 ** -24 * (want["logprob"].abs() + scale)),
                        ("top_logprobs", sums + 4 * 2.0 ** -24 * (want["top_logprobs"].abs() + scale[:, None])),
                        ("entropy", 2 * sums * (1 + scale + want["entropy"].abs()) + 4 * 2.0 ** -24 * scale)):
        a, b = got[name].double(), want[name]
        assert torch.equal(torch.isnan(a), torch.isnan(b)), name
        same = (a == b) | torch.isnan(b)                    # infinities
        assert bool((same | ((a - b).abs() <= bound)).all()), (name, (a - b).abs().nan_to_num().max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 0), (1, 1, 1), (3, 2, 2), (2, 63, 5), (5, 100, 32), (2, 513, 32), (4, 2047, 20),
                                            (3, 2048, 1), (2, 2049, 32), (3, 4099, 7), (2, 50001, 20), (300, 700, 5), (260, 5003, 32),
                                            (1, 151936, 20), (2, 300007, 32),
                                            (3, 64, 32), (5, 65, 12), (4, 127, 13), (9, 256, 32), (7, 257, 20), (6, 512, 32),
                                            (5, 515, 12), (6, 2050, 12), (3, 4096, 32), (5, 4097, 13), (1540, 4097, 32),
                                            (1539, 8193, 12), (1537, 16384, 32), (3, 16384, 32), (1600, 16385, 5)])
def test_logprobs(rows, vocab, top, dtype):
    g = torch.Generator().manual_seed(rows * vocab)
    wide = (2.5 * torch.randn((rows, vocab + 3), generator=g)).to(dtype).to(DEV)
    logits = wide[:, 1:vocab + 1]
    tokens = torch.randint(0, vocab, (rows,), generator=g).tolist()
    check_logprobs(logits, tokens, top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(11, 3001), (280, 3001), (11, 9001), (1540, 9001), (11, 40001), (280, 40001)])
def test_logprobs_of_odd_rows(rows, vocab, dtype):
    top = 20
    g = torch.Generator().manual_seed(rows)
    x = (2.5 * torch.randn((rows, vocab), generator=g)).to(dtype)
    inf = float("inf")
    tokens = torch.randint(0, vocab, (rows,), generator=g).tolist()
    x[0] = 1.5                                     # all equal
    x[1] = -inf; x[1, [5, 2500, 700]] = torch.tensor([1.0, 3.0, 1.0]).to(dtype); tokens[1] = 700       # masked but for three
    x[2] = -inf                                    # nothing left
    x[3, 40] = float("nan"); tokens[3] = 41        # a NaN
    x[4, 2999] = inf; tokens[4] = 2999             # an infinity
    x[5] = torch.arange(vocab).to(dtype); tokens[5] = 0               # ascending (with ties in bfloat16)
    x[6] = -torch.arange(vocab).to(dtype); tokens[6] = 2500
    x[7, ::2] = -inf; tokens[7] = 2                # half masked, the token too
    x[8] = 0.0; x[8, 1::2] = -0.0; tokens[8] = 3   # zeros of both signs are equal
    x[9, 30] = float("nan"); x[9, 35] = float("nan"); x[9, 2000] = float("nan"); tokens[9] = 35
    x[10, 17] = 3e38; tokens[10] = 18              # one large logit
    check_logprobs(x.to(DEV), tokens, top)
    for short in (40, 300, 515):
        check_logprobs(x.to(DEV)[:64, :short], [t % short for t in tokens[:64]], 32)


def test_tokens_outside_the_vocabulary():
    g = torch.Generator().manual_seed(1)
    x = torch.randn((4, 50), generator=g).to(DEV)
    check_logprobs(x, [-1, 50, 49, 2 ** 31 - 1], 3)


def test_a_row_has_the_same_bits_beside_others():
    g = torch.Generator().manual_seed(12)
    for dtype, vocab, rows in ((torch.float32, 20011, 600), (torch.bfloat16, 20011, 600), (torch.float32, 50021, 600),
                               (torch.bfloat16, 50021, 600), (torch.float32, 5003, 1600), (torch.bfloat16, 16381, 1600)):
        x = (2.5 * torch.randn((rows, vocab), generator=g)).to(dtype).to(DEV)
        tokens = torch.randint(0, vocab, (rows,), generator=g).tolist()
        many = run_logprobs(x, tokens, 5)
        for lo, hi in ((0, 1), (5, 22), (599, 600)):
            few = run_logprobs(x[lo:hi], tokens[lo:hi], 5)
            for name in few:
                assert torch.equal(few[name], many[name][lo:hi]), name


@pytest.mark.parametrize("rows,vocab,top", [((1 << 24) + 5, 3, 1), ((1 << 22) + 3, 16385, 0)])
def test_more_rows_than_a_launch_takes(rows, vocab, top):
    g = torch.Generator().manual_seed(15)
    some = torch.randn((1 if top == 0 else 64, vocab), generator=g).bfloat16().to(DEV)
    logits = some.expand(rows, vocab) if top == 0 else some[torch.arange(rows, device=DEV) % 64]
    f = lambda *s: torch.full(s, 9.0, device=DEV)  # noqa: E731
    i = lambda *s: torch.full(s, 9, dtype=torch.int32, device=DEV)  # noqa: E731
    out = [f(rows), f(rows), i(rows), i(rows, top), f(rows, top)]
    kernels().token_logprobs(logits, torch.ones(rows, dtype=torch.int32, device=DEV), *out)
    few = run_logprobs(some, [1] * len(some), top)
    for x, one in zip(out, few.values()):
        whole = rows // len(some) * len(some)
        assert bool((x[:whole].view(rows // len(some), *one.shape) == one).all()) and torch.equal(x[whole:], one[:rows - whole])


def test_logprobs_refusals():
    k = kernels()
    f, i = (lambda *s: torch.zeros(s, device=DEV)), (lambda *s: torch.zeros(s, dtype=torch.int32, device=DEV))
    base = dict(logits=f(3, 40), tokens=i(3), logprob=f(3), entropy=f(3), rank=i(3), top_ids=i(3, 2), top_logprobs=f(3, 2))
    k.token_logprobs(**base)
    for change in (dict(logits=f(3, 40).half()), dict(logits=f(40, 3).t()), dict(tokens=i(2)), dict(tokens=i(3).long()), dict(logprob=f(4)),
                   dict(entropy=i(3)), dict(rank=f(3)), dict(top_ids=i(3, 3)), dict(top_ids=i(3, 33), top_logprobs=f(3, 33)),
                   dict(logits=f(3, 1)), dict(logits=torch.empty((3, 0), device=DEV), top_ids=i(3, 0), top_logprobs=f(3, 0)),
                   dict(logits=torch.empty((3, 524289), device=DEV))):
        with pytest.raises(KernelError):
            k.token_logprobs(**{**base, **change})
    k.token_logprobs(f(0, 40), i(0), f(0), f(0), i(0), i(0, 2), f(0, 2))
    torch.cuda.synchronize()


# -- the two ways of a call ------------------------------------------------------------------------------------------------
def test_calls_by_the_module_and_by_python():
    """What the extension module accepts, it launches as Python does; what it does not accept, it leaves alone."""
    k = kernels()
    g = torch.Generator().manual_seed(16)
    make = lambda dtype, *s: torch.full(s, 9, dtype=dtype, device=DEV)  # noqa: E731
    ints = lambda *s: make(torch.int32, *s)  # noqa: E731
    kv = torch.randn((2, 9, 128), generator=g).to(DEV)
    q = torch.randn((9, 256), generator=g).to(DEV)
    logits = torch.randn((3, 70000), generator=g).to(DEV)

    def pass_over():
        pool = Fp4Pages.empty(120, 2, 16, 64, device=DEV)
        table = torch.full((2, 60), -1, dtype=torch.int32, device=DEV)
        table[0, :55] = torch.arange(55, dtype=torch.int32, device=DEV)
        tables = [ints(9), ints(9), ints(9), ints(3), ints(2), ints(2)]
        read = [make(torch.bfloat16, 9, 128), make(torch.bfloat16, 9, 128)]
        out, scores = make(torch.float32, 9, 256), [make(torch.float32, 3), make(torch.float32, 3), ints(3), ints(3, 4), make(torch.float32, 3, 4)]
        calls = [("step_tables", (i32([870, 0]), i32([1, 8]), table, 16, i32(list(range(60, 80))), i32([3]), *tables)),
                 ("fp4_write", (kv[0], kv[1], tables[0], pool)), ("fp4_read", None),
                 ("fp4_attention", (q, 4, 2, 64, pool, table, tables[3], tables[4], 8, 871, out, 0.125, 0)),
                 ("token_logprobs", (logits, i32([5, -1, 69999]), *scores))]
        for name, args in calls:
            if name == "fp4_read":
                args = (pool, tables[0], *read)
            getattr(k, name)(*args)
        torch.cuda.synchronize()
        calls[2] = ("fp4_read", (read[0], read[1], tables[0], pool))
        return calls, [table, *tables, *pool, *read, out, *scores]

    k.serving, k.fp4_attention_lib(64)
    assert k._calls is not None
    calls, by_module = pass_over()
    here, stream = torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream
    for name, args in calls:
        entry = getattr(k._calls, name)
        assert entry(here, stream, *args) is True, name
        for i, x in enumerate(args):            # another device, another type, not a tensor, one operand less
            if torch.is_tensor(x):
                assert entry(here, stream, *args[:i], x.cpu(), *args[i + 1:]) is False, (name, i)
                assert entry(here, stream, *args[:i], x.double(), *args[i + 1:]) is False, (name, i)
                assert entry(here, stream, *args[:i], None, *args[i + 1:]) is False, (name, i)
        assert entry(here + 1, stream, *args) is False and entry(here, stream, *args[:-1]) is False, name
    torch.cuda.synchronize()
    module, k._calls = k._calls, None
    try:
        _, by_python = pass_over()
    finally:
        k._calls = module
    for i, (a, b) in enumerate(zip(by_module, by_python)):
        # (step_tables ran twice on the first pass's table, with the same result)
        assert torch.equal(a.view(torch.uint8) if a.is_floating_point() else a, b.view(torch.uint8) if b.is_floating_point() else b), i


def test_the_module_takes_the_pages_that_python_takes(route):
    """Four tensors that are not an Fp4Pages are refused by both, before the library is loaded and afterwards."""
    k = kernels()
    pool = Fp4Pages.empty(2, 2, 16, 64, device=DEV)
    x, slots = torch.ones((3, 128), device=DEV), i32([0, 1, 2])
    q, out = torch.zeros((1, 256), device=DEV), torch.zeros((1, 256), device=DEV)
    table = torch.zeros((1, 2), dtype=torch.int32, device=DEV)
    k.fp4_write(x, x, slots, pool)
    for pages in (tuple(pool), list(pool)):
        for call in (lambda: k.fp4_write(x, x, slots, pages), lambda: k.fp4_read(pages, slots, x, x.clone()),
                     lambda: k.fp4_attention(q, 4, 2, 64, pages, table, i32([0, 1]), i32([3]), 1, 3, out, 0.1)):
            with pytest.raises(KernelError, match="Fp4Pages"):
                call()

    class Mine(Fp4Pages):
        pass

    k.fp4_read(Mine(*pool), slots, x, x.clone())
    torch.cuda.synchronize()


# -- together ---------------------------------------------------------------------------------------------------------------
class Serving:
    """A small decoder's serving state: a linear model of keys, values, queries and logits from token ids."""

    def __init__(self, requests, dtype, seed):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.page, self.columns = dtype, 8, 12
        self.heads, self.kv_heads, self.d, self.vocab = 4, 2, 64, 500
        make = lambda *s: torch.randn(s, generator=g).to(dtype).to(DEV)  # noqa: E731
        self.keys, self.values = make(self.vocab, 128), make(self.vocab, 128)
        self.queries, self.head = make(self.vocab, 256), make(self.vocab, 256) * 0.2
        self.pool = Fp4Pages.empty(requests * self.columns, self.kv_heads, self.page, self.d, device=DEV)
        self.table = torch.full((requests, self.columns), -1, dtype=torch.int32, device=DEV)
        self.free = torch.randperm(requests * self.columns, generator=g).to(torch.int32).to(DEV)
        self.lengths = torch.zeros(requests, dtype=torch.int32, device=DEV)
        self.cursor = i32([0])
        self.requests = requests

    def buffers(self, rows):
        i = lambda *s: torch.zeros(s, dtype=torch.int32, device=DEV)  # noqa: E731
        f = lambda *s: torch.zeros(s, device=DEV)  # noqa: E731
        return dict(slots=i(rows), tok_seq=i(rows), tok_pos=i(rows), offsets=i(self.requests + 1), new_lengths=i(self.requests),
                    progress=i(2), out=torch.zeros((rows, 256), dtype=self.dtype, device=DEV), logprob=f(rows), entropy=f(rows),
                    rank=i(rows), top_ids=i(rows, 3), top_logprobs=f(rows, 3))

    def step(self, tokens, news, most, b):
        k = kernels()
        k.step_tables(self.lengths, news, self.table, self.page, self.free, self.cursor, b["slots"], b["tok_seq"], b["tok_pos"],
                      b["offsets"], b["new_lengths"], b["progress"])
        ids = tokens.long()
        k.fp4_write(self.keys[ids], self.values[ids], b["slots"], self.pool)
        k.fp4_attention(self.queries[ids], self.heads, self.kv_heads, self.d, self.pool, self.table, b["offsets"], b["new_lengths"],
                        most, self.columns * self.page, b["out"], self.d ** -0.5)
        logits = torch.mm(b["out"].float(), self.head.float().t())
        k.token_logprobs(logits, tokens, b["logprob"], b["entropy"], b["rank"], b["top_ids"], b["top_logprobs"])
        self.lengths.copy_(b["new_lengths"])
        self.cursor.copy_(b["progress"][:1])
        return b["top_ids"][:, 0]


def serve(dtype, graph, stream=None):
    s = Serving(3, dtype, 7)
    g = torch.Generator().manual_seed(1)
    news = i32([5, 1, 30])
    tokens = torch.randint(0, s.vocab, (36,), generator=g).to(torch.int32).to(DEV)
    history = []
    prompt = s.buffers(36)
    picked = s.step(tokens, news, 30, prompt)
    history.append({k: v.clone() for k, v in prompt.items()})
    ends = prompt["offsets"][1:].long() - 1
    feed = picked[ends].clone()
    ones = i32([1, 1, 1])
    b = s.buffers(3)
    if graph:
        saved = [t.clone() for t in (s.lengths, s.cursor, s.table, *s.pool, feed)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            feed.copy_(s.step(feed, ones, 1, b))
        torch.cuda.current_stream().wait_stream(side)
        for t, old in zip((s.lengths, s.cursor, s.table, *s.pool, feed), saved):
            t.copy_(old)
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            feed.copy_(s.step(feed, ones, 1, b))
    for _ in range(9):
        if graph:
            captured.replay()
            (torch.ones(1000, device=DEV) * 2).sum().item()     # the program's own work in between
        else:
            feed.copy_(s.step(feed, ones, 1, b))
        history.append({k: v.clone() for k, v in b.items()})
    history.append({"table": s.table.clone(), "lengths": s.lengths.clone(), **{f"pool{i}": t.clone() for i, t in enumerate(s.pool)}})
    return history


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_run_of_them_together_eager_captured_and_on_two_streams(dtype):
    eager = serve(dtype, False)
    assert eager[-1]["lengths"].tolist() == [14, 10, 39] and eager[-2]["progress"].tolist() == [9, 0]
    replayed = serve(dtype, True)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    others = []
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            others.append(serve(dtype, False))
    torch.cuda.synchronize()
    for other in (replayed, *others):
        for a, b in zip(eager, other):
            for name in a:
                assert torch.equal(a[name], b[name]), name
    # and the last step against the plain implementations
    s = Serving(3, dtype, 7)
    pool = [eager[-1][f"pool{i}"] for i in range(4)]
    keys, values = plain.values_of_pages(pool)
    feed = eager[-3]["top_ids"][:, 0].long()
    last = eager[-2]
    want, spread, reach = plain.attention(s.queries[feed], 4, 2, 64, keys, values, eager[-1]["table"].tolist(), [0, 1, 2, 3],
                                          last["new_lengths"].tolist(), 8, 0.125, 0)
    bound = 2 * spread * (68 * 2.0 ** -24 * reach + 2.0 ** -21) + spread * (U[torch.bfloat16] + 2.0 ** -16) + U[dtype] * want.abs() + 1e-30
    assert bool(((last["out"].double().cpu() - want).abs() <= bound).all())


@pytest.mark.parametrize("tiny", ["A", "B"])
def test_scores_of_a_model(tiny_dirs, tiny):
    from plain.qwen3_plain import PlainModel

    from lockstep_amd import LLM, score

    folder = tiny_dirs[(tiny, "gen")]
    g = torch.Generator().manual_seed(13)
    tokens = torch.randint(0, 512, (41,), generator=g).tolist()
    logits = PlainModel(folder).logits(tokens)[:-1].double()
    want = plain.token_logprobs(logits, tokens[1:], 3)
    llm = LLM(folder, dtype="float32", num_pages=16)
    for found in (llm.score(tokens, top=3), score(llm.model, tokens, top=3, portion=7, page_size=8)):
        assert len(found) == 40
        # the float32 engine's logits agree with the plain ones to about 1e-6 of their spread
        spread = 1e-4 * float(logits.abs().max())
        assert max(abs(f["logprob"] - float(w)) for f, w in zip(found, want["logprob"])) < spread
        assert max(abs(f["entropy"] - float(w)) for f, w in zip(found, want["entropy"])) < spread
        assert [f["rank"] for f in found] == want["rank"]
        assert [[t for t, _ in f["top"]] for f in found] == want["top_ids"]
    assert llm.score(tokens[:1]) == [] and len(llm.score(tokens[:2])) == 1
    with pytest.raises(KernelError):
        llm.score(tokens, top=33)
