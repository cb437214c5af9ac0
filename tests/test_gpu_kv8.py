"""The kernels of a paged cache held in 8 bits against its definition in 64 bits.

What pages hold is compared for equality: scales are powers of two, a value times one
is exact, and one rounding to e4m3 is left. Attention: results are bf16, off by up to
2^-8 of themselves. Its scores are sums of D exact products in 32 bits, off by up to
2^-24 D of the sum of their sizes, and what the exponent is made of by 2^-22 more: a
weight is off by as much of itself, numerator and denominator. Weights of decoded rows
have two truncated bf16 terms, off by 2^-15 of themselves; those of prompts are
rounded to bf16, by e = 2^-8 / (1 + 2^-8) of themselves at most, and divided by the sum P of
the rounded ones: a result o is off by |sum (p' - p) (v - o)| / P, and with P at least
(1 - e) sum p = sum p / (1 + 2^-8) that is 2^-8 (sum p |v| / sum p + |o|) at most."""
import math

import pytest
import torch

from xllm_service_amd import ops

from kv8_oracle import Cache, attend, layout, same, slots_of

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rows(T, heads, dim, seed, big=1.0, beside=2):
    """bf16 rows in the middle of wider ones, on the CPU."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, (heads + beside) * dim, generator=g) * big)
    return x.to(torch.bfloat16)


def part(x, heads, dim):
    """Their heads, on the GPU, as a view of the wider rows."""
    return x.to(DEV)[:, dim:(1 + heads) * dim].unflatten(1, (heads, dim))


def ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


def filled(lens, heads, dim, seed, spare=3, big=1.0, width=None):
    """A cache of these sequences, written by the reference on the CPU, every other
    byte of it NaN and other scales 2^60: (cache on the GPU, oracle, table)."""
    table, pages = layout(lens, spare, seed, width)
    cache = ops.kv8_cache(pages, heads, dim)
    slots = slots_of(table, [0] * len(lens), [max(n, 0) for n in lens])
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(len(slots), heads, dim, generator=g) * big
            for _ in range(2))
    k = k.to(torch.bfloat16)
    v = (v * torch.exp2(torch.randn(heads, 1, generator=g))).to(torch.bfloat16)
    ops.reshape_and_cache_kv8(k, v, *cache, torch.tensor(slots).long())
    want = Cache(pages, heads, dim).load(*cache)
    live = torch.zeros(pages * 16, dtype=torch.bool)
    live[slots] = True
    live = live.view(pages, 16)
    kb, vb = (c.view(torch.uint8) for c in cache[:2])
    kb.transpose(2, 3).transpose(1, 2)[~live] = 0x7f
    vb.permute(0, 3, 1, 2)[~live] = 0x7f
    cache[2][~live.any(1)] = 2.0 ** 60
    return tuple(c.to(DEV) for c in cache), want, table


def close(got, q, want, table, cu, total, scale, weights):
    k, v = want.values(0), want.values(1)
    ref, big, most = attend(q, k, v, table, cu, total, scale)
    off = 2.0 ** -24 * q.shape[2] * most + 2.0 ** -22 * most.clamp(min=1.0)
    bound = (2.0 ** -8 + weights) * ref.abs() + (weights + 2 * off) * big + 1e-30
    diff = (got.cpu().double() - ref).abs()
    assert not diff.isnan().any()
    assert (diff <= bound).all(), float((diff / bound).max())


# ---- writing -----------------------------------------------------------------
@pytest.mark.parametrize("heads,dim", [(1, 64), (3, 128), (8, 128), (12, 64)])
def test_write(heads, dim):
    pages = 7
    cache = tuple(c.to(DEV) for c in ops.kv8_cache(pages, heads, dim))
    want = Cache(pages, heads, dim)
    steps = [list(range(16, 16 + 21)), [37], [38, 39], [40, -1, 41, 0],
             [1, 10 ** 9, -7, 112], [2, 2], [17, 17, 16, 19, 17],
             list(range(48, 64)) + list(range(95, 79, -1)),
             [9, 60, 100, 90, 30]]
    for n, slots in enumerate(steps):
        k, v = (rows(len(slots), heads, dim, 2 * n + i, 2.5 ** (n % 5 - 2))
                for i in range(2))
        gk, gv = part(k, heads, dim), part(v, heads, dim)
        ops.reshape_and_cache_kv8(gk, gv, *cache, ints(slots, torch.long))
        want.write(gk, gv, slots)
        got = Cache(pages, heads, dim).load(*cache)
        for i in range(2):
            assert same(got.x[i], want.x[i]), (n, i)
        assert same(got.scale, want.scale), n


def test_write_again_over_far_scales():
    """A page that goes on: from nothing, from NaN bytes, past what one power of
    two of fp32 spans, without growing, and with zeros."""
    cache = tuple(c.to(DEV) for c in ops.kv8_cache(2, 1, 64))
    want = Cache(2, 1, 64)
    for slot, big in ((3, 0.0), (4, 1e-38), (5, 1e-30), (6, 3e38), (7, 1.0),
                      (8, math.inf), (9, math.nan), (10, 0.0), (16, math.inf),
                      (17, -0.0)):
        x = torch.full((1, 1, 64), big).to(torch.bfloat16)
        x[0, 0, ::3] *= -0.5
        x = x.to(DEV)
        ops.reshape_and_cache_kv8(x, x, *cache, ints([slot], torch.long))
        want.write(x, x, [slot])
        got = Cache(2, 1, 64).load(*cache)
        for i in range(2):
            assert same(got.x[i], want.x[i]), slot
        assert same(got.scale, want.scale), slot


@pytest.mark.parametrize("offset", [0, 1, 8])
def test_write_rows_at_any_address(offset):
    """Keys are read by 16 B: rows that are not aligned are copied."""
    cache = tuple(c.to(DEV) for c in ops.kv8_cache(3, 2, 128))
    want = Cache(3, 2, 128)
    g = torch.Generator().manual_seed(3)
    x = torch.randn(20, 2 * 128 + 9, generator=g).to(torch.bfloat16).to(DEV)
    k = x[:, offset:offset + 256].unflatten(1, (2, 128))
    v = x[:, 9 - offset:265 - offset].unflatten(1, (2, 128))
    slots = list(range(5, 25))
    ops.reshape_and_cache_kv8(k, v, *cache, ints(slots, torch.long))
    want.write(k, v, slots)
    got = Cache(3, 2, 128).load(*cache)
    assert all(same(got.x[i], want.x[i]) for i in range(2))


# a wave looks over one token, two, four or eight: from 375, 750 and 1500 tokens of 8
# heads on, 250, 500 and 1000 of 12
@pytest.mark.parametrize("heads,dim,tokens", [
    (8, 128, 300), (8, 128, 400), (8, 128, 800), (8, 128, 1600), (8, 64, 1600),
    (12, 64, 260), (12, 64, 600), (12, 64, 1100)])
def test_write_by_windows(heads, dim, tokens):
    """Uneven sequences that begin anywhere in a page: several runs to a window, runs
    that begin in one and end in another, skipped tokens in and between them."""
    g = torch.Generator().manual_seed(tokens + heads)
    old, new = [], []
    while sum(new) < tokens:
        old.append(int(torch.randint(0, 40, (1,), generator=g)))
        long = torch.rand(1, generator=g) < 0.2
        new.append(int(torch.randint(1, 120 if long else 9, (1,), generator=g)))
    lens = [a + b for a, b in zip(old, new)]
    table, pages = layout(lens, 3, tokens)
    cache = tuple(c.to(DEV) for c in ops.kv8_cache(pages, heads, dim))
    want = Cache(pages, heads, dim)
    for n, (a, b) in enumerate([([0] * len(old), old), (old, lens)]):
        slots = []
        for s in slots_of(table, a, b):
            skip = torch.rand(2, generator=g)
            if skip[0] < 0.08:
                slots += [-1] * int(1 + 5 * skip[1])
            slots.append(s)
        k, v = (rows(len(slots), heads, dim, 2 * n + i, 3.0 ** n) for i in range(2))
        gk, gv = part(k, heads, dim), part(v, heads, dim)
        ops.reshape_and_cache_kv8(gk, gv, *cache, ints(slots, torch.long))
        want.write(gk, gv, slots)
        got = Cache(pages, heads, dim).load(*cache)
        assert same(got.scale, want.scale), n
        for i in range(2):
            assert same(got.x[i], want.x[i]), (n, i)


@pytest.mark.parametrize("heads,dim", [(3, 128), (2, 64)])
def test_write_twice_to_a_slot(heads, dim):
    """The later one stays; the scale holds all of a page's new tokens, those that
    do not stay among them, as it would after one call for each."""
    cache = tuple(c.to(DEV) for c in ops.kv8_cache(7, heads, dim))
    want = Cache(7, heads, dim)
    for n, (slots, big) in enumerate([
            ([2, 2], [300.0, 1.0]),
            ([5, 3, 5, 4, 3], [1.0, 9.0, 2000.0, 1.0, 1.0]),
            ([17, 17, 16, 19, 17], [50.0, 700.0, 1.0, 1.0, 1.0]),
            ([32, -1, 32, 33, 32], [1.0, 1e5, 77.0, 1.0, 1.0]),
            ([40, 40], [math.inf, 1.0]), ([41, 41, 41], [math.nan, 6e4, 1.0]),
            # more of them than a wave looks over at once
            ([64] + [65, 66] * 50 + [67], [1.0, 4000.0] + [1.0] * 100),
            ([70] * 90 + [71], [1.0] * 30 + [1e6] + [1.0] * 60),
            (list(range(80, 96)) * 5, [1.0] * 7 + [500.0] + [1.0] * 72)]):
        k, v = (rows(len(slots), heads, dim, 2 * n + i) for i in range(2))
        by = torch.tensor(big)[:, None]
        gk, gv = (part((x.float() * by).to(torch.bfloat16), heads, dim)
                  for x in (k, v))
        ops.reshape_and_cache_kv8(gk, gv, *cache, ints(slots, torch.long))
        want.write(gk, gv, slots)
        got = Cache(7, heads, dim).load(*cache)
        assert same(got.scale, want.scale), n
        for i in range(2):
            assert same(got.x[i], want.x[i]), (n, i)


@pytest.mark.parametrize("room", [50, 63, 64, 65, 1023, 1100, 8192, 20000])
def test_write_of_padded_rows(room):
    """Few tokens anywhere among rows without a slot: in front, behind, and a page's
    first and last ones far apart."""
    heads, dim = 1, 64
    k, v = (part(rows(room, heads, dim, i), heads, dim) for i in range(2))
    page = [*range(16, 30)]
    for where in (list(range(14)), list(range(room - 14, room)),
                  [0, *range(room - 13, room)], [*range(13), room - 1],
                  [room // 14 * i for i in range(14)], [*range(20, 33), room - 9]):
        cache = tuple(c.to(DEV) for c in ops.kv8_cache(3, heads, dim))
        want = Cache(3, heads, dim)
        slots = [-1] * room
        for at, s in zip(where, page):
            slots[at] = s
        if where[0] > 0:
            slots[where[0] - 1] = 40         # another page's, right before it
        if where[-1] < room - 3:
            slots[room - 2] = 5
        ops.reshape_and_cache_kv8(k, v, *cache, ints(slots, torch.long))
        want.write(k, v, slots)
        got = Cache(3, heads, dim).load(*cache)
        assert same(got.scale, want.scale), where
        assert all(same(got.x[i], want.x[i]) for i in range(2)), where


BIG = [3.3895313892515355e38, 3.3e38, 3.28e38, -3.3895313892515355e38, 3e38, 2.9e38,
       1e38, 1.0]


@pytest.mark.parametrize("heads,dim", [(3, 128), (2, 64)])
def test_the_largest_values_stay_finite(heads, dim):
    """448 times the largest scale passes fp32 and bf16: what would round to more
    than 240 of it is 240, within half a step of e4m3 of what it was."""
    cache = tuple(c.to(DEV) for c in ops.kv8_cache(4, heads, dim))
    plain = ops.kv8_cache(4, heads, dim)
    g = torch.Generator().manual_seed(1)
    for slots in (list(range(16, 32)), [0], [1], [2, 3]):
        x = torch.tensor(BIG)[torch.randint(len(BIG), (len(slots), heads, dim),
                                            generator=g)].to(torch.bfloat16)
        at = torch.tensor(slots)
        ops.reshape_and_cache_kv8(x, x, *plain, at)
        ops.reshape_and_cache_kv8(x.to(DEV), x.to(DEV), *cache, at.to(DEV))
        for a, b in zip(cache, plain):
            assert torch.equal(a.view(torch.uint8).cpu(), b.view(torch.uint8))
        got = Cache(4, heads, dim).load(*cache)
        for i in range(2):
            y = got.values(i)[at // 16, :, at % 16]
            assert (y.abs() < 2.0 ** 128 - 2.0 ** 119).all()     # bf16's largest
            # (below 2^-6 of the scale a step is 2^-9 of it)
            least = 2.0 ** -10 * got.scale[at // 16, :, i, None]
            assert ((y - x.double()).abs()
                    <= 2.0 ** -4 * x.double().abs() + least).all()


# ---- tables ------------------------------------------------------------------
@pytest.mark.parametrize("seqs,most_old,most_new,short", [
    (1, 0, 1, 0), (1, 100, 3, 0), (3, 40, 40, 0), (256, 300, 2, 0),
    (257, 300, 1, 0), (700, 90, 60, 0), (64, 2000, 1500, 0), (50, 60, 60, 9)])
def test_tables_from_lengths(seqs, most_old, most_new, short):
    g = torch.Generator().manual_seed(seqs)
    old = torch.randint(0, most_old + 1, (seqs,), generator=g).int()
    new = old + torch.randint(-2, most_new + 1, (seqs,), generator=g).int()
    width = (int(new.max()) + 47) // 16 - short // 4
    # rows of a wider table
    table = torch.randint(0, 10 ** 6, (seqs, width + 3), generator=g).int()
    pages = int(((new.clamp(min=0) + 15) // 16).sum())
    free = torch.randperm(pages + 5, generator=g).int()[short * 9:]
    room = int((new - old).clamp(min=0).sum()) + 7 - 11 * short
    there = table.to(DEV)
    got = ops.extend_block_tables(there[:, :width], old.to(DEV), new.to(DEV),
                                  free.to(DEV), room)
    want = ops.extend_block_tables(table[:, :width], old, new, free, room)
    assert torch.equal(there.cpu(), table)
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)


# sums of what is no length of a sequence would pass 32 bits
@pytest.mark.parametrize("seqs", [3, 256, 600, 1500])
@pytest.mark.parametrize("room", [0, 100])
def test_tables_from_lengths_of_any_size(seqs, room):
    most = 2 ** 31 - 1
    old = torch.zeros(seqs, dtype=torch.int32)
    new = torch.full_like(old, most)
    old[seqs // 2:], new[-1] = most, -most - 1
    old[:1], new[:1] = 3, 40
    free = torch.arange(7, dtype=torch.int32) * 3
    table = torch.arange(seqs * 3, dtype=torch.int32).reshape(seqs, 3)
    there = table.to(DEV)
    got = ops.extend_block_tables(there, old.to(DEV), new.to(DEV), free.to(DEV), room)
    want = ops.extend_block_tables(table, old, new, free, room)
    assert torch.equal(there.cpu(), table)
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)


# ---- attention ---------------------------------------------------------------
SHAPES = [(2, 4, 128), (1, 7, 128), (3, 1, 64), (2, 16, 128), (2, 12, 64),
          (1, 1, 128)]


@pytest.mark.parametrize("heads,per,dim", SHAPES)
@pytest.mark.parametrize("lens", [
    [1], [0, 1, 15, 16, 17, 31, 32, 33, 47, 48, 49, 64, 65], [300, 0, 129],
    [1500], [700, 3000, 5, 1029]], ids=lambda x: f"{len(x)}x{max(x)}")
def test_decode(heads, per, dim, lens):
    cache, want, table = filled(lens, heads, dim, len(lens))
    H, S = heads * per, len(lens)
    q = part(rows(S, H, dim, 5), H, dim)
    out = torch.full((S, H + 1, dim), 7.0, dtype=torch.bfloat16, device=DEV)
    ops.paged_attn_decode_kv8(q, *cache, table.to(DEV), ints(lens),
                              dim ** -0.5, out=out[:, :H])
    close(out[:, :H], q, want, table, list(range(S + 1)), lens, dim ** -0.5,
          2.0 ** -15)
    assert (out[:, H] == 7.0).all()
    plain = ops.paged_attn_decode_kv8(q, *cache, table.to(DEV), ints(lens),
                                      dim ** -0.5)
    assert torch.equal(plain, out[:, :H])


@pytest.mark.parametrize("seqs", [40, 90, 140])
def test_decode_many(seqs):
    """Sequences that fill the card once and more, lengths far apart."""
    lens = [(37 * i) % 601 for i in range(seqs)]
    cache, want, table = filled(lens, 2, 128, seqs)
    q = part(rows(seqs, 8, 128, 5), 8, 128)
    got = ops.paged_attn_decode_kv8(q, *cache, table.to(DEV), ints(lens), 0.09)
    close(got, q, want, table, list(range(seqs + 1)), lens, 0.09, 2.0 ** -15)


@pytest.mark.parametrize("heads,per,dim", SHAPES)
@pytest.mark.parametrize("new,old", [
    ([1], [0]), ([3, 1, 16, 0, 33], [0, 31, 16, 9, 0]), ([64, 65], [63, 0]),
    ([130], [0]), ([200], [1100]), ([70, 1, 300], [1000, 1200, 0]),
    ([17] * 70, [5] * 70)], ids=lambda x: f"{len(x)}x{max(x)}")
def test_prefill(heads, per, dim, new, old):
    lens = [n + o for n, o in zip(new, old)]
    cache, want, table = filled(lens, heads, dim, len(lens))
    H, T = heads * per, sum(new)
    q = part(rows(T + 3, H, dim, 6), H, dim)
    cu = [sum(new[:i]) for i in range(len(new) + 1)]
    out = torch.full((T + 3, H + 1, dim), 7.0, dtype=torch.bfloat16, device=DEV)
    ops.paged_attn_prefill_kv8(q, *cache, table.to(DEV), ints(cu), ints(lens),
                               dim ** -0.5, out=out[:, :H])
    close(out[:T, :H], q[:T], want, table, cu, lens, dim ** -0.5, 2.0 ** -8)
    assert (out[T:] == 7.0).all() and (out[:, H] == 7.0).all()


@pytest.mark.parametrize("heads,per,dim", [(8, 4, 128), (4, 7, 128), (12, 1, 64)])
@pytest.mark.parametrize("new,old", [
    ([1300], [0]), ([600, 900, 40], [700, 0, 2000]), ([400] * 5, [100] * 5)],
    ids=lambda x: f"{len(x)}x{max(x)}")
def test_prefill_of_full_steps(heads, per, dim, new, old):
    lens = [n + o for n, o in zip(new, old)]
    cache, want, table = filled(lens, heads, dim, len(lens), big=2.0)
    H, T = heads * per, sum(new)
    q = part(rows(T, H, dim, 6), H, dim)
    cu = [sum(new[:i]) for i in range(len(new) + 1)]
    got = ops.paged_attn_prefill_kv8(q, *cache, table.to(DEV), ints(cu),
                                     ints(lens), dim ** -0.5)
    close(got, q, want, table, cu, lens, dim ** -0.5, 2.0 ** -8)


# 440 to 512 workgroups of 256 rows, and fewer behind longer contexts
LONG = [(24, 8, [600], [0]), (21, 8, [300, 400], [100, 1700]),
        (28, 7, [513], [1600]), (64, 3, [512], [0]),
        (32, 4, [300, 270], [1900, 30]), (65, 1, [900], [200])]


@pytest.mark.parametrize("heads,per,new,old", LONG)
def test_prefill_of_whole_turns(heads, per, new, old):
    lens = [n + o for n, o in zip(new, old)]
    cache, want, table = filled(lens, heads, 128, len(lens), width=140)
    H, T = heads * per, sum(new)
    q = part(rows(T + 3, H, 128, 6), H, 128)
    cu = [sum(new[:i]) for i in range(len(new) + 1)]
    out = torch.full((T + 3, H, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    ops.paged_attn_prefill_kv8(q, *cache, table.to(DEV), ints(cu), ints(lens),
                               0.09, out=out)
    close(out[:T], q[:T], want, table, cu, lens, 0.09, 2.0 ** -8)
    assert (out[T:] == 7.0).all()
    again = ops.paged_attn_prefill_kv8(q, *cache, table.to(DEV), ints(cu),
                                       ints(lens), 0.09)
    assert torch.equal(again[:T], out[:T])


@pytest.mark.parametrize("total", [2300, 2240, 500, 300, 0, -9])
def test_prefill_of_whole_turns_and_odd_lengths(total):
    """A sequence longer than its table, shorter than its chunk, without keys."""
    heads, per, T = 24, 8, 600
    cache, want, table = filled([2240], heads, 128, 3, width=140)
    q = part(rows(T, heads * per, 128, 6), heads * per, 128)
    got = ops.paged_attn_prefill_kv8(q, *cache, table.to(DEV), ints([0, T]),
                                     ints([total]), 0.09)
    close(got, q, want, table, [0, T], [total], 0.09, 2.0 ** -8)
    if total < T:
        assert (got[:T - max(total, 0)] == 0).all()


@pytest.mark.parametrize("token", [0, 1, 200, 255, 511])
def test_prefill_of_whole_turns_and_values_that_are_not_finite(token):
    heads, per, T, old = 64, 3, 512, 17
    cache, _, table = filled([T + old], heads, 128, 3, width=140)
    q = part(rows(T, heads * per, 128, 6), heads * per, 128)
    at = token + old
    cache[1].view(torch.uint8)[table[0, at // 16], :, 77, at % 16] = 0xff
    got = ops.paged_attn_prefill_kv8(q, *cache, table.to(DEV), ints([0, T]),
                                     ints([T + old]), 0.09)
    assert got[token:, :, 77].isnan().all()
    got[token:, :, 77] = 0.0
    assert not got.isnan().any()


@pytest.mark.parametrize("heads,per,dim", [(2, 4, 128), (3, 1, 64), (1, 7, 128)])
@pytest.mark.parametrize("width", [10, 400])
@pytest.mark.parametrize("token", [0, 20, 63, 64, 130])
def test_values_that_are_not_finite_anywhere(token, heads, per, dim, width):
    T, old = 150, 5
    cache, _, table = filled([T + old], heads, dim, 3, width=width)
    q = part(rows(T, heads * per, dim, 6), heads * per, dim)
    at = token + old
    cache[1].view(torch.uint8)[table[0, at // 16], :, 33, at % 16] = 0xff
    got = ops.paged_attn_prefill_kv8(q, *cache, table.to(DEV), ints([0, T]),
                                     ints([T + old]), 0.09)
    assert got[token:, :, 33].isnan().all()
    got[token:, :, 33] = 0.0
    assert not got.isnan().any()



UNUSED = [([40, 3], [700, 90], 2, 4, 128, 400), ([300, 7], [20, 0], 16, 4, 128, 21),
          ([70] * 14, [3] * 14, 12, 3, 64, 6), ([600], [0], 24, 8, 128, 140),
          ([300, 410], [100, 1700], 21, 8, 128, 140), ([100], [5], 2, 4, 128, 12),
          ([150], [900], 2, 4, 64, 300), ([1] * 5, [0, 3, 40, 900, 31], 2, 12, 128, 60),
          ([1] * 5, [0, 3, 40, 900, 31], 2, 4, 64, 60)]


@pytest.mark.parametrize("what", [math.nan, math.inf])
@pytest.mark.parametrize("new,old,heads,per,dim,width", UNUSED)
def test_scales_of_pages_that_are_not_used(new, old, heads, per, dim, width, what):
    """Memory that nobody has cleared: page 0, which stands for what tables do not
    have, and other pages of no sequence have scales that are not finite."""
    lens = [n + o for n, o in zip(new, old)]
    spare = sum(-(-n // 16) for n in lens)
    for seed in range(99):
        table, _ = layout(lens, spare, seed)
        live = {int(p) for i, n in enumerate(lens) for p in table[i, :-(-n // 16)]}
        if 0 not in live:
            break
    cache, want, table = filled(lens, heads, dim, seed, spare=spare, width=width)
    cache[2][cache[2] == 2.0 ** 60] = what
    assert not cache[2][0].isfinite().any()
    for x in want.x:                             # (the oracle reads no such page)
        x[[p for p in range(len(x)) if p not in live]] = 0.0
    H, T = heads * per, sum(new)
    q = part(rows(T, H, dim, 6), H, dim)
    cu = [sum(new[:i]) for i in range(len(new) + 1)]
    got = ops.paged_attn_prefill_kv8(q, *cache, table.to(DEV), ints(cu), ints(lens),
                                     0.09)
    close(got, q, want, table, cu, lens, 0.09, 2.0 ** -8)
    if max(new) == 1:
        got = ops.paged_attn_decode_kv8(q, *cache, table.to(DEV), ints(lens), 0.09)
        close(got, q, want, table, cu, lens, 0.09, 2.0 ** -15)


@pytest.mark.parametrize("heads,per,dim,T,old,width", [
    (64, 3, 128, 512, 0, 140), (2, 4, 128, 150, 5, 10), (2, 4, 128, 150, 5, 400),
    (16, 4, 128, 600, 8, 38)])
def test_the_largest_values_reach_rows_that_see_them(heads, per, dim, T, old, width):
    """And no others, to which 0 times an infinity would bring a NaN."""
    total = T + old
    table, pages = layout([total], 3, 1, width)
    cache = ops.kv8_cache(pages, heads, dim, DEV)
    k, v = rows(total, heads, dim, 2), rows(total, heads, dim, 3)
    token = T - 70
    gv = part(v, heads, dim).clone()
    gv[token + old:] = 3.3895313892515355e38
    ops.reshape_and_cache_kv8(part(k, heads, dim), gv, *cache,
                              ints(slots_of(table, [0], [total]), torch.long))
    q = part(rows(T, heads * per, dim, 6), heads * per, dim)
    got = ops.paged_attn_prefill_kv8(q, *cache, table.to(DEV), ints([0, T]),
                                     ints([total]), 0.09)
    assert got[:token].isfinite().all()
    assert got[:token].abs().max() < 8.0


@pytest.mark.parametrize("heads,per,dim", [(2, 4, 128), (3, 1, 64), (1, 7, 128)])
def test_parts_without_keys_beside_values_that_are_not_finite(heads, per, dim):
    """Row tiles that see fewer tiles of keys than they have parts, by turns with
    calls whose every value is a NaN, which leave LDS full of what they noted."""
    T, width = 260, 400
    cache, want, table = filled([T], heads, dim, 3, width=width)
    bad = [c.clone() for c in cache]
    bad[1].view(torch.uint8).fill_(0x7f)
    q = part(rows(T, heads * per, dim, 6), heads * per, dim)
    for _ in range(4):
        got = ops.paged_attn_prefill_kv8(q, *bad, table.to(DEV), ints([0, T]),
                                         ints([T]), 0.09)
        assert got.isnan().all()
        got = ops.paged_attn_prefill_kv8(q, *cache, table.to(DEV), ints([0, T]),
                                         ints([T]), 0.09)
        close(got, q, want, table, [0, T], [T], 0.09, 2.0 ** -8)
        got = ops.paged_attn_prefill_kv8(q, *bad, table.to(DEV), ints([0, T]),
                                         ints([40]), 0.09)
        assert (got[:T - 40] == 0).all() and got[T - 40:].isnan().all()

# few rows over wide tables, whose keys are split over workgroups, and many over few keys
ROWS = [(2, 4, 128, [9], [1200], 300), (2, 4, 128, [40, 3], [700, 90], 400),
        (1, 8, 64, [30], [900], 260), (16, 4, 128, [80] * 9, [0] * 9, 8),
        (16, 4, 128, [300, 7], [20, 0], 21), (12, 3, 64, [70] * 14, [3] * 14, 6),
        (4, 4, 128, [600], [300], 600), (2, 5, 128, [11, 300, 1], [0, 5, 900], 700)]


@pytest.mark.parametrize("heads,per,dim,new,old,width", ROWS)
def test_prefill_by_tables(heads, per, dim, new, old, width):
    lens = [n + o for n, o in zip(new, old)]
    cache, want, table = filled(lens, heads, dim, len(lens), width=width)
    H, T = heads * per, sum(new)
    q = part(rows(T + 3, H, dim, 6), H, dim)
    cu = [sum(new[:i]) for i in range(len(new) + 1)]
    out = torch.full((T + 3, H, dim), 7.0, dtype=torch.bfloat16, device=DEV)
    ops.paged_attn_prefill_kv8(q, *cache, table.to(DEV), ints(cu), ints(lens),
                               dim ** -0.5, out=out)
    close(out[:T], q[:T], want, table, cu, lens, dim ** -0.5, 2.0 ** -8)
    assert (out[T:] == 7.0).all()


@pytest.mark.parametrize("heads,per,dim,width", [(2, 4, 128, 12), (3, 1, 64, 12),
                                                 (2, 4, 128, 400), (3, 1, 64, 400)])
@pytest.mark.parametrize("total", [400, 150, 60, 0, -9])
def test_prefill_and_odd_lengths(total, heads, per, dim, width):
    """A sequence longer than its table, shorter than its chunk, without keys."""
    T = 100
    cache, want, table = filled([192], heads, dim, 3, width=width)
    q = part(rows(T, heads * per, dim, 6), heads * per, dim)
    if width > 12:
        table = table[:, :12].repeat(1, -(-width // 12))[:, :width]
    got = ops.paged_attn_prefill_kv8(q, *cache, table.contiguous().to(DEV),
                                     ints([0, T]), ints([total]), 0.09)
    close(got, q, want, table, [0, T], [total], 0.09, 2.0 ** -8)



FAR, LOW = 2 ** 31 - 1, -2 ** 31


# a sequence's length need not be what its table holds: row tiles sorted and as they
# are, keys split over workgroups of one and of several sequences, whole turns, few rows
@pytest.mark.parametrize("heads,per,dim,new,lens,width", [
    (16, 4, 128, [80] * 9, [FAR, -9, 80, 2 ** 30, 128, LOW, 3 * 10 ** 8, 100, 0], 8),
    (24, 1, 128, [300] * 4, [FAR, -9, 300, 200], 19),
    (16, 1, 64, [300] * 9, [LOW, FAR, 304, 2 ** 30, -1, 5, 300, 0, FAR - 1], 19),
    (2, 4, 128, [40, 3], [FAR, 2 ** 30], 400),
    (1, 8, 128, [16] * 15 + [1600], [40000] * 15 + [2 ** 30], 700),
    (1, 8, 128, [16] * 15 + [1600], [FAR, LOW, 300] * 5 + [FAR], 700),
    (2, 4, 128, [9], [FAR], 300), (2, 4, 128, [9], [LOW], 300),
    (24, 8, 128, [600], [FAR], 140), (24, 8, 128, [600], [LOW], 140),
    (21, 8, 128, [300, 400], [FAR, -9], 140),
    (21, 8, 128, [300, 400], [LOW, 3 * 10 ** 8], 140),
    (2, 4, 128, [100], [FAR], 12), (2, 4, 128, [100, 7], [LOW, FAR], 12)])
def test_prefill_and_lengths_of_any_size(heads, per, dim, new, lens, width):
    cache, want, table = filled([192] * len(new), heads, dim, 3)
    table = table.repeat(1, -(-width // 12))[:, :width].contiguous()
    T = sum(new)
    q = part(rows(T + 3, heads * per, dim, 6), heads * per, dim)
    cu = [sum(new[:i]) for i in range(len(new) + 1)]
    out = torch.full((T + 3, heads * per, dim), 7.0, dtype=torch.bfloat16,
                     device=DEV)
    ops.paged_attn_prefill_kv8(q, *cache, table.to(DEV), ints(cu), ints(lens), 0.09,
                               out=out)
    close(out[:T], q[:T], want, table, cu, lens, 0.09, 2.0 ** -8)
    assert (out[T:] == 7.0).all()


@pytest.mark.parametrize("heads,per,dim", [(2, 4, 128), (1, 12, 64)])
def test_decode_and_lengths_of_any_size(heads, per, dim):
    lens = [FAR, LOW, -1, 2 ** 30, 33]
    cache, want, table = filled([192] * 5, heads, dim, 3)
    q = part(rows(5, heads * per, dim, 6), heads * per, dim)
    got = ops.paged_attn_decode_kv8(q, *cache, table.to(DEV), ints(lens), 0.09)
    close(got, q, want, table, list(range(6)), lens, 0.09, 2.0 ** -15)

def test_rows_without_keys():
    """Lengths of zero and below, chunks longer than their sequence, tables without
    columns."""
    cache, want, table = filled([20, 30], 2, 128, 1)
    q = part(rows(12, 4, 128, 2), 4, 128)
    tab = table.to(DEV)
    cu, total = [0, 5, 12], [2, -3]
    got = ops.paged_attn_prefill_kv8(q, *cache, tab, ints(cu), ints(total), 0.1)
    assert (got[:3] == 0).all() and (got[5:] == 0).all()
    close(got, q, want, table, cu, total, 0.1, 2.0 ** -8)
    got = ops.paged_attn_decode_kv8(q[:2], *cache, tab, ints([0, -100]), 0.1)
    assert (got == 0).all()
    none = tab[:, :0].contiguous()
    got = ops.paged_attn_decode_kv8(q[:2], *cache, none, ints([5, 9]), 0.1)
    assert (got == 0).all()
    got = ops.paged_attn_prefill_kv8(q, *cache, none, ints(cu), ints([5, 9]), 0.1)
    assert (got == 0).all()


def uneven(cache, want, seed):
    """Pages' scales far apart."""
    g = torch.Generator().manual_seed(seed)
    by = torch.exp2(torch.randint(-3, 4, want.scale.shape, generator=g).double())
    by[..., 0] = by[..., 0].clamp(max=1.0)
    cache[2].mul_(by.float().to(DEV))
    want.scale *= by


def close_rows(got, q, want, table, old, new, scale, weights, at):
    """Rows at[i] of every sequence, as those of a chunk that ends with them."""
    start = 0
    for i, (o, n) in enumerate(zip(old, new)):
        for a, b in at:
            a, b = min(a % n if a < 0 else a, n), min(b, n)
            if a < b:
                close(got[start + a:start + b], q[start + a:start + b], want,
                      table[i:i + 1], [0, b - a], [o + b], scale, weights)
        start += n


# Pages' ids and scales are looked up for 16, 32 or 64 tiles at a time: sequences that
# need a second and a third look, unsplit, in parts and by two groups of waves
@pytest.mark.parametrize("heads,per,dim", [(8, 4, 128), (8, 8, 64), (8, 12, 64),
                                           (8, 16, 128), (1, 4, 128), (1, 12, 128)])
@pytest.mark.parametrize("scale", [0.02, 0.3])
def test_decode_and_second_looks_at_tables(heads, per, dim, scale):
    lens = [13 * i % 41 for i in range(100)]
    lens[37], lens[71] = 9000, 4500
    if heads == 1:                           # in parts of over 16 tiles a wave
        lens = [90000, 3]
    cache, want, table = filled(lens, heads, dim, 2)
    uneven(cache, want, 1)
    S = len(lens)
    q = part(rows(S, heads * per, dim, 5), heads * per, dim)
    got = ops.paged_attn_decode_kv8(q, *cache, table.to(DEV), ints(lens), scale)
    close(got, q, want, table, list(range(S + 1)), lens, scale, 2.0 ** -15)


FEW = [25] * 60
SECOND = [(8, 4, 128, [200, 100], [4300, 10]), (8, 4, 64, [200, 100], [4300, 10]),
          (8, 4, 128, FEW, [4400] + [3] * 59), (12, 1, 64, [1200] * 3 + [150],
                                                [0, 0, 0, 8400]),
          (8, 4, 128, [500], [17500]), (24, 8, 128, [600], [4100]),
          (21, 8, 128, [300, 400], [100, 8300])]


@pytest.mark.parametrize("heads,per,dim,new,old", SECOND)
@pytest.mark.parametrize("scale", [0.02, 0.3])
def test_prefill_and_second_looks_at_tables(heads, per, dim, new, old, scale):
    lens = [a + b for a, b in zip(new, old)]
    cache, want, table = filled(lens, heads, dim, 2)
    uneven(cache, want, 1)
    T = sum(new)
    q = part(rows(T, heads * per, dim, 6), heads * per, dim)
    cu = [sum(new[:i]) for i in range(len(new) + 1)]
    got = ops.paged_attn_prefill_kv8(q, *cache, table.to(DEV), ints(cu), ints(lens),
                                     scale)
    close_rows(got, q, want, table, old, new, scale, 2.0 ** -8,
               [(0, 9), (127, 133), (-7, 10 ** 6)])


# many heads to one of the cache's, many sequences of few tokens, rows in front of the
# first sequence and more behind the last one than there are in all
OTHER = [(1, 32, 128, [40, 3], [500, 0], 60, 0, 3), (1, 71, 64, [33], [70], 300, 2, 1),
         (2, 24, 128, [300], [90], 30, 0, 0), (1, 100, 128, [700], [60], 140, 0, 5),
         (2, 4, 128, [i % 4 for i in range(300)], [7 * i % 101 for i in range(300)],
          300, 1, 9),
         (3, 1, 64, [i % 4 for i in range(300)], [7 * i % 101 for i in range(300)], 7,
          0, 2),
         (2, 4, 128, [20], [30], 4, 5, 700), (2, 4, 128, [20, 1], [1000, 30], 200, 5,
                                              700),
         (24, 8, 128, [600], [0], 140, 9, 800)]


@pytest.mark.parametrize("heads,per,dim,new,old,width,front,behind", OTHER)
def test_prefill_of_other_batches(heads, per, dim, new, old, width, front, behind):
    lens = [n + o for n, o in zip(new, old)]
    cache, want, table = filled(lens, heads, dim, 5, width=width)
    H, T = heads * per, front + sum(new)
    q = part(rows(T + behind, H, dim, 6), H, dim)
    cu = [front + sum(new[:i]) for i in range(len(new) + 1)]
    out = torch.full((T + behind, H, dim), 7.0, dtype=torch.bfloat16, device=DEV)
    ops.paged_attn_prefill_kv8(q, *cache, table.to(DEV), ints(cu), ints(lens),
                               dim ** -0.5, out=out)
    close(out[front:T], q[front:T], want, table, [c - front for c in cu], lens,
          dim ** -0.5, 2.0 ** -8)
    assert (out[:front] == 7.0).all() and (out[T:] == 7.0).all()


def test_entries_of_no_page_are_page_0():
    """Whatever it holds, and only where keys are seen there."""
    lens = [40, 25, 20]
    cache, want, table = filled(lens, 2, 64, 4)
    wild, zero = table.clone(), table.clone()
    wild[0, 1], zero[0, 1] = 10 ** 6, 0
    wild[1, 2], wild[2, 2] = -5, cache[2].shape[0]       # behind 32 keys
    cache[1].view(torch.uint8)[0] = 0x7f
    q = part(rows(9, 4, 64, 2), 4, 64)
    cu = ints([0, 4, 6, 9])
    for f, args in ((ops.paged_attn_decode_kv8, (q[:3],)),
                    (ops.paged_attn_prefill_kv8, (q,))):
        got = [f(*args, *cache, t.to(DEV), *((cu,) if len(args[0]) == 9 else ()),
                 ints(lens), 0.1) for t in (wild, zero)]
        bad = got[0].isnan()
        assert torch.equal(bad, got[1].isnan())
        assert torch.equal(got[0].nan_to_num(0.0), got[1].nan_to_num(0.0))
        first = 1 if len(args[0]) == 3 else 4
        assert bad[:first].all()
        live = 0 in table[1, :2] or 0 in table[2, :2]
        assert live or not bad[first:].any()


def test_tables_that_end_before_their_sequence():
    """Keys behind a table's end are not there; entries of no page are page 0."""
    lens = [40, 25]
    cache, want, table = filled(lens, 2, 64, 4)
    table[1, 1] = table[0, 0]
    wild = table.clone()
    table[table == table[0, 1]] = 0
    wild[wild == wild[0, 1]] = 10 ** 6
    wild[1, 2] = -5
    q = part(rows(9, 4, 64, 2), 4, 64)
    total = [100, 25]
    got = ops.paged_attn_decode_kv8(q[:2], *cache, wild.to(DEV), ints(total), 0.1)
    ok = want.values(1)[table[0, 2]][:, 8:].isnan()      # none of the oracle's
    assert not ok.any()
    # page 0 and what the last page holds behind 40 tokens: finite ones here
    for c in cache[:2]:
        c.view(torch.uint8)[c.view(torch.uint8) == 0x7f] = 0
    cache[2][cache[2] == 2.0 ** 60] = 1.0
    want.load(*cache)
    got = ops.paged_attn_decode_kv8(q[:2], *cache, wild.to(DEV), ints(total), 0.1)
    close(got, q[:2], want, table, [0, 1, 2], total, 0.1, 2.0 ** -15)
    got = ops.paged_attn_prefill_kv8(q, *cache, wild.to(DEV), ints([0, 4, 9]),
                                     ints(total), 0.1)
    close(got, q, want, table, [0, 4, 9], total, 0.1, 2.0 ** -8)


@pytest.mark.parametrize("offset", [1, 2, 3])
def test_rows_of_attention_at_any_address(offset):
    """Queries are read by 16 B, results written by 8: others are copied, and what
    is around the results stays."""
    lens, new = [70, 33], [9, 4]
    cache, want, table = filled(lens, 2, 64, 6)
    wide = rows(20, 4, 64, 2).to(DEV)
    q = wide[:13, offset:offset + 256].unflatten(1, (4, 64))
    big = torch.full((15, 261), 7.0, dtype=torch.bfloat16, device=DEV)
    out = big[:, offset:offset + 256].unflatten(1, (4, 64))
    cu = [0, 9, 13]
    got = ops.paged_attn_prefill_kv8(torch.cat((q, q[:2])), *cache, table.to(DEV),
                                     ints(cu), ints(lens), 0.1, out=out)
    assert got.data_ptr() == out.data_ptr()
    close(out[:13], q, want, table, cu, lens, 0.1, 2.0 ** -8)
    assert (big[13:] == 7.0).all() and (big[:, :offset] == 7.0).all()
    assert (big[:, offset + 256:] == 7.0).all()
    big.fill_(7.0)
    ops.paged_attn_decode_kv8(q[:2], *cache, table.to(DEV), ints(lens), 0.1,
                              out=out[:2])
    close(out[:2], q[:2], want, table, [0, 1, 2], lens, 0.1, 2.0 ** -15)
    assert (big[2:] == 7.0).all() and (big[:, :offset] == 7.0).all()


def test_nothing_to_do():
    cache, _, table = filled([20], 2, 64, 6)
    tab, none = table.to(DEV), ints([])
    q = torch.zeros(0, 4, 64, dtype=torch.bfloat16, device=DEV)
    assert ops.paged_attn_decode_kv8(q, *cache, tab, ints([20]), 0.1).shape == q.shape
    assert ops.paged_attn_prefill_kv8(q, *cache, tab, ints([0, 0]), ints([20]),
                                      0.1).shape == q.shape
    ops.reshape_and_cache_kv8(q[:, :2], q[:, :2], *cache, ints([], torch.long))
    slots, pos, cu, used = ops.extend_block_tables(tab[:0], none, none, none, 3)
    assert slots.tolist() == [-1] * 3 and pos.tolist() == [0] * 3
    assert cu.tolist() == [0] and used.tolist() == [0]
    slots, pos, cu, used = ops.extend_block_tables(tab, ints([20]), ints([20]), none,
                                                   0)
    assert slots.numel() == pos.numel() == 0
    assert cu.tolist() == [0, 0] and used.tolist() == [0]


def test_negative_scales_and_large_scores():
    lens = [50, 333]
    cache, want, table = filled(lens, 2, 128, 7, big=30.0)
    q = part(rows(2, 8, 128, 2, 9.0), 8, 128)
    for scale in (-0.3, 0.0, 2.0):
        got = ops.paged_attn_decode_kv8(q, *cache, table.to(DEV), ints(lens),
                                        scale)
        close(got, q, want, table, [0, 1, 2], lens, scale, 2.0 ** -15)
        got = ops.paged_attn_prefill_kv8(q, *cache, table.to(DEV),
                                         ints([0, 1, 2]), ints(lens), scale)
        close(got, q, want, table, [0, 1, 2], lens, scale, 2.0 ** -8)


def test_values_that_are_not_finite():
    """A NaN among a sequence's keys or values is seen by the rows that see it, and
    by no others."""
    lens = [40, 70]
    cache, want, table = filled(lens, 1, 64, 8)
    cache[1].view(torch.uint8)[table[1, 1], 0, 5, 4] = 0x7f      # token 20
    q = part(rows(110, 2, 64, 3), 2, 64)
    got = ops.paged_attn_prefill_kv8(q, *cache, table.to(DEV), ints([0, 40, 110]),
                                     ints(lens), 0.1).cpu()
    assert not got[:60].isnan().any()
    assert got[60:, :, 5].isnan().all()
    assert not got[60:, :, :5].isnan().any()
    got = ops.paged_attn_decode_kv8(q[:2], *cache, table.to(DEV), ints([40, 20]),
                                    0.1)
    assert not got.isnan().any()
    got = ops.paged_attn_decode_kv8(q[:2], *cache, table.to(DEV), ints([40, 21]),
                                    0.1).cpu()
    assert got[1, :, 5].isnan().all() and not got[0].isnan().any()


def test_pages_past_32_bits():
    """A pool of over 4 GiB of keys: its last pages are written and read."""
    heads, dim, pages = 8, 128, 270000
    cache = ops.kv8_cache(pages, heads, dim, DEV)
    table = torch.tensor([[pages - 1, 3, pages - 7, 262145]]).int()
    slots = slots_of(table, [0], [60])
    k, v = rows(60, heads, dim, 1), rows(60, heads, dim, 2)
    gk, gv = part(k, heads, dim), part(v, heads, dim)
    ops.reshape_and_cache_kv8(gk, gv, *cache, ints(slots, torch.long))
    want = Cache(4, heads, dim)
    want.write(gk, gv, list(range(60)))
    got = Cache(4, heads, dim).load(
        *(c.view(torch.uint8)[table[0].long().to(DEV)].view(c.dtype)
          if c.dtype == torch.float8_e4m3fn else c[table[0].long().to(DEV)]
          for c in cache))
    assert all(same(got.x[i], want.x[i]) for i in range(2))
    q = part(rows(60, 32, dim, 3), 32, dim)
    tab, near = table.to(DEV), torch.arange(4).int()[None]
    out = ops.paged_attn_prefill_kv8(q, *cache, tab, ints([0, 60]), ints([60]),
                                     0.1)
    close(out, q, want, near, [0, 60], [60], 0.1, 2.0 ** -8)
    out = ops.paged_attn_decode_kv8(q[:1], *cache, tab, ints([60]), 0.1)
    close(out, q[:1], want, near, [0, 1], [60], 0.1, 2.0 ** -15)


def test_long_sequence():
    lens = [40000, 33]
    cache, want, table = filled(lens, 1, 64, 9)
    q = part(rows(2, 4, 64, 3), 4, 64)
    got = ops.paged_attn_decode_kv8(q, *cache, table.to(DEV), ints(lens), 0.2)
    close(got, q, want, table, [0, 1, 2], lens, 0.2, 2.0 ** -15)


# ---- together, streams and graphs ----------------------------------------------
def step(cache, table, lens, new, free, k, v, q, out):
    slots, _, cu, used = ops.extend_block_tables(table, lens, new, free,
                                                 k.shape[0])
    ops.reshape_and_cache_kv8(k, v, *cache, slots)
    ops.paged_attn_prefill_kv8(q, *cache, table, cu, new, 0.1, out=out)
    return slots, cu, used


def test_a_run_of_them():
    heads, per, dim, S = 2, 4, 128, 3
    table = torch.zeros(S, 20, dtype=torch.int32, device=DEV)
    free = torch.randperm(64, generator=torch.Generator().manual_seed(1))
    free = free.int().to(DEV)
    cache = ops.kv8_cache(64, heads, dim, DEV)
    want = Cache(64, heads, dim)
    lens, at = torch.zeros(S, dtype=torch.int32, device=DEV), 0
    for n, grow in enumerate(([100, 0, 17], [1, 1, 1], [0, 130, 1], [1, 1, 14],
                              [1, 1, 1])):
        T = sum(grow)
        k, v, q = (part(rows(T, m, dim, 3 * n + i), m, dim) for i, m in
                   enumerate((heads, heads, heads * per)))
        out = torch.empty(q.shape, dtype=q.dtype, device=DEV)
        new = lens + ints(grow)
        slots, cu, used = step(cache, table, lens, new, free[at:], k, v, q, out)
        at += int(used)
        want.write(k, v, slots.tolist())
        close(out, q, want, table.cpu(), cu.tolist(), new.tolist(), 0.1,
              2.0 ** -8)
        if max(grow) == min(grow) == 1:
            one = ops.paged_attn_decode_kv8(q, *cache, table, new, 0.1)
            close(one, q, want, table.cpu(), cu.tolist(), new.tolist(), 0.1,
                  2.0 ** -15)
        lens = new


@torch.inference_mode()                       # as the engine's graphs are captured
def test_captured_steps():
    """Two captured steps that share a pool, replayed by turns with eager work
    between them: each replay is the eager result. Rows of padding have no slot."""
    heads, per, dim, S = 2, 4, 128, 4
    lens0 = [700, 3000, 30, 0]
    cache, _, table = filled([n + 64 for n in lens0], heads, dim, 3, spare=9)
    spare = sorted(set(range(cache[2].shape[0])) - set(table.flatten().tolist()))
    table = table.to(DEV)
    free, grow = ints(spare[:3]), ints([1, 1, 1, 0])
    x = part(rows(S, 2 * heads + heads * per, dim, 1), 2 * heads + heads * per,
             dim)

    def run(lens, x):
        new = lens + grow
        slots, *_ = ops.extend_block_tables(table, lens, new, free, S)
        ops.reshape_and_cache_kv8(x[:, :heads], x[:, heads:2 * heads], *cache,
                                  slots)
        return ops.paged_attn_decode_kv8(x[:, 2 * heads:], *cache, table, new,
                                         0.1)
    graphs, pool = [], None
    for g in range(2):
        lens, xx = ints(lens0), x.clone()
        run(lens, xx)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            out = run(lens, xx)
        pool = graph.pool()
        graphs.append((graph, lens, xx, out))
    for n in range(6):
        graph, lens, xx, out = graphs[n % 2]
        lens.copy_(ints([k + n for k in lens0[:3]] + [0]))
        xx.copy_(x * (1 + n))
        free.copy_(ints(spare[n:n + 3]))         # a page of its own for each
        keep = [c.clone() for c in cache]
        graph.replay()
        torch.cuda.synchronize()
        got, after = out.clone(), [c.clone() for c in cache]
        for c, was in zip(cache, keep):
            c.copy_(was)
        want = run(lens.clone(), xx.clone())
        assert torch.equal(got, want), n
        for c, b in zip(cache, after):
            assert torch.equal(c.view(torch.uint8), b.view(torch.uint8)), n
        assert (got[3] == 0).all()


def test_two_streams_at_once():
    lens = [900, 2500, 64]
    cache, want, table = filled(lens, 2, 128, 5)
    tab, n = table.to(DEV), ints(lens)
    q = [part(rows(3, 8, 128, i), 8, 128) for i in range(2)]
    alone = [ops.paged_attn_decode_kv8(x, *cache, tab, n, 0.1) for x in q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(ops.paged_attn_decode_kv8(q[i], *cache, tab, n,
                                                         0.1))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, alone[i]) for o in outs[i])


def test_refusals():
    k8, v8, s = ops.kv8_cache(3, 2, 64, DEV)
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device=DEV)
    at = torch.zeros(4, dtype=torch.long, device=DEV)
    tab, lens = ints([[0]] * 4), ints([1] * 4)
    cu = ints([0, 4])

    def no(f, *args, **kw):
        with pytest.raises(RuntimeError):
            f(*args, **kw)
    w = ops.reshape_and_cache_kv8
    no(w, x, x, k8, v8, s, at[:3])
    no(w, x, x[:3], k8, v8, s, at)
    no(w, x[:, :1], x, k8, v8, s, at)
    no(w, x, x, k8, v8, s, at.int())
    no(w, x, x, k8, v8, s, at.cpu())
    no(w, x.float(), x, k8, v8, s, at)
    no(w, x, x, k8.view(torch.uint8), v8, s, at)
    no(w, x, x, k8.cpu(), v8, s, at)
    no(w, x, x, k8, v8, s.double(), at)
    no(w, x, x, k8[:2], v8, s, at)
    no(w, x, x, v8, k8, s, at)
    no(w, x, x, k8[:0], v8[:0], s[:0], at)
    no(w, x.transpose(0, 1).contiguous().transpose(0, 1), x, k8, v8, s, at)
    d, p = ops.paged_attn_decode_kv8, ops.paged_attn_prefill_kv8
    no(d, x[:, :1], k8, v8, s, tab, lens, 1.0)
    no(d, x[..., :32], k8, v8, s, tab, lens, 1.0)
    no(d, x.half(), k8, v8, s, tab, lens, 1.0)
    no(d, x, k8, v8, s, tab.long(), lens, 1.0)
    no(d, x, k8, v8, s, tab[:3], lens, 1.0)
    no(d, x, k8, v8, s, tab, lens[:3], 1.0)
    no(d, x, k8, v8, s, tab, lens, 1.0, out=x[:3])
    no(d, x, k8, v8, s, tab, lens, 1.0, out=x[:1].expand(4, 2, 64))
    no(d, torch.zeros(4, 34, 64, dtype=x.dtype, device=DEV), k8, v8, s, tab, lens,
       1.0)
    no(p, x, k8, v8, s, tab, cu.long(), lens, 1.0)
    no(p, x, k8, v8, s, tab, cu[:0], lens, 1.0)
    no(p, x, k8, v8, s, tab[:0], cu, lens, 1.0)
    no(p, x, k8, v8, s[:2], tab, cu, lens, 1.0)
    many = ints([0]).expand(2 ** 21 + 1).contiguous()   # of two heads each
    with pytest.raises(RuntimeError, match="too many sequences"):
        d(x[:1].expand(2 ** 21, 2, 64), k8, v8, s, many[:, None], many, 1.0)
    with pytest.raises(RuntimeError, match="too many sequences"):
        p(x, k8, v8, s, many[:, None], many, many, 1.0)
    e = ops.extend_block_tables
    no(e, tab.long(), lens, lens, lens, 4)
    no(e, tab, lens, lens[:2], lens, 4)
    no(e, tab[:2], lens, lens, lens, 4)
    no(e, tab, lens.cpu(), lens, lens, 4)
    no(e, tab, lens, lens, lens, -1)
    no(e, tab, lens, lens, lens, 2 ** 20 + 1)
    no(e, tab.expand(4, 3), lens, lens, lens, 4)


@pytest.mark.parametrize("kind", ["fp8", None])
@pytest.mark.parametrize("tier", ["dram", "ssd"])
def test_engine_swaps_blocks(kind, tier, tmp_path):
    """Blocks out to the host or a file and back into others: the same bytes, those
    beside them untouched."""
    from xllm_service_amd.engine.engine import LLMEngine
    from xllm_service_amd.engine.sampling import SamplingParams
    from xllm_service_amd.engine.sequence import Sequence
    eng = LLMEngine("llama-tiny", device="cuda:0", max_kv_blocks=32, seed=3,
                    max_num_seqs=4, max_model_len=256, enable_graphs=False,
                    kv_cache_dtype=kind, enable_prefix_caching=False,
                    swap_space_mb=0 if tier == "ssd" else 64,
                    ssd_swap_dir=str(tmp_path / "spool"))
    assert (eng.cpu_block_manager is None) == (tier == "ssd")
    eng.generate([[5, 9, 2, 7] * 30, list(range(40, 100))],
                 SamplingParams(max_tokens=20, ignore_eos=True))
    tensors = eng.runner.paged_tensors()
    was = [c.clone() for c in tensors]
    assert all((c != 0).any() for c in was)
    seq = Sequence(request_id="s", prompt_token_ids=[1] * 70,
                   params=SamplingParams())
    seq.block_table = out = eng.block_manager.allocate_raw(5)
    seq.block_table = out = [out[i] for i in (3, 0, 1, 4, 2)]
    seq.cpu_block_table = eng._swap_out(seq)
    hold = eng.block_manager.allocate_raw(3)
    eng._swap_in(seq)
    into = seq.block_table
    assert not set(into) & set(out + hold)
    rest = [i for i in range(32) if i not in into]
    for c, w in zip(tensors, was):
        assert torch.equal(c[into], w[out])
        assert torch.equal(c[rest], w[rest])


@pytest.mark.parametrize("model", ["llama-tiny", "llama-debug-128", "opt-125m"])
def test_engine(model):
    """The engine over 8-bit pages: captured decode steps are the eager ones."""
    from xllm_service_amd.engine.engine import LLMEngine
    from xllm_service_amd.engine.sampling import SamplingParams
    prompts = [[5, 9, 2, 7] * 30, [3], list(range(40, 100))]
    sp = SamplingParams(max_tokens=20, ignore_eos=True)
    outs = []
    for graphs in (False, True):
        eng = LLMEngine(model, device="cuda:0", max_kv_blocks=64, seed=3,
                        max_num_seqs=4, max_batched_tokens=64, max_model_len=256,
                        enable_graphs=graphs, kv_cache_dtype="fp8")
        assert (eng.runner.graph_runner is not None) == graphs
        outs.append(eng.generate(prompts, sp))
        assert [len(o) for o in outs[-1]] == [20] * 3
        assert all(c[2].isfinite().all() for c in eng.runner.kv_caches)
        moved = eng.import_block_bytes([5], eng.export_block_bytes([1]))
        assert moved is None
        for c in eng.runner.paged_tensors():
            assert torch.equal(c[5], c[1])
        del eng
        torch.cuda.empty_cache()
    assert outs[0] == outs[1]
