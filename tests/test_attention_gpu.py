"""Rotary positions, the paged key-value cache and decode attention on the GPU, against their definitions in 64 bits.

What is stored and read back is defined to the bit.  The tolerances of the others are sums of half steps: fp16 2^-11 of a value
(2^-25 below the normal numbers), and the 32-bit arithmetic in front of it."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
HALF, TINY = 2.0 ** -11, 2.0 ** -25


def _gen(cuda, seed):
    g = cuda.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(cuda, g, *shape, scale=1.0):
    return (cuda.randn(shape, generator=g, device="cuda") * scale).to(cuda.float16)


# ---- rotary ----------------------------------------------------------------------------------------------------------

def _rotated(cuda, x, positions, table, interleaved):
    """(values, bound) in 64 bits; the angle from the table's words, whole turns taken off in integers."""
    rd = table.rotary_dim
    words = [int(w) % (1 << 64) for w in table.turns.cpu().tolist()]
    angle = np.array([[((int(p) * w) % (1 << 64)) / 2.0 ** 64 * 2 * math.pi for w in words] for p in positions.cpu().tolist()]).reshape(len(positions), rd // 2)
    cos, sin = (cuda.from_numpy(f(angle) * table.magnitude).cuda()[:, None] for f in (np.cos, np.sin))
    y, size = x.double(), x.double().abs()
    lo, hi = (slice(0, rd, 2), slice(1, rd, 2)) if interleaved else (slice(0, rd // 2), slice(rd // 2, rd))
    a, b = y[..., lo].clone(), y[..., hi].clone()
    y[..., lo], y[..., hi] = a * cos - b * sin, b * cos + a * sin
    bound = y.abs() * HALF + TINY
    # the angle is rounded to 24 bits (up to pi 2^-24 of a radian), sine and cosine to 2 units in the last place, three roundings more
    bound[..., lo] += (a.abs() + b.abs()) * table.magnitude * 2.0 ** -20
    bound[..., hi] += (a.abs() + b.abs()) * table.magnitude * 2.0 ** -20
    bound[..., rd:] = 0
    return y, bound


def _check_rotated(cuda, got, x, positions, table, interleaved):
    want, bound = _rotated(cuda, x, positions, table, interleaved)
    assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("tokens,hq,hk,d,rd", [(1, 1, 1, 16, 16), (1, 32, 32, 128, 128), (3, 5, 1, 64, 32), (17, 8, 2, 96, 96), (2, 7, 7, 96, 48), (33, 64, 8, 128, 64), (5, 3, 1, 256, 256),
                                               (4, 2, 1, 256, 16), (7, 9, 4, 80, 80), (6, 4, 4, 208, 112), (1100, 6, 2, 128, 128), (1025, 40, 1, 64, 64),
                                               # several heads a thread, some of whose turns have none
                                               (9001, 37, 5, 128, 128), (20000, 7, 2, 256, 64), (40000, 5, 3, 64, 32), (9001, 3, 37, 128, 96)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary(cuda, pplb200, tokens, hq, hk, d, rd, interleaved):
    g = _gen(cuda, tokens * 131 + d)
    q, k = _randn(cuda, g, tokens, hq, d), _randn(cuda, g, tokens, hk, d, scale=20.0)
    pos = cuda.randint(0, 5000, (tokens,), generator=g, device="cuda")
    table = pplb200.RotaryTable(rd, base=10000.0)
    qo, ko = pplb200.rotary_fp16(q, k, pos, table, interleaved)
    _check_rotated(cuda, qo, q, pos, table, interleaved)
    _check_rotated(cuda, ko, k, pos, table, interleaved)


@pytest.mark.parametrize("kind", ["linear", "ntk", "yarn", "wavelength"])
def test_rotary_far_positions_and_scalings(cuda, pplb200, kind):
    """Positions at both ends of 64 bits, negative ones among them: the angle is exact, not a product in 32 bits."""
    g = _gen(cuda, 5)
    table = pplb200.RotaryTable(128, base=500000.0, scaling=kind, factor=16.0, original_length=8192, keep_turns=32, stretch_turns=1)
    pos = cuda.tensor([0, 1, -1, 4095, 131071, -131072, 1 << 20, (1 << 31) - 1, -(1 << 31), 1 << 40, (1 << 63) - 1, -(1 << 63)], device="cuda")
    q = _randn(cuda, g, len(pos), 4, 128)
    qo, none = pplb200.rotary_fp16(q, None, pos, table)
    assert none is None
    _check_rotated(cuda, qo, q, pos, table, False)


def test_rotary_at_position_zero_is_the_identity(cuda, pplb200):
    q = _randn(cuda, _gen(cuda, 6), 9, 4, 128)
    q[0, 0, :4] = cuda.tensor([65504.0, -65504.0, 6e-8, -0.0])
    table = pplb200.RotaryTable(128)
    assert cuda.equal(pplb200.rotary_fp16(q, None, cuda.zeros(9, dtype=cuda.int64, device="cuda"), table)[0], q)


def test_rotary_special_values(cuda, pplb200):
    """An infinity or NaN stays in its plane; dimensions behind the rotated ones are copied bit for bit."""
    q = _randn(cuda, _gen(cuda, 7), 2, 2, 64)
    plain = pplb200.rotary_fp16(q, None, cuda.tensor([3, 4], device="cuda"), pplb200.RotaryTable(32))[0]
    q[0, 0, 5], q[1, 1, 20], q[1, 0, 40], q[0, 1, 50] = float("inf"), float("nan"), float("nan"), float("-inf")
    got = pplb200.rotary_fp16(q, None, cuda.tensor([3, 4], device="cuda"), pplb200.RotaryTable(32))[0]
    odd = ~cuda.isfinite(got)
    want = cuda.zeros_like(odd)
    want[0, 0, [5, 21]] = want[1, 1, [4, 20]] = want[1, 0, 40] = want[0, 1, 50] = True
    assert cuda.equal(odd, want) and cuda.equal(got[~want], plain[~want])


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_in_place_and_strided(cuda, pplb200, interleaved):
    """q and k inside the fused projection's rows, rotated where they lie; what lies around them is left alone."""
    g = _gen(cuda, 8)
    rows = _randn(cuda, g, 41, 14, 96)
    pos = cuda.randint(0, 100000, (41,), generator=g, device="cuda")
    table = pplb200.RotaryTable(64)
    apart = pplb200.rotary_fp16(rows[:, 1:9].contiguous(), rows[:, 9:11].contiguous(), pos, table, interleaved)
    before = rows.clone()
    q, k = rows[:, 1:9], rows[:, 9:11]
    qo, ko = pplb200.rotary_fp16(q, k, pos, table, interleaved, q_out=q, k_out=k)
    assert qo is q and ko is k and cuda.equal(q, apart[0]) and cuda.equal(k, apart[1])
    assert cuda.equal(rows[:, :1], before[:, :1]) and cuda.equal(rows[:, 11:], before[:, 11:])


# ---- the cache -------------------------------------------------------------------------------------------------------

def _quantized(x, group):
    """(int8 values, fp16 scales) of fp16 x in 64 bits; a group with an infinity has that for its scale, and zeros."""
    x = x.astype(np.float64)
    y = x.reshape(x.shape[:-1] + (-1, group))
    exact = np.abs(y).max(-1, keepdims=True) / 127
    s = exact.astype(np.float16)
    s = np.where(s.astype(np.float64) < exact, np.nextafter(s, np.float16(np.inf)), s)
    s = np.where(np.isinf(exact), np.float16(np.inf), np.clip(s, np.float16(2.0 ** -24), np.float16(515.5)))
    q = np.where(np.isinf(exact), 0, np.rint(np.where(np.isinf(exact), 0, y) / s.astype(np.float64)))
    return q.astype(np.int8).reshape(x.shape), s[..., 0]


def _cache(cuda, pplb200, pages, page, heads, d, group, order, fill):
    """A cache in one of two orders, everything set to `fill` first."""
    dt = cuda.int8 if group else cuda.float16
    shape = (pages, heads, page) if order == "heads" else (pages, page, heads)
    make = lambda n, t, v: cuda.full(shape + (n,), v, dtype=t, device="cuda")  # noqa: E731
    tensors = [make(d, dt, fill), make(d, dt, fill)] + ([make(d // group, cuda.float16, float(fill)) for _ in range(2)] if group else [])
    return pplb200.PagedKVCache(*(t if order == "heads" else t.transpose(1, 2) for t in tensors))


def _rows(t, slots, page):
    """[tokens, heads, ...] of a cache tensor at the slots."""
    return None if t is None else t[slots // page, :, slots % page]


STORED = [(1, 1, 16, 16, 1), (3, 2, 64, 8, 5), (29, 8, 128, 16, 3), (16, 32, 128, 16, 1), (50, 3, 96, 7, 2), (33, 1, 256, 64, 1), (12, 5, 80, 24, 4), (1200, 2, 128, 16, 1), (40, 4, 208, 1, 3),
          (12001, 7, 128, 16, 3), (14001, 3, 256, 7, 2)]  # several heads a thread, some of whose turns have none


@pytest.mark.parametrize("tokens,heads,d,page,spare", STORED)
@pytest.mark.parametrize("group", [0, 8, -1])
@pytest.mark.parametrize("order", ["heads", "tokens"])
def test_write_and_read(cuda, pplb200, tokens, heads, d, page, spare, group, order):
    """Stored to the bit, at the right place, everything else in the cache left as it was; read back to the bit."""
    group = d if group < 0 else group
    g = _gen(cuda, tokens + d)
    pages = (tokens + page - 1) // page + spare
    cache = _cache(cuda, pplb200, pages, page, heads, d, group, order, 77)
    k = _randn(cuda, g, tokens, heads, d) * cuda.exp(cuda.randn((tokens, heads, 1), generator=g, device="cuda") * 3).to(cuda.float16)
    v = _randn(cuda, g, tokens, heads + 2, d)[:, 1:heads + 1]  # not contiguous
    k[0, 0] = 0
    slots = cuda.randperm(pages * page, generator=g, device="cuda")[:tokens]
    if tokens > 2:
        slots[1] = -1                 # not stored
        slots[2] = pages * page + 5   # nor this
    pplb200.kv_cache_write(cache, k, v, slots)
    kept = (slots >= 0) & (slots < pages * page)
    for x, data, scale in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        touched = cuda.zeros((pages, page), dtype=cuda.bool, device="cuda")
        touched[slots[kept] // page, slots[kept] % page] = True
        for t in (data, scale) if group else (data,):
            assert bool((t.transpose(1, 2)[~touched] == 77).all())
        x = x[kept].cpu().numpy()
        if group:
            q, s = _quantized(x, group)
            assert np.array_equal(_rows(data, slots[kept], page).cpu().numpy(), q)
            assert np.array_equal(_rows(scale, slots[kept], page).cpu().numpy(), s)
        else:
            assert np.array_equal(_rows(data, slots[kept], page).cpu().numpy().view(np.int16), x.view(np.int16))
    for x, data, scale, back in zip((k, v), (cache.k, cache.v), (cache.k_scale, cache.v_scale), pplb200.kv_cache_read(cache, slots)):
        assert bool((back[~kept] == 0).all())
        want = _rows(data, slots[kept], page)
        if group:
            s = _rows(scale, slots[kept], page).cpu().numpy().astype(np.float64)
            want = cuda.from_numpy((want.cpu().numpy().astype(np.float64) * np.repeat(s, group, -1)).astype(np.float16)).cuda()
        assert bool(((back[kept] == want) | (back[kept].isnan() & want.isnan())).all())


@pytest.mark.parametrize("group", [8, 64])
def test_quantizer_at_its_edges(cuda, pplb200, group):
    """Quotients at half steps, the largest and the smallest numbers, zeros; infinities and NaN make their own group NaN and no other."""
    x = cuda.zeros((1, 8, 64), dtype=cuda.float16)
    x[0, 0, ::8] = 127.0
    x[0, 0, 1::8], x[0, 0, 2::8], x[0, 0, 3::8], x[0, 0, 4::8] = 0.5, 1.5, -2.5, 126.5
    x[0, 1, ::8], x[0, 1, 1::8] = 65504.0, -65504.0
    x[0, 2, ::8], x[0, 2, 1::8] = 2.0 ** -24, -(2.0 ** -23)
    x[0, 3] = cuda.arange(64) * 3e-7
    x[0, 4] = cuda.arange(64) * 1e-5
    x[0, 5, 3], x[0, 6, 9] = float("inf"), float("nan")
    x[0, 5, 10], x[0, 6, 1] = 3.0, 2.0
    x[0, 7] = -0.0
    cache = pplb200.PagedKVCache.allocate(2, 4, 8, 64, group)
    slot = cuda.tensor([6], device="cuda")
    pplb200.kv_cache_write(cache, x.cuda(), x.cuda(), slot)
    back, _ = pplb200.kv_cache_read(cache, slot)
    q, s = _quantized(x.numpy()[:, [0, 1, 2, 3, 4, 7]], group)
    fine = [0, 1, 2, 3, 4, 7]
    assert np.array_equal(cache.k[1, fine, 2].cpu().numpy(), q[0]) and np.array_equal(cache.k_scale[1, fine, 2].cpu().numpy(), s[0])
    odd = cuda.isnan(back[0].cpu())
    want = cuda.zeros((8, 64), dtype=cuda.bool)
    if group == 8:
        want[5, :8] = want[6, 8:16] = True
    else:
        want[5:7] = True
    assert cuda.equal(odd, want)
    # half a step of the scale that is stored, and the rounding of what is read back (half more at most than x)
    half = np.repeat(s[0].astype(np.float64), group, -1) / 2
    got, put = back[0].cpu().numpy().astype(np.float64)[fine], x[0].numpy().astype(np.float64)[fine]
    assert np.all(np.abs(got - put) <= half + (np.abs(put) + half) * HALF + TINY)


@pytest.mark.parametrize("tokens,hq,hk,d,rd,page", [(1, 8, 1, 128, 128, 16), (16, 32, 32, 128, 128, 16), (37, 7, 7, 96, 48, 5), (1030, 8, 2, 64, 64, 64), (3, 4, 2, 256, 128, 1),
                                                    (9001, 10, 3, 128, 128, 16), (16001, 13, 13, 64, 48, 16)])
@pytest.mark.parametrize("group", [0, 8, -1])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotating_write_is_the_two_calls(cuda, pplb200, tokens, hq, hk, d, rd, page, group, interleaved):
    group = d if group < 0 else group
    g = _gen(cuda, tokens)
    rows = _randn(cuda, g, tokens, hq + 2 * hk, d)
    q, k, v = rows[:, :hq], rows[:, hq:hq + hk], rows[:, hq + hk:]
    pos = cuda.randint(0, 1 << 20, (tokens,), generator=g, device="cuda")
    pages = (tokens + page - 1) // page + 1
    slots = cuda.randperm(pages * page, generator=g, device="cuda")[:tokens]
    slots[0] = -5
    table = pplb200.RotaryTable(rd, scaling="yarn", factor=4.0, original_length=4096, keep_turns=32, stretch_turns=1)
    one, two = (pplb200.PagedKVCache.allocate(pages, page, hk, d, group) for _ in range(2))
    q1 = pplb200.rotary_kv_cache_write(one, q, k, v, pos, slots, table, interleaved)
    q2, k2 = pplb200.rotary_fp16(q, k, pos, table, interleaved)
    pplb200.kv_cache_write(two, k2, v, slots)
    assert cuda.equal(q1, q2)
    for n in ("k", "v", "k_scale", "v_scale"):
        a, b = getattr(one, n), getattr(two, n)
        assert (a is None and b is None) or cuda.equal(a, b)
    # keys alone, and q rotated where it lies
    three = pplb200.PagedKVCache.allocate(pages, page, hk, d, group)
    assert pplb200.rotary_kv_cache_write(three, None, k, v, pos, slots, table, interleaved) is None and cuda.equal(three.k, two.k)
    pplb200.rotary_kv_cache_write(three, q, k, v, pos, slots, table, interleaved, q_out=q)
    assert cuda.equal(q, q2) and cuda.equal(three.v, two.v)


def test_read_takes_a_slot_several_times(cuda, pplb200):
    cache = pplb200.PagedKVCache.allocate(4, 16, 2, 128, 128)
    g = _gen(cuda, 3)
    k, v = _randn(cuda, g, 64, 2, 128), _randn(cuda, g, 64, 2, 128)
    pplb200.kv_cache_write(cache, k, v, cuda.arange(64, device="cuda"))
    slots = cuda.tensor([5, 5, -1, 63, 64, 5, 0], device="cuda")
    a, b = pplb200.kv_cache_read(cache, slots)
    one, _ = pplb200.kv_cache_read(cache, cuda.tensor([5], device="cuda"))
    assert cuda.equal(a[0], one[0]) and cuda.equal(a[1], one[0]) and cuda.equal(a[5], one[0])
    assert not a[2].any() and not b[2].any() and not a[4].any() and not b[4].any()


# ---- attention -------------------------------------------------------------------------------------------------------

def _stored(cuda, cache, slots):
    """(k, v) [tokens, heads, d] in 64 bits, what is stored at the slots: fp16, or whole numbers times scales."""
    rows = [None if t is None else _rows(t, slots, cache.page_size).double() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    return [x if s is None else x * s.repeat_interleave(cache.quant_group, -1) for x, s in (rows[::2], rows[1::2])]


def _attention(cuda, q, k, v, seen, scale, values_rounded=False):
    """One sequence in 64 bits: q [hq, d], k, v [tokens, hk, d], seen [tokens] -> out, lse and the bounds of both.  values_rounded: whole
    numbers times scales of groups of eight dimensions are rounded to fp16 before they are weighted."""
    hq, d = q.shape
    shared = hq // k.shape[1]
    out, lse = cuda.zeros((hq, d), dtype=cuda.float64, device="cuda"), cuda.full((hq,), -math.inf, dtype=cuda.float64, device="cuda")
    bound, lse_bound = cuda.full_like(out, TINY), cuda.zeros_like(lse)
    if not bool(seen.any()):
        return out, lse, bound, lse_bound
    k, v = k[seen].double().repeat_interleave(shared, 1), v[seen].double().repeat_interleave(shared, 1)
    score = cuda.einsum("hd,thd->ht", q.double(), k) * scale
    p = cuda.softmax(score, -1)
    lse = cuda.logsumexp(score, -1)
    out = cuda.einsum("ht,thd->hd", p, v)
    # a score: a sum of d products in 32 bits (whatever their order), the factors on it, the difference to the maximum
    size = cuda.einsum("hd,thd->ht", q.double().abs(), k.abs()).amax(-1) * abs(scale)
    off = size * (d + 8) * 2.0 ** -24 + 2.0 ** -20
    # a weight: that as a relative error (twice: the sum of the weights has it too), its rounding to fp16, sums over tokens in 32 bits
    weight = 2 * off + HALF + 2.0 ** -14
    if values_rounded:
        weight += HALF
        bound += TINY
    bound += out.abs() * HALF + weight[:, None] * cuda.einsum("ht,thd->hd", p, v.abs()) * (1 + HALF)
    return out, lse, bound, off + 2.0 ** -14 + lse.abs() * 2.0 ** -22


def _run_attention(cuda, pplb200, lengths, hq, hk, d, page, group, order="heads", window=0, scale=None, q_scale=2.0, holes=(), seed=0, poison=True, extra_pages=0, lse=True):
    """A filled cache, tables that scatter the sequences over it, everything that no sequence owns NaN (int8: NaN scales).
    Returns what the library and what the definition give."""
    g = _gen(cuda, seed + 17 * len(lengths) + d)
    counts = [-(-n // page) for n in lengths]
    width = max(counts + [1]) + extra_pages
    pages = sum(counts) + 3
    cache = _cache(cuda, pplb200, pages, page, hk, d, group, order, 1)
    cache.v.fill_(2)
    for t in ((cache.k_scale, cache.v_scale) if group else (cache.k, cache.v)) if poison else ():
        t.fill_(float("nan"))
    order_of_pages = cuda.randperm(pages, generator=g, device="cuda").tolist()
    table = cuda.full((len(lengths), width), pages + 1000, dtype=cuda.int32, device="cuda")  # behind a sequence's pages: no page
    q = _randn(cuda, g, len(lengths), hq, d, scale=q_scale)
    written = []
    for b, (n, c) in enumerate(zip(lengths, counts)):
        mine = [order_of_pages.pop() for _ in range(c)]
        if c:
            table[b, :c] = cuda.tensor(mine, dtype=cuda.int32, device="cuda")
        at = cuda.arange(n, device="cuda")
        slots = (table[b].long()[at // page] * page + at % page) if n else at
        k, v = _randn(cuda, g, n, hk, d), _randn(cuda, g, n, hk, d)
        if n:
            pplb200.kv_cache_write(cache, k, v, slots)
        written.append(_stored(cuda, cache, slots) if n else (k, v))
    for b, i, value in holes:
        table[b, i] = value
    lens = cuda.tensor(lengths, dtype=cuda.int32, device="cuda")
    att = pplb200.PagedDecodeAttention(cache, hq, max_batch=len(lengths), max_length=width * page, scale=scale, window=window)
    out = cuda.full((len(lengths), hq, d), 7.0, dtype=cuda.float16, device="cuda")
    got_lse = cuda.full((len(lengths), hq), 7.0, device="cuda") if lse else None
    att(q, table, lens, out=out, lse=got_lse)
    want = []
    for b, n in enumerate(lengths):
        at = cuda.arange(n, device="cuda")
        page_of = table[b].long()[at // page] if n else at
        seen = (page_of >= 0) & (page_of < pages) & ((at >= n - window) if window else (at >= 0))
        want.append(_attention(cuda, q[b], *written[b], seen, att.scale, group == 8))
    return out, got_lse, want, (att, q, table, lens, cache)


def _check_attention(out, lse, want):
    for b, (o, l, bound, lse_bound) in enumerate(want):
        off = (out[b].double() - o).abs()
        assert bool((off <= bound).all()), (b, float((off / bound).max()))
        if lse is not None:
            gone = l.isinf()
            assert bool((lse[b][gone] == -math.inf).all())
            assert bool(((lse[b].double() - l)[~gone].abs() <= lse_bound[~gone]).all()), b


@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("group", [0, 8, -1])
@pytest.mark.parametrize("hq,hk", [(1, 1), (4, 4), (8, 1), (10, 2), (32, 2), (40, 1)])
def test_attention_heads_and_types(cuda, pplb200, d, group, hq, hk):
    lengths = [1, 0, 2, 15, 16, 17, 63, 64, 65, 130, 333]
    _check_attention(*_run_attention(cuda, pplb200, lengths, hq, hk, d, 16, d if group < 0 else group)[:3])


@pytest.mark.parametrize("page", [1, 3, 8, 24, 64, 128, 1000])
@pytest.mark.parametrize("group", [0, 8, 128])
@pytest.mark.parametrize("order", ["heads", "tokens"])
def test_attention_pages_and_orders(cuda, pplb200, page, group, order):
    _check_attention(*_run_attention(cuda, pplb200, [5, 200, 1, 777, 64], 8, 2, 128, page, group, order=order, seed=page)[:3])


@pytest.mark.parametrize("group", [0, 8, 128])
@pytest.mark.parametrize("lengths", [[5000], [20011], [4096, 1, 9000, 0, 130], [70001]])
def test_attention_long(cuda, pplb200, lengths, group):
    """Sequences that are cut over many CTAs and joined."""
    _check_attention(*_run_attention(cuda, pplb200, lengths, 16, 2, 128, 64, group)[:3])


@pytest.mark.parametrize("d,group", [(64, 64), (96, 8), (128, 0), (256, 256)])
def test_attention_many_sequences(cuda, pplb200, d, group):
    """More sequences than CTAs, most of them short, empty ones between."""
    rng = np.random.default_rng(d)
    lengths = [int(n) for n in rng.integers(0, 90, 700)]
    lengths[3] = 2500
    _check_attention(*_run_attention(cuda, pplb200, lengths, 4, 2, d, 16, group)[:3])


def test_attention_all_empty(cuda, pplb200):
    out, lse, _, _ = _run_attention(cuda, pplb200, [0, 0, 0], 8, 2, 128, 16, 8, extra_pages=4)
    assert not out.any() and bool((lse == -math.inf).all())


@pytest.mark.parametrize("window", [1, 2, 16, 100, 129, 100000])
@pytest.mark.parametrize("group", [0, 8, 128])
@pytest.mark.parametrize("page", [16, 24])
def test_attention_window(cuda, pplb200, window, group, page):
    _check_attention(*_run_attention(cuda, pplb200, [1, 2, 15, 100, 101, 700, 0, 3001], 8, 2, 128, page, group, window=window)[:3])


@pytest.mark.parametrize("group", [0, 8, 128])
def test_attention_holes(cuda, pplb200, group):
    """Pages that are negative or beyond the cache take no part; one sequence has nothing but such pages."""
    holes = [(0, 0, -1), (0, 3, 1 << 30), (1, 0, -(1 << 31)), (1, 1, -7), (2, 5, -1), (3, 20, 1 << 20)]
    out, lse, want, _ = _run_attention(cuda, pplb200, [100, 30, 96, 1000], 8, 2, 128, 16, group, holes=holes)
    _check_attention(out, lse, want)
    assert not out[1].any() and bool((lse[1] == -math.inf).all())


@pytest.mark.parametrize("scale,q_scale", [(None, 20.0), (1.0, 8.0), (0.0, 1.0), (-0.1, 2.0), (1e-6, 1.0)])
@pytest.mark.parametrize("group", [0, 8])
def test_attention_scores_of_all_sizes(cuda, pplb200, scale, q_scale, group):
    """Softmaxes between uniform and one-hot, scores of some hundreds."""
    _check_attention(*_run_attention(cuda, pplb200, [1500, 40, 333], 8, 2, 128, 16, group, scale=scale, q_scale=q_scale)[:3])


@pytest.mark.parametrize("rising", [True, False])
@pytest.mark.parametrize("group", [0, 128])
def test_attention_scores_that_rise_or_fall(cuda, pplb200, rising, group):
    """The running maximum changes with every tile, or never after the first."""
    d, n = 128, 2000
    g = _gen(cuda, 1)
    cache = _cache(cuda, pplb200, 130, 16, 1, d, group, "heads", 0)
    k, v = cuda.zeros((n, 1, d), dtype=cuda.float16, device="cuda"), _randn(cuda, g, n, 1, d)
    ramp = cuda.linspace(0, 60, n, device="cuda")
    k[:, 0, 0] = (ramp if rising else ramp.flip(0)).to(cuda.float16)
    pplb200.kv_cache_write(cache, k, v, cuda.arange(n, device="cuda"))
    kr, vr = _stored(cuda, cache, cuda.arange(n, device="cuda"))
    q = cuda.zeros((1, 4, d), dtype=cuda.float16, device="cuda")
    q[0, :, 0] = cuda.tensor([1.0, 4.0, -4.0, 0.0])
    table = cuda.arange(125, dtype=cuda.int32, device="cuda")[None]
    att = pplb200.PagedDecodeAttention(cache, 4, 1, 2000, scale=1.0)
    lse = cuda.empty((1, 4), device="cuda")
    out = att(q, table, cuda.tensor([n], dtype=cuda.int32, device="cuda"), lse=lse)
    _check_attention(out, lse, [_attention(cuda, q[0], kr, vr, cuda.ones(n, dtype=cuda.bool, device="cuda"), 1.0)])


def test_attention_values_of_all_sizes(cuda, pplb200):
    """Values near the largest and the smallest of fp16: weights and sums neither overflow nor vanish."""
    for size in (60000.0, 1e-4, 1e-6):
        cache = pplb200.PagedKVCache.allocate(20, 16, 1, 128, 0)
        g = _gen(cuda, 2)
        k, v = _randn(cuda, g, 300, 1, 128), (cuda.rand((300, 1, 128), generator=g, device="cuda") * size).to(cuda.float16)
        pplb200.kv_cache_write(cache, k, v, cuda.arange(300, device="cuda"))
        q = _randn(cuda, g, 1, 2, 128)
        att = pplb200.PagedDecodeAttention(cache, 2, 1, 320)
        out = att(q, cuda.arange(20, dtype=cuda.int32, device="cuda")[None], cuda.tensor([300], dtype=cuda.int32, device="cuda"))
        _check_attention(out, None, [_attention(cuda, q[0], k, v, cuda.ones(300, dtype=cuda.bool, device="cuda"), att.scale)])


@pytest.mark.parametrize("group", [0, 8, 128])
@pytest.mark.parametrize("scale", [2.0 ** 50, -(2.0 ** 50)])
def test_attention_scores_at_the_largest_scale(cuda, pplb200, group, scale):
    """Scores of 1e20: one token has all the weight, and the reference exponent follows it far from where it begins."""
    d, n = 128, 300
    cache = _cache(cuda, pplb200, 20, 16, 1, d, group, "heads", 0)
    k = ((cuda.randperm(n, generator=_gen(cuda, 3), device="cuda") - 150.5) * 2).to(cuda.float16)[:, None, None].expand(n, 1, d).contiguous()
    pplb200.kv_cache_write(cache, k, _randn(cuda, _gen(cuda, 4), n, 1, d), cuda.arange(n, device="cuda"))
    kr, vr = _stored(cuda, cache, cuda.arange(n, device="cuda"))
    q = cuda.tensor([500.0, -500.0, 0.001], device="cuda").to(cuda.float16)[None, :, None].expand(1, 3, d).contiguous()
    att = pplb200.PagedDecodeAttention(cache, 3, 1, 320, scale=scale)
    out = att(q, cuda.arange(20, dtype=cuda.int32, device="cuda")[None], cuda.tensor([n], dtype=cuda.int32, device="cuda"))
    # neighbouring keys are 1 / 300 of the largest apart, 2^14 roundings to 32 bits: the same token wins.  Its value is rounded when it is
    # read with groups of 8, and rounded on output; the weights' sum is a power of two, and the quotient off by 2^-20 at most.
    score = cuda.einsum("hd,td->ht", q[0].double(), kr[:, 0]) * scale
    want = vr[score.argmax(-1), 0]
    assert bool(((out[0].double() - want).abs() <= want.abs() * (2 * HALF + 2.0 ** -20) + 2 * TINY).all())


@pytest.mark.parametrize("group", [8, 128])
def test_attention_scales_of_either_sign(cuda, pplb200, group):
    """Scales that another program stored may be negative."""
    n, d = 300, 128
    cache = _cache(cuda, pplb200, 20, 16, 1, d, group, "heads", 0)
    g = _gen(cuda, 5)
    pplb200.kv_cache_write(cache, _randn(cuda, g, n, 1, d), _randn(cuda, g, n, 1, d, scale=1000.0), cuda.arange(n, device="cuda"))
    for t in (cache.k_scale, cache.v_scale):
        t.mul_((cuda.rand(t.shape, generator=g, device="cuda") < 0.5) * 2 - 1)
    q = _randn(cuda, g, 1, 4, d)
    att = pplb200.PagedDecodeAttention(cache, 4, 1, 320)
    out = att(q, cuda.arange(20, dtype=cuda.int32, device="cuda")[None], cuda.tensor([n], dtype=cuda.int32, device="cuda"))
    kr, vr = _stored(cuda, cache, cuda.arange(n, device="cuda"))
    _check_attention(out, None, [_attention(cuda, q[0], kr, vr, cuda.ones(n, dtype=cuda.bool, device="cuda"), att.scale, group == 8)])


def test_attention_lengths_beyond_the_table_and_negative(cuda, pplb200):
    """No more is looked at than the table has pages for; a negative length is an empty sequence."""
    out, lse, want, (att, q, table, lens, cache) = _run_attention(cuda, pplb200, [64, 64, 33], 8, 2, 128, 16, 0)
    _check_attention(out, lse, want)
    far = cuda.tensor([1 << 30, -1, 33], dtype=cuda.int32, device="cuda")
    got = att(q, table, far)
    assert cuda.equal(got[0], out[0]) and cuda.equal(got[2], out[2]) and not got[1].any()
    got = att(q, table[:, :2], cuda.tensor([32, -(1 << 31), 20], dtype=cuda.int32, device="cuda"))
    same = att(q, table[:, :2].contiguous(), cuda.tensor([64, 0, 20], dtype=cuda.int32, device="cuda"))
    assert cuda.equal(got, same)
    assert not att(q, table[:, :0], lens).any()


def test_attention_special_values(cuda, pplb200):
    """A NaN or infinity among a sequence's own tokens reaches that sequence's heads and no other's; out of sight (another
    window, behind the length) it has no influence."""
    out, lse, want, (att, q, table, lens, cache) = _run_attention(cuda, pplb200, [100, 100, 50], 8, 2, 128, 16, 0, window=40)
    page, place = 97 // 16, 97 % 16
    cache.v[int(table[0, page]), 1, place, 5] = float("nan")
    cache.k[int(table[1, 1]), :, 3] = float("inf")       # token 19 of 100: outside the window
    cache.v[int(table[1, 1]), :, 3] = float("nan")
    cache.k[int(table[2, 3]), :, 10] = float("nan")      # token 58 of 50
    got = att(q, table, lens)
    assert cuda.equal(got[1:], out[1:]) and cuda.equal(got[0, :4], out[0, :4])
    assert bool(got[0, 4:, 5].isnan().all()) and bool(cuda.equal(got[0, 4:, 6:], out[0, 4:, 6:]))


def test_attention_strided_and_in_place(cuda, pplb200):
    """q inside the fused projection's rows, out in another tensor's, the table a slice of a wider one; then out on top of q."""
    out, _, want, (att, q, table, lens, cache) = _run_attention(cuda, pplb200, [70, 1, 300], 8, 2, 128, 16, 8, lse=False)
    rows, wide = cuda.zeros((3, 12, 128), dtype=cuda.float16, device="cuda"), cuda.zeros((3, 20, 128), dtype=cuda.float16, device="cuda")
    rows[:, 2:10] = q
    tables = cuda.full((3, table.shape[1] + 9), -1, dtype=cuda.int32, device="cuda")
    tables[:, 4:4 + table.shape[1]] = table
    att(rows[:, 2:10], tables[:, 4:4 + table.shape[1]], lens, out=wide[:, 5:13])
    assert cuda.equal(wide[:, 5:13], out) and not wide[:, :5].any() and not wide[:, 13:].any()
    att(rows[:, 2:10], table, lens, out=rows[:, 2:10])
    assert cuda.equal(rows[:, 2:10], out)


def test_attention_fewer_sequences_leave_the_rest_alone(cuda, pplb200):
    out, _, _, (att, q, table, lens, cache) = _run_attention(cuda, pplb200, [70, 1, 300, 9], 8, 2, 128, 16, 128, lse=False)
    more = cuda.full_like(out, 5.0)
    att(q[:2], table[:2], lens[:2], out=more[:2])
    assert cuda.equal(more[:2], out[:2]) and bool((more[2:] == 5).all())


@pytest.mark.parametrize("group", [0, 8, 128])
def test_attention_is_the_same_run_after_run(cuda, pplb200, group):
    out, lse, _, (att, q, table, lens, cache) = _run_attention(cuda, pplb200, [9000, 3, 500, 1234], 16, 2, 128, 16, group)
    for fill in (0, 255, 127):
        att.ws[14336:].fill_(fill)  # whatever an earlier call's sums were; the counters of arrivals lie in front of them
        again = cuda.empty_like(lse)
        assert cuda.equal(att(q, table, lens, lse=again), out) and cuda.equal(again, lse)


def test_attention_recovers_from_counters_that_were_left(cuda, pplb200):
    """Calls that overlapped on one workspace, against the rules, may leave counters of arrivals behind: the next call is right again."""
    out, _, _, (att, q, table, lens, cache) = _run_attention(cuda, pplb200, [9000, 3, 500, 1234], 16, 2, 128, 16, 128)
    for left in (1, 5, (1 << 16) + 3):
        att.ws[:3 * 592 * 8].view(cuda.int64).fill_(left)
        assert cuda.equal(att(q, table, lens), out)


@pytest.mark.parametrize("hq,hk,d", [(8, 1, 64), (4, 1, 128), (16, 1, 128), (3, 1, 256), (8, 4, 96)])
@pytest.mark.parametrize("group", [0, 8, -1])
def test_attention_of_few_heads_is_joined_from_many_parts(cuda, pplb200, hq, hk, d, group):
    """One or two sequences over the whole device: hundreds of parts of one item, beside items of one part."""
    for lengths in ([40000], [30001, 0, 5], [700, 20000], [2500]):
        _check_attention(*_run_attention(cuda, pplb200, lengths, hq, hk, d, 48, d if group < 0 else group)[:3])


@pytest.mark.parametrize("group", [0, 8, 128])
def test_attention_shared_pages(cuda, pplb200, group):
    """Sequences that share the pages of a common beginning, and one in which a page stands twice."""
    out, _, _, (att, q, table, lens, cache) = _run_attention(cuda, pplb200, [64, 64, 64], 8, 2, 128, 16, group)
    table[1, :2], table[2, 1] = table[0, :2], table[2, 0]
    got = att(q, table, lens)
    at = cuda.arange(64, device="cuda")
    for b in range(3):
        k, v = _stored(cuda, cache, table[b].long()[at // 16] * 16 + at % 16)
        _check_attention(got[b:b + 1], None, [_attention(cuda, q[b], k, v, at >= 0, att.scale, group == 8)])


@pytest.mark.parametrize("group,d,pages", [(0, 128, 36000), (8, 128, 70000), (128, 128, 70000)])
@pytest.mark.parametrize("order", ["heads", "tokens"])
def test_offsets_beyond_32_bits(cuda, pplb200, group, d, pages, order):
    """Keys and values of more than 2^32 bytes each: the last pages are written, read back and attended to."""
    page, heads, n = 64, 8, 200
    shape = (pages, heads, page) if order == "heads" else (pages, page, heads)
    make = lambda w, t: cuda.empty(shape + (w,), dtype=t, device="cuda")  # noqa: E731
    tensors = [make(d, cuda.int8 if group else cuda.float16) for _ in range(2)] + ([make(d // group, cuda.float16) for _ in range(2)] if group else [])
    assert tensors[0].numel() * tensors[0].element_size() > 1 << 32
    cache = pplb200.PagedKVCache(*(t if order == "heads" else t.transpose(1, 2) for t in tensors))
    g = _gen(cuda, 4)
    table = cuda.tensor([[pages - 1, 0, pages - 2, pages // 2]], dtype=cuda.int32, device="cuda")
    at = cuda.arange(n, device="cuda")
    slots = table[0].long()[at // page] * page + at % page
    k, v = _randn(cuda, g, n, heads, d), _randn(cuda, g, n, heads, d)
    pplb200.kv_cache_write(cache, k, v, slots)
    for x, back in zip((k, v), pplb200.kv_cache_read(cache, slots)):
        if group:
            q, s = _quantized(x.cpu().numpy(), group)
            x = cuda.from_numpy((q.astype(np.float64) * np.repeat(s.astype(np.float64), group, -1)).astype(np.float16)).cuda()
        assert cuda.equal(back, x)
    q = _randn(cuda, g, 1, 16, d)
    att = pplb200.PagedDecodeAttention(cache, 16, 1, 4 * page)
    out = att(q, table, cuda.tensor([n], dtype=cuda.int32, device="cuda"))
    _check_attention(out, None, [_attention(cuda, q[0], *_stored(cuda, cache, slots), at >= 0, att.scale, group == 8)])


def test_two_streams_at_once(cuda, pplb200):
    """Two objects on the same cache, each on its own stream, and rotations and stores beside them: no call disturbs another."""
    out, _, _, (att, q, table, lens, cache) = _run_attention(cuda, pplb200, [5000, 17, 900], 16, 2, 128, 16, 8, lse=False)
    other = pplb200.PagedDecodeAttention(cache, 16, 3, 5008)
    mine = pplb200.PagedKVCache.allocate(40, 16, 2, 128, 128)
    g = _gen(cuda, 12)
    k, v, pos, turns = _randn(cuda, g, 600, 2, 128), _randn(cuda, g, 600, 2, 128), cuda.arange(600, device="cuda"), pplb200.RotaryTable(128)
    plain = pplb200.PagedKVCache.allocate(40, 16, 2, 128, 128)
    pplb200.rotary_kv_cache_write(plain, None, k, v, pos, pos, turns)
    cuda.cuda.synchronize()
    streams = [cuda.cuda.Stream() for _ in range(3)]
    results = []
    for _ in range(20):
        for s, a in zip(streams, (att, other)):
            with cuda.cuda.stream(s):
                results.append(a(q, table, lens))
        with cuda.cuda.stream(streams[2]):
            pplb200.rotary_kv_cache_write(mine, None, k, v, pos, pos, turns)
    cuda.cuda.synchronize()
    assert all(cuda.equal(r, out) for r in results)
    assert cuda.equal(mine.k, plain.k) and cuda.equal(mine.v_scale, plain.v_scale)


def test_attention_parts_join_by_their_lse(cuda, pplb200):
    """Two halves of a context, joined by their sums, are the whole."""
    out, lse, want, (att, q, table, lens, cache) = _run_attention(cuda, pplb200, [512], 8, 2, 128, 16, 0)
    parts = []
    for half in (table[:, :16], table[:, 16:]):
        s = cuda.empty((1, 8), device="cuda")
        parts.append((att(q, half.contiguous(), cuda.tensor([256], dtype=cuda.int32, device="cuda"), lse=s).double(), s.double()))
    total = cuda.logaddexp(parts[0][1], parts[1][1])
    joined = sum(o * cuda.exp(s - total)[..., None] for o, s in parts)
    _, l, bound, lse_bound = want[0]
    assert bool(((joined[0] - want[0][0]).abs() <= 2 * bound).all()) and bool(((total[0] - l).abs() <= 2 * lse_bound).all())


def test_streams_and_graphs(cuda, pplb200):
    """Rotate + store + attend on a stream of its own, and captured and replayed with new tokens: the same as called in order."""
    g = _gen(cuda, 9)
    hq, hk, d, page, n = 8, 2, 128, 16, 90
    table = pplb200.RotaryTable(d)
    caches = [pplb200.PagedKVCache.allocate(12, page, hk, d, 8) for _ in range(2)]
    old = _randn(cuda, g, 2 * n, hk, d), _randn(cuda, g, 2 * n, hk, d)
    pages = cuda.arange(12, dtype=cuda.int32, device="cuda").view(2, 6)
    for c in caches:
        pplb200.kv_cache_write(c, *old, cuda.cat((cuda.arange(n, device="cuda"), 96 + cuda.arange(n, device="cuda"))))
    steps = [_randn(cuda, g, 2, hq + 2 * hk, d) for _ in range(4)]
    rows, lens = cuda.empty_like(steps[0]), cuda.empty(2, dtype=cuda.int32, device="cuda")
    pos, slots = (cuda.empty(2, dtype=cuda.int64, device="cuda") for _ in range(2))

    def step(cache, att):
        q = pplb200.rotary_kv_cache_write(cache, rows[:, :hq], rows[:, hq:hq + hk], rows[:, hq + hk:], pos, slots, table)
        return att(q, pages, lens)

    def feed(i):
        rows.copy_(steps[i])
        lens.fill_(n + 1 + i)
        pos.fill_(n + i)
        slots.copy_(cuda.tensor([n + i, 96 + n + i], device="cuda"))

    atts = [pplb200.PagedDecodeAttention(c, hq, 2, 96) for c in caches]
    want = []
    for i in range(4):
        feed(i)
        want.append(step(caches[0], atts[0]).clone())
    side = cuda.cuda.Stream()
    with cuda.cuda.stream(side):
        side.wait_stream(cuda.cuda.default_stream())
        feed(0)
        assert cuda.equal(step(caches[1], atts[1]), want[0])
        graph = cuda.cuda.CUDAGraph()
        with cuda.cuda.graph(graph, stream=side):
            out = step(caches[1], atts[1])
        for i in (1, 2, 3):
            feed(i)
            graph.replay()
            assert cuda.equal(out, want[i])
    cuda.cuda.synchronize()
    for a, b in ((caches[0].k, caches[1].k), (caches[0].v, caches[1].v), (caches[0].k_scale, caches[1].k_scale)):
        assert cuda.equal(a, b)


def test_a_layers_decode_step(cuda, pplb200):
    """norm + quantize, fused QKV in int32, dequantize + split, rotate + store, attend, W8A8 output projection: the new operators take what
    the others return, and the result is that of the same steps with attention in 64 bits."""
    g = _gen(cuda, 10)
    M, hidden, hq, hk, d, page, n = 5, 1024, 8, 2, 128, 16, 77
    qkv = (hq + 2 * hk) * d
    x, norm = _randn(cuda, g, M, hidden), cuda.ones(hidden, dtype=cuda.float16, device="cuda")
    w = cuda.randint(-127, 128, (qkv, hidden), generator=g, device="cuda", dtype=cuda.int8)
    sn = cuda.full((qkv,), 8192.0 / 73 / hidden ** 0.5, dtype=cuda.float16, device="cuda")
    wo = cuda.randint(-127, 128, (hidden, hq * d), generator=g, device="cuda", dtype=cuda.int8)
    sno = cuda.full((hidden,), 8192.0 / 73 / hidden ** 0.5, dtype=cuda.float16, device="cuda")
    cache = pplb200.PagedKVCache.allocate(M * 5, page, hk, d, 8)
    pages = cuda.randperm(M * 5, generator=g, device="cuda").to(cuda.int32).view(M, 5)
    at = cuda.arange(n, device="cuda")
    old = (pages.long()[:, at // page] * page + at % page).flatten()
    pplb200.kv_cache_write(cache, _randn(cuda, g, M * n, hk, d), _randn(cuda, g, M * n, hk, d), old)
    lens = cuda.full((M,), n + 1, dtype=cuda.int32, device="cuda")
    slots, pos = pages.long()[:, n // page] * page + n % page, cuda.full((M,), n, dtype=cuda.int64, device="cuda")
    table = pplb200.RotaryTable(d)

    _, xq, xs = pplb200.skip_rmsnorm_minmax_quantize_fp16(x, norm)
    acc = pplb200.column_parallel_linear(xq, w, xs, sn, None, hidden, qkv, gather_output=False)
    q, k, v = pplb200.minmax_dequantize_split3_fp16(acc, xs, sn, (hq * d, hk * d, hk * d))
    q, k, v = q.view(M, hq, d), k.view(M, hk, d), v.view(M, hk, d)
    qr = pplb200.rotary_kv_cache_write(cache, q, k, v, pos, slots, table)
    att = pplb200.PagedDecodeAttention(cache, hq, M, 80)
    out = att(qr, pages, lens)
    y = pplb200.W8A8Linear(wo, sno, max_tokens=M)(out.view(M, hq * d))
    cuda.cuda.synchronize()
    _check_rotated(cuda, qr, q, pos, table, False)
    at = cuda.arange(n + 1, device="cuda")
    for b in range(M):
        kr, vr = _stored(cuda, cache, pages.long()[b, at // page] * page + at % page)
        _check_attention(out[b:b + 1], None, [_attention(cuda, qr[b], kr, vr, at >= 0, att.scale, True)])
    oq, os_ = pplb200.minmax_quantize_fp16(out.view(M, hq * d))
    assert cuda.equal(y, pplb200.gemm_i8i8(oq, wo, pplb200.EPI_DEQUANT_F16, os_, sno)) and bool(cuda.isfinite(y).all()) and pplb200.gemm_status() == 0


@pytest.mark.parametrize("group", [0, 8, 128])
def test_an_allocated_cache_may_be_written_on_any_stream(cuda, pplb200, group):
    """The cache is zeroed on a stream that is busy for a while; what another stream stores meanwhile is not zeroed after it."""
    side, busy = cuda.cuda.Stream(), cuda.ones((4096, 4096), dtype=cuda.float16, device="cuda")
    k, slots = cuda.ones((64, 2, 128), dtype=cuda.float16, device="cuda"), cuda.arange(64, device="cuda")

    def stored():
        cache = pplb200.PagedKVCache.allocate(4, 16, 2, 128, group)
        with cuda.cuda.stream(side):
            pplb200.kv_cache_write(cache, k, k, slots)
        cuda.cuda.synchronize()
        return bool((cache.k != 0).all()) and bool((cache.v != 0).all()) and all(t is None or bool((t != 0).all()) for t in (cache.k_scale, cache.v_scale))

    stored()  # memory and kernels are at hand after this
    for _ in range(100):
        busy @ busy
    assert stored()
