"""Rotary positions of several axes, attention over a shared prefix, the bounds of blocks of keys and attention over the blocks that a score
selects, on the GPU, against their definitions in 64 bits.

What is chosen, and what the bounds are, is defined to the bit.  The other tolerances are those of test_attention_gpu.py: sums of half steps, fp16 2^-11 of a
value (weights of the prefix too), and the 32-bit arithmetic in front of it."""
import math

import numpy as np
import pytest

from test_attention_gpu import HALF, TINY, _attention, _cache, _check_attention, _gen, _randn, _stored

pytestmark = pytest.mark.gpu


# ---- rotary positions of several axes ----------------------------------------------------------------------------------

def _dealt(planes, alternating):
    left, out = list(planes), []
    while any(left):
        for axis in range(len(left)):
            n = min(left[axis], 1) if alternating else left[axis]
            out += [axis] * n
            left[axis] -= n
    return out


def _rotated_axes(cuda, x, positions, table, planes, alternating, interleaved):
    """(values, bound) in 64 bits, as for one axis: the angle from the table's words, whole turns taken off in integers."""
    rd = table.rotary_dim
    words, of = [int(w) % (1 << 64) for w in table.turns.cpu().tolist()], _dealt(planes, alternating)
    where = positions.cpu().tolist()
    angle = np.array([[((where[a][t] * w) % (1 << 64)) / 2.0 ** 64 * 2 * math.pi for a, w in zip(of, words)] for t in range(x.shape[0])]).reshape(-1, rd // 2)
    cos, sin = (cuda.from_numpy(f(angle) * table.magnitude).cuda()[:, None] for f in (np.cos, np.sin))
    y = x.double()
    lo, hi = (slice(0, rd, 2), slice(1, rd, 2)) if interleaved else (slice(0, rd // 2), slice(rd // 2, rd))
    a, b = y[..., lo].clone(), y[..., hi].clone()
    y[..., lo], y[..., hi] = a * cos - b * sin, b * cos + a * sin
    bound = y.abs() * HALF + TINY
    for part in (lo, hi):
        bound[..., part] += (a.abs() + b.abs()) * table.magnitude * 2.0 ** -20
    bound[..., rd:] = 0
    return y, bound


@pytest.mark.parametrize("tokens,hq,hk,d,rd,planes", [(1, 1, 1, 16, 16, (3, 5)), (24, 32, 8, 128, 128, (24, 20, 20)), (5, 3, 1, 64, 32, (16,)), (33, 4, 4, 80, 80, (20, 20)), (7, 5, 2, 96, 48, (1, 2, 3, 18)),
                                                      (1025, 16, 16, 64, 64, (0, 16, 16)), (3, 2, 2, 256, 256, (64, 0, 32, 32)), (9001, 9, 2, 128, 96, (7, 23, 18))])
@pytest.mark.parametrize("alternating", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_axes(cuda, pplb200, tokens, hq, hk, d, rd, planes, alternating, interleaved):
    g = _gen(cuda, tokens + rd)
    q, k = _randn(cuda, g, tokens, hq, d), _randn(cuda, g, tokens, hk, d, scale=20.0)
    pos = cuda.randint(-1000, 1 << 20, (len(planes), tokens + 3), generator=g, device="cuda")[:, 1:1 + tokens]  # rows further apart than long
    table = pplb200.RotaryTable(rd, axes=planes, alternating=alternating, restart=interleaved)
    qo, ko = pplb200.rotary_fp16(q, k, pos, table, interleaved)
    for got, x in ((qo, q), (ko, k)):
        want, bound = _rotated_axes(cuda, x, pos, table, planes, alternating, interleaved)
        assert bool(((got.double() - want).abs() <= bound).all())


def test_rotary_axes_far_positions(cuda, pplb200):
    far = [0, 1, -1, 131071, (1 << 31) - 1, -(1 << 31), 1 << 40, (1 << 63) - 1, -(1 << 63)]
    pos = cuda.tensor([far, far[::-1], [7] * len(far), far], device="cuda")
    q = _randn(cuda, _gen(cuda, 2), len(far), 4, 128)
    table = pplb200.RotaryTable(128, base=500000.0, scaling="yarn", factor=16.0, original_length=8192, keep_turns=32, stretch_turns=1, axes=(16, 16, 16, 16), alternating=True)
    got = pplb200.rotary_fp16(q, None, pos, table)[0]
    want, bound = _rotated_axes(cuda, q, pos, table, (16,) * 4, True, False)
    assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens", [5, 3001])
def test_equal_positions_on_all_axes_are_one_axis(cuda, pplb200, tokens, interleaved):
    """Text among the images: bit for bit what the call with one axis gives, in place too."""
    g = _gen(cuda, 3)
    rows = _randn(cuda, g, tokens, 14, 96)
    q, k = rows[:, 1:9], rows[:, 9:11]
    pos = cuda.randint(0, 100000, (tokens,), generator=g, device="cuda")
    one = pplb200.rotary_fp16(q, k, pos, pplb200.RotaryTable(64), interleaved)
    table = pplb200.RotaryTable(64, axes=(12, 10, 10), alternating=True)
    every = pos.expand(3, -1).contiguous()
    before = rows.clone()
    several = pplb200.rotary_fp16(q, k, every, table, interleaved, q_out=q, k_out=k)
    assert cuda.equal(several[0], one[0]) and cuda.equal(several[1], one[1])
    assert cuda.equal(rows[:, :1], before[:, :1]) and cuda.equal(rows[:, 11:], before[:, 11:])


@pytest.mark.parametrize("tokens,hq,hk,d,rd,page", [(1, 8, 1, 128, 128, 16), (37, 7, 7, 96, 48, 5), (1030, 8, 2, 64, 64, 64), (3, 4, 2, 256, 128, 1), (9001, 10, 3, 128, 128, 16)])
@pytest.mark.parametrize("group", [0, 8, -1])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotating_write_of_several_axes_is_the_two_calls(cuda, pplb200, tokens, hq, hk, d, rd, page, group, interleaved):
    group = d if group < 0 else group
    g = _gen(cuda, tokens)
    rows = _randn(cuda, g, tokens, hq + 2 * hk, d)
    q, k, v = rows[:, :hq], rows[:, hq:hq + hk], rows[:, hq + hk:]
    pos = cuda.randint(0, 1 << 20, (3, tokens), generator=g, device="cuda")
    pages = (tokens + page - 1) // page + 1
    slots = cuda.randperm(pages * page, generator=g, device="cuda")[:tokens]
    slots[0] = -5
    table = pplb200.RotaryTable(rd, axes=(rd // 4, rd // 8, rd // 8))
    one, two = (pplb200.PagedKVCache.allocate(pages, page, hk, d, group) for _ in range(2))
    q1 = pplb200.rotary_kv_cache_write(one, q, k, v, pos, slots, table, interleaved)
    q2, k2 = pplb200.rotary_fp16(q, k, pos, table, interleaved)
    pplb200.kv_cache_write(two, k2, v, slots)
    assert cuda.equal(q1, q2)
    for n in ("k", "v", "k_scale", "v_scale"):
        a, b = getattr(one, n), getattr(two, n)
        assert (a is None and b is None) or cuda.equal(a, b)


# ---- bounds of blocks ----------------------------------------------------------------------------------------------------

def _outer_scale(amax):
    """The smallest fp16, 2^-24 at least, of which 127 reach amax (64 bits)."""
    exact = amax / 127
    with np.errstate(over="ignore"):
        s = exact.astype(np.float16)
        s = np.where(s.astype(np.float64) < exact, np.nextafter(s, np.float16(np.inf)), s)
    return np.maximum(s, np.float16(2.0 ** -24))


def _bounds(cuda, cache, block):
    """int8 [pages, heads, blocks, 2, d], fp16 [pages, heads, blocks] of every block of the cache."""
    k = cache.k.cpu().numpy().astype(np.float64)
    if cache.quant_group:
        k = k * np.repeat(cache.k_scale.cpu().numpy().astype(np.float64), cache.quant_group, -1)
    k = k.reshape(k.shape[0], k.shape[1], -1, block, k.shape[3])
    bad = ~np.isfinite(k).all((-1, -2))
    k[bad] = 0
    lo, hi = k.min(-2), k.max(-2)
    s = _outer_scale(np.maximum(np.abs(lo), np.abs(hi)).max(-1))
    bad |= np.isinf(s)
    s64 = np.where(bad, 1.0, s.astype(np.float64))[..., None]
    both = np.stack((np.floor(lo / s64), np.ceil(hi / s64)), -2)
    both[bad] = 0
    return cuda.from_numpy(both.astype(np.int8)).cuda(), cuda.from_numpy(np.where(bad, np.float16(np.inf), s)).cuda()


def _filled(cuda, pplb200, g, pages, page, heads, d, group, order):
    cache = _cache(cuda, pplb200, pages, page, heads, d, group, order, 0)
    k, v = _randn(cuda, g, pages * page, heads, d), _randn(cuda, g, pages * page, heads, d)
    k *= cuda.exp(cuda.randn((pages * page, heads, 1), generator=g, device="cuda") * 2).to(cuda.float16)
    pplb200.kv_cache_write(cache, k, v, cuda.arange(pages * page, device="cuda"))
    return cache


@pytest.mark.parametrize("page,block,heads,d", [(16, 16, 3, 128), (64, 16, 1, 64), (64, 64, 8, 128), (48, 16, 2, 96), (96, 48, 5, 256), (256, 256, 1, 128), (32, 32, 37, 64)])
@pytest.mark.parametrize("group", [0, 8, -1])
@pytest.mark.parametrize("order", ["heads", "tokens"])
def test_bounds(cuda, pplb200, page, block, heads, d, group, order):
    """Of blocks whose last slot is named, and of no others."""
    g = _gen(cuda, page + d)
    pages = 7
    cache = _filled(cuda, pplb200, g, pages, page, heads, d, d if group < 0 else group, order)
    want, scale = _bounds(cuda, cache, block)
    for named in (1, 5, pages * page // block):
        bounds = pplb200.KeyBlockBounds(cache, block)
        bounds.bounds.fill_(55)
        bounds.scales.fill_(55)
        done = cuda.randperm(pages * page // block, generator=g, device="cuda")[:named]
        slots = cuda.cat([done * block + block - 1, done[: named // 2] * block, cuda.tensor([-1, pages * page + block - 1, -(1 << 40)], device="cuda")])
        pplb200.key_bounds_update(bounds, slots[cuda.randperm(len(slots), generator=g, device="cuda")])
        of = (done // (page // block), done % (page // block))
        hit = cuda.zeros((pages, page // block), dtype=cuda.bool, device="cuda")
        hit[of] = True
        hit = hit[:, None].expand(-1, heads, -1)
        assert cuda.equal(bounds.bounds[hit], want[hit]) and cuda.equal(bounds.scales[hit], scale[hit])
        assert bool((bounds.bounds[~hit] == 55).all()) and bool((bounds.scales[~hit] == 55).all())
        lo, hi = pplb200.key_bounds_read(bounds, cuda.cat([done, cuda.tensor([-1, pages * page // block], device="cuda")]))
        for x, got in ((0, lo), (1, hi)):
            assert cuda.equal(got[:named], (want[:, :, :, x].float() * scale[..., None].float())[of[0], :, of[1]]) and not got[named:].any()


def test_bounds_of_a_prompt(cuda, pplb200):
    """More slots than CTAs, every block of them; and none that ends one."""
    g = _gen(cuda, 4)
    cache = _filled(cuda, pplb200, g, 300, 64, 4, 64, 0, "heads")
    for block in (16, 32, 64):
        bounds = pplb200.KeyBlockBounds(cache, block)
        slots = cuda.arange(300 * 64, device="cuda").view(-1, 64)[cuda.randperm(300, generator=g, device="cuda")].flatten()
        pplb200.key_bounds_update(bounds, slots[slots % block != block - 1])
        assert not bounds.bounds.any() and not bounds.scales.any()
        pplb200.key_bounds_update(bounds, slots)
        want, scale = _bounds(cuda, cache, block)
        assert cuda.equal(bounds.bounds, want) and cuda.equal(bounds.scales, scale)


@pytest.mark.parametrize("group", [0, 8, 128])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_bounds_of_special_values(cuda, pplb200, group, value):
    """A key that is infinite or NaN, the largest and the smallest numbers, and zeros alone."""
    cache = _cache(cuda, pplb200, 4, 16, 2, 128, group, "heads", 0)
    k = cuda.zeros((64, 2, 128), dtype=cuda.float16, device="cuda")
    k[5, 0, 77] = value
    k[16:32, 0], k[20, 0, 3], k[21, 0, 4] = 1.0, 65504.0, -65504.0
    k[40, 1, 9] = 2.0 ** -24
    pplb200.kv_cache_write(cache, k, k, cuda.arange(64, device="cuda"))
    bounds = pplb200.KeyBlockBounds(cache, 16)
    pplb200.key_bounds_update(bounds, cuda.arange(64, device="cuda"))
    want, scale = _bounds(cuda, cache, 16)
    assert cuda.equal(bounds.bounds, want) and cuda.equal(bounds.scales, scale) and scale[0, 0, 0] == math.inf
    lo, hi = pplb200.key_bounds_read(bounds, cuda.arange(4, device="cuda"))
    assert bool((lo[0, 0] == -math.inf).all()) and bool((hi[0, 0] == math.inf).all()) and not lo[3].any() and not hi[3].any()


def test_bounds_of_scales_beyond_fp16(cuda, pplb200):
    """An int8 cache of another program: scales near fp16's largest, negative ones, a value of -128."""
    cache = _cache(cuda, pplb200, 2, 16, 1, 64, 64, "heads", 0)
    g = _gen(cuda, 9)
    cache.k.copy_(cuda.randint(-127, 128, cache.k.shape, generator=g, device="cuda"))
    cache.k_scale.copy_(cuda.randn(cache.k_scale.shape, generator=g, device="cuda") * 20000)
    cache.k[1, 0, 3, 7], cache.k_scale[1, 0, 3] = -128, 65504.0
    bounds = pplb200.KeyBlockBounds(cache, 16)
    pplb200.key_bounds_update(bounds, cuda.arange(32, device="cuda"))
    want, scale = _bounds(cuda, cache, 16)
    assert scale[1, 0, 0] == math.inf and cuda.equal(bounds.bounds, want) and cuda.equal(bounds.scales, scale)


# ---- attention over chosen blocks ----------------------------------------------------------------------------------------

def _choice(cuda, q, bounds, table, n, first, last, top, pages):
    """The blocks of one sequence, for each key head in ascending order: the definition in whole numbers."""
    cache, block = bounds.cache, bounds.block
    per_page, hk = cache.page_size // block, cache.kv_heads
    blocks = -(-n // block)
    if blocks <= first + last + top:
        return [list(range(blocks))] * hk
    number = np.arange(first, blocks - last)
    page, x = table.cpu().numpy().astype(np.int64)[number // per_page], number % per_page
    there = (page >= 0) & (page < pages)
    page = np.where(there, page, 0)
    low, high = (bounds.bounds[:, :, :, i].cpu().numpy().astype(np.int64) for i in (0, 1))
    scales = bounds.scales.cpu().numpy()
    queries = q.cpu().numpy().astype(np.float64).reshape(hk, -1, q.shape[-1])
    out = []
    for h in range(hk):
        best = np.full(len(number), -np.inf)
        for row in queries[h]:
            if not np.isfinite(row).all():
                continue
            s = np.float64(_outer_scale(np.abs(row).max()[None])[0])
            q8 = np.rint(row / s).astype(np.int64)
            dot = np.maximum(q8 * low[page, h, x], q8 * high[page, h, x]).sum(-1)
            with np.errstate(invalid="ignore"):
                best = np.fmax(best, (dot * (s * scales[page, h, x].astype(np.float64))).astype(np.float32).astype(np.float64))
        best = np.where(np.isinf(scales[page, h, x]), np.inf, best)
        order = sorted(range(len(number)), key=lambda i: (not there[i], -best[i], i))
        out.append(sorted(list(range(first)) + [first + i for i in order[:top]] + list(range(blocks - last, blocks))))
    return out


def _run_sparse(cuda, pplb200, lengths, hq, hk, d, page, block, group, first, last, top, order="heads", seed=0, extra_pages=0, spoil=None, q_scale=2.0):
    g = _gen(cuda, seed + 31 * len(lengths) + d)
    counts = [-(-n // page) for n in lengths]
    width = max(counts + [1]) + extra_pages
    pages = sum(counts) + 2
    cache = _filled(cuda, pplb200, g, pages, page, hk, d, group, order)
    bounds = pplb200.KeyBlockBounds(cache, block)
    pplb200.key_bounds_update(bounds, cuda.arange(pages * page, device="cuda"))
    table = cuda.full((len(lengths), width), pages + 1000, dtype=cuda.int32, device="cuda")
    at = cuda.randperm(pages, generator=g, device="cuda").to(cuda.int32)
    for b, c in enumerate(counts):
        table[b, :c] = at[sum(counts[:b]):sum(counts[:b + 1])]
    q = _randn(cuda, g, len(lengths), hq, d, scale=q_scale)
    if spoil:
        spoil(q, table, cache, bounds)
    att = pplb200.BlockSparseDecodeAttention(bounds, hq, len(lengths), width * page, first, last, top)
    out = cuda.full((len(lengths), hq, d), 7.0, dtype=cuda.float16, device="cuda")
    lse = cuda.full((len(lengths), hq), 7.0, device="cuda")
    blocks = cuda.full((len(lengths), hk, first + last + top), 7, dtype=cuda.int32, device="cuda")
    lens = cuda.tensor(lengths, dtype=cuda.int32, device="cuda")
    att(q, table, lens, out=out, lse=lse, blocks=blocks)
    want, shared = [], hq // hk
    for b, n in enumerate(lengths):
        n = min(max(n, 0), width * page)
        chosen = _choice(cuda, q[b], bounds, table[b], n, first, last, top, pages)
        parts = []
        for h in range(hk):
            assert blocks[b, h].tolist() == chosen[h] + [-1] * (first + last + top - len(chosen[h])), (b, h)
            token = (cuda.tensor(chosen[h], dtype=cuda.int64, device="cuda")[:, None] * block + cuda.arange(block, device="cuda")).flatten()
            token = token[token < n]
            of = table[b].long()[token // page]
            seen = (of >= 0) & (of < pages)
            k, v = _stored(cuda, cache, cuda.where(seen, of, 0) * page + token % page)
            parts.append(_attention(cuda, q[b, h * shared:(h + 1) * shared], k[:, h:h + 1], v[:, h:h + 1], seen, att.scale, group == 8))
        want.append(tuple(cuda.cat(x) for x in zip(*parts)))
    return out, lse, want, (att, q, table, lens, cache, bounds, blocks)


@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("group", [0, 8, -1])
@pytest.mark.parametrize("hq,hk", [(1, 1), (8, 1), (10, 2), (32, 2), (5, 5)])
def test_sparse_heads_and_types(cuda, pplb200, d, group, hq, hk):
    _check_attention(*_run_sparse(cuda, pplb200, [1, 0, 16, 17, 95, 96, 97, 112, 113, 500, 1025], hq, hk, d, 16, 16, d if group < 0 else group, 1, 2, 3)[:3])


@pytest.mark.parametrize("page,block", [(16, 16), (64, 16), (64, 64), (48, 16), (96, 48), (256, 32)])
@pytest.mark.parametrize("group", [0, 8, 128])
@pytest.mark.parametrize("order", ["heads", "tokens"])
def test_sparse_pages_and_orders(cuda, pplb200, page, block, group, order):
    _check_attention(*_run_sparse(cuda, pplb200, [5, 1200, 777, 64, 3001], 8, 2, 128, page, block, group, 1, 1, 4, order=order, seed=page)[:3])


@pytest.mark.parametrize("first,last,top", [(0, 1, 0), (0, 1, 1), (3, 1, 0), (0, 4, 9), (2, 2, 100), (0, 1, 200), (5, 8, 31)])
def test_sparse_choices(cuda, pplb200, first, last, top):
    _check_attention(*_run_sparse(cuda, pplb200, [2000, 100, 1, 2001, 1600, 3184], 8, 2, 64, 16, 16, 0, first, last, top)[:3])


@pytest.mark.parametrize("lengths,top", [([70001], 100), ([140000, 9], 1), ([40000, 33333, 16], 1500)])
@pytest.mark.parametrize("group", [0, 128])
def test_sparse_long(cuda, pplb200, lengths, top, group):
    """Choices that a cluster of CTAs makes, thresholds within and between the CTAs' shares."""
    _check_attention(*_run_sparse(cuda, pplb200, lengths, 4, 1, 128, 64, 16, group, 1, 2, top)[:3])


def test_sparse_many_sequences(cuda, pplb200):
    rng = np.random.default_rng(5)
    lengths = [int(n) for n in rng.integers(0, 400, 300)]
    _check_attention(*_run_sparse(cuda, pplb200, lengths, 4, 2, 64, 32, 16, 64, 1, 1, 5)[:3])


def test_sparse_more_scores_than_a_launch_has_room_for_unasked(cuda, pplb200):
    """Over 8192 blocks a CTA, which shared memory has to be asked for; a long table, a shorter sequence."""
    _check_attention(*_run_sparse(cuda, pplb200, [180000, 100], 1, 1, 64, 16, 16, 64, 1, 1, 3, extra_pages=240000)[:3])


def test_sparse_of_few_blocks_is_attention_over_all(cuda, pplb200):
    lengths = [700, 1, 0, 333]
    out, lse, _, (att, q, table, lens, cache, _, _) = _run_sparse(cuda, pplb200, lengths, 8, 2, 128, 16, 16, 0, 2, 2, 60)
    full_lse = cuda.empty_like(lse)
    full = pplb200.PagedDecodeAttention(cache, 8, 4, table.shape[1] * 16)(q, table, lens, lse=full_lse)
    assert cuda.equal(out, full) and cuda.equal(lse, full_lse)


@pytest.mark.parametrize("top", [1, 7, 40])
def test_sparse_ties_go_to_the_lowest(cuda, pplb200, top):
    """Equal bounds everywhere but for a few blocks: what is at the threshold is taken from the front."""
    def spoil(q, table, cache, bounds):
        bounds.bounds[:] = bounds.bounds[0, 0, 0]
        bounds.scales.fill_(1.0)
        bounds.scales[table[0, 33].long()] = 2.0
        bounds.scales[table[0, 50].long()] = 0.5
        bounds.scales[table[0, 51].long()] = 0.0
    _check_attention(*_run_sparse(cuda, pplb200, [1500, 800], 4, 2, 128, 16, 16, 0, 1, 1, top, spoil=spoil)[:3])


@pytest.mark.parametrize("group", [0, 128])
def test_sparse_holes_and_infinite_scales(cuda, pplb200, group):
    """Blocks with an infinite scale come first, those on pages that are not there last, and take no part; rows with holes only, or chosen ones."""
    def spoil(q, table, cache, bounds):
        table[0, 3], table[0, 40], table[0, 7] = -1, 1 << 30, -(1 << 31)
        bounds.scales[table[0, 20].long(), 0] = math.inf
        bounds.scales[table[0, 21].long(), 1] = math.inf
        bounds.bounds[table[0, 21].long(), 1] = 0
        table[1, :] = -5
        table[2, 2:60] = -1
    out, lse, want, (*_, blocks) = _run_sparse(cuda, pplb200, [1000, 900, 1200], 8, 2, 128, 16, 16, group, 1, 1, 12, spoil=spoil)
    _check_attention(out, lse, want)
    assert not out[1].any() and bool((lse[1] == -math.inf).all())
    assert 20 in blocks[0, 0].tolist() and 21 in blocks[0, 1].tolist() and not {3, 7, 40} & set(blocks[0].flatten().tolist())


def test_sparse_queries_without_a_say(cuda, pplb200):
    """An infinity or NaN in a query head: its own output is lost, its neighbours' choice is as if it were not there; all of them: the lowest blocks."""
    def spoil(q, table, cache, bounds):
        q[0, 1, 5], q[0, 4:8, 0] = math.nan, math.inf
        q[1, :, 3] = math.nan
    out, lse, want, _ = _run_sparse(cuda, pplb200, [1000, 700], 8, 2, 128, 16, 16, 0, 1, 1, 9, spoil=spoil)
    _check_attention(out[:1, [0, 2, 3]], lse[:1, [0, 2, 3]], [tuple(x[[0, 2, 3]] for x in want[0])])
    assert bool(out[0, 1].isnan().all()) and bool(out[1].isnan().all())


@pytest.mark.parametrize("scale", [0.0, 6e-8, 1e-3, 60000.0])
def test_sparse_queries_of_all_sizes(cuda, pplb200, scale):
    def spoil(q, table, cache, bounds):
        q.copy_((q.float().clamp(-1, 1) * scale).to(cuda.float16))
    _, _, _, (att, q, table, lens, cache, bounds, blocks) = _run_sparse(cuda, pplb200, [1000], 4, 2, 128, 16, 16, 0, 1, 1, 9, spoil=spoil, q_scale=1.0)
    assert blocks.shape == (1, 2, 11)  # what they are has been checked


def test_sparse_lengths_beyond_the_table_and_negative(cuda, pplb200):
    _check_attention(*_run_sparse(cuda, pplb200, [500, 640], 8, 2, 128, 16, 16, 0, 1, 1, 4)[:3])
    out, lse, want, (att, q, table, lens, *_) = _run_sparse(cuda, pplb200, [640, 100, 33], 8, 2, 128, 16, 16, 0, 1, 1, 4)
    odd = cuda.tensor([641, -3, 33], dtype=cuda.int32, device="cuda")
    again = att(q, table, odd)
    assert cuda.equal(again[0], out[0]) and not again[1].any() and cuda.equal(again[2], out[2])


@pytest.mark.parametrize("group", [0, 8, 128])
def test_bounds_hold_every_key(cuda, pplb200, group):
    """No key is outside of its block's bounds, so that no product of a block's keys with a query is above what the bounds give."""
    g = _gen(cuda, 12)
    cache = _filled(cuda, pplb200, g, 30, 32, 2, 128, group, "heads")
    bounds = pplb200.KeyBlockBounds(cache, 16)
    pplb200.key_bounds_update(bounds, cuda.arange(30 * 32, device="cuda"))
    lo, hi = (x.double().repeat_interleave(16, 0) for x in pplb200.key_bounds_read(bounds, cuda.arange(60, device="cuda")))
    k, _ = _stored(cuda, cache, cuda.arange(30 * 32, device="cuda"))
    assert bool((lo <= k).all()) and bool((k <= hi).all())
    q = _randn(cuda, g, 2, 128).double()
    assert bool((cuda.einsum("hd,thd->ht", q, k) <= (cuda.maximum(q * lo, q * hi)).sum(-1).T + 1e-9).all())


# ---- attention over a shared prefix --------------------------------------------------------------------------------------

def _run_prefix(cuda, pplb200, prefix, lengths, hq, hk, d, page, group, order="heads", seed=0, holes=(), prefix_holes=(), extra_pages=0, scale=None, q_scale=2.0, poison=True, rising=0.0):
    """As _run_attention: pages scattered over a cache in which everything that nobody owns is NaN."""
    g = _gen(cuda, seed + 17 * len(lengths) + d + prefix)
    counts = [-(-max(n, 0) // page) for n in [prefix] + lengths]
    pages = sum(counts) + 3
    cache = _cache(cuda, pplb200, pages, page, hk, d, group, order, 1)
    cache.v.fill_(2)
    for t in ((cache.k_scale, cache.v_scale) if group else (cache.k, cache.v)) if poison else ():
        t.fill_(float("nan"))
    at = cuda.randperm(pages, generator=g, device="cuda").to(cuda.int32)
    tables, written = [], []
    for i, (n, c) in enumerate(zip([prefix] + lengths, counts)):
        table = cuda.full((max(counts[1:] + [1] if i else [counts[0]]) + extra_pages,), pages + 1000, dtype=cuda.int32, device="cuda")
        table[:c] = at[sum(counts[:i]):sum(counts[:i + 1])]
        n = max(n, 0)
        token = cuda.arange(n, device="cuda")
        slots = table.long()[token // page] * page + token % page if n else token
        k, v = _randn(cuda, g, n, hk, d), _randn(cuda, g, n, hk, d)
        if rising:
            k[..., 0] += (cuda.linspace(0, rising, n, device="cuda")).to(cuda.float16)[:, None]
        if n:
            pplb200.kv_cache_write(cache, k, v, slots)
        tables.append(table)
        written.append(_stored(cuda, cache, slots) if n else (k, v))
    for b, i, value in holes:
        tables[1 + b][i] = value
    for i, value in prefix_holes:
        tables[0][i] = value
    q = _randn(cuda, g, len(lengths), hq, d, scale=q_scale)
    att = pplb200.SharedPrefixDecodeAttention(cache, hq, len(lengths), len(tables[1]) * page if lengths else 0, len(tables[0]) * page, scale=scale)
    out = cuda.full((len(lengths), hq, d), 7.0, dtype=cuda.float16, device="cuda")
    lse = cuda.full((len(lengths), hq), 7.0, device="cuda")
    call = (q, tables[0], cuda.tensor([prefix], dtype=cuda.int32, device="cuda"), cuda.stack(tables[1:]), cuda.tensor(lengths, dtype=cuda.int32, device="cuda"))
    att(*call, out=out, lse=lse)
    want, shared = [], []
    for i, table in enumerate(tables):
        of = table.long()[cuda.arange(max(0, ([prefix] + lengths)[i]), device="cuda") // page]
        shared.append((of >= 0) & (of < pages))
    for b, n in enumerate(lengths):
        k, v = (cuda.cat([written[0][x], written[1 + b][x]]) for x in (0, 1))
        seen = cuda.cat([shared[0], shared[1 + b]])
        want.append(_attention(cuda, q[b], k, v, seen if n >= 0 else cuda.zeros_like(seen), att.scale, group > 0))  # v of int8 caches is rounded to fp16
    return out, lse, want, (att, call, cache)


@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("group", [0, 8, -1])
@pytest.mark.parametrize("hq,hk", [(1, 1), (4, 4), (10, 2), (32, 2), (40, 1)])
def test_prefix_heads_and_types(cuda, pplb200, d, group, hq, hk):
    """One to 440 rows a key head; sequences with nothing of their own, one that is none."""
    group = d if group < 0 else group
    _check_attention(*_run_prefix(cuda, pplb200, 333, [1, 0, 2, 15, 16, 17, -1, 64, 65, 130, 333], hq, hk, d, 16, group)[:3])
    _check_attention(*_run_prefix(cuda, pplb200, 130, [3], hq, hk, d, 16, group)[:3])


@pytest.mark.parametrize("prefix", [0, 1, 15, 16, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1000, 5003])
@pytest.mark.parametrize("group", [0, 8, 128])
@pytest.mark.parametrize("batch", [2, 40])
def test_prefix_lengths(cuda, pplb200, prefix, group, batch):
    _check_attention(*_run_prefix(cuda, pplb200, prefix, [7, 0, -2, 30][:batch] + list(range(batch - 4)), 8, 2, 128, 16, group)[:3])


@pytest.mark.parametrize("page", [1, 3, 8, 24, 64, 1000])
@pytest.mark.parametrize("group", [0, 8, 128])
@pytest.mark.parametrize("order", ["heads", "tokens"])
def test_prefix_pages_and_orders(cuda, pplb200, page, group, order):
    _check_attention(*_run_prefix(cuda, pplb200, 777, [5, 200, 1, 64] * 6, 8, 2, 128, page, group, order=order, seed=page)[:3])


@pytest.mark.parametrize("prefix,batch,hq,hk,d,group", [(20011, 3, 8, 8, 128, 128), (9000, 70, 16, 2, 128, 0), (9000, 33, 16, 2, 64, 8), (3000, 700, 4, 1, 128, 128), (3000, 257, 1, 1, 96, 0), (6001, 20, 16, 1, 256, 8),
                                                        (12345, 256, 8, 1, 128, 0)])
def test_prefix_long_and_many(cuda, pplb200, prefix, batch, hq, hk, d, group):
    rng = np.random.default_rng(batch)
    _check_attention(*_run_prefix(cuda, pplb200, prefix, [int(n) for n in rng.integers(-1, 60, batch)], hq, hk, d, 64, group)[:3])


@pytest.mark.parametrize("group", [0, 8, 128])
@pytest.mark.parametrize("batch", [1, 24])
def test_prefix_holes(cuda, pplb200, group, batch):
    """Pages of the prefix and of the sequences that are not there; sequences of which nothing is seen at all."""
    lengths = [100, 0, 33, 16] * 6
    holes = [(0, 0, -1), (0, 3, 1 << 30), (2, 0, -7)]
    _check_attention(*_run_prefix(cuda, pplb200, 700, lengths[:batch], 8, 2, 128, 16, group, holes=holes[:2] if batch == 1 else holes, prefix_holes=[(0, -1), (7, 1 << 30), (8, -3), (20, -(1 << 31)), (43, -1)])[:3])
    out, lse, want, _ = _run_prefix(cuda, pplb200, 40, lengths[:batch], 8, 2, 128, 16, group, prefix_holes=[(0, -1), (1, -1), (2, 1 << 30)])
    _check_attention(out, lse, want)
    if batch > 1:
        assert not out[1].any() and bool((lse[1] == -math.inf).all())


@pytest.mark.parametrize("scale,q_scale", [(None, 20.0), (1.0, 8.0), (0.0, 1.0), (-0.1, 2.0), (1e-6, 1.0)])
@pytest.mark.parametrize("group", [0, 8, 128])
def test_prefix_scores_of_all_sizes(cuda, pplb200, scale, q_scale, group):
    _check_attention(*_run_prefix(cuda, pplb200, 1500, [40, 333, 0] * 8, 8, 2, 128, 16, group, scale=scale, q_scale=q_scale)[:3])


@pytest.mark.parametrize("rising", [60.0, -60.0])
@pytest.mark.parametrize("group", [0, 128])
def test_prefix_scores_that_rise_or_fall(cuda, pplb200, rising, group):
    """The reference exponent moves with every tile, or never after the first."""
    _check_attention(*_run_prefix(cuda, pplb200, 2500, [1, 100] * 20, 4, 1, 128, 16, group, q_scale=4.0, scale=0.3, rising=rising)[:3])


@pytest.mark.parametrize("batch", [1, 40])
def test_prefix_queries_of_padding_reach_nobody(cuda, pplb200, batch):
    """Rows that are no sequence may hold anything, NaN among it."""
    out, lse, want, (att, call, _) = _run_prefix(cuda, pplb200, 500, [9, -1] * batch, 8, 2, 128, 16, 0)
    call[0][1::2] = math.nan
    again_lse = cuda.empty_like(lse)
    again = att(*call, lse=again_lse)
    assert cuda.equal(again, out) and cuda.equal(again_lse, lse) and not again[1::2].any() and bool((lse[1::2] == -math.inf).all())


@pytest.mark.parametrize("value", [math.inf, math.nan])
@pytest.mark.parametrize("group", [0, 8, 128])
@pytest.mark.parametrize("batch", [1, 24])
def test_prefix_special_values(cuda, pplb200, value, group, batch):
    """A key of the prefix that is lost makes its head's outputs NaN; a value that is lost its own dimensions (those that share its scale)."""
    d = 128
    out, _, _, (att, call, cache) = _run_prefix(cuda, pplb200, 300, [5] * batch, 8, 2, d, 16, group, poison=False)
    place = (int(call[1][6]), 1, 3)
    k, v = _stored(cuda, cache, cuda.tensor([place[0] * 16 + 3], device="cuda"))
    k, v = k.to(cuda.float16), v.to(cuda.float16)
    slot = cuda.tensor([place[0] * 16 + 3], device="cuda")
    lost = v.clone()
    lost[0, 1, 21] = value
    pplb200.kv_cache_write(cache, k, lost, slot)
    got = att(*call)
    odd = cuda.zeros_like(out, dtype=cuda.bool)
    at = 21 // max(group, 1) * max(group, 1)
    odd[:, 4:, at:at + max(group, 1)] = True
    assert cuda.equal(~cuda.isfinite(got), odd)
    lost = k.clone()
    lost[0, 1, 21] = math.nan
    pplb200.kv_cache_write(cache, lost, v, slot)
    got = att(*call)
    assert bool(got[:, 4:].isnan().all()) and bool(cuda.isfinite(got[:, :4]).all())


def test_prefix_beyond_its_table_and_negative(cuda, pplb200):
    out, lse, want, (att, call, _) = _run_prefix(cuda, pplb200, 160, [20, 40] * 10, 8, 2, 128, 16, 0)
    more = list(call)
    more[2] = cuda.tensor([100000], dtype=cuda.int32, device="cuda")
    assert cuda.equal(att(*more), out)
    more[2] = cuda.tensor([-4], dtype=cuda.int32, device="cuda")
    none = list(call)
    none[2] = cuda.tensor([0], dtype=cuda.int32, device="cuda")
    assert cuda.equal(att(*more), att(*none))


@pytest.mark.parametrize("group", [0, 128])
def test_prefix_strided_and_in_place(cuda, pplb200, group):
    """q inside the fused projection's rows, the output where q was; fewer sequences than the object was made for."""
    out, _, _, (att, call, _) = _run_prefix(cuda, pplb200, 700, [20, 3] * 10, 8, 2, 128, 16, group)
    rows = cuda.full((20, 12, 128), 3.0, dtype=cuda.float16, device="cuda")
    rows[:, :8] = call[0]
    q = rows[:, :8]
    assert att(q, *call[1:], out=q) is q and cuda.equal(q, out) and bool((rows[:, 8:] == 3.0).all())
    few = att(call[0][:3].contiguous(), call[1], call[2], call[3][:3], call[4][:3])
    assert bool(((few - out[:3]).abs() <= out[:3].abs() * 4 * HALF + 1e-3).all())


@pytest.mark.parametrize("hq,hk,d,group", [(8, 2, 128, 0), (8, 1, 64, 64), (32, 1, 256, 8)])
def test_prefix_batches_of_all_sizes_on_one_workspace(cuda, pplb200, hq, hk, d, group):
    """One object for them all, in turn: what a large batch leaves in the workspace is nothing to a small one, whose kernels are others."""
    lengths = [4000, 3, 0, 777, 1200] * 13
    _, _, _, (att, call, cache) = _run_prefix(cuda, pplb200, 3000, lengths, hq, hk, d, 16, group)
    for n in (65, 1, 64, 2, 33, 1, 65, 16, 3, 9):
        mine = pplb200.SharedPrefixDecodeAttention(cache, hq, n, att.max_pages * 16, 3000)
        part = (call[0][:n], call[1], call[2], call[3][:n], call[4][:n])
        assert cuda.equal(att(*part), mine(*part)), n


@pytest.mark.parametrize("prefix,batch,hq,hk,d,group,own", [
    (900, 32, 16, 4, 128, 0, 1000),     # own tokens by a CTA each, on SMs that are left to them
    (900, 40, 8, 8, 64, 64, 513),       # the same, where they fill them all
    (9000, 32, 32, 8, 128, 0, 900),     # no SMs left: shared out
    (300, 5, 4, 1, 96, 8, 511),         # few items, a CTA each
    (300, 5, 4, 1, 256, 0, 2100),       # few and long: shared out
    (40, 300, 4, 4, 128, 128, 130),     # more CTAs than the device holds
    (9000, 4, 4, 4, 128, 8, 600),       # few rows of an int8 cache, which the decode kernel takes
    (9000, 2, 4, 1, 256, 8, 40),
    (9000, 4, 32, 8, 256, 256, 50),
    (17000, 4, 32, 8, 96, 96, 50),
    (17000, 16, 8, 8, 64, 8, 50),
])
def test_prefix_own_tokens_dealt_out(cuda, pplb200, prefix, batch, hq, hk, d, group, own):
    lengths = [own, 0, -1, 1, own - 1, own // 2, 17] * (batch // 7) + [own] * (batch % 7)
    _check_attention(*_run_prefix(cuda, pplb200, prefix, lengths, hq, hk, d, 16, group)[:3])


def test_prefix_without_own_pages(cuda, pplb200):
    """A table of no pages: the lengths are not looked at, but for their sign."""
    out, lse, _, (att, call, cache) = _run_prefix(cuda, pplb200, 500, [0, 0, -1] * 4, 8, 2, 128, 16, 128)
    none = pplb200.SharedPrefixDecodeAttention(cache, 8, 12, 0, 500)
    table, lengths = cuda.empty((12, 0), dtype=cuda.int32, device="cuda"), cuda.tensor([0, 99, -1] * 4, dtype=cuda.int32, device="cuda")
    assert cuda.equal(none(call[0], call[1], call[2], table, lengths), out) and not bool(out[2::3].any())


def test_no_wait_has_given_up(cuda, pplb200):
    _run_prefix(cuda, pplb200, 400, [5] * 20, 4, 1, 64, 16, 0)
    cuda.cuda.synchronize()
    assert pplb200.shared_prefix_status(reset=False) == 0 == pplb200.shared_prefix_status()


# ---- streams, graphs, runs together --------------------------------------------------------------------------------------

@pytest.mark.parametrize("group", [0, 8, 128])
def test_same_run_after_run_and_in_a_graph(cuda, pplb200, group):
    """On another stream than the tensors' own, captured, and replayed on new contents."""
    _, _, _, (att, q, table, lens, _, _, blocks) = _run_sparse(cuda, pplb200, [3000, 40, 999], 8, 2, 128, 16, 16, group, 1, 2, 9)
    _, _, _, (prefix, call, _) = _run_prefix(cuda, pplb200, 2000, [30, 0, 7] * 9, 8, 2, 128, 16, group)
    one, two = att(q, table, lens), prefix(*call)
    for _ in range(3):
        assert cuda.equal(att(q, table, lens), one) and cuda.equal(prefix(*call), two)
    side = cuda.cuda.Stream()
    side.wait_stream(cuda.cuda.current_stream())
    a, b = cuda.empty_like(one), cuda.empty_like(two)
    graph = cuda.cuda.CUDAGraph()
    with cuda.cuda.graph(graph, stream=side):
        att(q, table, lens, out=a, blocks=blocks)
        prefix(*call, out=b)
        att(q, table, lens, out=a, blocks=blocks)
    for turn in range(3):
        if turn:
            q.mul_(0.5)
            lens[0] -= 100
            call[0].mul_(0.7)
            call[2][0] -= 300
        a.zero_(), b.zero_()
        graph.replay()
        cuda.cuda.synchronize()
        assert cuda.equal(a, att(q, table, lens)) and cuda.equal(b, prefix(*call))


@pytest.mark.parametrize("group", [0, 128])
def test_two_graphs_at_once(cuda, pplb200, group):
    """Calls on two streams, each with workspaces of its own, over one cache each."""
    graphs = []
    for seed in (1, 2):
        _, _, _, (att, q, table, lens, _, _, _) = _run_sparse(cuda, pplb200, [3000, 40, 999], 8, 2, 128, 16, 16, group, 1, 2, 9, seed=seed)
        _, _, _, (prefix, call, _) = _run_prefix(cuda, pplb200, 2500, [30, 600, 7] * 9, 8, 2, 128, 16, group, seed=seed)
        want = att(q, table, lens), prefix(*call)
        out = tuple(cuda.zeros_like(t) for t in want)
        graph, stream = cuda.cuda.CUDAGraph(), cuda.cuda.Stream()
        stream.wait_stream(cuda.cuda.current_stream())
        with cuda.cuda.graph(graph, stream=stream):
            for _ in range(3):
                prefix(*call, out=out[1])
                att(q, table, lens, out=out[0])
        graphs.append((graph, stream, want, out, (att, prefix, q, table, lens, call)))
    for _ in range(5):
        cuda.cuda.synchronize()
        for _, _, _, out, _ in graphs:
            [t.zero_() for t in out]
        cuda.cuda.synchronize()
        for graph, stream, _, _, _ in graphs:
            with cuda.cuda.stream(stream):
                graph.replay()
        cuda.cuda.synchronize()
        assert all(cuda.equal(a, b) for _, _, want, out, _ in graphs for a, b in zip(want, out))


def test_a_decode_step_behind_a_shared_image(cuda, pplb200):
    """Prompt with positions of three axes, bounds, then steps: rotate and store, complete blocks, attend over the prefix and over chosen blocks.  What the
    chain gives is what its parts give, and where every block is chosen, what attention over all tokens gives."""
    b, hq, hk, d, page, group = 3, 8, 2, 128, 32, 128
    g = _gen(cuda, 77)
    prefix, steps = 96, 20
    cache = pplb200.PagedKVCache.allocate(20, page, hk, d, group)
    bounds = pplb200.KeyBlockBounds(cache, 16)
    table = pplb200.RotaryTable(d, axes=(24, 20, 20), alternating=True)
    rows = _randn(cuda, g, prefix, hq + 2 * hk, d)
    at = cuda.arange(prefix, device="cuda")
    pos = cuda.stack([cuda.zeros_like(at), at // 12, at % 12])
    pplb200.rotary_kv_cache_write(cache, rows[:, :hq], rows[:, hq:hq + hk], rows[:, hq + hk:], pos, at, table)
    pplb200.key_bounds_update(bounds, at)
    pages = cuda.cat([cuda.arange(3, dtype=cuda.int32, device="cuda").expand(b, -1), 3 + cuda.arange(b, dtype=cuda.int32, device="cuda")[:, None]], 1).contiguous()
    mine = pages[:, 3:].contiguous()
    shared = pplb200.SharedPrefixDecodeAttention(cache, hq, b, page, prefix)
    full = pplb200.PagedDecodeAttention(cache, hq, b, prefix + page)
    some, every = (pplb200.BlockSparseDecodeAttention(bounds, hq, b, prefix + page, 1, 1, top) for top in (2, 6))
    length = cuda.tensor([prefix], dtype=cuda.int32, device="cuda")
    for step in range(steps):
        rows = _randn(cuda, g, b, hq + 2 * hk, d)
        slots = mine[:, 0].long() * page + step
        q = pplb200.rotary_kv_cache_write(cache, rows[:, :hq], rows[:, hq:hq + hk], rows[:, hq + hk:], cuda.full((3, b), 12 + step, device="cuda"), slots, table)
        pplb200.key_bounds_update(bounds, slots)
        lens = cuda.full((b,), prefix + step + 1, dtype=cuda.int32, device="cuda")
        want = full(q, pages, lens)
        assert cuda.equal(every(q, pages, lens), want)
        got = shared(q, pages[0, :3].contiguous(), length, mine, lens - prefix)
        assert bool(((got - want).abs().float() <= want.abs().float() * 4 * HALF + 1e-3).all())
        blocks = cuda.empty((b, hk, 4), dtype=cuda.int32, device="cuda")
        out, lse = cuda.empty_like(want), cuda.empty((b, hq), device="cuda")
        some(q, pages, lens, out=out, lse=lse, blocks=blocks)
        for i in range(b):
            n = prefix + step + 1
            assert blocks[i].tolist() == _choice(cuda, q[i], bounds, pages[i], n, 1, 1, 2, 20)
    done = cuda.cat([cuda.arange(6, device="cuda"), mine[:, 0].long() * 2])
    want, scale = _bounds(cuda, cache, 16)
    of = (done // 2, done % 2)
    assert cuda.equal(bounds.bounds[of[0], :, of[1]], want[of[0], :, of[1]]) and cuda.equal(bounds.scales[of[0], :, of[1]], scale[of[0], :, of[1]])
