"""What decode attention keeps of its numbers, where roundings would show: scores, weights, values and their scales at the ends of
their ranges, infinities, against definitions in 64 bits over what the cache holds.

The bounds count roundings: 2^-24 of a value for one in 32 bits, 2^-11 for the output's, 2^-25 below fp16's normal numbers."""
import math

import pytest

from test_attention_gpu import HALF, TINY, _cache, _check_attention, _gen, _randn, _run_attention, _stored

pytestmark = pytest.mark.gpu


def _one_sequence(cuda, pplb200, cache, q, n, scale=None):
    """Attention of q [hq, d] over the first n tokens of the cache's pages in order: out, lse and the scale."""
    att = pplb200.PagedDecodeAttention(cache, q.shape[0], 1, cache.num_pages * cache.page_size, scale=scale)
    lse = cuda.empty((1, q.shape[0]), device="cuda")
    pages = cuda.arange(cache.num_pages, dtype=cuda.int32, device="cuda")[None]
    out = att(q[None].contiguous(), pages, cuda.tensor([n], dtype=cuda.int32, device="cuda"), lse=lse)
    return out[0].double(), lse[0].double(), att.scale


@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("hq", [4, 16])
@pytest.mark.parametrize("group", [0, 8, -1])
@pytest.mark.parametrize("page", [16, 5])
def test_scores_beside_a_dimension_that_the_query_does_not_see(cuda, pplb200, d, hq, group, page):
    """Keys of a step or two of a scale that one outlier sets, queries of one sign that do not see the outlier: what is small in a key counts
    in full, whatever its row's scale.  The score of a single token is its lse."""
    group = d if group < 0 else group
    n = 16 * page
    g = _gen(cuda, d + hq)
    cache = _cache(cuda, pplb200, 16, page, 1, d, group, "heads", 0)
    k = cuda.randint(-2, 3, (n, 1, d), generator=g, device="cuda").to(cuda.float16)
    k[:, 0, 3] = 127
    pplb200.kv_cache_write(cache, k, k, cuda.arange(n, device="cuda"))
    q = _randn(cuda, g, hq, d).abs() * 20
    q[:, 3] = 0
    att = pplb200.PagedDecodeAttention(cache, hq, n, page, window=1)
    at, lse = cuda.arange(n, device="cuda"), cuda.empty((n, hq), device="cuda")
    att(q.expand(n, -1, -1).contiguous(), (at // page).to(cuda.int32)[:, None].contiguous(), (at % page + 1).to(cuda.int32), lse=lse)
    keys = _stored(cuda, cache, at)[0][:, 0]
    score, size = keys @ q.double().T * att.scale, keys.abs() @ q.double().abs().T * att.scale
    # d products and d - 1 sums in 32 bits, in any order; scale, scale * log2(e), their product with a row's scale and with the sum, back to
    # natural logarithms (three of those); beside them the difference to and from the reference exponent, 8 away
    assert bool(((lse.double() - score).abs() <= size * (d + 8) * 2.0 ** -24 + 2.0 ** -20).all())


@pytest.mark.parametrize("d,shared", [(64, 1), (96, 3), (128, 1), (128, 16), (256, 2)])
@pytest.mark.parametrize("group", [0, 8, -1])
def test_weights_keep_22_bits(cuda, pplb200, d, shared, group):
    """Tokens in pairs whose weighted values nearly cancel: what a rounding of the weights leaves is not hidden by the output's own.  Keys
    with one dimension, so that scores are exact products; values of whole numbers times a power of two, so that no cache rounds them."""
    group = d if group < 0 else group
    hk, lengths, page = 8, [2, 4, 8, 32], 16
    g = _gen(cuda, d + shared)
    n = sum(lengths)
    q = cuda.zeros((1, hk * shared, d), dtype=cuda.float16, device="cuda")
    q[..., 1] = 4.0
    a = cuda.rand((n // 2, hk), generator=g, device="cuda", dtype=cuda.float64) - 0.5
    m = cuda.randint(64, 128, (2, n // 2, hk), generator=g, device="cuda").double()
    sign = (cuda.randint(0, 2, (1, hk, d), generator=g, device="cuda") * 2 - 1).double()
    k, v = cuda.zeros((n, hk, d), dtype=cuda.float64, device="cuda"), cuda.empty((n, hk, d), dtype=cuda.float64, device="cuda")
    k[0::2, :, 1] = a
    k[1::2, :, 1] = a + (m[0] / m[1]).log() / 4  # e^(4 k) m is the same for both
    v[0::2], v[1::2] = m[0][..., None] * sign / 64, -m[1][..., None] * sign / 64
    v[..., 7::8] = 127 / 64  # the largest of every group, so that its scale is a power of two
    k, v = k.to(cuda.float16), v.to(cuda.float16)
    cache = _cache(cuda, pplb200, 8, page, hk, d, group, "heads", 0)
    pages = cuda.tensor([[0, 0], [1, 1], [2, 2], [3, 4]], dtype=cuda.int32, device="cuda")
    slots = [pages[b].long()[cuda.arange(c, device="cuda") // page] * page + cuda.arange(c, device="cuda") % page for b, c in enumerate(lengths)]
    pplb200.kv_cache_write(cache, k, v, cuda.cat(slots))
    att = pplb200.PagedDecodeAttention(cache, hk * shared, 4, 2 * page, scale=1.0)
    out = att(q.expand(4, -1, -1).contiguous(), pages, cuda.tensor(lengths, dtype=cuda.int32, device="cuda")).double()
    for b, c in enumerate(lengths):
        keys, values = _stored(cuda, cache, slots[b])
        p = cuda.softmax(4 * keys[..., 1], 0)
        want, size = (cuda.einsum("th,thd->hd", p, x).repeat_interleave(shared, 0) for x in (values, values.abs()))
        # scores up to 4: four roundings of six, two of up to sixteen, 2^-22 of the power of two, 2^-22 left of the weight: below 2^-18,
        # twice, since the weights' sum has it too; c sums in 32 bits, cut off rather than rounded, in both; joining the warps' sums
        bound = size * (2.0 ** -17 + c * 2.0 ** -22 + 2.0 ** -21) + want.abs() * HALF + TINY
        assert bool(((out[b] - want).abs() <= bound).all()), c


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("group", [0, 8, 128])
@pytest.mark.parametrize("n", [40, 5000])
def test_what_a_value_is_does_not_reach_the_lse(cuda, pplb200, value, group, n):
    """An infinity or NaN among the values: its dimensions (those that share its scale) of its heads' output are lost, and nothing else."""
    d, page = 128, 16
    g = _gen(cuda, n)
    cache = _cache(cuda, pplb200, -(-n // page), page, 2, d, group, "heads", 0)
    k, v, q = _randn(cuda, g, n, 2, d), _randn(cuda, g, n, 2, d), _randn(cuda, g, 6, d)
    at = cuda.arange(n, device="cuda")
    pplb200.kv_cache_write(cache, k, v, at)
    out, lse, scale = _one_sequence(cuda, pplb200, cache, q, n)
    v[n - 3, 1, 21] = value
    pplb200.kv_cache_write(cache, k, v, at)
    lost, same, _ = _one_sequence(cuda, pplb200, cache, q, n)
    keys = _stored(cuda, cache, at)[0].repeat_interleave(3, 1)
    score, size = cuda.einsum("hd,thd->ht", q.double(), keys) * scale, cuda.einsum("hd,thd->ht", q.double().abs(), keys.abs()).amax(-1) * scale
    # a score's products and sums and its factors, and n sums of weights, all in 32 bits
    bound = size * (d + 8) * 2.0 ** -24 + 2.0 ** -20 + n * 2.0 ** -23
    for x in (lse, same):
        assert bool(((x - cuda.logsumexp(score, -1)).abs() <= bound).all())
    odd = cuda.zeros_like(out, dtype=cuda.bool)
    first = 21 // max(group, 1) * max(group, 1)
    odd[3:, first:first + max(group, 1)] = True
    assert cuda.equal(~cuda.isfinite(lost), odd) and cuda.equal(lost[~odd], out[~odd])


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("group", [8, 128])
def test_a_lost_key_is_not_left_out(cuda, pplb200, value, group):
    """Keys that read back as NaN make their heads' output and lse NaN, whatever the query's signs."""
    d, n, page = 128, 50, 16
    for seed in range(8):
        g = _gen(cuda, seed)
        cache = _cache(cuda, pplb200, 4, page, 2, d, group, "heads", 0)
        k, v, q = _randn(cuda, g, n, 2, d), _randn(cuda, g, n, 2, d), _randn(cuda, g, 16, d, scale=30.0)
        k[7 * seed % n, 0, 3] = value
        pplb200.kv_cache_write(cache, k, v, cuda.arange(n, device="cuda"))
        out, lse, _ = _one_sequence(cuda, pplb200, cache, q, n)
        assert bool(out[:8].isnan().all()) and bool(lse[:8].isnan().all())
        assert bool(cuda.isfinite(out[8:]).all()) and bool(cuda.isfinite(lse[8:]).all())


@pytest.mark.parametrize("lengths", [[1], [20, 0, 3], [4000]])
def test_scores_of_minus_infinity_only(cuda, pplb200, lengths):
    """Tokens that are seen, but whose scores are all minus infinity: their sum is zero, as the definition has it, and the quotient NaN; zeros
    are for sequences of which nothing is seen.  Beside finite scores such tokens have no weight."""
    d, page = 128, 16
    g = _gen(cuda, 2)
    width = -(-max(lengths) // page)
    cache = _cache(cuda, pplb200, width, page, 1, d, 0, "heads", 0)
    n = width * page
    v = _randn(cuda, g, n, 1, d)
    k = cuda.zeros_like(v)
    k[..., 9], k[..., 10] = math.inf, 0.5
    pplb200.kv_cache_write(cache, k, v, cuda.arange(n, device="cuda"))
    q = cuda.ones((len(lengths), 3, d), dtype=cuda.float16, device="cuda")
    q[:, :, 9] = -1.0
    q[:, 0, 10] = 0.0
    pages = cuda.arange(width, dtype=cuda.int32, device="cuda").expand(len(lengths), -1)
    lens = cuda.tensor(lengths, dtype=cuda.int32, device="cuda")
    att = pplb200.PagedDecodeAttention(cache, 3, len(lengths), n, scale=1.0)
    lse = cuda.empty((len(lengths), 3), device="cuda")
    out = att(q, pages.contiguous(), lens, lse=lse)
    assert bool((lse == -math.inf).all())
    for b, c in enumerate(lengths):
        assert bool(out[b].isnan().all()) if c else not bool(out[b].any())
    cache.k[0, 0, 0, 9] = 0.0  # one token's score is finite
    out = att(q, pages.contiguous(), lens, lse=lse)
    for b, c in enumerate(lengths):
        assert not bool(out[b].any()) if c == 0 else bool((out[b] == cache.v[0, 0, 0]).all())
        want = cuda.tensor([0.0, 0.5, 0.5] if c else [-math.inf] * 3, device="cuda")
        # 0.5 by way of base 2: the factor, the product, 8 off and on, and back, each rounded to 32 bits
        assert cuda.equal(lse[b], want) or bool(((lse[b] - want).abs() <= 2.0 ** -20).all())


def _foreign(cuda, pplb200, n, hk, d, group, k_scale, v_scale, seed):
    """A cache that another program filled: any whole numbers, scales [n, hk, d / group] (sizes; their signs are drawn)."""
    g = _gen(cuda, seed)
    cache = _cache(cuda, pplb200, -(-n // 16), 16, hk, d, group, "heads", 0)
    at = cuda.arange(n, device="cuda")
    for x, s, size in ((cache.k, cache.k_scale, k_scale), (cache.v, cache.v_scale, v_scale)):
        x.copy_(cuda.randint(-127, 128, x.shape, generator=g, device="cuda"))
        sign = cuda.randint(0, 2, size.shape, generator=g, device="cuda") * 2 - 1
        s[at // 16, :, at % 16] = (size * sign).to(cuda.float16)
    return cache


def _check(cuda, cache, out, lse, q, n, scale, group, extra=0.0):
    """Against the definition; group: of the cache, 8: values are rounded to fp16.  extra [hq]: of the weights' products with values' scales."""
    shared = q.shape[0] // cache.kv_heads
    k, v = (x.repeat_interleave(shared, 1) for x in _stored(cuda, cache, cuda.arange(n, device="cuda")))
    score = cuda.einsum("hd,thd->ht", q.double(), k) * scale
    p = cuda.softmax(score, -1)
    want, size = cuda.einsum("ht,thd->hd", p, v), cuda.einsum("ht,thd->hd", p, v.abs())
    # a score as above; a weight: twice that, 22 bits, n sums in 32 bits in it and in the product with values
    off = cuda.einsum("hd,thd->ht", q.double().abs(), k.abs()).amax(-1) * abs(scale) * (q.shape[1] + 8) * 2.0 ** -24 + 2.0 ** -20
    weight = 2 * off + n * 2.0 ** -22 + 2.0 ** -20 + (HALF if group == 8 else 0)
    bound = weight[:, None] * size * (1 + HALF) + (want.abs() * HALF + 2 * TINY) + extra
    assert bool(((out - want).abs() <= bound).all())
    assert bool(((lse - cuda.logsumexp(score, -1)).abs() <= off + n * 2.0 ** -23).all())


@pytest.mark.parametrize("n", [37, 3000])
def test_rows_whose_scales_differ_by_all_of_fp16(cuda, pplb200, n):
    """Values whose scales span fp16, from one token to the next and zeros among them, while the weights span as much the other way: the
    reference exponent follows their product."""
    d, hk = 128, 2
    g = _gen(cuda, n)
    u = cuda.rand((n, hk, 1), generator=g, device="cuda")
    v_scale = cuda.exp2(40 * u - 24).clamp_max(1000.0)
    v_scale[cuda.rand((n, hk, 1), generator=g, device="cuda") < 0.1] = 0.0
    cache = _foreign(cuda, pplb200, n, hk, d, d, cuda.full((n, hk, 1), 1e-2, device="cuda"), v_scale, n)
    cache.v.clamp_(-60, 60)  # of 1000: within fp16 on output
    # a dimension that raises the score of tokens with small scales
    at = cuda.arange(n, device="cuda")
    cache.k[at // 16, :, at % 16, 0] = (127 * (1 - 2 * u[..., 0])).round().to(cuda.int8)
    q = _randn(cuda, g, 6, d) * 0.1
    q[:, 0] = cuda.tensor([0.0, 12.0, -12.0, 6.0, 20.0, -3.0])
    out, lse, scale = _one_sequence(cuda, pplb200, cache, q, n, scale=1.0)
    k, v = _stored(cuda, cache, at)
    p = cuda.softmax(cuda.einsum("hd,thd->ht", q.double(), k.repeat_interleave(3, 1)), -1)
    s = cache.v_scale[at // 16, :, at % 16, 0].double().abs().T.repeat_interleave(3, 0)
    # what is left of weight x scale is rounded at 2^-25 where the largest is 2^8 at least: of every token, times up to 60 steps
    extra = (n * 60 * 2.0 ** -33 * (p * s).amax(-1))[:, None]
    _check(cuda, cache, out, lse, q, n, scale, d, extra)


@pytest.mark.parametrize("group", [8, 128])
def test_scales_up_to_the_largest(cuda, pplb200, group):
    """Keys and values of the largest steps that the writer stores, 515.5; rows that share a scale take larger keys as well."""
    n, d = 200, 128
    for k_size, v_size in ((515.5, 1.0), (1e-3, 515.5)) + (((60000.0, 1.0),) if group == d else ()):
        scales = [cuda.full((n, 1, d // group), x, device="cuda") for x in (k_size, v_size)]
        cache = _foreign(cuda, pplb200, n, 1, d, group, *scales, 3)
        q = _randn(cuda, _gen(cuda, 4), 3, d)
        out, lse, scale = _one_sequence(cuda, pplb200, cache, q, n, scale=0.05 / k_size)
        _check(cuda, cache, out, lse, q, n, scale, group)


def test_products_beyond_fp16_are_not_silent(cuda, pplb200):
    """Groups of 8: a key beyond fp16's range makes its heads NaN, and no other's; a small number of large steps is a key like any."""
    n, d = 50, 128
    scales = cuda.full((n, 2, d // 8), 0.01, device="cuda")
    cache = _foreign(cuda, pplb200, n, 2, d, 8, scales, scales, 5)
    cache.k_scale[1, 0, 4, 3], cache.k[1, 0, 4, 24:32] = 4000.0, 16
    q = _randn(cuda, _gen(cuda, 6), 4, d) * 0.01
    out, lse, scale = _one_sequence(cuda, pplb200, cache, q, n)
    _check(cuda, cache, out, lse, q, n, scale, 8)
    cache.k[1, 0, 4, 25] = 17
    lost, lost_lse, _ = _one_sequence(cuda, pplb200, cache, q, n)
    assert bool(lost[:2].isnan().all()) and bool(lost_lse[:2].isnan().all())
    assert cuda.equal(lost[2:], out[2:]) and cuda.equal(lost_lse[2:], lse[2:])


@pytest.mark.parametrize("scale,q_scale", [(None, 20.0), (1.0, 8.0), (0.0, 1.0), (-0.1, 2.0), (1e-6, 1.0)])
@pytest.mark.parametrize("hq", [2, 32])
def test_rows_scores_of_all_sizes(cuda, pplb200, scale, q_scale, hq):
    """Softmaxes between uniform and one-hot over int8 rows, scores of some hundreds."""
    _check_attention(*_run_attention(cuda, pplb200, [1500, 40, 333], hq, 2, 128, 16, 128, scale=scale, q_scale=q_scale)[:3])


@pytest.mark.parametrize("group", [8, 128])
@pytest.mark.parametrize("size", [60000.0, 1e-4, 1e-6])
def test_int8_values_of_all_sizes(cuda, pplb200, group, size):
    """Values near the largest and the smallest of fp16, whose scales are the largest and subnormal: nothing overflows or vanishes."""
    n, d = 300, 128
    g = _gen(cuda, 2)
    cache = _cache(cuda, pplb200, 20, 16, 1, d, group, "heads", 0)
    v = (cuda.rand((n, 1, d), generator=g, device="cuda") * size).to(cuda.float16)
    pplb200.kv_cache_write(cache, _randn(cuda, g, n, 1, d), v, cuda.arange(n, device="cuda"))
    q = _randn(cuda, g, 2, d)
    out, lse, scale = _one_sequence(cuda, pplb200, cache, q, n)
    _check(cuda, cache, out, lse, q, n, scale, group)


@pytest.mark.parametrize("group", [8, 128])
def test_int8_special_values_out_of_sight(cuda, pplb200, group):
    """NaN scales outside the window, behind the length and in another sequence's pages have no influence."""
    out, lse, want, (att, q, table, lens, cache) = _run_attention(cuda, pplb200, [100, 100, 50], 8, 2, 128, 16, group, window=40)
    _check_attention(out, lse, want)
    nan = float("nan")
    cache.k_scale[int(table[1, 1]), :, 3], cache.v_scale[int(table[1, 1]), :, 3] = nan, nan    # token 19 of 100: outside the window
    cache.k_scale[int(table[2, 3]), :, 10], cache.v_scale[int(table[2, 3]), :, 10] = nan, nan  # token 58 of 50
    cache.v_scale[int(table[0, 6]), 1, 1] = nan                                                # token 97 of 100: seen
    got = att(q, table, lens)
    assert cuda.equal(got[1:], out[1:]) and cuda.equal(got[0, :4], out[0, :4])
    assert bool(got[0, 4:].isnan().all())


@pytest.mark.parametrize("batch,heads", [(65535, 1), (3, 65535), (9000, 40)])
@pytest.mark.parametrize("group", [0, 64])
def test_the_most_sequences_and_heads(cuda, pplb200, batch, heads, group):
    """As many sequences and heads as are taken, of none to three tokens: every row is written, from its own pages.  With values that are the
    same for all tokens of a sequence and head, the output is that value, whatever the weights."""
    d, page = 64, 3
    g = _gen(cuda, batch)
    pages = batch
    cache = _cache(cuda, pplb200, pages, page, heads, d, group, "heads", 0)
    size = cuda.randint(1, 100, (pages, heads), generator=g, device="cuda").to(cuda.float16)
    cache.k.copy_(cuda.randint(-3, 4, (1, 1, page, d), generator=g, device="cuda").expand(cache.k.shape))
    if group:
        cache.k_scale.fill_(0.125)
        cache.v.fill_(1)
        cache.v_scale.copy_(size[:, :, None, None].expand(cache.v_scale.shape))
    else:
        cache.v.copy_(size[:, :, None, None].expand(cache.v.shape))
    table = cuda.randperm(pages, generator=g, device="cuda").to(cuda.int32)[:, None].contiguous()
    lens = cuda.randint(0, page + 1, (batch,), generator=g, device="cuda").to(cuda.int32)
    q = _randn(cuda, g, 1, 1, d).expand(batch, heads, d).contiguous()
    att = pplb200.PagedDecodeAttention(cache, heads, batch, page)
    out = att(q, table, lens, out=cuda.full_like(q, 7.0))
    want = size[table[:, 0].long()].float()
    want[lens == 0] = 0
    # three weights and their sum: a few roundings at 2^-22, and the output's
    assert bool(((out.float() - want[..., None]).abs() <= want[..., None] * (HALF + 2.0 ** -19)).all())
