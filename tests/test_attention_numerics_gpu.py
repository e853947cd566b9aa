"""What decode attention keeps of its numbers, where roundings would show: scores, weights, values and their scales at the ends of
their ranges, infinities, against definitions in 64 bits over what the cache holds.

The bounds count roundings: 2^-24 of a value for one in 32 bits, 2^-11 for the output's, 2^-25 below fp16's normal numbers."""
import math

import pytest

from test_attention_gpu import HALF, TINY, _cache, _gen, _randn, _stored

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
