"""Attention behind a shared prefix, over chosen blocks and over all tokens, on the GPU, where the usual cases do not go.  Tolerances as in test_attention_gpu.py: sums of half
steps."""
import pytest

from test_attention_gpu import HALF, TINY, _cache, _gen, _randn, _stored

pytestmark = pytest.mark.gpu


# ---- scores beyond 2^24 ------------------------------------------------------------------------------------------------

# base-2 scores near 2^30, and at the largest scale that is taken
@pytest.mark.parametrize("scale", [2.0 ** 15, 2.0 ** 50, -(2.0 ** 50)])
@pytest.mark.parametrize("group", [0, 8, 128])
@pytest.mark.parametrize("kind", ["decode", "sparse", "prefix few", "prefix many"])
def test_scores_far_beyond_what_their_steps_resolve(cuda, pplb200, kind, group, scale):
    """One token has all the weight.  Neighbouring keys are a 300th of the largest apart, 2^13 roundings to 32 bits, so that it is the same as in 64: its value, rounded when it is
    read where rows have groups of 8, and rounded on output."""
    d, n, rows = 128, 300, 64
    cache = _cache(cuda, pplb200, 20, 16, 1, d, group, "heads", 0)
    k = ((cuda.randperm(n, generator=_gen(cuda, 3), device="cuda") - 150.5) * 2).to(cuda.float16)[:, None, None].expand(n, 1, d).contiguous()
    pplb200.kv_cache_write(cache, k, _randn(cuda, _gen(cuda, 4), n, 1, d), cuda.arange(n, device="cuda"))
    kr, vr = _stored(cuda, cache, cuda.arange(n, device="cuda"))
    batch = 1 if kind in ("decode", "sparse") else 1 if kind == "prefix few" else 4
    q = cuda.linspace(0.62, 1.15, batch * rows, device="cuda").to(cuda.float16).view(batch, rows, 1).expand(-1, -1, d).contiguous()
    q[:, ::3] *= -1
    table, i32 = cuda.arange(20, dtype=cuda.int32, device="cuda"), dict(dtype=cuda.int32, device="cuda")
    if kind == "decode":
        out = pplb200.PagedDecodeAttention(cache, rows, 1, 320, scale=scale)(q, table[None], cuda.tensor([n], **i32))
    elif kind == "sparse":
        bounds = pplb200.KeyBlockBounds(cache, 16)
        out = pplb200.BlockSparseDecodeAttention(bounds, rows, 1, 320, 1, 1, 30, scale=scale)(q, table[None], cuda.tensor([n], **i32))
    else:  # 13 pages of the prefix, the others each sequence's own
        att = pplb200.SharedPrefixDecodeAttention(cache, rows, batch, 112, 208, scale=scale)
        out = att(q, table[:13].contiguous(), cuda.tensor([208], **i32), table[13:].expand(batch, -1).contiguous(), cuda.full((batch,), n - 208, **i32))
    score = cuda.einsum("bhd,td->bht", q.double(), kr[:, 0]) * scale
    want = vr[score.argmax(-1), 0]
    assert bool(((out.double() - want).abs() <= want.abs() * (2 * HALF + 2.0 ** -20) + 2 * TINY).all())
