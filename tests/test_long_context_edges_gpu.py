"""Attention behind a shared prefix, over chosen blocks and over all tokens, on the GPU, where the usual cases do not go.  Tolerances as in test_attention_gpu.py: sums of half
steps."""
import ctypes
import os
import struct
import threading

import numpy as np
import pytest

from test_attention_gpu import HALF, TINY, _attention, _cache, _check_attention, _gen, _randn, _rows, _run_attention, _stored
from test_long_context_gpu import _choice, _run_prefix, _run_sparse

pytestmark = pytest.mark.gpu


# ---- scores beyond 2^24 ------------------------------------------------------------------------------------------------

# base-2 scores of up to 2^27 to 2^28, where 8 lies half way between two numbers of 32 bits; near 2^30; the largest scale that is taken
@pytest.mark.parametrize("scale", [2.0 ** 12, -(2.0 ** 12), 2.0 ** 15, 2.0 ** 50, -(2.0 ** 50)])
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


@pytest.mark.parametrize("step", [1, 2, 4, 8, 16, 32])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("group", [0, 8, 128])
@pytest.mark.parametrize("kind", ["decode", "sparse", "prefix few", "prefix many"])
def test_scores_that_rise_by_what_32_bits_resolve(cuda, pplb200, kind, group, sign, step):
    """Base-2 scores of +-2^23 step and a multiple of `step` more: every number on the way is exact in 32 bits, every weight a power of two.  So the outputs are off by their own rounding, by
    the sums' of 300 tokens in 32 bits, and by that of values which are rounded when they are read."""
    d, n, rows = 128, 300, 16
    cache = _cache(cuda, pplb200, 20, 16, 1, d, group, "heads", 0)
    at = cuda.arange(n, device="cuda")
    k = cuda.zeros((n, 1, d), dtype=cuda.float16, device="cuda")
    k[:, 0, 0], k[:, 0, 8] = 4.0 * sign, (at // 3 * 2.0 ** -4).to(cuda.float16)
    pplb200.kv_cache_write(cache, k, _randn(cuda, _gen(cuda, 4), n, 1, d), at)
    if group:  # whole numbers times 2^-4
        cache.k.view(20, 16, d)[at // 16, at % 16] = (k[:, 0] * 16).to(cuda.int8)
        cache.k_scale.fill_(2.0 ** -4)
    kr, vr = _stored(cuda, cache, at)
    assert cuda.equal(kr, k.double())
    batch = 12 if kind == "prefix many" else 1
    q = cuda.zeros((batch, rows, d), dtype=cuda.float16, device="cuda")
    q[..., 0], q[..., 8] = 8192.0, 2.0 ** -4
    scale = np.float32(step * 256.0 / 1.4426950408889634)
    while scale * np.float32(1.4426950408889634) < step * 256:
        scale = np.nextafter(scale, np.float32(np.inf))
    while scale * np.float32(1.4426950408889634) > step * 256:
        scale = np.nextafter(scale, np.float32(0))
    assert scale * np.float32(1.4426950408889634) == step * 256  # so that a score is 2^15 times step 2^8, and 2^-8 times that for a third of the token's number
    table, i32 = cuda.arange(20, dtype=cuda.int32, device="cuda"), dict(dtype=cuda.int32, device="cuda")
    if kind == "decode":
        out = pplb200.PagedDecodeAttention(cache, rows, 1, 320, scale=float(scale))(q, table[None], cuda.tensor([n], **i32))
    elif kind == "sparse":
        out = pplb200.BlockSparseDecodeAttention(pplb200.KeyBlockBounds(cache, 16), rows, 1, 320, 1, 1, 30, scale=float(scale))(q, table[None], cuda.tensor([n], **i32))
    else:
        att = pplb200.SharedPrefixDecodeAttention(cache, rows, batch, 112, 208, scale=float(scale))
        out = att(q, table[:13].contiguous(), cuda.tensor([208], **i32), table[13:].expand(batch, -1).contiguous(), cuda.full((batch,), n - 208, **i32))
    weight = 2.0 ** (step * (at // 3 - (n - 1) // 3).double())
    weight /= weight.sum()
    want, size = weight @ vr[:, 0], weight @ vr[:, 0].abs()
    assert bool(((out.double() - want).abs() <= want.abs() * HALF + size * (HALF * (group > 0) + 2.0 ** -14) + 2 * TINY).all())


# ---- scales of an int8 cache ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("prefix,batch", [(500, 24), (500, 1), (9000, 2), (9000, 40)])
@pytest.mark.parametrize("q_scale", [0.5, 20.0])
def test_prefix_of_rows_of_any_finite_scale(cuda, pplb200, prefix, batch, d, q_scale):
    """Values whose product with their scale fp16 does not hold, on the way from 2^-24 to 65504, of either sign: by tiles and by the decode kernel, whatever the number of rows."""
    g, page, own, hq, hk = _gen(cuda, 7), 16, 32, 8, 2
    n, pages = prefix + batch * own, -(-prefix // page) + batch * own // page
    cache = _cache(cuda, pplb200, pages, page, hk, d, d, "heads", 0)
    pplb200.kv_cache_write(cache, _randn(cuda, g, pages * page, hk, d), _randn(cuda, g, pages * page, hk, d), cuda.arange(pages * page, device="cuda"))
    size = cuda.exp2(cuda.rand(cache.v_scale.shape, generator=g, device="cuda") * 31 - 24)
    big = cuda.rand(size.shape, generator=g, device="cuda") < 8 / n  # 127 times 520 and more is beyond fp16; eight of them or so, so that a mean of all stays below
    size = cuda.where(big, 520.0 + cuda.rand(size.shape, generator=g, device="cuda") * (2000 if q_scale < 1 else 64984), size)
    cache.v_scale.copy_(size * ((cuda.rand(size.shape, generator=g, device="cuda") < 0.5) * 2 - 1))
    table = cuda.randperm(pages, generator=g, device="cuda").to(cuda.int32)
    shared, mine = table[:-(-prefix // page)].contiguous(), table[-(-prefix // page):].view(batch, -1).contiguous()
    att = pplb200.SharedPrefixDecodeAttention(cache, hq, batch, own, len(shared) * page)
    q, i32 = _randn(cuda, g, batch, hq, d, scale=q_scale), dict(dtype=cuda.int32, device="cuda")
    lse = cuda.empty((batch, hq), device="cuda")
    out = att(q, shared, cuda.tensor([prefix], **i32), mine, cuda.full((batch,), own, **i32), lse=lse)
    want = []
    for b in range(batch):
        token = cuda.arange(prefix, device="cuda")
        slots = cuda.cat([shared.long()[token // page] * page + token % page, (mine[b].long()[:, None] * page + cuda.arange(page, device="cuda")).flatten()])
        k, v = _stored(cuda, cache, slots)
        o, l, bound, lse_bound = _attention(cuda, q[b], k, v, cuda.ones(len(slots), dtype=cuda.bool, device="cuda"), att.scale)
        # A weight times its scale is the sum of two fp16, the second of which is off by half a step, 2^-25 at least.  The reference exponent is up to 4 above a score and the size of
        # the scales beside it, of which the least may be 5 below: the largest product is 2^(8 - 4 - 5) or more, so that a token loses 2^-24 of it.
        s = _rows(cache.v_scale, slots, page).double().abs()[..., 0].repeat_interleave(hq // hk, 1).T
        p = cuda.softmax(cuda.einsum("hd,thd->ht", q[b].double(), k.repeat_interleave(hq // hk, 1)) * att.scale, -1)
        bound += 2.0 ** -24 * (p * s).amax(-1, keepdim=True) * (v.abs().repeat_interleave(hq // hk, 1) / s.T[..., None]).sum(0)
        want.append((o, l, bound, lse_bound))
    inside = cuda.stack([w[0] for w in want]).abs() < 65000.0
    assert float(inside.double().mean()) > 0.9
    for b, (o, l, bound, lse_bound) in enumerate(want):
        assert bool(((out[b].double() - o).abs() <= bound)[inside[b]].all()), b
        assert bool(((lse[b].double() - l).abs() <= lse_bound).all()), b


@pytest.mark.parametrize("d", [64, 128, 256])
def test_prefix_of_rows_is_as_exact_as_decode_attention(cuda, pplb200, d):
    """Whole numbers times weights of 22 bits: no value is rounded.  48 rows of 1000 tokens behind a shared prefix, and by the decode kernel over all."""
    out, lse, _, (att, call, cache) = _run_prefix(cuda, pplb200, 968, [32] * 24, 8, 2, d, 16, d)
    rows = lambda table, n: _stored(cuda, cache, (table.long()[:, None] * 16 + cuda.arange(16, device="cuda")).flatten()[:n])  # noqa: E731
    k, v = rows(call[1], 968)
    error = []
    for b in range(24):
        own = rows(call[3][b], 32)
        want = _attention(cuda, call[0][b], cuda.cat([k, own[0]]), cuda.cat([v, own[1]]), cuda.ones(1000, dtype=cuda.bool, device="cuda"), att.scale)[0]
        error.append(((out[b].double() - want), want))
    # the output's rounding, evenly spread over a step of 2^-11 to 2^-10 of the value: the 2-norm of the errors is 2^-11 / sqrt(3) of the values' at most, 0.00028, and over a whole octave 0.00021
    # in the mean; a tenth more for the weights' and the sums' roundings
    off, size = (cuda.stack([e[i] for e in error]).norm() for i in (0, 1))
    assert float(off / size) < 0.00023


# ---- waits that give up ----------------------------------------------------------------------------------------------------

@pytest.fixture(scope="module")
def impatient(pplb200):
    """The library in which the warp that issues a prefix's products does not wait for the values of its last two tasks.  Everybody else arrives and waits as ever: the scores of these
    tasks are there, so that no other wait runs out."""
    lib = ctypes.CDLL(os.path.join(os.path.dirname(pplb200.LIB_PATH), "libpplb200_impatient_prefix.so"))
    lib.pplb200_shared_prefix_attention_fp16.argtypes = [ctypes.c_void_p] + [ctypes.c_char_p] * 3
    lib.pplb200_shared_prefix_attention_status.argtypes = [ctypes.c_int32]
    return lib


@pytest.mark.parametrize("group,d", [(0, 64), (0, 128), (128, 128), (64, 64)])
@pytest.mark.parametrize("prefix,batch,page", [(100, 24, 16), (3, 40, 16), (2100, 64, 64), (2100, 64, 24), (300, 1, 16)])
def test_products_that_are_not_all_there_leave_nan(cuda, pplb200, impatient, prefix, batch, page, group, d):
    """One task of a CTA, two, and several: no finite sum without all of its values."""
    hq, hk = 64, 8
    out, lse, _, (att, call, cache) = _run_prefix(cuda, pplb200, prefix, ([5, 0, -1, 40] * batch)[:batch], hq, hk, d, page, group)
    cuda.cuda.synchronize()
    lost, lost_lse = cuda.full_like(out, 7.0), cuda.full_like(lse, 7.0)
    q, shared, length, pages, lengths = call
    args = struct.pack("=6Q6q2ifi", q.data_ptr(), lost.data_ptr(), lost_lse.data_ptr(), pages.data_ptr(), lengths.data_ptr(), att.ws.data_ptr(), att.ws.numel(), batch, pages.shape[1], pages.stride(0),
                       q.stride(0), lost.stride(0), hq, 0, att.scale, 0)
    stream = cuda.cuda.current_stream().cuda_stream
    impatient.pplb200_shared_prefix_attention_status(1)
    assert impatient.pplb200_shared_prefix_attention_fp16(stream, cache._args[0], args, struct.pack("=2Qq", shared.data_ptr(), length.data_ptr(), shared.shape[0])) == 0
    cuda.cuda.synchronize()
    assert impatient.pplb200_shared_prefix_attention_status(1) == 2 and impatient.pplb200_shared_prefix_attention_status(0) == 0  # the code of the products' warp
    there = lengths >= 0
    assert bool(lost[there].isnan().all()) and bool(lost_lse[there].isnan().all())
    assert not lost[~there].any() and bool((lost_lse[~there] == -float("inf")).all())
    assert cuda.equal(att(*call), out) and pplb200.shared_prefix_status() == 0  # the workspace is fit for the next call


# ---- calls of several threads ----------------------------------------------------------------------------------------------

def test_choices_of_several_threads(cuda, pplb200):
    """Tables that need different amounts of shared memory, on a stream and a workspace each: no thread's launch depends on what another is doing."""
    cache = _cache(cuda, pplb200, 200, 16, 1, 128, 0, "heads", 0)
    pplb200.kv_cache_write(cache, _randn(cuda, _gen(cuda, 1), 3200, 1, 128), _randn(cuda, _gen(cuda, 2), 3200, 1, 128), cuda.arange(3200, device="cuda"))
    bounds = pplb200.KeyBlockBounds(cache, 16)
    pplb200.key_bounds_update(bounds, cuda.arange(3200, device="cuda"))
    q, lengths = _randn(cuda, _gen(cuda, 3), 1, 4, 128), cuda.tensor([3200], dtype=cuda.int32, device="cuda")
    jobs = []
    for blocks in (9000, 16000, 11000, 200):
        table = cuda.full((1, blocks), -1, dtype=cuda.int32, device="cuda")
        table[0, :200] = cuda.arange(200, dtype=cuda.int32, device="cuda")
        att = pplb200.BlockSparseDecodeAttention(bounds, 4, 1, blocks * 16, 1, 1, 30)
        jobs.append((att, table, cuda.cuda.Stream(), cuda.empty_like(q)))
    want = jobs[0][0](q, jobs[0][1], lengths)
    cuda.cuda.synchronize()
    failed = []

    def work(att, table, stream, out):
        try:
            with cuda.cuda.stream(stream):
                for _ in range(3000):
                    att(q, table, lengths, out=out)
        except Exception as e:
            failed.append(e)

    threads = [threading.Thread(target=work, args=job) for job in jobs]
    [t.start() for t in threads]
    [t.join() for t in threads]
    cuda.cuda.synchronize()
    assert not failed, failed
    for _, _, _, out in jobs:
        assert bool(((out - want).abs().float() <= want.abs().float() * 2 * HALF + 2.0 ** -14).all())  # the order in which parts are joined may differ


# ---- one workspace ------------------------------------------------------------------------------------------------------------

def test_one_workspace_for_all_forms_of_attention(cuda, pplb200):
    """As large as the largest of them needs, zeroed once: what a call leaves in it is nothing to the next, whatever that is."""
    calls = []
    for d, group in ((128, 128), (64, 0)):
        for lengths, hq, hk in (([9000, 3, 500], 16, 2), ([20000], 4, 1)):
            _, _, _, (att, q, table, lens, cache) = _run_attention(cuda, pplb200, lengths, hq, hk, d, 16, group)
            calls.append((att, (q, table, lens), cache))
        for prefix, lengths, hq, hk in ((300, [2100] * 5, 4, 1), (9000, [40] * 4, 4, 4), (9000, [3000, 0, 5], 32, 2), (700, [900] * 40, 8, 2)):
            _, _, _, (att, call, cache) = _run_prefix(cuda, pplb200, prefix, lengths, hq, hk, d, 16, group)
            calls.append((att, call, cache))
        _, _, _, (att, q, table, lens, cache, bounds, _) = _run_sparse(cuda, pplb200, [9000, 40, 3000], 8, 2, d, 16, 16, group, 1, 2, 400)
        calls.append((att, (q, table, lens), cache))
    want = [att(*call) for att, call, _ in calls]
    ws = cuda.zeros(max(att.ws.numel() for att, _, _ in calls), dtype=cuda.uint8, device="cuda")
    for att, _, _ in calls:  # (an object's workspace is its own: a caller of the C functions brings one)
        args = att._args
        object.__setattr__(att, "_args", args[:3] + (ws.data_ptr(), ws.numel()) + args[5:])
    order = list(range(len(calls))) * 3
    np.random.default_rng(1).shuffle(order)
    for i in order + order[::-1]:
        att, call, _ = calls[i]
        assert cuda.equal(att(*call, out=cuda.full_like(want[i], 7.0)), want[i]), i


# ---- chains of steps --------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("batch,hq,hk,d,group,prefix", [(16, 8, 8, 128, 0, 2000), (4, 32, 8, 128, 128, 9000), (40, 16, 2, 64, 8, 700), (100, 8, 1, 256, 256, 3000), (2, 4, 4, 96, 0, 200)])
def test_steps_in_one_captured_chain(cuda, pplb200, batch, hq, hk, d, group, prefix):
    """Lengths, page tables, positions and the cache are advanced by kernels between the calls of one graph, each call's own tokens' kernel beginning beside its prefix's: what a step gives is what it
    gives with the device waited for in front of every kernel."""
    g, page, steps, most = _gen(cuda, 21), 16, 24, 64
    own = most // page
    pages = -(-prefix // page) + batch * own
    table = pplb200.RotaryTable(d)
    shared = cuda.arange(pages - batch * own, dtype=cuda.int32, device="cuda")
    every = len(shared) + cuda.randperm(batch * own, generator=g, device="cuda").to(cuda.int32).view(batch, own)
    rows = _randn(cuda, g, steps, batch, hq + 2 * hk, d)
    at = cuda.arange(len(shared) * page, device="cuda")
    k, v = (_randn(cuda, g, len(at), hk, d) for _ in range(2))

    def run(settled):
        cache = pplb200.PagedKVCache.allocate(pages, page, hk, d, group)
        cache.v.fill_(1)
        for t in (cache.k_scale, cache.v_scale) if group else (cache.k, cache.v):
            t.fill_(float("nan"))  # what is read too early is lost
        att = pplb200.SharedPrefixDecodeAttention(cache, hq, batch, most, prefix)
        pages_now, lengths, length = cuda.full_like(every, -1), cuda.zeros(batch, dtype=cuda.int32, device="cuda"), cuda.zeros(1, dtype=cuda.int32, device="cuda")
        slots, positions = cuda.zeros(batch, dtype=cuda.int64, device="cuda"), cuda.zeros(batch, dtype=cuda.int64, device="cuda")
        outs, lses = cuda.zeros((steps, batch, hq, d), dtype=cuda.float16, device="cuda"), cuda.zeros((steps, batch, hq), device="cuda")
        number = cuda.arange(batch, device="cuda")

        def chain():
            wait = cuda.cuda.synchronize if settled else (lambda: None)
            lengths.zero_(), pages_now.fill_(-1), length.fill_(prefix - steps)
            pplb200.kv_cache_write(cache, k, v, at)
            for i in range(steps):
                positions.copy_(lengths)
                pages_now[:, i // page] = every[:, i // page]
                slots.copy_(every[number, i // page].long() * page + i % page)
                wait()
                q = pplb200.rotary_kv_cache_write(cache, rows[i, :, :hq], rows[i, :, hq:hq + hk], rows[i, :, hq + hk:], positions, slots, table)
                wait()
                lengths.add_(1), length.add_(1)
                wait()
                att(q, shared, length, pages_now, lengths, out=outs[i], lse=lses[i])
                wait()
        if settled:
            chain()
        else:
            graph, stream = cuda.cuda.CUDAGraph(), cuda.cuda.Stream()
            stream.wait_stream(cuda.cuda.current_stream())
            with cuda.cuda.graph(graph, stream=stream):
                chain()
            for _ in range(3):
                outs.zero_(), lses.zero_()
                graph.replay()
        cuda.cuda.synchronize()
        assert int(att.ws[3 * 592 * 8:3 * 592 * 8 + 4].view(cuda.int32)) == 0  # the word by which the next call's kernel goes ahead
        return outs, lses

    want, got = run(True), run(False)
    assert bool(cuda.isfinite(want[0]).all()) and cuda.equal(got[0], want[0]) and cuda.equal(got[1], want[1])


# ---- positions ----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("tokens", [1, 5, 3001])
@pytest.mark.parametrize("interleaved", [False, True])
def test_positions_expanded_over_the_axes(cuda, pplb200, tokens, interleaved):
    """A token of text has the same position on every axis: one row stands for all, in both calls, bit for bit as the rows written out and as one axis."""
    g = _gen(cuda, 5)
    q, k, v = _randn(cuda, g, tokens, 8, 64), _randn(cuda, g, tokens, 2, 64), _randn(cuda, g, tokens, 2, 64)
    pos, slots = cuda.randint(0, 100000, (tokens,), generator=g, device="cuda"), cuda.arange(tokens, device="cuda")
    one, table = pplb200.RotaryTable(64), pplb200.RotaryTable(64, axes=(12, 10, 10), alternating=True)
    caches = [pplb200.PagedKVCache.allocate(-(-tokens // 16), 16, 2, 64, 8) for _ in range(3)]
    got = [(pplb200.rotary_fp16(q, k, p, t, interleaved), pplb200.rotary_kv_cache_write(c, q, k, v, p, slots, t, interleaved))
           for c, p, t in zip(caches, (pos.expand(3, -1), pos.expand(3, -1).contiguous(), pos), (table, table, one))]
    for (qo, ko), qc in got:
        assert cuda.equal(qo, got[2][0][0]) and cuda.equal(ko, got[2][0][1]) and cuda.equal(qc, qo)
    for c in caches[:2]:
        assert cuda.equal(c.k, caches[2].k) and cuda.equal(c.k_scale, caches[2].k_scale)


# ---- choices among more blocks than the CTAs of a cluster tell each other -----------------------------------------------------

@pytest.mark.parametrize("lengths,hk,first,last,top", [([300000], 1, 1, 2, 40), ([270001, 290000], 1, 0, 1, 3000), ([280000], 2, 5, 3, 17000), ([400000, 7, 262145], 1, 3, 1, 1), ([300000], 1, 0, 1, 18000)])
def test_sparse_scores_across_a_cluster(cuda, pplb200, lengths, hk, first, last, top):
    """Over 16384 blocks: every CTA keeps the scores of its own share, and the threshold is found by all together.  Among so many keys some are infinite; their blocks are chosen first, and a
    head that has one attends to it has NaN by the definition too."""
    out, lse, want, _ = _run_sparse(cuda, pplb200, lengths, 2 * hk, hk, 64, 16, 16, 0, first, last, top)
    for b, (o, l, bound, lse_bound) in enumerate(want):
        lost = o.isnan().any(-1)
        assert bool(out[b][lost].isnan().all()) and bool(lse[b][lost].isnan().all())
        _check_attention(out[b:b + 1][:, ~lost], lse[b:b + 1][:, ~lost], [(o[~lost], l[~lost], bound[~lost], lse_bound[~lost])])


@pytest.mark.parametrize("top", [1, 300, 5000, 18747])
def test_sparse_ties_across_a_cluster(cuda, pplb200, top):
    """Equal scores in all shares but for a few blocks, holes among them: what is at the threshold is taken from the first share on."""
    def spoil(q, table, cache, bounds):
        bounds.bounds[:] = bounds.bounds[0, 0, 0]
        bounds.scales.fill_(1.0)
        for number, scale in ((40, 0.5), (5000, 2.0), (9999, 0.0), (18000, 2.0), (18001, float("inf"))):
            bounds.scales[table[0, number].long()] = scale
        table[0, 7000:7010] = -1
    _check_attention(*_run_sparse(cuda, pplb200, [300000], 2, 1, 64, 16, 16, 0, 1, 1, top, spoil=spoil)[:3])


# ---- caches of more than 2^32 bytes -------------------------------------------------------------------------------------------

@pytest.mark.parametrize("group,pages,page", [(0, 36000, 64), (0, 96000, 24), (8, 70000, 64), (128, 70000, 64)])
@pytest.mark.parametrize("order", ["heads", "tokens"])
def test_offsets_beyond_32_bits(cuda, pplb200, group, pages, page, order):
    """A prefix and own tokens on the cache's last pages, by tiles and by the decode kernel; blocks there, their bounds and the choice among them."""
    d, heads, n = 128, 8, 2000
    shape = (pages, heads, page) if order == "heads" else (pages, page, heads)
    make = lambda w, t: cuda.empty(shape + (w,), dtype=t, device="cuda")  # noqa: E731
    tensors = [make(d, cuda.int8 if group else cuda.float16) for _ in range(2)] + ([make(d // group, cuda.float16) for _ in range(2)] if group else [])
    assert tensors[0].numel() * tensors[0].element_size() > 1 << 32
    cache = pplb200.PagedKVCache(*(t if order == "heads" else t.transpose(1, 2) for t in tensors))
    g, count, i32 = _gen(cuda, 4), -(-n // page), dict(dtype=cuda.int32, device="cuda")
    table = (pages - 1 - cuda.randperm(2 * count, generator=g, device="cuda")[:count]).to(cuda.int32)
    table[::3] = cuda.arange(len(table[::3]), **i32)
    at = cuda.arange(count * page, device="cuda")
    slots = table.long()[at // page] * page + at % page
    pplb200.kv_cache_write(cache, _randn(cuda, g, len(at), heads, d), _randn(cuda, g, len(at), heads, d), slots)
    k, v = _stored(cuda, cache, slots[:n])
    first = n // 2 // page * page
    for batch in (2, 20):
        q = _randn(cuda, g, batch, 16, d)
        att = pplb200.SharedPrefixDecodeAttention(cache, 16, batch, (count - first // page) * page, first)
        out = att(q, table[:first // page].contiguous(), cuda.tensor([first], **i32), table[first // page:].expand(batch, -1).contiguous(), cuda.full((batch,), n - first, **i32))
        _check_attention(out, None, [_attention(cuda, x, k, v, at[:n] >= 0, att.scale, group == 8) for x in q])
    if page % 16:
        return
    bounds = pplb200.KeyBlockBounds(cache, 16)
    pplb200.key_bounds_update(bounds, slots)
    q, blocks = _randn(cuda, g, 1, 16, d), cuda.empty((1, heads, 33), **i32)
    att = pplb200.BlockSparseDecodeAttention(bounds, 16, 1, count * page, 1, 2, 30)
    out = att(q, table[None], cuda.tensor([n], **i32), blocks=blocks)
    chosen, parts = _choice(cuda, q[0], bounds, table, n, 1, 2, 30, pages), []
    for h in range(heads):
        assert blocks[0, h].tolist() == chosen[h]
        token = (cuda.tensor(chosen[h], device="cuda")[:, None] * 16 + cuda.arange(16, device="cuda")).flatten()
        token = token[token < n]
        parts.append(_attention(cuda, q[0, 2 * h:2 * h + 2], k[token, h:h + 1], v[token, h:h + 1], token >= 0, att.scale, group == 8))
    _check_attention(out, None, [tuple(cuda.cat(x) for x in zip(*parts))])


# ---- layouts of the cache -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("group", [0, 8, 128])
@pytest.mark.parametrize("layout", ["keys and values side by side", "one head for all", "wider rows", "a window of the pages"])
def test_layouts_of_the_cache(cuda, pplb200, layout, group):
    """Strides other than a dense tensor's: the same bits as over a dense copy, whichever way the tokens are brought.  (Rows further apart than long are other forms of the kernels.)"""
    g, pages, page, heads, d = _gen(cuda, 31), 90, 16, 4, 128
    wide = {"keys and values side by side": (pages, 2, heads, page), "one head for all": (pages, 2, 1, page), "wider rows": (pages, 2, heads, page), "a window of the pages": (pages + 9, 2, heads, page)}[layout]

    def laid(width, dtype):
        extra = 32 if layout == "wider rows" else 0
        t = cuda.randn(wide + (width + extra,), generator=g, device="cuda")
        t = (t * 40).clamp(-127, 127).to(cuda.int8) if dtype == cuda.int8 else (t.abs() * 0.02 if group else t).to(dtype)
        out = [t[:, i, ..., :width] for i in (0, 1)]
        if layout == "one head for all":
            return [x.expand(-1, heads, -1, -1) for x in out]
        return [x[4:4 + pages] for x in out] if layout == "a window of the pages" else out

    kv = laid(d, cuda.int8 if group else cuda.float16)
    scales = laid(d // group, cuda.float16) if group else []
    caches = [pplb200.PagedKVCache(*kv, *scales), pplb200.PagedKVCache(*(t.contiguous() for t in kv + scales))]
    i32 = dict(dtype=cuda.int32, device="cuda")
    table = cuda.randperm(pages, generator=g, device="cuda").to(cuda.int32)
    exact = layout != "wider rows"
    for batch, prefix in ((1, 900), (30, 900), (2, 60)):
        q, own = _randn(cuda, g, batch, 8, d), table[60:].view(1, -1).expand(batch, -1).contiguous()
        a, b = (pplb200.SharedPrefixDecodeAttention(c, 8, batch, 480, 960)(q, table[:60].contiguous(), cuda.tensor([prefix], **i32), own, cuda.full((batch,), 333, **i32)) for c in caches)
        assert bool(((a - b).abs().float() <= b.abs().float() * 4 * HALF + 2.0 ** -12).all()) and (cuda.equal(a, b) or not exact)
    both = [pplb200.KeyBlockBounds(c, 16) for c in caches]
    at = cuda.arange(pages * page, device="cuda")
    for b in both:
        pplb200.key_bounds_update(b, at)
    assert cuda.equal(both[0].bounds, both[1].bounds) and cuda.equal(both[0].scales, both[1].scales)
    q, blocks = _randn(cuda, g, 1, 8, d), [cuda.empty((1, heads, 20), **i32) for _ in caches]
    a, b = (pplb200.BlockSparseDecodeAttention(k, 8, 1, pages * page, 1, 2, 17)(q, table[None], cuda.tensor([1400], **i32), blocks=x) for k, x in zip(both, blocks))
    assert cuda.equal(*blocks) and bool(((a - b).abs().float() <= b.abs().float() * 4 * HALF + 2.0 ** -12).all()) and (cuda.equal(a, b) or not exact)


@pytest.mark.parametrize("group", [0, 8, 128])
def test_a_cache_without_pages(cuda, pplb200, group):
    """Every page is a hole: zeros and -inf, blocks chosen from the front."""
    cache = pplb200.PagedKVCache.allocate(0, 16, 2, 128, group)
    bounds = pplb200.KeyBlockBounds(cache, 16)
    i32 = dict(dtype=cuda.int32, device="cuda")
    pplb200.key_bounds_update(bounds, cuda.arange(64, device="cuda"))
    lo, hi = pplb200.key_bounds_read(bounds, cuda.arange(-1, 3, device="cuda"))
    assert not lo.any() and not hi.any()
    table = cuda.arange(100, **i32)
    for batch in (1, 40):
        q, out, lse = _randn(cuda, _gen(cuda, 1), batch, 8, 128), cuda.full((batch, 8, 128), 7.0, dtype=cuda.float16, device="cuda"), cuda.zeros((batch, 8), device="cuda")
        pplb200.SharedPrefixDecodeAttention(cache, 8, batch, 160, 1600)(q, table, cuda.tensor([1500], **i32), table[:10].expand(batch, -1).contiguous(), cuda.full((batch,), 99, **i32), out=out, lse=lse)
        assert not out.any() and bool((lse == -float("inf")).all())
        out.fill_(7.0), lse.zero_()
        blocks = cuda.empty((batch, 2, 9), **i32)
        pplb200.BlockSparseDecodeAttention(bounds, 8, batch, 1600, 1, 2, 6)(q, table.expand(batch, -1).contiguous(), cuda.full((batch,), 1590, **i32), out=out, lse=lse, blocks=blocks)
        assert not out.any() and bool((lse == -float("inf")).all()) and bool((blocks == cuda.tensor([0, 1, 2, 3, 4, 5, 6, 98, 99], **i32)).all())
