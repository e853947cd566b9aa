"""GPU-less checks of rotary positions of several axes, attention over a shared prefix, key bounds and attention over chosen blocks: the frequencies,
argument blocks, and every refusal (which come before anything is launched)."""
import ctypes
import os
import struct
import subprocess

import numpy as np
import pytest

from test_attention_cpu import AT, ATTEND, BAD_CACHES, ROOT, ROTARY, WRITE, _cache, _frequencies

AXES = dict(axis_of_plane=AT, stride=4, axes=3, reserved=0)
PREFIX = dict(pages=AT, length=AT, num_pages=10)
BOUNDS = dict(bounds=AT, scale=AT, block=16, reserved=0)
CHOICE = dict(first=1, last=2, top=3, reserved=0, blocks=0)


def _calls():
    from pplb200 import lib
    attend = lambda kw: struct.pack("=6Q6q2ifi", *dict(ATTEND, **kw).values())  # noqa: E731
    bounds = lambda kw: struct.pack("=2Q2i", *dict(BOUNDS, **kw).values())  # noqa: E731
    return dict(
        rotary=lambda axes={}, **kw: lib.pplb200_rotary_axes_fp16(None, struct.pack("=6Q5q5if", *dict(ROTARY, **kw).values()), struct.pack("=Qq2i", *dict(AXES, **axes).values())),
        write=lambda c, axes={}, **kw: lib.pplb200_kv_cache_write_axes_fp16(None, c, struct.pack("=7Q5q3if", *dict(WRITE, **kw).values()), struct.pack("=Qq2i", *dict(AXES, **axes).values())),
        prefix=lambda c, prefix={}, **kw: lib.pplb200_shared_prefix_attention_fp16(None, c, attend(kw), struct.pack("=2Qq", *dict(PREFIX, **prefix).values())),
        sparse=lambda c, k={}, choice={}, **kw: lib.pplb200_block_sparse_attention_fp16(None, c, bounds(k), attend(kw), struct.pack("=4iQ", *dict(CHOICE, **choice).values())),
        update=lambda c, slots=AT, tokens=4, **kw: lib.pplb200_key_bounds_update(None, c, bounds(kw), slots, tokens),
        read=lambda c, blocks=AT, count=4, lo=AT, hi=AT, **kw: lib.pplb200_key_bounds_read(None, c, bounds(kw), blocks, count, lo, hi))


def test_blocks_are_packed_as_declared(tmp_path):
    src = tmp_path / "c_caller.c"
    src.write_text('#include "pplb200_attention.h"\n#include <stdio.h>\n#include <stddef.h>\n'
                   'int main(void) {\n'
                   '    printf("%d %d %d %d\\n", (int)sizeof(pplb200_rotary_axes), (int)sizeof(pplb200_shared_prefix), (int)sizeof(pplb200_key_bounds), (int)sizeof(pplb200_block_choice));\n'
                   '    printf("%d %d %d %d\\n", (int)offsetof(pplb200_rotary_axes, axes), (int)offsetof(pplb200_shared_prefix, num_pages),\n'
                   '           (int)offsetof(pplb200_key_bounds, block), (int)offsetof(pplb200_block_choice, optional_blocks));\n'
                   '    return pplb200_block_sparse_attention_workspace_bytes(1, 3, 2, 128, 4) == -1 && PPLB200_ROTARY_MAX_AXES == 4 ? 0 : 1;\n}\n')
    exe = tmp_path / "c_caller"
    lib_dir = os.path.join(ROOT, "ppl.llm.kernel.cuda_b200", "lib")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Wextra", "-Werror", "-pedantic", "-I" + os.path.join(ROOT, "include"),
                    str(src), "-o", str(exe), "-L" + lib_dir, "-lpplb200_i8i8", "-Wl,-rpath," + lib_dir], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()
    assert [int(v) for v in out] == [struct.calcsize(f) for f in ("=Qq2i", "=2Qq", "=2Q2i", "=4iQ", "=Qq", "=2Q", "=2Q", "=4i")]


# ---- frequencies of several axes -----------------------------------------------------------------------------------

def _axis_of_plane(planes, alternating):
    if not alternating:
        return [a for a, n in enumerate(planes) for _ in range(n)]
    return [a for turn in range(max(planes)) for a, n in enumerate(planes) if turn < n]


SCALINGS = [("none", 1.0, 0, 0, 0), ("linear", 4.0, 0, 0, 0), ("ntk", 8.0, 0, 0, 0), ("yarn", 32.0, 4096, 32, 1), ("wavelength", 8.0, 8192, 4, 1)]


@pytest.mark.parametrize("kind,factor,original,keep,stretch", SCALINGS)
@pytest.mark.parametrize("planes", [(24, 20, 20), (64,), (1, 63), (0, 32, 0, 32), (16, 16, 16, 16), (1, 1, 1, 61)])
@pytest.mark.parametrize("alternating", [False, True])
@pytest.mark.parametrize("restart", [False, True])
def test_frequencies_of_axes(kind, factor, original, keep, stretch, planes, alternating, restart):
    import pplb200
    t = pplb200.RotaryTable(128, base=10000.0, scaling=kind, factor=factor, original_length=original, keep_turns=keep, stretch_turns=stretch, device="cpu",
                            axes=planes, alternating=alternating, restart=restart)
    of = _axis_of_plane(planes, alternating)
    assert t.axis_of_plane.tolist() == of and t.axes == planes
    plain = pplb200.RotaryTable(128, base=10000.0, scaling=kind, factor=factor, original_length=original, keep_turns=keep, stretch_turns=stretch, device="cpu")
    assert t.magnitude == plain.magnitude
    if not restart:
        assert t.turns.tolist() == plain.turns.tolist()
        return
    got = t.turns.numpy().view(np.uint64).astype(np.longdouble) / np.longdouble(2.0) ** 64 * 2 * np.longdouble("3.14159265358979323846264338327950288")
    for axis, n in enumerate(planes):
        if n == 1:  # the first plane of a series: whatever the base, NTK's too, one radian a position before the scaling
            want = np.array([np.longdouble(1.0)]) if kind in ("none", "ntk") else _frequencies(2, 10000.0, kind, factor, original, keep, stretch)
        elif n:
            want = _frequencies(2 * n, 10000.0, kind, factor, original, keep, stretch)
        else:
            continue
        mine = got[[i for i, a in enumerate(of) if a == axis]]
        # pow and a few products in 64 bits; the word itself resolves 2^-64 of a turn
        assert np.all(np.abs(mine - want) <= np.abs(want) * 64 * 2.0 ** -53 + 8 * 2.0 ** -64)


@pytest.mark.parametrize("args,rc", [(dict(axes=()), 2), (dict(axes=(8,) * 5), 2), (dict(axes=(16, 15)), 4), (dict(axes=(16, 17)), 4), (dict(axes=(33, -1)), 4), (dict(axes=(1 << 31 - 1, 32)), 4),
                                     (dict(axes=(16, 16), base=1.0), 4), (dict(axes=(16, 16), scaling="yarn", factor=2.0), 4), (dict(axes=(10, 10), rotary_dim=40), 4)])
def test_frequency_refusals_of_axes(args, rc):
    import pplb200
    with pytest.raises(pplb200.PplError) as e:
        pplb200.RotaryTable(**dict(dict(rotary_dim=64, device="cpu"), **args))
    assert e.value.rc == rc and pplb200.last_error()


def test_frequency_refusals_of_pointers():
    from pplb200 import lib
    good = [(ctypes.c_int32 * 2)(16, 16), 0, 0, (ctypes.c_uint64 * 32)(), (ctypes.c_uint8 * 32)(), ctypes.byref(ctypes.c_float())]
    call = lambda a: lib.pplb200_rotary_axes_frequencies(64, 1e4, 0, 1.0, 0.0, 0.0, 0.0, 2, *a)  # noqa: E731
    assert call(good) == 0
    for i in (0, 3, 4, 5):
        assert call([None if j == i else x for j, x in enumerate(good)]) == 4


def test_arrangements_are_of_axes():
    import pplb200
    for kw in (dict(alternating=True), dict(restart=True)):
        with pytest.raises(ValueError):
            pplb200.RotaryTable(64, device="cpu", **kw)


# ---- refusals --------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("axes,rc", [(dict(axes=0), 2), (dict(axes=5), 2), (dict(axes=-1), 2), (dict(axis_of_plane=0), 4), (dict(axis_of_plane=AT + 2), 4), (dict(stride=3), 4), (dict(stride=-4), 4), (dict(axes=1, stride=-1), 4)])
def test_axes_refusals(axes, rc):
    import pplb200
    c = _calls()
    assert c["rotary"](axes) == c["write"](_cache(), axes) == rc and pplb200.last_error()


@pytest.mark.parametrize("bad,rc", [(dict(tokens=-1), 4), (dict(rd=24), 4), (dict(turns=0), 4), (dict(positions=0), 4), (dict(q=0), 4), (dict(k=AT + 2), 4), (dict(q_stride=512), 4)])
def test_calls_with_axes_refuse_what_those_with_one_do(bad, rc):
    c = _calls()
    assert c["rotary"](**bad) == c["write"](_cache(), **bad) == rc


def test_axes_without_a_rotation():
    c = _calls()
    assert c["write"](_cache(), rd=0) == 4 and c["write"](_cache(), tokens=0) == c["rotary"](tokens=0) == 0
    from pplb200 import lib
    assert lib.pplb200_rotary_axes_fp16(None, struct.pack("=6Q5q5if", *ROTARY.values()), None) == 4
    assert lib.pplb200_kv_cache_write_axes_fp16(None, _cache(), struct.pack("=7Q5q3if", *WRITE.values()), None) == 4


@pytest.mark.parametrize("bad,rc", BAD_CACHES)
def test_bad_caches(bad, rc):
    c, cache = _calls(), _cache(**bad)
    assert c["prefix"](cache) == c["sparse"](cache) == c["update"](cache) == c["read"](cache) == c["write"](cache) == rc


@pytest.mark.parametrize("bad,rc", [
    (dict(batch=-1), 4), (dict(batch=70000), 2), (dict(width=-1), 4), (dict(width=1 << 40, pages_stride=1 << 40), 2), (dict(q_heads=0), 4), (dict(q_heads=12), 4), (dict(scale=float("nan")), 4),
    (dict(q=0), 4), (dict(out=AT + 2), 4), (dict(q_stride=1020), 4), (dict(out_stride=512), 4), (dict(pages=0), 4), (dict(lengths=0), 4), (dict(pages=AT + 2), 4), (dict(lse=AT + 2), 4),
    (dict(pages_stride=9), 4), (dict(ws=0), 4), (dict(ws=AT + 16), 4), (dict(ws_bytes=16), 4), (dict(window=5), 2)])
def test_attention_refusals(bad, rc):
    import pplb200
    c = _calls()
    assert c["prefix"](_cache(), **bad) == c["sparse"](_cache(), **bad) == rc and pplb200.last_error()


@pytest.mark.parametrize("hq,hk", [(1, 1), (8, 1), (32, 8), (64, 8), (20, 20), (256, 1), (300, 300)])
@pytest.mark.parametrize("d", [64, 256])
def test_a_workspace_fits_every_smaller_batch(hq, hk, d):
    from pplb200 import lib
    sizes = [lib.pplb200_shared_prefix_attention_workspace_bytes(b, hq, hk, d) for b in list(range(1100)) + list(range(1100, 40000, 997))]
    assert all(s > 0 and s % 256 == 0 for s in sizes) and sizes == sorted(sizes)


@pytest.mark.parametrize("bad,rc", [(dict(pages=0), 4), (dict(length=0), 4), (dict(pages=AT + 2), 4), (dict(length=AT + 1), 4), (dict(num_pages=-1), 4), (dict(num_pages=1 << 40), 2)])
def test_prefix_refusals(bad, rc):
    import pplb200
    assert _calls()["prefix"](_cache(), bad) == rc and pplb200.last_error()


def test_prefix_rows():
    from pplb200 import lib
    big = dict(q_heads=65528, q_stride=65528 * 128, out_stride=65528 * 128)
    assert _calls()["prefix"](_cache(), batch=300, **big) == 2
    need = lib.pplb200_shared_prefix_attention_workspace_bytes
    assert need(300, 65528, 8, 128) == need(-1, 8, 8, 128) == need(1, 0, 8, 128) == need(1, 9, 8, 128) == need(1, 8, 0, 128) == need(1, 8, 8, 0) == -1
    sizes = [need(b, 64, 8, 128) for b in (0, 1, 2, 16, 300, 65535)]
    assert all(s > 0 and s % 256 == 0 for s in sizes) and sizes == sorted(sizes)


@pytest.mark.parametrize("k,rc", [(dict(block=0), 4), (dict(block=-16), 4), (dict(block=8), 4), (dict(block=32), 4), (dict(bounds=0), 4), (dict(scale=0), 4), (dict(bounds=AT + 8), 4), (dict(scale=AT + 1), 4)])
def test_bounds_refusals(k, rc):
    import pplb200
    c = _calls()
    assert c["sparse"](_cache(), k) == c["update"](_cache(), **k) == c["read"](_cache(), **k) == rc and pplb200.last_error()


def test_bounds_of_blocks_beyond_all_measure():
    c, page = _calls(), (1 << 31) - 16
    cache = _cache(page=page, token_stride=0, head_stride=0, page_stride=0, stoken=0, shead=0, spage=0)
    assert c["update"](cache, block=page) == c["read"](cache, block=page) == 2


def test_bounds_refusals_of_calls():
    c = _calls()
    assert c["update"](_cache(), tokens=-1) == c["update"](_cache(), slots=0) == c["update"](_cache(), slots=AT + 4) == 4 and c["update"](_cache(), tokens=1 << 31) == 2
    assert c["read"](_cache(), count=-1) == c["read"](_cache(), blocks=0) == c["read"](_cache(), blocks=AT + 4) == c["read"](_cache(), lo=0) == c["read"](_cache(), hi=AT + 8) == 4
    assert c["read"](_cache(), count=1 << 40) == 2
    assert c["update"](_cache(), tokens=0, slots=0) == c["read"](_cache(), count=0, blocks=0, lo=0, hi=0) == c["sparse"](_cache(), batch=0) == c["prefix"](_cache(), batch=0) == 0
    for dim in (16, 80, 112, 160):
        cache = _cache(dim=dim, group=dim, token_stride=dim, head_stride=16 * dim, page_stride=128 * dim)
        stride = dict(q_stride=8 * dim, out_stride=8 * dim)
        assert c["update"](cache) == c["read"](cache) == c["sparse"](cache, **stride) == c["prefix"](cache, **stride) == 2


@pytest.mark.parametrize("choice,rc", [(dict(first=-1), 4), (dict(last=0), 4), (dict(top=-1), 4), (dict(top=65534), 2), (dict(first=1 << 30, top=1 << 30, last=1 << 30), 2), (dict(blocks=AT + 2), 4)])
def test_choice_refusals(choice, rc):
    import pplb200
    assert _calls()["sparse"](_cache(), {}, choice) == rc and pplb200.last_error()


def test_choice_refusals_of_extents():
    from pplb200 import lib
    c = _calls()
    assert c["sparse"](_cache(), width=(1 << 18) + 1, pages_stride=1 << 20) == 2  # blocks of a row
    many = _cache(pages=1 << 30, page=64, page_stride=0, head_stride=0, token_stride=0, spage=0, shead=0, stoken=0)
    assert c["sparse"](many) == 2  # blocks of the cache
    heads = _cache(heads=65528, head_stride=0, shead=0)
    assert c["sparse"](heads, q_heads=65528, q_stride=65528 * 128, out_stride=65528 * 128, batch=300) == 2
    need = lib.pplb200_block_sparse_attention_workspace_bytes
    assert need(-1, 8, 8, 128, 4) == need(1, 0, 8, 128, 4) == need(1, 9, 8, 128, 4) == need(1, 8, 0, 128, 4) == need(1, 8, 8, 128, -1) == need(300, 65528, 65528, 128, 4) == -1
    sizes = [need(b, 64, 8, 128, n) for b, n in ((0, 0), (1, 4), (16, 64), (256, 128), (256, 65536))]
    assert all(s > 0 and s % 256 == 0 for s in sizes) and sizes == sorted(sizes)


def test_null_blocks():
    from pplb200 import lib
    attend, k = struct.pack("=6Q6q2ifi", *ATTEND.values()), struct.pack("=2Q2i", *BOUNDS.values())
    assert lib.pplb200_shared_prefix_attention_fp16(None, _cache(), attend, None) == lib.pplb200_shared_prefix_attention_fp16(None, _cache(), None, attend) == 4
    assert lib.pplb200_block_sparse_attention_fp16(None, _cache(), k, attend, None) == lib.pplb200_block_sparse_attention_fp16(None, _cache(), None, attend, attend) == 4
    assert lib.pplb200_key_bounds_update(None, _cache(), None, AT, 4) == lib.pplb200_key_bounds_read(None, _cache(), None, AT, 4, AT, AT) == 4


def test_status_without_a_device():
    import pplb200
    import torch
    if not torch.cuda.is_available():
        assert pplb200.shared_prefix_status() == -1


# ---- the binding: types, shapes and devices (the tensors are on the CPU, which is never the current device) ---------

@pytest.fixture
def here(monkeypatch):
    """The binding with CPU tensors taken for the current device's and the C calls recorded, their last argument block as bytes."""
    from pplb200 import attention
    calls, keep = [], []
    monkeypatch.setattr(attention, "_here", lambda: (-1, 0))
    vp, i64 = ctypes.c_void_p, ctypes.c_int64
    for n, types, size in (("_rotary_axes", (vp, vp, vp), 24), ("_write_axes", (vp, vp, vp, vp), 24), ("_attend_prefix", (vp, vp, vp, vp), 24), ("_attend_blocks", (vp, vp, vp, vp, vp), 24),
                           ("_bounds_update", (vp, vp, vp, vp, i64), 0), ("_bounds_read", (vp, vp, vp, vp, i64, vp, vp), 0)):
        f = ctypes.CFUNCTYPE(ctypes.c_int32, *types)(lambda *a, n=n, size=size: calls.append((n, a[:-1] + (ctypes.string_at(a[-1], size),) if size else a)) or 0)
        keep.append(f)
        monkeypatch.setattr(attention, n, ctypes.cast(f, vp).value)
    yield calls
    del keep


def _objects(pplb200):
    cache = pplb200.PagedKVCache.allocate(6, 32, 2, 64, 0, device="cpu")
    bounds = pplb200.KeyBlockBounds(cache, 16)
    return (cache, bounds, pplb200.SharedPrefixDecodeAttention(cache, 4, 3, 64, 96), pplb200.BlockSparseDecodeAttention(bounds, 4, 3, 64, 1, 1, 2),
            pplb200.RotaryTable(64, device="cpu", axes=(16, 8, 8)))


def test_binding_passes_what_it_is_given(here):
    import torch
    import pplb200
    cache, bounds, shared, sparse, table = _objects(pplb200)
    f16 = lambda *s: torch.zeros(s, dtype=torch.float16)  # noqa: E731
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    pos = torch.zeros((3, 9), dtype=torch.int64)[:, 2:7]
    pplb200.rotary_fp16(f16(5, 4, 64), f16(5, 2, 64), pos, table)
    assert struct.unpack("=Qq2i", here[-1][1][-1]) == (table.axis_of_plane.data_ptr(), 9, 3, 0)
    pplb200.rotary_kv_cache_write(cache, None, f16(5, 2, 64), f16(5, 2, 64), pos, torch.zeros(5, dtype=torch.int64), table)
    assert here[-1][0] == "_write_axes" and struct.unpack("=Qq2i", here[-1][1][-1])[1:3] == (9, 3)
    prefix, length = i32(3), i32(1)
    shared(f16(2, 4, 64), prefix, length, i32(2, 2), i32(2), lse=torch.zeros((2, 4)))
    assert struct.unpack("=2Qq", here[-1][1][-1]) == (prefix.data_ptr(), length.data_ptr(), 3)
    blocks = i32(2, 2, 4)
    sparse(f16(2, 4, 64), i32(2, 2), i32(2), blocks=blocks)
    assert struct.unpack("=4iQ", here[-1][1][-1]) == (1, 1, 2, 0, blocks.data_ptr())
    slots = torch.zeros(7, dtype=torch.int64)
    pplb200.key_bounds_update(bounds, slots)
    assert here[-1][0] == "_bounds_update" and here[-1][1][3:] == (slots.data_ptr(), 7)
    lo, hi = pplb200.key_bounds_read(bounds, slots)
    assert lo.shape == hi.shape == (7, 2, 64) and here[-1][1][3:] == (slots.data_ptr(), 7, lo.data_ptr(), hi.data_ptr())


def test_binding_refusals(here):
    import torch
    import pplb200
    cache, bounds, shared, sparse, table = _objects(pplb200)
    f16 = lambda *s: torch.zeros(s, dtype=torch.float16)  # noqa: E731
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    i64 = lambda *s: torch.zeros(s, dtype=torch.int64)  # noqa: E731
    q, p, n, pages, lens = f16(2, 4, 64), i32(3), i32(1), i32(2, 2), i32(2)
    for x in (i64(2), i64(2, 2), i64(3, 3), i32(3, 2), i64(2, 3).T):
        with pytest.raises(ValueError):
            pplb200.rotary_fp16(q, None, x, table)
    for args in ((q, i32(4), n, pages, lens), (q, i64(3), n, pages, lens), (q, i32(1, 3), n, pages, lens), (q, i32(6)[::2], n, pages, lens), (q, p, i32(2), pages, lens), (q, p, i64(1), pages, lens),
                 (f16(4, 4, 64), p, n, i32(4, 2), i32(4)), (f16(2, 2, 64), p, n, pages, lens), (q, p, n, i32(2, 3), lens), (q, p, n, pages, i32(3)), (q, p, n, pages, i64(2))):
        with pytest.raises(ValueError):
            shared(*args)
    for kw in (dict(blocks=i32(2, 2, 5)), dict(blocks=i64(2, 2, 4)), dict(blocks=i32(2, 4, 4)), dict(lse=f16(2, 4)), dict(out=f16(2, 4, 32))):
        with pytest.raises(ValueError):
            sparse(q, pages, lens, **kw)
    for x in (i32(4), i64(4, 1), i64(8)[::2]):
        with pytest.raises(ValueError):
            pplb200.key_bounds_update(bounds, x)
    with pytest.raises(ValueError):
        pplb200.key_bounds_read(bounds, i64(4), lo_out=torch.zeros((4, 2, 32)))
    for kw in (dict(block=0), dict(block=8), dict(block=64), dict(block=16, bounds=bounds.bounds), dict(block=16, bounds=bounds.bounds, scales=bounds.scales[:5]), dict(block=32, bounds=bounds.bounds, scales=bounds.scales),
               dict(block=16, bounds=bounds.bounds.float(), scales=bounds.scales)):
        with pytest.raises(ValueError):
            pplb200.KeyBlockBounds(cache, **kw)
    for kw in (dict(first=-1), dict(last=0), dict(top=-2), dict(top=70000), dict(q_heads=3), dict(max_batch=-1)):
        with pytest.raises(ValueError):
            pplb200.BlockSparseDecodeAttention(bounds, **dict(dict(q_heads=4, max_batch=1, max_length=9, first=1, last=1, top=1), **kw))
    for kw in (dict(q_heads=3), dict(max_batch=-1), dict(max_length=-1), dict(max_prefix=-1)):
        with pytest.raises(ValueError):
            pplb200.SharedPrefixDecodeAttention(cache, **dict(dict(q_heads=4, max_batch=1, max_length=9, max_prefix=9), **kw))
    assert not here
    for o in (bounds, shared, sparse):
        with pytest.raises(AttributeError):
            o.cache = None
