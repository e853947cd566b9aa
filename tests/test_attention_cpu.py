"""GPU-less checks of rotary positions, the paged cache and decode attention: the C header and its argument blocks, the
frequencies, the index arithmetic of the cache, and every refusal (which come before anything is launched)."""
import ctypes
import math
import os
import re
import struct
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "pplb200_attention.h")


def test_library_exports_every_declared_symbol():
    import pplb200
    from pplb200 import attention
    src = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = set(re.findall(r"\b(pplb200_[a-z0-9_]+)\s*\(", src))
    assert names == set(attention.EXPORTS)
    assert all(hasattr(pplb200.lib, n) for n in names)


def test_header_is_plain_c99_and_blocks_are_packed_as_declared(tmp_path):
    src = tmp_path / "c_caller.c"
    src.write_text('#include "pplb200_attention.h"\n#include <stdio.h>\n#include <stddef.h>\n'
                   'int main(void) {\n'
                   '    printf("%d %d %d %d\\n", (int)sizeof(pplb200_kv_cache), (int)sizeof(pplb200_rotary_args),\n'
                   '           (int)sizeof(pplb200_kv_write_args), (int)sizeof(pplb200_paged_attention_args));\n'
                   '    printf("%d %d %d %d\\n", (int)offsetof(pplb200_kv_cache, page_size), (int)offsetof(pplb200_rotary_args, magnitude),\n'
                   '           (int)offsetof(pplb200_kv_write_args, q_heads), (int)offsetof(pplb200_paged_attention_args, scale));\n'
                   '    return pplb200_paged_decode_attention_workspace_bytes(1, 16, 3, 2, 128) == -1 ? 0 : 1;\n}\n')
    exe = tmp_path / "c_caller"
    lib_dir = os.path.join(ROOT, "ppl.llm.kernel.cuda_b200", "lib")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Wextra", "-Werror", "-pedantic", "-I" + os.path.join(ROOT, "include"),
                    str(src), "-o", str(exe), "-L" + lib_dir, "-lpplb200_i8i8", "-Wl,-rpath," + lib_dir], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()
    formats = ("=4Q7q4i", "=6Q5q5if", "=7Q5q3if", "=6Q6q2ifi")
    assert [int(v) for v in out[:4]] == [struct.calcsize(f) for f in formats]
    assert [int(v) for v in out[4:]] == [struct.calcsize(f) for f in ("=4Q7q", "=6Q5q5i", "=7Q5q", "=6Q6q2i")]


# ---- frequencies ---------------------------------------------------------------------------------------------------

def _frequencies(rd, base, kind, factor, original, keep, stretch):
    """The definitions, plane by plane, in extended precision."""
    ld = np.longdouble
    out = []
    for i in range(rd // 2):
        f = ld(base) ** (ld(-2 * i) / rd)
        if kind == "linear":
            f /= factor
        elif kind == "ntk":
            f = (ld(base) * ld(factor) ** (ld(rd) / (rd - 2))) ** (ld(-2 * i) / rd)
        elif kind == "yarn":
            ends = [rd * math.log(original / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (keep, stretch)]
            first, last = max(math.floor(ends[0]), 0), min(math.ceil(ends[1]), rd - 1)
            part = min(1.0, max(0.0, (i - first) / max(last - first, 0.001)))
            f = f * (1 - part) + f / factor * part
        elif kind == "wavelength":
            turns = original * f / (2 * ld(math.pi))
            part = min(ld(1), max(ld(0), (turns - stretch) / (keep - stretch)))
            f = f * part + f / factor * (1 - part)
        out.append(f)
    return np.array(out)


@pytest.mark.parametrize("kind,factor,original,keep,stretch", [
    ("none", 1.0, 0, 0, 0), ("linear", 4.0, 0, 0, 0), ("ntk", 8.0, 0, 0, 0), ("yarn", 32.0, 4096, 32, 1), ("wavelength", 8.0, 8192, 4, 1),
    ("yarn", 1.0, 4096, 32, 1), ("yarn", 4.0, 8, 32, 1)])
@pytest.mark.parametrize("rd,base", [(16, 10000.0), (64, 10000.0), (96, 500000.0), (128, 1000000.0), (256, 10000.0)])
def test_frequencies(kind, factor, original, keep, stretch, rd, base):
    import pplb200
    t = pplb200.RotaryTable(rd, base=base, scaling=kind, factor=factor, original_length=original, keep_turns=keep, stretch_turns=stretch, device="cpu")
    got = t.turns.numpy().view(np.uint64).astype(np.longdouble) / np.longdouble(2.0) ** 64 * 2 * np.longdouble("3.14159265358979323846264338327950288")
    want = _frequencies(rd, base, kind, factor, original, keep, stretch)
    assert got.shape == (rd // 2,)
    # pow and a few products in 64 bits; the word itself resolves 2^-64 of a turn
    assert np.all(np.abs(got - want) <= np.abs(want) * 64 * 2.0 ** -53 + 8 * 2.0 ** -64)
    assert t.magnitude == np.float32(0.1 * math.log(factor) + 1.0 if kind == "yarn" else 1.0)


@pytest.mark.parametrize("kind,factor,original,keep,stretch", [
    ("none", 1.0, 0, 0, 0), ("linear", 3.0, 0, 0, 0), ("ntk", 8.0, 0, 0, 0), ("yarn", 32.0, 4096, 32, 1), ("wavelength", 7.0, 8192, 4, 1)])
@pytest.mark.parametrize("rd,base", [(16, 10000.0), (96, 500000.0), (128, 10000.0), (256, 1000000.0)])
def test_words_of_a_turn_hold_to_their_last_bits(kind, factor, original, keep, stretch, rd, base):
    """An error of a word grows with the position; in the words of 64-bit arithmetic it was 2^-56 of a turn."""
    import decimal
    import pplb200
    D = decimal.Decimal
    t = pplb200.RotaryTable(rd, base=base, scaling=kind, factor=factor, original_length=original, keep_turns=keep, stretch_turns=stretch, device="cpu")
    with decimal.localcontext() as context:
        context.prec = 60
        two_pi = 2 * D("3.14159265358979323846264338327950288419716939937510582097494459")
        for i, word in enumerate(t.turns.numpy().view(np.uint64)):
            b = D(base) * D(factor) ** (D(rd) / (rd - 2)) if kind == "ntk" else D(base)
            f = b ** (D(-2 * i) / rd)
            part = D(1)
            if kind == "yarn":
                ends = [rd * math.log(original / (x * 2 * math.pi)) / (2 * math.log(base)) for x in (keep, stretch)]
                first, last = max(math.floor(ends[0]), 0), min(math.ceil(ends[1]), rd - 1)
                part = 1 - D(i - first) / max(last - first, D("0.001"))
            elif kind == "wavelength":
                part = (original * f / two_pi - D(stretch)) / (D(keep) - D(stretch))
            part = min(D(1), max(D(0), part)) if kind != "linear" else D(0)
            f = f * part + f / D(factor) * (1 - part)
            # half a unit for the word; in front of it some ten roundings to 64 bits of numbers below 2^62 of these units
            assert abs(D(int(word)) - f / two_pi * 2 ** 64) <= 4


@pytest.mark.parametrize("args,rc", [
    (dict(rotary_dim=0), 4), (dict(rotary_dim=24), 4), (dict(rotary_dim=272), 4), (dict(rotary_dim=64, base=1.0), 4), (dict(rotary_dim=64, base=float("nan")), 4),
    (dict(rotary_dim=64, base=float("inf")), 4), (dict(rotary_dim=64, scaling="linear", factor=0.5), 4), (dict(rotary_dim=64, scaling="ntk", factor=float("nan")), 4),
    (dict(rotary_dim=64, scaling="yarn", factor=2.0), 4), (dict(rotary_dim=64, scaling="yarn", factor=2.0, original_length=4096, keep_turns=1, stretch_turns=1), 4),
    (dict(rotary_dim=64, scaling="wavelength", factor=2.0, original_length=4096, keep_turns=4, stretch_turns=0), 4)])
def test_frequency_refusals(args, rc):
    import pplb200
    with pytest.raises(pplb200.PplError) as e:
        pplb200.RotaryTable(device="cpu", **args)
    assert e.value.rc == rc and pplb200.last_error()


def test_unknown_scaling():
    import pplb200
    with pytest.raises(ValueError):
        pplb200.RotaryTable(64, scaling="dynamic", device="cpu")
    words, mag = (ctypes.c_uint64 * 32)(), ctypes.c_float()
    assert pplb200.lib.pplb200_rotary_frequencies(64, 1e4, 5, 1.0, 0.0, 0.0, 0.0, words, ctypes.byref(mag)) == pplb200.RC_UNSUPPORTED
    assert pplb200.lib.pplb200_rotary_frequencies(64, 1e4, 0, 1.0, 0.0, 0.0, 0.0, None, ctypes.byref(mag)) == pplb200.RC_INVALID_VALUE


# ---- the cache: where rows lie, what is refused --------------------------------------------------------------------

AT = 1 << 20  # an aligned address; nothing in this file gets as far as using one
CACHE = dict(k=AT, v=AT, ks=AT, vs=AT, pages=100, page_stride=8 * 16 * 128, head_stride=16 * 128, token_stride=128,
             spage=8 * 16, shead=16, stoken=1, page=16, heads=8, dim=128, group=128)


def _cache(**kw):
    return struct.pack("=4Q7q4i", *dict(CACHE, **kw).values())


def test_offsets():
    import pplb200
    at = lambda slot, head, **kw: pplb200.lib.pplb200_kv_cache_offset(_cache(**kw), slot, head)  # noqa: E731
    assert at(0, 0) == 0 and at(17, 3) == 16384 + 3 * 2048 + 128
    assert at(1599, 7) == 99 * 16384 + 7 * 2048 + 15 * 128
    # slots that the cache does not have
    assert at(-1, 0) == at(1600, 0) == at(-1 << 62, 0) == at(1 << 40, 0) == at((1 << 63) - 1, 0) == at(0, 8) == at(0, -1) == -1
    # a page of one token, an odd page, tokens first, and rows beyond 2^31 and 2^32 elements
    assert at(99, 0, page=1) == 99 * 16384 and at(100, 0, page=1) == -1
    assert at(23, 1, page=7) == 3 * 16384 + 2048 + 2 * 128
    assert at(17, 3, head_stride=128, token_stride=1024) == 16384 + 3 * 128 + 1024
    big = 1 << 33
    assert at(big - 1, 7, pages=big // 16) == (big // 16 - 1) * 16384 + 7 * 2048 + 15 * 128
    assert at(big, 7, pages=big // 16) == -1


def test_int32_boundaries_of_the_slot_division():
    import pplb200
    for page in (1, 3, 16, 24, 1000003):
        pages = (1 << 34) // page
        for slot in (0, (1 << 31) - 1, 1 << 31, (1 << 32) - 1, 1 << 32, (1 << 32) + 12345, pages * page - 1):
            got = pplb200.lib.pplb200_kv_cache_offset(_cache(page=page, pages=pages, page_stride=16 * 1000003, head_stride=0, token_stride=16), slot, 0)
            assert got == slot // page * 16 * 1000003 + slot % page * 16


BAD_CACHES = [(dict(pages=-1), 4), (dict(page=0), 4), (dict(heads=0), 4), (dict(heads=70000), 4), (dict(dim=0), 2), (dict(dim=100), 2), (dict(dim=272), 2), (dict(group=16), 2),
              (dict(group=-8), 2), (dict(k=0), 4), (dict(v=0), 4), (dict(ks=0), 4), (dict(vs=0), 4), (dict(k=AT + 8), 4), (dict(v=AT + 1), 4),
              (dict(page_stride=-16), 4), (dict(head_stride=8), 4), (dict(token_stride=100), 4), (dict(group=0, token_stride=100), 4),
              (dict(spage=-1), 4), (dict(shead=-1), 4), (dict(stoken=-1), 4), (dict(ks=AT + 1), 4)]
WRITE = dict(q=AT, k=AT, v=AT, q_out=AT, positions=AT, slots=AT, turns=AT, tokens=4, q_stride=1024, k_stride=1024, v_stride=1024, qo_stride=1024,
             q_heads=8, rd=128, interleaved=0, magnitude=1.0)
ROTARY = dict(q=AT, k=AT, q_out=AT, k_out=AT, positions=AT, turns=AT, tokens=4, q_stride=1024, k_stride=1024, qo_stride=1024, ko_stride=1024,
              q_heads=8, k_heads=8, dim=128, rd=128, interleaved=0, magnitude=1.0)
ATTEND = dict(q=AT, out=AT, lse=0, pages=AT, lengths=AT, ws=AT, ws_bytes=1 << 40, batch=4, width=10, pages_stride=10, q_stride=1024, out_stride=1024,
              q_heads=8, window=0, scale=0.1, reserved=0)


def _calls():
    import pplb200
    return (lambda c, **kw: pplb200.lib.pplb200_kv_cache_write_fp16(None, c, struct.pack("=7Q5q3if", *dict(WRITE, **kw).values())),
            lambda **kw: pplb200.lib.pplb200_rotary_fp16(None, struct.pack("=6Q5q5if", *dict(ROTARY, **kw).values())),
            lambda c, **kw: pplb200.lib.pplb200_paged_decode_attention_fp16(None, c, struct.pack("=6Q6q2ifi", *dict(ATTEND, **kw).values())))


@pytest.mark.parametrize("bad,rc", BAD_CACHES)
def test_bad_caches(bad, rc):
    import pplb200
    write, _, attend = _calls()
    c = _cache(**bad)
    assert write(c) == attend(c) == rc and pplb200.last_error()
    assert pplb200.lib.pplb200_kv_cache_read_fp16(None, c, AT, 4, AT, AT) == rc
    assert pplb200.lib.pplb200_kv_cache_offset(c, 0, 0) == -1


@pytest.mark.parametrize("bad,rc", [
    (dict(tokens=-1), 4), (dict(tokens=1 << 31), 2), (dict(slots=0), 4), (dict(slots=AT + 4), 4), (dict(rd=-16), 4), (dict(rd=24), 4), (dict(rd=144), 4),
    (dict(turns=0), 4), (dict(positions=0), 4), (dict(positions=AT + 4), 4), (dict(turns=AT + 4), 4), (dict(q=0), 4), (dict(q=AT + 2), 4), (dict(q_out=0), 4),
    (dict(q_out=AT + 8), 4), (dict(k=0), 4), (dict(v=0), 4), (dict(k=AT + 2), 4), (dict(v=AT + 8), 4), (dict(q_stride=1020), 4), (dict(k_stride=1016), 4), (dict(v_stride=-1024), 4),
    (dict(qo_stride=512), 4), (dict(q_heads=-1), 4), (dict(q_heads=1 << 20, q_stride=1 << 40), 4)])
def test_write_refusals(bad, rc):
    import pplb200
    assert _calls()[0](_cache(), **bad) == rc and pplb200.last_error()


@pytest.mark.parametrize("bad,rc", [
    (dict(tokens=-1), 4), (dict(tokens=1 << 31), 2), (dict(dim=0), 2), (dict(dim=72), 2), (dict(dim=512), 2), (dict(rd=-16), 4), (dict(rd=40), 4), (dict(rd=144), 4),
    (dict(turns=0), 4), (dict(positions=0), 4), (dict(q=0), 4), (dict(k=0), 4), (dict(q_out=0), 4), (dict(k_out=AT + 4), 4), (dict(q_stride=1022), 4),
    (dict(k_stride=896), 4), (dict(qo_stride=1016), 4), (dict(ko_stride=-1024), 4), (dict(q_heads=-2), 4), (dict(k_heads=70000, k_stride=1 << 40), 4)])
def test_rotary_refusals(bad, rc):
    import pplb200
    assert _calls()[1](**bad) == rc and pplb200.last_error()


def test_read_refusals():
    import pplb200
    read = lambda slots=AT, tokens=4, k=AT, v=AT: pplb200.lib.pplb200_kv_cache_read_fp16(None, _cache(), slots, tokens, k, v)  # noqa: E731
    assert read(tokens=-1) == read(slots=0) == read(slots=AT + 4) == read(k=0) == read(v=0) == read(k=AT + 8) == read(v=AT + 2) == pplb200.RC_INVALID_VALUE
    assert read(tokens=1 << 40) == pplb200.RC_UNSUPPORTED


@pytest.mark.parametrize("bad,rc", [
    (dict(batch=-1), 4), (dict(batch=70000), 2), (dict(width=-1), 4), (dict(width=1 << 40, pages_stride=1 << 40), 2), (dict(q_heads=0), 4), (dict(q_heads=12), 4), (dict(q_heads=-8), 4), (dict(scale=float("nan")), 4),
    (dict(scale=float("inf")), 4), (dict(scale=1.2e15), 4), (dict(scale=-2.0 ** 51), 4), (dict(q=0), 4), (dict(out=0), 4), (dict(q=AT + 8), 4), (dict(out=AT + 2), 4), (dict(q_stride=1020), 4), (dict(q_stride=512), 4),
    (dict(out_stride=1016), 4), (dict(pages=0), 4), (dict(lengths=0), 4), (dict(pages=AT + 2), 4), (dict(lengths=AT + 1), 4), (dict(lse=AT + 2), 4), (dict(pages_stride=9), 4),
    (dict(ws=0), 4), (dict(ws=AT + 16), 4), (dict(ws_bytes=16), 4)])
def test_attention_refusals(bad, rc):
    import pplb200
    assert _calls()[2](_cache(), **bad) == rc and pplb200.last_error()


@pytest.mark.parametrize("cache,rc", [
    # scales of groups of 8 are read two at a time
    (dict(group=8, ks=AT + 2), 4), (dict(group=8, vs=AT + 2), 4), (dict(group=8, spage=8 * 256 + 1), 4), (dict(group=8, shead=255), 4), (dict(group=8, stoken=17), 4),
    # rows of a head 2^32 times their alignment apart, in keys and values, and in scales
    (dict(pages=(1 << 28) + 1, page_stride=(1 << 8) + 16, token_stride=0), 2), (dict(group=0, pages=(1 << 31) - 1, page_stride=24, token_stride=8), 2),
    (dict(pages=1 << 30, page_stride=0, token_stride=0, spage=9), 2), (dict(pages=1 << 30, page_stride=0, token_stride=0, group=8, spage=18, stoken=0), 2)])
def test_attention_refusals_of_caches(cache, rc):
    import pplb200
    assert _calls()[2](_cache(**cache)) == rc and pplb200.last_error()


@pytest.mark.parametrize("bad", [dict(page_stride=1 << 62), dict(pages=1 << 60, page_stride=16), dict(head_stride=1 << 60), dict(token_stride=(1 << 58)), dict(page=1 << 30, token_stride=1 << 40),
                                 dict(spage=1 << 62), dict(shead=1 << 60), dict(page=1 << 30, stoken=1 << 40), dict(group=0, ks=0, vs=0, page_stride=1 << 62)])
def test_caches_beyond_any_memory(bad):
    """Offsets whose products would not fit 64 bits."""
    import pplb200
    write, _, attend = _calls()
    c = _cache(**bad)
    assert write(c) == attend(c) == pplb200.lib.pplb200_kv_cache_read_fp16(None, c, AT, 4, AT, AT) == 4 and pplb200.last_error()
    assert pplb200.lib.pplb200_kv_cache_offset(c, 0, 0) == pplb200.lib.pplb200_paged_attention_offset(c, 0, 0) == -1


def test_attention_offsets_are_the_caches():
    """Attention's kernel computes them with 32-bit numbers of a unit of its own; up to the largest that it takes."""
    import pplb200
    lib = pplb200.lib
    edge = 1 << 32  # units
    for kw in (dict(), dict(group=0), dict(page=1), dict(page=7, head_stride=7 * 128, page_stride=7 * 1024), dict(head_stride=128, token_stride=1024), dict(pages=70000, page=64, page_stride=64 * 1024, head_stride=64 * 128),
               dict(group=0, pages=36000, page=64, page_stride=64 * 1024, head_stride=64 * 128), dict(pages=1, page_stride=16), dict(page=1, token_stride=0), dict(page_stride=0, head_stride=0, token_stride=0),
               # the last row is the last unit, of 16 bytes (int8: 16 elements, fp16: 8) and of more
               dict(pages=edge, page=1, page_stride=16), dict(pages=edge // 16, page_stride=256, token_stride=16), dict(group=0, pages=edge, page=1, page_stride=8),
               dict(pages=edge, page=1, page_stride=4096), dict(pages=edge // 2, page=2, page_stride=48, token_stride=16), dict(pages=1 << 22, page=64, page_stride=64 * 1024 * 16, head_stride=16, token_stride=1024 * 16)):
        c = _cache(**dict(dict(spage=0, shead=0, stoken=0), **kw))
        full = dict(CACHE, **kw)
        slots = full["pages"] * full["page"]
        for slot in (0, 1, full["page"] - 1, full["page"], slots // 2, slots // 3, slots - 1):
            for head in (0, 3, 7):
                want = lib.pplb200_kv_cache_offset(c, slot, head)
                if kw == dict(pages=edge // 2, page=2, page_stride=48, token_stride=16):  # 3 / 2 times as far as it takes
                    assert want >= 0 and lib.pplb200_paged_attention_offset(c, slot, head) == -1
                elif slot < slots:
                    assert want >= 0 and lib.pplb200_paged_attention_offset(c, slot, head) == want, (kw, slot, head)
        assert lib.pplb200_paged_attention_offset(c, slots, 0) == lib.pplb200_paged_attention_offset(c, -1, 0) == lib.pplb200_paged_attention_offset(c, 0, 8) == -1
    assert lib.pplb200_paged_attention_offset(_cache(pages=edge + 1, page=1, page_stride=16, spage=0, shead=0, stoken=0), 0, 0) == -1


def test_attention_head_dimensions():
    import pplb200
    attend = _calls()[2]
    for dim in (16, 80, 112, 160, 192):
        c = _cache(dim=dim, group=dim, token_stride=dim, head_stride=16 * dim, page_stride=128 * dim)
        assert attend(c, q_stride=8 * dim, out_stride=8 * dim) == pplb200.RC_UNSUPPORTED


def test_empty_calls_succeed():
    import pplb200
    write, rotary, attend = _calls()
    assert write(_cache(), tokens=0) == rotary(tokens=0) == attend(_cache(), batch=0) == 0
    assert pplb200.lib.pplb200_kv_cache_read_fp16(None, _cache(), None, 0, None, None) == 0


def test_null_blocks():
    import pplb200
    lib = pplb200.lib
    assert lib.pplb200_rotary_fp16(None, None) == lib.pplb200_kv_cache_write_fp16(None, _cache(), None) == 4
    assert lib.pplb200_kv_cache_write_fp16(None, None, None) == lib.pplb200_paged_decode_attention_fp16(None, _cache(), None) == 4
    assert lib.pplb200_kv_cache_read_fp16(None, None, AT, 1, AT, AT) == 4


def test_attention_workspace():
    import pplb200
    need = pplb200.lib.pplb200_paged_decode_attention_workspace_bytes
    assert need(-1, 16, 8, 8, 128) == need(1, -1, 8, 8, 128) == need(1, 16, 0, 8, 128) == need(1, 16, 9, 8, 128) == need(1, 16, 8, 0, 128) == -1
    sizes = [need(b, n, 64, 8, 128) for b, n in ((0, 0), (1, 16), (1, 131072), (16, 4096), (256, 8192), (65535, 1 << 20))]
    assert all(s > 0 and s % 256 == 0 for s in sizes) and sizes == sorted(sizes) and sizes[-1] <= 64 << 20


# ---- the binding: types, shapes and devices (the tensors are on the CPU, which is never the current device) ---------

@pytest.fixture
def here(monkeypatch):
    """The binding with CPU tensors taken for the current device's and the C calls recorded, their last argument block as bytes."""
    from pplb200 import attention
    calls, keep = [], []
    monkeypatch.setattr(attention, "_here", lambda: (-1, 0))
    vp, i64 = ctypes.c_void_p, ctypes.c_int64
    for n, types, size in (("_rotary", (vp, vp), 112), ("_write", (vp, vp, vp), 112), ("_read", (vp, vp, vp, i64, vp, vp), 0), ("_attend", (vp, vp, vp), 112)):
        f = ctypes.CFUNCTYPE(ctypes.c_int32, *types)(lambda *a, n=n, size=size: calls.append((n, a[:-1] + (ctypes.string_at(a[-1], size),) if size else a)) or 0)
        keep.append(f)
        monkeypatch.setattr(attention, n, ctypes.cast(f, vp).value)
    yield calls
    del keep


def test_binding_takes_strided_heads(here):
    import torch
    import pplb200
    rows = torch.zeros((5, 12, 64), dtype=torch.float16)
    table = pplb200.RotaryTable(32, device="cpu")
    q, k = pplb200.rotary_fp16(rows[:, :8], rows[:, 8:10], torch.zeros(5, dtype=torch.int64), table, q_out=rows[:, :8])
    assert q.data_ptr() == rows.data_ptr() and tuple(k.shape) == (5, 2, 64)
    block = struct.unpack("=6Q5q5if", here[0][1][1])
    assert block[0] == block[2] == rows.data_ptr() and block[1] == rows.data_ptr() + 8 * 64 * 2 and block[3] == k.data_ptr()
    assert block[6:11] == (5, 12 * 64, 12 * 64, 12 * 64, 128) and block[11:16] == (8, 2, 64, 32, 0)
    pplb200.rotary_fp16(None, rows[:, 8:], torch.zeros(5, dtype=torch.int64), table, interleaved=True)
    assert struct.unpack("=6Q5q5if", here[1][1][1])[11:16] == (0, 4, 64, 32, 1)


def test_binding_refuses_other_types_shapes_and_devices(here, monkeypatch):
    import torch
    import pplb200
    from pplb200 import attention
    f16, i64, i32 = torch.float16, torch.int64, torch.int32
    z = lambda *s, t=f16: torch.zeros(s, dtype=t)  # noqa: E731
    table, pos = pplb200.RotaryTable(64, device="cpu"), z(4, t=i64)
    cache = pplb200.PagedKVCache.allocate(10, 16, 2, 64, 8, device="cpu")
    att = pplb200.PagedDecodeAttention(cache, 8, max_batch=4, max_length=100)
    assert att.max_pages == 7
    good = dict(q=z(4, 8, 64), pages=z(4, 7, t=i32), lengths=z(4, t=i32))
    att(**good)
    kv = z(4, 2, 64)
    for call in (
            lambda: pplb200.rotary_fp16(z(4, 8, 64, t=torch.bfloat16), None, pos, table), lambda: pplb200.rotary_fp16(z(4, 8, 64), z(3, 8, 64), pos, table),
            lambda: pplb200.rotary_fp16(z(4, 8, 64), None, z(3, t=i64), table), lambda: pplb200.rotary_fp16(z(4, 8, 64), None, z(4, t=i32), table),
            lambda: pplb200.rotary_fp16(z(4, 8, 128)[..., ::2], None, pos, table), lambda: pplb200.rotary_fp16(z(4, 16, 64)[:, ::2], None, pos, table),
            lambda: pplb200.rotary_fp16(z(4, 8, 64), None, pos, table, q_out=z(4, 7, 64)), lambda: pplb200.rotary_fp16(z(4, 512), None, pos, table),
            lambda: pplb200.rotary_fp16(None, None, pos, table), lambda: pplb200.rotary_kv_cache_write(cache, z(4, 8, 64), kv, kv, pos, pos, None),
            lambda: pplb200.kv_cache_write(cache, z(4, 3, 64), kv, pos), lambda: pplb200.kv_cache_write(cache, kv, z(4, 2, 32), pos),
            lambda: pplb200.kv_cache_write(cache, kv, kv, z(8, t=i64)[::2]), lambda: pplb200.kv_cache_write(cache, kv, kv.float(), pos),
            lambda: pplb200.rotary_kv_cache_write(cache, z(4, 8, 64), kv, kv, pos, pos, table, q_out=z(4, 6, 64)),
            lambda: pplb200.kv_cache_read(cache, pos, k_out=z(4, 2, 32)), lambda: pplb200.kv_cache_read(cache, pos, v_out=z(4, 4, 64)[:, ::2]),
            lambda: pplb200.kv_cache_read(cache, z(4, t=i32)),
            lambda: att(**dict(good, q=z(4, 16, 64))), lambda: att(**dict(good, q=z(4, 8, 64).float())), lambda: att(**dict(good, pages=z(4, 7, t=i64))),
            lambda: att(**dict(good, pages=z(4, 8, t=i32))), lambda: att(**dict(good, pages=z(3, 7, t=i32))), lambda: att(**dict(good, lengths=z(5, t=i32))),
            lambda: att(**dict(good, lengths=z(8, t=i32)[::2])), lambda: att(**dict(good, pages=z(4, 14, t=i32)[:, ::2])), lambda: att(**good, lse=z(4, 8)),
            lambda: att(**good, out=z(4, 4, 64)), lambda: att(z(5, 8, 64), z(5, 7, t=i32), z(5, t=i32)),
            lambda: pplb200.PagedDecodeAttention(cache, 7, 1, 16), lambda: pplb200.PagedDecodeAttention(cache, 8, -1, 16)):
        before = len(here)
        with pytest.raises(ValueError):
            call()
        assert len(here) == before
    # a tensor, a cache or a table on another device than the current one
    monkeypatch.setattr(attention, "_here", lambda: (0, 0))
    for call in (lambda: pplb200.rotary_fp16(z(4, 8, 64), None, pos, table), lambda: pplb200.kv_cache_write(cache, kv, kv, pos),
                 lambda: pplb200.kv_cache_read(cache, pos), lambda: att(**good)):
        with pytest.raises(ValueError):
            call()


def test_binding_takes_tensors_and_truth_values(here):
    import torch
    import pplb200
    q, pos, table = torch.zeros((2, 1, 64), dtype=torch.float16), torch.zeros(2, dtype=torch.int64), pplb200.RotaryTable(64, device="cpu")
    cache = pplb200.PagedKVCache.allocate(10, 16, 1, 64, device="cpu")
    for call in (lambda: pplb200.rotary_fp16(q, None, [0, 1], table), lambda: pplb200.kv_cache_write(cache, q, q, None), lambda: pplb200.kv_cache_read(cache, pos, k_out=3)):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(ValueError):
        pplb200.rotary_fp16(q, None, pos, table, interleaved=np.zeros(2))
    assert not here
    for on, flag in ((True, 1), (1, 1), (np.bool_(False), 0), (0, 0)):
        pplb200.rotary_fp16(q, None, pos, table, interleaved=on)
        assert struct.unpack("=6Q5q5if", here[-1][1][1])[15] == flag


def test_objects_are_laid_out_once():
    import torch
    import pplb200
    table = pplb200.RotaryTable(64, device="cpu")
    cache = pplb200.PagedKVCache.allocate(10, 16, 1, 64, 8, device="cpu")
    att = pplb200.PagedDecodeAttention(cache, 4, 1, 160)
    for o, name, value in ((table, "turns", table.turns.clone()), (cache, "k", torch.zeros_like(cache.k)), (cache, "v_scale", None), (att, "ws", att.ws.clone()), (att, "scale", 1.0), (att, "window", 5), (att, "cache", cache)):
        with pytest.raises(AttributeError):
            setattr(o, name, value)


def test_binding_describes_the_cache():
    import torch
    import pplb200
    k, v = (torch.zeros((6, 24, 4, 96), dtype=torch.int8) for _ in range(2))
    ks, vs = (torch.zeros((6, 24, 4, 12), dtype=torch.float16) for _ in range(2))
    c = pplb200.PagedKVCache(*(t.transpose(1, 2) for t in (k, v, ks, vs)))  # stored token by token
    assert (c.num_pages, c.kv_heads, c.page_size, c.head_dim, c.quant_group) == (6, 4, 24, 96, 8)
    assert struct.unpack("=4Q7q4i", c._args[0]) == (k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), 6, 24 * 384, 96, 384, 24 * 48, 12, 48, 24, 4, 96, 8)
    h = torch.float16
    for bad in (lambda: pplb200.PagedKVCache(k, v), lambda: pplb200.PagedKVCache(k.to(h), v.to(h), ks, vs), lambda: pplb200.PagedKVCache(k, v, ks, None),
                lambda: pplb200.PagedKVCache(k, v[:5], ks, vs), lambda: pplb200.PagedKVCache(k, v, ks.float(), vs.float()), lambda: pplb200.PagedKVCache(k, v, ks[..., :5], vs[..., :5]),
                lambda: pplb200.PagedKVCache(k.float(), v.float()), lambda: pplb200.PagedKVCache(k, v.transpose(1, 2).contiguous().transpose(1, 2), ks, vs),
                lambda: pplb200.PagedKVCache(k[..., ::2], v[..., ::2], ks, vs), lambda: pplb200.PagedKVCache.allocate(1, 1, 1, 64, 16, device="cpu")):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("group", [0, 8, 64])
def test_an_allocated_cache_is_there_before_its_first_call(monkeypatch, group):
    import pplb200
    from pplb200 import attention
    settled = []
    monkeypatch.setattr(attention, "_settle", settled.append)
    cache = pplb200.PagedKVCache.allocate(10, 16, 1, 64, group, device="cpu")
    assert settled == [cache.k.device]
