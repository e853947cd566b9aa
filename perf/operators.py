"""What lies between a quantized layer's fused QKV projection and its output projection, as timed cases: rotary positions
on the query and key heads, the paged key-value cache written (fp16, or int8 with fp16 scales) and read back, and attention
of one new token a sequence over that cache.

`listed()` are fixed cases, `draw(rng)` gives more of the same ranges.  A case is run with `run(prepare(case, seed))`: in
plain tensor operations, or, where `own` is true, by the library's calls.  `exact` computes the same in 64 bits.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False


def _lib():
    at = os.path.join(os.getcwd(), "ppl.llm.kernel.cuda_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import pplb200
    return pplb200


# ---- cases -------------------------------------------------------------------------------------------------------
# t tokens, hq query and hk key-value heads of d dimensions; rd of them rotated; group: dimensions that share a scale of the
# int8 cache (0: the cache holds fp16); page: tokens a page; b sequences of up to `longest` tokens.

def listed():
    return [
        # sixteen conversations being decoded, 4096-wide layer
        dict(name="rotary t16", kind="rotary", t=16, hq=32, hk=32, d=128, rd=128, interleaved=False, scaling="none", far=4096, packed=False),
        # an odd prompt, neighbouring pairs, half of each head, q and k still inside the fused projection's rows
        dict(name="rotary t1999 partial", kind="rotary", t=1999, hq=32, hk=32, d=128, rd=64, interleaved=True, scaling="ntk", far=16384, packed=True),
        # the largest prefill of an 8192-wide layer, at positions far beyond the original context
        dict(name="rotary t8192 far", kind="rotary", t=8192, hq=64, hk=8, d=128, rd=128, interleaved=False, scaling="yarn", far=131072, packed=False),
        # batched decode: q and k rotated, k and v quantized into the cache in one call, what was stored read back
        dict(name="write t128 i8", kind="write", t=128, hq=32, hk=32, d=128, rd=128, interleaved=False, scaling="none", far=4096, group=8, page=16),
        # a prompt's keys and values (already rotated) quantized with one scale a head, what was stored read back
        dict(name="write t4096 i8", kind="write", t=4096, hq=0, hk=8, d=128, rd=0, interleaved=False, scaling="none", far=4096, group=128, page=64),
        # the largest prefill of an 8192-wide layer, rotated, stored as fp16
        dict(name="write t8192 fp16", kind="write", t=8192, hq=64, hk=8, d=128, rd=128, interleaved=False, scaling="linear", far=32768, group=0, page=64),
        # a long cached prefix, scattered over pages, read back for a prompt that continues it
        dict(name="read t32768 i8", kind="read", t=32768, hk=8, d=128, group=8, page=16),
        # one short conversation being decoded, every head its own keys
        dict(name="attend b1", kind="attend", b=1, longest=333, hq=32, hk=32, d=128, group=8, page=16, window=0),
        # sixteen conversations of all lengths, 4096-wide layer
        dict(name="attend b16", kind="attend", b=16, longest=4096, hq=32, hk=32, d=128, group=8, page=16, window=0),
        # one rank's eighth of an 8192-wide layer, 96 conversations, one shared key-value head
        dict(name="attend b96 shard", kind="attend", b=96, longest=2048, hq=8, hk=1, d=128, group=128, page=64, window=0),
        # many long conversations, grouped heads
        dict(name="attend b64 long", kind="attend", b=64, longest=8192, hq=64, hk=8, d=128, group=128, page=64, window=0),
        # one very long context, unquantized
        dict(name="attend b1 long", kind="attend", b=1, longest=131072, hq=64, hk=8, d=128, group=0, page=64, window=0),
    ]


def _log_int(rng, lo, hi):
    return int(min(hi, max(lo, round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["rotary", "write", "read", "attend", "attend", "attend"])
    d = rng.choice([64, 96, 128, 128, 256])
    hk = rng.choice([1, 2, 4, 8, 8, 32])
    hq = hk * (1 if hk == 32 else rng.choice([1, 2, 4, 5, 8, 8, 16]))
    page = rng.choice([1, 8, 16, 16, 24, 32, 64, 128])
    group = rng.choice([0, 8, 8, d, d])
    if kind == "attend":
        b = _log_int(rng, 1, 256)
        most = int(650e6 / (2 * b * hk * d * (1 + 2 / group if group else 2)))  # of bytes in the cache, if every length were the greatest
        return dict(kind=kind, b=b, longest=_log_int(rng, 16, max(16, min(131072, most))), hq=hq, hk=hk, d=d, group=group, page=page,
                    window=rng.choice([0, 0, 0, 100, 1024]))
    widest = (hq + 2 * hk) * d
    if kind == "read":
        return dict(kind=kind, t=_log_int(rng, 1, min(32768, 33_000_000 // (hk * d))), hk=hk, d=d, group=group, page=page)
    rd = rng.choice([d, d, d // 2])
    c = dict(kind=kind, t=_log_int(rng, 1, min(8192, 80_000_000 // widest)), hq=hq, hk=hk, d=d, rd=rd, interleaved=rng.random() < 0.4,
             scaling=rng.choice(["none", "linear", "ntk", "yarn", "wavelength"]), far=_log_int(rng, 1024, 1 << 20))
    if kind == "rotary":
        return dict(c, packed=rng.random() < 0.5)
    return dict(c, group=group, page=page)


#: base, and what the scaling takes: factor, original length, and how often a plane turns within that to be kept, or at most to be stretched
BASE, FACTOR, ORIGINAL = 10000.0, 8.0, 4096
LIMITS = {"yarn": (32.0, 1.0), "wavelength": (4.0, 1.0)}


def _lengths(case):
    """Tokens in the cache of each sequence, the new one among them: one whole length, the others spread below it, one empty."""
    rng = random.Random(case["b"] * 1000003 + case["longest"])
    n = [case["longest"]] + [rng.randint(max(1, case["longest"] // 8), case["longest"]) for _ in range(case["b"] - 1)]
    if case["b"] >= 8:
        n[rng.randrange(1, case["b"])] = 0
    return n


# ---- inputs ------------------------------------------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(0x0B200 + int(seed))
    return g


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda").to(torch.float16)


def _keys(g, *shape):
    """As keys come: some dimensions of every head are several times larger than the others."""
    x = torch.randn(shape, generator=g, device="cuda")
    x *= 1.0 + 5.0 * (torch.rand(shape[-1:], generator=g, device="cuda") < 0.05)
    return x.to(torch.float16)


def _frequencies(case):
    """Angle a position in each of the rd / 2 planes, and the factor on the rotated values, in plain operations."""
    rd, scaling = case["rd"], case["scaling"]
    i = torch.arange(rd // 2, dtype=torch.float64, device="cuda")
    base = BASE * FACTOR ** (rd / (rd - 2)) if scaling == "ntk" else BASE
    f = base ** (-2.0 * i / rd)
    if scaling == "linear":
        f = f / FACTOR
    elif scaling == "yarn":  # planes with many turns within the original length stay, those with few are interpolated
        lo, hi = (rd * math.log(ORIGINAL / (turns * 2 * math.pi)) / (2 * math.log(BASE)) for turns in LIMITS["yarn"])
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), rd - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        f = f * (1 - ramp) + f / FACTOR * ramp
    elif scaling == "wavelength":
        most, least = LIMITS["wavelength"]
        keep = ((ORIGINAL * f / (2 * math.pi) - least) / (most - least)).clamp(0, 1)
        f = f * keep + f / FACTOR * (1 - keep)
    return f, (0.1 * math.log(FACTOR) + 1.0 if scaling == "yarn" else 1.0)


def _rotary_table(lib, case):
    s = case["scaling"]
    keep, stretch = LIMITS.get(s, (0.0, 0.0))
    return lib.RotaryTable(case["rd"], base=BASE, scaling=s, factor=FACTOR, original_length=ORIGINAL, keep_turns=keep, stretch_turns=stretch)


def _empty_cache(pages, heads, page, d, group):
    """Keys, values and, for int8, their scales: [pages, heads, tokens of a page, ...]"""
    data = [torch.zeros((pages, heads, page, d), dtype=torch.int8 if group else torch.float16, device="cuda") for _ in range(2)]
    scales = [torch.zeros((pages, heads, page, d // group), dtype=torch.float16, device="cuda") for _ in range(2)] if group else [None, None]
    return data + scales


def _filled_cache(g, pages, heads, page, d, group):
    if not group:
        return [_keys(g, pages, heads, page, d), _normal(g, pages, heads, page, d), None, None]
    c = _empty_cache(pages, heads, page, d, group)
    for n, make in enumerate((_keys, _normal)):
        for at in range(0, pages, max(1, pages // 8)):  # by parts: several copies in 32 bits of a large cache need not fit
            part = slice(at, at + max(1, pages // 8))
            x = make(g, *c[n][part].shape)
            c[n][part], c[2 + n][part] = _quantize(x, group)
    return c


def _scattered(g, n, of):
    return torch.randperm(of, generator=g, device="cuda")[:n]


def prepare(case, seed):
    g = _generator(seed)
    s = dict(case)
    kind, d = case["kind"], case["d"]
    if kind in ("rotary", "write"):
        t, hq, hk = case["t"], case["hq"], case["hk"]
        if case.get("packed"):
            rows = _normal(g, t, hq + 2 * hk, d)
            s["q"], s["k"] = rows[:, :hq], rows[:, hq:hq + hk]
        else:
            s["q"], s["k"] = _normal(g, t, hq, d), _keys(g, t, hk, d)
        s["positions"] = torch.randint(0, case["far"], (t,), generator=g, device="cuda")
        if case["rd"]:
            s["f"], s["magnitude"] = _frequencies(case)
        s["q_out"] = torch.empty((t, hq, d), dtype=torch.float16, device="cuda")
        s["k_out"] = torch.empty((t, hk, d), dtype=torch.float16, device="cuda")
    if kind == "write":
        s["v"] = _normal(g, case["t"], case["hk"], d)
        pages = -(-2 * case["t"] // case["page"]) + 1  # as many tokens again are another request's
        s["cache"] = _empty_cache(pages, case["hk"], case["page"], d, case["group"])
        s["slots"] = _scattered(g, case["t"], 2 * case["t"])
        s["v_out"] = torch.empty_like(s["k_out"])
    elif kind == "read":
        pages = -(-case["t"] // case["page"])
        s["cache"] = _filled_cache(g, pages, case["hk"], case["page"], d, case["group"])
        at = torch.arange(case["t"], device="cuda")
        s["slots"] = _scattered(g, pages, pages)[at // case["page"]] * case["page"] + at % case["page"]
        s["k_out"], s["v_out"] = (torch.empty((case["t"], case["hk"], d), dtype=torch.float16, device="cuda") for _ in range(2))
    elif kind == "attend":
        b, page = case["b"], case["page"]
        lengths = _lengths(case)
        counts = [-(-n // page) for n in lengths]
        s["cache"] = _filled_cache(g, max(1, sum(counts)), case["hk"], page, d, case["group"])
        table = np.zeros((b, max(counts)), dtype=np.int32)
        table[np.arange(max(counts))[None] < np.array(counts)[:, None]] = _scattered(g, sum(counts), sum(counts)).cpu().numpy()
        s["pages"] = torch.from_numpy(table).cuda()
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        s["q"] = _normal(g, b, case["hq"], d) * 2
        s["out"] = torch.empty((b, case["hq"], d), dtype=torch.float16, device="cuda")
    if own:
        lib = _lib()
        if case.get("rd"):
            s["rotary"] = _rotary_table(lib, case)
        if "cache" in s:
            s["kv"] = lib.PagedKVCache(*s["cache"])
        if kind == "attend":
            s["attention"] = lib.PagedDecodeAttention(s["kv"], case["hq"], max_batch=case["b"], max_length=case["longest"], window=case["window"])
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------

def _quantize(x, group):
    """int8 values and fp16 scales: a group's largest magnitude is 127 steps, or barely less, since the scale is rounded up."""
    x = x.float().unflatten(-1, (-1, group))
    step = x.abs().amax(-1, keepdim=True) / 127
    scale = step.to(torch.float16)
    scale = (scale.view(torch.int16) + (scale.float() < step)).view(torch.float16).clamp_min(2.0 ** -24)
    q = torch.round(x / scale.float()).to(torch.int8)
    return q.flatten(-2), scale.squeeze(-1)


def _values(q, scale):
    """What a cache's elements stand for, in 32 bits."""
    if scale is None:
        return q.float()
    return (q.unflatten(-1, (scale.shape[-1], -1)).float() * scale.float().unsqueeze(-1)).flatten(-2)


def _rotate(x, s):
    rd, x = s["rd"], x.float()
    angle = s["positions"].double()[:, None, None] * s["f"]
    cos, sin = (angle.cos() * s["magnitude"]).float(), (angle.sin() * s["magnitude"]).float()
    if s["interleaved"]:
        a, b = x[..., 0:rd:2], x[..., 1:rd:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :rd // 2], x[..., rd // 2:rd]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., rd:]), -1).to(torch.float16)


def _store(s, k, v):
    page, at = s["slots"] // s["page"], s["slots"] % s["page"]
    for n, x in enumerate((k, v)):
        if s["group"]:
            s["cache"][n][page, :, at], s["cache"][2 + n][page, :, at] = _quantize(x, s["group"])
        else:
            s["cache"][n][page, :, at] = x


def _stored(s):
    page, at = s["slots"] // s["page"], s["slots"] % s["page"]
    rows = [None if c is None else c[page, :, at] for c in s["cache"]]
    return [_values(rows[n], rows[2 + n]).to(torch.float16) for n in (0, 1)]


def _attend(s):
    b, hk, d, page = s["b"], s["hk"], s["d"], s["page"]
    at = torch.arange(s["pages"].shape[1] * page, device="cuda")
    n = s["lengths"].long()[:, None]
    seen = at < n
    if s["window"]:
        seen = seen & (at >= n - s["window"])
    seen = seen[:, None, None]
    rows = [None if c is None else c[s["pages"].long()].transpose(1, 2).flatten(2, 3) for c in s["cache"]]  # [b, heads, tokens, ...]
    score = s["q"].float().view(b, hk, -1, d) @ _values(rows[0], rows[2]).transpose(-1, -2) / math.sqrt(d)
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True).clamp_min(-3e38)
    p = torch.exp(score - top)
    out = p @ _values(rows[1], rows[3])
    return (out / p.sum(-1, keepdim=True).clamp_min(1e-30)).view(b, -1, d).to(torch.float16)


def run(state):
    s, kind = state, state["kind"]
    if own:
        lib = _lib()
        if kind == "rotary":
            return lib.rotary_fp16(s["q"], s["k"], s["positions"], s["rotary"], interleaved=s["interleaved"], q_out=s["q_out"], k_out=s["k_out"])
        if kind == "attend":
            return s["attention"](s["q"], s["pages"], s["lengths"], out=s["out"])
        if kind == "read":
            return lib.kv_cache_read(s["kv"], s["slots"], k_out=s["k_out"], v_out=s["v_out"])
        outs = []
        if s["rd"]:
            outs.append(lib.rotary_kv_cache_write(s["kv"], s["q"], s["k"], s["v"], s["positions"], s["slots"], s["rotary"],
                                                  interleaved=s["interleaved"], q_out=s["q_out"]))
        else:
            lib.kv_cache_write(s["kv"], s["k"], s["v"], s["slots"])
        if not s["group"]:
            return outs + s["cache"][:2]
        return outs + list(lib.kv_cache_read(s["kv"], s["slots"], k_out=s["k_out"], v_out=s["v_out"]))
    if kind == "rotary":
        return _rotate(s["q"], s), _rotate(s["k"], s)
    if kind == "attend":
        return _attend(s)
    if kind == "read":
        return _stored(s)
    outs = [_rotate(s["q"], s)] if s["rd"] else []
    _store(s, _rotate(s["k"], s) if s["rd"] else s["k"], s["v"])
    return outs + (_stored(s) if s["group"] else s["cache"][:2])


# ---- the same from the definitions, in 64 bits -------------------------------------------------------------------

def _exact_rotary(case, x, positions):
    """Complex multiplication by magnitude * e^(i angle), plane by plane; the angle in whole turns and a fraction."""
    rd, s = case["rd"], case["scaling"]
    planes = []
    for i in range(rd // 2):
        f = (BASE * FACTOR ** (rd / (rd - 2)) if s == "ntk" else BASE) ** (-2 * i / rd)
        if s == "linear":
            f /= FACTOR
        elif s == "yarn":
            first = max(math.floor(rd / 2 * math.log(ORIGINAL / (2 * math.pi * LIMITS[s][0]), BASE)), 0)
            last = min(math.ceil(rd / 2 * math.log(ORIGINAL / (2 * math.pi * LIMITS[s][1]), BASE)), rd - 1)
            part = min(1.0, max(0.0, (i - first) / max(last - first, 0.001)))
            f = f + part * (f / FACTOR - f)
        elif s == "wavelength":
            turns = ORIGINAL * f / (2 * math.pi)
            most, least = LIMITS[s]
            part = 0.0 if turns <= least else 1.0 if turns >= most else (turns - least) / (most - least)
            f = f / FACTOR + part * (f - f / FACTOR)
        planes.append(f)
    angle = positions.double().unsqueeze(1) * torch.tensor(planes, dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.full_like(angle, 1 + math.log(FACTOR) / 10 if s == "yarn" else 1.0), angle).unsqueeze(1)
    out = x.double()
    first, second = (slice(0, rd, 2), slice(1, rd, 2)) if case["interleaved"] else (slice(0, rd // 2), slice(rd // 2, rd))
    z = torch.complex(out[..., first], out[..., second]) * turn
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _exact_stored(x, group):
    """What is read back for x (fp16): whole multiples of a group's scale, the smallest fp16 that puts the group within 127 of them."""
    y = x.double().reshape(*x.shape[:-1], -1, group)
    least = y.abs().amax(-1, keepdim=True).cpu().numpy() / 127
    scale = least.astype(np.float16)
    scale = np.where(scale < least, np.nextafter(scale, np.float16(np.inf)), scale).astype(np.float64)
    scale = torch.from_numpy(np.maximum(scale, 2.0 ** -24)).cuda()
    return (torch.round(y / scale) * scale).reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    kind, d, page = case["kind"], case["d"], case["page"] if "page" in case else 0
    if kind == "rotary":
        return tuple(_exact_rotary(case, s[n], s["positions"]) for n in ("q", "k"))
    if kind == "read":
        outs = []
        for n in (0, 1):
            x = s["cache"][n].double()
            if case["group"]:
                x = x * s["cache"][2 + n].double().repeat_interleave(case["group"], -1)
            outs.append(x.transpose(1, 2).reshape(-1, case["hk"], d)[s["slots"]])
        return outs
    if kind == "write":
        outs, k = [], s["k"]
        if case["rd"]:
            outs.append(_exact_rotary(case, s["q"], s["positions"]))
            k = _exact_rotary(case, k, s["positions"])
        if case["group"]:
            return outs + [_exact_stored(x.half(), case["group"]) for x in (k, s["v"])]
        for x in (k, s["v"]):
            rows = torch.zeros((s["cache"][0].shape[0] * page, case["hk"], d), dtype=torch.float64, device="cuda")
            rows[s["slots"]] = x.double()
            outs.append(rows.view(-1, page, case["hk"], d).transpose(1, 2))
        return outs
    out = torch.zeros((case["b"], case["hq"], d), dtype=torch.float64, device="cuda")
    shared = case["hq"] // case["hk"]
    for i, n in enumerate(_lengths(case)):
        first = max(0, n - case["window"]) if case["window"] else 0
        if n == 0:
            continue
        at = torch.arange(first, n, device="cuda")
        at = s["pages"][i].long()[at // page], at % page
        for h in range(case["hk"]):
            k, v = (s["cache"][m][at[0], h, at[1]].double() for m in (0, 1))
            if case["group"]:
                k, v = (x * s["cache"][2 + m][at[0], h, at[1]].double().repeat_interleave(case["group"], -1) for m, x in ((0, k), (1, v)))
            heads = slice(h * shared, (h + 1) * shared)
            weight = torch.softmax(s["q"][i, heads].double() @ k.T * d ** -0.5, -1)
            out[i, heads] = weight @ v
    return out


# ---- what a pass cannot do without -------------------------------------------------------------------------------

def work(case):
    """Inputs read once, results written once.  Rotation: six operations a pair; quantizing: two an element; attention: two
    multiply-adds for every query head and dimension of a token that is seen."""
    d = case["d"]
    element = 2 if not case.get("group") else 1 + 2 / case["group"]  # bytes in the cache, scales included
    if case["kind"] == "attend":
        seen = sum(min(n, case["window"] or n) for n in _lengths(case))
        table = 4 * sum(-(-n // case["page"]) for n in _lengths(case)) + 4 * case["b"]
        return {"bytes": int(2 * seen * case["hk"] * d * element) + 4 * case["b"] * case["hq"] * d + table, "flops": 4 * seen * case["hq"] * d}
    t, hk = case["t"], case["hk"]
    if case["kind"] == "read":
        return {"bytes": int(2 * t * hk * d * (element + 2)) + 8 * t, "flops": 2 * t * hk * d if case["group"] else 0}
    hq, rd = case["hq"], case["rd"]
    turned = t * (hq + hk) * rd * 3
    if case["kind"] == "rotary":
        return {"bytes": 4 * t * (hq + hk) * d + 8 * t, "flops": turned}
    # into the cache, and for int8 the values read back
    moved = 2 * t * hk * d * (2 + element + (2 if case["group"] else 0)) + 8 * t
    if rd:
        moved += 4 * t * hq * d + 8 * t
    return {"bytes": int(moved), "flops": turned + (4 * t * hk * d if case["group"] else 0)}
