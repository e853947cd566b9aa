"""Decoding over long and shared contexts, as timed cases: rotary positions of several axes (time, height, width), attention of a
batch over a prefix that its sequences share, and attention over the blocks of a cache that a cheap score selects, with the bounds
of the blocks' keys that the score is made of.

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
# hq query and hk key-value heads of d dimensions; group: dimensions that share a scale of the int8 cache (0: the cache holds fp16);
# page: tokens a page.
# axes: t tokens, rd dimensions rotated, p0 + p1 + p2 planes of the axes; alternating: planes dealt out to the axes in turn; restart: each axis
#       has frequencies of its own; store: into the cache too.
# bounds: of the blocks of `block` tokens that t new tokens complete; whole: the tokens of prompts, else one token each of t sequences.
# prefix: b sequences share `prefix` tokens and have up to `longest` of their own.
# sparse: b sequences of up to `longest` tokens, of whose blocks the first, the last and the best of the others are attended.

def listed():
    return [
        # a decode step of a model that sees images: 24 conversations, time, height and width dealt out in turn
        dict(name="axes t24", kind="axes", t=24, hq=32, hk=8, d=128, rd=128, p0=24, p1=20, p2=20, alternating=True, restart=False, interleaved=False, scaling="none", store=False, group=0, page=16),
        # an odd number of image patches: half of each head for height, half for width, neighbouring pairs, inside the projection's rows
        dict(name="axes t1999 patches", kind="axes", t=1999, hq=16, hk=16, d=64, rd=64, p0=16, p1=16, p2=0, alternating=False, restart=True, interleaved=True, scaling="none", store=False, group=0, page=16),
        # a video's prefill in an 8192-wide layer, quantized into the cache, what was stored read back
        dict(name="axes t8192 store", kind="axes", t=8192, hq=64, hk=8, d=128, rd=128, p0=16, p1=24, p2=24, alternating=False, restart=False, interleaved=False, scaling="yarn", store=True, group=128, page=64),
        # 96 conversations being decoded, six of whose new tokens complete a block
        dict(name="bounds t96", kind="bounds", t=96, whole=False, hk=8, d=128, group=8, page=64, block=16),
        # the largest prefill: every block of it
        dict(name="bounds t16384", kind="bounds", t=16384, whole=True, hk=8, d=128, group=0, page=64, block=64),
        # four answers to one odd prompt, every head its own keys
        dict(name="prefix b4", kind="prefix", b=4, prefix=999, longest=77, hq=32, hk=32, d=128, group=8, page=16),
        # 48 conversations behind one system prompt, grouped heads
        dict(name="prefix b48 i8", kind="prefix", b=48, prefix=4000, longest=1024, hq=64, hk=8, d=128, group=128, page=64),
        # one rank's eighth of an 8192-wide layer, 256 samples of one long question
        dict(name="prefix b256 shard", kind="prefix", b=256, prefix=12345, longest=300, hq=8, hk=1, d=128, group=0, page=64),
        # 64 questions about one long document, unquantized
        dict(name="prefix b64 long", kind="prefix", b=64, prefix=32768, longest=256, hq=64, hk=8, d=128, group=0, page=64),
        # one conversation being decoded, every head its own keys
        dict(name="sparse b1", kind="sparse", b=1, longest=4099, hq=32, hk=32, d=128, group=8, page=16, block=16, first=1, last=4, top=27),
        # sixteen long conversations, grouped heads
        dict(name="sparse b16", kind="sparse", b=16, longest=16384, hq=64, hk=8, d=128, group=128, page=64, block=32, first=1, last=2, top=61),
        # one very long context, unquantized
        dict(name="sparse b1 long", kind="sparse", b=1, longest=131072, hq=64, hk=8, d=128, group=0, page=64, block=64, first=1, last=2, top=125),
    ]


def _log_int(rng, lo, hi):
    return int(min(hi, max(lo, round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["axes", "bounds", "prefix", "prefix", "sparse", "sparse"])
    d = rng.choice([64, 96, 128, 128, 256])
    hk = rng.choice([1, 2, 4, 8, 8, 32])
    hq = hk * (1 if hk == 32 else rng.choice([1, 2, 4, 5, 8, 8, 16]))
    group = rng.choice([0, 8, d, d])
    page = rng.choice([16, 16, 32, 64, 64, 128])
    block = rng.choice([n for n in (16, 32, 64, 128) if page % n == 0])
    element = 1 + 2 / group if group else 2
    c = dict(kind=kind, hq=hq, hk=hk, d=d, group=group, page=page)
    if kind == "axes":
        rd = rng.choice([d, d, d // 2])
        p0, p1 = rng.randint(1, rd // 2 - 2), 0
        p1 = rng.randint(1, rd // 2 - p0)
        restart = rng.random() < 0.3
        return dict(c, t=_log_int(rng, 1, min(8192, 80_000_000 // ((hq + 2 * hk) * d))), rd=rd, p0=p0, p1=p1, p2=rd // 2 - p0 - p1,
                    alternating=rng.random() < 0.5, restart=restart, interleaved=rng.random() < 0.4,
                    scaling=rng.choice(["none", "linear"] if restart else ["none", "linear", "ntk", "yarn", "wavelength"]), store=rng.random() < 0.5)
    if kind == "bounds":
        return dict(kind=kind, hk=hk, d=d, group=group, page=page, block=block, whole=rng.random() < 0.6, t=_log_int(rng, max(16, block), min(16384, 30_000_000 // (hk * d))))
    if kind == "prefix":
        b = _log_int(rng, 1, 256)
        most = min(64 * 64 * 32768 * 128 // (b * hq * d), int(400e6 / (2 * hk * d * element)))
        prefix = _log_int(rng, 16, max(16, min(32768, most)))
        own_most = min(2048, int(200e6 / (2 * b * hk * d * element)), max(1, most // 4))
        return dict(c, page=rng.choice([1, 8, page, page, page]), b=b, prefix=prefix, longest=_log_int(rng, 1, max(1, own_most)))
    b = _log_int(rng, 1, 128)
    most = int(600e6 / (2 * b * hk * d * element))
    longest = _log_int(rng, 16, max(16, min(131072, most)))
    return dict(c, block=block, b=b, longest=longest, first=rng.choice([0, 1, 2]), last=rng.choice([1, 2, 4, 8]), top=_log_int(rng, 1, max(1, 4096 // block)))


#: base, and what the scaling takes: factor, original length, and how often a plane turns within that to be kept, or at most to be stretched
BASE, FACTOR, ORIGINAL = 10000.0, 8.0, 4096
LIMITS = {"yarn": (32.0, 1.0), "wavelength": (4.0, 1.0)}


def _sections(case):
    return [n for n in (case["p0"], case["p1"], case["p2"]) if n]


def _axis_of_plane(case):
    """The axis whose position turns each plane: one axis behind the other, or in turn as long as an axis has planes left."""
    left = _sections(case)
    if not case["alternating"]:
        return [axis for axis, n in enumerate(left) for _ in range(n)]
    out = []
    while any(left):
        for axis, n in enumerate(left):
            if n:
                out.append(axis)
                left[axis] -= 1
    return out


def _spread(n, longest, b, least):
    """One whole length, the others spread below it."""
    rng = random.Random(n * 1000003 + longest)
    return [longest] + [rng.randint(max(least, longest // 8), longest) for _ in range(b - 1)]


def _lengths(case):
    """Tokens of each sequence, the new one among them; prefix: behind the prefix, one sequence that has nothing but the prefix, one row of
    padding; sparse: one empty sequence."""
    b, kind = case["b"], case["kind"]
    n = _spread(b, case["longest"], b, 1)
    if b >= 8:
        n[b // 2] = 0
        if kind == "prefix":
            n[b - 1] = -1
    return n


# ---- inputs ------------------------------------------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(0xB200 + 7919 * int(seed))
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
    scaling = case["scaling"]
    if case["restart"]:
        f = torch.empty(case["rd"] // 2, dtype=torch.float64, device="cuda")
        of = torch.tensor(_axis_of_plane(case), device="cuda")
        for axis, n in enumerate(_sections(case)):
            f[of == axis] = BASE ** (-torch.arange(n, dtype=torch.float64, device="cuda") / n)
        return (f / FACTOR if scaling == "linear" else f), 1.0
    rd = case["rd"]
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
    return lib.RotaryTable(case["rd"], base=BASE, scaling=s, factor=FACTOR, original_length=ORIGINAL, keep_turns=keep, stretch_turns=stretch,
                           axes=_sections(case), alternating=case["alternating"], restart=case["restart"])


def _empty_cache(pages, heads, page, d, group):
    """Keys, values and, for int8, their scales: [pages, heads, tokens of a page, ...]"""
    data = [torch.zeros((pages, heads, page, d), dtype=torch.int8 if group else torch.float16, device="cuda") for _ in range(2)]
    scales = [torch.zeros((pages, heads, page, d // group), dtype=torch.float16, device="cuda") for _ in range(2)] if group else [None, None]
    return data + scales


def _filled_cache(g, pages, heads, page, d, group, drift=0):
    """drift: keys of neighbouring pages resemble each other, as those of neighbouring tokens of a text do."""
    c = _empty_cache(pages, heads, page, d, group)
    step = max(1, pages // 8)
    for n, make in enumerate((_keys, _normal)):
        for at in range(0, pages, step):  # by parts: several copies in 32 bits of a large cache need not fit
            part = slice(at, at + step)
            x = make(g, *c[n][part].shape)
            if drift and n == 0:
                x += (torch.randn((x.shape[0], heads, 1, d), generator=g, device="cuda") * drift).to(torch.float16)
            if group:
                c[n][part], c[2 + n][part] = _quantize(x, group)
            else:
                c[n][part] = x
    return c


def _scattered(g, n, of):
    return torch.randperm(of, generator=g, device="cuda")[:n]


def _tables(g, lengths, page, ahead):
    """Page table of the sequences over scattered pages, behind `ahead` pages that are another's; pages in all, and that other's pages."""
    counts = [-(-max(0, n) // page) for n in lengths]
    at = _scattered(g, ahead + sum(counts), ahead + sum(counts))
    table = np.zeros((len(lengths), max(1, max(counts))), dtype=np.int32)
    table[np.arange(table.shape[1])[None] < np.array(counts)[:, None]] = at[ahead:].cpu().numpy()
    return torch.from_numpy(table).cuda(), max(1, ahead + sum(counts)), at[:ahead].to(torch.int32)


def prepare(case, seed):
    g = _generator(seed)
    s = dict(case)
    kind, d, hk, page, group = case["kind"], case["d"], case["hk"], case["page"], case["group"]
    if kind == "axes":
        t, hq = case["t"], case["hq"]
        rows = _normal(g, t, hq + 2 * hk, d)  # of the fused projection
        s["q"], s["k"], s["v"] = rows[:, :hq], rows[:, hq:hq + hk], rows[:, hq + hk:]
        s["positions"] = torch.stack([torch.randint(0, far, (t,), generator=g, device="cuda") for far in (65536, 128, 128)[-len(_sections(case)):]])
        s["axis"] = torch.tensor(_axis_of_plane(case), device="cuda")
        s["f"], s["magnitude"] = _frequencies(case)
        s["q_out"] = torch.empty((t, hq, d), dtype=torch.float16, device="cuda")
        s["k_out"], s["v_out"] = (torch.empty((t, hk, d), dtype=torch.float16, device="cuda") for _ in range(2))
        if case["store"]:
            s["cache"] = _empty_cache(-(-t // page), hk, page, d, group)
            s["slots"] = _scattered(g, t, -(-t // page) * page)
    elif kind == "bounds":
        t, block = case["t"], case["block"]
        if case["whole"]:  # consecutive tokens, whose blocks lie scattered
            blocks = -(-t // block)
            at = torch.arange(t, device="cuda")
            s["slots"] = _scattered(g, blocks, -(-blocks * block // page) * (page // block))[at // block] * block + at % block
            s["done"] = s["slots"][block - 1::block] // block
            pages = -(-blocks * block // page)
        else:  # one token each of t sequences, every sixteenth of which completes its block
            pages = -(-t * block // page)
            at = _scattered(g, t, pages * (page // block))
            s["slots"] = at * block + torch.where(torch.arange(t, device="cuda") % 16 == 15, block - 1, torch.arange(t, device="cuda") % (block - 1))
            s["done"] = at[15::16].contiguous()
        s["cache"] = _filled_cache(g, pages, hk, page, d, group)
        s["bounds"], s["bound_scales"] = _no_bounds(case, pages)
        s["lo"], s["hi"] = (torch.empty((s["done"].shape[0], hk, d), device="cuda") for _ in range(2))
    else:
        b = case["b"]
        lengths = _lengths(case)
        ahead = -(-case["prefix"] // page) if kind == "prefix" else 0
        s["pages"], pages, s["prefix_pages"] = _tables(g, lengths, page, ahead)
        s["cache"] = _filled_cache(g, pages, hk, page, d, group, drift=0.5 if kind == "sparse" else 0)
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        s["q"] = _normal(g, b, case["hq"], d) * 2
        s["out"] = torch.empty((b, case["hq"], d), dtype=torch.float16, device="cuda")
        if kind == "prefix":
            s["prefix_length"] = torch.tensor([case["prefix"]], dtype=torch.int32, device="cuda")
        else:
            s["bounds"], s["bound_scales"] = _no_bounds(case, pages)
            step = max(1, pages // 8)
            for at in range(0, pages, step):
                part = slice(at, at + step)
                k = _values(s["cache"][0][part], None if s["cache"][2] is None else s["cache"][2][part])
                s["bounds"][part], s["bound_scales"][part] = _bounds(k.unflatten(2, (-1, case["block"])))
    if own:
        lib = _lib()
        if kind == "axes":
            s["rotary"] = _rotary_table(lib, case)
        if "cache" in s:
            s["kv"] = lib.PagedKVCache(*s["cache"])
        if "bounds" in s:
            s["key_bounds"] = lib.KeyBlockBounds(s["kv"], case["block"], s["bounds"], s["bound_scales"])
        if kind == "prefix":
            s["attention"] = lib.SharedPrefixDecodeAttention(s["kv"], case["hq"], max_batch=case["b"], max_length=case["longest"], max_prefix=case["prefix"])
        if kind == "sparse":
            s["attention"] = lib.BlockSparseDecodeAttention(s["key_bounds"], case["hq"], max_batch=case["b"], max_length=case["longest"],
                                                            first=case["first"], last=case["last"], top=case["top"])
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------

def _scale(amax):
    """The smallest fp16 that puts amax within 127 of it."""
    step = amax / 127
    scale = step.to(torch.float16)
    return (scale.view(torch.int16) + (scale.float() < step)).view(torch.float16).clamp_min(2.0 ** -24)


def _quantize(x, group):
    """int8 values and fp16 scales: a group's largest magnitude is 127 steps, or barely less, since the scale is rounded up."""
    x = x.float().unflatten(-1, (-1, group))
    scale = _scale(x.abs().amax(-1, keepdim=True))
    q = torch.round(x / scale.float()).to(torch.int8)
    return q.flatten(-2), scale.squeeze(-1)


def _values(q, scale):
    """What a cache's elements stand for, in 32 bits."""
    if scale is None:
        return q.float()
    return (q.unflatten(-1, (scale.shape[-1], -1)).float() * scale.float().unsqueeze(-1)).flatten(-2)


def _rotate(x, s):
    rd, x = s["rd"], x.float()
    angle = (s["positions"][s["axis"]].T.double() * s["f"])[:, None]
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


def _no_bounds(case, pages):
    """int8 [pages, heads, blocks of a page, least and greatest, dimensions] and a scale a block and head, of blocks that nothing is known of."""
    blocks = case["page"] // case["block"]
    return (torch.zeros((pages, case["hk"], blocks, 2, case["d"]), dtype=torch.int8, device="cuda"),
            torch.zeros((pages, case["hk"], blocks), dtype=torch.float16, device="cuda"))


def _bounds(k):
    """[..., tokens of a block, dimensions] -> the least and the greatest as whole steps outwards, and the step."""
    lo, hi = k.amin(-2), k.amax(-2)
    scale = _scale(torch.maximum(lo.abs(), hi.abs()).amax(-1))
    step = scale.float().unsqueeze(-1)
    return torch.stack((torch.floor(lo / step), torch.ceil(hi / step)), -2).to(torch.int8), scale


def _complete(s):
    """Bounds of the blocks whose last token is among the slots."""
    block, page, hk = s["block"], s["page"], s["hk"]
    done = s["slots"][s["slots"] % block == block - 1] // block
    at = (done // (page // block), done % (page // block))
    tokens = torch.arange(block, device="cuda") + at[1][:, None] * block
    rows = [None if c is None else c[at[0][:, None], :, tokens] for c in (s["cache"][0], s["cache"][2])]  # [blocks, tokens, heads, ...]
    s["bounds"][at[0], :, at[1]], s["bound_scales"][at[0], :, at[1]] = _bounds(_values(*rows).transpose(1, 2))


def _bound_values(s):
    at = (s["done"] // (s["page"] // s["block"]), s["done"] % (s["page"] // s["block"]))
    both = s["bounds"][at[0], :, at[1]].float() * s["bound_scales"][at[0], :, at[1]].float()[..., None, None]
    return both[:, :, 0], both[:, :, 1]


def _softmax(parts):
    """sum w v / sum w over several (scores, values) with one reference exponent; scores of -inf have no weight."""
    top = torch.cat([score.amax(-1, keepdim=True) for score, _ in parts], -1).amax(-1, keepdim=True).clamp_min(-3e38)
    out = norm = 0
    for score, v in parts:
        p = torch.exp(score - top)
        out, norm = out + p @ v, norm + p.sum(-1, keepdim=True)
    return out / norm.clamp_min(1e-30)


def _gathered(s, pages):
    """Values of keys and values of whole pages [n, ...] in order: [heads, tokens, dimensions] with n's leading extents ahead."""
    out = []
    for n in (0, 1):
        rows = [None if c is None else c[pages.long()].transpose(-4, -3).flatten(-3, -2) for c in (s["cache"][n], s["cache"][2 + n])]
        out.append(_values(*rows))
    return out


def _attend_prefix(s):
    b, hk, d = s["b"], s["hk"], s["d"]
    q = s["q"].float().view(b, hk, -1, d) / math.sqrt(d)
    k, v = _gathered(s, s["prefix_pages"])
    k, v = k[:, :s["prefix"]], v[:, :s["prefix"]]
    rows = q.transpose(0, 1).flatten(1, 2)  # [heads, sequences x query heads, dimensions]
    ahead = (rows @ k.transpose(-1, -2)).view(hk, b, -1, s["prefix"])
    own_k, own_v = _gathered(s, s["pages"])
    seen = torch.arange(own_k.shape[2], device="cuda") < s["lengths"][:, None]
    behind = (q @ own_k.transpose(-1, -2)).masked_fill(~seen[:, None, None], -math.inf).transpose(0, 1)
    top = torch.maximum(ahead.amax(-1, keepdim=True), behind.amax(-1, keepdim=True))
    ahead, behind = torch.exp(ahead - top), torch.exp(behind - top)
    out = (ahead.flatten(1, 2) @ v).view(hk, b, -1, d) + (behind.transpose(0, 1) @ own_v).transpose(0, 1)
    out = out / (ahead.sum(-1, keepdim=True) + behind.sum(-1, keepdim=True))
    return torch.where(s["lengths"][:, None, None, None] < 0, 0.0, out.transpose(0, 1)).reshape(b, -1, d).to(torch.float16)


def _attend_sparse(s):
    b, hk, d, block, per_page = s["b"], s["hk"], s["d"], s["block"], s["page"] // s["block"]
    n = s["lengths"].long()
    blocks = (n + block - 1) // block
    q8, q_scale = _quantize(s["q"].view(b, hk, -1, d), d)
    q = q8.float()
    at = s["pages"].long()
    both = s["bounds"][at].transpose(1, 2).flatten(2, 3).float()  # [b, heads, blocks, 2, dimensions]
    scale = s["bound_scales"][at].transpose(1, 2).flatten(2, 3).float()
    dot = q.clamp_max(0) @ both[:, :, :, 0].transpose(-1, -2) + q.clamp_min(0) @ both[:, :, :, 1].transpose(-1, -2)  # whole numbers below 2^24
    score = (dot * (q_scale.float() * scale[:, :, None])).amax(2)  # [b, heads, blocks]
    number = torch.arange(score.shape[-1], device="cuda")
    total = s["first"] + s["last"] + s["top"]
    kept = (number < s["first"]) | (number >= (blocks - s["last"])[:, None])
    there = number < blocks[:, None]
    score = torch.where(kept[:, None], math.inf, score).masked_fill(~there[:, None], -math.inf)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :total]
    chosen = torch.sort(torch.where(there[:, None].expand_as(score).gather(-1, order), order, 1 << 30), dim=-1).values
    token = (chosen[..., None] * block + torch.arange(block, device="cuda")).flatten(-2)
    seen = token < n[:, None, None]
    token = torch.where(seen, token, 0)
    slot = at[:, None].expand(-1, hk, -1).gather(-1, token // s["page"]), token % s["page"]
    head = torch.arange(hk, device="cuda")[None, :, None]
    rows = [None if c is None else c[slot[0], head, slot[1]] for c in s["cache"]]
    score = s["q"].float().view(b, hk, -1, d) @ _values(rows[0], rows[2]).transpose(-1, -2) / math.sqrt(d)
    return _softmax([(score.masked_fill(~seen[:, :, None], -math.inf), _values(rows[1], rows[3]))]).view(b, -1, d).to(torch.float16)


def run(state):
    s, kind = state, state["kind"]
    if own:
        lib = _lib()
        if kind == "prefix":
            return s["attention"](s["q"], s["prefix_pages"], s["prefix_length"], s["pages"], s["lengths"], out=s["out"])
        if kind == "sparse":
            return s["attention"](s["q"], s["pages"], s["lengths"], out=s["out"])
        if kind == "bounds":
            lib.key_bounds_update(s["key_bounds"], s["slots"])
            return lib.key_bounds_read(s["key_bounds"], s["done"], lo_out=s["lo"], hi_out=s["hi"])
        if not s["store"]:
            return lib.rotary_fp16(s["q"], s["k"], s["positions"], s["rotary"], interleaved=s["interleaved"], q_out=s["q_out"], k_out=s["k_out"])
        q = lib.rotary_kv_cache_write(s["kv"], s["q"], s["k"], s["v"], s["positions"], s["slots"], s["rotary"], interleaved=s["interleaved"], q_out=s["q_out"])
        return [q] + (list(lib.kv_cache_read(s["kv"], s["slots"], k_out=s["k_out"], v_out=s["v_out"])) if s["group"] else s["cache"][:2])
    if kind == "prefix":
        return _attend_prefix(s)
    if kind == "sparse":
        return _attend_sparse(s)
    if kind == "bounds":
        _complete(s)
        return _bound_values(s)
    if not s["store"]:
        return _rotate(s["q"], s), _rotate(s["k"], s)
    _store(s, _rotate(s["k"], s), s["v"])
    return [_rotate(s["q"], s)] + (_stored(s) if s["group"] else s["cache"][:2])


# ---- the same from the definitions, in 64 bits -------------------------------------------------------------------

def _exact_planes(case):
    """(axis, angle a position) of every plane."""
    rd, s, out = case["rd"], case["scaling"], []
    taken = [0, 0, 0]
    sections = _sections(case)
    for i in range(rd // 2):
        if case["alternating"]:  # the axis that has had the fewest, as long as it has planes left
            axis = min((a for a in range(len(sections)) if taken[a] < sections[a]), key=lambda a: (taken[a], a))
        else:
            axis = next(a for a in range(len(sections)) if i < sum(sections[:a + 1]))
        part = taken[axis] / sections[axis] if case["restart"] else 2 * i / rd
        taken[axis] += 1
        f = (BASE * FACTOR ** (rd / (rd - 2)) if s == "ntk" else BASE) ** -part
        if s == "linear":
            f /= FACTOR
        elif s == "yarn":
            begin = max(math.floor(rd / 2 * math.log(ORIGINAL / (2 * math.pi * LIMITS[s][0]), BASE)), 0)
            end = min(math.ceil(rd / 2 * math.log(ORIGINAL / (2 * math.pi * LIMITS[s][1]), BASE)), rd - 1)
            mix = min(1.0, max(0.0, (i - begin) / max(end - begin, 0.001)))
            f = f + mix * (f / FACTOR - f)
        elif s == "wavelength":
            turns = ORIGINAL * f / (2 * math.pi)
            most, least = LIMITS[s]
            mix = 0.0 if turns <= least else 1.0 if turns >= most else (turns - least) / (most - least)
            f = f / FACTOR + mix * (f - f / FACTOR)
        out.append((axis, f))
    return out


def _exact_rotary(case, x, positions):
    """Complex multiplication by magnitude * e^(i angle), plane by plane."""
    rd = case["rd"]
    planes = _exact_planes(case)
    angle = torch.stack([positions[axis].double() * f for axis, f in planes], -1)
    turn = torch.polar(torch.full_like(angle, 1 + math.log(FACTOR) / 10 if case["scaling"] == "yarn" else 1.0), angle).unsqueeze(1)
    out = x.double().clone()
    one, two = (slice(0, rd, 2), slice(1, rd, 2)) if case["interleaved"] else (slice(0, rd // 2), slice(rd // 2, rd))
    z = torch.complex(out[..., one], out[..., two]) * turn
    out[..., one], out[..., two] = z.real, z.imag
    return out


def _exact_scale(amax):
    """The smallest fp16 of which 127 are at least amax (64 bits), in 64 bits."""
    least = amax.cpu().numpy() / 127
    scale = least.astype(np.float16)
    scale = np.where(scale < least, np.nextafter(scale, np.float16(np.inf)), scale).astype(np.float64)
    return torch.from_numpy(np.maximum(scale, 2.0 ** -24)).cuda()


def _exact_stored(x, group):
    y = x.double().reshape(*x.shape[:-1], -1, group)
    scale = _exact_scale(y.abs().amax(-1, keepdim=True))
    return (torch.round(y / scale) * scale).reshape(x.shape)


def _exact_rows(case, s, n, page, head, at):
    """What keys (n = 0) or values (n = 1) of one head stand for, tokens `at` of pages `page`."""
    x = s["cache"][n][page, head, at].double()
    return x * s["cache"][2 + n][page, head, at].double().repeat_interleave(case["group"], -1) if case["group"] else x


def exact(case, seed):
    s = prepare(case, seed)
    kind, d, hk, page = case["kind"], case["d"], case["hk"], case["page"]
    if kind == "axes":
        q, k = (_exact_rotary(case, s[n], s["positions"]) for n in ("q", "k"))
        if not case["store"]:
            return q, k
        if case["group"]:
            return [q] + [_exact_stored(x.half(), case["group"]) for x in (k, s["v"])]
        outs = [q]
        for x in (k, s["v"]):
            rows = torch.zeros((s["cache"][0].shape[0] * page, hk, d), dtype=torch.float64, device="cuda")
            rows[s["slots"]] = x.double()
            outs.append(rows.view(-1, page, hk, d).transpose(1, 2))
        return outs
    if kind == "bounds":
        per_page = page // case["block"]
        lo, hi = (torch.empty(s["lo"].shape, dtype=torch.float64, device="cuda") for _ in range(2))
        token = torch.arange(case["block"], device="cuda")
        where = s["done"] // per_page, s["done"] % per_page
        for h in range(hk):
            k = _exact_rows(case, s, 0, where[0][:, None], h, where[1][:, None] * case["block"] + token)
            scale = _exact_scale(k.abs().amax((1, 2)))[:, None]
            lo[:, h], hi[:, h] = torch.floor(k.amin(1) / scale) * scale, torch.ceil(k.amax(1) / scale) * scale
        return lo, hi
    out = torch.zeros((case["b"], case["hq"], d), dtype=torch.float64, device="cuda")
    shared = case["hq"] // hk
    if kind == "prefix":
        token = torch.arange(case["prefix"], device="cuda")
        ahead = s["prefix_pages"].long()[token // page], token % page
        for h in range(hk):
            heads = slice(h * shared, (h + 1) * shared)
            k, v = (_exact_rows(case, s, n, ahead[0], h, ahead[1]) for n in (0, 1))
            score = (s["q"][:, heads].double().reshape(-1, d) @ k.T * d ** -0.5).view(case["b"], shared, -1)
            norm = torch.logsumexp(score, -1)
            part = (torch.exp(score - norm[..., None]).flatten(0, 1) @ v).view(case["b"], shared, d)
            del score
            for i, n in enumerate(_lengths(case)):
                if n < 0:
                    continue
                if n == 0:
                    out[i, heads] = part[i]
                    continue
                at = token.new_tensor(range(n))
                at = s["pages"][i].long()[at // page], at % page
                k2, v2 = (_exact_rows(case, s, m, at[0], h, at[1]) for m in (0, 1))
                mine = s["q"][i, heads].double() @ k2.T * d ** -0.5
                both = torch.logaddexp(norm[i], torch.logsumexp(mine, -1))[:, None]
                out[i, heads] = torch.exp(norm[i][:, None] - both) * part[i] + torch.exp(mine - both) @ v2
        return out
    block, per_page = case["block"], page // case["block"]
    for i, n in enumerate(_lengths(case)):
        if n == 0:
            continue
        blocks = -(-n // block)
        table = s["pages"][i].long()
        for h in range(hk):
            heads = slice(h * shared, (h + 1) * shared)
            q = s["q"][i, heads].double()
            inner = range(min(case["first"], blocks), max(min(case["first"], blocks), blocks - case["last"]))
            chosen = set(range(blocks)) - set(inner)
            if len(inner) > case["top"]:
                number = torch.arange(inner.start, inner.stop, device="cuda")
                where = table[number // per_page], number % per_page
                low, high = (s["bounds"][where[0], h, where[1], x].double() for x in (0, 1))
                step = _exact_scale(q.abs().amax(-1, keepdim=True))
                whole = torch.round(q / step)
                dot = (torch.where(whole < 0, whole, 0.0) @ low.T) + (torch.where(whole > 0, whole, 0.0) @ high.T)
                score = (dot * (step * s["bound_scales"][where[0], h, where[1]].double())).float().amax(0)  # a score has 32 bits
                best = sorted(range(len(inner)), key=lambda x, v=score.tolist(): (-v[x], x))[:case["top"]]
                chosen |= {inner.start + x for x in best}
            else:
                chosen |= set(inner)
            at = (torch.tensor(sorted(chosen), device="cuda")[:, None] * block + torch.arange(block, device="cuda")).flatten()
            at = at[at < n]
            at = table[at // page], at % page
            k, v = (_exact_rows(case, s, m, at[0], h, at[1]) for m in (0, 1))
            out[i, heads] = torch.softmax(q @ k.T * d ** -0.5, -1) @ v
    return out


# ---- what a pass cannot do without -------------------------------------------------------------------------------

def _tokens_attended(case, n):
    """(blocks whose bounds are looked at, tokens attended) of a sequence of n tokens."""
    blocks = -(-n // case["block"])
    total = case["first"] + case["last"] + case["top"]
    if blocks <= total:
        return 0, n
    return blocks - case["first"] - case["last"], total * case["block"] - (blocks * case["block"] - n)


def work(case):
    """Inputs read once, results written once.  Rotation: six operations a pair; quantizing: two an element; bounds: two an element; attention: two
    multiply-adds for every query head and dimension of a token that is seen; a score: one for every dimension of a block and query head."""
    d, hk, kind = case["d"], case["hk"], case["kind"]
    element = 2 if not case["group"] else 1 + 2 / case["group"]  # bytes in the cache, scales included
    if kind == "axes":
        t, hq, rd = case["t"], case["hq"], case["rd"]
        moved = 4 * t * hq * d + 8 * t * len(_sections(case))
        turned = t * (hq + hk) * rd * 3
        if not case["store"]:
            return {"bytes": moved + 4 * t * hk * d, "flops": turned}
        # into the cache, and for int8 the values read back
        return {"bytes": int(moved + 2 * t * hk * d * (2 + element + (2 if case["group"] else 0)) + 8 * t), "flops": turned + (4 * t * hk * d if case["group"] else 0)}
    if kind == "bounds":
        done = case["t"] // case["block"] if case["whole"] else case["t"] // 16
        return {"bytes": int(done * hk * d * (case["block"] * element + 2 + 8)) + 2 * done * hk + 8 * case["t"], "flops": 2 * done * hk * d * case["block"]}
    b, hq = case["b"], case["hq"]
    if kind == "prefix":
        own_tokens = sum(max(0, n) for n in _lengths(case))
        rows = sum(n >= 0 for n in _lengths(case))
        table = 4 * sum(-(-max(0, n) // case["page"]) for n in _lengths(case)) + 4 * -(-case["prefix"] // case["page"]) + 4 * b
        return {"bytes": int(2 * (case["prefix"] + own_tokens) * hk * d * element) + 4 * b * hq * d + table,
                "flops": 4 * hq * d * (case["prefix"] * rows + own_tokens)}
    scored, seen = (sum(x) for x in zip(*(_tokens_attended(case, n) for n in _lengths(case))))
    table = 4 * sum(-(-n // case["page"]) for n in _lengths(case)) + 4 * b
    return {"bytes": int(2 * seen * hk * d * element) + scored * hk * (2 * d + 2) + 4 * b * hq * d + table, "flops": 4 * seen * hq * d + 2 * scored * hq * d}
