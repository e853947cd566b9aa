"""Rotary positions, the paged key-value cache and attention of one new token a sequence: the binding of
include/pplb200_attention.h, where the operators, their layouts and what they refuse are described.

Tensors are checked for type, shape and device here; sizes, alignment and strides by the C ABI, whose refusals raise PplError.
"""
import ctypes
import struct

import torch

from . import PplError, _check, lib

EXPORTS = [
    "pplb200_rotary_frequencies", "pplb200_rotary_fp16", "pplb200_kv_cache_write_fp16", "pplb200_kv_cache_read_fp16",
    "pplb200_paged_decode_attention_workspace_bytes", "pplb200_paged_decode_attention_fp16", "pplb200_kv_cache_offset",
]
ROTARY_SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3, "wavelength": 4}

_vp, _i64, _i32, _f64, _blk = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_double, ctypes.c_char_p
lib.pplb200_rotary_frequencies.argtypes = [_i32, _f64, _i32, _f64, _f64, _f64, _f64, _vp, _vp]
lib.pplb200_rotary_fp16.argtypes = [_vp, _blk]
lib.pplb200_kv_cache_write_fp16.argtypes = [_vp, _blk, _blk]
lib.pplb200_kv_cache_read_fp16.argtypes = [_vp, _blk, _vp, _i64, _vp, _vp]
lib.pplb200_paged_decode_attention_workspace_bytes.argtypes = [_i64, _i64, _i32, _i32, _i32]
lib.pplb200_paged_decode_attention_workspace_bytes.restype = _i64
lib.pplb200_paged_decode_attention_fp16.argtypes = [_vp, _blk, _blk]
lib.pplb200_kv_cache_offset.argtypes = [_blk, _i64, _i32]
lib.pplb200_kv_cache_offset.restype = _i64

# the argument blocks of the header, packed: a call converts three or four arguments instead of twenty
_pack_cache = struct.Struct("=4Q7q4i").pack
_pack_rotary = struct.Struct("=6Q5q5if").pack
_pack_write = struct.Struct("=7Q5q3if").pack
_pack_attention = struct.Struct("=6Q6q2ifi").pack
_rotary, _write = lib.pplb200_rotary_fp16, lib.pplb200_kv_cache_write_fp16
_read, _attend = lib.pplb200_kv_cache_read_fp16, lib.pplb200_paged_decode_attention_fp16


def _need(ok, what):
    if not ok:
        raise ValueError(what)


_F16, _I64, _I32 = torch.float16, torch.int64, torch.int32


# These run on every call, and a small call's kernel takes two microseconds: one look at each property, the text only where it is needed.
def _heads(t, name, tokens, head_dim, device):
    """(heads, elements between tokens) of an fp16 [tokens, heads, head_dim] tensor whose heads are contiguous."""
    shape, stride = t.shape, t.stride()
    if (len(shape) != 3 or shape[0] != tokens or shape[2] != head_dim or stride[2] != 1 or (stride[1] != head_dim and shape[1] > 1)
            or t.dtype is not _F16 or t.get_device() != device):
        raise ValueError("%s must be fp16 [%d, heads, %d] on device %d, the heads of a token contiguous; got %s %s, strides %s, on device %d"
                         % (name, tokens, head_dim, device, t.dtype, tuple(shape), stride, t.get_device()))
    return shape[1], stride[0]


def _indices(t, name, tokens, device):
    if t.shape != (tokens,) or t.dtype is not _I64 or (t.stride(0) != 1 and tokens > 1) or t.get_device() != device:
        raise ValueError("%s must be a contiguous int64 [%d] tensor on device %d" % (name, tokens, device))
    return t.data_ptr()


def _here():
    """(current device, handle of its current stream): tensors have to be on that device.  The first call puts the look-up in its place."""
    global _here
    torch.cuda.init()
    device, raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream

    def _here():
        d = device()
        return d, raw_stream(d)
    return _here()


def _settle(device):
    """What an object has just laid out on the device is there before the object is: its calls may come on any stream."""
    if device.type == "cuda":
        torch.cuda.current_stream(device).synchronize()


class RotaryTable:
    """Frequencies of the rotated planes, laid out once on `device`.  scaling: "none", "linear", "ntk", "yarn" or "wavelength"."""

    def __init__(self, rotary_dim, base=10000.0, scaling="none", factor=1.0, original_length=0, keep_turns=0.0, stretch_turns=0.0,
                 device="cuda"):
        _need(scaling in ROTARY_SCALINGS, "unknown scaling %r" % (scaling,))
        words, magnitude = (ctypes.c_uint64 * max(1, rotary_dim // 2))(), ctypes.c_float()
        _check(lib.pplb200_rotary_frequencies(rotary_dim, base, ROTARY_SCALINGS[scaling], factor, original_length, keep_turns,
                                              stretch_turns, words, ctypes.byref(magnitude)))
        self.rotary_dim, self.magnitude = rotary_dim, magnitude.value
        self.turns = torch.frombuffer(words, dtype=_I64).to(device, copy=True)
        self.device_index, self.address = self.turns.get_device(), self.turns.data_ptr()
        _settle(self.turns.device)


def rotary_fp16(q, k, positions, table, interleaved=False, q_out=None, k_out=None):
    """q [tokens, q_heads, head_dim], k [tokens, k_heads, head_dim] fp16 (either may be None) -> both rotated by `positions` (int64
    [tokens]).  q_out=q and k_out=k rotate in place."""
    dev, stream = _here()
    if q is None and k is None:
        raise ValueError("neither q nor k is given")
    tokens, _, head_dim = (k if q is None else q).shape
    qp = qo = qh = qs = qos = kp = ko = kh = ks = kos = 0
    if q is not None:
        qh, qs = _heads(q, "q", tokens, head_dim, dev)
        if q_out is None:
            q_out = torch.empty((tokens, qh, head_dim), dtype=_F16, device=q.device)
        heads, qos = _heads(q_out, "q_out", tokens, head_dim, dev)
        qp, qo = q.data_ptr(), q_out.data_ptr()
        if heads != qh:
            raise ValueError("q_out must have the heads of q")
    if k is not None:
        kh, ks = _heads(k, "k", tokens, head_dim, dev)
        if k_out is None:
            k_out = torch.empty((tokens, kh, head_dim), dtype=_F16, device=k.device)
        heads, kos = _heads(k_out, "k_out", tokens, head_dim, dev)
        kp, ko = k.data_ptr(), k_out.data_ptr()
        if heads != kh:
            raise ValueError("k_out must have the heads of k")
    if table.device_index != dev:
        raise ValueError("the rotary table is on another device")
    rc = _rotary(stream, _pack_rotary(qp, kp, qo, ko, _indices(positions, "positions", tokens, dev), table.address, tokens,
                                      qs, ks, qos, kos, qh, kh, head_dim, table.rotary_dim, 1 if interleaved else 0, table.magnitude))
    if rc:
        raise PplError(rc)
    return (None if q is None else q_out), (None if k is None else k_out)


class PagedKVCache:
    """One layer's cache over the caller's tensors: k, v [pages, kv_heads, tokens of a page, head_dim], fp16, or int8 with fp16
    k_scale, v_scale [pages, kv_heads, tokens of a page, head_dim / group].  Any strides (k as v, k_scale as v_scale) with contiguous
    dimensions: a cache that is stored token by token is passed as its transpose(1, 2)."""

    def __init__(self, k, v, k_scale=None, v_scale=None):
        _need(k.dim() == 4 and v.shape == k.shape and v.stride() == k.stride(), "k and v must be [pages, heads, tokens, dimensions], laid out alike")
        _need(k.dtype == v.dtype and k.dtype in (torch.float16, torch.int8), "k and v must be fp16 or int8")
        _need((k.dtype == torch.int8) == (k_scale is not None) == (v_scale is not None), "an int8 cache has scales, an fp16 cache none")
        _need(k.stride(3) == 1, "a row's dimensions must be contiguous")
        pages, heads, page, dim = k.shape
        strides, group = [0, 0, 0], 0
        _need(all(t is None or t.device == k.device for t in (v, k_scale, v_scale)), "the cache must be on one device")
        if k_scale is not None:
            _need(k_scale.dtype == v_scale.dtype == torch.float16, "scales must be fp16")
            _need(k_scale.shape[:3] == k.shape[:3] and k_scale.dim() == 4 and v_scale.shape == k_scale.shape and v_scale.stride() == k_scale.stride(),
                  "scales must be [pages, heads, tokens, dimensions / group], laid out alike")
            groups = k_scale.shape[3]
            _need(groups > 0 and dim % groups == 0 and (groups == 1 or k_scale.stride(3) == 1), "a row's scales must be contiguous and divide it")
            strides, group = k_scale.stride()[:3], dim // groups
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.num_pages, self.kv_heads, self.page_size, self.head_dim, self.quant_group = pages, heads, page, dim, group
        self.device_index = k.get_device()
        self._block = _pack_cache(k.data_ptr(), v.data_ptr(), *(0 if t is None else t.data_ptr() for t in (k_scale, v_scale)), pages,
                                  *k.stride()[:3], *strides, page, heads, dim, group)

    @classmethod
    def allocate(cls, num_pages, page_size, kv_heads, head_dim, quant_group=0, device="cuda"):
        """A zeroed cache; quant_group 0 (fp16), 8 or head_dim (int8)."""
        _need(quant_group in (0, 8, head_dim), "quant_group must be 0, 8 or head_dim")
        k, v = (torch.zeros((num_pages, kv_heads, page_size, head_dim), dtype=torch.int8 if quant_group else torch.float16, device=device)
                for _ in range(2))
        if not quant_group:
            return cls(k, v)
        return cls(k, v, *(torch.zeros((num_pages, kv_heads, page_size, head_dim // quant_group), dtype=torch.float16, device=device)
                           for _ in range(2)))


def _store(cache, q, k, v, positions, slots, table, interleaved, q_out):
    dev, stream = _here()
    tokens, dim = k.shape[0], cache.head_dim
    kh, ks = _heads(k, "k", tokens, dim, dev)
    vh, vs = _heads(v, "v", tokens, dim, dev)
    if kh != cache.kv_heads or vh != kh or cache.device_index != dev:
        raise ValueError("k and v must have the cache's %d heads, and the cache be on device %d" % (cache.kv_heads, dev))
    qp = qo = qh = qs = qos = pos = turns = rotary_dim = 0
    magnitude = 1.0
    if table is not None:
        if q is not None:
            qh, qs = _heads(q, "q", tokens, dim, dev)
            heads, qos = _heads(q_out, "q_out", tokens, dim, dev)
            qp, qo = q.data_ptr(), q_out.data_ptr()
            if heads != qh:
                raise ValueError("q_out must have the heads of q")
        if table.device_index != dev:
            raise ValueError("the rotary table is on another device")
        pos, turns, rotary_dim, magnitude = _indices(positions, "positions", tokens, dev), table.address, table.rotary_dim, table.magnitude
    rc = _write(stream, cache._block, _pack_write(qp, k.data_ptr(), v.data_ptr(), qo, pos, _indices(slots, "slots", tokens, dev), turns,
                                                  tokens, qs, ks, vs, qos, qh, rotary_dim, 1 if interleaved else 0, magnitude))
    if rc:
        raise PplError(rc)


def kv_cache_write(cache, k, v, slots):
    """Stores k, v fp16 [tokens, kv_heads, head_dim] at `slots` (int64 [tokens]: page * page_size + place; negative: not stored)."""
    _store(cache, None, k, v, None, slots, None, False, None)


def rotary_kv_cache_write(cache, q, k, v, positions, slots, table, interleaved=False, q_out=None):
    """rotary_fp16 of q and k and kv_cache_write of the rotated k and of v, in one pass.  Returns the rotated q."""
    if table is None:
        raise ValueError("a rotary table is needed")
    if q is not None and q_out is None:
        q_out = torch.empty(q.shape, dtype=torch.float16, device=q.device)
    _store(cache, q, k, v, positions, slots, table, interleaved, q_out)
    return q_out


def kv_cache_read(cache, slots, k_out=None, v_out=None):
    """-> (k, v) fp16 [tokens, kv_heads, head_dim], what is stored at `slots` (int64 [tokens]; negative: zeros)."""
    dev, stream = _here()
    tokens, heads, dim = slots.shape[0], cache.kv_heads, cache.head_dim
    if cache.device_index != dev:
        raise ValueError("the cache is not on the current device")
    if k_out is None:
        k_out = torch.empty((tokens, heads, dim), dtype=_F16, device=cache.k.device)
    if v_out is None:
        v_out = torch.empty((tokens, heads, dim), dtype=_F16, device=cache.k.device)
    for name, t in (("k_out", k_out), ("v_out", v_out)):
        if t.shape != (tokens, heads, dim) or t.dtype is not _F16 or not t.is_contiguous() or t.get_device() != dev:
            raise ValueError("%s must be a contiguous fp16 [%d, %d, %d] on device %d" % (name, tokens, heads, dim, dev))
    rc = _read(stream, cache._block, _indices(slots, "slots", tokens, dev), tokens, k_out.data_ptr(), v_out.data_ptr())
    if rc:
        raise PplError(rc)
    return k_out, v_out


class PagedDecodeAttention:
    """Attention of one new token a sequence over a PagedKVCache.  Owns the workspace for `max_batch` sequences of `max_length` tokens, so
    one object serves one stream at a time.  scale: 1 / sqrt(head_dim) unless given; window: how many of the last tokens are seen (0: all)."""

    def __init__(self, cache, q_heads, max_batch, max_length, scale=None, window=0):
        _need(q_heads > 0 and q_heads % cache.kv_heads == 0, "q_heads must be a multiple of the cache's heads")
        _need(max_batch >= 0 and max_length >= 0 and window >= 0, "negative extent")
        self.cache, self.q_heads, self.max_batch, self.window = cache, q_heads, max_batch, window
        self.max_pages = -(-max_length // cache.page_size)
        self.scale = cache.head_dim ** -0.5 if scale is None else scale
        need = lib.pplb200_paged_decode_attention_workspace_bytes(max_batch, self.max_pages * cache.page_size, q_heads, cache.kv_heads, cache.head_dim)
        self.ws = torch.zeros((need,), dtype=torch.uint8, device=cache.k.device)
        self._ws, self._ws_bytes = self.ws.data_ptr(), need
        _settle(cache.k.device)

    def __call__(self, q, pages, lengths, out=None, lse=None):
        """q fp16 [batch, q_heads, head_dim], pages int32 [batch, pages a sequence] (negative: a hole), lengths int32 [batch] -> out as q;
        lse fp32 [batch, q_heads], where given, receives log(sum exp(scores))."""
        (dev, stream), cache = _here(), self.cache
        batch, heads, dim = q.shape[0], self.q_heads, cache.head_dim
        if out is None:
            out = torch.empty((batch, heads, dim), dtype=_F16, device=q.device)
        qh, qs = _heads(q, "q", batch, dim, dev)
        oh, os_ = _heads(out, "out", batch, dim, dev)
        if qh != heads or oh != heads or batch > self.max_batch or cache.device_index != dev:
            raise ValueError("expected at most %d sequences of %d heads on the cache's device %d" % (self.max_batch, heads, cache.device_index))
        shape, stride = pages.shape, pages.stride()
        if (len(shape) != 2 or shape[0] != batch or shape[1] > self.max_pages or (stride[1] != 1 and shape[1] > 1) or pages.dtype is not _I32
                or pages.get_device() != dev):
            raise ValueError("pages must be int32 [%d, at most %d] with contiguous rows on device %d" % (batch, self.max_pages, dev))
        if lengths.shape != (batch,) or lengths.dtype is not _I32 or (lengths.stride(0) != 1 and batch > 1) or lengths.get_device() != dev:
            raise ValueError("lengths must be a contiguous int32 [%d] tensor on device %d" % (batch, dev))
        lse_ptr = 0
        if lse is not None:
            if lse.shape != (batch, heads) or lse.dtype is not torch.float32 or not lse.is_contiguous() or lse.get_device() != dev:
                raise ValueError("lse must be a contiguous fp32 [%d, %d] tensor on device %d" % (batch, heads, dev))
            lse_ptr = lse.data_ptr()
        rc = _attend(stream, cache._block, _pack_attention(q.data_ptr(), out.data_ptr(), lse_ptr, pages.data_ptr(), lengths.data_ptr(), self._ws, self._ws_bytes,
                                                           batch, shape[1], stride[0], qs, os_, heads, self.window, self.scale, 0))
        if rc:
            raise PplError(rc)
        return out
