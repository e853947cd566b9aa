"""Rotary positions, the paged key-value cache and attention of one new token a sequence: the binding of
include/pplb200_attention.h, where the operators, their layouts and what they refuse are described.

Tensors are checked for type, shape and device by the compiled part of the binding (csrc/attention_binding.cpp: ValueError); sizes,
alignment and strides by the C ABI, whose refusals raise PplError.
"""
import ctypes
import importlib.util
import os
import struct
import sys

import torch

from . import LIB_PATH, PplError, _check, lib

EXPORTS = [
    "pplb200_rotary_frequencies", "pplb200_rotary_fp16", "pplb200_kv_cache_write_fp16", "pplb200_kv_cache_read_fp16",
    "pplb200_paged_decode_attention_workspace_bytes", "pplb200_paged_decode_attention_fp16", "pplb200_kv_cache_offset",
    "pplb200_paged_attention_offset",
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
lib.pplb200_kv_cache_offset.argtypes = lib.pplb200_paged_attention_offset.argtypes = [_blk, _i64, _i32]
lib.pplb200_kv_cache_offset.restype = lib.pplb200_paged_attention_offset.restype = _i64

_pack_cache = struct.Struct("=4Q7q4i").pack


def binding_path():
    """Compiled for this Python and this torch, as build.py names it."""
    return os.path.join(os.path.dirname(LIB_PATH), "pplb200_attention_binding.%s.torch-%s.so" % (sys.implementation.cache_tag, torch.__version__))


def _load_binding():
    path = binding_path()
    if not os.path.exists(path):
        raise ImportError("the compiled part of the binding is not built (%s); run `python ppl.llm.kernel.cuda_b200/build.py`." % os.path.normpath(path))
    spec = importlib.util.spec_from_file_location("pplb200_attention_binding", os.path.normpath(path))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


_binding = _load_binding()
# what the compiled functions call
_rotary, _write, _read, _attend = (ctypes.cast(f, ctypes.c_void_p).value for f in (
    lib.pplb200_rotary_fp16, lib.pplb200_kv_cache_write_fp16, lib.pplb200_kv_cache_read_fp16, lib.pplb200_paged_decode_attention_fp16))


def _need(ok, what):
    if not ok:
        raise ValueError(what)


_F16, _I64, _I32 = torch.float16, torch.int64, torch.int32


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


class _LaidOutOnce:
    """Calls are given what an object laid out when it was made: its attributes do not change."""

    def __setattr__(self, name, value):
        if name in self.__dict__:
            raise AttributeError("%s of a %s is laid out once; make a new one" % (name, type(self).__name__))
        object.__setattr__(self, name, value)


class RotaryTable(_LaidOutOnce):
    """Frequencies of the rotated planes, laid out once on `device`.  scaling: "none", "linear", "ntk", "yarn" or "wavelength"."""

    def __init__(self, rotary_dim, base=10000.0, scaling="none", factor=1.0, original_length=0, keep_turns=0.0, stretch_turns=0.0,
                 device="cuda"):
        _need(scaling in ROTARY_SCALINGS, "unknown scaling %r" % (scaling,))
        words, magnitude = (ctypes.c_uint64 * max(1, rotary_dim // 2))(), ctypes.c_float()
        _check(lib.pplb200_rotary_frequencies(rotary_dim, base, ROTARY_SCALINGS[scaling], factor, original_length, keep_turns,
                                              stretch_turns, words, ctypes.byref(magnitude)))
        self.rotary_dim, self.magnitude = rotary_dim, magnitude.value
        self.turns = torch.frombuffer(words, dtype=_I64).to(device, copy=True)
        self._args = (self.turns.data_ptr(), self.turns.get_device(), rotary_dim, self.magnitude)
        _settle(self.turns.device)


def rotary_fp16(q, k, positions, table, interleaved=False, q_out=None, k_out=None):
    """q [tokens, q_heads, head_dim], k [tokens, k_heads, head_dim] fp16 (either may be None) -> both rotated by `positions` (int64
    [tokens]).  q_out=q and k_out=k rotate in place."""
    dev, stream = _here()
    if q is not None and q_out is None:
        q_out = torch.empty(q.shape, dtype=_F16, device=q.device)
    if k is not None and k_out is None:
        k_out = torch.empty(k.shape, dtype=_F16, device=k.device)
    rc = _binding.rotary(_rotary, stream, dev, q, k, positions, table._args, interleaved, q_out, k_out)
    if rc:
        raise PplError(rc)
    return (None if q is None else q_out), (None if k is None else k_out)


class PagedKVCache(_LaidOutOnce):
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
        block = _pack_cache(k.data_ptr(), v.data_ptr(), *(0 if t is None else t.data_ptr() for t in (k_scale, v_scale)), pages,
                            *k.stride()[:3], *strides, page, heads, dim, group)
        self._args = (block, k.get_device())

    @classmethod
    def allocate(cls, num_pages, page_size, kv_heads, head_dim, quant_group=0, device="cuda"):
        """A zeroed cache; quant_group 0 (fp16), 8 or head_dim (int8)."""
        _need(quant_group in (0, 8, head_dim), "quant_group must be 0, 8 or head_dim")
        k, v = (torch.zeros((num_pages, kv_heads, page_size, head_dim), dtype=torch.int8 if quant_group else torch.float16, device=device)
                for _ in range(2))
        scales = (torch.zeros((num_pages, kv_heads, page_size, head_dim // quant_group), dtype=torch.float16, device=device)
                  for _ in range(2 if quant_group else 0))
        cache = cls(k, v, *scales)
        _settle(k.device)
        return cache


def kv_cache_write(cache, k, v, slots):
    """Stores k, v fp16 [tokens, kv_heads, head_dim] at `slots` (int64 [tokens]: page * page_size + place; negative: not stored)."""
    dev, stream = _here()
    rc = _binding.write(_write, stream, dev, cache._args, None, k, v, None, slots, None, False, None)
    if rc:
        raise PplError(rc)


def rotary_kv_cache_write(cache, q, k, v, positions, slots, table, interleaved=False, q_out=None):
    """rotary_fp16 of q and k and kv_cache_write of the rotated k and of v, in one pass.  Returns the rotated q."""
    _need(table is not None, "a rotary table is needed")
    dev, stream = _here()
    if q is not None and q_out is None:
        q_out = torch.empty(q.shape, dtype=_F16, device=q.device)
    rc = _binding.write(_write, stream, dev, cache._args, q, k, v, positions, slots, table._args, interleaved, q_out)
    if rc:
        raise PplError(rc)
    return q_out


def kv_cache_read(cache, slots, k_out=None, v_out=None):
    """-> (k, v) fp16 [tokens, kv_heads, head_dim], what is stored at `slots` (int64 [tokens]; negative: zeros)."""
    dev, stream = _here()
    if k_out is None:
        k_out = torch.empty((slots.shape[0], cache.kv_heads, cache.head_dim), dtype=_F16, device=cache.k.device)
    if v_out is None:
        v_out = torch.empty((slots.shape[0], cache.kv_heads, cache.head_dim), dtype=_F16, device=cache.k.device)
    rc = _binding.read(_read, stream, dev, cache._args, slots, k_out, v_out)
    if rc:
        raise PplError(rc)
    return k_out, v_out


class PagedDecodeAttention(_LaidOutOnce):
    """Attention of one new token a sequence over a PagedKVCache.  Owns the workspace for `max_batch` sequences of `max_length` tokens, so
    one object serves one stream at a time, and is kept until its calls have run.  scale: 1 / sqrt(head_dim) unless given; window: how many of the last tokens are seen (0: all)."""

    def __init__(self, cache, q_heads, max_batch, max_length, scale=None, window=0):
        _need(q_heads > 0 and q_heads % cache.kv_heads == 0, "q_heads must be a multiple of the cache's heads")
        _need(max_batch >= 0 and max_length >= 0 and window >= 0, "negative extent")
        self.cache, self.q_heads, self.max_batch, self.window = cache, q_heads, max_batch, window
        self.max_pages = -(-max_length // cache.page_size)
        self.scale = cache.head_dim ** -0.5 if scale is None else scale
        need = lib.pplb200_paged_decode_attention_workspace_bytes(max_batch, self.max_pages * cache.page_size, q_heads, cache.kv_heads, cache.head_dim)
        self.ws = torch.zeros((need,), dtype=torch.uint8, device=cache.k.device)
        self._args = (q_heads, max_batch, self.max_pages, self.ws.data_ptr(), need, window, self.scale)
        _settle(cache.k.device)

    def __call__(self, q, pages, lengths, out=None, lse=None):
        """q fp16 [batch, q_heads, head_dim], pages int32 [batch, pages a sequence] (negative: a hole), lengths int32 [batch] -> out as q;
        lse fp32 [batch, q_heads], where given, receives log(sum exp(scores))."""
        dev, stream = _here()
        if out is None:
            out = torch.empty(q.shape, dtype=_F16, device=q.device)
        rc = _binding.attend(_attend, stream, dev, self.cache._args, self._args, q, pages, lengths, out, lse)
        if rc:
            raise PplError(rc)
        return out
