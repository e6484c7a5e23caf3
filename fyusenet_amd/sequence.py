"""Attention over sequences, and the paged cache of their keys and values (the "sequences" part of include/fynhip.h).

Tensors are device memory of the caller's: anything with data_ptr(), dtype, shape and stride() (torch tensors), anything
with __cuda_array_interface__, a capi.TensorView as custom layers get them, or a DeviceArray.  `stream` is a hipStream_t as
an integer (torch.cuda.current_stream().cuda_stream), 0 the default stream.  Calls return before the work is done.
"""
import array
import ctypes
import struct

import numpy as np

from . import capi

_SIZE = {capi.STORAGE_F16: 2, capi.STORAGE_F32: 4}


class DeviceArray:
    """Device memory: address, element type ("float16", "float32" or "int32"), shape, and distances in elements (dense if
    not given)."""

    __slots__ = ("ptr", "dtype", "shape", "strides")

    def __init__(self, ptr, dtype, shape, strides=None):
        self.ptr, self.dtype, self.shape = int(ptr), str(dtype), tuple(shape)
        if strides is None:
            strides, n = [], 1
            for m in reversed(self.shape):
                strides.insert(0, n)
                n *= m
        self.strides = tuple(strides)

    @staticmethod
    def of(x, name, heads=0):
        """`x` as a DeviceArray; a TensorView [height, width, channels] becomes [height, width, heads, channels / heads]."""
        if isinstance(x, DeviceArray):
            return x
        if hasattr(x, "data_ptr"):
            if not getattr(x, "is_cuda", True):
                raise capi.FynException(capi.ERR_INVALID, "%s: not device memory" % name)
            return DeviceArray(x.data_ptr(), str(x.dtype).rpartition(".")[2], x.shape, x.stride())
        if isinstance(x, capi.TensorView):
            if x.channels % max(1, heads):
                raise capi.FynException(capi.ERR_INVALID, "%s: %d channels are not %d heads" % (name, x.channels, heads))
            wide, dim = x.width + 2 * x.padding, x.channels // max(1, heads)
            typ = "float16" if x.storage == capi.STORAGE_F16 else "float32"
            return DeviceArray((x.data or 0) + (x.padding * wide + x.padding) * x.channel_pitch * _SIZE[x.storage], typ,
                               (x.height, x.width, heads, dim), (wide * x.channel_pitch, x.channel_pitch, dim, 1))
        if hasattr(x, "__cuda_array_interface__"):
            a = x.__cuda_array_interface__
            dtype = np.dtype(a["typestr"])
            strides = a.get("strides")
            return DeviceArray(a["data"][0], dtype.name, a["shape"], strides and [s // dtype.itemsize for s in strides])
        raise capi.FynException(capi.ERR_INVALID, "%s: not device memory" % name)


_TYPES = {capi.STORAGE_F16: "float16", capi.STORAGE_F32: "float32"}
_STORAGES = {"float16": capi.STORAGE_F16, "float32": capi.STORAGE_F32}

# The structs of the calls that a step makes, packed at once (field by field takes longer than the launch).
_ROWS = "Q3q"
_ATTENTION = struct.Struct("=I9if4xQ" + 4 * _ROWS)
_ATTEND = struct.Struct("=I3if4x" + 2 * _ROWS)
_ONE = struct.Struct("=" + _ROWS)
assert _ATTENTION.size == ctypes.sizeof(capi.AttentionDesc) and _ATTEND.size == ctypes.sizeof(capi.AttendDesc) and _ONE.size == ctypes.sizeof(capi.Rows)

_V = ctypes.c_void_p
_calls = {}


def _call(name, *args):
    """An entry point that takes packed structs (bytes) where its prototype has pointers to them."""
    fn = _calls.get(name)
    if fn is None:
        capi.lib()
        fn = _calls[name] = ctypes.CFUNCTYPE(ctypes.c_int, *args)((name, capi.lib()))
    return fn


_dtypes = {}   # element types of tensors that have been seen -> their names


def _take(x, name, heads=0):
    """Address, element type, shape and strides of a tensor."""
    try:
        known = _dtypes.get(x.dtype)
        if known is None:
            known = _dtypes[x.dtype] = str(x.dtype).rpartition(".")[2]
        if x.is_cuda:
            return x.data_ptr(), known, x.shape, x.stride()
    except (AttributeError, TypeError):
        pass
    a = DeviceArray.of(x, name, heads)
    return a.ptr, a.dtype, a.shape, a.strides


def _rows(a, name, typ, shape):
    """Address and pitches (sequence, token, head) of a tensor [.., token, head, dim] that has to have this type and shape."""
    ptr, dtype, have, st = a
    if dtype != typ:
        raise capi.FynException(capi.ERR_INVALID, "%s: %s values, %s are expected" % (name, dtype, typ))
    if have != shape and tuple(have) != tuple(shape):
        raise capi.FynException(capi.ERR_INVALID, "%s: shape %s, %s is expected" % (name, tuple(have), tuple(shape)))
    if st[-1] != 1 and shape[-1] > 1:
        raise capi.FynException(capi.ERR_INVALID, "%s: the values of a head have to lie side by side" % name)
    # (a distance that nothing is multiplied with may be anything)
    return (ptr, st[0] if len(shape) == 4 and shape[0] > 1 else 0, st[-3] if shape[-3] > 1 else 0, st[-2] if shape[-2] > 1 else 0)


def attention(queries, keys, values, result, lengths=None, causal=True, window=0, sinks=0, scale=0.0, heads=0, kv_heads=0, stream=0):
    """fyn_attention: queries and result [batch, tokens, heads, dim], keys and values [batch, tokens, kv_heads, dim].
    lengths: int32 [batch] or None.  heads and kv_heads are asked for only where tensors are given as TensorViews, whose
    rows are the sequences."""
    q, k = _take(queries, "queries", heads), _take(keys, "keys", kv_heads or heads)
    shape, kv_shape = q[2], k[2]
    if len(shape) != 4 or len(kv_shape) != 4:
        raise capi.FynException(capi.ERR_INVALID, "attention: tensors [batch, tokens, heads, dim] are expected")
    batch, tokens, nheads, dim = shape
    typ = q[1]
    kv_shape = (batch, tokens, kv_shape[2], dim)
    storage = _STORAGES.get(typ)
    if storage is None:
        raise capi.FynException(capi.ERR_INVALID, "queries: %s values are not supported" % typ)
    at = 0
    if lengths is not None:
        n = _take(lengths, "lengths")
        if n[1] != "int32" or tuple(n[2]) != (batch,) or (batch > 1 and n[3][0] != 1):
            raise capi.FynException(capi.ERR_INVALID, "lengths: %d int32 values side by side are expected" % batch)
        at = n[0]
    try:
        d = _ATTENTION.pack(_ATTENTION.size, storage, batch, tokens, nheads, kv_shape[2], dim, 1 if causal else 0, window, sinks, scale, at,
                            *_rows(q, "queries", typ, shape), *_rows(k, "keys", typ, kv_shape),
                            *_rows(_take(values, "values", kv_heads or heads), "values", typ, kv_shape),
                            *_rows(_take(result, "result", heads), "result", typ, shape))
    except (struct.error, OverflowError) as e:
        raise capi.FynException(capi.ERR_INVALID, "attention: %s" % e)
    status = _call("fyn_attention", _V, _V)(d, stream)
    if status:
        capi.check(status)


_arrays = {}


def _ints(v):
    """int32 values as a call's argument.  (ctypes by itself takes any integer, and its last 32 bits.)"""
    n = len(v)
    t = _arrays.get(n)
    if t is None:
        t = _arrays[n] = ctypes.c_int32 * n
    if n < 8:   # (two values: 0.4 us, and 0.7 by way of an array; 1000: 18 us by way of an array, and 80)
        return t(*map(capi.int32, v))
    try:
        return t.from_buffer(array.array("i", v))
    except (OverflowError, TypeError) as e:
        raise capi.FynException(capi.ERR_INVALID, "int32 values are expected: %s" % e)


class SequenceCache:
    """fyn_cache: keys and values of `sequences` sequences in `pages` pages of `page_tokens` tokens, for `layers` attention
    layers of `heads` heads that share `kv_heads` key heads of `head_dim` values.

    A step: extend(sequences, tokens) names the sequences that get new tokens and how many; then, for each layer,
    write(layer, keys, values) and attend(layer, queries, result) take these tokens' rows, sequence after sequence, as
    [rows, heads, dim]."""

    def __init__(self, storage, layers, heads, kv_heads, head_dim, page_tokens, pages, sequences, most_tokens=0, device=0):
        self._h = ctypes.c_void_p()
        d = capi.CacheDesc(ctypes.sizeof(capi.CacheDesc), *map(capi.int32, (storage, layers, heads, kv_heads, head_dim, page_tokens, pages, sequences, most_tokens)))
        capi.check(capi.lib().fyn_cache_create(capi.int32(device), ctypes.byref(d), ctypes.byref(self._h)))
        self.storage, self.layers, self.heads, self.kv_heads, self.head_dim = storage, layers, heads, kv_heads, head_dim
        self.page_tokens, self.sequences = page_tokens, sequences
        self._type = _TYPES[storage]

    def _same(self, a, b, what):
        if len(a) != len(b):
            raise capi.FynException(capi.ERR_INVALID, "%s: %d sequences and %d values" % (what, len(a), len(b)))

    def extend(self, sequences, tokens, stream=0):
        self._same(sequences, tokens, "extend")
        capi.check(capi.lib().fyn_cache_extend(self._h, len(sequences), _ints(sequences), _ints(tokens), stream))

    def _kv(self, keys, values):
        k = _take(keys, "keys")
        shape = (k[2][0] if len(k[2]) == 3 else 0, self.kv_heads, self.head_dim)
        return _ONE.pack(*_rows(k, "keys", self._type, shape)), _ONE.pack(*_rows(_take(values, "values"), "values", self._type, shape)), shape[0]

    def write(self, layer, keys, values, stream=0):
        k, v, rows = self._kv(keys, values)
        capi.check(_call("fyn_cache_write", _V, ctypes.c_int, _V, _V, ctypes.c_int, _V)(self._h, capi.int32(layer), k, v, capi.int32(rows), stream))

    def attend(self, layer, queries, result, window=0, sinks=0, scale=0.0, stream=0):
        q = _take(queries, "queries")
        shape = (q[2][0] if len(q[2]) == 3 else 0, self.heads, self.head_dim)
        try:
            d = _ATTEND.pack(_ATTEND.size, shape[0], window, sinks, scale, *_rows(q, "queries", self._type, shape),
                             *_rows(_take(result, "result"), "result", self._type, shape))
        except (struct.error, OverflowError) as e:
            raise capi.FynException(capi.ERR_INVALID, "attend: %s" % e)
        status = _call("fyn_cache_attend", _V, ctypes.c_int, _V, _V)(self._h, capi.int32(layer), d, stream)
        if status:
            capi.check(status)

    def read(self, sequences, layer, keys, values, stream=0):
        """Keys and values of whole sequences into [tokens of all of them, kv_heads, dim]."""
        k, v, rows = self._kv(keys, values)
        capi.check(_call("fyn_cache_read", _V, ctypes.c_int, _V, ctypes.c_int, _V, _V, ctypes.c_int, _V)(
            self._h, len(sequences), _ints(sequences), capi.int32(layer), k, v, capi.int32(rows), stream))

    def fork(self, source, targets, tokens=-1, stream=0):
        capi.check(capi.lib().fyn_cache_fork(self._h, capi.int32(source), len(targets), _ints(targets), capi.int32(tokens), stream))

    def copy(self, sources, targets, stream=0):
        self._same(sources, targets, "copy")
        capi.check(capi.lib().fyn_cache_copy(self._h, len(sources), _ints(sources), _ints(targets), stream))

    def truncate(self, sequences, tokens, stream=0):
        self._same(sequences, tokens, "truncate")
        capi.check(capi.lib().fyn_cache_truncate(self._h, len(sequences), _ints(sequences), _ints(tokens), stream))

    def free(self, sequences, stream=0):
        capi.check(capi.lib().fyn_cache_free(self._h, len(sequences), _ints(sequences), stream))

    def compact(self, stream=0):
        """-> the number of used pages, which are the first ones now."""
        used = ctypes.c_int(0)
        capi.check(capi.lib().fyn_cache_compact(self._h, ctypes.byref(used), stream))
        return used.value

    def lengths(self, sequences):
        got = (ctypes.c_int32 * len(sequences))()
        capi.check(capi.lib().fyn_cache_lengths(self._h, len(sequences), _ints(sequences), got))
        return list(got)

    def pages(self):
        """-> pages in use, pages that are free."""
        used, left = ctypes.c_int(0), ctypes.c_int(0)
        capi.check(capi.lib().fyn_cache_pages(self._h, ctypes.byref(used), ctypes.byref(left)))
        return used.value, left.value

    def order(self, stream):
        """What this cache's calls have queued comes before what is queued on this stream from now on."""
        capi.check(capi.lib().fyn_cache_order(self._h, stream))

    def close(self):
        if self._h:
            capi.check(capi.lib().fyn_cache_destroy(self._h))
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
