"""A key-value cache in 8-bit codes and attention over it, or over the blocks
that a bound on their keys selects: Python front-end of include/dance_kv.h.

    cache = KVCache.empty(blocks, kv_heads, dim, block_tokens=64)
    append(cache, k, v, table, lengths)                      # a step's or a prompt's tokens
    o = attention(cache, q, table, lengths)                  # over all tokens
    chosen = select(cache, q, table, lengths, 64, sink=1, recent=2)
    o = sparse_attention(cache, q, chosen, table, lengths)   # over 64 blocks a query

Arguments that all calls share:
    table    [sequences, blocks] int32: the cache block of each part of a
             sequence; entries outside the cache are holes
    lengths  [sequences] int32: the sequences' tokens, this call's included
    offsets  [sequences + 1] int32: a sequence's token rows are offsets[b] up to
             offsets[b + 1]; None: one row for each sequence
    max_tokens   the most rows of a sequence, on the host (default: all rows)
    max_length   the longest length, on the host (default: the table's width)
Rows are [tokens, heads, dim] in float16 or bfloat16 with adjacent dimensions.
Row i of a sequence's n stands at position length - n + i and sees the
positions up to its own.

The calls run on torch's current stream, wait for nothing and can be captured
into a graph. As with any torch call, tensors made on another stream have to be
ready on this one. Outputs of rows beyond the last offset are undefined. There
are no gradients (codes are for serving) and no CPU path.
"""
from __future__ import annotations

import ctypes as C
import struct

import torch

from . import lib as _lib

DTYPES = {torch.float16: 2, torch.bfloat16: 3}
DIMS = (64, 96, 128, 192, 256)
BLOCK_TOKENS = (16, 32, 64, 128)


class DanceKvCache(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("scale", C.c_void_p), ("bound", C.c_void_p),
                ("blocks", C.c_uint32), ("kv_heads", C.c_uint32), ("dim", C.c_uint32), ("block_tokens", C.c_uint32)]


class DanceKvBatch(C.Structure):
    _fields_ = [("table", C.c_void_p), ("lengths", C.c_void_p), ("offsets", C.c_void_p), ("seqs", C.c_uint32),
                ("tokens", C.c_uint32), ("table_width", C.c_uint32), ("max_tokens", C.c_uint32),
                ("max_length", C.c_uint64)]


class DanceKvRows(C.Structure):
    _fields_ = [("data", C.c_void_p), ("token_stride", C.c_int64), ("head_stride", C.c_int64), ("heads", C.c_uint32),
                ("dtype", C.c_int)]


# The same structs as bytes, which a call takes as it takes a pointer: a small
# attention is 8 us of host time, and the three ctypes objects would be another 1.5.
_CACHE, _BATCH, _ROWS = struct.Struct("@PPPPIIII"), struct.Struct("@PPPIIIIQ"), struct.Struct("@PqqIi")
assert [_CACHE.size, _BATCH.size, _ROWS.size] == [C.sizeof(t) for t in (DanceKvCache, DanceKvBatch, DanceKvRows)]

# torch's handle of the current stream, without the Stream object around it where torch has that
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_bound = None
_fast = {}


def _stream(index):
    return _raw_stream(index) if _raw_stream else torch.cuda.current_stream(index).cuda_stream


def _bind():
    global _bound
    if _bound is None:
        L = _lib()
        vp, u32, f32, sz = C.c_void_p, C.c_uint32, C.c_float, C.c_size_t
        cache, batch, rows = C.POINTER(DanceKvCache), C.POINTER(DanceKvBatch), C.POINTER(DanceKvRows)
        for name, args, res in (
                ("append", [cache, batch, rows, rows, vp], C.c_int),
                ("attention", [cache, batch, rows, f32, vp, vp, vp, sz, vp], C.c_int),
                ("attention_work", [cache, batch, u32], sz),
                ("select", [cache, batch, rows, u32, u32, u32, vp, vp, sz, vp], C.c_int),
                ("select_work", [cache, batch, u32, u32], sz),
                ("sparse_attention", [cache, batch, rows, vp, u32, f32, vp, vp, vp, sz, vp], C.c_int),
                ("sparse_attention_work", [cache, batch, u32, u32], sz)):
            fn = getattr(L, "dance_kv_" + name)
            fn.argtypes, fn.restype = args, res
            as_bytes = [C.c_char_p if t in (cache, batch, rows) else t for t in args]
            _fast[name] = C.CFUNCTYPE(res, *as_bytes)(("dance_kv_" + name, L))
        _bound = L
    return _bound


class KVCache:
    """The cache's four arrays:
        k     [blocks, kv_heads, block_tokens, dim] int8   codes of the keys
        v     [blocks, kv_heads, dim, block_tokens] int8   codes of the values
        scale [blocks, kv_heads, 2] float32                a key is k * scale[0], a value v * scale[1]
        bound [blocks, kv_heads, 2, dim] int8              largest and least key code of a block
    """

    def __init__(self, k, v, scale, bound):
        for name, t, dtype, nd in (("k", k, torch.int8, 4), ("v", v, torch.int8, 4), ("scale", scale, torch.float32, 3),
                                   ("bound", bound, torch.int8, 4)):
            if t.dtype != dtype or t.ndim != nd:
                raise TypeError(f"{name} must be a {nd}-dimensional {dtype} tensor")
            if not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
            if t.device != k.device:
                raise ValueError("the cache's arrays must be on one device")
        blocks, heads, block_tokens, dim = k.shape
        if (v.shape != (blocks, heads, dim, block_tokens) or scale.shape != (blocks, heads, 2)
                or bound.shape != (blocks, heads, 2, dim)):
            raise ValueError("the cache's arrays do not fit together")
        if dim not in DIMS or block_tokens not in BLOCK_TOKENS:
            raise ValueError(f"dim must be one of {DIMS} and block_tokens one of {BLOCK_TOKENS}")
        if blocks < 1 or heads < 1:
            raise ValueError("a cache has at least one block and one head")
        if k.device.type != "cuda":
            raise ValueError("the cache must be in GPU memory")
        self.k, self.v, self.scale, self.bound = k, v, scale, bound
        self.blocks, self.kv_heads, self.block_tokens, self.dim = blocks, heads, block_tokens, dim
        self.device = k.device
        self._bytes = _CACHE.pack(k.data_ptr(), v.data_ptr(), scale.data_ptr(), bound.data_ptr(), blocks, heads, dim,
                                  block_tokens)
        _bind()

    @classmethod
    def empty(cls, blocks, kv_heads, dim, block_tokens=64, device="cuda"):
        """A cache whose blocks hold nothing yet: append fills them."""
        def make(shape, dtype):
            return torch.zeros(shape, dtype=dtype, device=device)
        return cls(make((blocks, kv_heads, block_tokens, dim), torch.int8),
                   make((blocks, kv_heads, dim, block_tokens), torch.int8), make((blocks, kv_heads, 2), torch.float32),
                   make((blocks, kv_heads, 2, dim), torch.int8))


def _ints(name, t, shape, device):
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32")
    if t.shape != shape:
        raise ValueError(f"{name} must have the shape {tuple(shape)}")
    if t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous and on the cache's device")


def _rows(cache, name, t, heads=None):
    """Checks rows of keys, values or queries; (their struct's bytes, tokens, heads)."""
    shape = t.shape
    if len(shape) != 3 or shape[2] != cache.dim:
        raise ValueError(f"{name} must be [tokens, heads, {cache.dim}]")
    dtype = DTYPES.get(t.dtype)
    if dtype is None:
        raise TypeError(f"{name} must be float16 or bfloat16")
    if t.device != cache.device:
        raise ValueError(f"{name} must be on the cache's device")
    token_stride, head_stride, one = t.stride()
    if one != 1:
        raise ValueError(f"the dimensions of {name} must be adjacent")
    tokens, n, _ = shape
    if n != heads if heads else n == 0 or n % cache.kv_heads:
        raise ValueError(f"{name} must have {heads} heads" if heads else
                         f"{name} must have a multiple of {cache.kv_heads} heads")
    return _ROWS.pack(t.data_ptr(), token_stride, head_stride, n, dtype), tokens, n


def _batch(cache, tokens, table, lengths, offsets, max_tokens, max_length):
    """Checks a batch; its struct's bytes."""
    shape = table.shape
    if len(shape) != 2:
        raise ValueError("table must be [sequences, blocks]")
    seqs, width = shape
    _ints("table", table, shape, cache.device)
    _ints("lengths", lengths, (seqs,), cache.device)
    if offsets is None:
        if tokens != seqs:
            raise ValueError("without offsets there is one row for each sequence")
        max_tokens, at = 1, 0
    else:
        _ints("offsets", offsets, (seqs + 1,), cache.device)
        if max_tokens is None:
            max_tokens = tokens
        elif max_tokens < 1:
            raise ValueError("max_tokens must be positive")
        at = offsets.data_ptr()
    if max_length is not None and max_length < 1:
        raise ValueError("max_length must be positive")
    return _BATCH.pack(table.data_ptr(), lengths.data_ptr(), at, seqs, tokens, width, min(max_tokens, tokens),
                       max_length or 0)


def _call(name, cache, *args):
    index = cache.device.index
    if torch.cuda.current_device() != index:
        with torch.cuda.device(index):
            rc = _fast[name](cache._bytes, *args, _stream(index))
    else:
        rc = _fast[name](cache._bytes, *args, _stream(index))
    if rc != 0:
        raise RuntimeError(f"dance_kv_{name} failed with return code {rc}")


def _work(cache, size):
    return torch.empty(size, dtype=torch.uint8, device=cache.device) if size else None


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _out(t, q):
    if t is None:
        return torch.empty_like(q, memory_format=torch.contiguous_format)
    if t.shape != q.shape or t.dtype != q.dtype or t.device != q.device or not t.is_contiguous():
        raise ValueError(f"out must be a contiguous {q.dtype} tensor of q's shape on the cache's device")
    return t


def append(cache, k, v, table, lengths, offsets=None, max_tokens=None):
    """Writes the rows' keys and values into the cache's blocks; scales and bounds follow."""
    kr, tokens, _ = _rows(cache, "k", k, cache.kv_heads)
    vr, others, _ = _rows(cache, "v", v, cache.kv_heads)
    if tokens != others or k.dtype != v.dtype:
        raise ValueError("k and v must have one shape and type")
    b = _batch(cache, tokens, table, lengths, offsets, max_tokens, None)
    if tokens:
        _call("append", cache, b, kr, vr)


def attention(cache, q, table, lengths, offsets=None, *, scale=None, max_tokens=None, max_length=None, out=None,
              return_lse=False):
    """Softmax attention of the rows over their sequences' tokens: [tokens, heads,
    dim] of q's type. With return_lse also the logarithm of each row's sum
    [tokens, heads] in float32. Rows that see nothing give zeros and -inf.
    scale defaults to dim ** -0.5."""
    r, tokens, heads = _rows(cache, "q", q)
    b = _batch(cache, tokens, table, lengths, offsets, max_tokens, max_length)
    out = _out(out, q)
    lse = torch.empty((tokens, heads), dtype=torch.float32, device=cache.device) if return_lse else None
    if tokens:
        size = _fast["attention_work"](cache._bytes, b, heads)
        work = _work(cache, size)
        _call("attention", cache, b, r, cache.dim ** -0.5 if scale is None else scale, out.data_ptr(), _ptr(lse),
              _ptr(work), size)
    return (out, lse) if return_lse else out


def select(cache, q, table, lengths, count, offsets=None, *, sink=0, recent=0, max_tokens=None, max_length=None):
    """The `count` blocks of each row and kv head whose keys may have the largest
    products with the head group's queries, by an upper bound that 8-bit codes
    of the queries give exactly: [tokens, kv_heads, count] int32, logical blocks
    in ascending order, -1 behind them. Equal bounds go to the lower block. The
    first `sink` and the last `recent` blocks that a row sees are always among
    them."""
    r, tokens, heads = _rows(cache, "q", q)
    b = _batch(cache, tokens, table, lengths, offsets, max_tokens, max_length)
    if count < 1 or sink < 0 or recent < 0 or sink + recent > count:
        raise ValueError("count must be positive and hold sink and recent")
    chosen = torch.empty((tokens, cache.kv_heads, count), dtype=torch.int32, device=cache.device)
    if tokens:
        size = _fast["select_work"](cache._bytes, b, heads, count)
        work = _work(cache, size)
        _call("select", cache, b, r, count, sink, recent, chosen.data_ptr(), _ptr(work), size)
    return chosen


def sparse_attention(cache, q, chosen, table, lengths, offsets=None, *, scale=None, max_tokens=None, out=None,
                     return_lse=False):
    """attention over the blocks that `chosen` [tokens, kv_heads, count] int32 lists
    for each row and kv head: logical blocks in any order, each at most once;
    negative ones and those the row does not see are left out."""
    r, tokens, heads = _rows(cache, "q", q)
    b = _batch(cache, tokens, table, lengths, offsets, max_tokens, None)
    if chosen.ndim != 3 or chosen.shape[2] < 1:
        raise ValueError("chosen must be [tokens, kv_heads, count]")
    count = chosen.shape[2]
    _ints("chosen", chosen, (tokens, cache.kv_heads, count), cache.device)
    out = _out(out, q)
    lse = torch.empty((tokens, heads), dtype=torch.float32, device=cache.device) if return_lse else None
    if tokens:
        size = _fast["sparse_attention_work"](cache._bytes, b, heads, count)
        work = _work(cache, size)
        _call("sparse_attention", cache, b, r, chosen.data_ptr(), count, cache.dim ** -0.5 if scale is None else scale,
              out.data_ptr(), _ptr(lse), _ptr(work), size)
    return (out, lse) if return_lse else out
