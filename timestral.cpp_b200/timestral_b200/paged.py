"""Attention over a paged cache on caller-owned device arrays (tsb_norm_rope, tsb_paged_append
and tsb_paged_attention of include/timestral_b200.h, which documents what each computes).

The arrays are objects with data_ptr(), stride(), shape and dtype on the current device, such as
torch tensors; this module does not import torch. Results go into arrays the caller gives; a
call enqueues its kernels on `stream` (a cudaStream_t as an integer, 0: the legacy default
stream) and returns. The arrays must live until that work is done.

A decoded token's calls are small, so what stands between them and the launch is kept short: each
array is looked at once, and the C structures (NormRopeArgs and the others of the package) are
packed by struct in one go."""
from __future__ import annotations

import ctypes as C
import struct

from . import PagedAppendArgs, PagedAttentionArgs, PagedBatchArgs, PagedCacheArgs, NormRopeArgs, TimestralError, lib

_HEADS = "Pqq"
_ROTATION = "PPqiiP"
_NORM_ROPE = struct.Struct("@5if" + 4 * _HEADS + "PP" + _ROTATION + "P")
_APPEND = struct.Struct("@PP" + 2 * _HEADS + "ifP" + _ROTATION + "P")
_ATTENTION = struct.Struct("@PP" + 3 * _HEADS + "4ifiPqPNP")
for _s, _c in ((_NORM_ROPE, NormRopeArgs), (_APPEND, PagedAppendArgs), (_ATTENTION, PagedAttentionArgs)):
    assert _s.size == C.sizeof(_c), (_s.size, C.sizeof(_c))
_NO_HEADS = (0, 0, 0)
_NO_ROTATION = (0, 0, 0, 0, 0, 0)

# What a dtype is: (GGUF type number or 0, name), by the dtype object.
_KINDS = {}
_VALUES = {"float16": 1, "bfloat16": 30}


def _kind(dtype):
    k = _KINDS.get(dtype)
    if k is None:
        name = str(dtype).rsplit(".", 1)[-1]
        k = _KINDS[dtype] = (_VALUES.get(name, 0), name)
    return k


def _type(a, name):
    t = _kind(a.dtype)[0]
    if not t:
        raise TimestralError(f"{name} is {a.dtype}, not float16 or bfloat16")
    return t


def _heads(a, name, dtype, shape):
    """The C view (address, token and head stride) of a [tokens, heads, head_dim] array."""
    if a.dtype != dtype:
        raise TimestralError(f"{name} is {a.dtype}, unlike the other arrays")
    if a.shape != shape:
        raise TimestralError(f"{name} has shape {tuple(a.shape)}, not {tuple(shape)}")
    token, head, last = a.stride()
    if last != 1:
        raise TimestralError(f"{name} is strided along its last axis")
    return a.data_ptr(), token, head if shape[1] > 1 else 0


def _vector(a, name, kind, length):
    """The address of a dense vector of the given type and length, 0 for None."""
    if a is None:
        return 0
    if _kind(a.dtype)[1] != kind:
        raise TimestralError(f"{name} is {a.dtype}, not {kind}")
    if a.shape != (length,):
        raise TimestralError(f"{name} has shape {tuple(a.shape)}, not ({length},)")
    if length > 1 and a.stride() != (1,):
        raise TimestralError(f"{name} is strided")
    return a.data_ptr()


def _matrix(a, name, kind):
    """(address, rows, columns, row stride) of a matrix whose rows are dense."""
    if _kind(a.dtype)[1] != kind:
        raise TimestralError(f"{name} is {a.dtype}, not {kind}")
    if len(a.shape) != 2:
        raise TimestralError(f"{name} has shape {tuple(a.shape)}, not [rows, entries]")
    rows, columns = a.shape
    stride, last = a.stride()
    if last != 1 and columns > 1:
        raise TimestralError(f"{name} is strided along its last axis")
    return a.data_ptr(), rows, columns, stride


def _rotation(cos, sin, positions, tokens):
    if cos is None and sin is None:
        return _NO_ROTATION
    if cos is None or sin is None:
        raise TimestralError("one of cos and sin is missing")
    c, s = _matrix(cos, "cos", "float32"), _matrix(sin, "sin", "float32")
    if c[1:] != s[1:]:
        raise TimestralError("cos and sin are not two [positions, rope_dim / 2] tables alike")
    at, rows, half, stride = c
    if rows == 0 or half == 0:                        # their address would be NULL, which means no rotation
        raise TimestralError(f"the rotation tables have {rows} rows of {half}")
    return at, s[0], stride, rows, 2 * half, _vector(positions, "positions", "int32", tokens)


def _run(rc, name):
    if rc != 0:
        raise TimestralError(f"{name} failed ({rc}): {lib().timestral_capi_last_error(None).decode()}")


class PagedCache:
    """Pages of keys and values, k and v [pages, kv_heads, page_size, head_dim] with any strides
    (head_dim contiguous), and table [sequences, entries] int32: the page of position p of
    sequence s is table[s, p // page_size]."""

    __slots__ = ("arrays", "dtype", "heads", "head_dim", "sequences", "args", "address")

    def __init__(self, k, v, table):
        shape = k.shape
        if len(shape) != 4 or v.shape != shape:
            raise TimestralError(f"k {tuple(k.shape)} and v {tuple(v.shape)} are not [pages, heads, page_size, head_dim] alike")
        kind = _type(k, "k")
        if v.dtype != k.dtype:
            raise TimestralError("k and v have different types")
        ks, vs = k.stride(), v.stride()
        if ks[3] != 1 or vs[3] != 1:
            raise TimestralError("the cache is strided along its last axis")
        pages, heads, slots, dim = shape
        at, rows, entries, stride = _matrix(table, "table", "int32")
        self.arrays = (k, v, table)
        self.dtype, self.heads, self.head_dim, self.sequences = k.dtype, heads, dim, rows
        self.args = PagedCacheArgs(k.data_ptr(), v.data_ptr(), ks[0], ks[1] if heads > 1 else 0, ks[2], vs[0],
                                   vs[1] if heads > 1 else 0, vs[2], at, stride, entries, kind, pages, slots, heads, dim)
        self.address = C.addressof(self.args)


class PagedBatch:
    """The new tokens of each sequence: q_start [sequences + 1] and lengths [sequences] int32 on the
    device, lengths counting the new tokens, and bounds of both that hold for every sequence."""

    __slots__ = ("arrays", "sequences", "args", "address")

    def __init__(self, q_start, lengths, max_chunk, max_length):
        n = lengths.shape[0]
        if max_chunk >= 2 ** 31 or max_length >= 2 ** 31:          # a C int would take them for something else
            raise TimestralError(f"max_chunk {max_chunk} or max_length {max_length} is above 2^31 - 1")
        self.arrays = (q_start, lengths)
        self.sequences = n
        self.args = PagedBatchArgs(_vector(q_start, "q_start", "int32", n + 1), _vector(lengths, "lengths", "int32", n), n,
                                   max_chunk, max_length)
        self.address = C.addressof(self.args)


def _together(cache, batch):
    if batch.sequences > cache.sequences:
        raise TimestralError(f"the batch has {batch.sequences} sequences, the cache's table {cache.sequences}")


def norm_rope(q, q_out, k=None, k_out=None, *, q_weight=None, k_weight=None, eps=1e-6, cos=None, sin=None, positions=None,
              error=None, stream=0):
    """RMS norm of every head of q (and k) with its weight [head_dim] f32 (None: no norm), then the
    rotation by cos/sin [positions, rope_dim / 2] f32 at positions [tokens] int32 (None: no
    rotation). q_out may be q, k_out may be k."""
    shape, dtype = q.shape, q.dtype
    if len(shape) != 3:
        raise TimestralError(f"q has shape {tuple(shape)}, not [tokens, heads, head_dim]")
    tokens, heads, dim = shape
    k_heads, k_view, k_to = 0, _NO_HEADS, _NO_HEADS
    if k is not None:
        k_shape = k.shape
        if len(k_shape) != 3 or k_shape[0] != tokens or k_shape[2] != dim:
            raise TimestralError(f"k has shape {tuple(k_shape)}, not [{tokens}, heads, {dim}]")
        if k_out is None:
            raise TimestralError("k_out is missing")
        k_heads, k_view, k_to = k_shape[1], _heads(k, "k", dtype, k_shape), _heads(k_out, "k_out", dtype, k_shape)
    a = _NORM_ROPE.pack(_type(q, "q"), tokens, dim, heads, k_heads, eps, *_heads(q, "q", dtype, shape),
                        *_heads(q_out, "q_out", dtype, shape), *k_view, *k_to, _vector(q_weight, "q_weight", "float32", dim),
                        _vector(k_weight, "k_weight", "float32", dim), *_rotation(cos, sin, positions, tokens),
                        0 if error is None else _vector(error, "error", "int32", 1))
    _run(lib().tsb_norm_rope(a, stream), "tsb_norm_rope")


def paged_append(cache, batch, k, v, *, k_weight=None, eps=1e-6, cos=None, sin=None, positions=None, error=None, stream=0):
    """Write k and v [tokens, kv_heads, head_dim] at the new tokens' positions of the cache, k normed
    with k_weight and rotated on the way as norm_rope does (positions None: the positions in the
    cache)."""
    _together(cache, batch)
    tokens, dim, dtype = k.shape[0], cache.head_dim, cache.dtype
    shape = (tokens, cache.heads, dim)
    a = _APPEND.pack(cache.address, batch.address, *_heads(k, "k", dtype, shape), *_heads(v, "v", dtype, shape), tokens, eps,
                     _vector(k_weight, "k_weight", "float32", dim), *_rotation(cos, sin, positions, tokens),
                     0 if error is None else _vector(error, "error", "int32", 1))
    _run(lib().tsb_paged_append(a, stream), "tsb_paged_append")


def paged_attention(cache, batch, q, out, *, scale=0.0, window=0, key_valid=None, key_valid_positions=None, self_visible=False,
                    gate=None, workspace=None, error=None, stream=0):
    """out = gate * attention of q [tokens, q_heads, head_dim] over the cache. key_valid
    [sequences, words] int32: bit p % 32 of word p // 32 says whether position p may be seen, for the
    first key_valid_positions positions (None: all the bits there are). workspace: any dense
    device array; its bytes bound how far the keys are split."""
    _together(cache, batch)
    shape, dtype = q.shape, cache.dtype
    if len(shape) != 3 or shape[2] != cache.head_dim:
        raise TimestralError(f"q has shape {tuple(shape)}, not [tokens, heads, {cache.head_dim}]")
    bits_at = bits = bits_stride = 0
    if key_valid is not None:
        bits_at, rows, words, bits_stride = _matrix(key_valid, "key_valid", "int32")
        if rows < batch.sequences:
            raise TimestralError(f"key_valid has shape {tuple(key_valid.shape)}, not [{batch.sequences}, words]")
        bits = 32 * words if key_valid_positions is None else key_valid_positions
        if not 0 <= bits <= 32 * words:
            raise TimestralError(f"key_valid holds {32 * words} bits, not {key_valid_positions}")
    space = held = 0
    if workspace is not None:
        if not workspace.is_contiguous():
            raise TimestralError("workspace is not dense")
        space, held = workspace.data_ptr(), workspace.nbytes
    a = _ATTENTION.pack(cache.address, batch.address, *_heads(q, "q", dtype, shape), *_heads(out, "out", dtype, shape),
                        *(_NO_HEADS if gate is None else _heads(gate, "gate", dtype, shape)), shape[0], shape[1], window,
                        bool(self_visible), scale, bits, bits_at, bits_stride, space, held,
                        0 if error is None else _vector(error, "error", "int32", 1))
    _run(lib().tsb_paged_attention(a, stream), "tsb_paged_attention")


def paged_attention_workspace(cache, batch, tokens, q_heads, window=0) -> int:
    """Bytes of workspace with which paged_attention splits the keys as far as it would like to."""
    _together(cache, batch)
    a = _ATTENTION.pack(cache.address, batch.address, *_NO_HEADS, *_NO_HEADS, *_NO_HEADS, tokens, q_heads, window, 0, 0.0, 0, 0, 0,
                        0, 0, 0)
    return lib().tsb_paged_attention_workspace(a)
