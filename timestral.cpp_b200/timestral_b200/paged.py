"""Attention over a paged cache on caller-owned device arrays (tsb_norm_rope, tsb_paged_append
and tsb_paged_attention of include/timestral_b200.h, which documents what each computes).

The arrays are objects with data_ptr(), stride(), shape and dtype on the current device, such as
torch tensors; this module does not import torch. Results go into arrays the caller gives; a
call enqueues its kernels on `stream` (a cudaStream_t as an integer, 0: the legacy default
stream) and returns. The arrays must live until that work is done."""
from __future__ import annotations

import ctypes as C

from . import (Heads, NormRopeArgs, PagedAppendArgs, PagedAttentionArgs, PagedBatchArgs, PagedCacheArgs, Rotation,
               TimestralError, lib)

_TYPES = {}          # dtype object -> GGUF type number (0: not a value type of these operators)
_WANTED = {"float16": 1, "bfloat16": 30}


def _type(a, name):
    t = _TYPES.get(a.dtype)
    if t is None:
        t = _TYPES[a.dtype] = _WANTED.get(str(a.dtype).rsplit(".", 1)[-1], 0)
    if not t:
        raise TimestralError(f"{name} is {a.dtype}, not float16 or bfloat16")
    return t


def _of(a, name, kind):
    """The address of an index, bit, weight or table array of the given kind, checked to be dense
    along its last axis."""
    if not str(a.dtype).endswith(kind):
        raise TimestralError(f"{name} is {a.dtype}, not {kind}")
    if a.stride()[-1] != 1 and a.shape[-1] > 1:
        raise TimestralError(f"{name} is strided along its last axis")
    return a.data_ptr()


def _vector(a, name, kind, length):
    if a is None:
        return None
    if len(a.shape) != 1 or a.shape[0] != length:
        raise TimestralError(f"{name} has shape {tuple(a.shape)}, not ({length},)")
    return _of(a, name, kind)


def _heads(a, name, want_type, shape):
    """The C view of a [tokens, heads, head_dim] array."""
    if _type(a, name) != want_type:
        raise TimestralError(f"{name} is {a.dtype}, unlike the other arrays")
    got = a.shape
    if len(got) != 3 or got[0] != shape[0] or got[1] != shape[1] or got[2] != shape[2]:
        raise TimestralError(f"{name} has shape {tuple(got)}, not {tuple(shape)}")
    token, head, last = a.stride()
    if last != 1:
        raise TimestralError(f"{name} is strided along its last axis")
    return Heads(a.data_ptr(), token, head if shape[1] > 1 else 0)


def _rotation(cos, sin, positions, tokens):
    if cos is None and sin is None:
        return Rotation()
    if cos is None or sin is None:
        raise TimestralError("one of cos and sin is missing")
    if cos.shape != sin.shape or cos.stride() != sin.stride() or len(cos.shape) != 2:
        raise TimestralError("cos and sin are not two [positions, rope_dim / 2] tables alike")
    if cos.shape[0] == 0 or cos.shape[1] == 0:       # their address would be NULL, which means no rotation
        raise TimestralError(f"the rotation tables have {cos.shape[0]} rows of {cos.shape[1]}")
    return Rotation(_of(cos, "cos", "float32"), _of(sin, "sin", "float32"), cos.stride()[0], cos.shape[0], 2 * cos.shape[1],
                    _vector(positions, "positions", "int32", tokens))


def _run(rc, name):
    if rc != 0:
        raise TimestralError(f"{name} failed ({rc}): {lib().timestral_capi_last_error(None).decode()}")


class PagedCache:
    """Pages of keys and values, k and v [pages, kv_heads, page_size, head_dim] with any strides
    (head_dim contiguous), and table [sequences, entries] int32: the page of position p of
    sequence s is table[s, p // page_size]."""

    def __init__(self, k, v, table):
        if len(k.shape) != 4 or k.shape != v.shape:
            raise TimestralError(f"k {tuple(k.shape)} and v {tuple(v.shape)} are not [pages, heads, page_size, head_dim] alike")
        if len(table.shape) != 2:
            raise TimestralError(f"table has shape {tuple(table.shape)}, not [sequences, entries]")
        kind = _type(k, "k")
        if _type(v, "v") != kind:
            raise TimestralError("k and v have different types")
        ks, vs = k.stride(), v.stride()
        if ks[3] != 1 or vs[3] != 1:
            raise TimestralError("the cache is strided along its last axis")
        pages, heads, slots, dim = k.shape
        self.arrays = (k, v, table)
        self.kind, self.heads, self.head_dim, self.sequences = kind, heads, dim, table.shape[0]
        self.args = PagedCacheArgs(k.data_ptr(), v.data_ptr(), ks[0], ks[1] if heads > 1 else 0, ks[2], vs[0],
                                   vs[1] if heads > 1 else 0, vs[2], _of(table, "table", "int32"), table.stride()[0],
                                   table.shape[1], kind, pages, slots, heads, dim)


class PagedBatch:
    """The new tokens of each sequence: q_start [sequences + 1] and lengths [sequences] int32 on the
    device, lengths counting the new tokens, and bounds of both that hold for every sequence."""

    def __init__(self, q_start, lengths, max_chunk, max_length):
        n = lengths.shape[0]
        self.arrays = (q_start, lengths)
        self.sequences = n
        self.args = PagedBatchArgs(_vector(q_start, "q_start", "int32", n + 1), _vector(lengths, "lengths", "int32", n), n,
                                   max_chunk, max_length)


def _together(cache, batch):
    if batch.sequences > cache.sequences:
        raise TimestralError(f"the batch has {batch.sequences} sequences, the cache's table {cache.sequences}")


def norm_rope(q, q_out, k=None, k_out=None, *, q_weight=None, k_weight=None, eps=1e-6, cos=None, sin=None, positions=None,
              error=None, stream=0):
    """RMS norm of every head of q (and k) with its weight [head_dim] f32 (None: no norm), then the
    rotation by cos/sin [positions, rope_dim / 2] f32 at positions [tokens] int32 (None: no
    rotation). q_out may be q, k_out may be k."""
    tokens, heads, dim = q.shape
    kind = _type(q, "q")
    a = NormRopeArgs(kind, tokens, dim, heads, 0, eps, _heads(q, "q", kind, q.shape), _heads(q_out, "q_out", kind, q.shape))
    if k is not None:
        shape = (tokens, k.shape[1], dim)
        a.k_heads, a.k, a.k_out = shape[1], _heads(k, "k", kind, shape), _heads(k_out, "k_out", kind, shape)
    a.q_weight, a.k_weight = _vector(q_weight, "q_weight", "float32", dim), _vector(k_weight, "k_weight", "float32", dim)
    a.rotation = _rotation(cos, sin, positions, tokens)
    if error is not None:
        a.error = _vector(error, "error", "int32", 1)
    _run(lib().tsb_norm_rope(C.byref(a), stream), "tsb_norm_rope")


def paged_append(cache, batch, k, v, *, k_weight=None, eps=1e-6, cos=None, sin=None, positions=None, error=None, stream=0):
    """Write k and v [tokens, kv_heads, head_dim] at the new tokens' positions of the cache, k normed
    with k_weight and rotated on the way as norm_rope does (positions None: the positions in the
    cache)."""
    _together(cache, batch)
    shape = (k.shape[0], cache.heads, cache.head_dim)
    a = PagedAppendArgs(C.pointer(cache.args), C.pointer(batch.args), _heads(k, "k", cache.kind, shape),
                        _heads(v, "v", cache.kind, shape), shape[0], eps, _vector(k_weight, "k_weight", "float32", shape[2]),
                        _rotation(cos, sin, positions, shape[0]))
    if error is not None:
        a.error = _vector(error, "error", "int32", 1)
    _run(lib().tsb_paged_append(C.byref(a), stream), "tsb_paged_append")


def paged_attention(cache, batch, q, out, *, scale=0.0, window=0, key_valid=None, key_valid_positions=None, self_visible=False,
                    gate=None, workspace=None, error=None, stream=0):
    """out = gate * attention of q [tokens, q_heads, head_dim] over the cache. key_valid
    [sequences, words] int32: bit p % 32 of word p // 32 says whether position p may be seen, for the
    first key_valid_positions positions (None: all the bits there are). workspace: any dense
    device array; its bytes bound how far the keys are split."""
    _together(cache, batch)
    shape = q.shape
    if len(shape) != 3 or shape[2] != cache.head_dim:
        raise TimestralError(f"q has shape {tuple(shape)}, not [tokens, heads, {cache.head_dim}]")
    a = PagedAttentionArgs(C.pointer(cache.args), C.pointer(batch.args), _heads(q, "q", cache.kind, shape),
                           _heads(out, "out", cache.kind, shape))
    a.tokens, a.q_heads, a.window, a.self_visible, a.scale = shape[0], shape[1], window, bool(self_visible), scale
    if gate is not None:
        a.gate = _heads(gate, "gate", cache.kind, shape)
    if key_valid is not None:
        if len(key_valid.shape) != 2 or key_valid.shape[0] < batch.sequences:
            raise TimestralError(f"key_valid has shape {tuple(key_valid.shape)}, not [{batch.sequences}, words]")
        words = key_valid.shape[1]
        a.key_valid, a.key_valid_stride = _of(key_valid, "key_valid", "int32"), key_valid.stride()[0]
        a.key_valid_positions = 32 * words if key_valid_positions is None else key_valid_positions
        if not 0 <= a.key_valid_positions <= 32 * words:
            raise TimestralError(f"key_valid holds {32 * words} bits, not {key_valid_positions}")
    if workspace is not None:
        if not workspace.is_contiguous():
            raise TimestralError("workspace is not dense")
        a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    if error is not None:
        a.error = _vector(error, "error", "int32", 1)
    _run(lib().tsb_paged_attention(C.byref(a), stream), "tsb_paged_attention")


def paged_attention_workspace(cache, batch, tokens, q_heads, window=0) -> int:
    """Bytes of workspace with which paged_attention splits the keys as far as it would like to."""
    _together(cache, batch)
    a = PagedAttentionArgs(C.pointer(cache.args), C.pointer(batch.args))
    a.tokens, a.q_heads, a.window = tokens, q_heads, window
    return lib().tsb_paged_attention_workspace(C.byref(a))
