"""Attention over a paged cache of keys and values, next to the search over its keys.

A decoder keeps the keys and values of its tokens in pages and reaches back over a context that is too long to be read in full by a
search over the keys.  A step of several sequences, one token each, then is::

    slots, q = kv_cache.append(keys, values, new_keys, new_values, pages, positions, queries=queries, frequencies=frequencies)
    near = kv_cache.attention(keys, values, q, pages, lengths, window=window)
    # index[i][h]: over the keys of sequence i and key head h before the window, in float32, whose source ids are slots
    own = q.float().unflatten(1, (n_heads, -1))
    candidates = torch.stack([torch.cat([ivf_pq.search(params, index[i][h], own[i, h], k)[1] for h in range(n_heads)])
                              for i in range(len(own))])
    far = kv_cache.attend_candidates(keys, values, q, candidates)               # [n_sequences, n_query_heads, k]
    out, lse = kv_cache.merge_parts(torch.stack((near[0], far[0])), torch.stack((near[1], far[1])))

An index that several sequences share would name slots of all of them for each: :func:`attend_candidates` attends to whatever a list names.

``keys`` and ``values`` are ``[n_pages, page_size, n_heads, dim]`` tensors of float16, bfloat16 or float32, of any strides that leave the
rows of ``dim`` elements contiguous and on 16-byte boundaries.  A token's slot is ``page * page_size + place``, and is the id under which
its key is put into an index.  ``pages`` (int32 ``[n_sequences, width]``) names the pages of each sequence in the order of its positions;
an entry that is no page of the cache, such as -1, holds no tokens.  Query head ``i`` reads the rows of head
``i // (n_query_heads // n_heads)``.  Softmax and sums are held in 32 bits, outputs are rounded once; where nothing may be attended to, the
output is 0 and its ``lse`` is -inf.  Weights below 2^-100 of the largest may count as 0, in :func:`attention` over float16 those below 2^-38
(times an infinite value that is no number).

These calls serve: they have no gradients.  They enqueue their work on the stream of ``resources`` (torch's current stream by default) and
wait for it unless ``sync=False``, which is what a captured call needs.
"""
from __future__ import annotations

import ctypes as C
import functools
import operator
import struct

import torch

from . import _lib as L
from .common import Resources, _default_resources, default_resources

# ndim | dtype code << 32 | bits << 40 | lanes << 48
_WORD = {t: (code << 32) | (bits << 40) | (1 << 48)
         for t, code, bits in ((torch.float16, 2, 16), (torch.bfloat16, 4, 16), (torch.float32, 2, 32), (torch.float64, 2, 64),
                               (torch.int32, 0, 32), (torch.int64, 0, 64), (torch.uint32, 1, 32), (torch.uint8, 1, 8))}
_APPEND, _ATTENTION, _CANDIDATES, _MERGE = range(4)
_f32 = struct.Struct("<f")
_u32 = struct.Struct("<I")


def _words(tensors, scalars):
    """The words that describe a call's tensors (the order of the C interface) and its scalars, and how many they are.  One array of
    integers for all of them: a descriptor structure for each took longer than the kernels of a small call."""
    words = []
    for t in tensors:
        if t is None:
            words.append(0)
            continue
        shape, word, at = t.shape, _WORD.get(t.dtype), t.get_device()
        if word is None:
            raise ValueError(f"unsupported element type {t.dtype}")
        if not 1 <= len(shape) <= 4:
            raise ValueError(f"tensors have 1 to 4 dimensions, not {len(shape)}")
        words += (word | len(shape), t.data_ptr(), (at << 32) | L.kDLCUDA if at >= 0 else L.kDLCPU, *shape, *t.stride())
    words += scalars
    n = len(words)
    return _packer(n).pack(*words), n


@functools.lru_cache(maxsize=256)
def _packer(n):
    return struct.Struct(f"{n}q")


def _bits(scale):
    return _u32.unpack(_f32.pack(scale))[0]


def _handle(tensor, resources):
    """The handle for a call on this tensor's device, and its stream."""
    device = tensor.get_device() if isinstance(tensor, torch.Tensor) else -1
    if device < 0:
        raise ValueError("expected CUDA tensors")
    if resources is None:
        resources = _default_resources.get(device)
        if resources is None:
            with torch.cuda.device(device):
                resources = default_resources(device)
    return resources, resources.stream_at_call(device)


def _window(window):
    """The window as a number of 64 bits; 0: none.  Positions are below 2^31."""
    if window is None:
        return 0
    if window <= 0:
        raise ValueError("window must be positive, or None")
    return min(operator.index(window), 1 << 31)


def _on(stream, tensor):
    return torch.cuda.stream(torch.cuda.ExternalStream(stream, device=tensor.device))


def _rows_like(rows, resources, stream):
    """A result of the shape and type of these rows that belongs to the stream which writes it."""
    if resources._fixed_stream is None:
        return torch.empty_like(rows)
    with _on(stream, rows):
        return torch.empty_like(rows)


def _empty(dtype, tensor, resources, stream, *shape):
    if resources._fixed_stream is None:
        return torch.empty(*shape, dtype=dtype, device=tensor.device)
    with _on(stream, tensor):
        return torch.empty(*shape, dtype=dtype, device=tensor.device)


def _call(resources, stream, op, tensors, integer, scale, sync):
    """`tensors`: those of the call in the order of the C interface, filled up with None to eleven.  False: the call is being captured, and
    needs a workspace to itself."""
    for t in tensors:
        if t is not None and type(t) is not _Tensor:
            return _call(resources, stream, op, tuple(_plain(t) for t in tensors), integer, scale, sync)
    if _tensors is None:
        scalars = ((integer,), (integer, _bits(scale)), (_bits(scale),), ())[op]
        status = _arrays(resources.handle, stream, op, *_words(tensors[:_COUNTS[op]], scalars), sync)
    else:
        status = _tensors(resources.handle, stream, op, *tensors, integer, scale, sync)
    if status == _NEEDS_WORKSPACE:
        return False
    if status != L.CUVS_SUCCESS:
        L.check(L.CUVS_ERROR)
    if not sync:
        resources._last.stream = stream  # what resources.sync() waits for
    elif _tensors is not None:
        L.check(_wait(resources.handle, stream))
    return True


def _plain(t):
    """Parameters and other subclasses as the tensors that they are."""
    if t is not None and not isinstance(t, _Tensor):
        raise TypeError(f"expected torch tensors, not {type(t).__name__}")
    return t if t is None or type(t) is _Tensor else t.as_subclass(_Tensor)


def _tensor_calls():
    """The entry point that reads tensors in place, through torch's table of DLPack exchange functions: describing them in Python took as long
    as everything else of a small call together.  None where torch has no such table."""
    capsule = getattr(torch.Tensor, "__dlpack_c_exchange_api__", None)
    if capsule is None:
        return None
    pointer = C.pythonapi.PyCapsule_GetPointer
    pointer.restype, pointer.argtypes = C.c_void_p, [C.py_object, C.c_char_p]
    if L.load().cuvsB200SetTensorExchange(pointer(capsule, b"dlpack_exchange_api"), id(None)) != L.CUVS_SUCCESS:
        return None
    call = C.PyDLL(L.LIB_PATH).cuvsB200KvCacheTensors  # keeps the interpreter's lock: it reads Python objects
    call.restype, call.argtypes = C.c_int, L.SIGNATURES["cuvsB200KvCacheTensors"]
    return call


_COUNTS = (11, 9, 7, 4)
_NEEDS_WORKSPACE = 2
_Tensor = torch.Tensor
_arrays = L.load().cuvsB200KvCacheArrays
_workspace = L.load().cuvsB200KvCacheWorkspaceArrays
_wait = L.load().cuvsB200KvCacheWait
_tensors = _tensor_calls()


def append(keys, values, new_keys, new_values, pages, positions, sequences=None, queries=None, frequencies=None, interleaved=False,
           slots=None, rotated=None, resources: Resources | None = None, sync: bool = True):
    """Writes the rows of new tokens to their places in the cache and returns ``(slots, rotated)``: the tokens' slots (int64), and their
    turned queries (None without ``queries``).

    ``new_keys``, ``new_values``: ``[n_tokens, n_heads, dim]``, any strides with rows on 16-byte boundaries (a part of a fused projection, say);
    ``positions``: int32 ``[n_tokens]``; ``sequences``: int32 ``[n_tokens]``, which sequence each token belongs to -- without it, token ``i`` is
    one of sequence ``i``; ``queries``: ``[n_tokens, n_query_heads, dim]``, with ``rotated`` to receive them (it may be ``queries``).

    ``frequencies`` (float64 or float32 ``[n_pairs]``, ``2 * n_pairs <= dim``): the pairs of columns ``(i, i + n_pairs)`` -- with
    ``interleaved`` ``(2i, 2i + 1)`` -- of keys and queries are turned by ``position * frequencies[i]`` radians; columns behind them stay.
    Angles are formed in 64 bits.

    A token whose position is negative (padding), whose sequence does not exist or whose page is not in the cache gets slot -1 and is not
    written; the query row of a token with a negative position is copied as it is.  Two tokens of a call must not have the same slot."""
    resources, stream = _handle(keys, resources)
    if slots is None:
        slots = _empty(torch.int64, keys, resources, stream, new_keys.shape[0])
    if queries is not None and rotated is None:
        rotated = _rows_like(queries, resources, stream)
    _call(resources, stream, _APPEND, (keys, values, new_keys, new_values, pages, positions, sequences, queries, frequencies, slots, rotated),
          1 if interleaved else 0, 0.0, sync)
    return slots, rotated


def attention(keys, values, queries, pages, lengths, scale=None, window=None, filter=None, out=None, lse=None, workspace=None,
              resources: Resources | None = None, sync: bool = True):
    """Attention of one token per sequence to the positions ``0 .. lengths[i] - 1`` of its sequence, or the last ``window`` of them.  Returns
    ``(out, lse)``: ``[n_sequences, n_query_heads, dim]`` of the cache's element type, and the natural logarithm of the softmax's
    denominator, float32 ``[n_sequences, n_query_heads]``.

    ``queries``: ``[n_sequences, n_query_heads, dim]``; ``pages``: int32 ``[n_sequences, width]``; ``lengths``: int32 ``[n_sequences]`` (0: nothing;
    positions past the table's width are not there); ``scale``: of the scores, by default ``dim ** -0.5``; ``filter``: uint32 tensor, the slot
    ``i`` may be attended only if bit ``i % 32`` of word ``i // 32`` is set, as in ``ivf_pq.search``.

    ``workspace``: uint8 tensor of at least ``attention_workspace(...)`` bytes that nothing else uses until the work is done; by default
    the handle's own for the stream, and one allocated for the call while it is captured."""
    window = _window(window)
    resources, stream = _handle(keys, resources)
    if queries.dim() != 3:
        raise ValueError(f"queries: 3 dimensions, not {queries.dim()}")
    n, n_heads, dim = queries.shape
    if out is None:
        out = _rows_like(queries, resources, stream)
    if lse is None:
        lse = _empty(torch.float32, keys, resources, stream, n, n_heads)
    if scale is None:
        scale = dim ** -0.5
    if not _call(resources, stream, _ATTENTION, (keys, values, queries, pages, lengths, filter, out, lse, workspace, None, None), window, scale,
                 sync):
        # what is replayed needs a workspace to itself; else the handle has one for the stream
        workspace = _empty(torch.uint8, keys, resources, stream, _attention_workspace(resources, keys, queries, pages, window))
        _call(resources, stream, _ATTENTION, (keys, values, queries, pages, lengths, filter, out, lse, workspace, None, None), window, scale,
              sync)
    return out, lse


def attention_workspace(keys, queries, pages, window=None, resources: Resources | None = None):
    """Bytes of workspace that :func:`attention` needs for tensors of these shapes."""
    return _attention_workspace(_handle(keys, resources)[0], keys, queries, pages, _window(window or None))


def _attention_workspace(resources, keys, queries, pages, window):
    size = C.c_size_t()
    L.check(_workspace(resources.handle, *_words((keys, queries, pages), (window,)), size))
    return size.value


def attend_candidates(keys, values, queries, candidates, scale=None, filter=None, out=None, lse=None,
                      resources: Resources | None = None, sync: bool = True):
    """Attention of every query head of a token to the slots that its list names: ``candidates``, int64 ``[n_tokens, n_query_heads, k]``, as
    searches over the keys of the token's sequence return them (whose slots they are is not looked at).  Ids that are no slots (the search's "no such neighbour", -1) and slots that ``filter`` leaves out
    are skipped; a slot that is named twice counts twice.  Returns ``(out, lse)`` as :func:`attention` does."""
    resources, stream = _handle(keys, resources)
    if queries.dim() != 3:
        raise ValueError(f"queries: 3 dimensions, not {queries.dim()}")
    n, n_heads, dim = queries.shape
    if out is None:
        out = _rows_like(queries, resources, stream)
    if lse is None:
        lse = _empty(torch.float32, keys, resources, stream, n, n_heads)
    _call(resources, stream, _CANDIDATES, (keys, values, queries, candidates, filter, out, lse, None, None, None, None), 0,
          dim ** -0.5 if scale is None else scale, sync)
    return out, lse


def merge_parts(parts, parts_lse, out=None, lse=None, resources: Resources | None = None, sync: bool = True):
    """Joins parts of one softmax over disjoint sets of rows: ``parts`` ``[n_parts, n_tokens, n_heads, dim]`` and their ``parts_lse``, float32
    ``[n_parts, n_tokens, n_heads]``, both of any strides between rows (blocks gathered from several GPUs, say).  Returns ``(out, lse)``.  What
    the row of a part holds whose lse is -inf does not count.  Parts have been rounded to their type before, the joined rows are once more."""
    resources, stream = _handle(parts, resources)
    if parts.dim() != 4:
        raise ValueError(f"parts: 4 dimensions, not {parts.dim()}")
    n_parts, n, n_heads, dim = parts.shape
    if out is None:
        out = _empty(parts.dtype, parts, resources, stream, n, n_heads, dim)
    if lse is None:
        lse = _empty(torch.float32, parts, resources, stream, n, n_heads)
    _call(resources, stream, _MERGE, (parts, parts_lse, out, lse, None, None, None, None, None, None, None), 0, 0.0, sync)
    return out, lse
