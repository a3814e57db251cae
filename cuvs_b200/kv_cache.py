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

A decoder that drafts several tokens per sequence, a tree of them, and keeps the path that it accepts has as its step::

    mask, positions = kv_cache.draft_tree(parents, lengths)                     # [n_sequences, n_drafted]; lengths: without the drafted tokens
    places = torch.where(positions >= 0, lengths[:, None] + torch.arange(n_drafted, dtype=torch.int32, device="cuda"), -1).flatten()
    # these hold for all layers; for each of them
    slots, q = kv_cache.append(keys, values, new_keys.flatten(0, 1), new_values.flatten(0, 1), pages, places, sequences=sequences,
                               queries=queries.flatten(0, 1), frequencies=frequencies, turns=positions.flatten())
    out, lse = kv_cache.attend_tree(keys, values, q.view(queries.shape), pages, lengths, positions, mask)
    lengths = kv_cache.keep_path(keys, values, pages, lengths, paths)           # paths: which of the drafted tokens stay, in order

The drafted token ``j`` of a sequence is stored behind the sequence's own tokens, at place ``lengths[i] + j``, whatever its depth in the tree: its
position, by which it is turned, is that of its depth.  Where a sequence goes on in several ways they have its full pages in common, and
:func:`copy_pages` copies the last one.

These calls serve: they have no gradients.  They enqueue their work on the stream of ``resources`` (torch's current stream by default) and
wait for it unless ``sync=False``, which is what a captured call needs.  :func:`attend_tree` of 16-bit rows waits inside its kernel, with limits of seconds:
should one run out, the next call that waits for that stream, or ``Resources.sync``, raises an error (of a captured call, the next on any stream).
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
_APPEND, _ATTENTION, _CANDIDATES, _MERGE, _APPEND_TURNED, _DRAFT_TREE, _ATTEND_TREE, _KEEP_PATH, _COPY_PAGES = range(9)
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


def _call(resources, stream, op, tensors, integer, scale, sync, cap=0.0):
    """`tensors`: those of the call in the order of the C interface, filled up with None to eleven, from the fifth call on to thirteen.  False:
    the call is being captured, and needs a workspace to itself."""
    for t in tensors:
        if t is not None and type(t) is not _Tensor:
            return _call(resources, stream, op, tuple(_plain(t) for t in tensors), integer, scale, sync, cap)
    if _tensors is None:
        scalars = ((integer,), (integer, _bits(scale)), (_bits(scale),), (), (integer,), (), (integer, _bits(scale), _bits(cap)), (), ())[op]
        status = _arrays(resources.handle, stream, op, *_words(tensors[:_COUNTS[op]], scalars), sync)
    elif op < _APPEND_TURNED:
        status = _tensors(resources.handle, stream, op, *tensors, integer, scale, sync)
    else:
        status = _more_tensors(resources.handle, stream, op, *tensors, integer, scale, cap, sync)
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
    """The entry points that read tensors in place, through torch's table of DLPack exchange functions: describing them in Python took as long
    as everything else of a small call together.  None where torch has no such table."""
    capsule = getattr(torch.Tensor, "__dlpack_c_exchange_api__", None)
    if capsule is None:
        return None, None
    pointer = C.pythonapi.PyCapsule_GetPointer
    pointer.restype, pointer.argtypes = C.c_void_p, [C.py_object, C.c_char_p]
    if L.load().cuvsB200SetTensorExchange(pointer(capsule, b"dlpack_exchange_api"), id(None)) != L.CUVS_SUCCESS:
        return None, None
    lib, calls = C.PyDLL(L.LIB_PATH), []  # keeps the interpreter's lock: it reads Python objects
    for name in ("cuvsB200KvCacheTensors", "cuvsB200KvCacheMoreTensors"):
        call = getattr(lib, name)
        call.restype, call.argtypes = C.c_int, L.SIGNATURES[name]
        calls.append(call)
    return calls


_COUNTS = (11, 9, 7, 4, 13, 4, 12, 6, 4)
_NEEDS_WORKSPACE = 2
_Tensor = torch.Tensor
_arrays = L.load().cuvsB200KvCacheArrays
_workspace = L.load().cuvsB200KvCacheWorkspaceArrays
_tree_workspace = L.load().cuvsB200KvCacheTreeWorkspaceArrays
_wait = L.load().cuvsB200KvCacheWait
_tensors, _more_tensors = _tensor_calls()


def append(keys, values, new_keys, new_values, pages, positions, sequences=None, queries=None, frequencies=None, interleaved=False,
           slots=None, rotated=None, resources: Resources | None = None, sync: bool = True, *, turns=None, axes=None):
    """Writes the rows of new tokens to their places in the cache and returns ``(slots, rotated)``: the tokens' slots (int64), and their
    turned queries (None without ``queries``).

    ``new_keys``, ``new_values``: ``[n_tokens, n_heads, dim]``, any strides with rows on 16-byte boundaries (a part of a fused projection, say);
    ``positions``: int32 ``[n_tokens]``; ``sequences``: int32 ``[n_tokens]``, which sequence each token belongs to -- without it, token ``i`` is
    one of sequence ``i``; ``queries``: ``[n_tokens, n_query_heads, dim]``, with ``rotated`` to receive them (it may be ``queries``).

    ``frequencies`` (float64 or float32 ``[n_pairs]``, ``2 * n_pairs <= dim``): the pairs of columns ``(i, i + n_pairs)`` -- with
    ``interleaved`` ``(2i, 2i + 1)`` -- of keys and queries are turned by ``position * frequencies[i]`` radians; columns behind them stay.
    Angles are formed in 64 bits.

    ``turns`` (int32 ``[n_tokens]`` or ``[n_tokens, n_axes]``) turns keys and queries by other positions than those that say where the tokens go:
    pair ``i`` of token ``t`` by ``turns[t, axes[i]] * frequencies[i]`` radians, either way round; ``axes``: int32 ``[n_pairs]``, not needed where there is one axis;
    a pair whose axis is none of them stays.  (Tokens of images and videos have a time, a row and a column; a drafted token's position is
    its depth in the tree, not its place.)

    A token whose position is negative (padding), whose sequence does not exist or whose page is not in the cache gets slot -1 and is not
    written; the query row of a token with a negative position is copied as it is.  Two tokens of a call must not have the same slot."""
    resources, stream = _handle(keys, resources)
    if slots is None:
        slots = _empty(torch.int64, keys, resources, stream, new_keys.shape[0])
    if queries is not None and rotated is None:
        rotated = _rows_like(queries, resources, stream)
    tensors = (keys, values, new_keys, new_values, pages, positions, sequences, queries, frequencies, slots, rotated)
    if turns is not None:
        _call(resources, stream, _APPEND_TURNED, (*tensors, turns, axes), 1 if interleaved else 0, 0.0, sync)
    elif axes is not None:
        raise ValueError("axes go with turns")
    else:
        _call(resources, stream, _APPEND, tensors, 1 if interleaved else 0, 0.0, sync)
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


def draft_tree(parents, lengths, mask=None, positions=None, resources: Resources | None = None, sync: bool = True):
    """Who reaches whom in the trees of a step's drafted tokens.  ``parents``: int32 ``[n_sequences, n_drafted]`` (at most 1024; sequences may
    share a row, as ``expand`` makes it), the index of the token that each one follows, in whatever order they stand, or -1: it follows the
    sequence itself; any other value, and what follows it, is no token.  ``lengths``: int32 ``[n_sequences]``, the sequences' tokens without them.

    Returns ``(mask, positions)``: uint32 ``[n_sequences, n_drafted, ceil(n_drafted / 32)]``, in whose row ``j`` bit ``k % 32`` of word ``k // 32`` says that
    ``k`` is ``j`` or one of its ancestors, and int32 ``[n_sequences, n_drafted]``, the length plus the number of ancestors; 0 and -1 for what is no token.
    They hold for all layers of a step."""
    resources, stream = _handle(parents, resources)
    if parents.dim() != 2:
        raise ValueError(f"parents: 2 dimensions, not {parents.dim()}")
    n, m = parents.shape
    if mask is None:
        mask = _empty(torch.uint32, parents, resources, stream, n, m, (m + 31) // 32)
    if positions is None:
        positions = _empty(torch.int32, parents, resources, stream, n, m)
    _call(resources, stream, _DRAFT_TREE, (parents, lengths, mask, positions, *(None,) * 9), 0, 0.0, sync)
    return mask, positions


def attend_tree(keys, values, queries, pages, lengths, positions, mask, scale=None, window=None, cap=None, slopes=None, filter=None, out=None,
                lse=None, workspace=None, resources: Resources | None = None, sync: bool = True):
    """Attention of the drafted tokens of each sequence, ``queries`` ``[n_sequences, n_drafted, n_query_heads, dim]``, to the sequence's positions
    ``0 .. lengths[i] - 1`` and to those of its drafted tokens that ``mask`` names.  Returns ``(out, lse)``: of the queries' shape, and float32
    ``[n_sequences, n_drafted, n_query_heads]``.

    ``lengths``: int32 ``[n_sequences]``, without the drafted tokens, of which number ``k`` is stored at place ``lengths[i] + k``; ``positions`` (int32
    ``[n_sequences, n_drafted]``) and ``mask`` (uint32 ``[n_sequences, n_drafted, words]``) as :func:`draft_tree` returns them, or any others, sequences may share
    them; a token whose position is below its sequence's length is none: it attends to nothing, and none to it.

    Scores are ``s = scale * q.k`` (``dim ** -0.5``), with ``cap`` (1e-30 to 1e30, ``scale / cap`` in the range of 32-bit numbers) then ``cap *
    tanh(s / cap)``, with ``slopes`` (float32 ``[n_query_heads]``) then less ``slope * distance`` of the two positions.  ``window``: only what is less than so many positions before the token's own; ``filter``, ``workspace`` as in
    :func:`attention`.  Of 16-bit rows, weights below 2^-30 of the largest may count as 0."""
    window = _window(window)
    resources, stream = _handle(keys, resources)
    if queries.dim() != 4:
        raise ValueError(f"queries: 4 dimensions, not {queries.dim()}")
    if cap is not None and not 1e-30 <= cap <= 1e30:
        raise ValueError("cap must be between 1e-30 and 1e30, or None")
    n, m, n_heads, dim = queries.shape
    if out is None:
        out = _empty(queries.dtype, keys, resources, stream, n, m, n_heads, dim)
    if lse is None:
        lse = _empty(torch.float32, keys, resources, stream, n, m, n_heads)
    scale, cap = dim ** -0.5 if scale is None else scale, cap or 0.0
    tensors = (keys, values, queries, pages, lengths, positions, mask, slopes, filter, out, lse)
    if not _call(resources, stream, _ATTEND_TREE, (*tensors, workspace, None), window, scale, sync, cap):
        # what is replayed needs a workspace to itself; else the handle has one for the stream
        workspace = _empty(torch.uint8, keys, resources, stream, _attend_tree_workspace(resources, keys, queries, pages, window))
        _call(resources, stream, _ATTEND_TREE, (*tensors, workspace, None), window, scale, sync, cap)
    return out, lse


def attend_tree_workspace(keys, queries, pages, window=None, resources: Resources | None = None):
    """Bytes of workspace that :func:`attend_tree` needs for tensors of these shapes."""
    return _attend_tree_workspace(_handle(keys, resources)[0], keys, queries, pages, _window(window or None))


def _attend_tree_workspace(resources, keys, queries, pages, window):
    size = C.c_size_t()
    L.check(_tree_workspace(resources.handle, *_words((keys, queries, pages), (window,)), size))
    return size.value


def keep_path(keys, values, pages, lengths, paths, kept=None, resources: Resources | None = None, sync: bool = True):
    """Moves the rows of the drafted tokens that stay up to their sequences' ends, and returns the sequences' new lengths, int32 ``[n_sequences]``.

    ``paths``: int32 ``[n_sequences, n_entries]``, which of the drafted tokens stay, in ascending order; a path ends at its first entry that is not
    greater than the one before it, such as -1.  The row at place ``lengths[i] + paths[i, m]`` goes to place ``lengths[i] + m`` where the cache has both;
    it has been turned by its position before, which stays the same where a path goes from parent to child.  ``kept`` receives the new lengths, in memory of
    its own.  Pages that are written belong to one sequence alone."""
    resources, stream = _handle(keys, resources)
    if kept is None:
        kept = _empty(torch.int32, keys, resources, stream, lengths.shape[0])
    _call(resources, stream, _KEEP_PATH, (keys, values, pages, lengths, paths, kept, *(None,) * 7), 0, 0.0, sync)
    return kept


def copy_pages(keys, values, sources, targets, resources: Resources | None = None, sync: bool = True):
    """Copies the pages ``sources[m]`` of keys and values to the pages ``targets[m]``, int32 ``[n_pairs]`` each.  A pair with a number that is no page of the
    cache is skipped; no page may be the target of two pairs, or a target and a source.

    Where a sequence goes on in several ways, the new ones have its full pages in common, and a copy of the last::

        last = pages[sources, lengths[sources] // page_size]
        kv_cache.copy_pages(keys, values, last, free)
        pages[targets] = pages[sources]
        pages[targets, lengths[sources] // page_size] = free"""
    resources, stream = _handle(keys, resources)
    _call(resources, stream, _COPY_PAGES, (keys, values, sources, targets, *(None,) * 9), 0, 0.0, sync)
