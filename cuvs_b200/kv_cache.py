"""Attention over a paged cache of keys and values, next to the search over its keys.

A decoder keeps the keys and values of its tokens in pages and reaches back over a context that is too long to be read in full by a
search over the keys.  A step then is::

    slots, q = kv_cache.append(keys, values, new_keys, new_values, pages, positions, queries=queries, frequencies=frequencies)
    _, candidates = ivf_pq.search(params, index_of_head, q[:, head], k)         # an index whose source ids are slots
    near = kv_cache.attention(keys, values, q, pages, lengths, window=window)
    far = kv_cache.attend_candidates(keys, values, q, candidates)               # [n_tokens, n_query_heads, k]
    out, lse = kv_cache.merge_parts(torch.stack((near[0], far[0])), torch.stack((near[1], far[1])))

``keys`` and ``values`` are ``[n_pages, page_size, n_heads, dim]`` tensors of float16, bfloat16 or float32, of any strides that leave the
rows of ``dim`` elements contiguous and on 16-byte boundaries.  A token's slot is ``page * page_size + place``, and is the id under which
its key is put into an index.  ``pages`` (int32 ``[n_sequences, width]``) names the pages of each sequence in the order of its positions;
an entry that is no page of the cache, such as -1, holds no tokens.  Query head ``i`` reads the rows of head
``i // (n_query_heads // n_heads)``.  Softmax and sums are held in 32 bits, outputs are rounded once; where nothing may be attended to, the
output is 0 and its ``lse`` is -inf.

These calls serve: they have no gradients.  They enqueue their work on the stream of ``resources`` (torch's current stream by default) and
wait for it unless ``sync=False``, which is what a captured call needs.
"""
from __future__ import annotations

import ctypes as C
import struct

import torch

from . import _lib as L
from .common import Resources, default_resources

# ndim | dtype code << 32 | bits << 40 | lanes << 48
_WORD = {t: (code << 32) | (bits << 40) | (1 << 48)
         for t, code, bits in ((torch.float16, 2, 16), (torch.bfloat16, 4, 16), (torch.float32, 2, 32), (torch.float64, 2, 64),
                               (torch.int32, 0, 32), (torch.int64, 0, 64), (torch.uint32, 1, 32), (torch.uint8, 1, 8))}
_PAD = [(0,) * n for n in range(5)]
_ABSENT = (0,) * 11
_APPEND, _ATTENTION, _CANDIDATES, _MERGE = range(4)


def _words(tensors, device, scalars):
    """The words that describe a call's tensors (the order of the C interface) and its scalars."""
    words = []
    for t in tensors:
        if t is None:
            words += _ABSENT
            continue
        word, n, at = _WORD.get(t.dtype), t.dim(), t.get_device()
        if word is None:
            raise ValueError(f"unsupported element type {t.dtype}")
        if not 1 <= n <= 4:
            raise ValueError(f"tensors have 1 to 4 dimensions, not {n}")
        pad = _PAD[4 - n]
        words += (t.data_ptr(), word | n, (L.kDLCUDA | (at << 32)) if at >= 0 else L.kDLCPU, *t.shape, *pad, *t.stride(), *pad)
    words += scalars
    return (C.c_int64 * len(words))(*words)


def _bits(scale):
    return struct.unpack("<I", struct.pack("<f", scale))[0]


class _Call:
    """Where a call's work goes and where its results are allocated: the tensors' device and the stream of the handle."""

    __slots__ = ("res", "stream", "device", "_scope")

    def __init__(self, tensor, resources):
        if not isinstance(tensor, torch.Tensor) or not tensor.is_cuda:
            raise ValueError("expected CUDA tensors")
        self.device = tensor.get_device()
        self._scope = None
        if resources is None:
            if torch.cuda.current_device() == self.device:
                resources = default_resources(self.device)
            else:
                with torch.cuda.device(self.device):
                    resources = default_resources(self.device)
        self.res = resources
        self.stream = resources.stream_at_call(self.device)
        if resources._fixed_stream is not None:
            # results belong to the stream that writes them
            self._scope = torch.cuda.stream(torch.cuda.ExternalStream(self.stream, device=self.device))

    def __enter__(self):
        if self._scope is not None:
            self._scope.__enter__()
        return self

    def __exit__(self, *what):
        if self._scope is not None:
            self._scope.__exit__(*what)

    def run(self, op, tensors, scalars, sync):
        words = _words(tensors, self.device, scalars)
        L.check(L.load().cuvsB200KvCacheArrays(self.res.handle, self.stream, op, words, len(words), bool(sync)))


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
    with _Call(keys, resources) as call:
        if slots is None:
            slots = torch.empty((new_keys.shape[0],), dtype=torch.int64, device=keys.device)
        if queries is not None and rotated is None:
            rotated = queries.new_empty(queries.shape)
        call.run(_APPEND, (keys, values, new_keys, new_values, pages, positions, sequences, queries, frequencies, slots, rotated),
                 (int(bool(interleaved)),), sync)
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
    one is allocated for the call."""
    if window is not None and window <= 0:
        raise ValueError("window must be positive, or None")
    if scale is None:
        scale = queries.shape[-1] ** -0.5
    with _Call(keys, resources) as call:
        if out is None:
            out = queries.new_empty(queries.shape)
        if lse is None:
            lse = torch.empty(queries.shape[:2], dtype=torch.float32, device=keys.device)
        if workspace is None:
            need = _attention_workspace(call, keys, queries, pages, window)
            if need:
                workspace = torch.empty((need,), dtype=torch.uint8, device=keys.device)
        call.run(_ATTENTION, (keys, values, queries, pages, lengths, filter, out, lse, workspace), (window or 0, _bits(scale)), sync)
    return out, lse


def _attention_workspace(call, keys, queries, pages, window):
    return 0


def attend_candidates(keys, values, queries, candidates, scale=None, filter=None, out=None, lse=None,
                      resources: Resources | None = None, sync: bool = True):
    """Attention of every query head of a token to the slots that its list names: ``candidates``, int64 ``[n_tokens, n_query_heads, k]``, as
    searches over the keys return them.  Ids that are no slots (the search's "no such neighbour", -1) and slots that ``filter`` leaves out
    are skipped; a slot that is named twice counts twice.  Returns ``(out, lse)`` as :func:`attention` does."""
    if scale is None:
        scale = queries.shape[-1] ** -0.5
    with _Call(keys, resources) as call:
        if out is None:
            out = queries.new_empty(queries.shape)
        if lse is None:
            lse = torch.empty(queries.shape[:2], dtype=torch.float32, device=keys.device)
        call.run(_CANDIDATES, (keys, values, queries, candidates, filter, out, lse), (_bits(scale),), sync)
    return out, lse


def merge_parts(parts, parts_lse, out=None, lse=None, resources: Resources | None = None, sync: bool = True):
    """Joins parts of one softmax over disjoint sets of rows: ``parts`` ``[n_parts, n_tokens, n_heads, dim]`` and their ``parts_lse``, float32
    ``[n_parts, n_tokens, n_heads]``, both of any strides between rows (blocks gathered from several GPUs, say).  Returns ``(out, lse)``.  A
    part whose lse is -inf is not read."""
    with _Call(parts, resources) as call:
        if out is None:
            out = parts.new_empty(parts.shape[1:])
        if lse is None:
            lse = torch.empty(parts.shape[1:3], dtype=torch.float32, device=parts.device)
        call.run(_MERGE, (parts, parts_lse, out, lse), (), sync)
    return out, lse
