"""A paged K/V cache and the attention that reads it (include/gfx950_fmha.h):

* ``assign_slots``: block tables and slot maps from request lengths, on the GPU;
* ``write_cache``: K and V rows into the cache at those slots;
* ``tree_attention``: attention of a tree of drafted tokens over the cache; one
  token per request is plain decoding.

A cache is a (blocks, block_size, K/V heads, head dim) tensor, or a view of that
shape of any other storage order with a unit head-dim stride.  No reference
counterpart: it has no cache."""

from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _lib
from . import _launch
from ._launch import ptr, sig, strides

MAX_REQUESTS = 4096  # of one assign_slots call (G9_SLOTS_MAX_REQUESTS)


class Slots(NamedTuple):
    """Where a step's tokens go (``assign_slots``)."""

    cu_seqlens: torch.Tensor  # (B + 1,) int32: each request's rows in the packed batch
    slots: torch.Tensor  # (T,) int64: block * block_size + offset, -1 where there is none
    positions: torch.Tensor  # (T,) int64: the token's position in its request
    taken: torch.Tensor  # (1,) int32: new blocks


def assign_slots(lengths: torch.Tensor, counts: torch.Tensor, block_table: torch.Tensor, free_blocks: torch.Tensor,
                 block_size: int, num_tokens: int, *, free_start: torch.Tensor | None = None) -> Slots:
    """Slots for the next ``counts[b]`` tokens of each request, and the blocks
    they need entered into ``block_table``.

    ``lengths`` (B,) int32 are the tokens already in the cache, whose blocks fill
    the first ceil(length / block_size) entries of the request's table row; new
    blocks are the next of ``free_blocks`` (int32), from ``free_start[0]`` on (a
    (1,) int32 tensor; 0 by default), in the order of the requests.  Everything
    stays on the GPU: a program that keeps its free list there adds ``taken`` to
    ``free_start`` for the next step, and returns blocks at the list's end.

    ``num_tokens`` is the packed batch's row count; rows behind the last token get
    slot -1 and position 0.  A token for which the free list or the table's width
    does not reach gets slot -1 (``taken`` above what the list holds says so).
    At most ``MAX_REQUESTS`` requests."""
    block_size, num_tokens = int(block_size), int(num_tokens)
    key = ("slots", block_size, num_tokens, sig(lengths), sig(counts), sig(block_table), sig(free_blocks),
           free_start is not None and sig(free_start))
    dev, B, args = _launch.planned(key) or _plan_slots(key, lengths, counts, block_table, free_blocks, block_size,
                                                       num_tokens, free_start)
    longs = torch.empty((2, num_tokens), dtype=torch.int64, device=dev)
    ints = torch.empty(B + 2, dtype=torch.int32, device=dev)
    slots, positions = longs.unbind(0)
    cu, taken = ints.split_with_sizes((B + 1, 1))
    at, cu_at = longs.data_ptr(), ints.data_ptr()
    _launch.call("g9_assign_slots", dev, lengths.data_ptr(), counts.data_ptr(), B, block_table.data_ptr(), *args[:2],
                 free_blocks.data_ptr(), args[2], ptr(free_start), block_size, num_tokens, cu_at, at, at + 8 * num_tokens,
                 cu_at + 4 * (B + 1))
    return Slots(cu, slots, positions, taken)


def _plan_slots(key, lengths, counts, block_table, free_blocks, block_size, num_tokens, free_start):
    dev = _launch.gpu_of(lengths, counts, block_table, free_blocks, free_start)
    for name, t, n in (("lengths", lengths, 1), ("counts", counts, 1), ("block_table", block_table, 2),
                       ("free_blocks", free_blocks, 1)):
        _launch.int32_of(name, t, n)
    B = lengths.shape[0]
    if counts.shape[0] != B or block_table.shape[0] != B:
        raise ValueError(f"lengths, counts and block_table hold {B}, {counts.shape[0]} and {block_table.shape[0]} requests")
    if B > MAX_REQUESTS:
        raise ValueError(f"{B} requests; at most {MAX_REQUESTS} in one call")
    if num_tokens < 0:
        raise ValueError(f"num_tokens is {num_tokens}")
    if free_start is not None:
        _launch.int32_of("free_start", free_start, 1)
        if free_start.shape[0] != 1:
            raise ValueError("free_start must hold one value")
    return _launch.keep(key, dev, (dev, B, (block_table.stride(0), block_table.shape[1], free_blocks.shape[0])))


def _cache_of(k_cache, v_cache):
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or k_cache.dtype != v_cache.dtype:
        raise ValueError("k_cache and v_cache must be (blocks, block_size, heads, head dim) of one shape and dtype; got "
                         f"{tuple(k_cache.shape)} and {tuple(v_cache.shape)}")
    if k_cache.stride(3) != 1 or v_cache.stride(3) != 1:
        raise ValueError("the caches need a unit head-dim stride")
    return k_cache.shape


def write_cache(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                slots: torch.Tensor) -> None:
    """Copies row t of k and v (T, HK, D) to slot ``slots[t]`` (int64) of the
    caches.  Rows whose slot is negative or behind the cache are skipped; slots
    must be distinct (two rows of one slot may leave a mixture of both there).

    fp16 or bf16, head dim 64 or 128; block_size a power of two from 16 to 1024."""
    key = ("write", sig(k), sig(v), sig(k_cache), sig(v_cache), sig(slots))
    dev, rest = _launch.planned(key) or _plan_write(key, k, v, k_cache, v_cache, slots)
    _launch.plain(k, v, k_cache, v_cache)
    _launch.call("g9_write_cache", dev, k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                 slots.data_ptr(), *rest)


def _plan_write(key, k, v, k_cache, v_cache, slots):
    dev = _launch.gpu_of(k, v, k_cache, v_cache, slots)
    T, HK, D = _launch.rows_of("k", k)
    _launch.rows_of("v", v)
    blocks, size, heads, dim = _cache_of(k_cache, v_cache)
    if v.shape != k.shape or (heads, dim) != (HK, D):
        raise ValueError(f"k {tuple(k.shape)}, v {tuple(v.shape)} do not fit a cache of {heads} heads of {dim}")
    if slots.dtype != torch.int64 or slots.dim() != 1 or slots.shape[0] != T or not slots.is_contiguous():
        raise ValueError(f"slots must be {T} contiguous int64 values")
    _launch.dtype_of(k, v, k_cache, v_cache)
    return _launch.keep(key, dev, (dev, (T, HK, D, blocks, size, strides(k), strides(v), strides(k_cache),
                                         strides(v_cache))))


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                   lengths: torch.Tensor, cu_seqlens: torch.Tensor, tree_mask: torch.Tensor | None = None,
                   o: torch.Tensor | None = None, *, sm_scale: float | None = None,
                   lse: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of drafted tokens over a paged cache.

    Request b brings the query rows [cu_seqlens[b], cu_seqlens[b + 1]) of q
    (T, HQ, D), the nodes of its draft.  ``block_table`` (B, width) int32 names the
    blocks of its ``lengths[b]`` context tokens and, at the positions behind them,
    of the nodes themselves: their K and V are in the cache already
    (``assign_slots``, ``write_cache``).  Every node reads the whole context and
    the nodes j whose bit j % 64 is set in word j // 64 of its ``tree_mask`` row,
    int64 (T, words) or (T,); a node that is to read itself has its own bit set.
    Without a mask the draft is a chain: node i reads the nodes j <= i, and one
    node per request is plain decoding.

    fp16 or bf16, head dim 64 or 128, grouped heads; block_size a power of two
    from 16 to 1024.  Returns ``o`` (T, HQ, D), allocated when not given; rows
    behind the last request are left as they were, a row that reads nothing gives
    zeros.  ``lse`` and the arithmetic as in ``varlen_attention``.  Asynchronous on
    the current stream; forward only."""
    sm_scale = None if sm_scale is None else float(sm_scale)
    key = ("tree", sm_scale, sig(q), sig(k_cache), sig(v_cache), sig(block_table), sig(lengths), sig(cu_seqlens),
           tree_mask is not None and sig(tree_mask), o is not None and sig(o), lse is not None and sig(lse))
    dev, need, table, words, rest = _launch.planned(key) or _plan_tree(
        key, q, k_cache, v_cache, block_table, lengths, cu_seqlens, tree_mask, o, lse, sm_scale)
    _launch.plain(q, k_cache, v_cache, o, lse)
    if o is None:
        o = torch.empty(q.shape, dtype=q.dtype, device=dev)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    _launch.call("g9_tree_fwd", dev, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), o.data_ptr(), ptr(lse),
                 block_table.data_ptr(), *table, lengths.data_ptr(), cu_seqlens.data_ptr(), ptr(tree_mask), words, *rest,
                 ws.data_ptr(), need)
    return o


def _plan_tree(key, q, k_cache, v_cache, block_table, lengths, cu_seqlens, tree_mask, o, lse, sm_scale):
    dev = _launch.gpu_of(q, k_cache, v_cache, block_table, lengths, cu_seqlens, tree_mask, o, lse)
    T, HQ, D = _launch.rows_of("q", q)
    blocks, size, HK, dim = _cache_of(k_cache, v_cache)
    if dim != D:
        raise ValueError(f"q has head dim {D}, the cache {dim}")
    B = _launch.offsets_of("cu_seqlens", cu_seqlens)
    _launch.int32_of("lengths", lengths, 1)
    _launch.int32_of("block_table", block_table, 2)
    if lengths.shape[0] != B or block_table.shape[0] != B:
        raise ValueError(f"cu_seqlens, lengths and block_table hold {B}, {lengths.shape[0]} and {block_table.shape[0]} requests")
    words = _launch.mask_words(tree_mask, T)
    _launch.heads_fit(HQ, HK, D)
    if o is not None:
        _launch.rows_of("o", o)
        if o.shape != q.shape:
            raise ValueError(f"o is {tuple(o.shape)}, q {tuple(q.shape)}")
    dtype = _launch.dtype_of(q, k_cache, v_cache, *([o] if o is not None else []))
    _launch.lse_fits(lse, HQ, T)
    os = _launch.array(HQ * D, D) if o is None else strides(o)
    return _launch.keep(key, dev, (
        dev, _lib.load().g9_tree_workspace_size(B, T, HQ, HK, D), (block_table.stride(0), block_table.shape[1]), words,
        (B, T, HQ, HK, D, blocks, size, strides(q), strides(k_cache), strides(v_cache), os,
         D**-0.5 if sm_scale is None else sm_scale, dtype)))
