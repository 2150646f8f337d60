"""Latent attention (include/gfx950_fmha.h): every head's keys and values come from
one latent of 512 values a token, beside a rotated key of 64 values that all heads
share.

* ``write_latent``: norm, rotation and write of a step's tokens into a paged cache;
* ``latent_attention``: the absorbed form over that cache, where the heads'
  projections are applied to the query and to the output: single tokens and drafts;
* ``latent_varlen_attention``: the expanded form over packed prompts, where they
  are applied to the latents.

A cache is a (blocks, block_size, 576) tensor with a unit last stride, a row the
latent and behind it the rotated key; ``assign_slots`` keeps its books.  No reference
counterpart."""

from __future__ import annotations

import math

import torch

from .. import _lib
from . import _launch
from ._launch import ptr, sig, strides
from .rotary import check_turns

RANK, ROPE = 512, 64  # values of a latent, of a rotated key
NOPE, VALUE = 128, 128  # of an expanded key's own part, of an expanded value


def _rows(name, t, width):
    if t.dim() != 2 or t.shape[1] != width or t.stride(1) != 1:
        raise ValueError(f"{name} must be (rows, {width}) with a unit last stride; got {tuple(t.shape)}, strides {t.stride()}")
    return t.shape[0]


def _cache(cache):
    if cache.dim() != 3 or cache.shape[2] != RANK + ROPE or cache.stride(2) != 1:
        raise ValueError(f"the cache must be (blocks, block_size, {RANK + ROPE}) with a unit last stride; got "
                         f"{tuple(cache.shape)}, strides {cache.stride()}")
    return cache.shape[:2]


def write_latent(c: torch.Tensor, k_rope: torch.Tensor, cache: torch.Tensor, slots: torch.Tensor, *,
                 weight: torch.Tensor | None = None, eps: float = 1e-6, positions: torch.Tensor | None = None,
                 freqs: torch.Tensor | None = None, interleaved: bool = False, scale: float = 1.0,
                 c_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None) -> None:
    """Row t of c (T, 512) and k_rope (T, 64) to slot ``slots[t]`` (int64) of the cache.

    With ``weight`` (512,) the latent is normalised on the way: c / sqrt(mean(c^2) +
    eps) * weight; with ``positions`` and ``freqs`` (32,) the key is turned as by
    ``rotary`` (``interleaved`` and ``scale`` as there).  Both in fp32, rounded once.
    ``c_out`` (T, 512) and ``k_out`` (T, 64), if given, receive every row as the cache
    does, for the expansion of a prompt's keys and values; they may be c and k_rope
    themselves and must not overlap the inputs, each other or the cache otherwise.

    Rows whose slot is negative or behind the cache are skipped (in ``c_out`` and
    ``k_out`` they are not); slots must be distinct.  fp16 or bf16; row steps of 16
    bytes, so c and k_rope may be parts of one projection; block_size a power of two
    from 16 to 1024.  Asynchronous on the current stream; forward only."""
    eps, interleaved, scale = float(eps), bool(interleaved), float(scale)
    key = ("write_latent", eps, interleaved, scale, sig(c), sig(k_rope), sig(cache), sig(slots),
           *(t is not None and sig(t) for t in (weight, positions, freqs, c_out, k_out)))
    dev, rest = _launch.planned(key) or _plan_write(key, c, k_rope, cache, slots, weight, eps, positions, freqs,
                                                    interleaved, scale, c_out, k_out)
    _launch.plain(c, k_rope, cache, weight, freqs, c_out, k_out)
    _launch.call("g9_write_latent", dev, c.data_ptr(), k_rope.data_ptr(), cache.data_ptr(), slots.data_ptr(), ptr(weight),
                 eps, ptr(positions), ptr(freqs), ptr(c_out), ptr(k_out), *rest)


def _plan_write(key, c, k_rope, cache, slots, weight, eps, positions, freqs, interleaved, scale, c_out, k_out):
    dev = _launch.gpu_of(c, k_rope, cache, slots, weight, positions, freqs, c_out, k_out)
    T = _rows("c", c, RANK)
    blocks, size = _cache(cache)
    for name, t, width in (("k_rope", k_rope, ROPE), ("c_out", c_out, RANK), ("k_out", k_out, ROPE)):
        if t is not None and _rows(name, t, width) != T:
            raise ValueError(f"c has {T} rows, {name} {t.shape[0]}")
    if slots.dtype != torch.int64 or slots.shape != (T,) or not slots.is_contiguous():
        raise ValueError(f"slots must be {T} contiguous int64 values")
    if weight is not None and (weight.shape != (RANK,) or not weight.is_contiguous()):
        raise ValueError(f"weight must be {RANK} contiguous values")
    if (positions is None) != (freqs is None):
        raise ValueError("positions and freqs come together")
    if positions is not None:
        check_turns("c", T, positions, freqs, ROPE // 2)
    if not (math.isfinite(eps) and eps >= 0 and math.isfinite(scale)):
        raise ValueError(f"eps is {eps}, scale {scale}")
    dtype = _launch.dtype_of(c, k_rope, cache, *(t for t in (weight, c_out, k_out) if t is not None))
    return _launch.keep(key, dev, (dev, (T, blocks, size, c.stride(0), k_rope.stride(0), strides(cache),
                                         0 if c_out is None else c_out.stride(0), 0 if k_out is None else k_out.stride(0),
                                         scale, interleaved, dtype)))


def latent_attention(q: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor,
                     cu_seqlens: torch.Tensor, tree_mask: torch.Tensor | None = None, o: torch.Tensor | None = None, *,
                     sm_scale: float, lse: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of single or drafted tokens over a paged cache of latents.

    q (T, H, 576) holds each head's query times its key projection (512 values) and
    its rotated part (64); the score of a token is ``sm_scale`` times the product with
    its row, and ``o`` (T, H, 512) the weighted sum of the latents, to be multiplied by
    the heads' value projections.  ``sm_scale`` is that of the expanded form, whose keys
    are shorter: it does not follow from q.  Requests, ``block_table``, ``lengths``,
    ``cu_seqlens`` and ``tree_mask`` as in ``tree_attention``.

    fp16 or bf16, any number of heads; block_size a power of two from 16 to 1024.
    Returns ``o``, allocated when not given; rows behind the last request are left as
    they were, a row that reads nothing gives zeros.  ``lse`` (H, T) and the
    arithmetic as in ``varlen_attention``, but for scores of any finite size.  A call's
    workspace is 34 to 135 MB, by T / B times H.  Asynchronous on the current stream;
    forward only."""
    sm_scale = float(sm_scale)
    key = ("latent", sm_scale, sig(q), sig(cache), sig(block_table), sig(lengths), sig(cu_seqlens),
           tree_mask is not None and sig(tree_mask), o is not None and sig(o), lse is not None and sig(lse))
    dev, need, table, words, shape, rest = _launch.planned(key) or _plan_latent(
        key, q, cache, block_table, lengths, cu_seqlens, tree_mask, o, lse, sm_scale)
    _launch.plain(q, cache, o, lse)
    if o is None:
        o = torch.empty(shape, dtype=q.dtype, device=dev)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    _launch.call("g9_latent_fwd", dev, q.data_ptr(), cache.data_ptr(), o.data_ptr(), ptr(lse), block_table.data_ptr(),
                 *table, lengths.data_ptr(), cu_seqlens.data_ptr(), ptr(tree_mask), words, *rest, ws.data_ptr(), need)
    return o


def _plan_latent(key, q, cache, block_table, lengths, cu_seqlens, tree_mask, o, lse, sm_scale):
    dev = _launch.gpu_of(q, cache, block_table, lengths, cu_seqlens, tree_mask, o, lse)
    T, H, D = _launch.rows_of("q", q)
    if D != RANK + ROPE or H == 0:
        raise ValueError(f"q must be (rows, heads, {RANK + ROPE}); got {tuple(q.shape)}")
    blocks, size = _cache(cache)
    B = _launch.offsets_of("cu_seqlens", cu_seqlens)
    _launch.int32_of("lengths", lengths, 1)
    _launch.int32_of("block_table", block_table, 2)
    if lengths.shape[0] != B or block_table.shape[0] != B:
        raise ValueError(f"cu_seqlens, lengths and block_table hold {B}, {lengths.shape[0]} and {block_table.shape[0]} requests")
    words = _launch.mask_words(tree_mask, T)
    if o is not None:
        _launch.rows_of("o", o)
        if o.shape != (T, H, RANK):
            raise ValueError(f"o is {tuple(o.shape)}, not {(T, H, RANK)}")
    dtype = _launch.dtype_of(q, cache, *([o] if o is not None else []))
    _launch.lse_fits(lse, H, T)
    os = _launch.array(H * RANK, RANK) if o is None else strides(o)
    return _launch.keep(key, dev, (
        dev, _lib.load().g9_latent_workspace_size(B, T, H), (block_table.stride(0), block_table.shape[1]), words,
        (T, H, RANK), (B, T, H, blocks, size, strides(q), strides(cache), os, sm_scale, dtype)))


def latent_varlen_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_rope: torch.Tensor,
                            cu_seqlens: torch.Tensor, o: torch.Tensor | None = None, *,
                            cu_seqlens_k: torch.Tensor | None = None, causal: bool = True,
                            sm_scale: float | None = None, lse: torch.Tensor | None = None) -> torch.Tensor:
    """Latent attention within each sequence of a packed batch, its keys and values
    expanded: softmax(sm_scale (q[..., :128] k^T + q[..., 128:] k_rope^T)) v.

    q is (T, HQ, 192), its last 64 values rotated; k and v are (TK, HK, 128), the
    latents times the heads' projections (slices of one product are read in place); k_rope (TK,
    64) the rotated keys that all heads share.  ``sm_scale`` is 192^-0.5 by default.
    Sequences, ``cu_seqlens_k``, ``causal``, ``o`` (T, HQ, 128), ``lse``, strides and the
    arithmetic as in ``varlen_attention``."""
    causal, sm_scale = bool(causal), None if sm_scale is None else float(sm_scale)
    key = ("latent_varlen", causal, sm_scale, sig(q), sig(k), sig(v), sig(k_rope), sig(cu_seqlens),
           cu_seqlens_k is not None and sig(cu_seqlens_k), o is not None and sig(o), lse is not None and sig(lse))
    dev, shape, rest = _launch.planned(key) or _plan_varlen(key, q, k, v, k_rope, cu_seqlens, cu_seqlens_k, o, lse, causal,
                                                            sm_scale)
    _launch.plain(q, k, v, k_rope, o, lse)
    if o is None:
        o = torch.empty(shape, dtype=q.dtype, device=dev)
    cu = cu_seqlens.data_ptr()
    _launch.call("g9_latent_varlen_fwd", dev, q.data_ptr(), k.data_ptr(), v.data_ptr(), k_rope.data_ptr(), o.data_ptr(),
                 ptr(lse), cu, cu if cu_seqlens_k is None else cu_seqlens_k.data_ptr(), *rest)
    return o


def _plan_varlen(key, q, k, v, k_rope, cu_seqlens, cu_seqlens_k, o, lse, causal, sm_scale):
    dev = _launch.gpu_of(q, k, v, k_rope, cu_seqlens, cu_seqlens_k, o, lse)
    T, HQ, D = _launch.rows_of("q", q)
    TK, HK, _ = _launch.rows_of("k", k)
    _launch.rows_of("v", v)
    if D != NOPE + ROPE or k.shape[2] != NOPE or v.shape != (TK, HK, VALUE) or _rows("k_rope", k_rope, ROPE) != TK:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}, k_rope {tuple(k_rope.shape)} do not "
                         f"fit; a head's key has {NOPE} values of its own and {ROPE} shared ones, its value {VALUE}")
    if HK == 0 or HQ == 0 or HQ % HK:
        raise ValueError(f"query heads {HQ} not a multiple of key/value heads {HK}")
    if cu_seqlens_k is None and TK != T:
        raise ValueError(f"{TK} keys for {T} queries need cu_seqlens_k")
    B = _launch.offsets_of("cu_seqlens", cu_seqlens)
    if cu_seqlens_k is not None and _launch.offsets_of("cu_seqlens_k", cu_seqlens_k) != B:
        raise ValueError("cu_seqlens and cu_seqlens_k hold different numbers of sequences")
    if o is not None:
        _launch.rows_of("o", o)
        if o.shape != (T, HQ, VALUE):
            raise ValueError(f"o is {tuple(o.shape)}, not {(T, HQ, VALUE)}")
    dtype = _launch.dtype_of(q, k, v, k_rope, *([o] if o is not None else []))
    _launch.lse_fits(lse, HQ, T)
    os = _launch.array(HQ * VALUE, VALUE) if o is None else strides(o)
    return _launch.keep(key, dev, (dev, (T, HQ, VALUE), (
        B, T, TK, HQ, HK, strides(q), strides(k), strides(v), k_rope.stride(0), os,
        (NOPE + ROPE) ** -0.5 if sm_scale is None else sm_scale, dtype, 1 if causal else 0)))
