"""Attention over packed sequences of different lengths: whole prompts in one
call, causal or not, with grouped K/V heads (``g9_varlen_fwd``,
include/gfx950_fmha.h).  No reference counterpart: its attention is
non-causal over equal lengths."""

from __future__ import annotations

import torch

from . import _launch
from ._launch import ptr, strides


def varlen_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                     o: torch.Tensor | None = None, *, cu_seqlens_k: torch.Tensor | None = None, causal: bool = True,
                     sm_scale: float | None = None, lse: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(q k^T * sm_scale) v within each sequence of a packed batch.

    q is (T, HQ, D), k and v are (TK, HK, D) with HQ a multiple of HK, fp16 or
    bf16, head dim 64 or 128; any strides with a unit head-dim stride and steps
    of 16 bytes, so slices of one fused q/k/v projection are read in place.
    ``cu_seqlens`` (B + 1, int32, on the GPU) holds the sequences' row offsets in
    q, and in k and v unless ``cu_seqlens_k`` gives theirs.  With ``causal`` query
    i of Lq reads the keys j <= i + Lk - Lq: where a prompt's first part is
    cached already, its new queries read all of it.  A query without a key gives
    zeros (lse -inf).

    Returns ``o`` (T, HQ, D), allocated when not given; rows behind the last
    sequence are left as they were.  ``lse``, if given, is a contiguous fp32
    (HQ, T) tensor that receives each query's natural-log log-sum-exp.
    Asynchronous on the current stream; forward only."""
    dev = _launch.gpu_of(q, k, v, cu_seqlens, cu_seqlens_k, o, lse)
    T, HQ, D = _launch.rows_of("q", q)
    TK, HK, _ = _launch.rows_of("k", k)
    if k.shape != v.shape or k.shape[2] != D:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} do not fit")
    if cu_seqlens_k is None:
        if TK != T:
            raise ValueError(f"{TK} keys for {T} queries need cu_seqlens_k")
        cu_seqlens_k = cu_seqlens
    B = _launch.offsets_of("cu_seqlens", cu_seqlens)
    if _launch.offsets_of("cu_seqlens_k", cu_seqlens_k) != B:
        raise ValueError("cu_seqlens and cu_seqlens_k hold different numbers of sequences")
    _launch.heads_fit(HQ, HK, D)
    if o is None:
        o = torch.empty((T, HQ, D), dtype=q.dtype, device=dev)
    elif o.shape != q.shape:
        raise ValueError(f"o is {tuple(o.shape)}, q {tuple(q.shape)}")
    dtype = _launch.dtype_of(q, k, v, o)
    _launch.lse_fits(lse, HQ, T)
    _launch.forward_only(q, k, v)
    _launch.call("g9_varlen_fwd", dev, ptr(q), ptr(k), ptr(v), ptr(o), ptr(lse), ptr(cu_seqlens), ptr(cu_seqlens_k),
                 B, T, TK, HQ, HK, D, strides(q), strides(k), strides(v), strides(o),
                 D**-0.5 if sm_scale is None else float(sm_scale), dtype, 1 if causal else 0)
    return o
