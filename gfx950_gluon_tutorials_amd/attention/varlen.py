"""Attention over packed sequences of different lengths: whole prompts in one
call, causal or not, with grouped K/V heads (``g9_varlen_fwd``,
include/gfx950_fmha.h).  No reference counterpart: its attention is
non-causal over equal lengths."""

from __future__ import annotations

import torch

from . import _launch
from ._launch import ptr, sig, strides


def varlen_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                     o: torch.Tensor | None = None, *, cu_seqlens_k: torch.Tensor | None = None, causal: bool = True,
                     sm_scale: float | None = None, lse: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(q k^T * sm_scale) v within each sequence of a packed batch.

    q is (T, HQ, D), k and v are (TK, HK, D) with HQ a multiple of HK, fp16 or
    bf16, head dim 64 or 128; any strides with a unit head-dim stride and steps
    of 16 bytes, below 8 MiB a token, so slices of one fused q/k/v projection, and
    expanded or overlapping q, k and v, are read in place.
    ``cu_seqlens`` (B + 1, int32, on the GPU) holds the sequences' row offsets in
    q, and in k and v unless ``cu_seqlens_k`` gives theirs.  With ``causal`` query
    i of Lq reads the keys j <= i + Lk - Lq: where a prompt's first part is
    cached already, its new queries read all of it (a sequence's keys are not divided
    among workgroups here: few queries behind thousands of keys are faster through
    ``tree_attention``, which does that).  A query without a key gives zeros (lse
    -inf).

    Returns ``o`` (T, HQ, D), allocated when not given; rows behind the last
    sequence are left as they were.  ``lse``, if given, is a contiguous fp32
    (HQ, T) tensor that receives each query's natural-log log-sum-exp.
    Scores, softmax and sums are fp32, each weight is rounded to the input type for
    its product with v; scaled scores up to 2^26 in magnitude.  Asynchronous on the
    current stream; forward only."""
    causal, sm_scale = bool(causal), None if sm_scale is None else float(sm_scale)
    key = ("varlen", causal, sm_scale, sig(q), sig(k), sig(v), sig(cu_seqlens), cu_seqlens_k is not None and sig(cu_seqlens_k),
           o is not None and sig(o), lse is not None and sig(lse))
    dev, rest = _launch.planned(key) or _plan(key, q, k, v, cu_seqlens, cu_seqlens_k, o, lse, causal, sm_scale)
    _launch.plain(q, k, v, o, lse)
    if o is None:
        o = torch.empty(q.shape, dtype=q.dtype, device=dev)
    cu = cu_seqlens.data_ptr()
    _launch.call("g9_varlen_fwd", dev, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), ptr(lse), cu,
                 cu if cu_seqlens_k is None else cu_seqlens_k.data_ptr(), *rest)
    return o


def _plan(key, q, k, v, cu_seqlens, cu_seqlens_k, o, lse, causal, sm_scale):
    """The checks, and the C call's arguments behind the pointers."""
    dev = _launch.gpu_of(q, k, v, cu_seqlens, cu_seqlens_k, o, lse)
    T, HQ, D = _launch.rows_of("q", q)
    TK, HK, _ = _launch.rows_of("k", k)
    _launch.rows_of("v", v)
    if k.shape != v.shape or k.shape[2] != D:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} do not fit")
    if cu_seqlens_k is None and TK != T:
        raise ValueError(f"{TK} keys for {T} queries need cu_seqlens_k")
    B = _launch.offsets_of("cu_seqlens", cu_seqlens)
    if cu_seqlens_k is not None and _launch.offsets_of("cu_seqlens_k", cu_seqlens_k) != B:
        raise ValueError("cu_seqlens and cu_seqlens_k hold different numbers of sequences")
    _launch.heads_fit(HQ, HK, D)
    if o is not None:
        _launch.rows_of("o", o)
        if o.shape != q.shape:
            raise ValueError(f"o is {tuple(o.shape)}, q {tuple(q.shape)}")
    dtype = _launch.dtype_of(q, k, v, *([o] if o is not None else []))
    _launch.lse_fits(lse, HQ, T)
    os = _launch.array(HQ * D, D) if o is None else strides(o)
    return _launch.keep(key, dev, (dev, (B, T, TK, HQ, HK, D, strides(q), strides(k), strides(v), os,
                                         D**-0.5 if sm_scale is None else sm_scale, dtype, 1 if causal else 0)))
