"""Launch of the gfx950 attention kernels from torch tensors: argument checks
(for ``g9_fmha_fwd`` those of the reference launchers), then one call through
the C ABI on the current stream.  No fallback: without the built library the
call raises."""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from .. import _lib
from .common import get_shape_from_layout, get_strides_from_layout

BLOCK_N = 64  # keys per tile: the sequence length must be a multiple of it
HEAD_DIMS = (64, 128)
_DTYPES = {torch.float16: _lib.G9_F16, torch.bfloat16: _lib.G9_BF16}


def fmha_forward(q, k, v, o, metadata, scale_on_q: bool, variant: int, lse=None) -> None:
    """Writes softmax(q k^T * sm_scale) v into ``o``.

    The checks follow run_gluon_attention (kernels/attention/fmha_v4.py:761-775):
    non-causal only, K sequence length a multiple of 64, Q and K sequence
    lengths equal (assertions there and here); beyond those this kernel needs
    head dim 64 or 128 and 16-bit tensors on one GPU (ValueError).  ``lse``, if
    given, is a contiguous fp32 (batch, query heads, seq) tensor that receives
    each query's natural-log log-sum-exp of its scaled scores."""
    assert not metadata.causal, "the gfx950 FMHA kernel supports non-causal attention only"
    assert metadata.max_seqlens_k % BLOCK_N == 0, "K seqlen must be a multiple of BLOCK_N (64)"
    assert metadata.max_seqlens_q == metadata.max_seqlens_k, "combined N_CTX requires Q seqlen == K seqlen"
    batch, nheads_q, nheads_k, head_size = get_shape_from_layout(q, k, metadata)
    assert head_size & (head_size - 1) == 0, "head dim must be a power of two"
    if head_size not in HEAD_DIMS:
        raise ValueError(f"head dim {head_size} unsupported: the gfx950 kernels are built for {HEAD_DIMS}")
    if q.dtype not in _DTYPES or any(t.dtype != q.dtype for t in (k, v, o)):
        raise ValueError(f"q, k, v, o must share one of {list(_DTYPES)}; got {[t.dtype for t in (q, k, v, o)]}")
    dev = q.device
    if dev.type != "cuda" or any(t.device != dev for t in (k, v, o)):
        raise ValueError("q, k, v, o must be on one GPU")
    S = metadata.max_seqlens_q
    order = (0, 1, 2, 3) if metadata.layout == "bhsd" else (0, 2, 1, 3)
    want_q = (batch, nheads_q, S, head_size)
    want_k = (batch, nheads_k, S, head_size)
    for name, t, want in (("q", q, want_q), ("k", k, want_k), ("v", v, want_k), ("o", o, want_q)):
        got = tuple(t.shape[i] for i in order)
        if got != want:
            raise ValueError(f"{name} has (batch, head, seq, dim) {got}, expected {want}")
    if nheads_q % nheads_k != 0:
        raise ValueError(f"query heads {nheads_q} not a multiple of key/value heads {nheads_k}")
    if lse is not None:
        if (lse.dtype != torch.float32 or not lse.is_contiguous() or tuple(lse.shape) != (batch, nheads_q, S)
                or lse.device != dev):
            raise ValueError("lse must be a contiguous fp32 (batch, query heads, seq) tensor on the same GPU")
    strides = get_strides_from_layout(q, k, v, o, metadata)
    arr = [(_lib.ctypes.c_int64 * 4)(*st) for st in strides]
    lib = _lib.load()
    args = (q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr() if lse is not None else None, batch,
            nheads_q, nheads_k, S, head_size, arr[0], arr[1], arr[2], arr[3], float(metadata.sm_scale),
            _DTYPES[q.dtype], 1 if scale_on_q else 0, variant, torch._C._cuda_getCurrentRawStream(dev.index))
    if torch._C._cuda_getDevice() == dev.index:
        rc = lib.g9_fmha_fwd(*args)
    else:
        with torch.cuda.device(dev):
            rc = lib.g9_fmha_fwd(*args)
    _lib.check(rc, "g9_fmha_fwd")


# --- packed and paged attention -----------------------------------------------


def ptr(t):
    return t.data_ptr() if t is not None else None


def array(*values):
    return (_lib.ctypes.c_int64 * len(values))(*values)


def strides(t):
    """Element strides but the last dimension's."""
    return array(*t.stride()[:-1])


def gpu_of(first, *others) -> torch.device:
    """The one GPU that holds every given tensor."""
    dev = first.device
    if dev.type != "cuda" or any(t is not None and t.device != dev for t in others):
        raise ValueError(f"all tensors must be on one GPU; got {[str(t.device) for t in (first, *others) if t is not None]}")
    return dev


def rows_of(name, t) -> tuple[int, int, int]:
    if t.dim() != 3 or t.stride(2) != 1:
        raise ValueError(f"{name} must be (rows, heads, head dim) with a unit head-dim stride; got {tuple(t.shape)}, "
                         f"strides {t.stride()}")
    return t.shape


def offsets_of(name, t) -> int:
    """The number of sequences of a cu_seqlens tensor."""
    if t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] < 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of sequences + 1 values")
    return t.shape[0] - 1


def int32_of(name, t, dims) -> None:
    """Rows of contiguous int32 values."""
    if t.dtype != torch.int32 or t.dim() != dims or (t.stride(-1) != 1 and t.shape[-1] > 1):
        raise ValueError(f"{name} must be a {dims}-dimensional int32 tensor with contiguous rows; got {t.dtype} "
                         f"{tuple(t.shape)}, strides {t.stride()}")


def heads_fit(HQ, HK, D) -> None:
    if HK == 0 or HQ == 0 or HQ % HK:
        raise ValueError(f"query heads {HQ} not a multiple of key/value heads {HK}")
    if D not in HEAD_DIMS:
        raise ValueError(f"head dim {D} unsupported: the gfx950 kernels are built for {HEAD_DIMS}")


def dtype_of(first, *others) -> int:
    if first.dtype not in _DTYPES or any(t.dtype != first.dtype for t in others):
        raise ValueError(f"the tensors must share one of {list(_DTYPES)}; got {[t.dtype for t in (first, *others)]}")
    return _DTYPES[first.dtype]


def lse_fits(lse, HQ, T) -> None:
    if lse is not None and (lse.dtype != torch.float32 or lse.shape != (HQ, T) or not lse.is_contiguous()):
        raise ValueError("lse must be a contiguous fp32 (query heads, rows) tensor")


def mask_words(tree_mask, T) -> int:
    """64-bit words of a node's row of a tree mask, 0 without one."""
    if tree_mask is None:
        return 0
    if tree_mask.dtype != torch.int64 or tree_mask.dim() not in (1, 2) or not tree_mask.is_contiguous():
        raise ValueError("tree_mask must be a contiguous int64 (T, words) or (T,) tensor")
    words = 1 if tree_mask.dim() == 1 else tree_mask.shape[1]
    if tree_mask.shape[0] != T or words == 0:
        raise ValueError(f"tree_mask {tuple(tree_mask.shape)} does not fit {T} rows")
    return words


def plain(*tensors) -> None:
    """Refuses what the kernels would silently lose: a gradient, a tangent, a pending negation."""
    dual = forward_ad._current_level >= 0
    for t in tensors:
        if t is None:
            continue
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError("forward only: call it under torch.no_grad(), or detach the tensors that require a gradient")
        if dual and forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError("forward only: a tensor has a forward-mode tangent; pass its primal")
        if t.is_neg():
            raise ValueError("a lazily negated view: call resolve_neg() first")


# What a call's arguments are but for their addresses and contents, to the
# arguments of the C call that follow from it: a call of the same kind as an
# earlier one is not checked again (a call's host time: write_cache 8.5 us instead of
# 13.8, varlen_attention 10.8 instead of 16.7, decoding 16.8 instead of 24.5).
_plans: dict = {}


def sig(t):
    return (t.shape, t.stride(), t.dtype, t.get_device())


def planned(key):
    return _plans.get(key)


def keep(key, dev, plan):
    if dev.type == "cuda":
        if len(_plans) >= 4096:
            _plans.clear()
        _plans[key] = plan
    return plan


def call(entry: str, dev: torch.device, *args) -> None:
    """One C call on the current stream of `dev`."""
    fn = getattr(_lib.load(), entry)
    stream = torch._C._cuda_getCurrentRawStream(dev.index)
    if torch._C._cuda_getDevice() == dev.index:
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, stream)
    if rc:
        _lib.check(rc, entry)
