"""Rotary positions (``g9_rotary``, include/gfx950_fmha.h): the pairs of a query's or
key's values turned by angles that grow with its position.  No reference
counterpart."""

from __future__ import annotations

import math

import torch

from . import _launch
from ._launch import sig, strides

SCALINGS = (None, "linear", "base", "turns", "index")


def rotary_frequencies(dim: int, base: float = 10000.0, *, scaling: str | None = None, factor: float = 1.0,
                       original_length: int | None = None, fast: float = 32.0, slow: float = 1.0,
                       device=None) -> torch.Tensor:
    """The dim / 2 frequencies f_i = base^(-2 i / dim) in radians a position, float64.

    ``scaling`` stretches them for contexts ``factor`` times as long as the
    ``original_length`` that a model was trained with:

    * ``"linear"``: f_i / factor (positions interpolated);
    * ``"base"``: base * factor^(dim / (dim - 2)) in place of base: the slowest pair
      is slowed by the factor, the fastest kept;
    * ``"turns"``: f_i (w + (1 - w) / factor), w falling from 1 for pairs that turn
      ``fast`` times or more over the original length to 0 for those that turn
      ``slow`` times or less, linearly in the turns;
    * ``"index"``: the same with w linear in the pair's index, between the indexes
      (rounded outward) whose pairs turn ``fast`` and ``slow`` times."""
    if dim < 2 or dim % 2:
        raise ValueError(f"dim is {dim}: an even number of values is turned")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling {scaling!r} is none of {SCALINGS}")
    if not (base > 0 and factor > 0 and math.isfinite(base) and math.isfinite(factor)):
        raise ValueError(f"base {base} and factor {factor} must be positive")
    if scaling in ("turns", "index") and not (original_length and original_length > 0 and fast > slow > 0):
        raise ValueError(f"scaling {scaling!r} needs the original length and fast > slow > 0")
    if scaling == "index" and base <= 1:
        raise ValueError("scaling 'index' needs a base above 1")
    if scaling == "base":
        if dim == 2:
            raise ValueError("scaling 'base' needs more than one pair")
        base = base * factor ** (dim / (dim - 2))
    f = [base ** (-2 * i / dim) for i in range(dim // 2)]
    if scaling == "linear":
        f = [x / factor for x in f]
    elif scaling in ("turns", "index"):
        if scaling == "turns":
            w = [(original_length * x / (2 * math.pi) - slow) / (fast - slow) for x in f]
        else:
            def index(turns):
                return dim * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))

            lo, hi = max(math.floor(index(fast)), 0), min(math.ceil(index(slow)), dim - 1)
            w = [1 - (i - lo) / max(hi - lo, 1e-3) for i in range(dim // 2)]
        w = [min(max(x, 0.0), 1.0) for x in w]
        f = [x * (y + (1 - y) / factor) for x, y in zip(f, w)]
    return torch.tensor(f, dtype=torch.float64, device=device)


def check_turns(name, rows, positions, freqs, pairs=None) -> None:
    """Positions (rows,) int64 and frequencies (pairs,) float64."""
    if positions.dtype != torch.int64 or positions.shape != (rows,) or not positions.is_contiguous():
        raise ValueError(f"positions must be {rows} contiguous int64 values, one for each row of {name}")
    if freqs.dtype != torch.float64 or freqs.dim() != 1 or not freqs.is_contiguous():
        raise ValueError("freqs must be contiguous float64 values (rotary_frequencies)")
    if pairs is not None and freqs.shape[0] != pairs:
        raise ValueError(f"{freqs.shape[0]} frequencies for {pairs} pairs")


def rotary(x: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, o: torch.Tensor | None = None, *,
           first: int = 0, interleaved: bool = False, inverse: bool = False, scale: float = 1.0) -> torch.Tensor:
    """Turns the pairs of x (T, H, D) by ``positions[t] * freqs[i]``.

    Of each row the 2 * len(freqs) values from ``first`` on are turned and multiplied
    by ``scale`` (a magnitude correction for long contexts), the others copied.
    Pair i is (x[first + i], x[first + len(freqs) + i]), or with ``interleaved``
    neighbours (x[first + 2 i], x[first + 2 i + 1]).  ``positions`` (T,) int64, as
    ``assign_slots`` gives them; ``freqs`` float64 (``rotary_frequencies``): angles
    are formed in 64 bits, so far positions lose nothing.  Turned in fp32, rounded
    once.

    With ``inverse`` the pairs are turned back (and multiplied by ``scale`` as before).
    That is the operator's backward pass: ``rotary(grad_o, positions, freqs,
    inverse=True, ...)`` with the other arguments the same is the gradient of x.

    fp16 or bf16; any strides with a unit last one and steps of 16 bytes: the query
    and key heads of one fused projection are one x.  D and ``first`` are multiples of
    8, len(freqs) too.  Returns ``o``, allocated when not given; ``o`` may be x itself
    (in place) and must not overlap it otherwise.  Asynchronous on the current stream;
    tensors that require a gradient are refused while gradients are enabled."""
    first, interleaved, inverse, scale = int(first), bool(interleaved), bool(inverse), float(scale)
    key = ("rotary", first, interleaved, inverse, scale, sig(x), sig(positions), sig(freqs), o is not None and sig(o))
    dev, rest = _launch.planned(key) or _plan(key, x, positions, freqs, o, first, interleaved, inverse, scale)
    _launch.plain(x, o, freqs)
    if o is None:
        o = torch.empty(x.shape, dtype=x.dtype, device=dev)
    _launch.call("g9_rotary", dev, x.data_ptr(), o.data_ptr(), positions.data_ptr(), freqs.data_ptr(), *rest)
    return o


def _plan(key, x, positions, freqs, o, first, interleaved, inverse, scale):
    dev = _launch.gpu_of(x, positions, freqs, o)
    T, H, D = _launch.rows_of("x", x)
    check_turns("x", T, positions, freqs)
    dim = 2 * freqs.shape[0]
    if first < 0 or first % 8 or D % 8 or dim == 0 or dim % 16 or first + dim > D:
        raise ValueError(f"{dim} values from {first} on of rows of {D}: row length and first must be multiples of 8, the "
                         "turned values a multiple of 16 within the row")
    if not math.isfinite(scale):
        raise ValueError(f"scale is {scale}")
    if o is not None:
        _launch.rows_of("o", o)
        if o.shape != x.shape:
            raise ValueError(f"o is {tuple(o.shape)}, x {tuple(x.shape)}")
    dtype = _launch.dtype_of(x, *([o] if o is not None else []))
    os = _launch.array(H * D, D) if o is None else strides(o)
    return _launch.keep(key, dev, (dev, (T, H, D, first, dim, strides(x), os, scale, interleaved, inverse, dtype)))
