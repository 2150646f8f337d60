"""Flash-attention forward for gfx950: the drop-in for the reference's
``kernels/attention`` launchers (``fmha_v3.run_gluon_attention``,
``fmha_v4.run_gluon_attention``) and their host-side helpers (``common``).

Beside it, without reference counterparts, the attention of a serving loop:
``varlen_attention`` over packed prompts, and a paged cache with
``assign_slots``, ``write_cache`` and ``tree_attention`` (``paged``).

The kernels are hand-written HIP behind include/gfx950_fmha.h.
"""

from .common import MetaData, compute_flops, get_shape_from_layout, get_strides_from_layout, input_helper
from .fmha_v4 import run_gluon_attention
from .paged import Slots, assign_slots, tree_attention, write_cache
from .varlen import varlen_attention

__all__ = [
    "MetaData",
    "Slots",
    "assign_slots",
    "compute_flops",
    "get_shape_from_layout",
    "get_strides_from_layout",
    "input_helper",
    "run_gluon_attention",
    "tree_attention",
    "varlen_attention",
    "write_cache",
]
