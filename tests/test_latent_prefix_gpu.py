"""latent_varlen_attention of chunks behind prefixes, on both sides of where the prefix decides
the launch's form, against the float64 oracle."""

import numpy as np
import pytest
import torch

from gfx950_gluon_tutorials_amd.attention import latent_varlen_attention
from oracle import latent_ref as L
from oracle import serving_ref as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,n,prefix,HQ,HK", [(4, 100, 499, 64, 64), (4, 100, 500, 64, 64), (2, 33, 501, 320, 32), (20, 32, 510, 40, 8)])
def test_chunks_behind_prefixes(gpu, B, n, prefix, HQ, HK):
    g = torch.Generator().manual_seed(prefix)
    r = lambda *s: torch.randn(*s, generator=g).bfloat16()
    T, TK = B * n, B * (n + prefix)
    q, k, v, kr = r(T, HQ, 192), r(TK, HK, 128), r(TK, HK, 128), r(TK, 64)
    cq, ck = np.arange(B + 1) * n, np.arange(B + 1) * (n + prefix)
    i = lambda x: torch.tensor(x, dtype=torch.int32).to(gpu)
    got = latent_varlen_attention(*(t.to(gpu) for t in (q, k, v, kr)), i(cq), cu_seqlens_k=i(ck))
    torch.cuda.synchronize()
    f = lambda t: t.float().numpy()
    ref, lse, mag, spread = L.packed(f(q), f(k), f(v), f(kr), cq, ck, True, 192**-0.5)
    to, _ = R.tolerances(ref, lse, mag, spread, torch.finfo(torch.bfloat16).eps, n + prefix, 192, float(v.abs().max()), 0.0)
    off = np.abs(f(got.cpu()) - ref) - to
    assert (off <= 0).all(), f"{off.max():.3g} past its bound"
