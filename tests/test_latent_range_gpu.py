"""Large scores against the float64 oracle: latent_attention over the whole range of finite
ones, the packed and paged forms up to 2^26.

The query has one value that is not zero, so a score is one exact product; keys come in
levels, whose scores differ by far more than an exponential can tell from zero.  A row's
result is then the mean of its highest level's values, all of one weight."""

import numpy as np
import pytest
import torch

from gfx950_gluon_tutorials_amd.attention import latent_attention, latent_varlen_attention, tree_attention, varlen_attention
from oracle import latent_ref as L
from oracle import serving_ref as R

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
# Scores (natural log), one for each 32 keys of the beginning and one for the rest.  fp16: by
# values up to 2^15 and a scale of 2^6.
RISING = [-1.4e38, -1.1e38, -6e37, -1e30, 1e20, 1.5e38]
LEVELS = {
    "bf16": [[-1.4e38, 0.0], [-1.4e38], [-2.3e38], [2.3e38], [0.0, -1.4e38], RISING, RISING[::-1], [-2.2e38, -1.4e38],
             [-3e9, 5e9, 4e9], [2.0**24, 2.0**25 + 2.0**20]],
    "fp16": [[-2.0**34, -2.0**33 - 2.0**30], [2.0**28], [-2.0**29 - 2.0**22], [2.0**34, 2.0**33, 2.0**34 + 2.0**26]],
}


def _case(dev, dtype, levels, context, nodes, H, sign, size=16):
    """Heads of which every second sees the scores negated, where `sign` is -1."""
    g = torch.Generator().manual_seed(context + H)
    a, scale = (2.0**60, 1.0) if dtype == "bf16" else (2.0**14, 2.0**6)
    n = context + nodes
    per_key = [levels[min(j // 32, len(levels) - 1)] / (a * scale) for j in range(n)]
    rows = torch.randn(n, 576, generator=g).to(DT[dtype])
    rows[:, 512] = torch.tensor(per_key, dtype=torch.float64).to(DT[dtype])
    used = -(-n // size)
    table = torch.randperm(used + 2, generator=g)[:used]
    cache = torch.randn(used + 2, size, 576, generator=g).to(DT[dtype])
    at = torch.arange(n)
    cache[table[at // size], at % size] = rows
    q = torch.zeros(nodes, H, 576, dtype=DT[dtype])
    q[:, 0::2, 512] = a
    q[:, 1::2, 512] = a * sign
    assert q.isfinite().all() and cache.isfinite().all()
    return q.to(dev), cache.to(dev), table[None].int().to(dev), scale


def _check(dev, dtype, levels, context, nodes, H, sign):
    q, cache, table, scale = _case(dev, dtype, levels, context, nodes, H, sign)
    lse = torch.empty(H, nodes, device=dev)
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)
    got = latent_attention(q, cache, table, i(context), i(0, nodes), sm_scale=scale, lse=lse)
    torch.cuda.synchronize()
    n = lambda t: t.double().cpu().numpy()
    # The heads are of two kinds.
    want, lse_want, mag, _ = L.paged(n(q)[:, :2], n(cache), table.cpu().numpy(), [context], [0, nodes], None, scale)
    kind = np.arange(H) % 2
    want, lse_want, mag = want[:, kind], lse_want[kind], mag[:, kind]
    # Weights of 1 and 0 are exact.  Their sum over the keys is fp32, its quotient and two products
    # are 2^-22 at most; then half a step.  lse: its maximum is a product with the scale by log2 e,
    # itself rounded twice, a sum, and a product with ln 2, rounded too: seven times 2^-24 at most.
    h = torch.finfo(DT[dtype]).eps / 2
    tol = h * np.abs(want) * (1 + h) + ((context + nodes) * 2.0**-24 + 2.0**-22) * (1 + h) * mag
    tol += 2.0**-25 if dtype == "fp16" else 0
    off = np.abs(n(got) - want)
    assert (off <= tol).all(), f"{(off - tol).max():.3g} past its bound, or not finite"
    assert (np.abs(n(lse) - lse_want) <= 2.0**-21 * np.abs(lse_want) + 1e-6).all()


@pytest.mark.parametrize("H,nodes", [(1, 1), (16, 1), (40, 1), (128, 1), (16, 9)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_scores_of_any_finite_size(gpu, dtype, H, nodes):
    for levels in LEVELS[dtype]:
        for context in (1, 33, 100, 1000):
            for sign in (1, -1):
                _check(gpu, dtype, levels, context, nodes, H, sign)


def test_scores_of_any_finite_size_in_many_parts(gpu):
    for H in (16, 128):
        for levels in (RISING, RISING[::-1], [-1.4e38, 0.0]):
            _check(gpu, "bf16", levels, 20000, 1, H, -1)


@pytest.mark.parametrize("H", [16, 64, 128])
def test_large_scores_leave_the_other_rows_as_they_are(gpu, H):
    """Rows of one wave: the others' bits do not depend on them."""
    g = torch.Generator().manual_seed(H)
    cache = torch.randn(70, 16, 576, generator=g).bfloat16().to(gpu)
    q = (torch.randn(1, H, 576, generator=g) * 0.6).bfloat16().to(gpu)
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device=gpu)
    run = lambda: latent_attention(q, cache, torch.arange(70, dtype=torch.int32, device=gpu)[None], i(1000), i(0, 1), sm_scale=192**-0.5)
    clean = run().clone()
    for size in (2.0**40, 2.0**100, float("inf")):
        q[:, 3::32] = size
        got, rest = run(), torch.arange(H) % 32 != 3
        assert torch.equal(got[:, rest], clean[:, rest]) and got[:, 3::32].isfinite().all() == (size < float("inf"))


# --- the packed forms and the paged cache of keys and values --------------------------------

UP_TO_2_26 = [[2.0**26], [-2.0**26], [-2.0**26, -2.0**26 + 2.0**20], [2.0**26, 2.0**25 + 2.0**22, 2.0**26],
              [-2.0**26, -2.0**25, -2.0**23, 0.0, 2.0**22, 2.0**26]]


@pytest.mark.parametrize("form", ["latent", "d128", "d64", "tree"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_scores_up_to_2_26(gpu, dtype, form):
    """Queries and heads on both sides of where the launches change their form."""
    a, scale = (2.0**20, 1.0) if dtype == "bf16" else (2.0**14, 2.0**-3)
    D, VD = {"latent": (192, 128), "d64": (64, 64)}.get(form, (128, 128))
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device=gpu)
    n = lambda t: t.double().cpu().numpy()
    for T, H in ((197, 2), (1400, 32)) if form != "tree" else ((1, 16), (9, 32)):
        g = torch.Generator().manual_seed(T)
        TK = T if form != "tree" else 700
        for at, levels in enumerate(UP_TO_2_26):
            q, k = torch.zeros(T, H, D, dtype=DT[dtype]), torch.randn(TK, H, D, generator=g).to(DT[dtype])
            v = torch.randn(TK, H, VD, generator=g).to(DT[dtype])
            q[:, 0::2, 0], q[:, 1::2, 0] = a, -a
            per_key = [levels[min(j // 64, len(levels) - 1)] / (a * scale) for j in range(TK)]
            k[..., 0] = torch.tensor(per_key, dtype=torch.float64).to(DT[dtype])[:, None]
            lse, causal = torch.empty(H, T, device=gpu), form == "tree" or at % 2 == 0
            qd, kd, vd = q.to(gpu), k.to(gpu), v.to(gpu)
            kw = dict(sm_scale=scale, lse=lse)
            if form == "latent":
                got = latent_varlen_attention(qd, kd[..., :128], vd, torch.zeros(TK, 64, dtype=DT[dtype], device=gpu), i(0, T),
                                              causal=causal, **kw)
            elif form == "tree":
                pages = torch.zeros(2, 704, H, 128, dtype=DT[dtype], device=gpu)
                pages[0, :TK], pages[1, :TK] = kd, vd
                pages = pages.view(2, 44, 16, H, 128)
                got = tree_attention(qd, pages[0], pages[1], torch.arange(44, dtype=torch.int32, device=gpu)[None], i(TK - T), i(0, T), **kw)
            else:
                got = varlen_attention(qd, kd, vd, i(0, T), causal=causal, **kw)
            torch.cuda.synchronize()
            # Two heads of each kind against the oracle, which has no shared keys here.
            reads = R.causal_reads(T, TK, causal)
            want, lse_want, mag, _ = L.attend(n(q)[:, :4], n(k)[:, :4], n(v)[:, :4], reads, scale)
            # All weights alike, 2^x with |x| at most 4 (half a step of the maximum): each half a step, the
            # sum over the keys, the quotient.
            h = torch.finfo(DT[dtype]).eps / 2
            tol = h * np.abs(want) * (1 + h) + (h + TK * 2.0**-24 + 2.0**-20) * (1 + h) * mag + (2.0**-25 if dtype == "fp16" else 0)
            off = np.abs(n(got)[:, :4] - want)
            assert (off <= tol).all(), f"{T} by {H}, {levels}: {(off - tol).max():.3g} past its bound, or not finite"
            assert np.isfinite(n(got)).all()
            assert (np.abs(n(lse)[:4] - lse_want) <= 2.0**-21 * np.abs(lse_want) + 1e-5).all()
