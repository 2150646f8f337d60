"""CPU checks of rotary positions and latent attention: what the Python functions and
the C entries refuse (before anything reaches a GPU), what they pass on, and the
frequencies."""

import ctypes
import math

import numpy as np
import pytest
import torch

from gfx950_gluon_tutorials_amd import _lib
from gfx950_gluon_tutorials_amd.attention import (_launch, latent_attention, latent_varlen_attention, rotary,
                                                  rotary_frequencies, write_latent)
from oracle import latent_ref as L
from oracle import serving_ref as R

FAKE = 0x10000  # 16-byte aligned non-null address; never dereferenced on these paths


@pytest.fixture
def calls(monkeypatch):
    """The C calls that the functions would make of CPU tensors."""
    out = []
    monkeypatch.setattr(_launch, "gpu_of", lambda first, *rest: torch.device("cpu"))
    monkeypatch.setattr(_launch, "call", lambda entry, dev, *args: out.append((entry, args)))
    return out


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32)


def _bf(*shape):
    return torch.zeros(*shape).bfloat16()


def _rotary(**kw):
    a = dict(x=_bf(6, 4, 64), positions=torch.arange(6), freqs=rotary_frequencies(32))
    a.update(kw)
    return rotary(**a)


def _write(**kw):
    a = dict(c=_bf(6, 512), k_rope=_bf(6, 64), cache=_bf(3, 16, 576), slots=torch.arange(6))
    a.update(kw)
    return write_latent(**a)


def _paged(**kw):
    a = dict(q=_bf(6, 4, 576), cache=_bf(3, 16, 576), block_table=torch.zeros(2, 2, dtype=torch.int32), lengths=_i32(3, 4),
             cu_seqlens=_i32(0, 2, 6), sm_scale=0.1)
    a.update(kw)
    return latent_attention(**a)


def _prompt(**kw):
    a = dict(q=_bf(6, 4, 192), k=_bf(6, 2, 128), v=_bf(6, 2, 128), k_rope=_bf(6, 64), cu_seqlens=_i32(0, 6))
    a.update(kw)
    return latent_varlen_attention(**a)


def test_good_calls_reach_their_entries(calls):
    assert _rotary().shape == (6, 4, 64)
    x = _bf(6, 4, 64)
    assert _rotary(x=x, o=x, first=16, interleaved=True, inverse=True, scale=2) is x
    assert _write() is None
    _write(weight=_bf(512), positions=torch.arange(6), freqs=rotary_frequencies(64), c_out=_bf(6, 512), k_out=_bf(6, 64))
    assert _paged().shape == (6, 4, 512)
    _paged(tree_mask=torch.zeros(6, dtype=torch.int64))
    _paged(tree_mask=torch.zeros(6, 2, dtype=torch.int64), lse=torch.zeros(4, 6), o=_bf(6, 4, 512))
    assert _prompt().shape == (6, 4, 128)
    _prompt(cu_seqlens_k=_i32(0, 4), k=_bf(4, 2, 128), v=_bf(4, 2, 128), k_rope=_bf(4, 64))
    assert [c[0] for c in calls] == (["g9_rotary"] * 2 + ["g9_write_latent"] * 2 + ["g9_latent_fwd"] * 3
                                     + ["g9_latent_varlen_fwd"] * 2)
    assert 192**-0.5 in calls[-2][1]


@pytest.mark.parametrize("kw", [
    dict(x=torch.zeros(6, 4, 64)), dict(x=_bf(6, 64)), dict(x=_bf(6, 4, 128)[..., ::2]), dict(x=_bf(6, 4, 60)),
    dict(positions=torch.arange(5)), dict(positions=torch.arange(6).int()), dict(positions=torch.arange(12)[::2]),
    dict(freqs=rotary_frequencies(32).float()), dict(freqs=rotary_frequencies(128)), dict(freqs=rotary_frequencies(24)),
    dict(freqs=rotary_frequencies(64)[::2]), dict(freqs=torch.zeros(0, dtype=torch.float64)), dict(first=4), dict(first=40),
    dict(first=-8), dict(scale=math.nan), dict(scale=math.inf), dict(o=_bf(6, 4, 128)), dict(o=torch.zeros(6, 4, 64).half()),
    dict(x=_bf(6, 4, 64).requires_grad_()),
])
def test_rotary_refuses(calls, kw):
    with pytest.raises(ValueError):
        _rotary(**kw)
    assert not calls


@pytest.mark.parametrize("kw", [
    dict(c=_bf(6, 256)), dict(c=_bf(512, 6).t()), dict(k_rope=_bf(5, 64)), dict(k_rope=_bf(6, 32)), dict(cache=_bf(3, 16, 512)),
    dict(cache=_bf(3, 16, 1, 576)), dict(cache=torch.zeros(3, 16, 576).half()), dict(slots=torch.arange(6).int()),
    dict(slots=torch.arange(5)), dict(slots=torch.arange(12)[::2]), dict(weight=_bf(64)), dict(weight=torch.zeros(512)),
    dict(positions=torch.arange(6)), dict(freqs=rotary_frequencies(64)),
    dict(positions=torch.arange(6), freqs=rotary_frequencies(32)), dict(c_out=_bf(5, 512)), dict(k_out=_bf(6, 128)),
    dict(c_out=torch.zeros(6, 512)), dict(eps=-1.0), dict(eps=math.nan), dict(scale=math.inf), dict(c=_bf(6, 512).requires_grad_()),
    dict(weight=_bf(512).requires_grad_()),
])
def test_write_refuses(calls, kw):
    with pytest.raises(ValueError):
        _write(**kw)
    assert not calls


@pytest.mark.parametrize("kw", [
    dict(q=_bf(6, 4, 512)), dict(q=_bf(6, 0, 576)), dict(q=torch.zeros(6, 4, 576).half()), dict(q=torch.zeros(6, 4, 576), cache=torch.zeros(3, 16, 576)),
    dict(cache=_bf(3, 16, 512)), dict(cache=_bf(3, 16, 1152)[..., ::2]), dict(block_table=torch.zeros(3, 2, dtype=torch.int32)),
    dict(block_table=torch.zeros(2, 2, dtype=torch.int64)), dict(block_table=torch.zeros(2, 4, dtype=torch.int32)[:, ::2]),
    dict(lengths=_i32(3)), dict(lengths=torch.tensor([3, 4])), dict(cu_seqlens=torch.tensor([0, 2, 6])),
    dict(tree_mask=torch.zeros(6, dtype=torch.int32)), dict(tree_mask=torch.zeros(5, dtype=torch.int64)),
    dict(tree_mask=torch.zeros(6, 0, dtype=torch.int64)), dict(o=_bf(6, 4, 576)), dict(lse=torch.zeros(6, 4)),
    dict(lse=torch.zeros(4, 6).double()), dict(q=_bf(6, 4, 576).requires_grad_()),
])
def test_paged_refuses(calls, kw):
    with pytest.raises(ValueError):
        _paged(**kw)
    assert not calls


@pytest.mark.parametrize("kw", [
    dict(q=_bf(6, 3, 192)), dict(q=_bf(6, 4, 128)), dict(q=torch.zeros(6, 4, 192).half()), dict(k=_bf(6, 2, 192)),
    dict(v=_bf(6, 4, 128)), dict(v=_bf(5, 2, 128)), dict(k_rope=_bf(6, 128)), dict(k_rope=_bf(6, 2, 64)), dict(k_rope=_bf(5, 64)),
    dict(k=_bf(5, 2, 128), v=_bf(5, 2, 128), k_rope=_bf(5, 64)), dict(cu_seqlens=_i32(0, 6)[None]),
    dict(cu_seqlens_k=_i32(0, 3, 6)), dict(o=_bf(6, 4, 192)), dict(lse=torch.zeros(6, 4)), dict(k=_bf(6, 2, 128).requires_grad_()),
])
def test_prompt_refuses(calls, kw):
    with pytest.raises(ValueError):
        _prompt(**kw)
    assert not calls


def test_tensors_off_the_gpu_are_refused():
    for f in (_rotary, _write, _paged, _prompt):
        with pytest.raises(ValueError, match="one GPU"):
            f()


# --- the C entries, before any launch -----------------------------------------------

def _arr(*v):
    return (ctypes.c_int64 * len(v))(*v)


def _c_rotary(x=FAKE, o=FAKE + 1024, pos=FAKE, freqs=FAKE, T=4, H=2, D=64, first=0, dim=64, xs=(128, 64), os=(128, 64), scale=1.0,
              dtype=1):
    return _lib.load().g9_rotary(x, o, pos, freqs, T, H, D, first, dim, _arr(*xs) if xs else None, _arr(*os), scale, 0, 0, dtype,
                                 None)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=2), _lib.G9_ERR_DTYPE), (dict(T=-1), _lib.G9_ERR_SHAPE), (dict(H=0), _lib.G9_ERR_SHAPE),
    (dict(D=60), _lib.G9_ERR_SHAPE), (dict(dim=72), _lib.G9_ERR_SHAPE), (dict(dim=24), _lib.G9_ERR_SHAPE),
    (dict(first=8), _lib.G9_ERR_SHAPE), (dict(first=-8, dim=16), _lib.G9_ERR_SHAPE), (dict(scale=math.nan), _lib.G9_ERR_SHAPE),
    (dict(xs=None), _lib.G9_ERR_LAYOUT), (dict(xs=(128, 60)), _lib.G9_ERR_LAYOUT), (dict(xs=(-128, 64)), _lib.G9_ERR_LAYOUT),
    (dict(os=(64, 64)), _lib.G9_ERR_LAYOUT), (dict(os=(0, 64)), _lib.G9_ERR_LAYOUT), (dict(x=None), _lib.G9_ERR_LAYOUT),
    (dict(x=FAKE + 2), _lib.G9_ERR_LAYOUT), (dict(pos=None), _lib.G9_ERR_LAYOUT), (dict(freqs=FAKE + 4), _lib.G9_ERR_LAYOUT),
    (dict(o=FAKE, os=(256, 128)), _lib.G9_ERR_LAYOUT), (dict(T=0), _lib.G9_OK),
])
def test_c_rotary(kw, code):
    assert _c_rotary(**kw) == code


def _c_write(c=FAKE, k=FAKE, cache=FAKE, slots=FAKE, weight=None, eps=1e-6, pos=None, freqs=None, c_out=None, k_out=None, T=4,
             blocks=2, size=16, cs=576, ks=576, st=(9216, 576), cos=512, kos=64, scale=1.0, dtype=1):
    return _lib.load().g9_write_latent(c, k, cache, slots, weight, eps, pos, freqs, c_out, k_out, T, blocks, size, cs, ks,
                                       _arr(*st) if st else None, cos, kos, scale, 0, dtype, None)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=2), _lib.G9_ERR_DTYPE), (dict(T=-1), _lib.G9_ERR_SHAPE), (dict(size=24), _lib.G9_ERR_SHAPE),
    (dict(size=8), _lib.G9_ERR_SHAPE), (dict(eps=-1.0), _lib.G9_ERR_SHAPE), (dict(eps=math.inf), _lib.G9_ERR_SHAPE),
    (dict(scale=math.nan), _lib.G9_ERR_SHAPE), (dict(st=None), _lib.G9_ERR_LAYOUT), (dict(st=(9216, 568)), _lib.G9_ERR_LAYOUT),
    (dict(st=(576, 576)), _lib.G9_ERR_LAYOUT), (dict(cs=577), _lib.G9_ERR_LAYOUT), (dict(cs=-576), _lib.G9_ERR_LAYOUT),
    (dict(c_out=FAKE, cos=256), _lib.G9_ERR_LAYOUT), (dict(k_out=FAKE, kos=0), _lib.G9_ERR_LAYOUT),
    (dict(c=None), _lib.G9_ERR_LAYOUT), (dict(slots=None), _lib.G9_ERR_LAYOUT), (dict(k=FAKE + 8), _lib.G9_ERR_LAYOUT),
    (dict(weight=FAKE + 2), _lib.G9_ERR_LAYOUT), (dict(freqs=FAKE), _lib.G9_ERR_LAYOUT),
    (dict(slots=FAKE + 4), _lib.G9_ERR_LAYOUT), (dict(T=0), _lib.G9_OK),
])
def test_c_write(kw, code):
    assert _c_write(**kw) == code


@pytest.mark.parametrize("kw", [dict(c_out=FAKE), dict(c_out=FAKE, cos=640), dict(k_out=FAKE), dict(k_out=FAKE, kos=584, T=2),
                                dict(c_out=FAKE, cs=0)])
def test_c_write_in_place_needs_the_rows_of_the_input(kw):
    """With other steps a row would land on inputs that are not read yet."""
    assert _c_write(**kw) == _lib.G9_ERR_LAYOUT


def _c_paged(q=FAKE, cache=FAKE, o=FAKE, lse=None, table=FAKE, ts=4, width=4, lengths=FAKE, cu=FAKE, mask=None, words=0, B=2, T=4,
             H=2, blocks=3, size=16, qs=(1152, 576), cs=(9216, 576), os=(1024, 512), scale=1.0, dtype=1, ws=FAKE, wsb=1 << 40):
    return _lib.load().g9_latent_fwd(q, cache, o, lse, table, ts, width, lengths, cu, mask, words, B, T, H, blocks, size,
                                     _arr(*qs), _arr(*cs), _arr(*os), scale, dtype, ws, wsb, None)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=2), _lib.G9_ERR_DTYPE), (dict(H=0), _lib.G9_ERR_SHAPE), (dict(B=8193), _lib.G9_ERR_SHAPE),
    (dict(T=1 << 31), _lib.G9_ERR_SHAPE), (dict(size=48), _lib.G9_ERR_SHAPE), (dict(width=1 << 27, ts=1 << 27), _lib.G9_ERR_SHAPE),
    (dict(scale=0.0), _lib.G9_ERR_SHAPE), (dict(scale=-1.0), _lib.G9_ERR_SHAPE), (dict(mask=FAKE), _lib.G9_ERR_SHAPE),
    (dict(words=1025), _lib.G9_ERR_SHAPE), (dict(T=1 << 20, H=1 << 12, qs=(0, 0), os=(512 << 12, 512)), _lib.G9_ERR_SHAPE),
    (dict(qs=(1152, 575)), _lib.G9_ERR_LAYOUT), (dict(cs=(9216, 568)), _lib.G9_ERR_LAYOUT), (dict(os=(512, 512)), _lib.G9_ERR_LAYOUT),
    (dict(ts=3), _lib.G9_ERR_LAYOUT), (dict(q=None), _lib.G9_ERR_LAYOUT), (dict(cache=None), _lib.G9_ERR_LAYOUT),
    (dict(lengths=None), _lib.G9_ERR_LAYOUT), (dict(o=FAKE + 8), _lib.G9_ERR_LAYOUT), (dict(lse=FAKE + 2), _lib.G9_ERR_LAYOUT),
    (dict(ws=None), _lib.G9_ERR_WORKSPACE), (dict(ws=FAKE + 16), _lib.G9_ERR_WORKSPACE), (dict(wsb=0), _lib.G9_ERR_WORKSPACE),
    (dict(B=0), _lib.G9_OK), (dict(T=0), _lib.G9_OK),
])
def test_c_paged(kw, code):
    assert _c_paged(**kw) == code


def test_paged_workspace():
    size = _lib.load().g9_latent_workspace_size
    assert size(0, 4, 2) == size(2, 0, 2) == size(2, 4, 0) == size(-1, 4, 2) == 0
    assert size(2, 4, 2) > 0 and size(8192, 8192, 128) < 1 << 30


def _c_prompt(q=FAKE, k=FAKE, v=FAKE, r=FAKE, o=FAKE, lse=None, cq=FAKE, ck=FAKE, B=1, T=4, TK=4, HQ=2, HK=2, qs=(384, 192),
              ks=(512, 256), vs=(512, 256), rs=64, os=(256, 128), scale=1.0, dtype=1):
    return _lib.load().g9_latent_varlen_fwd(q, k, v, r, o, lse, cq, ck, B, T, TK, HQ, HK, _arr(*qs), _arr(*ks), _arr(*vs), rs,
                                            _arr(*os), scale, dtype, 1, None)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=3), _lib.G9_ERR_DTYPE), (dict(HQ=3), _lib.G9_ERR_SHAPE), (dict(HK=0), _lib.G9_ERR_SHAPE), (dict(B=-1), _lib.G9_ERR_SHAPE),
    (dict(scale=math.inf), _lib.G9_ERR_SHAPE), (dict(qs=(384, 190)), _lib.G9_ERR_LAYOUT), (dict(rs=-64), _lib.G9_ERR_LAYOUT),
    (dict(rs=60), _lib.G9_ERR_LAYOUT), (dict(os=(128, 128)), _lib.G9_ERR_LAYOUT), (dict(ks=(1 << 23, 256)), _lib.G9_ERR_LAYOUT),
    (dict(q=None), _lib.G9_ERR_LAYOUT), (dict(r=None), _lib.G9_ERR_LAYOUT), (dict(r=FAKE + 4), _lib.G9_ERR_LAYOUT),
    (dict(ck=None), _lib.G9_ERR_LAYOUT), (dict(lse=FAKE + 1), _lib.G9_ERR_LAYOUT), (dict(T=0), _lib.G9_OK), (dict(B=0), _lib.G9_OK),
])
def test_c_prompt(kw, code):
    assert _c_prompt(**kw) == code


# --- frequencies and the oracle -------------------------------------------------------

def test_frequencies():
    f = rotary_frequencies(64)
    assert f.dtype == torch.float64 and f.shape == (32,) and f[0] == 1 and torch.all(f[1:] < f[:-1])
    assert torch.allclose(f[-1], torch.tensor(10000.0 ** (-62 / 64), dtype=torch.float64), rtol=1e-15)
    assert torch.allclose(rotary_frequencies(64, scaling="linear", factor=4.0), f / 4, rtol=1e-15)
    g = rotary_frequencies(64, scaling="base", factor=8.0)
    assert g[0] == 1 and torch.allclose(g[-1], f[-1] / 8, rtol=1e-12)
    for scaling in ("turns", "index"):
        g = rotary_frequencies(64, scaling=scaling, factor=8.0, original_length=4096)
        turns = 4096 * f / (2 * math.pi)
        ratio = g / f
        assert torch.allclose(ratio[turns >= 40], torch.ones(1, dtype=torch.float64), rtol=1e-12)
        assert torch.allclose(ratio[turns <= 0.8], torch.full((1,), 1 / 8, dtype=torch.float64), rtol=1e-12)
        assert torch.all(ratio[1:] <= ratio[:-1] + 1e-12)
    # Halfway between slow and fast: the mean of both.
    i = (turns - 16.5).abs().argmin()
    w = (turns[i] - 1) / 31
    g = rotary_frequencies(64, scaling="turns", factor=8.0, original_length=4096)
    assert torch.allclose(g[i] / f[i], w + (1 - w) / 8, rtol=1e-12)
    lo = math.floor(64 * math.log(4096 / (32 * 2 * math.pi)) / (2 * math.log(10000)))
    hi = math.ceil(64 * math.log(4096 / (2 * math.pi)) / (2 * math.log(10000)))
    g = rotary_frequencies(64, scaling="index", factor=8.0, original_length=4096)
    w = 1 - 3 / (hi - lo)
    assert torch.allclose(g[lo + 3] / f[lo + 3], torch.tensor(w + (1 - w) / 8, dtype=torch.float64), rtol=1e-12)


@pytest.mark.parametrize("a,kw", [
    ((0,), {}), ((7,), {}), ((64, -1.0), {}), ((64, math.inf), {}), ((64,), dict(scaling="other")), ((64,), dict(factor=0.0)),
    ((64,), dict(scaling="turns", factor=2.0)), ((64,), dict(scaling="index", factor=2.0, original_length=4096, fast=1, slow=2)),
    ((64, 0.5), dict(scaling="index", original_length=4096)), ((2,), dict(scaling="base", factor=2.0)),
])
def test_frequencies_refuse(a, kw):
    with pytest.raises(ValueError):
        rotary_frequencies(*a, **kw)


def test_oracle_rotation_is_a_rotation():
    rng = np.random.default_rng(0)
    x, pos, f = rng.standard_normal((5, 2, 48)), np.array([0, 1, 7, -3, 10**6]), rotary_frequencies(32).numpy()
    for inter in (False, True):
        y = L.rotate(x, pos, f, 8, inter)
        assert np.allclose(L.rotate(y, pos, f, 8, inter, inverse=True), x, atol=1e-9)
        assert np.array_equal(y[0], x[0]) and np.array_equal(y[..., :8], x[..., :8]) and np.array_equal(y[..., 40:], x[..., 40:])
        # Products depend on the distance alone.
        q, k = rng.standard_normal((2, 1, 1, 32))
        d = [(L.rotate(q, [a + 5], f, 0, inter) * L.rotate(k, [a], f, 0, inter)).sum() for a in (0, 11, 500)]
        assert np.allclose(d, d[0])


def test_oracle_attention_forms_agree():
    """The absorbed form over latents is the expanded form over their projections, and both the plain oracle's."""
    rng = np.random.default_rng(1)
    n, H, C, P, K, V = 9, 3, 16, 4, 6, 5
    c, kr, up_k, up_v = rng.standard_normal((n, C)), rng.standard_normal((n, P)), rng.standard_normal((H, K, C)), rng.standard_normal((H, V, C))
    q = rng.standard_normal((n, H, K + P))
    reads = R.causal_reads(n, n)
    keys = np.concatenate([np.einsum("tc,hkc->thk", c, up_k), np.broadcast_to(kr[:, None], (n, H, P))], -1)
    vals = np.einsum("tc,hvc->thv", c, up_v)
    o, lse, _, _ = L.attend(q, keys, vals, reads, 0.3)
    absorbed = np.concatenate([np.einsum("thk,hkc->thc", q[..., :K], up_k), q[..., K:]], -1)
    rows = np.concatenate([c, kr], -1)
    a, lse2, _, _ = L.attend(absorbed, rows[:, None], c[:, None], reads, 0.3)
    assert np.allclose(np.einsum("thc,hvc->thv", a, up_v), o) and np.allclose(lse, lse2)
    for h in range(H):
        want, w_lse, _, _ = R.masked_attention(q[:, h], keys[:, h], vals[:, h], reads, 0.3)
        assert np.allclose(o[:, h], want) and np.allclose(lse[h], w_lse)


def test_rotation_bound_counts_the_roundings():
    """The angle's 64-bit part, as the kernel forms it, against 60 digits; and the bound's fp32 terms."""
    import random
    from fractions import Fraction

    pi = Fraction("3.14159265358979323846264338327950288419716939937510582097494459")
    inv, rng, top = float(0.15915494309189533577), random.Random(0), 0
    assert abs(Fraction(inv) * 2 * pi - 1) <= Fraction(1, 2**53)
    for _ in range(20000):
        n, f = rng.randrange(1, 2**31), 10.0 ** rng.uniform(-4, 0)
        t = n * (f * inv)
        off = abs(Fraction(t) * 2 * pi - Fraction(n) * Fraction(f)) / (Fraction(n) * Fraction(f))
        top = max(top, off)
    # Three roundings (the constant's, two products'); with the oracle's own product four.
    assert 2.0**-53 < top <= 3 * 2.0**-53
    angle, sine, products = 2 * math.pi * 2.0**-26, 2.0**-24, 4 * 2.0**-24
    assert angle + sine + products < 2.0**-21
    x, n, f = np.ones((1, 1, 2)), 2**31, 1.0
    y = L.rotate(x, [n], [f])
    bound = L.rotate_bound(x, y, [n], [f], 0.0, 0.0)
    assert (bound >= 2 * (angle + sine + products + 4 * 2.0**-53 * n * f)).all()
