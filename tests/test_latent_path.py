"""Serving with latent attention, stage by stage: slots, norm, rotation and writes, prompts
through the expanded form, decoding through the absorbed one, the framework's products
between.  Each stage is held against the float64 oracle of the rounded inputs that it was
given, so that its bound is that of its own roundings; a CPU test plants mistakes in the
oracle and sees every one of them leave the bounds."""

import numpy as np
import pytest
import torch

from gfx950_gluon_tutorials_amd.attention import (assign_slots, latent_attention, latent_varlen_attention, rotary,
                                                  rotary_frequencies, write_latent)
from gfx950_gluon_tutorials_amd.gemm.intra_wave.a16w16 import matmul
from gfx950_gluon_tutorials_amd.gemm.moe import moe_matmul
from oracle import latent_ref as L
from oracle import serving_ref as R

DT, EPS, SCALE = torch.bfloat16, torch.finfo(torch.bfloat16).eps, 192**-0.5
H, HIDDEN, SIZE = 4, 256, 16
FREQS = dict(scaling="turns", factor=4.0, original_length=4096)


def _np(t):
    return t.detach().double().cpu().numpy()


def _bf(x):
    """A float64 array rounded to bf16 values."""
    return _np(torch.tensor(x).to(DT))


def _off(got, ref, tol):
    """How many of the outputs are outside their bounds (or not numbers)."""
    return int((~(np.abs(got - ref) <= tol)).sum())


def product_off(got, x, w):
    """got = x w^T over the last axis, heads in the middle where w has them.  K exact products summed in
    fp32: K 2^-24 of the products' magnitudes; then half a step."""
    f = "thk,hnk->thn" if w.ndim == 3 else "tk,nk->tn"
    ref, mag = np.einsum(f, x, w), np.einsum(f, np.abs(x), np.abs(w))
    return _off(got, ref, EPS / 2 * np.abs(ref) * (1 + EPS) + 2 * w.shape[-1] * 2.0**-24 * mag)


def decode_off(got, q, cache, table, lengths, cu, scale=SCALE, mask=None):
    ref, lse, mag, spread = L.paged(q, cache, table, lengths, cu, mask, scale)
    longest = max(int(n) for n in lengths) + int(np.diff(cu).max())
    return _off(got, ref, R.tolerances(ref, lse, mag, spread, EPS, longest, 576, np.abs(cache).max(), 0.0)[0])


def prompt_off(got, q, k, v, k_rope, cu, causal=True, scale=SCALE):
    ref, lse, mag, spread = L.packed(q, k, v, k_rope, cu, cu, causal, scale)
    return _off(got, ref, R.tolerances(ref, lse, mag, spread, EPS, int(np.diff(cu).max()), 192, np.abs(v).max(), 0.0)[0])


def write_off(c_out, k_out, down, weight, positions, freqs, interleaved):
    """The bounds of tests/test_rotary_gpu.py."""
    want = L.rms(down[:, :512], weight, 1e-6)
    turned = L.rotate(down[:, None, 512:], positions, freqs, 0, interleaved)
    bound = L.rotate_bound(down[:, None, 512:], turned, positions, freqs, EPS, 0.0, 0, interleaved)
    return _off(c_out, want, (EPS / 2 + 2.0**-20) * np.abs(want) * (1 + EPS)) + _off(k_out, turned[:, 0], bound[:, 0])


def _weights(g):
    r = lambda *s: torch.randn(*s, generator=g)
    w_up = (r(H, 256, 512) / 23).to(DT)  # a head's key rows, then its value rows
    return dict(q=(r(H * 192, HIDDEN) / 16).to(DT), down=(r(576, HIDDEN) / 16).to(DT), up=w_up,
                k=w_up[:, :128].transpose(1, 2).contiguous(), v=w_up[:, 128:].contiguous(), norm=(1 + 0.1 * r(512)).to(DT))


def test_mistakes_leave_the_bounds():
    """The stages' outputs as the oracle gives them, rounded, against oracles with a mistake each."""
    g = torch.Generator().manual_seed(1)
    w = {k: _np(t) for k, t in _weights(g).items()}
    freqs = rotary_frequencies(64, **FREQS).numpy()
    n, context = [2, 1], [37, 20]
    cu, table = np.array([0, 2, 3]), np.array([[5, 0, 3], [1, 4, 0]])
    cache = np.zeros((6, SIZE, 576))
    for b, pages in enumerate(table):
        rows = _bf(torch.randn(context[b] + n[b], HIDDEN, generator=g).numpy()) @ w["down"].T
        at = np.arange(len(rows))
        kr = L.rotate(_bf(rows)[:, None, 512:], at, freqs)[:, 0]
        cache[pages[at // SIZE], at % SIZE] = _bf(np.concatenate([L.rms(_bf(rows)[:, :512], w["norm"], 1e-6), kr], -1))
    q = _bf((_bf(torch.randn(3, HIDDEN, generator=g).numpy()) @ w["q"].T).reshape(3, H, 192))
    full = _bf(np.concatenate([np.einsum("thd,hcd->thc", q[..., :128], w["k"]), q[..., 128:]], -1))
    got = _bf(L.paged(full, cache, table, context, cu, None, SCALE)[0])
    assert decode_off(got, full, cache, table, context, cu) == 0
    out = got.size
    turned = np.concatenate([full[..., :512], np.zeros_like(full[..., 512:])], -1)
    own = np.array([[0], [1], [0]], np.uint64)  # the nodes before a row's own
    wrong = [decode_off(got, full, cache, table, context, cu, scale=576**-0.5), decode_off(got, turned, cache, table, context, cu),
             decode_off(got, full, cache, table, context, cu, mask=own),
             decode_off(got, full, cache, table, [c + 1 for c in context], cu),
             decode_off(got, full, cache, table[:, [1, 0, 2]], context, cu), decode_off(0 * got, full, cache, table, context, cu)]
    assert min(wrong) > out / 4, wrong
    # The value projection, and its heads in another order.
    o = _bf(np.einsum("thc,hvc->thv", got, w["v"]))
    assert product_off(o, got, w["v"]) == 0 and product_off(o, got, w["v"][::-1]) > o.size / 2
    assert product_off(0 * o, got, w["v"]) > o.size / 2
    # A prompt: no mask, no shared keys, another scale.
    T = 30
    cu = np.array([0, 17, 30])
    q, kr = _bf(torch.randn(T, H, 192, generator=g).numpy()), _bf(torch.randn(T, 64, generator=g).numpy())
    k, v = (_bf(torch.randn(T, H, 128, generator=g).numpy()) for _ in range(2))
    o = _bf(L.packed(q, k, v, kr, cu, cu, True, SCALE)[0])
    assert prompt_off(o, q, k, v, kr, cu) == 0
    wrong = [prompt_off(o, q, k, v, kr, cu, causal=False), prompt_off(o, q, k, v, 0 * kr, cu), prompt_off(o, q, k, v, kr, cu, scale=128**-0.5),
             prompt_off(o, q, k, v, kr[::-1], cu), prompt_off(0 * o, q, k, v, kr, cu)]
    assert min(wrong) > o.size / 4, wrong
    # Writes: positions one further, the other pairs, no norm's weight.
    down, at = _bf(torch.randn(9, 576, generator=g).numpy()), np.arange(9) + 3
    c, kr = _bf(L.rms(down[:, :512], w["norm"], 1e-6)), _bf(L.rotate(down[:, None, 512:], at, freqs)[:, 0])
    assert write_off(c, kr, down, w["norm"], at, freqs, False) == 0
    for wrong in ((w["norm"], at + 1, freqs, False), (w["norm"], at, freqs, True), (1 + 0 * w["norm"], at, freqs, False)):
        assert write_off(c, kr, down, *wrong) > kr.size / 4


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_each_stage_of_a_prompt_and_of_decoding(gpu, interleaved):
    g = torch.Generator().manual_seed(2)
    w = {k: t.to(gpu) for k, t in _weights(g).items()}
    ref = {k: _np(t) for k, t in w.items()}
    freqs = rotary_frequencies(64, device=gpu, **FREQS)
    B = 2
    cache = torch.zeros(12, SIZE, 576, dtype=DT, device=gpu)
    table = torch.zeros(B, 5, dtype=torch.int32, device=gpu)
    free, start = torch.randperm(12, generator=g).int().to(gpu), torch.zeros(1, dtype=torch.int32, device=gpu)
    lengths = torch.zeros(B, dtype=torch.int32, device=gpu)

    def per_head(x, m):  # the grouped product with heads as experts
        T = x.shape[0]
        off = torch.arange(0, (H + 1) * T, T, dtype=torch.int32, device=gpu)
        return moe_matmul(x.transpose(0, 1).reshape(H * T, -1), m, off).view(H, T, -1).transpose(0, 1)

    for counts, prompt in (([37, 20], True), ([1, 1], False), ([2, 1], False), ([1, 3], False)):
        T = sum(counts)
        n = torch.tensor(counts, dtype=torch.int32, device=gpu)
        x = torch.randn(T, HIDDEN, generator=g).to(DT).to(gpu)
        s = assign_slots(lengths, n, table, free, SIZE, T, free_start=start)
        q = matmul(x, w["q"].T).view(T, H, 192)
        before = _np(q)
        rotary(q, s.positions, freqs, q, first=128, interleaved=interleaved)
        pos, f = _np(s.positions), _np(freqs)
        turned = L.rotate(before, pos, f, 128, interleaved)
        assert _off(_np(q), turned, L.rotate_bound(before, turned, pos, f, EPS, 0.0, 128, interleaved)) == 0
        down = matmul(x, w["down"].T)
        c, kr = torch.empty(T, 512, dtype=DT, device=gpu), torch.empty(T, 64, dtype=DT, device=gpu)
        write_latent(down[:, :512], down[:, 512:], cache, s.slots, weight=w["norm"], positions=s.positions, freqs=freqs,
                     interleaved=interleaved, c_out=c, k_out=kr)
        assert write_off(_np(c), _np(kr), _np(down), ref["norm"], pos, f, interleaved) == 0
        assert torch.equal(cache.view(-1, 576)[s.slots], torch.cat((c, kr), 1))
        cu = s.cu_seqlens.cpu().numpy()
        if prompt:
            kv = matmul(c, w["up"].reshape(H * 256, 512).T).view(T, H, 256)
            o = latent_varlen_attention(q, kv[..., :128], kv[..., 128:], kr, s.cu_seqlens)
            assert prompt_off(_np(o), _np(q), _np(kv[..., :128]), _np(kv[..., 128:]), _np(kr), cu) == 0
        else:
            full = torch.empty(T, H, 576, dtype=DT, device=gpu)
            full[..., :512] = per_head(q[..., :128], w["k"])
            full[..., 512:] = q[..., 128:]
            assert product_off(_np(full[..., :512]), _np(q[..., :128]), ref["k"]) == 0
            latent = latent_attention(full, cache, table, lengths, s.cu_seqlens, sm_scale=SCALE)
            assert decode_off(_np(latent), _np(full), _np(cache), table.cpu().numpy(), lengths.tolist(), cu) == 0
            assert product_off(_np(per_head(latent, w["v"])), _np(latent), ref["v"]) == 0
        lengths += n
        start.add_(s.taken)
