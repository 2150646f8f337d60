"""GPU parity of the rotary positions and of the latents' writes against the float64
oracle (oracle/latent_ref.py).  Bounds come from the arithmetic (there); copies must
be equal."""

import numpy as np
import pytest
import torch

from gfx950_gluon_tutorials_amd.attention import rotary, rotary_frequencies, write_latent
from oracle import latent_ref as R

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
SUBNORMAL = {"fp16": 2.0**-25, "bf16": 0.0}


def _np(t):
    return t.detach().double().cpu().numpy()


def _check(got, x, positions, freqs, dtype, first=0, interleaved=False, inverse=False, scale=1.0):
    x, freqs, positions = _np(x), _np(freqs), positions.cpu().numpy()
    want = R.rotate(x, positions, freqs, first, interleaved, inverse, scale)
    bound = R.rotate_bound(x, want, positions, freqs, torch.finfo(DT[dtype]).eps, SUBNORMAL[dtype], first, interleaved, scale)
    off = np.abs(_np(got) - want) - bound
    assert (off <= 0).all(), f"{off.max():.3g} past its bound at {np.unravel_index(off.argmax(), off.shape)}"


@pytest.mark.parametrize("T,H,D,first,dim", [
    (1, 1, 64, 0, 64), (3, 5, 128, 0, 128), (7, 2, 192, 128, 64), (64, 40, 128, 0, 128), (33, 3, 80, 0, 32), (5, 1, 96, 48, 48),
    (2, 7, 256, 8, 16), (1000, 4, 64, 0, 64), (9, 128, 192, 128, 64), (130, 1, 576, 512, 64),
])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_rotary(gpu, T, H, D, first, dim, interleaved, dtype):
    g = torch.Generator().manual_seed(T + D)
    x = torch.randn(T, H, D, generator=g).to(DT[dtype]).to(gpu)
    pos = torch.randint(0, 200000, (T,), generator=g).to(gpu)
    freqs = rotary_frequencies(dim, device=gpu)
    for inverse, scale in ((False, 1.0), (True, 1.25)):
        o = rotary(x, pos, freqs, first=first, interleaved=interleaved, inverse=inverse, scale=scale)
        _check(o, x, pos, freqs, dtype, first, interleaved, inverse, scale)
        same = x.clone()
        assert rotary(same, pos, freqs, same, first=first, interleaved=interleaved, inverse=inverse, scale=scale) is same
        assert torch.equal(same, o)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_of_a_fused_projection_in_place(gpu, interleaved):
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(50, 12, 128, generator=g).to(torch.bfloat16).to(gpu)
    before = qkv.clone()
    pos, freqs = torch.arange(50, device=gpu) * 3, rotary_frequencies(64, device=gpu)
    qk = qkv[:, :10]
    rotary(qk, pos, freqs, qk, interleaved=interleaved)
    assert torch.equal(qkv[:, 10:], before[:, 10:]) and torch.equal(qkv[..., 64:], before[..., 64:])
    assert torch.equal(qk, rotary(before[:, :10], pos, freqs, interleaved=interleaved))


def test_rotary_strides(gpu):
    g = torch.Generator().manual_seed(2)
    T, H, D = 37, 4, 64
    x = torch.randn(H, 2 * T, D + 8, generator=g).to(torch.float16).to(gpu)[:, ::2, :D].transpose(0, 1)
    buf = torch.full((T, H, 576), 7.0, dtype=torch.float16, device=gpu)
    pos, freqs = torch.arange(T, device=gpu), rotary_frequencies(D, device=gpu)
    rotary(x, pos, freqs, buf[..., 512:])
    assert (buf[..., :512] == 7).all()
    assert torch.equal(buf[..., 512:], rotary(x.contiguous(), pos, freqs))
    one = torch.randn(1, 1, D, generator=g).half().to(gpu)
    wide = rotary(one.expand(T, H, D), pos, freqs)
    assert torch.equal(wide, rotary(one.expand(T, H, D).contiguous(), pos, freqs))


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_far_and_negative_positions(gpu, interleaved):
    g = torch.Generator().manual_seed(3)
    pos = torch.tensor([0, 1, -1, 2**20 + 1, 2**24 + 1, 2**31 - 1, -(2**31), 10**7], device=gpu)
    x = torch.randn(len(pos), 3, 128, generator=g).half().to(gpu)
    freqs = rotary_frequencies(128, device=gpu)
    _check(rotary(x, pos, freqs, interleaved=interleaved), x, pos, freqs, "fp16", 0, interleaved)


def test_rotary_of_special_values_stays_within_its_pair(gpu):
    x = torch.ones(4, 2, 64, device=gpu, dtype=torch.bfloat16)
    pos, freqs = torch.arange(4, device=gpu), rotary_frequencies(32, device=gpu)
    clean = rotary(x, pos, freqs)
    x[1, 0, 3], x[2, 1, 40] = float("nan"), float("inf")
    got = rotary(x, pos, freqs)
    keep = torch.ones_like(x, dtype=torch.bool)
    keep[1, 0, [3, 19]], keep[2, 1, 40] = False, False
    assert torch.equal(got[keep], clean[keep])
    assert got[1, 0, [3, 19]].isnan().all() and got[2, 1, 40] == float("inf")


def test_rotary_gradient(gpu):
    """The gradient against the formula's, by autograd in 64 bits, and against differences."""
    g = torch.Generator().manual_seed(4)
    T, H, D, first, dim, scale = 6, 2, 96, 16, 64, 0.75
    pos, freqs = torch.randint(0, 5000, (T,), generator=g), rotary_frequencies(dim)
    for interleaved in (False, True):
        x = torch.randn(T, H, D, generator=g, dtype=torch.float64, requires_grad=True)
        w = torch.randn(T, H, D, generator=g).half()
        t = pos.double()[:, None, None] * freqs
        part = x[..., first:first + dim]
        a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else part.chunk(2, -1)
        u, v = scale * (a * t.cos() - b * t.sin()), scale * (a * t.sin() + b * t.cos())
        y = torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)
        loss = (torch.cat((x[..., :first], y, x[..., first + dim:]), -1) * w.double()).sum()
        (want,) = torch.autograd.grad(loss, x)
        got = rotary(w.to(gpu), pos.to(gpu), freqs.to(gpu), first=first, interleaved=interleaved, inverse=True, scale=scale)
        bound = R.rotate_bound(w.double().numpy(), want.numpy(), pos.numpy(), freqs.numpy(), 2.0**-10, 2.0**-25, first,
                               interleaved, scale)
        assert (np.abs(_np(got) - want.numpy()) <= bound).all()
        # Differences of the oracle's forward: it is linear, so a step of 1 is exact to 64 bits.
        d = torch.randn(T, H, D, generator=g, dtype=torch.float64).numpy()
        diff = (R.rotate(d, pos.numpy(), freqs.numpy(), first, interleaved, False, scale) * w.double().numpy()).sum()
        assert abs(diff - (d * _np(got)).sum()) <= (np.abs(d) * bound).sum() + 1e-9


def test_rotary_nothing_to_do(gpu):
    x = torch.empty(0, 4, 64, dtype=torch.float16, device=gpu)
    assert rotary(x, torch.empty(0, dtype=torch.int64, device=gpu), rotary_frequencies(64, device=gpu)).shape == x.shape


def test_rotary_past_32_bit_offsets(gpu):
    T, H, D = 2**15 + 3, 128, 576
    x = torch.zeros(T, H, D, dtype=torch.bfloat16, device=gpu)
    assert x.numel() > 2**31
    x[-3:] = torch.randn(3, H, D, device=gpu).bfloat16()
    pos, freqs = torch.arange(T, device=gpu), rotary_frequencies(64, device=gpu)
    want = rotary(x[-3:].clone(), pos[-3:].clone(), freqs, first=512, interleaved=True)
    rotary(x, pos, freqs, x, first=512, interleaved=True)
    assert torch.equal(x[-3:], want) and not x[:-3].any()
    del x
    torch.cuda.empty_cache()


def test_rotary_streams_and_graphs(gpu):
    x = torch.randn(100, 8, 128, device=gpu).bfloat16()
    pos, freqs, o = torch.arange(100, device=gpu), rotary_frequencies(128, device=gpu), torch.empty_like(x)
    want = rotary(x, pos, freqs)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        rotary(x, pos, freqs, o)
    s.synchronize()
    assert torch.equal(o, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rotary(x, pos, freqs, o)
    for i in range(3):
        x.normal_()
        pos.add_(i)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, rotary(x, pos, freqs))


# --- latents into the cache -----------------------------------------------------

def _write_case(gpu, T, blocks, size, dtype, seed, wide=False):
    g = torch.Generator().manual_seed(seed)
    down = torch.randn(T, 576 + (16 if wide else 0), generator=g).to(DT[dtype]).to(gpu)
    cache = torch.randn(blocks, size, 576, generator=g).to(DT[dtype]).to(gpu)
    slots = torch.randperm(blocks * size, generator=g)[:T]
    slots[::7] = torch.tensor([-1, blocks * size, -2**40, 2**40])[torch.arange(len(slots[::7])) % 4]
    weight = (1 + 0.3 * torch.randn(512, generator=g)).to(DT[dtype]).to(gpu)
    pos = torch.randint(0, 100000, (T,), generator=g).to(gpu)
    return down[:, :512], down[:, 512:576], cache, slots.to(gpu), weight, pos


def _check_latents(c_out, k_out, c, k, weight, eps, pos, freqs, interleaved, scale, dtype):
    h = torch.finfo(DT[dtype]).eps / 2
    if weight is None:
        assert torch.equal(c_out, c)
    else:
        want = R.rms(_np(c), _np(weight), eps)
        # Sum of 512 squares: 8 + 6 additions on the way, halved by the root; root, quotient
        # and two products 2^-23 at most: less than 2^-20 together; then half a step.
        assert (np.abs(_np(c_out) - want) <= (h + 2.0**-20) * np.abs(want) * (1 + h) + SUBNORMAL[dtype]).all()
    if freqs is None:
        assert torch.equal(k_out, k)
    else:
        _check(k_out[:, None], k[:, None], pos, freqs, dtype, 0, interleaved, False, scale)


@pytest.mark.parametrize("T,size,wide", [(1, 16, False), (5, 16, True), (130, 64, False), (1003, 32, False), (77, 1024, True)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("norm,turn", [(True, True), (True, False), (False, True), (False, False)])
def test_write_latent(gpu, T, size, wide, interleaved, dtype, norm, turn):
    blocks = 3 + 2 * T // size
    c, k, cache, slots, weight, pos = _write_case(gpu, T, blocks, size, dtype, T, wide)
    freqs = rotary_frequencies(64, device=gpu)
    kw = dict(interleaved=interleaved, scale=1.1)
    if norm:
        kw.update(weight=weight, eps=1e-5)
    if turn:
        kw.update(positions=pos, freqs=freqs)
    before = cache.clone()
    c_out, k_out = torch.empty(T, 512, dtype=c.dtype, device=gpu), torch.empty(T, 64, dtype=c.dtype, device=gpu)
    assert write_latent(c, k, cache, slots, c_out=c_out, k_out=k_out, **kw) is None
    _check_latents(c_out, k_out, c, k, weight if norm else None, 1e-5, pos, freqs if turn else None, interleaved, 1.1, dtype)
    want = before.view(-1, 576)
    ok = (slots >= 0) & (slots < blocks * size)
    want[slots[ok]] = torch.cat((c_out, k_out), 1)[ok]
    assert torch.equal(cache.view(-1, 576), want)
    # Without the outputs, and with the inputs as outputs.
    again = before.clone()
    write_latent(c, k, again, slots, **kw)
    assert torch.equal(again, cache)
    write_latent(c, k, again, slots, c_out=c, k_out=k, **kw)
    assert torch.equal(again, cache) and torch.equal(c, c_out) and torch.equal(k, k_out)


@pytest.mark.parametrize("value", [0.0, 1e-7, 3e4])
def test_write_latent_of_small_and_large_rows(gpu, value):
    c = torch.full((3, 512), value, dtype=torch.float16, device=gpu)
    k = torch.zeros(3, 64, dtype=torch.float16, device=gpu)
    weight = torch.ones(512, dtype=torch.float16, device=gpu)
    out = torch.empty_like(c)
    cache = torch.zeros(1, 16, 576, dtype=torch.float16, device=gpu)
    write_latent(c, k, cache, torch.arange(3, device=gpu), weight=weight, eps=1e-6, c_out=out)
    want = R.rms(_np(c), _np(weight), 1e-6)
    assert (np.abs(_np(out) - want) <= (2.0**-11 + 2.0**-19) * np.abs(want) + 2.0**-25).all()


def test_write_latent_cache_strides_and_far_slots(gpu):
    """A cache of more than 4 GiB, its blocks further apart than they are long."""
    blocks, size = 2**15 + 5, 64
    base = torch.zeros(blocks, size + 16, 640, dtype=torch.bfloat16, device=gpu)
    cache = base[:, :size, 32:608]
    assert base.numel() * 2 > 2**31
    c, k = torch.randn(3, 512, device=gpu).bfloat16(), torch.randn(3, 64, device=gpu).bfloat16()
    slots = torch.tensor([blocks * size - 1, 2**20 + 5, 0], device=gpu)
    write_latent(c, k, cache, slots)
    for t, s in enumerate(slots.tolist()):
        assert torch.equal(cache[s // size, s % size], torch.cat((c[t], k[t])))
        cache[s // size, s % size] = 0
    assert not base.any()
    del base, cache
    torch.cuda.empty_cache()


def test_write_latent_streams_graphs_and_nothing(gpu):
    c, k, cache, slots, weight, pos = _write_case(gpu, 60, 9, 16, "bf16", 5)
    freqs = rotary_frequencies(64, device=gpu)
    c, k = c.clone(), k.clone()
    write_latent(c[:0], k[:0], cache, slots[:0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        write_latent(c, k, cache, slots, weight=weight, positions=pos, freqs=freqs)
    for _ in range(3):
        c.normal_()
        k.normal_()
        want = cache.clone()
        write_latent(c, k, want, slots, weight=weight, positions=pos, freqs=freqs)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(cache, want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    other = torch.zeros_like(cache)
    with torch.cuda.stream(s):
        s.wait_stream(torch.cuda.default_stream())
        write_latent(c, k, other, slots, weight=weight, positions=pos, freqs=freqs)
    s.synchronize()
    ok = (slots >= 0) & (slots < 9 * 16)
    assert torch.equal(other.view(-1, 576)[slots[ok]], cache.view(-1, 576)[slots[ok]])
