"""GPU parity of latent attention, over a paged cache and over packed prompts, against
the float64 oracle (oracle/latent_ref.py), at the sizes and masks where it can go
wrong.  Tolerances come from the arithmetic (serving_ref.tolerances)."""

import itertools

import numpy as np
import pytest
import torch

from gfx950_gluon_tutorials_amd.attention import (assign_slots, latent_attention, latent_varlen_attention, rotary,
                                                  rotary_frequencies, write_latent)
from gfx950_gluon_tutorials_amd.gemm.intra_wave.a16w16 import matmul
from gfx950_gluon_tutorials_amd.gemm.moe import moe_matmul
from oracle import latent_ref as L
from oracle import serving_ref as R

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
SUBNORMAL = {"fp16": 2.0**-25, "bf16": 0.0}
SCALE = 192**-0.5


def _cu(lengths):
    return np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)


def _np(t):
    return t.detach().float().cpu().numpy()


def _dev(x, dev, dtype=torch.int32):
    return torch.tensor(np.asarray(x), dtype=dtype).to(dev)


def _check(got, lse, ref, lse_ref, mag, spread, dtype, longest, D, vmax, rows):
    to, tl = R.tolerances(ref, lse_ref, mag, spread, torch.finfo(DT[dtype]).eps, longest, D, vmax, SUBNORMAL[dtype])
    got, ref, to = _np(got)[:rows], ref[:rows], to[:rows]
    assert np.isfinite(got).all()
    off = np.abs(got - ref) - to
    assert (off <= 0).all(), f"o is {off.max():.3g} past its bound at {np.unravel_index(off.argmax(), off.shape)}"
    if lse is None:
        return
    lse, lse_ref, tl = _np(lse)[:, :rows], lse_ref[:, :rows], tl[:, :rows]
    none = np.isneginf(lse_ref)
    assert (np.isneginf(lse) == none).all()
    off = np.abs(np.where(none, 0, lse) - np.where(none, 0, lse_ref)) - np.where(none, 0, tl)
    assert (off <= 0).all(), f"lse is {off.max():.3g} past its bound"


# --- the absorbed form over a paged cache ---------------------------------------

def _paged(dev, dtype, context, nodes, H, size, seed, mask=None, pad=0, qscale=0.6, spare=3, width=None, wide=False):
    g = torch.Generator().manual_seed(seed)
    total = [c + n for c, n in zip(context, nodes)]
    used = [-(-t // size) for t in total]
    blocks = sum(used) + spare
    ids = torch.randperm(blocks, generator=g).tolist()
    W = max(max(used, default=0), 1) if width is None else width
    table = np.zeros((len(context), W), np.int32)
    for b, n in enumerate(used):
        for j in range(n):
            page = ids.pop()
            if j < W:
                table[b, j] = page
    cache = torch.randn(blocks, size, 576 + (24 if wide else 0), generator=g).to(DT[dtype])
    T = sum(nodes) + pad
    q = (torch.randn(T, H, 576 + (8 if wide else 0), generator=g) * qscale).to(DT[dtype])
    return dict(q=q.to(dev)[..., :576], cache=cache.to(dev)[..., :576], table=table, context=context, cu=_cu(nodes), mask=mask)


def _run_paged(dev, a, o=None, lse=None, scale=SCALE):
    mask = None if a["mask"] is None else torch.from_numpy(a["mask"].astype(np.uint64).view(np.int64)).to(dev)
    return latent_attention(a["q"], a["cache"], _dev(a["table"], dev), _dev(a["context"], dev), _dev(a["cu"], dev), mask, o,
                            sm_scale=scale, lse=lse)


def _check_paged(dev, dtype, a, scale=SCALE):
    T, H = a["q"].shape[:2]
    rows = int(a["cu"][-1])
    o = torch.full((T, H, 512), 7.0, dtype=DT[dtype], device=dev)
    lse = torch.full((H, T), 7.0, device=dev)
    assert _run_paged(dev, a, o, lse, scale) is o
    torch.cuda.synchronize()
    ref = L.paged(_np(a["q"]), _np(a["cache"]), a["table"], a["context"], a["cu"], a["mask"], scale)
    longest = max((c + n for c, n in zip(a["context"], np.diff(a["cu"]))), default=1)
    _check(o, lse, *ref, dtype, longest, 576, float(np.abs(_np(a["cache"])).max(initial=0)), rows)
    assert (_np(o)[rows:] == 7).all() and (_np(lse)[:, rows:] == 7).all(), "rows behind the last request changed"
    return o, lse


def _tree(rng, n, words):
    mask = np.zeros((n, words), np.uint64)
    for i in range(n):
        if i:
            mask[i] = mask[rng.integers(max(0, i - 4), i)]
        mask[i, i // 64] |= np.uint64(1) << np.uint64(i % 64)
    return mask


LENGTHS = [
    ([0], [1]), ([1], [1]), ([31], [1]), ([32], [1]), ([700], [1]), ([0, 5, 0], [1, 0, 3]),
    ([15, 16, 17, 63, 64, 65, 127, 128, 129], [1] * 9), ([100, 0, 1000, 3], [2, 1, 5, 1]), ([257], [33]), ([2000, 1], [1, 1]),
]


@pytest.mark.parametrize("context,nodes", LENGTHS, ids=lambda x: "_".join(map(str, x)))
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("H,size", [(16, 16), (128, 64), (5, 32)])
def test_paged_lengths(gpu, context, nodes, dtype, H, size):
    _check_paged(gpu, dtype, _paged(gpu, dtype, context, nodes, H, size, sum(context) + H, pad=2))


@pytest.mark.parametrize("H", [1, 2, 7, 16, 20, 31, 32, 33, 40, 64, 65, 96, 100, 128, 129, 200])
@pytest.mark.parametrize("nodes", [1, 3])
def test_paged_heads(gpu, H, nodes):
    _check_paged(gpu, "bf16", _paged(gpu, "bf16", [300, 77], [nodes, 1], H, 16, H))


@pytest.mark.parametrize("size", [16, 32, 64, 128, 1024])
@pytest.mark.parametrize("H", [16, 64, 128])
def test_paged_block_sizes(gpu, size, H):
    _check_paged(gpu, "fp16", _paged(gpu, "fp16", [1500, 9, 640], [1, 2, 1], H, size, size))


@pytest.mark.parametrize("n,words", [(1, 1), (12, 1), (64, 1), (65, 2), (100, 2), (130, 3)])
@pytest.mark.parametrize("H", [2, 32])
def test_paged_trees(gpu, n, words, H):
    rng = np.random.default_rng(n)
    nodes = [n, max(1, n // 2), 1]
    mask = np.concatenate([_tree(rng, m, words) for m in nodes])
    _check_paged(gpu, "bf16", _paged(gpu, "bf16", [200, 0, 33], nodes, H, 32, n, mask))


def test_paged_rows_that_read_nothing(gpu):
    """Nodes whose bits are all zero: without a context they read nothing, with one only that."""
    mask = np.array([[1], [0], [4], [0], [2], [0]], np.uint64)
    for H in (3, 32, 128):
        a = _paged(gpu, "fp16", [0, 40], [4, 2], H, 16, H, mask)
        o, lse = _check_paged(gpu, "fp16", a)
        assert (o[1] == 0).all() and torch.isneginf(lse[:, 1]).all()


def test_paged_mask_with_few_words(gpu):
    """Nodes behind the last word's are read by none."""
    mask = np.full((80, 1), 2**64 - 1, np.uint64)
    _check_paged(gpu, "bf16", _paged(gpu, "bf16", [10], [80], 4, 16, 1, mask))


@pytest.mark.parametrize("B,H", [(300, 16), (700, 4), (65, 128), (257, 33)])
def test_paged_many_requests(gpu, B, H):
    rng = np.random.default_rng(B)
    context = rng.integers(0, 90, B).tolist()
    nodes = rng.integers(0, 3, B).tolist()
    _check_paged(gpu, "bf16", _paged(gpu, "bf16", context, nodes, H, 16, B, pad=1))


@pytest.mark.parametrize("H", [16, 40, 128])
@pytest.mark.parametrize("context", [[20000], [9000, 10, 4000], [33000, 1]])
def test_paged_long_contexts(gpu, H, context):
    """Contexts that many workgroups share."""
    _check_paged(gpu, "bf16", _paged(gpu, "bf16", context, [1] * len(context), H, 64, H))


@pytest.mark.parametrize("H", [16, 64, 128])
def test_paged_long_parts(gpu, H):
    """A workgroup's part of more than the 32 tiles whose pages it holds at once.  The
    requests share their pages."""
    B, n = 24, 14000
    a = _paged(gpu, "bf16", [n], [1], H, 64, H)
    g = torch.Generator().manual_seed(H)
    a["q"] = (torch.randn(B, H, 576, generator=g) * 0.6).to(torch.bfloat16).to(gpu)
    a["table"] = np.repeat(a["table"], B, 0)
    a["context"] = [n - 7 * b for b in range(B)]
    a["cu"] = _cu([1] * B)
    _check_paged(gpu, "bf16", a)


@pytest.mark.parametrize("qscale", [0.0, 1e-3, 6.0, 40.0])
@pytest.mark.parametrize("H", [16, 128])
def test_paged_score_ranges(gpu, qscale, H):
    _check_paged(gpu, "bf16", _paged(gpu, "bf16", [900], [2], H, 16, 9, qscale=qscale))


def test_paged_maxima_that_keep_growing(gpu):
    """Scores that rise from tile to tile, so that every tile moves the maximum."""
    a = _paged(gpu, "bf16", [1200], [1], 16, 16, 3)
    a["q"][:] = 0.25
    ramp = torch.linspace(-1, 1, 1201, device=gpu)[:, None].expand(-1, 576)
    at = torch.arange(1201, device=gpu)
    page = _dev(a["table"][0], gpu).long()
    a["cache"][page[at // 16], at % 16] = ramp.to(torch.bfloat16)
    _check_paged(gpu, "bf16", a, scale=1.0)
    a["cache"][page[at // 16], at % 16] = ramp.flip(0).to(torch.bfloat16)
    _check_paged(gpu, "bf16", a, scale=1.0)


def test_paged_strides(gpu):
    a = _paged(gpu, "bf16", [200, 50], [2, 1], 6, 16, 2, wide=True)
    o = torch.full((6, 3, 520), 7.0, dtype=torch.bfloat16, device=gpu).transpose(0, 1)
    r = _run_paged(gpu, a, o[..., :512])
    b = {**a, "q": a["q"].contiguous(), "cache": a["cache"].contiguous()}
    assert torch.equal(r, _run_paged(gpu, b)) and (o[..., 512:] == 7).all()
    h = {**a, "q": a["q"].transpose(0, 1).contiguous().transpose(0, 1)}
    assert torch.equal(r, _run_paged(gpu, h))
    e = {**a, "q": a["q"][:1, :1].expand(3, 6, 576)}
    assert torch.equal(_run_paged(gpu, e), _run_paged(gpu, {**e, "q": e["q"].contiguous()}))


@pytest.mark.parametrize("H", [16, 64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_paged_values_that_no_row_reads(gpu, H, bad):
    """Rows behind a request, unused blocks, and a node that only itself reads."""
    mask = np.array([[1], [3], [4], [1]], np.uint64)
    a = _paged(gpu, "bf16", [70, 33], [3, 1], H, 16, H, mask)
    clean = _run_paged(gpu, a).clone()
    cache = a["cache"]
    used = np.zeros(cache.shape[:2], bool)
    for b, n in enumerate((73, 34)):
        at = np.arange(n)
        used[a["table"][b][at // 16], at % 16] = True
    used[a["table"][0][72 // 16], 72 % 16] = False  # node 2, read by itself alone
    cache[torch.from_numpy(~used).to(gpu)] = bad
    a["q"][4:] = bad
    got = _run_paged(gpu, a)
    assert torch.equal(got[[0, 1, 3]], clean[[0, 1, 3]])
    assert not torch.isfinite(got[2]).all()


@pytest.mark.parametrize("H", [16, 128])
@pytest.mark.parametrize("context", [[40], [3000, 500]])
def test_paged_values_that_rows_read(gpu, H, context):
    """A NaN in one row of a context shows in that request's outputs, an infinite latent in its column."""
    a = _paged(gpu, "bf16", context, [1] * len(context), H, 16, 7)
    clean = _run_paged(gpu, a).clone()
    page, off = int(a["table"][0][1]), 3
    a["q"][..., 100] = 0  # the infinity does not enter the scores as 0 * inf ...
    keep = a["cache"][page, off].clone()
    a["cache"][page, off, 512] = float("nan")
    got = _run_paged(gpu, a)
    assert got[0].isnan().all()
    assert torch.equal(got[1:], _run_paged(gpu, {**a, "q": a["q"]})[1:])
    a["cache"][page, off] = keep
    assert torch.isfinite(clean).all()


def test_paged_tables_and_offsets_that_lie(gpu):
    """Whatever the table, lengths and offsets hold, nothing outside the tensors is touched."""
    a = _paged(gpu, "bf16", [50, 20], [2, 1], 32, 16, 3)
    base = torch.full((20, 32, 512), 7.0, dtype=torch.bfloat16, device=gpu)
    for table, context, cu in (([[-1, 10**9, 3, 0], [99, 1, 2, 3]], [50, 20], [0, 2, 3]),
                               (a["table"], [10**9, -5], [0, 2, 3]), (a["table"], [50, 20], [-5, 2, 900]),
                               (a["table"], [50, 20], [3, 1, 0])):
        r = latent_attention(a["q"], a["cache"], _dev(table, gpu), _dev(context, gpu), _dev(cu, gpu), None, base[5:8],
                             sm_scale=SCALE)
        torch.cuda.synchronize()
        assert (base[:5] == 7).all() and (base[8:] == 7).all() and r.isfinite().all()
    # An entry outside the cache reads as zeros.
    table = np.array(a["table"])
    zero = a["cache"].clone()
    zero[int(table[0, 1])] = 0
    want = _run_paged(gpu, {**a, "cache": zero})
    table[0, 1] = 10**6
    assert torch.equal(_run_paged(gpu, {**a, "table": table}), want)


def test_paged_keys_behind_the_tables_width(gpu):
    for H in (16, 128):
        _check_paged(gpu, "bf16", _paged(gpu, "bf16", [100, 30], [2, 1], H, 16, 2, width=4))


def test_paged_nothing_to_do(gpu):
    cache = torch.zeros(2, 16, 576, dtype=torch.float16, device=gpu)
    z = torch.empty(0, 4, 576, dtype=torch.float16, device=gpu)
    i = lambda *v: _dev(v, gpu)
    assert latent_attention(z, cache, torch.zeros(0, 1, dtype=torch.int32, device=gpu), i(), i(0), sm_scale=1.0).shape == (0, 4, 512)
    assert latent_attention(z, cache, torch.zeros(1, 1, dtype=torch.int32, device=gpu), i(5), i(0, 0), sm_scale=1.0).shape == (0, 4, 512)
    q = torch.ones(2, 4, 576, dtype=torch.float16, device=gpu)
    o = torch.full((2, 4, 512), 7.0, dtype=torch.float16, device=gpu)
    latent_attention(q, cache, torch.zeros(1, 1, dtype=torch.int32, device=gpu), i(5), i(0, 0), None, o, sm_scale=1.0)
    assert (o == 7).all()
    lse = torch.zeros(4, 2, device=gpu)
    latent_attention(q, cache[:0], torch.zeros(1, 0, dtype=torch.int32, device=gpu), i(0), i(0, 2), None, o, sm_scale=1.0, lse=lse)
    assert (o == 0).all() and torch.isneginf(lse).all()


def test_paged_past_32_bit_offsets(gpu):
    """A cache of more than 4 GiB, rows at its far end, blocks and tokens further apart than they are long."""
    blocks, size = 2**15 + 9, 64
    base = torch.zeros(blocks, size, 1160, dtype=torch.bfloat16, device=gpu)
    cache = base[..., 8:584]
    assert base.numel() > 2**31
    table = np.array([[blocks - 1, 3, blocks - 2]], np.int32)
    for page in table[0]:
        cache[int(page)] = torch.randn(size, 576, device=gpu).bfloat16()
    small = torch.stack([cache[int(p)] for p in table[0]])
    for H in (16, 128):
        q = (torch.randn(2, H, 576, device=gpu) * 0.6).bfloat16()
        a = dict(q=q, cache=cache, table=table, context=[180], cu=_cu([2]), mask=None)
        assert torch.equal(_run_paged(gpu, a), _run_paged(gpu, {**a, "cache": small, "table": np.arange(3)[None]}))
    del base, cache
    torch.cuda.empty_cache()


@pytest.mark.parametrize("H", [16, 128])
def test_paged_is_deterministic_and_runs_on_another_stream(gpu, H):
    a = _paged(gpu, "bf16", [3000, 10, 500], [1, 2, 1], H, 64, 4)
    want = _run_paged(gpu, a)
    for _ in range(3):
        assert torch.equal(_run_paged(gpu, a), want)
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    out = []
    torch.cuda.synchronize()
    for st in (s, t, s, t):  # two streams at once
        with torch.cuda.stream(st):
            out.append(_run_paged(gpu, a))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in out)


@pytest.mark.parametrize("H", [16, 128])
def test_paged_graphs(gpu, H):
    """Two captured graphs, replayed with lengths and values that changed."""
    a = _paged(gpu, "bf16", [700, 90], [1, 1], H, 64, 6)
    table, context, cu = _dev(a["table"], gpu), _dev(a["context"], gpu), _dev(a["cu"], gpu)
    q, cache = a["q"].clone(), a["cache"]
    _run_paged(gpu, a)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(latent_attention(q, cache, table, context, cu, sm_scale=SCALE))
        graphs.append(g)
    for i in range(4):
        q.normal_()
        context.copy_(torch.tensor([700 - 150 * i, 90 - 30 * i]))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = latent_attention(q, cache, table, context, cu, sm_scale=SCALE)
        assert all(torch.equal(o, want) for o in outs)


# --- the expanded form over packed prompts -----------------------------------------

def _prompt(dev, dtype, lq, lk, HQ, HK, causal, seed, pad=0, split=False, scale=None, qscale=1.0):
    g = torch.Generator().manual_seed(seed)
    T, TK = sum(lq) + pad, sum(lk) + pad
    q = (torch.randn(T, HQ, 192, generator=g) * qscale).to(DT[dtype]).to(dev)
    kv = torch.randn(TK, HK, 256, generator=g).to(DT[dtype]).to(dev)
    k, v = kv[..., :128], kv[..., 128:]
    if split:
        k, v = k.contiguous(), v.transpose(0, 1).contiguous().transpose(0, 1)
    kr = torch.randn(TK, 64, generator=g).to(DT[dtype]).to(dev)
    cq, ck = _cu(lq), _cu(lk)
    o = torch.full((T, HQ, 128), 7.0, dtype=DT[dtype], device=dev)
    lse = torch.full((HQ, T), 7.0, device=dev)
    r = latent_varlen_attention(q, k, v, kr, _dev(cq, dev), o, cu_seqlens_k=None if lq == lk else _dev(ck, dev), causal=causal,
                                sm_scale=scale, lse=lse)
    assert r is o
    torch.cuda.synchronize()
    scale = SCALE if scale is None else scale
    ref = L.packed(_np(q), _np(k), _np(v), _np(kr), cq, ck, causal, scale)
    _check(o, lse, *ref, dtype, max(lk, default=1), 192, float(np.abs(_np(v)).max(initial=0)), sum(lq))
    if pad:
        assert (_np(o)[sum(lq):] == 7).all() and (_np(lse)[:, sum(lq):] == 7).all(), "rows behind the last sequence changed"


PROMPTS = [
    ([1], None), ([63, 64, 65], None), ([0, 1, 31, 0, 33, 0], None), ([255, 256, 257, 2], None), ([700], None),
    ([513, 5, 129], None), ([1, 3, 70], [200, 3, 75]), ([5, 70, 300], [2, 0, 260]),
    ([64] * 9, [1, 63, 64, 65, 127, 128, 129, 191, 300]),
]


@pytest.mark.parametrize("lq,lk", PROMPTS, ids=lambda x: "_".join(map(str, x)) if x else "same")
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_lengths(gpu, lq, lk, dtype, causal):
    _prompt(gpu, dtype, lq, lk or lq, 2, 2, causal, seed=len(lq) * 1000 + sum(lq), pad=3)


@pytest.mark.parametrize("HQ,HK", [(1, 1), (4, 4), (6, 2), (5, 1), (16, 16), (40, 8), (16, 1), (128, 128)])
def test_prompt_heads(gpu, HQ, HK):
    _prompt(gpu, "bf16", [70, 130], [70, 130], HQ, HK, True, seed=HQ, split=HK % 2 == 0)


# Rows by heads on both sides of where the launch changes its form.
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lq,lk,H", [([3000, 700], None, 16), ([900, 1, 257], [1500, 700, 300], 64), ([2100] * 2, [2000, 2500], 16)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_prompt_of_many_rows(gpu, lq, lk, H, causal, dtype):
    _prompt(gpu, dtype, lq, lk or lq, H, H, causal, seed=H)


def test_prompt_many_short_sequences(gpu):
    rng = np.random.default_rng(0)
    lq = rng.integers(0, 9, 300).tolist()
    _prompt(gpu, "fp16", lq, lq, 2, 2, True, seed=3)
    lq = rng.integers(0, 90, 100).tolist()
    _prompt(gpu, "bf16", lq, lq, 16, 16, True, seed=4)


@pytest.mark.parametrize("B", [64, 65, 129])
def test_prompt_batches_around_a_wave(gpu, B):
    lq = [(7 * b) % 11 for b in range(B)]
    lq[B // 2] = 600
    _prompt(gpu, "bf16", lq, lq, 1, 1, True, seed=B)


@pytest.mark.parametrize("qscale", [0.0, 1e-3, 8.0, 40.0])
@pytest.mark.parametrize("n,H", [(260, 1), (1700, 32)])
def test_prompt_score_ranges(gpu, qscale, n, H):
    _prompt(gpu, "bf16", [n], [n], H, H, True, seed=9, qscale=qscale)


def test_prompt_scale(gpu):
    _prompt(gpu, "fp16", [100], [100], 1, 1, True, seed=9, scale=0.5)


def _prompt_inputs(gpu, T, H, dtype=torch.bfloat16, seed=2):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(*s, generator=g).to(dtype).to(gpu) for s in ((T, H, 192), (T, H, 128), (T, H, 128), (T, 64))]


def test_prompt_strides(gpu):
    q, k, v, kr = _prompt_inputs(gpu, 130, 4)
    cu = _dev([0, 90, 130], gpu)
    want = latent_varlen_attention(q, k, v, kr, cu)
    hm = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)
    wide = lambda t: torch.cat((t, t[..., :24]), -1)[..., :t.shape[-1]]
    o = torch.full((4, 130, 136), 7.0, dtype=q.dtype, device=gpu).transpose(0, 1)
    assert torch.equal(latent_varlen_attention(hm(q), wide(k), hm(v), wide(kr), cu, o[..., :128]), want)
    assert (o[..., 128:] == 7).all()
    one = [q[:1, :1].expand(130, 4, 192), k[:1, :1].expand(130, 4, 128), v[:1].expand(130, 4, 128), kr[:1].expand(130, 64)]
    assert torch.equal(latent_varlen_attention(*one, cu), latent_varlen_attention(*(t.contiguous() for t in one), cu))


@pytest.mark.parametrize("T,H", [(200, 2), (1300, 64)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_prompt_values_that_no_row_reads(gpu, T, H, bad):
    """Other sequences and rows behind the last one hold NaN or infinities; so does
    the last key, which the last query alone reads."""
    q, k, v, kr = _prompt_inputs(gpu, T, H)
    n = T // 2
    cu = _dev([0, n, T - 23], gpu)
    clean = latent_varlen_attention(q, k, v, kr, cu).clone()
    for t in (k, v, kr):
        t[n - 1] = bad
        t[T - 23:] = bad
    q[T - 23:] = bad
    got = latent_varlen_attention(q, k, v, kr, cu)
    keep = [i for i in range(T - 23) if i != n - 1]
    assert torch.equal(got[keep], clean[keep])
    assert not torch.isfinite(got[n - 1]).all()


@pytest.mark.parametrize("T,H", [(900, 4), (1000, 64)])
def test_prompt_is_deterministic_streams_and_graphs(gpu, T, H):
    q, k, v, kr = _prompt_inputs(gpu, T, H)
    cu = _dev([0, 1, 400, T], gpu)
    want = latent_varlen_attention(q, k, v, kr, cu)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = latent_varlen_attention(q, k, v, kr, cu)
    s.synchronize()
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = latent_varlen_attention(q, k, v, kr, cu)
    for i in range(3):
        q.normal_()
        cu.copy_(torch.tensor([0, 1 + i, 400 - i, T]))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, latent_varlen_attention(q, k, v, kr, cu))


def test_prompt_offsets_that_lie_are_held_inside_the_tensors(gpu):
    q, k, v, kr = _prompt_inputs(gpu, 50, 1)
    base = torch.full((80, 1, 128), 7.0, device=gpu, dtype=torch.bfloat16)
    for cu in ([0, 500], [-5, 30, 20, 70], [40, 10, 60]):
        latent_varlen_attention(q, k, v, kr, _dev(cu, gpu), base[10:60])
        torch.cuda.synchronize()
        assert (base[:10] == 7).all() and (base[60:] == 7).all()


def test_prompt_nothing_to_do(gpu):
    q, k, v, kr = _prompt_inputs(gpu, 3, 2)
    for cu in ([0], [0, 0, 0]):
        assert latent_varlen_attention(q[:0], k[:0], v[:0], kr[:0], _dev(cu, gpu)).shape == (0, 2, 128)
    r = latent_varlen_attention(q, k[:0], v[:0], kr[:0], _dev([0, 3], gpu), cu_seqlens_k=_dev([0, 0], gpu))
    assert (r == 0).all()


def test_prompt_past_32_bit_offsets(gpu):
    T, H = 2**15 + 70, 128
    kv = torch.zeros(T, H, 640, dtype=torch.bfloat16, device=gpu)
    assert kv.numel() > 2**31
    g = torch.Generator().manual_seed(0)
    n = 70
    kv[-n:] = torch.randn(n, H, 640, generator=g).bfloat16().to(gpu)
    q = torch.randn(n, H, 192, generator=g).bfloat16().to(gpu)
    kr = torch.zeros(T, 64, dtype=torch.bfloat16, device=gpu)
    kr[-n:] = torch.randn(n, 64, generator=g).bfloat16().to(gpu)
    got = latent_varlen_attention(q, kv[..., :128], kv[..., 512:], kr, _dev([0, n], gpu), cu_seqlens_k=_dev([T - n, T], gpu))
    cut = kv[-n:].clone()
    assert torch.equal(got, latent_varlen_attention(q, cut[..., :128], cut[..., 512:], kr[-n:].clone(), _dev([0, n], gpu)))
    del kv
    torch.cuda.empty_cache()


# --- together --------------------------------------------------------------------

@pytest.mark.parametrize("interleaved", [False, True])
def test_a_prompt_and_decoding_together(gpu, interleaved):
    """Two prompts through the expanded form, then two steps through the absorbed one, with the framework's products
    between: slots, norm, rotation and writes, expansion, attention, the heads' projections.  Every step's output
    against the expanded form in 64 bits of the rounded latents, queries and weights."""
    dt, H, hidden, size = torch.bfloat16, 4, 256, 16
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g)
    w_q, w_down = (r(H * 192, hidden) / 16).to(dt).to(gpu), (r(576, hidden) / 16).to(dt).to(gpu)
    w_up = (r(H, 256, 512) / 23).to(dt).to(gpu)  # a head's key rows, then its value rows
    w_k = w_up[:, :128].transpose(1, 2).contiguous()  # (H, 512, 128): the query's side of the key projection
    w_v = w_up[:, 128:].contiguous()  # (H, 128, 512)
    norm = (1 + 0.1 * r(512)).to(dt).to(gpu)
    freqs = rotary_frequencies(64, scaling="turns", factor=4.0, original_length=4096, device=gpu)
    B, lens = 2, [37, 20]
    cache = torch.zeros(12, size, 576, dtype=dt, device=gpu)
    table = torch.zeros(B, 5, dtype=torch.int32, device=gpu)
    free, start = torch.randperm(12, generator=g).int().to(gpu), torch.zeros(1, dtype=torch.int32, device=gpu)
    lengths = torch.zeros(B, dtype=torch.int32, device=gpu)
    seen = [[] for _ in range(B)]  # each request's latents and rotated keys, as rounded

    def per_head(x, w):  # (T, H, K) by (H, N, K): the grouped product with heads as experts
        T = x.shape[0]
        off = torch.arange(0, (H + 1) * T, T, dtype=torch.int32, device=gpu)
        y = moe_matmul(x.transpose(0, 1).reshape(H * T, -1), w, off)
        return y.view(H, T, -1).transpose(0, 1)

    def step(counts, prompt):
        nonlocal lengths
        T = sum(counts)
        x = r(T, hidden).to(dt).to(gpu)
        s = assign_slots(lengths, _dev(counts, gpu), table, free, size, T, free_start=start)
        q = matmul(x, w_q.T).view(T, H, 192)
        rotary(q, s.positions, freqs, q, first=128, interleaved=interleaved)
        down = matmul(x, w_down.T)
        c, kr = torch.empty(T, 512, dtype=dt, device=gpu), torch.empty(T, 64, dtype=dt, device=gpu)
        write_latent(down[:, :512], down[:, 512:], cache, s.slots, weight=norm, positions=s.positions, freqs=freqs,
                     interleaved=interleaved, c_out=c, k_out=kr)
        want = L.rotate(_np(down)[:, None, 512:], s.positions.cpu().numpy(), freqs.cpu().numpy(), 0, interleaved)
        assert np.abs(_np(kr) - want[:, 0]).max() <= 2.0**-7 * np.abs(want).max()
        if prompt:
            kv = matmul(c, w_up.reshape(H * 256, 512).T).view(T, H, 256)
            o = latent_varlen_attention(q, kv[..., :128], kv[..., 128:], kr, s.cu_seqlens)
        else:
            full = torch.empty(T, H, 576, dtype=dt, device=gpu)
            full[..., :512] = per_head(q[..., :128], w_k)
            full[..., 512:] = q[..., 128:]
            o = per_head(latent_attention(full, cache, table, lengths, s.cu_seqlens, sm_scale=SCALE), w_v)
        lengths += _dev(counts, gpu)
        start.add_(s.taken)
        # The reference: keys and values from the rounded latents, in 64 bits.
        up, row = _np(w_up).astype(np.float64), 0
        for b, n in enumerate(counts):
            seen[b] += [(_np(c[row + i]), _np(kr[row + i])) for i in range(n)]
            lat, rope = (np.stack([t[j] for t in seen[b]]).astype(np.float64) for j in (0, 1))
            keys = np.einsum("tc,hdc->thd", lat, up[:, :128])
            vals = np.einsum("tc,hdc->thd", lat, up[:, 128:])
            keys = np.concatenate([keys, np.broadcast_to(rope[:, None], keys.shape[:2] + (64,))], -1)
            ref, _, mag, spread = L.attend(_np(q[row:row + n]), keys, vals, R.causal_reads(n, len(lat)), SCALE)
            # Expanded: keys and values rounded (half a step each, so scores by 2^-9 of the spread), then the
            # weights and the output.  Absorbed: the query rounded, the latents' sum and the output: the sum's
            # rounding, half a step of 512 latents, goes through the value projection.
            h = 2.0**-9
            tol = (np.exp(2 * h * spread * 2) - 1 + 4 * h) * mag
            if not prompt:
                top = np.abs(lat).max() * np.abs(up[:, 128:]).sum(-1).max()
                tol = tol + 2 * h * top
            assert (np.abs(_np(o[row:row + n]) - ref) <= tol + 1e-3).all()
            row += n

    step(lens, True)
    step([1, 1], False)
    step([2, 1], False)  # a drafted chain of two beside a single token
