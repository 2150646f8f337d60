"""GPU parity of the packed prompt attention, the paged cache and the tree
attention against the float64 oracle (oracle/serving_ref.py), at the sizes and
masks where they can go wrong.  Tolerances come from the arithmetic
(serving_ref.tolerances); integers and copies must be equal."""

import itertools

import numpy as np
import pytest
import torch

from gfx950_gluon_tutorials_amd.attention import assign_slots, tree_attention, varlen_attention, write_cache
from oracle import serving_ref as R

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
SUBNORMAL = {"fp16": 2.0**-25, "bf16": 0.0}



def _cu(lengths):
    return np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)


def _np(t):
    return t.detach().float().cpu().numpy()


def _check(got, lse, ref, lse_ref, mag, spread, dtype, longest, D, vmax, rows):
    to, tl = R.tolerances(ref, lse_ref, mag, spread, torch.finfo(DT[dtype]).eps, longest, D, vmax, SUBNORMAL[dtype])
    got, ref, to = _np(got)[:rows], ref[:rows], to[:rows]
    assert np.isfinite(got).all()
    off = np.abs(got - ref) - to
    assert (off <= 0).all(), f"o is {off.max():.3g} past its bound at {np.unravel_index(off.argmax(), off.shape)}"
    lse, lse_ref, tl = _np(lse)[:, :rows], lse_ref[:, :rows], tl[:, :rows]
    none = np.isneginf(lse_ref)
    assert (np.isneginf(lse) == none).all()
    off = np.abs(np.where(none, 0, lse) - np.where(none, 0, lse_ref)) - np.where(none, 0, tl)
    assert (off <= 0).all(), f"lse is {off.max():.3g} past its bound"


# --- packed prompts -----------------------------------------------------------

def _prompt(dev, dtype, lq, lk, HQ, HK, D, causal, seed, pad=0, fused=False, scale=None, qscale=1.0):
    g = torch.Generator().manual_seed(seed)
    T, TK = sum(lq) + pad, sum(lk) + pad
    if fused:
        qkv = torch.randn(T, HQ + 2 * HK, D, generator=g).to(DT[dtype]).to(dev)
        q, k, v = qkv[:, :HQ], qkv[:, HQ:HQ + HK], qkv[:, HQ + HK:]
    else:
        q = (torch.randn(T, HQ, D, generator=g) * qscale).to(DT[dtype]).to(dev)
        k, v = (torch.randn(TK, HK, D, generator=g).to(DT[dtype]).to(dev) for _ in range(2))
    cq, ck = _cu(lq), _cu(lk)
    o = torch.full((T, HQ, D), 7.0, dtype=DT[dtype], device=dev)
    lse = torch.full((HQ, T), 7.0, device=dev)
    scale = D**-0.5 if scale is None else scale
    same = lq == lk
    r = varlen_attention(q, k, v, torch.from_numpy(cq).to(dev), o,
                         cu_seqlens_k=None if same else torch.from_numpy(ck).to(dev), causal=causal, sm_scale=scale,
                         lse=lse)
    assert r is o
    torch.cuda.synchronize()
    ref = R.packed_attention(_np(q), _np(k), _np(v), cq, ck, lambda b: R.causal_reads(lq[b], lk[b], causal), scale)
    _check(o, lse, *ref, dtype, max(lk, default=1), D, float(np.abs(_np(v)).max(initial=0)), sum(lq))
    if pad:
        assert (_np(o)[sum(lq):] == 7).all() and (_np(lse)[:, sum(lq):] == 7).all(), "rows behind the last sequence changed"


PROMPTS = [
    ([1], None),
    ([63, 64, 65], None),
    ([0, 1, 31, 0, 33, 0], None),
    ([255, 256, 257, 2], None),
    ([700], None),
    ([513, 5, 129], None),
    ([1, 3, 70], [200, 3, 75]),      # cached prefixes
    ([5, 70, 300], [2, 0, 260]),     # fewer keys than queries: rows that read nothing
    ([64] * 9, [1, 63, 64, 65, 127, 128, 129, 191, 300]),
]


@pytest.mark.parametrize("lq,lk", PROMPTS, ids=lambda x: "_".join(map(str, x)) if x else "same")
@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("fp16", 128), ("bf16", 64), ("fp16", 64)])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_lengths(gpu, lq, lk, dtype, D, causal):
    _prompt(gpu, dtype, lq, lk or lq, 2, 1, D, causal, seed=len(lq) * 1000 + sum(lq), pad=3)


@pytest.mark.parametrize("HQ,HK", [(1, 1), (4, 4), (6, 2), (5, 1), (16, 8), (40, 8), (16, 1)])
def test_prompt_heads(gpu, HQ, HK):
    _prompt(gpu, "bf16", [70, 130], [70, 130], HQ, HK, 128, True, seed=HQ)


def test_prompt_many_short_sequences(gpu):
    rng = np.random.default_rng(0)
    lq = rng.integers(0, 9, 300).tolist()
    _prompt(gpu, "fp16", lq, lq, 2, 2, 64, True, seed=3)


@pytest.mark.parametrize("B", [64, 65, 129])
def test_prompt_batches_around_a_wave(gpu, B):
    lq = [(7 * b) % 11 for b in range(B)]
    lq[B // 2] = 600
    _prompt(gpu, "bf16", lq, lq, 1, 1, 64, True, seed=B)


def test_prompt_fused_projection(gpu):
    _prompt(gpu, "bf16", [200, 61], [200, 61], 8, 2, 128, True, seed=5, fused=True, pad=1)


def test_prompt_head_major_and_wide_strides(gpu):
    g = torch.Generator().manual_seed(1)
    lq, HQ, HK, D = [90, 40], 4, 2, 64
    T = sum(lq)
    q = torch.randn(HQ, T, D, generator=g).to(DT["bf16"]).to(gpu).transpose(0, 1)
    k = torch.randn(T, HK, D + 8, generator=g).to(DT["bf16"]).to(gpu)[:, :, :D]
    v = torch.randn(HK, 2 * T, D, generator=g).to(DT["bf16"]).to(gpu)[:, ::2].transpose(0, 1)
    o = torch.empty(HQ, T, D, dtype=q.dtype, device=gpu).transpose(0, 1)
    cu = _cu(lq)
    lse = torch.empty(HQ, T, device=gpu)
    varlen_attention(q, k, v, torch.from_numpy(cu).to(gpu), o, lse=lse)
    ref = R.packed_attention(_np(q), _np(k), _np(v), cu, cu, lambda b: R.causal_reads(lq[b], lq[b]), D**-0.5)
    _check(o, lse, *ref, "bf16", 90, D, float(np.abs(_np(v)).max()), T)


@pytest.mark.parametrize("qscale", [0.0, 1e-3, 8.0, 40.0])
def test_prompt_score_ranges(gpu, qscale):
    _prompt(gpu, "bf16", [260], [260], 1, 1, 128, True, seed=9, qscale=qscale)


def test_prompt_scale(gpu):
    _prompt(gpu, "fp16", [100], [100], 1, 1, 128, True, seed=9, scale=0.5)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_prompt_values_that_no_row_reads(gpu, D, bad):
    """Other sequences and rows behind the last one hold NaN or infinities; so does
    the last key, which the last query alone reads."""
    g = torch.Generator().manual_seed(2)
    lq = [100, 77]
    cu = _cu(lq)
    q, k, v = (torch.randn(200, 1, D, generator=g).to(DT["bf16"]) for _ in range(3))
    clean = varlen_attention(*(t.to(gpu) for t in (q, k, v)), torch.from_numpy(cu).to(gpu))
    for t in (k, v):
        t[99] = bad
        t[177:] = bad
    q[177:] = bad
    got = varlen_attention(*(t.to(gpu) for t in (q, k, v)), torch.from_numpy(cu).to(gpu))
    keep = [i for i in range(177) if i != 99]
    assert torch.equal(got[keep], clean[keep])
    assert not torch.isfinite(got[99]).all()


def test_prompt_is_deterministic_and_runs_on_another_stream(gpu):
    g = torch.Generator().manual_seed(4)
    q, k, v = (torch.randn(900, 4, 128, generator=g).to(DT["bf16"]).to(gpu) for _ in range(3))
    cu = torch.tensor([0, 1, 400, 900], dtype=torch.int32, device=gpu)
    a = varlen_attention(q, k, v, cu)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = varlen_attention(q, k, v, cu)
    s.synchronize()
    assert torch.equal(a, b)


def test_prompt_offsets_that_lie_are_held_inside_the_tensors(gpu):
    """Offsets past the packed rows or out of order read and write nothing outside."""
    q = torch.randn(50, 1, 64, device=gpu, dtype=torch.bfloat16)
    base = torch.full((80, 1, 64), 7.0, device=gpu, dtype=torch.bfloat16)
    for cu in ([0, 500], [-5, 30, 20, 70], [40, 10, 60]):
        varlen_attention(q, q, q, torch.tensor(cu, dtype=torch.int32, device=gpu), base[10:60])
        torch.cuda.synchronize()
        assert (base[:10] == 7).all() and (base[60:] == 7).all()


def test_prompt_nothing_to_do(gpu):
    z = torch.empty(0, 2, 64, device=gpu, dtype=torch.float16)
    assert varlen_attention(z, z, z, torch.zeros(1, dtype=torch.int32, device=gpu)).shape == (0, 2, 64)
    assert varlen_attention(z, z, z, torch.zeros(4, dtype=torch.int32, device=gpu)).shape == (0, 2, 64)
    q = torch.ones(3, 2, 64, device=gpu, dtype=torch.float16)
    cu = torch.tensor([0, 3], dtype=torch.int32, device=gpu)
    assert (varlen_attention(q, z, z, cu, cu_seqlens_k=torch.zeros(2, dtype=torch.int32, device=gpu)) == 0).all()


# --- the paged cache ------------------------------------------------------------

def _cache(g, blocks, size, HK, D, dtype, dev, order="bshd", fill=None):
    shape = (blocks, size, HK, D) if order == "bshd" else (blocks, HK, size, D)
    out = []
    for _ in range(2):
        t = torch.randn(shape, generator=g) if fill is None else torch.full(shape, fill)
        t = t.to(DT[dtype]).to(dev)
        out.append(t if order == "bshd" else t.transpose(1, 2))
    return out


@pytest.mark.parametrize("T,HK,D,size,order", [
    (1, 1, 64, 16, "bshd"), (5, 3, 128, 16, "bhsd"), (130, 8, 128, 64, "bshd"), (77, 2, 64, 1024, "bhsd"),
    (1000, 16, 64, 32, "bshd"), (64, 5, 128, 16, "bhsd"),
])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_write_cache(gpu, T, HK, D, size, order, dtype):
    g = torch.Generator().manual_seed(T)
    blocks = 3 + 2 * T // size
    kc, vc = _cache(g, blocks, size, HK, D, dtype, gpu, order)
    qkv = torch.randn(T, 2 * HK + 1, D, generator=g).to(DT[dtype]).to(gpu)
    k, v = qkv[:, :HK], qkv[:, HK:2 * HK]
    slots = torch.randperm(blocks * size, generator=g)[:T]
    slots[::7] = torch.tensor([-1, blocks * size, -2**40, 2**40])[torch.arange(len(slots[::7])) % 4]
    wk, wv = (t.contiguous().reshape(-1, HK, D).cpu().clone() for t in (kc, vc))
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < blocks * size:
            wk[s], wv[s] = k[t].cpu(), v[t].cpu()
    write_cache(k, v, kc, vc, slots.to(gpu))
    assert torch.equal(kc.contiguous().reshape(-1, HK, D).cpu(), wk)
    assert torch.equal(vc.contiguous().reshape(-1, HK, D).cpu(), wv)


def test_write_cache_past_32_bit_offsets(gpu):
    """A cache of more than 4 GiB per tensor."""
    blocks, size, HK, D = 2**16 + 9, 64, 8, 64
    kc, vc = (torch.zeros(blocks, size, HK, D, dtype=torch.bfloat16, device=gpu) for _ in range(2))
    k, v = (torch.randn(2, HK, D, device=gpu).bfloat16() for _ in range(2))
    write_cache(k, v, kc, vc, torch.tensor([blocks * size - 1, 2**22 + 5], device=gpu))
    for t, s in enumerate((blocks * size - 1, 2**22 + 5)):
        assert torch.equal(kc[s // size, s % size], k[t]) and torch.equal(vc[s // size, s % size], v[t])
    # The attention reads the same rows back: one key's softmax is that key's value.
    table = torch.tensor([[blocks - 1]], dtype=torch.int32, device=gpu)
    kc[blocks - 1, 0], vc[blocks - 1, 0] = k[0], v[0]
    o = tree_attention(k[:1], kc, vc, table, torch.zeros(1, dtype=torch.int32, device=gpu),
                       torch.tensor([0, 1], dtype=torch.int32, device=gpu))
    assert torch.equal(o[0], v[0])
    del kc, vc
    torch.cuda.empty_cache()


def test_write_cache_of_more_rows_than_a_launch_has_waves(gpu):
    T, HK, D, blocks, size = 2**26 + 77, 8, 64, 3, 16
    kc, vc = (torch.zeros(blocks, size, HK, D, dtype=torch.float16, device=gpu) for _ in range(2))
    k, v = (torch.randn(1, HK, D, device=gpu).half().expand(T, HK, D) for _ in range(2))
    slots = torch.full((T,), -1, dtype=torch.int64, device=gpu)
    taken = {0: 5, 2**24 - 1: 6, 2**24: 7, T // 2: 40, T - 1: 47}
    for t, s in taken.items():
        slots[t] = s
    write_cache(k, v, kc, vc, slots)
    for got, row in ((kc, k[0]), (vc, v[0])):
        want = torch.zeros_like(got).view(-1, HK, D)
        want[list(taken.values())] = row
        assert torch.equal(got.view(-1, HK, D), want)


SLOTS = [
    # lengths, counts, size, width, free, start, T - sum(counts)
    ([0], [1], 16, 4, 4, None, 0),
    ([5, 16, 0, 15, 33], [1, 1, 0, 1, 30], 16, 8, 20, 0, 5),
    ([0, 0, 0], [100, 1, 64], 32, 8, 20, 3, 0),
    ([7, 9], [40, 40], 16, 8, 4, 1, 0),      # the free list runs out
    ([7, 9], [40, 40], 16, 2, 50, 0, 3),     # the table is too narrow
    ([3, 200], [5, 9], 16, 4, 50, 0, 0),     # a context past the table's width already
    ([-4, 3], [-2, 5], 16, 4, 50, 0, 2),     # negative counts as none
    ([4, 4], [0, 0], 16, 4, 9, 0, 4),
    ([4, 10], [9, 9], 16, 4, 9, 0, -5),      # fewer rows than tokens
    ([1], [100000], 16, 7000, 7000, 0, 1),
    ([10], [50], 7, 20, 20, 0, 0),           # any block size
]


@pytest.mark.parametrize("lengths,counts,size,width,free,start,pad", SLOTS)
def test_assign_slots(gpu, lengths, counts, size, width, free, start, pad):
    _slots(gpu, lengths, counts, size, width, free, start, sum(max(c, 0) for c in counts) + pad)


@pytest.mark.parametrize("B", [63, 64, 255, 256, 257, 1000, 4096])
def test_assign_slots_batches(gpu, B):
    rng = np.random.default_rng(B)
    counts = rng.integers(0, 40, B).tolist()
    _slots(gpu, rng.integers(0, 200, B).tolist(), counts, 16, 16, 16 * B, 2, sum(counts) + 9)


def _slots(dev, lengths, counts, size, width, free, start, T):
    rng = np.random.default_rng(len(lengths))
    ids = rng.permutation(free + len(lengths) * width).astype(np.int32)
    table = ids[free:].reshape(len(lengths), width).copy()
    cu, slots, pos, taken, after = R.slots(lengths, counts, table, ids[:free], start or 0, size, T)
    dt = torch.from_numpy(table).to(dev)
    args = [torch.tensor(x, dtype=torch.int32, device=dev) for x in (lengths, counts)]
    for _ in range(2):  # the same call twice gives the same
        r = assign_slots(*args, dt, torch.from_numpy(ids[:free]).to(dev), size, T,
                         free_start=None if start is None else torch.tensor([start], dtype=torch.int32, device=dev))
        assert r.cu_seqlens.tolist() == cu.tolist()
        assert r.taken.tolist() == [taken]
        assert np.array_equal(r.positions.cpu().numpy(), pos)
        assert np.array_equal(r.slots.cpu().numpy(), slots)
        assert np.array_equal(dt.cpu().numpy(), after)


def test_assign_slots_nothing_to_do(gpu):
    e = torch.empty(0, dtype=torch.int32, device=gpu)
    r = assign_slots(e, e, e.reshape(0, 4), e, 16, 3)
    assert r.cu_seqlens.tolist() == [0] and r.taken.tolist() == [0] and r.slots.tolist() == [-1] * 3
    assert assign_slots(e, e, e.reshape(0, 4), e, 16, 0).slots.shape == (0,)


# --- attention over the cache -----------------------------------------------------

def _bits(rows, words):
    out = np.zeros((len(rows), words), np.uint64)
    for i, r in enumerate(rows):
        for j in r:
            out[i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return out


def _tree(dev, dtype, ctx, nodes, HQ, HK, D, size, order="bshd", mask="chain", seed=0, pad=0, poison=None, scale=None,
          qscale=1.0, width=None):
    g = torch.Generator().manual_seed(seed)
    rng = np.random.default_rng(seed)
    total = [c + n for c, n in zip(ctx, nodes)]
    used = [-(-t // size) for t in total]
    width = width or max(1, max(used)) + 2
    blocks = sum(used) + 3
    ids = rng.permutation(blocks).astype(np.int32)
    table = np.full((len(ctx), width), 2**30, np.int32)  # entries that nobody may read
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = ids[at:at + n]
        at += n
    kc, vc = _cache(g, blocks, size, HK, D, dtype, dev, order)
    T = sum(nodes) + pad
    q = (torch.randn(T, HQ, D, generator=g) * qscale).to(DT[dtype]).to(dev)
    if poison is not None:  # every cache row that no request holds
        held = torch.zeros(blocks * size, dtype=torch.bool)
        for b, t in enumerate(total):
            for p in range(t):
                held[int(table[b, p // size]) * size + p % size] = True
        for c in (kc, vc):
            c[(~held).reshape(blocks, size).to(dev)] = poison
    words, bits = 0, None
    if mask != "chain":
        words = max(1, -(-max(nodes) // 64))
        rows = []
        for n in nodes:
            sees = []
            for i in range(n):
                if mask == "tree":
                    p = int(rng.integers(max(0, i - 4), i)) if i and rng.random() < 0.9 else -1
                    sees.append((sees[p] if p >= 0 else set()) | {i})
                elif mask == "random":
                    sees.append(set(np.flatnonzero(rng.random(n) < 0.5).tolist()))
                else:
                    sees.append(set())
            rows += sees
        bits = _bits(rows + [set()] * pad, words)
    cu = _cu(nodes)
    o = torch.full((T, HQ, D), 7.0, dtype=DT[dtype], device=dev)
    lse = torch.full((HQ, T), 7.0, device=dev)
    scale = D**-0.5 if scale is None else scale
    dmask = None if bits is None else torch.from_numpy(bits.view(np.int64)).to(dev)
    if dmask is not None and words == 1:
        dmask = dmask.reshape(-1)
    r = tree_attention(q, kc, vc, torch.from_numpy(table).to(dev), torch.tensor(ctx, dtype=torch.int32, device=dev),
                       torch.from_numpy(cu).to(dev), dmask, o, sm_scale=scale, lse=lse)
    assert r is o
    torch.cuda.synchronize()
    fk, fv = (_np(c.contiguous().reshape(-1, HK, D)) for c in (kc, vc))
    rows_of = [[int(table[b, p // size]) * size + p % size for p in range(t)] for b, t in enumerate(total)]
    flat = list(itertools.chain(*rows_of))
    ref = R.packed_attention(_np(q), fk[flat], fv[flat], cu, _cu(total), lambda b: R.tree_reads(
        None if bits is None else bits[cu[b]:cu[b + 1]], ctx[b], nodes[b]), scale)
    _check(o, lse, *ref, dtype, max(total), D, float(np.abs(np.nan_to_num(fv[flat])).max(initial=0)), sum(nodes))
    if pad:
        assert (_np(o)[sum(nodes):] == 7).all() and (_np(lse)[:, sum(nodes):] == 7).all()


TREES = [
    ([0], [1]), ([1], [1]), ([15, 16, 17], [1, 1, 1]), ([31, 32, 33, 63, 64, 65, 127, 128, 129], [1] * 9),
    ([700], [1]), ([0, 5, 300], [3, 1, 7]), ([100, 0, 40], [0, 2, 0]), ([33, 2000], [16, 17]), ([50], [64]),
    ([128, 3], [65, 130]),
]


@pytest.mark.parametrize("ctx,nodes", TREES, ids=lambda x: "_".join(map(str, x)))
@pytest.mark.parametrize("dtype,D,size,order", [("bf16", 128, 16, "bshd"), ("fp16", 64, 64, "bhsd"),
                                                ("fp16", 128, 128, "bhsd"), ("bf16", 64, 32, "bshd")])
@pytest.mark.parametrize("mask", ["chain", "tree"])
def test_tree_lengths(gpu, ctx, nodes, dtype, D, size, order, mask):
    _tree(gpu, dtype, ctx, nodes, 4, 2, D, size, order, mask, seed=sum(ctx) + sum(nodes), pad=2)


@pytest.mark.parametrize("mask", ["random", "none"])
@pytest.mark.parametrize("ctx", [[0, 0], [0, 90]])
def test_tree_rows_that_read_few_or_none(gpu, mask, ctx):
    _tree(gpu, "bf16", ctx, [20, 70], 4, 2, 128, 16, mask=mask, seed=11)


@pytest.mark.parametrize("HQ,HK", [(1, 1), (8, 8), (5, 1), (6, 2), (16, 1), (17, 1), (24, 2), (64, 8), (33, 1), (64, 1), (80, 1)])
@pytest.mark.parametrize("n", [1, 3, 20])
def test_tree_heads(gpu, HQ, HK, n):
    _tree(gpu, "bf16", [77, 300], [n, 2], HQ, HK, 128, 16, seed=HQ)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype,D,size,order", [("bf16", 128, 16, "bshd"), ("fp16", 64, 64, "bhsd")])
def test_tree_cache_rows_that_nobody_holds(gpu, bad, dtype, D, size, order):
    _tree(gpu, dtype, [1, 40, 200], [1, 3, 2], 4, 2, D, size, order, "tree", seed=5, poison=bad)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("n", [2, 30])
def test_tree_nodes_that_a_row_does_not_read(gpu, bad, n):
    """A node's NaN stays with the rows that read it."""
    g = torch.Generator().manual_seed(8)
    kc, vc = _cache(g, 12, 16, 1, 128, "bf16", gpu)
    q = torch.randn(n, 4, 128, generator=g).to(DT["bf16"]).to(gpu)
    table = torch.arange(12, dtype=torch.int32, device=gpu)[None]
    ctx = torch.tensor([50], dtype=torch.int32, device=gpu)
    cu = torch.tensor([0, n], dtype=torch.int32, device=gpu)
    mask = torch.tensor([1 << i for i in range(n)], device=gpu)  # each node itself alone
    clean = tree_attention(q, kc, vc, table, ctx, cu, mask)
    for c in (kc, vc):
        c.reshape(-1, 128)[50 + n - 1] = bad
    got = tree_attention(q, kc, vc, table, ctx, cu, mask)
    assert torch.equal(got[:-1], clean[:-1])
    assert not torch.isfinite(got[-1]).all()


@pytest.mark.parametrize("qscale", [0.0, 8.0, 40.0])
def test_tree_score_ranges(gpu, qscale):
    _tree(gpu, "bf16", [500, 20], [4, 3], 8, 2, 128, 16, mask="tree", seed=6, qscale=qscale)


def test_tree_long_and_short_requests_together(gpu):
    _tree(gpu, "bf16", [9000] + [30] * 20, [2] + [1] * 20, 8, 1, 128, 64, seed=4)


def test_tree_many_requests(gpu):
    rng = np.random.default_rng(3)
    ctx = rng.integers(0, 60, 300).tolist()
    _tree(gpu, "fp16", ctx, rng.integers(0, 3, 300).tolist(), 4, 4, 64, 16, seed=4)


def test_tree_table_entries_outside_the_cache_read_as_zeros(gpu):
    g = torch.Generator().manual_seed(8)
    kc, vc = _cache(g, 4, 16, 1, 64, "fp16", gpu)
    q = torch.randn(1, 1, 64, generator=g).to(DT["fp16"]).to(gpu)
    ctx = torch.tensor([40], dtype=torch.int32, device=gpu)
    cu = torch.tensor([0, 1], dtype=torch.int32, device=gpu)
    want_k, want_v = kc.clone(), vc.clone()
    want_k[1], want_v[1] = 0, 0
    good = torch.tensor([[0, 1, 2]], dtype=torch.int32, device=gpu)
    want = tree_attention(q, want_k, want_v, good, ctx, cu)
    for bad in (-1, 4, 2**31 - 1, -2**31):
        table = good.clone()
        table[0, 1] = bad
        assert torch.equal(tree_attention(q, kc, vc, table, ctx, cu), want)


def test_tree_keys_behind_the_table_are_left_out(gpu):
    g = torch.Generator().manual_seed(8)
    kc, vc = _cache(g, 4, 16, 1, 64, "fp16", gpu)
    q = torch.randn(1, 1, 64, generator=g).to(DT["fp16"]).to(gpu)
    cu = torch.tensor([0, 1], dtype=torch.int32, device=gpu)
    table = torch.tensor([[2, 0]], dtype=torch.int32, device=gpu)
    a = tree_attention(q, kc, vc, table, torch.tensor([31], dtype=torch.int32, device=gpu), cu)
    for ctx in (32, 500, 2**31 - 1):
        assert torch.equal(tree_attention(q, kc, vc, table, torch.tensor([ctx], dtype=torch.int32, device=gpu), cu), a)
    one = tree_attention(q, kc, vc, table, torch.tensor([-9], dtype=torch.int32, device=gpu), cu)
    assert torch.equal(one, vc[2, 0][None])


# --- together -----------------------------------------------------------------------

def test_prompts_then_decoding_then_a_draft(gpu):
    """Slots, rows into the cache and attention as a serving loop runs them: the
    prompts, then steps of one token, then a drafted chain, each against the
    attention over the whole sequence at once."""
    torch.manual_seed(0)
    HQ, HK, D, size = 8, 2, 128, 16
    prompt, steps, draft = [33, 1, 160], 3, 4
    final = [p + steps + draft for p in prompt]
    B = len(prompt)
    q, k, v = ([torch.randn(n, h, D, device=gpu).bfloat16() for n in final] for h in (HQ, HK, HK))
    kc, vc = (torch.full((64, size, HK, D), float("nan"), device=gpu, dtype=torch.bfloat16) for _ in range(2))
    free = torch.randperm(64, device=gpu).int()
    table = torch.full((B, 16), -1, dtype=torch.int32, device=gpu)
    start = torch.zeros(1, dtype=torch.int32, device=gpu)
    lengths = torch.zeros(B, dtype=torch.int32, device=gpu)
    got = [[] for _ in range(B)]
    done = [0] * B
    for counts in [prompt] + [[1] * B] * steps + [[draft] * B]:
        c = torch.tensor(counts, dtype=torch.int32, device=gpu)
        r = assign_slots(lengths, c, table, free, size, sum(counts), free_start=start)
        qs, ks, vs = (torch.cat([x[b][done[b]:done[b] + counts[b]] for b in range(B)]) for x in (q, k, v))
        write_cache(ks, vs, kc, vc, r.slots)
        if done[0] == 0:
            o = varlen_attention(qs, ks, vs, r.cu_seqlens)
        else:
            o = tree_attention(qs, kc, vc, table, lengths, r.cu_seqlens)
        for b, part in enumerate(torch.split(o, counts)):
            got[b].append(part)
        start += r.taken
        lengths += c
        done = [a + n for a, n in zip(done, counts)]
    assert int(start) == sum(-(-n // size) for n in final)
    for b in range(B):
        n = final[b]
        lse = torch.empty(HQ, n, device=gpu)
        ref = R.packed_attention(_np(q[b]), _np(k[b]), _np(v[b]), [0, n], [0, n], lambda _: R.causal_reads(n, n), D**-0.5)
        varlen_attention(q[b], k[b], v[b], torch.tensor([0, n], dtype=torch.int32, device=gpu), lse=lse)
        _check(torch.cat(got[b]), lse, *ref, "bf16", n, D, 6.0, n)


def test_a_step_captured_into_a_graph(gpu):
    """One decoding step replayed with new lengths: the eager results each time."""
    torch.manual_seed(1)
    B, HQ, HK, D, size = 5, 8, 2, 64, 16
    kc, vc = (torch.randn(40, size, HK, D, device=gpu).half() for _ in range(2))
    free = torch.randperm(40, device=gpu).int()
    table = torch.full((B, 8), -1, dtype=torch.int32, device=gpu)
    lengths = torch.zeros(B, dtype=torch.int32, device=gpu)
    start = torch.zeros(1, dtype=torch.int32, device=gpu)
    counts = torch.ones(B, dtype=torch.int32, device=gpu)
    qkv = torch.randn(B + 3, HQ + 2 * HK, D, device=gpu).half()
    q, k, v = qkv[:, :HQ], qkv[:, HQ:HQ + HK], qkv[:, HQ + HK:]
    o = torch.zeros(B + 3, HQ, D, device=gpu, dtype=torch.half)

    def step():
        r = assign_slots(lengths, counts, table, free, size, B + 3, free_start=start)
        write_cache(k, v, kc, vc, r.slots)
        tree_attention(q, kc, vc, table, lengths, r.cu_seqlens, o=o)
        p = varlen_attention(q, k, v, r.cu_seqlens)
        return r, p

    r, _ = step()
    start += r.taken
    lengths += counts
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        rg, pg = step()
    for _ in range(40):
        qkv.copy_(torch.randn_like(qkv))
        o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        want = (o.clone(), pg[:B].clone(), rg.slots.clone(), kc.clone(), table.clone())
        o.zero_()
        re, pe = step()
        for a, b in zip(want, (o, pe[:B], re.slots, kc, table)):
            assert torch.equal(a, b)
        start += re.taken
        lengths += counts


def test_two_streams_at_once(gpu):
    torch.manual_seed(2)
    kc, vc = (torch.randn(600, 16, 2, 128, device=gpu).bfloat16() for _ in range(2))
    table = torch.randperm(600, device=gpu).int().reshape(2, 300).contiguous()
    lengths = torch.tensor([4700, 900], dtype=torch.int32, device=gpu)
    cu = torch.tensor([0, 1, 6], dtype=torch.int32, device=gpu)
    qs = [torch.randn(6, 16, 128, device=gpu).bfloat16() for _ in range(8)]
    want = [tree_attention(q, kc, vc, table, lengths, cu) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = [None] * 8
    torch.cuda.synchronize()
    for n, q in enumerate(qs):
        with torch.cuda.stream(streams[n % 4]):
            got[n] = tree_attention(q, kc, vc, table, lengths, cu)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
