"""The forms that the packed and the paged attention choose between by size
(few queries or the pipeline; blocks of 32, 64 or 256 query rows), each at the
lengths where its tiles, blocks and parts end, against plain attention in 64
bits on the GPU; large offsets, long contexts and values that no row reads.
Tolerances from the arithmetic (serving_ref.tolerances)."""

import random

import pytest
import torch

from gfx950_gluon_tutorials_amd.attention import tree_attention, varlen_attention
from oracle import serving_ref as R

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
SUBNORMAL = {"fp16": 2.0**-25, "bf16": 0.0}
SHORT_ROWS = 48 * 1024  # queries by heads up to which the short form runs


def _i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _cu(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _check(o, lse, q, k, v, reads, scale, dtype):
    """One sequence: o, q (Lq, HQ, D), lse (HQ, Lq), k and v (Lk, HK, D), reads (Lq, Lk).  Heads by 8."""
    HQ, D = q.shape[1:]
    group = HQ // k.shape[1]
    eps = torch.finfo(DT[dtype]).eps
    for h0 in range(0, HQ, 8):
        h = list(range(h0, min(HQ, h0 + 8)))
        g = [x // group for x in h]
        qq, kk, vv = (x.double().transpose(0, 1).contiguous() for x in (q[:, h], k[:, g], v[:, g]))
        s = torch.matmul(qq, kk.transpose(1, 2).contiguous()) * scale
        s = s.masked_fill(~reads, float("-inf"))
        top = s.amax(-1, keepdim=True) if s.shape[-1] else s.new_full(s.shape[:-1] + (1,), float("-inf"))
        none = torch.isneginf(top)
        w = torch.exp(s - torch.where(none, 0.0, top))
        z = w.sum(-1, keepdim=True)
        p = w / torch.where(z == 0, 1.0, z)
        ref = torch.matmul(p, vv)
        mag = torch.matmul(p, vv.abs())
        lref = torch.where(none, float("-inf"), top + z.log())[..., 0]
        spread = float(torch.matmul(qq.abs(), kk.abs().transpose(1, 2).contiguous()).max()) * scale if kk.shape[1] else 0.0
        vmax = float(vv.abs().max()) if kk.shape[1] else 0.0
        to, tl = R.tolerances(ref.cpu().numpy(), torch.where(torch.isneginf(lref), 0.0, lref).cpu().numpy(),
                              mag.cpu().numpy(), spread, eps, max(1, kk.shape[1]), D, vmax, SUBNORMAL[dtype])
        got, lgot = o[:, h].double().transpose(0, 1), lse[h].double()
        assert torch.isfinite(got).all()
        off = (got - ref).abs().cpu().numpy() - to
        assert (off <= 0).all(), f"heads {h[0]}..: o is {off.max():.3g} past its bound"
        assert torch.equal(torch.isneginf(lgot), torch.isneginf(lref))
        off = (torch.where(torch.isneginf(lref), 0.0, lgot) - torch.where(torch.isneginf(lref), 0.0, lref)).abs().cpu().numpy() - tl
        assert (off <= 0).all(), f"heads {h[0]}..: lse is {off.max():.3g} past its bound"


def _causal(lq, lk, causal, dev):
    i, j = torch.arange(lq, device=dev)[:, None], torch.arange(lk, device=dev)[None]
    return j <= i + lk - lq if causal else torch.ones(lq, lk, dtype=torch.bool, device=dev)


def _prompt(dev, dtype, lq, lk, HQ, HK, D, causal, seed, short):
    T, TK = sum(lq), sum(lk)
    assert (T * HQ <= SHORT_ROWS) == short
    gen = torch.Generator(device=dev).manual_seed(seed)
    q = torch.randn(T + 2, HQ, D, generator=gen, device=dev).to(DT[dtype])
    k, v = (torch.randn(TK + 2, HK, D, generator=gen, device=dev).to(DT[dtype]) for _ in range(2))
    o, lse = torch.full_like(q, 7.0), torch.full((HQ, T + 2), 7.0, device=dev)
    cq, ck = _cu(lq), _cu(lk)
    scale = D**-0.5
    varlen_attention(q, k, v, _i32(cq, dev), o, cu_seqlens_k=_i32(ck, dev), causal=causal, lse=lse)
    assert (o[T:] == 7).all() and (lse[:, T:] == 7).all()
    for b in range(len(lq)):
        r, c = slice(cq[b], cq[b + 1]), slice(ck[b], ck[b + 1])
        if lq[b]:
            _check(o[r], lse[:, r], q[r], k[c], v[c], _causal(lq[b], lk[b], causal, dev), scale, dtype)


PIPELINE = [
    ([255, 256, 257, 2], None), ([1100], None), ([513, 5, 300], None), ([0, 900, 0, 31, 1], None), ([64] * 13, None),
    ([300, 500, 70], [900, 500, 75]), ([400, 300, 200], [130, 0, 64]), ([129] * 7, [1, 127, 128, 129, 383, 384, 385]),
]


@pytest.mark.parametrize("lq,lk", PIPELINE, ids=lambda x: "_".join(map(str, x)) if x else "same")
@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("fp16", 128), ("bf16", 64), ("fp16", 64)])
@pytest.mark.parametrize("causal", [True, False])
def test_pipeline_lengths(gpu, lq, lk, dtype, D, causal):
    _prompt(gpu, dtype, lq, lk or lq, 64, 8, D, causal, seed=sum(lq), short=False)


@pytest.mark.parametrize("lq,lk", PIPELINE[:6], ids=lambda x: "_".join(map(str, x)) if x else "same")
@pytest.mark.parametrize("HQ,HK,D", [(16, 4, 128), (15, 3, 64)])
def test_short_form_lengths(gpu, lq, lk, HQ, HK, D):
    _prompt(gpu, "bf16", lq, lk or lq, HQ, HK, D, True, seed=sum(lq), short=True)


@pytest.mark.parametrize("B", [64, 65, 129, 600])
def test_pipeline_batches_around_a_wave(gpu, B):
    lq = [(7 * b) % 23 for b in range(B)]
    lq[B // 2], lq[B // 3] = 700, 300
    _prompt(gpu, "bf16", lq, lq, 64, 64, 64, True, seed=B, short=False)


@pytest.mark.parametrize("HQ,HK", [(60, 5), (64, 1), (63, 9), (64, 16)])
def test_pipeline_heads(gpu, HQ, HK):
    _prompt(gpu, "fp16", [500, 400], [500, 400], HQ, HK, 128, True, seed=HQ, short=False)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("HQ", [4, 64])
def test_values_that_no_row_reads(gpu, bad, D, HQ):
    """NaN or infinities behind the sequences and in keys that only the last
    queries read: the others' bits stay."""
    gen = torch.Generator(device=gpu).manual_seed(2)
    q, k, v = (torch.randn(1000, h, D, generator=gen, device=gpu).bfloat16() for h in (HQ, 2, 2))
    cu = _i32([0, 500, 900], gpu)
    clean = varlen_attention(q, k, v, cu)
    for t in (k, v):
        t[470] = bad
        t[899, 1] = bad
        t[900:] = bad
    q[900:] = bad
    got = varlen_attention(q, k, v, cu)
    assert torch.equal(got[:470], clean[:470]) and torch.equal(got[500:899], clean[500:899])
    assert torch.equal(got[899, :HQ // 2], clean[899, :HQ // 2])
    assert not torch.isfinite(got[470:500]).all(-1).any()
    assert not torch.isfinite(got[899, HQ // 2:]).all(-1).any()


@pytest.mark.parametrize("HQ", [8, 64])
def test_rows_past_32_bit_offsets(gpu, HQ):
    """Sequences at the end of a fused projection of more than 4 GiB."""
    T, HK, D = 420_000 if HQ == 8 else 240_000, 16 if HQ == 8 else 8, 128
    L = 900
    HK = min(HK, HQ)
    big = torch.zeros(T, HQ + 2 * HK if HQ == 64 else 48, D, dtype=torch.bfloat16, device=gpu)
    assert big.numel() * 2 > 2**32
    gen = torch.Generator(device=gpu).manual_seed(5)
    big[-L:] = torch.randn(L, big.shape[1], D, generator=gen, device=gpu).bfloat16()
    q, k, v = big[:, :HQ], big[:, HQ:HQ + HK], big[:, HQ + HK:HQ + 2 * HK]
    cu = _i32([T - L, T - 300, T], gpu)
    o = torch.empty(T, HQ, D, dtype=torch.bfloat16, device=gpu)
    varlen_attention(q, k, v, cu, o)
    want = varlen_attention(q[-L:].contiguous(), k[-L:].contiguous(), v[-L:].contiguous(), _i32([0, L - 300, L], gpu))
    if (T * HQ <= SHORT_ROWS) == (L * HQ <= SHORT_ROWS):
        assert torch.equal(o[-L:], want)
    else:
        assert torch.allclose(o[-L:].float(), want.float(), rtol=2.0**-7, atol=2.0**-7)
    del big, q, k, v, o
    torch.cuda.empty_cache()


# --- over the cache ---------------------------------------------------------------

def _tree(dev, dtype, ctx, nodes, HQ, HK, D, size, mask, seed, order="bshd", heads=None):
    gen = torch.Generator(device=dev).manual_seed(seed)
    rng = random.Random(seed)
    total = [c + n for c, n in zip(ctx, nodes)]
    used = [-(-t // size) for t in total]
    blocks = sum(used) + 2
    ids = torch.randperm(blocks, generator=gen, device=dev).int()
    table = torch.full((len(ctx), max(1, max(used))), -7, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = ids[at:at + n]
        at += n
    shape = (blocks, size, HK, D) if order == "bshd" else (blocks, HK, size, D)
    kc, vc = (torch.randn(shape, generator=gen, device=dev).to(DT[dtype]) for _ in range(2))
    if order == "bhsd":
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    T = sum(nodes)
    q = torch.randn(T, HQ, D, generator=gen, device=dev).to(DT[dtype])
    cu = _cu(nodes)
    sees, words = [], max(1, -(-max(nodes) // 64))
    for n in nodes:
        m = torch.zeros(n, n, dtype=torch.bool)
        for i in range(n):
            p = i - 1 if mask == "chain" else rng.randint(max(-1, i - 5), i - 1)
            if p >= 0:
                m[i] = m[p]
            m[i, i] = True
        sees.append(m)
    bits = None
    if mask == "tree":
        rows = []
        for m in sees:
            for i in range(len(m)):
                x = sum(1 << j for j in torch.nonzero(m[i]).flatten().tolist())
                w = [(x >> 64 * k) & (2**64 - 1) for k in range(words)]
                rows.append([y - 2**64 if y >> 63 else y for y in w])
        bits = torch.tensor(rows, dtype=torch.int64, device=dev)
    lse = torch.empty(HQ, T, device=dev)
    o = tree_attention(q, kc, vc, table, _i32(ctx, dev), _i32(cu, dev), bits, lse=lse)
    for b in range(len(ctx)):
        if not nodes[b]:
            continue
        pos = torch.arange(total[b], device=dev)
        page = table[b][pos // size].long()
        h = list(range(HQ)) if heads is None else heads
        g = sorted({x * HK // HQ for x in h})
        assert heads is None or len(g) == 1
        k, v = (c[page, pos % size][:, g] for c in (kc, vc))
        reads = torch.ones(nodes[b], total[b], dtype=torch.bool, device=dev)
        reads[:, ctx[b]:] = sees[b].to(dev)
        r = slice(cu[b], cu[b + 1])
        _check(o[r][:, h], lse[h][:, r], q[r][:, h], k, v, reads, D**-0.5, dtype)


@pytest.mark.parametrize("rows", [32, 33, 64, 65, 128, 129, 256, 257, 300])
@pytest.mark.parametrize("D,dtype,size,order", [(128, "bf16", 16, "bshd"), (64, "fp16", 64, "bhsd")])
@pytest.mark.parametrize("mask", ["chain", "tree"])
def test_blocks_of_rows(gpu, rows, D, dtype, size, order, mask):
    """One query head a K/V head, so that a request's nodes are its rows."""
    _tree(gpu, dtype, [200, 1000, 0, 63], [rows, rows, rows, rows], 3, 3, D, size, mask, seed=rows, order=order)


@pytest.mark.parametrize("nodes", [[1] * 20 + [130], [200, 1, 0, 3], [40] * 5 + [1] * 30, [150, 150, 1, 0, 149]])
@pytest.mark.parametrize("D", [64, 128])
def test_uneven_batches(gpu, nodes, D):
    ctx = [(37 * b * b) % 1500 for b in range(len(nodes))]
    _tree(gpu, "bf16", ctx, nodes, 8, 2, D, 32, "tree", seed=len(nodes))


@pytest.mark.parametrize("D,nodes", [(128, 3), (128, 40), (64, 3), (64, 20), (64, 100)])
def test_a_long_request_among_short_ones(gpu, D, nodes):
    _tree(gpu, "bf16", [20000] + [50] * 9, [nodes] * 10, 8, 2, D, 64, "chain", seed=nodes)


@pytest.mark.parametrize("D,nodes,B", [(128, 24, 300), (64, 70, 200), (64, 20, 300), (128, 5, 400)])
def test_many_short_requests_among_long_ones(gpu, D, nodes, B):
    """Parts of many blocks, of one, and of a piece of one."""
    ctx = [0, 1, 63, 90, 40] * (B // 5)
    ctx[B // 3], ctx[-1] = 9000, 4000
    _tree(gpu, "fp16", ctx, [nodes] * B, 4, 2, D, 16, "chain", seed=B)


@pytest.mark.parametrize("ctx", [0, 1, 50, 130, 800])
@pytest.mark.parametrize("D,HK", [(128, 1), (64, 3)])
def test_fewer_tiles_than_workers(gpu, ctx, D, HK):
    _tree(gpu, "bf16", [ctx], [140], HK, HK, D, 16, "tree", seed=ctx)


@pytest.mark.parametrize("D,nodes", [(128, 1), (128, 24), (64, 20), (64, 80)])
def test_long_contexts(gpu, D, nodes):
    """More than 64 tiles for every part: parts that cross heads, pages asked for
    again."""
    _tree(gpu, "bf16", [150_000], [nodes], 32, 16, D, 16, "chain", seed=D + nodes, heads=[0, 1])
    torch.cuda.empty_cache()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [10, 60, 150])
def test_nodes_that_a_row_does_not_read(gpu, bad, D, n):
    gen = torch.Generator(device=gpu).manual_seed(8)
    kc, vc = (torch.randn(60, 16, 2, D, generator=gen, device=gpu).bfloat16() for _ in range(2))
    q = torch.randn(n, 4, D, generator=gen, device=gpu).bfloat16()
    table = torch.randperm(60, generator=gen, device=gpu).int()[None]
    ctx, cu = _i32([700], gpu), _i32([0, n], gpu)
    words = -(-n // 64)
    rows = [[0] * words for _ in range(n)]
    for i in range(n):
        rows[i][i // 64] = 1 << (i % 64) if i % 64 < 63 else -(1 << 63)
    mask = torch.tensor(rows, dtype=torch.int64, device=gpu)
    clean = tree_attention(q, kc, vc, table, ctx, cu, mask)
    at = 700 + n // 2
    blk = int(table[0, at // 16])
    for c in (kc, vc):
        c[blk, at % 16] = bad
    got = tree_attention(q, kc, vc, table, ctx, cu, mask)
    keep = [i for i in range(n) if i != n // 2]
    assert torch.equal(got[keep], clean[keep])
    assert not torch.isfinite(got[n // 2]).all()


@pytest.mark.parametrize("seed", range(12))
def test_drawn_batches(gpu, seed):
    rng = random.Random(seed)
    B = rng.choice([1, 2, 7, 40])
    HK = rng.choice([1, 2, 5])
    HQ = HK * rng.choice([1, 3, 8])
    D, dtype = rng.choice([64, 128]), rng.choice(["fp16", "bf16"])
    ctx = [rng.choice([0, 1, rng.randint(0, 100), rng.randint(0, 3000)]) for _ in range(B)]
    nodes = [rng.choice([0, 1, 1, rng.randint(1, 70)]) for _ in range(B)]
    nodes[0] = max(nodes[0], 1)
    _tree(gpu, dtype, ctx, nodes, HQ, HK, D, rng.choice([16, 128, 1024]), rng.choice(["chain", "tree"]), seed,
          order=rng.choice(["bshd", "bhsd"]))


# --- the inputs that would be lost -------------------------------------------------

def test_lazily_negated_views_are_refused(gpu):
    q = torch.randn(4, 1, 64, device=gpu).half()
    cu = _i32([0, 4], gpu)
    varlen_attention(q, q, q, cu)
    with pytest.raises(ValueError, match="negated"):
        varlen_attention(torch._neg_view(q), q, q, cu)


def test_a_scale_tensor_is_taken_by_value(gpu):
    q = torch.randn(4, 1, 64, device=gpu).half()
    cu = _i32([0, 4], gpu)
    s = torch.tensor(0.5)
    a = varlen_attention(q, q, q, cu, sm_scale=s)
    s.fill_(0.01)
    b = varlen_attention(q, q, q, cu, sm_scale=s)
    assert torch.equal(a, varlen_attention(q, q, q, cu, sm_scale=0.5))
    assert torch.equal(b, varlen_attention(q, q, q, cu, sm_scale=float(s))) and not torch.equal(a, b)


def test_a_causal_flag_tensor_is_taken_by_value(gpu):
    q = torch.randn(4, 1, 64, device=gpu).half()
    cu = _i32([0, 4], gpu)
    flag = torch.tensor(True)
    a = varlen_attention(q, q, q, cu, causal=flag)
    flag.fill_(False)
    b = varlen_attention(q, q, q, cu, causal=flag)
    assert torch.equal(a, varlen_attention(q, q, q, cu, causal=True))
    assert torch.equal(b, varlen_attention(q, q, q, cu, causal=False)) and not torch.equal(a, b)


def test_a_negated_or_differentiable_lse_is_refused(gpu):
    q = torch.randn(1, 1, 64, device=gpu).half()
    cu = _i32([0, 1], gpu)
    lse = torch.zeros(1, 1, device=gpu)
    varlen_attention(q, q, q, cu, lse=lse)
    for bad in (torch._neg_view(lse), torch.zeros(1, 1, device=gpu, requires_grad=True)):
        with pytest.raises(ValueError):
            varlen_attention(q, q, q, cu, lse=bad)


def test_a_batch_of_too_many_requests_is_refused(gpu):
    B = 8193
    q = torch.zeros(1, 1, 64, device=gpu, dtype=torch.half)
    kc = torch.zeros(1, 16, 1, 64, device=gpu, dtype=torch.half)
    z = torch.zeros(B, dtype=torch.int32, device=gpu)
    with pytest.raises(ValueError):
        tree_attention(q, kc, kc, z[:, None], z, torch.zeros(B + 1, dtype=torch.int32, device=gpu))
