"""The packed attention on queries, keys and values whose rows are closer than
they are long: one row for all tokens (stride 0), rows that overlap, and a single
row of any stride.  The same values in rows of their own give the same bits."""

import numpy as np
import pytest
import torch

from gfx950_gluon_tutorials_amd.attention import varlen_attention
from oracle import serving_ref as R

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
SUBNORMAL = {"fp16": 2.0**-25, "bf16": 0.0}
SHORT_ROWS = 48 * 1024  # queries by heads up to which the short form runs


def _rows(gen, T, H, D, step, dtype, dev):
    """(T, H, D) with `step` elements between tokens, heads apart."""
    span = step * (T - 1) + D
    base = torch.randn(H, span, generator=gen).to(DT[dtype]).to(dev)
    return base.as_strided((T, H, D), (step, span, 1))


def _steps(D):
    return [0, 8, D // 2, D - 8]


def _call(q, k, v, lq, lk, causal):
    cq, ck = (torch.tensor(np.concatenate([[0], np.cumsum(x)]), dtype=torch.int32, device=q.device) for x in (lq, lk))
    lse = torch.empty(q.shape[1], q.shape[0], device=q.device)
    return varlen_attention(q, k, v, cq, cu_seqlens_k=ck, causal=causal, lse=lse), lse


# Span of a head is a multiple of 8 elements for every step above.
@pytest.mark.parametrize("which", ["q", "k", "v", "qkv"])
@pytest.mark.parametrize("D,dtype,causal", [(64, "fp16", True), (64, "bf16", False), (128, "bf16", True), (128, "fp16", False)])
@pytest.mark.parametrize("HQ", [4, 64])
def test_rows_closer_than_they_are_long(gpu, which, D, dtype, causal, HQ):
    lq, lk = [300, 1, 0, 513, 70], [300, 33, 5, 600, 64]
    T, TK, HK = sum(lq), sum(lk), 2
    assert (T * HQ <= SHORT_ROWS) == (HQ == 4)
    for step in _steps(D):
        gen = torch.Generator().manual_seed(step)
        q = _rows(gen, T, HQ, D, step if "q" in which else D, dtype, gpu)
        k = _rows(gen, TK, HK, D, step if "k" in which else D, dtype, gpu)
        v = _rows(gen, TK, HK, D, step if "v" in which else D, dtype, gpu)
        got, lse = _call(q, k, v, lq, lk, causal)
        want, wlse = _call(q.contiguous(), k.contiguous(), v.contiguous(), lq, lk, causal)
        assert torch.equal(got, want), f"step {step}"
        assert torch.equal(lse, wlse), f"step {step}"


@pytest.mark.parametrize("D,dtype", [(64, "fp16"), (128, "bf16")])
@pytest.mark.parametrize("HQ", [2, 400])
def test_expanded_tensors_against_the_oracle(gpu, D, dtype, HQ):
    lens, HK = [70, 129], 1
    T = sum(lens)
    assert (T * HQ <= SHORT_ROWS) == (HQ == 2)
    gen = torch.Generator().manual_seed(D)
    q = torch.randn(T, HQ, D, generator=gen).to(DT[dtype]).to(gpu)
    k, v = (torch.randn(1, HK, D, generator=gen).to(DT[dtype]).to(gpu).expand(T, HK, D) for _ in range(2))
    o, lse = _call(q, k, v, lens, lens, True)
    qn, kn, vn, on = (t.float().cpu().numpy() for t in (q[:, :2], k, v, o[:, :2]))
    cu = [0, lens[0], T]
    ref, lref, mag, spread = R.packed_attention(qn, kn, vn, cu, cu, lambda b: R.causal_reads(lens[b], lens[b]), D**-0.5)
    to, tl = R.tolerances(ref, lref, mag, spread, torch.finfo(DT[dtype]).eps, max(lens), D, float(np.abs(vn).max()),
                          SUBNORMAL[dtype])
    assert (np.abs(on - ref) <= to).all() and (np.abs(lse[:2].cpu().numpy() - lref) <= tl).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("step", [0, 3, 8, 4096])
def test_a_single_row_of_any_stride(gpu, D, step):
    gen = torch.Generator().manual_seed(D)
    q, k, v = (torch.randn(1, 2, D, generator=gen).half().to(gpu) for _ in range(3))
    got, lse = _call(*(t.as_strided((1, 2, D), (step, D, 1)) for t in (q, k, v)), [1], [1], True)
    want, wlse = _call(q, k, v, [1], [1], True)
    assert torch.equal(got, v) and torch.equal(want, v) and torch.equal(lse, wlse)
    q64 = torch.randn(1, 50_000, D, generator=gen).half().to(gpu)  # one row of many heads: the pipeline
    got, lse = _call(q64.as_strided(q64.shape, (step, D, 1)), *(t.as_strided((1, 2, D), (step, D, 1)) for t in (k, v)),
                     [1], [1], True)
    assert torch.equal(got, v.repeat_interleave(25_000, 1))


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("HQ", [4, 64])
def test_overlapping_rows_behind_a_sequence_stay_out(gpu, bad, D, HQ):
    """The first row behind a sequence shares its first half with the sequence's last
    one; its other half, and all that follows, is not finite."""
    L, T = 850, 900
    gen = torch.Generator().manual_seed(7)
    q = torch.randn(T, HQ, D, generator=gen).bfloat16().to(gpu)
    k, v = (_rows(gen, T, 1, D, D // 2, "bf16", gpu) for _ in range(2))
    cu = torch.tensor([0, L], dtype=torch.int32, device=gpu)
    clean = varlen_attention(q, k, v, cu)[:L]
    for t in (k, v):
        t[L:, :, D // 2:] = bad
    assert torch.isfinite(k[:L]).all() and torch.isfinite(v[:L]).all()
    assert torch.equal(varlen_attention(q, k, v, cu)[:L], clean)
