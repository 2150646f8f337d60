"""CPU checks of the packed and paged attention entry points: what the Python
functions and the C entries refuse (before anything reaches a GPU), what they
pass on, and the oracle against plain torch."""

import ctypes
import re
import os

import numpy as np
import pytest
import torch

from gfx950_gluon_tutorials_amd import _lib
from gfx950_gluon_tutorials_amd.attention import _launch, assign_slots, paged, tree_attention, varlen_attention, write_cache
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


def _prompt(**kw):
    a = dict(q=torch.zeros(6, 4, 64).bfloat16(), k=torch.zeros(6, 2, 64).bfloat16(), v=torch.zeros(6, 2, 64).bfloat16(),
             cu_seqlens=_i32(0, 6))
    a.update(kw)
    return varlen_attention(**a)


def _tree(**kw):
    a = dict(q=torch.zeros(6, 4, 64).bfloat16(), k_cache=torch.zeros(3, 16, 2, 64).bfloat16(),
             v_cache=torch.zeros(3, 16, 2, 64).bfloat16(), block_table=torch.zeros(2, 2, dtype=torch.int32),
             lengths=_i32(3, 4), cu_seqlens=_i32(0, 2, 6))
    a.update(kw)
    return tree_attention(**a)


def _write(**kw):
    a = dict(k=torch.zeros(6, 2, 64).half(), v=torch.zeros(6, 2, 64).half(), k_cache=torch.zeros(3, 16, 2, 64).half(),
             v_cache=torch.zeros(3, 16, 2, 64).half(), slots=torch.arange(6))
    a.update(kw)
    return write_cache(**a)


def _assign(**kw):
    a = dict(lengths=_i32(3, 4), counts=_i32(1, 1), block_table=torch.zeros(2, 2, dtype=torch.int32),
             free_blocks=_i32(5, 6), block_size=16, num_tokens=2)
    a.update(kw)
    return assign_slots(**a)


def test_good_calls_reach_their_entries(calls):
    assert _prompt().shape == (6, 4, 64)
    _prompt(cu_seqlens_k=_i32(0, 4), k=torch.zeros(4, 2, 64).bfloat16(), v=torch.zeros(4, 2, 64).bfloat16())
    assert _tree().shape == (6, 4, 64)
    _tree(tree_mask=torch.zeros(6, dtype=torch.int64))
    _tree(tree_mask=torch.zeros(6, 2, dtype=torch.int64), lse=torch.zeros(4, 6))
    _write()
    r = _assign()
    assert r.cu_seqlens.shape == (3,) and r.slots.shape == r.positions.shape == (2,) and r.taken.shape == (1,)
    assert [c[0] for c in calls] == ["g9_varlen_fwd"] * 2 + ["g9_tree_fwd"] * 3 + ["g9_write_cache", "g9_assign_slots"]


@pytest.mark.parametrize("kw", [
    dict(q=torch.zeros(6, 3, 64).bfloat16()),                        # heads that do not divide
    dict(q=torch.zeros(6, 4, 32).bfloat16(), k=torch.zeros(6, 2, 32).bfloat16(), v=torch.zeros(6, 2, 32).bfloat16()),
    dict(q=torch.zeros(6, 4, 64).half()),                            # mixed types
    dict(q=torch.zeros(6, 4, 64), k=torch.zeros(6, 2, 64), v=torch.zeros(6, 2, 64)),
    dict(v=torch.zeros(5, 2, 64).bfloat16()),
    dict(k=torch.zeros(5, 2, 64).bfloat16(), v=torch.zeros(5, 2, 64).bfloat16()),  # other lengths, no cu_seqlens_k
    dict(q=torch.zeros(6, 4, 128).bfloat16()[:, :, ::2]),            # head-dim stride
    dict(q=torch.zeros(24, 64).bfloat16()),
    dict(cu_seqlens=torch.tensor([0, 6])),                           # int64
    dict(cu_seqlens=torch.zeros(0, dtype=torch.int32)),
    dict(cu_seqlens=_i32(0, 1, 6, 9)[::2]),
    dict(cu_seqlens_k=_i32(0, 3, 6)),
    dict(o=torch.zeros(6, 4, 64).half()),
    dict(o=torch.zeros(5, 4, 64).bfloat16()),
    dict(lse=torch.zeros(6, 4)),
    dict(lse=torch.zeros(4, 6).bfloat16()),
    dict(lse=torch.zeros(4, 12)[:, ::2]),
    dict(q=torch.zeros(6, 4, 64).bfloat16().requires_grad_()),
    dict(v=torch.zeros(6, 2, 64).bfloat16().requires_grad_()),
])
def test_prompt_refusals(calls, kw):
    with pytest.raises(ValueError):
        _prompt(**kw)
    assert not calls


@pytest.mark.parametrize("kw", [
    dict(q=torch.zeros(6, 3, 64).bfloat16()),
    dict(q=torch.zeros(6, 4, 128).bfloat16()),
    dict(k_cache=torch.zeros(3, 16, 2, 64).half()),
    dict(v_cache=torch.zeros(2, 16, 2, 64).bfloat16()),
    dict(k_cache=torch.zeros(3, 16, 128).bfloat16(), v_cache=torch.zeros(3, 16, 128).bfloat16()),
    dict(k_cache=torch.zeros(3, 16, 2, 128).bfloat16()[..., ::2]),
    dict(block_table=torch.zeros(2, 2)),
    dict(block_table=torch.zeros(3, 2, dtype=torch.int32)),
    dict(block_table=torch.zeros(2, 4, dtype=torch.int32)[:, ::2]),
    dict(block_table=torch.zeros(4, dtype=torch.int32)),
    dict(lengths=torch.tensor([3, 4])),
    dict(lengths=_i32(3)),
    dict(cu_seqlens=_i32(0, 6)),
    dict(tree_mask=torch.zeros(6, dtype=torch.int32)),
    dict(tree_mask=torch.zeros(5, dtype=torch.int64)),
    dict(tree_mask=torch.zeros(6, 0, dtype=torch.int64)),
    dict(tree_mask=torch.zeros(6, 4, dtype=torch.int64)[:, ::2]),
    dict(tree_mask=torch.zeros(6, 6, dtype=torch.bool)),
    dict(lse=torch.zeros(6, 4)),
    dict(o=torch.zeros(6, 4, 64)),
    dict(q=torch.zeros(6, 4, 64).bfloat16().requires_grad_()),
])
def test_tree_refusals(calls, kw):
    with pytest.raises(ValueError):
        _tree(**kw)
    assert not calls


@pytest.mark.parametrize("kw", [
    dict(k=torch.zeros(5, 2, 64).half()),
    dict(k=torch.zeros(6, 3, 64).half(), v=torch.zeros(6, 3, 64).half()),
    dict(k=torch.zeros(6, 2, 64).bfloat16(), v=torch.zeros(6, 2, 64).bfloat16()),
    dict(slots=torch.arange(5)),
    dict(slots=torch.arange(6).int()),
    dict(slots=torch.arange(12)[::2]),
    dict(v_cache=torch.zeros(3, 16, 2, 128).half()[..., ::2]),
    dict(k=torch.zeros(6, 2, 64).half().requires_grad_()),
])
def test_write_refusals(calls, kw):
    with pytest.raises(ValueError):
        _write(**kw)
    assert not calls


@pytest.mark.parametrize("kw", [
    dict(counts=_i32(1)),
    dict(lengths=torch.tensor([3, 4])),
    dict(free_blocks=torch.tensor([3, 4])),
    dict(free_blocks=_i32(1, 2, 3, 4)[::2]),
    dict(block_table=torch.zeros(3, 2, dtype=torch.int32)),
    dict(free_start=_i32(0, 1)),
    dict(free_start=torch.tensor([0])),
    dict(lengths=torch.zeros(5000, dtype=torch.int32), counts=torch.zeros(5000, dtype=torch.int32),
         block_table=torch.zeros(5000, 2, dtype=torch.int32)),
])
def test_assign_refusals(calls, kw):
    with pytest.raises(ValueError):
        _assign(**kw)
    assert not calls


def test_tensors_off_the_gpu_are_refused():
    for f in (_prompt, _tree, _write, _assign):
        with pytest.raises(ValueError, match="on one GPU"):
            f()


def test_requires_grad_is_fine_without_a_graph(calls):
    with torch.no_grad():
        _prompt(q=torch.zeros(6, 4, 64).bfloat16().requires_grad_())
    assert len(calls) == 1


def test_forward_mode_tangents_are_refused(calls):
    """Of anything read or written, with grad mode off too; not of plain tensors
    inside the level, nor outside of one."""
    def dual(t):
        return torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))

    with torch.autograd.forward_ad.dual_level():
        _prompt(), _tree(), _write()
        assert len(calls) == 3
        calls.clear()
        bad = [(_prompt, dict(q=dual(torch.zeros(6, 4, 64).bfloat16()))), (_prompt, dict(v=dual(torch.zeros(6, 2, 64).bfloat16()))),
               (_prompt, dict(o=dual(torch.zeros(6, 4, 64).bfloat16()))), (_prompt, dict(lse=dual(torch.zeros(4, 6)))),
               (_tree, dict(q=dual(torch.zeros(6, 4, 64).bfloat16()))), (_tree, dict(k_cache=dual(torch.zeros(3, 16, 2, 64).bfloat16()))),
               (_write, dict(k=dual(torch.zeros(6, 2, 64).half()))), (_write, dict(v_cache=dual(torch.zeros(3, 16, 2, 64).half())))]
        for f, kw in bad:
            with pytest.raises(ValueError, match="forward only"):
                f(**kw)
            with pytest.raises(ValueError, match="forward only"), torch.no_grad():
                f(**kw)
    assert not calls


# --- the C entries -------------------------------------------------------------

def _arr(*v):
    return (ctypes.c_int64 * len(v))(*v)


VARLEN = dict(q=FAKE, k=FAKE, v=FAKE, o=FAKE, lse=None, cu_q=FAKE, cu_k=FAKE, B=1, T=6, TK=6, HQ=4, HK=2, D=64,
              qs=(256, 64), ks=(128, 64), vs=(128, 64), os=(256, 64), scale=0.125, dtype=_lib.G9_BF16, causal=1)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=_lib.G9_BF8), _lib.G9_ERR_DTYPE),
    (dict(D=96), _lib.G9_ERR_SHAPE),
    (dict(HQ=5), _lib.G9_ERR_SHAPE),
    (dict(HK=0), _lib.G9_ERR_SHAPE),
    (dict(T=-1), _lib.G9_ERR_SHAPE),
    (dict(T=2**31), _lib.G9_ERR_SHAPE),
    (dict(TK=2**31), _lib.G9_ERR_SHAPE),
    (dict(B=2**21, T=2**21), _lib.G9_ERR_SHAPE),  # workgroups of a launch
    (dict(scale=0.0), _lib.G9_ERR_SHAPE),
    (dict(scale=-1.0), _lib.G9_ERR_SHAPE),
    (dict(scale=float("nan")), _lib.G9_ERR_SHAPE),
    (dict(scale=float("inf")), _lib.G9_ERR_SHAPE),
    (dict(qs=(250, 64)), _lib.G9_ERR_LAYOUT),
    (dict(ks=(-128, 64)), _lib.G9_ERR_LAYOUT),
    (dict(os=(0, 64)), _lib.G9_ERR_LAYOUT),      # rows of o on top of each other
    (dict(os=(128, 64)), _lib.G9_ERR_LAYOUT),
    (dict(os=(256, 56)), _lib.G9_ERR_LAYOUT),
    (dict(q=FAKE + 2), _lib.G9_ERR_LAYOUT),
    (dict(k=None), _lib.G9_ERR_LAYOUT),
    (dict(lse=FAKE + 1), _lib.G9_ERR_LAYOUT),
    (dict(cu_k=None), _lib.G9_ERR_LAYOUT),
    (dict(T=0), _lib.G9_OK),
    (dict(B=0), _lib.G9_OK),
])
def test_varlen_entry_validation(kw, code):
    a = dict(VARLEN, **kw)
    assert _lib.load().g9_varlen_fwd(a["q"], a["k"], a["v"], a["o"], a["lse"], a["cu_q"], a["cu_k"], a["B"], a["T"],
                                     a["TK"], a["HQ"], a["HK"], a["D"], _arr(*a["qs"]), _arr(*a["ks"]), _arr(*a["vs"]),
                                     _arr(*a["os"]), a["scale"], a["dtype"], a["causal"], None) == code


TREE = dict(q=FAKE, k=FAKE, v=FAKE, o=FAKE, lse=None, table=FAKE, ts=4, width=4, lengths=FAKE, cu=FAKE, mask=FAKE,
            words=1, B=2, T=6, HQ=4, HK=2, D=64, nb=8, bs=16, qs=(256, 64), ks=(2048, 128, 64), vs=(2048, 128, 64),
            os=(256, 64), scale=0.125, dtype=_lib.G9_F16, ws=FAKE, ws_bytes=2**40)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=_lib.G9_FP4), _lib.G9_ERR_DTYPE),
    (dict(D=32), _lib.G9_ERR_SHAPE),
    (dict(HQ=3), _lib.G9_ERR_SHAPE),
    (dict(bs=8), _lib.G9_ERR_SHAPE),
    (dict(bs=48), _lib.G9_ERR_SHAPE),
    (dict(bs=2048), _lib.G9_ERR_SHAPE),
    (dict(words=0), _lib.G9_ERR_SHAPE),
    (dict(words=-1), _lib.G9_ERR_SHAPE),
    (dict(width=2**28, ts=2**28), _lib.G9_ERR_SHAPE),
    (dict(scale=float("nan")), _lib.G9_ERR_SHAPE),
    (dict(ts=3), _lib.G9_ERR_LAYOUT),
    (dict(ks=(2048, 128, 60)), _lib.G9_ERR_LAYOUT),
    (dict(os=(64, 64)), _lib.G9_ERR_LAYOUT),
    (dict(table=None), _lib.G9_ERR_LAYOUT),
    (dict(lengths=None), _lib.G9_ERR_LAYOUT),
    (dict(mask=FAKE + 4), _lib.G9_ERR_LAYOUT),
    (dict(v=FAKE + 8), _lib.G9_ERR_LAYOUT),
    (dict(B=0), _lib.G9_OK),
    (dict(T=0), _lib.G9_OK),
])
def test_tree_entry_validation(kw, code):
    a = dict(TREE, **kw)
    assert _lib.load().g9_tree_fwd(a["q"], a["k"], a["v"], a["o"], a["lse"], a["table"], a["ts"], a["width"],
                                   a["lengths"], a["cu"], a["mask"], a["words"], a["B"], a["T"], a["HQ"], a["HK"],
                                   a["D"], a["nb"], a["bs"], _arr(*a["qs"]), _arr(*a["ks"]), _arr(*a["vs"]),
                                   _arr(*a["os"]), a["scale"], a["dtype"], a["ws"], a["ws_bytes"], None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(D=100), _lib.G9_ERR_SHAPE),
    (dict(bs=20), _lib.G9_ERR_SHAPE),
    (dict(T=-1), _lib.G9_ERR_SHAPE),
    (dict(kc=(0, 128, 64)), _lib.G9_ERR_LAYOUT),       # blocks on top of each other
    (dict(vc=(2048, 64, 64)), _lib.G9_ERR_LAYOUT),
    (dict(kc=(2048, 128, 32)), _lib.G9_ERR_LAYOUT),
    (dict(slots=FAKE + 4), _lib.G9_ERR_LAYOUT),
    (dict(k=FAKE + 8), _lib.G9_ERR_LAYOUT),
    (dict(T=0), _lib.G9_OK),
    (dict(nb=0), _lib.G9_OK),
])
def test_write_entry_validation(kw, code):
    a = dict(k=FAKE, slots=FAKE, T=6, HK=2, D=64, nb=8, bs=16, kc=(2048, 128, 64), vc=(2048, 128, 64))
    a.update(kw)
    assert _lib.load().g9_write_cache(a["k"], FAKE, FAKE, FAKE, a["slots"], a["T"], a["HK"], a["D"], a["nb"], a["bs"],
                                      _arr(128, 64), _arr(128, 64), _arr(*a["kc"]), _arr(*a["vc"]), None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(B=4097), _lib.G9_ERR_SHAPE),
    (dict(B=-1), _lib.G9_ERR_SHAPE),
    (dict(bs=0), _lib.G9_ERR_SHAPE),
    (dict(T=2**31), _lib.G9_ERR_SHAPE),
    (dict(ts=3), _lib.G9_ERR_LAYOUT),
    (dict(lengths=None), _lib.G9_ERR_LAYOUT),
    (dict(slots=None), _lib.G9_ERR_LAYOUT),
    (dict(taken=None), _lib.G9_ERR_LAYOUT),
])
def test_assign_entry_validation(kw, code):
    a = dict(lengths=FAKE, B=2, ts=4, width=4, bs=16, T=6, slots=FAKE, taken=FAKE)
    a.update(kw)
    assert _lib.load().g9_assign_slots(a["lengths"], FAKE, a["B"], FAKE, a["ts"], a["width"], FAKE, 9, None, a["bs"],
                                       a["T"], FAKE, a["slots"], FAKE, a["taken"], None) == code


def test_most_requests_matches_the_header():
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "gfx950_fmha.h")).read()
    assert int(re.search(r"#define G9_SLOTS_MAX_REQUESTS (\d+)", text).group(1)) == paged.MAX_REQUESTS


# --- the oracle -------------------------------------------------------------------

@pytest.mark.parametrize("lq,lk", [(5, 5), (3, 9), (9, 3), (1, 1), (4, 0)])
@pytest.mark.parametrize("causal", [True, False])
def test_oracle_attention_against_torch(lq, lk, causal):
    rng = np.random.default_rng(lq * 10 + lk)
    q, k, v = (torch.from_numpy(rng.standard_normal((n, 16))) for n in (lq, lk, lk))
    o, lse, _, _ = R.masked_attention(q, k, v, R.causal_reads(lq, lk, causal), 0.25)
    x = q @ k.T * 0.25
    if causal:
        i, j = torch.arange(lq)[:, None], torch.arange(lk)[None]
        x = x.masked_fill(j > i + lk - lq, float("-inf"))
    want = torch.nan_to_num(torch.softmax(x, 1) @ v, nan=0.0) if lk else torch.zeros(lq, 16, dtype=torch.float64)
    assert np.allclose(o, want.numpy(), atol=1e-12)
    assert np.allclose(lse, torch.logsumexp(x, 1).numpy(), atol=1e-12)


@pytest.mark.parametrize("n", [1100, 3000, 9000])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_the_bound_tells_a_wrong_output_at_the_longest_lengths(n, D, dtype):
    """Outputs of zeros, and those of the first half of the keys, leave it nearly
    everywhere; the weights and the output rounded to 16 bits do not."""
    gen = torch.Generator().manual_seed(n + D)
    q, k, v = (torch.randn(m, D, generator=gen).to(dtype).double().numpy() for m in (8, n, n))
    reads = np.ones((8, n), bool)
    o, lse, mag, spread = R.masked_attention(q, k, v, reads, D**-0.5)
    subnormal = 2.0**-25 if dtype == torch.float16 else 0.0
    to, _ = R.tolerances(o, lse, mag, spread, torch.finfo(dtype).eps, n, D, float(np.abs(v).max()), subnormal)
    half = R.masked_attention(q, k[:n // 2], v[:n // 2], reads[:, :n // 2], D**-0.5)[0]
    assert (np.abs(o) > to).mean() > 0.5 and (np.abs(half - o) > to).mean() > 0.5
    for lag in (0.0, 8.0):  # of the running maximum, in powers of two
        s = torch.from_numpy(q @ k.T * D**-0.5 / np.log(2.0))
        w = torch.exp2(s - (s.amax(1, keepdim=True) - lag))
        got = (w.to(dtype).double() @ torch.from_numpy(v) / w.sum(1, keepdim=True)).to(dtype).double().numpy()
        assert (np.abs(got - o) <= to).all()


def test_oracle_slots_by_hand():
    cu, slots, pos, taken, table = R.slots([3, 4], [2, 5], np.array([[9, 0, 0], [7, 0, 0]], np.int32), [5, 6], 0, 4, 8)
    assert cu.tolist() == [0, 2, 7] and taken == 3
    assert slots.tolist() == [39, 20, 24, 25, 26, 27, -1, -1]
    assert pos.tolist() == [3, 4, 4, 5, 6, 7, 8, 0]
    assert table.tolist() == [[9, 5, 0], [7, 6, -1]]
