"""latent_attention over infinite and NaN values that rows read: what shows in the rows that
read them, and that nothing shows in the others."""

import numpy as np
import pytest
import torch

from gfx950_gluon_tutorials_amd.attention import latent_attention

pytestmark = pytest.mark.gpu

SCALE, SIZE, COLUMN = 192**-0.5, 16, 100


def _inputs(dev, context, H, seed):
    """One token a request; the queries' value in COLUMN is 1 in even heads, -1 in odd ones."""
    g = torch.Generator().manual_seed(seed)
    B, used = len(context), [-(-(n + 1) // SIZE) for n in context]
    ids = torch.randperm(sum(used) + 2, generator=g).tolist()
    table = np.zeros((B, max(used)), np.int32)
    for b, n in enumerate(used):
        table[b, :n] = [ids.pop() for _ in range(n)]
    cache = torch.randn(sum(used) + 2, SIZE, 576, generator=g).bfloat16().to(dev)
    q = (torch.randn(B, H, 576, generator=g) * 0.6).bfloat16().to(dev)
    q[:, 0::2, COLUMN], q[:, 1::2, COLUMN] = 1, -1
    i = lambda x: torch.tensor(x, dtype=torch.int32).to(dev)
    args = (i(table), i(context), i(list(range(B + 1))))
    return q, cache, table, lambda: latent_attention(q, cache, *args, sm_scale=SCALE)


# Contexts of one part and of many; a key of a tile (32 keys) that every row reads whole, and one of the last.
CASES = [([40], 19), ([40], 35), ([3000, 500], 19), ([3000, 500], 1601), ([3000, 500], 2999), ([33000, 7], 20000)]


@pytest.mark.parametrize("context,key", CASES, ids=str)
def test_a_latent_that_one_request_reads(gpu, context, key):
    for H in (16, 64, 128):
        q, cache, table, run = _inputs(gpu, context, H, H + key)
        clean = run().clone()
        assert clean.isfinite().all()
        at = (int(table[0][key // SIZE]), key % SIZE, COLUMN)
        odd, rest = torch.arange(H, device=gpu) % 2 == 1, torch.arange(512, device=gpu) != COLUMN
        for bad in (float("inf"), float("-inf"), float("nan")):
            cache[at] = bad
            got = run()
            assert torch.equal(got[1:], clean[1:])
            # A weight of 0 does not keep the value out of its column; a score of infinity or NaN takes the row.
            up = odd | ~odd if bad != bad else odd if bad < 0 else ~odd
            assert got[0, :, COLUMN].isnan().all() and got[0][up].isnan().all()
            # Heads whose score is -infinity: where every row reads the tile, the key's weight is 0, as with
            # a finite value of a score as far below the others, but in that column.
            if (key // 32 + 1) * 32 <= context[0] and not up.all():
                cache[at] = 1e30 if bad > 0 else -1e30
                want = run()[0][~up][:, rest]
                assert want.isfinite().all() and torch.equal(got[0][~up][:, rest], want)


@pytest.mark.parametrize("context,key", CASES, ids=str)
def test_a_rotated_key_that_one_request_reads(gpu, context, key):
    for H in (16, 128):
        q, cache, table, run = _inputs(gpu, context, H, key)
        clean = run().clone()
        cache[int(table[0][key // SIZE]), key % SIZE, 512 + 9] = float("nan")
        got = run()
        assert got[0].isnan().all() and torch.equal(got[1:], clean[1:])
