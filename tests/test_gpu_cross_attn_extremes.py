"""GPU: cross_attn at the ends of what it accepts: rows far apart, scales and scores of any size, large values.  Tolerances are
those of test_gpu_cross_attn.py; where a call is the same up to powers of two, the answers have to be equal."""
import math

import pytest
import torch

from tests.test_gpu_cross_attn import BF, F32, U, check, inputs, ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dims,dt", [((1, 128, 20, 1, 1, 32), F32), ((1, 200, 30, 2, 2, 64), F32), ((1, 150, 20, 2, 1, 24), F32),
                                     ((1, 128, 17, 1, 1, 128), BF), ((1, 190, 32, 1, 1, 96), BF)],
                         ids=lambda d: "x".join(map(str, d)) if isinstance(d, tuple) else str(d).split(".")[-1])
def test_rows_20_mb_apart(ops, dims, dt):
    """q and dout as columns of one matrix whose rows are 20 MB apart: a tile of 128 rows spans more than 2^31 bytes."""
    B, nq, nk, H, KV, hd = dims
    t = inputs(*dims, "none", dt, seed=sum(dims))
    es = 2 if dt == BF else 4
    wide = torch.empty(B * nq, 20 * 2 ** 20 // es, dtype=dt, device="cuda")
    for i, name in enumerate(("q", "do")):
        cols = wide[:, 256 * i:256 * i + H * hd]
        cols.copy_(t[name])
        t[name] = cols
    check(ops, t, dims)
