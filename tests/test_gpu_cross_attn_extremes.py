"""GPU: cross_attn at the ends of what it accepts: rows far apart, scales and scores of any size, large values.  Tolerances are
those of test_gpu_cross_attn.py; where a call is the same up to powers of two, the answers have to be equal."""
import math

import pytest
import torch

from tests.test_gpu_cross_attn import BF, F32, U, check, close, inputs, ops, reference  # noqa: F401

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


def call(ops, t, dims, scale):
    B, nq, nk, H, KV, hd = dims
    dt = t["q"].dtype
    nan = lambda *s, d=dt: torch.full(s, float("nan"), dtype=d, device="cuda")  # noqa: E731
    r = dict(out=nan(B * nq, H * hd), lse=nan(B, H, nq, d=F32), dq=nan(B * nq, H * hd), dk=nan(B * nk, KV * hd), dv=nan(B * nk, KV * hd))
    nb = max(ops.cross_attn_workspace_bytes(*dims, dt), ops.cross_attn_backward_workspace_bytes(*dims, dt))
    ws = torch.full((nb,), 0xff, dtype=torch.uint8, device="cuda")
    kw = dict(key_lens=t["lens"], key_mask=t["mask"])
    ops.cross_attn(t["q"], t["k"], t["v"], *dims, scale, r["out"], ws, lse=r["lse"], **kw)
    ops.cross_attn_backward(t["q"], t["k"], t["v"], r["out"], r["lse"], t["do"], *dims, scale, r["dq"], r["dk"], r["dv"], ws, **kw)
    return r


@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("dims", [(2, 70, 100, 2, 2, 32), (2, 300, 400, 4, 2, 64), (1, 40, 20, 1, 1, 128), (2, 1, 400, 4, 2, 64),
                                  (16, 2053, 100, 8, 8, 32)], ids=lambda d: "x".join(map(str, d)))
def test_scale_of_any_size(ops, dims, dt):
    """q and k smaller and the scale larger by the same powers of two (and the other way round): the same scores, bit for bit, with
    units of 32 keys that the mask hides wholly at the start and beside shown ones."""
    B, nq, nk, H, KV, hd = dims
    t = inputs(*dims, "mask", dt, seed=nk)
    t["mask"][:, :32] = nk <= 32
    t["mask"][:, 64:96] = False
    t["mask"][0, 40:] = True
    want = call(ops, t, dims, hd ** -0.5)
    assert all(bool(torch.isfinite(want[n]).all()) for n in ("out", "dq", "dk", "dv"))
    for e in (17, 32, -30):     # scales 3e9 and up, 3e18 and up, 3e-19 and down
        s = dict(t, q=t["q"] * 2.0 ** -e, k=t["k"] * 2.0 ** -e)
        got = call(ops, s, dims, hd ** -0.5 * 4.0 ** e)
        for n in ("out", "lse", "dv"):
            assert torch.equal(got[n], want[n]), (n, e)
        for n in ("dq", "dk"):
            assert torch.equal(got[n], want[n] * 2.0 ** e), (n, e)


@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("nq", [1, 50])
def test_scores_far_below_zero(ops, nq, dt):
    """Every product q k is -1e31 or -2e31: the former share the row evenly, the latter get nothing.  lse = -8 2^34 + log(count): the
    sum is lost in the product's rounding, one of fp32 for the product and one for the logarithm's base each way: 4 u of it."""
    dims = B, nq, nk, H, KV, hd = (1, nq, 90, 2, 2, 8)
    t = inputs(*dims, "none", dt, seed=5)
    t["q"] = torch.full_like(t["q"], 2.0 ** 50)
    near = torch.arange(nk, device="cuda") % 3 == 0
    t["k"] = torch.where(near[:, None], -2.0 ** 50, -2.0 ** 51).to(dt).expand(nk, H * hd).contiguous()
    r = call(ops, t, dims, 2.0 ** -66)
    mean = t["v"].double()[near].mean(0)
    # 30 equal probabilities: 1/30 formed by a reciprocal (u), sums of 30 terms, the store's half step
    tol = 40 * U * t["v"].double()[near].abs().mean(0) + (2.0 ** -8 if dt == BF else U) * mean.abs()
    assert bool(((r["out"].double() - mean).abs() <= tol).all())
    lse = -8 * 2.0 ** 34 + math.log(30)
    assert bool(((r["lse"].double() - lse).abs() <= 4 * U * abs(lse)).all())


@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("dims", [(2, 70, 300, 2, 2, 16), (2, 2, 300, 2, 2, 16), (16, 2053, 300, 8, 8, 16)], ids=lambda d: "x".join(map(str, d)))
def test_large_values_under_rising_scores(ops, dims, dt):
    """v of 1e22 beside scores that rise from 0 to 40 along the keys: e^40 1e22 would pass the fp32 range, the answer does not."""
    B, nq, nk, H, KV, hd = dims
    t = inputs(*dims, "none", dt, seed=7)
    q, k = torch.zeros(B * nq, H, hd, device="cuda"), torch.zeros(B, nk, KV, hd, device="cuda")
    q[..., 0] = 4        # scale 1/4
    k[:, 128:, :, 0] = 40
    t["q"], t["k"] = q.reshape(B * nq, -1).to(dt), k.reshape(B * nk, -1).to(dt)
    t["v"] = (t["v"].float() * 1e22).to(dt)
    check(ops, t, dims, grads=nq < 100)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("dims", [(2, 5, 300, 4, 2, 64), (2, 300, 77, 4, 2, 32), (2, 300, 400, 2, 2, 96), (8, 2053, 300, 8, 8, 24)],
                         ids=lambda d: "x".join(map(str, d)))
def test_a_bad_query_stays_in_its_row(ops, dims, dt, bad):
    """A query row of NaN or infinities (and a gradient row) leaves the answers and dq of all other rows right."""
    B, nq, nk, H, KV, hd = dims
    t = inputs(*dims, "mask", dt, seed=13)
    rows = torch.tensor([0, nq + nq // 2, B * nq - 1], device="cuda")
    ok = torch.ones(B * nq, dtype=torch.bool, device="cuda")
    ok[rows] = False
    hit = dict(t, q=t["q"].clone(), do=t["do"].clone())
    hit["q"][rows] = bad
    hit["do"][rows] = bad
    r, w = reference(t, *dims), call(ops, hit, dims, hd ** -0.5)
    close("out", w["out"][ok], r["o"][ok], r["to"][ok], r["h"])
    close("dq", w["dq"][ok], r["dq"][ok], r["tdq"][ok], r["h"])
