"""GPU: the variants of group_norm_act and cross_attn_backward that only large calls select.  Tolerances are those of
test_gpu_group_norm_act.py and test_gpu_cross_attn.py."""
import pytest
import torch

from tests.test_gpu_cross_attn import BF, check, inputs, ops  # noqa: F401
from tests.test_gpu_group_norm_act import EPS, HALF, U, close, make, reference

pytestmark = pytest.mark.gpu
F32 = torch.float32


@pytest.mark.parametrize("dims,keys", [((8, 2053, 300, 8, 8, 64), "none"), ((8, 2053, 300, 8, 8, 64), "mask"), ((8, 1030, 300, 16, 8, 24), "none"),
                                       ((8, 1030, 300, 16, 8, 24), "mask"), ((24, 3000, 257, 8, 8, 32), "lens"),
                                       ((29, 2100, 290, 16, 8, 40), "both")],
                         ids=lambda d: "x".join(map(str, d)) if isinstance(d, tuple) else d)
def test_gradients_with_two_row_groups_a_wave(ops, dims, keys):
    """bf16, more than 256 keys, up to 64 columns and 512 blocks of 256 rows (2048 with lengths): ragged last row tiles, waves and second
    groups without a row, shared heads, images that show nothing."""
    B, nq, nk, H, KV, hd = dims
    assert -(-nq * (H // KV) // 256) * B * KV >= (2048 if keys in ("lens", "both") else 512) and nk > 256
    check(ops, inputs(*dims, keys, BF, seed=sum(dims)), dims)


def image(t, b, n):
    return None if t is None else t[b * n:(b + 1) * n]


@pytest.mark.parametrize("C,G", [(64, 32), (63, 9)])
@pytest.mark.parametrize("dt,do", [(BF, BF), (F32, F32), (F32, BF)], ids=["bf16", "f32", "f32-bf16"])
def test_forward_past_the_caches(ops, dt, do, C, G):
    """Rows in and out above 192 MB are written past the caches: 16 images of 256 x 256, vectors of 16 bytes and of one element, in
    place as well."""
    B, n = 16, 65536
    x, gamma, beta, ss, _ = make(B, n, C, True, dt, seed=C)
    assert x.nbytes + x.numel() * (2 if do == BF else 4) > 192 << 20
    ws = torch.empty(ops.group_norm_act_workspace_bytes(B, n, C, G), dtype=torch.uint8, device="cuda")
    out = torch.full((B * n, C), float("nan"), dtype=do, device="cuda")
    ops.group_norm_act(x, B, n, C, G, EPS, gamma, beta, out, ws, act=ops.ACT_SILU, scale_shift=ss)
    for b in range(B):
        r = reference(image(x, b, n), gamma, beta, ss[b:b + 1], 1, n, C, G, True)
        close(image(out, b, n), r["y"], r["ty"], HALF[do])
    if do == dt:
        ops.group_norm_act(x, B, n, C, G, EPS, gamma, beta, x, ws, act=ops.ACT_SILU, scale_shift=ss)
        assert torch.equal(x, out)


@pytest.mark.parametrize("C,G", [(64, 32), (63, 9)])
@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "f32"])
def test_backward_past_the_caches(ops, dt, C, G):
    B, n = 16, 65536
    x, gamma, beta, ss, dy = make(B, n, C, True, dt, seed=C + 1)
    assert 3 * x.nbytes > 192 << 20
    ws = torch.empty(ops.group_norm_act_workspace_bytes(B, n, C, G), dtype=torch.uint8, device="cuda")
    mean, rstd = torch.empty(B, G, device="cuda"), torch.empty(B, G, device="cuda")
    dx = torch.empty_like(x)
    ops.group_norm_act(x, B, n, C, G, EPS, gamma, beta, dx, ws, act=ops.ACT_SILU, scale_shift=ss, mean=mean, rstd=rstd)
    dx.fill_(float("nan"))
    e = lambda *s: torch.full(s, float("nan"), device="cuda")  # noqa: E731
    dg, db, dss = e(C), e(C), e(B, 2 * C)
    kw = dict(act=ops.ACT_SILU, scale_shift=ss, dscale_shift=dss)
    ops.group_norm_act_backward(dy, x, B, n, C, G, gamma, beta, mean, rstd, dx, dg, db, ws, **kw)
    sums = dict(dgamma=0, tdgamma=0, dbeta=0, tdbeta=0)
    for b in range(B):
        r = reference(image(x, b, n), gamma, beta, ss[b:b + 1], 1, n, C, G, True, dy=image(dy, b, n))
        close(image(dx, b, n), r["dx"], r["tdx"], HALF[dt])
        close(dss[b:b + 1], r["dss"], r["tdss"], 4 * U)
        sums = {k: v + r[k] for k, v in sums.items()}
    close(dg, sums["dgamma"], sums["tdgamma"], 4 * U)
    close(db, sums["dbeta"], sums["tdbeta"], 4 * U)
    for into in (dy, x):      # in place: first of dy, then of x
        d2 = dy.clone()
        x2 = x.clone()
        target = d2 if into is dy else x2
        ops.group_norm_act_backward(d2, x2, B, n, C, G, gamma, beta, mean, rstd, target, dg, db, ws, **kw)
        assert torch.equal(target, dx)
