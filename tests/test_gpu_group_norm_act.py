"""GPU: group_norm_act and its backward (uwir_group_norm_act*) against the operator's definition in 64 bits.

Tolerances, per element, from the roundings on the way (u = 2^-24, the half step of fp32; h = half a step of the output type,
2^-8 for bf16, u for fp32):
  forward   z = (x - m) a + s with m, a, s each rounded a few times and statistics whose fp32 part is a few roundings of a
            thread's own rows: |dz| <= 16 u (|m a| + |(x - m) a| + |s|);  |act'| <= 1.1;  SiLU's own error is that of
            exp2 at an argument rounded to |z| u: <= 4 u (1 + |z|) |y|;  then the store: h |y|.
  backward  dz = dy act'(z), so |d dz| <= 16 u |dy| (1 + |dz/z error|);  S1, S2 are sums of n rows: the terms' own errors
            plus 64 u sum |terms| (fp32 chains of at most 64 merged batches, fp64 beyond);  dx = r (w dz - m1 - xh m2)
            adds up the errors of its three parts."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8}
EPS = 1e-5


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from underwater_image_restoration_amd import _lib, ops as o
    _lib.load()
    return o


def make(B, n, C, ss, dt, seed=0, offset=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x = (r(B * n, C) * (0.5 + r(C).abs()) + r(C) + offset).to(dt)
    return x, 1 + 0.2 * r(C), 0.2 * r(C), (0.3 * r(B, 2 * C) if ss else None), r(B * n, C).to(dt)


def reference(x, gamma, beta, ss, B, n, C, G, silu, eps=EPS, dy=None):
    """fp64: (y, tolerance of y in fp32 arithmetic, mean, rstd) and, with dy, the gradients and their tolerances."""
    X = x.double().view(B, n, G, C // G)
    m = X.mean((1, 3), keepdim=True)
    r = ((X - m).square().mean((1, 3), keepdim=True) + eps).rsqrt()
    flat = lambda t: t.expand(B, n, G, C // G).reshape(B, n, C)  # noqa: E731
    M, Rr = flat(m), flat(r)
    xh = (X.reshape(B, n, C) - M) * Rr
    f = 1.0 if ss is None else 1.0 + ss.double()[:, None, :C]
    sh = 0.0 if ss is None else ss.double()[:, None, C:]
    w = gamma.double() * f
    s = beta.double() * f + sh + torch.zeros_like(xh)
    z = xh * w + s
    tz = 16 * U * ((M * Rr * w).abs() + (xh * w).abs() + s.abs())
    sg = torch.sigmoid(z)
    y = z * sg if silu else z
    ty = (1.1 * tz + 4 * U * (1 + z.abs()) * y.abs()) if silu else tz
    out = dict(y=y.reshape(B * n, C), ty=ty.reshape(B * n, C), mean=m.view(B, G), rstd=r.view(B, G))
    if dy is None:
        return out
    DY = dy.double().view(B, n, C)
    da = sg * (1 + z * (1 - sg)) if silu else torch.ones_like(z)
    dz = DY * da
    # act'' of SiLU is at most 0.5; sigmoid at an argument off by |z| u
    tdz = DY.abs() * (0.5 * tz + 8 * U * (1 + z.abs())) + 4 * U * dz.abs() if silu else torch.zeros_like(dz)
    txh = 4 * U * ((M * Rr).abs() + xh.abs())
    s1, s2 = dz.sum(1), (dz * xh).sum(1)
    t1 = tdz.sum(1) + 64 * U * dz.abs().sum(1)
    t2 = (tdz * xh.abs() + dz.abs() * txh).sum(1) + 64 * U * (dz * xh).abs().sum(1)
    N = n * (C // G)
    W = w + torch.zeros(B, 1, C, dtype=torch.float64, device="cuda")
    grp = lambda t: (t.view(B, G, C // G).sum(2) / N)[:, None, :, None]  # noqa: E731
    m1, m2 = flat(grp(W[:, 0] * s1)), flat(grp(W[:, 0] * s2))
    e1, e2 = flat(grp(W[:, 0].abs() * t1)), flat(grp(W[:, 0].abs() * t2))
    dx = Rr * (W * dz - m1 - xh * m2)
    tdx = Rr * (W.abs() * tdz + e1 + xh.abs() * e2 + txh * m2.abs()
                + 16 * U * ((W * dz).abs() + m1.abs() + (xh * m2).abs()))
    F = W[:, 0] / gamma.double()
    out.update(dx=dx.reshape(B * n, C), tdx=tdx.reshape(B * n, C), dgamma=(F * s2).sum(0), tdgamma=(F.abs() * t2).sum(0),
               dbeta=(F * s1).sum(0), tdbeta=(F.abs() * t1).sum(0))
    if ss is not None:
        out["dss"] = torch.cat([gamma.double() * s2 + beta.double() * s1, s1], 1)
        out["tdss"] = torch.cat([gamma.double().abs() * t2 + beta.double().abs() * t1, t1], 1)
    return out


def close(got, want, tol, half):
    e = (got.double() - want).abs()
    lim = tol + half * want.abs() * 1.01 + 1e-30
    bad = e > lim
    assert bool(torch.isfinite(got).all()) and not bool(bad.any()), \
        f"{int(bad.sum())} of {bad.numel()} off, worst {float((e / lim).max()):.2f} of the tolerance"


# n = 1, one element a group (variance 0), odd channel counts, unaligned groups, both forms, one group over everything
SHAPES = [(1, 1, 8, 8), (2, 1, 32, 4), (1, 64, 512, 32), (3, 418, 96, 32), (2, 33, 15, 5), (2, 1500, 30, 3), (1, 5000, 64, 32),
          (2, 700, 1024, 1), (5, 17, 2048, 32), (1, 2049, 2048, 2048), (2, 4100, 396, 4), (16, 1024, 128, 32), (1, 70001, 6, 2),
          (2, 900, 1026, 2), (2, 900, 1026, 1), (1, 700, 2047, 1), (3, 5000, 192, 64), (1, 3000, 160, 4)]


@pytest.mark.parametrize("dt,do", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16),
                                   (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("B,n,C,G", SHAPES)
def test_forward(ops, B, n, C, G, dt, do):
    for silu, ss in ((True, True), (False, False)):
        x, gamma, beta, sst, _ = make(B, n, C, ss, dt, seed=n + C)
        out = torch.full((B * n, C), float("nan"), dtype=do, device="cuda")
        mean, rstd = torch.empty(B, G, device="cuda"), torch.empty(B, G, device="cuda")
        ws = torch.empty(ops.group_norm_act_workspace_bytes(B, n, C, G), dtype=torch.uint8, device="cuda")
        ops.group_norm_act(x, B, n, C, G, EPS, gamma, beta, out, ws, act=ops.ACT_SILU if silu else ops.ACT_NONE,
                           scale_shift=sst, mean=mean, rstd=rstd)
        r = reference(x, gamma, beta, sst, B, n, C, G, silu)
        close(out, r["y"], r["ty"], HALF[do])
        close(mean, r["mean"], 4 * U * x.double().abs().max(), U)
        close(rstd, r["rstd"], 8 * U * r["rstd"], U)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,n,C,G", SHAPES)
def test_backward(ops, B, n, C, G, dt):
    for silu, ss in ((True, True), (False, False), (True, False)):
        x, gamma, beta, sst, dy = make(B, n, C, ss, dt, seed=n + C)
        act = ops.ACT_SILU if silu else ops.ACT_NONE
        ws = torch.empty(ops.group_norm_act_workspace_bytes(B, n, C, G), dtype=torch.uint8, device="cuda")
        y, mean, rstd = torch.empty_like(x), torch.empty(B, G, device="cuda"), torch.empty(B, G, device="cuda")
        ops.group_norm_act(x, B, n, C, G, EPS, gamma, beta, y, ws, act=act, scale_shift=sst, mean=mean, rstd=rstd)
        dx = torch.full_like(x, float("nan"))
        dg, db = (torch.full((C,), float("nan"), device="cuda") for _ in range(2))
        dss = torch.full((B, 2 * C), float("nan"), device="cuda") if ss else None
        ops.group_norm_act_backward(dy, x, B, n, C, G, gamma, beta, mean, rstd, dx, dg, db, ws, act=act, scale_shift=sst,
                                    dscale_shift=dss)
        r = reference(x, gamma, beta, sst, B, n, C, G, silu, dy=dy)
        close(dx, r["dx"], r["tdx"], HALF[dt])
        close(dg, r["dgamma"], r["tdgamma"], 4 * U)
        close(db, r["dbeta"], r["tdbeta"], 4 * U)
        if ss:
            close(dss, r["dss"], r["tdss"], 4 * U)


def test_mean_far_from_zero_and_stray_element(ops):
    """The statistics lose no digits to a large mean, nor to one element far from all others (the first of its group)."""
    for n in (300, 30000):
        x, gamma, beta, _, _ = make(2, n, 64, False, torch.float32, seed=3, offset=2000.0)
        x[0, 0] = -3.0e4
        out, ws = torch.empty_like(x), torch.empty(ops.group_norm_act_workspace_bytes(2, n, 64, 8), dtype=torch.uint8, device="cuda")
        ops.group_norm_act(x, 2, n, 64, 8, EPS, gamma, beta, out, ws)
        r = reference(x, gamma, beta, None, 2, n, 64, 8, False)
        close(out, r["y"], r["ty"], U)


def test_strides_in_place_and_untouched_memory(ops):
    B, n, C, G = 2, 300, 24, 3
    for dt in (torch.float32, torch.bfloat16):
        for pad in (8, 3, 1):     # row strides that allow 16-byte, 2- and 4-byte accesses only
            x, gamma, beta, _, dy = make(B, n, C, False, dt, seed=pad)
            wide = torch.full((B * n + 2, C + 2 * pad), 7.0, dtype=dt, device="cuda")
            view = wide[1:-1, pad:pad + C]
            view.copy_(x)
            ws = torch.empty(ops.group_norm_act_workspace_bytes(B, n, C, G), dtype=torch.uint8, device="cuda")
            r = reference(x, gamma, beta, None, B, n, C, G, True)
            out = torch.full((B * n + 2, C + pad), 7.0, dtype=dt, device="cuda")
            ops.group_norm_act(view, B, n, C, G, EPS, gamma, beta, out[1:-1, :C], ws, act=ops.ACT_SILU)
            close(out[1:-1, :C], r["y"], r["ty"], HALF[dt])
            assert bool((out[0] == 7).all() and (out[-1] == 7).all() and (out[:, C:] == 7).all())
            ops.group_norm_act(view, B, n, C, G, EPS, gamma, beta, view, ws, act=ops.ACT_SILU)     # in place
            assert torch.equal(view, out[1:-1, :C])
            assert bool((wide[0] == 7).all() and (wide[-1] == 7).all() and (wide[:, :pad] == 7).all() and (wide[:, pad + C:] == 7).all())
            # backward in place of dy
            mean, rstd = r["mean"].float().contiguous(), r["rstd"].float().contiguous()
            dg, db = torch.empty(C, device="cuda"), torch.empty(C, device="cuda")
            d1, d2 = torch.empty_like(x), dy.clone()
            ops.group_norm_act_backward(dy, x, B, n, C, G, gamma, beta, mean, rstd, d1, dg, db, ws, act=ops.ACT_SILU)
            ops.group_norm_act_backward(d2, x, B, n, C, G, gamma, beta, mean, rstd, d2, dg, db, ws, act=ops.ACT_SILU)
            assert torch.equal(d1, d2)


def test_rows_beyond_32_bit_offsets(ops):
    """Row strides that put the last rows past 2^32 bytes and 2^31 elements."""
    n, C, G, ld = 70000, 32, 8, 1 << 15
    x, gamma, beta, _, _ = make(1, n, C, False, torch.bfloat16, seed=5)
    wide = torch.empty(n, ld, dtype=torch.bfloat16, device="cuda")
    wide[:, :C] = x
    out = torch.empty_like(x)
    ws = torch.empty(ops.group_norm_act_workspace_bytes(1, n, C, G), dtype=torch.uint8, device="cuda")
    ops.group_norm_act(wide[:, :C], 1, n, C, G, EPS, gamma, beta, out, ws, act=ops.ACT_SILU)
    want = torch.empty_like(x)
    ops.group_norm_act(x, 1, n, C, G, EPS, gamma, beta, want, ws, act=ops.ACT_SILU)
    assert torch.equal(out, want)


def test_gradient_against_differences(ops):
    """Directional differences of the forward kernel: with L = sum(y w) and u = dx / |dx| the slope along u is |dx|.  Central
    differences at step e are off by e^2 / 6 times the third derivative along u, at most (3 |dx| / spread)^2-ish of the
    slope: e = 2^-4 of a unit direction in n C = 6400 dimensions moves an element by ~8e-4 sigma, so truncation is below
    1e-5 of the slope; noise is sqrt(6400) roundings of y (6e-8 each) over 2 e |dx| ~ 8: < 1e-5.  Bound: 1e-3."""
    B, n, C, G = 2, 200, 16, 4
    x, gamma, beta, ss, w = make(B, n, C, True, torch.float32, seed=9)
    ws = torch.empty(ops.group_norm_act_workspace_bytes(B, n, C, G), dtype=torch.uint8, device="cuda")
    mean, rstd = torch.empty(B, G, device="cuda"), torch.empty(B, G, device="cuda")

    def loss(x, gamma, beta, ss):
        y = torch.empty_like(x)
        ops.group_norm_act(x, B, n, C, G, EPS, gamma, beta, y, ws, act=ops.ACT_SILU, scale_shift=ss, mean=mean, rstd=rstd)
        return float((y.double() * w.double()).sum())

    loss(x, gamma, beta, ss)
    dx, dg, db, dss = torch.empty_like(x), torch.empty(C, device="cuda"), torch.empty(C, device="cuda"), torch.empty(B, 2 * C, device="cuda")
    ops.group_norm_act_backward(w, x, B, n, C, G, gamma, beta, mean, rstd, dx, dg, db, ws, act=ops.ACT_SILU, scale_shift=ss,
                                dscale_shift=dss)
    args = [x, gamma, beta, ss]
    for i, d in enumerate((dx, dg, db, dss)):
        norm, e = float(d.norm()), 2.0 ** -4
        u = d / norm
        hi, lo = list(args), list(args)
        hi[i], lo[i] = args[i] + e * u, args[i] - e * u
        # the step actually taken (fp32 sums round it)
        step = float(((hi[i] - lo[i]).double() * u.double()).sum())
        slope = (loss(*hi) - loss(*lo)) / step
        assert abs(slope - norm) < 1e-3 * norm, (i, slope, norm)


def test_captured_and_replayed(ops):
    """A captured forward + backward replays to the eager results, also beside eager calls with a workspace of their own."""
    for n in (64, 9000):
        B, C, G = 2, 64, 32
        x, gamma, beta, ss, dy = make(B, n, C, True, torch.bfloat16, seed=n)
        nb = ops.group_norm_act_workspace_bytes(B, n, C, G)

        def buffers():
            e = lambda *s: torch.empty(*s, device="cuda")  # noqa: E731
            return dict(ws=torch.empty(nb, dtype=torch.uint8, device="cuda"), y=torch.empty_like(x), mean=e(B, G), rstd=e(B, G),
                        dx=torch.empty_like(x), dg=e(C), db=e(C), dss=e(B, 2 * C))

        def step(t):
            ops.group_norm_act(x, B, n, C, G, EPS, gamma, beta, t["y"], t["ws"], act=ops.ACT_SILU, scale_shift=ss, mean=t["mean"],
                               rstd=t["rstd"])
            ops.group_norm_act_backward(dy, x, B, n, C, G, gamma, beta, t["mean"], t["rstd"], t["dx"], t["dg"], t["db"], t["ws"],
                                        act=ops.ACT_SILU, scale_shift=ss, dscale_shift=t["dss"])

        eager, cap = buffers(), buffers()
        step(eager)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(cap)
        for i in range(4):
            x.copy_(torch.roll(x, 1, 0))
            for k in ("y", "dx", "dg", "db", "dss"):
                cap[k].fill_(float("nan"))
            graph.replay()
            step(eager)
            torch.cuda.synchronize()
            for k in ("y", "mean", "rstd", "dx", "dg", "db", "dss"):
                assert torch.equal(cap[k], eager[k]), (n, i, k)


def test_side_stream(ops):
    B, n, C, G = 2, 5000, 64, 8
    x, gamma, beta, _, _ = make(B, n, C, False, torch.float32)
    ws = torch.empty(ops.group_norm_act_workspace_bytes(B, n, C, G), dtype=torch.uint8, device="cuda")
    a, b = torch.empty_like(x), torch.empty_like(x)
    ops.group_norm_act(x, B, n, C, G, EPS, gamma, beta, a, ws)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        ops.group_norm_act(x, B, n, C, G, EPS, gamma, beta, b, ws)
    s.synchronize()
    assert torch.equal(a, b)
