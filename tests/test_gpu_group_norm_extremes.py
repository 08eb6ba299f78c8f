"""GPU: group_norm_act on values that leave the range of squares, on infinities and NaN, and on rows so many that one thread takes
thousands.  Tolerances are those of test_gpu_group_norm_act.py."""
import pytest
import torch

from tests.test_gpu_group_norm_act import EPS, HALF, U, close, make, ops, reference  # noqa: F401

pytestmark = pytest.mark.gpu


def forward(ops, x, gamma, beta, B, n, C, G, act=0, ss=None):
    y, mean, rstd = torch.full_like(x, float("nan")), torch.empty(B, G, device="cuda"), torch.empty(B, G, device="cuda")
    ws = torch.empty(ops.group_norm_act_workspace_bytes(B, n, C, G), dtype=torch.uint8, device="cuda")
    ops.group_norm_act(x, B, n, C, G, EPS, gamma, beta, y, ws, act=act, scale_shift=ss, mean=mean, rstd=rstd)
    return y, mean, rstd, ws


# one launch and two, one element a vector and many, one group wider than a block
SHAPES = [(1, 64, 64, 8), (2, 33, 15, 5), (2, 5000, 64, 8), (2, 3000, 30, 3), (1, 700, 2047, 1)]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("B,n,C,G", SHAPES)
def test_mean_whose_square_leaves_the_range(ops, B, n, C, G, dt):
    """Values of 3e19 (1 +- 1e-2): the mean's square is past fp32, the variance is not.  rstd: a thread's mean of up to 8 rows is a sum
    and a product in fp32, off by d <= 8 u |m|; the variance is that of the threads' means as they are held, plus the squares about
    them, so it is off by 2 cov(means, d) <= 2 sigma d: 16 u |m| / sigma of itself, rstd by half of that.  (|m| / sigma is 150
    here, not the 1 for which 8 u hold.)"""
    x, gamma, beta, _, _ = make(B, n, C, False, torch.float32, seed=n)
    x = (3e19 * (1 + 0.01 * torch.tanh(x))).to(dt)
    y, mean, rstd, _ = forward(ops, x, gamma, beta, B, n, C, G)
    r = reference(x, gamma, beta, None, B, n, C, G, False)
    close(y, r["y"], r["ty"], HALF[dt])
    close(mean, r["mean"], 4 * U * x.double().abs().max(), U)
    close(rstd, r["rstd"], 8 * U * r["rstd"] * (1 + r["mean"].abs() * r["rstd"]), U)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("B,n,C,G", SHAPES)
def test_a_diverged_group_shows(ops, B, n, C, G, dt, bad):
    """One infinity or NaN makes its own group NaN, statistics included, and leaves the others as they were."""
    x, gamma, beta, _, _ = make(B, n, C, False, dt, seed=n)
    want, wm, wr, _ = forward(ops, x, gamma, beta, B, n, C, G)
    hit = x.clone()
    hit[n - 1, C - 1] = bad     # the last group of the first image
    y, mean, rstd, _ = forward(ops, hit, gamma, beta, B, n, C, G)
    assert bool(torch.isnan(rstd[0, -1])) and not bool(torch.isfinite(mean[0, -1]))
    group = torch.zeros(B * n, C, dtype=torch.bool, device="cuda")
    group[:n, C - C // G:] = True
    assert bool(torch.isnan(y[group]).all()) and torch.equal(y[~group], want[~group])
    stats = torch.zeros(B, G, dtype=torch.bool, device="cuda")
    stats[0, -1] = True
    assert torch.equal(mean[~stats], wm[~stats]) and torch.equal(rstd[~stats], wr[~stats])


def test_statistics_of_many_rows_a_thread(ops):
    """256 images of 1024 rows, one group of 2048: a thread walks a thousand rows of ones, the second half 2^-17 larger.  Added row by
    row, each of those small steps is below half a step of the mean in fp32, and the mean would stay where it was."""
    B, n, C = 256, 1024, 2048
    x = torch.ones(B, n, C, device="cuda")
    x[:, n // 2:] += 2.0 ** -17
    one, zero = torch.ones(C, device="cuda"), torch.zeros(C, device="cuda")
    y, mean, _, _ = forward(ops, x.view(B * n, C), one, zero, B, n, C, 1)
    assert float((mean.double() - (1 + 2.0 ** -18)).abs().max()) <= 4 * U
    r = (2.0 ** -36 + EPS) ** -0.5
    want = 2.0 ** -18 * r
    # the file's 16 u (|m a| + |(x - m) a|) with a = r
    tol = 16 * U * (r + want) + U * want
    y = y.view(B, n, C)
    assert float((y[:, :n // 2] + want).abs().max()) <= tol and float((y[:, n // 2:] - want).abs().max()) <= tol


def test_gradients_of_many_rows_a_thread(ops):
    """256 images of 2048 rows, one group of 2048 channels, dy = 1 + 230 2^-23 everywhere: past 1024, a running fp32 sum of pairs
    loses 0.45 of a step at every addition.  S1 and S2 within the tolerance of 64 merged batches: 64 u, and the store's."""
    B, n, C = 256, 2048, 2048
    d = 1 + 230 * 2.0 ** -23
    x, dy = torch.ones(B * n, C, device="cuda"), torch.full((B * n, C), d, device="cuda")
    one, zero = torch.ones(C, device="cuda"), torch.zeros(C, device="cuda")
    ss, dss = torch.zeros(B, 2 * C, device="cuda"), torch.empty(B, 2 * C, device="cuda")
    mean, rstd = torch.zeros(B, 1, device="cuda"), torch.ones(B, 1, device="cuda")
    dg, db = torch.empty(C, device="cuda"), torch.empty(C, device="cuda")
    ws = torch.empty(ops.group_norm_act_workspace_bytes(B, n, C, 1), dtype=torch.uint8, device="cuda")
    ops.group_norm_act_backward(dy, x, B, n, C, 1, one, zero, mean, rstd, dy, dg, db, ws, scale_shift=ss, dscale_shift=dss)
    for got, want in ((dss, n * d), (dg, B * n * d), (db, B * n * d)):
        assert float((got.double() - want).abs().max()) <= 66 * U * want


# so many images that a block has all rows of one: several runs of 128 rows a thread, the last ones ragged; one group wider than a block,
# vectors of 16 bytes and the most LDS, several groups a slab
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("B,n,C,G", [(256, 300, 2047, 1), (257, 601, 2048, 1), (256, 400, 1024, 2), (256, 70001, 24, 3), (256, 33100, 32, 8)])
def test_runs_of_rows(ops, B, n, C, G, dt):
    """y has one tolerance more than test_gpu_group_norm_act.py's: s = beta (1 + scale) + shift with 1 + scale rounded to fp32 is off by
    u |beta (1 + scale)|, however small s is where the two parts cancel (half a million channels and images have some that do), and
    |act'| <= 1.1 takes that to y."""
    x, gamma, beta, ss, dy = make(B, n, C, True, dt, seed=n)
    y, mean, rstd, ws = forward(ops, x, gamma, beta, B, n, C, G, act=ops.ACT_SILU, ss=ss)
    dx, dg, db, dss = torch.empty_like(x), torch.empty(C, device="cuda"), torch.empty(C, device="cuda"), torch.empty(B, 2 * C, device="cuda")
    ops.group_norm_act_backward(dy, x, B, n, C, G, gamma, beta, mean, rstd, dx, dg, db, ws, act=ops.ACT_SILU, scale_shift=ss,
                                dscale_shift=dss)
    sums = dict(dgamma=0, tdgamma=0, dbeta=0, tdbeta=0)
    for b in range(B):
        rows = slice(b * n, (b + 1) * n)
        r = reference(x[rows], gamma, beta, ss[b:b + 1], 1, n, C, G, True, dy=dy[rows])
        sums = {k: v + r[k] for k, v in sums.items()}
        if b % 51 and b != B - 1:
            continue
        close(y[rows], r["y"], r["ty"] + 1.1 * U * (beta * (1 + ss[b, :C])).double().abs(), HALF[dt])
        close(mean[b:b + 1], r["mean"], 4 * U * x[rows].double().abs().max(), U)
        close(rstd[b:b + 1], r["rstd"], 8 * U * r["rstd"], U)
        close(dx[rows], r["dx"], r["tdx"], HALF[dt])
        close(dss[b:b + 1], r["dss"], r["tdss"], 4 * U)
    close(dg, sums["dgamma"], sums["tdgamma"], 4 * U)
    close(db, sums["dbeta"], sums["tdbeta"], 4 * U)
