"""Layer norm and its backward pass against the formulas in float64.

Tolerances.  u = 2^-24.  A sum over a row is a chain of at most D - 12
additions in a thread and 10 in two warps' trees, so it is off by at most
D u times the sum of the magnitudes.  Forward: the mean is off by
D u mean|x|, the variance by (D + 4) u relative (a shifted mean changes it in
second order only), rstd by half of that, and the rest are four roundings:
  |y - y*| <= u (|gamma| (rstd D mean|x| + (D + 8) |xhat|) + 2 |y|).
Backward (mean and rstd are inputs): xhat is off by 2 u, v = dy gamma by u,
and the two row sums by D u of their magnitudes, giving
  |dx - dx*| <= u rstd (8 |v| + (D + 4) (mean|v| + |xhat| mean|v xhat|)).
A column sum over R rows is a chain of at most R / 148 + 96 additions.
"""
import pytest

from minixla_b200 import lib as mlib
from tests.operator_calls import U, captured, current_stream, fake_context, ok, pitched, ptr, within

D = 64
EPS = 1e-5


def forward(lib, ctx, x, gamma, beta, y=None, stats=True, eps=EPS, stream=None):
    import torch

    rows, cols = x.shape
    y = torch.empty(rows, cols, device="cuda") if y is None else y
    mean, rstd = (torch.empty(rows, device="cuda") for _ in range(2)) if stats else (None, None)
    ok(lib.mxb_layer_norm(ctx, ptr(x), x.stride(0), ptr(gamma), ptr(beta), eps, ptr(y), y.stride(0), ptr(mean),
                          ptr(rstd), rows, cols, stream or current_stream()))
    return y, mean, rstd


def backward(lib, ctx, dy, x, gamma, mean, rstd, dx=None, dgamma=True, dbeta=True, want_dx=True, stream=None):
    import torch

    rows, cols = x.shape
    if want_dx and dx is None:
        dx = torch.empty(rows, cols, device="cuda")
    dgamma, dbeta = (torch.full((cols,), float("nan"), device="cuda") if w else None for w in (dgamma, dbeta))
    ok(lib.mxb_layer_norm_backward(ctx, ptr(dy), dy.stride(0), ptr(x), x.stride(0), ptr(gamma), ptr(mean), ptr(rstd),
                                   ptr(dx), dx.stride(0) if dx is not None else 0, ptr(dgamma), ptr(dbeta), rows, cols,
                                   stream or current_stream()))
    return dx, dgamma, dbeta


def make(rows, cols, seed=0, offset=0.5):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, cols, device="cuda", generator=g) * 2 + offset
    dy = torch.randn(rows, cols, device="cuda", generator=g)
    gamma = 1 + 0.3 * torch.randn(cols, device="cuda", generator=g)
    beta = torch.randn(cols, device="cuda", generator=g)
    return x, dy, gamma, beta


def check_forward(x, gamma, beta, y, mean, rstd, eps=EPS):
    xd = x.double()
    m = xd.mean(1, keepdim=True)
    var = (xd - m).square().mean(1, keepdim=True)
    r = (var + eps).rsqrt()
    xh = (xd - m) * r
    g = gamma.double() if gamma is not None else 1.0
    want = xh * g + (beta.double() if beta is not None else 0.0)
    mag = xd.abs().mean(1, keepdim=True)
    gabs = gamma.double().abs() if gamma is not None else 1.0
    within(y, want, U * (gabs * (r * D * mag + (D + 8) * xh.abs()) + 2 * want.abs()), "y")
    if mean is not None:
        within(mean, m[:, 0], U * D * mag[:, 0], "mean")
        within(rstd, r[:, 0], U * (D + 8) * r[:, 0], "rstd")


def check_backward(dy, x, gamma, mean, rstd, dx, dgamma, dbeta):
    xh = (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
    r = rstd.double()[:, None]
    d = dy.double()
    v = d * gamma.double() if gamma is not None else d
    vx = v * xh
    if dx is not None:
        want = r * (v - v.mean(1, keepdim=True) - xh * vx.mean(1, keepdim=True))
        tol = U * r * (8 * v.abs() + (D + 4) * (v.abs().mean(1, keepdim=True)
                                                + xh.abs() * vx.abs().mean(1, keepdim=True)))
        within(dx, want, tol, "dx")
    chain = x.shape[0] / 148 + 96
    if dgamma is not None:
        within(dgamma, (d * xh).sum(0), U * (chain + 4) * (d * xh).abs().sum(0), "dgamma")
    if dbeta is not None:
        within(dbeta, d.sum(0), U * chain * d.abs().sum(0), "dbeta")


# Widths around the warp / block / long-row borders, odd ones among them.
SHAPES = [(1, 1), (3, 2), (1, 4096), (7, 31), (300, 33), (2000, 127), (401, 128), (4097, 256), (513, 512), (700, 516),
          (333, 1024), (1200, 1027), (600, 2048), (311, 4100), (500, 8192), (310, 8196), (320, 12001), (5, 16384),
          (330, 16384), (3, 32768), (2, 32772), (3, 40001), (301, 40000)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward_and_backward(lib, gpu_ctx, rows, cols):
    x, dy, gamma, beta = make(rows, cols, rows + cols)
    y, mean, rstd = forward(lib, gpu_ctx, x, gamma, beta)
    check_forward(x, gamma, beta, y, mean, rstd)
    check_backward(dy, x, gamma, mean, rstd, *backward(lib, gpu_ctx, dy, x, gamma, mean, rstd))


# Rows for which every block of the ring kernels refills each slot at least once: a block of t threads has at most
# 2048 / t neighbours on one of 148 SMs, and a ring at most eight slots.
@pytest.mark.gpu
@pytest.mark.parametrize("cols,threads", [(1027, 64), (1028, 64), (2051, 128), (2052, 128), (4099, 256), (4100, 256),
                                          (8191, 512), (8192, 512)])
def test_ring_refills_its_slots(lib, gpu_ctx, cols, threads):
    """Widths of a block's rows, odd ones (a refilled slot then has another skip) and multiples of four."""
    rows = 2 * 8 * 148 * (2048 // threads) + 5
    x, dy, gamma, beta = make(rows, cols, cols)
    y, mean, rstd = forward(lib, gpu_ctx, x, gamma, beta)
    got = backward(lib, gpu_ctx, dy, x, gamma, mean, rstd)
    part = 4096
    for r in range(0, rows, part):
        s = slice(r, min(rows, r + part))
        check_forward(x[s], gamma, beta, y[s], mean[s], rstd[s])
        check_backward(dy[s], x[s], gamma, mean[s], rstd[s], got[0][s], None, None)
    check_backward(dy, x, gamma, mean, rstd, None, *got[1:])
    assert lib.mxb_check_device_error(gpu_ctx) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("cols,pitch", [(96, 100), (96, 97), (1023, 1024), (1030, 1031), (5000, 5004)])
def test_pitches_and_unaligned_bases(lib, gpu_ctx, cols, pitch):
    import torch

    x, dy, gamma, beta = make(37, cols, cols)
    xp, dyp = pitched(x, pitch), pitched(dy, pitch)
    yp = pitched(torch.zeros_like(x), pitch, 7.0)
    _, mean, rstd = forward(lib, gpu_ctx, xp, gamma, beta, y=yp)
    check_forward(x, gamma, beta, yp, mean, rstd)
    full = yp.as_strided((37, pitch), (pitch, 1))
    assert (full[:, cols:] == 7.0).all(), "the gap between rows was written"
    dxp = pitched(torch.zeros_like(x), pitch, 7.0)
    check_backward(dy, x, gamma, mean, rstd, *backward(lib, gpu_ctx, dyp, xp, gamma, mean, rstd, dx=dxp))
    assert (dxp.as_strided((37, pitch), (pitch, 1))[:, cols:] == 7.0).all()
    # Bases off by one float.
    xo = torch.empty(37 * cols + 1, device="cuda")[1:].view(37, cols).copy_(x)
    go = torch.empty(cols + 1, device="cuda")[1:].copy_(gamma)
    y, mean, rstd = forward(lib, gpu_ctx, xo, go, beta)
    check_forward(x, gamma, beta, y, mean, rstd)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [64, 516, 4096, 40000])
def test_optional_parts_and_in_place(lib, gpu_ctx, cols):
    x, dy, gamma, beta = make(50, cols, 3)
    y, _, _ = forward(lib, gpu_ctx, x, None, None, stats=False)
    check_forward(x, None, None, y, None, None)
    want, mean, rstd = forward(lib, gpu_ctx, x, gamma, beta)
    xi = x.clone()
    got, _, _ = forward(lib, gpu_ctx, xi, gamma, beta, y=xi)
    assert (got == want).all()
    full = backward(lib, gpu_ctx, dy, x, gamma, mean, rstd)
    for kw in (dict(dgamma=False), dict(dbeta=False), dict(want_dx=False), dict(dgamma=False, dbeta=False)):
        part = backward(lib, gpu_ctx, dy, x, gamma, mean, rstd, **kw)
        for a, b in zip(part, full):
            assert a is None or (a == b).all(), kw
    check_backward(dy, x, None, mean, rstd, *backward(lib, gpu_ctx, dy, x, None, mean, rstd))
    for which in ("dy", "x"):
        d, xx = dy.clone(), x.clone()
        got = backward(lib, gpu_ctx, d, xx, gamma, mean, rstd, dx=d if which == "dy" else xx)
        assert all((a == b).all() for a, b in zip(got, full)), which


@pytest.mark.gpu
def test_constant_rows_and_far_offsets(lib, gpu_ctx):
    import torch

    # A constant row has variance 0 (exactly: the mean of equal values in
    # powers of two is exact), so y = beta; an offset of 1000 spreads costs
    # what the bound says and no more.
    x = torch.full((4, 1024), 0.75, device="cuda")
    _, _, gamma, beta = make(4, 1024)
    y, mean, rstd = forward(lib, gpu_ctx, x, gamma, beta)
    assert (y == beta).all() and (mean == 0.75).all()
    for cols in (1024, 4096):
        x, _, gamma, beta = make(200, cols, 1, offset=2000.0)
        check_forward(x, gamma, beta, *forward(lib, gpu_ctx, x, gamma, beta))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(3, 5), (900, 30), (900, 129), (400, 1030), (400, 1027), (2, 515), (400, 12001),
                                       (400, 12002), (3, 40001), (3, 40002)])
def test_mean_far_past_the_spread(lib, gpu_ctx, rows, cols):
    """Rows of one value 1e37: xhat is 0 and dx what is left of dy, though mean times rstd is past fp32's range."""
    import torch

    _, dy, gamma, _ = make(rows, cols, cols)
    x = torch.full((rows, cols), 2.0 ** 123, device="cuda")
    mean, rstd = x[:, 0].contiguous(), torch.full((rows,), 316.0, device="cuda")
    pitch = (cols + 3) // 4 * 4
    for p in (cols, pitch):
        check_backward(dy, x, gamma, mean, rstd, *backward(lib, gpu_ctx, pitched(dy, p), pitched(x, p), gamma, mean, rstd,
                                                           dx=pitched(torch.zeros_like(x), p)))


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [200, 3000, 40000])
def test_bad_values_stay_in_their_row(lib, gpu_ctx, cols):
    import torch

    x, dy, gamma, beta = make(40, cols, 5)
    y0, mean, rstd = forward(lib, gpu_ctx, x, gamma, beta)
    dx0, _, _ = backward(lib, gpu_ctx, dy, x, gamma, mean, rstd)
    bad = x.clone()
    bad[7, 3], bad[9, 0] = float("nan"), float("inf")
    y, mean2, rstd2 = forward(lib, gpu_ctx, bad, gamma, beta)
    dx, _, _ = backward(lib, gpu_ctx, dy, bad, gamma, mean2, rstd2)
    keep = torch.ones(40, dtype=torch.bool, device="cuda")
    keep[7] = keep[9] = False
    assert (y[keep] == y0[keep]).all() and (dx[keep] == dx0[keep]).all()
    assert torch.isnan(y[7]).all() and torch.isnan(dx[7]).all()


@pytest.mark.gpu
def test_no_rows(lib, gpu_ctx):
    import torch

    x = torch.empty(0, 100, device="cuda")
    ok(lib.mxb_layer_norm(gpu_ctx, None, 100, None, None, EPS, None, 100, None, None, 0, 100, current_stream()))
    dg, db = torch.ones(2, 100, device="cuda")
    ok(lib.mxb_layer_norm_backward(gpu_ctx, None, 100, None, 100, None, None, None, None, 100, ptr(dg), ptr(db), 0,
                                   100, current_stream()))
    torch.cuda.synchronize()
    assert (dg == 0).all() and (db == 0).all() and x.numel() == 0


@pytest.mark.gpu
def test_gradient_against_differences(lib, gpu_ctx):
    """Central differences of sum(w * y) in float64 along random directions.
    The difference is off by h^2 / 6 of the third derivative (below 1e-3 for
    h = 1e-4, rstd <= 1, unit directions) plus the kernel's own bound."""
    import torch

    x, w, gamma, beta = make(6, 700, 11)
    _, mean, rstd = forward(lib, gpu_ctx, x, gamma, beta)
    dx, dgamma, dbeta = backward(lib, gpu_ctx, w, x, gamma, mean, rstd)

    def loss(x, gamma, beta):
        m = x.mean(1, keepdim=True)
        r = ((x - m).square().mean(1, keepdim=True) + EPS).rsqrt()
        return (w.double() * ((x - m) * r * gamma + beta)).sum().item()

    args = [x.double(), gamma.double(), beta.double()]
    gen = torch.Generator(device="cuda").manual_seed(1)
    h = 1e-4
    for i, grad in enumerate((dx, dgamma, dbeta)):
        d = torch.randn(args[i].shape, device="cuda", generator=gen, dtype=torch.float64)
        d /= d.norm()
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + h * d, args[i] - h * d
        diff = (loss(*up) - loss(*down)) / (2 * h)
        got = (grad.double() * d).sum().item()
        assert abs(diff - got) <= 1e-6 + 1e-5 * grad.double().norm().item(), (i, diff, got)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [96, 2000])
def test_captured_beside_eager_calls(lib, gpu_ctx, cols):
    """Two graphs and eager calls in between keep their partial sums apart."""
    import torch

    x, dy, gamma, beta = make(900, cols, 21)
    x2, dy2, _, _ = make(900, cols, 22)
    _, mean, rstd = forward(lib, gpu_ctx, x, gamma, beta)
    _, mean2, rstd2 = forward(lib, gpu_ctx, x2, gamma, beta)
    want = backward(lib, gpu_ctx, dy, x, gamma, mean, rstd)
    want2 = backward(lib, gpu_ctx, dy2, x2, gamma, mean2, rstd2)
    got, got2 = {}, {}
    ga = captured(lambda: got.update(r=backward(lib, gpu_ctx, dy, x, gamma, mean, rstd)))
    gb = captured(lambda: got2.update(r=backward(lib, gpu_ctx, dy2, x2, gamma, mean2, rstd2)))
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(sa):
            ga.replay()
        with torch.cuda.stream(sb):
            gb.replay()
        eager = backward(lib, gpu_ctx, dy, x, gamma, mean, rstd)
    torch.cuda.synchronize()
    for a, b, c in zip(got["r"], want, eager):
        assert (a == b).all() and (c == b).all()
    assert all((a == b).all() for a, b in zip(got2["r"], want2))


@pytest.mark.gpu
def test_streams_and_the_contexts_own(lib, gpu_ctx):
    import torch

    x, dy, gamma, beta = make(500, 1000, 31)
    want, mean, rstd = forward(lib, gpu_ctx, x, gamma, beta)
    full = backward(lib, gpu_ctx, dy, x, gamma, mean, rstd)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(backward(lib, gpu_ctx, dy, x, gamma, mean, rstd))
    y = torch.empty_like(x)
    torch.cuda.synchronize()
    ok(lib.mxb_layer_norm(gpu_ctx, ptr(x), 1000, ptr(gamma), ptr(beta), EPS, ptr(y), 1000, None, None, 500, 1000, None))
    assert lib.mxb_check_device_error(gpu_ctx) == 0
    assert (y == want).all()
    for g in got:
        assert all((a == b).all() for a, b in zip(g, full))


@pytest.mark.gpu
def test_rows_at_the_ends_of_an_allocation(lib, gpu_ctx):
    """The copies of unaligned rows reach past a row's ends, never past the matrix's: with NaN right before and behind
    it, and rows of every alignment, nothing changes."""
    import torch

    for cols in (1029, 2050, 4099):
        x, dy, gamma, beta = make(9, cols, cols)
        buf = torch.full((3, 9 * cols + 8), float("nan"), device="cuda")
        xv, dv = (buf[i][4:4 + 9 * cols].view(9, cols).copy_(t) for i, t in ((0, x), (1, dy)))
        y, mean, rstd = forward(lib, gpu_ctx, xv, gamma, beta)
        check_forward(x, gamma, beta, y, mean, rstd)
        check_backward(dy, x, gamma, mean, rstd, *backward(lib, gpu_ctx, dv, xv, gamma, mean, rstd))


def test_columns_past_the_limit(lib):
    n = (1 << 30) + 4
    assert lib.mxb_layer_norm(fake_context(), 4096, n, None, None, EPS, 8192, n, None, None, 1, n, None) == mlib.MXB_E_UNSUPPORTED
    assert lib.mxb_layer_norm_backward(fake_context(), 4096, n, 8192, n, None, 64, 64, 16384, n, None, None, 1, n,
                                       None) == mlib.MXB_E_UNSUPPORTED
    assert "2^30" in mlib.last_error()


REFUSED = [
    dict(ctx=None), dict(x=None), dict(y=None), dict(cols=0), dict(rows=-1), dict(ldx=15), dict(ldy=15),
    dict(y="x", ldy=20),
]


@pytest.mark.parametrize("change", REFUSED, ids=str)
def test_forward_refusals(lib, change):
    a = dict(ctx=fake_context(), x=4096, ldx=16, gamma=None, beta=None, eps=EPS, y=8192, ldy=16, mean=None, rstd=None,
             rows=2, cols=16, stream=None)
    a.update(change)
    if a["y"] == "x":
        a["y"] = a["x"]
    assert lib.mxb_layer_norm(*a.values()) == mlib.MXB_E_ARG
    assert "mxb_layer_norm" in mlib.last_error()


REFUSED_BACKWARD = [
    dict(ctx=None), dict(dy=None), dict(x=None), dict(mean=None), dict(rstd=None), dict(cols=0), dict(rows=-1),
    dict(ldx=15), dict(lddy=15), dict(lddx=15), dict(dx=None, dgamma=None, dbeta=None), dict(dx="dy", lddx=20),
    dict(dx="x", lddx=20),
]


@pytest.mark.parametrize("change", REFUSED_BACKWARD, ids=str)
def test_backward_refusals(lib, change):
    a = dict(ctx=fake_context(), dy=4096, lddy=16, x=8192, ldx=16, gamma=None, mean=12288, rstd=16384, dx=20480,
             lddx=16, dgamma=24576, dbeta=28672, rows=2, cols=16, stream=None)
    a.update(change)
    if isinstance(a["dx"], str):
        a["dx"] = a[a["dx"]]
    assert lib.mxb_layer_norm_backward(*a.values()) == mlib.MXB_E_ARG
    assert "mxb_layer_norm_backward" in mlib.last_error()
