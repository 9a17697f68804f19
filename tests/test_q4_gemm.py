"""Products with 4-bit weights against the definition in float64.

Tolerance.  An activation enters as three bf16 parts whose sum is exact, q - z
is exact in bf16, and a group's sum is accumulated by matrix instructions that
may cut each partial sum to 23 bits: with three parts and 16 values to an
instruction, at most 24 cuts in 128 values, each below 2^-23 of the sum of
magnitudes S = sum |a| |w|.  The scale and the sum over the groups (or over
runs of 128 values) add ceil(K / 32) roundings of u = 2^-24 at most, and the
steps a few: |out - out*| <= (24 * 2^-23 + (K / 32 + 16) * 2^-24) S + 4 u |out|.
"""
import pytest

from minixla_b200 import lib as mlib
from tests.operator_calls import U, captured, current_stream, fake_context, ok, pitched, ptr, steps, within


def make(m, n, k, group, scale="f32", zeros=True, seed=0, lda=None, ldq=None, lds=None):
    import torch

    dt = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[scale]
    g = torch.Generator(device="cuda").manual_seed(seed)
    kg = -(-k // group)
    a = torch.randn(m, k, device="cuda", generator=g)
    a = pitched(a, lda or (k + 3) // 4 * 4)
    q = torch.randint(0, 256, (n, ldq or ((k + 1) // 2 + 15) // 16 * 16), dtype=torch.uint8, device="cuda", generator=g)
    s = ((torch.rand(n, kg, device="cuda", generator=g) + 0.5) * 0.1).to(dt)
    z = torch.randint(0, 16, (n, kg), dtype=torch.uint8, device="cuda", generator=g)
    if lds:
        s = pitched(s, lds)
        z = pitched(z, lds, 255)
    return dict(a=a, q=q, s=s, z=z if zeros else None, group=group, m=m, n=n, k=k, scale=scale)


def weight(c):
    """W [K, N] in float64."""
    import torch

    q = torch.stack((c["q"] & 15, c["q"] >> 4), 2).flatten(1)[:, : c["k"]].double()
    col = torch.arange(c["k"], device="cuda") // c["group"]
    z = c["z"].double()[:, col] if c["z"] is not None else 8.0
    return ((q - z) * c["s"].double()[:, col]).t()


def run(lib, ctx, c, st=None, out=None, stream=None):
    import torch

    out = torch.full((c["m"], c["n"]), float("nan"), device="cuda") if out is None else out
    arr, cnt = st or steps()
    kind = {"f32": mlib.MXB_SCALE_F32, "f16": mlib.MXB_SCALE_F16, "bf16": mlib.MXB_SCALE_BF16}[c["scale"]]
    ok(lib.mxb_q4_gemm(ctx, ptr(c["a"]), c["a"].stride(0), ptr(c["q"]), c["q"].stride(0), ptr(c["s"]), kind, ptr(c["z"]),
                       c["s"].stride(0), c["group"], ptr(out), out.stride(0), c["m"], c["n"], c["k"], arr, cnt,
                       stream or current_stream()))
    return out


def check(c, out, post=lambda y: y):
    w = weight(c)
    a = c["a"].double()
    want = post(a @ w)
    mag = a.abs() @ w.abs()
    tol = (24 * 2.0 ** -23 + (c["k"] / 32 + 16) * U) * mag + 4 * U * want.abs()
    within(out, want, tol, str((c["m"], c["n"], c["k"], c["group"])))


SHAPES = [(1, 1, 1, 32), (1, 1, 2, 32), (2, 7, 31, 32), (3, 16, 33, 32), (1, 129, 100, 64), (4, 63, 4095, 128),
          (5, 200, 128, 128), (6, 31, 1000, 96), (7, 257, 513, 256), (8, 512, 512, 64), (9, 65, 300, 512),
          (11, 40, 2049, 128), (13, 33, 96, 32), (16, 1000, 1000, 128), (17, 300, 700, 32), (31, 128, 256, 64),
          (64, 130, 1024, 128), (100, 257, 1031, 96), (129, 1000, 320, 64), (300, 515, 2050, 128), (1, 4096, 8192, 128),
          (700, 384, 4096, 4096), (257, 129, 64, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,group", SHAPES)
def test_against_definition(lib, gpu_ctx, m, n, k, group):
    for i, scale in enumerate(("f32", "f16", "bf16")):
        for zeros in (False, True):
            c = make(m, n, k, group, scale, zeros, seed=m + n + k + i)
            check(c, run(lib, gpu_ctx, c))


# Weights wide enough for the wider tiles of the few-row kernel (32 columns a warp tile from 24 columns an SM, 64 for more than
# eight rows from 32) and long enough that each warp's ring goes round more than once; widths that end inside a tile.
WIDE = [(1, 3555, 8200, 128), (1, 5000, 8200, 96), (2, 4100, 8200, 128), (2, 4100, 8200, 32), (2, 1000, 16500, 64),
        (4, 3601, 4200, 256), (8, 4097, 8192, 32), (8, 4097, 8192, 128), (12, 3600, 4200, 64), (12, 3600, 4200, 128),
        (9, 4800, 2049, 32), (16, 5000, 8200, 32), (16, 5000, 8200, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,group", WIDE)
def test_wide_weights_for_few_rows(lib, gpu_ctx, m, n, k, group):
    for scale, zeros in (("f32", True), ("f16", False), ("bf16", True)):
        c = make(m, n, k, group, scale, zeros, seed=m + n + k)
        check(c, run(lib, gpu_ctx, c))
    assert lib.mxb_check_device_error(gpu_ctx) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(1, 4000), (2, 150), (2, 4000), (8, 4000), (13, 4000), (16, 5000)])
def test_wide_weights_exactly(lib, gpu_ctx, m, n):
    """Integer activations of very different sizes in the rows, scales of one: every sum is exact."""
    import torch

    k = 3000
    c = make(m, n, k, 96 if n == 150 else 128, seed=m)
    big = 2.0 ** (torch.arange(m, device="cuda") % 5 * 20 - 40)
    c["a"] = torch.randint(-9, 10, (m, k), device="cuda").float() * big[:, None]
    c["s"].fill_(1.0)
    assert (run(lib, gpu_ctx, c).double() == c["a"].double() @ weight(c)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 2])
@pytest.mark.parametrize("size", [1e-20, 1e-3, 1e20])
def test_large_and_tiny_activations_of_one_or_two_rows(lib, gpu_ctx, m, size):
    c = make(m, 4000, 3000, 128, seed=m)
    c["a"] = c["a"] * size
    check(c, run(lib, gpu_ctx, c))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 3, 8, 16, 40, 200])
def test_exact_small_integers(lib, gpu_ctx, m):
    """Integer activations and scales of one: every sum is exact, whatever its order."""
    import torch

    c = make(m, 150, 777, 96, seed=m)
    c["a"] = pitched(torch.randint(-9, 10, (m, 777), device="cuda").float(), 780)
    c["s"].fill_(1.0)
    assert (run(lib, gpu_ctx, c).double() == c["a"].double() @ weight(c)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 6, 16, 33, 150])
def test_pitches_steps_and_gaps(lib, gpu_ctx, m):
    import torch

    n, k = 203, 330
    c = make(m, n, k, 64, "bf16", True, seed=m, lda=352, ldq=192, lds=9)
    out = pitched(torch.zeros(m, n, device="cuda"), 211, 5.0)
    add = pitched(torch.randn(m, n, device="cuda"), 207)
    row, mod = torch.randn(n, device="cuda"), torch.randn(n * 3 + 1, device="cuda")
    st = steps((mlib.MXB_EP_ADD_ROW, row, 0, 0), (mlib.MXB_EP_ADD_FULL, add, 207, 0), (mlib.MXB_EP_RELU, None, 0, 0),
               (mlib.MXB_EP_SCALE, None, 0, 1.5), (mlib.MXB_EP_ADD_MOD, mod, mod.numel(), 0))
    run(lib, gpu_ctx, c, st, out)
    idx = torch.arange(m * n, device="cuda").view(m, n) % mod.numel()
    # The steps after the sum see its error times 1.5 and round five times more.
    w, a = weight(c), c["a"].double()
    pre = a @ w
    want = ((pre + row.double() + add.double()).clamp(min=0) * 1.5) + mod.double()[idx]
    tol = 1.5 * (24 * 2.0 ** -23 + (k / 32 + 16) * U) * (a.abs() @ w.abs()) + 8 * U * (
        pre.abs() + row.double().abs() + add.double().abs() + mod.double()[idx].abs()) * 1.5
    within(out, want, tol)
    assert (out.as_strided((m, 211), (211, 1))[:, n:] == 5.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 8, 16, 64, 300])
def test_large_and_tiny_activations(lib, gpu_ctx, m):
    """Magnitudes from 1e-20 to 1e20 keep the same relative bound; a row of zeros gives zeros."""
    import torch

    c = make(m, 96, 512, 128, seed=m)
    c["a"] = c["a"] * (10.0 ** torch.linspace(-20, 20, m, device="cuda"))[:, None]
    c["a"][m // 2] = 0
    out = run(lib, gpu_ctx, c)
    check(c, out)
    assert (out[m // 2] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [2, 16, 40, 200])
def test_bad_rows_stay_alone(lib, gpu_ctx, m):
    import torch

    c = make(m, 70, 200, 32, seed=m)
    good = run(lib, gpu_ctx, c)
    c["a"][0, 5] = float("nan")
    out = run(lib, gpu_ctx, c)
    assert torch.isnan(out[0]).all() and (out[1:] == good[1:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n,k,group", [(70, 200, 32), (5000, 700, 128), (4100, 8200, 32)])
@pytest.mark.parametrize("m", [1, 2, 3, 8, 16, 40, 200])
def test_infinite_activations(lib, gpu_ctx, m, n, k, group):
    """An infinity gives what fp32 gives: infinity with its weight's sign, NaN against a weight of zero or against another
    infinity of the other sign; the relu that follows keeps the positive ones.  NaN stays NaN whatever its payload."""
    import torch

    c = make(m, n, k, group, seed=m)
    good = run(lib, gpu_ctx, c)
    inf = float("inf")
    c["a"][0, 5] = inf
    if m > 2:
        c["a"][2, k - 1], c["a"][2, 40] = -inf, inf
    if m > 7:
        c["a"][6, 7] = torch.tensor([0x7F800001], dtype=torch.int32, device="cuda").view(torch.float32)[0]  # NaN
    out = run(lib, gpu_ctx, c)
    want = c["a"].double() @ weight(c)
    bad = ~torch.isfinite(want)
    assert bad[0].all() and (torch.isinf(want[0]).any() and torch.isnan(want[0]).any())
    assert torch.equal(out[bad].nan_to_num(7.0), want[bad].float().nan_to_num(7.0))
    assert torch.equal(out[~bad], good[~bad])
    relu = run(lib, gpu_ctx, c, steps((mlib.MXB_EP_RELU, None, 0, 0)))
    assert torch.equal(relu, torch.where(out > 0, out, 0.0))
    assert torch.isinf(relu[0]).any()
    # Added to the output itself: once, though some sums are made a second time.
    added = torch.ones_like(out)
    run(lib, gpu_ctx, c, steps((mlib.MXB_EP_ADD_FULL, added, n, 0)), added)
    assert torch.equal(added.nan_to_num(7.0), (out + 1).nan_to_num(7.0))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 2, 5, 16, 40, 300])
@pytest.mark.parametrize("k", [1, 33, 500])
def test_columns_of_a_wider_weight(lib, gpu_ctx, m, k):
    """The last columns of K of a wider matrix, whose last row ends where the memory does: the copies read K columns of
    a row, not its pitch."""
    import torch

    c = make(m, 100, k, 32, seed=m + k)
    keep = -(-k // 32) * 16
    wide = torch.randint(0, 256, (100, 512 + keep), dtype=torch.uint8, device="cuda")
    wide[:, 512:512 + (k + 1) // 2] = c["q"][:, :(k + 1) // 2]
    assert torch.equal(run(lib, gpu_ctx, dict(c, q=wide[:, 512:])), run(lib, gpu_ctx, c))


@pytest.mark.gpu
def test_rows_do_not_depend_on_their_number(lib, gpu_ctx):
    """Every row of a larger product is within the bound of the same row alone."""
    c = make(40, 333, 1000, 128, seed=3)
    whole = run(lib, gpu_ctx, c)
    check(c, whole)
    for m in (1, 2, 5, 16):
        part = dict(c, a=c["a"][:m], m=m)
        check(part, run(lib, gpu_ctx, part))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 16, 300])
def test_captured_and_on_other_streams(lib, gpu_ctx, m):
    import torch

    c = make(m, 500, 1000, 128, seed=9)
    want = run(lib, gpu_ctx, c)
    got = {}
    g1 = captured(lambda: got.update(a=run(lib, gpu_ctx, c)))
    c2 = make(m, 500, 1000, 128, seed=10)
    want2 = run(lib, gpu_ctx, c2)
    g2 = captured(lambda: got.update(b=run(lib, gpu_ctx, c2)))
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(4):
        with torch.cuda.stream(s1):
            g1.replay()
        with torch.cuda.stream(s2):
            g2.replay()
        eager = run(lib, gpu_ctx, c2)
    torch.cuda.synchronize()
    assert (got["a"] == want).all() and (got["b"] == want2).all() and (eager == want2).all()
    outs = []
    for s in (torch.cuda.Stream(), torch.cuda.Stream()):
        with torch.cuda.stream(s):
            outs.append(run(lib, gpu_ctx, c))
    torch.cuda.synchronize()
    assert all((o == want).all() for o in outs)
    assert lib.mxb_check_device_error(gpu_ctx) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 8, 16, 200])
def test_added_to_the_output_itself(lib, gpu_ctx, m):
    import torch

    c = make(m, 300, 512, 64, seed=m)
    c["a"] = torch.randint(-9, 10, (m, 512), device="cuda").float()
    c["s"].fill_(1.0)
    out = torch.randint(-9, 10, (m, 300), device="cuda").float()
    want = out.double() + c["a"].double() @ weight(c)
    run(lib, gpu_ctx, c, steps((mlib.MXB_EP_ADD_FULL, out, 300, 0)), out)
    assert (out == want).all()


@pytest.mark.gpu
def test_norm_then_two_products_serve_a_block(lib, gpu_ctx):
    """norm -> 4-bit product (bias, relu) -> 4-bit product added to the block's input, for one row and for a prompt,
    the calls one after the other on one stream: within 1e-5 of the norm of the float64 block (each call is within
    about 1e-6 of its own norm, and the block's condition is about one)."""
    import torch
    from tests.test_layer_norm import forward as norm

    d, h = 384, 1000
    up, down = make(1, h, d, 64, "bf16", seed=1), make(1, d, h, 128, "f16", seed=2)
    gamma, beta, bias = torch.randn(d, device="cuda"), torch.randn(d, device="cuda"), torch.randn(h, device="cuda")
    for m in (1, 7, 150):
        x = torch.randn(m, d, device="cuda")
        y, _, _ = norm(lib, gpu_ctx, x, gamma, beta)
        hid = run(lib, gpu_ctx, dict(up, a=y, m=m), steps((mlib.MXB_EP_ADD_ROW, bias, 0, 0), (mlib.MXB_EP_RELU, None, 0, 0)))
        out = run(lib, gpu_ctx, dict(down, a=hid, m=m), steps((mlib.MXB_EP_ADD_FULL, x, d, 0)))
        X = x.double()
        c = X - X.mean(1, keepdim=True)
        Y = c * (c.square().mean(1, keepdim=True) + 1e-5).rsqrt() * gamma.double() + beta.double()
        want = torch.relu(Y @ weight(up) + bias.double()) @ weight(down) + X
        assert ((out.double() - want).norm() / want.norm()).item() <= 1e-5


@pytest.mark.gpu
def test_weight_past_32_bit_offsets(lib, gpu_ctx):
    """A weight of more than 2^32 bytes: the last columns are read at their place."""
    import torch

    k, n = 65536, 140000  # 4.6 GB
    c = make(1, 64, k, 128, seed=1)
    q = torch.zeros(n, k // 2, dtype=torch.uint8, device="cuda")
    s = torch.zeros(n, k // 128, device="cuda")
    q[-64:], s[-64:] = c["q"], c["s"]
    z = torch.zeros(n, k // 128, dtype=torch.uint8, device="cuda")
    z[-64:] = c["z"]
    for m in (1, 24):
        small = dict(c, a=torch.randn(m, k, device="cuda"), m=m)
        big = dict(small, q=q, s=s, z=z, n=n)
        out = run(lib, gpu_ctx, big)
        check(small, out[:, -64:])
        assert (out[:, :-64] == 0).all()


REFUSED = [
    dict(ctx=None), dict(A=None), dict(Q=None), dict(scales=None), dict(out=None), dict(M=0), dict(N=0), dict(K=0),
    dict(lda=60), dict(lda=65), dict(ldq=31), dict(ldq=40), dict(A=4100), dict(Q=8200), dict(scales=12289),
    dict(scale_type=3), dict(scale_type=-1), dict(group=16), dict(group=48), dict(group=0), dict(lds=1), dict(ldo=15),
    dict(n_steps=1), dict(n_steps=17), dict(n_steps=-1), dict(kind=mlib.MXB_EP_RELU_GRAD),
    dict(kind=mlib.MXB_EP_ADD_PRODUCT), dict(kind=mlib.MXB_EP_ADD_FULL), dict(kind=99),
]


@pytest.mark.parametrize("change", REFUSED, ids=str)
def test_refusals(lib, change):
    a = dict(ctx=fake_context(), A=4096, lda=64, Q=8192, ldq=32, scales=12288, scale_type=0, zeros=None, lds=2, group=32,
             out=16384, ldo=16, M=2, N=16, K=64, steps=None, n_steps=0, stream=None)
    change = dict(change)
    if "kind" in change:
        a["steps"], a["n_steps"] = steps((change.pop("kind"), None, 16, 1.0))
    a.update(change)
    assert lib.mxb_q4_gemm(*a.values()) == mlib.MXB_E_ARG
    assert "mxb_q4_gemm" in mlib.last_error()
