"""Products grouped by expert and their gradients against float64.

Tolerances, with S the sum of the magnitudes of an output's products.
3xTF32: an operand is split into big + small with |small| <= 2^-10 of it; what
is dropped is small * small (2^-20) and the cut of each small part to 11 bits
(2^-21 each, rounded to nearest), together below 2^-19 S.  The tensor core cuts
each partial sum to 24 bits: at most 48 accumulations (128 values of the sum
dimension, three products) below 2^-23 each before the sums go to fp32 registers,
whose additions round ceil(K / 64) times by u = 2^-24 at most:
  (2^-19 + 48 * 2^-23 + (K / 64 + 8) u) S.
TF32: both operands are rounded to 11 bits, 2^-11 each: 2^-10 S besides the sums.
Sums of small integers are exact in both modes.
"""
import pytest

from minixla_b200 import lib as mlib
from tests.operator_calls import U, captured, current_stream, fake_context, ok, pitched, ptr, steps, within

TF32, X3 = mlib.GPU_PRECISION_TF32, mlib.GPU_PRECISION_3XTF32


def bound(mag, length, precision):
    split = 2.0 ** -19 if precision == X3 else 1.01 * 2.0 ** -10
    return (split + 48 * 2.0 ** -23 + (length / 64 + 8) * U) * mag


def make(sizes, k, n, seed=0, before=0, behind=0, ints=False, pad=0):
    """Rows `before` the first group and `behind` the last belong to none."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    at = [before]
    for s in sizes:
        at.append(at[-1] + s)
    rows, groups = at[-1] + behind, len(sizes)

    def mat(*shape):
        if ints:
            return torch.randint(-6, 7, shape, device="cuda", generator=g).float()
        return torch.randn(shape, device="cuda", generator=g)

    up = lambda v: (v + 3) // 4 * 4 + pad  # noqa: E731
    return dict(a=pitched(mat(rows, k), up(k)), dy=pitched(mat(rows, n), up(n)), b=pitched(mat(groups, k, n), up(n)),
                at=at, off=torch.tensor(at, dtype=torch.int32, device="cuda"), rows=rows, groups=groups, k=k, n=n)


def forward(lib, ctx, c, precision=X3, st=None, out=None, stream=None):
    import torch

    out = torch.full((c["rows"], c["n"]), 77.0, device="cuda") if out is None else out
    arr, cnt = st or steps()
    ok(lib.mxb_grouped_gemm(ctx, ptr(c["a"]), c["a"].stride(0), ptr(c["b"]), c["b"].stride(1), c["b"].stride(0),
                            ptr(c["off"]), c["groups"], ptr(out), out.stride(0), c["rows"], c["n"], c["k"], arr, cnt,
                            precision, stream or current_stream()))
    return out


def grad_a(lib, ctx, c, precision=X3, st=None, out=None, stream=None):
    import torch

    out = torch.full((c["rows"], c["k"]), 77.0, device="cuda") if out is None else out
    arr, cnt = st or steps()
    ok(lib.mxb_grouped_gemm_grad_a(ctx, ptr(c["dy"]), c["dy"].stride(0), ptr(c["b"]), c["b"].stride(1),
                                   c["b"].stride(0), ptr(c["off"]), c["groups"], ptr(out), out.stride(0), c["rows"],
                                   c["n"], c["k"], arr, cnt, precision, stream or current_stream()))
    return out


def grad_b(lib, ctx, c, precision=X3, db=None, dbias=True, stream=None):
    import torch

    db = torch.full((c["groups"], c["k"], c["n"]), 77.0, device="cuda") if db is None else db
    dbias = torch.full((c["groups"], c["n"]), 77.0, device="cuda") if dbias else None
    ok(lib.mxb_grouped_gemm_grad_b(ctx, ptr(c["a"]), c["a"].stride(0), ptr(c["dy"]), c["dy"].stride(0), ptr(c["off"]),
                                   c["groups"], ptr(db), db.stride(1), db.stride(0), ptr(dbias), c["rows"], c["n"],
                                   c["k"], precision, stream or current_stream()))
    return db, dbias


def check_all(c, out, da, db, dbias, precision):
    """Each of the four outputs (or None), and that rows outside the groups kept their 77."""
    import torch

    inside = torch.zeros(c["rows"], dtype=torch.bool, device="cuda")
    inside[c["at"][0]: c["at"][-1]] = True
    for got in (out, da):
        if got is not None:
            assert (got[~inside] == 77.0).all(), "a row outside the groups was written"
    for e in range(c["groups"]):
        r = slice(c["at"][e], c["at"][e + 1])
        a, dy, b = (t.double() for t in (c["a"][r], c["dy"][r], c["b"][e]))
        if out is not None:
            within(out[r], a @ b, bound(a.abs() @ b.abs(), c["k"], precision), f"out {e}") if len(a) else None
        if da is not None:
            within(da[r], dy @ b.t(), bound(dy.abs() @ b.abs().t(), c["n"], precision), f"da {e}") if len(a) else None
        if db is not None:
            within(db[e], a.t() @ dy, bound(a.abs().t() @ dy.abs(), len(a), precision), f"db {e}")
        if dbias is not None:
            within(dbias[e], dy.sum(0), (len(a) + 4) * U * dy.abs().sum(0), f"dbias {e}")


CASES = [
    ([1], 1, 1), ([1], 4, 4), ([1, 0, 1], 33, 17), ([2, 0, 3, 1], 100, 130), ([0, 0, 5], 64, 128),
    ([16, 16], 32, 32), ([17, 15, 1, 33], 257, 129), ([128, 0, 127, 129], 320, 200), ([31, 65, 250], 96, 515),
    ([300], 1000, 100), ([0, 0, 0], 40, 40), ([256, 256, 1], 256, 256), ([513, 7, 270], 128, 384),
    ([1] * 20, 512, 1030), ([5, 90, 0, 40, 700, 3], 1024, 300), ([1100, 260], 515, 1024), ([3, 1, 2, 2], 2048, 2048),
]


@pytest.mark.gpu
@pytest.mark.parametrize("precision", [X3, TF32], ids=["3xtf32", "tf32"])
@pytest.mark.parametrize("sizes,k,n", CASES, ids=lambda v: "x".join(map(str, v)) if isinstance(v, list) else str(v))
def test_against_definition(lib, gpu_ctx, sizes, k, n, precision):
    c = make(sizes, k, n, seed=sum(sizes) + k, before=3, behind=5)
    check_all(c, forward(lib, gpu_ctx, c, precision), grad_a(lib, gpu_ctx, c, precision),
              *grad_b(lib, gpu_ctx, c, precision), precision)
    assert lib.mxb_check_device_error(gpu_ctx) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("precision", [X3, TF32], ids=["3xtf32", "tf32"])
@pytest.mark.parametrize("sizes,k,n", [([2, 0, 1], 70, 90), ([40, 3, 0, 100], 130, 260), ([300, 290, 10], 512, 515)],
                         ids=["few", "some", "many"])
def test_exact_small_integers(lib, gpu_ctx, sizes, k, n, precision):
    c = make(sizes, k, n, seed=1, ints=True)
    out, da, (db, dbias) = (f(lib, gpu_ctx, c, precision) for f in (forward, grad_a, grad_b))
    for e in range(c["groups"]):
        r = slice(c["at"][e], c["at"][e + 1])
        a, dy, b = (t.double() for t in (c["a"][r], c["dy"][r], c["b"][e]))
        assert (out[r] == a @ b).all() and (da[r] == dy @ b.t()).all()
        assert (db[e] == a.t() @ dy).all() and (dbias[e] == dy.sum(0)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [[1, 0, 4], [50, 20, 70], [300, 0, 260]], ids=["few", "some", "many"])
def test_steps_pitches_and_gaps(lib, gpu_ctx, sizes):
    import torch

    k, n = 150, 203
    c = make(sizes, k, n, seed=4, before=2, behind=3, pad=8)
    groups, rows = c["groups"], c["rows"]
    bias = pitched(torch.randn(groups, n, device="cuda"), 207)
    one = torch.randn(n, device="cuda")
    full = pitched(torch.randn(rows, n, device="cuda"), 209)
    gate = pitched(torch.randn(rows, n, device="cuda"), 205)
    out = pitched(torch.full((rows, n), 77.0, device="cuda"), 211, 5.0)
    st = steps((mlib.MXB_EP_ADD_ROW, bias, 207, 0), (mlib.MXB_EP_ADD_ROW, one, 0, 0), (mlib.MXB_EP_ADD_FULL, full, 209, 0),
               (mlib.MXB_EP_RELU, None, 0, 0), (mlib.MXB_EP_SCALE, None, 0, -0.5), (mlib.MXB_EP_RELU_GRAD, gate, 205, 0))
    forward(lib, gpu_ctx, c, X3, st, out)
    for e in range(groups):
        r = slice(c["at"][e], c["at"][e + 1])
        if c["at"][e] == c["at"][e + 1]:
            continue
        a, b = c["a"][r].double(), c["b"][e].double()
        pre = a @ b
        added = bias[e].double() + one.double() + full[r].double()
        want = torch.where(gate[r] > 0, (pre + added).clamp(min=0) * -0.5, 0.0)
        tol = bound(a.abs() @ b.abs(), k, X3) + 8 * U * (pre.abs() + bias[e].double().abs() + one.double().abs()
                                                         + full[r].double().abs())
        within(out[r], want, tol)
    assert (out.as_strided((rows, 211), (211, 1))[:, n:] == 5.0).all()
    assert (out[:2] == 77.0).all() and (out[rows - 3:] == 77.0).all()
    # Gradients with gaps between the rows of each result.
    da = pitched(torch.full((rows, k), 77.0, device="cuda"), 155, 5.0)
    db = pitched(torch.full((groups, k, n), 77.0, device="cuda"), 205, 5.0)
    grad_a(lib, gpu_ctx, c, out=da)
    _, dbias = grad_b(lib, gpu_ctx, c, db=db)
    check_all(c, None, da, db, dbias, X3)
    assert (da.as_strided((rows, 155), (155, 1))[:, k:] == 5.0).all()
    assert (db.as_strided((groups * k, 205), (205, 1))[:, n:] == 5.0).all()
    db2, none = grad_b(lib, gpu_ctx, c, dbias=False)
    assert none is None and (db2 == db).all()


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [[3, 2], [40, 90], [300, 280]], ids=["few", "some", "many"])
def test_bad_values_stay_in_their_group(lib, gpu_ctx, sizes):
    """NaN and infinities in rows of no group, in another group's rows and in
    an unused group's weights reach nothing else."""
    import torch

    c = make([sizes[0], 0, sizes[1]], 200, 136, seed=7, before=2, behind=4)
    good = [forward(lib, gpu_ctx, c), grad_a(lib, gpu_ctx, c), *grad_b(lib, gpu_ctx, c)]
    nan = float("nan")
    for t in (c["a"], c["dy"]):
        t[:2], t[-4:] = nan, float("inf")
        t[c["at"][2]] = nan  # the third group's first row
    c["b"][1] = nan
    out, da, db, dbias = forward(lib, gpu_ctx, c), grad_a(lib, gpu_ctx, c), *grad_b(lib, gpu_ctx, c)
    r = torch.arange(c["rows"], device="cuda")
    keep = (r >= c["at"][0]) & (r < c["at"][3]) & (r != c["at"][2])
    assert (out[keep] == good[0][keep]).all() and (da[keep] == good[1][keep]).all()
    assert torch.isnan(out[c["at"][2]]).all() and torch.isnan(da[c["at"][2]]).all()
    assert (db[:2] == good[2][:2]).all() and (dbias[:2] == good[3][:2]).all()
    assert (db[1] == 0).all() and (dbias[1] == 0).all() and torch.isnan(db[2]).all() and torch.isnan(dbias[2]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("offsets,meant", [
    ([0, 9, 4, 20], [(0, 9), (9, 9), (4, 20)]), ([-7, 3, 500, 600], [(0, 3), (3, 30), (30, 30)]),
    ([40, 2, 2, 2 ** 31 - 1], [(30, 30), (2, 2), (2, 30)]), ([-2 ** 31, -5, -1, 0], [(0, 0), (0, 0), (0, 0)]),
], ids=["decreasing", "past the end", "wild", "negative"])
def test_offsets_out_of_range_are_clamped(lib, gpu_ctx, offsets, meant):
    """Each group is clamp(offsets[e], 0, rows) .. clamp(offsets[e+1], start, rows)."""
    import torch

    c = make([10, 10, 10], 64, 48, seed=5, ints=True)
    c["off"] = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    db, dbias = grad_b(lib, gpu_ctx, c)
    for e, (r0, r1) in enumerate(meant):
        a, dy = c["a"][r0:r1].double(), c["dy"][r0:r1].double()
        assert (db[e] == a.t() @ dy).all() and (dbias[e] == dy.sum(0)).all()
    out, da = forward(lib, gpu_ctx, c), grad_a(lib, gpu_ctx, c)
    cover = [[e for e, (r0, r1) in enumerate(meant) if r0 <= r < r1] for r in range(30)]
    for r, es in enumerate(cover):
        a, dy = c["a"][r].double(), c["dy"][r].double()
        if not es:
            assert (out[r] == 77.0).all() and (da[r] == 77.0).all()
        else:  # each value of a row that two groups claim is one of the two results: their tiles run at the same time
            assert torch.stack([out[r] == a @ c["b"][e].double() for e in es]).any(0).all()
            assert torch.stack([da[r] == dy @ c["b"][e].double().t() for e in es]).any(0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width,length,groups,overlaps", [(130, 64, 512, 5, 3), (640, 128, 1024, 3, 2)])
def test_decreasing_offsets_where_clusters_share_sums(lib, gpu_ctx, rows, width, length, groups, overlaps):
    """Offsets 0, rows, 0, rows, ... make every other group all of the rows: more tiles (64 rows, 128 columns) than
    non-decreasing offsets can give, from which the grid of clusters was sized."""
    import torch

    assert overlaps * -(-rows // 64) > rows // 64 + groups, "a tile more than clusters"
    assert mlib.grouped_plan(mlib.MXB_GROUPED_FORWARD, rows, groups, width, length).k_splits == 8
    assert mlib.grouped_plan(mlib.MXB_GROUPED_GRAD_A, rows, groups, length, width).k_splits == 8
    offsets = torch.tensor([e % 2 * rows for e in range(groups + 1)], dtype=torch.int32, device="cuda")
    for f, k, n in ((forward, length, width), (grad_a, width, length)):
        c = make([rows] + [0] * (groups - 1), k, n, seed=rows, ints=True)
        c["off"] = offsets
        got = f(lib, gpu_ctx, c)
        x = (c["a"] if f is forward else c["dy"]).double()
        meant = torch.stack([x @ (b if f is forward else b.t()) for b in c["b"][::2].double()])
        assert (got == meant).any(0).all()
        # Increasing ones again, of the same extents: clusters.
        c["off"] = torch.tensor([0] + [rows] * groups, dtype=torch.int32, device="cuda")
        assert (f(lib, gpu_ctx, c) == meant[0]).all()
    assert lib.mxb_check_device_error(gpu_ctx) == 0


@pytest.mark.gpu
def test_no_rows(lib, gpu_ctx):
    import torch

    c = make([0, 0], 20, 12, seed=1)
    db, dbias = grad_b(lib, gpu_ctx, c)
    assert (db == 0).all() and (dbias == 0).all()
    off = torch.zeros(3, dtype=torch.int32, device="cuda")
    arr, cnt = steps()
    for f in (lib.mxb_grouped_gemm, lib.mxb_grouped_gemm_grad_a):
        ok(f(gpu_ctx, None, 20, None, 20, 400, ptr(off), 2, None, 20, 0, 12, 20, arr, cnt, X3, current_stream()))
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_most_groups(lib, gpu_ctx):
    import torch

    g = torch.Generator().manual_seed(3)
    sizes = (torch.rand(mlib.MXB_MAX_GROUPS, generator=g) ** 4 * 6).int().tolist()
    c = make(sizes, 48, 40, seed=2, ints=True)
    out, da, (db, dbias) = forward(lib, gpu_ctx, c), grad_a(lib, gpu_ctx, c), grad_b(lib, gpu_ctx, c)
    e = torch.repeat_interleave(torch.arange(len(sizes)), torch.tensor(sizes)).cuda()
    assert (out == torch.einsum("rk,rkn->rn", c["a"].double(), c["b"].double()[e])).all()
    assert (da == torch.einsum("rn,rkn->rk", c["dy"].double(), c["b"].double()[e])).all()
    outer = torch.einsum("rk,rn->rkn", c["a"].double(), c["dy"].double())
    want = torch.zeros(len(sizes), 48, 40, dtype=torch.float64, device="cuda").index_add_(0, e, outer)
    assert (db == want).all()
    assert (dbias == torch.zeros(len(sizes), 40, dtype=torch.float64, device="cuda").index_add_(0, e, c["dy"].double())).all()


@pytest.mark.gpu
def test_weights_past_32_bit_offsets(lib, gpu_ctx):
    """More than 2^31 weights: the last group's are read, and its gradient written, at their place."""
    import torch

    groups, k, n = 9, 16384, 16384  # 9.7 GB
    c = make([3], k, n, seed=1)
    b = torch.zeros(groups, k, n, device="cuda")
    b[-1] = c["b"][0]
    big = dict(c, b=b, groups=groups, at=[0] * groups + [3],
               off=torch.tensor([0] * groups + [3], dtype=torch.int32, device="cuda"))
    out, da = forward(lib, gpu_ctx, big), grad_a(lib, gpu_ctx, big)
    check_all(c, out, da, None, None, X3)
    db, dbias = grad_b(lib, gpu_ctx, big, db=b)
    check_all(c, None, None, db[-1:], dbias[-1:], X3)
    assert not db[:-1].any() and not dbias[:-1].any()


@pytest.mark.gpu
def test_large_groups(lib, gpu_ctx):
    """Long sums and many tiles per group, ragged, in all three directions."""
    c = make([1500, 3, 2100, 0, 700], 1030, 2060, seed=8, behind=9)
    check_all(c, forward(lib, gpu_ctx, c), grad_a(lib, gpu_ctx, c), *grad_b(lib, gpu_ctx, c), X3)


@pytest.mark.gpu
@pytest.mark.parametrize("precision", [X3, TF32], ids=["3xtf32", "tf32"])
def test_large_groups_exactly(lib, gpu_ctx, precision):
    """Enough tiles for every SM, small integers: each product lands where it belongs, and nothing behind the groups."""
    c = make([700, 0, 33, 1300, 256, 1], 1024, 1500, seed=15, before=1, behind=2, ints=True)
    out, da, (db, dbias) = (f(lib, gpu_ctx, c, precision) for f in (forward, grad_a, grad_b))
    for e in range(c["groups"]):
        r = slice(c["at"][e], c["at"][e + 1])
        a, dy, b = (t.double() for t in (c["a"][r], c["dy"][r], c["b"][e]))
        assert (out[r] == a @ b).all() and (da[r] == dy @ b.t()).all()
        assert (db[e] == a.t() @ dy).all() and (dbias[e] == dy.sum(0)).all()
    assert (out[:1] == 77).all() and (out[-2:] == 77).all() and (da[:1] == 77).all() and (da[-2:] == 77).all()


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [[3, 2], [60, 90], [700, 900]], ids=["few", "some", "many"])
def test_added_to_the_output_itself(lib, gpu_ctx, sizes):
    import torch

    c = make(sizes, 96, 1400, seed=3, ints=True)
    out = torch.randint(-9, 10, (c["rows"], c["n"]), device="cuda").float()
    want = out.double() + torch.cat([c["a"][:sizes[0]].double() @ c["b"][0].double(),
                                     c["a"][sizes[0]:].double() @ c["b"][1].double()])
    forward(lib, gpu_ctx, c, st=steps((mlib.MXB_EP_ADD_FULL, out, out.stride(0), 0)), out=out)
    assert (out == want).all()


@pytest.mark.gpu
def test_two_threads_share_a_context(lib, gpu_ctx):
    """Calls from two host threads on streams of their own give what one thread gives."""
    import threading

    import torch

    cases = [make([40, 0, 70], 200, 300, seed=s) for s in (1, 2)]
    want = [(forward(lib, gpu_ctx, c), grad_a(lib, gpu_ctx, c), *grad_b(lib, gpu_ctx, c)) for c in cases]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[i] = (forward(lib, gpu_ctx, cases[i]), grad_a(lib, gpu_ctx, cases[i]), *grad_b(lib, gpu_ctx, cases[i]))
                torch.cuda.current_stream().synchronize()
        except BaseException as e:  # noqa: BLE001 - reported by the main thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for w, g in zip(want, got):
        assert all((a == b).all() for a, b in zip(w, g))


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [[2, 0, 1], [60, 0, 30], [400, 0, 300]], ids=["few", "some", "many"])
def test_captured_and_on_other_streams(lib, gpu_ctx, sizes):
    import torch

    c = make(sizes, 300, 260, seed=9)
    calls = lambda: (forward(lib, gpu_ctx, c), grad_a(lib, gpu_ctx, c), *grad_b(lib, gpu_ctx, c))  # noqa: E731
    want = calls()
    again = calls()
    assert all((a == b).all() for a, b in zip(want, again)), "the same inputs gave other bits"
    got = {}
    graph = captured(lambda: got.update(r=calls()))
    # New offsets in the same buffer: the replay follows them.
    other = make(sizes[::-1], 300, 260, seed=9)
    c["off"].copy_(other["off"])
    graph.replay()
    torch.cuda.synchronize()
    moved = calls()
    assert all((a == b).all() for a, b in zip(got["r"], moved))
    c["off"].copy_(torch.tensor(c["at"], dtype=torch.int32))
    torch.cuda.synchronize()
    outs = []
    for s in (torch.cuda.Stream(), torch.cuda.Stream()):
        with torch.cuda.stream(s):
            outs.append(calls())
    torch.cuda.synchronize()
    assert all((a == b).all() for o in outs for a, b in zip(o, want))
    assert lib.mxb_check_device_error(gpu_ctx) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [[3, 0, 4], [90, 0, 60]], ids=["few", "some"])
def test_gradients_against_differences(lib, gpu_ctx, sizes):
    """The product is linear in each operand, so a difference of two float64
    products is the gradient's value along that direction, up to rounding."""
    import torch

    c = make(sizes, 130, 70, seed=13)
    da, (db, dbias) = grad_a(lib, gpu_ctx, c), grad_b(lib, gpu_ctx, c)

    def loss(a, b, bias):
        return sum((c["dy"][r].double() * (a[r] @ b[e] + bias[e])).sum().item()
                   for e in range(3) for r in [slice(c["at"][e], c["at"][e + 1])])

    args = [c["a"].double(), c["b"].double(), torch.zeros(3, 70, dtype=torch.float64, device="cuda")]
    for i, grad in enumerate((da, db, dbias)):
        d = torch.randn(args[i].shape, dtype=torch.float64, device="cuda", generator=torch.Generator("cuda").manual_seed(i))
        d /= d.norm()
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + d, args[i] - d
        diff = (loss(*up) - loss(*down)) / 2
        assert abs(diff - (grad.double() * d).sum().item()) <= 1e-5 * grad.double().norm().item(), i


@pytest.mark.gpu
def test_block_of_an_expert_mlp_trains_and_serves(lib, gpu_ctx):
    """norm -> experts (bias, relu) -> experts (bias) and the backward pass of
    all of it, the calls one after the other on one stream, against float64
    autograd of the same block.  Five products or sums in a row, each within
    1e-5 of its norm by the bounds above, and their condition here is about
    one: 1e-4 of each gradient's norm."""
    import torch
    from tests.test_layer_norm import backward as norm_backward, forward as norm_forward

    d, h, sizes = 96, 260, [70, 0, 1, 200]
    c1 = make(sizes, d, h, seed=1)
    c2 = make(sizes, h, d, seed=2)
    rows, groups = c1["rows"], 4
    x, dy, gamma, beta = (torch.randn(s, device="cuda") for s in ((rows, d), (rows, d), (d,), (d,)))
    w1, w2 = c1["b"] / d ** 0.5, c2["b"] / h ** 0.5
    b1, b2 = torch.randn(groups, h, device="cuda"), torch.randn(groups, d, device="cuda")
    y, mean, rstd = norm_forward(lib, gpu_ctx, x, gamma, beta)
    hid = forward(lib, gpu_ctx, dict(c1, a=y, b=w1), st=steps((mlib.MXB_EP_ADD_ROW, b1, h, 0), (mlib.MXB_EP_RELU, None, 0, 0)))
    out = forward(lib, gpu_ctx, dict(c2, a=hid, b=w2), st=steps((mlib.MXB_EP_ADD_ROW, b2, d, 0)))
    dhid = grad_a(lib, gpu_ctx, dict(c2, dy=dy, b=w2), st=steps((mlib.MXB_EP_RELU_GRAD, hid, h, 0)))
    dw2, db2 = grad_b(lib, gpu_ctx, dict(c2, a=hid, dy=dy))
    dn = grad_a(lib, gpu_ctx, dict(c1, dy=dhid, b=w1))
    dw1, db1 = grad_b(lib, gpu_ctx, dict(c1, a=y, dy=dhid))
    dx, dgamma, dbeta = norm_backward(lib, gpu_ctx, dn, x, gamma, mean, rstd)

    leaves = [t.double().requires_grad_() for t in (x, gamma, beta, w1, b1, w2, b2)]
    X, G, Be, W1, B1, W2, B2 = leaves
    m = X.mean(1, keepdim=True)
    Y = (X - m) * ((X - m).square().mean(1, keepdim=True) + 1e-5).rsqrt() * G + Be
    parts = []
    for e in range(groups):
        r = slice(c1["at"][e], c1["at"][e + 1])
        parts.append(torch.relu(Y[r] @ W1[e] + B1[e]) @ W2[e] + B2[e])
    O = torch.cat(parts)
    want = torch.autograd.grad(O, leaves, dy.double())
    for name, got, ref in zip(("out", "dx", "dgamma", "dbeta", "dw1", "db1", "dw2", "db2"),
                              (out, dx, dgamma, dbeta, dw1, db1, dw2, db2), (O, *want)):
        err = ((got.double() - ref).norm() / ref.norm()).item()
        assert err <= 1e-4, (name, err)


# ---- the CTA-pair kernel, which takes groups of more than 84 rows where there are enough tiles

PAIR_SIZES, PAIR_K, PAIR_N = [300, 0, 190, 257, 1, 256, 400, 196], 1030, 1100


def make_for_pairs(**kw):
    """A case whose three products all run there (of this or of the full GPU's SMs)."""
    c = make(PAIR_SIZES, PAIR_K, PAIR_N, **kw)
    for product in (mlib.MXB_GROUPED_FORWARD, mlib.MXB_GROUPED_GRAD_A, mlib.MXB_GROUPED_GRAD_B):
        assert mlib.grouped_plan(product, c["rows"], c["groups"], PAIR_N, PAIR_K).kernel == mlib.MXB_KERNEL_CTA_PAIR
    return c


@pytest.mark.gpu
@pytest.mark.parametrize("precision", [X3, TF32], ids=["3xtf32", "tf32"])
def test_pairs_against_definition(lib, gpu_ctx, precision):
    c = make_for_pairs(seed=21, before=3, behind=5)
    check_all(c, forward(lib, gpu_ctx, c, precision), grad_a(lib, gpu_ctx, c, precision),
              *grad_b(lib, gpu_ctx, c, precision), precision)
    assert lib.mxb_check_device_error(gpu_ctx) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("precision", [X3, TF32], ids=["3xtf32", "tf32"])
def test_pairs_steps_pitches_and_gaps(lib, gpu_ctx, precision):
    import torch

    c = make_for_pairs(seed=22, before=2, behind=3, pad=8)
    groups, rows = c["groups"], c["rows"]
    for f, x, width, length in ((forward, c["a"], PAIR_N, PAIR_K), (grad_a, c["dy"], PAIR_K, PAIR_N)):
        bias = pitched(torch.randn(groups, width, device="cuda"), width + 5)
        one = torch.randn(width, device="cuda")
        full = pitched(torch.randn(rows, width, device="cuda"), width + 7)
        gate = pitched(torch.randn(rows, width, device="cuda"), width + 3)
        out = pitched(torch.full((rows, width), 77.0, device="cuda"), width + 9, 5.0)
        st = steps((mlib.MXB_EP_ADD_ROW, bias, width + 5, 0), (mlib.MXB_EP_ADD_ROW, one, 0, 0),
                   (mlib.MXB_EP_ADD_FULL, full, width + 7, 0), (mlib.MXB_EP_RELU, None, 0, 0),
                   (mlib.MXB_EP_SCALE, None, 0, -0.5), (mlib.MXB_EP_RELU_GRAD, gate, width + 3, 0))
        f(lib, gpu_ctx, c, precision, st, out)
        for e in range(groups):
            r = slice(c["at"][e], c["at"][e + 1])
            if c["at"][e] == c["at"][e + 1]:
                continue
            a, b = x[r].double(), c["b"][e].double() if f is forward else c["b"][e].double().t()
            pre = a @ b
            added = bias[e].double() + one.double() + full[r].double()
            want = torch.where(gate[r] > 0, (pre + added).clamp(min=0) * -0.5, 0.0)
            tol = bound(a.abs() @ b.abs(), length, precision) + 8 * U * (
                pre.abs() + bias[e].double().abs() + one.double().abs() + full[r].double().abs())
            within(out[r], want, tol)
        assert (out.as_strided((rows, width + 9), (width + 9, 1))[:, width:] == 5.0).all()
        assert (out[:2] == 77.0).all() and (out[rows - 3:] == 77.0).all()
    db = pitched(torch.full((groups, PAIR_K, PAIR_N), 77.0, device="cuda"), PAIR_N + 3, 5.0)
    _, dbias = grad_b(lib, gpu_ctx, c, precision, db=db)
    check_all(c, None, None, db, dbias, precision)
    assert (db.as_strided((groups * PAIR_K, PAIR_N + 3), (PAIR_N + 3, 1))[:, PAIR_N:] == 5.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("precision", [X3, TF32], ids=["3xtf32", "tf32"])
def test_pairs_bad_values_stay_in_their_group(lib, gpu_ctx, precision):
    import torch

    c = make_for_pairs(seed=23, before=2, behind=4)
    at = c["at"]
    good = [forward(lib, gpu_ctx, c, precision), grad_a(lib, gpu_ctx, c, precision), *grad_b(lib, gpu_ctx, c, precision)]
    nan = float("nan")
    for t in (c["a"], c["dy"]):
        t[:2], t[-4:] = nan, float("inf")
        t[at[3]] = nan  # the first row of the group behind two others in its tiles' boxes
    c["b"][1] = nan     # of an empty group
    out, da = forward(lib, gpu_ctx, c, precision), grad_a(lib, gpu_ctx, c, precision)
    db, dbias = grad_b(lib, gpu_ctx, c, precision)
    r = torch.arange(c["rows"], device="cuda")
    keep = (r >= at[0]) & (r < at[-1]) & (r != at[3])
    assert (out[keep] == good[0][keep]).all() and (da[keep] == good[1][keep]).all()
    assert torch.isnan(out[at[3]]).all() and torch.isnan(da[at[3]]).all()
    others = [0, 1, 2, 4, 5, 6, 7]
    assert (db[others] == good[2][others]).all() and (dbias[others] == good[3][others]).all()
    assert torch.isnan(db[3]).all() and torch.isnan(dbias[3]).all() and (db[1] == 0).all() and (dbias[1] == 0).all()


@pytest.mark.gpu
def test_pairs_added_to_the_output_itself(lib, gpu_ctx):
    import torch

    c = make_for_pairs(seed=24, ints=True)
    for f, x, width in ((forward, c["a"], PAIR_N), (grad_a, c["dy"], PAIR_K)):
        out = torch.randint(-9, 10, (c["rows"], width), device="cuda").float()
        want = out.double()
        for e in range(c["groups"]):
            r = slice(c["at"][e], c["at"][e + 1])
            b = c["b"][e].double()
            want[r] += x[r].double() @ (b if f is forward else b.t())
        f(lib, gpu_ctx, c, st=steps((mlib.MXB_EP_ADD_FULL, out, out.stride(0), 0)), out=out)
        assert (out == want).all()


@pytest.mark.gpu
def test_pairs_with_decreasing_offsets(lib, gpu_ctx):
    """Four groups of all the rows: more tiles than the grid was sized for."""
    import torch

    c = make_for_pairs(seed=25, ints=True)
    c["off"] = torch.tensor([e % 2 * c["rows"] for e in range(9)], dtype=torch.int32, device="cuda")
    for f, x in ((forward, c["a"]), (grad_a, c["dy"])):
        got = f(lib, gpu_ctx, c)
        found = torch.zeros_like(got, dtype=torch.bool)
        for b in c["b"][::2].double():
            found |= got == x.double() @ (b if f is forward else b.t())
        assert found.all()


@pytest.mark.gpu
@pytest.mark.parametrize("precision", [X3, TF32], ids=["3xtf32", "tf32"])
def test_pairs_captured_and_on_other_streams(lib, gpu_ctx, precision):
    import torch

    c = make_for_pairs(seed=26)
    calls = lambda: (forward(lib, gpu_ctx, c, precision), grad_a(lib, gpu_ctx, c, precision),  # noqa: E731
                     *grad_b(lib, gpu_ctx, c, precision))
    want, again = calls(), calls()
    assert all((a == b).all() for a, b in zip(want, again)), "the same inputs gave other bits"
    got = {}
    graph = captured(lambda: got.update(r=calls()))
    at = [0]
    for size in PAIR_SIZES[::-1]:
        at.append(at[-1] + size)
    c["off"].copy_(torch.tensor(at, dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    moved = calls()
    assert all((a == b).all() for a, b in zip(got["r"], moved))
    c["off"].copy_(torch.tensor(c["at"], dtype=torch.int32))
    torch.cuda.synchronize()
    outs = []
    for s in (torch.cuda.Stream(), torch.cuda.Stream()):
        with torch.cuda.stream(s):
            outs.append(calls())
    torch.cuda.synchronize()
    assert all((a == b).all() for o in outs for a, b in zip(o, want))
    assert lib.mxb_check_device_error(gpu_ctx) == 0
    del graph


@pytest.mark.parametrize("which", ["mxb_grouped_gemm", "mxb_grouped_gemm_grad_a"])
def test_extents_past_the_limit(lib, which):
    n = (1 << 30) + 4
    rc = getattr(lib, which)(fake_context(), 4096, n, 8192, n, 0, 12288, 1, 16384, n, 4, n, n, None, 0, X3, None)
    assert rc == mlib.MXB_E_UNSUPPORTED and "2^30" in mlib.last_error()


A, B, OFF, OUT = 4096, 8192, 12288, 16384
REFUSED = [
    dict(ctx=None), dict(A=None), dict(B=None), dict(offsets=None), dict(out=None), dict(groups=0), dict(groups=1025),
    dict(rows=-1), dict(N=0), dict(K=0), dict(lda=7), dict(lda=9), dict(ldb=13), dict(ldb=18), dict(b_stride=64),
    dict(b_stride=130), dict(A=4100), dict(B=8200), dict(ldo=5), dict(n_steps=1), dict(n_steps=17), dict(n_steps=-1),
    dict(precision=2), dict(kind=mlib.MXB_EP_ADD_MOD), dict(kind=mlib.MXB_EP_ADD_PRODUCT),
    dict(kind=mlib.MXB_EP_ADD_FULL), dict(kind=mlib.MXB_EP_RELU_GRAD), dict(kind=-1),
]


@pytest.mark.parametrize("which", ["mxb_grouped_gemm", "mxb_grouped_gemm_grad_a"])
@pytest.mark.parametrize("change", REFUSED, ids=str)
def test_refusals(lib, which, change):
    n, k = (16, 8) if which == "mxb_grouped_gemm" else (8, 8)
    a = dict(ctx=fake_context(), A=A, lda=8, B=B, ldb=16, b_stride=128, offsets=OFF, groups=2, out=OUT, ldo=16, rows=4,
             N=n, K=k, steps=None, n_steps=0, precision=X3, stream=None)
    change = dict(change)
    if "ldb" in change and which.endswith("grad_a"):
        change["ldb"] = 6 if change["ldb"] == 13 else 18
    if "kind" in change:
        a["steps"], a["n_steps"] = steps((change.pop("kind"), None, 16, 1.0))
    a.update(change)
    if change.get("b_stride") == 64 and which.endswith("grad_a"):
        a["b_stride"] = 100
    assert getattr(lib, which)(*a.values()) == mlib.MXB_E_ARG
    assert which in mlib.last_error()


REFUSED_B = [
    dict(ctx=None), dict(A=None), dict(dY=None), dict(offsets=None), dict(dB=None), dict(groups=0), dict(groups=1025),
    dict(rows=-1), dict(N=0), dict(K=0), dict(lda=7), dict(lda=9), dict(lddy=13), dict(lddy=18), dict(A=4100),
    dict(dY=8200), dict(lddb=15), dict(db_stride=100), dict(precision=0),
]


@pytest.mark.parametrize("change", REFUSED_B, ids=str)
def test_refusals_of_the_weight_gradient(lib, change):
    a = dict(ctx=fake_context(), A=A, lda=8, dY=B, lddy=16, offsets=OFF, groups=2, dB=OUT, lddb=16, db_stride=128,
             dbias=None, rows=4, N=16, K=8, precision=X3, stream=None)
    a.update(change)
    assert lib.mxb_grouped_gemm_grad_b(*a.values()) == mlib.MXB_E_ARG
    assert "mxb_grouped_gemm_grad_b" in mlib.last_error()
