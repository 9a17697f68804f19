"""Layer norm, products with 4-bit weights and products grouped by expert: what is measured of them.

A case names one pass through one entry point of the library.  ``prepare``
makes its inputs on the GPU, ``run`` runs it -- in plain torch operations
(``own`` false) or through the library's C ABI (``own`` true) -- and ``exact``
gives the same outputs from the definition in float64.

Formulas (rows r, columns j; everything is stored in fp32 unless said):

* layer norm      y = (x - mean) * rstd * gamma + beta,  rstd = (var + eps)^-1/2;
                  its backward pass gives dx, dgamma, dbeta;
* q4 product      out = relu(A @ W + bias), W[k, n] = (q[n, k] - z[n, k/G]) * s[n, k/G]
                  with q in 0..15, two to a byte along k (low nibble first);
* grouped product out[r] = relu(A[r] @ B[e] + bias[e]) for offsets[e] <= r < offsets[e+1];
                  grad_a: dA[r] = (dY[r] @ B[e]^T) where the saved activation is positive, else 0;
                  grad_b: dB[e] = A_e^T @ dY_e and dbias[e] = the column sums of dY_e.
"""
import torch

own = False

EPS = 1e-5
SCALES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- cases


def listed():
    return [
        # The norm in front of an MLP block while eight sequences decode: latency.
        dict(name="norm decode 8x4096", op="norm", rows=8, cols=4096),
        # The same norm over a prompt of 16384 rows: two streams of 268 MB.
        dict(name="norm prompt 16384x4096", op="norm", rows=16384, cols=4096),
        # A short ragged batch with a width that no vector divides.
        dict(name="norm grad 5003x1027", op="norm_grad", rows=5003, cols=1027),
        # A training batch: x, dy and dx are 268 MB each.
        dict(name="norm grad 8192x8192", op="norm_grad", rows=8192, cols=8192),
        # One token through a 4096 x 4096 weight in 4 bits, bf16 scales, no zero points.
        dict(name="q4 1x4096x4096", op="q4", m=1, n=4096, k=4096, group=128, scale="bf16", zeros=False),
        # Eight decoding sequences, small groups with fp32 scales and zero points.
        dict(name="q4 8x8192x8192", op="q4", m=8, n=8192, k=8192, group=32, scale="f32", zeros=True),
        # A prompt of 1000 rows through the same weight.
        dict(name="q4 1000x8192x8192", op="q4", m=1000, n=8192, k=8192, group=128, scale="f16", zeros=True),
        # One token sent to two of eight experts (1024 -> 4096, the sizes of the 3-layer MLP).
        dict(name="grouped 2 rows, 8 experts", op="grouped", rows=2, groups=8, k=1024, n=4096),
        # 64 tokens to two of 64 experts each: the weights (537 MB) are read for one or two rows apiece.
        dict(name="grouped 128 rows, 64 experts", op="grouped", rows=128, groups=64, k=1024, n=2048),
        # A prompt: 4096 tokens to two of eight experts of 4096 x 4096.
        dict(name="grouped 8192 rows, 8 experts", op="grouped", rows=8192, groups=8, k=4096, n=4096),
        # The gradient of the same layer's input, more and smaller experts, ragged.
        dict(name="grouped grad a 4001, 16 experts", op="grouped_grad_a", rows=4001, groups=16, k=1024, n=4096),
        # The gradient of the weights and of the bias.
        dict(name="grouped grad b 8191, 8 experts", op="grouped_grad_b", rows=8191, groups=8, k=1024, n=4096),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "q4", "q4", "grouped", "grouped", "grouped_grad_a", "grouped_grad_b"])
    if op in ("norm", "norm_grad"):
        cols = _log(rng, 64, 16384)
        return dict(op=op, rows=_log(rng, 1, min(16384, (1 << 26) // cols)), cols=cols)
    if op == "q4":
        return dict(op=op, m=_log(rng, 1, 512), n=_log(rng, 100, 8192), k=_log(rng, 100, 8192),
                    group=rng.choice([32, 64, 128]), scale=rng.choice(sorted(SCALES)), zeros=rng.random() < 0.5)
    return dict(op=op, rows=_log(rng, 1, 8192), groups=_log(rng, 1, 32), k=_log(rng, 64, 4096), n=_log(rng, 64, 4096))


def work(case):
    op = case["op"]
    if op == "norm":
        r, c = case["rows"], case["cols"]
        return {"bytes": 4 * (2 * r * c + 2 * c + 2 * r), "flops": 8 * r * c}
    if op == "norm_grad":
        r, c = case["rows"], case["cols"]
        return {"bytes": 4 * (3 * r * c + 3 * c + 2 * r), "flops": 14 * r * c}
    if op == "q4":
        m, n, k = case["m"], case["n"], case["k"]
        per = SCALES[case["scale"]].itemsize + (1 if case["zeros"] else 0)
        return {"bytes": n * ((k + 1) // 2 + -(-k // case["group"]) * per) + 4 * (m * k + m * n + n),
                "flops": 2 * m * n * k}
    r, k, n, g = case["rows"], case["k"], case["n"], case["groups"]
    used = min(g, r)  # no more groups than rows have weights that are read
    if op == "grouped":
        b = 4 * (r * k + used * (k * n + n) + r * n)
    elif op == "grouped_grad_a":
        b = 4 * (r * n + used * k * n + 2 * r * k)
    else:
        b = 4 * (r * k + r * n + g * (k * n + n))
    return {"bytes": b + 4 * (g + 1), "flops": 2 * r * k * n}


# ---------------------------------------------------------------- inputs


def _pitched(rows, cols, gen, scale=1.0):
    """A [rows, cols] matrix whose rows start on 16-byte boundaries, as the library's products ask."""
    pitch = (cols + 3) // 4 * 4
    return torch.randn(rows, pitch, device="cuda", generator=gen).mul_(scale)[:, :cols]


def _offsets(rows, groups, gen):
    """Row counts as a router gives them: popular and rare experts, some without a row."""
    p = torch.rand(groups, device="cuda", generator=gen) ** 2 + 0.01
    e = torch.multinomial(p, rows, replacement=True, generator=gen)
    sizes = torch.bincount(e, minlength=groups).tolist()
    at = [0]
    for s in sizes:
        at.append(at[-1] + s)
    return at, torch.tensor(at, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s, op = {"op": case["op"]}, case["op"]
    if op in ("norm", "norm_grad"):
        r, c = case["rows"], case["cols"]
        # Activations of a residual stream: every row with its own spread and offset.
        spread = torch.rand(r, 1, device="cuda", generator=gen) * 3 + 0.1
        s["x"] = torch.randn(r, c, device="cuda", generator=gen).mul_(spread).add_(spread * 0.3)
        s["gamma"] = 1 + 0.1 * torch.randn(c, device="cuda", generator=gen)
        s["beta"] = 0.1 * torch.randn(c, device="cuda", generator=gen)
        if op == "norm_grad":
            s["dy"] = torch.randn(r, c, device="cuda", generator=gen)
            x = s["x"]
            s["mean"] = x.double().mean(1).float()
            s["rstd"] = (x.double().var(1, unbiased=False) + EPS).rsqrt().float()
        return s
    if op == "q4":
        m, n, k, group = case["m"], case["n"], case["k"], case["group"]
        kg = -(-k // group)
        pitch = ((k + 1) // 2 + 15) // 16 * 16
        s.update(m=m, n=n, k=k, group=group, scale=case["scale"])
        s["a"] = _pitched(m, k, gen)
        s["q"] = torch.randint(0, 256, (n, pitch), dtype=torch.uint8, device="cuda", generator=gen)
        s["scales"] = ((torch.rand(n, kg, device="cuda", generator=gen) + 0.5) * (0.25 / k ** 0.5)).to(SCALES[case["scale"]])
        s["zeros"] = torch.randint(5, 11, (n, kg), dtype=torch.uint8, device="cuda", generator=gen) if case["zeros"] else None
        s["bias"] = 0.1 * torch.randn(n, device="cuda", generator=gen)
        return s
    r, k, n, g = case["rows"], case["k"], case["n"], case["groups"]
    s.update(rows=r, k=k, n=n, groups=g)
    s["at"], s["offsets"] = _offsets(r, g, gen)
    if op != "grouped_grad_b":
        s["b"] = _pitched(g * k, n, gen, 1 / k ** 0.5).unflatten(0, (g, k))
    if op == "grouped":
        s["a"] = _pitched(r, k, gen)
        s["bias"] = 0.1 * torch.randn(g, n, device="cuda", generator=gen)
    else:
        s["dy"] = _pitched(r, n, gen)
        # The layer's input: the relu of the layer before it, about half of it zero.
        s["act"] = _pitched(r, k, gen).clamp_(min=0)
    return s


# ---------------------------------------------------------------- plain forms


def _dequantised(s):
    """W [K, N] in fp32."""
    n, k, group = s["n"], s["k"], s["group"]
    q = torch.stack((s["q"] & 15, s["q"] >> 4), dim=2).view(n, -1)[:, :k].float()
    col = torch.arange(k, device="cuda") // group
    z = s["zeros"].float()[:, col] if s["zeros"] is not None else 8.0
    return ((q - z) * s["scales"].float()[:, col]).t()


def _plain(s):
    op = s["op"]
    if op == "norm":
        x = s["x"]
        mean = x.mean(1, keepdim=True)
        d = x - mean
        rstd = (d.square().mean(1, keepdim=True) + EPS).rsqrt()
        return d * rstd * s["gamma"] + s["beta"], mean.squeeze(1), rstd.squeeze(1)
    if op == "norm_grad":
        xhat = (s["x"] - s["mean"][:, None]) * s["rstd"][:, None]
        g = s["dy"] * s["gamma"]
        dx = (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True)) * s["rstd"][:, None]
        return dx, (s["dy"] * xhat).sum(0), s["dy"].sum(0)
    if op == "q4":
        return (s["a"] @ _dequantised(s) + s["bias"]).clamp(min=0)
    at, g = s["at"], s["groups"]
    if op == "grouped":
        out = torch.empty(s["rows"], s["n"], device="cuda")
        for e in range(g):
            if at[e] < at[e + 1]:
                out[at[e]:at[e + 1]] = (s["a"][at[e]:at[e + 1]] @ s["b"][e] + s["bias"][e]).clamp(min=0)
        return out
    if op == "grouped_grad_a":
        da = torch.empty(s["rows"], s["k"], device="cuda")
        for e in range(g):
            if at[e] < at[e + 1]:
                da[at[e]:at[e + 1]] = s["dy"][at[e]:at[e + 1]] @ s["b"][e].t()
        return da * (s["act"] > 0)
    db = torch.zeros(g, s["k"], s["n"], device="cuda")
    dbias = torch.zeros(g, s["n"], device="cuda")
    for e in range(g):
        if at[e] < at[e + 1]:
            db[e] = s["act"][at[e]:at[e + 1]].t() @ s["dy"][at[e]:at[e + 1]]
            dbias[e] = s["dy"][at[e]:at[e + 1]].sum(0)
    return db, dbias


# ---------------------------------------------------------------- the library's calls

_handles = {}


def _library():
    """(library, context) of the current device, made once as a program does."""
    dev = torch.cuda.current_device()
    if dev not in _handles:
        from minixla_b200 import lib as mlib

        L = mlib.load()
        ctx = L.gpu_ctx_create_on(dev)
        if not ctx:
            raise RuntimeError(mlib.last_error())
        _handles[dev] = (mlib, L, ctx)
    return _handles[dev]


def _own(s):
    mlib, L, ctx = _library()
    op = s["op"]
    stream = torch.cuda.current_stream().cuda_stream or mlib.CUDA_STREAM_LEGACY
    p = lambda t: t.data_ptr() if t is not None else None  # noqa: E731

    def new(*shape):
        return torch.empty(shape, device="cuda")

    def checked(rc):
        if rc != 0:
            raise RuntimeError(mlib.last_error())

    if op == "norm":
        r, c = s["x"].shape
        y, mean, rstd = new(r, c), new(r), new(r)
        checked(L.mxb_layer_norm(ctx, p(s["x"]), c, p(s["gamma"]), p(s["beta"]), EPS, p(y), c, p(mean), p(rstd), r, c, stream))
        return y, mean, rstd
    if op == "norm_grad":
        r, c = s["x"].shape
        dx, dgamma, dbeta = new(r, c), new(c), new(c)
        checked(L.mxb_layer_norm_backward(ctx, p(s["dy"]), c, p(s["x"]), c, p(s["gamma"]), p(s["mean"]), p(s["rstd"]),
                                          p(dx), c, p(dgamma), p(dbeta), r, c, stream))
        return dx, dgamma, dbeta
    if op == "q4":
        m, n, k = s["m"], s["n"], s["k"]
        steps = (mlib.EpStepDev * 2)()
        steps[0].kind, steps[0].operand = mlib.MXB_EP_ADD_ROW, p(s["bias"])
        steps[1].kind = mlib.MXB_EP_RELU
        out = new(m, n)
        kind = {"f32": mlib.MXB_SCALE_F32, "f16": mlib.MXB_SCALE_F16, "bf16": mlib.MXB_SCALE_BF16}[s["scale"]]
        checked(L.mxb_q4_gemm(ctx, p(s["a"]), s["a"].stride(0), p(s["q"]), s["q"].stride(0), p(s["scales"]), kind, p(s["zeros"]),
                              s["scales"].stride(0), s["group"], p(out), n, m, n, k, steps, 2, stream))
        return out
    r, k, n, g = s["rows"], s["k"], s["n"], s["groups"]
    x3 = mlib.GPU_PRECISION_3XTF32
    if op == "grouped":
        steps = (mlib.EpStepDev * 2)()
        steps[0].kind, steps[0].operand, steps[0].ld_or_size = mlib.MXB_EP_ADD_ROW, p(s["bias"]), n
        steps[1].kind = mlib.MXB_EP_RELU
        out = new(r, n)
        checked(L.mxb_grouped_gemm(ctx, p(s["a"]), s["a"].stride(0), p(s["b"]), s["b"].stride(1), s["b"].stride(0), p(s["offsets"]), g,
                                   p(out), n, r, n, k, steps, 2, x3, stream))
        return out
    if op == "grouped_grad_a":
        steps = (mlib.EpStepDev * 1)()
        steps[0].kind, steps[0].operand, steps[0].ld_or_size = mlib.MXB_EP_RELU_GRAD, p(s["act"]), s["act"].stride(0)
        da = new(r, k)
        checked(L.mxb_grouped_gemm_grad_a(ctx, p(s["dy"]), s["dy"].stride(0), p(s["b"]), s["b"].stride(1), s["b"].stride(0), p(s["offsets"]), g,
                                          p(da), k, r, n, k, steps, 1, x3, stream))
        return da
    db, dbias = new(g, k, n), new(g, n)
    checked(L.mxb_grouped_gemm_grad_b(ctx, p(s["act"]), s["act"].stride(0), p(s["dy"]), s["dy"].stride(0), p(s["offsets"]), g,
                                      p(db), n, k * n, p(dbias), r, n, k, x3, stream))
    return db, dbias


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------- 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    d = {key: v.double() for key, v in s.items() if torch.is_tensor(v) and v.is_floating_point()}
    op = case["op"]
    if op == "norm":
        var, mean = torch.var_mean(d["x"], dim=1, correction=0)
        rstd = 1 / torch.sqrt(var + EPS)
        return d["gamma"] * torch.einsum("rc,r->rc", d["x"] - mean.unsqueeze(1), rstd) + d["beta"], mean, rstd
    if op == "norm_grad":
        # Through the Jacobian: dx = rstd (I - 11'/c - xhat xhat'/c) (gamma * dy), row by row.
        c = case["cols"]
        rstd = d["rstd"].unsqueeze(1)
        xhat = rstd * d["x"] - rstd * d["mean"].unsqueeze(1)
        v = torch.einsum("rc,c->rc", d["dy"], d["gamma"])
        dot = torch.einsum("rc,rc->r", v, xhat).unsqueeze(1)
        dx = rstd * v - rstd * (v.sum(1, keepdim=True) + dot * xhat) / c
        return dx, torch.einsum("rc,rc->c", d["dy"], xhat), torch.einsum("rc->c", d["dy"])
    if op == "q4":
        m, n, k, group = (case[x] for x in ("m", "n", "k", "group"))
        kg = -(-k // group)
        w = torch.zeros(n, kg * group, dtype=torch.float64, device="cuda")
        q = s["q"][:, :(k + 1) // 2].to(torch.int16)
        w[:, 0:k:2] = (q % 16).double()[:, :(k + 1) // 2]
        w[:, 1:k:2] = (q // 16).double()[:, :k // 2]
        w = w.view(n, kg, group)
        w = (w - (s["zeros"].double().unsqueeze(2) if s["zeros"] is not None else 8)) * d["scales"].unsqueeze(2)
        return torch.relu(torch.einsum("mk,nk->mn", d["a"], w.view(n, -1)[:, :k]) + d["bias"])
    sizes = (s["offsets"][1:] - s["offsets"][:-1]).tolist()
    if op == "grouped":
        parts = [torch.relu(torch.addmm(d["bias"][e], x, d["b"][e])) for e, x in enumerate(d["a"].split(sizes))]
        return torch.cat(parts)
    if op == "grouped_grad_a":
        da = torch.cat([torch.einsum("rn,kn->rk", y, d["b"][e]) for e, y in enumerate(d["dy"].split(sizes))])
        return torch.where(s["act"] > 0, da, torch.zeros_like(da))
    pairs = list(zip(d["act"].split(sizes), d["dy"].split(sizes)))
    return torch.stack([torch.einsum("rk,rn->kn", a, y) for a, y in pairs]), torch.stack([y.sum(0) for _, y in pairs])
