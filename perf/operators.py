"""The channels-last layer operators -- group norm with an activation, and the matrix product with bias, activation and residual --
as measurable cases: their inputs, their plain form in elementary torch operations, their use through the library, and their values in 64 bits.

`own` False: `run` computes the plain form (32-bit arithmetic whatever the inputs' type, rounded once at the end).
`own` True:  `run` makes the calls a user makes of `ttc._lib.Context`.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"fp32": 4, "fp16": 2, "bf16": 2}
EPS = 1e-5

TILE_PIXELS = 36 * 158 * 158          # output pixels of the 36 windows of one 618 x 618 tile
MAX_NORM = 36 * 172 * 172 * 64        # elements of the bi-ConvGRU output of one tile
MAX_BYTES = 4 * TILE_PIXELS * 64 * 4
MAX_FLOPS = {"fp32": 2 * 65536 * 256 * 256, "fp16": 2 * 8192 * 1024 * 4096, "bf16": 2 * 8192 * 1024 * 4096}


def listed():
    def gn(name, dtype, n, h, w, c, groups, act, train=False, extra=0):
        return dict(name=name, op="group_norm", dtype=dtype, n=n, h=h, w=w, c=c, groups=groups, act=act, train=train, extra=extra)

    def lin(name, dtype, rows, k, n, act, bias=True, residual=False, scale=1.0, train=False, extra=0):
        return dict(name=name, op="linear", dtype=dtype, rows=rows, k=k, n=n, act=act, bias=bias, residual=residual, scale=scale, train=train,
                    extra=extra)
    return [
        # one 14 x 14 training patch: the smallest call, latency only
        gn("norm_patch_f32", "fp32", 1, 14, 14, 64, 8, "swish"),
        # the recurrent features of a whole tile (36 windows of 172 x 172, 64 channels)
        gn("norm_tile_f32", "fp32", 36, 172, 172, 64, 8, "swish"),
        # a U-Net level of a whole tile at half precision, gate activation
        gn("norm_level_bf16", "bf16", 36, 84, 84, 128, 8, "sigmoid"),
        # odd sizes, channels taken out of a wider concatenated tensor, forward and backward
        gn("norm_slice_train_f16", "fp16", 5, 61, 47, 40, 5, "tanh", train=True, extra=24),
        # a training batch of the reference's 28 x 28 patches
        gn("norm_batch_train_f32", "fp32", 32, 28, 28, 64, 8, "swish", train=True),
        # a training step over a whole tile's features
        gn("norm_tile_train_bf16", "bf16", 36, 172, 172, 64, 8, "swish", train=True),
        # one row through a wide layer: a single vector, latency and weight streaming
        lin("product_row_bf16", "bf16", 1, 1024, 4096, "gelu"),
        # the 1 x 1 sigmoid head over the features of a tile
        lin("product_head_f32", "fp32", TILE_PIXELS, 64, 1, "sigmoid"),
        # a wide layer over many rows: bound by the matrix cores
        lin("product_wide_bf16", "bf16", 8192, 1024, 4096, "gelu"),
        # a pointwise residual layer over the features of a tile, forward and backward
        lin("product_tile_train_bf16", "bf16", TILE_PIXELS, 64, 64, "swish", residual=True, scale=0.1, train=True),
        # the deepest U-Net level (40 x 40, 36 windows) reduced to half its channels, forward and backward
        lin("product_level_train_f32", "fp32", 36 * 40 * 40, 256, 128, "tanh", train=True),
        # ragged sizes, rows of a wider tensor, no activation, forward and backward
        lin("product_ragged_train_f16", "fp16", 5003, 177, 93, None, residual=True, train=True, extra=7),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    train = rng.random() < 0.5
    if rng.random() < 0.5:
        while True:
            groups = rng.choice([1, 2, 4, 5, 8, 16, 32])
            c = groups * _log(rng, 2, 64)
            n, h, w = _log(rng, 1, 36), _log(rng, 3, 172), _log(rng, 3, 172)
            extra = rng.choice([0, 0, 3, 8, 64])
            if c <= 512 and n * h * w * (c + extra) <= MAX_NORM:
                break
        return dict(op="group_norm", dtype=dtype, n=n, h=h, w=w, c=c, groups=groups, act=rng.choice([None, "swish", "sigmoid", "tanh", "gelu"]),
                    train=train, extra=extra)
    while True:
        rows, k, n = _log(rng, 1, TILE_PIXELS), _log(rng, 1, 1024), _log(rng, 1, 4096)
        if rng.random() < 0.5:                       # whole 16-byte vectors as often as odd sizes
            k, n = -(-k // 8) * 8, -(-n // 8) * 8
        case = dict(op="linear", dtype=dtype, rows=rows, k=k, n=n, act=rng.choice([None, "swish", "sigmoid", "tanh", "gelu"]),
                    bias=rng.random() < 0.8, residual=rng.random() < 0.5, scale=rng.choice([1.0, 0.1]), train=train, extra=rng.choice([0, 0, 0, 5, 64]))
        if work(case)["flops"] <= MAX_FLOPS[dtype] and work(case)["bytes"] <= MAX_BYTES and rows * (k + case["extra"]) * 4 <= MAX_BYTES // 2:
            return case


_ctx = None


def _context():
    """the library context a program keeps; its window geometry is the smallest the model takes"""
    global _ctx
    if _ctx is None:
        from ttc import _lib
        _ctx = _lib.Context(win_in=44, length=1, max_windows=1)
    return _ctx


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0, shift=0.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)

    st = {"case": case, "ctx": _context() if own else None}
    if case["op"] == "group_norm":
        n, h, w, c = case["n"], case["h"], case["w"], case["c"]
        # channel means and spreads differ, as those of a convolution's raw outputs do
        spread = torch.rand(c + case["extra"], generator=g, device="cuda") * 1.5 + 0.5
        level = torch.randn(c + case["extra"], generator=g, device="cuda")
        wide = (torch.randn(n, h, w, c + case["extra"], generator=g, device="cuda") * spread + level).to(dt)
        st["x"] = wide[..., case["extra"]:]
        st["gamma"] = randn(c, scale=0.1, shift=1.0, dtype=torch.float32)
        st["beta"] = randn(c, scale=0.1, dtype=torch.float32)
        if case["train"]:
            st["dy"] = randn(n, h, w, c)
    else:
        rows, k, n = case["rows"], case["k"], case["n"]
        st["x"] = randn(rows, k + case["extra"])[:, case["extra"]:]
        st["w"] = randn(k, n, scale=1.0 / math.sqrt(k))
        st["bias"] = randn(n, scale=0.1, dtype=torch.float32) if case["bias"] else None
        st["residual"] = randn(rows, n) if case["residual"] else None
        if case["train"]:
            st["dy"] = randn(rows, n)
    return st


# ---- plain form ---------------------------------------------------------------------------------------------------------------

def _activate(z, act):
    if act is None:
        return z
    if act == "swish":
        return z / (1.0 + torch.exp(-z))
    if act == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-z))
    if act == "tanh":
        return torch.tanh(z)
    if act == "gelu":
        return 0.5 * z * torch.erfc(z * -math.sqrt(0.5))
    raise ValueError(act)


def _slope(z, act):
    if act == "swish":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s + z * s * (1.0 - s)
    if act == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 - s)
    if act == "tanh":
        t = torch.tanh(z)
        return 1.0 - t * t
    if act == "gelu":
        return 0.5 * torch.erfc(z * -math.sqrt(0.5)) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    raise ValueError(act)


def _plain_norm(st):
    case, x = st["case"], st["x"]
    n, c, g = case["n"], case["c"], case["groups"]
    xf = x.float().reshape(n, -1, g, c // g)
    d = xf - xf.mean(dim=(1, 3), keepdim=True)
    rstd = 1.0 / torch.sqrt((d * d).mean(dim=(1, 3), keepdim=True) + EPS)
    xhat = (d * rstd).reshape(n, -1, c)
    z = xhat * st["gamma"] + st["beta"]
    y = _activate(z, case["act"]).reshape(x.shape).to(x.dtype)
    if not case["train"]:
        return (y,)
    dz = st["dy"].float().reshape(n, -1, c)
    if case["act"] is not None:
        dz = dz * _slope(z, case["act"])
    dbeta = dz.sum(dim=(0, 1))
    dgamma = (dz * xhat).sum(dim=(0, 1))
    t = (dz * st["gamma"]).reshape(n, -1, g, c // g)
    xh = xhat.reshape(n, -1, g, c // g)
    dx = rstd * (t - t.mean(dim=(1, 3), keepdim=True) - xh * (t * xh).mean(dim=(1, 3), keepdim=True))
    return y, dx.reshape(x.shape).to(x.dtype), dgamma, dbeta


def _plain_product(st):
    case, x, w = st["case"], st["x"].float(), st["w"].float()
    z = torch.matmul(x, w)
    if st["bias"] is not None:
        z = z + st["bias"]
    y = _activate(z, case["act"]) * case["scale"]
    if st["residual"] is not None:
        y = y + st["residual"].float()
    y = y.to(st["x"].dtype)
    if not case["train"]:
        return (y,)
    dz = st["dy"].float() * case["scale"]
    if case["act"] is not None:
        dz = dz * _slope(z, case["act"])
    dx = torch.matmul(dz, w.t()).to(st["x"].dtype)
    dw = torch.matmul(x.t(), dz).to(st["w"].dtype)
    return (y, dx, dw, dz.sum(dim=0)) if case["bias"] else (y, dx, dw)


# ---- the library's form -------------------------------------------------------------------------------------------------------

def _own_norm(st):
    case, ctx, x = st["case"], st["ctx"], st["x"]
    if not case["train"]:
        return (ctx.group_norm(x, st["gamma"], st["beta"], groups=case["groups"], eps=EPS, activation=case["act"]),)
    y, stats = ctx.group_norm(x, st["gamma"], st["beta"], groups=case["groups"], eps=EPS, activation=case["act"], want_stats=True)
    dx, dgamma, dbeta = ctx.group_norm_backward(st["dy"], x, st["gamma"], st["beta"], stats, activation=case["act"])
    return y, dx, dgamma, dbeta


def _own_product(st):
    case, ctx, x, w = st["case"], st["ctx"], st["x"], st["w"]
    keep = case["train"] and case["act"] is not None
    out = ctx.linear(x, w, bias=st["bias"], residual=st["residual"], activation=case["act"], scale=case["scale"], want_preact=keep)
    y, preact = out if keep else (out, None)
    if not case["train"]:
        return (y,)
    dx, dw, dbias = ctx.linear_backward(st["dy"], x, w, preact, st["bias"], activation=case["act"], scale=case["scale"], want_dbias=case["bias"])
    return (y, dx, dw, dbias) if case["bias"] else (y, dx, dw)


def run(state):
    norm = state["case"]["op"] == "group_norm"
    if own:
        return _own_norm(state) if norm else _own_product(state)
    return _plain_norm(state) if norm else _plain_product(state)


def work(case):
    s = SIZES[case["dtype"]]
    if case["op"] == "group_norm":
        e = case["n"] * case["h"] * case["w"] * case["c"]
        # forward: x in, y out; a training step also takes dy in and dx out
        return {"bytes": (4 if case["train"] else 2) * e * s + 4 * case["c"] * (4 if case["train"] else 2), "flops": (30 if case["train"] else 10) * e}
    m, k, n = case["rows"], case["k"], case["n"]
    b = (m * k + k * n + m * n * (2 if case["residual"] else 1)) * s + (4 * n if case["bias"] else 0)
    if case["train"]:
        b += (m * n + m * k + k * n) * s + (4 * n if case["bias"] else 0)
    return {"bytes": b, "flops": (6 if case["train"] else 2) * m * k * n}


# ---- values in 64 bits, from the definitions -------------------------------------------------------------------------------------

def _f64(z, act):
    """act(z) and act'(z) in float64"""
    if act is None:
        return z, torch.ones_like(z)
    if act == "tanh":
        t = torch.tanh(z)
        return t, (1 - t) * (1 + t)
    if act == "gelu":
        cdf = torch.special.ndtr(z)
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(z)
    if act == "sigmoid":
        return s, s * torch.sigmoid(-z)
    return z * s, s * (1 + z * torch.sigmoid(-z))


def _exact_norm(st, case):
    # one sample at a time: a sample's channels are independent of every other sample's
    ys, dxs, dgamma, dbeta = [], [], 0, 0
    gamma, beta = st["gamma"].double(), st["beta"].double()
    cpg = case["c"] // case["groups"]
    for i in range(case["n"]):
        x = st["x"][i].double().reshape(-1, case["c"])
        rows = x.shape[0]
        m = rows * cpg

        def spread(per_channel):                     # sums over the rows -> sums over the group, back on the channels
            return per_channel.reshape(case["groups"], cpg).sum(1).repeat_interleave(cpg)
        mean = spread(x.sum(0)) / m
        std = torch.sqrt(spread(((x - mean) ** 2).sum(0)) / m + EPS)
        xhat = (x - mean) / std
        y, slope = _f64(gamma * xhat + beta, case["act"])
        ys.append(y.reshape(st["x"].shape[1:]))
        if case["train"]:
            dz = st["dy"][i].double().reshape(rows, -1) * slope
            dbeta = dbeta + dz.sum(0)
            dgamma = dgamma + (dz * xhat).sum(0)
            t = dz * gamma
            dxs.append(((t - spread(t.sum(0)) / m - xhat * (spread((t * xhat).sum(0)) / m)) / std).reshape(st["x"].shape[1:]))
    if not case["train"]:
        return (torch.stack(ys),)
    return torch.stack(ys), torch.stack(dxs), dgamma, dbeta


def _exact_product(st, case):
    x, w = st["x"].double(), st["w"].double()
    z = torch.mm(x, w)
    if case["bias"]:
        z += st["bias"].double()
    y, slope = _f64(z, case["act"])
    y = y * case["scale"]
    if case["residual"]:
        y = y + st["residual"].double()
    if not case["train"]:
        return (y,)
    dz = st["dy"].double() * slope * case["scale"]
    dx, dw = torch.mm(dz, w.t().contiguous()), torch.mm(x.t().contiguous(), dz)
    return (y, dx, dw, dz.sum(0)) if case["bias"] else (y, dx, dw)


def exact(case, seed):
    global own
    keep, own = own, False                           # the inputs alone: no handle of the library
    try:
        st = prepare(case, seed)
    finally:
        own = keep
    return _exact_norm(st, case) if case["op"] == "group_norm" else _exact_product(st, case)
