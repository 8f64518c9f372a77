"""GPU: the channels-last layer operators (group norm with an activation; product with bias, activation and residual), forward and backward, against
their definitions in 64 bits.

Tolerances are bounds, per element, formed in 64 bits next to the reference value.  H = half a step of the result's type (finfo.eps / 2: fp32 2^-24,
fp16 2^-11, bf16 2^-8; U = 2^-24 for what is held in fp32; TINY = half the spacing of fp16 subnormals).
 * a sum of k fp32 products in any order is within (k + 2) U of the sum of their magnitudes;
 * activations are 1.13-Lipschitz (gelu; swish 1.10, the others <= 1) and their fp32 evaluation is within 64 U max(1, |z|) of |value| + U (exp with a
   relative error growing like |z|);
 * |z act''(z)| <= 0.8: a preact rounded by H moves the slope by at most 0.8 H.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U = 2.0 ** -24
DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
ACTS = [None, "relu", "swish", "sigmoid", "tanh", "gelu"]


def H(dt):
    return torch.finfo(dt).eps / 2


def TINY(dt):
    return 2.0 ** -25 if dt == torch.float16 else 0.0


@pytest.fixture(scope="module")
def ctx():
    from ttc import _lib
    return _lib.Context(win_in=44, length=1, max_windows=1)


def act64(z, act):
    """value and slope in float64"""
    if act is None:
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "tanh":
        t = torch.tanh(z)
        return t, 1 - t * t
    if act == "gelu":
        cdf = torch.special.ndtr(z)
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / np.sqrt(2 * np.pi)
    s = torch.sigmoid(z)
    return (s, s * (1 - s)) if act == "sigmoid" else (z * s, s + z * s * (1 - s))


def within(name, got, ref, tol):
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    d = (got.double() - ref).abs()
    bad = ~(d <= tol)                                   # NaN counts as bad
    assert not bool(bad.any()), f"{name}: {int(bad.sum())} of {bad.numel()} off; worst |d| {float(d.max()):.3e}, tol there {float(tol.flatten()[d.flatten().argmax()]):.3e}"


def randn(shape, dt, seed, scale=1.0, shift=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale + shift).to(dt)


# ---- group norm -------------------------------------------------------------------------------------------------------------------

def norm64(x, gamma, beta, G, eps, act):
    """y, and everything its bound and the backward pass need, in float64; x [n, rows, c]"""
    n, r, c = x.shape
    x = x.double()
    xg = x.reshape(n, r, G, c // G)
    mean = xg.mean(dim=(1, 3), keepdim=True)
    var = ((xg - mean) ** 2).mean(dim=(1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xhat = ((xg - mean) * rstd).reshape(n, r, c)
    z = xhat * gamma.double() + beta.double()
    y, slope = act64(z, act)
    # error of xhat: up to 128 rows are summed in fp32 about a sample of the data (|x - x0| <= 2 max|x - mean|), the mean is rounded to fp32
    dev = (xg - mean).abs().amax(dim=(1, 3), keepdim=True)
    k = min(128, r) + 8
    e_mean = U * (k * 2 * dev + mean.abs()) * rstd
    e_rstd = U * (k * 4 * dev * dev * rstd * rstd + 4)
    e = (e_mean + 2 * U * (xg - mean).abs() * rstd).expand(n, r, G, c // G).reshape(n, r, c) + xhat.abs() * e_rstd.expand(n, r, G, c // G).reshape(n, r, c)
    return y, slope, z, xhat, mean, rstd, e


def check_norm(ctx, x, gamma, beta, G, act, eps=1e-5, dy=None):
    """x [n, .., c] as given (any strides) -> forward and backward against float64"""
    n, c = x.shape[0], x.shape[-1]
    dt, h = x.dtype, H(x.dtype)
    g64 = torch.ones(c, device="cuda") if gamma is None else gamma
    b64 = torch.zeros(c, device="cuda") if beta is None else beta
    y, stats = ctx.group_norm(x, gamma, beta, groups=G, eps=eps, activation=act, want_stats=True)
    assert y.dtype == dt and y.shape == x.shape and y.is_contiguous()
    assert torch.equal(y, ctx.group_norm(x, gamma, beta, groups=G, eps=eps, activation=act)), "statistics asked for or not: the same bits"
    x3 = x.reshape(n, -1, c)
    ry, slope, z, xhat, mean, rstd, e = norm64(x3, g64, b64, G, eps, act)
    ez = e * g64.double().abs() + 3 * U * (z.abs() + b64.double().abs())
    within("y", y.reshape(x3.shape), ry, h * ry.abs() * (1 + h) + 1.13 * ez + 64 * U * z.abs().clamp(min=1) * (ry.abs() + U) + TINY(dt))
    within("rstd", stats[..., 1], rstd.reshape(n, G), rstd.reshape(n, G) * (U * 2) + (rstd ** 3).reshape(n, G) * U * 4 * (min(128, x3.shape[1]) + 8)
           * ((x3.double().reshape(n, -1, G, c // G) - mean).abs().amax(dim=(1, 3)) ** 2))
    if dy is None:
        return y
    dx, dg, db = ctx.group_norm_backward(dy, x, gamma, beta, stats, activation=act)
    d3 = dy.reshape(x3.shape).double()
    dz = d3 * slope
    edz = d3.abs() * (0.8 * (ez if act != "relu" else 0 * ez) + 64 * U * z.abs().clamp(min=1) * (slope.abs() + U)) + 2 * U * dz.abs()
    R = x3.shape[1]
    ks = R + 8                                                   # every sum over the rows, in any order
    within("dbeta", db, dz.sum((0, 1)), edz.sum((0, 1)) + ks * U * dz.abs().sum((0, 1)) + U)
    eb = (edz * xhat.abs() + dz.abs() * e).sum((0, 1)) + ks * U * (dz * xhat).abs().sum((0, 1))
    within("dgamma", dg, (dz * xhat).sum((0, 1)), eb + U)
    t, et = dz * g64.double(), (edz + 2 * U * dz.abs()) * g64.double().abs()
    grp = lambda a: a.reshape(n, R, G, c // G).mean(dim=(1, 3), keepdim=True).expand(n, R, G, c // G).reshape(n, R, c)      # noqa: E731
    rs = rstd.expand(n, R, G, c // G).reshape(n, R, c)
    s1, s2 = grp(t), grp(t * xhat)
    es1, es2 = grp(et) + ks * U * grp(t.abs()), grp(et * xhat.abs() + t.abs() * e) + ks * U * grp((t * xhat).abs())
    ref = rs * (t - s1 - xhat * s2)
    e_r = U * (8 + 4 * (min(128, R) + 8) * ((x3.double().reshape(n, R, G, c // G) - mean).abs().amax(dim=(1, 3), keepdim=True) * rstd) ** 2)
    e_r = e_r.expand(n, R, G, c // G).reshape(n, R, c)
    tol = h * ref.abs() * (1 + h) + rs * (et + es1 + xhat.abs() * es2 + e * s2.abs() + 6 * U * (t.abs() + s1.abs() + (xhat * s2).abs())) + e_r * rs * (
        t.abs() + s1.abs() + (xhat * s2).abs()) + TINY(dt)
    within("dx", dx.reshape(x3.shape), ref, tol)
    return y


NORM_SHAPES = [  # n, rows, channels, groups
    (1, 1, 1, 1), (2, 1, 64, 8), (3, 2, 6, 3), (1, 7, 23, 1), (2, 196, 64, 8), (5, 129, 40, 5), (2, 1000, 12, 4), (1, 5000, 64, 8), (70, 9, 16, 16),
    (2, 33, 512, 32), (1, 11, 4096, 8), (2, 3, 1000, 125), (1, 40, 2056, 8), (3, 257, 130, 2), (1, 30000, 8, 8), (2, 700, 257, 257),
    (300, 512, 64, 8),
]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", NORM_SHAPES, ids=str)
def test_group_norm(ctx, dtype, shape):
    n, r, c, G = shape
    i = NORM_SHAPES.index(shape)
    act = ACTS[(i + list(DT).index(dtype)) % len(ACTS)]
    x = randn((n, r, c), DT[dtype], i, 1.5, 0.7)
    gamma, beta = randn((c,), torch.float32, 100 + i, 0.3, 1.0), randn((c,), torch.float32, 200 + i, 0.3)
    check_norm(ctx, x, gamma, beta, G, act, dy=randn((n, r, c), DT[dtype], 300 + i))


@pytest.mark.parametrize("act", ACTS, ids=str)
@pytest.mark.parametrize("dtype", list(DT))
def test_group_norm_activations_and_no_affine(ctx, dtype, act):
    x, dy = randn((2, 13, 9, 48), DT[dtype], 1, 3.0), randn((2, 13, 9, 48), DT[dtype], 2)
    check_norm(ctx, x, None, None, 6, act, dy=dy)
    wide = randn((48,), torch.float32, 3, 20.0)                       # activations far into both tails
    check_norm(ctx, x, wide, None, 6, act, dy=dy)
    check_norm(ctx, x, None, wide, 6, act, eps=0.0, dy=dy)


@pytest.mark.parametrize("dtype", list(DT))
def test_group_norm_strided_inputs(ctx, dtype):
    wide, dwide = randn((3, 10, 7, 96), DT[dtype], 5), randn((3, 10, 7, 80), DT[dtype], 6)
    gamma, beta = randn((40,), torch.float32, 7, 0.2, 1.0), randn((40,), torch.float32, 8)
    for lo in (0, 3, 8, 56):                                          # rows that start at any element
        check_norm(ctx, wide[..., lo:lo + 40], gamma, beta, 8, "swish", dy=dwide[..., 1:41])
    check_norm(ctx, wide[:, 2:3, ::2, 8:48], gamma, beta, 8, "tanh", dy=dwide[:, 1:2, :4, :40])
    check_norm(ctx, wide.transpose(1, 2)[..., :40], gamma, beta, 8, None, dy=randn((1, 1, 1, 40), DT[dtype], 9).expand(3, 7, 10, 40))
    check_norm(ctx, wide[::2, ..., 5:45], gamma, beta, 8, "gelu", dy=dwide[:2, ..., :40])
    check_norm(ctx, wide[:, 0, 0, :40], gamma, beta, 4, "sigmoid", dy=dwide[:, 0, 0, :40])        # [n, c]: one row per sample


def test_group_norm_hard_values(ctx):
    # a mean 3000 spreads away, one outlier, and a group with no spread at all: y = act(beta) exactly there
    x = randn((2, 400, 16), torch.float32, 11, 1.0, 3000.0)
    x[0, 5, 3] = 1e6
    x[1, :, 8:12] = 0.1
    gamma, beta = randn((16,), torch.float32, 12, 0.3, 1.0), randn((16,), torch.float32, 13)
    y = check_norm(ctx, x, gamma, beta, 4, None, dy=randn((2, 400, 16), torch.float32, 14))
    assert torch.equal(y[1, :, 8:12], beta[8:12].expand(400, 4))
    # NaN / inf in one group of one sample stay in that group
    for v in (float("nan"), float("inf")):
        bad = randn((3, 50, 16), torch.float32, 15)
        bad[1, 7, 5] = v
        y = ctx.group_norm(bad, gamma, beta, groups=4)
        assert bool(y[1, :, 4:8].isnan().all())
        y[1, :, 4:8] = 0
        assert bool(y.isfinite().all())


def test_group_norm_empty(ctx):
    gamma = torch.ones(16, device="cuda")
    for shape in ((0, 5, 16), (4, 0, 16), (0, 0, 16)):
        x = torch.zeros(shape, device="cuda")
        y, stats = ctx.group_norm(x, gamma, None, groups=4, want_stats=True)
        assert y.shape == x.shape and stats.shape == (shape[0], 4, 2)
        dx, dg, db = ctx.group_norm_backward(x, x, gamma, None, stats)
        assert dx.shape == x.shape and not dg.any() and not db.any()


# ---- product -----------------------------------------------------------------------------------------------------------------------

def check_linear(ctx, x, w, bias, res, act, scale=1.0, dy=None):
    dt, h = x.dtype, H(x.dtype)
    k, n = w.shape[-2:]
    y, pre = ctx.linear(x, w, bias, res, activation=act, scale=scale, want_preact=True)
    assert y.dtype == dt and y.is_contiguous() and y.shape == x.shape[:-1] + (n,)
    assert torch.equal(y, ctx.linear(x, w, bias, res, activation=act, scale=scale)), "preact asked for or not: the same bits"
    x2, w2 = x.reshape(-1, k).double(), w.reshape(k, n).double()
    z, S = x2 @ w2, x2.abs() @ w2.abs()
    if bias is not None:
        z, S = z + bias.double(), S + bias.double().abs()
    ez = (k + 4) * U * S
    if pre is not None:
        assert pre.dtype == torch.float32 and act
        within("preact", pre.reshape(-1, n), z, ez)
    v, slope = act64(z, act)
    r = res.reshape(-1, n).double() if res is not None else torch.zeros_like(z)
    ref = r + scale * v
    e = abs(scale) * (1.13 * ez + 64 * U * z.abs().clamp(min=1) * (v.abs() + U)) + 3 * U * (r.abs() + abs(scale) * v.abs())
    within("y", y.reshape(-1, n), ref, e + h * (ref.abs() + e) + TINY(dt))
    if dy is None:
        return y
    if act:                                              # the kept argument, or the same formed again: both within the bounds
        kept = pre if pre is not None else z.float().reshape(y.shape)
        linear_grads(dy, x, w, bias, act, scale, z, slope, ez, ctx.linear_backward(dy, x, w, kept, activation=act, scale=scale))
    linear_grads(dy, x, w, bias, act, scale, z, slope, ez, ctx.linear_backward(dy, x, w, None, bias, activation=act, scale=scale))
    return y


def linear_grads(dy, x, w, bias, act, scale, z, slope, ez, got):
    dt, h = x.dtype, H(x.dtype)
    k, n = w.shape[-2:]
    x2, w2 = x.reshape(-1, k).double(), w.reshape(k, n).double()
    dx, dw, db = got
    assert dx.dtype == dt and dw.dtype == dt and dw.shape == w.shape and db.dtype == torch.float32
    d = dy.reshape(-1, n).double()
    dz = scale * d * slope
    # the slope comes from a preact off by ez; relu's is exact but where z is within its error of 0
    es = 0.8 * (ez + 2 * U * z.abs()) + 64 * U * z.abs().clamp(min=1) * (slope.abs() + U) if act not in (None, "relu") else 0 * z
    if act == "relu":
        es = (z.abs() <= ez).double()
    edz = abs(scale) * d.abs() * es + 3 * U * dz.abs()
    within("dbias", db, dz.sum(0), edz.sum(0) + (dz.shape[0] + 8) * U * dz.abs().sum(0) + U * TINY(torch.float16))
    rdz = edz + (h * (dz.abs() + edz) + TINY(dt) if act else 0)      # rounded to the type for the products
    ref = dz @ w2.t()
    e = rdz @ w2.abs().t() + (n + 4) * U * (dz.abs() @ w2.abs().t())
    within("dx", dx.reshape(-1, k), ref, e + h * (ref.abs() + e) + TINY(dt))
    ref = x2.t() @ dz
    e = x2.abs().t() @ rdz + (dz.shape[0] + 8) * U * (x2.abs().t() @ dz.abs())
    within("dw", dw.reshape(k, n), ref, e + h * (ref.abs() + e) + TINY(dt))


LIN_SHAPES = [  # rows, cin, cout
    (1, 1, 1), (1, 64, 1), (1, 1024, 4096), (2, 3, 5), (3, 17, 33), (7, 8, 16), (16, 256, 512), (17, 100, 1), (64, 64, 64), (129, 65, 127), (128, 128, 128),
    (200, 31, 200), (1000, 64, 32), (1037, 177, 93), (2500, 1, 40), (2500, 40, 1), (5000, 64, 64), (4099, 24, 8), (300, 1000, 130), (2100, 256, 128), (515, 300, 264),
]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", LIN_SHAPES, ids=str)
def test_linear(ctx, dtype, shape):
    m, k, n = shape
    i = LIN_SHAPES.index(shape)
    act = ACTS[(i + list(DT).index(dtype)) % len(ACTS)]
    dt = DT[dtype]
    check_linear(ctx, randn((m, k), dt, i), randn((k, n), dt, 50 + i, k ** -0.5), randn((n,), torch.float32, 100 + i, 0.3) if i % 3 else None,
                 randn((m, n), dt, 150 + i) if i % 2 else None, act, scale=(1.0, 0.1)[i // 2 % 2], dy=randn((m, n), dt, 200 + i))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", [(9999, 64, 640), (9999, 640, 64), (64, 9996, 640), (3333, 128, 3848), (3333, 3848, 128), (192, 3336, 3848), (1000, 12352, 1000), (3584, 64, 4096)], ids=str)
def test_linear_wide(ctx, dtype, shape):
    """products of many 256 x 256 or 256 x 128 tiles, ragged at the far edges: in y, in dx, in dw, with the contracted index split; the strided and the
    misaligned call give the aligned call's bits or stay within the bounds"""
    m, k, n = shape
    dt = DT[dtype]
    x, w, dy = randn((m, k), dt, 1), randn((k, n), dt, 2, k ** -0.5), randn((m, n), dt, 3)
    bias, res = randn((n,), torch.float32, 4, 0.3), randn((m, n), dt, 5)
    y = check_linear(ctx, x, w, bias, res, "swish", scale=0.5, dy=dy)
    ws, xs = randn((k, n + 24), dt, 6)[:, 8:n + 8], randn((m, k + 16), dt, 7)[:, 16:]
    ws.copy_(w), xs.copy_(x)
    assert torch.equal(y, ctx.linear(xs, ws, bias, res, activation="swish", scale=0.5))
    off = randn((m, k + 3), dt, 8)[:, 3:]
    off.copy_(x)
    check_linear(ctx, off, w, bias, res, "swish", scale=0.5)


@pytest.mark.parametrize("rows", list(range(1, 19)) + [31, 33, 63, 65])
def test_linear_row_counts(ctx, rows):
    """every count of a few rows, which take paths of their own, at sizes with and without whole vectors"""
    for j, (dtype, k, n) in enumerate((("bf16", 192, 136), ("fp16", 77, 51), ("fp32", 130, 70), ("bf16", 520, 8))):
        check_linear(ctx, randn((rows, k), DT[dtype], rows), randn((k, n), DT[dtype], j, k ** -0.5), randn((n,), torch.float32, 3), randn((rows, n), DT[dtype], 4),
                     "swish", dy=randn((rows, n), DT[dtype], 5))


@pytest.mark.parametrize("act", ACTS, ids=str)
@pytest.mark.parametrize("dtype", list(DT))
def test_linear_activations(ctx, dtype, act):
    dt = DT[dtype]
    for scale in (6.0, 0.02):                                          # far into both tails; next to 0
        check_linear(ctx, randn((150, 72), dt, 1, scale), randn((72, 56), dt, 2, 0.3), randn((56,), torch.float32, 3, 0.01), None, act, scale=-0.5,
                     dy=randn((150, 56), dt, 4))


@pytest.mark.parametrize("dtype", list(DT))
def test_linear_strided_inputs(ctx, dtype):
    dt = DT[dtype]
    wide, wres, wdy = randn((3, 11, 5, 90), dt, 1), randn((3, 11, 5, 70), dt, 2), randn((3, 11, 5, 61), dt, 3)
    wts, bias = randn((48, 99), dt, 4, 0.2), randn((40,), torch.float32, 5)
    for lo in (0, 1, 8, 42):
        check_linear(ctx, wide[..., lo:lo + 48], wts[:, lo:lo + 40], bias, wres[..., 3:43], "tanh", dy=wdy[..., 2:42])
    check_linear(ctx, wide[:, ::2, 1, :48], wts[:, :40], bias, wres[:, ::2, 1, :40], "swish", dy=wdy[:, ::2, 0, :40])
    check_linear(ctx, wide.transpose(0, 1)[..., :48], randn((40, 48), dt, 6, 0.2).t(), None, None, None, dy=randn((1, 1, 1, 40), dt, 7).expand(11, 3, 5, 40))
    check_linear(ctx, wide[0, 0, 0, :48], wts[:, :40].reshape(1, 1, 48, 40), bias, None, "gelu", dy=wdy[0, 0, 0, :40])       # one vector, TF kernel


def test_linear_hard_values(ctx):
    # NaN and inf stay in their row
    for dt in DT.values():
        x, w = randn((40, 30), dt, 1), randn((30, 20), dt, 2)
        x[3, 4], x[9, 0] = float("nan"), float("inf")
        y = ctx.linear(x, w)
        ok = torch.ones(40, dtype=torch.bool, device="cuda")
        ok[[3, 9]] = False
        assert bool(y[3].isnan().all()) and not bool(y[9].isfinite().any()) and bool(y[ok].isfinite().all())
    # fp16: an argument past the type's range or below its smallest value keeps its side of 0 and a finite slope, kept or formed again
    x = torch.tensor([[300.0], [-300.0], [1e-4], [-1e-4]], device="cuda").half()
    w = torch.tensor([[300.0, 1e-4]], device="cuda").half()
    for act in ("swish", "gelu", "tanh", "sigmoid", "relu"):
        for kept in (None, x.float() * w.float()):
            dx, dw, db = ctx.linear_backward(torch.ones(4, 2, device="cuda").half(), x, w, kept, activation=act)
            assert bool(dx.isfinite().all()) and bool(dw.isfinite().all()) and bool(db.isfinite().all())
            if act == "relu":
                assert torch.equal(db, torch.full_like(db, 2.0))


def test_linear_empty(ctx):
    for shape in ((0, 12), (3, 0, 12)):
        x, w = torch.zeros(shape, device="cuda"), torch.ones(12, 5, device="cuda")
        y, pre = ctx.linear(x, w, torch.ones(5, device="cuda"), activation="tanh", want_preact=True)
        assert y.shape == shape[:-1] + (5,)
        dx, dw, db = ctx.linear_backward(y, x, w, pre, activation="tanh")
        assert dx.shape == x.shape and not dw.any() and not db.any()


def test_outputs_not_wanted(ctx):
    for k, n in ((24, 12), (300, 280)):                  # a narrow layer and a wide one
        x, w, dy = randn((50, k), torch.float32, 1), randn((k, n), torch.float32, 2), randn((50, n), torch.float32, 3)
        _, pre = ctx.linear(x, w, activation="tanh", want_preact=True)
        full = ctx.linear_backward(dy, x, w, pre, activation="tanh")
        for keep in range(8):
            got = ctx.linear_backward(dy, x, w, pre, activation="tanh", want_dx=bool(keep & 1), want_dw=bool(keep & 2), want_dbias=bool(keep & 4))
            for i in range(3):
                assert (got[i] is None) if not keep >> i & 1 else torch.equal(got[i], full[i])
    xs, g, b = randn((2, 30, 24), torch.float32, 4), randn((24,), torch.float32, 5), randn((24,), torch.float32, 6)
    _, st = ctx.group_norm(xs, g, b, 4, activation="tanh", want_stats=True)
    full = ctx.group_norm_backward(xs, xs, g, b, st, activation="tanh")
    for keep in range(8):
        got = ctx.group_norm_backward(xs, xs, g, b, st, activation="tanh", want_dx=bool(keep & 1), want_dgamma=bool(keep & 2), want_dbeta=bool(keep & 4))
        for i in range(3):
            assert (got[i] is None) if not keep >> i & 1 else torch.equal(got[i], full[i])


# ---- refusals, streams, graphs -------------------------------------------------------------------------------------------------------

def test_refusals_on_the_device(ctx):
    x, w = torch.zeros(6, 16, device="cuda"), torch.zeros(16, 8, device="cuda")
    for call in (lambda: ctx.linear(x.cpu(), w), lambda: ctx.linear(x, w.half()), lambda: ctx.linear(x, w, bias=torch.zeros(7, device="cuda")),
                 lambda: ctx.linear(x, w, residual=torch.zeros(6, 7, device="cuda")), lambda: ctx.linear(x, w, residual=torch.zeros(6, 8, device="cuda").half()),
                 lambda: ctx.linear(x, w, activation="softplus"), lambda: ctx.linear_backward(torch.zeros(6, 8, device="cuda"), x, w, torch.zeros(6, 8, device="cuda").half(), activation="swish"),
                 lambda: ctx.linear_backward(torch.zeros(6, 8, device="cuda"), x, w, None, torch.zeros(9, device="cuda"), activation="swish"),
                 lambda: ctx.linear_backward(torch.zeros(6, 7, device="cuda"), x, w), lambda: ctx.group_norm(x, torch.ones(8, device="cuda")),
                 lambda: ctx.group_norm_backward(x, x, None, None, torch.zeros(5, 8, 2, device="cuda")),
                 lambda: ctx.group_norm_backward(x.half(), x, None, None, torch.zeros(6, 8, 2, device="cuda"))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: ctx.group_norm(x, groups=5), lambda: ctx.group_norm(x, groups=0), lambda: ctx.group_norm(x, eps=float("nan")),
                 lambda: ctx.linear(x, w, scale=float("nan")), lambda: ctx.linear(torch.zeros(6, 0, device="cuda"), torch.zeros(0, 8, device="cuda"))):
        with pytest.raises(RuntimeError, match="status 1"):
            call()
    # the C entries themselves: null pointers and a short workspace are errors, not launches
    import ctypes as C
    from ttc import _lib
    lib, p = ctx.lib, x.data_ptr()
    d = _lib.TTCGroupNormDesc(0, 0, 1, 1 << 20, 16, 4, 96, 16, 1e-5)         # long enough to need scratch memory
    assert lib.ttc_group_norm(ctx._h, C.byref(d), p, None, None, p, None, p, 8, None) == 1 and b"workspace" in lib.ttc_last_error(ctx._h)
    assert lib.ttc_group_norm(ctx._h, C.byref(d), None, None, None, p, None, p, 1 << 20, None) == 1
    assert lib.ttc_group_norm_backward(ctx._h, C.byref(d), p, 96, 16, p, None, None, p, p, None, None, p, 8, None) == 1 and b"workspace" in lib.ttc_last_error(ctx._h)
    assert lib.ttc_group_norm(ctx._h, C.byref(d), p, None, None, p, None, p + 4, 1 << 30, None) == 1 and b"aligned" in lib.ttc_last_error(ctx._h)
    d = _lib.TTCGroupNormDesc(0, 0, 1, 6, 16, 4, 96, 16, 1e-5)
    assert lib.ttc_group_norm(ctx._h, C.byref(d), None, None, None, p, None, p, 1 << 20, None) == 1
    assert lib.ttc_group_norm_backward(ctx._h, C.byref(d), p, 96, 16, p, None, None, None, p, None, None, p, 1 << 20, None) == 1
    l = _lib.TTCLinearDesc(0, 2, 6, 16, 8, 16, 8, 8, 8, 1.0)
    assert lib.ttc_linear(ctx._h, C.byref(l), None, p, None, None, p, None, None, 0, None) == 1
    assert lib.ttc_linear_backward(ctx._h, C.byref(l), p, p, None, None, None, p, p, None, p, 1 << 20, None) == 1
    for px, pw, dx, dw in ((None, p, p, None), (p, None, None, p)):          # one gradient alone: the narrow pass still reads all three arrays
        l.activation = 0
        assert lib.ttc_linear_backward(ctx._h, C.byref(l), p, px, pw, None, None, dx, dw, None, p, 1 << 20, None) == 1 and b"null" in lib.ttc_last_error(ctx._h)
        l.activation = 2
    assert lib.ttc_linear_backward(ctx._h, C.byref(l), p, p, p, None, None, p, p, p, p, 1, None) == 1 and b"workspace" in lib.ttc_last_error(ctx._h)
    assert lib.ttc_linear_backward(ctx._h, C.byref(l), p, p, p, None, None, p, p, p, p + 8, 1 << 30, None) == 1 and b"aligned" in lib.ttc_last_error(ctx._h)
    torch.cuda.synchronize()


def test_two_runs_give_the_same_bits(ctx):
    x, w, dy = randn((40000, 64), torch.bfloat16, 1), randn((64, 48), torch.bfloat16, 2, 0.1), randn((40000, 48), torch.bfloat16, 3)
    xs, g = randn((3, 9000, 64), torch.float32, 4), randn((64,), torch.float32, 5)

    def once():
        y, pre = ctx.linear(x, w, activation="swish", want_preact=True)
        z, st = ctx.group_norm(xs, g, None, activation="tanh", want_stats=True)
        return (y,) + ctx.linear_backward(dy, x, w, pre, activation="swish") + (z, st) + ctx.group_norm_backward(xs, xs, g, None, st, activation="tanh")
    a, b = once(), once()
    assert all(torch.equal(u, v) for u, v in zip(a, b))


def _block(ctx, x, p, dy):
    """a residual block of the two operators, forward and backward, with explicit calls"""
    h, pre = ctx.linear(x, p["w1"], p["b1"], activation="swish", want_preact=True)
    nrm, st = ctx.group_norm(h, p["g"], p["be"], groups=8, activation="tanh", want_stats=True)
    y = ctx.linear(nrm, p["w2"], p["b2"], residual=x, scale=0.1)
    dn, dw2, db2 = ctx.linear_backward(dy, nrm, p["w2"], scale=0.1)
    dh, dg, dbe = ctx.group_norm_backward(dn, h, p["g"], p["be"], st, activation="tanh")
    dx, dw1, db1 = ctx.linear_backward(dh, x, p["w1"], pre, p["b1"], activation="swish")
    return [y, dx + dy, dw1, db1, dg, dbe, dw2, db2]


def _block_params(dt, cin=64, mid=96):
    return dict(w1=randn((cin, mid), dt, 1, cin ** -0.5), b1=randn((mid,), torch.float32, 2, 0.1), g=randn((mid,), torch.float32, 3, 0.1, 1.0),
                be=randn((mid,), torch.float32, 4, 0.1), w2=randn((mid, cin), dt, 5, mid ** -0.5), b2=randn((cin,), torch.float32, 6, 0.1))


def test_block_on_another_stream_and_in_two_graphs(ctx):
    """two graphs captured from one context, replayed in turn and at once on two streams, between eager calls: every replay equals the eager result"""
    dt = torch.bfloat16
    p = _block_params(dt)
    xs = [randn((2, 30, 31, 64), dt, 10 + i) for i in range(2)]
    dys = [randn((2, 30, 31, 64), dt, 20 + i) for i in range(2)]
    want = [_block(ctx, x, p, dy) for x, dy in zip(xs, dys)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _block(ctx, xs[0], p, dys[0])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    graphs, outs = [], []
    for x, dy in zip(xs, dys):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_block(ctx, x, p, dy))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for rep in range(4):
        for o in outs:
            for a in o:
                a.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            if rep % 2:
                g.replay()
            else:
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for o, r in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(o, r))
        again = _block(ctx, xs[rep % 2], p, dys[rep % 2])
        assert all(torch.equal(a, b) for a, b in zip(again, want[rep % 2]))


# ---- autograd, and the operators on the model's own features ---------------------------------------------------------------------------

def test_autograd_block_matches_formula_and_differences(ctx):
    p = {k: v.requires_grad_() for k, v in _block_params(torch.float32, 16, 24).items()}
    x = randn((2, 6, 5, 16), torch.float32, 30).requires_grad_()
    dy = randn((2, 6, 5, 16), torch.float32, 31)

    def fwd(x, p):
        h = ctx.linear(x, p["w1"], p["b1"], activation="swish")
        return ctx.linear(ctx.group_norm(h, p["g"], p["be"], activation="tanh"), p["w2"], p["b2"], residual=x, scale=0.1)

    def ref(x, p):
        x = x.double()
        q = {k: v.double() for k, v in p.items()}
        z = x @ q["w1"] + q["b1"]
        h = z * torch.sigmoid(z)
        g = h.reshape(2, -1, 8, 3)
        m = g.mean((1, 3), keepdim=True)
        g = ((g - m) / torch.sqrt(((g - m) ** 2).mean((1, 3), keepdim=True) + 1e-5)).reshape(h.shape)
        return x + 0.1 * (torch.tanh(g * q["g"] + q["be"]) @ q["w2"] + q["b2"])
    y = fwd(x, p)
    (y * dy).sum().backward()
    got = {k: v.grad.clone() for k, v in list(p.items()) + [("x", x)]}
    x.grad = None
    for v in p.values():
        v.grad = None
    (ref(x, p) * dy).sum().backward()
    for k, v in list(p.items()) + [("x", x)]:
        # 60 rows of O(1) values through three layers of up to 24 products each, every one within 100 U of its magnitude sums
        assert float((got[k] - v.grad).abs().max()) <= 1e-4 * float(v.grad.abs().max()), k
    # against central differences of the operators' own float64 definition along one direction
    with torch.no_grad():
        t, h = {k: randn(v.shape, torch.float32, 40) for k, v in p.items()}, 1e-4
        up, dn = ({k: v.double() + s * h * t[k].double() for k, v in p.items()} for s in (1, -1))
        num = float(((ref(x, up) - ref(x, dn)) * dy).sum()) / (2 * h)
        ana = sum(float((got[k].double() * t[k].double()).sum()) for k in p)
    mag = sum(float((got[k].double() * t[k].double()).abs().sum()) for k in p)
    assert abs(num - ana) <= 1e-4 * mag                       # h^2 truncation 1e-8, gradients within 1e-4
    # one input alone; a leaf of another type gets its own type back
    b = torch.zeros(24, device="cuda", dtype=torch.float16, requires_grad=True)
    ctx.linear(x.detach(), p["w1"].detach(), b).sum().backward()
    assert b.grad.dtype == torch.float16 and torch.equal(b.grad, torch.full_like(b.grad, 60.0))
    for call in (lambda: ctx.linear(x, p["w1"], want_preact=True), lambda: ctx.group_norm(x, want_stats=True)):
        with pytest.raises(ValueError, match="autograd"):
            call()


def test_recording_gradients_in_a_capture_is_refused(ctx):
    x, w = randn((8, 16), torch.float32, 1).requires_grad_(), randn((16, 8), torch.float32, 2)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="capture"):
            ctx.linear(x, w)
        with pytest.raises(RuntimeError, match="capture"):
            ctx.group_norm(x)
        with torch.no_grad():
            y = ctx.linear(x, w)
    for _ in range(3):
        y.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ctx.linear(x.detach(), w))


def test_head_on_exported_features_is_the_models_own(ctx):
    """linear(late features, head) = the probabilities of the same forward pass; the graph's head is this 1x1 convolution"""
    from tests.helpers import synth
    from ttc import _lib, weights as Wt
    w = Wt.synth_weights(0)
    m = _lib.Context(win_in=44, length=1, max_windows=2)
    m.load_weights(w)
    probs, early, late = m.forward_taps(synth.synth_windows(seed=1, N=2, L=1, W=44))
    got = m.linear(late, w["head/kernel"], w["head/bias"], activation="sigmoid")[..., 0]
    z = (late.double() * torch.from_numpy(w["head/kernel"][0, 0, :, 0]).cuda().double()).abs().sum(-1)
    # both sum the same 64 fp32 products in their own order (66 U of the magnitudes each) and sigmoid's slope is at most 1/4
    assert bool(((got - probs).abs().double() <= 2 * 0.25 * 66 * U * (z + 3) + 8 * U).all())
    # a head of another kind on the recurrent features, in 16 bits: norm, product, norm -- as a fine-tune would
    f = early.bfloat16()
    k = randn((64, 32), torch.bfloat16, 3, 0.125)
    out = m.linear(m.group_norm(f, groups=8, activation="swish"), k, activation="gelu")
    assert out.shape == early.shape[:-1] + (32,) and bool(out.isfinite().all())
