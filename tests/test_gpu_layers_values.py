"""GPU: the channels-last layer operators where a wrong value hides inside a wide tolerance -- gradients of 16-bit arrays held to their own final rounding.

The bounds are formed as in test_gpu_layers (H, U, TINY: half a step of the result's type, 2^-24, half the spacing of fp16 subnormals)."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from tests.test_gpu_layers import DT, H, TINY, U, act64, check_norm, randn, within      # noqa: E402


@pytest.fixture(scope="module")
def ctx():
    from ttc import _lib
    return _lib.Context(win_in=44, length=1, max_windows=1)


# ---- product: dz = dy act'(z) keeps more bits than the arrays' type --------------------------------------------------------------------

def check_grads(dy, x, w, bias, act, scale, got):
    """linear_backward's gradients with dz as a pair of 16-bit values: hi within H, what is left within H again (bf16 2^-16 in all, fp16 2^-22), fp16 no
    finer than 2^-35 (half the spacing of the low half, 2^-25, is 2^-11 of its own scale, twice that for the halved value); in fp16 x as factor of the low
    half may be off by 2^-25 against a factor of at most |dz| / 2, twice that again for the halved value"""
    dt, h = x.dtype, H(x.dtype)
    x2, w2, d = x.double(), w.double(), dy.double()
    z, S = x2 @ w2 + bias.double(), x2.abs() @ w2.abs() + bias.double().abs()
    ez = (x.shape[1] + 4) * U * S
    _, slope = act64(z, act)
    dz = scale * d * slope
    e = abs(scale) * d.abs() * (0.8 * (ez + 2 * U * z.abs()) + 64 * U * z.abs().clamp(min=1) * (slope.abs() + U)) + 3 * U * dz.abs()
    e = e + h * h * (dz.abs() + e) + (2.0 ** -35 * abs(scale) if dt == torch.float16 else 0.0)
    dx, dw, db = got
    n, m = w.shape[1], x.shape[0]
    ref = dz @ w2.t()
    b = e @ w2.abs().t() + (2 * n + 8) * U * (dz.abs() @ w2.abs().t())
    within("dx", dx, ref, b + h * (ref.abs() + b) + TINY(dt))
    ref = x2.t() @ dz
    b = x2.abs().t() @ e + (2 * m + 8) * U * (x2.abs().t() @ dz.abs()) + (2.0 ** -25 * dz.abs().sum(0) if dt == torch.float16 else 0.0)
    within("dw", dw, ref, b + h * (ref.abs() + b) + TINY(dt))
    within("dbias", db, dz.sum(0), e.sum(0) + (m + 8) * U * dz.abs().sum(0) + U * TINY(torch.float16))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("shape", [(640, 64, 64), (700, 50, 33), (301, 40, 128), (301, 128, 40), (77, 64, 1), (900, 61, 30), (333, 64, 32), (600, 177, 93), (515, 300, 264), (300, 264, 1024),
                                   (1024, 65, 129), (6400, 640, 128), (128, 6400, 640), (64, 2048, 2048), (2048, 2048, 64)], ids=str)
def test_linear_gradients_are_rounded_once(ctx, dtype, shape):
    m, k, n = shape
    dt, act = DT[dtype], ("swish", "sigmoid", "gelu", "tanh")[(m + k + n) % 4]
    x, w, dy, bias = randn((m, k), dt, 1), randn((k, n), dt, 2, k ** -0.5), randn((m, n), dt, 3), randn((n,), torch.float32, 4, 0.3)
    _, pre = ctx.linear(x, w, bias, activation=act, want_preact=True)
    for kept in {id(None): None, id(pre): pre}.values():
        check_grads(dy, x, w, bias, act, 0.5, ctx.linear_backward(dy, x, w, kept, bias, activation=act, scale=0.5))


@pytest.mark.parametrize("shape", [(2000, 64, 64), (2000, 60, 40), (2000, 177, 93), (128, 6400, 640)], ids=str)
def test_linear_fp16_slopes_below_and_above_the_types_range(ctx, shape):
    m, k, n = shape
    # dy act' about 1e-7, below fp16's smallest normal value: sums over many rows are not
    x, w, dy = randn((m, k), torch.float16, 1, 8.0), randn((k, n), torch.float16, 2, 0.02 * k ** -0.5), randn((m, n), torch.float16, 3, 1e-3)
    bias = randn((n,), torch.float32, 4, 0.3, 9.0)
    _, pre = ctx.linear(x, w, bias, activation="sigmoid", want_preact=True)
    check_grads(dy, x, w, bias, "sigmoid", 1.0, ctx.linear_backward(dy, x, w, pre, bias, activation="sigmoid"))
    # dy act' past its largest value, gradients well inside
    x, w = randn((m, k), torch.float16, 5, 1e-4), randn((k, n), torch.float16, 6, 1e-3)
    bias, dy = torch.full((n,), 1.4, device="cuda"), torch.full((m, n), 64000.0, device="cuda", dtype=torch.float16)
    _, pre = ctx.linear(x, w, bias, activation="gelu", want_preact=True)
    check_grads(dy, x, w, bias, "gelu", 1.0, ctx.linear_backward(dy, x, w, pre, bias, activation="gelu"))


# ---- infinities and NaN in the backward passes -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("act", ["relu", "sigmoid", "tanh"])
def test_linear_gradients_of_rows_with_infinities_and_nan(ctx, dtype, act):
    """an infinite x has an infinite argument and a slope of 0 or 1: that row's dx is finite, at widths with and without padded columns alike; a NaN stays in
    its row, and neither reaches another row"""
    dt = DT[dtype]
    for m, k, n in ((100, 64, 64), (100, 64, 1), (100, 64, 20), (101, 50, 33), (70, 33, 63), (90, 64, 128), (90, 128, 50), (150, 200, 150), (2, 64, 5)):
        x, w, dy = randn((m, k), dt, 1), randn((k, n), dt, 2, k ** -0.5), randn((m, n), dt, 3)
        w = torch.where(w == 0, torch.ones_like(w), w)
        bias = randn((n,), torch.float32, 4, 0.3)
        bad = x.clone()
        rows = {0: float("inf"), m - 1: float("nan")} if m < 50 else {3: float("inf"), 17: float("-inf"), m - 1: float("inf"), 40: float("nan")}
        for r, v in rows.items():
            bad[r, (7 * r) % k] = v
        pre = bad.double() @ w.double() + bias.double()
        dx0, _, _ = ctx.linear_backward(dy, x, w, None, bias, activation=act)
        for kept in (None, pre.float()):
            dx, dw, db = ctx.linear_backward(dy, bad, w, kept, bias, activation=act)
            slope = {"relu": (pre > 0).double(), "sigmoid": torch.zeros_like(pre), "tanh": torch.zeros_like(pre)}[act]
            for r, v in rows.items():
                if v != v:
                    assert bool(dx[r].isnan().all()), (m, k, n, r)
                    continue
                assert bool(pre[r].isinf().all())
                dz = dy[r].double() * slope[r]
                ref, mag = dz @ w.double().t(), dz.abs() @ w.double().abs().t()
                within(f"dx of row {r} of {(m, k, n)}", dx[r], ref, (n + 8) * U * mag + H(dt) * (ref.abs() + (n + 8) * U * mag) + TINY(dt))
            if kept is None:
                others = [r for r in range(m) if r not in rows]
                assert torch.equal(dx[others], dx0[others])


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("rows", [50, 40000])
def test_group_norm_gradients_of_a_group_with_nan(ctx, dtype, rows):
    """NaN and infinities stay in their sample's group, and in the parameter gradients of its channels: one launch and several"""
    dt = DT[dtype]
    x, dy, gamma = randn((3, rows, 16), dt, 1), randn((3, rows, 16), dt, 2), randn((16,), torch.float32, 3)
    for v in (float("nan"), float("inf")):
        bad = x.clone()
        bad[1, 7, 5] = v
        _, st = ctx.group_norm(bad, gamma, None, groups=4, activation="tanh", want_stats=True)
        dx, dg, db = ctx.group_norm_backward(dy, bad, gamma, None, st, activation="tanh")
        assert bool(dx[1, :, 4:8].isnan().all()) and bool(dg[4:8].isnan().all()) and bool(db[4:8].isnan().all())
        dx[1, :, 4:8], dg[4:8], db[4:8] = 0, 0, 0
        assert bool(dx.isfinite().all()) and bool(dg.isfinite().all()) and bool(db.isfinite().all())


# ---- group norm: sums over many rows ---------------------------------------------------------------------------------------------------

def test_group_norm_gradients_of_many_samples_of_many_rows(ctx):
    """one large dy and 16383 small ones per channel: a 32-bit run of all rows drops every small one (2^14 + 2^-11 is 2^14 there).  513 samples, the number
    from which their count alone fills the chip; they are one sample read 513 times (sample stride 0)"""
    n, rows, c = 513, 16384, 2048
    dy = torch.full((1, rows, c), 2.0 ** -11, device="cuda", dtype=torch.float16)
    dy[:, 0] = 2.0 ** 14
    x = torch.ones((1, rows, c), device="cuda", dtype=torch.float16)
    x[:, 1::2] = -1.0                                             # mean 0, variance 1
    st = torch.zeros((n, 8, 2), device="cuda")
    st[..., 1] = (1 + 1e-5) ** -0.5
    dx, dg, db = ctx.group_norm_backward(dy.expand(n, rows, c), x.expand(n, rows, c), None, None, st, want_dx=False)
    assert dx is None
    d = dy[0].double()
    tol = (512 + 16) * U * n * d.abs().sum(0)                     # runs of 512 rows in any order; everything joined is in 64 bits
    within("dbeta", db, n * d.sum(0), tol)
    within("dgamma", dg, n * float(st[0, 0, 1]) * (d * x[0].double()).sum(0), tol)


# ---- the ends of the sizes -------------------------------------------------------------------------------------------------------------

def test_linear_gradient_of_no_rows_at_the_largest_weights(ctx):
    w = torch.empty((65536, 65536), device="cuda", dtype=torch.bfloat16)
    x = torch.empty((0, 65536), device="cuda", dtype=torch.bfloat16)
    dx, dw, db = ctx.linear_backward(x, x, w, None, None)
    assert dx.shape == x.shape and dw.shape == w.shape and not db.any()
    assert not any(bool(part.any()) for part in dw.split(8192))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", [(32, 784, 64, 8), (32, 841, 64, 8), (32, 961, 64, 8), (32, 1024, 64, 8), (32, 1025, 64, 8), (8, 480, 128, 8), (8, 481, 128, 8),
                                   (1, 500, 64, 8), (257, 16, 64, 8)], ids=str)
def test_group_norm_both_sides_of_one_launch(ctx, dtype, shape):
    """sizes next to the ones from which a sample is no longer held by one workgroup"""
    n, r, c, G = shape
    x, gamma, beta = randn((n, r, c), DT[dtype], 1, 1.5, 0.7), randn((c,), torch.float32, 2, 0.3, 1.0), randn((c,), torch.float32, 3, 0.3)
    check_norm(ctx, x, gamma, beta, G, "swish", dy=randn((n, r, c), DT[dtype], 4))


# ---- whole numbers: every sum is exact in 32 bits, so every result is the exact value rounded once, and one lost row or column shows ---------------------

def ints(shape, dt, seed, hi=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-hi, hi + 1, shape, generator=g, device="cuda").to(dt)


def exact_linear(ctx, x, w, bias, res, act, dy):
    """x, w, dy, res, bias of whole numbers, act None or relu: bits of y, dx, dw, dbias"""
    dt = x.dtype
    y, pre = ctx.linear(x, w, bias, res, activation=act, want_preact=True)
    z = x.double() @ w.double() + bias.double()
    v = z.clamp(min=0) if act else z
    assert torch.equal(y, (v + (0 if res is None else res.double())).to(dt))
    dz = dy.double() * ((z > 0) if act else 1)
    ref = ((dz @ w.double().t()).to(dt), (x.double().t() @ dz).to(dt), dz.sum(0).float())
    for kept in ([pre, None] if pre is not None else [None]):
        for got, want, name in zip(ctx.linear_backward(dy, x, w, kept, bias, activation=act), ref, ("dx", "dw", "dbias")):
            assert torch.equal(got, want), (name, tuple(x.shape), tuple(w.shape), int((got != want).sum()))


INT_SHAPES = [(2500, 64, 64), (4099, 64, 48), (30000, 64, 1), (30000, 50, 33), (4099, 24, 128), (2500, 128, 60), (2500, 177, 93), (9999, 256, 128), (4099, 300, 264),
              (100, 5000, 60), (37, 70, 9000), (9999, 64, 640), (9984, 64, 640), (128, 6400, 640), (6400, 640, 128), (1, 1000, 999), (3, 999, 64), (8, 513, 77)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", INT_SHAPES, ids=str)
def test_linear_whole_numbers(ctx, dtype, shape):
    m, k, n = shape
    dt = DT[dtype]
    for act in (None, "relu"):
        exact_linear(ctx, ints((m, k), dt, 1), ints((k, n), dt, 2), ints((n,), torch.float32, 3, 3), ints((m, n), dt, 4) if n % 2 else None, act, ints((m, n), dt, 5))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", [(1000, 64, 64), (2500, 177, 93), (2500, 300, 264), (2560, 320, 1024), (6400, 640, 128)], ids=str)
def test_linear_whole_numbers_in_rows_of_wider_arrays(ctx, dtype, shape):
    """x, w, residual and dy as slices that start anywhere, at narrow, ordinary and wide sizes"""
    m, k, n = shape
    dt = DT[dtype]
    for lo, act in ((0, None), (8, "relu"), (3, None), (5, "relu")):
        x, w = ints((m, k + 24), dt, 1)[:, lo:lo + k], ints((k, n + 16), dt, 2)[:, lo:lo + n]
        exact_linear(ctx, x, w, ints((n,), torch.float32, 3, 3), ints((m, n + 40), dt, 4)[:, lo:lo + n], act, ints((m, n + 8 + lo), dt, 5)[:, 8:8 + n])


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", [(1, 2500, 64, 8), (3, 4099, 40, 5), (2, 9999, 24, 2), (1, 30000, 8, 4), (1, 30001, 64, 8), (40, 784, 64, 8), (300, 33, 256, 32),
                                   (1, 777, 1030, 5), (600, 2000, 8, 1)], ids=str)
def test_group_norm_whole_numbers(ctx, dtype, shape):
    """x is 1 and -1 in neighbouring channels: mean 0, variance 1 and, without eps, x itself normalised; dbeta and dgamma are whole sums"""
    n, r, c, G = shape
    dt = DT[dtype]
    x = torch.ones((n, r, c), device="cuda")
    x[..., 1::2] = -1
    x = (x * (2 * ints((n, r, 1), torch.float32, 1).clamp(min=0) - 1)).to(dt)
    y, st = ctx.group_norm(x, groups=G, eps=0.0, want_stats=True)
    assert torch.equal(y, x) and not st[..., 0].any() and bool((st[..., 1] == 1).all())
    dy = ints((n, r, c), dt, 2)
    _, dg, db = ctx.group_norm_backward(dy, x, None, None, st)
    assert torch.equal(db, dy.double().sum((0, 1)).float()) and torch.equal(dg, (dy.double() * x.double()).sum((0, 1)).float())
    assert ctx.group_norm_backward(dy, x, None, None, st, want_dx=False)[1].equal(dg)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 29584, 512, 32), (1, 14000, 512, 512), (1, 3000, 4096, 32), (1, 3000, 2049, 2049)], ids=str)
def test_group_norm_of_one_sample_with_many_groups(ctx, dtype, shape):
    n, r, c, G = shape
    x, gamma, beta = randn((n, r, c), DT[dtype], 1, 1.5, 0.7), randn((c,), torch.float32, 2, 0.3, 1.0), randn((c,), torch.float32, 3, 0.3)
    check_norm(ctx, x, gamma, beta, G, "swish", dy=randn((n, r, c), DT[dtype], 4))


# ---- autograd in every type, narrow and wide, on slices: the gradients of the explicit calls ---------------------------------------------------

@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", [(64, 24), (64, 1), (200, 136)], ids=str)
def test_autograd_gives_the_explicit_calls_gradients(ctx, dtype, shape):
    k, n = shape
    dt = DT[dtype]
    wide = randn((2, 9, 31, k + 16), dt, 1)
    for lo in (0, 3, 8):
        x = wide[..., lo:lo + k].detach().requires_grad_()
        w, bias = randn((k, n), dt, 2, k ** -0.5).requires_grad_(), randn((n,), torch.float32, 3, 0.3).requires_grad_()
        gamma, beta = randn((k,), torch.float32, 4, 0.3, 1.0).requires_grad_(), randn((k,), torch.float32, 5).requires_grad_()
        res = randn((2, 9, 31, n), dt, 6).requires_grad_()
        dy = randn((2, 9, 31, n + 4), dt, 7)[..., 4:]
        assert not x.is_contiguous()
        h = ctx.group_norm(x, gamma, beta, groups=8, activation="swish")
        y = ctx.linear(h, w, bias, residual=res, activation="tanh", scale=0.5)
        y.backward(dy)
        with torch.no_grad():
            h2, st = ctx.group_norm(x, gamma, beta, groups=8, activation="swish", want_stats=True)
            y2, pre = ctx.linear(h2, w, bias, residual=res, activation="tanh", scale=0.5, want_preact=True)
            dh, dw, db = ctx.linear_backward(dy, h2, w, pre, bias, activation="tanh", scale=0.5)
            dx, dg, dbe = ctx.group_norm_backward(dh, x, gamma, beta, st, activation="swish")
        assert (pre is None) == (n != 136)
        for got, want in ((y, y2), (x.grad, dx), (w.grad, dw), (bias.grad, db), (gamma.grad, dg), (beta.grad, dbe), (res.grad, dy)):
            assert got.dtype == want.dtype and torch.equal(got, want)
        # one leaf at a time: what is not wanted is not formed, the rest keeps its bits
        for leaf, want in ((x, dx), (w, dw), (bias, db), (gamma, dg)):
            a = {id(t): t.detach().clone() if t is not x else t.detach() for t in (x, w, bias, gamma, beta, res)}
            a[id(leaf)].requires_grad_()
            out = ctx.linear(ctx.group_norm(a[id(x)], a[id(gamma)], a[id(beta)], groups=8, activation="swish"), a[id(w)], a[id(bias)], residual=a[id(res)],
                             activation="tanh", scale=0.5)
            got, = torch.autograd.grad(out, a[id(leaf)], dy)
            assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", [(100, 64, 64), (100, 64, 1), (101, 50, 33), (300, 200, 150), (3200, 512, 640)], ids=str)
def test_linear_relu_weight_gradient_of_an_infinite_x(ctx, dtype, shape):
    """inf * dz is an infinity of dz's sign, NaN where relu's slope or dy is 0; the other rows of dw are exact"""
    m, k, n = shape
    dt = DT[dtype]
    x, w, dy, bias = ints((m, k), dt, 1), ints((k, n), dt, 2), ints((m, n), dt, 3), torch.zeros(n, device="cuda")
    w[5] = w[5].abs() * 2 - 1                                     # the infinite element has weights 1 and -1
    x[7, 5] = float("inf")
    z = torch.cat([x[:7].double() @ w.double(), w[5:6].double() * float("inf"), x[8:].double() @ w.double()])
    dz = dy.double() * (z > 0)
    want = x.double().nan_to_num(posinf=0).t() @ dz
    want[5] += float("inf") * dz[7]
    _, pre = ctx.linear(x, w, bias, activation="relu", want_preact=True)
    for kept in ([pre, None] if pre is not None else [None]):
        dx, dw, db = ctx.linear_backward(dy, x, w, kept, bias, activation="relu")
        assert torch.equal(dw.isnan(), want.isnan()) and torch.equal(dw.nan_to_num(), want.to(dt).nan_to_num())
        assert torch.equal(dx, (dz @ w.double().t()).to(dt)) and torch.equal(db, dz.sum(0).float())


# ---- offsets past 32 bits ----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("cin,cout", [(64, 64), (64, 1), (264, 136)], ids=str)
def test_linear_past_two_to_the_31_elements(ctx, cin, cout):
    """x of more than 2^31 elements whose rows are zero but at both ends and next to the offsets of 2^31 elements and bytes"""
    dt, m = torch.bfloat16, (1 << 31) // cin + 1003
    x, dy = torch.zeros((m, cin), device="cuda", dtype=dt), torch.zeros((m, cout), device="cuda", dtype=dt)
    at = [r for c in (0, (1 << 31) // cin, (1 << 30) // cin, (1 << 31) // max(cout, 64), (1 << 30) // max(cout, 64), m) for r in range(c - 20, c + 20) if 0 <= r < m]
    at = torch.tensor(sorted(set(at)), device="cuda")
    x[at], dy[at] = ints((len(at), cin), dt, 1), ints((len(at), cout), dt, 2)
    w, bias = ints((cin, cout), dt, 3), torch.zeros(cout, device="cuda")
    y, pre = ctx.linear(x, w, bias, activation="relu", want_preact=True)
    z = x[at].double() @ w.double()
    assert torch.equal(y[at], z.clamp(min=0).to(dt)) and int(torch.count_nonzero(y)) == int((z > 0).sum())
    dx, dw, db = ctx.linear_backward(dy, x, w, pre, bias, activation="relu")
    dz = dy[at].double() * (z > 0)
    want = (dz @ w.double().t()).to(dt)
    assert torch.equal(dx[at], want) and int(torch.count_nonzero(dx)) == int(torch.count_nonzero(want))
    assert torch.equal(dw, (x[at].double().t() @ dz).to(dt)) and torch.equal(db, dz.sum(0).float())


def test_group_norm_past_two_to_the_31_elements(ctx):
    dt, n, r, c = torch.bfloat16, 3, (1 << 30) // 64 + 77, 64
    x = torch.ones((n, r, c), device="cuda", dtype=dt)
    x[..., 1::2] = -1
    dy = torch.zeros_like(x)
    at = torch.tensor([0, 1, 2, r - 3, r - 2, r - 1], device="cuda")
    dy[:, at] = ints((n, 6, c), dt, 1)
    y, st = ctx.group_norm(x, groups=8, eps=0.0, want_stats=True)
    assert torch.equal(y, x)
    del y
    dx, dg, db = ctx.group_norm_backward(dy, x, None, None, st)
    d = dy[:, at].double()
    assert torch.equal(db, d.sum((0, 1)).float()) and torch.equal(dg, (d * x[:, at].double()).sum((0, 1)).float())
    # the group means are at most 48 / 1.3e8, below what the type resolves next to 1; where dy is 0 they are what is left
    assert bool(((dx[:, at].double() - d).abs() <= 1e-6).all()) and bool((dx.abs().amax(2).float()[:, 3:-3] <= 1e-6).all())
