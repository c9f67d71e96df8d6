"""The dense operators against their definitions in double: product with bias, activation and residual, layer norm, distillation loss, and
their backward passes."""
import math

import pytest
import torch

from drone_b200 import dense

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF_STEP = {t: torch.finfo(t).eps / 2 for t in TYPES}      # of a rounding to the type, relative to the value
STEP = 2.0 ** -23                                            # an addition in 32 bits, also where it is cut off instead of rounded
SMALLEST = {t: torch.finfo(t).smallest_normal * torch.finfo(t).eps for t in TYPES}      # below the normal numbers steps have this size


def rows_of(gen, n, f, dtype, pad=0, lead=0, scale=1.0):
    """[n, f] random values whose rows lie pad + lead values further apart and begin `lead` values behind an aligned address."""
    base = torch.randn((n, lead + f + pad), device="cuda", generator=gen) * scale
    return base.to(dtype)[:, lead:lead + f]


def activated(z, name):
    return {"none": lambda v: v, "relu": torch.relu, "gelu": lambda v: v * torch.special.ndtr(v),
            "silu": lambda v: v * torch.sigmoid(v)}[name or "none"](z)


def slope(z, name):
    if name == "relu":
        return (z > 0).double()
    if name == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "silu":
        return torch.sigmoid(z) * (1 + z * torch.sigmoid(-z))
    return torch.ones_like(z)


def check_rounded(got, want, bound, dtype):
    """got is want rounded once to its type, after an error of at most `bound`."""
    assert got.dtype == dtype and got.shape == want.shape
    err = (got.double() - want).abs()
    allowed = bound + HALF_STEP[dtype] * (want.abs() + bound) + SMALLEST[dtype]
    worst = (err / allowed).max().item() if err.numel() else 0.0
    assert worst <= 1, "%g times the allowed error" % worst


def product_bound(x, w, extra=0.0):
    """Of a sum of K products: each off by a step (what splitting a float leaves out), as is each of K additions."""
    return (x.shape[1] + 16) * STEP * (x.double().abs() @ w.double().abs() + extra)


def check_linear(gen, n, k, m, dtype, activation="none", bias=False, residual=False, transposed=False, keep=False, pad=0, lead=0):
    x = rows_of(gen, n, k, dtype, pad, lead)
    w = rows_of(gen, m, k, dtype, pad, lead, 0.5) if transposed else rows_of(gen, k, m, dtype, pad, lead, 0.5)
    b = torch.randn(m, device="cuda", generator=gen) if bias else None
    r = rows_of(gen, n, m, dtype, pad, lead) if residual else None
    pre = torch.full((n, m + pad), 7.0, dtype=dtype, device="cuda")[:, :m] if keep else None
    out = torch.full((n + 3, m + pad), 9.0, dtype=dtype, device="cuda")
    got = dense.linear(x, w, bias=b, activation=activation, residual=r, transposed=transposed, out=out[1:n + 1, :m], pre=pre)
    assert (out[0] == 9).all() and (out[n + 1:] == 9).all() and (out[:, m:] == 9).all()      # nothing beside the rows is written
    wd = w.double().t() if transposed else w.double()
    z = x.double() @ wd
    bound = product_bound(x, wd, z.abs())
    if bias:
        z = z + b.double()
        bound = bound + STEP * z.abs()
    want = activated(z, activation)
    # an activation of slope 1.13 at most, a few roundings of its own
    total = 1.13 * bound + 8 * STEP * z.abs() * (activation not in ("none", "relu"))
    if residual:
        want = want + r.double()
        total = total + STEP * want.abs()
    check_rounded(got, want, total, dtype)
    if keep:
        check_rounded(pre, z, bound, dtype)
    assert torch.equal(dense.linear(x, w, bias=b, activation=activation, residual=r, transposed=transposed), got)
    return x, w


SHAPES = [(1, 1, 1), (1, 602, 128), (1, 4096, 1000), (2, 3, 5), (3, 64, 64), (5, 129, 257), (8, 300, 41), (9, 17, 15), (16, 33, 7), (17, 100, 47),
          (31, 31, 31), (64, 16, 16), (65, 65, 65), (127, 32, 128), (128, 64, 129), (129, 63, 127), (200, 128, 256), (255, 602, 128),
          (257, 100, 300), (1000, 41, 128), (3001, 128, 41), (20011, 256, 47), (5003, 1000, 7)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k,m", SHAPES)
def test_linear(cuda_device, n, k, m, dtype):
    gen = torch.Generator(cuda_device).manual_seed(n + k + m)
    check_linear(gen, n, k, m, dtype)
    check_linear(gen, n, k, m, dtype, transposed=True, bias=True, activation="relu")
    check_linear(gen, n, k, m, dtype, bias=True, residual=True, activation="gelu", keep=True, pad=8)
    check_linear(gen, n, k, m, dtype, transposed=True, residual=True, activation="silu", keep=True, pad=2, lead=1)
    check_linear(gen, n, k, m, dtype, residual=True, pad=1, lead=3)


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_many_rows(cuda_device, dtype):
    """More tiles than the GPU holds at once; every row and column against double."""
    gen = torch.Generator(cuda_device).manual_seed(1)
    check_linear(gen, 100003, 96, 72, dtype, bias=True, activation="relu")
    check_linear(gen, 70001, 40, 520, dtype, residual=True, transposed=True)


def test_products_of_floats_are_floats(cuda_device):
    """One product per output, of full mantissas: within two steps of the exact one, whatever the factors' sizes.  Very small and very large
    factors among them, down to subnormal ones and up to the largest."""
    gen = torch.Generator(cuda_device).manual_seed(2)
    x = rows_of(gen, 300, 1, torch.float32) * torch.exp2(torch.randint(-60, 60, (300, 1), device="cuda", generator=gen).float())
    w = rows_of(gen, 1, 200, torch.float32) * torch.exp2(torch.randint(-60, 60, (1, 200), device="cuda", generator=gen).float())
    want = x.double() * w.double()
    got = dense.linear(x, w)
    # the smallest factors are 2^-60 times a value that may be far below 1, so that products fall below 2^-126, where floats are the
    # multiples of 2^-149: the product is formed of six products of a float's parts, and each of them, cut off there, is off by less than
    # one of these whatever its size
    assert ((got - want).abs() <= 2 * STEP * want.abs() + 6 * 2.0 ** -149).all()
    big = torch.tensor([[3.4028235e38], [-3.4028235e38], [3.39e38], [1e-38], [1e-44]], device="cuda")
    got = dense.linear(big, torch.tensor([[1.0, 0.5, -1.0, 1e-30]], device="cuda"))
    want = big.double() * torch.tensor([[1.0, 0.5, -1.0, 1e-30]], device="cuda").double()
    assert ((got - want).abs() <= 2 * STEP * want.abs() + 2.0 ** -133).all()


def test_large_floats_in_tiles(cuda_device):
    """The same through many rows: values up to the largest float beside others, weights of 0, products that leave the range."""
    gen = torch.Generator(cuda_device).manual_seed(12)
    top = 3.4028234663852886e38
    x = rows_of(gen, 700, 40, torch.float32)
    w = rows_of(gen, 40, 200, torch.float32)
    x[5], x[6], x[7], x[8, 3] = 0, 0, 0, 0
    x[5, 1], x[6, 2], x[7, 30], x[8, 3] = top, -top, 3.39e38, 1e-44
    w[1, 7], w[2, 9], w[30, 11], w[1, 12] = 0, 0, 0, 1e-30
    got, want = dense.linear(x, w), x.double() @ w.double()
    finite = want.abs() <= top
    assert torch.equal(got.isfinite(), finite) and torch.equal(torch.sign(got[~finite]).double(), torch.sign(want[~finite]))
    bound = (40 + 16) * STEP * (x.double().abs() @ w.double().abs()) + 2.0 ** -133
    assert ((got - want).abs()[finite] <= bound[finite]).all()
    g = torch.zeros((700, 200), device="cuda")
    g[5, 3], g[6, 3], g[9, 4] = 1e-3, 1e-3, 2
    dw = dense.linear_backward(g, x, w, input_gradient=False)[1]
    want = x.double().t() @ g.double()
    assert ((dw - want).abs() <= (700 + 16) * STEP * (x.double().abs().t() @ g.double().abs()) + 2.0 ** -133).all()
    x[9, 5], x[10, 6] = math.inf, math.nan
    dw = dense.linear_backward(g + 1e-3, x, w, input_gradient=False)[1]
    assert (dw[5] == math.inf).all() and dw[6].isnan().all() and dw[7:].isfinite().all() and dw[:1].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [3, 300])
def test_linear_of_infinities(cuda_device, dtype, n):
    """Infinities and NaN reach exactly the outputs that they reach in the formula, whichever k they stand at."""
    gen = torch.Generator(cuda_device).manual_seed(3)
    x, w = rows_of(gen, n, 70, dtype), rows_of(gen, 70, 50, dtype)
    x[0, 3], x[1, 69], x[2, 40] = math.inf, -math.inf, math.nan
    w[10, 7], w[69, 8] = math.inf, 0
    got, want = dense.linear(x, w), x.double() @ w.double()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    assert torch.equal(got[want.isinf()].double(), want[want.isinf()])
    fine = want.isfinite()
    bound = (70 + 16) * STEP * (x.double().abs().nan_to_num(0, 0, 0) @ w.double().abs().nan_to_num(0, 0, 0))
    check_rounded(got[fine], want[fine], bound[fine], dtype)
    assert dense.linear(x, w, activation="relu")[2].isnan().all()      # as max(0, NaN) of torch


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("n,k,m", [(0, 5, 6), (1, 1, 1), (2, 9, 3), (63, 16, 16), (65, 40, 33), (129, 129, 65), (1000, 602, 41), (4097, 64, 128), (20011, 47, 256),
                                   (100003, 24, 40)])
def test_linear_backward(cuda_device, n, k, m, dtype, transposed):
    gen = torch.Generator(cuda_device).manual_seed(n + k + m)
    for activation, pad, lead in (("none", 0, 0), ("relu", 3, 1), ("gelu", 8, 0), ("silu", 0, 0)):
        x, g = rows_of(gen, n, k, dtype, pad, lead), rows_of(gen, n, m, dtype, pad, lead)
        w = rows_of(gen, m, k, dtype, pad, lead) if transposed else rows_of(gen, k, m, dtype, pad, lead)
        pre = rows_of(gen, n, m, dtype, pad, lead) if activation != "none" else None
        dx, dw, db = dense.linear_backward(g, x, w, pre=pre, activation=activation, transposed=transposed)
        wd = w.double().t() if transposed else w.double()
        dz = g.double() * slope(pre.double(), activation) if pre is not None else g.double()
        # what the rounding of dz to the rows' type and its own arithmetic leave
        off = dz.abs() * (HALF_STEP[dtype] + 8 * STEP) + 8 * STEP * g.double().abs() + SMALLEST[dtype] if pre is not None else dz.abs() * 0
        check_rounded(dx, dz @ wd.t(), (m + 16) * STEP * (dz.abs() @ wd.t().abs()) + off @ wd.t().abs(), dtype)
        bound = (n + 16) * STEP * (x.double().abs().t() @ dz.abs()) + x.double().abs().t() @ off
        want = x.double().t() @ dz
        check_rounded(dw, want.t() if transposed else want, bound.t() if transposed else bound, dtype)
        check_rounded(db, dz.sum(dim=0), ((n + 16) * STEP * dz.abs() + 8 * STEP * g.double().abs()).sum(dim=0), torch.float32)
        again = dense.linear_backward(g, x, w, pre=pre, activation=activation, transposed=transposed)
        assert all(torch.equal(a, b) for a, b in zip((dx, dw, db), again))
        some = dense.linear_backward(g, x, w, pre=pre, activation=activation, transposed=transposed, bias=False, input_gradient=False)
        assert some[0] is None and some[2] is None and torch.equal(some[1], dw)


def test_linear_backward_against_differences(cuda_device):
    """The gradients against differences of the forward pass: (f(x + h) - f(x - h)) / 2h in the direction of a random matrix.  The forward
    pass is good to about K steps, so with h = 2^-6 and values of size 1 the difference is off by K * 2^-23 * 2^6, and by h^2."""
    gen = torch.Generator(cuda_device).manual_seed(4)
    n, k, m, h = 50, 40, 30, 2.0 ** -6
    x, w, b = rows_of(gen, n, k, torch.float32), rows_of(gen, k, m, torch.float32, scale=0.2), torch.randn(m, device="cuda", generator=gen)
    r, g = rows_of(gen, n, m, torch.float32), rows_of(gen, n, m, torch.float32)
    pre = torch.empty((n, m), device="cuda")
    for activation in ("gelu", "silu"):
        dense.linear(x, w, bias=b, activation=activation, residual=r, pre=pre)
        dx, dw, db = dense.linear_backward(g, x, w, pre=pre, activation=activation)
        f = lambda *a: (dense.linear(a[0], a[1], bias=a[2], activation=activation, residual=r).double() * g.double()).sum().item()
        for i, grad in enumerate((dx, dw, db)):
            at = [x, w, b]
            d = torch.randn(at[i].shape, device="cuda", generator=gen)
            d /= d.norm()
            moved = [[t + s * h * d if j == i else t for j, t in enumerate(at)] for s in (1, -1)]
            want = (f(*moved[0]) - f(*moved[1])) / (2 * h)
            assert abs((grad.double() * d.double()).sum().item() - want) <= 2e-2


def norm_of(x, scale, shift, eps, relu):
    x = x.double()
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    rstd = (var + eps) ** -0.5
    y = (x - mean) * rstd * scale.double() + shift.double()
    return (torch.relu(y) if relu else y), mean[:, 0], rstd[:, 0]


NORM_WIDTHS = [1, 2, 7, 8, 32, 33, 41, 64, 100, 128, 256, 300, 512, 602, 1000, 1024, 2048, 2049, 4104, 8192, 8200, 16384, 16392, 20001]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("f", NORM_WIDTHS)
def test_layer_norm(cuda_device, f, dtype):
    gen = torch.Generator(cuda_device).manual_seed(f)
    scale, shift = (torch.randn(f, device="cuda", generator=gen) for _ in range(2))
    for n, pad, lead, relu in ((1, 0, 0, False), (37, 8, 0, True), (33, 3, 1, False), (1 + (1 << 21) // (f + 100), 0, 0, True)):
        x = rows_of(gen, n, f, dtype, pad, lead, 1.5)
        out = torch.full((n + 2, f + pad), 9.0, dtype=dtype, device="cuda")
        y, mean, rstd = dense.layer_norm(x, scale, shift, eps=1e-3, relu=relu, out=out[1:n + 1, :f])
        assert (out[0] == 9).all() and (out[n + 1:] == 9).all() and (out[:, f:] == 9).all()
        want, want_mean, want_rstd = norm_of(x, scale, shift, 1e-3, relu)
        # sums of up to f / 8 values a lane; mean, deviation and quotient by a few steps each
        steps = (16 + f / 256) * STEP
        size = x.double().abs().amax(dim=1)
        assert ((mean - want_mean).abs() <= steps * size).all()
        assert ((rstd - want_rstd).abs() <= steps * want_rstd * (1 + (size * want_rstd) ** 2 * steps)).all()
        bound = steps * (want_rstd * size)[:, None] * scale.double().abs() + STEP * shift.double().abs() + steps * want.abs()
        check_rounded(y, want, bound, dtype)
        # in place: the same bits as beside, of rows that lie the same way (how they lie decides the order of a row's sums)
        at_x = x.clone()
        beside = dense.layer_norm(at_x, scale, shift, eps=1e-3, relu=relu)[0]
        assert torch.equal(dense.layer_norm(at_x, scale, shift, eps=1e-3, relu=relu, out=at_x)[0], beside)


def test_layer_norm_of_constant_and_distant_rows(cuda_device):
    """Rows without variance give the shift; rows far from 0 keep the digits that their differences have."""
    scale, shift = torch.full((96,), 2.0, device="cuda"), torch.arange(96, device="cuda").float()
    x = torch.full((5, 96), 3.25, device="cuda")
    x[1], x[2] = 0, -1e30
    y, mean, rstd = dense.layer_norm(x, scale, shift, eps=1e-5)
    assert torch.equal(y, shift.expand(5, 96))
    far = 4096 + torch.arange(96, device="cuda").float().expand(3, 96) / 8
    y, _, _ = dense.layer_norm(far.contiguous(), scale, shift, eps=1e-5)
    want = norm_of(far, scale, shift, 1e-5, False)[0]
    # the mean is off by a few steps of 4096, the differences by as much
    assert (y - want).abs().max() <= 16 * STEP * 4096 / 3.4 * 2 + 1e-4
    x = torch.ones((3, 96), device="cuda")
    x[1, 5] = math.nan
    y, mean, rstd = dense.layer_norm(x, scale, shift)
    assert y[1].isnan().all() and torch.equal(y[0], shift) and torch.equal(y[2], shift)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("f", NORM_WIDTHS)
def test_layer_norm_backward(cuda_device, f, dtype):
    gen = torch.Generator(cuda_device).manual_seed(f)
    scale, shift = (torch.randn(f, device="cuda", generator=gen) for _ in range(2))
    for n, pad, lead, relu, mirrors in ((1, 0, 0, False, False), (37, 8, 0, True, True), (33, 3, 1, False, True), (1 + (1 << 21) // (f + 100), 0, 0, True, False)):
        x, g = rows_of(gen, n, f, dtype, pad, lead, 1.5), rows_of(gen, n, f, dtype, pad, lead)
        y, mean, rstd = dense.layer_norm(x, scale, shift, eps=1e-3, relu=relu)
        m2w = torch.where(torch.rand(n, device="cuda", generator=gen) < 0.3, 2, -1).int() if mirrors else None
        dx, ds, dt = dense.layer_norm_backward(g, x, scale, mean, rstd, out=y if relu else None, mirror_rows=m2w)
        gd = g.double() * (y > 0) if relu else g.double()
        hat = (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
        h = gd * scale.double()
        r = rstd.double()[:, None]
        want = r * (h - h.mean(dim=1, keepdim=True) - hat * (h * hat).mean(dim=1, keepdim=True))
        steps = (16 + f / 128) * STEP
        size = (x.double().abs() + mean.double().abs()[:, None]) * r      # what xhat's difference was formed of
        bound = steps * r * (h.abs() + h.abs().mean(dim=1, keepdim=True) + size * (h * hat).abs().mean(dim=1, keepdim=True)
                             + hat.abs() * (h.abs() * size).mean(dim=1, keepdim=True))
        check_rounded(dx, want, bound, dtype)
        own = (m2w == -1).double()[:, None] if mirrors else torch.ones((n, 1), dtype=torch.float64, device="cuda")
        rows = (16 + n / 8) * STEP      # a chain over the rows of a thread
        check_rounded(ds, (own * gd * hat).sum(dim=0), rows * (own * gd.abs() * size).sum(dim=0), torch.float32)
        check_rounded(dt, (own * gd).sum(dim=0), rows * (own * gd.abs()).sum(dim=0), torch.float32)
        again = dense.layer_norm_backward(g, x, scale, mean, rstd, out=y if relu else None, mirror_rows=m2w)
        assert all(torch.equal(a, b) for a, b in zip((dx, ds, dt), again))


def test_layer_norm_backward_against_differences(cuda_device):
    gen = torch.Generator(cuda_device).manual_seed(6)
    n, f, h = 20, 24, 2.0 ** -6
    x, g = rows_of(gen, n, f, torch.float32), rows_of(gen, n, f, torch.float32)
    scale, shift = (torch.randn(f, device="cuda", generator=gen) for _ in range(2))
    _, mean, rstd = dense.layer_norm(x, scale, shift)
    grads = dense.layer_norm_backward(g, x, scale, mean, rstd)
    f_of = lambda *a: (dense.layer_norm(*a)[0].double() * g.double()).sum().item()
    for i, grad in enumerate(grads):
        at = [x, scale, shift]
        d = torch.randn(at[i].shape, device="cuda", generator=gen)
        d /= d.norm()
        moved = [[t + s * h * d if j == i else t for j, t in enumerate(at)] for s in (1, -1)]
        want = (f_of(*moved[0]) - f_of(*moved[1])) / (2 * h)
        # n f values of a few steps each over h, and h^2 times a third derivative of size 10
        assert abs((grad.double() * d.double()).sum().item() - want) <= n * f * 8 * STEP / h + 10 * h * h


def distilled(logits, teacher, classes, t, truth, labelled, soft, hard):
    """Loss and gradient in double, from the definition."""
    z = logits.double()
    has_entry = (classes >= 0) & (teacher.double() > -math.inf)
    some = has_entry.any(dim=1)
    q = torch.softmax(torch.where(has_entry, teacher.double() / t, -1e300), dim=1) * has_entry
    target = torch.zeros_like(z).scatter_add_(1, classes.clamp(min=0), q)
    log_p = torch.log_softmax(z / t, dim=1)
    terms = torch.where(q > 0, q * (torch.log(q.clamp(min=1e-300)) - log_p.gather(1, classes.clamp(min=0))), 0.0)
    rows = t * t * terms.sum(dim=1) * some
    grad = soft * t * (log_p.exp() - target) * some[:, None]
    loss = [rows.sum() / max(int(some.sum()), 1), torch.zeros((), dtype=torch.float64, device=z.device)]
    if truth is not None:
        log_p = torch.log_softmax(z, dim=1)
        loss[1] = -(log_p.gather(1, truth[:, None])[:, 0] * labelled).sum() / max(int(labelled.sum()), 1)
        grad = grad + hard * (log_p.exp() - torch.nn.functional.one_hot(truth, z.shape[1])) * labelled[:, None]
    return torch.stack(loss), grad


def check_distillation(logits, teacher, classes, t=1.0, truth=None, labelled=None, soft=1.0, hard=0.0):
    loss, grad = dense.distillation_loss(logits, teacher, classes, temperature=t, truth=truth, labelled=labelled, soft=soft, hard=hard)
    want_loss, want = distilled(logits, teacher, classes, t, truth, labelled, soft, hard)
    # exponents of size |z| / t, off by two steps; a sum of `classes` exponentials, a thread's share in a chain; a quotient
    size = (logits.double().max(dim=1).values - logits.double().min(dim=1).values).clamp(max=100).max().item() if logits.numel() else 0
    off = (16 + 2 * size / min(t, 1.0) + logits.shape[1] / 64) * STEP
    check_rounded(grad, want, off * (abs(soft) * t + abs(hard)) * torch.ones_like(want), logits.dtype)
    assert ((loss - want_loss).abs() <= off * (t * t + 1) * (4 + size)).all()
    again = dense.distillation_loss(logits, teacher, classes, temperature=t, truth=truth, labelled=labelled, soft=soft, hard=hard)
    assert torch.equal(again[0], loss) and torch.equal(again[1], grad)
    return loss, grad


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c", [1, 2, 7, 8, 9, 16, 17, 33, 41, 47, 64, 65, 200, 256, 257, 1000, 4099, 32000, 70001])
def test_distillation(cuda_device, c, dtype):
    gen = torch.Generator(cuda_device).manual_seed(c)
    for n, k, t, hard, pad in ((1, 1, 1.0, False, 0), (37, 8, 2.0, True, 0), (300, 64, 4.0, True, 3), (1 + 200000 // c, 5, 0.5, False, 8), (70, 256, 2.0, False, 0)):
        logits = rows_of(gen, n, c, dtype, pad, scale=3.0)
        teacher = rows_of(gen, n, k, [torch.float32, dtype][n % 2], pad, scale=3.0)
        # classes may be there twice; some rows have fewer entries, some none
        classes = torch.randint(0, c, (n, k + pad), device="cuda", generator=gen)[:, :k]
        classes[torch.rand((n, k), device="cuda", generator=gen) < 0.2] = -1
        if n > 9:
            classes[3], teacher[5], teacher[7, 0] = -7, -math.inf, torch.finfo(teacher.dtype).min
            classes[9, :] = classes[9, 0].clamp(min=0)
        truth = torch.randint(0, c, (n,), device="cuda", generator=gen) if hard else None
        labelled = torch.rand(n, device="cuda", generator=gen) < 0.5 if hard else None
        loss, grad = check_distillation(logits, teacher, classes, t, truth, labelled, *((0.25, 0.75) if hard else (1.0, 0.0)))
        if n > 9 and not hard:
            assert (grad[3] == 0).all() and (grad[5] == 0).all()


def test_distillation_of_rows_that_count_for_nothing(cuda_device):
    gen = torch.Generator(cuda_device).manual_seed(8)
    for c in (5, 47, 300):
        logits, teacher = rows_of(gen, 12, c, torch.float32), rows_of(gen, 12, 3, torch.float32)
        none = torch.full((12, 3), -1, device="cuda")
        loss, grad = dense.distillation_loss(logits, teacher, none)
        assert (loss == 0).all() and (grad == 0).all()
        no_rows = dense.distillation_loss(logits[:0], teacher[:0], none[:0])
        assert (no_rows[0] == 0).all() and no_rows[1].shape == (0, c)
        # minus infinity among the logits: a class without a share; where the teacher wants it the loss is infinite
        classes = torch.tensor([[0, 1, 2]], device="cuda").expand(12, 3).contiguous()
        logits[4, 3:] = -math.inf
        logits[4, 4] = 0
        check_distillation(logits, teacher, classes)
        logits[4, 1] = -math.inf
        assert dense.distillation_loss(logits, teacher, classes)[0][0] == math.inf
        logits[4] = -math.inf
        loss, grad = dense.distillation_loss(logits, teacher, classes)
        assert loss[0].isnan() and grad[4].isnan().all() and grad[:4].isfinite().all() and grad[5:].isfinite().all()


def test_distillation_classes_that_do_not_exist(cuda_device):
    gen = torch.Generator(cuda_device).manual_seed(9)
    for c in (5, 47, 300):
        logits, teacher = rows_of(gen, 12, c, torch.float32), rows_of(gen, 12, 3, torch.float32)
        classes = torch.randint(0, c, (12, 3), device="cuda", generator=gen)
        truth, labelled = torch.randint(0, c, (12,), device="cuda", generator=gen), torch.ones(12, dtype=torch.bool, device="cuda")
        for bad in (c, 1 << 40):
            wrong = classes.clone()
            wrong[7, 1] = bad
            loss, grad = dense.distillation_loss(logits, teacher, wrong)
            assert loss[0].isnan() and grad[7].isnan().all() and grad[:7].isfinite().all() and grad[8:].isfinite().all()
        for bad in (-1, c):
            wrong = truth.clone()
            wrong[2] = bad
            loss, grad = dense.distillation_loss(logits, teacher, classes, truth=wrong, labelled=labelled, hard=0.5)
            assert loss[0].isfinite() and loss[1].isnan() and grad[2].isnan().all() and grad[3:].isfinite().all()


def test_distillation_gradient_against_differences(cuda_device):
    """Summed over rows, as the gradient is: differences of the mean loss times the number of rows."""
    gen = torch.Generator(cuda_device).manual_seed(10)
    for c in (9, 400):
        n, h = 6, 2.0 ** -6
        logits, teacher = rows_of(gen, n, c, torch.float32), rows_of(gen, n, 4, torch.float32)
        classes, truth = torch.randint(0, c, (n, 4), device="cuda", generator=gen), torch.randint(0, c, (n,), device="cuda", generator=gen)
        rest = dict(temperature=2.0, truth=truth, labelled=torch.ones(n, dtype=torch.bool, device="cuda"), soft=0.3, hard=0.7)
        grad = dense.distillation_loss(logits, teacher, classes, **rest)[1]
        d = torch.randn((n, c), device="cuda", generator=gen)
        d /= d.norm()
        value = lambda z: n * (torch.tensor([0.3, 0.7], device="cuda").double() @ dense.distillation_loss(z, teacher, classes, **rest)[0].double()).item()
        want = (value(logits + h * d) - value(logits - h * d)) / (2 * h)
        # a loss of size n * 10, good to 32 steps, over h, and h^2
        assert abs((grad.double() * d.double()).sum().item() - want) <= 32 * STEP * n * 10 / h + h * h


@pytest.mark.parametrize("dtype", TYPES)
def test_distillation_of_masked_logits(cuda_device, dtype):
    """Logits and entries of the type's lowest value: no share beside others, equal shares where there is nothing else."""
    gen = torch.Generator(cuda_device).manual_seed(11)
    low = torch.finfo(dtype).min
    for c in (7, 47, 100, 500, 9000):
        logits, teacher = rows_of(gen, 6, c, dtype), rows_of(gen, 6, 4, dtype)
        classes = torch.arange(4, device="cuda").expand(6, 4).contiguous()
        logits[1, 5:], logits[2], teacher[3, 1:], teacher[4] = low, low, low, low
        check_distillation(logits, teacher, classes, 1.0)
        check_distillation(logits, teacher, classes, 4.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k,m", [(2, 1, 1), (600, 5, 1), (513, 1, 128), (70001, 16, 8), (9999, 128, 1), (300007, 3, 20), (5, 2, 64)])
def test_narrow_products_and_their_gradients(cuda_device, n, k, m, dtype):
    """Few products a row: forward, and the weights' gradient in both orders."""
    gen = torch.Generator(cuda_device).manual_seed(n + k + m)
    for pad, lead in ((0, 0), (3, 1)):
        check_linear(gen, n, k, m, dtype, bias=True, residual=True, activation="silu", keep=True, pad=pad, lead=lead)
        x, g = rows_of(gen, n, k, dtype, pad, lead), rows_of(gen, n, m, dtype, pad, lead)
        for transposed in (False, True):
            check_linear(gen, n, k, m, dtype, transposed=transposed, pad=pad, lead=lead)
            w = rows_of(gen, m, k, dtype) if transposed else rows_of(gen, k, m, dtype)
            dx, dw, db = dense.linear_backward(g, x, w, transposed=transposed)
            wd = w.double().t() if transposed else w.double()
            want, bound = x.double().t() @ g.double(), (n + 16) * STEP * (x.double().abs().t() @ g.double().abs())
            check_rounded(dw, want.t() if transposed else want, bound.t() if transposed else bound, dtype)
            check_rounded(dx, g.double() @ wd.t(), (m + 16) * STEP * (g.double().abs() @ wd.t().abs()), dtype)
