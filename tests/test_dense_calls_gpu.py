"""The dense operators as programs call them: other streams, several calls at once, captured and replayed, operands beyond 32 bits, the largest widths, views, and what
the Python calls refuse."""
import pytest
import torch

from drone_b200 import dense

pytestmark = pytest.mark.gpu


def calls(gen, dtype, n=3000):
    """Each operator on inputs of its own, as functions of nothing that return new outputs."""
    r = lambda *shape: torch.randn(shape, device="cuda", generator=gen).to(dtype)
    f = lambda m: torch.randn(m, device="cuda", generator=gen)
    x, w, wt, bias, res, g = r(n, 200), r(200, 136), r(136, 200), f(136), r(n, 136), r(n, 136)
    odd, odd_w = r(n, 201)[:, :199], r(199, 47)
    scale, shift = f(200), f(200)
    logits, teacher = r(n, 41), r(n, 5)
    many, best = r(200, 5000), r(200, 20)
    classes, ids = torch.randint(-1, 41, (n, 5), device="cuda", generator=gen), torch.randint(0, 5000, (200, 20), device="cuda", generator=gen)
    truth, labelled = torch.randint(0, 41, (n,), device="cuda", generator=gen), torch.rand(n, device="cuda", generator=gen) < 0.5
    y, mean, rstd = dense.layer_norm(x, scale, shift, relu=True)
    inputs = (x, w, wt, bias, res, g, odd, odd_w, scale, shift, logits, teacher, many, best)
    return inputs, [
        lambda: dense.linear(x, w, bias=bias, activation="gelu", residual=res),
        lambda: dense.linear(x, wt, transposed=True),
        lambda: dense.linear(odd, odd_w, activation="silu"),
        lambda: dense.linear(x[:3], w, bias=bias),
        lambda: dense.linear(x[:, :9], w[:9, :12]),
        lambda: dense.linear_backward(g, x, w, pre=res, activation="gelu"),
        lambda: dense.layer_norm(x, scale, shift),
        lambda: dense.layer_norm_backward(x, x, scale, mean, rstd, out=y),
        lambda: dense.distillation_loss(logits, teacher, classes, temperature=2.0, truth=truth, labelled=labelled, soft=0.5, hard=0.5),
        lambda: dense.distillation_loss(many, best, ids),
    ]


def flat(out):
    return [out] if isinstance(out, torch.Tensor) else [t for t in out if t is not None]


def same(a, b):
    return len(flat(a)) == len(flat(b)) and all(torch.equal(x, y) for x, y in zip(flat(a), flat(b)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_streams(cuda_device, dtype):
    """Calls on two streams at once give the bits of calls one after the other; a call waits for what its own stream did before."""
    gen = torch.Generator(cuda_device).manual_seed(1)
    inputs, functions = calls(gen, dtype)
    want = [f() for f in functions]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(3):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        got = [[], []]
        for f in functions:
            for i, s in enumerate(streams):
                with torch.cuda.stream(s):
                    got[i].append(f())
        torch.cuda.synchronize()
        assert all(same(a, w) for own in got for a, w in zip(own, want))
    x, w = torch.zeros((100000, 128), device="cuda", dtype=dtype), torch.randn((128, 64), device="cuda", generator=gen).to(dtype)
    source = torch.randn((100000, 128), device="cuda", generator=gen).to(dtype)
    torch.cuda.synchronize()
    with torch.cuda.stream(streams[0]):
        x.copy_(source)
        late = dense.linear(x, w)
    torch.cuda.synchronize()
    assert torch.equal(late, dense.linear(source, w))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_captured_and_replayed(cuda_device, dtype):
    """Each call captured twice, into graphs that are replayed in turn on other inputs: the bits of the eager calls on these."""
    gen = torch.Generator(cuda_device).manual_seed(2)
    inputs, functions = calls(gen, dtype)
    for f in functions:
        f()
    torch.cuda.synchronize()
    graphs = []
    for f in functions:
        pair = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = f()
            pair.append((g, out))
        graphs.append(pair)
    for _ in range(2):
        for t in inputs:
            t.copy_(torch.randn(t.shape, device="cuda", generator=gen))
        want = [f() for f in functions]
        for pair in graphs:
            for g, _ in pair:
                g.replay()
        torch.cuda.synchronize()
        for (a, b), w in zip(graphs, want):
            assert same(a[1], w) and same(b[1], w)


@pytest.mark.parametrize("dtype,rows,width", [(torch.bfloat16, 17_000_001, 256), (torch.float32, 8_500_001, 256)])
def test_operands_beyond_32_bits(cuda_device, dtype, rows, width):
    """More than 2^32 bytes, and for 16 bits than 2^32 values, to the last row: rows from all over equal the same rows by themselves."""
    gen = torch.Generator(cuda_device).manual_seed(3)
    x = torch.empty((rows, width), dtype=dtype, device="cuda")
    for r in range(0, rows, 1 << 20):
        x[r:r + (1 << 20)] = torch.randn(x[r:r + (1 << 20)].shape, device="cuda", generator=gen).to(dtype)
    at = torch.cat([torch.arange(0, 300), torch.arange((1 << 31) // width - 150, (1 << 31) // width + 150), torch.arange(rows - 300, rows)]).cuda()
    some = x[at].contiguous()
    w, scale = torch.randn((width, 40), device="cuda", generator=gen).to(dtype), torch.randn(width, device="cuda", generator=gen)
    # more than a few rows, so that the same kernel and order of sums serve both
    assert torch.equal(dense.linear(x, w)[at], dense.linear(some, w))
    y, mean, rstd = dense.layer_norm(x, scale, scale)
    want = dense.layer_norm(some, scale, scale)
    assert torch.equal(y[at], want[0]) and torch.equal(mean[at], want[1]) and torch.equal(rstd[at], want[2])
    dx = dense.layer_norm_backward(y, x, scale, mean, rstd)[0]
    assert torch.equal(dx[at], dense.layer_norm_backward(want[0], some, scale, want[1], want[2])[0])
    del y, dx
    teacher, classes = x[:, :4], torch.randint(0, width, (rows, 4), device="cuda", generator=gen)
    grad = dense.distillation_loss(x, teacher, classes)[1]
    assert torch.equal(grad[at], dense.distillation_loss(some, some[:, :4], classes[at])[1])
    del grad
    g = torch.zeros((rows, 24), dtype=dtype, device="cuda")
    g[at] = torch.randn((len(at), 24), device="cuda", generator=gen).to(dtype)
    dw, db = dense.linear_backward(g, x, torch.zeros((width, 24), dtype=dtype, device="cuda"), input_gradient=False)[1:]
    want = some.double().t() @ g[at].double()
    bound = some.double().abs().t() @ g[at].double().abs()
    step = torch.finfo(dtype).eps / 2 + (len(at) + 16) * 2.0 ** -23
    assert ((dw - want).abs() <= step * bound + 1e-30).all()
    assert ((db - g[at].double().sum(dim=0)).abs() <= (len(at) + 16) * 2.0 ** -23 * g[at].double().abs().sum(dim=0)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,k,m", [(1, 32768, 8), (3, 32768, 33), (300, 32768, 9), (2000, 32767, 70), (1, 8, 32768), (3, 5, 32768), (300, 9, 32768), (600, 1, 300), (600, 300, 1)])
def test_widest_products(cuda_device, n, k, m, dtype):
    """Values from -1, 0, 1 with one entry a row, so that every sum is exact in every type."""
    gen = torch.Generator(cuda_device).manual_seed(4)
    at = torch.randint(0, k, (n, 1), device="cuda", generator=gen)
    x = torch.zeros((n, k), dtype=dtype, device="cuda").scatter_(1, at, 1)
    w = torch.randint(-1, 2, (k, m), device="cuda", generator=gen).to(dtype)
    want = w[at[:, 0]]
    assert torch.equal(dense.linear(x, w), want) and torch.equal(dense.linear(x, w.t().contiguous(), transposed=True), want)
    g = torch.randint(-1, 2, (n, m), device="cuda", generator=gen).to(dtype)
    dx, dw, db = dense.linear_backward(g, x, w)
    assert torch.equal(dw.double(), x.double().t() @ g.double()) and torch.equal(db.double(), g.double().sum(dim=0))
    exact = g.double() @ w.double().t()      # whole numbers up to m: exact as floats, then rounded once
    assert torch.equal(dx, exact.to(dtype))


def test_views_and_empty_operands(cuda_device):
    gen = torch.Generator(cuda_device).manual_seed(5)
    x, w = torch.randn((70, 30), device="cuda", generator=gen), torch.randn((30, 20), device="cuda", generator=gen)
    want = dense.linear(x, w)
    assert torch.equal(dense.linear(x, w.t().contiguous().t()), dense.linear(x, w.t().contiguous(), transposed=True))
    assert torch.equal(dense.linear(x, w.t(), transposed=True), want)
    gx, gw, gb = dense.linear_backward(want, x, w.t(), transposed=True)
    assert gw.shape == (20, 30) and torch.equal(gx, dense.linear_backward(want, x, w)[0])
    for rows in (x[::2], torch.cat([x, x], dim=1)[:, 30:], x[5:6]):
        assert (dense.linear(rows, w) - rows.double() @ w.double()).abs().max() < 1e-4
        assert (dense.layer_norm(rows, x[0], x[1])[0] - dense.layer_norm(rows.contiguous(), x[0], x[1])[0]).abs().max() < 1e-5
    column = torch.randn((70, 4), device="cuda", generator=gen)[:, 2:3]
    assert torch.equal(dense.linear(column, w[:1]), dense.linear(column.contiguous(), w[:1]))
    none = x[:0]
    assert dense.linear(none, w).shape == (0, 20)
    gx, gw, gb = dense.linear_backward(none[:, :20], none, w)
    assert gx.shape == (0, 30) and (gw == 0).all() and gw.shape == (30, 20) and (gb == 0).all()
    y, mean, rstd = dense.layer_norm(none, x[0], x[1])
    assert y.shape == (0, 30) and mean.shape == (0,)
    gx, gs, gt = dense.layer_norm_backward(none, none, x[0], mean, rstd)
    assert gx.shape == (0, 30) and (gs == 0).all() and (gt == 0).all()
    # in place where that is allowed
    residual = torch.randn((70, 20), device="cuda", generator=gen)
    beside = dense.linear(x, w, residual=residual)
    assert dense.linear(x, w, residual=residual, out=residual) is residual and torch.equal(residual, beside)


def test_refusals(cuda_device):
    x, w, b = torch.zeros((9, 6), device="cuda"), torch.zeros((6, 7), device="cuda"), torch.zeros(7, device="cuda")
    y, v, m = torch.zeros((9, 7), device="cuda"), torch.zeros(6, device="cuda"), torch.zeros(9, device="cuda")
    ids = torch.zeros((9, 2), dtype=torch.int64, device="cuda")
    linear = [dict(x=x.double()), dict(x=x.int()), dict(x=x[0]), dict(x=x.t()), dict(x=x[:1].expand(9, 6)), dict(x=x[:, :5]), dict(x=x[:, ::2]), dict(w=w.half()), dict(w=w.cpu()),
              dict(w=w[:, :0]), dict(bias=b[:6]), dict(bias=b.half()), dict(bias=b.cpu()), dict(bias=torch.zeros(14, device="cuda")[::2]), dict(activation="tanh"),
              dict(residual=y[:8]), dict(residual=y.half()), dict(residual=x), dict(out=y[:, :6]), dict(out=y.half()), dict(pre=y[:5]), dict(transposed=True), dict(out=y, pre=y)]
    for change in linear:
        with pytest.raises(ValueError):
            dense.linear(**{**dict(x=x, w=w), **change})
    square = torch.zeros((6, 6), device="cuda")
    for change in (dict(out=x), dict(pre=x), dict(out=torch.zeros(100, device="cuda").as_strided((9, 6), (6, 1)), residual=None, w=square, x=None)):
        big = torch.zeros(100, device="cuda")
        given = {**dict(x=x, w=square), **change}
        if given["x"] is None:
            given["x"], given["out"] = big.as_strided((9, 6), (6, 1)), big.as_strided((9, 6), (6, 1), 12)
        with pytest.raises(ValueError, match="overlaps"):
            dense.linear(**given)
    for change in (dict(grad=x), dict(grad=y.half()), dict(activation="relu"), dict(activation="relu", pre=x), dict(activation="none", x=x[:, :5]), dict(activation="x")):
        with pytest.raises(ValueError):
            dense.linear_backward(**{**dict(grad=y, x=x, w=w), **change})
    for change in (dict(scale=v[:5]), dict(shift=v.half()), dict(eps=0), dict(eps=-1e-5), dict(x=x.double()), dict(out=x.half()), dict(out=y), dict(scale=v.cpu())):
        with pytest.raises(ValueError):
            dense.layer_norm(**{**dict(x=x, scale=v, shift=v), **change})
    big = torch.zeros(100, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        dense.layer_norm(big.as_strided((9, 6), (6, 1)), v, v, out=big.as_strided((9, 6), (6, 1), 6))
    for change in (dict(grad=y), dict(mean=m[:8]), dict(rstd=m.half()), dict(out=y), dict(scale=m), dict(mirror_rows=m), dict(mirror_rows=m.int()[:3])):
        with pytest.raises(ValueError):
            dense.layer_norm_backward(**{**dict(grad=x, x=x, scale=v, mean=m, rstd=m), **change})
    for change in (dict(teacher=x[:8, :2]), dict(classes=ids.int()), dict(classes=ids[:, :1]), dict(temperature=0.0), dict(temperature=1e9), dict(truth=ids[:, 0].contiguous()),
                   dict(labelled=m > 0), dict(truth=ids[:, 0], labelled=m > 0), dict(truth=ids[:, 0].int(), labelled=m > 0), dict(logits=x.double()), dict(teacher=x[:, :2].cpu()),
                   dict(teacher=torch.zeros((9, 257), device="cuda"), classes=torch.zeros((9, 257), dtype=torch.int64, device="cuda"))):
        with pytest.raises(ValueError):
            dense.distillation_loss(**{**dict(logits=x, teacher=x[:, :2], classes=ids), **change})


def test_what_lies_behind_the_last_row_stays(cuda_device):
    """Outputs in a larger buffer: rows behind the last and values behind a row's last are left as they were."""
    gen = torch.Generator(cuda_device).manual_seed(6)
    for dtype in (torch.float32, torch.bfloat16):
        for n in (1, 200, 5000):
            x, w = torch.randn((n, 64), device="cuda", generator=gen).to(dtype), torch.randn((64, 96), device="cuda", generator=gen).to(dtype)
            out, pre = (torch.full((n + 130, 104), 5.0, dtype=dtype, device="cuda") for _ in range(2))
            dense.linear(x, w, out=out[:n, :96], pre=pre[:n, :96])
            for t in (out, pre):
                assert (t[n:] == 5).all() and (t[:, 96:] == 5).all() and not (t[:n, :96] == 5).all()
