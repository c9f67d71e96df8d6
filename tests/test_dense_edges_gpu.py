"""Edges of the dense operators: infinities through the activations, tails, logits with an offset, values at the ends of their type, rows that count for nothing, sums over very
many rows."""
import ctypes as C
import math

import pytest
import torch

from drone_b200 import _lib, dense, gcn
from test_dense_gpu import STEP, TYPES, activated, check_linear, check_rounded, distilled, rows_of, slope
from test_residual_gcn_gpu import graph_of, parameters

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 3, 700])
@pytest.mark.parametrize("activation", ["relu", "gelu", "silu"])
def test_activations_of_infinities(cuda_device, activation, n, dtype):
    """An infinite or undefined value before the activation comes out as the formula has it: z Phi(z) and z / (1 + exp(-z)) are infinite at +infinity,
    undefined at -infinity."""
    gen = torch.Generator(cuda_device).manual_seed(n)
    for k, m in ((2, 8), (70, 200)):      # by itself and in tiles
        x, w, bias = rows_of(gen, n, k, dtype), rows_of(gen, k, m, dtype), torch.randn(m, device="cuda", generator=gen)
        bias[1], bias[2], bias[3], bias[4], bias[5] = math.inf, -math.inf, math.nan, 1e30, -1e30
        pre = torch.empty((n, m), dtype=dtype, device="cuda")
        got = dense.linear(x, w, bias=bias, activation=activation, pre=pre)
        z = x.double() @ w.double() + bias.double()
        want = activated(z, activation)
        top = torch.finfo(dtype).max
        inf = want.abs() > top      # 1e30 is infinite in 16 bits of a 5-bit exponent
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), inf) and (got[inf] > 0).all()
        assert torch.equal(pre.isnan(), z.isnan()) and torch.equal(pre.isinf(), z.abs() > top)


def test_gelu_tails_of_16_bits(cuda_device):
    """z Phi(z) and its slope as good as their types as far out as there is anything.  The tail's polynomial is good to 4.4e-5 of the value; the exponent of its
    bell, up to 126 and off by three half steps, makes 126 * 3 * 2^-24 * ln 2 = 1.6e-5 of it; together 2^-14.  Below 2^-126 the exponential is 0."""
    for dtype in (torch.bfloat16, torch.float16):
        z = torch.linspace(-14, 14, 4001, device="cuda").to(dtype)[:, None]
        one = torch.ones((1, 1), dtype=dtype, device="cuda")
        phi = lambda v: 0.5 * torch.special.erfc(-v * math.sqrt(0.5))      # torch.special.ndtr is a difference from 1, good to 2^-53 of that
        got, want = dense.linear(z, one, activation="gelu"), z.double() * phi(z.double())
        gone = 16 * 2.0 ** -126
        tail = z.double().abs() * phi(-z.double().abs())
        check_rounded(got, want, 2.0 ** -14 * tail + 2 * STEP * want.abs() + gone, dtype)
        # of one row the bias gradient is the gradient before the activation, not rounded
        pre = z.t().contiguous()
        got = dense.linear_backward(torch.ones_like(pre), one, one.expand(1, pre.shape[1]).contiguous(), pre=pre, activation="gelu")[2]
        v = pre.double()[0]
        bell = torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
        size = phi(-v.abs()) + v.abs() * bell
        assert ((got - (phi(v) + v * bell)).abs() <= 2.0 ** -14 * size + 2 * STEP * (v >= 0) + gone).all()


@pytest.mark.parametrize("c", [47, 200, 257, 4096, 9001])
@pytest.mark.parametrize("t", [1.0, 4.0, 1e-3, 1e-6])
def test_logits_with_an_offset(cuda_device, c, t):
    """What all logits of a row have in common leaves no trace, however large: a row's shares follow from differences, which are exact or off by half a step.  An exponent x
    that is off by 4 half steps moves exp(-x) by x exp(-x) of them, less than one."""
    gen = torch.Generator(cuda_device).manual_seed(c)
    offsets = [0.0, 100.0, -1e4, 1e4, 1e5, 1e6, -1e9, 1e10, -1e10, 1e20, 3e30, -3e38]
    n = len(offsets)
    logits = rows_of(gen, n, c, torch.float32, scale=3.0 * min(t, 1.0)) + torch.tensor(offsets, device="cuda")[:, None]
    logits[::2, 5:9] = -3e38      # classes that are masked with a low value beside the others
    teacher, classes = rows_of(gen, n, 4, torch.float32, scale=min(t, 1.0)), torch.randint(9, c, (n, 4), device="cuda", generator=gen)
    truth, labelled = torch.randint(9, c, (n,), device="cuda", generator=gen), torch.ones(n, dtype=torch.bool, device="cuda")
    off = (16 + c / 64) * STEP
    for r in range(n):      # a row at a time, so that each has its own bound
        at = slice(r, r + 1)
        loss, grad = dense.distillation_loss(logits[at], teacher[at], classes[at], temperature=t, truth=truth[at], labelled=labelled[at], soft=0.5, hard=0.5)
        want_loss, want = distilled(logits[at], teacher[at], classes[at], t, truth[at], labelled[at], 0.5, 0.5)
        check_rounded(grad, want, off * (0.5 * t + 0.5) * torch.ones_like(want), torch.float32)
        apart = (logits[at].double().max() - logits[at].double().gather(1, torch.cat([classes[at], truth[at][:, None]], dim=1))).abs().max().item()
        assert abs(loss[0] - want_loss[0]) <= off * t * t * (8 + (apart + 10 * t) / t), (offsets[r], loss, want_loss)
        assert abs(loss[1] - want_loss[1]) <= off * (8 + apart), (offsets[r], loss, want_loss)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c", [7, 47, 200, 300])
def test_teachers_of_extreme_values(cuda_device, c, dtype):
    """Entries at either end of their type, at temperatures whose quotient with them is no float: equal entries have equal shares, the others none."""
    gen = torch.Generator(cuda_device).manual_seed(c)
    low, top = torch.finfo(dtype).min, torch.finfo(dtype).max
    for t in (1.0, 0.5, 1e-3, 1e-6):
        logits, teacher = rows_of(gen, 6, c, torch.float32, scale=min(t, 1.0)), rows_of(gen, 6, 4, dtype)
        classes = torch.arange(4, device="cuda").expand(6, 4).contiguous()
        teacher[1], teacher[2, 1:], teacher[3], teacher[4, 2], teacher[5] = low, low, top, top, torch.tensor([low, top, -math.inf, low]).to(teacher)
        loss, grad = dense.distillation_loss(logits, teacher, classes, temperature=t)
        want_loss, want = distilled(logits, teacher, classes, t, None, None, 1.0, 0.0)
        # teachers' values around 1 over t = 1e-6: a share is exp(-x) with x off by 4 half steps
        check_rounded(grad, want, (16 + c / 64) * STEP * t * torch.ones_like(want), torch.float32)
        assert abs(loss[0] - want_loss[0]) <= (16 + c / 64) * STEP * t * t * (20 + (teacher[0].max() - teacher[0].min()).item() / t)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c", [5, 47, 200, 300])
def test_rows_without_a_label_need_none(cuda_device, c, dtype):
    """-1 for vertices without a label, as the graph models' own truth has it: the bits of any other class there."""
    gen = torch.Generator(cuda_device).manual_seed(c)
    n = 70
    logits, teacher, classes = rows_of(gen, n, c, dtype), rows_of(gen, n, 3, dtype), torch.randint(-1, c, (n, 3), device="cuda", generator=gen)
    truth = torch.randint(0, c, (n,), device="cuda", generator=gen)
    labelled = torch.rand(n, device="cuda", generator=gen) < 0.4
    run = lambda given: dense.distillation_loss(logits, teacher, classes, truth=given, labelled=labelled, soft=0.5, hard=0.5)
    want = run(truth)
    for none in (-1, c, -(1 << 40), 1 << 40):
        got = run(torch.where(labelled, truth, none))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and got[0].isfinite().all() and got[1].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c", [5, 47, 200, 300])
def test_rows_that_count_for_nothing_may_hold_anything(cuda_device, c, dtype):
    """Rows without entry and label, such as padding: whatever their logits are, their gradient is 0 and the others' results are what they are without them."""
    gen = torch.Generator(cuda_device).manual_seed(c)
    n = 40
    logits, teacher, classes = rows_of(gen, n, c, dtype), rows_of(gen, n, 3, dtype), torch.randint(0, c, (n, 3), device="cuda", generator=gen)
    truth, labelled = torch.randint(0, c, (n,), device="cuda", generator=gen), torch.rand(n, device="cuda", generator=gen) < 0.5
    none = torch.zeros(n, dtype=torch.bool, device="cuda")
    none[3::5] = True
    classes[none], labelled = -1, labelled & ~none
    for hard in (False, True):
        run = lambda: dense.distillation_loss(logits, teacher, classes, **(dict(truth=truth, labelled=labelled, soft=0.5, hard=0.5) if hard else {}))
        logits[none] = 0
        want = run()
        for value in (math.nan, math.inf, -math.inf, torch.finfo(dtype).min):
            logits[none] = value
            got = run()
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and (got[1][none] == 0).all(), value


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_weight_gradients_over_very_many_rows(cuda_device, dtype, transposed):
    """Tiles that fill the GPU by themselves, so that none is cut along the rows, and factors of one sign: an accumulator that cuts off with every addition must not run through
    all of them.  It runs through 8192 rows, 512 additions of 16 products, which lose a step of the sum each (measured: 0.8 of one); what it holds then is added 49 times."""
    gen = torch.Generator(cuda_device).manual_seed(1)
    n, k, m = 400_003, 2048, 1280
    x, g = (torch.rand((n, f), device="cuda", generator=gen).add_(0.5).to(dtype) for f in (k, m))
    w = torch.zeros((m, k) if transposed else (k, m), dtype=dtype, device="cuda")
    g *= 2.0 ** -8      # sums of 400,003 products stay below the largest of any type
    dw = dense.linear_backward(g, x, w, transposed=transposed, bias=False, input_gradient=False)[1]
    for i, j in ((0, 0), (k - 100, m - 100), (1000, 200)):
        want = x[:, i:i + 100].double().t() @ g[:, j:j + 100].double()
        got = dw[j:j + 100, i:i + 100].t() if transposed else dw[i:i + 100, j:j + 100]
        check_rounded(got, want, (512 + 49 + 16) * STEP * want, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [4, 9, 15, 16, 17, 31, 33, 47, 48, 49, 63, 65, 97, 129, 145, 257, 300])
def test_tiles_of_few_columns(cuda_device, m, dtype):
    """The warps that take a tile out share its columns, however few they are, also where the last tile of a row of tiles has fewer than the others; rows that lie any distance
    apart are taken out a value a lane, the others 4 or 8."""
    gen = torch.Generator(cuda_device).manual_seed(m)
    for pad, lead in ((0, 0), (1, 0), (3, 1), (8, 0)):
        check_linear(gen, 40011, 40, m, dtype, bias=True, residual=True, activation="gelu", keep=True, pad=pad, lead=lead)
        check_linear(gen, 40011, 33, m, dtype, activation="silu", transposed=True, pad=pad, lead=lead)
        check_linear(gen, 2100, 600, m, dtype, residual=True, pad=pad, lead=lead)


def in_tiles(x, w, transposed=False):
    """Whether such a product of floats goes through tiles, whose operands are split: it asks for an image of the weights."""
    size = C.c_longlong(0)
    rows, outputs = x.shape[0], w.shape[0 if transposed else 1]
    _lib.check(_lib.lib().drone_linear_scratch(_lib.F32, rows, x.shape[1], outputs, x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), int(transposed), C.byref(size)))
    return size.value > 0


@pytest.mark.parametrize("transposed", [False, True])
def test_split_products_one_by_one(cuda_device, transposed):
    """One product an output, beside others with 0, of full mantissas and any size: six products of a float's parts leave two steps of it, or six of the smallest floats."""
    gen = torch.Generator(cuda_device).manual_seed(2)
    x = rows_of(gen, 700, 1, torch.float32) * torch.exp2(torch.randint(-60, 60, (700, 1), device="cuda", generator=gen).float())
    w = rows_of(gen, 40, 200, torch.float32) * torch.exp2(torch.randint(-60, 60, (1, 200), device="cuda", generator=gen).float())
    at = torch.randint(0, 40, (700, 1), device="cuda", generator=gen)
    x = torch.zeros((700, 40), device="cuda").scatter_(1, at, x)
    given = w.t().contiguous() if transposed else w
    assert in_tiles(x, given, transposed)
    want, got = x.double() @ w.double(), dense.linear(x, given, transposed=transposed)
    assert ((got - want).abs() <= 2 * STEP * want.abs() + 6 * 2.0 ** -149).all()


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("n,k,m", [(513, 255, 33), (1400, 600, 32), (1744, 601, 9), (1745, 601, 9), (8192, 100, 33), (8192, 128, 32), (8192, 129, 32), (8192, 3, 31), (8193, 17, 30), (20011, 9, 17)])
def test_more_rows_of_few_columns(cuda_device, n, k, m, transposed):
    """Floats of at most 32 columns, on both sides of the number of rows up to which they go eight at a time."""
    gen = torch.Generator(cuda_device).manual_seed(n)
    for pad, lead in ((0, 0), (3, 1)):
        check_linear(gen, n, k, m, torch.float32, bias=True, residual=True, activation="gelu", keep=True, transposed=transposed, pad=pad, lead=lead)
        check_linear(gen, n, k, m, torch.float32, transposed=transposed, pad=pad, lead=lead)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k,m", [(513, 129, 1), (600, 4096, 2), (700, 8192, 1), (700, 8193, 1), (3001, 2048, 4), (3001, 2049, 3), (20011, 33, 4), (20011, 200, 3), (5003, 602, 2), (70001, 65, 2),
                                   (513, 1, 129), (600, 2, 65), (2100, 3, 43), (2100, 4, 128), (2100, 4, 1000), (3001, 1, 447), (3001, 3, 32768), (70001, 2, 131), (20011, 4, 33)])
def test_thin_products_and_their_gradients(cuda_device, n, k, m, dtype):
    """Weights of a few rows or columns: forward with everything that an epilogue may have, both orders of the weights, and all three gradients; some rows far apart, not on 16 bytes."""
    gen = torch.Generator(cuda_device).manual_seed(n + k + m)
    for pad, lead in ((0, 0), (3, 1)):
        check_linear(gen, n, k, m, dtype, bias=True, residual=True, activation="gelu", keep=True, pad=pad, lead=lead)
        check_linear(gen, n, k, m, dtype, transposed=True, activation="silu", pad=pad, lead=lead)
        x, g = rows_of(gen, n, k, dtype, pad, lead), rows_of(gen, n, m, dtype, pad, lead)
        for transposed in (False, True):
            w = rows_of(gen, m, k, dtype) if transposed else rows_of(gen, k, m, dtype)
            dx, dw, db = dense.linear_backward(g, x, w, transposed=transposed)
            wd = w.double().t() if transposed else w.double()
            want, bound = x.double().t() @ g.double(), (n + 16) * STEP * (x.double().abs().t() @ g.double().abs())
            check_rounded(dw, want.t() if transposed else want, bound.t() if transposed else bound, dtype)
            check_rounded(dx, g.double() @ wd.t(), (m + 16) * STEP * (g.double().abs() @ wd.t().abs()), dtype)
            check_rounded(db, g.double().sum(dim=0), (n + 16) * STEP * g.double().abs().sum(dim=0), torch.float32)
            again = dense.linear_backward(g, x, w, transposed=transposed)
            assert all(torch.equal(a, b) for a, b in zip((dx, dw, db), again))


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("n,k,m", [(700, 256, 200), (700, 602, 128), (1000, 1025, 41), (600, 4096, 130)])
def test_split_products_are_as_good_as_floats(cuda_device, n, k, m, transposed):
    """Factors of one sign, where what is left out or cut off adds up: a product is off by 2 steps, an accumulator by one with each of its 16 additions of 16 products (times
    two: there are two accumulators, the second far smaller), and every 256 of K the sum is rounded.  Without the third parts it would be 256 steps."""
    gen = torch.Generator(cuda_device).manual_seed(k)
    x, w = (torch.rand(shape, device="cuda", generator=gen) + 0.5 for shape in ((n, k), (k, m)))
    given = w.t().contiguous() if transposed else w
    assert in_tiles(x, given, transposed)
    want, got = x.double() @ w.double(), dense.linear(x, given, transposed=transposed)
    assert ((got - want).abs() <= (2 + 18 + k / 256) * STEP * want).all()


@pytest.mark.parametrize("transposed", [False, True])
def test_split_products_of_infinities(cuda_device, transposed):
    """Infinities and NaN in float tiles reach the outputs that they reach in the formula, forward and in the gradient of the rows."""
    gen = torch.Generator(cuda_device).manual_seed(3)
    x, w = rows_of(gen, 700, 70, torch.float32), rows_of(gen, 70, 150, torch.float32)
    x[0, 3], x[1, 69], x[2, 40], x[650, 0] = math.inf, -math.inf, math.nan, math.inf
    w[10, 7], w[69, 8], w[0, 149] = math.inf, 0, -math.inf
    for rows, weights in ((x, w), (rows_of(gen, 700, 150, torch.float32), w.t())):
        given = weights.t().contiguous() if transposed else weights.contiguous()
        assert in_tiles(rows, given, transposed)
        got, want = dense.linear(rows, given, transposed=transposed), rows.double() @ weights.double()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf()) and torch.equal(got[want.isinf()].double(), want[want.isinf()])
        fine = want.isfinite()
        size = rows.double().abs().nan_to_num(0, 0, 0) @ weights.double().abs().nan_to_num(0, 0, 0)
        check_rounded(got[fine], want[fine], ((rows.shape[1] + 16) * STEP * size)[fine], torch.float32)


def test_captured_step_on_other_inputs(cuda_device, oracle):
    """Captured on one input and replayed on two others, beside a second graph of the same model: the bits of the eager steps on these."""
    n, _, (graph,) = graph_of(cuda_device, oracle)
    gen = torch.Generator(cuda_device).manual_seed(7)
    dims = (40, 32, 7)
    inputs = [torch.randn((n, dims[0]), device=cuda_device, generator=gen) for _ in range(3)]
    truth = torch.randint(-1, dims[2], (n,), device=cuda_device, generator=gen, dtype=torch.int32)
    model = gcn.ResidualGCN(graph, inputs[0].clone(), truth, *parameters(cuda_device, gen, dims, 2))

    def eager(rows):
        model.x.copy_(rows)
        return [model.forward().clone(), *(g.clone() for g in model.backward())]
    wanted = [eager(rows) for rows in inputs]
    assert all(not torch.equal(a, b) for i in range(3) for a, b in zip(wanted[i], wanted[i - 1]))
    model.x.copy_(inputs[2])
    captured = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outputs = [model.forward(), *model.backward()]
        captured.append((g, outputs))
    for rows, want in zip(inputs, wanted):
        model.x.copy_(rows)
        for g, outputs in captured:
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outputs, want))
