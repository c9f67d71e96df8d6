"""The dense operators beside the aggregation, as a list of measured cases: what a training step or an answer of a residual graph
network needs besides its aggregations, and what the model that is taught by it needs.

A case is a plain dict.  Its "kind" names the entry point of drone_b200.dense it goes through:

  linear            Y = activation(X . W + bias) + residual, on request with the values before the activation
  linear_backward   the gradients of X, W and the bias from that of Y, with the values before the activation kept
  norm              layer norm of the rows, on request with a ReLU behind it; mean and reciprocal deviation come with it
  norm_backward     the gradients of its input, scale and shift
  distillation      loss and gradient of logits against a teacher's top logits, with a share of labelled rows

Widths and numbers of rows are those of the graphs the benchmark uses (Reddit-shaped: 232,965 vertices, 602-128-41;
products-shaped: 2,449,029 vertices, 100-256-256-47), of its small test graphs, and generic ones.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5


def listed():
    linear = dict(kind="linear", type="f32", bias=True, activation="none", residual=False, transposed=False, pad=0, keep=False)
    back = dict(kind="linear_backward", type="f32", bias=True, activation="none", transposed=False, pad=0)
    norm = dict(kind="norm", type="f32", relu=False, pad=0)
    norm_back = dict(kind="norm_backward", type="f32", relu=False, pad=0)
    taught = dict(kind="distillation", type="f32", temperature=2.0, hard=0.0, pad=0)
    return [
        # the answer for one vertex that has just been asked for: the first layer of the Reddit-shaped model on a single row
        dict(linear, name="linear_one_row", rows=1, inputs=602, outputs=128, activation="relu"),
        # the first layer over all vertices of the Reddit-shaped graph; rows of 2408 bytes
        dict(linear, name="linear_reddit_602_128", rows=232965, inputs=602, outputs=128, activation="relu"),
        # a residual block of the products-shaped model in half the memory, as a training step runs it
        dict(linear, name="linear_products_256_bf16", rows=2449029, inputs=256, outputs=256, type="bf16", activation="gelu",
             residual=True, keep=True),
        # logits of a mini-batch of vertices: an odd width
        dict(linear, name="linear_logits_47_f16", rows=20011, inputs=256, outputs=47, type="f16"),
        # the backward pass of the Reddit-shaped model's first layer, the gradient of its input among it
        dict(back, name="linear_backward_reddit_602_128", rows=232965, inputs=602, outputs=128, activation="relu"),
        # the backward pass of a hidden layer in 16 bits with weights kept as [outputs, inputs], rows that fill no tile
        dict(back, name="linear_backward_512_bf16", rows=100003, inputs=512, outputs=512, type="bf16", activation="gelu",
             transposed=True),
        # the norm ahead of a block of the products-shaped model: one pass over 2.5 GB
        dict(norm, name="norm_products_256", rows=2449029, width=256, relu=True),
        # the same for a handful of asked-for vertices of an odd width
        dict(norm, name="norm_few_rows_f16", rows=37, width=41, type="f16"),
        # its backward pass on the Reddit-shaped graph's hidden width
        dict(norm_back, name="norm_backward_reddit_128", rows=232965, width=128, relu=True),
        # the backward pass of a wide norm in 16 bits
        dict(norm_back, name="norm_backward_1024_bf16", rows=65537, width=1024, type="bf16"),
        # all vertices of the products-shaped graph taught by a larger model's best eight of 47 classes, some labelled
        dict(taught, name="distillation_products_47", rows=2449029, classes=47, top=8, hard=0.5),
        # many classes: a mini-batch over 32,000 of them, the teacher's best 64
        dict(taught, name="distillation_32000_bf16", rows=8192, classes=32000, top=64, type="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear"] * 3 + ["linear_backward"] * 2 + ["norm", "norm_backward"] + ["distillation"] * 2)
    case = dict(kind=kind, type=rng.choice(sorted(TYPES)), pad=rng.choice([0, 0, 1, 3, 8]))
    rows = _log_int(rng, 1, 2449029)
    if kind in ("linear", "linear_backward"):
        inputs, outputs = _log_int(rng, 1, 1024), _log_int(rng, 1, 1024)
        # no more values and products than the largest listed case of the kind
        most, products = (1.2e9, 1.5e11) if kind == "linear" else (1.7e8, 1.8e10)
        rows = max(1, min(rows, int(most / (inputs + 2 * outputs)), int(products / (inputs * outputs))))
        case.update(rows=rows, inputs=inputs, outputs=outputs, bias=rng.random() < 0.7, transposed=rng.random() < 0.4,
                    activation=rng.choice(["none", "relu", "gelu", "silu"]))
        if kind == "linear":
            case.update(residual=rng.random() < 0.5, keep=rng.random() < 0.3)
    elif kind in ("norm", "norm_backward"):
        width = _log_int(rng, 2, 4096)
        case.update(rows=max(1, min(rows, int((6.2e8 if kind == "norm" else 6.5e7) / width))), width=width, relu=rng.random() < 0.5)
    else:
        classes = _log_int(rng, 2, 32000)
        case.update(rows=max(1, min(rows, int((1.1e8 if classes < 1000 else 2.6e8) / classes))), classes=classes,
                    top=min(_log_int(rng, 1, 128), classes), temperature=rng.choice([1.0, 2.0, 4.0]), hard=rng.choice([0.0, 0.5]))
    return case


def _rows(gen, rows, width, dtype, pad, scale=1.0, shift=0.0):
    """Rows that lie `pad` values further apart than they are wide."""
    t = torch.empty((rows, width + pad), dtype=dtype, device="cuda")[:, :width]
    step = max(1, (1 << 27) // width)
    for r in range(0, rows, step):
        part = torch.randn((min(step, rows - r), width), device="cuda", generator=gen)
        t[r:r + step] = part.mul_(scale).add_(shift)
    return t


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    dtype, rows, pad, kind = TYPES[case["type"]], case["rows"], case["pad"], case["kind"]
    s = dict(case=case)
    if kind in ("linear", "linear_backward"):
        k, n = case["inputs"], case["outputs"]
        s["x"] = _rows(gen, rows, k, dtype, pad)
        # uniform weights of the usual size, rows [inputs, outputs] or [outputs, inputs]
        w = ((torch.rand((k, n), device="cuda", generator=gen) - 0.5) * 2 * math.sqrt(6.0 / (k + n))).to(dtype)
        s["w"] = w.t().contiguous() if case["transposed"] else w
        s["bias"] = torch.randn(n, device="cuda", generator=gen) / 8 if case["bias"] else None
        if kind == "linear":
            s["residual"] = _rows(gen, rows, n, dtype, pad) if case["residual"] else None
        else:
            s["grad"] = _rows(gen, rows, n, dtype, pad, 0.1)
            # values before the activation: of the size that the product of such inputs has
            s["pre"] = None if case["activation"] == "none" else _rows(gen, rows, n, dtype, pad, math.sqrt(2.0 * k / (k + n)))
    elif kind in ("norm", "norm_backward"):
        f = case["width"]
        s["x"] = _rows(gen, rows, f, dtype, pad, 1.5, 0.3)
        s["scale"] = 1 + torch.randn(f, device="cuda", generator=gen) / 8
        s["shift"] = torch.randn(f, device="cuda", generator=gen) / 8
        if kind == "norm_backward":
            s["grad"] = _rows(gen, rows, f, dtype, pad, 0.1)
            x = s["x"].float()
            mean = x.mean(dim=1, dtype=torch.float64)
            var = (x - mean[:, None].float()).square_().mean(dim=1, dtype=torch.float64)
            s["mean"], s["rstd"] = mean.float(), (var + EPS).rsqrt().float()
            # the forward pass's output says where the ReLU let a value through
            s["out"] = None
            if case["relu"]:
                y = (x - s["mean"][:, None]) * s["rstd"][:, None] * s["scale"] + s["shift"]
                s["out"] = y.clamp_(min=0).to(dtype)
    else:
        c, k = case["classes"], case["top"]
        s["logits"] = _rows(gen, rows, c, dtype, pad, 2.0)
        # the teacher's best classes of a row, best first: k different ones, a few rows with fewer of them or none
        step = torch.randint(1, max(2, c // k + 1), (rows, k), device="cuda", generator=gen)
        first = torch.randint(0, c, (rows, 1), device="cuda", generator=gen)
        classes = (first + step.cumsum(dim=1) - step[:, :1]) % c
        fewer = torch.rand((rows, 1), device="cuda", generator=gen)
        known = torch.where(fewer < 0.05, (fewer * 20 * (k + 1)).long(), k)
        s["classes"] = torch.where(torch.arange(k, device="cuda") < known, classes, -1)
        s["teacher"] = (torch.randn((rows, k), device="cuda", generator=gen).mul_(2).sort(dim=1, descending=True).values + 4).to(dtype)
        s["truth"] = torch.randint(0, c, (rows,), device="cuda", generator=gen)
        s["labelled"] = torch.rand(rows, device="cuda", generator=gen) < 0.3
    return s


# ----- the plain forms -----

def _weights(s):
    w = s["w"].float()
    return w.t() if s["case"]["transposed"] else w


def _activate(z, name):
    if name == "relu":
        return z.clamp(min=0)
    if name == "gelu":
        return z * (0.5 * (1 + torch.erf(z * math.sqrt(0.5))))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    if name == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    return torch.ones_like(z)


def _plain_linear(s):
    case, dtype = s["case"], s["x"].dtype
    z = s["x"].float() @ _weights(s)
    if s["bias"] is not None:
        z += s["bias"]
    y = _activate(z, case["activation"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return (y.to(dtype), z.to(dtype)) if case["keep"] else y.to(dtype)


def _plain_linear_backward(s):
    case, dtype = s["case"], s["x"].dtype
    dz = s["grad"].float()
    if s["pre"] is not None:
        dz = dz * _slope(s["pre"].float(), case["activation"])
    dw = s["x"].float().t() @ dz
    if case["transposed"]:
        dw = dw.t()
    dx = dz @ _weights(s).t()
    return dx.to(dtype), dw.to(dtype), dz.sum(dim=0, dtype=torch.float64).float() if case["bias"] else None


def _plain_norm(s):
    x = s["x"].float()
    mean = x.mean(dim=1, keepdim=True)
    off = x - mean
    rstd = 1 / torch.sqrt((off * off).mean(dim=1, keepdim=True) + EPS)
    y = off * rstd * s["scale"] + s["shift"]
    if s["case"]["relu"]:
        y = y.clamp(min=0)
    return y.to(s["x"].dtype), mean[:, 0], rstd[:, 0]


def _plain_norm_backward(s):
    g = s["grad"].float()
    if s["out"] is not None:
        g = g * (s["out"] > 0)
    hat = (s["x"].float() - s["mean"][:, None]) * s["rstd"][:, None]
    gs = g * s["scale"]
    dx = s["rstd"][:, None] * (gs - gs.mean(dim=1, keepdim=True) - hat * (gs * hat).mean(dim=1, keepdim=True))
    return dx.to(s["x"].dtype), (g * hat).sum(dim=0, dtype=torch.float64).float(), g.sum(dim=0, dtype=torch.float64).float()


def _plain_distillation(s):
    case, t = s["case"], s["case"]["temperature"]
    z = s["logits"].float()
    z = z - z.max(dim=1, keepdim=True).values
    known = s["classes"] >= 0
    some = known.any(dim=1)
    at = s["classes"].clamp(min=0)
    q = torch.where(known, s["teacher"].float() / t, -math.inf)
    q = torch.where(known, torch.exp(q - q.max(dim=1, keepdim=True).values), 0.0)
    q = q / torch.where(some, q.sum(dim=1), 1.0)[:, None]
    e = torch.exp(z / t)
    total = e.sum(dim=1, keepdim=True)
    log_p = z.gather(1, at) / t - torch.log(total)
    soft = t * t * (q * (torch.log(torch.where(q > 0, q, 1.0)) - log_p)).sum(dim=1)
    grad = e / total * t * some[:, None]
    grad.scatter_add_(1, at, -t * q)
    loss = torch.zeros(2, dtype=torch.float64, device=z.device)
    loss[0] = (soft * some).sum(dtype=torch.float64) / some.sum().clamp(min=1)
    if case["hard"]:
        e = torch.exp(z)
        total = e.sum(dim=1, keepdim=True)
        truth = s["truth"][:, None]
        hard = torch.log(total) - z.gather(1, truth)
        p = e / total
        p.scatter_add_(1, truth, -torch.ones_like(hard))
        grad = (1 - case["hard"]) * grad + case["hard"] * p * s["labelled"][:, None]
        loss[1] = (hard[:, 0] * s["labelled"]).sum(dtype=torch.float64) / s["labelled"].sum().clamp(min=1)
    return loss.float(), grad.to(s["logits"].dtype)


def _own(s):
    from drone_b200 import dense
    case, kind = s["case"], s["case"]["kind"]
    if kind == "linear":
        pre = s["x"].new_empty((case["rows"], case["outputs"])) if case["keep"] else None
        y = dense.linear(s["x"], s["w"], bias=s["bias"], activation=case["activation"], residual=s["residual"],
                         transposed=case["transposed"], pre=pre)
        return (y, pre) if case["keep"] else y
    if kind == "linear_backward":
        return dense.linear_backward(s["grad"], s["x"], s["w"], pre=s["pre"], activation=case["activation"],
                                     transposed=case["transposed"], bias=case["bias"])
    if kind == "norm":
        return dense.layer_norm(s["x"], s["scale"], s["shift"], eps=EPS, relu=case["relu"])
    if kind == "norm_backward":
        return dense.layer_norm_backward(s["grad"], s["x"], s["scale"], s["mean"], s["rstd"], out=s["out"])
    hard = dict(truth=s["truth"], labelled=s["labelled"], soft=1 - case["hard"], hard=case["hard"]) if case["hard"] else {}
    return dense.distillation_loss(s["logits"], s["teacher"], s["classes"], temperature=case["temperature"], **hard)


def run(state):
    if own:
        return _own(state)
    return {"linear": _plain_linear, "linear_backward": _plain_linear_backward, "norm": _plain_norm,
            "norm_backward": _plain_norm_backward, "distillation": _plain_distillation}[state["case"]["kind"]](state)


def work(case):
    size, rows = SIZE[case["type"]], case["rows"]
    if case["kind"] in ("linear", "linear_backward"):
        k, n = case["inputs"], case["outputs"]
        if case["kind"] == "linear":
            values = rows * k + k * n + rows * n * (1 + case["residual"] + case["keep"])
            return {"bytes": size * values + 4 * n * case["bias"], "flops": 2 * rows * k * n}
        values = 2 * rows * k + 2 * k * n + rows * n * (1 + (case["activation"] != "none"))
        return {"bytes": size * values + 4 * n * case["bias"], "flops": 4 * rows * k * n}
    if case["kind"] == "norm":
        return {"bytes": rows * (2 * case["width"] * size + 8) + 8 * case["width"], "flops": 8 * rows * case["width"]}
    if case["kind"] == "norm_backward":
        return {"bytes": rows * ((3 + case["relu"]) * case["width"] * size + 8) + 12 * case["width"], "flops": 14 * rows * case["width"]}
    per_row = 2 * case["classes"] * size + case["top"] * (8 + size) + (9 if case["hard"] else 0)
    return {"bytes": rows * per_row + 8, "flops": rows * case["classes"] * (14 if case["hard"] else 8)}


# ----- the definitions in 64 bits -----

def _blocks(rows, width):
    """Row ranges whose values take about 2 GB as doubles."""
    step = max(1, (1 << 28) // max(1, width))
    return [slice(r, min(r + step, rows)) for r in range(0, rows, step)]


def _exact_linear(s, case):
    w = s["w"].double()
    w = w.t() if case["transposed"] else w
    dtype, ys, zs = s["x"].dtype, [], []
    out = torch.float64 if dtype == torch.float32 else torch.float32
    for b in _blocks(case["rows"], case["inputs"] + 3 * case["outputs"]):
        z = torch.matmul(s["x"][b].double(), w)
        if s["bias"] is not None:
            z = z + s["bias"].double()
        y = {"none": lambda v: v, "relu": torch.relu, "gelu": lambda v: v * torch.special.ndtr(v),
             "silu": lambda v: v * torch.sigmoid(v)}[case["activation"]](z)
        if s["residual"] is not None:
            y = y + s["residual"][b].double()
        ys.append(y.to(out))
        if case["keep"]:
            zs.append(z.to(out))
    return (torch.cat(ys), torch.cat(zs)) if case["keep"] else torch.cat(ys)


def _exact_linear_backward(s, case):
    w = s["w"].double()
    w = w.t() if case["transposed"] else w
    dtype, dxs = s["x"].dtype, []
    dw = torch.zeros_like(w)
    db = torch.zeros(case["outputs"], dtype=torch.float64, device="cuda")
    for b in _blocks(case["rows"], 2 * case["inputs"] + 3 * case["outputs"]):
        dz = s["grad"][b].double()
        if s["pre"] is not None:
            v = s["pre"][b].double()
            if case["activation"] == "relu":
                dz = torch.where(v > 0, dz, 0.0)
            elif case["activation"] == "gelu":
                dz = dz * (torch.special.ndtr(v) + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi))
            else:
                dz = dz * (torch.sigmoid(v) + v * torch.sigmoid(v) * torch.sigmoid(-v))
        dxs.append(torch.matmul(dz, w.t()))
        dw += torch.matmul(s["x"][b].double().t(), dz)
        db += dz.sum(dim=0)
    return torch.cat(dxs), dw.t() if case["transposed"] else dw, db if case["bias"] else None


def _exact_norm(s, case):
    ys, means, rstds = [], [], []
    out = torch.float64 if s["x"].dtype == torch.float32 else torch.float32
    for b in _blocks(case["rows"], 3 * case["width"]):
        x = s["x"][b].double()
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        rstd = (var + EPS) ** -0.5
        y = torch.addcmul(s["shift"].double(), (x - mean) * rstd, s["scale"].double())
        ys.append((torch.relu(y) if case["relu"] else y).to(out))
        means.append(mean.flatten())
        rstds.append(rstd.flatten())
    return torch.cat(ys), torch.cat(means), torch.cat(rstds)


def _exact_norm_backward(s, case):
    f = case["width"]
    dxs = []
    d_scale, d_shift = (torch.zeros(f, dtype=torch.float64, device="cuda") for _ in range(2))
    for b in _blocks(case["rows"], 5 * f):
        g = s["grad"][b].double()
        if s["out"] is not None:
            g = torch.where(s["out"][b] > 0, g, 0.0)
        rstd = s["rstd"][b].double()[:, None]
        hat = (s["x"][b].double() - s["mean"][b].double()[:, None]) * rstd
        d_hat = g * s["scale"].double()
        dxs.append(rstd / f * (f * d_hat - d_hat.sum(dim=1, keepdim=True) - hat * torch.linalg.vecdot(d_hat, hat)[:, None]))
        d_scale += torch.einsum("rf,rf->f", g, hat)
        d_shift += g.sum(dim=0)
    return torch.cat(dxs), d_scale, d_shift


def _exact_distillation(s, case):
    t, grads = case["temperature"], []
    out = torch.float64 if s["logits"].dtype == torch.float32 else torch.float32
    sums = torch.zeros(4, dtype=torch.float64, device="cuda")
    for b in _blocks(case["rows"], 4 * case["classes"]):
        z, classes = s["logits"][b].double(), s["classes"][b]
        teacher = torch.where(classes >= 0, s["teacher"][b].double() / t, -math.inf)
        has = (classes >= 0).sum(dim=1) > 0
        log_q = torch.log_softmax(torch.where(has[:, None], teacher, 0.0), dim=1)
        q = torch.where(classes >= 0, log_q.exp(), 0.0)
        log_p = torch.log_softmax(z / t, dim=1)
        apart = torch.where(q > 0, q * (log_q - log_p.gather(1, classes.clamp(min=0))), 0.0).sum(dim=1)
        sums[0] += t * t * apart[has].sum()
        sums[1] += has.sum()
        target = torch.zeros_like(z).scatter_add_(1, classes.clamp(min=0), q)
        grad = torch.where(has[:, None], t * (log_p.exp() - target), 0.0)
        if case["hard"]:
            log_p = torch.log_softmax(z, dim=1)
            truth, lab = s["truth"][b], s["labelled"][b]
            sums[2] -= log_p.gather(1, truth[:, None])[:, 0][lab].sum()
            sums[3] += lab.sum()
            hard = log_p.exp()
            hard[torch.arange(len(truth), device="cuda"), truth] -= 1
            grad = (1 - case["hard"]) * grad + torch.where(lab[:, None], case["hard"] * hard, 0.0)
        grads.append(grad.to(out))
    return torch.stack([sums[0] / sums[1].clamp(min=1), sums[2] / sums[3].clamp(min=1)]), torch.cat(grads)


def exact(case, seed):
    state = prepare(case, seed)
    return {"linear": _exact_linear, "linear_backward": _exact_linear_backward, "norm": _exact_norm,
            "norm_backward": _exact_norm_backward, "distillation": _exact_distillation}[case["kind"]](state, case)
