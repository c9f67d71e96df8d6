"""The dense operators together, as a model runs them: a residual graph network's step against the same model in double, on the labels and taught by
another model, as one part and as two parts of one graph, eagerly and captured."""
import numpy as np
import pytest
import torch

from drone_b200 import gcn, graphgen as gg, graphsum as gs, partition as pt
from helpers import graph_case

pytestmark = pytest.mark.gpu


def graph_of(device, oracle, scale=9, parts=1):
    n, u, v = gg.rmat_graph(scale, 8, seed=61, symmetrise=True, self_loops="add")
    u, v = u.numpy(), v.numpy()
    index, dst, in_deg, out_deg, val = graph_case(gg, oracle, n, u, v)
    adjacency = torch.zeros((n, n), dtype=torch.float64, device=device)      # A[source, destination]
    src = np.repeat(np.arange(n), np.diff(index))
    adjacency[torch.as_tensor(src, device=device), torch.as_tensor(dst, device=device).long()] = torch.as_tensor(val, device=device).double()
    part = pt.ebv_partition(n, u, v, parts)
    graphs = [gs.DeviceGraph(part.local_graph(p), in_deg, out_deg, device, max_features=64) for p in range(parts)]
    return n, adjacency, graphs


def parameters(device, gen, dims, layers):
    widths = [(dims[0], dims[1])] + [(dims[1], dims[1])] * layers + [(dims[1], dims[2])]
    r = lambda *shape: torch.randn(shape, device=device, generator=gen)
    weights = [r(a, b) / a ** 0.5 for a, b in widths]
    biases = [r(b) / 4 for _, b in widths]
    norms = [(1 + r(dims[1]) / 4, r(dims[1]) / 4) for _ in range(layers + 1)]
    return weights, biases, norms


def step_in_double(adjacency, x, weights, biases, norms, loss_of):
    """Loss and gradients by automatic differentiation of the formulas in double."""
    leaves = [t.double().requires_grad_() for t in (*weights, *biases, *(t for pair in norms for t in pair))]
    w, b, flat = leaves[:len(weights)], leaves[len(weights):2 * len(weights)], leaves[2 * len(weights):]
    pairs = list(zip(flat[::2], flat[1::2]))
    norm = lambda z, l: torch.relu(torch.nn.functional.layer_norm(z, z.shape[1:], *pairs[l], eps=1e-5))
    z = x.double() @ w[0] + b[0]
    for l in range(1, len(weights) - 1):
        z = z + (adjacency.t() @ norm(z, l - 1)) @ w[l] + b[l]
    logits = norm(z, len(weights) - 2) @ w[-1] + b[-1]
    loss, total = loss_of(logits)
    return logits, loss, torch.autograd.grad(total, leaves)


def cross_entropy(truth):
    def of(logits):
        rows = torch.nn.functional.cross_entropy(logits, truth.clamp(min=0).long(), reduction="none") * (truth >= 0)
        return rows.sum() / (truth >= 0).sum(), rows.sum()
    return of


def taught(truth, values, classes, t, soft, hard):
    def of(logits):
        known = classes >= 0
        q = torch.softmax(torch.where(known, values.double() / t, -1e300), dim=1) * known
        log_p = torch.log_softmax(logits / t, dim=1).gather(1, classes.clamp(min=0))
        rows = t * t * (torch.where(q > 0, q * (torch.log(q.clamp(min=1e-300)) - log_p), 0.0)).sum(dim=1)
        labels = torch.nn.functional.cross_entropy(logits, truth.clamp(min=0).long(), reduction="none") * (truth >= 0)
        some = known.any(dim=1)
        return soft * rows.sum() / some.sum() + hard * labels.sum() / (truth >= 0).sum(), soft * rows.sum() + hard * labels.sum()
    return of


def rel(got, want):
    return ((got.double() - want).abs().max() / want.abs().max().clamp(min=1e-30)).item()


# The bound the path's specification gives for outputs and gradients of the graph models, for each of the few products and norms in a row.  A ReLU that
# falls the other way in float moves its entry's gradient by all of it: the chance is 1e-6 an entry, and the seeds below have none.
TOL = 5e-5


@pytest.mark.parametrize("layers", [0, 1, 3])
@pytest.mark.parametrize("dims", [(40, 32, 7), (33, 20, 41), (602, 64, 13)])
def test_step(cuda_device, oracle, dims, layers):
    n, adjacency, (graph,) = graph_of(cuda_device, oracle)
    gen = torch.Generator(cuda_device).manual_seed(sum(dims) + layers)
    order = torch.as_tensor(graph.host.l2g, device=cuda_device).long()
    x = torch.randn((n, dims[0]), device=cuda_device, generator=gen)
    truth = torch.randint(-1, dims[2], (n,), device=cuda_device, generator=gen, dtype=torch.int32)
    weights, biases, norms = parameters(cuda_device, gen, dims, layers)
    model = gcn.ResidualGCN(graph, x[order], truth[order], weights, biases, norms)
    loss = model.forward()
    grads = model.backward()
    logits, want, want_grads = step_in_double(adjacency, x, weights, biases, norms, cross_entropy(truth))
    assert rel(model.logits, logits[order]) < TOL and abs(loss.item() - want.item()) < TOL * want.item()
    assert len(grads) == len(want_grads) == len(model.parameters())
    for got, expected, parameter in zip(grads, want_grads, model.parameters()):
        assert got.shape == parameter.shape and rel(got, expected) < TOL
    before = [loss.clone(), *(g.clone() for g in grads)]
    assert all(torch.equal(a, b) for a, b in zip(before, [model.forward(), *model.backward()]))


def test_taught_step(cuda_device, oracle):
    """A small model taught by the best three classes of a wider one, half of it, and by labels."""
    n, adjacency, (graph,) = graph_of(cuda_device, oracle)
    gen = torch.Generator(cuda_device).manual_seed(3)
    order = torch.as_tensor(graph.host.l2g, device=cuda_device).long()
    dims = (24, 16, 9)
    x = torch.randn((n, dims[0]), device=cuda_device, generator=gen)
    truth = torch.randint(-1, dims[2], (n,), device=cuda_device, generator=gen, dtype=torch.int32)
    big = gcn.ResidualGCN(graph, x[order], truth[order], *parameters(cuda_device, gen, (dims[0], 48, dims[2]), 2))
    big.forward()
    values, classes = big.logits.topk(3, dim=1)
    classes[::5, 2], classes[7] = -1, -1
    weights, biases, norms = parameters(cuda_device, gen, dims, 1)
    model = gcn.ResidualGCN(graph, x[order], truth[order], weights, biases, norms, teacher=(values, classes), temperature=2.0, soft=0.5, hard=0.25)
    loss = model.forward()
    grads = model.backward()
    back = torch.argsort(order)
    _, want, want_grads = step_in_double(adjacency, x, weights, biases, norms, taught(truth, values[back], classes[back], 2.0, 0.5, 0.25))
    assert abs(loss.item() - want.item()) < TOL * want.item()
    for got, expected in zip(grads, want_grads):
        assert rel(got, expected) < TOL


def test_two_parts_on_one_device(cuda_device, oracle):
    """Two parts of a partition, their aggregations summed over the replicas on one device: the gradients of both parts add up to those of the whole, every
    replicated vertex counted once in weights, biases and norms."""
    n, adjacency, graphs = graph_of(cuda_device, oracle, parts=2)
    gen = torch.Generator(cuda_device).manual_seed(5)
    dims, layers = (24, 32, 7), 2
    x = torch.randn((n, dims[0]), device=cuda_device, generator=gen)
    truth = torch.randint(-1, dims[2], (n,), device=cuda_device, generator=gen, dtype=torch.int32)
    weights, biases, norms = parameters(cuda_device, gen, dims, layers)
    orders = [torch.as_tensor(g.host.l2g, device=cuda_device).long() for g in graphs]
    # The parts run in turn, so that each step's exchange has the other part's rows from an earlier run: after as many runs as there are exchanges all
    # of them are right.
    rows, at = [{}, {}], [0, 0]

    def sync_of(p):
        def sync(own):
            step, at[p] = at[p], at[p] + 1
            rows[p][step] = own.clone()
            other = rows[1 - p].get(step, torch.zeros_like(own[:1]).expand(len(orders[1 - p]), own.shape[1]))
            total = torch.zeros((n, own.shape[1]), device=own.device).index_add_(0, orders[p], own).index_add_(0, orders[1 - p], other)
            own.copy_(total[orders[p]])
        return sync
    models = []
    for p, g in enumerate(graphs):
        aggregate = lambda op, src, out, plan=g.plan: plan.spmm(op, src, out=out)
        model = gcn.ResidualGCN(g, x[orders[p]], truth[orders[p]], weights, biases, norms, worker_num=2, aggregate=aggregate, sync=sync_of(p))
        models.append(model)
    assert sum(int((m.mirror2worker != -1).sum()) for m in models) > 0
    for _ in range(2 * layers + 1):
        for p, m in enumerate(models):
            at[p] = 0
            m.forward()
            m.backward()
    owned = [(m.mirror2worker == -1) for m in models]
    # the loss's gradient counts a row wherever it is; weights, biases and norms where its master is
    logits, _, want = step_in_double(adjacency, x, weights, biases, norms, cross_entropy(truth))
    for m, order, own in zip(models, orders, owned):
        assert rel(m.logits, logits[order]) < TOL
    for a, b, expected in zip(models[0].gradients(), models[1].gradients(), want):
        assert rel(a + b, expected) < TOL


def test_captured_step(cuda_device, oracle):
    """A step captured into a graph and replayed on other inputs, beside a second graph of the same model: the bits of the eager step."""
    n, _, (graph,) = graph_of(cuda_device, oracle)
    gen = torch.Generator(cuda_device).manual_seed(7)
    dims = (40, 32, 7)
    x = torch.randn((n, dims[0]), device=cuda_device, generator=gen)
    truth = torch.randint(-1, dims[2], (n,), device=cuda_device, generator=gen, dtype=torch.int32)
    model = gcn.ResidualGCN(graph, x, truth, *parameters(cuda_device, gen, dims, 2))
    other = torch.randn((n, dims[0]), device=cuda_device, generator=gen)

    def eager(rows):
        model.x.copy_(rows)
        return [model.forward().clone(), *(g.clone() for g in model.backward())]
    wanted = [eager(rows) for rows in (x.clone(), other)]
    first = x.clone()
    captured = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outputs = [model.forward(), *model.backward()]
        captured.append((g, outputs))
    for (g, outputs), (h, more) in (captured, captured[::-1]):
        for rows in (first, other):
            model.x.copy_(rows)
            g.replay()
            h.replay()
            torch.cuda.synchronize()
            model.x.copy_(rows)
            want = eager(rows)
            assert all(torch.equal(a, b) for a, b in zip(outputs, want)) and all(torch.equal(a, b) for a, b in zip(more, want))
    assert all(torch.isfinite(w[0]) for w in wanted)


def test_models_that_are_none(cuda_device):
    x, truth = torch.zeros((4, 3), device=cuda_device), torch.zeros(4, dtype=torch.int32, device=cuda_device)
    w = [torch.zeros((3, 5), device=cuda_device), torch.zeros((5, 2), device=cuda_device)]
    b = [torch.zeros(5, device=cuda_device), torch.zeros(2, device=cuda_device)]
    norm = (torch.ones(5, device=cuda_device), torch.zeros(5, device=cuda_device))
    with pytest.raises(ValueError, match="no model"):
        gcn.ResidualGCN(None, x, truth, w, b, [], aggregate=lambda *a: None)
    with pytest.raises(ValueError, match="no model"):
        gcn.ResidualGCN(None, x, truth, w, b[:1], [norm], aggregate=lambda *a: None)
    with pytest.raises(ValueError, match="float32"):
        gcn.ResidualGCN(None, x.half(), truth, w, b, [norm], aggregate=lambda *a: None)
    with pytest.raises(ValueError, match="label"):
        gcn.ResidualGCN(None, x, truth + 2, w, b, [norm], aggregate=lambda *a: None)
