"""Edges of the dense operators: infinities through the activations, tails, logits with an offset, values at the ends of their type, rows that count for nothing, sums over very
many rows."""
import math

import pytest
import torch

from drone_b200 import dense
from test_dense_gpu import TYPES, activated, rows_of

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
