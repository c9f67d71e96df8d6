"""What the dense operators refuse, before anything reaches a device: the C ABI by its codes and messages, the Python calls by ValueError."""
import ctypes as C

import pytest
import torch

from drone_b200 import _lib, dense

P = 1 << 12      # an address that is never read: every call here is refused


def refused(name, *args):
    rc = getattr(_lib.lib(), name)(*args)
    assert rc == -1, (name, args, rc)
    return _lib.lib().drone_last_error().decode()


def linear_args(**change):
    a = dict(type=0, rows=5000, K=60, N=70, X=P, ldx=60, W=P, ldw=70, transposed=0, bias=None, act=0, R=None, ldr=0, Y=P, ldy=70, pre=None, ldp=0, scratch=P, floats=1 << 24, stream=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change", [
    dict(type=3), dict(type=-1), dict(rows=-1), dict(rows=(1 << 30) + 1), dict(K=0), dict(K=(1 << 15) + 1, ldx=1 << 16), dict(N=0), dict(N=-3), dict(ldx=59), dict(ldw=69),
    dict(transposed=1, ldw=59), dict(transposed=2), dict(act=4), dict(act=-1), dict(R=P, ldr=69), dict(ldy=69), dict(pre=P, ldp=69), dict(X=None), dict(W=None),
    dict(Y=None), dict(X=P + 2), dict(type=1, Y=P + 1), dict(R=P + 1, ldr=70), dict(type=2, pre=P + 1, ldp=70), dict(scratch=None), dict(scratch=P + 4), dict(floats=16), dict(bias=P + 2)])
def test_linear_refuses(change):
    assert "drone_linear" in refused("drone_linear", *linear_args(**change))


def test_linear_without_rows_is_nothing():
    assert _lib.lib().drone_linear(*linear_args(rows=0, X=None, Y=None)) == 0


@pytest.mark.parametrize("change", [dict(type=5), dict(rows=-1), dict(N=0), dict(act=7), dict(ldg=3), dict(act=1, ldp=3), dict(ldz=3), dict(G=None),
                                    dict(act=1, pre=None), dict(G=P + 1), dict(Z=P + 2)])
def test_activation_gradient_refuses(change):
    a = dict(type=0, rows=5, N=7, G=P, ldg=7, pre=P, ldp=7, act=0, Z=P, ldz=7, bias=None, scratch=None, floats=0, stream=None)
    a.update(change)
    assert "drone_activation_gradient" in refused("drone_activation_gradient", *a.values())


@pytest.mark.parametrize("change", [dict(type=5), dict(rows=-1), dict(K=0), dict(N=1 << 16, ldz=1 << 16), dict(ldx=5), dict(ldz=6), dict(ldw=6), dict(transposed=1, ldw=5),
                                    dict(transposed=3), dict(X=None), dict(Z=None), dict(W=None), dict(W=P + 2)])
def test_weight_gradient_refuses(change):
    a = dict(type=0, rows=5, K=6, N=7, X=P, ldx=6, Z=P, ldz=7, transposed=0, W=P, ldw=7, scratch=P, floats=1 << 20, stream=None)
    a.update(change)
    assert "drone_linear_weight_gradient" in refused("drone_linear_weight_gradient", *a.values())


@pytest.mark.parametrize("change", [dict(type=4), dict(rows=-1), dict(F=0), dict(F=65537, ldx=1 << 17, ldy=1 << 17), dict(ldx=6), dict(ldy=6), dict(eps=0.0), dict(eps=-1.0),
                                    dict(eps=float("nan")), dict(relu=2), dict(X=None), dict(scale=None), dict(shift=None), dict(Y=None), dict(X=P + 1)])
def test_layer_norm_refuses(change):
    a = dict(type=0, rows=5, F=7, X=P, ldx=7, scale=P, shift=P, eps=1e-5, relu=0, Y=P, ldy=7, mean=None, rstd=None, stream=None)
    a.update(change)
    assert "drone_layer_norm" in refused("drone_layer_norm", *a.values())


@pytest.mark.parametrize("change", [dict(type=4), dict(rows=-1), dict(F=0), dict(F=65537), dict(ldg=6), dict(ldx=6), dict(out=P, ldo=6), dict(ld=6), dict(G=None),
                                    dict(X=None), dict(scale=None), dict(mean=None), dict(rstd=None), dict(dX=None), dict(out=P + 2), dict(G=P + 3)])
def test_layer_norm_backward_refuses(change):
    a = dict(type=0, rows=5, F=7, G=P, ldg=7, X=P, ldx=7, scale=P, mean=P, rstd=P, out=None, ldo=0, mirrors=None, dX=P, ld=7, ds=None, dt=None, scratch=P,
             floats=1 << 24, stream=None)
    a.update(change)
    assert "drone_layer_norm_backward" in refused("drone_layer_norm_backward", *a.values())


@pytest.mark.parametrize("change", [dict(type=3), dict(teacher_type=-2), dict(rows=-1), dict(classes=0), dict(ld=6), dict(top=0), dict(top=257, ldt=300, ldc=300), dict(ldt=2),
                                    dict(ldc=2), dict(t=0.0), dict(t=-1.0), dict(t=float("nan")), dict(t=float("inf")), dict(truth=P), dict(labelled=P), dict(ldg=6),
                                    dict(logits=None), dict(teacher=None), dict(ids=None), dict(grad=None), dict(loss=None), dict(scratch=None), dict(scratch=P + 4),
                                    dict(grad=P + 1), dict(teacher=P + 2)])
def test_distillation_refuses(change):
    a = dict(type=0, rows=5, classes=7, logits=P, ld=7, teacher_type=0, top=3, teacher=P, ldt=3, ids=P, ldc=3, t=1.0, truth=None, labelled=None, soft=1.0, hard=0.0,
             grad=P, ldg=7, loss=P, scratch=P, stream=None)
    a.update(change)
    assert "drone_distillation_loss" in refused("drone_distillation_loss", *a.values())


def test_scratch_sizes_refuse():
    size = C.c_longlong(0)
    for name, args in (("drone_linear_scratch", (3, 5, 4, 4, P, 4, P, 4, 0)), ("drone_linear_scratch", (0, -1, 4, 4, P, 4, P, 4, 0)),
                       ("drone_linear_scratch", (0, 5, 0, 4, P, 4, P, 4, 0)), ("drone_linear_scratch", (0, 5, 4, 4, P, 4, P, 4, 3)), 
                       ("drone_activation_gradient_scratch", (0, -1, 4)), ("drone_activation_gradient_scratch", (0, 5, 0)), ("drone_activation_gradient_scratch", (1, (1 << 30) + 1, 4)),
                       ("drone_activation_gradient_scratch", (7, 5, 4)),
                       ("drone_linear_weight_gradient_scratch", (0, -1, 4, 4, P, 4, P, 4, 0)), ("drone_linear_weight_gradient_scratch", (9, 5, 4, 4, P, 4, P, 4, 0)),
                       ("drone_linear_weight_gradient_scratch", (0, 5, 4, 4, P, 4, P, 4, 2)), ("drone_layer_norm_backward_scratch", (0, -1, 4)),
                       ("drone_layer_norm_backward_scratch", (0, 5, 65537)), ("drone_layer_norm_backward_scratch", (3, 5, 4))):
        assert name in refused(name, *args, C.byref(size))


def test_operands_on_the_host_are_refused():
    x, w, v = torch.zeros(5, 6), torch.zeros(6, 7), torch.zeros(6)
    for call in (lambda: dense.linear(x, w), lambda: dense.linear_backward(torch.zeros(5, 7), x, w), lambda: dense.layer_norm(x, v, v),
                 lambda: dense.layer_norm_backward(x, x, v, torch.zeros(5), torch.zeros(5)),
                 lambda: dense.distillation_loss(x, torch.zeros(5, 2), torch.zeros(5, 2, dtype=torch.int64))):
        with pytest.raises(ValueError, match="CUDA device"):
            call()
    for wrong in (None, torch.zeros(3), torch.zeros(2, 2, 2), [[1.0]]):
        with pytest.raises(ValueError, match="not a matrix"):
            dense.layer_norm(wrong, v, v)


def test_constants_are_the_headers():
    import os
    import re
    text = open(os.path.join(os.path.dirname(_lib.PKG), "include", "drone_b200.h")).read()
    defined = {name: int(value) for name, value in re.findall(r"#define DRONE_(\w+)\s+(-?\d+)\b", text)}
    for name in ("F32", "BF16", "F16", "ACT_NONE", "ACT_RELU", "ACT_GELU", "ACT_SILU", "NORM_MAX_WIDTH", "DISTILLATION_MAX_TOP", "DISTILLATION_SCRATCH"):
        assert getattr(_lib, name) == defined[name], name


def test_widths_beyond_an_int_are_refused():
    """A single row may be as long as memory is; the C ABI takes its length as an int, which 2^32 + 7 would reach as 7."""
    for f in ((1 << 31) - 1, 1 << 31, (1 << 32) + 7):
        row = torch.empty((1, f), dtype=torch.bfloat16, device="meta")
        if f < 1 << 31:
            assert dense._matrix("x", row, device=row.device) == f
        else:
            with pytest.raises(ValueError, match="x has 1 rows of %d" % f):
                dense._matrix("x", row, device=row.device)
