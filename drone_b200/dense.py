"""Dense operators beside the aggregation, over the C ABI: product with bias, activation and residual, layer norm, the loss against a
teacher's top logits, and their backward passes.  What a layer of a residual graph network or a model taught by one does to the
vertices' rows between its aggregations; gcn.ResidualGCN is made of them.

The rows of a call are a CUDA matrix of float32, bfloat16 or float16 whose rows lie one after the other (any distance apart); weights
have the rows' type, bias, scale, shift and their gradients are float32.  Gradients are returned, no autograd graph is recorded.  Calls run on the
current stream of the rows' device and may be captured; nothing is kept from one call to the next.  ValueError says what does not fit.
"""
import ctypes as C

import torch

from ._lib import (ACT_GELU, ACT_NONE, ACT_RELU, ACT_SILU, BF16, DISTILLATION_MAX_TOP, DISTILLATION_SCRATCH, F16, F32, NORM_MAX_WIDTH, check,
                   lib)

_TYPES = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}
_ACTIVATIONS = {None: ACT_NONE, "none": ACT_NONE, "relu": ACT_RELU, "gelu": ACT_GELU, "silu": ACT_SILU}
_MAX_WIDTH, _MAX_ROWS = 1 << 15, 1 << 30


def _require(condition, message, *values):
    if not condition:
        raise ValueError(message % values)


def _matrix(name, t, rows=None, width=None, dtype=None, device=None):
    """t's distance between rows, once it is a matrix that the kernels can read or write."""
    try:
        (n, f), (apart, step), its = t.shape, t.stride(), t.dtype
        if ((its in _TYPES if dtype is None else its is dtype) and (t.is_cuda if device is None else t.device == device)
                and (rows is None or n == rows) and (width is None or f == width) and f >= 1 and f <= (apart if n > 1 else f) < 1 << 31
                and (step == 1 or f == 1 or n == 0) and n <= _MAX_ROWS):
            return apart if n > 1 else f
    except (AttributeError, TypeError, ValueError):
        pass
    _refuse_matrix(name, t, rows, width, dtype, device)


def _refuse_matrix(name, t, rows, width, dtype, device):
    _require(isinstance(t, torch.Tensor) and t.dim() == 2, "%s is not a matrix", name)
    _require(t.is_cuda if device is None else t.device == device, "%s is on %s, not on %s", name, t.device, device or "a CUDA device")
    _require(t.dtype in _TYPES if dtype is None else t.dtype == dtype, "%s is of %s", name, t.dtype)
    _require((rows is None or t.shape[0] == rows) and (width is None or t.shape[1] == width), "%s is %d x %d where %s x %s are needed", name,
             *t.shape, "any" if rows is None else rows, "any" if width is None else width)
    raise ValueError("%s has %d rows of %d values, %d apart, with values %d apart" % (name, *t.shape, *t.stride()))


def _vector(name, t, size, dtype, device):
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == (size,) and t.device == device and t.is_contiguous()):
        raise ValueError("%s is not %d values of %s side by side on %s" % (name, size, dtype, device))


def _span(t):
    if t.numel() == 0:
        return 0, 0
    first = t.data_ptr()
    return first, first + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _apart(name, out, *others):
    """An output overlaps no operand but those that it may lie on exactly."""
    a, b = _span(out)
    for other, may_be_same in others:
        if other is None:
            continue
        c, d = _span(other)
        same = may_be_same and a == c and out.shape == other.shape and out.stride() == other.stride() and out.dtype == other.dtype
        _require(same or b <= c or d <= a, "%s overlaps another operand", name)


def _pointer(t):
    return None if t is None else t.data_ptr()


def _activation(name):
    if name not in _ACTIVATIONS:
        raise ValueError("activation %r is none of none, relu, gelu, silu" % (name,))
    return _ACTIVATIONS[name]


class _Call:
    """Library calls on a device and its current stream."""

    def __init__(self, device):
        self.device = device
        self.guard = None if torch._C._cuda_getDevice() == device.index else torch.cuda.device(device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        self.stream = torch._C._cuda_getCurrentRawStream(self.device.index)
        self.lib = lib()
        return self

    def __exit__(self, *error):
        if self.guard is not None:
            self.guard.__exit__(*error)

    def __call__(self, name, *args):
        code = getattr(self.lib, name)(*args, self.stream)
        if code:
            check(code)

    def scratch(self, name, *sizes):
        """Scratch for a call of these sizes and its number of floats."""
        floats = C.c_longlong(0)
        check(getattr(self.lib, name)(*sizes, C.byref(floats)))
        return (torch.empty(floats.value, dtype=torch.float32, device=self.device) if floats.value else None), floats.value


def _weights(w, inputs, dtype, device, transposed):
    """Distance between the weights' rows, their other width and whether they lie as [outputs, inputs].  The transposed view of a
    contiguous matrix is read as that matrix."""
    if not isinstance(w, torch.Tensor) or w.dim() != 2:
        raise ValueError("the weights are not a matrix")
    if w.stride(1) != 1 and w.stride(0) == 1:
        w, transposed = w.t(), not transposed
    ldw = _matrix("the weights", w, dtype=dtype, device=device)
    rows, columns = w.shape
    taken, outputs = (columns, rows) if transposed else (rows, columns)
    if taken != inputs:
        raise ValueError("the weights are for rows of %d, not of %d" % (taken, inputs))
    if rows > _MAX_WIDTH or columns > _MAX_WIDTH:
        raise ValueError("weights of %d x %d: at most %d each way" % (rows, columns, _MAX_WIDTH))
    return ldw, outputs, transposed


def linear(x, w, bias=None, activation=None, residual=None, transposed=False, out=None, pre=None):
    """activation(x . w + bias) + residual for rows x [n, inputs] and weights w [inputs, outputs], or [outputs, inputs] with
    `transposed`.  activation: None, "relu", "gelu" (exact) or "silu".  `out` may be the residual itself; `pre` receives the
    values before the activation, which the backward pass wants."""
    ldx = _matrix("x", x)
    n, dtype, device = x.shape[0], x.dtype, x.device
    ldw, outputs, flipped = _weights(w, x.shape[1], dtype, device, bool(transposed))
    if bias is not None:
        _vector("the bias", bias, outputs, torch.float32, device)
    act = _activation(activation)
    made = out is None
    if made:
        out = x.new_empty((n, outputs))
    ldy = outputs if made else _matrix("out", out, n, outputs, dtype, device)
    ldr = _matrix("the residual", residual, n, outputs, dtype, device) if residual is not None else 0
    ldp = _matrix("pre", pre, n, outputs, dtype, device) if pre is not None else 0
    if not made:
        _apart("out", out, (x, False), (w, False), (bias, False), (residual, True), (pre, False))
    if pre is not None:
        _apart("pre", pre, (x, False), (w, False), (bias, False), (residual, False))
    with _Call(device) as call:
        image, floats = call.scratch("drone_linear_scratch", _TYPES[dtype], n, x.shape[1], outputs, x.data_ptr(), ldx, w.data_ptr(), ldw, int(flipped))
        call("drone_linear", _TYPES[dtype], n, x.shape[1], outputs, x.data_ptr(), ldx, w.data_ptr(), ldw, int(flipped), _pointer(bias), act,
             _pointer(residual), ldr, out.data_ptr(), ldy, _pointer(pre), ldp, _pointer(image), floats)
    return out


def linear_backward(grad, x, w, pre=None, activation=None, transposed=False, bias=True, input_gradient=True):
    """Gradients of x, the weights and the bias from that of linear(x, w, ...).  pre: the values before the activation (for the ReLU
    its output will do where no residual was added); not needed without one.  The residual's gradient is `grad` itself.  Between the activation and
    the products the gradient is rounded to the rows' type.  None stands for what is not asked for (bias, input_gradient)."""
    ldx = _matrix("x", x)
    n, dtype, device = x.shape[0], x.dtype, x.device
    inputs = x.shape[1]
    ldw, outputs, flipped = _weights(w, inputs, dtype, device, bool(transposed))
    ldg = _matrix("grad", grad, n, outputs, dtype, device)
    act = _activation(activation)
    if act != ACT_NONE:
        _require(pre is not None, "the backward pass of %s needs the values before it", activation)
        ldp = _matrix("pre", pre, n, outputs, dtype, device)
    kind = _TYPES[dtype]
    grad_w = torch.empty(w.shape, dtype=dtype, device=device)
    grad_x = torch.empty((n, inputs), dtype=dtype, device=device) if input_gradient else None
    grad_b = torch.empty(outputs, dtype=torch.float32, device=device) if bias else None
    with _Call(device) as call:
        dz, ldz = grad, ldg
        # 16-bit rows that are not on 16 bytes are copied to rows that are here, once for both products
        own = act != ACT_NONE or (dtype != torch.float32 and (ldg % 8 != 0 or grad.data_ptr() % 16 != 0))
        if own:
            ldz = outputs if dtype == torch.float32 else (outputs + 7) // 8 * 8      # rows on 16 bytes, as the products want them
            dz = torch.empty((n, ldz), dtype=dtype, device=device)
        if own or bias:
            size = call.scratch("drone_activation_gradient_scratch", kind, n, outputs) if bias else (None, 0)
            call("drone_activation_gradient", kind, n, outputs, grad.data_ptr(), ldg, _pointer(pre) if act != ACT_NONE else None,
                 ldp if act != ACT_NONE else 0, act, dz.data_ptr() if own else None, ldz, _pointer(grad_b), _pointer(size[0]), size[1])
        if input_gradient:
            size = call.scratch("drone_linear_scratch", kind, n, outputs, inputs, dz.data_ptr(), ldz, w.data_ptr(), ldw, int(not flipped))
            call("drone_linear", kind, n, outputs, inputs, dz.data_ptr(), ldz, w.data_ptr(), ldw, int(not flipped), None, ACT_NONE, None, 0,
                 grad_x.data_ptr(), inputs, None, 0, _pointer(size[0]), size[1])
        # in the weights' own order
        size = call.scratch("drone_linear_weight_gradient_scratch", kind, n, inputs, outputs, x.data_ptr(), ldx, dz.data_ptr(), ldz,
                            int(bool(transposed)))
        call("drone_linear_weight_gradient", kind, n, inputs, outputs, x.data_ptr(), ldx, dz.data_ptr(), ldz, int(bool(transposed)),
             grad_w.data_ptr(), grad_w.shape[1], _pointer(size[0]), size[1])
    return grad_x, grad_w, grad_b


def layer_norm(x, scale, shift, eps=1e-5, relu=False, out=None):
    """(y, mean, rstd) with y = (x - mean) * rstd * scale + shift over each row, rstd = 1 / sqrt(variance + eps), and max(y, 0) with
    `relu`.  `out` may be x."""
    ldx = _matrix("x", x)
    n, f, device = x.shape[0], x.shape[1], x.device
    _require(f <= NORM_MAX_WIDTH, "rows of %d: at most %d", f, NORM_MAX_WIDTH)
    _vector("scale", scale, f, torch.float32, device)
    _vector("shift", shift, f, torch.float32, device)
    _require(eps > 0, "eps=%r", eps)
    if out is None:
        out, ldy = x.new_empty((n, f)), f
    else:
        ldy = _matrix("out", out, n, f, x.dtype, device)
        _apart("out", out, (x, True), (scale, False), (shift, False))
    mean, rstd = scale.new_empty(n), scale.new_empty(n)
    with _Call(device) as call:
        call("drone_layer_norm", _TYPES[x.dtype], n, f, x.data_ptr(), ldx, scale.data_ptr(), shift.data_ptr(), float(eps), int(bool(relu)),
             out.data_ptr(), ldy, mean.data_ptr(), rstd.data_ptr())
    return out, mean, rstd


def layer_norm_backward(grad, x, scale, mean, rstd, out=None, mirror_rows=None):
    """Gradients of x, scale and shift from that of layer_norm(x, ...)[0].  out: what layer_norm returned, where it had a ReLU.
    mirror_rows: Mirror2Worker of a part of a graph; rows with an entry other than -1 are left out of the sums over rows."""
    ldx = _matrix("x", x)
    n, f, dtype, device = x.shape[0], x.shape[1], x.dtype, x.device
    _require(f <= NORM_MAX_WIDTH, "rows of %d: at most %d", f, NORM_MAX_WIDTH)
    ldg = _matrix("grad", grad, n, f, dtype, device)
    ldo = _matrix("out", out, n, f, dtype, device) if out is not None else 0
    _vector("scale", scale, f, torch.float32, device)
    _vector("mean", mean, n, torch.float32, device)
    _vector("rstd", rstd, n, torch.float32, device)
    if mirror_rows is not None:
        _vector("mirror_rows", mirror_rows, n, torch.int32, device)
    grad_x = x.new_empty((n, f))
    grad_scale, grad_shift = scale.new_empty(f), scale.new_empty(f)
    with _Call(device) as call:
        sums, floats = call.scratch("drone_layer_norm_backward_scratch", _TYPES[dtype], n, f)
        call("drone_layer_norm_backward", _TYPES[dtype], n, f, grad.data_ptr(), ldg, x.data_ptr(), ldx, scale.data_ptr(), mean.data_ptr(),
             rstd.data_ptr(), _pointer(out), ldo, _pointer(mirror_rows), grad_x.data_ptr(), f, grad_scale.data_ptr(), grad_shift.data_ptr(),
             _pointer(sums), floats)
    return grad_x, grad_scale, grad_shift


def distillation_loss(logits, teacher, classes, temperature=1.0, truth=None, labelled=None, soft=1.0, hard=0.0):
    """(loss, gradient) of logits [n, classes] against a teacher's top logits: values `teacher` [n, top] of the classes `classes`
    [n, top] (int64; negative: no entry).  loss[0]: mean over the rows with an entry of temperature^2 * KL(teacher || model) over the
    entries; loss[1]: mean cross-entropy over the labelled rows (truth int64, labelled bool; where a row is
    not labelled its truth may be anything, such as -1).  The gradient is soft times that of the first sum over rows plus hard times that of the
    second, not divided by the numbers of rows, as the graph model's own loss has it."""
    ld = _matrix("logits", logits)
    n, c, device = logits.shape[0], logits.shape[1], logits.device
    ldt = _matrix("teacher", teacher, n, device=device)
    top = teacher.shape[1]
    _require(top <= DISTILLATION_MAX_TOP, "%d entries of the teacher: at most %d", top, DISTILLATION_MAX_TOP)
    ldc = _matrix("classes", classes, n, top, torch.int64, device)
    _require(1e-6 <= temperature <= 1e6, "temperature=%r", temperature)
    _require((truth is None) == (labelled is None), "truth and labelled come together")
    if truth is not None:
        _vector("truth", truth, n, torch.int64, device)
        _vector("labelled", labelled, n, torch.bool, device)
    loss, grad = torch.empty(2, dtype=torch.float32, device=device), torch.empty((n, c), dtype=logits.dtype, device=device)
    with _Call(device) as call:
        scratch = torch.empty(DISTILLATION_SCRATCH, dtype=torch.float64, device=device)
        call("drone_distillation_loss", _TYPES[logits.dtype], n, c, logits.data_ptr(), ld, _TYPES[teacher.dtype], top, teacher.data_ptr(), ldt,
             classes.data_ptr(), ldc, float(temperature), _pointer(truth), _pointer(labelled), float(soft), float(hard), grad.data_ptr(), c,
             loss.data_ptr(), scratch.data_ptr())
    return loss, grad
