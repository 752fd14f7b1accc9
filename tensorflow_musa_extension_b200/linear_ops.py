"""Op front end of the matrix products with bias, activation and residual in
their epilogue: MusaMatMulBiasAct, its gradient, and the 8-bit form.

The reference fuses these chains into MusaLinearActivation and
MusaMatMulBiasAdd, a library matmul followed by separate passes
(musa_ext/graph/fusion/linear_activation_fusion.cc:68-263,
musa_ext/graph/fusion/matmul_biasadd_fusion.cc:153-347,
musa_ext/kernels/fusion/musa_linear_relu_op.cc:30-217); here one kernel does
the product and what follows it."""
import collections

import torch

from .errors import InternalError, InvalidArgumentError
from . import raw_ops as _r

_DTYPES = (torch.float16, torch.bfloat16)
ACTIVATIONS = {"Identity": _r.ACT_IDENTITY, "Relu": _r.ACT_RELU, "Sigmoid": _r.ACT_SIGMOID,
               "Silu": _r.ACT_SILU, "Gelu": _r.ACT_GELU}

MusaMatMulBiasActOutput = collections.namedtuple("MusaMatMulBiasAct", ["y", "preactivation"])
MusaMatMulBiasActGradOutput = collections.namedtuple(
    "MusaMatMulBiasActGrad", ["da", "db", "dbias"])


def _activation(opname, activation):
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise InvalidArgumentError(
            "%s: activation must be one of %s, got %r"
            % (opname, ", ".join(sorted(ACTIVATIONS)), activation))
    return act


def _same(opname, name, t, like, dtype):
    if t is None:
        return
    if t.dtype != dtype:
        raise InvalidArgumentError(
            "%s: %s dtype %s does not match %s" % (opname, name, t.dtype, dtype))
    if t.device != like.device:
        raise InvalidArgumentError(
            "%s: %s is on %s, not on %s" % (opname, name, t.device, like.device))


def _factor(t):
    """(tensor, line stride, transposed) of a 2-D tensor: taken as it lies where
    either axis is contiguous, copied otherwise."""
    rows, cols = t.shape
    for transposed in (False, True):
        lines, length = (cols, rows) if transposed else (rows, cols)
        line, step = (t.stride(1), t.stride(0)) if transposed else (t.stride(0), t.stride(1))
        if (step == 1 or length <= 1) and (lines <= 1 or line >= length):
            return t, line if lines > 1 else length, transposed
    t = t.contiguous()
    return t, cols, False


def _operands(opname, a, b, transpose_a, transpose_b):
    """2-D views of the factors, the leading shape of the product, m, n, k."""
    if a.dim() < 2 or b.dim() != 2:
        raise InvalidArgumentError(
            "%s: a must be at least 2D and b 2D: %s, %s" % (opname, tuple(a.shape),
                                                            tuple(b.shape)))
    if transpose_a and a.dim() != 2:
        raise InvalidArgumentError("%s: transpose_a needs a 2D a: %s" % (opname, tuple(a.shape)))
    if b.dtype != a.dtype or b.device != a.device:
        raise InvalidArgumentError(
            "%s: b (%s on %s) does not match a (%s on %s)"
            % (opname, b.dtype, b.device, a.dtype, a.device))
    if transpose_a:
        lead, (k, m), a2 = (a.shape[1],), a.shape, a
    else:
        lead, k = tuple(a.shape[:-1]), a.shape[-1]
        m = 1
        for d in lead:
            m *= d
        a2 = a if a.dim() == 2 else a.reshape(m, k)
    n, kb = b.shape if transpose_b else (b.shape[1], b.shape[0])
    if k != kb:
        raise InvalidArgumentError(
            "%s: matrix size-incompatible: a %s, b %s" % (opname, tuple(a.shape),
                                                          tuple(b.shape)))
    return a2, lead, m, n, k


def _epilogue(opname, like, bias, residual, shape, dtype):
    n = shape[-1]
    _same(opname, "bias", bias, like, dtype)
    _same(opname, "residual", residual, like, dtype)
    if bias is not None and tuple(bias.shape) != (n,):
        raise InvalidArgumentError(
            "%s: bias must have the shape (%d,), got %s" % (opname, n, tuple(bias.shape)))
    if residual is not None and tuple(residual.shape) != tuple(shape):
        raise InvalidArgumentError(
            "%s: residual must have the shape %s, got %s"
            % (opname, tuple(shape), tuple(residual.shape)))
    return (None if bias is None else bias.contiguous(),
            None if residual is None else residual.contiguous())


def MusaMatMulBiasAct(a, b, bias=None, residual=None, activation="Identity", transpose_a=False,
                      transpose_b=False, return_preactivation=False, name=None):
    """y = act(op(a) op(b) + bias) + residual for T in {half, bfloat16}.

    a: [..., k] (or [k, m] with transpose_a), b: [k, n] (or [n, k] with
    transpose_b), bias [n], residual of y's shape [..., n]; bias and residual may be
    None.  activation: "Identity", "Relu", "Sigmoid", "Silu" (z * sigmoid(z); not
    MusaBiasAddSwish, whose factor is the input before the bias) or "Gelu" (z *
    Phi(z), good to 8e-7 of |z|; of the value, which is small there, to 0.4 % at
    z = -6 and 1 % at -8).  The product and what follows are fp32, y is rounded
    once.  With return_preactivation returns (y, preactivation): z = op(a) op(b) + bias rounded
    to T, which MusaMatMulBiasActGrad takes.  The order of the sums is fixed by the
    sizes; float is not taken: the tensor cores would keep 11 of its 24 bits."""
    what = "MusaMatMulBiasAct"
    act = _activation(what, activation)
    out = _r._native().matmul_bias_act(a, b, bias, residual, act, transpose_a, transpose_b,
                                       return_preactivation)
    if out is not None:
        return _r._native_result(
            out, MusaMatMulBiasActOutput if return_preactivation else None, what)
    _r._require_cuda()
    hf = _r._HostForm()
    ad, bd, bias, residual = (hf.to_device(t) for t in (a, b, bias, residual))
    if ad.dtype not in _DTYPES:
        raise InvalidArgumentError("%s: unsupported dtype %s" % (what, ad.dtype))
    a2, lead, m, n, k = _operands(what, ad, bd, transpose_a, transpose_b)
    bias, residual = _epilogue(what, ad, bias, residual, lead + (n,), ad.dtype)
    with torch.cuda.device(ad.device):
        y = torch.empty(lead + (n,), dtype=ad.dtype, device=ad.device)
        z = torch.empty_like(y) if return_preactivation else None
        lib = _r._lib()
        fa, lda, ta = _factor(a2)
        fb, ldb, tb = _factor(bd)
        factors = (_r._ptr(fa), lda, ta != bool(transpose_a), _r._ptr(fb), ldb,
                   tb != bool(transpose_b))
        ws = _r._scratch(lib.MatMulWorkspaceBytes(2, *factors, m, n, k), ad.device)
        rc = lib.LaunchMatMulBiasAct(
            _r._DT_CODE[ad.dtype], *factors, _r._ptr(bias), _r._ptr(residual), _r._ptr(y),
            _r._ptr(z), m, n, k, act, _r._ptr(ws), ws.numel(), _r._stream())
        _r._check(rc, what)
    if return_preactivation:
        return MusaMatMulBiasActOutput(*hf.back_many([y, z]))
    return hf.back(y)


def MusaMatMulBiasActGrad(dy, a, b, preactivation=None, activation="Identity",
                          transpose_a=False, transpose_b=False, name=None):
    """The gradient of MusaMatMulBiasAct: returns (da, db, dbias), shaped like a, b
    and [n].  `preactivation` is the z that the forward returned (None with
    "Identity"); Relu has the slope 0 at 0.  dz = dy * act'(z) is rounded to T for
    the two products, dbias sums the unrounded dz in a fixed order.  The gradient of
    the residual is dy itself."""
    what = "MusaMatMulBiasActGrad"
    act = _activation(what, activation)
    out = _r._native().matmul_bias_act_grad(dy, a, b, preactivation, act, transpose_a,
                                            transpose_b)
    if out is not None:
        return _r._native_result(out, MusaMatMulBiasActGradOutput, what)
    _r._require_cuda()
    hf = _r._HostForm()
    d, ad, bd, z = (hf.to_device(t) for t in (dy, a, b, preactivation))
    if ad.dtype not in _DTYPES:
        raise InvalidArgumentError("%s: unsupported dtype %s" % (what, ad.dtype))
    a2, lead, m, n, k = _operands(what, ad, bd, transpose_a, transpose_b)
    _same(what, "dy", d, ad, ad.dtype)
    _same(what, "preactivation", z, ad, ad.dtype)
    if z is None and act != _r.ACT_IDENTITY:
        raise InvalidArgumentError("%s: %s needs the preactivation" % (what, activation))
    for label, t in (("dy", d), ("preactivation", z)):
        if t is not None and tuple(t.shape) != lead + (n,):
            raise InvalidArgumentError(
                "%s: %s must have the shape %s, got %s"
                % (what, label, lead + (n,), tuple(t.shape)))
    d = d.contiguous()
    z = None if z is None else z.contiguous()
    with torch.cuda.device(ad.device):
        da = torch.empty(ad.shape, dtype=ad.dtype, device=ad.device)
        db = torch.empty(bd.shape, dtype=bd.dtype, device=bd.device)
        dbias = torch.empty((n,), dtype=ad.dtype, device=ad.device)
        lib = _r._lib()
        # The gradients have the layout of a and b as they are given: [k, m] where
        # transposed; a factor that lies the other way round is copied.
        fa, fb = a2.contiguous(), bd.contiguous()
        factors = (_r._ptr(fa), a2.shape[1], bool(transpose_a), _r._ptr(fb), bd.shape[1],
                   bool(transpose_b))
        ws = _r._scratch(lib.MatMulGradWorkspaceBytes(_r._ptr(d), *factors, _r._ptr(z), m, n, k,
                                                      act), ad.device)
        rc = lib.LaunchMatMulBiasActGrad(
            _r._DT_CODE[ad.dtype], _r._ptr(d), *factors, _r._ptr(z), _r._ptr(da), _r._ptr(db),
            _r._ptr(dbias), m, n, k, act, _r._ptr(ws), ws.numel(), _r._stream())
        _r._check(rc, what)
    return MusaMatMulBiasActGradOutput(*hf.back_many([da, db, dbias]))


def MusaQuantizedMatMulBiasAct(a, a_scale, b, b_scale, bias=None, residual=None,
                               activation="Identity", out_dtype=torch.bfloat16, name=None):
    """y = act((a * a_scale) (b * b_scale)^T + bias) + residual for float8_e4m3fn a
    [..., k] and b [n, k] with fp32 scales, one per row of each (MusaQuantizeRows,
    MusaAddRmsNormQuantize), which the product takes one after the other; bias [n], residual [..., n] and y are of out_dtype,
    half or bfloat16.  Device tensors only."""
    what = "MusaQuantizedMatMulBiasAct"
    act = _activation(what, activation)
    out = _r._native().quantized_matmul_bias_act(a, a_scale, b, b_scale, bias, residual, act,
                                                 _r._DT_CODE.get(out_dtype, -1))
    if out is not None:
        return _r._native_result(out, None, what)
    _r._require_cuda()
    if out_dtype not in _DTYPES:
        raise InvalidArgumentError("%s: unsupported out_dtype %s" % (what, out_dtype))
    for label, t in (("a", a), ("a_scale", a_scale), ("b", b), ("b_scale", b_scale)):
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise InvalidArgumentError("%s: %s must be a device tensor" % (what, label))
    if a.dtype != torch.float8_e4m3fn:
        raise InvalidArgumentError("%s: unsupported dtype %s" % (what, a.dtype))
    a2, lead, m, n, k = _operands(what, a, b, False, True)
    _same(what, "a_scale", a_scale, a, torch.float32)
    _same(what, "b_scale", b_scale, a, torch.float32)
    if a_scale.numel() != m or b_scale.numel() != n:
        raise InvalidArgumentError(
            "%s: one scale per row is needed: %d and %d, got %d and %d"
            % (what, m, n, a_scale.numel(), b_scale.numel()))
    bias, residual = _epilogue(what, a, bias, residual, lead + (n,), out_dtype)
    with torch.cuda.device(a.device):
        y = torch.empty(lead + (n,), dtype=out_dtype, device=a.device)
        lib = _r._lib()
        fa, lda, ta = _factor(a2)
        fb, ldb, tb = _factor(b)
        if ta:                     # the 8-bit products read both factors along k
            fa, lda = a2.contiguous(), k
        if tb:
            fb, ldb = b.contiguous(), k
        # Copies are held until the launch: the block of one that is gone is the next one's.
        sa, sb = a_scale.contiguous(), b_scale.contiguous()
        ws = _r._scratch(lib.MatMulWorkspaceBytes(1, _r._ptr(fa), lda, False, _r._ptr(fb), ldb,
                                                  True, m, n, k), a.device)
        rc = lib.LaunchQuantizedMatMulBiasAct(
            _r._DT_CODE[out_dtype], _r._ptr(fa), lda, _r._ptr(sa), _r._ptr(fb), ldb, _r._ptr(sb),
            _r._ptr(bias), _r._ptr(residual), _r._ptr(y), m, n, k, act, _r._ptr(ws), ws.numel(),
            _r._stream())
        _r._check(rc, what)
    return y


def check_products():
    """Raises InternalError if a product's kernel on the current device has given up a
    wait since the library was loaded (its outputs are then not valid; the kernels'
    waits end after about two seconds).  Synchronises with the device: not to be called while
    a stream is captured."""
    rc = _r._lib().MusaMatMulStatus()
    if rc != 0:
        raise InternalError("matrix products: %s" % _r._capi.ERROR_NAMES.get(rc, rc))
