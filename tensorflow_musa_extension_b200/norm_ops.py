"""Op front end of the row normalisations: MusaLayerNorm, MusaLayerNormGrad,
MusaRmsNorm, MusaRmsNormGradDx.  Same names, argument meaning, checks and error
text as the reference ops; one launch each through the C ABI.

New here, beyond the reference's ops: the residual's addition with the RMS norm
behind it (MusaAddRmsNorm, MusaAddRmsNormGrad) and the same forward with an
8-bit output (MusaAddRmsNormQuantize, MusaQuantizeRows), which the 8-bit
product of linear_ops takes."""
import collections

import torch

from .errors import InvalidArgumentError
from . import raw_ops as _r

_LN_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
_RMS_DTYPES = (torch.float32, torch.bfloat16)
_SCALE_MIN = 2.0 ** -126

MusaLayerNormGradOutput = collections.namedtuple(
    "MusaLayerNormGrad", ["dx", "dgamma", "dbeta"])
MusaRmsNormOutput = collections.namedtuple(
    "MusaRmsNorm", ["y", "normalized", "inv_rms"])
MusaAddRmsNormOutput = collections.namedtuple("MusaAddRmsNorm", ["y", "sum", "inv_rms"])
MusaAddRmsNormGradOutput = collections.namedtuple("MusaAddRmsNormGrad", ["dx", "dgamma"])
MusaAddRmsNormQuantizeOutput = collections.namedtuple(
    "MusaAddRmsNormQuantize", ["q", "scale", "sum"])
MusaQuantizeRowsOutput = collections.namedtuple("MusaQuantizeRows", ["q", "scale"])


def _rows(x):
    if x.dim() < 1:
        raise InvalidArgumentError("Input rank must be >= 1")
    last = x.shape[-1]
    return (x.numel() // last if last else 0), last


def _check_vector(v, name, last):
    if v.numel() != last:
        raise InvalidArgumentError(
            "%s size mismatch: expected %d, got %d" % (name, last, v.numel()))


def MusaLayerNorm(x, gamma, beta, epsilon=0.00001, name=None):
    """MusaLayerNorm for T in {float, half, bfloat16}: normalises the last
    axis, y = (x - mean) * rsqrt(var + epsilon) * gamma + beta
    (musa_ext/kernels/fusion/musa_layernorm_op.cc:26-100, op definition
    :118-124)."""
    out = _r._native().layer_norm(x, gamma, beta, epsilon)
    if out is not None:
        return _r._native_result(out, None, "MusaLayerNorm")
    _r._require_cuda()
    hf = _r._HostForm()
    xd, g, b = hf.to_device(x), hf.to_device(gamma), hf.to_device(beta)
    if xd.dtype not in _LN_DTYPES:
        raise InvalidArgumentError("MusaLayerNorm: unsupported dtype %s" % (xd.dtype,))
    if g.dtype != xd.dtype or b.dtype != xd.dtype:
        raise InvalidArgumentError("MusaLayerNorm: x, gamma and beta must share a dtype")
    rows, last = _rows(xd)
    _check_vector(g, "Gamma", last)
    _check_vector(b, "Beta", last)
    # Copies are held until the launch: the block of one that is gone is the next one's.
    xd, g, b = xd.contiguous(), g.contiguous(), b.contiguous()
    with torch.cuda.device(xd.device):
        y = torch.empty_like(xd)
        if xd.numel():
            fn = getattr(_r._lib(), "LaunchLayerNorm_" + _r._SUFFIX[xd.dtype])
            rc = fn(_r._ptr(xd), _r._ptr(g), _r._ptr(b), _r._ptr(y), None, None, rows, last,
                    float(epsilon), _r._stream())
            _r._check(rc, "MusaLayerNorm")
    return hf.back(y)


def MusaLayerNormGrad(dy, x, gamma, beta, epsilon=0.00001, name=None):
    """MusaLayerNormGrad: (dx, dgamma, dbeta) from dy, x, gamma; the row
    statistics are recomputed from x
    (musa_ext/kernels/fusion/musa_layernorm_grad_op.cc:23-141, op definition
    :143-158)."""
    out = _r._native().layer_norm_grad(dy, x, gamma, beta, epsilon)
    if out is not None:
        return _r._native_result(out, MusaLayerNormGradOutput, "MusaLayerNormGrad")
    _r._require_cuda()
    hf = _r._HostForm()
    d, xd, g, b = (hf.to_device(t) for t in (dy, x, gamma, beta))
    if xd.dtype not in _LN_DTYPES:
        raise InvalidArgumentError("MusaLayerNormGrad: unsupported dtype %s" % (xd.dtype,))
    if any(t.dtype != xd.dtype for t in (d, g, b)):
        raise InvalidArgumentError("MusaLayerNormGrad: all inputs must share a dtype")
    if xd.dim() < 1:
        raise InvalidArgumentError("Input rank must be >= 1")
    if tuple(d.shape) != tuple(xd.shape):
        raise InvalidArgumentError(
            "dy and x must have the same shape: dy=%s, x=%s"
            % (tuple(d.shape), tuple(xd.shape)))
    rows, last = _rows(xd)
    _check_vector(g, "Gamma", last)
    _check_vector(b, "Beta", last)
    xd, d, g = xd.contiguous(), d.contiguous(), g.contiguous()
    with torch.cuda.device(xd.device):
        dx = torch.empty_like(xd)
        dgamma = torch.empty_like(g)
        dbeta = torch.empty_like(b, memory_format=torch.contiguous_format)
        if last:
            lib = _r._lib()
            nbytes = lib.LayerNormGradWorkspaceBytes(rows, last)
            ws = _r._workspace(nbytes, xd.device)
            fn = getattr(lib, "LaunchLayerNormGrad_" + _r._SUFFIX[xd.dtype])
            rc = fn(_r._ptr(d), _r._ptr(xd), _r._ptr(g), _r._ptr(dx), _r._ptr(dgamma),
                    _r._ptr(dbeta), rows, last, float(epsilon), _r._ptr(ws), ws.numel(),
                    _r._stream())
            _r._check(rc, "MusaLayerNormGrad")
    return MusaLayerNormGradOutput(*hf.back_many([dx, dgamma, dbeta]))


def MusaRmsNorm(x, gamma, epsilon=0.00001, name=None):
    """MusaRmsNorm for T in {float, bfloat16}: returns (y, normalized,
    inv_rms), inv_rms shaped like x with a last axis of 1
    (musa_ext/kernels/nn/musa_rmsnorm_op.cc:24-87, op definition :175-201)."""
    out = _r._native().rms_norm(x, gamma, epsilon)
    if out is not None:
        return _r._native_result(out, MusaRmsNormOutput, "MusaRmsNorm")
    _r._require_cuda()
    hf = _r._HostForm()
    xd, g = hf.to_device(x), hf.to_device(gamma)
    if xd.dtype not in _RMS_DTYPES or g.dtype != xd.dtype:
        raise InvalidArgumentError("MusaRmsNorm expects float/bfloat16 inputs")
    if xd.dim() < 1:
        raise InvalidArgumentError("Input rank must be >= 1")
    last = xd.shape[-1]
    if last <= 0:
        raise InvalidArgumentError("Last dimension must be positive")
    _check_vector(g, "Gamma", last)
    rows = xd.numel() // last
    xd, g = xd.contiguous(), g.contiguous()
    with torch.cuda.device(xd.device):
        y = torch.empty_like(xd)
        normalized = torch.empty_like(xd)
        inv = torch.empty(tuple(xd.shape[:-1]) + (1,), dtype=xd.dtype, device=xd.device)
        if xd.numel():
            lib = _r._lib()
            fn = lib.LaunchRmsNormFloat if xd.dtype == torch.float32 else lib.LaunchRmsNormBFloat16
            fn(_r._ptr(xd), _r._ptr(g), _r._ptr(y), _r._ptr(normalized), _r._ptr(inv), rows,
               last, float(epsilon), _r._stream())
    return MusaRmsNormOutput(*hf.back_many([y, normalized, inv]))


def MusaRmsNormGradDx(x, inv_rms, gamma, dy, name=None):
    """MusaRmsNormGradDx: the gradient of MusaRmsNorm with respect to x
    (musa_ext/kernels/nn/musa_rmsnorm_op.cc:96-146, op definition :163-173)."""
    out = _r._native().rms_norm_grad_dx(x, inv_rms, gamma, dy)
    if out is not None:
        return _r._native_result(out, None, "MusaRmsNormGradDx")
    _r._require_cuda()
    hf = _r._HostForm()
    xd, inv, g, d = (hf.to_device(t) for t in (x, inv_rms, gamma, dy))
    if xd.dtype not in _RMS_DTYPES or any(t.dtype != xd.dtype for t in (inv, g, d)):
        raise InvalidArgumentError("MusaRmsNormGradDx expects float/bfloat16 inputs")
    if tuple(xd.shape) != tuple(d.shape):
        raise InvalidArgumentError("MusaRmsNormGradDx x/dy shape mismatch")
    if g.dim() != 1:
        raise InvalidArgumentError("MusaRmsNormGradDx gamma must be rank 1")
    last = g.numel()
    if last <= 0 or xd.numel() % last != 0:
        raise InvalidArgumentError("MusaRmsNormGradDx invalid row size")
    rows = xd.numel() // last
    if inv.numel() != rows:
        raise InvalidArgumentError("MusaRmsNormGradDx inv size mismatch")
    xd, inv, g, d = (t.contiguous() for t in (xd, inv, g, d))
    with torch.cuda.device(xd.device):
        dx = torch.empty_like(xd)
        if xd.numel():
            lib = _r._lib()
            fn = (lib.LaunchRmsNormGradDxFloat if xd.dtype == torch.float32
                  else lib.LaunchRmsNormGradDxBFloat16)
            fn(_r._ptr(xd), _r._ptr(inv), _r._ptr(g), _r._ptr(d), _r._ptr(dx), rows, last,
               _r._stream())
    return hf.back(dx)


# ------------------------------------------ RMS norm of a residual's sum --

def _check_rows(opname, x, others, normed=True):
    """x's rows and their length; `others`: (name, tensor, like x or a vector).  Rows of length
    0 have no norm."""
    if x.dtype not in _LN_DTYPES:
        raise InvalidArgumentError("%s: unsupported dtype %s" % (opname, x.dtype))
    if x.dim() < 1:
        raise InvalidArgumentError("Input rank must be >= 1")
    rows, last = _rows(x)
    if normed and not last:
        raise InvalidArgumentError("%s: the last dimension must be positive" % opname)
    for name, t, vector in others:
        if t is None:
            continue
        if t.dtype != x.dtype:
            raise InvalidArgumentError(
                "%s: %s dtype %s does not match %s" % (opname, name, t.dtype, x.dtype))
        if t.device != x.device:
            raise InvalidArgumentError(
                "%s: %s is on %s, not on %s" % (opname, name, t.device, x.device))
        if vector:
            _check_vector(t, name.capitalize(), last)
        elif tuple(t.shape) != tuple(x.shape):
            raise InvalidArgumentError(
                "%s: %s must have the shape %s, got %s"
                % (opname, name, tuple(x.shape), tuple(t.shape)))
    return rows, last


def MusaAddRmsNorm(x, residual, gamma, epsilon=0.00001, name=None):
    """The residual's addition with the RMS norm of the last axis behind it, for
    T in {float, half, bfloat16}: returns (y, sum, inv_rms) with sum = x +
    residual, inv_rms = rsqrt(mean(sum^2) + epsilon) (fp32, shaped like x with a
    last axis of 1) and y = sum * inv_rms * gamma.  The norm is that of the
    unrounded sum; `sum` holds it rounded to T.  One launch where Add and
    MusaRmsNorm are two with the sum written and read between.  Rows of length 0
    have no norm and are refused."""
    out = _r._native().add_rms_norm(x, residual, gamma, epsilon)
    if out is not None:
        return _r._native_result(out, MusaAddRmsNormOutput, "MusaAddRmsNorm")
    _r._require_cuda()
    hf = _r._HostForm()
    xd, rd, g = (hf.to_device(t) for t in (x, residual, gamma))
    rows, last = _check_rows("MusaAddRmsNorm", xd, [("residual", rd, False), ("gamma", g, True)])
    xd, rd, g = xd.contiguous(), rd.contiguous(), g.contiguous()
    with torch.cuda.device(xd.device):
        y, total = torch.empty_like(xd), torch.empty_like(xd)
        inv = torch.empty(tuple(xd.shape[:-1]) + (1,), dtype=torch.float32, device=xd.device)
        fn = getattr(_r._lib(), "LaunchAddRmsNorm_" + _r._SUFFIX[xd.dtype])
        rc = fn(_r._ptr(xd), _r._ptr(rd), _r._ptr(g), _r._ptr(y), _r._ptr(total), _r._ptr(inv),
                rows, last, float(epsilon), _r._stream())
        _r._check(rc, "MusaAddRmsNorm")
    return MusaAddRmsNormOutput(*hf.back_many([y, total, inv]))


def MusaAddRmsNormGrad(dy, dsum, sum, inv_rms, gamma, name=None):
    """The gradient of MusaAddRmsNorm from its stored sum and inv_rms: returns
    (dx, dgamma).  dx is the gradient of x and of the residual alike; `dsum` is
    the gradient that reaches `sum` past the norm (None: none does).  dgamma is
    summed over the rows in a fixed order."""
    out = _r._native().add_rms_norm_grad(dy, dsum, sum, inv_rms, gamma)
    if out is not None:
        return _r._native_result(out, MusaAddRmsNormGradOutput, "MusaAddRmsNormGrad")
    _r._require_cuda()
    hf = _r._HostForm()
    d, ds, s, inv, g = (hf.to_device(t) for t in (dy, dsum, sum, inv_rms, gamma))
    rows, last = _check_rows("MusaAddRmsNormGrad", s, [
        ("dy", d, False), ("dsum", ds, False), ("gamma", g, True)])
    if inv.dtype != torch.float32 or inv.numel() != rows or inv.device != s.device:
        raise InvalidArgumentError(
            "MusaAddRmsNormGrad: inv_rms must be float32 with one value per row (%d)" % rows)
    # Copies are held until the launch: the block of one that is gone is the next one's.
    s, d, inv, g = (t.contiguous() for t in (s, d, inv, g))
    ds = None if ds is None else ds.contiguous()
    with torch.cuda.device(s.device):
        dx, dgamma = torch.empty_like(s), torch.empty_like(g)
        lib = _r._lib()
        ws = _r._scratch(lib.AddRmsNormGradWorkspaceBytes(rows, last), s.device)
        fn = getattr(lib, "LaunchAddRmsNormGrad_" + _r._SUFFIX[s.dtype])
        rc = fn(_r._ptr(d), _r._ptr(ds), _r._ptr(s), _r._ptr(inv), _r._ptr(g), _r._ptr(dx),
                _r._ptr(dgamma), rows, last, _r._ptr(ws), ws.numel(), _r._stream())
        _r._check(rc, "MusaAddRmsNormGrad")
    return MusaAddRmsNormGradOutput(*hf.back_many([dx, dgamma]))


def _quantize(opname, x, residual, gamma, epsilon):
    out = _r._native().add_rms_norm_quantize(x, residual, gamma, epsilon)
    if out is not None:
        return _r._native_result(out, tuple, opname)
    _r._require_cuda()
    hf = _r._HostForm()
    xd, rd, g = (hf.to_device(t) for t in (x, residual, gamma))
    if hf.kind is not None:
        raise InvalidArgumentError(
            "%s: 8-bit outputs have no host form: pass device tensors" % opname)
    rows, last = _check_rows(opname, xd, [("residual", rd, False), ("gamma", g, True)],
                             normed=g is not None)
    xd = xd.contiguous()
    rd, g = (None if t is None else t.contiguous() for t in (rd, g))
    with torch.cuda.device(xd.device):
        q = torch.empty(xd.shape, dtype=torch.float8_e4m3fn, device=xd.device)
        scale = torch.empty(tuple(xd.shape[:-1]) + (1,), dtype=torch.float32, device=xd.device)
        if not last:                 # nothing is launched: the least scale, as for a row of zeros
            scale.fill_(_SCALE_MIN)
        total = None if rd is None else torch.empty_like(xd)
        fn = getattr(_r._lib(), "LaunchAddRmsNormQuantize_" + _r._SUFFIX[xd.dtype])
        rc = fn(_r._ptr(xd), _r._ptr(rd), _r._ptr(g), _r._ptr(q), _r._ptr(scale),
                _r._ptr(total), rows, last, float(epsilon), _r._stream())
        _r._check(rc, opname)
    return q, scale, total


def MusaAddRmsNormQuantize(x, residual, gamma, epsilon=0.00001, name=None):
    """MusaAddRmsNorm with its output in 8 bits: returns (q, scale, sum), q in
    float8_e4m3fn and scale = max(max|y| / 448, 2^-126) of each row (fp32, shaped
    like x with a last axis of 1), so that y = q * scale; y itself is not written.
    `residual` None: the norm of x alone, and sum is None.  A row with a NaN has a
    NaN scale; rows of length 0 have no norm and are refused."""
    if gamma is None:
        raise InvalidArgumentError("MusaAddRmsNormQuantize: gamma is missing")
    out = _quantize("MusaAddRmsNormQuantize", x, residual, gamma, epsilon)
    return MusaAddRmsNormQuantizeOutput(*out)


def MusaQuantizeRows(x, name=None):
    """The rows of x (T in {float, half, bfloat16}) in 8 bits: returns (q, scale),
    x = q * scale, as MusaAddRmsNormQuantize returns them; what lays out the weights
    [n, k] of MusaQuantizedMatMulBiasAct once.  A row of length 0 has the least scale,
    2^-126, as a row of zeros has."""
    return MusaQuantizeRowsOutput(*_quantize("MusaQuantizeRows", x, None, None, 0.0)[:2])
