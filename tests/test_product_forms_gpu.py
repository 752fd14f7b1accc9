"""Every tile of the matrix products' split form, and the operators of a transformer block
one behind the other, against the formulas in 64 bits.  The tolerances are those of
test_linear_gpu.py; each step of a run is checked on the inputs that it got."""
import pytest
import torch

import test_linear_gpu as linear
from tensorflow_musa_extension_b200 import raw_ops

pytestmark = pytest.mark.gpu

F16, BF16 = linear.F16, linear.BF16
_rand, _check = linear._rand, linear._check


@pytest.fixture
def forced(kernel_lib):
    old = kernel_lib.MusaKernelsSetTuning(29, 0)
    yield lambda rows, splits: kernel_lib.MusaKernelsSetTuning(29, rows + splits)
    kernel_lib.MusaKernelsSetTuning(29, old)


# Two and more tiles of every height, the last of them short; one and many blocks of depth.
@pytest.mark.parametrize("splits", [1, 2, 4, 8])
@pytest.mark.parametrize("rows", [16, 32, 64, 128, 256])
def test_row_tiles(forced, rows, splits):
    forced(rows, splits)
    for m, n, k in ((2 * rows + 5, 200, 1030), (rows, 129, 520), (3 * rows - 1, 64, 513),
                    (1, 130, 512)):
        for ta, tb in ((False, True), (True, False)):
            a = _rand((k, m) if ta else (m, k), BF16, 1)
            b = _rand((n, k) if tb else (k, n), BF16, 2, k ** -0.5)
            bias, res = _rand((n,), BF16, 3), _rand((m, n), BF16, 4)
            want, wz, tol, tz = linear._forward(a, b, bias, res, "Silu", ta, tb, BF16)
            y, z = raw_ops.MusaMatMulBiasAct(a, b, bias, res, "Silu", ta, tb,
                                             return_preactivation=True)
            _check(y, want, tol, "y %s" % ((m, n, k, ta, tb),))
            _check(z, wz, tz, "z %s" % ((m, n, k, ta, tb),))
        k -= k % 16
        (q, s), (w, ws) = linear._quantized(m, k, 5), linear._quantized(n, k, 6, k ** -0.5)
        want, _, tol, _ = linear._forward(q.double() * s, (w.double() * ws).mT, bias, res, "Gelu",
                                          False, False, F16)
        y = raw_ops.MusaQuantizedMatMulBiasAct(q, s, w, ws, bias.half(), res.half(), "Gelu", F16)
        _check(y, want, tol, "8 bit %s" % ((m, n, k),))
    raw_ops.check_products()


def _norm(x, residual, gamma):
    h = x.double() + residual.double()
    inv = ((h * h).mean(-1, keepdim=True) + 1e-5).rsqrt()
    return h, inv, h * inv * gamma.double()


def _norm_tol(v, dtype, cols):
    """Tolerance of values of a norm (fp32 sums of `cols` terms, one rounding)."""
    return ((cols / 32 + 40) * 2.0 ** -23 + torch.finfo(dtype).eps / 2) * v.abs() + 2.0 ** -18


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens,width,hidden", [(1, 64, 256), (130, 192, 520), (301, 515, 1030)])
def test_training_step_of_a_block(kernel_lib, dtype, tokens, width, hidden):
    """norm -> up-projection with Gelu -> down-projection with the residual, and back."""
    x, r, dout = (_rand((2, tokens, width), dtype, i) for i in (1, 2, 3))
    gamma = 1 + _rand((width,), dtype, 4, 0.2)
    up, b_up = _rand((width, hidden), dtype, 5, width ** -0.5), _rand((hidden,), dtype, 6)
    down, b_down = _rand((width, hidden), dtype, 7, hidden ** -0.5), _rand((width,), dtype, 8)
    n = raw_ops.MusaAddRmsNorm(x, r, gamma)
    u = raw_ops.MusaMatMulBiasAct(n.y, up, b_up, activation="Gelu", return_preactivation=True)
    out = raw_ops.MusaMatMulBiasAct(u.y, down, b_down, n.sum, transpose_b=True)
    d2 = raw_ops.MusaMatMulBiasActGrad(dout, u.y, down, transpose_b=True)
    d1 = raw_ops.MusaMatMulBiasActGrad(d2.da, n.y, up, u.preactivation, "Gelu")
    d0 = raw_ops.MusaAddRmsNormGrad(d1.da, dout, n.sum, n.inv_rms, gamma)

    h, inv, y = _norm(x, r, gamma)
    _check(n.sum, h, _norm_tol(h, dtype, 1), "sum")
    _check(n.y, y, _norm_tol(y, dtype, width), "norm")

    def flat(t):
        return t.reshape(-1, t.shape[-1])
    want, wz, tol, tz = linear._forward(flat(n.y), up, b_up, None, "Gelu", False, False, dtype)
    _check(flat(u.y), want, tol, "up")
    _check(flat(u.preactivation), wz, tz, "preactivation")
    want, _, tol, _ = linear._forward(flat(u.y), down, b_down, flat(n.sum), "Identity", False,
                                      True, dtype)
    _check(flat(out), want, tol, "down")
    for got, wants in ((d2, linear._backward(flat(dout), flat(u.y), down, None, "Identity", False,
                                             True, dtype)),
                       (d1, linear._backward(flat(d2.da), flat(n.y), up, flat(u.preactivation),
                                             "Gelu", False, False, dtype))):
        for name, g, (want, tol) in zip(got._fields, got, wants):
            _check(flat(g) if name == "da" else g, want, tol, name)
    s, dy, iv = flat(n.sum).double(), flat(d1.da).double(), n.inv_rms.double().reshape(-1, 1)
    g, hat = dy * gamma.double(), s * iv
    dx = flat(dout).double() + iv * (g - hat * (g * hat).mean(-1, keepdim=True))
    spread = iv * (g.abs() + hat.abs() * (g * hat).abs().mean(-1, keepdim=True))
    _check(flat(d0.dx), dx, _norm_tol(dx, dtype, 1) + (width / 32 + 40) * 2.0 ** -22 * spread,
           "dx")
    want, total = (dy * hat).sum(0), (dy * hat).abs().sum(0)
    _check(d0.dgamma, want, (2 * tokens + 8) * 2.0 ** -23 * total + _norm_tol(want, dtype, 1),
           "dgamma")
    raw_ops.check_products()


@pytest.mark.parametrize("tokens", [1, 16, 333])
def test_serving_step_of_a_block(kernel_lib, tokens):
    """The same block in 8 bits: norm and quantise -> up -> quantise -> down + residual."""
    width, hidden = 512, 1408
    x, r = _rand((tokens, width), BF16, 1), _rand((tokens, width), BF16, 2, 3.0)
    gamma = 1 + _rand((width,), BF16, 3, 0.2)
    up, down = linear._quantized(hidden, width, 4), linear._quantized(width, hidden, 5)
    n = raw_ops.MusaAddRmsNormQuantize(x, r, gamma)
    u = raw_ops.MusaQuantizedMatMulBiasAct(n.q, n.scale, up.q, up.scale, activation="Silu")
    q = raw_ops.MusaQuantizeRows(u)
    out = raw_ops.MusaQuantizedMatMulBiasAct(q.q, q.scale, down.q, down.scale, residual=n.sum)
    # A step of e4m3 is at most 2^-3 of a value, a rounding half of that; below 2^-6 the steps
    # are 2^-9 (in units of the scale).
    _, _, y = _norm(x, r, gamma)
    for what, v, got in (("norm", y, n), ("up", u.double(), q)):
        _check(got.q.double() * got.scale, v, 2.0 ** -4 * 1.001 * v.abs() + 2.0 ** -10 * got.scale,
               what)
    for what, got, a, b, res, act in (("up", u, n, up, None, "Silu"),
                                      ("down", out, q, down, n.sum, "Identity")):
        want, _, tol, _ = linear._forward(a.q.double() * a.scale, b.q.double() * b.scale, None, res,
                                          act, False, True, BF16)
        _check(got, want, tol, what)
    raw_ops.check_products()
