"""Vector arguments that are not contiguous, several of them in one call: the bits of the
call with contiguous copies, and the formulas in 64 bits.  The tolerances are those of
test_linear_gpu.py."""
import pytest
import torch

import test_linear_gpu as linear
from tensorflow_musa_extension_b200 import raw_ops

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
_rand, _check = linear._rand, linear._check


def _every_second(t):
    return torch.stack((t, torch.full_like(t, 3.0)), -1).flatten(-2)[..., ::2]


def _column(t):
    """t as a column of a table."""
    flat = t.reshape(-1)
    return torch.stack((torch.full_like(flat, 5.0), flat, flat + 1), 1)[:, 1].view(t.shape)


STORED = [_every_second, _column]


@pytest.mark.parametrize("stored", STORED)
@pytest.mark.parametrize("m,n,k", [(64, 64, 64), (1, 128, 96), (130, 100, 48), (300, 300, 272)])
def test_scales_of_8bit_products(kernel_lib, stored, m, n, k):
    a, sa = linear._quantized(m, k, 1)
    b, sb = linear._quantized(n, k, 2, k ** -0.5)
    want, _, tol, _ = linear._forward(a.double() * sa, (b.double() * sb).mT, None, None, "Silu",
                                      False, False, BF16)
    plain = raw_ops.MusaQuantizedMatMulBiasAct(a, sa, b, sb, activation="Silu")
    y = raw_ops.MusaQuantizedMatMulBiasAct(a, stored(sa), b, stored(sb), activation="Silu")
    _check(y, want, tol, "strided scales")
    assert torch.equal(y, plain)


def test_one_scale_for_all_rows(kernel_lib):
    m, n, k = 64, 64, 128
    a, b = (linear._quantized(s, k, i).q for i, s in enumerate((m, n)))
    sa, sb = torch.full((1, 1), 0.25, device="cuda"), torch.full((1, 1), 8.0, device="cuda")
    want, _, tol, _ = linear._forward(a.double() * 0.25, (b.double() * 8.0).mT, None, None,
                                      "Identity", False, False, F16)
    y = raw_ops.MusaQuantizedMatMulBiasAct(a, sa.expand(m, 1), b, sb.expand(n, 1), out_dtype=F16)
    # Half ends at 65504; what rounds to 65520 and more is infinite.
    inside, beyond = want.abs() + tol < 65504, want.abs() - tol >= 65520
    assert inside.any() and torch.equal(y[beyond].double(), want[beyond].sign() * float("inf"))
    _check(y[inside], want[inside], tol[inside], "expanded scales")


@pytest.mark.parametrize("stored", STORED)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,cols", [(64, 64), (100, 100), (300, 512)])
def test_vectors_of_the_residual_norm(kernel_lib, stored, dtype, rows, cols):
    x, r, dy = (_rand((rows, cols), dtype, i) for i in (1, 2, 3))
    g = _rand((cols,), dtype, 4)
    f = raw_ops.MusaAddRmsNorm(x, r, g)
    want = (*f, *raw_ops.MusaAddRmsNormGrad(dy, r, f.sum, f.inv_rms, g),
            *raw_ops.MusaAddRmsNormQuantize(x, r, g))
    got = (*raw_ops.MusaAddRmsNorm(x, r, stored(g)),
           *raw_ops.MusaAddRmsNormGrad(dy, r, f.sum, stored(f.inv_rms), stored(g)),
           *raw_ops.MusaAddRmsNormQuantize(x, r, stored(g)))
    for a, b in zip(got, want):
        assert a.shape == b.shape and torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("stored", STORED)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,cols", [(64, 64), (100, 100), (300, 512)])
def test_vectors_of_the_row_norms(kernel_lib, stored, dtype, rows, cols):
    x, dy = (_rand((rows, cols), dtype, i) for i in (1, 2))
    g, b = _rand((cols,), dtype, 3), _rand((cols,), dtype, 4)
    inv = raw_ops.MusaRmsNorm(x, g).inv_rms

    def all_of(g, b, inv):
        return (raw_ops.MusaLayerNorm(x, g, b), *raw_ops.MusaLayerNormGrad(dy, x, g, b),
                *raw_ops.MusaRmsNorm(x, g), raw_ops.MusaRmsNormGradDx(x, inv, g, dy))
    for got, want in zip(all_of(stored(g), stored(b), stored(inv)), all_of(g, b, inv)):
        assert got.shape == want.shape and torch.equal(got, want)


def test_gradients_of_vectors_with_two_axes(kernel_lib):
    """Vectors are taken by their number of values; one of two axes, stored with the first
    contiguous, has its gradients in the order of its values."""
    x, dy = _rand((70, 24), F32, 1), _rand((70, 24), F32, 2)
    g, b = _rand((24,), F32, 3), _rand((24,), F32, 4)
    inv = raw_ops.MusaRmsNorm(x, g).inv_rms

    def both(g, b):
        return (*raw_ops.MusaLayerNormGrad(dy, x, g, b)[1:],
                raw_ops.MusaAddRmsNormGrad(dy, None, x, inv, g).dgamma)
    tables = (t.view(4, 6).t().contiguous().t() for t in (g, b))
    for got, want in zip(both(*tables), both(g, b)):
        assert got.shape == (4, 6) and torch.equal(got.reshape(-1), want)
