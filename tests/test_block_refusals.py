"""What the launchers of the residual RMS norm and of the matrix products refuse before they
touch the device: the addresses below are never read."""
import pytest

OK, EINVAL, EWORKSPACE, EUNSUPPORTED, ETOOLARGE = 0, -1, -2, -3, -4
P, ODD = 1 << 20, (1 << 20) + 2     # on and off a 16-byte boundary
F32, F16, BF16 = 0, 1, 2
TOO_MANY = 65535 * 256 + 1


def _product(lib, dtype=BF16, a=P, lda=64, ta=False, b=P, ldb=32, tb=False, y=P, m=8, n=32, k=64,
             act=0, ws=None, size=0):
    return lib.LaunchMatMulBiasAct(dtype, a, lda, ta, b, ldb, tb, None, None, y, None, m, n, k,
                                   act, ws, size, None)


@pytest.mark.parametrize("want,change", [
    (EUNSUPPORTED, dict(dtype=F32)), (EUNSUPPORTED, dict(dtype=7)),
    (EUNSUPPORTED, dict(act=2)),                      # Swish: its factor is not z
    (EUNSUPPORTED, dict(act=-1)), (EUNSUPPORTED, dict(act=6)),
    (EINVAL, dict(m=-1)), (EINVAL, dict(n=-1)), (EINVAL, dict(k=-1)),
    (ETOOLARGE, dict(m=TOO_MANY)), (ETOOLARGE, dict(n=TOO_MANY)),
    (EINVAL, dict(y=None)), (EINVAL, dict(a=None)), (EINVAL, dict(b=None)),
    (EINVAL, dict(lda=63)), (EINVAL, dict(ldb=31)),
    (EINVAL, dict(ta=True, lda=7)), (EINVAL, dict(tb=True, ldb=63)),
    (EWORKSPACE, dict(a=ODD)), (EWORKSPACE, dict(ldb=33)),
    (EWORKSPACE, dict(a=ODD, ws=P, size=16)), (EWORKSPACE, dict(a=ODD, ws=ODD, size=1 << 20)),
    (OK, dict(m=0)), (OK, dict(n=0)), (OK, dict(m=0, a=None, y=None)),
])
def test_products(kernel_lib, want, change):
    assert _product(kernel_lib, **change) == want


def _gradient(lib, dtype=BF16, dy=P, a=P, b=P, z=P, m=8, n=32, k=64, act=1, ws=P, size=1 << 20):
    return lib.LaunchMatMulBiasActGrad(dtype, dy, a, k, False, b, n, False, z, P, P, P, m, n, k,
                                       act, ws, size, None)


@pytest.mark.parametrize("want,change", [
    (EUNSUPPORTED, dict(dtype=F32)), (EUNSUPPORTED, dict(act=2)), (EINVAL, dict(m=-1)),
    (ETOOLARGE, dict(k=TOO_MANY)), (EINVAL, dict(dy=None)), (EINVAL, dict(z=None)),
    (EINVAL, dict(a=None)), (EINVAL, dict(b=None)), (EWORKSPACE, dict(ws=None)),
    (EWORKSPACE, dict(size=16)), (EWORKSPACE, dict(ws=ODD)),
])
def test_product_gradients(kernel_lib, want, change):
    assert _gradient(kernel_lib, **change) == want


def _bytes(lib, dtype=BF16, a=P, lda=64, sa=P, b=P, ldb=64, sb=P, y=P, m=8, n=32, k=64, act=0,
           ws=None, size=0):
    return lib.LaunchQuantizedMatMulBiasAct(dtype, a, lda, sa, b, ldb, sb, None, None, y, m, n, k,
                                            act, ws, size, None)


@pytest.mark.parametrize("want,change", [
    (EUNSUPPORTED, dict(dtype=F32)), (EUNSUPPORTED, dict(act=2)), (EINVAL, dict(k=-1)),
    (ETOOLARGE, dict(n=TOO_MANY)), (EINVAL, dict(sa=None)), (EINVAL, dict(sb=None)),
    (EINVAL, dict(y=None)), (EINVAL, dict(lda=63)), (EINVAL, dict(ldb=63)),
    (EWORKSPACE, dict(lda=65)), (EWORKSPACE, dict(b=ODD)), (OK, dict(m=0)),
])
def test_8bit_products(kernel_lib, want, change):
    assert _bytes(kernel_lib, **change) == want


def test_workspace_queries(kernel_lib):
    lib = kernel_lib

    def need(a=P, lda=64, b=P, ldb=32, m=8, elem=2):
        return lib.MatMulWorkspaceBytes(elem, a, lda, False, b, ldb, False, m, 32, 64)
    assert need() == 0 and need(m=-1) == 0 and need(elem=4) == 0
    assert need(a=ODD) >= 8 * 64 * 2 and need(ldb=33) >= 64 * 32 * 2
    assert need(a=ODD, ldb=33) >= need(a=ODD) + need(ldb=33)


@pytest.mark.parametrize("suffix", ["F32", "F16", "BF16"])
def test_norms(kernel_lib, suffix):
    norm = getattr(kernel_lib, "LaunchAddRmsNorm_" + suffix)
    quantize = getattr(kernel_lib, "LaunchAddRmsNormQuantize_" + suffix)
    grad = getattr(kernel_lib, "LaunchAddRmsNormGrad_" + suffix)
    for missing in range(6):
        p = [None if i == missing else P for i in range(6)]
        assert norm(*p, 4, 64, 1e-5, None) == EINVAL
    for rows, size in ((-1, 64), (4, -1), (4, (1 << 24) + 1)):
        assert norm(*[P] * 6, rows, size, 1e-5, None) == EINVAL
        assert quantize(*[P] * 6, rows, size, 1e-5, None) == EINVAL
        assert grad(*[P] * 7, rows, size, P, 1 << 30, None) == EINVAL
    assert norm(*[None] * 6, 0, 64, 1e-5, None) == OK
    assert norm(*[None] * 6, 4, 0, 1e-5, None) == OK
    # x, residual, gamma, q, scale, sum
    for p in ((None, P, P, P, P, P), (P, P, P, None, P, P), (P, P, P, P, None, P),
              (P, P, P, P, P, None), (P, None, P, P, P, P), (P, P, None, P, P, P)):
        assert quantize(*p, 4, 64, 1e-5, None) == EINVAL
    # dy, dsum, sum, inv_rms, gamma, dx, dgamma
    need = kernel_lib.AddRmsNormGradWorkspaceBytes(4, 64)
    for missing in (0, 2, 3, 4, 5, 6):
        p = [None if i == missing else P for i in range(7)]
        assert grad(*p, 4, 64, P, need, None) == EINVAL
    for ws, size in ((None, need), (P, need - 1), (ODD, need)):
        assert grad(*[P] * 7, 4, 64, ws, size, None) == EWORKSPACE
    assert grad(*[None] * 7, 4, 0, None, 0, None) == OK
