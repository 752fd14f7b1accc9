"""Scales whose product no fp32 number holds: z = product * a_scale * b_scale, one after the
other."""
import pytest
import torch

import test_linear_gpu as linear
from tensorflow_musa_extension_b200 import raw_ops

pytestmark = pytest.mark.gpu
form = linear.form


@pytest.mark.parametrize("m,n,k", [(20, 140, 64), (300, 264, 256)])
def test_scales_far_from_one(form, m, n, k):
    a, b = linear._quantized(m, k, 1).q, linear._quantized(n, k, 2).q

    def scales(of_a, of_b):
        return (torch.full((m, 1), of_a, device="cuda"), torch.full((n, 1), of_b, device="cuda"))
    # Zeros stay zeros.
    y = raw_ops.MusaQuantizedMatMulBiasAct(torch.zeros_like(a), scales(2.0 ** 70, 1)[0], b,
                                           scales(1, 2.0 ** 70)[1])
    assert not y.any()
    # The scales' product, some 2^-144, keeps five bits in fp32; z, 2^22 and more times as large,
    # is normal.
    for of_a, of_b in ((1.7 * 2.0 ** -100, 1.3 * 2.0 ** -45), (1.3 * 2.0 ** -20, 1.7 * 2.0 ** -124)):
        sa, sb = scales(of_a, of_b)
        ones = (torch.full_like(a.float(), 448.0).to(a.dtype), torch.full_like(
            b.float(), 256.0).to(b.dtype))
        want = 448.0 * 256.0 * k * sa.double() * sb.double().mT
        y = raw_ops.MusaQuantizedMatMulBiasAct(ones[0], sa, ones[1], sb)
        # Two fp32 products and one rounding to bfloat16, whose smallest step is 2^-133.
        tol = (2.0 ** -8 + 2.0 ** -22) * want + 2.0 ** -134
        linear._check(y, want, tol, "small scales")
