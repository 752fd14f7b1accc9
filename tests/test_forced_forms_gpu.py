"""The forced form of a product on depths that its CTAs cannot all share."""
import pytest
import torch

import test_linear_gpu as linear
from tensorflow_musa_extension_b200 import raw_ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [16, 64, 256])
@pytest.mark.parametrize("splits", [2, 4, 8])
@pytest.mark.parametrize("k", [0, 16, 128, 256, 384])
def test_more_ctas_than_blocks_of_depth(kernel_lib, rows, splits, k):
    m, n = rows + 5, 200
    one = torch.ones(m, 1, device="cuda"), torch.ones(n, 1, device="cuda")
    a, b = linear._quantized(m, k, 1).q, linear._quantized(n, k, 2).q
    want, _, tol, _ = linear._forward(a.double(), b.double().mT, None, None, "Identity", False,
                                      False, torch.bfloat16)
    # What another product left in tensor memory would be seen with scales of one.
    big = torch.full((512, 512), 300.0, dtype=torch.bfloat16, device="cuda")
    old = kernel_lib.MusaKernelsSetTuning(29, 0)
    try:
        for _ in range(4):
            kernel_lib.MusaKernelsSetTuning(29, 3)
            raw_ops.MusaMatMulBiasAct(big, big)
            assert kernel_lib.MusaKernelsSetTuning(29, rows + splits) == 3
            y = raw_ops.MusaQuantizedMatMulBiasAct(a, one[0], b, one[1])
            linear._check(y, want, tol, "forced")
    finally:
        kernel_lib.MusaKernelsSetTuning(29, old)
    raw_ops.check_products()
