"""check_products() waits for everything that the device has to do."""
import pytest
import torch

from tensorflow_musa_extension_b200 import raw_ops

pytestmark = pytest.mark.gpu


def test_status_waits_for_streams_that_do_not_block(kernel_lib):
    a = torch.ones(64, 64, dtype=torch.bfloat16, device="cuda")
    raw_ops.MusaMatMulBiasAct(a, a)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(400_000_000)     # 0.2 s at 1.965 GHz
        raw_ops.MusaMatMulBiasAct(a, a)
    raw_ops.check_products()
    done = side.query()
    side.synchronize()
    assert done
