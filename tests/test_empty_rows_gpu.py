"""Norms of rows of length 0: MusaRmsNorm refuses them, and so do these; a row without values
is quantised with the smallest scale."""
import pytest
import torch

from tensorflow_musa_extension_b200 import errors, raw_ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lead", [(3,), (2, 3), (0,)])
def test_rows_of_length_0(monkeypatch, kernel_lib, dtype, lead, native):
    if not native:
        monkeypatch.setattr(raw_ops, "_native", lambda: raw_ops._NoNativePath())
    x = torch.empty(lead + (0,), dtype=dtype, device="cuda")
    g = torch.empty(0, dtype=dtype, device="cuda")
    inv = torch.ones(lead + (1,), device="cuda")
    for call in (lambda: raw_ops.MusaAddRmsNorm(x, x, g),
                 lambda: raw_ops.MusaAddRmsNormGrad(x, None, x, inv, g),
                 lambda: raw_ops.MusaAddRmsNormQuantize(x, x, g),
                 lambda: raw_ops.MusaAddRmsNormQuantize(x, None, g)):
        with pytest.raises(errors.InvalidArgumentError):
            call()
    # What the allocator hands out next is not zero.
    dirty = torch.full(inv.shape, float("nan"), device="cuda")
    del dirty
    q, scale = raw_ops.MusaQuantizeRows(x)
    assert q.shape == x.shape and scale.shape == inv.shape and scale.dtype == torch.float32
    assert (scale == 2.0 ** -126).all()
    if lead == (3,):
        w, ws = q.new_empty(5, 0), torch.ones(5, 1, device="cuda")
        assert not raw_ops.MusaQuantizedMatMulBiasAct(q, scale, w, ws).any()
