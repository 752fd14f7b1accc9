"""The form of the matrix products that can be forced: only values that name one."""
import pytest

FORM = 29


@pytest.fixture
def restored(kernel_lib):
    old = kernel_lib.MusaKernelsGetTuning(FORM)
    yield kernel_lib
    kernel_lib.MusaKernelsSetTuning(FORM, old)


def test_forms_that_there_are(restored):
    before = restored.MusaKernelsGetTuning(FORM)
    for value in (1, 2, 3, *(r + s for r in range(16, 257, 16) for s in (1, 2, 4, 8)), 0):
        assert restored.MusaKernelsSetTuning(FORM, value) == before
        assert restored.MusaKernelsGetTuning(FORM) == value
        before = value


@pytest.mark.parametrize("value", [-1, 4, 8, 15, 16, 32, 16 + 3, 64 + 5, 128 + 6, 256 + 9, 240 + 15,
                                   256, 272 + 1, 512 + 1, 1 << 20, -16 + 1, -(1 << 31)])
def test_forms_that_there_are_not(restored, value):
    before = restored.MusaKernelsGetTuning(FORM)
    assert restored.MusaKernelsSetTuning(FORM, value) == -1
    assert restored.MusaKernelsGetTuning(FORM) == before
