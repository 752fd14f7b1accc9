"""The residual RMS norm of rows around a pack: the copies that the kernel makes, for every
small shape on the host (csrc/row_layout.h), and the values on the GPU.  The tolerances are
those of test_add_rms_norm_gpu.py."""
import os
import subprocess

import pytest
import torch

import test_add_rms_norm_gpu as norms
from conftest import ROOT
from tensorflow_musa_extension_b200 import raw_ops

PROGRAM = r"""
#include <cstdio>
#include "row_layout.h"
using namespace musa_b200;
template <int vec>
bool Inside(int n, int64_t rows) {
  bool ok = true;
  const int64_t tail = FirstTailRow<vec>(rows, n);
  for (int64_t row = 0; row < rows; ++row) {
    const int shift = RowShift<vec>(row, n), packs = ShiftedPacks<vec>(n, shift);
    const int64_t first = row * n - shift;
    int64_t end = first;
    for (int p = 0; p < packs; ++p) {
      const int e = ElementsInside<vec>(row, rows, tail, n, shift, p, packs);
      ok = ok && end == first + p * vec && e > 0 && e <= vec;
      // A shorter copy only where the tensor ends.
      ok = ok && (e == vec || end + e == rows * n) && end + e <= rows * n;
      end += e;
    }
    ok = ok && end >= (row + 1) * n;
  }
  if (!ok) std::printf("packs of %d: [%d, %d]\n", vec, (int)rows, n);
  return ok;
}
int main() {
  bool ok = true;
  for (int n = 1; n <= 40; ++n)
    for (int64_t rows = 1; rows <= 40; ++rows) ok = Inside<4>(n, rows) && Inside<8>(n, rows) && ok;
  return !ok;
}
"""


def test_forward_copies_stay_inside_the_tensor(tmp_path):
    src, exe = tmp_path / "rows.cc", tmp_path / "rows"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(
        ROOT, "tensorflow_musa_extension_b200", "csrc"), str(src), "-o", str(exe)], check=True)
    got = subprocess.run([str(exe)], capture_output=True, text=True)
    assert got.returncode == 0, got.stdout


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", norms.DTYPES)
@pytest.mark.parametrize("cols", [1, 2, 3, 5, 7, 9, 13])
def test_values_of_short_rows(kernel_lib, dtype, cols):
    for rows in (*range(1, 18), 1000, 1001, 1013):
        x, r = norms._rand((rows, cols), dtype, 1), norms._rand((rows, cols), dtype, 2, 3.0)
        g = norms._rand((cols,), dtype, 3)
        h, inv, y = norms._norm(x, r, g)
        lost = 2.0 ** -24 * (x.double().abs() + r.double().abs())
        got = raw_ops.MusaAddRmsNorm(x, r, g, epsilon=norms.EPS)
        half, small = norms._half(dtype), norms._small(dtype)
        norms._check(got.sum, h, lost + half * h.abs() + small, "sum of %d rows" % rows)
        # The sum that cancels takes its error into the mean of squares too.
        off = norms._rel(cols) * y.abs() + lost * inv * g.double().abs()
        off = off + y.abs() * (lost * h.abs()).sum(-1, keepdim=True) * inv ** 2
        norms._check(got.y, y, off + half * (y.abs() + off) + small, "y of %d rows" % rows)
        q = raw_ops.MusaQuantizeRows(x)
        scale = (x.double().abs().amax(-1, keepdim=True) / 448).clamp(min=2.0 ** -126)
        norms._check(q.scale, scale, 2.0 ** -22 * scale, "scale of %d rows" % rows)
        assert torch.equal(q.q.double(), norms._to_e4m3(x.float() / q.scale))
