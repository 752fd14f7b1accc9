"""MusaAddRmsNorm, its gradient, MusaAddRmsNormQuantize and MusaQuantizeRows on the GPU
against the formulas in 64 bits.

Tolerances.  A row's fp32 sum of squares adds at most row_size / 32 + 32 terms one after the
other, all of one sign: (row_size / 32 + 32) * 2^-24 relative; its root, the division and
the products behind it are good to 2^-21.  An output is rounded once: half a step."""
import pytest
import torch

from tensorflow_musa_extension_b200 import errors, raw_ops

pytestmark = pytest.mark.gpu

F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
DTYPES = [F32, F16, BF16]
EPS = 1e-5
# One element, below and around a pack, every width of row group, rows that are no whole
# packs, rows beyond what the threads of a CTA hold.
COLS = [1, 2, 3, 7, 8, 9, 31, 32, 33, 64, 100, 128, 255, 256, 257, 500, 512, 513, 1000, 1024,
        1025, 2047, 2048, 4096, 4100, 5001, 8192, 8200, 16384, 16390, 20000, 32768, 33000]


def _rand(shape, dtype, seed, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _rows(cols):
    return 37 if cols < 4096 else 5


def _half(t):
    return torch.finfo(t).eps / 2


def _small(t):
    """Half the smallest step of the type."""
    return torch.finfo(t).tiny * torch.finfo(t).eps / 2


def _rel(cols):
    return (cols / 32 + 32) * 2.0 ** -24 + 2.0 ** -21


def _check(got, want, tol, what):
    assert got.shape == want.shape, what
    off = (got.double() - want).abs() - tol
    assert float(off.max()) <= 0, "%s: off by %g more than allowed" % (what, float(off.max()))


def _norm(x, residual, gamma):
    h = x.double() + residual.double()
    inv = ((h * h).mean(-1, keepdim=True) + EPS).rsqrt()
    return h, inv, h * inv * gamma.double()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", COLS)
def test_forward(kernel_lib, dtype, cols):
    x, r = _rand((_rows(cols), cols), dtype, 1), _rand((_rows(cols), cols), dtype, 2, 3.0)
    g = _rand((cols,), dtype, 3)
    h, inv, y = _norm(x, r, g)
    got = raw_ops.MusaAddRmsNorm(x, r, g, epsilon=EPS)
    # The fp32 sum is off by 2^-24 of itself, which may be what cancels in h.
    lost = 2.0 ** -24 * (x.double().abs() + r.double().abs())
    _check(got.sum, h, lost + _half(dtype) * h.abs() + _small(dtype), "sum")
    assert got.inv_rms.dtype == F32 and got.inv_rms.shape == (x.shape[0], 1)
    _check(got.inv_rms, inv, _rel(cols) * inv, "inv_rms")
    off = _rel(cols) * y.abs() + lost * inv * g.double().abs()
    _check(got.y, y, off + _half(dtype) * (y.abs() + off) + _small(dtype), "y")


def _to_e4m3(v):
    """The nearest of the type's values, ties to the even one."""
    return v.float().to(E4M3).double()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", COLS)
def test_quantize(kernel_lib, dtype, cols):
    x, r = _rand((_rows(cols), cols), dtype, 1), _rand((_rows(cols), cols), dtype, 2, 3.0)
    g = _rand((cols,), dtype, 3)
    x[1] = 0
    r[1] = 0
    h, inv, y = _norm(x, r, g)
    for args, want, total in (((x, r, g), y, h), ((x, None, g), _norm(x, 0 * x, g)[2], None),
                              ((x, None, None), x.double(), None)):
        if args[2] is None:
            got = raw_ops.MusaQuantizeRows(x)
        else:
            got = raw_ops.MusaAddRmsNormQuantize(*args, epsilon=EPS)
            assert (got.sum is None) == (total is None)
            if total is not None:
                assert torch.equal(got.sum, raw_ops.MusaAddRmsNorm(*args, epsilon=EPS).sum)
        scale = (want.abs().amax(-1, keepdim=True) / 448).clamp(min=2.0 ** -126)
        assert got.q.dtype == E4M3 and got.scale.shape == (x.shape[0], 1)
        rel = 2 * _rel(cols) + 2.0 ** -22
        _check(got.scale, scale, rel * scale, "scale")
        # The fp32 arithmetic moves y / scale by rel (and what cancels in h) at most; rounding
        # is monotone, so q lies between the roundings of the two ends.  (No count of values
        # that differ from the nearest: quotients of 16-bit values fall on a border often.)
        v = want / scale
        off = (2 * rel + 2.0 ** -23) * v.abs()
        if args[1] is not None:
            off = off + (2.0 ** -24 * (x.double().abs() + r.double().abs()) * inv
                         * g.double().abs() / scale)
        q = got.q.double()
        assert (q >= _to_e4m3((v - off).clamp(-448, 448))).all()
        assert (q <= _to_e4m3((v + off).clamp(-448, 448))).all()
        if args[2] is None:     # one division, rounded once
            assert torch.equal(q, _to_e4m3(x.float() / got.scale))
        assert (got.q.double().abs().amax(-1) >= 447).sum() == (want.abs().amax(-1) > 0).sum()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", COLS)
def test_gradient(kernel_lib, dtype, cols):
    rows = _rows(cols)
    s, dy, ds = (_rand((rows, cols), dtype, i, 2.0) for i in (1, 2, 3))
    g = _rand((cols,), dtype, 4)
    inv = ((s.double() ** 2).mean(-1, keepdim=True) + EPS).rsqrt().float()
    for dsum in (ds, None):
        got = raw_ops.MusaAddRmsNormGrad(dy, dsum, s, inv, g)
        hat, u = s.double() * inv.double(), dy.double() * g.double()
        dot, dots = (u * hat).mean(-1, keepdim=True), (u * hat).abs().mean(-1, keepdim=True)
        dx = inv.double() * (u - hat * dot)
        off = inv.double() * (2.0 ** -22 * u.abs() + hat.abs() * (_rel(cols) * dots
                                                                  + 2.0 ** -21 * dot.abs()))
        if dsum is not None:
            dx = dx + dsum.double()
            off = off + 2.0 ** -24 * dx.abs()
        _check(got.dx, dx, off + _half(dtype) * (dx.abs() + off) + _small(dtype), "dx")
        dg, dgs = (dy.double() * hat).sum(0), (dy.double() * hat).abs().sum(0)
        off = (rows + 8) * 2.0 ** -23 * dgs
        _check(got.dgamma, dg, off + _half(dtype) * (dg.abs() + off) + _small(dtype), "dgamma")


@pytest.mark.parametrize("dtype,rows,cols", [(BF16, 70001, 96), (F16, 20011, 333), (F32, 9001, 1024),
                                             (BF16, 5003, 2999), (F32, 4001, 4097)])
def test_many_rows(kernel_lib, dtype, rows, cols):
    """More rows than one round of the CTAs; two runs give the same bits."""
    s, dy, x = (_rand((rows, cols), dtype, i) for i in (1, 2, 3))
    g = _rand((cols,), dtype, 4)
    f = raw_ops.MusaAddRmsNorm(x, s, g)
    h, inv, y = _norm(x, s, g)
    lost = 2.0 ** -24 * (x.double().abs() + s.double().abs()) * inv * g.double().abs()
    off = _rel(cols) * y.abs() + lost
    _check(f.y, y, off + _half(dtype) * (y.abs() + off) + _small(dtype), "y")
    a = raw_ops.MusaAddRmsNormGrad(dy, None, f.sum, f.inv_rms, g)
    b = raw_ops.MusaAddRmsNormGrad(dy, None, f.sum, f.inv_rms, g)
    assert torch.equal(a.dx, b.dx) and torch.equal(a.dgamma, b.dgamma)
    hat = f.sum.double() * f.inv_rms.double()
    dg, dgs = (dy.double() * hat).sum(0), (dy.double() * hat).abs().sum(0)
    # A thread adds the rows of its CTA, at most rows / 8 + 16; the rest is fp64.
    off = (rows / 8 + 16) * 2.0 ** -24 * dgs + 2.0 ** -22 * dgs
    _check(a.dgamma, dg, off + _half(dtype) * (dg.abs() + off), "dgamma")


def test_gradient_against_differences(kernel_lib):
    """Central differences of the 64-bit forward: fp32 rows of 11, both outputs used."""
    x, r, g = _rand((4, 11), F32, 1), _rand((4, 11), F32, 2), _rand((11,), F32, 3)
    dy, ds = _rand((4, 11), F32, 4), _rand((4, 11), F32, 5)
    f = raw_ops.MusaAddRmsNorm(x, r, g, epsilon=EPS)
    got = raw_ops.MusaAddRmsNormGrad(dy, ds, f.sum, f.inv_rms, g)

    def loss(x, g):
        h, _, y = _norm(x, r, g)
        return float((y * dy.double()).sum() + (h * ds.double()).sum())
    h = 1e-5
    for i, want_of in enumerate((got.dx, got.dgamma)):
        args = [x.double(), g.double()]
        want = torch.zeros_like(args[i])
        for j in range(want.numel()):
            ends = []
            for sign in (1, -1):
                moved = [t.clone() for t in args]
                moved[i].view(-1)[j] += sign * h
                ends.append(loss(*moved))
            want.view(-1)[j] = (ends[0] - ends[1]) / (2 * h)
        # fp32 sums of 11 and 4 terms of size 10 at most; differences good to h^2 and 1e-16 / h.
        _check(want_of, want, 2e-5 * (1 + want.abs()), "argument %d" % i)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [5, 256, 1000, 20000])
def test_values_that_are_not_finite(kernel_lib, dtype, cols):
    x, r = _rand((6, cols), dtype, 1), _rand((6, cols), dtype, 2)
    g = _rand((cols,), dtype, 3).abs() + 0.5
    want = raw_ops.MusaAddRmsNorm(x, r, g)
    q_want = raw_ops.MusaAddRmsNormQuantize(x, r, g)
    x[1, 2] = float("nan")
    x[3, 0] = float("inf")
    x[4] = 0
    r[4] = 0
    got = raw_ops.MusaAddRmsNorm(x, r, g)
    q = raw_ops.MusaAddRmsNormQuantize(x, r, g)
    assert got.y[1].isnan().all() and q.scale[1].isnan() and q.q[1].float().isnan().all()
    assert got.y[3, 0].isnan() and not got.y[3, 1:].any() and q.scale[3].isnan()
    assert not got.y[4].any() and not q.q[4].float().any() and q.scale[4] == 2.0 ** -126
    for i in (0, 2, 5):
        assert torch.equal(got.y[i], want.y[i]) and q.scale[i] == q_want.scale[i]
    p = raw_ops.MusaQuantizeRows(x)
    assert p.scale[1].isnan() and p.scale[3] == float("inf") and p.q[3, 0].float().isnan()
    assert not p.q[3, 1:].float().any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(6, 64), (3, 2, 37), (4, 5, 1000)])
def test_forms_and_paths(monkeypatch, kernel_lib, dtype, shape):
    """Storage other than the tested one, on the native and the general path."""
    def forms(t):
        yield t
        yield t.transpose(0, 1).contiguous().transpose(0, 1)
        yield torch.stack((t, t), -1).flatten(-2)[..., ::2]
        yield torch.cat((t.new_zeros(1), t.reshape(-1)))[1:].view(t.shape)
        yield t[:1].expand(t.shape)
    x, r, dy = (_rand(shape, dtype, i) for i in (1, 2, 3))
    g = _rand(shape[-1:], dtype, 4)

    def all_of(x, r, dy, g):
        f = raw_ops.MusaAddRmsNorm(x, r, g)
        return (*f, *raw_ops.MusaAddRmsNormGrad(dy, r, f.sum, f.inv_rms, g),
                *raw_ops.MusaAddRmsNormQuantize(x, r, g), *raw_ops.MusaQuantizeRows(x))

    def bits(t):
        return t.view(torch.uint8)
    for fx, fr, fd in zip(forms(x), forms(r), forms(dy)):
        got = all_of(fx, fr, fd, g)
        with monkeypatch.context() as m:
            m.setattr(raw_ops, "_native", lambda: raw_ops._NoNativePath())
            want = all_of(fx, fr, fd, g)
        for a, b in zip(got, want):
            assert a.shape == b.shape and torch.equal(bits(a), bits(b))
        # Off a 16-byte boundary the sums take another order.
        plain = all_of(*(t.clone(memory_format=torch.contiguous_format) for t in (fx, fr, fd, g)))
        for a, b in zip(got[:5], plain):
            tol = (4 * _half(a.dtype) + 2.0 ** -19) * (1 + b.double().abs())
            _check(a, b.double(), tol, "form")


def test_outputs_stay_inside_their_tensors(kernel_lib):
    st = torch.cuda.current_stream().cuda_stream
    for cols in (3, 37, 100, 1001):
        x, r, g = _rand((9, cols), BF16, 1), _rand((9, cols), BF16, 2), _rand((cols,), BF16, 3)
        n = 9 * cols
        y, s = (torch.full((n + 128,), 7.0, dtype=BF16, device="cuda") for _ in range(2))
        q = torch.full((n + 128,), 7, dtype=torch.uint8, device="cuda")
        inv = torch.empty(9, device="cuda")
        assert kernel_lib.LaunchAddRmsNorm_BF16(x.data_ptr(), r.data_ptr(), g.data_ptr(),
                                                y.data_ptr() + 128, s.data_ptr() + 128,
                                                inv.data_ptr(), 9, cols, EPS, st) == 0
        assert kernel_lib.LaunchAddRmsNormQuantize_BF16(x.data_ptr(), r.data_ptr(), g.data_ptr(),
                                                        q.data_ptr() + 64, inv.data_ptr(),
                                                        s.data_ptr() + 128, 9, cols, EPS, st) == 0
        for t in (y, s, q):
            assert (t[:64] == 7).all() and (t[-64:] == 7).all()
        assert torch.equal(y[64:-64].view(9, cols), raw_ops.MusaAddRmsNorm(x, r, g, EPS).y)


def test_empty_and_refusals(kernel_lib):
    x, g = _rand((3, 8), BF16, 1), _rand((8,), BF16, 2)
    inv = torch.ones(3, 1, device="cuda")
    f = raw_ops.MusaAddRmsNorm(x[:0], x[:0], g)
    assert f.y.shape == (0, 8) and f.inv_rms.shape == (0, 1)
    d = raw_ops.MusaAddRmsNormGrad(x[:0], None, x[:0], inv[:0], g)
    assert d.dx.shape == (0, 8) and not d.dgamma.any()
    assert raw_ops.MusaAddRmsNormQuantize(x[:0], None, g).q.shape == (0, 8)
    assert raw_ops.MusaQuantizeRows(x[:, :0]).q.shape == (3, 0)
    for call in (lambda: raw_ops.MusaAddRmsNorm(x, x[:2], g),
                 lambda: raw_ops.MusaAddRmsNorm(x, x.half(), g),
                 lambda: raw_ops.MusaAddRmsNorm(x, x, g[:7]),
                 lambda: raw_ops.MusaAddRmsNorm(x.int(), x.int(), g.int()),
                 lambda: raw_ops.MusaAddRmsNorm(x.sum(), x.sum(), g),
                 lambda: raw_ops.MusaAddRmsNormGrad(x, x[:2], x, inv, g),
                 lambda: raw_ops.MusaAddRmsNormGrad(x, None, x, inv[:2], g),
                 lambda: raw_ops.MusaAddRmsNormGrad(x, None, x, inv.half(), g),
                 lambda: raw_ops.MusaAddRmsNormQuantize(x, x, None),
                 lambda: raw_ops.MusaAddRmsNormQuantize(x, x[:, :4], g),
                 lambda: raw_ops.MusaQuantizeRows(x.double()),
                 lambda: raw_ops.MusaQuantizeRows(x.cpu())):
        with pytest.raises(errors.InvalidArgumentError):
            call()
