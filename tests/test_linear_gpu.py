"""MusaMatMulBiasAct, its gradient and MusaQuantizedMatMulBiasAct on the GPU against
the formulas in 64 bits.

Tolerances.  With S = sum_k |a||b| of an element, an fp32 accumulator that adds the
products of 8 or more depths at a time, and may truncate (2^-23 of what it holds, at
most S), is off by (k / 8 + 16) * 2^-23 * S.  The activations have slopes below 1.2, and
their fp32 forms are good to 2^-19.  An output is rounded once: half a step, eps / 2.
The gradient's dz is rounded to T before its products: eps / 2 of S more."""
import threading

import pytest
import torch

from tensorflow_musa_extension_b200 import errors, raw_ops

pytestmark = pytest.mark.gpu

F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn
ACTS = sorted(raw_ops.ACTIVATIONS)
# Sizes of one line, around the tiles and the widths of vector accesses and boxes.
SIZES = [(1, 1, 1), (1, 128, 64), (2, 3, 5), (1, 1000, 4096), (7, 40, 2048), (16, 128, 128),
         (17, 129, 65), (64, 64, 64), (65, 200, 72), (100, 1030, 515), (128, 256, 192),
         (129, 127, 1000), (256, 512, 320), (257, 130, 8), (333, 2047, 1001), (512, 384, 4104),
         (1000, 72, 24), (3, 4099, 777)]


def _rand(shape, dtype, seed, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _act(z, act):
    if act == "Relu":
        return z.clamp(min=0)
    if act == "Sigmoid":
        return torch.sigmoid(z)
    if act == "Silu":
        return z * torch.sigmoid(z)
    if act == "Gelu":
        return z * 0.5 * torch.special.erfc(-z * 0.5 ** 0.5)
    return z


def _slope(z, act):
    """act'(z) from differentiating the formula."""
    z = z.clone().requires_grad_()
    with torch.enable_grad():
        return torch.autograd.grad(_act(z, act).sum(), z)[0]


def _sums(k):
    return (k / 8 + 16) * 2.0 ** -23


def _check(got, want, tol, what):
    assert got.shape == want.shape, what
    if not got.numel():
        return
    off = (got.double() - want).abs() - tol
    i = int(off.argmax())
    assert float(off.max()) <= 0, "%s: %r against %r, off by %g more than allowed" % (
        what, float(got.reshape(-1)[i]), float(want.reshape(-1)[i]), float(off.max()))


def _half(t):
    return torch.finfo(t).eps / 2


def _forward(a, b, bias, residual, act, ta, tb, dtype):
    """y, z and their tolerances."""
    a, b = a.double(), b.double()
    a, b = (a.mT if ta else a), (b.mT if tb else b)
    z, s = a @ b, a.abs() @ b.abs()
    if bias is not None:
        z = z + bias.double()
    # The accumulator, the fp32 additions behind it, a subnormal of T at most.
    off = _sums(a.shape[-1]) * s + 2.0 ** -22 * z.abs() + 2.0 ** -25
    h = _act(z, act)
    y = h if residual is None else h + residual.double()
    y_off = 1.2 * off + 2.0 ** -19 * h.abs() + 2.0 ** -23 * y.abs()
    return y, z, y_off + _half(dtype) * (y.abs() + y_off), off + _half(dtype) * (z.abs() + off)


@pytest.fixture(params=["by rule", "split", "pairs of 256", "pairs of 128"])
def form(request, kernel_lib):
    """Every form of the products on every size."""
    old = kernel_lib.MusaKernelsSetTuning(29, ["by rule", "split", "pairs of 256",
                                               "pairs of 128"].index(request.param))
    yield request.param
    kernel_lib.MusaKernelsSetTuning(29, old)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_forward(form, dtype, m, n, k):
    for i, (ta, tb) in enumerate(((False, False), (False, True), (True, False), (True, True))):
        act = ACTS[(m + n + i) % len(ACTS)]
        a = _rand((k, m) if ta else (m, k), dtype, 1)
        b = _rand((n, k) if tb else (k, n), dtype, 2, k ** -0.5)
        bias, res = _rand((n,), dtype, 3), _rand((m, n), dtype, 4)
        want, wz, tol, tz = _forward(a, b, bias, res, act, ta, tb, dtype)
        y, z = raw_ops.MusaMatMulBiasAct(a, b, bias, res, act, ta, tb, return_preactivation=True)
        _check(z, wz, tz, "z %s %s" % (ta, tb))
        _check(y, want, tol, "y %s %s %s" % (act, ta, tb))
        want, _, tol, _ = _forward(a, b, None, None, "Identity", ta, tb, dtype)
        y = raw_ops.MusaMatMulBiasAct(a, b, transpose_a=ta, transpose_b=tb)
        _check(y, want, tol, "plain %s %s" % (ta, tb))
    raw_ops.check_products()


def _backward(dy, a, b, z, act, ta, tb, dtype):
    """da, db, dbias and their tolerances."""
    a, b, dy = a.double(), b.double(), dy.double()
    oa, ob = (a.mT if ta else a), (b.mT if tb else b)
    slope = torch.ones_like(dy) if z is None else _slope(z.double(), act)
    dz = dy * slope
    # |slope| is good to 2^-19 of at most 1.2; dz is rounded to T, a subnormal at most.
    dz_off = 2.0 ** -19 * 1.2 * dy.abs()
    round_off = _half(dtype) * (dz.abs() + dz_off) + 2.0 ** -25 if act != "Identity" else 0 * dz
    out = []
    for x, y, off_x, flip in ((dz, ob.mT, dz_off + round_off, ta), (oa.mT, dz, None, tb)):
        want, s = x @ y, x.abs() @ y.abs()
        spread = off_x @ y.abs() if off_x is not None else x.abs() @ (dz_off + round_off)
        tol = spread + _sums(x.shape[-1]) * s + 2.0 ** -25
        tol = tol + _half(dtype) * (want.abs() + tol)
        out += [(want.mT, tol.mT) if flip else (want, tol)]
    want, s = dz.sum(0), dz.abs().sum(0)
    tol = dz_off.sum(0) + dy.shape[0] * 2.0 ** -24 * s + 2.0 ** -25
    return out + [(want, tol + _half(dtype) * (want.abs() + tol))]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_gradient(form, dtype, m, n, k):
    for i, (ta, tb) in enumerate(((False, False), (False, True), (True, False), (True, True))):
        act = ACTS[(m + n + i) % len(ACTS)]
        a = _rand((k, m) if ta else (m, k), dtype, 1)
        b = _rand((n, k) if tb else (k, n), dtype, 2, k ** -0.5)
        dy, z = _rand((m, n), dtype, 3), _rand((m, n), dtype, 4, 2.0)
        z = None if act == "Identity" else z
        got = raw_ops.MusaMatMulBiasActGrad(dy, a, b, z, act, ta, tb)
        wants = _backward(dy, a, b, z, act, ta, tb, dtype)
        for name, g, (want, tol) in zip(got._fields, got, wants):
            _check(g, want, tol, "%s %s %s %s" % (name, act, ta, tb))
    raw_ops.check_products()


@pytest.mark.parametrize("act", ACTS)
def test_gradient_against_differences(kernel_lib, act):
    """Central differences of the 64-bit forward, through the op's own preactivation (its
    rounding moves the slope by at most eps / 2 * |z| * 1.1)."""
    m, n, k, h = 5, 7, 6, 1e-5
    a, b = _rand((m, k), F16, 1), _rand((k, n), F16, 2, 0.5)
    bias, dy = _rand((n,), F16, 3), _rand((m, n), F16, 4)
    # Relu has no difference quotient at its bend.
    z = raw_ops.MusaMatMulBiasAct(a, b, bias, None, act, return_preactivation=True).preactivation
    assert float(z.abs().min()) > 1e-3
    got = raw_ops.MusaMatMulBiasActGrad(dy, a, b, z, act)

    def loss(a, b, bias):
        return float((_act(a @ b + bias, act) * dy.double()).sum())
    args = [a.double(), b.double(), bias.double()]
    z_off = 1.1 * _half(F16) * z.double().abs() * dy.double().abs()
    spread = (z_off @ b.double().abs().mT, a.double().abs().mT @ z_off, z_off.sum(0))
    tols = [t for _, t in _backward(dy, a, b, z, act, False, False, F16)]
    for i, name in enumerate(got._fields):
        want = torch.zeros_like(args[i])
        for j in range(args[i].numel()):
            ends = []
            for sign in (1, -1):
                moved = [t.clone() for t in args]
                moved[i].view(-1)[j] += sign * h
                ends.append(loss(*moved))
            want.view(-1)[j] = (ends[0] - ends[1]) / (2 * h)
        _check(got[i], want, tols[i] + spread[i] + 1e-7, name)


def _quantized(m, k, seed, std=1.0):
    return raw_ops.MusaQuantizeRows(_rand((m, k), BF16, seed, std))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_quantized(form, dtype, m, n, k):
    act = ACTS[(m + n) % len(ACTS)]
    a, sa = _quantized(m, k, 1)
    b, sb = _quantized(n, k, 2, k ** -0.5)
    bias, res = _rand((n,), dtype, 3), _rand((m, n), dtype, 4)
    fa, fb = a.double() * sa, b.double() * sb
    for bias, res, act in ((bias, res, act), (None, None, "Identity")):
        want, _, tol, _ = _forward(fa, fb.mT, bias, res, act, False, False, dtype)
        y = raw_ops.MusaQuantizedMatMulBiasAct(a, sa, b, sb, bias, res, act, dtype)
        assert y.dtype == dtype
        _check(y, want, tol, act)
    raw_ops.check_products()


@pytest.mark.parametrize("m,n,k", [(2049, 1300, 700), (700, 5000, 1100), (4100, 520, 2050),
                                   (300, 300, 20000)])
def test_larger_sizes(form, m, n, k):
    a, b = _rand((m, k), BF16, 1), _rand((k, n), BF16, 2, k ** -0.5)
    bias, res, dy = _rand((n,), BF16, 3), _rand((m, n), BF16, 4), _rand((m, n), BF16, 5)
    want, wz, tol, tz = _forward(a, b, bias, res, "Gelu", False, False, BF16)
    y, z = raw_ops.MusaMatMulBiasAct(a, b, bias, res, "Gelu", return_preactivation=True)
    _check(y, want, tol, "y")
    _check(z, wz, tz, "z")
    got = raw_ops.MusaMatMulBiasActGrad(dy, a, b, z, "Gelu")
    for name, g, (want, tol) in zip(got._fields, got,
                                    _backward(dy, a, b, z, "Gelu", False, False, BF16)):
        _check(g, want, tol, name)


def test_leading_axes_and_empty_sizes(kernel_lib):
    a, b = _rand((2, 3, 4, 24), BF16, 1), _rand((24, 10), BF16, 2)
    bias = _rand((10,), BF16, 3)
    y, z = raw_ops.MusaMatMulBiasAct(a, b, bias, None, "Relu", return_preactivation=True)
    flat = raw_ops.MusaMatMulBiasAct(a.view(24, 24), b, bias, None, "Relu")
    assert y.shape == (2, 3, 4, 10) and torch.equal(y.view(24, 10), flat)
    g = raw_ops.MusaMatMulBiasActGrad(y, a, b, z, "Relu")
    assert g.da.shape == a.shape and g.db.shape == b.shape and g.dbias.shape == bias.shape
    # No depth: the epilogue alone.
    res = _rand((4, 10), BF16, 4)
    y = raw_ops.MusaMatMulBiasAct(a.new_empty(4, 0), b[:0], bias, res, "Sigmoid")
    want = (torch.sigmoid(bias.double()) + res.double())
    _check(y, want, _half(BF16) * want.abs() + 2.0 ** -18, "k = 0")
    y = raw_ops.MusaMatMulBiasAct(a.new_empty(4, 0), b[:0])
    assert y.shape == (4, 10) and not y.any()
    # No rows, no columns.
    assert raw_ops.MusaMatMulBiasAct(a.new_empty(0, 24), b, bias).shape == (0, 10)
    assert raw_ops.MusaMatMulBiasAct(a, b[:, :0]).shape == (2, 3, 4, 0)
    g = raw_ops.MusaMatMulBiasActGrad(a.new_empty(0, 10), a.new_empty(0, 24), b)
    assert g.da.shape == (0, 24) and not g.db.any() and not g.dbias.any()
    g = raw_ops.MusaMatMulBiasActGrad(a.new_empty(4, 0), a.view(24, 24)[:4], b[:, :0])
    assert not g.da.any() and g.db.shape == (24, 0) and g.dbias.shape == (0,)
    g = raw_ops.MusaMatMulBiasActGrad(res, a.new_empty(4, 0), b[:0])
    assert g.da.shape == (4, 0) and g.db.shape == (0, 10)
    _check(g.dbias, res.double().sum(0), _half(BF16) * 10 + 0 * res.double().sum(0), "dbias")
    e = a.new_empty(3, 0).to(E4M3)
    y = raw_ops.MusaQuantizedMatMulBiasAct(e, _rand((3, 1), torch.float32, 1), e[:2],
                                           _rand((2, 1), torch.float32, 2))
    assert y.shape == (3, 2) and not y.any()


def _forms(t):
    """The values of t, stored otherwise: transposed, lines apart, off a 16-byte boundary,
    every second column, lines of an odd pitch."""
    rows, cols = t.shape
    yield t.t().contiguous().t()
    wide = t.new_zeros(rows, cols + 8)
    wide[:, :cols] = t
    yield wide[:, :cols]
    yield torch.cat((t.new_zeros(1), t.reshape(-1)))[1:].view(rows, cols)
    yield torch.stack((t, t), -1).flatten(1)[:, ::2]
    odd = t.new_zeros(rows, cols + 3)
    odd[:, :cols] = t
    yield odd[:, :cols]
    yield t[0].expand(rows, cols)


@pytest.mark.parametrize("m,n,k", [(5, 48, 72), (300, 264, 520)])
def test_strides_and_alignment(form, m, n, k):
    a, b = _rand((m, k), BF16, 1), _rand((k, n), BF16, 2, k ** -0.5)
    dy, z = _rand((m, n), BF16, 3), _rand((m, n), BF16, 4)
    bias, res = _rand((n,), BF16, 5), _rand((m, n), BF16, 6)

    def both(a, b, dy, z, bias, res):
        return (raw_ops.MusaMatMulBiasAct(a, b, bias, res, "Silu"),
                *raw_ops.MusaMatMulBiasActGrad(dy, a, b, z, "Silu"))
    for fa, fb, fd, fz, fr in zip(*(_forms(t) for t in (a, b, dy, z, res))):
        fbias = torch.stack((bias, bias), 1)[:, 0]
        want = both(*(t.contiguous() for t in (fa, fb, fd, fz, fbias, fr)))
        for got, w in zip(both(fa, fb, fd, fz, fbias, fr), want):
            assert torch.equal(got, w)
        a8, sa = raw_ops.MusaQuantizeRows(fa)
        b8, sb = raw_ops.MusaQuantizeRows(fb.t())
        want = raw_ops.MusaQuantizedMatMulBiasAct(a8, sa, b8, sb, fbias, fr, "Silu")
        for ga, gb in zip(_forms(a8.view(torch.uint8)), _forms(b8.view(torch.uint8))):
            if (ga != a8.view(torch.uint8)).any() or (gb != b8.view(torch.uint8)).any():
                continue                               # the expanded form holds other values
            y = raw_ops.MusaQuantizedMatMulBiasAct(ga.view(E4M3), sa, gb.view(E4M3), sb, fbias,
                                                   fr, "Silu")
            assert torch.equal(y, want)


def test_values_that_are_not_finite(form):
    """They stay in their row or column: no element reads its neighbours' masked lanes."""
    a, b = _rand((20, 30), BF16, 1), _rand((30, 50), BF16, 2)
    want = raw_ops.MusaMatMulBiasAct(a, b)
    a[3, 4], b[6, 7] = float("nan"), float("inf")
    got = raw_ops.MusaMatMulBiasAct(a, b, activation="Relu")
    assert got[3].isnan().all()
    rows = [i for i in range(20) if i != 3]
    cols = [j for j in range(50) if j != 7]
    assert torch.equal(got[rows][:, cols], want[rows][:, cols].clamp(min=0))
    column = got[rows, 7]
    assert ((column == float("inf")) | (column == 0) | column.isnan()).all()
    # What lies behind the last line of a factor is not read into a sum.
    store = torch.full((40, 64), float("nan"), dtype=BF16, device="cuda")
    store[:20, :30] = a.nan_to_num(0.0)
    assert raw_ops.MusaMatMulBiasAct(store[:20, :30], b.nan_to_num(0.0, 0.0, 0.0)).isfinite().all()


def test_outputs_stay_inside_their_tensors(form, kernel_lib):
    """Launchers on a part of a larger buffer: what surrounds it keeps its values."""
    lib = kernel_lib
    for m, n, k in ((3, 5, 7), (130, 257, 64), (300, 600, 128), (600, 1001, 72)):
        a, b = _rand((m, k), BF16, 1), _rand((n, k), BF16, 2)
        ys = [torch.full((m * n + 128,), 7.0, dtype=BF16, device="cuda") for _ in range(2)]
        ptr = [y.data_ptr() + 64 * 2 for y in ys]
        need = lib.MatMulWorkspaceBytes(2, a.data_ptr(), k, False, b.data_ptr(), k, True, m, n, k)
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
        st = torch.cuda.current_stream().cuda_stream
        assert lib.LaunchMatMulBiasAct(2, a.data_ptr(), k, False, b.data_ptr(), k, True, None,
                                       None, ptr[0], ptr[1], m, n, k, 0, ws.data_ptr(),
                                       ws.numel(), st) == 0
        want = raw_ops.MusaMatMulBiasAct(a, b, transpose_b=True).view(-1)
        for y in ys:
            assert torch.equal(y[64:-64], want) and (y[:64] == 7).all() and (y[-64:] == 7).all()


def _step(x, w, dy, bias):
    f = raw_ops.MusaMatMulBiasAct(x, w, bias, dy, "Gelu", return_preactivation=True)
    g = raw_ops.MusaMatMulBiasActGrad(dy, x, w, f.preactivation, "Gelu")
    q, s = raw_ops.MusaQuantizeRows(x)
    q2, s2 = raw_ops.MusaQuantizeRows(w.t().contiguous())
    return (*f, *g, raw_ops.MusaQuantizedMatMulBiasAct(q, s, q2, s2, bias, dy, "Relu"))


def _step_inputs(seed, odd):
    m, k, n = (259, 515, 333) if odd else (384, 512, 640)
    return (_rand((m, k), BF16, seed), _rand((k, n), BF16, seed + 1, k ** -0.5),
            _rand((m, n), BF16, seed + 2), _rand((n,), BF16, seed + 3))


@pytest.mark.parametrize("odd", [False, True])
def test_several_threads_and_streams(form, odd):
    inputs = [_step_inputs(10 * i, odd) for i in range(4)]
    want = [_step(*a) for a in inputs]
    torch.cuda.synchronize()
    got, failed = [None] * 4, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[i] = _step(*inputs[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:   # reported by the assertion below
            failed.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for a, b in zip(got, want):
        for u, v in zip(a, b):
            assert torch.equal(u, v)
    raw_ops.check_products()


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("odd", [False, True])
def test_graph_capture(monkeypatch, form, odd, native):
    """Two captured graphs replayed at once on streams of their own, on new inputs: the bits
    of the eager calls (each graph has its own scratch)."""
    if not native:
        monkeypatch.setattr(raw_ops, "_native", lambda: raw_ops._NoNativePath())
    inputs = [_step_inputs(30, odd), _step_inputs(40, odd)]
    graphs, outs = [], []
    for buffers in inputs:
        _step(*buffers)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_step(*buffers))
        graphs.append(graph)
    for round_ in range(3):
        for i, buffers in enumerate(inputs):
            for t, v in zip(buffers, _step_inputs(100 * round_ + i, odd)):
                t.copy_(v)
        torch.cuda.synchronize()
        for graph in graphs:
            with torch.cuda.stream(torch.cuda.Stream()):
                graph.replay()
        torch.cuda.synchronize()
        for buffers, out in zip(inputs, outs):
            for u, v in zip(out, _step(*buffers)):
                assert torch.equal(u, v)
    del graphs, graph


def test_native_and_general_path_agree(monkeypatch, kernel_lib):
    for odd in (False, True):
        args = _step_inputs(7, odd)
        got = _step(*args)
        with monkeypatch.context() as m:
            m.setattr(raw_ops, "_native", lambda: raw_ops._NoNativePath())
            want = _step(*args)
        for u, v in zip(got, want):
            assert u.dtype == v.dtype and torch.equal(u, v)


def test_host_buffers(kernel_lib):
    a, b, bias = (_rand(s, F16, i).cpu() for i, s in enumerate(((5, 8), (8, 3), (3,))))
    y = raw_ops.MusaMatMulBiasAct(a, b, bias, activation="Relu")
    assert not y.is_cuda
    want = raw_ops.MusaMatMulBiasAct(a.cuda(), b.cuda(), bias.cuda(), activation="Relu")
    assert torch.equal(y.cuda(), want)
    y = raw_ops.MusaMatMulBiasAct(a.numpy(), b.numpy(), bias.numpy(), activation="Relu")
    assert torch.equal(torch.from_numpy(y).cuda(), want)


def test_refusals(kernel_lib):
    a, b, v = _rand((4, 8), BF16, 1), _rand((8, 6), BF16, 2), _rand((6,), BF16, 3)
    y = _rand((4, 6), BF16, 4)
    q, s = raw_ops.MusaQuantizeRows(a)
    w, ws = raw_ops.MusaQuantizeRows(b.t().contiguous())
    calls = [
        lambda: raw_ops.MusaMatMulBiasAct(a.float(), b.float()),
        lambda: raw_ops.MusaMatMulBiasAct(a, b.half()),
        lambda: raw_ops.MusaMatMulBiasAct(a, b[:7]),
        lambda: raw_ops.MusaMatMulBiasAct(a, b, transpose_b=True),
        lambda: raw_ops.MusaMatMulBiasAct(a[0], b),
        lambda: raw_ops.MusaMatMulBiasAct(a[None], b, transpose_a=True),
        lambda: raw_ops.MusaMatMulBiasAct(a, b[None]),
        lambda: raw_ops.MusaMatMulBiasAct(a, b, v[:5]),
        lambda: raw_ops.MusaMatMulBiasAct(a, b, v[None]),
        lambda: raw_ops.MusaMatMulBiasAct(a, b, v.half()),
        lambda: raw_ops.MusaMatMulBiasAct(a, b, v, v),
        lambda: raw_ops.MusaMatMulBiasAct(a, b, v, y.float()),
        lambda: raw_ops.MusaMatMulBiasAct(a, b, activation="Swish"),
        lambda: raw_ops.MusaMatMulBiasActGrad(y[:3], a, b),
        lambda: raw_ops.MusaMatMulBiasActGrad(y, a, b, None, "Relu"),
        lambda: raw_ops.MusaMatMulBiasActGrad(y, a, b, y[:, :5], "Relu"),
        lambda: raw_ops.MusaMatMulBiasActGrad(y.half(), a, b),
        lambda: raw_ops.MusaQuantizedMatMulBiasAct(a, s, b, s),
        lambda: raw_ops.MusaQuantizedMatMulBiasAct(q, s[:3], w, ws),
        lambda: raw_ops.MusaQuantizedMatMulBiasAct(q, s.half(), w, ws),
        lambda: raw_ops.MusaQuantizedMatMulBiasAct(q, s, w[:, :7], ws),
        lambda: raw_ops.MusaQuantizedMatMulBiasAct(q, s, w, ws, out_dtype=torch.float32),
        lambda: raw_ops.MusaQuantizedMatMulBiasAct(q, s, w, ws, v.half()),
        lambda: raw_ops.MusaQuantizedMatMulBiasAct(q.view(torch.uint8), s, w, ws),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(errors.InvalidArgumentError):
            call()
            pytest.fail("call %d was not refused" % i)
