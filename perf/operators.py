"""Performance cases of the transformer-block operators: the residual addition
with its RMS norm (forward, gradient, 8-bit output), and the matrix product with
bias, activation and residual in its epilogue (forward, gradient, 8-bit inputs).

`run` computes an operator in elementary torch operations in 32 bits, or, with
`own` set, through the framework's ops.  Both take the tensors of `prepare`.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_EPSILON = 1e-5
_E4M3_MAX = 448.0
_SCALE_MIN = 2.0 ** -126


def listed():
    return [
        # One decoding step of four sequences: the call is all latency.
        dict(name="norm-decode", op="norm", rows=4, cols=4096, dtype="bf16"),
        # A packed batch of sequences whose width is no multiple of a vector access.
        dict(name="norm-ragged", op="norm", rows=6001, cols=2999, dtype="f16"),
        # Backward of a training step, 16384 tokens: HBM-bound.
        dict(name="norm-grad-train", op="norm_grad", rows=16384, cols=4096, dtype="bf16"),
        # Serving: the norm in front of an 8-bit product, one token.
        dict(name="norm-quantize-decode", op="norm_quantize", rows=1, cols=8192, dtype="bf16"),
        # Serving: the same over a prefill of 8192 tokens.
        dict(name="norm-quantize-prefill", op="norm_quantize", rows=8192, cols=8192,
             dtype="bf16"),
        # The up-projection of one decoding token: the weights are read once.
        dict(name="linear-decode", op="linear", m=1, k=4096, n=16384, dtype="bf16",
             act="Silu", bias=False, residual=False, save=False, transpose_b=True),
        # Odd in every dimension, everything in the epilogue, output before the
        # activation kept for the backward pass.
        dict(name="linear-odd", op="linear", m=333, k=1001, n=2047, dtype="f16",
             act="Gelu", bias=True, residual=True, save=True, transpose_b=False),
        # The up-projection of a training step.
        dict(name="linear-train", op="linear", m=8192, k=4096, n=16384, dtype="bf16",
             act="Gelu", bias=True, residual=False, save=True, transpose_b=False),
        # Backward of a narrow layer with odd sizes.
        dict(name="linear-grad-odd", op="linear_grad", m=1500, k=515, n=1030, dtype="f16",
             act="Relu", transpose_b=False),
        # Backward of a training step: two products and a column sum.
        dict(name="linear-grad-train", op="linear_grad", m=8192, k=4096, n=8192, dtype="bf16",
             act="Gelu", transpose_b=False),
        # Decoding of 16 sequences with 8-bit weights, the residual in the epilogue.
        dict(name="linear-8bit-decode", op="linear_8bit", m=16, k=8192, n=8192, dtype="bf16",
             act="Identity", bias=False, residual=True),
        # Prefill with 8-bit inputs on both sides.
        dict(name="linear-8bit-prefill", op="linear_8bit", m=8192, k=8192, n=8192,
             dtype="bf16", act="Silu", bias=True, residual=False),
    ]


def _log_size(rng, low, high):
    """A size spread over the logarithm of the range; every other one a multiple of 64."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.5 and n >= 64:
        n = n // 64 * 64
    return n


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "norm_quantize", "linear", "linear_grad",
                     "linear_8bit"])
    if op.startswith("norm"):
        cols = _log_size(rng, 64, 16384)
        rows = min(_log_size(rng, 1, 16384), (1 << 26) // cols)
        return dict(op=op, rows=rows, cols=cols, dtype=rng.choice(["bf16", "f16", "f32"]))
    limit = 8192 * 4096 * (8192 if op == "linear_grad" else 16384)
    while True:
        m = _log_size(rng, 1, 8192)
        k = _log_size(rng, 64, 16384)
        n = _log_size(rng, 64, 16384)
        if m * k * n <= limit:
            break
    act = rng.choice(["Identity", "Relu", "Sigmoid", "Silu", "Gelu"])
    dtype = rng.choice(["bf16", "f16"])
    case = dict(op=op, m=m, k=k, n=n, dtype=dtype, act=act)
    if op == "linear_8bit":
        case.update(k=max(k // 16, 4) * 16, bias=rng.random() < 0.5, residual=rng.random() < 0.5)
    else:
        case.update(transpose_b=rng.random() < 0.5)
    if op == "linear":
        case.update(bias=rng.random() < 0.5, residual=rng.random() < 0.5,
                    save=rng.random() < 0.5)
    return case


# ------------------------------------------------------------------ inputs --

def _quantized_rows(x):
    """e4m3 rows and their fp32 scales."""
    amax = x.abs().amax(dim=-1, keepdim=True)
    scale = (amax / _E4M3_MAX).clamp(min=_SCALE_MIN)
    return (x / scale).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = _DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=t):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    s = {"case": case}
    if case["op"].startswith("norm"):
        rows, cols = case["rows"], case["cols"]
        # A residual stream: wider than the branch added to it, some channels far out.
        spread = torch.rand(cols, generator=g, device="cuda").pow(-0.3)
        stream = torch.randn(rows, cols, generator=g, device="cuda") * spread * 3.0
        s["gamma"] = (1.0 + 0.2 * torch.randn(cols, generator=g, device="cuda")).to(t)
        if case["op"] == "norm_grad":
            s["sum"] = stream.to(t)
            mean = s["sum"].double().square().mean(dim=-1, keepdim=True)
            s["inv_rms"] = (mean + _EPSILON).rsqrt().float()
            s["dy"] = normal(rows, cols, std=1e-2)
            s["dsum"] = normal(rows, cols, std=1e-2)
        else:
            s["residual"] = stream.to(t)
            s["x"] = normal(rows, cols)
        return s
    m, k, n = case["m"], case["k"], case["n"]
    std = 1.0 / math.sqrt(k)
    if case["op"] == "linear_8bit":
        # Activations with far-out channels, weights quantised once per output row.
        spread = torch.rand(k, generator=g, device="cuda").pow(-0.3)
        s["a"], s["a_scale"] = _quantized_rows(
            torch.randn(m, k, generator=g, device="cuda") * spread)
        s["b"], s["b_scale"] = _quantized_rows(
            torch.randn(n, k, generator=g, device="cuda") * std)
    else:
        s["a"] = normal(m, k)
        s["b"] = normal(n, k, std=std) if case["transpose_b"] else normal(k, n, std=std)
    if case["op"] == "linear_grad":
        s["dy"] = normal(m, n, std=1e-2)
        s["z"] = None if case["act"] == "Identity" else normal(m, n)
    else:
        s["bias"] = normal(n, std=0.1) if case["bias"] else None
        s["residual"] = normal(m, n) if case["residual"] else None
    return s


# ------------------------------------------------------------- plain forms --

def _plain_activation(z, act):
    if act == "Relu":
        return z.clamp(min=0)
    if act == "Sigmoid":
        return 1 / (1 + torch.exp(-z))
    if act == "Silu":
        return z / (1 + torch.exp(-z))
    if act == "Gelu":
        return z * 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
    return z


def _plain_activation_grad(z, act):
    if act == "Relu":
        return (z > 0).float()
    if act == "Gelu":
        density = torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * density
    p = 1 / (1 + torch.exp(-z))
    if act == "Sigmoid":
        return p * (1 - p)
    return p * (1 + z * (1 - p))


def _plain_norm(s):
    total = s["x"].float() + s["residual"].float()
    inv = torch.rsqrt(total.square().mean(dim=-1, keepdim=True) + _EPSILON)
    return total, inv, total * inv * s["gamma"].float()


def _plain_norm_grad(s):
    x, inv, dy = s["sum"].float(), s["inv_rms"], s["dy"].float()
    hat = x * inv
    g = dy * s["gamma"].float()
    dx = s["dsum"].float() + inv * (g - hat * (g * hat).mean(dim=-1, keepdim=True))
    # A sum over all rows: in 64 bits.
    dgamma = (dy * hat).sum(dim=0, dtype=torch.float64)
    return dx, dgamma


def _plain_linear(s, product):
    c = s["case"]
    z = product
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _plain_activation(z, c["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y, z


def _plain_linear_grad(s):
    c = s["case"]
    a, b = s["a"].float(), s["b"].float()
    dz = s["dy"].float()
    if c["act"] != "Identity":
        dz = dz * _plain_activation_grad(s["z"].float(), c["act"])
    da = dz @ (b if c["transpose_b"] else b.T)
    db = dz.T @ a if c["transpose_b"] else a.T @ dz
    return da, db, dz.sum(dim=0, dtype=torch.float64)


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_plain(s):
    c = s["case"]
    t = _DTYPES[c["dtype"]]
    if c["op"] == "norm":
        total, inv, y = _plain_norm(s)
        return {"y": y.to(t), "sum": total.to(t), "inv_rms": inv}
    if c["op"] == "norm_quantize":
        total, _, y = _plain_norm(s)
        q, scale = _quantized_rows(y)
        return {"q": q, "scale": scale, "sum": total.to(t)}
    if c["op"] == "norm_grad":
        dx, dgamma = _plain_norm_grad(s)
        return {"dx": dx.to(t), "dgamma": dgamma.to(t)}
    if c["op"] == "linear":
        b = s["b"].float()
        y, z = _plain_linear(s, s["a"].float() @ (b.T if c["transpose_b"] else b))
        return {"y": y.to(t), "z": z.to(t)} if c["save"] else {"y": y.to(t)}
    if c["op"] == "linear_8bit":
        product = s["a"].float() @ s["b"].float().T
        y, _ = _plain_linear(s, product * s["a_scale"] * s["b_scale"].T)
        return {"y": y.to(t)}
    da, db, dbias = _plain_linear_grad(s)
    return {"da": da.to(t), "db": db.to(t), "dbias": dbias.to(t)}


# -------------------------------------------------------- the framework's ops --

def _run_own(s):
    from tensorflow_musa_extension_b200 import raw_ops
    c = s["case"]
    if c["op"] == "norm":
        out = raw_ops.MusaAddRmsNorm(s["x"], s["residual"], s["gamma"], epsilon=_EPSILON)
        return {"y": out.y, "sum": out.sum, "inv_rms": out.inv_rms}
    if c["op"] == "norm_quantize":
        out = raw_ops.MusaAddRmsNormQuantize(s["x"], s["residual"], s["gamma"],
                                             epsilon=_EPSILON)
        return {"q": out.q, "scale": out.scale, "sum": out.sum}
    if c["op"] == "norm_grad":
        out = raw_ops.MusaAddRmsNormGrad(s["dy"], s["dsum"], s["sum"], s["inv_rms"],
                                         s["gamma"])
        return {"dx": out.dx, "dgamma": out.dgamma}
    if c["op"] == "linear":
        out = raw_ops.MusaMatMulBiasAct(
            s["a"], s["b"], bias=s["bias"], residual=s["residual"], activation=c["act"],
            transpose_b=c["transpose_b"], return_preactivation=c["save"])
        return {"y": out.y, "z": out.preactivation} if c["save"] else {"y": out}
    if c["op"] == "linear_8bit":
        y = raw_ops.MusaQuantizedMatMulBiasAct(
            s["a"], s["a_scale"], s["b"], s["b_scale"], bias=s["bias"],
            residual=s["residual"], activation=c["act"], out_dtype=_DTYPES[c["dtype"]])
        return {"y": y}
    out = raw_ops.MusaMatMulBiasActGrad(s["dy"], s["a"], s["b"], preactivation=s["z"],
                                        activation=c["act"], transpose_b=c["transpose_b"])
    return {"da": out.da, "db": out.db, "dbias": out.dbias}


# ------------------------------------------------------ work and exact values --

def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"].startswith("norm"):
        rows, cols = case["rows"], case["cols"]
        e = rows * cols
        if case["op"] == "norm":          # x, residual -> y, sum; gamma; inv_rms
            return {"bytes": 4 * size * e + size * cols + 4 * rows, "flops": 5 * e}
        if case["op"] == "norm_quantize":  # x, residual -> sum, q; gamma; scale
            return {"bytes": (3 * size + 1) * e + size * cols + 4 * rows, "flops": 7 * e}
        # dy, dsum, sum -> dx; gamma, inv_rms; dgamma
        return {"bytes": 4 * size * e + 2 * size * cols + 4 * rows, "flops": 10 * e}
    m, k, n = case["m"], case["k"], case["n"]
    if case["op"] == "linear":
        out = 1 + case["residual"] + case["save"]
        return {"bytes": size * (m * k + k * n + out * m * n + case["bias"] * n),
                "flops": 2 * m * n * k}
    if case["op"] == "linear_8bit":
        out = 1 + case["residual"]
        return {"bytes": m * k + k * n + 4 * (m + n) + size * (out * m * n + case["bias"] * n),
                "flops": 2 * m * n * k}
    saved = 1 if case["act"] == "Identity" else 2
    return {"bytes": size * (saved * m * n + 2 * m * k + 2 * k * n + n),
            "flops": 4 * m * n * k}


def exact(case, seed):
    """The operators' definitions in 64 bits."""
    s = {key: (v.double() if isinstance(v, torch.Tensor) else v)
         for key, v in prepare(case, seed).items()}
    op = case["op"]
    if op in ("norm", "norm_quantize"):
        h = s["x"] + s["residual"]
        rms = ((h * h).sum(-1, keepdim=True) / h.shape[-1] + _EPSILON).sqrt()
        y = h / rms * s["gamma"]
        if op == "norm":
            return {"y": y, "sum": h, "inv_rms": 1 / rms}
        step = torch.clamp(y.abs().max(-1, keepdim=True).values / _E4M3_MAX, min=_SCALE_MIN)
        return {"q": y / step, "scale": step, "sum": h}
    if op == "norm_grad":
        n = s["sum"].shape[-1]
        u = s["dy"] * s["gamma"]
        along = (u * s["sum"]).sum(-1, keepdim=True)
        dx = s["dsum"] + u * s["inv_rms"] - s["sum"] * along * s["inv_rms"] ** 3 / n
        return {"dx": dx, "dgamma": torch.einsum("rc,rc,rk->c", s["dy"], s["sum"],
                                                 s["inv_rms"])}
    act = case["act"]

    def cdf(v):
        return 0.5 * torch.special.erfc(-v / math.sqrt(2.0))

    if op == "linear_grad":
        d = s["dy"]
        if act != "Identity":
            z = s["z"]
            p = torch.sigmoid(z)
            slope = {"Relu": lambda: torch.where(z > 0, 1.0, 0.0),
                     "Sigmoid": lambda: p - p * p,
                     "Silu": lambda: p + z * p - z * p * p,
                     "Gelu": lambda: cdf(z) + z * torch.exp(z * z / -2) / (2 * math.pi) ** 0.5}
            d = d * slope[act]()
        if case["transpose_b"]:
            return {"da": torch.matmul(d, s["b"]), "db": torch.matmul(d.mT, s["a"]),
                    "dbias": d.sum(0)}
        return {"da": torch.matmul(d, s["b"].mT), "db": torch.matmul(s["a"].mT, d),
                "dbias": d.sum(0)}
    if op == "linear_8bit":
        z = torch.matmul(s["a"] * s["a_scale"], (s["b"] * s["b_scale"]).mT)
    else:
        z = torch.matmul(s["a"], s["b"].mT if case["transpose_b"] else s["b"])
    if s["bias"] is not None:
        z = z + s["bias"]
    y = {"Identity": lambda: z, "Relu": lambda: torch.where(z > 0, z, 0.0 * z),
         "Sigmoid": lambda: torch.sigmoid(z), "Silu": lambda: z * torch.sigmoid(z),
         "Gelu": lambda: z * cdf(z)}[act]()
    if s["residual"] is not None:
        y = y + s["residual"]
    return {"y": y, "z": z} if case.get("save") else {"y": y}
