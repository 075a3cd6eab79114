"""The layers of a feed-forward block as cases that can be timed and compared.

Four passes, each in a plain form (elementary torch operations) and through
this package's kernel-level calls:

  linear            y = act(x . w + bias) + residual; optionally z = x . w + bias
  linear_grad       dz = dy * act'(z), dbias = sum over rows of dz,
                    dw = x^T . dz, dx = (dz . w^T) * act'(z of the layer
                    before) + residual
  layer_norm        y = (x - mean) * rstd * gamma + beta, with mean and rstd
  layer_norm_grad   dx (+ residual), dgamma, dbeta

x is [m][k], w is [k][n], row-major, as hexir.linear has them.  dz is an
output of its own and is held in the inputs' type: dw, dx and dbias are
products and sums of dz as it is stored.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32,
          "f64": torch.float64}


def linear(name, m, n, k, dtype, act, **more):
    return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "dtype": dtype,
            "act": act, "bias": True, "residual": False, "preact": False,
            "pad": 0, **more}


def linear_grad(name, m, n, k, dtype, act, **more):
    return {"name": name, "op": "linear_grad", "m": m, "n": n, "k": k,
            "dtype": dtype, "act": act, "prev_act": "none", "residual": False,
            "pad": 0, **more}


def layer_norm(name, rows, cols, dtype, **more):
    return {"name": name, "op": "layer_norm", "rows": rows, "cols": cols,
            "dtype": dtype, "pad": 0, **more}


def layer_norm_grad(name, rows, cols, dtype, **more):
    return {"name": name, "op": "layer_norm_grad", "rows": rows, "cols": cols,
            "dtype": dtype, "residual": False, "pad": 0, **more}


def listed():
    return [
        # Answering with one sequence: one token's output projection, added
        # to the residual stream.
        linear("linear-token", 1, 8192, 8192, "bf16", "none", residual=True),
        # Answering sixteen sequences at once: the up projection.
        linear("linear-tokens16", 16, 8192, 2048, "f16", "gelu"),
        # One training sequence's up projection; z is kept for the gradient.
        linear("linear-up", 2048, 8192, 2048, "bf16", "gelu", preact=True),
        # A large batch through a square projection with the residual add.
        linear("linear-large", 8192, 8192, 8192, "bf16", "none", residual=True),
        # Sizes without any alignment: rows that start on odd elements.
        linear("linear-odd", 777, 1001, 1537, "f16", "swish", residual=True),
        # The gradient of the up projection.
        linear_grad("linear-grad-up", 2048, 8192, 2048, "bf16", "gelu"),
        # A packed batch of ragged length: rows inside wider buffers, the
        # activation before this layer and the residual's gradient folded in.
        linear_grad("linear-grad-ragged", 1237, 1000, 520, "f16", "swish",
                    prev_act="gelu", residual=True, pad=24),
        # One token's norm.
        layer_norm("norm-token", 1, 8192, "bf16"),
        # A long prompt's norm.
        layer_norm("norm-large", 16384, 8192, "bf16"),
        # f64 rows of odd length, as the f64 programs have them.
        layer_norm("norm-odd", 4099, 1025, "f64"),
        # A training batch's norm with the residual branch's gradient.
        layer_norm_grad("norm-grad-large", 16384, 4096, "bf16", residual=True),
        # f32 rows of odd length.
        layer_norm_grad("norm-grad-odd", 2047, 2049, "f32"),
    ]


def spread(rng, low, high):
    """A whole number from low to high, even over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low),
                                                         math.log(high + 1))))))


def width(rng, low, high):
    """A row length: mostly a multiple of 8, one in four any number."""
    v = spread(rng, low, high)
    return v if rng.random() < 0.25 else max(8, v // 8 * 8)


def draw(rng):
    op = rng.choice(["linear", "linear", "linear_grad", "layer_norm",
                     "layer_norm_grad"])
    pad = rng.choice([0, 0, 8, 24, 5])
    acts = ["none", "relu", "gelu", "swish", "tanh", "sigmoid", "leaky_relu",
            "elu", "mish"]
    if op == "linear":
        m = spread(rng, 1, 64) if rng.random() < 0.4 else spread(rng, 65, 8192)
        return {"op": op, "m": m, "n": width(rng, 256, 8192),
                "k": width(rng, 256, 8192), "dtype": rng.choice(["bf16", "f16"]),
                "act": rng.choice(acts), "bias": rng.random() < 0.7,
                "residual": rng.random() < 0.5, "preact": rng.random() < 0.3,
                "pad": pad}
    if op == "linear_grad":
        return {"op": op, "m": spread(rng, 128, 4096), "n": width(rng, 256, 8192),
                "k": width(rng, 256, 8192), "dtype": rng.choice(["bf16", "f16"]),
                "act": rng.choice(acts), "prev_act": rng.choice(["none"] + acts),
                "residual": rng.random() < 0.5, "pad": pad}
    cols = width(rng, 64, 16384)
    dtype = rng.choice(["bf16", "f16", "f32", "f64"])
    rows = spread(rng, 1, 2 ** 27 // cols // DTYPES[dtype].itemsize)
    case = {"op": op, "rows": rows, "cols": cols, "dtype": dtype, "pad": pad}
    if op == "layer_norm_grad":
        case["residual"] = rng.random() < 0.5
    return case


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    pad = case["pad"]
    wide = torch.float64 if dtype == torch.float64 else torch.float32

    def empty(rows, cols, of=dtype):
        return torch.empty(rows, cols + pad, device="cuda", dtype=of)[:, :cols]

    def normal(rows, cols, std=1.0, mean=0.0):
        t = empty(rows, cols)
        t.copy_(torch.randn(rows, cols, generator=gen, device="cuda",
                            dtype=torch.float32).mul_(std).add_(mean))
        return t

    def vector(size, std, mean=0.0):
        return normal(1, size, std, mean).reshape(-1).clone()

    s = {"case": case, "out": {}}
    out = s["out"]
    if case["op"] in ("linear", "linear_grad"):
        m, n, k = case["m"], case["n"], case["k"]
        s["x"] = normal(m, k)
        s["w"] = normal(k, n, 1.0 / math.sqrt(k))
    if case["op"] == "linear":
        s["bias"] = vector(n, 0.1) if case["bias"] else None
        s["residual"] = normal(m, n) if case["residual"] else None
        out["y"] = empty(m, n)
        out["z"] = empty(m, n) if case["preact"] else None
    elif case["op"] == "linear_grad":
        # Gradients of a mean over m tokens, scaled up as mixed precision
        # training scales its loss.
        s["dy"] = normal(m, n, 0.1)
        s["z"] = normal(m, n) if case["act"] != "none" else None
        s["prev_z"] = normal(m, k) if case["prev_act"] != "none" else None
        s["residual"] = normal(m, k, 0.1) if case["residual"] else None
        out["dz"] = empty(m, n) if case["act"] != "none" else None
        out["dx"], out["dw"] = empty(m, k), empty(k, n)
        out["dbias"] = torch.empty(n, device="cuda", dtype=dtype)
        # The size grad_workspace_bytes(n, dtype) asks for.
        out["workspace"] = torch.empty(640 * n * 4, device="cuda", dtype=torch.uint8)
    else:
        rows, cols = case["rows"], case["cols"]
        s["eps"] = 1e-5
        s["x"] = normal(rows, cols, 2.0, 0.5)
        s["gamma"] = vector(cols, 0.1, 1.0)
        out["mean"] = torch.empty(rows, device="cuda", dtype=wide)
        out["rstd"] = torch.empty(rows, device="cuda", dtype=wide)
        if case["op"] == "layer_norm":
            s["beta"] = vector(cols, 0.1)
            out["y"] = empty(rows, cols)
        else:
            x = s["x"].double()
            s["mean"] = x.mean(1).to(wide)
            s["rstd"] = (x.var(1, unbiased=False) + s["eps"]).rsqrt().to(wide)
            del x
            s["dy"] = normal(rows, cols, 0.1)
            s["residual"] = normal(rows, cols, 0.1) if case["residual"] else None
            out["dx"] = empty(rows, cols)
            out["dgamma"] = torch.empty(cols, device="cuda", dtype=dtype)
            out["dbeta"] = torch.empty(cols, device="cuda", dtype=dtype)
            out["workspace"] = torch.empty(640 * cols * wide.itemsize,
                                           device="cuda", dtype=torch.uint8)
    return s


# ------------------------------------------------------------- plain form


def act_plain(act, z):
    if act == "none":
        return z
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "leaky_relu":
        return torch.where(z > 0, z, 0.01 * z)
    if act == "elu":
        return torch.where(z > 0, z, torch.expm1(z))
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    if act == "tanh":
        return torch.tanh(z)
    if act == "gelu":
        return 0.5 * z * torch.erfc(-z * math.sqrt(0.5))
    if act == "swish":
        return z / (1 + torch.exp(-z))
    return z * torch.tanh(torch.log1p(torch.exp(-z.abs())) + z.clamp(min=0))  # mish


def slope_plain(act, z):
    one = torch.ones_like(z)
    if act == "none":
        return one
    if act == "relu":
        return torch.where(z > 0, one, 0 * one)
    if act == "leaky_relu":
        return torch.where(z > 0, one, 0.01 * one)
    if act == "elu":
        return torch.where(z > 0, one, torch.exp(z))
    if act == "tanh":
        t = torch.tanh(z)
        return 1 - t * t
    if act == "gelu":
        return (0.5 * torch.erfc(-z * math.sqrt(0.5))
                + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi))
    s = 1 / (1 + torch.exp(-z))
    if act == "sigmoid":
        return s * (1 - s)
    if act == "swish":
        return s * (1 + z * (1 - s))
    t = torch.tanh(torch.log1p(torch.exp(-z.abs())) + z.clamp(min=0))  # mish
    return t + z * (1 - t * t) * s


def run_plain(s):
    case = s["case"]
    dtype = DTYPES[case["dtype"]]
    wide = torch.float64 if dtype == torch.float64 else torch.float32

    def up(t):
        return t.to(wide)

    if case["op"] == "linear":
        z = up(s["x"]) @ up(s["w"])
        if s["bias"] is not None:
            z = z + up(s["bias"])
        y = act_plain(case["act"], z)
        if s["residual"] is not None:
            y = y + up(s["residual"])
        return (y.to(dtype), z.to(dtype)) if case["preact"] else y.to(dtype)
    if case["op"] == "linear_grad":
        dz = s["dy"]
        if case["act"] != "none":
            dz = (up(dz) * slope_plain(case["act"], up(s["z"]))).to(dtype)
        wide_dz = up(dz)
        dbias = wide_dz.sum(0)
        dw = up(s["x"]).t() @ wide_dz
        dx = wide_dz @ up(s["w"]).t()
        if case["prev_act"] != "none":
            dx = dx * slope_plain(case["prev_act"], up(s["prev_z"]))
        if s["residual"] is not None:
            dx = dx + up(s["residual"])
        grads = (dx.to(dtype), dw.to(dtype), dbias.to(dtype))
        return grads + (dz,) if case["act"] != "none" else grads
    x, gamma = up(s["x"]), up(s["gamma"])
    if case["op"] == "layer_norm":
        mean = x.sum(1) / case["cols"]
        x = x - mean[:, None]
        rstd = 1 / torch.sqrt((x * x).sum(1) / case["cols"] + s["eps"])
        return ((x * rstd[:, None] * gamma + up(s["beta"])).to(dtype), mean, rstd)
    dy = up(s["dy"])
    xhat = (x - s["mean"][:, None]) * s["rstd"][:, None]
    g = dy * gamma
    a = g.sum(1) / case["cols"]
    b = (g * xhat).sum(1) / case["cols"]
    dx = (g - a[:, None] - xhat * b[:, None]) * s["rstd"][:, None]
    if s["residual"] is not None:
        dx = dx + up(s["residual"])
    return dx.to(dtype), (dy * xhat).sum(0).to(dtype), dy.sum(0).to(dtype)


# ------------------------------------------------------ this package's calls


def at(t):
    return 0 if t is None else t.data_ptr()


def ld(t):
    return 0 if t is None else t.stride(0)


def run_own(s):
    import hexir_b200 as hx

    case, out = s["case"], s["out"]
    dtype = case["dtype"]
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        x, w, residual, y, z = s["x"], s["w"], s["residual"], out["y"], out["z"]
        hx.cuda_linear(0, at(x), at(w), at(y), m, n, k, dtype, case["act"],
                       bias=at(s["bias"]), residual=at(residual), preact=at(z),
                       ldx=ld(x), ldw=ld(w), ldy=ld(y), ldr=ld(residual),
                       ldp=ld(z), stream=stream)
        return (y, z) if case["preact"] else y
    if case["op"] == "linear_grad":
        m, n, k = case["m"], case["n"], case["k"]
        x, w, dy, z, prev_z = s["x"], s["w"], s["dy"], s["z"], s["prev_z"]
        residual, dz, dx, dw = s["residual"], out["dz"], out["dx"], out["dw"]
        hx.cuda_linear_output_grad(0, at(dy), m, n, dtype, case["act"],
                                   preact=at(z), dz=at(dz), dbias=at(out["dbias"]),
                                   workspace=at(out["workspace"]),
                                   workspace_bytes=out["workspace"].numel(),
                                   lddy=ld(dy), ldp=ld(z), lddz=ld(dz),
                                   stream=stream)
        if dz is None:
            dz = dy
        hx.cuda_linear_weight_grad(0, at(x), at(dz), at(dw), m, n, k, dtype,
                                   ldx=ld(x), lddz=ld(dz), lddw=ld(dw),
                                   stream=stream)
        hx.cuda_linear_input_grad(0, at(dz), at(w), at(dx), m, n, k, dtype,
                                  case["prev_act"], preact=at(prev_z),
                                  residual=at(residual), lddz=ld(dz), ldw=ld(w),
                                  lddx=ld(dx), ldp=ld(prev_z), ldr=ld(residual),
                                  stream=stream)
        grads = (dx, dw, out["dbias"])
        return grads + (dz,) if case["act"] != "none" else grads
    rows, cols = case["rows"], case["cols"]
    x, mean, rstd = s["x"], out["mean"], out["rstd"]
    if case["op"] == "layer_norm":
        y = out["y"]
        hx.cuda_layer_norm(0, at(x), at(y), rows, cols, dtype,
                           gamma=at(s["gamma"]), beta=at(s["beta"]),
                           mean=at(mean), rstd=at(rstd), eps=s["eps"], ldx=ld(x),
                           ldy=ld(y), stream=stream)
        return y, mean, rstd
    dy, dx, residual = s["dy"], out["dx"], s["residual"]
    hx.cuda_layer_norm_grad(0, at(dy), at(x), at(s["mean"]), at(s["rstd"]), at(dx),
                            rows, cols, dtype, gamma=at(s["gamma"]),
                            dgamma=at(out["dgamma"]), dbeta=at(out["dbeta"]),
                            residual=at(residual),
                            workspace=at(out["workspace"]),
                            workspace_bytes=out["workspace"].numel(), lddy=ld(dy),
                            ldx=ld(x), lddx=ld(dx), ldr=ld(residual),
                            stream=stream)
    return dx, out["dgamma"], out["dbeta"]


def run(state):
    return run_own(state) if own else run_plain(state)


# ------------------------------------------------------------ work and truth


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    if case["op"] in ("linear", "linear_grad"):
        m, n, k = case["m"], case["n"], case["k"]
        if case["op"] == "linear":
            count = (m * k + k * n + m * n * (1 + case["residual"] + case["preact"])
                     + n * case["bias"])
            return {"bytes": size * count, "flops": 2 * m * n * k}
        count = (m * n * (3 if case["act"] != "none" else 1) + 2 * k * n
                 + m * k * (2 + (case["prev_act"] != "none") + case["residual"]) + n)
        return {"bytes": size * count, "flops": 4 * m * n * k}
    rows, cols = case["rows"], case["cols"]
    stats = 2 * rows * max(size, 4)
    if case["op"] == "layer_norm":
        return {"bytes": size * (2 * rows * cols + 2 * cols) + stats,
                "flops": 8 * rows * cols}
    return {"bytes": size * (rows * cols * (3 + case["residual"]) + 3 * cols) + stats,
            "flops": 14 * rows * cols}


def normal_cdf(z):
    return torch.special.erfc(z / -(2.0 ** 0.5)) / 2


def act_exact(act, z):
    inf = float("inf")
    table = {
        "none": lambda: z, "relu": lambda: z.clamp(0, inf),
        "leaky_relu": lambda: z.clamp(0, inf) + z.clamp(-inf, 0) / 100,
        "elu": lambda: z.clamp(0, inf) + torch.special.expm1(z.clamp(-inf, 0)),
        "sigmoid": lambda: torch.special.expit(z), "tanh": lambda: z.tanh(),
        "gelu": lambda: z * normal_cdf(z),
        "swish": lambda: z * torch.special.expit(z),
        "mish": lambda: z * torch.logaddexp(z, torch.zeros_like(z)).tanh(),
    }
    return table[act]()


def slope_exact(act, z):
    """act'(z) as d act / dz, each from the function's own closed form."""
    sigma = torch.special.expit
    table = {
        "none": lambda: torch.ones_like(z),
        "relu": lambda: (z > 0).double(),
        "leaky_relu": lambda: (z > 0).double() * 0.99 + 0.01,
        "elu": lambda: z.clamp(-float("inf"), 0).exp(),
        "sigmoid": lambda: sigma(z) * sigma(-z),
        "tanh": lambda: z.cosh().pow(-2),
        "gelu": lambda: normal_cdf(z) + z * (z.square() / -2).exp() / (2 * math.pi) ** 0.5,
        "swish": lambda: sigma(z) + z * sigma(z) * sigma(-z),
    }
    if act != "mish":
        return table[act]()
    soft = torch.logaddexp(z, torch.zeros_like(z))
    return soft.tanh() + z * sigma(z) / soft.cosh().square()


def exact(case, seed):
    s = prepare(case, seed)

    def of(name):
        return None if s[name] is None else s[name].to(torch.float64)

    if case["op"] == "linear":
        z = torch.matmul(of("x"), of("w"))
        if case["bias"]:
            z += of("bias")
        y = act_exact(case["act"], z)
        if case["residual"]:
            y = y + of("residual")
        return (y, z) if case["preact"] else y
    if case["op"] == "linear_grad":
        dz = of("dy")
        if case["act"] != "none":
            dz = dz * slope_exact(case["act"], of("z"))
        # The products take dz as it is stored.
        held = dz.to(DTYPES[case["dtype"]]).to(torch.float64)
        dx = torch.einsum("mn,kn->mk", held, of("w"))
        if case["prev_act"] != "none":
            dx *= slope_exact(case["prev_act"], of("prev_z"))
        if case["residual"]:
            dx += of("residual")
        grads = (dx, torch.einsum("mk,mn->kn", of("x"), held), held.sum(dim=0))
        return grads + (dz,) if case["act"] != "none" else grads
    x, gamma = of("x"), of("gamma")
    if case["op"] == "layer_norm":
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        rstd = (var + s["eps"]).pow(-0.5)
        y = torch.addcmul(of("beta"), (x - mean) * rstd, gamma)
        return y, mean.squeeze(1), rstd.squeeze(1)
    dy, rstd = of("dy"), s["rstd"].double().unsqueeze(1)
    xhat = (x - s["mean"].double().unsqueeze(1)) * rstd
    g = dy * gamma
    dx = rstd * (g - g.mean(dim=1, keepdim=True)
                 - xhat * (g * xhat).mean(dim=1, keepdim=True))
    if case["residual"]:
        dx = dx + of("residual")
    return dx, torch.einsum("rc,rc->c", dy, xhat), dy.sum(dim=0)
