"""The layer operators of networks that the fused renderer kernels do not cover, as measurable cases: a linear layer with
its epilogue (forward and backward), the residual addition with a root-mean-square norm (forward, backward, and with an
8-bit output), and the linear layer on 8-bit operands with scales.

Three kinds of case, by "op":

  linear      y = act(x W^T + b) + r; x may come in two pieces along its columns (a skip connection: [points | hidden]).
              With train, the gradients of x (each piece), W, b and r for a given dL/dy as well.
  norm        h = x + r,  y = w h / sqrt(mean(h^2) + eps). With q8, y leaves as e4m3 numbers and one float32 scale a row.
              With train, the gradients of x (= of r) and w for given dL/dy and dL/dh.
  linear_q8   y = act(s_x s_w (q_x q_w^T) + b) + r on e4m3 operands with a float32 scale for each row of x and of W.

`run` computes them in their plain form, or, where `own` is true, with the framework's operators.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
E4M3_MAX = 448.0
SCALE_MIN = 2.0 ** -126
EPS = 1e-6


def _linear(name, dtype, m, n, k, k2=0, act="relu", residual=False, train=False):
    return {"name": name, "op": "linear", "dtype": dtype, "m": m, "n": n, "k": k, "k2": k2, "act": act,
            "residual": residual, "train": train}


def _norm(name, dtype, m, n, residual=True, q8=False, train=False):
    return {"name": name, "op": "norm", "dtype": dtype, "m": m, "n": n, "residual": residual, "q8": q8, "train": train}


def _q8(name, dtype, m, n, k, act="relu", residual=True):
    return {"name": name, "op": "linear_q8", "dtype": dtype, "m": m, "n": n, "k": k, "act": act, "residual": residual}


def listed():
    return [
        # one row through a wide layer: what a single query costs, latency alone
        _linear("linear_one_row_bf16", "bf16", 1, 1024, 1024, act="silu", residual=True),
        # a handful of rows through a large layer: the weights have to be read once, nothing else counts
        _linear("linear_few_rows_fp16", "fp16", 13, 4096, 4096, act="gelu"),
        # a trunk layer of the 256-wide network over a training batch's fine samples (4096 rays x 192)
        _linear("linear_trunk_bf16", "bf16", 786432, 256, 256, act="relu"),
        # the layer after the skip connection, [63 encoded coordinates | 256 hidden], over one network chunk of 65536
        _linear("linear_skip_fp32", "fp32", 65536, 256, 63, k2=256, act="relu"),
        # a square layer of a wide network: matrix-core bound
        _linear("linear_wide_bf16", "bf16", 8192, 4096, 4096, act="gelu", residual=True),
        # forward and backward of a trunk layer over 1024 rays x 192 samples
        _linear("linear_train_trunk_bf16", "bf16", 196608, 256, 256, act="relu", train=True),
        # forward and backward at sizes that fit no tile, every gradient needed, rows that are not 16-byte aligned
        _linear("linear_train_odd_fp16", "fp16", 4097, 515, 1021, act="gelu", residual=True, train=True),
        # one row between two 8-bit layers: latency alone
        _norm("norm_one_row_q8", "bf16", 1, 4096, q8=True),
        # forward and backward between two 1024-wide layers over a network chunk
        _norm("norm_train_bf16", "bf16", 65536, 1024, train=True),
        # the input of a large 8-bit layer, one row short of a round number
        _norm("norm_rows_q8", "bf16", 16383, 4096, q8=True),
        # a few rows through a large 8-bit layer: weight bytes alone
        _q8("linear_q8_few_rows", "bf16", 5, 4096, 4096, act="silu"),
        # a square layer of a wide network in 8 bits
        _q8("linear_q8_wide", "bf16", 8192, 4096, 4096, act="gelu"),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm; every third one round."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.34 and v >= 16:
        v -= v % (64 if v >= 256 else 16)
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "norm", "norm", "linear_q8"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    act = rng.choice(["none", "relu", "gelu", "silu"])
    residual = rng.random() < 0.5
    while True:
        if op == "norm":
            q8 = rng.random() < 0.4
            c = {"op": op, "dtype": dtype, "m": _spread(rng, 1, 65536), "n": _spread(rng, 1, 8192), "residual": residual,
                 "q8": q8, "train": not q8 and rng.random() < 0.5}
            if c["m"] * c["n"] <= 1 << 26:
                return c
        elif op == "linear_q8":
            c = {"op": op, "dtype": dtype, "m": _spread(rng, 1, 65536), "n": _spread(rng, 1, 4096),
                 "k": _spread(rng, 16, 4096), "act": act, "residual": residual}
            if c["m"] * c["n"] * c["k"] <= 1 << 36 and c["m"] * (c["n"] + c["k"]) <= 1 << 27:
                return c
        else:
            train = rng.random() < 0.5
            c = {"op": op, "dtype": dtype, "m": _spread(rng, 1, 262144), "n": _spread(rng, 1, 4096),
                 "k": _spread(rng, 1, 4096), "k2": _spread(rng, 1, 512) if rng.random() < 0.3 else 0, "act": act,
                 "residual": residual, "train": train}
            k = c["k"] + c["k2"]
            if c["m"] * c["n"] * k <= 1 << (34 if train else 36) and c["m"] * (c["n"] + k) <= 1 << 27:
                return c


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    m, n = case["m"], case["n"]

    def normal(*shape, scale=1.0, offset=0.0):
        return (torch.randn(*shape, device="cuda", generator=g) * scale + offset).to(dt)

    s = {"case": dict(case)}
    if case["op"] == "norm":
        s["x"] = normal(m, n)
        s["w"] = normal(n, scale=0.2, offset=1.0)
        s["r"] = normal(m, n, scale=2.0) if case["residual"] else None
        if case["train"]:
            s["gy"], s["gh"] = normal(m, n), normal(m, n)
            for key in ("x", "w", "r"):
                if s[key] is not None:
                    s[key].requires_grad_()
        return s
    if case["op"] == "linear_q8":
        k = case["k"]
        s["xq"], s["xs"] = _quantised(torch.randn(m, k, device="cuda", generator=g))
        s["wq"], s["ws"] = _quantised(torch.randn(n, k, device="cuda", generator=g) / math.sqrt(k))
        s["b"] = normal(n, scale=0.1)
        s["r"] = normal(m, n) if case["residual"] else None
        return s
    k, k2 = case["k"], case["k2"]
    s["x"] = normal(m, k)
    s["x2"] = normal(m, k2) if k2 else None
    s["w"] = normal(n, k + k2, scale=1.0 / math.sqrt(k + k2))
    s["b"] = normal(n, scale=0.1)
    s["r"] = normal(m, n) if case["residual"] else None
    if case["train"]:
        s["gy"] = normal(m, n)
        for key in ("x", "x2", "w", "b", "r"):
            if s[key] is not None:
                s[key].requires_grad_()
    return s


def run(s):
    return _run_own(s) if own else _run_plain(s)


def work(case):
    """Inputs read once and outputs written once; the products' multiplications and additions."""
    m, n = case["m"], case["n"]
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm":
        streams = 3 + (1 if case["residual"] else 0)              # x, (r), y, h
        if case["q8"]:
            return {"bytes": m * n * e * (streams - 1) + n * e + m * n + 4 * m, "flops": 5.0 * m * n}
        if case["train"]:                                         # dL/dy, dL/dh, dx read and written besides
            return {"bytes": m * n * e * (streams + 3) + 2 * n * e, "flops": 16.0 * m * n}
        return {"bytes": m * n * e * streams + n * e, "flops": 5.0 * m * n}
    if case["op"] == "linear_q8":
        k = case["k"]
        return {"bytes": m * k + n * k + 4 * (m + n) + n * e + m * n * e * (2 if case["residual"] else 1),
                "flops": 2.0 * m * n * k}
    k = case["k"] + case["k2"]
    forward = e * (m * k + n * k + n + m * n * (2 if case["residual"] else 1))
    if not case["train"]:
        return {"bytes": forward, "flops": 2.0 * m * n * k}
    # dL/dy read; dx, dW, db written (dr is dL/dy itself)
    return {"bytes": forward + e * (m * n + m * k + n * k + n), "flops": 6.0 * m * n * k}


# ---------------------------------------------------------------------------- the framework's operators
def _run_own(s):
    from nerf_loc_amd import layers
    c = s["case"]
    if c["op"] == "norm":
        if c["q8"]:
            q, scale, h = layers.add_rms_norm_q8(s["x"], s["w"], residual=s["r"], eps=EPS)
            return {"q": q, "scale": scale, "h": h}
        y, h = layers.add_rms_norm(s["x"], s["w"], residual=s["r"], eps=EPS)
        if not c["train"]:
            return {"y": y, "h": h}
        leaves = [t for t in (s["x"], s["w"], s["r"]) if t is not None]
        grads = torch.autograd.grad([y, h], leaves, [s["gy"], s["gh"]])
        return {"y": y, "h": h, "grads": list(grads)}
    if c["op"] == "linear_q8":
        return layers.linear_q8(s["xq"], s["xs"], s["wq"], s["ws"], s["b"], activation=c["act"], residual=s["r"],
                                out_dtype=DTYPES[c["dtype"]])
    x = s["x"] if s["x2"] is None else (s["x"], s["x2"])
    y = layers.linear(x, s["w"], s["b"], activation=c["act"], residual=s["r"])
    if not c["train"]:
        return y
    leaves = [t for t in (s["x"], s["x2"], s["w"], s["b"], s["r"]) if t is not None]
    return {"y": y, "grads": list(torch.autograd.grad(y, leaves, s["gy"]))}


# ---------------------------------------------------------------------------- the plain forms
def _quantised(x):
    """e4m3 numbers and the float32 scale of each row: amax / 448."""
    scale = (x.abs().amax(-1) / E4M3_MAX).clamp_min(SCALE_MIN)
    return (x / scale[:, None]).to(torch.float8_e4m3fn), scale


def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if act == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    return torch.ones_like(z)


@torch.no_grad()
def _run_plain(s):
    c = s["case"]
    dt = DTYPES[c["dtype"]]
    if c["op"] == "norm":
        h, w = s["x"].float(), s["w"].float()
        if s["r"] is not None:
            h = h + s["r"].float()
        rstd = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS)
        y = h * rstd * w
        if c["q8"]:
            q, scale = _quantised(y)
            return {"q": q, "scale": scale, "h": h.to(dt)}
        if not c["train"]:
            return {"y": y.to(dt), "h": h.to(dt)}
        gy = s["gy"].float()
        gn = gy * w
        gx = s["gh"].float() + rstd * (gn - h * rstd * rstd * (gn * h).mean(-1, keepdim=True))
        gw = (gy * h * rstd).sum(0)
        gx = gx.to(dt)
        return {"y": y.to(dt), "h": h.to(dt), "grads": [gx, gw.to(dt)] + ([gx] if s["r"] is not None else [])}
    if c["op"] == "linear_q8":
        z = s["xq"].float() @ s["wq"].float().T
        z = z * s["xs"][:, None] * s["ws"] + s["b"].float()
        y = _act(z, c["act"])
        return (y + s["r"].float() if s["r"] is not None else y).to(dt)
    x = s["x"].float() if s["x2"] is None else torch.cat([s["x"].float(), s["x2"].float()], -1)
    w = s["w"].float()
    z = x @ w.T + s["b"].float()
    y = _act(z, c["act"])
    y = (y + s["r"].float() if s["r"] is not None else y).to(dt)
    if not c["train"]:
        return y
    gz = s["gy"].float() * _act_grad(z, c["act"])
    gx = (gz @ w).to(dt)
    grads = [gx] if s["x2"] is None else [gx[:, :c["k"]], gx[:, c["k"]:]]
    grads += [(gz.T @ x).to(dt), gz.sum(0).to(dt)] + ([s["gy"]] if s["r"] is not None else [])
    return {"y": y, "grads": grads}


# ---------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    with torch.no_grad():
        s = prepare(case, seed)
        with torch.enable_grad():
            return _exact_norm(s) if case["op"] == "norm" else _exact_linear(s)


def _exact_norm(s):
    """The gradients come from differentiating the definition."""
    c = s["case"]
    x, w = s["x"].detach().double().requires_grad_(), s["w"].detach().double().requires_grad_()
    h = x if s["r"] is None else x + s["r"].detach().double()
    y = w * (h / (h.square().mean(-1, keepdim=True) + EPS).sqrt())
    if c["q8"]:
        y = y.detach()
        scale = torch.clamp(y.abs().max(-1).values / E4M3_MAX, min=SCALE_MIN)
        return {"q": (y / scale.unsqueeze(-1)).to(torch.float8_e4m3fn), "scale": scale, "h": h.detach()}
    if not c["train"]:
        return {"y": y.detach(), "h": h.detach()}
    gx, gw = torch.autograd.grad((y * s["gy"].double()).sum() + (h * s["gh"].double()).sum(), [x, w])
    return {"y": y.detach(), "h": h.detach(), "grads": [gx, gw] + ([gx] if s["r"] is not None else [])}


def _exact_linear(s):
    c = s["case"]
    fn = {"none": lambda z: z, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu}[c["act"]]
    r = None if s["r"] is None else s["r"].detach().double()
    b = s["b"].detach().double()
    if c["op"] == "linear_q8":
        x = s["xq"].double() * s["xs"].double().unsqueeze(-1)
        w = s["wq"].double() * s["ws"].double().unsqueeze(-1)
        y = fn(torch.mm(x, w.t()).add_(b))
        return y if r is None else y.add_(r)
    pieces = [t.detach().double() for t in (s["x"], s["x2"]) if t is not None]
    w = s["w"].detach().double()
    if c["train"]:
        leaves = [t.requires_grad_() for t in pieces + [w, b] + ([r] if r is not None else [])]
    x = torch.cat(pieces, -1)
    y = fn(torch.mm(x, w.t()) + b)
    if r is not None:
        y = y + r
    if not c["train"]:
        return y
    return {"y": y.detach(), "grads": list(torch.autograd.grad(y, leaves, s["gy"].double()))}
