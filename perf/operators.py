"""Performance cases of the operators around the residual MLP block: the
root-mean-square norm in front of it (float32, 16 and 8 bits out, with its
gradient) and the products with bias, activation and residual inside it
(bfloat16, float16 and 8 bits, with their gradient).

  norm         h = x + residual; y = h / sqrt(mean(h^2) + eps) * weight,
               rounded to x's type or to 8 bits (e4m3) with one scale a row
  norm_grad    dx (with the gradient that reaches h added) and dweight
  linear       act(x @ w + bias) + residual, the pre-activation kept on demand
  linear_grad  dx, dw and dbias from dy and the kept pre-activation
  linear8      the 8-bit product with a scale a row and a scale a column; x is
               given in 8 bits, or in bfloat16 and quantised row by row first

`own` selects the framework's kernels; without it the same operators run as
elementary torch operations in float32, rounded once at the end.
"""

import math

import torch

own = False

EPS = 1e-6
F8 = torch.float8_e4m3fn
F8_MAX = 448.0
TINY = 2.0 ** -100  # a row's largest magnitude is taken as at least this
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ACTS = ("none", "relu", "gelu", "silu")

# The largest product a drawn case may have (multiply-adds), and the longest norm (elements).
MOST_MNK = 8192 ** 3
MOST_ELEMENTS = 16384 * 8192


def _norm(rows, d, dtype, wtype, quantize, residual, name=None):
    c = {"op": "norm", "rows": rows, "d": d, "dtype": dtype, "wtype": wtype, "quantize": quantize, "residual": residual}
    return c if name is None else {"name": name, **c}


def _norm_grad(rows, d, dtype, wtype, residual, name=None):
    c = {"op": "norm_grad", "rows": rows, "d": d, "dtype": dtype, "wtype": wtype, "residual": residual}
    return c if name is None else {"name": name, **c}


def _linear(m, n, k, dtype, act, order, bias, residual, keep, name=None):
    c = {"op": "linear", "m": m, "n": n, "k": k, "dtype": dtype, "act": act, "order": order, "bias": bias,
         "residual": residual, "keep": keep}
    return c if name is None else {"name": name, **c}


def _linear_grad(m, n, k, dtype, act, order, bias, name=None):
    c = {"op": "linear_grad", "m": m, "n": n, "k": k, "dtype": dtype, "act": act, "order": order, "bias": bias}
    return c if name is None else {"name": name, **c}


def _linear8(m, n, k, act, bias, residual, quantize, name=None):
    c = {"op": "linear8", "m": m, "n": n, "k": k, "act": act, "bias": bias, "residual": residual, "quantize": quantize}
    return c if name is None else {"name": name, **c}


def listed():
    return [
        # Serving one token: the norm in front of an 8-bit layer, where only latency counts.
        _norm(1, 2048, "bf16", "bf16", True, True, "norm_token_8bit"),
        # A long prompt's norm into 8 bits: bound by memory.
        _norm(16384, 8192, "bf16", "bf16", True, True, "norm_prompt_8bit"),
        # The norm's gradient in a float32 model of odd width.
        _norm_grad(777, 1111, "f32", "f32", False, "norm_grad_ragged"),
        # The norm's gradient in a training step, the residual stream's gradient added on the way.
        _norm_grad(8192, 4096, "bf16", "bf16", True, "norm_grad_train"),
        # One token through a layer whose weights lie row by output: bound by reading the weights.
        _linear(1, 4096, 4096, "bf16", "silu", "nk", True, False, False, "linear_token"),
        # A small batch (the 64-row layer) on weights as the framework's programs hold them.
        _linear(64, 4096, 4096, "bf16", "gelu", "kn", True, True, False, "linear_rows64"),
        # Odd sizes throughout: no row but the first is aligned.
        _linear(777, 1111, 333, "f16", "relu", "kn", True, True, False, "linear_ragged"),
        # The residual block's first layer in training, the pre-activation kept.
        _linear(4096, 8192, 2048, "bf16", "gelu", "kn", True, False, True, "linear_up_train"),
        # A small layer's gradient (examples/mbr.mlir's sizes): many short steps.
        _linear_grad(256, 256, 128, "f16", "relu", "kn", True, "linear_grad_small"),
        # The first layer's gradient in training.
        _linear_grad(4096, 8192, 2048, "bf16", "gelu", "kn", True, "linear_grad_train"),
        # A few tokens through an 8-bit second layer with the residual.
        _linear8(16, 2048, 8192, "none", True, True, False, "linear8_tokens"),
        # A long prompt through a large 8-bit layer, its input quantised on the way.
        _linear8(8192, 8192, 8192, "none", False, True, True, "linear8_prompt"),
    ]


def _log(rng, lo, hi):
    """A size between lo and hi, even over its logarithm; a multiple of 64 or 8 half of the time where it is large enough."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    step = rng.choice([1, 1, 8, 64])
    return max(lo, min(hi, v if v < 4 * step else v // step * step))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_grad", "linear", "linear", "linear", "linear_grad", "linear_grad", "linear8",
                     "linear8"])
    if op in ("norm", "norm_grad"):
        d = _log(rng, 32, 8192)
        rows = _log(rng, 1, min(16384, MOST_ELEMENTS // d))
        dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
        wtype = rng.choice([dtype, "f32"])
        residual = rng.random() < 0.6
        if op == "norm":
            return _norm(rows, d, dtype, wtype, rng.random() < 0.5, residual)
        return _norm_grad(rows, d, dtype, wtype, residual)
    n, k = _log(rng, 64, 8192), _log(rng, 64, 8192)
    m = _log(rng, 1, min(8192, max(1, MOST_MNK // (4 * n * k))))
    act, bias, residual = rng.choice(ACTS), rng.random() < 0.7, rng.random() < 0.5
    if op == "linear8":
        k = max(64, k // 16 * 16)  # 8-bit rows are whole 16-byte pieces
        return _linear8(m, n, k, act, bias, residual, rng.random() < 0.5)
    dtype, order = rng.choice(["bf16", "bf16", "f16"]), rng.choice(["kn", "nk"])
    if op == "linear":
        return _linear(m, n, k, dtype, act, order, bias, residual, rng.random() < 0.4)
    return _linear_grad(m, n, k, dtype, act, order, bias)


def _to_f8(v):
    """(codes, scale) of v (float32) row by row: scale = max|v| / 448, codes nearest (ties to even) to v / scale."""
    top = v.abs().amax(-1).clamp_min(TINY)
    return (v * (F8_MAX / top)[:, None]).to(F8), top / F8_MAX


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(sigma, *shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * sigma

    op = case["op"]
    if op in ("norm", "norm_grad"):
        t, tw, rows, d = DTYPES[case["dtype"]], DTYPES[case["wtype"]], case["rows"], case["d"]
        # Activations: rows of different sizes, a few channels that stand out.
        size = torch.exp(normal(0.5, rows, 1))
        channel = 1 + 8 * (torch.rand((d,), generator=gen, device="cuda") < 0.01)
        s = {"x": (normal(1.0, rows, d) * size * channel).to(t), "w": (1 + normal(0.1, d)).to(tw)}
        if case["residual"]:
            s["r"] = normal(0.7, rows, d).to(t)
        if op == "norm_grad":
            s["dy"] = normal(0.02, rows, d).to(t)
        return s
    m, n, k = case["m"], case["n"], case["k"]
    if op == "linear8":
        x = normal(1.0, m, k) * torch.exp(normal(0.5, m, 1))
        codes, scale = _to_f8(normal(k ** -0.5, n, k))
        s = {"w": codes, "ws": scale}
        if case["quantize"]:
            s["x"] = x.to(torch.bfloat16)
        else:
            s["x"], s["xs"] = _to_f8(x)
        if case["bias"]:
            s["bias"] = normal(0.02, n)
        if case["residual"]:
            s["r"] = normal(1.0, m, n).to(torch.bfloat16)
        return s
    t = DTYPES[case["dtype"]]
    s = {"x": normal(1.0, m, k).to(t)}
    s["w"] = (normal(k ** -0.5, n, k).to(t).t() if case["order"] == "nk" else normal(k ** -0.5, k, n).to(t))
    if op == "linear_grad":
        s["dy"] = normal(0.02, m, n).to(t)
        if case["act"] != "none":
            s["z"] = normal(1.0, m, n).to(t)
        return s
    if case["bias"]:
        s["bias"] = normal(0.02, n).to(t)
    if case["residual"]:
        s["r"] = normal(1.0, m, n).to(t)
    return s


def prepare(case, seed):
    return {"case": case, **_inputs(case, seed)}


def _run_own(s):
    from tensorforge_amd import tforge_nn as nn
    c = s["case"]
    op = c["op"]
    if op == "norm":
        if c["quantize"]:
            q, scale, h = nn.rms_norm(s["x"], s["w"], residual=s.get("r"), eps=EPS, quantize=True)
            return {"q": q, "scale": scale, "h": h} if c["residual"] else {"q": q, "scale": scale}
        y, h = nn.rms_norm(s["x"], s["w"], residual=s.get("r"), eps=EPS)
        return {"y": y, "h": h} if c["residual"] else {"y": y}
    if op == "norm_grad":
        dx, dw = nn.rms_norm_grad(s["dy"], s["x"], s["w"], eps=EPS, dh=s.get("r"))
        return {"dx": dx, "dw": dw}
    if op == "linear":
        if c["keep"]:
            out, z = nn.linear(s["x"], s["w"], s.get("bias"), c["act"], s.get("r"), keep=True)
            return {"out": out, "z": z}
        return {"out": nn.linear(s["x"], s["w"], s.get("bias"), c["act"], s.get("r"))}
    if op == "linear_grad":
        dx, dw, dbias = nn.linear_grad(s["dy"], s["x"], s["w"], s.get("z"), c["act"],
                                       bias_dtype=s["x"].dtype if c["bias"] else None)
        return {"dx": dx, "dw": dw, "dbias": dbias} if c["bias"] else {"dx": dx, "dw": dw}
    if c["quantize"]:
        q, scale = nn.quantize_rows(s["x"])
        out = nn.linear(q, s["w"].t(), s.get("bias"), c["act"], s.get("r"), x_scale=scale, w_scale=s["ws"])
        return {"out": out, "q": q, "scale": scale}
    return {"out": nn.linear(s["x"], s["w"].t(), s.get("bias"), c["act"], s.get("r"), x_scale=s["xs"],
                             w_scale=s["ws"])}


def _act(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).float()
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    s = 1 / (1 + torch.exp(-z))
    return s * (1 + z * (1 - s))


def run(state):
    if own:
        return _run_own(state)
    s, c = state, state["case"]
    op = c["op"]
    if op == "norm":
        t = s["x"].dtype
        h = s["x"].float() + s["r"].float() if c["residual"] else s["x"].float()
        y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * s["w"].float()
        if c["quantize"]:
            q, scale = _to_f8(y)
            out = {"q": q, "scale": scale}
        else:
            out = {"y": y.to(t)}
        if c["residual"]:
            out["h"] = h.to(t)
        return out
    if op == "norm_grad":
        h, dy, w = s["x"].float(), s["dy"].float(), s["w"].float()
        r = torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)
        xhat, g = h * r, dy * w
        dx = r * (g - xhat * (g * xhat).mean(-1, keepdim=True))
        if c["residual"]:
            dx = dx + s["r"].float()
        return {"dx": dx.to(s["x"].dtype), "dw": (dy * xhat).sum(0).to(s["w"].dtype)}
    if op == "linear_grad":
        t = s["x"].dtype
        dz = s["dy"].float()
        if c["act"] != "none":
            dz = dz * _act_slope(s["z"].float(), c["act"])
        out = {"dx": (dz @ s["w"].float().t()).to(t)}
        if c["order"] == "nk":  # the weights' gradient lies in memory as the weights do
            out["dw"] = (dz.t() @ s["x"].float()).to(t).t()
        else:
            out["dw"] = (s["x"].float().t() @ dz).to(t)
        if c["bias"]:
            out["dbias"] = dz.sum(0).to(t)
        return out
    more = {}
    if op == "linear8":
        t = torch.bfloat16
        x, xs = s["x"], s.get("xs")
        if c["quantize"]:
            x, xs = _to_f8(x.float())
            more = {"q": x, "scale": xs}
        z = (x.float() @ s["w"].float().t()) * xs[:, None] * s["ws"]
    else:
        t = s["x"].dtype
        z = s["x"].float() @ s["w"].float()
    if c["bias"]:
        z = z + s["bias"].float()
    if c.get("keep"):
        more = {"z": z.to(t)}
    out = _act(z, c["act"])
    if c["residual"]:
        out = out + s["r"].float()
    return {"out": out.to(t), **more}


def work(case):
    c, op = case, case["op"]
    size = {"f32": 4, "bf16": 2, "f16": 2}
    if op in ("norm", "norm_grad"):
        e, n = size[c["dtype"]], c["rows"] * c["d"]
        if op == "norm":
            tensors = 3 if c["residual"] else 1  # x, residual in, h out
            out = n + 4 * c["rows"] if c["quantize"] else e * n
            return {"bytes": tensors * e * n + out + size[c["wtype"]] * c["d"], "flops": 5 * n}
        tensors = 4 if c["residual"] else 3  # dy, h, (dh) in, dx out
        return {"bytes": tensors * e * n + 2 * size[c["wtype"]] * c["d"], "flops": 10 * n}
    m, n, k = c["m"], c["n"], c["k"]
    if op == "linear8":
        x = (2 * m * k + m * k if c["quantize"] else m * k) + 4 * m
        extra = (4 * n if c["bias"] else 0) + (2 * m * n if c["residual"] else 0)
        return {"bytes": x + n * k + 4 * n + 2 * m * n + extra, "flops": 2 * m * n * k}
    if op == "linear":
        extra = (n if c["bias"] else 0) + m * n * (int(c["residual"]) + int(c["keep"]))
        return {"bytes": 2 * (m * k + k * n + m * n + extra), "flops": 2 * m * n * k}
    read = m * n * (1 if c["act"] == "none" else 2) + m * k + k * n
    return {"bytes": 2 * (read + m * k + k * n + (n if c["bias"] else 0)), "flops": 4 * m * n * k}


def exact(case, seed):
    """The outputs in 64 bits from the definitions.  8-bit codes appear as the values that they round: y / scale."""
    i = {k: v.double() for k, v in _inputs(case, seed).items()}
    op = case["op"]
    if op == "norm":
        h = i["x"] + i["r"] if case["residual"] else i["x"]
        y = h / (h.pow(2).mean(1, keepdim=True) + EPS).sqrt() * i["w"]
        out = {"h": h} if case["residual"] else {}
        if not case["quantize"]:
            return {"y": y, **out}
        scale = y.abs().max(1).values.clamp_min(TINY) / F8_MAX
        return {"q": y / scale[:, None], "scale": scale, **out}
    if op == "norm_grad":
        h, d = i["x"], case["d"]
        var = h.pow(2).sum(1, keepdim=True) / d + EPS
        g = i["dy"] * i["w"]
        dx = g / var.sqrt() - h * (g * h).sum(1, keepdim=True) / (d * var.pow(1.5))
        if case["residual"]:
            dx = dx + i["r"]
        return {"dx": dx, "dw": (i["dy"] * h / var.sqrt()).sum(0)}
    act = case["act"]
    if op == "linear_grad":
        dz = i["dy"]
        if act == "relu":
            dz = torch.where(i["z"] > 0, dz, torch.zeros_like(dz))
        elif act == "gelu":
            z = i["z"]
            dz = dz * (torch.special.erfc(-z / 2 ** 0.5) / 2 + z * torch.exp(-z * z / 2) / (2 * math.pi) ** 0.5)
        elif act == "silu":
            s = torch.sigmoid(i["z"])
            dz = dz * (s + i["z"] * s * (1 - s))
        out = {"dx": torch.matmul(dz, i["w"].t().contiguous())}
        out["dw"] = torch.matmul(i["x"].t().contiguous(), dz)
        if case["bias"]:
            out["dbias"] = dz.sum(0)
        return out
    more = {}
    if op == "linear8":
        x, w = i["x"], i["w"].t().contiguous() * i["ws"]
        if case["quantize"]:
            # The product takes the rounded codes.
            scale = x.abs().max(1).values.clamp_min(TINY) / F8_MAX
            more = {"q": x / scale[:, None], "scale": scale}
            x = (x / scale[:, None]).float().to(F8).double() * scale[:, None]
        else:
            x = x * i["xs"][:, None]
        z = torch.matmul(x, w)
    else:
        z = torch.matmul(i["x"], i["w"].contiguous())
    if case["bias"]:
        z = z + i["bias"]
    if case.get("keep"):
        more = {"z": z}
    if act == "relu":
        out = torch.where(z > 0, z, torch.zeros_like(z))
    elif act == "gelu":
        out = z * torch.special.erfc(-z / 2 ** 0.5) / 2
    elif act == "silu":
        out = z * torch.sigmoid(z)
    else:
        out = z
    if case["residual"]:
        out = out + i["r"]
    return {"out": out, **more}
