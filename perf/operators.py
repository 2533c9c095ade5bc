"""Timed cases of the dense linear and layer norm operators.

The two operators are one half of a transformer block in trainable form: a
layer norm (affine, or modulated per sample), and a matrix product whose
epilogue adds the bias, applies the activation, scales by a gate and adds the
residual.  ``run`` computes them either in plain torch operations in 32 bits
(``own`` false) or through the framework's public calls (``own`` true).
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
GELU_K = math.sqrt(2.0 / math.pi)
GELU_C = 0.044715
EPS = 1e-6


# ---------------------------------------------------------------------------- cases

def _linear(name, train, dtype, samples, rows, k, n, act, bias=True, gate=False, residual=False):
    return {"name": name, "op": "linear", "train": train, "dtype": dtype, "samples": samples, "rows": rows, "k": k,
            "n": n, "act": act, "bias": bias, "gate": gate, "residual": residual}


def _norm(name, train, dtype, samples, rows, d, form, vec_dtype=None):
    return {"name": name, "op": "norm", "train": train, "dtype": dtype, "samples": samples, "rows": rows, "d": d,
            "form": form, "vec_dtype": vec_dtype or dtype}


def listed():
    return [
        # image feed-forward on dense weights, 3456 image tokens: the product that widens, with its GELU
        _linear("linear_fc1_gelu", False, "bf16", 1, 3456, 3072, 12288, "gelu_tanh"),
        # the product that narrows, two samples of 1728 tokens, each with its own gate, onto the residual
        _linear("linear_fc2_gated", False, "bf16", 2, 1728, 12288, 3072, "none", gate=True, residual=True),
        # the text stream's 256 tokens through the same product: few tiles, a long sum
        _linear("linear_text_fc2", False, "bf16", 1, 256, 12288, 3072, "none", gate=True, residual=True),
        # timestep embedding of a batch of sixteen
        _linear("linear_rows16_silu", False, "fp16", 1, 16, 3072, 3072, "silu"),
        # modulation vectors of one sample: one row against a large weight, latency and bandwidth
        _linear("linear_row1", False, "bf16", 1, 1, 3072, 18432, "none"),
        # a training step of the widening product at the image's length
        _linear("linear_fc1_train", True, "bf16", 1, 3456, 3072, 12288, "gelu_tanh"),
        # a ragged training step: odd widths, short samples, every optional operand
        _linear("linear_odd_train", True, "fp16", 2, 333, 1001, 777, "silu", gate=True, residual=True),
        # the block's norm with one sample's and stream's modulation vectors
        _norm("norm_modulate", False, "bf16", 2, 3456, 3072, "modulate"),
        # a single token's affine norm: latency
        _norm("norm_row1", False, "bf16", 1, 1, 3072, "affine"),
        # a training step of the modulated norm, gradients of both vectors per sample
        _norm("norm_modulate_train", True, "bf16", 2, 3456, 3072, "modulate"),
        # long batch of narrower rows in half precision with 32-bit weights
        _norm("norm_long_train", True, "fp16", 1, 65536, 1024, "affine", "fp32"),
        # a ragged 32-bit norm of odd width
        _norm("norm_odd_train", True, "fp32", 1, 999, 1001, "affine"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    train = rng.random() < 0.5
    if rng.random() < 0.6:
        most = 3456 * 3072 * 12288 * (1 if train else 3)
        while True:
            samples = rng.choice([1, 1, 2, 3, 4])
            rows, k, n = _log_int(rng, 1, 4096), _log_int(rng, 16, 12288), _log_int(rng, 16, 18432)
            if rng.random() < 0.6:  # widths of real layers are mostly multiples of eight
                k, n = (k + 7) // 8 * 8, (n + 7) // 8 * 8
            if samples * rows <= 8192 and samples * rows * k * n <= most:
                break
        return {"op": "linear", "train": train, "dtype": rng.choice(["bf16", "bf16", "fp16"]), "samples": samples,
                "rows": rows, "k": k, "n": n, "act": rng.choice(["none", "gelu_tanh", "silu"]),
                "bias": rng.random() < 0.8, "gate": rng.random() < 0.4, "residual": rng.random() < 0.4}
    while True:
        samples = rng.choice([1, 1, 2, 3, 4])
        rows, d = _log_int(rng, 1, 65536), _log_int(rng, 8, 12288)
        if rng.random() < 0.6:
            d = (d + 7) // 8 * 8
        if samples * rows * d <= 65536 * 1024:
            break
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    form = rng.choice(["affine", "modulate"])
    vec = "fp32" if form == "affine" and rng.random() < 0.5 else dtype
    return {"op": "norm", "train": train, "dtype": dtype, "samples": samples, "rows": rows, "d": d, "form": form,
            "vec_dtype": vec}


def work(case):
    m = case["samples"] * case["rows"]
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "linear":
        k, n = case["k"], case["n"]
        moved = m * k + n * k + m * n + (n if case["bias"] else 0) + (m * n if case["residual"] else 0) \
            + (case["samples"] * n if case["gate"] else 0)
        flops = 2 * m * n * k
        if case["train"]:  # reads dy; writes dx, dW, db, d gate
            moved += m * n + m * k + n * k + (n if case["bias"] else 0) + (case["samples"] * n if case["gate"] else 0)
            flops *= 3
        return {"bytes": moved * e, "flops": flops}
    d = case["d"]
    vecs = case["samples"] if case["form"] == "modulate" else 1
    ve = 4 if case["vec_dtype"] == "fp32" else 2
    passes, vec_passes = (4, 4) if case["train"] else (2, 2)  # x, y (dy, dx); weight, bias (and their gradients)
    return {"bytes": passes * m * d * e + vec_passes * vecs * d * ve, "flops": (22 if case["train"] else 8) * m * d}


# --------------------------------------------------------------------------- inputs

def _shape(case, width):
    return (case["samples"], case["rows"], width)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def normal(shape, std, mean=0.0, dtype=dt):
        return (torch.randn(shape, generator=g, device="cuda") * std + mean).to(dtype)

    state = {"case": case}
    if case["op"] == "linear":
        k, n = case["k"], case["n"]
        state["x"] = normal(_shape(case, k), 1.0)
        state["w"] = normal((n, k), 1.0 / math.sqrt(k))
        state["b"] = normal((n,), 0.1) if case["bias"] else None
        state["gate"] = normal((case["samples"], n), 0.5) if case["gate"] else None
        state["res"] = normal(_shape(case, n), 1.0) if case["residual"] else None
        names = ("x", "w", "b", "gate", "res")
        out = n
    else:
        d, vdt = case["d"], DTYPES[case["vec_dtype"]]
        # hidden states: a spread of row scales, and channels with an offset of their own
        scale = torch.rand(_shape(case, 1), generator=g, device="cuda") * 3.0 + 0.5
        offset = torch.randn((d,), generator=g, device="cuda") * 0.5
        state["x"] = (torch.randn(_shape(case, d), generator=g, device="cuda") * scale + offset).to(dt)
        if case["form"] == "modulate":
            state["shift"] = normal((case["samples"], d), 0.3, dtype=vdt)
            state["scale"] = normal((case["samples"], d), 0.3, dtype=vdt)
            names = ("x", "shift", "scale")
        else:
            state["w"] = normal((d,), 0.2, 1.0, dtype=vdt)
            state["b"] = normal((d,), 0.2, dtype=vdt)
            names = ("x", "w", "b")
        out = d
    if case["train"]:
        state["dy"] = normal(_shape(case, out), 1.0)
        state["leaves"] = [name for name in names if state[name] is not None]
        for name in state["leaves"]:
            state[name].requires_grad_(True)
    return state


# ------------------------------------------------------------------------ one pass

def _plain_act(z, act):
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(GELU_K * (z + GELU_C * z * z * z)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _plain_act_grad(z, act):
    if act == "gelu_tanh":
        t = torch.tanh(GELU_K * (z + GELU_C * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * GELU_K * (1.0 + 3.0 * GELU_C * z * z)
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    return None


def _plain_linear(state, case):
    x, w = state["x"].float(), state["w"].float()
    dt = state["x"].dtype
    z = x.reshape(-1, case["k"]) @ w.t()
    z = z.reshape(_shape(case, case["n"]))
    if state["b"] is not None:
        z = z + state["b"].float()
    a = _plain_act(z, case["act"])
    y = a
    gate = None if state["gate"] is None else state["gate"].float()[:, None, :]
    if gate is not None:
        y = gate * y
    if state["res"] is not None:
        y = state["res"].float() + y
    if not case["train"]:
        return y.to(dt)
    dy = state["dy"].float()
    dz = dy if gate is None else dy * gate
    slope = _plain_act_grad(z, case["act"])
    if slope is not None:
        dz = dz * slope
    flat = dz.reshape(-1, case["n"])
    grads = {"x": (flat @ w).reshape(x.shape), "w": flat.t() @ x.reshape(-1, case["k"])}
    if state["b"] is not None:
        grads["b"] = flat.sum(0)
    if gate is not None:
        grads["gate"] = (dy * a).sum(1)
    if state["res"] is not None:
        grads["res"] = dy
    return [y.to(dt)] + [grads[name].to(dt) for name in state["leaves"]]


def _plain_norm(state, case):
    x = state["x"].float()
    modulate = case["form"] == "modulate"
    weight = 1.0 + state["scale"].float()[:, None, :] if modulate else state["w"].float()
    bias = state["shift"].float()[:, None, :] if modulate else state["b"].float()
    centred = x - x.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + EPS)
    xh = centred * rstd
    y = (xh * weight + bias).to(state["x"].dtype)
    if not case["train"]:
        return y
    dy = state["dy"].float()
    a = dy * weight
    dx = rstd * (a - a.mean(-1, keepdim=True) - xh * (a * xh).mean(-1, keepdim=True))
    over = (1,) if modulate else (0, 1)
    dweight, dbias = (dy * xh).sum(over), dy.sum(over)
    grads = {"x": dx, "scale": dweight, "shift": dbias, "w": dweight, "b": dbias}
    return [y] + [grads[name].to(state[name].dtype) for name in state["leaves"]]


def _own_forward(state, case):
    from qwen_image_shardedit_mlx_b200 import dense_linear, layer_norm, layer_norm_modulate

    if case["op"] == "linear":
        act = None if case["act"] == "none" else case["act"]
        return dense_linear(state["x"], state["w"], state["b"], activation=act, residual=state["res"],
                            gate=state["gate"])
    if case["form"] == "modulate":
        return layer_norm_modulate(state["x"], state["shift"], state["scale"], eps=EPS)
    return layer_norm(state["x"], state["w"], state["b"], eps=EPS)


def run(state):
    case = state["case"]
    if own:
        y = _own_forward(state, case)
        if not case["train"]:
            return y
        return [y.detach(), *torch.autograd.grad(y, [state[name] for name in state["leaves"]], state["dy"])]
    with torch.no_grad():
        return _plain_linear(state, case) if case["op"] == "linear" else _plain_norm(state, case)


# --------------------------------------------------------------------- 64-bit values

def exact(case, seed):
    """The operators by their definitions in 64 bits; the gradients by
    differentiating that definition."""

    state = prepare(case, seed)
    v = {name: t.detach().double() for name, t in state.items() if isinstance(t, torch.Tensor)}
    for name in state.get("leaves", ()):
        v[name].requires_grad_(True)
    if case["op"] == "linear":
        y = torch.einsum("stk,nk->stn", v["x"], v["w"])
        if "b" in v:
            y = y + v["b"]
        if case["act"] == "silu":
            y = y * torch.sigmoid(y)
        elif case["act"] == "gelu_tanh":  # 0.5 (1 + tanh u) = sigmoid(2 u)
            y = y * torch.sigmoid(2.0 * GELU_K * (y + GELU_C * y ** 3))
        if "gate" in v:
            y = torch.einsum("stn,sn->stn", y, v["gate"])
        if "res" in v:
            y = y + v["res"]
    else:
        var, mean = torch.var_mean(v["x"], dim=-1, keepdim=True, correction=0)
        y = (v["x"] - mean) / (var + EPS).sqrt()
        if case["form"] == "modulate":
            y = y + y * v["scale"].unsqueeze(1) + v["shift"].unsqueeze(1)
        else:
            y = y * v["w"] + v["b"]
    if not case["train"]:
        return y
    return [y.detach(), *torch.autograd.grad(y, [v[name] for name in state["leaves"]], v["dy"])]
