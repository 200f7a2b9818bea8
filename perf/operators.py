"""The feed-forward operators of a transformer layer: what is measured of them, and their plain forms.

Three operators, each with its backward pass:

  linear          out = act(x @ w + bias) + residual
  gated_linear    h = act(x @ w_gate) * (x @ w_up)
  residual_norm   sum = scale * residual + gate * post(block),  normed = norm(sum) * weight + bias

`run` computes them from elementary torch operations in 32 bits, rounded once at the end, or - where
the module's `own` is true - through this package's kernels.  `exact` computes them in 64 bits.
"""

import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _functional():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "triton-metal_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from triton_metal import functional
    return functional


# ---- cases ---------------------------------------------------------------------------------

def _linear(op, dtype, M, K, N, activation="none", bias=False, residual=False, w_layout="kn", pad=0):
    """x [M, K] with rows K + pad apart, w [K, N]; w_layout "nk": stored as the [N, K] of a transposed weight."""
    return {"op": op, "dtype": dtype, "M": M, "K": K, "N": N, "activation": activation, "bias": bias,
            "residual": residual, "w_layout": w_layout, "pad": pad}


def _gated(op, dtype, M, K, N, activation="silu", save=False, w_layout="kn"):
    return {"op": op, "dtype": dtype, "M": M, "K": K, "N": N, "activation": activation, "save": save,
            "w_layout": w_layout}


def _norm(op, dtype, M, D, kind="rms", block=True, post=False, gate=False, bias=False, scale=1.0):
    return {"op": op, "dtype": dtype, "M": M, "D": D, "kind": kind, "block": block, "post": post, "gate": gate,
            "bias": bias, "scale": scale}


def listed():
    return [
        # one token of a decoding step through the down projection, joined with the residual stream
        dict(_linear("linear", "bf16", 1, 11008, 4096, residual=True), name="linear 1 token"),
        # the up projection of a plain feed-forward block over a prompt
        dict(_linear("linear", "bf16", 8192, 4096, 16384, "gelu", bias=True), name="linear prompt gelu"),
        # a single-precision layer with a bias, weights stored as [out, in]
        dict(_linear("linear", "f32", 2048, 1024, 4096, "relu", bias=True, w_layout="nk"), name="linear f32"),
        # a training step of the same block on a ragged batch: dx, dw, dbias
        dict(_linear("linear_backward", "f16", 1999, 1096, 4104, "gelu_tanh", bias=True), name="linear backward ragged"),
        # a handful of sequences decoding together: gate and up projections
        dict(_gated("gated_linear", "bf16", 16, 4096, 11008), name="gated 16 tokens"),
        # the same over a training batch, keeping what the backward pass reads
        dict(_gated("gated_linear", "bf16", 8192, 4096, 11008, save=True), name="gated batch"),
        # gradients of that step: dx, dw_gate, dw_up
        dict(_gated("gated_linear_backward", "bf16", 4096, 4096, 11008), name="gated backward"),
        # a small model whose sizes are odd, so that no row starts on a 16-byte boundary
        dict(_gated("gated_linear", "f16", 777, 1023, 2731, "gelu", w_layout="nk"), name="gated odd"),
        # the norm in front of a decoding step's block
        dict(_norm("residual_norm", "bf16", 1, 4096), name="norm 1 token"),
        # the join of a training batch: norm of the block's output, its gate, the residual, the next norm
        dict(_norm("residual_norm", "bf16", 16384, 4096, post=True, gate=True, scale=0.5), name="norm batch"),
        # its gradients
        dict(_norm("residual_norm_backward", "bf16", 16384, 4096, post=True, gate=True, scale=0.5), name="norm backward"),
        # layer norm of a single-precision model of odd width, gradients
        dict(_norm("residual_norm_backward", "f32", 3001, 1023, kind="layer", bias=True), name="layer norm backward odd"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """Any operator, type and layout; 1 to 8192 rows, widths of 64 to 11008 (16384 rows and widths of 16 to 8192
    for the norms), two in five of the widths odd or not a multiple of 8."""
    def width(low, high):
        n = _spread(rng, low, high)
        return n if rng.random() < 0.4 else max(8, n // 8 * 8)

    op = rng.choice(["linear", "linear", "linear_backward", "gated_linear", "gated_linear", "gated_linear_backward",
                     "residual_norm", "residual_norm_backward"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op.startswith("residual_norm"):
        kind = rng.choice(["rms", "layer"])
        block = op.endswith("backward") or rng.random() < 0.8
        M, D = _spread(rng, 1, 16384), width(16, 8192 if dtype != "f32" else 4096)
        while M * D > 16384 * (4096 if dtype != "f32" else 2048):
            M = (M + 1) // 2
        return _norm(op, dtype, M, D, kind, block,
                     block and rng.random() < 0.4, block and rng.random() < 0.4, rng.random() < 0.5,
                     rng.choice([1.0, 0.5, 0.8]) if block else 1.0)
    M, K, N = _spread(rng, 1, 8192), width(64, 8192), width(64, 11008)
    most = 1.0e11 if dtype == "f32" else 6.0e11      # products of all the sizes: less than the largest listed case
    while float(M) * K * N > (most / 4 if op.startswith("gated") else most / 2):
        M = (M + 1) // 2
    layout = rng.choice(["kn", "nk"])
    if op.startswith("gated"):
        return _gated(op, dtype, M, K, N, rng.choice(["silu", "gelu", "gelu_tanh", "relu", "sigmoid"]),
                      op == "gated_linear" and rng.random() < 0.5, layout)
    return _linear(op, dtype, M, K, N, rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu", "sigmoid"]),
                   rng.random() < 0.5, op == "linear" and rng.random() < 0.5, layout, rng.choice([0, 0, 8, 24]))


# ---- inputs ---------------------------------------------------------------------------------

def prepare(case, seed):
    """Activations, pre-activations and gradients N(0, 1); weights N(0, 1) / sqrt(fan-in)."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = TYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0):
        t = torch.empty(shape, device="cuda", dtype=dtype)
        return t.normal_(mean, std, generator=g)

    state = {"case": case}
    M = case["M"]
    if case["op"].startswith("residual_norm"):
        D = case["D"]
        state["weight"] = normal(D, mean=1.0, std=0.1)
        if case["bias"]:
            state["bias"] = normal(D, std=0.1)
        if case["block"]:
            state["block"] = normal(M, D, std=1.5)
        if case["gate"]:
            state["gate"] = normal(D, mean=0.5, std=0.2)
        if case["post"]:
            state["post_weight"] = normal(D, mean=1.0, std=0.1)
        if case["op"] == "residual_norm":
            state["residual"] = normal(M, D, std=2.0)
        else:
            state["sum"] = normal(M, D, std=2.0)
            state["dsum"], state["dnormed"] = normal(M, D), normal(M, D)
            # the row statistics that the forward pass keeps: mean and 1/deviation of sum, then of block
            state["stats"] = torch.cat([_statistics(state["sum"].float(), case["kind"]),
                                        _statistics(state["block"].float(), case["kind"])], dim=1).contiguous()
        return state
    K, N = case["K"], case["N"]

    def weight():
        w = normal(K, N, std=K ** -0.5) if case["w_layout"] == "kn" else normal(N, K, std=K ** -0.5).t()
        return w

    if case["op"].startswith("linear"):
        state["x"] = normal(M, K + case["pad"])[:, :K]
        state["w"] = weight()
        if case["op"] == "linear":
            if case["bias"]:
                state["bias"] = normal(N, std=0.1)
            if case["residual"]:
                state["residual"] = normal(M, N)
        else:
            state["dout"] = normal(M, N)
            if case["activation"] != "none":
                state["pre"] = normal(M, N)
    else:
        state["x"] = normal(M, K)
        state["w_gate"], state["w_up"] = weight(), weight()
        if case["op"] == "gated_linear_backward":
            state["dh"], state["pre_gate"], state["pre_up"] = normal(M, N), normal(M, N), normal(M, N)
    return state


EPS = 1e-6


def _statistics(v, kind):
    """[M, 2]: mean (0 for the root-mean-square norm) and reciprocal deviation of each row."""
    if kind == "layer":
        mean = v.mean(dim=1, keepdim=True)
        return torch.cat([mean, ((v - mean).square().mean(dim=1, keepdim=True) + EPS).rsqrt()], dim=1)
    square = v.square().mean(dim=1, keepdim=True)
    return torch.cat([torch.zeros_like(square), (square + EPS).rsqrt()], dim=1)


# ---- the plain forms ---------------------------------------------------------------------------

SQRT_HALF = math.sqrt(0.5)
TANH_A, TANH_B = math.sqrt(2.0 / math.pi), 0.044715


def _act(z, name):
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * SQRT_HALF))
    if name == "gelu_tanh":
        return z / (1 + torch.exp(-2 * TANH_A * (z + TANH_B * z * z * z)))
    return z


def _dact(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if name == "sigmoid":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 - s)
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * SQRT_HALF)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        s = 1 / (1 + torch.exp(-2 * TANH_A * (z + TANH_B * z * z * z)))
        return s + z * s * (1 - s) * 2 * TANH_A * (1 + 3 * TANH_B * z * z)
    return torch.ones_like(z)


def _plain(state):
    case = state["case"]
    op, dtype = case["op"], TYPES[case["dtype"]]
    f = {k: v.float() for k, v in state.items() if k != "case"}
    if op == "linear":
        z = f["x"] @ f["w"]
        if "bias" in f:
            z = z + f["bias"]
        out = _act(z, case["activation"])
        return (out + f["residual"] if "residual" in f else out).to(dtype)
    if op == "linear_backward":
        dz = f["dout"] * _dact(f["pre"], case["activation"]) if "pre" in f else f["dout"]
        grads = [dz @ f["w"].t(), f["x"].t() @ dz] + ([dz.sum(dim=0)] if case["bias"] else [])
        return tuple(v.to(dtype) for v in grads)
    if op == "gated_linear":
        g, u = f["x"] @ f["w_gate"], f["x"] @ f["w_up"]
        h = _act(g, case["activation"]) * u
        return tuple(v.to(dtype) for v in (h, g, u)) if case["save"] else h.to(dtype)
    if op == "gated_linear_backward":
        g, u, dh = f["pre_gate"], f["pre_up"], f["dh"]
        dg, du = dh * u * _dact(g, case["activation"]), dh * _act(g, case["activation"])
        dx = dg @ f["w_gate"].t() + du @ f["w_up"].t()
        return tuple(v.to(dtype) for v in (dx, f["x"].t() @ dg, f["x"].t() @ du))
    if op == "residual_norm":
        total = f["residual"] * case["scale"]
        if "block" in f:
            t = f["block"]
            if "post_weight" in f:
                sy = _statistics(t, case["kind"])
                t = (t - sy[:, :1]) * sy[:, 1:] * f["post_weight"]
            total = total + (t * f["gate"] if "gate" in f else t)
        st = _statistics(total, case["kind"])
        n = (total - st[:, :1]) * st[:, 1:] * f["weight"]
        n = n + f["bias"] if "bias" in f else n
        return (total.to(dtype), n.to(dtype)) if "block" in f else n.to(dtype)
    # residual_norm_backward
    st, layer = f["stats"], case["kind"] == "layer"

    def norm_grad(v, mean, rstd, dhat):
        hat = (v - mean) * rstd
        d = dhat - hat * (dhat * hat).mean(dim=1, keepdim=True)
        if layer:
            d = d - dhat.mean(dim=1, keepdim=True)
        return hat, d * rstd

    hat, through = norm_grad(f["sum"], st[:, 0:1], st[:, 1:2], f["dnormed"] * f["weight"])
    ds = f["dsum"] + through
    grads = [ds * case["scale"]]
    dt = ds * f["gate"] if "gate" in f else ds
    t = f["block"]
    extra = []
    if "post_weight" in f:
        hat_y, dy = norm_grad(f["block"], st[:, 2:3], st[:, 3:4], dt * f["post_weight"])
        t = hat_y * f["post_weight"]
        extra = [(dt * hat_y).sum(dim=0)]
        grads.append(dy)
    else:
        grads.append(dt)
    grads.append((f["dnormed"] * hat).sum(dim=0))
    if "bias" in f:
        grads.append(f["dnormed"].sum(dim=0))
    if "gate" in f:
        grads.append((ds * t).sum(dim=0))
    return tuple(v.to(dtype) for v in grads + extra)


# ---- one pass -------------------------------------------------------------------------------------

def run(state):
    if not own:
        return _plain(state)
    F = _functional()
    case = state["case"]
    op, get = case["op"], state.get
    if op == "linear":
        return F.linear(get("x"), get("w"), get("bias"), get("residual"), activation=case["activation"])
    if op == "linear_backward":
        dx, dw, db = F.linear_backward(get("dout"), get("x"), get("w"), get("pre"), activation=case["activation"],
                                       bias=case["bias"])
        return (dx, dw, db) if case["bias"] else (dx, dw)
    if op == "gated_linear":
        return F.gated_linear(get("x"), get("w_gate"), get("w_up"), activation=case["activation"], save=case["save"])
    if op == "gated_linear_backward":
        return F.gated_linear_backward(get("dh"), get("x"), get("w_gate"), get("w_up"), get("pre_gate"),
                                       get("pre_up"), activation=case["activation"])
    if op == "residual_norm":
        total, normed = F.residual_norm(get("residual"), get("block"), get("weight"), get("bias"), get("gate"),
                                        get("post_weight"), kind=case["kind"], scale=case["scale"], eps=EPS)
        return (total, normed) if case["block"] else normed
    grads = F.residual_norm_backward(get("dnormed"), get("dsum"), get("sum"), get("stats"), get("weight"),
                                     get("block"), get("gate"), get("post_weight"), kind=case["kind"],
                                     scale=case["scale"], bias=case["bias"])
    return tuple(v for v in grads if v is not None)


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    M = case["M"]
    if case["op"].startswith("residual_norm"):
        D = case["D"]
        vectors = 1 + case["bias"] + case["gate"] + case["post"]
        if case["op"] == "residual_norm":
            return {"bytes": size * (M * D * (4 if case["block"] else 2) + D * vectors), "flops": 10.0 * M * D}
        return {"bytes": size * (M * D * 6 + D * 2 * vectors) + 16 * M, "flops": 20.0 * M * D}
    K, N = case["K"], case["N"]
    if case["op"] == "linear":
        return {"bytes": size * (M * K + K * N + M * N * (1 + case["residual"]) + N * case["bias"]),
                "flops": 2.0 * M * K * N}
    if case["op"] == "linear_backward":
        return {"bytes": size * (2 * M * K + 2 * K * N + M * N * (1 + (case["activation"] != "none")) + N * case["bias"]),
                "flops": 4.0 * M * K * N}
    if case["op"] == "gated_linear":
        return {"bytes": size * (M * K + 2 * K * N + M * N * (3 if case["save"] else 1)), "flops": 4.0 * M * K * N}
    return {"bytes": size * (2 * M * K + 4 * K * N + 3 * M * N), "flops": 8.0 * M * K * N}


# ---- the definition in 64 bits ---------------------------------------------------------------------

def _act64(z, name):
    return {"none": lambda: z, "relu": lambda: z.clamp(min=0), "silu": lambda: z * torch.sigmoid(z),
            "sigmoid": lambda: torch.sigmoid(z), "gelu": lambda: z * torch.special.ndtr(z),
            "gelu_tanh": lambda: z / 2 * (1 + torch.tanh((2 / math.pi) ** 0.5 * (z + 0.044715 * z ** 3)))}[name]()


def _norm64(v, kind):
    centred = v - v.mean(-1, keepdim=True) if kind == "layer" else v
    return centred / torch.sqrt(centred.pow(2).mean(-1, keepdim=True) + EPS)


def exact(case, seed):
    """Gradients by differentiating the forward definition."""
    state = prepare(case, seed)
    d = {k: v.double() for k, v in state.items() if k not in ("case", "stats")}
    op, name = case["op"], case.get("activation")
    if op == "linear":
        out = _act64(torch.matmul(d["x"], d["w"]) + d.get("bias", 0.0), name)
        return out + d.get("residual", 0.0)
    if op == "linear_backward":
        dz = d["dout"]
        if "pre" in d:
            z = d["pre"].requires_grad_(True)
            dz, = torch.autograd.grad(_act64(z, name), z, dz)
        return tuple([torch.matmul(dz, d["w"].mT), torch.matmul(d["x"].mT, dz)] + ([dz.sum(0)] if case["bias"] else []))
    if op == "gated_linear":
        g, u = torch.matmul(d["x"], d["w_gate"]), torch.matmul(d["x"], d["w_up"])
        h = _act64(g, name) * u
        return (h, g, u) if case["save"] else h
    if op == "gated_linear_backward":
        g, u = d["pre_gate"].requires_grad_(True), d["pre_up"].requires_grad_(True)
        dg, du = torch.autograd.grad(_act64(g, name) * u, (g, u), d["dh"])
        return (torch.matmul(torch.cat([dg, du], 1), torch.cat([d["w_gate"], d["w_up"]], 1).mT),
                torch.matmul(d["x"].mT, dg), torch.matmul(d["x"].mT, du))
    if op == "residual_norm":
        total = case["scale"] * d["residual"]
        if case["block"]:
            t = _norm64(d["block"], case["kind"]) * d["post_weight"] if case["post"] else d["block"]
            total = total + d.get("gate", 1.0) * t
        n = _norm64(total, case["kind"]) * d["weight"] + d.get("bias", 0.0)
        return (total, n) if case["block"] else n
    wanted = [k for k in ("block", "weight", "bias", "gate", "post_weight") if k in d]
    leaves = {k: d[k].requires_grad_(True) for k in wanted}
    total = d["sum"].requires_grad_(True)
    ds, dw, *db = torch.autograd.grad(_norm64(total, case["kind"]) * d["weight"] + d.get("bias", 0.0),
                                      [total] + [leaves[k] for k in ("weight", "bias") if k in leaves], d["dnormed"])
    ds = ds + d["dsum"]
    t = _norm64(d["block"], case["kind"]) * d["post_weight"] if case["post"] else d["block"]
    branch = [k for k in ("block", "gate", "post_weight") if k in leaves]
    dy, *rest = torch.autograd.grad(d.get("gate", 1.0) * t, [leaves[k] for k in branch], ds)
    return tuple([case["scale"] * ds, dy, dw] + db + rest)
