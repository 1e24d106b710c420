"""Cases of the dense operators: the linear map with its epilogue and the gated feed-forward block.

    linear   out = residual + scale * act(x W^T + bias)
    ffn      a   = act(x Wg^T) * (x Wu^T)

Each runs as a forward pass alone (``"mode": "fwd"``: serving, a prompt or one token) or as a forward
pass and the gradients of every input that has one (``"mode": "train"``).  With ``own`` false ``run``
computes the plain form in float32; with ``own`` true it calls the library's operators.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}

# A case: op, mode, m rows (tokens), k input features, n output features (the inner width of the ffn), the
# type of x, W and the result; for the linear map also act, bias (float32 or the type, "none" without), scale
# (float32 per output feature), residual ("none", "same": the type, "f32") and out (the result's type);
# xpad: x is a column slice of rows that are xpad elements longer.
LINEAR = {"act": "none", "bias": "none", "scale": False, "residual": "none", "out": "same", "xpad": 0}


def _linear(name, mode, dtype, m, k, n, **more):
    return {"name": name, "op": "linear", "mode": mode, "dtype": dtype, "m": m, "k": k, "n": n, **LINEAR, **more}


def _ffn(name, mode, dtype, m, k, n, act="silu", xpad=0):
    return {"name": name, "op": "ffn", "mode": mode, "dtype": dtype, "m": m, "k": k, "n": n, "act": act, "xpad": xpad}


def listed():
    return [
        # one decoded token through the block's down projection: gate and float32 residual stream in the epilogue
        _linear("linear token", "fwd", "bf16", 1, 1248, 640, scale=True, residual="f32", out="f32"),
        # 48 requests' tokens through the attention layer's stacked input projection (latent, queries, index, gate)
        _linear("linear batch of tokens", "fwd", "bf16", 48, 640, 1544, bias="f32"),
        # a prompt batch (8 x 8192 tokens) through the down projection into the residual stream
        _linear("linear prompt batch", "fwd", "bf16", 65536, 1248, 640, scale=True, residual="f32", out="f32"),
        # a short ragged prompt, odd widths, a slice of a wider buffer
        _linear("linear odd", "fwd", "fp16", 777, 641, 1003, act="gelu", bias="same", residual="same", xpad=3),
        # a float32 parity run of the same projection
        _linear("linear float32", "fwd", "fp32", 4096, 640, 1544, act="silu", bias="f32"),
        # a training step's projection: every gradient, the bias' and the residual gate's among them
        _linear("linear train", "train", "bf16", 16384, 640, 2560, act="silu", bias="same", scale=True, residual="same"),
        # one decoded token through the block
        _ffn("ffn token", "fwd", "bf16", 1, 640, 1248),
        # a short prompt
        _ffn("ffn prompt", "fwd", "bf16", 200, 640, 1728),
        # a prompt batch (8 x 8192 tokens)
        _ffn("ffn prompt batch", "fwd", "bf16", 65536, 640, 1248),
        # a ragged training batch, odd widths
        _ffn("ffn train odd", "train", "fp16", 1001, 650, 1251, act="gelu", xpad=1),
        # a training step of a wide block: the largest
        _ffn("ffn train wide", "train", "bf16", 8192, 2048, 5632),
        # a float32 training step
        _ffn("ffn train float32", "train", "fp32", 2048, 640, 1248),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    while True:
        op = rng.choice(["linear", "ffn"])
        mode = rng.choice(["fwd", "fwd", "train"])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        m = log_int(1, 65536)
        k, n = log_int(64, 4096), log_int(64, 8192)
        if rng.random() < 0.6:  # most layers have widths that are multiples of eight
            k, n = (k + 7) // 8 * 8, (n + 7) // 8 * 8
        xpad = rng.choice([0, 0, 0, 8, 5])
        if op == "linear":
            case = _linear("", mode, dtype, m, k, n, act=rng.choice(["none", "none", "relu", "silu", "gelu"]),
                           bias=rng.choice(["none", "same", "f32"]), scale=rng.random() < 0.4,
                           residual=rng.choice(["none", "same", "f32"]), out=rng.choice(["same", "same", "f32"]), xpad=xpad)
        else:
            case = _ffn("", mode, dtype, m, k, n, act=rng.choice(["silu", "silu", "gelu", "relu"]), xpad=xpad)
        del case["name"]
        w = work(case)
        if w["flops"] <= (1e11 if dtype == "fp32" else 1e12) and w["bytes"] <= 2e9:
            return case


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    m, k, n = case["m"], case["k"], case["n"]

    def randn(*shape, std=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dtype)

    state = {"case": case, "x": randn(m, k + case["xpad"])[:, case["xpad"]:]}  # normalised activations
    if case["op"] == "linear":
        state["w"] = randn(n, k, std=k ** -0.5)
        state["bias"] = None if case["bias"] == "none" else randn(n, std=0.1, dtype=dt if case["bias"] == "same" else torch.float32)
        state["scale"] = torch.sigmoid(randn(n, std=0.3, dtype=torch.float32) + 2.0) if case["scale"] else None
        state["residual"] = None if case["residual"] == "none" else randn(m, n, dtype=dt if case["residual"] == "same" else torch.float32)
        out = dt if case["out"] == "same" else torch.float32
    else:
        state["w_gate"], state["w_up"] = randn(n, k, std=k ** -0.5), randn(n, k, std=k ** -0.5)
        out = dt
    if case["mode"] == "train":
        state["grad"] = randn(m, n, std=0.05, dtype=out)
    return state


# ---------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------
def _act(z, act):
    if act == "relu":
        return torch.where(z <= 0, torch.zeros_like(z), z)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    return torch.ones_like(z)


def _plain_linear(s):
    case, x, w = s["case"], s["x"].float(), s["w"].float()
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _act(z, case["act"])
    out = y if s["scale"] is None else y * s["scale"]
    if s["residual"] is not None:
        out = out + s["residual"].float()
    got = {"out": out.to(DTYPES[case["dtype"]] if case["out"] == "same" else torch.float32)}
    if case["mode"] == "train":
        g = s["grad"].float()
        dy = g if s["scale"] is None else g * s["scale"]
        dz = dy * _act_slope(z, case["act"])
        got["dx"] = (dz @ w).to(s["x"].dtype)
        got["dw"] = (dz.t() @ x).to(s["w"].dtype)
        if s["bias"] is not None:
            got["dbias"] = dz.sum(0).to(s["bias"].dtype)
        if s["scale"] is not None:
            got["dscale"] = (g * y).sum(0)
    return got


def _plain_ffn(s):
    case, x, wg, wu = s["case"], s["x"].float(), s["w_gate"].float(), s["w_up"].float()
    zg, zu = x @ wg.t(), x @ wu.t()
    a = _act(zg, case["act"])
    got = {"out": (a * zu).to(s["x"].dtype)}
    if case["mode"] == "train":
        g = s["grad"].float()
        dg, du = g * zu * _act_slope(zg, case["act"]), g * a
        got["dx"] = (dg @ wg + du @ wu).to(s["x"].dtype)
        got["dw_gate"] = (dg.t() @ x).to(s["w_gate"].dtype)
        got["dw_up"] = (du.t() @ x).to(s["w_up"].dtype)
    return got


# ---------------------------------------------------------------------------
# the library's operators
# ---------------------------------------------------------------------------
def _own_linear(s):
    import maba_v2_architecture_b200 as mb

    case = s["case"]
    out_dtype = None if case["out"] == "same" else torch.float32
    got = {"out": mb.b200_linear(s["x"], s["w"], s["bias"], activation=case["act"], scale=s["scale"],
                                 residual=s["residual"], out_dtype=out_dtype)}
    if case["mode"] == "train":
        dx, dw, dbias, dscale = mb.b200_linear_backward(s["grad"], s["x"], s["w"], s["bias"], activation=case["act"],
                                                        scale=s["scale"])
        got.update(dx=dx, dw=dw)
        if dbias is not None:
            got["dbias"] = dbias
        if dscale is not None:
            got["dscale"] = dscale
    return got


def _own_ffn(s):
    import maba_v2_architecture_b200 as mb

    case = s["case"]
    got = {"out": mb.b200_gated_ffn(s["x"], s["w_gate"], s["w_up"], activation=case["act"])}
    if case["mode"] == "train":
        got["dx"], got["dw_gate"], got["dw_up"] = mb.b200_gated_ffn_backward(s["grad"], s["x"], s["w_gate"], s["w_up"],
                                                                             activation=case["act"])
    return got


def run(state):
    if own:
        return _own_linear(state) if state["case"]["op"] == "linear" else _own_ffn(state)
    return _plain_linear(state) if state["case"]["op"] == "linear" else _plain_ffn(state)


def work(case):
    m, k, n = case["m"], case["k"], case["n"]
    el = 4 if case["dtype"] == "fp32" else 2
    nw = 1 if case["op"] == "linear" else 2
    out_el = 4 if case.get("out") == "f32" else el
    nbytes = (m * k + nw * n * k) * el + m * n * out_el
    flops = 2.0 * m * n * k * nw
    if case["op"] == "linear":
        nbytes += 0 if case["bias"] == "none" else n * (el if case["bias"] == "same" else 4)
        nbytes += 4 * n if case["scale"] else 0
        nbytes += 0 if case["residual"] == "none" else m * n * (el if case["residual"] == "same" else 4)
    if case["mode"] == "train":  # the incoming gradient read, dx and dW (and the vectors') written
        nbytes += m * n * out_el + (m * k + nw * n * k) * el
        if case["op"] == "linear":
            nbytes += 0 if case["bias"] == "none" else n * (el if case["bias"] == "same" else 4)
            nbytes += 4 * n if case["scale"] else 0
        flops *= 3
    return {"bytes": nbytes, "flops": flops}


# ---------------------------------------------------------------------------
# the definition in 64 bits: the gradients by differentiation
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    train = case["mode"] == "train"
    wide = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    names = [k for k in ("x", "w", "bias", "scale", "w_gate", "w_up") if k in wide]
    for k in names if train else ():
        wide[k].requires_grad_(True)
    phi = {"none": lambda z: z, "relu": torch.nn.functional.relu, "silu": torch.nn.functional.silu,
           "gelu": torch.nn.functional.gelu}[case["act"]]
    with torch.enable_grad() if train else torch.no_grad():
        if case["op"] == "linear":
            out = phi(torch.nn.functional.linear(wide["x"], wide["w"], wide.get("bias")))
            if "scale" in wide:
                out = wide["scale"] * out
            if "residual" in wide:
                out = out + wide["residual"]
        else:
            out = phi(torch.nn.functional.linear(wide["x"], wide["w_gate"])) * torch.nn.functional.linear(wide["x"], wide["w_up"])
    got = {"out": out.detach()}
    if train:
        grads = torch.autograd.grad(out, [wide[k] for k in names], wide["grad"])
        got.update({"d" + k: g for k, g in zip(names, grads)})
    return got
