"""The position-wise operators' measured cases: `linear` (matrix product with bias, activation and residual in its epilogue) and
`gated_linear` (both projections of a gated feed-forward block, activation and product in one kernel), forward and training step,
and the block the two make together.

Shapes: x (rows, k); linear's weight (n, k), gated_linear's weight (2 n, k) -- the gate's n rows first, then the n rows of the other
factor.  A case's `kind` is
    linear    y = act(x W^T + b) + r                                                    (infer | train)
    gated     h = act(x Wg^T + bg) * (x Wu^T + bu)                                      (infer | train)
    block     y = gated(x) Wd^T + bd + x, Wd (k, n)                                     (infer | train)
`train` is the forward and the backward pass for a given upstream gradient; it returns the output and every input's gradient.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _case(name, kind, mode, dtype, rows, k, n, act, bias=True, residual=False):
    return {"name": name, "kind": kind, "mode": mode, "dtype": dtype, "rows": rows, "k": k, "n": n, "act": act, "bias": bias, "residual": residual}


def listed():
    return [
        # one new position of a stream: the weights are read once, latency and bandwidth count
        _case("linear_one_row_bf16", "linear", "infer", "bf16", 1, 2048, 2048, "none", residual=True),
        _case("gated_one_row_bf16", "gated", "infer", "bf16", 1, 4096, 8192, "silu", bias=False),
        # a few streams at once, odd sizes: rows that no vector load fits
        _case("gated_few_rows_odd_fp16", "gated", "infer", "fp16", 13, 1003, 1337, "gelu"),
        # the rectification network's own widths at its batch of 32 sequences of 16, trained in fp32
        _case("linear_sequences_train_fp32", "linear", "train", "fp32", 32 * 16, 384, 128, "leaky_relu"),
        # a middling batch: too few output tiles to fill the card by themselves
        _case("linear_batch_fp16", "linear", "infer", "fp16", 200, 4096, 1024, "relu", residual=True),
        # many positions at once, the ordinary wide products
        _case("linear_wide_bf16", "linear", "infer", "bf16", 4096, 4096, 4096, "gelu", residual=True),
        _case("linear_wide_train_fp32", "linear", "train", "fp32", 4096, 1024, 4096, "gelu_tanh"),
        _case("gated_ragged_train_bf16", "gated", "train", "bf16", 2999, 1000, 2504, "sigmoid"),
        _case("gated_wide_fp32", "gated", "infer", "fp32", 2048, 2048, 4096, "silu", bias=False),
        _case("gated_wide_bf16", "gated", "infer", "bf16", 8192, 4096, 8192, "silu", bias=False),
        # the whole block as a model uses it: one training step, and one row of a stream
        _case("block_train_bf16", "block", "train", "bf16", 8192, 2048, 5504, "silu", bias=False),
        _case("block_one_row_fp16", "block", "infer", "fp16", 1, 2048, 5504, "silu", bias=False),
    ]


ACTS = ("none", "leaky_relu", "sigmoid", "relu", "silu", "gelu", "gelu_tanh")


def _log_int(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    v = min(max(v, lo), hi)
    if v >= 64 and rng.random() < 0.6:            # most widths are whole vectors, the rest stay odd
        v = (v + 31) // 32 * 32
    return min(v, hi)


def draw(rng):
    kind = rng.choice(("linear", "gated", "block"))
    mode = rng.choice(("infer", "train"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    rows = rng.choice((_log_int(rng, 1, 64), _log_int(rng, 16, 8192), _log_int(rng, 1024, 8192)))
    k = _log_int(rng, 64, 4096)
    n = _log_int(rng, 64, 6144)
    return {"kind": kind, "mode": mode, "dtype": dtype, "rows": rows, "k": k, "n": n, "act": rng.choice(ACTS if kind == "linear" else ACTS[2:]),
            "bias": rng.random() < 0.5, "residual": kind == "linear" and rng.random() < 0.5}


def _sizes(case):
    return case["rows"], case["k"], case["n"]


def prepare(case, seed):
    rows, k, n = _sizes(case)
    dtype = DTYPES[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)

    def uniform(bound, *shape):
        return ((torch.rand(shape, generator=gen, device="cuda") * 2 - 1) * bound).to(dtype)

    wide = 2 * n if case["kind"] != "linear" else n
    leaves = {"x": normal(rows, k), "w": uniform(1.7 / math.sqrt(k), wide, k)}
    if case["bias"]:
        leaves["b"] = uniform(0.5, wide)
    if case["kind"] == "block":
        leaves["wd"] = uniform(1.7 / math.sqrt(n), k, n)
        if case["bias"]:
            leaves["bd"] = uniform(0.5, k)
    if case["residual"]:
        leaves["r"] = normal(rows, n)
    train = case["mode"] == "train"
    state = {"case": case, **{name: t.requires_grad_(train) for name, t in leaves.items()}, "names": list(leaves)}
    if train:
        state["dy"] = normal(rows, k if case["kind"] == "block" else n, scale=0.1)
    return state


# ------------------------------------------------------------------------------------------ the plain form: elementary operations in 32 bits
def _erf(z):
    return torch.erf(z)


def _act(z, act):
    if act == "none":
        return z
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "leaky_relu":
        return torch.where(z > 0, z, 0.01 * z)
    if act == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-z))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1.0 + _erf(z * math.sqrt(0.5)))
    c = math.sqrt(2.0 / math.pi)
    return 0.5 * z * (1.0 + torch.tanh(c * (z + 0.044715 * z * z * z)))


def _act_grad(z, act):
    if act == "none":
        return torch.ones_like(z)
    if act == "relu":
        return torch.where(z > 0, torch.ones_like(z), torch.zeros_like(z))
    if act == "leaky_relu":
        return torch.where(z > 0, torch.ones_like(z), torch.full_like(z, 0.01))
    if act == "gelu":
        return 0.5 * (1.0 + _erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if act == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * z * z)
    s = 1.0 / (1.0 + torch.exp(-z))
    return s * (1.0 - s) if act == "sigmoid" else s * (1.0 + z * (1.0 - s))


@torch.no_grad()
def _plain(state):
    case = state["case"]
    act, kind, n = case["act"], case["kind"], case["n"]
    dtype = DTYPES[case["dtype"]]
    f = {name: state[name].detach().float() for name in state["names"]}
    z = f["x"] @ f["w"].t()
    if "b" in f:
        z = z + f["b"]
    if kind == "linear":
        y = _act(z, act)
        if "r" in f:
            y = y + f["r"]
    else:
        g, u = z[:, :n], z[:, n:]
        h = _act(g, act) * u
        y = h
        if kind == "block":
            y = h @ f["wd"].t() + f["x"]
            if "bd" in f:
                y = y + f["bd"]
    if case["mode"] == "infer":
        return y.to(dtype)
    dy = state["dy"].float()
    grads = {}
    if kind == "linear":
        dz = dy * _act_grad(z, act)
    else:
        dh = dy
        if kind == "block":
            dh = dy @ f["wd"]
            grads["wd"] = dy.t() @ h
            if "bd" in f:
                grads["bd"] = dy.sum(0)
        dz = torch.cat([dh * u * _act_grad(g, act), dh * _act(g, act)], 1)
    grads["x"] = dz @ f["w"]
    if kind == "block":
        grads["x"] = grads["x"] + dy
    grads["w"] = dz.t() @ f["x"]
    if "b" in f:
        grads["b"] = dz.sum(0)
    if "r" in f:
        grads["r"] = dy
    return {"y": y.to(dtype), **{name: grads[name].to(dtype) for name in state["names"]}}


# ------------------------------------------------------------------------------------------ the framework's calls
def _own(state):
    from tracknetv3_amd import feedforward as ff
    case = state["case"]
    train = case["mode"] == "train"
    with torch.set_grad_enabled(train):
        if case["kind"] == "linear":
            y = ff.linear(state["x"], state["w"], state.get("b"), residual=state.get("r"), act=case["act"])
        elif case["kind"] == "gated":
            y = ff.gated_linear(state["x"], state["w"], state.get("b"), act=case["act"])
        else:
            h = ff.gated_linear(state["x"], state["w"], state.get("b"), act=case["act"])
            y = ff.linear(h, state["wd"], state.get("bd"), residual=state["x"])
    if not train:
        return y
    grads = torch.autograd.grad(y, [state[name] for name in state["names"]], state["dy"])
    return {"y": y.detach(), **dict(zip(state["names"], grads))}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    rows, k, n = _sizes(case)
    size = 4 if case["dtype"] == "fp32" else 2
    wide = n if case["kind"] == "linear" else 2 * n
    weights = wide * k + (wide if case["bias"] else 0)
    products = rows * k * wide
    out = n
    if case["kind"] == "block":
        weights += k * n + (k if case["bias"] else 0)
        products += rows * k * n
        out = k
    elements = rows * k + weights + rows * out + (rows * n if case["residual"] else 0)
    if case["mode"] == "train":               # + the upstream gradient in, the gradients of x, the weights and the residual out
        elements += rows * out + rows * k + weights + (rows * n if case["residual"] else 0)
        products *= 3
    return {"bytes": size * elements, "flops": 2 * products}


# ------------------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    n, act = case["n"], case["act"]
    d = {name: state[name].detach().double().requires_grad_(case["mode"] == "train") for name in state["names"]}
    F = torch.nn.functional
    fn = {"none": lambda t: t, "leaky_relu": lambda t: F.leaky_relu(t, 0.01), "sigmoid": torch.sigmoid, "relu": F.relu, "silu": F.silu,
          "gelu": F.gelu, "gelu_tanh": lambda t: F.gelu(t, approximate="tanh")}[act]
    if case["kind"] == "linear":
        y = fn(F.linear(d["x"], d["w"], d.get("b")))
        y = y + d["r"] if "r" in d else y
    else:
        gate, other = F.linear(d["x"], d["w"], d.get("b")).split(n, dim=1)
        y = fn(gate) * other
        if case["kind"] == "block":
            y = F.linear(y, d["wd"], d.get("bd")) + d["x"]
    if case["mode"] == "infer":
        return y
    grads = torch.autograd.grad(y, [d[name] for name in state["names"]], state["dy"].double())
    return {"y": y.detach(), **dict(zip(state["names"], grads))}
