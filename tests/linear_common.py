"""Shared by the CPU (emulator) and GPU tests of the position-wise layers: 64-bit oracles, element-wise error bounds derived from the types, and the
exact integer cases (operands in {-1, 0, 1} whose sums every type holds exactly: any wrong, missing or doubled index shows)."""
import torch
import torch.nn.functional as F

ACTS = ("none", "leaky_relu", "sigmoid", "relu", "silu", "gelu", "gelu_tanh")
DTYPES = (torch.float32, torch.bfloat16, torch.float16)
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}      # below: absolute instead of relative rounding
LARGEST_EXACT = {torch.float32: 1 << 24, torch.bfloat16: 1 << 8, torch.float16: 1 << 11}


def act64(z, act):
    return {"none": lambda t: t, "leaky_relu": lambda t: F.leaky_relu(t, 0.01), "sigmoid": torch.sigmoid, "relu": F.relu, "silu": F.silu, "gelu": F.gelu,
            "gelu_tanh": lambda t: F.gelu(t, approximate="tanh")}[act](z)


def oracle(x, w, b=None, r=None, act="none", gated=False, dy=None):
    """{y, z[, dz, x, w, b, r gradients]} in float64 on the CPU."""
    d = {k: t.detach().cpu().double().requires_grad_() for k, t in (("x", x), ("w", w), ("b", b), ("r", r)) if t is not None}
    z = F.linear(d["x"], d["w"], d.get("b"))
    z.retain_grad()
    if gated:
        g, u = z.chunk(2, -1)
        y = act64(g, act) * u
    else:
        y = act64(z, act)
        y = y + d["r"] if "r" in d else y
    out = {"y": y.detach(), "z": z.detach()}
    if dy is not None:
        y.backward(dy.cpu().double())
        out["dz"] = z.grad
        out.update({"d" + k: t.grad for k, t in d.items()})
    return out


# |act''| <= 1.2 and |act'| <= 1.13 for every activation of ACTS away from the kinks of relu / leaky_relu
L1, L2 = 1.13, 1.2


def bounds(x, w, b, r, act, gated, dy, dtype):
    """Largest allowed |error| per element of y and the gradients, from: inputs exact; sums in fp32 (a chain of at most 6 / 16 roundings per term
    of the contraction plus 64, and 2^-23 per term left out of the fp32 split); the activation within 2^-18 of its scale; one rounding of
    z, dz and each output to the type."""
    u, tiny = HALF_STEP[dtype], TINY[dtype]
    o = oracle(x, w, b, r, act, gated, dy)
    x64, w64 = x.detach().cpu().double().abs(), w.detach().cpu().double().abs()
    x2 = x64.reshape(-1, x64.shape[-1])

    def chain(terms):
        return (6 * terms / 16 + 64) * 2.0 ** -24 + 2.0 ** -23

    e_act = 2.0 ** -18 if dtype != torch.float32 else 2.0 ** -21
    z = o["z"].abs().reshape(-1, w64.shape[0])
    ez = chain(x2.shape[1]) * (x2 @ w64.t() + (0 if b is None else b.detach().cpu().double().abs()))          # of the fp32 sum
    y = o["y"].abs().reshape(z.shape[0], -1)
    out = {}
    if gated:
        g, uu = z.chunk(2, -1)
        eg, eu = ez.chunk(2, -1)
        a = g + 1
        out["y"] = u * y + tiny + (L1 * eg + e_act * a) * (uu + eu) + a * eu
    else:
        rr = 0 if r is None else r.detach().cpu().double().abs().reshape(y.shape)
        out["y"] = u * y + tiny + L1 * ez + e_act * (z + 1) + 2.0 ** -23 * (z + rr)
    if dy is None:
        return out
    d = dy.cpu().double().abs().reshape(y.shape)
    ezs = ez + (2.0 ** -24 if gated else u) * z + tiny       # of the pre-activation as it is kept: fp32 / the type
    if gated:
        g, uu = z.chunk(2, -1)
        eg, eu = ezs.chunk(2, -1)
        edz = torch.cat([d * (L1 * eu + (L2 * eg + e_act * (g + 1)) * (uu + eu)), d * (L1 * eg + e_act * (g + 1))], -1)
        act_pass = True
    else:
        act_pass = act != "none"
        edz = d * (L2 * ezs + e_act * (z + 1)) if act_pass else torch.zeros_like(z)
    dz = o["dz"].abs().reshape(z.shape)
    edb = edz + 2.0 ** -23 * dz
    if act_pass:
        edz = edz + (u + 2.0 ** -23) * dz + tiny
    rows = z.shape[0]
    out["dx"] = (edz + chain(z.shape[1]) * (dz + edz)) @ w64 + u * o["dx"].abs().reshape(x2.shape) + tiny
    out["dw"] = (edz + chain(rows) * (dz + edz)).t() @ x2 + u * o["dw"].abs() + tiny
    if b is not None:
        out["db"] = (edb + chain(rows) * (dz + edb)).sum(0) + u * o["db"].abs() + tiny
    return out


def make(rows, k, n, dtype, gated=False, bias=True, residual=False, seed=0, device="cpu", scale=1.0):
    g = torch.Generator().manual_seed(seed)
    wide = 2 * n if gated else n
    x = (torch.randn(rows, k, generator=g) * scale).to(dtype).to(device)
    w = (torch.randn(wide, k, generator=g) / k ** 0.5).to(dtype).to(device)
    b = torch.randn(wide, generator=g).to(dtype).to(device) if bias else None
    r = torch.randn(rows, n, generator=g).to(dtype).to(device) if residual else None
    dy = torch.randn(rows, n, generator=g).to(dtype).to(device)
    return x, w, b, r, dy


def run(x, w, b, r, act, gated, dy):
    """The framework's forward and backward: {y, dx, dw[, db, dr]}."""
    from tracknetv3_amd import feedforward as ff
    leaves = {k: t.detach().requires_grad_() for k, t in (("x", x), ("w", w), ("b", b), ("r", r)) if t is not None}
    if gated:
        y = ff.gated_linear(leaves["x"], leaves["w"], leaves.get("b"), act=act)
    else:
        y = ff.linear(leaves["x"], leaves["w"], leaves.get("b"), residual=leaves.get("r"), act=act)
    grads = torch.autograd.grad(y, list(leaves.values()), dy)
    return {"y": y.detach(), **{"d" + k: g for k, g in zip(leaves, grads)}}


def check_close(rows, k, n, dtype, act, gated, bias, residual, device, seed=0):
    x, w, b, r, dy = make(rows, k, n, dtype, gated, bias, residual, seed, device)
    got = run(x, w, b, r, act, gated, dy)
    if act in ("relu", "leaky_relu"):
        # away from the kink: a sum within its own error of 0 has no determined derivative
        z = oracle(x, w, b, r, act, gated)["z"]
        z = z.chunk(2, -1)[0] if gated else z
        assert (z.abs() > 1e-6).all()
    want, tol = oracle(x, w, b, r, act, gated, dy), bounds(x, w, b, r, act, gated, dy, dtype)
    for name, limit in tol.items():
        err = (got[name].cpu().double() - want[name]).abs().reshape(limit.shape)
        assert torch.isfinite(got[name]).all(), name
        worst = (err / limit).max().item()
        assert worst <= 1.0, (name, worst, err.max().item())
    if r is not None:
        assert torch.equal(got["dr"], dy)


def sparse_signs(shape, density, gen):
    return torch.randint(0, 2, shape, generator=gen) * 2.0 - 1.0 if density >= 1 else \
        (torch.rand(shape, generator=gen) < density).float() * (torch.randint(0, 2, shape, generator=gen) * 2.0 - 1.0)


def check_exact(rows, k, n, dtype, gated, bias, residual, device, act="relu", seed=0):
    """Integer operands: every sum, product and rounding is exact, so the results are equal to the oracle's.  Densities keep the sums far below the
    largest integer up to which the type holds all."""
    g = torch.Generator().manual_seed(seed)
    wide = 2 * n if gated else n

    def density(terms):                   # about 12 nonzero products at most, each of size 1
        return min(1.0, (12.0 / terms) ** 0.5)

    # two factors of a product share the density of its length; the longest contraction decides
    p = density(max(rows, k, wide))
    x = sparse_signs((rows, k), max(p, density(k)), g)
    w = sparse_signs((wide, k), max(p, density(k)), g)
    dy = sparse_signs((rows, n), min(p, density(max(rows, wide))), g)
    b = torch.randint(-2, 3, (wide,), generator=g).float() if bias else None
    r = torch.randint(-2, 3, (rows, n), generator=g).float() if residual else None
    act = "none" if act == "none" else "relu"
    want = oracle(x, w, b, r, act, gated, dy)
    lim = LARGEST_EXACT[dtype]
    assert all(v.abs().max() <= lim for v in want.values()), {q: v.abs().max().item() for q, v in want.items()}
    cast = [None if t is None else t.to(dtype).to(device) for t in (x, w, b, r, dy)]
    got = run(*cast[:4], act, gated, cast[4])
    for name, v in got.items():
        assert torch.equal(v.cpu().double(), want[name]), (name, (v.cpu().double() != want[name]).nonzero()[:4].tolist())
    return cast, want


def check_exact_subsets(rows, k, n, dtype, gated, device):
    from tracknetv3_amd import ops
    (x, w, b, _, dy), want = check_exact(rows, k, n, dtype, gated, True, False, device)
    act = ops.ACT_RELU
    _, pre = ops.gated_linear(x, w, b, act, want_pre=True) if gated else ops.linear(x, w, b, None, act, want_pre=True)
    call = ops.gated_linear_backward if gated else ops.linear_backward
    for mask in range(1, 8):
        asked = [bool(mask & 1), bool(mask & 2), bool(mask & 4)]
        for name, on, g in zip(("dx", "dw", "db"), asked, call(dy, x, w, pre, act, asked)):
            assert (g is None) == (not on)
            assert g is None or torch.equal(g.cpu().double(), want[name]), (name, asked)


def check_nan_stays_in_place(rows, k, n, dtype, gated, device, seed=0):
    """A NaN row of x, of dy or of the weight reaches the results that it enters and leaves every other one as it was, to the bit: nothing of a
    neighbouring row is read into a product, nothing is multiplied by a zero that stands for "not there"."""
    act = "silu"
    x, w, b, _, dy = make(rows, k, n, dtype, gated, True, False, seed, device)
    clean = run(x, w, b, None, act, gated, dy)
    for r in sorted({0, rows // 2, rows - 1}):
        others = torch.arange(rows, device=device) != r
        bad = x.clone()
        bad[r] = float("nan")
        got = run(bad, w, b, None, act, gated, dy)
        assert torch.isnan(got["y"][r]).all() and torch.isnan(got["dx"][r]).all() and torch.isnan(got["dw"]).all()
        assert torch.equal(got["y"][others], clean["y"][others]) and torch.equal(got["dx"][others], clean["dx"][others]), ("x", r)
        bad = dy.clone()
        bad[r] = float("nan")
        got = run(x, w, b, None, act, gated, bad)
        assert torch.equal(got["y"], clean["y"]) and torch.equal(got["dx"][others], clean["dx"][others]), ("dy", r)
        assert torch.isnan(got["dx"][r]).all() and torch.isnan(got["dw"]).all() and torch.isnan(got["db"]).all()
    wide = w.shape[0]
    for j in sorted({0, n - 1, wide - 1}):
        others = torch.arange(wide, device=device) != j
        if gated:
            others = others & (torch.arange(wide, device=device) % n != j % n)        # the pair's other row sees the NaN in its factor
        bad = w.clone()
        bad[j] = float("nan")
        got = run(x, bad, b, None, act, gated, dy)
        cols = torch.arange(n, device=device) != j % n
        assert torch.isnan(got["y"][:, j % n]).all() and torch.equal(got["y"][:, cols], clean["y"][:, cols]), ("w", j)
        assert torch.isnan(got["dx"]).all() and torch.isnan(got["dw"][j % n]).all()         # (gated: act'(g) u, whichever is NaN)
        assert torch.equal(got["dw"][others], clean["dw"][others]) and torch.equal(got["db"][others], clean["db"][others]), ("w", j)


def check_sigmoid_derivative(dtype, device):
    """sigmoid'(z) = s(z) s(-z) falls by e per unit on BOTH sides; 1 - s would be 0 from z = 17 on.  One row, W = 0, z = the bias; bounds as in
    check_far_gates."""
    u, k = HALF_STEP[dtype], 8
    b = torch.tensor([-60.0, -30.0, -17.0, -8.0, 0.0, 8.0, 12.0, 17.0, 30.0, 60.0]).to(dtype)
    scale = 1024.0 if dtype == torch.float16 else 1.0                  # (keeps fp16's results normal a little longer)
    x, w, dy = torch.ones(1, k, dtype=dtype), torch.zeros(len(b), k, dtype=dtype), torch.full((1, len(b)), scale, dtype=dtype)
    got = run(*(t.to(device) for t in (x, w, b)), None, "sigmoid", False, dy.to(device))["db"].cpu().double()
    want = scale * torch.sigmoid(b.double()) * torch.sigmoid(-b.double())              # (autograd's s (1 - s) cancels in 64 bits too: 0 at 60)
    assert ((got - want).abs() <= (2 * u + 2.0 ** -15) * want + TINY[dtype]).all(), (got.tolist(), want.tolist())


FAR_GATES = (-30.0, -70.0, -100.0, -1e3, -6e4, -1e20, -1e30, -3e38, 30.0, 70.0, 1e3, 6e4)


def check_far_gates(act, dtype, device):
    """Gates far from 0 (masks, large biases): one row, W = 0, so g and u are the biases; dh = 1, x = 1.  du = dh act(g) must be what the forward pass
    multiplies with, dg = dh u act'(g) the derivative there.  Bounds: the exponential's argument carries |g| 2^-24 and the function 2^-21, so 2^-15
    relative at |g| <= 128; below, either side is 0 to within 128 times the least normal number; one rounding to the type for dz and one for each
    result."""
    u, k = HALF_STEP[dtype], 8
    gates = torch.tensor([g for g in FAR_GATES if abs(g) <= torch.finfo(dtype).max], dtype=torch.float64).to(dtype)
    n = len(gates)
    b = torch.cat([gates, torch.full((n,), 1.5).to(dtype)])
    x, w, dy = torch.ones(1, k, dtype=dtype), torch.zeros(2 * n, k, dtype=dtype), torch.ones(1, n, dtype=dtype)
    got = {q: v.cpu().double() for q, v in run(*(t.to(device) for t in (x, w, b)), None, act, True, dy.to(device)).items()}
    want = oracle(x, w, b, None, act, True, dy)
    if act == "sigmoid":                                               # (autograd's s (1 - s) cancels in 64 bits too)
        dg = 1.5 * torch.sigmoid(gates.double()) * torch.sigmoid(-gates.double())
        want["db"][:n], want["dw"][:n] = dg, dg[:, None].expand(n, k)
    floor = 2 * max(TINY[dtype], 128 * 2.0 ** -126)
    for name, rel in (("y", u + 2.0 ** -15), ("db", 2 * u + 2.0 ** -15), ("dw", 2 * u + 2.0 ** -15)):
        fits = want[name].abs() <= torch.finfo(dtype).max              # 1.5 * 6e4 is beyond fp16's largest: infinite
        assert torch.equal(torch.isfinite(got[name]), fits), name
        err = (got[name] - want[name]).abs()
        assert (err <= rel * want[name].abs() + floor)[fits].all(), (name, got[name].tolist(), want[name].tolist())
    # the same activation in both directions: y = 1.5 act(g), db's second half act(g)
    fits = torch.isfinite(got["y"][0])
    assert ((got["y"][0] - 1.5 * got["db"][n:]).abs() <= 4 * u * got["y"][0].abs() + 2 * floor)[fits].all()


def check_gelu_tail(act, dtype, device):
    """GELU and its derivative for z in [-10, -3], RELATIVE: y is a product z Phi(z), and Phi is known to its own rounding there.  One row, W = 0, z = the
    bias.  The exponent (up to 87 in the tanh form, after four roundings) carries 87 * 4 * 2^-24, the fitted factor 2^-17: 2^-14 together, and Phi + z phi
    amplifies it by at most (z^2 + 1) / (z^2 - 1) <= 1.25."""
    u, k = HALF_STEP[dtype], 8
    b = torch.linspace(-10.0, -3.0, 57).to(dtype)
    z = b.double()
    if act == "gelu":
        p, dp = 0.5 * torch.special.erfc(-z / 2 ** 0.5), torch.exp(-0.5 * z * z) / (2 * torch.pi) ** 0.5
    else:                                                              # (1 + tanh a) / 2 = sigmoid(2 a)
        c = (2 / torch.pi) ** 0.5
        a = 2 * c * (z + 0.044715 * z ** 3)
        p = torch.sigmoid(a)
        dp = p * torch.sigmoid(-a) * 2 * c * (1 + 3 * 0.044715 * z * z)
    want = {"y": (z * p)[None], "db": p + z * dp}
    x, w, dy = torch.ones(1, k, dtype=dtype), torch.zeros(len(b), k, dtype=dtype), torch.ones(1, len(b), dtype=dtype)
    got = run(*(t.to(device) for t in (x, w, b)), None, act, False, dy.to(device))
    for name, rel in (("y", u + 2.0 ** -14), ("db", 2 * u + 2.0 ** -13)):
        err = (got[name].cpu().double() - want[name]).abs()
        assert (err <= rel * want[name].abs() + TINY[dtype]).all(), (name, (err / want[name].abs()).tolist())


def check_least_positive(rows, k, n, act, device):
    """fp16: a positive pre-activation below the type's least subnormal has the derivative 1, not that of 0.  z = 2^-14 * 2^-13 in every element (exact),
    so y rounds to 0 while dz = dy."""
    x, w = torch.zeros(rows, k, dtype=torch.float16), torch.zeros(n, k, dtype=torch.float16)
    x[:, -1], w[:, -1] = 2.0 ** -14, 2.0 ** -13
    dy = torch.ones(rows, n, dtype=torch.float16)
    got = run(x.to(device), w.to(device), torch.zeros(n, dtype=torch.float16, device=device), None, act, False, dy.to(device))
    assert not got["y"].any()
    assert (got["db"].cpu() == rows).all() and (got["dx"][:, -1].cpu().double() == n * 2.0 ** -13).all()


# Every product kernel by sizes that are planned on it: (16-bit types?, gated, which: 0 forward, 1 both gradients, tile: 0 64 x 64, 1 128 x 128 with four LDS
# stages, 2 128 x 128 / fp32 128 x 64, 3 256 x 256 / fp32 256 x 128, contraction in parts?, sizes).  For the emulator's CU count (first column) and the card's 256.
KERNELS_EMU = [
    (1, True, False, 0, 0, False, (65, 40, 40)), (1, True, False, 0, 1, False, (65, 200, 72)), (1, True, False, 0, 2, False, (65, 40, 72)),
    (1, True, False, 0, 3, False, (130, 264, 136)), (2, True, True, 0, 0, False, (65, 40, 40)), (1, True, True, 0, 1, False, (65, 200, 40)),
    (1, True, True, 0, 2, False, (65, 40, 40)), (1, True, True, 0, 3, False, (130, 264, 72)),
    (4, True, False, 1, 1, False, (257, 40, 40)), (4, True, False, 1, 2, True, (200, 40, 40)), (4, True, False, 1, 3, False, (130, 264, 136)),
    (4, True, False, 1, 3, True, (130, 136, 392)), (4, True, True, 1, 1, False, (65, 40, 136)), (2, True, True, 1, 2, True, (65, 40, 520)),
    (4, True, True, 1, 3, True, (130, 136, 200)),
    (1, False, False, 0, 2, False, (65, 40, 40)), (2, False, False, 0, 2, True, (65, 136, 40)), (1, False, False, 0, 3, False, (130, 72, 72)),
    (4, False, True, 0, 2, True, (65, 136, 40)), (1, False, True, 0, 3, False, (130, 72, 40)),
    (4, False, False, 1, 2, True, (130, 40, 40)), (1, False, False, 1, 3, False, (130, 72, 136)), (1, False, False, 1, 3, True, (130, 72, 520)),
    (1, False, True, 1, 2, True, (65, 40, 200)), (4, False, True, 1, 3, True, (130, 72, 136)),
]
KERNELS_GPU = [(256,) + e for e in (
    (True, False, 0, 0, True, (65, 776, 72)), (True, False, 0, 1, False, (1500, 200, 2056)), (True, False, 0, 1, True, (65, 4104, 4104)),
    (True, False, 0, 2, False, (1500, 40, 2056)), (True, False, 0, 2, True, (2500, 4104, 776)), (True, False, 0, 3, False, (3001, 264, 4104)),
    (True, True, 0, 0, True, (65, 776, 72)), (True, True, 0, 1, False, (260, 200, 5000)), (True, True, 0, 1, True, (65, 2056, 4104)),
    (True, True, 0, 2, False, (260, 40, 5000)), (True, True, 0, 2, True, (200, 4104, 4104)), (True, True, 0, 3, False, (4100, 72, 5000)),
    (True, False, 1, 1, True, (200, 40, 4104)), (True, False, 1, 2, True, (200, 40, 72)), (True, False, 1, 3, False, (1500, 4104, 1544)),
    (True, False, 1, 3, True, (4100, 1544, 520)), (True, True, 1, 1, True, (65, 40, 4104)), (True, True, 1, 2, True, (200, 40, 72)),
    (True, True, 1, 3, False, (1500, 4104, 776)), (True, True, 1, 3, True, (65, 4104, 4104)),
    (False, False, 0, 2, True, (65, 136, 72)), (False, False, 0, 3, False, (1500, 72, 4104)), (False, False, 0, 3, True, (130, 2056, 4104)),
    (False, True, 0, 2, True, (65, 136, 72)), (False, True, 0, 3, False, (520, 72, 5000)), (False, True, 0, 3, True, (130, 520, 4104)),
    (False, False, 1, 2, True, (65, 40, 136)), (False, False, 1, 3, False, (520, 4104, 520)), (False, False, 1, 3, True, (130, 520, 4104)),
    (False, True, 1, 2, True, (65, 40, 72)), (False, True, 1, 3, False, (520, 4104, 264)), (False, True, 1, 3, True, (130, 520, 2056)))]


def check_kernel(half, gated, rows, k, n, device, exact_only=False):
    """One kernel of KERNELS_*: bias, activation, residual and a kept pre-activation in the epilogue; real values against the bounds, integers exactly, and in
    fp32 integers that fill all three planes."""
    if exact_only:
        check_exact(rows, k, n, torch.bfloat16 if half else torch.float32, gated, bias=True, residual=not gated, device=device, seed=rows + n)
        return
    for dtype in ((torch.bfloat16, torch.float16) if half else (torch.float32,)):
        check_close(rows, k, n, dtype, "silu", gated, bias=True, residual=not gated, device=device, seed=rows + k + n)
        check_exact(rows, k, n, dtype, gated, bias=True, residual=not gated, device=device, seed=rows + n)
        if dtype == torch.float32:
            check_exact_planes(rows, k, n, gated, device)


def check_exact_planes(rows, k, n, gated, device):
    """fp32 products of integers of up to 24 bits: three planes on one side, or two on both, so that every one of the six plane products carries part of the
    result.  All sums of absolute values stay within 2^24: exact in any order, so the results are equal."""
    gen = torch.Generator().manual_seed(rows + k + n)

    def integers(shape, bits, density):
        v = torch.randint(1, 1 << bits, shape, generator=gen) * (torch.randint(0, 2, shape, generator=gen) * 2 - 1) if bits else \
            torch.randint(0, 2, shape, generator=gen) * 2 - 1
        return (v * (torch.rand(shape, generator=gen) < density)).double()
    for bits_x, bits_w in ((20, 0), (0, 20), (10, 10)):
        # x, w and dy meet pairwise over k, n and rows; about 1.5 products per sum, of up to 2^20
        p = (1.5 / max(k, n, rows)) ** 0.5
        x, w, dy = integers((rows, k), bits_x, p), integers((n, k), bits_w, p), integers((rows, n), 0, p)
        if gated:                             # u = 1 by a column of its own: h = g
            x[:, 0], w[:, 0] = 1, 0
            up = torch.zeros(n, k, dtype=torch.float64)
            up[:, 0] = 1
            got = ops_call("gated_linear", x, torch.cat([w, up]), device)
            assert (x.abs() @ w.abs().t()).max() <= 1 << 24
            assert torch.equal(got, x @ w.t()), (bits_x, bits_w)
            continue
        sums = [(x, w.t()), (dy, w), (dy.t(), x)]
        assert all((a.abs() @ b.abs()).max() <= 1 << 24 for a, b in sums)
        y = ops_call("linear", x, w, device)
        dx, dw, _ = ops_call("linear_backward", dy, x, w, device)
        for name, got, (a, b) in zip(("y", "dx", "dw"), (y, dx, dw), sums):
            assert torch.equal(got, a @ b), (name, bits_x, bits_w, (got != a @ b).nonzero()[:4].tolist())


def ops_call(name, *args):
    """ops.<name> of float64 tensors in fp32 on the device that comes last, without an activation; float64 results."""
    from tracknetv3_amd import ops
    out = getattr(ops, name)(*(t.float().to(args[-1]) for t in args[:-1]), act=ops.ACT_NONE)
    return tuple(t if t is None else t.cpu().double() for t in out) if isinstance(out, tuple) else out.cpu().double()


def check_nonfinite_products(rows, k, n, device, seed=0):
    """fp32, all three products (y = x w^T, dx = dy w, dw = dy^T x), with infinities of either sign, NaN and values beyond bf16's largest in either operand:
    NaN, infinities and their signs where fp32 arithmetic has them, the finite rest to its usual accuracy."""
    from tracknetv3_amd import ops
    inf, nan, big = float("inf"), float("nan"), 3.4e38
    for where in ("x", "w", "dy"):
        gen = torch.Generator().manual_seed(seed + rows + n)
        t = {"x": torch.randn(rows, k, generator=gen), "w": torch.randn(n, k, generator=gen), "dy": torch.randn(rows, n, generator=gen)}
        # beyond bf16's largest: only products with factors of at most 1/8 in size, so that no sum of them passes fp32's largest
        for q in t:
            t[q] = t[q].clamp(-4, 4) if q == where else t[q].clamp(-4, 4) / 64
        a, b = t[where].shape
        for at, v in (((1, 3), inf), ((2, 7), -inf), ((3, 2), nan), ((4, 0), big), ((a - 1, b - 1), -inf), ((a // 2, b // 2), -big)):
            t[where][at] = v
        for q in t:                            # inf * 0 = NaN
            if q != where:
                t[q][5, 3] = t[q][3, 5] = 0.0
        x, w, dy = (t[q].to(device) for q in ("x", "w", "dy"))
        y = ops.linear(x, w)
        dx, dw, _ = ops.linear_backward(dy, x, w)
        for name, got, (p, q) in (("y", y, ("x", "wt")), ("dx", dx, ("dy", "w")), ("dw", dw, ("dyt", "x"))):
            p, q = ((t[s[:-1]].t() if s.endswith("t") else t[s]).double() for s in (p, q))
            want, got = (p @ q).float(), got.cpu()
            assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want)), (where, name)
            at = torch.isinf(want)
            assert torch.equal(torch.sign(got[at]), torch.sign(want[at])), (where, name)
            ok = torch.isfinite(want)
            # a finite sum: the chain's roundings and the split's 2^-23 per term, relative to the sum of the sizes
            size = torch.where(torch.isfinite(p), p, 0.0).abs() @ torch.where(torch.isfinite(q), q, 0.0).abs()
            limit = ((6 * p.shape[1] / 16 + 64) * 2.0 ** -24 + 2.0 ** -23) * size + 2.0 ** -126
            assert ((got.double() - p @ q).abs()[ok] <= limit[ok]).all(), (where, name)
