"""CPU: the position-wise layers (linear, gated_linear and their backward passes) on the host SIMT emulator -- index arithmetic, tails and write-out
of the unchanged kernels -- and the refusals of their entry points."""
import ctypes

import pytest
import torch

import linear_common as lc
from tracknetv3_amd import _lib, feedforward as ff, ops


@pytest.mark.parametrize("dtype", lc.DTYPES)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows,k,n", [(1, 1, 1), (1, 64, 32), (3, 5, 7), (17, 72, 40), (33, 129, 65), (5, 200, 20), (66, 70, 33), (67, 33, 66), (130, 40, 136)])
def test_exact_integers(emu, rows, k, n, gated, dtype):
    lc.check_exact(rows, k, n, dtype, gated, bias=True, residual=not gated, device="cpu", seed=rows + k)


@pytest.mark.parametrize("dtype", lc.DTYPES)
@pytest.mark.parametrize("gated,act", [(False, a) for a in lc.ACTS] + [(True, a) for a in lc.ACTS if a != "none"])
def test_activations_and_gradients(emu, act, gated, dtype):
    lc.check_close(9, 40, 24, dtype, act, gated, bias=True, residual=not gated, device="cpu", seed=3)


def test_no_bias_no_residual_and_leading_shape(emu):
    x = torch.randn(2, 3, 16)
    w = torch.randn(8, 16) / 4
    y = ff.linear(x, w)
    assert y.shape == (2, 3, 8) and torch.allclose(y, x @ w.t(), atol=1e-6)
    h = ff.gated_linear(x.transpose(0, 1), w)                     # not contiguous: copied by the differentiable entry
    assert h.shape == (3, 2, 4)


def test_split_contraction_joins_all_parts(emu, monkeypatch):
    """Few rows and a long contraction: the parts' partial sums are joined."""
    lib = _lib.load()
    assert lib.tnv3_linear_forward_workspace_bytes(70, 1100, 24, 0) > 0
    for dtype in lc.DTYPES:
        lc.check_exact(70, 1100, 24, dtype, False, True, True, "cpu")
        lc.check_exact(70, 1100, 24, dtype, True, True, False, "cpu")


@pytest.mark.parametrize("lazy", ["0", "1"])
@pytest.mark.parametrize("rows,k,n", [(17, 4104, 40), (40, 2104, 24), (64, 2100, 72), (64, 2104, 72)])
def test_few_rows_of_a_long_contraction(emu, monkeypatch, rows, k, n, lazy):
    """Up to 64 rows on tiles: steps of fewer elements than stages, of as many and of more."""
    monkeypatch.setenv("TNV3_EMU_LAZY_DMA", lazy)
    # parts to join: not the few-rows kernel, which wins where the tiles would need a copy into whole pieces
    assert (_lib.load().tnv3_linear_forward_workspace_bytes(rows, k, n, 1) > 0) == (k % 8 == 0)
    for cus in ("256", "8", "1"):
        monkeypatch.setenv("TNV3_EMU_CUS", cus)
        for dtype in lc.DTYPES:
            lc.check_exact(rows, k, n, dtype, False, True, True, "cpu")
        lc.check_exact(rows, k, n, torch.bfloat16, True, True, False, "cpu")


@pytest.mark.parametrize("lazy", ["0", "1"])
@pytest.mark.parametrize("cus", ["1", "256"])
def test_direct_loads_land_before_they_are_read(emu, monkeypatch, cus, lazy):
    """16-bit operands that move by direct loads: pieces landing as early or as late as the program's waits allow; one CU makes the wide tiles
    the choice."""
    monkeypatch.setenv("TNV3_EMU_CUS", cus)
    monkeypatch.setenv("TNV3_EMU_LAZY_DMA", lazy)
    for dtype in lc.DTYPES:
        lc.check_exact(70, 200, 264, dtype, False, True, True, "cpu")
        lc.check_exact(130, 264, 136, dtype, True, True, False, "cpu")
        lc.check_exact(75, 131, 69, dtype, True, True, False, "cpu")


@pytest.mark.parametrize("cus", ["1", "256"])
def test_fp32_keeps_infinities_and_nan_where_they_belong(emu, monkeypatch, cus):
    monkeypatch.setenv("TNV3_EMU_CUS", cus)
    inf, nan = float("inf"), float("nan")
    x = torch.randn(5, 40)
    w = torch.randn(6, 40)
    x[1, 3], x[2, 7], x[3, 2], x[4, 0] = inf, -inf, nan, 3.4e38       # 3.4e38: beyond bf16's largest, finite in fp32
    w[:, 0] = torch.tensor([0.25, -0.25, 0.5, -0.5, 0.125, 0.0])
    w[5, 3] = 0.0                                                     # inf * 0 = NaN
    y = ff.linear(x, w)
    want = (x.double() @ w.double().t()).float()
    assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(torch.isinf(y), torch.isinf(want))
    ok = torch.isfinite(want)
    assert torch.allclose(y[ok], want[ok], rtol=1e-5, atol=1e-5)
    assert torch.equal(torch.sign(y[torch.isinf(want)]), torch.sign(want[torch.isinf(want)]))


@pytest.mark.parametrize("dtype", lc.DTYPES)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows,k,n", [(1, 5, 3), (6, 70, 9), (19, 33, 17), (70, 67, 35), (66, 136, 72)])
def test_nan_stays_in_its_row(emu, rows, k, n, gated, dtype):
    lc.check_nan_stays_in_place(rows, k, n, dtype, gated, "cpu")


def test_zero_rows(emu):
    x = torch.zeros(0, 12, requires_grad=True)
    w = torch.randn(10, 12, requires_grad=True)
    b = torch.randn(10, requires_grad=True)
    for y in (ff.linear(x, w, b, act="gelu"), ff.gated_linear(x, w, b)):
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
        assert dx.shape == (0, 12) and not dw.any() and not db.any()


def test_only_the_gradients_that_are_wanted(emu):
    x, w, b, r, dy = lc.make(6, 24, 16, torch.float32, residual=True)
    w.requires_grad_()
    y = ff.linear(x, w, b, r, act="silu")
    (dw,) = torch.autograd.grad(y, (w,), dy)
    want = lc.oracle(x, w, b, r, "silu", False, dy)["dw"]
    assert torch.allclose(dw.double(), want, atol=1e-5)
    r.requires_grad_()
    y = ff.linear(x, w.detach(), b, r)
    (dr,) = torch.autograd.grad(y, (r,), dy)
    assert torch.equal(dr, dy)


@pytest.mark.parametrize("dtype", lc.DTYPES)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows,k,n", [(9, 40, 24), (70, 136, 130)])
def test_each_subset_of_the_gradients(emu, rows, k, n, gated, dtype):
    """Exact integers: whatever else is asked for, a gradient is the same."""
    lc.check_exact_subsets(rows, k, n, dtype, gated, "cpu")


def test_a_second_derivative_is_refused(emu):
    x, w, b, r, dy = lc.make(3, 8, 6, torch.float32, residual=True)
    w.requires_grad_()
    for y in (ff.linear(x, w, b, r, act="silu"), ff.gated_linear(x, torch.cat([w, w]), act="silu")):
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(y, (w,), dy, create_graph=True)


def test_gradients_against_differences(emu):
    """Central differences of sum(y * dy) along random directions; fp32 forward, step 2^-7: the difference's own error is about
    (step^2 |third derivative| + 2^-24 |value| / step) -- 1e-3 of the gradient's scale."""
    for gated in (False, True):
        x, w, b, _, dy = lc.make(7, 20, 12, torch.float32, gated)
        got = lc.run(x, w, b, None, "gelu", gated, dy)
        gen = torch.Generator().manual_seed(9)
        for name, t in (("dx", x), ("dw", w), ("db", b)):
            v = torch.randn(t.shape, generator=gen)
            h = 2.0 ** -7

            def f(s):
                a = {"dx": x, "dw": w, "db": b}
                a[name] = t + s * v
                y = ff.gated_linear(a["dx"], a["dw"], a["db"], act="gelu") if gated else ff.linear(a["dx"], a["dw"], a["db"], act="gelu")
                return (y.double() * dy.double()).sum()
            num, ana = ((f(h) - f(-h)) / (2 * h)).item(), (got[name].double() * v.double()).sum().item()
            assert abs(num - ana) <= 3e-3 * (got[name].double().norm() * v.double().norm()).item(), (gated, name, num, ana)


def test_block_runs_as_a_model_uses_it(emu):
    torch.manual_seed(1)
    block = ff.GatedFeedForward(24, 40, bias=True)
    assert list(block.state_dict()) == ["weight", "weight_out", "bias", "bias_out"]
    x = torch.randn(3, 5, 24, requires_grad=True)
    y = block(x)
    y.square().mean().backward()
    p = {k: v.detach().double().requires_grad_() for k, v in block.named_parameters()}
    x64 = x.detach().double().requires_grad_()
    g, u = torch.nn.functional.linear(x64, p["weight"], p["bias"]).chunk(2, -1)
    ref = torch.nn.functional.linear(torch.nn.functional.silu(g) * u, p["weight_out"], p["bias_out"]) + x64
    ref.square().mean().backward()
    assert torch.allclose(y.double(), ref, atol=1e-5)
    for got, want in [(x.grad, x64.grad)] + [(q.grad, p[k].grad) for k, q in block.named_parameters()]:
        assert torch.allclose(got.double(), want, rtol=1e-4, atol=1e-6)
    lin = ff.Linear(24, 8, act="relu")
    assert list(lin.state_dict()) == ["weight", "bias"] and torch.allclose(lin(x), torch.relu(torch.nn.functional.linear(x, lin.weight, lin.bias)), atol=1e-5)


def test_refusals(emu):
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    err = _lib.Tnv3Error
    for call, text in ((lambda: ops.linear(x.double(), w.double()), "float32, bfloat16 or float16"),
                       (lambda: ops.linear(x, w.bfloat16()), "must be"),
                       (lambda: ops.linear(x, torch.zeros(6, 9)), "does not match"),
                       (lambda: ops.linear(x, w, torch.zeros(5)), "bias"),
                       (lambda: ops.linear(x, w, None, torch.zeros(4, 1)), "residual"),
                       (lambda: ops.linear(x, w, act=7), "unknown activation"),
                       (lambda: ops.linear(x.t().contiguous().t(), w), "contiguous"),
                       (lambda: ops.gated_linear(x, torch.zeros(5, 8)), "even number"),
                       (lambda: ops.gated_linear(torch.zeros(4, 0), torch.zeros(6, 0)), "bad weight"),
                       (lambda: ops.linear_backward(torch.zeros(4, 6), x, w, None, ops.ACT_SILU), "pre-activation"),
                       (lambda: ops.gated_linear_backward(torch.zeros(4, 3), x, w, None), "pre-activation"),
                       (lambda: ops.linear_backward(torch.zeros(4, 5), x, w), "upstream"),
                       (lambda: ops.gated_linear_backward(torch.zeros(4, 3), x, w, torch.zeros(4, 3)), "pre")):
        with pytest.raises(err, match=text):
            call()
    with pytest.raises(ValueError, match="unknown activation"):
        ff.linear(x, w, act="tanh")
    with pytest.raises(ValueError, match="expects"):
        ff.GatedFeedForward(8, 4)(torch.zeros(2, 7))
    # the C entries themselves
    lib = _lib.load()
    p, null = _lib.ptr, ctypes.c_void_p(0)
    y = torch.zeros(4, 6)

    def fwd(rows=4, k=8, n=6, act=0, dtype=0, xp=None, ws=null, nws=0):
        return lib.tnv3_linear_forward(p(x) if xp is None else xp, p(w), null, null, p(y), null, ws, nws, rows, k, n, act, dtype, null)
    assert fwd() == 0
    for bad in (dict(rows=0), dict(k=0), dict(n=-1), dict(rows=(1 << 30) + 1), dict(k=(1 << 20) + 1), dict(n=(1 << 20) + 1), dict(act=7), dict(act=-1),
                dict(dtype=3), dict(xp=null)):
        assert fwd(**bad) != 0, bad
    assert lib.tnv3_linear_backward(p(y), p(x), p(w), null, p(x), null, null, null, 0, 4, 8, 6, 0, 0, null) != 0           # no workspace
    long_k = lib.tnv3_linear_forward_workspace_bytes(70, 1100, 24, 0)
    big = [torch.zeros(s) for s in ((70, 1100), (24, 1100), (70, 24))]
    ws = torch.zeros(long_k // 4)
    args = [p(big[0]), p(big[1]), null, null, p(big[2]), null]
    assert lib.tnv3_linear_forward(*args, p(ws), long_k - 4, 70, 1100, 24, 0, 0, null) != 0                                  # too small
    assert lib.tnv3_linear_forward(*args, p(ws), long_k, 70, 1100, 24, 0, 0, null) == 0
    assert lib.tnv3_linear_forward_workspace_bytes(0, 1, 1, 0) == 0
    off = torch.zeros(4 * 8 + 1)[1:].view(4, 8)                                                                              # 4 bytes off the boundary
    assert fwd(xp=p(off)) != 0 and fwd() == 0
    assert torch.equal(ops.linear(off + 1, torch.ones(6, 8)), torch.full((4, 6), 8.0))
    assert torch.equal(ops.linear(off, w), torch.zeros(4, 6))                                                                # the op copies such a view


def test_a_launch_that_counts_more_than_32_bits_of_work_items_is_refused(emu):
    """2^30 rows of 33 elements: the copy into whole pieces would be 2^24 and more workgroups of 256; refused before anything is launched, so the
    tensors and the workspace need not be there in full."""
    lib, p = _lib.load(), _lib.ptr
    t = torch.zeros(64, dtype=torch.bfloat16)
    rows = 1 << 30
    need = lib.tnv3_linear_forward_workspace_bytes(rows, 33, 8, 1)
    assert need > rows * 80 - 1
    assert lib.tnv3_linear_forward(p(t), p(t), None, None, p(t), None, p(t), need, rows, 33, 8, 0, 1, None) != 0
    assert b"more than one launch takes" in lib.tnv3_last_error()


@pytest.mark.parametrize("dtype", lc.DTYPES)
def test_sigmoid_derivative_at_large_arguments(emu, dtype):
    lc.check_sigmoid_derivative(dtype, "cpu")


@pytest.mark.parametrize("dtype", lc.DTYPES)
@pytest.mark.parametrize("act", [a for a in lc.ACTS if a != "none"])
def test_gates_far_from_zero(emu, act, dtype):
    lc.check_far_gates(act, dtype, "cpu")


@pytest.mark.parametrize("dtype", lc.DTYPES)
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh"])
def test_gelu_of_negative_arguments_to_relative_accuracy(emu, act, dtype):
    lc.check_gelu_tail(act, dtype, "cpu")


@pytest.mark.parametrize("act", ["relu", "leaky_relu"])
@pytest.mark.parametrize("rows,k,n", [(2, 24, 16), (3, 9, 11), (70, 72, 24), (70, 1096, 20)])         # few rows; odd; tiles; tiles with parts to join
def test_least_positive_pre_activation(emu, rows, k, n, act):
    lc.check_least_positive(rows, k, n, act, "cpu")


def _plan(emu, which, rows, k, n, half, gated):
    """(tile, parts of the contraction: the most of both products') of a launch; the few-rows kernel has tile -1."""
    call = emu.load().tnv3_emu_linear_plan
    call.argtypes = [ctypes.c_int, ctypes.c_long] + [ctypes.c_int] * 4
    got = [call(q, rows, k, n, int(half), int(gated)) for q in ((0,) if which == 0 else (1, 2))]
    return (-1, 1) if got[0] < 0 else (got[0] % 256, max(g // 256 for g in got))


@pytest.mark.parametrize("cus,half,gated,which,tile,parts,sizes", lc.KERNELS_EMU + lc.KERNELS_GPU)
def test_sizes_are_planned_on_the_kernel_they_are_to_test(emu, monkeypatch, cus, half, gated, which, tile, parts, sizes):
    monkeypatch.setenv("TNV3_EMU_CUS", str(cus))
    got = _plan(emu, which, *sizes, half, gated)
    assert (got[0], got[1] > 1) == (tile, parts)


def test_every_kernel_is_listed():
    want = {(half, gated, which, tile) for half in (True, False) for gated in (False, True) for which in (0, 1) for tile in range(4)
            if (tile >= 2 or half) and (tile or which == 0)}
    for table in (lc.KERNELS_EMU, lc.KERNELS_GPU):
        assert {e[1:5] for e in table} == want


@pytest.mark.parametrize("lazy", ["0", "1"])
@pytest.mark.parametrize("cus,half,gated,which,tile,parts,sizes", lc.KERNELS_EMU)
def test_every_kernel_by_the_sizes_that_choose_it(emu, monkeypatch, cus, half, gated, which, tile, parts, sizes, lazy):
    """(lazy: direct loads land as early or as late as the program's waits allow)"""
    if lazy == "1" and not half:
        pytest.skip("fp32 products have no direct loads")
    monkeypatch.setenv("TNV3_EMU_CUS", str(cus))
    monkeypatch.setenv("TNV3_EMU_LAZY_DMA", lazy)
    lc.check_kernel(half, gated, *sizes, "cpu", exact_only=half and lazy == "0")


@pytest.mark.parametrize("cus,tiles,sizes", [(1, (2, 2), (70, 40, 40)), (1, (3, 2), (130, 72, 72)), (1, (2, 3), (130, 72, 136)), (4, (2, 2), (65, 136, 40))])
def test_fp32_tiles_keep_infinities_and_nan_where_they_belong(emu, monkeypatch, cus, tiles, sizes):
    """The products that are computed a second time, forward and backward, in both tiles, whole and in parts."""
    monkeypatch.setenv("TNV3_EMU_CUS", str(cus))
    assert tuple(_plan(emu, which, *sizes, False, False)[0] for which in (0, 1)) == tiles
    lc.check_nonfinite_products(*sizes, "cpu")


@pytest.mark.parametrize("frozen", [False, True])
def test_a_forward_mode_tangent_is_refused(emu, frozen):
    """Whether or not anything requires a gradient, and whichever input carries it."""
    import torch.autograd.forward_ad as fwd
    x, w, b, r, _ = lc.make(3, 8, 6, torch.float32, residual=True)
    w.requires_grad_(not frozen)
    for i in range(4):
        with fwd.dual_level():
            args = [x, w, b, r]
            args[i] = fwd.make_dual(args[i].detach(), torch.ones_like(args[i]))
            with pytest.raises(NotImplementedError):
                ff.linear(*args)
            if i < 3:
                with pytest.raises(NotImplementedError):
                    ff.gated_linear(*args[:3])
            assert ff.linear(x, w.detach(), b, r).shape == (3, 6)                # a level is open, no input carries a tangent
    with fwd.dual_level(), torch.no_grad(), pytest.raises(NotImplementedError):
        ff.GatedFeedForward(8, 4)(fwd.make_dual(x, torch.ones_like(x)))


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("frozen", [False, True])
def test_tracing_is_refused(emu, frozen):
    """A traced block would return uninitialised memory."""
    block = ff.GatedFeedForward(8, 16).requires_grad_(not frozen)
    for check in (True, False):
        with pytest.raises(RuntimeError, match="torch.jit.trace"):
            torch.jit.trace(block, torch.randn(3, 8), check_trace=check)
    x, w = torch.randn(3, 8), torch.randn(6, 8)
    for call in (lambda t: ops.linear(t, w), lambda t: ops.gated_linear(t, w), lambda t: ops.linear_backward(t, x, torch.randn(8, 8))[0]):
        with pytest.raises(RuntimeError, match="torch.jit.trace"):
            torch.jit.trace(call, x, check_trace=False)
    assert block(x).shape == (3, 8)


def test_streams_of_the_nodes_that_take_the_gradients():
    """What a captured backward pass is judged by: one entry per gradient that this pass wants, read from autograd's nodes whatever operation made them.
    (On the CPU a node has no stream, -1.)"""
    seen = []

    class Probe(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w, b, r):
            return x * w + r

        @staticmethod
        def backward(ctx, g):
            seen.append(_lib.gradient_streams(ctx))
            return g, g, None, g
    x, w, r = torch.ones(3), torch.ones(3, requires_grad=True), torch.ones(3, requires_grad=True)
    inner = w * 2
    y = Probe.apply(x, inner, None, r)
    torch.autograd.grad(y, [r], torch.ones(3), retain_graph=True)
    torch.autograd.grad(y, [r, w], torch.ones(3), retain_graph=True)
    y.sum().backward()
    assert seen == [[-1], [-1, -1], [-1, -1]]


@pytest.mark.parametrize("streams,refused", [([], False), ([-1], False), ([0], True), ([94, 0], True), ([94, 7, 94], False)])
def test_which_captured_backward_passes_are_refused(streams, refused):
    if not refused:
        return ff._refuse_default_stream(streams)
    with pytest.raises(RuntimeError, match="eager graph"):
        ff._refuse_default_stream(streams)


def test_refusals_of_the_modules(emu):
    for make, text in ((lambda: ff.GatedFeedForward(8, 0), "widths must be positive"), (lambda: ff.GatedFeedForward(0, 8), "widths must be positive"),
                       (lambda: ff.GatedFeedForward(8, -1), "widths must be positive"), (lambda: ff.Linear(8, 0), "widths must be positive"),
                       (lambda: ff.Linear(0, 8), "widths must be positive"), (lambda: ff.GatedFeedForward(8, 4, act=9), "unknown activation"),
                       (lambda: ff.Linear(8, 4, act=None), "unknown activation"), (lambda: ff.Linear(8, 4, act=-1), "unknown activation"),
                       (lambda: ff.GatedFeedForward(8, 4)(torch.tensor(1.0)), "expects")):
        with pytest.raises(ValueError, match=text):
            make()
    with torch.autocast("cpu", torch.bfloat16), pytest.raises(_lib.Tnv3Error, match="must be torch.bfloat16"):
        ff.Linear(8, 4)(torch.zeros(2, 8, dtype=torch.bfloat16))
    assert ff.Linear(8, 4, act=ops.ACT_GELU).act == ops.ACT_GELU


def test_inputs_that_are_not_contiguous(emu):
    """Strides of every kind: the same results and gradients, which have the inputs' shapes; the layer's edges lead to the caller's own nodes (what a
    captured backward pass is judged by), not to a copy's."""
    for gated in (False, True):
        x, w, b, r, dy = lc.make(6, 10, 8, torch.float32, gated, True, True, 4)
        want = lc.run(x, w, b, None if gated else r, "silu", gated, dy)

        def strided(t):                       # the same values, every second element of a larger tensor, transposed
            big = torch.zeros(*(2 * s for s in reversed(t.shape)))
            v = big[tuple(slice(None, None, 2) for _ in t.shape)]
            v = v.t() if t.dim() == 2 else v
            return v.copy_(t).detach()
        leaves = [strided(t).requires_grad_() for t in ([x, w, b] if gated else [x, w, b, r])]
        assert not any(t.is_contiguous() for t in leaves)
        y = ff.gated_linear(*leaves, act="silu") if gated else ff.linear(*leaves, act="silu")
        assert [node.variable.data_ptr() for node, _ in y.grad_fn.next_functions] == [t.data_ptr() for t in leaves]
        grads = torch.autograd.grad(y, leaves, strided(dy))
        assert torch.equal(y, want["y"])
        for name, g, t in zip(("dx", "dw", "db", "dr"), grads, leaves):
            assert g.shape == t.shape and torch.equal(g, want[name]), name
        with torch.no_grad():
            assert torch.equal(ff.gated_linear(*leaves, act="silu") if gated else ff.linear(*leaves, act="silu"), want["y"])
    # a copy of the input as it was: changing it afterwards does not reach the backward pass
    xt = torch.randn(10, 6).t()
    w = torch.randn(8, 10, requires_grad=True)
    y, x0 = ff.linear(xt, w), xt.clone()
    xt.mul_(2)
    assert torch.allclose(torch.autograd.grad(y.sum(), [w])[0], torch.ones(8, 6) @ x0, atol=1e-5)
