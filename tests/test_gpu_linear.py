"""GPU: the position-wise layers on the MI355X through the public entry points -- every kernel variant's sizes, alignments, streams, graph replay."""
import gc

import pytest
import torch

import linear_common as lc
from tracknetv3_amd import feedforward as ff, ops

pytestmark = pytest.mark.gpu

# one row, a few, the border of the few-rows kernels, ragged tiles, whole tiles, long contractions with few tiles, many tiles
SHAPES = [(1, 1, 1), (1, 64, 32), (1, 2048, 512), (2, 40, 24), (13, 1003, 137), (16, 256, 256), (17, 72, 40), (31, 130, 66), (33, 512, 200), (64, 1000, 264),
          (65, 33, 1030), (128, 128, 128), (130, 40, 136), (200, 4096, 96), (257, 264, 520), (300, 1001, 333), (512, 384, 128), (1000, 600, 1000),
          (2048, 512, 768), (4099, 72, 136), (3000, 2000, 1504)]


@pytest.mark.parametrize("dtype", lc.DTYPES)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows,k,n", SHAPES)
def test_exact_integers(gpu_device, rows, k, n, gated, dtype):
    lc.check_exact(rows, k, n, dtype, gated, bias=True, residual=not gated, device=gpu_device, seed=rows + k)


@pytest.mark.parametrize("dtype", lc.DTYPES)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows,k,n", [(17, 8192, 40), (33, 8200, 1000), (40, 2104, 24), (64, 4096, 4096), (65, 128, 4096), (100, 192, 520), (200, 4096, 2056),
                                      (400, 2048, 4096), (260, 320, 8192)])
def test_exact_integers_at_some_hundred_rows(gpu_device, rows, k, n, gated, dtype):
    """Around the border between the few-rows kernel and tiles, contractions of fewer steps than LDS stages and of many, one and two workgroups per CU."""
    lc.check_exact(rows, k, n, dtype, gated, bias=True, residual=not gated, device=gpu_device, seed=rows + k)


@pytest.mark.parametrize("dtype", lc.DTYPES)
@pytest.mark.parametrize("gated,act", [(False, a) for a in lc.ACTS] + [(True, a) for a in lc.ACTS if a != "none"])
@pytest.mark.parametrize("rows,k,n", [(1, 96, 40), (9, 40, 24), (150, 264, 136)])
def test_activations_and_gradients(gpu_device, rows, k, n, act, gated, dtype):
    lc.check_close(rows, k, n, dtype, act, gated, bias=True, residual=not gated, device=gpu_device, seed=3)


@pytest.mark.parametrize("dtype", lc.DTYPES)
@pytest.mark.parametrize("gated", [False, True])
def test_large_against_64_bits(gpu_device, gated, dtype):
    lc.check_close(1027, 776, 1048, dtype, "silu" if gated else "gelu", gated, bias=True, residual=not gated, device=gpu_device, seed=5)
    lc.check_close(520, 1031, 517, dtype, "sigmoid", gated, bias=False, residual=False, device=gpu_device, seed=6)


@pytest.mark.parametrize("dtype", lc.DTYPES)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows,k,n", [(9, 40, 24), (200, 2048, 515), (1030, 520, 264), (600, 2048, 2048)])
def test_each_subset_of_the_gradients(gpu_device, rows, k, n, gated, dtype):
    """Exact integers: whatever else is asked for, a gradient is the same."""
    lc.check_exact_subsets(rows, k, n, dtype, gated, gpu_device)


@pytest.mark.parametrize("dtype", lc.DTYPES)
@pytest.mark.parametrize("rows", [1, 40, 300])
def test_views_whose_base_is_not_aligned(gpu_device, rows, dtype):
    """Contiguous tensors that start one element into their storage."""
    k, n = 264, 136

    def shifted(t):
        s = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:]
        s.copy_(t.reshape(-1))
        return s.view(t.shape)
    for gated in (False, True):
        x, w, b, r, dy = lc.make(rows, k, n, dtype, gated, True, not gated, 2, gpu_device)
        want = lc.run(x, w, b, r, "silu", gated, dy)
        got = lc.run(shifted(x), shifted(w), shifted(b), None if r is None else shifted(r), "silu", gated, shifted(dy))
        tol = lc.bounds(x, w, b, r, "silu", gated, dy, dtype)
        for name, limit in tol.items():
            assert ((got[name] - want[name]).cpu().double().abs().reshape(limit.shape) <= 2 * limit).all(), name


def test_fp32_keeps_infinities_and_nan_where_they_belong(gpu_device):
    inf, nan = float("inf"), float("nan")
    for rows in (5, 200):
        x, w = torch.randn(rows, 40), torch.randn(66, 40)
        x[1, 3], x[2, 7], x[3, 2], x[4, 0] = inf, -inf, nan, 3.4e38
        w[:, 0] = torch.randn(66).sign() * 0.25
        w[5, 3] = 0.0
        y = ff.linear(x.to(gpu_device), w.to(gpu_device)).cpu()
        want = (x.double() @ w.double().t()).float()
        assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(torch.isinf(y), torch.isinf(want))
        ok = torch.isfinite(want)
        assert torch.allclose(y[ok], want[ok], rtol=1e-5, atol=1e-4)
        assert torch.equal(torch.sign(y[torch.isinf(want)]), torch.sign(want[torch.isinf(want)]))


@pytest.mark.parametrize("dtype", lc.DTYPES)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows,k,n", [(1, 5, 3), (6, 70, 9), (33, 513, 40), (70, 67, 35), (130, 72, 140), (300, 1001, 333), (700, 2050, 600)])
def test_nan_stays_in_its_row(gpu_device, rows, k, n, gated, dtype):
    lc.check_nan_stays_in_place(rows, k, n, dtype, gated, gpu_device)


@pytest.mark.parametrize("dtype", lc.DTYPES)
def test_rows_behind_the_last_stay_as_they_were(gpu_device, dtype):
    """Outputs are written up to their last element and not beyond, at sizes that end inside a tile, a vector and a row block."""
    lib, p = ops._lib.load(), ops._lib.ptr
    code = ops._LINEAR_DTYPES[dtype]
    for rows, k, n in ((1, 40, 24), (5, 33, 17), (37, 136, 72), (130, 72, 140)):
        x, w, _, _, dy = lc.make(rows, k, n, dtype, device=gpu_device)
        outs = {name: torch.full((size + 64,), 7.0, dtype=dtype, device=gpu_device) for name, size in
                (("y", rows * n), ("pre", rows * n), ("dx", rows * k), ("dw", n * k), ("db", n))}
        s = ops._lib.stream_ptr(x)
        nf, nb = lib.tnv3_linear_forward_workspace_bytes(rows, k, n, code), lib.tnv3_linear_backward_workspace_bytes(rows, k, n, 4, code)
        guard = 4096
        ws = torch.full((max(nf, nb) + guard,), 85, dtype=torch.uint8, device=gpu_device)
        assert lib.tnv3_linear_forward(p(x), p(w), None, None, p(outs["y"]), p(outs["pre"]), p(ws), nf, rows, k, n, 4, code, s) == 0
        assert lib.tnv3_linear_backward(p(dy), p(x), p(w), p(outs["pre"]), p(outs["dx"]), p(outs["dw"]), p(outs["db"]), p(ws), nb, rows, k, n, 4, code, s) == 0
        for name, t in outs.items():
            assert (t[-64:] == 7).all() and torch.isfinite(t).all(), (name, rows)
        assert (ws[-guard:] == 85).all()


@pytest.mark.parametrize("dtype", lc.DTYPES)
def test_same_bits_from_run_to_run_and_on_another_stream(gpu_device, dtype):
    side = torch.cuda.Stream(gpu_device)
    for rows, k, n in ((1, 1024, 512), (48, 2048, 256), (700, 512, 640)):
        x, w, b, _, dy = lc.make(rows, k, n, dtype, True, device=gpu_device)
        first = lc.run(x, w, b, None, "silu", True, dy)
        again = lc.run(x, w, b, None, "silu", True, dy)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = lc.run(x, w, b, None, "silu", True, dy)
        torch.cuda.current_stream().wait_stream(side)
        for name in first:
            assert torch.equal(first[name], again[name]) and torch.equal(first[name], other[name]), name


@pytest.mark.parametrize("rows", [1, 24, 400])
def test_block_captured_and_replayed(gpu_device, rows):
    """The whole block, forward and backward, in one graph: replays on new inputs equal the eager results, with eager work in between."""
    torch.manual_seed(0)
    block = ff.GatedFeedForward(256, 640, bias=True).to(gpu_device, torch.bfloat16)
    params = list(block.parameters())
    x = torch.randn(rows, 256, device=gpu_device, dtype=torch.bfloat16, requires_grad=True)
    dy = torch.randn(rows, 256, device=gpu_device, dtype=torch.bfloat16)

    def step():
        y = block(x)
        return [y.detach()] + list(torch.autograd.grad(y, [x] + params, dy))
    side = torch.cuda.Stream(gpu_device)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for i in range(3):
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
            dy.copy_(torch.randn_like(dy))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        for a, b in zip(got, step()):
            assert torch.equal(a, b), i


def test_captured_backward_beside_an_eager_graph_of_the_same_leaves_is_refused(gpu_device):
    """The refusal comes before anything of the backward pass is launched; afterwards eager and captured steps work as before."""
    block = ff.GatedFeedForward(64, 96).to(gpu_device)
    params = list(block.parameters())
    x = torch.randn(20, 64, device=gpu_device)
    dy = torch.randn(20, 64, device=gpu_device)
    eager = block(x)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(graph):
            y = block(x)
            torch.autograd.grad(y, params, dy)
    del graph, y
    want = torch.autograd.grad(eager, params, dy)
    del eager
    gc.collect()                       # the exception's frames hold the refused graph
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(block(x), params, dy)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_two_graphs_keep_their_own_workspaces(gpu_device):
    x = [torch.randn(40, 2048, device=gpu_device) for _ in range(2)]
    w = torch.randn(64, 2048, device=gpu_device) / 45
    want = [ff.linear(t, w) for t in x]
    graphs, outs = [], []
    for t in x:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ff.linear(t, w))
        graphs.append(g)
    streams = [torch.cuda.Stream(gpu_device) for _ in x]
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


def test_masked_rows_of_zero_and_large_values(gpu_device):
    """Rows that are all zero give the bias alone; 16-bit sums that pass the type's largest value become infinite, not wrapped."""
    w = torch.randn(96, 64, device=gpu_device)
    b = torch.randn(96, device=gpu_device)
    y = ff.linear(torch.zeros(33, 64, device=gpu_device), w, b)
    assert torch.equal(y, b.expand(33, 96))
    x = torch.full((20, 64), 100.0, device=gpu_device, dtype=torch.float16)
    y = ff.linear(x, torch.full((40, 64), 100.0, device=gpu_device, dtype=torch.float16))
    assert torch.isinf(y).all() and (y > 0).all()


def test_training_step_of_the_block_follows_the_oracle(gpu_device):
    """The block under the framework's own optimizer for three steps against the same steps in 64 bits."""
    from tracknetv3_amd.optim import FusedSGD
    torch.manual_seed(2)
    block = ff.GatedFeedForward(64, 176, bias=True).to(gpu_device)
    ref = {k: v.detach().cpu().double().requires_grad_() for k, v in block.named_parameters()}
    opt = FusedSGD(block.parameters(), lr=0.05)
    x, t = torch.randn(48, 64), torch.randn(48, 64)
    for _ in range(3):
        opt.zero_grad()
        ((block(x.to(gpu_device)) - t.to(gpu_device)) ** 2).mean().backward()
        opt.step()
        x64 = x.double()
        g, u = torch.nn.functional.linear(x64, ref["weight"], ref["bias"]).chunk(2, -1)
        y = torch.nn.functional.linear(torch.nn.functional.silu(g) * u, ref["weight_out"], ref["bias_out"]) + x64
        grads = torch.autograd.grad(((y - t.double()) ** 2).mean(), list(ref.values()))
        with torch.no_grad():
            for p, gr in zip(ref.values(), grads):
                p -= 0.05 * gr
    for k, v in block.named_parameters():
        # three updates of lr * gradient (|gradient| < 1 here), each within fp32's 2^-18 of the gradient's norm, plus the parameter's rounding
        assert (v.cpu().double() - ref[k]).abs().max() <= 2.0 ** -20, k


def _signs(shape, keep, device, gen, dtype):
    """-1, 0, 1 with about `keep` nonzero; exact in every type."""
    r = torch.rand(shape, generator=gen, device=device)
    return ((r < keep / 2).to(dtype) - (r > 1 - keep / 2).to(dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_operands_beyond_2_to_the_32_bytes_and_elements(gpu_device, dtype):
    """Long batches and large weights: the offsets pass 32 bits.  Integer operands, so the compared parts are equal."""
    gen = torch.Generator(device=gpu_device).manual_seed(1)
    # rows x k beyond 2^31 elements (2^32 bytes in bf16): x, dx and the contraction of dW are long
    rows, k, n = (1 << 19) + 131, 4160, 72
    x = _signs((rows, k), 0.002, gpu_device, gen, dtype)
    w = _signs((n, k), 0.1, gpu_device, gen, dtype)
    dy = _signs((rows, n), 0.002, gpu_device, gen, dtype)
    y = ops.linear(x, w)
    dx, dw, db = ops.linear_backward(dy, x, w)
    for part in (slice(0, 300), slice(rows // 2, rows // 2 + 300), slice(rows - 300, rows)):
        assert torch.equal(y[part].float(), x[part].float() @ w.float().t())
        assert torch.equal(dx[part].float(), dy[part].float() @ w.float())
    want = torch.zeros(n, k, device=gpu_device)
    for at in range(0, rows, 1 << 16):
        want += dy[at:at + (1 << 16)].float().t() @ x[at:at + (1 << 16)].float()
    assert want.abs().max() <= 256 and torch.equal(dw.float(), want)
    assert torch.equal(db.float(), dy.float().sum(0).to(dtype).float())
    del x, y, dx, dy
    # a weight beyond 2^31 elements, few and more rows; its gradient is as large
    n, k = 1 << 19, 4168
    w = _signs((n, k), 0.003, gpu_device, gen, dtype)
    for rows in (3, 70):
        x = _signs((rows, k), 0.5, gpu_device, gen, dtype)
        y, h = ops.linear(x, w), ops.gated_linear(x, w, act=ops.ACT_RELU)
        for part in (slice(0, 300), slice(n // 2 - 300, n // 2), slice(n - 300, n)):
            assert torch.equal(y[:, part].float(), x.float() @ w[part].float().t())
        last = slice(n // 2 - 300, n // 2)
        g, u = (x.float() @ w[r].float().t() for r in (last, slice(n - 300, n)))
        assert torch.equal(h[:, last].float(), torch.relu(g) * u)
    dy = _signs((70, n), 0.001, gpu_device, gen, dtype)
    dx, dw, _ = ops.linear_backward(dy, x, w, want=(True, True, False))
    assert torch.equal(dw[-300:].float(), dy[:, -300:].float().t() @ x.float())
    want = torch.zeros(70, k, device=gpu_device)
    for at in range(0, n, 1 << 16):
        want += dy[:, at:at + (1 << 16)].float() @ w[at:at + (1 << 16)].float()
    assert want.abs().max() <= 256 and torch.equal(dx.float(), want)


@pytest.mark.parametrize("dtype", lc.DTYPES)
def test_sigmoid_derivative_at_large_arguments(gpu_device, dtype):
    lc.check_sigmoid_derivative(dtype, gpu_device)


@pytest.mark.parametrize("dtype", lc.DTYPES)
@pytest.mark.parametrize("act", [a for a in lc.ACTS if a != "none"])
def test_gates_far_from_zero(gpu_device, act, dtype):
    lc.check_far_gates(act, dtype, gpu_device)


@pytest.mark.parametrize("dtype", lc.DTYPES)
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh"])
def test_gelu_of_negative_arguments_to_relative_accuracy(gpu_device, act, dtype):
    lc.check_gelu_tail(act, dtype, gpu_device)


@pytest.mark.parametrize("act", ["relu", "leaky_relu"])
@pytest.mark.parametrize("rows,k,n", [(2, 24, 16), (3, 9, 11), (70, 72, 24), (70, 1096, 20), (1500, 520, 1032)])
def test_least_positive_pre_activation(gpu_device, rows, k, n, act):
    lc.check_least_positive(rows, k, n, act, gpu_device)


@pytest.mark.parametrize("cus,half,gated,which,tile,parts,sizes", lc.KERNELS_GPU)
def test_every_kernel_by_the_sizes_that_choose_it(gpu_device, cus, half, gated, which, tile, parts, sizes):
    """(The CPU tests check that these sizes are planned on these kernels.)"""
    if torch.cuda.get_device_properties(gpu_device).multi_processor_count != cus:
        pytest.skip("other CU counts plan other tiles")
    lc.check_kernel(half, gated, *sizes, gpu_device)


@pytest.mark.parametrize("sizes", [(70, 40, 40), (200, 40, 66), (1500, 72, 4104), (520, 4104, 520), (130, 520, 4104)])
def test_fp32_tiles_keep_infinities_and_nan_where_they_belong(gpu_device, sizes):
    """The products that are computed a second time, forward and backward: tiles of 128 x 64 and 256 x 128, whole and in parts."""
    lc.check_nonfinite_products(*sizes, gpu_device)


def _captured_gradients(block, x, dy, params):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(block(x), params, dy)
    return graph, got


def _replays_equal(graph, got, want):
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_accumulators_that_another_operation_made(gpu_device):
    """A leaf whose first graph is another operation's: on the default stream and alive, the captured backward pass is refused; on a side stream, or inside
    the capture itself, it runs."""
    block = ff.GatedFeedForward(64, 96).to(gpu_device)
    params = list(block.parameters())
    x = torch.randn(20, 64, device=gpu_device, requires_grad=True)
    dy = torch.randn(20, 64, device=gpu_device)
    want = torch.autograd.grad(block(x), params + [x], dy)
    side = torch.cuda.Stream(gpu_device)
    for penalty_of in (params[0], params[1], x):
        penalty = penalty_of.square().sum()                            # alive, on the default stream
        assert penalty.requires_grad
        with pytest.raises(RuntimeError, match="eager graph"):
            _captured_gradients(block, x, dy, params + [x])
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):                                  # a first call of the block on a side stream does not hide it
            beside = block(x)
        with pytest.raises(RuntimeError, match="eager graph"):
            _captured_gradients(block, x, dy, params + [x])
        del penalty, beside
        gc.collect()
    with torch.cuda.stream(side):
        penalty = (params[0].square().sum(), x.square().sum(), block(x))
    torch.cuda.synchronize()
    _replays_equal(*_captured_gradients(block, x, dy, params + [x]), want)
    del penalty
    gc.collect()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h = x * 1.0
        got = torch.autograd.grad(ff.linear(h, params[1].t()[:64], residual=x), [x], dy)
    _replays_equal(graph, got, torch.autograd.grad(ff.linear(x * 1.0, params[1].t()[:64], residual=x), [x], dy))


def test_a_gradient_that_is_not_computed_does_not_refuse_a_capture(gpu_device):
    x = torch.randn(20, 64, device=gpu_device, requires_grad=True)
    w = torch.randn(32, 64, device=gpu_device, requires_grad=True)
    dy = torch.randn(20, 32, device=gpu_device)
    want = torch.autograd.grad(ff.linear(x, w), [x], dy)
    penalty = w.square().sum()                                         # alive, on the default stream
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(ff.linear(x, w), [x], dy)
    _replays_equal(graph, got, want)
    assert penalty.requires_grad


def test_a_leaf_that_is_not_contiguous_is_seen_by_the_refusal(gpu_device):
    x = torch.randn(20, 64, device=gpu_device)
    w = torch.randn(64, 32, device=gpu_device).t().requires_grad_()
    dy = torch.randn(20, 32, device=gpu_device)
    want = torch.autograd.grad(ff.linear(x, w), [w], dy)
    penalty = w.square().sum()                                         # alive, on the default stream
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(graph):
            torch.autograd.grad(ff.linear(x, w), [w], dy)
    del penalty, graph
    gc.collect()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(ff.linear(x, w), [w], dy)
    _replays_equal(graph, got, want)
