"""gated_linear against its formula in float64: sizes that end inside a tile, one row and one
feature, unaligned rows and views, every activation and type, its gradients against float64 and
against differences, saturated units, non-finite values, streams and graphs, and its refusals."""

from __future__ import annotations

import math

import pytest
import torch

import fused_hoad
from gpu_helpers import require_gpu_extension
from network_helpers import HALF_ULP, contraction_tolerance, double, leaf, norm_error, normal, show

ACTIVATIONS = {
    "silu": torch.nn.functional.silu,
    "tanh": torch.tanh,
    "gelu": torch.nn.functional.gelu,
    "sigmoid": torch.sigmoid,
}
F32, BF16 = torch.float32, torch.bfloat16


def formula(x, gate_weight, up_weight, gate_bias, up_bias, activation):
    linear = torch.nn.functional.linear
    return ACTIVATIONS[activation](linear(x, gate_weight, gate_bias)) * linear(x, up_weight, up_bias)


def inputs(rows, width, hidden, dtype, bias=True, seed=0):
    scale = 1.0 / math.sqrt(width)
    tensors = [normal(rows, width, seed=seed, dtype=dtype),
               normal(hidden, width, seed=seed + 1, dtype=dtype, scale=scale),
               normal(hidden, width, seed=seed + 2, dtype=dtype, scale=scale)]
    if bias:
        return tensors + [normal(hidden, seed=seed + 3, dtype=dtype, scale=0.3),
                          normal(hidden, seed=seed + 4, dtype=dtype, scale=0.3)]
    return tensors + [None, None]


def call(tensors, activation):
    return fused_hoad.gated_linear(*tensors, activation=activation)


def check(rows, width, hidden, dtype, activation="silu", bias=True, seed=0, tensors=None):
    require_gpu_extension()
    show(f"gated_linear {rows} x {width} x {hidden} {dtype} {activation} bias={bias}")
    tensors = [leaf(t) for t in (tensors or inputs(rows, width, hidden, dtype, bias, seed))]
    upstream = normal(rows, hidden, seed=seed + 5, dtype=dtype)
    h = call(tensors, activation)
    assert h.shape == (rows, hidden) and h.dtype == dtype
    wanted = [t for t in tensors if t is not None]
    grads = torch.autograd.grad(h, wanted, upstream)
    exact = [double(t) for t in tensors]
    h64 = formula(*exact, activation)
    grads64 = torch.autograd.grad(h64, [t for t in exact if t is not None], upstream.double())

    # The forward, element by element. g and u are sums of `width` products: at most 8 roundings for
    # every 16 of them (six part products), each 2^-23 (a matrix instruction may truncate) of the sum
    # of magnitudes. |act'| is at most 1.13 and the activation formulas are good to 8 units of
    # 2^-24 (1 + |g|); bfloat16 rounds the result once.
    with torch.no_grad():
        magnitudes = [torch.nn.functional.linear(exact[0].abs(), w.abs(), None if b is None else b.abs())
                      for w, b in ((exact[1], exact[3]), (exact[2], exact[4]))]
        gamma = (8 * math.ceil(width / 16) + 8) * 2.0**-23
        g = torch.nn.functional.linear(exact[0], exact[1], exact[3])
        u = torch.nn.functional.linear(exact[0], exact[2], exact[4])
        act = ACTIVATIONS[activation](g)
        bound = (1.13 * gamma * magnitudes[0] + 2.0**-21 * (1 + g.abs())) * (u.abs() + gamma * magnitudes[1])
        bound += act.abs() * gamma * magnitudes[1]
        bound += HALF_ULP[dtype] * h64.abs()
        assert bool(((h.double() - h64).abs() <= bound).all())
    names = [name for name, t in zip(("x", "gate_weight", "up_weight", "gate_bias", "up_bias"), tensors) if t is not None]
    depths = {"x": 2 * hidden + width, "gate_weight": rows + width, "up_weight": rows + width,
              "gate_bias": rows + width, "up_bias": rows + width}
    for name, got, want in zip(names, grads, grads64):
        assert got.dtype == dtype and got.shape == want.shape
        error = norm_error(got, want)
        assert error <= contraction_tolerance(dtype, depths[name]), f"{name}: {error:.3e}"
    return h, grads


SIZES = [
    (1, 1, 1), (1, 64, 48), (1, 257, 3), (3, 16, 33), (16, 100, 65), (17, 129, 40), (32, 72, 200),
    (33, 40, 70), (64, 64, 64), (65, 66, 127), (130, 200, 96), (300, 31, 257), (513, 520, 264),
    (2000, 24, 40),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows, width, hidden", SIZES)
def test_sizes(rows, width, hidden, dtype) -> None:
    check(rows, width, hidden, dtype, seed=rows + width)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows, width, hidden", [(6000, 264, 1100), (5003, 129, 1365), (40000, 136, 70)])
def test_large_tiles(rows, width, hidden, dtype) -> None:
    """Enough tiles for the large ones, whole and odd rows, and depths that are cut into runs."""
    check(rows, width, hidden, dtype, seed=3)


@pytest.mark.gpu
@pytest.mark.parametrize("rows, width, hidden", [(2047, 777, 2300), (4100, 777, 2300), (8200, 1025, 1100)])
def test_operands_split_before(rows, width, hidden) -> None:
    """float32 layers whose second operands are split before the products, and one row too few for it:
    odd widths, and gradients whose depth is cut into runs."""
    check(rows, width, hidden, F32, seed=4)


@pytest.mark.gpu
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("rows, width, hidden", [(33, 17, 1), (33, 1, 33), (255, 700, 1023), (256, 300, 1024),
                                                 (257, 300, 1025), (600, 100, 700), (1000, 255, 1365)])
def test_few_and_many_tiles(rows, width, hidden, bias) -> None:
    """float32 layers on both sides of a workgroup of 32 rows and 32 features for every CU."""
    check(rows, width, hidden, F32, "gelu", bias, seed=rows)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("activation", sorted(ACTIVATIONS))
@pytest.mark.parametrize("bias", [False, True])
def test_activations(activation, bias, dtype) -> None:
    check(70, 48, 90, dtype, activation, bias, seed=11)


@pytest.mark.gpu
@pytest.mark.parametrize("activation", sorted(ACTIVATIONS))
def test_activation_over_its_range(activation) -> None:
    """g from -30 to 30 through a one-wide layer, u = 1: the activation, and by an upstream gradient of
    one its slope, element by element. Tails keep a relative precision of 2^-18 down to 2^-100 (the
    exponent's rounding grows with |g|), and elsewhere 8 units of 2^-24."""
    require_gpu_extension()
    show(f"activation {activation}")
    x = torch.linspace(-30, 30, 24001, device="cuda").unsqueeze(1)
    one, zero = torch.ones(1, 1, device="cuda"), torch.zeros(1, 1, device="cuda")
    up_bias = torch.ones(1, device="cuda")
    x = leaf(x)
    h = fused_hoad.gated_linear(x, one, zero, None, up_bias, activation=activation)
    slope, = torch.autograd.grad(h, x, torch.ones_like(h))
    exact = double(x)
    h64 = ACTIVATIONS[activation](exact)
    slope64, = torch.autograd.grad(h64, exact, torch.ones_like(h64))
    # Differences from one lose float64's digits in the tails too.
    if activation == "sigmoid":
        slope64 = torch.sigmoid(exact) * torch.sigmoid(-exact)
    elif activation == "tanh":
        slope64 = 4 * torch.sigmoid(2 * exact) * torch.sigmoid(-2 * exact)
    for got, want in ((h, h64), (slope, slope64)):
        error = (got.double() - want).abs()
        assert bool((error <= 2.0**-18 * want.abs() + 2.0**-100).logical_or(error <= 2.0**-21).all())
        tail = want.abs() < 2.0**-12
        # gelu's slope crosses zero; where it does not, the tail's relative error counts.
        if activation != "gelu" and not (activation == "silu" and got is slope):
            assert bool((error[tail] <= 2.0**-18 * want[tail].abs() + 2.0**-100).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_unaligned_and_strided_inputs(dtype) -> None:
    """Views at odd offsets, transposed and expanded inputs give bitwise what aligned contiguous
    copies give, for the same way of staging (odd rows) and for both (whole rows)."""
    require_gpu_extension()
    rows, width, hidden = 150, 40, 72
    tensors = inputs(rows, width, hidden, dtype, seed=21)
    for t in (0, 1, 2):
        storage = torch.empty(tensors[t].numel() + 1, dtype=dtype, device="cuda")
        view = storage[1:].view(tensors[t].shape)
        view.copy_(tensors[t])
        moved = list(tensors)
        moved[t] = view
        show(f"unaligned input {t} {dtype}")
        check(rows, width, hidden, dtype, seed=21, tensors=moved)
    plain = call(tensors, "silu")
    strided = [tensors[0].t().contiguous().t(), tensors[1].t().contiguous().t(), tensors[2], tensors[3], tensors[4]]
    assert torch.equal(call(strided, "silu"), plain)
    row = tensors[0][:1]
    x = leaf(row)
    h = fused_hoad.gated_linear(x.expand(rows, width), *tensors[1:], activation="silu")
    upstream = normal(rows, hidden, seed=5, dtype=dtype)
    got, = torch.autograd.grad(h, x, upstream)
    exact = double(row)
    h64 = formula(exact.expand(rows, width), *[t.double() for t in tensors[1:]], "silu")
    want, = torch.autograd.grad(h64, exact, upstream.double())
    assert norm_error(got, want) <= contraction_tolerance(dtype, 2 * hidden + width + rows)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_leading_dimensions_and_empty(dtype) -> None:
    require_gpu_extension()
    x, *rest = inputs(24, 32, 40, dtype, seed=8)
    shaped = fused_hoad.gated_linear(x.view(2, 3, 4, 32), *rest)
    assert shaped.shape == (2, 3, 4, 40) and torch.equal(shaped.view(24, 40), fused_hoad.gated_linear(x, *rest))
    one = fused_hoad.gated_linear(x[0], *rest)
    assert one.shape == (40,)
    tensors = [leaf(t) for t in (x[:0], *rest)]
    h = fused_hoad.gated_linear(*tensors)
    assert h.shape == (0, 40)
    for t, grad in zip(tensors, torch.autograd.grad(h.sum(), tensors)):
        assert grad.shape == t.shape and not grad.any()


@pytest.mark.gpu
def test_gradient_against_differences() -> None:
    """Directional derivatives of sum(h upstream) by central differences of the kernel's own forward,
    summed in float64: the third-order term is about step^2, the forward's rounding 2^-21 over
    the step, so a step of 2^-7 leaves 2e-4 or less of the derivative's scale; 2e-3 is allowed."""
    require_gpu_extension()
    tensors = [leaf(t) for t in inputs(60, 48, 56, F32, seed=31)]
    upstream = normal(60, 56, seed=40)
    for activation in sorted(ACTIVATIONS):
        show(f"differences {activation}")
        grads = torch.autograd.grad(call(tensors, activation), tensors, upstream)
        for k, grad in enumerate(grads):
            direction = normal(*tensors[k].shape, seed=50 + k)
            direction = direction * (tensors[k].detach().norm() / direction.norm())
            values = []
            for sign in (1, -1):
                moved = [t.detach() for t in tensors]
                moved[k] = moved[k] + sign * 2.0**-7 * direction
                values.append((call(moved, activation).double() * upstream).sum())
            slope = (values[0] - values[1]) / 2.0**-6
            want = (grad.double() * direction).sum()
            scale = grad.double().norm() * direction.double().norm()
            assert abs(float(slope - want)) <= 2e-3 * float(scale), (activation, k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_results_repeat_and_need_no_gradients(dtype) -> None:
    """Bitwise the same with and without gradients and on a second call; only the gradients that are
    asked for are formed."""
    require_gpu_extension()
    tensors = inputs(700, 130, 200, dtype, seed=2)
    upstream = normal(700, 200, seed=3, dtype=dtype)
    plain = call(tensors, "gelu")
    leaves = [leaf(t) for t in tensors]
    h = call(leaves, "gelu")
    assert torch.equal(h, plain)
    grads = torch.autograd.grad(h, leaves, upstream)
    again = torch.autograd.grad(call(leaves, "gelu"), leaves, upstream)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    for k in range(5):
        some = [leaf(t) if k == i else t for i, t in enumerate(tensors)]
        grad, = torch.autograd.grad(call(some, "gelu"), some[k], upstream)
        assert torch.equal(grad, grads[k]), k


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows, width, hidden", [(5, 50, 60), (90, 50, 60), (5000, 520, 1100)])
def test_non_finite_values_stay_in_their_rows(dtype, rows, width, hidden) -> None:
    require_gpu_extension()
    show(f"non-finite {dtype} {rows}")
    tensors = inputs(rows, width, hidden, dtype, seed=12)
    clean = call(tensors, "silu")
    for value in (math.nan, math.inf, -math.inf):
        x = tensors[0].clone()
        x[2, 7] = value
        h = call([x, *tensors[1:]], "silu")
        assert not torch.isfinite(h[2]).all()
        others = [r for r in range(rows) if r != 2]
        assert torch.equal(h[others], clean[others])


@pytest.mark.gpu
def test_large_and_small_values() -> None:
    """float32 values up to 1e18 and down to 1e-15 keep float32 precision (products up to 1e36)."""
    require_gpu_extension()
    for scale in (1e18, 1e-15):
        x, gw, uw, _, _ = inputs(70, 40, 50, F32, bias=False, seed=4)
        u = fused_hoad.gated_linear(x * scale, torch.zeros_like(gw), uw, torch.full((50,), 2.0, device="cuda"),
                                    activation="sigmoid")
        want = (x.double() * scale) @ uw.double().t() * torch.sigmoid(torch.tensor(2.0, dtype=torch.float64))
        assert norm_error(u, want) <= contraction_tolerance(F32, 40)


@pytest.mark.gpu
@pytest.mark.parametrize("rows, width, hidden", [(90, 48, 70), (5000, 520, 1100)])
def test_rows_of_very_different_sizes(rows, width, hidden) -> None:
    """Rows of x, of the up weights and of the upstream gradient scaled by powers of two from 2^-40 to 2^40:
    every row and column of h, every row of the input's gradient and every row of the up weights'
    gradient (one feature's) keeps the relative precision that unscaled ones have. g is 2 throughout
    (no gate weights), so h = sigmoid(2) u."""
    require_gpu_extension()
    show(f"row sizes {rows}")
    x, gw, uw, _, _ = inputs(rows, width, hidden, F32, bias=False, seed=14)
    gate_bias = torch.full((hidden,), 2.0, device="cuda")
    factor = torch.sigmoid(torch.tensor(2.0, dtype=torch.float64)).item()

    def scales(count, most, seed):
        return 2.0 ** torch.randint(-most, most + 1, (count, 1), generator=torch.Generator().manual_seed(seed)).cuda()

    def up_only(x, uw):
        return fused_hoad.gated_linear(x, torch.zeros_like(gw), uw, gate_bias, activation="sigmoid")

    by_row, by_feature = scales(rows, 40, 1), scales(hidden, 40, 2)
    h = up_only(x * by_row, uw * by_feature).double() / by_row.double() / by_feature.double().t()
    h64 = factor * (x.double() @ uw.double().t())
    error = (h - h64).abs()
    for dim in (0, 1):
        assert bool((error.norm(dim=dim) <= contraction_tolerance(F32, width) * h64.norm(dim=dim)).all())
    x, uw, by_row = leaf(x), leaf(uw), scales(rows, 40, 3)
    upstream = normal(rows, hidden, seed=15) * by_row
    dx, duw = torch.autograd.grad(up_only(x, uw), (x, uw), upstream)
    du = factor * upstream.double()
    dx64, duw64 = du @ uw.detach().double(), du.t() @ x.detach().double()
    assert bool(((dx.double() - dx64).norm(dim=1) <= contraction_tolerance(F32, 2 * hidden) * dx64.norm(dim=1)).all())
    assert bool(((duw.double() - duw64).norm(dim=1) <= contraction_tolerance(F32, rows) * duw64.norm(dim=1)).all())


@pytest.mark.gpu
def test_columns_of_very_different_sizes() -> None:
    """Columns of x and of the up weights scaled against each other by up to 2^20 (features of very
    different units, and weights that make up for them): the products are those of unscaled ones, and
    so is h's precision, row by row."""
    require_gpu_extension()
    show("column sizes")
    for rows, width, hidden in ((90, 48, 70), (5000, 520, 1100)):
        x, gw, uw, _, _ = inputs(rows, width, hidden, F32, bias=False, seed=16)
        by_column = 2.0 ** torch.randint(-10, 11, (width,), generator=torch.Generator().manual_seed(4)).cuda()
        gate_bias = torch.full((hidden,), 2.0, device="cuda")
        h = fused_hoad.gated_linear(x * by_column, torch.zeros_like(gw), uw / by_column, gate_bias, activation="sigmoid")
        h64 = torch.sigmoid(torch.tensor(2.0, dtype=torch.float64)) * (x.double() @ uw.double().t())
        error = (h.double() - h64).norm(dim=1)
        assert bool((error <= contraction_tolerance(F32, width) * h64.norm(dim=1)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_own_stream_and_graph_replays(dtype) -> None:
    """On a stream of its own, and captured with its backward and replayed on new inputs with eager
    work between the replays: each bitwise the eager result."""
    require_gpu_extension()
    show(f"graph {dtype}")
    tensors = [leaf(t) for t in inputs(200, 72, 136, dtype, seed=6)]
    upstream = normal(200, 136, seed=7, dtype=dtype)

    def run():
        h = call(tensors, "silu")
        # Detached: a graph that is kept would hold the leaves' gradient nodes on this stream.
        return [h.detach(), *torch.autograd.grad(h, tensors, upstream)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(on_side, run()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = run()
    for seed in (61, 62, 63):
        with torch.no_grad():
            for t, new in zip(tensors, inputs(200, 72, 136, dtype, seed=seed)):
                t.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(static, run()))


def test_refusals_on_the_cpu() -> None:
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    with pytest.raises(RuntimeError, match="x must be a CUDA tensor"):
        fused_hoad.gated_linear(x, w, w)
    with pytest.raises(RuntimeError, match="activation must be"):
        fused_hoad.gated_linear(x, w, w, activation="relu")


@pytest.mark.gpu
def test_refusals() -> None:
    require_gpu_extension()
    x, gw, uw, gb, ub = inputs(4, 8, 6, F32)
    gated_linear = fused_hoad.gated_linear
    for bad, message in (
        (lambda: gated_linear(x.half(), gw, uw), "float32 or bfloat16"),
        (lambda: gated_linear(x, gw.bfloat16(), uw), "gate_weight must have x's dtype"),
        (lambda: gated_linear(x, gw, uw.cpu()), "up_weight must be a CUDA tensor"),
        (lambda: gated_linear(x, gw[:, :7], uw), "gate_weight must have shape"),
        (lambda: gated_linear(x, gw, uw[:5]), "up_weight must have gate_weight's shape"),
        (lambda: gated_linear(x, gw, uw, gb[:5]), r"gate_bias must have shape \[6\]"),
        (lambda: gated_linear(x, gw, uw, gb, ub.view(1, 6)), r"up_bias must have shape \[6\]"),
        (lambda: gated_linear(x[0, 0], gw, uw), "x must have shape"),
    ):
        with pytest.raises(RuntimeError, match=message):
            bad()
    leaves = [leaf(t) for t in (x, gw, uw)]
    grad, = torch.autograd.grad(gated_linear(*leaves).sum(), leaves[0])
    assert grad.shape == x.shape
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(gated_linear(*leaves).sum(), leaves[0], create_graph=True)
    h = gated_linear(*leaves)
    with torch.no_grad():
        leaves[1].add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()


def saturating_values(dtype):
    """g from -1e30 to 1e30, dense where e^-g ends (88.7) and beyond, each value the same in every format."""
    pieces = [torch.linspace(-200, 200, 1201), torch.linspace(85, 95, 201), torch.linspace(-95, -85, 201)]
    far = torch.tensor([250.0, 500, 1000, 5000, 6899, 9999, 1e4, 1.1e4, 1e5, 1e10, 1e19, 1e30])
    values = torch.cat([*pieces, far, -far]).to(dtype).float()
    bits = values.view(torch.int32) & ~0xFF  # 16 significant bits: exact as two float16 parts
    return bits.view(torch.float32).to(device="cuda", dtype=dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("rows, width", [(5, 8), (64, 8), (600, 8), (700, 2048), (4000, 520)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("activation", sorted(ACTIVATIONS))
def test_saturated_units(activation, dtype, rows, width) -> None:
    """Finite g from -1e30 to 1e30, one value a feature (x is one in its first column and zero elsewhere, u is
    one): h, and by the gradients of the gate's bias and weights the slope, are finite and close to float64,
    in the kernels for few rows, few tiles and the tiles of every format. An activation's relative error
    grows with |g| 2^-23 in its tail, where it is below 2^-20: 2^-18 of a value and 2^-20 are allowed, and the
    sums over equal rows at most rows 2^-24 beside it; bfloat16 rounds dg and the results."""
    require_gpu_extension()
    show(f"saturated {activation} {dtype} {rows} x {width}")
    values = saturating_values(dtype)
    hidden = values.numel()
    x = torch.zeros(rows, width, device="cuda", dtype=dtype)
    x[:, 0] = 1
    gate_weight = torch.zeros(hidden, width, device="cuda", dtype=dtype)
    gate_weight[:, 0] = values
    zero, one = torch.zeros(hidden, device="cuda", dtype=dtype), torch.ones(hidden, device="cuda", dtype=dtype)
    tensors = [leaf(t) for t in (x, gate_weight, torch.zeros_like(gate_weight), zero, one)]
    h = call(tensors, activation)
    grads = torch.autograd.grad(h, tensors, torch.ones_like(h))
    assert all(bool(torch.isfinite(t).all()) for t in (h, *grads))
    exact = values.double().requires_grad_()
    h64 = ACTIVATIONS[activation](exact)
    slope64, = torch.autograd.grad(h64.sum(), exact)
    rounding = HALF_ULP[BF16] if dtype == BF16 else 0.0
    relative = 2.0**-18 + rounding
    assert bool(((h.double() - h64).abs() <= relative * h64.abs() + 2.0**-20).all())
    # Of the gate's weights: of their first column; x is zero in the others.
    for got in (grads[3], grads[1][:, 0]):
        error = (got.double() / rows - slope64).abs()
        assert bool((error <= (relative + rounding + rows * 2.0**-24) * slope64.abs() + 2.0**-20).all())
    assert not grads[1][:, 1:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows, width, hidden", [(5, 50, 60), (90, 50, 60), (600, 40, 700), (5000, 520, 1100)])
def test_non_finite_operands_leave_nothing_finite(dtype, rows, width, hidden) -> None:
    """A NaN or infinite value of x makes the whole of its row of h and of the input's gradient non-finite,
    and leaves every other row of both bitwise alone."""
    require_gpu_extension()
    show(f"non-finite row {dtype} {rows}")
    tensors = inputs(rows, width, hidden, dtype, seed=12)
    upstream = normal(rows, hidden, seed=13, dtype=dtype)

    def run(x):
        x = leaf(x)
        h = call([x, *tensors[1:]], "silu")
        return h.detach(), torch.autograd.grad(h, x, upstream)[0]

    clean = run(tensors[0])
    others = [r for r in range(rows) if r != 2]
    for value in (math.nan, math.inf, -math.inf):
        x = tensors[0].clone()
        x[2, 7] = value
        for got, want in zip(run(x), clean):
            assert not torch.isfinite(got[2]).any()
            assert torch.equal(got[others], want[others])


@pytest.mark.gpu
@pytest.mark.parametrize("needs_grad", [False, True])
def test_forward_mode_is_refused(needs_grad) -> None:
    """A dual tensor in any place raises, with and without gradient mode, instead of losing its tangent;
    the tensors that lie in it are taken as before."""
    from torch.autograd import forward_ad

    require_gpu_extension()
    show("gated_linear dual tensors")
    tensors = inputs(4, 8, 6, F32)
    plain = call(tensors, "silu")
    with forward_ad.dual_level(), torch.set_grad_enabled(needs_grad):
        for k, t in enumerate(tensors):
            some = list(tensors)
            some[k] = forward_ad.make_dual(leaf(t) if needs_grad else t, torch.ones_like(t))
            with pytest.raises(RuntimeError, match="gated_linear has no forward-mode derivative"):
                call(some, "silu")
            some[k] = forward_ad.unpack_dual(some[k]).primal
            assert torch.equal(call(some, "silu"), plain)


@pytest.mark.gpu
@pytest.mark.parametrize("rows, width, hidden", [(5, 40, 70), (64, 40, 70), (600, 40, 700), (700, 2048, 300),
                                                 (4000, 520, 1700)])
def test_the_largest_float32_values(rows, width, hidden) -> None:
    """Operands next to the largest float32 value, which bfloat16 rounds to infinity, with others that make
    up for them: h, the input's gradient and the up weights' gradient element by element. The gate is
    tanh(30), one, so the products are u = x Wu^T, dx = dh Wu and dWu = dh^T x, whose sums of n products
    have at most 8 roundings for every 16 of them, 2^-23 each of the sum of magnitudes. The matrix cores
    take bfloat16 parts below 2^-126 as zero, which changes an operand by at most 2^-126 + 2^-134: that much of
    each operand's values counts beside it."""
    require_gpu_extension()
    show(f"largest values {rows} x {width} x {hidden}")
    largest = torch.finfo(F32).max
    edges = [largest, -largest, float.fromhex("0x1.FFp127"), -float.fromhex("0x1.FEFFFEp127"),
             float.fromhex("0x1.FEp127")]

    def with_edges(t):
        for k, value in enumerate(edges):
            t[k, 3 * k + 1] = value
        return t

    gate_bias = torch.full((hidden,), 30.0, device="cuda")
    small = 2.0**-115

    def run(x, up_weight, upstream):
        x, up_weight = leaf(x), leaf(up_weight)
        h = fused_hoad.gated_linear(x, torch.zeros_like(up_weight), up_weight, gate_bias, activation="tanh")
        return h.detach(), *torch.autograd.grad(h, (x, up_weight), upstream)

    def close(got, a, b):
        """got = a b, element by element."""
        a, b = a.double(), b.double()
        gamma = (8 * math.ceil(a.shape[1] / 16) + 8) * 2.0**-23
        lost = (2.0**-126 + 2.0**-134) * (a.abs().sum(1, keepdim=True) + b.abs().sum(0, keepdim=True))
        assert bool(((got.double() - a @ b).abs() <= gamma * (a.abs() @ b.abs()) + lost).all())

    x, w = normal(rows, width, seed=1), normal(hidden, width, seed=2)
    upstream = normal(rows, hidden, seed=3)
    close(run(with_edges(x.clone()), w * small, upstream)[0], with_edges(x.clone()), w.t() * small)
    close(run(x * small, with_edges(w.clone()), upstream)[0], x * small, with_edges(w.clone()).t())
    close(run(x * small, w * small, with_edges(upstream.clone()))[1], with_edges(upstream.clone()), w * small)
    close(run(x * small, with_edges(w.clone()), upstream * small)[1], upstream * small, with_edges(w.clone()))
    close(run(x * small, w * small, with_edges(upstream.clone()))[2], with_edges(upstream.clone()).t(), x * small)
    close(run(with_edges(x.clone()), w * small, upstream * small)[2], upstream.t() * small, with_edges(x.clone()))


@pytest.mark.gpu
@pytest.mark.parametrize("rows, width, hidden", [(5, 64, 70), (64, 64, 70), (600, 40, 700), (700, 2048, 1700),
                                                 (4000, 520, 1700)])
def test_operands_whose_low_parts_are_largest(rows, width, hidden) -> None:
    """Operands of 1 + 2^-11, halfway between two float16 values, where the product of the low parts that the
    larger layers leave out is largest and of one sign: the products, 1 + 2^-10 + 2^-22, are good to 2^-21
    and their sums, of equal terms, to that and eight roundings of 2^-24. The gate is tanh(30), one, so h is
    x Wu^T, the input's gradient dh Wu and the up weights' gradient dh^T x."""
    require_gpu_extension()
    show(f"low parts {rows} x {width} x {hidden}")
    value = 1.0 + 2.0**-11
    x, up_weight = leaf(torch.full((rows, width), value, device="cuda")), leaf(torch.full((hidden, width), -value, device="cuda"))
    gate_bias = torch.full((hidden,), 30.0, device="cuda")
    h = fused_hoad.gated_linear(x, torch.zeros_like(up_weight), up_weight, gate_bias, activation="tanh")
    dx, dw = torch.autograd.grad(h, (x, up_weight), torch.full_like(h, value))
    for got, count, sign in ((h, width, -1), (dx, hidden, -1), (dw, rows, 1)):
        want = sign * count * value * value
        assert float((got.double() - want).abs().max()) <= (2.0**-21 + 8 * 2.0**-24) * abs(want)
