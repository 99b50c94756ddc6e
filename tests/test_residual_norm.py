"""residual_norm against its formula in float64: every kind of gate and norm, widths that end inside
a vector, rows of one value and of the widest, shared gates and broadcast inputs, gradients against
float64 and differences, offsets far above the spread, zero rows, non-finite values, and refusals."""

from __future__ import annotations

import math

import pytest
import torch

import fused_hoad
from gpu_helpers import require_gpu_extension
from network_helpers import HALF_ULP, double, leaf, norm_error, normal, show

F32, BF16 = torch.float32, torch.bfloat16
NAMES = ("residual", "block", "gate", "weight", "bias", "post_weight", "post_bias")


def formula(t, scale, kind, eps):
    def norm(x, weight, bias):
        if kind == "layer":
            x = x - x.mean(-1, keepdim=True)
        x = x / ((x * x).mean(-1, keepdim=True) + eps).sqrt() * weight
        return x if bias is None else x + bias

    if t["block"] is None:
        return t["residual"], norm(t["residual"], t["weight"], t["bias"])
    n = t["block"]
    if t["post_weight"] is not None:
        n = norm(n, t["post_weight"], t["post_bias"])
    if t["gate"] is not None:
        n = t["gate"] * n
    hidden = scale * t["residual"] + n
    return hidden, norm(hidden, t["weight"], t["bias"])


def inputs(shape, dtype, kind, gate, post, bias, seed, offset=0.25):
    width = shape[-1]
    t = dict.fromkeys(NAMES)
    t["residual"] = normal(*shape, seed=seed, dtype=dtype, scale=2.0)
    t["block"] = (normal(*shape, seed=seed + 1) + offset).to(dtype)
    t["weight"] = (1 + normal(width, seed=seed + 2, scale=0.2)).to(dtype)
    if bias:
        t["bias"] = normal(width, seed=seed + 3, dtype=dtype, scale=0.2)
    if post:
        t["post_weight"] = (1 + normal(width, seed=seed + 4, scale=0.2)).to(dtype)
        if bias:
            t["post_bias"] = normal(width, seed=seed + 5, dtype=dtype, scale=0.2)
    if gate is not None:
        t["gate"] = (0.5 + normal(*gate, seed=seed + 6, scale=0.3)).to(dtype)
    return t


def call(t, scale=1.0, kind="rms", eps=1e-6):
    return fused_hoad.residual_norm(t["residual"], t["block"], t["gate"], weight=t["weight"], bias=t["bias"],
                                    post_weight=t["post_weight"], post_bias=t["post_bias"],
                                    residual_scale=scale, kind=kind, eps=eps)


def tolerance(dtype, terms) -> float:
    """Relative 2-norm error: statistics and sums of ``terms`` values in float32 (pairwise or in runs:
    at most 2^-24 sqrt(terms) for random signs), a dozen roundings of each value on its way, and for
    bfloat16 the result's one rounding."""
    return 2.0**-23 * (12 + math.sqrt(terms)) + (HALF_ULP[BF16] if dtype == BF16 else 0.0)


def check(shape, dtype=F32, kind="rms", gate=None, post=True, bias=False, scale=1.0, seed=0, tensors=None):
    require_gpu_extension()
    show(f"residual_norm {shape} {dtype} {kind} gate={gate} post={post} bias={bias} scale={scale}")
    t = {k: leaf(v) for k, v in (tensors or inputs(shape, dtype, kind, gate, post, bias, seed)).items()}
    up = [normal(*shape, seed=seed + 7, dtype=dtype), normal(*shape, seed=seed + 8, dtype=dtype)]
    outputs = call(t, scale, kind)
    wanted = [k for k in NAMES if t[k] is not None]
    grads = dict(zip(wanted, torch.autograd.grad(outputs, [t[k] for k in wanted], up)))
    exact = {k: double(v) for k, v in t.items()}
    outputs64 = formula(exact, scale, kind, 1e-6)
    grads64 = dict(zip(wanted, torch.autograd.grad(outputs64, [exact[k] for k in wanted], [u.double() for u in up])))
    rows = math.prod(shape[:-1])
    for name, got, want in (("hidden", outputs[0], outputs64[0]), ("normed", outputs[1], outputs64[1])):
        assert got.dtype == dtype and got.shape == want.shape
        error = norm_error(got, want)
        assert error <= tolerance(dtype, shape[-1]), f"{name}: {error:.3e}"
    for name in wanted:
        assert grads[name].dtype == dtype and grads[name].shape == t[name].shape
        error = norm_error(grads[name], grads64[name])
        assert error <= tolerance(dtype, rows + shape[-1]), f"{name}: {error:.3e}"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("width", [2, 3, 7, 8, 63, 64, 65, 255, 256, 511, 512, 513, 1000, 1024, 1025, 2047, 2049,
                                   4096, 4099, 8191, 8192, 8200, 16381, 16384])
def test_widths(width, dtype) -> None:
    # A layer norm of two values is +-1 whatever they are, and its gradient rounding alone.
    check((9, width), dtype, "layer" if width > 2 else "rms", (width,), bias=True, seed=width)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 2, 5, 257, 3001])
def test_rows(rows, dtype) -> None:
    check((rows, 96), dtype, "rms", (96,), seed=rows)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("post, bias", [(False, False), (True, False), (True, True), (False, True)])
@pytest.mark.parametrize("gate", ["none", "channel", "sample", "element"])
def test_forms(gate, post, bias, kind, dtype) -> None:
    shapes = {"none": None, "channel": (80,), "sample": (6, 1, 80), "element": (6, 11, 80)}
    check((6, 11, 80), dtype, kind, shapes[gate], post, bias, scale=1.5, seed=17)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("post, bias", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("gate", ["none", "channel", "sample", "element"])
@pytest.mark.parametrize("width", [8201, 10001, 16384])
def test_forms_of_wide_rows(width, gate, post, bias, dtype) -> None:
    """Two rows to a workgroup, in layouts that read a row's values again in each pass."""
    shape = (3, 100, width)
    gates = {"none": None, "channel": (width,), "sample": (3, 1, width), "element": shape}
    check(shape, dtype, "layer" if bias else "rms", gates[gate], post=post, bias=bias, scale=0.7, seed=width)


@pytest.mark.gpu
@pytest.mark.parametrize("shape, gate", [
    ((3000, 2, 72), (3000, 1, 72)),     # more gate rows than workgroups
    ((2, 3000, 72), (2, 1, 72)),        # few gate rows, split over workgroups
    ((5, 700, 1365), (5, 1, 1365)),     # the same with a workgroup to a row, odd width
    ((4, 3, 5, 40), (4, 3, 1, 40)),     # two leading dimensions
    ((4, 3, 5, 40), (4, 1, 1, 40)),     # one leading dimension, shared over two
    ((4, 3, 5, 40), (1, 1, 1, 40)),     # a channel gate with dimensions of one
    ((1, 7, 40), (1, 1, 40)),
    ((7, 1, 40), (7, 1, 40)),
    ((1, 1, 40), (40,)),
])
def test_shared_gates(shape, gate) -> None:
    check(shape, F32, "rms", gate, seed=23)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("shape", [(1, 256), (33, 77), (2, 5, 1030)])
def test_without_a_block(shape, kind, dtype) -> None:
    tensors = inputs(shape, dtype, kind, None, False, kind == "layer", 3)
    tensors["block"] = None
    check(shape, dtype, kind, tensors=tensors)


@pytest.mark.gpu
def test_one_output_alone() -> None:
    """A loss on one of the outputs only: the other's gradient counts as zero."""
    require_gpu_extension()
    t = {k: leaf(v) for k, v in inputs((40, 60), F32, "layer", (60,), True, True, 5).items()}
    up = normal(40, 60, seed=9)
    for which in (0, 1):
        grads = torch.autograd.grad(call(t, kind="layer")[which], list(t.values()), up, allow_unused=True)
        exact = {k: double(v) for k, v in t.items()}
        want = torch.autograd.grad(formula(exact, 1.0, "layer", 1e-6)[which], list(exact.values()), up.double(),
                                   allow_unused=True)
        for name, got, expected in zip(t, grads, want):
            if expected is None:  # the gradient of what the output does not depend on
                assert got is None or not got.any(), name
            else:
                assert norm_error(got, expected) <= tolerance(F32, 100), name


@pytest.mark.gpu
@pytest.mark.parametrize("width", [300, 3000])
def test_offset_far_above_the_spread(width) -> None:
    """A layer norm of values about 1,000 with a spread of one: the mean is taken out before squares are
    summed, so the error is that of the inputs' own rounding, 2^-24 of 1,000 over the spread (6e-5),
    and not of squares of a million (6e-2)."""
    require_gpu_extension()
    t = inputs((20, width), F32, "layer", None, True, False, 1, offset=1000.0)
    t["residual"] += 1000.0
    hidden, normed = call(t, kind="layer")
    hidden64, normed64 = formula({k: double(v) for k, v in t.items()}, 1.0, "layer", 1e-6)
    assert norm_error(hidden, hidden64) <= 2e-6
    assert norm_error(normed, normed64) <= 2e-4


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_zero_and_non_finite_rows(dtype) -> None:
    """A row of zeros is normalised to zeros (to the bias with one); a NaN or an infinity makes its
    own row non-finite and leaves the others bitwise alone."""
    require_gpu_extension()
    t = inputs((12, 200), dtype, "rms", (200,), True, True, 2)
    t["post_bias"] = None
    t["residual"][3] = 0
    t["block"][3] = 0
    hidden, normed = call(t)
    assert not hidden[3].any() and torch.equal(normed[3], t["bias"])
    for value in (math.nan, math.inf):
        bad = {k: v if v is None else v.clone() for k, v in t.items()}
        bad["block"][5, 17] = value
        hidden2, normed2 = call(bad)
        assert torch.isnan(normed2[5]).any()
        rest = [r for r in range(12) if r != 5]
        assert torch.equal(hidden2[rest], hidden[rest]) and torch.equal(normed2[rest], normed[rest])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("width", [77, 1365, 7013])
@pytest.mark.parametrize("column", [-1, -3, 0])
def test_infinite_weight(column, width, dtype) -> None:
    """Its own gradient is NaN and the other columns' infinite, as in the formula, wherever it lies in
    the row: in the last columns, too, which a thread holds beside zeros."""
    require_gpu_extension()
    show(f"residual_norm infinite weight at {column} of {width} {dtype}")
    residual, weight = normal(3, width, seed=width, dtype=dtype), torch.ones(width, device="cuda", dtype=dtype)
    weight[column] = math.inf
    up = torch.where(normal(3, width, seed=width + 1) > 0, 1.0, -1.0).to(dtype)
    got, want = [], []
    for x, w, into in ((leaf(residual), weight, got), (double(residual), weight.double(), want)):
        if into is got:
            outputs = fused_hoad.residual_norm(x, weight=w)
        else:
            outputs = formula(dict.fromkeys(NAMES) | {"residual": x, "weight": w}, 1.0, "rms", 1e-6)
        into.append(torch.autograd.grad(outputs[1], x, up.to(x.dtype))[0].double())
    assert torch.equal(got[0].isnan(), want[0].isnan()) and got[0].isnan().sum() == 3
    keep = ~want[0].isnan()
    assert torch.equal(got[0][keep], want[0][keep]) and got[0][keep].isinf().all()


@pytest.mark.gpu
def test_gradient_against_differences() -> None:
    """Central differences of the kernel's own forward, as for gated_linear: step 2^-7 of the input's
    size, 2e-3 of the scale allowed."""
    require_gpu_extension()
    for kind, gate in (("rms", (64,)), ("layer", (4, 1, 64)), ("layer", (4, 9, 64))):
        show(f"differences {kind} {gate}")
        t = {k: leaf(v) for k, v in inputs((4, 9, 64), F32, kind, gate, True, True, 41).items()}
        up = [normal(4, 9, 64, seed=50), normal(4, 9, 64, seed=51)]
        grads = dict(zip(t, torch.autograd.grad(call(t, 1.25, kind), list(t.values()), up)))
        for name, grad in grads.items():
            direction = normal(*t[name].shape, seed=60)
            direction = direction * (t[name].detach().norm() / direction.norm())
            values = []
            for sign in (1, -1):
                moved = {k: v.detach() for k, v in t.items()}
                moved[name] = moved[name] + sign * 2.0**-7 * direction
                values.append(sum((o.double() * u).sum() for o, u in zip(call(moved, 1.25, kind), up)))
            slope = (values[0] - values[1]) / 2.0**-6
            scale = grad.double().norm() * direction.double().norm()
            assert abs(float(slope - (grad.double() * direction).sum())) <= 2e-3 * float(scale), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_unaligned_strided_and_broadcast_inputs(dtype) -> None:
    require_gpu_extension()
    t = inputs((30, 48), dtype, "rms", (48,), True, False, 6)
    plain = call(t)
    for name in ("residual", "block", "gate", "weight", "post_weight"):
        storage = torch.empty(t[name].numel() + 1, dtype=dtype, device="cuda")
        view = storage[1:].view(t[name].shape)
        view.copy_(t[name])
        assert all(torch.equal(a, b) for a, b in zip(call({**t, name: view}), plain)), name
    strided = {**t, "residual": t["residual"].t().contiguous().t()}
    assert all(torch.equal(a, b) for a, b in zip(call(strided), plain))
    row = leaf(t["block"][:1])
    hidden, normed = call({**t, "block": row.expand(30, 48)})
    up = [normal(30, 48, seed=7, dtype=dtype), normal(30, 48, seed=8, dtype=dtype)]
    got, = torch.autograd.grad((hidden, normed), row, up)
    exact = double(row)
    want, = torch.autograd.grad(formula({**{k: double(v) for k, v in t.items()}, "block": exact.expand(30, 48)},
                                        1.0, "rms", 1e-6), exact, [u.double() for u in up])
    # Each of the 30 rows' gradients is rounded, and their sum once more.
    assert norm_error(got, want) <= tolerance(dtype, 30 + 48) * 2


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_repeats_graphs_and_empty(dtype) -> None:
    require_gpu_extension()
    t = {k: leaf(v) for k, v in inputs((8, 90, 136), dtype, "layer", (8, 1, 136), True, True, 12).items()}
    up = [normal(8, 90, 136, seed=13, dtype=dtype), normal(8, 90, 136, seed=14, dtype=dtype)]

    def run():
        outputs = call(t, kind="layer")
        # Detached: a graph that is kept would hold the leaves' gradient nodes on this stream, and a
        # capture cannot wait on the default stream.
        return [o.detach() for o in outputs] + list(torch.autograd.grad(outputs, list(t.values()), up))

    first = run()
    assert all(torch.equal(a, b) for a, b in zip(first, run()))
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(call(t, kind="layer"), first))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = run()
    for seed in (71, 72, 73):
        with torch.no_grad():
            t["residual"].copy_(normal(8, 90, 136, seed=seed, dtype=dtype))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(static, run()))
    empty = {k: leaf(v) for k, v in inputs((0, 40), dtype, "layer", (40,), True, True, 1).items()}
    outputs = call(empty, kind="layer")
    assert outputs[0].shape == (0, 40) and outputs[1].shape == (0, 40)
    for name, grad in zip(empty, torch.autograd.grad(outputs, list(empty.values()), [o.detach() for o in outputs])):
        assert grad.shape == empty[name].shape and not grad.any()


def test_refusals_on_the_cpu() -> None:
    with pytest.raises(RuntimeError, match="residual must be a CUDA tensor"):
        fused_hoad.residual_norm(torch.zeros(2, 4), weight=torch.zeros(4))
    with pytest.raises(RuntimeError, match="kind must be"):
        fused_hoad.residual_norm(torch.zeros(2, 4), weight=torch.zeros(4), kind="batch")


@pytest.mark.gpu
def test_refusals() -> None:
    require_gpu_extension()
    x, w = normal(3, 5, 8, seed=0), normal(8, seed=1)
    norm = fused_hoad.residual_norm
    for bad, message in (
        (lambda: norm(x.double(), weight=w), "float32 or bfloat16"),
        (lambda: norm(x, weight=w.bfloat16()), "weight must have residual's dtype"),
        (lambda: norm(x, weight=w[:7]), r"weight must have shape \[8\]"),
        (lambda: norm(x, x[:, :4], weight=w), "block must have residual's shape"),
        (lambda: norm(x, x.cpu(), weight=w), "block must be a CUDA tensor"),
        (lambda: norm(x, weight=w, post_weight=w), "need a block"),
        (lambda: norm(x, weight=w, residual_scale=2.0), "need a block"),
        (lambda: norm(x, x, weight=w, post_bias=w), "post_bias needs post_weight"),
        (lambda: norm(x, x, normal(1, 5, 8, seed=2), weight=w), "first dimensions"),
        (lambda: norm(x, x, normal(3, 4, 8, seed=2), weight=w), "gate must broadcast"),
        (lambda: norm(x, x, normal(3, 5, 1, seed=2), weight=w), "gate must broadcast"),
        (lambda: norm(x, x, weight=w, eps=-1.0), "eps must be non-negative"),
        (lambda: norm(normal(1, 16385, seed=3), weight=normal(16385, seed=4)), "width must be at most 16384"),
    ):
        with pytest.raises(RuntimeError, match=message):
            bad()
    leaves = [leaf(x), leaf(w)]
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(norm(leaves[0], weight=leaves[1])[1].sum(), leaves[0], create_graph=True)


@pytest.mark.gpu
@pytest.mark.parametrize("needs_grad", [False, True])
def test_forward_mode_is_refused(needs_grad) -> None:
    """A dual tensor in any place raises, with and without gradient mode, instead of losing its tangent;
    the tensors that lie in it are taken as before."""
    from torch.autograd import forward_ad

    require_gpu_extension()
    show("residual_norm dual tensors")
    t = inputs((4, 8), F32, "layer", (8,), True, True, 3)
    plain = call(t, kind="layer")
    with forward_ad.dual_level(), torch.set_grad_enabled(needs_grad):
        for name, value in t.items():
            dual = forward_ad.make_dual(leaf(value) if needs_grad else value, torch.ones_like(value))
            with pytest.raises(RuntimeError, match="residual_norm has no forward-mode derivative"):
                call({**t, name: dual}, kind="layer")
            outputs = call({**t, name: forward_ad.unpack_dual(dual).primal}, kind="layer")
            assert all(torch.equal(a, b) for a, b in zip(outputs, plain))
        dual = forward_ad.make_dual(t["residual"], torch.ones_like(t["residual"]))
        with pytest.raises(RuntimeError, match="residual_norm has no forward-mode derivative"):
            fused_hoad.residual_norm(dual, weight=t["weight"])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("width", [8201, 10001, 16381])
@pytest.mark.parametrize("column", [-1, -3, 0])
def test_infinite_weight_of_wide_rows(column, width, dtype) -> None:
    """As test_infinite_weight, where a row's values are read again in each pass."""
    test_infinite_weight(column, width, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("unaligned", [False, True])
@pytest.mark.parametrize("gate", ["none", "channel", "sample", "element"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_rows_of_one_value(kind, gate, unaligned, dtype) -> None:
    """Rows shorter than any vector, element by element against float64, where norms cancel: each rounding
    counts as 2^-24 of a term, sixteen of them to a value, forty-eight more to a sum over the rows, and in
    bfloat16 the result's.

    RMS: the gradient through a norm, eps / (x^2 + eps)^(3/2) w dy, is what two terms of about w dy / |x|
    leave. Layer: a value is its own mean, so a norm gives its bias exactly, and nothing goes back through the
    first norm. Through the second goes what one rounding of hidden (below 8, formed again in the backward) makes
    of it at 1 / sqrt(eps) = 1,000: a unit value of u = 1,000 x 2^-20 instead of zero, and by its square and the
    rounding of w dy 1,000 (u^2 + 2^-23) = 0.00103 of w dy."""
    require_gpu_extension()
    show(f"residual_norm one value {kind} {gate} {unaligned} {dtype}")
    shape = (3, 50, 1)
    gates = {"none": None, "channel": (1,), "sample": (3, 1, 1), "element": shape}
    t = inputs(shape, dtype, kind, gates[gate], True, kind == "layer", 5)
    for name in ("residual", "block"):  # away from zero, where what cancels has no bound
        t[name] = (t[name].abs().clamp(max=3.0) + 1.0).to(dtype)
    if unaligned:
        for name, value in t.items():
            if value is not None:
                t[name] = torch.empty(value.numel() + 1, dtype=dtype, device="cuda")[1:].view(value.shape).copy_(value)
    t = {k: None if v is None else v.requires_grad_(True) for k, v in t.items()}
    up = [normal(*shape, seed=9, dtype=dtype), normal(*shape, seed=10, dtype=dtype)]
    outputs = call(t, 1.5, kind)
    wanted = [k for k in NAMES if t[k] is not None]
    grads = dict(zip(wanted, torch.autograd.grad(outputs, [t[k] for k in wanted], up)))
    exact = {k: double(v) for k, v in t.items()}
    outputs64 = formula(exact, 1.5, kind, 1e-6)
    grads64 = dict(zip(wanted, torch.autograd.grad(outputs64, [exact[k] for k in wanted], [u.double() for u in up])))
    rounding = HALF_ULP[BF16] if dtype == BF16 else 0.0
    one = torch.ones(1, device="cuda", dtype=torch.float64)

    def size(name):
        return one if exact[name] is None else exact[name].detach().abs()

    def summed(values, like):
        values = values.expand(shape)
        return values if like.shape == shape else values.sum((0, 1) if like.dim() == 1 else 1).reshape(like.shape)

    if kind == "layer":
        assert torch.equal(outputs[1], t["bias"].detach().expand(shape))
        assert not grads["block"].any() and not grads["post_weight"].any()
    for got, want in zip(outputs, outputs64):
        assert bool(((got.double() - want).abs() <= (2.0**-20 + rounding) * want.abs() + 2.0**-20).all())
    dh, dy = (u.double().abs() for u in up)
    unit = 1000 * 2.0**-20 if kind == "layer" else 0.0
    through = 0.00103 * size("weight") * dy if kind == "layer" else 2.0**-20 * size("weight") * dy / outputs64[0].detach().abs()
    total = dh + size("weight") * dy / (outputs64[0].detach().abs() if kind == "rms" else one)
    branch = size("post_weight") if kind == "rms" else size("post_bias")
    bounds = {
        "residual": 1.5 * (through + 2.0**-20 * dh),
        "block": 2.0**-20 * size("gate") * total * size("post_weight") / size("block"),
        "gate": branch * (2.0**-18 * total + through),
        "weight": (2.0**-18 + unit) * dy * 1.01,
        "bias": 2.0**-18 * dy,
        "post_weight": size("gate") * (2.0**-18 * total + through) * 1.01,
        "post_bias": size("gate") * (2.0**-18 * total + through),
    }
    for name in wanted:
        want = grads64[name]
        bound = summed(bounds[name], want) + rounding * want.abs()
        assert bool(((grads[name].double() - want).abs() <= bound).all()), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", ["none", "channel", "element"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("width", [40, 1365, 6001, 12001])
def test_hidden_alone_with_a_masked_row(width, kind, gate, post, dtype) -> None:
    """A loss on hidden alone, whose mask leaves out a row that holds an infinity in the residual: nothing goes
    through the second norm, so the row's gradients are zeros, the other rows' and the sums are finite and
    as in float64, and the second norm's weight and bias have none."""
    require_gpu_extension()
    show(f"residual_norm hidden alone {width} {kind} {gate} post={post} {dtype}")
    shape = (7, width)
    t = inputs(shape, dtype, kind, {"none": None, "channel": (width,), "element": shape}[gate], post, kind == "layer", 8)
    t["residual"][2, width // 2] = math.inf
    t = {k: leaf(v) for k, v in t.items()}
    up = normal(*shape, seed=9, dtype=dtype)
    up[2] = 0
    wanted = [k for k in NAMES if t[k] is not None]
    grads = dict(zip(wanted, torch.autograd.grad(call(t, 1.5, kind)[0], [t[k] for k in wanted], up, allow_unused=True)))
    exact = {k: double(v) for k, v in t.items()}
    want = dict(zip(wanted, torch.autograd.grad(formula(exact, 1.5, kind, 1e-6)[0], [exact[k] for k in wanted],
                                                up.double(), allow_unused=True)))
    for name in wanted:
        if want[name] is None:
            assert grads[name] is None or not grads[name].any(), name
            continue
        if name in ("residual", "block") or (name == "gate" and gate == "element"):
            assert not grads[name][2].any(), name
        assert norm_error(grads[name], want[name]) <= tolerance(dtype, 7 + width), name
