"""adamw_step and FusedAdamW: 32-bit results to the bit against the formula evaluated step by step in
float32 and close to float64 and torch.optim.AdamW; 8-bit states against the codes' definition;
tensors of every size and alignment, missing gradients, many tensors, non-finite gradients, rounding
without bias, state dicts, graphs and refusals."""

from __future__ import annotations

import collections
import copy
import math

import pytest
import torch

import fused_hoad
from fused_hoad.optim import STATE_BLOCK, state_span
from gpu_helpers import require_gpu_extension
from network_helpers import norm_error, normal, show

F32, BF16 = torch.float32, torch.bfloat16
OPTIONS = {"lr": 2e-3, "betas": (0.9, 0.99), "eps": 1e-8, "weight_decay": 0.05}
SHAPES = [(1,), (3,), (255,), (256,), (257,), (0,), (7, 11), (64, 171), (2, 3, 4), (5000,), (4096,), (4097,), (20011,)]


def packed(tensors):
    """Float32 values of the tensors in the packed layout, zeros between them."""
    pieces = []
    for t in tensors:
        flat = t.detach().reshape(-1).float()
        pieces += [flat, flat.new_zeros(state_span(flat.numel()) - flat.numel())]
    return torch.cat(pieces)


def unpacked(flat, like):
    out, at = [], 0
    for t in like:
        out.append(flat[at : at + t.numel()].view(t.shape))
        at += state_span(t.numel())
    return out


class Plain:
    """The step in elementary float32 operations on the packed layout, each rounded by itself."""

    def __init__(self, tensors, options, bits, seed):
        self.options, self.bits, self.seed = options, bits, seed
        self.like = tensors
        self.counts = torch.tensor([state_span(t.numel()) for t in tensors], device="cuda")
        self.steps = torch.zeros(len(tensors), dtype=torch.int64, device="cuda")
        size = fused_hoad.packed_state_size(tensors)
        self.mean = torch.zeros(size, device="cuda")
        self.square = torch.zeros(size, device="cuda")
        self.codes = None

    def each(self, values):
        return torch.repeat_interleave(values, self.counts)

    def step(self, parameters, gradients):
        o, (beta1, beta2) = self.options, self.options["betas"]
        has = torch.tensor([g is not None for g in gradients], device="cuda")
        self.steps += has
        t = self.steps.clamp(min=1).double()
        size = self.each((o["lr"] / (1 - beta1**t)).float())
        root = self.each((1 / torch.sqrt(1 - beta2**t)).float())
        on = self.each(has)
        p = packed(parameters)
        g = packed([torch.zeros_like(a) if b is None else b for a, b in zip(parameters, gradients)])
        mean = self.mean * beta1 + g * (1 - beta1)
        square = self.square * beta2 + g * g * (1 - beta2)
        deviation = torch.sqrt(square)
        new = p * (1 - o["lr"] * o["weight_decay"]) - size * (mean / (deviation * root + o["eps"]))
        if self.bits == 8:
            random = random_bits(p.numel(), self.seed, self.each(self.steps))
            codes = encode(mean, random >> 16, 3) + encode(deviation, random & 0xFFFF, 4)
            mean, deviation = decode(codes[0], codes[1], 3), decode(codes[2], codes[3], 4)
            square = deviation * deviation
            old = self.codes or codes
            blocks = on.view(-1, STATE_BLOCK)[:, 0]
            self.codes = tuple(torch.where(on if c.numel() == on.numel() else blocks, c, b) for c, b in zip(codes, old))
        self.mean = torch.where(on, mean, self.mean)
        self.square = torch.where(on, square, self.square)
        return [v.to(a.dtype) if b is not None else a
                for v, a, b in zip(unpacked(new, parameters), parameters, gradients)]


def mix(x):
    x = ((x ^ (x >> 16)) * 0x9E3779B9) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x6A09E667) & 0xFFFFFFFF
    return x ^ (x >> 16)


def random_bits(count, seed, steps):
    key = mix((steps + mix(torch.full_like(steps, seed))) & 0xFFFFFFFF)
    return mix(torch.arange(count, device=steps.device) ^ key)


def values_of_codes(mantissa):
    """What each code stands for before its scale, from the format's definition."""
    codes = torch.arange(256, dtype=torch.float64)
    magnitude = codes % 128 if mantissa == 3 else codes
    exponent = torch.floor(magnitude / 2**mantissa)
    fraction = magnitude - exponent * 2**mantissa
    value = torch.where(exponent > 0, (1 + fraction / 2**mantissa) * 2.0 ** (exponent - 15),
                        fraction / 2**mantissa * 2.0**-14)
    return torch.where(codes >= 128, -value, value) if mantissa == 3 else value


def decode(codes, scales, mantissa):
    table = values_of_codes(mantissa).float().to(codes.device)
    return (table[codes.long()].view(-1, STATE_BLOCK) * scales[:, None]).view(-1)


def encode(x, random, mantissa):
    """Codes by search in the table of values: the largest one not above |x| / scale, or the next with
    the probability of the remainder (16 random bits)."""
    largest = 2.0 - 2.0**-mantissa
    top = x.abs().view(-1, STATE_BLOCK).amax(1)
    top = torch.where(top < 2.0**-100, 0.0, top)
    scale = top * (1 / largest)
    inverse = torch.where(top > 0, 1 / scale, 0.0)
    y = (x.abs().view(-1, STATE_BLOCK) * inverse[:, None]).view(-1).double()
    table = values_of_codes(mantissa)[: 128 if mantissa == 3 else 256].to(x.device)
    last = table.numel() - 1
    below = (torch.searchsorted(table, y, right=True) - 1).clamp(max=last)
    spacing = 2.0 ** (torch.floor(torch.log2(y.clamp(min=2.0**-14))) - mantissa)
    code = below + (torch.floor((y - table[below]) / spacing * 65536) + random >= 65536)
    code = code.clamp(max=last)
    if mantissa == 3:
        return (code + 128 * (x < 0)).to(torch.uint8), scale
    return torch.where(y > 0, code.clamp(min=1), code).to(torch.uint8), scale


def tensors_of(shapes, dtype, seed=0, scale=1.0):
    return [normal(*s, seed=seed + k, dtype=dtype, scale=scale) for k, s in enumerate(shapes)]


def state_of(optimizer):
    return optimizer._packs[0]


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_steps_to_the_bit(dtype, bits) -> None:
    """Five steps over tensors of every size, one of them without a gradient in two of the steps:
    parameters, moments (codes and scales) and step counts equal the plain form's exactly."""
    require_gpu_extension()
    show(f"adamw {dtype} {bits}")
    parameters = [torch.nn.Parameter(p) for p in tensors_of(SHAPES, dtype)]
    optimizer = fused_hoad.FusedAdamW(parameters, state_bits=bits, seed=77, **OPTIONS)
    plain = Plain(parameters, OPTIONS, bits, 77)
    expected = [p.detach().clone() for p in parameters]
    for step in range(5):
        gradients = tensors_of(SHAPES, dtype, seed=100 * (step + 1), scale=10.0 ** (step - 3))
        if step in (1, 3):
            gradients[7] = None
        for p, g in zip(parameters, gradients):
            p.grad = g
        optimizer.step()
        expected = plain.step(expected, gradients)
        for k, (p, e) in enumerate(zip(parameters, expected)):
            assert torch.equal(p.detach(), e), (step, k)
        pack = state_of(optimizer)
        assert torch.equal(pack["step"].long(), plain.steps)
        if bits == 32:
            assert torch.equal(pack["exp_avg"], plain.mean) and torch.equal(pack["exp_avg_sq"], plain.square)
        else:
            names = ("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale")
            for name, want in zip(names, plain.codes):
                assert torch.equal(pack[name], want), (step, name)
            for k, p in enumerate(parameters):
                mean, square = optimizer.moments(p)
                assert torch.equal(mean, unpacked(plain.mean, parameters)[k])
                assert torch.equal(square, unpacked(plain.square, parameters)[k])


@pytest.mark.gpu
def test_against_torch_adamw_in_float64() -> None:
    """Twenty steps against torch.optim.AdamW in float64. A parameter's relative error grows by at
    most a few roundings (2^-24) a step: 20 x 4 x 2^-24 = 5e-6 of its size."""
    require_gpu_extension()
    start = tensors_of([(64, 171), (171,), (1000,)], F32)
    ours = [torch.nn.Parameter(p.clone()) for p in start]
    theirs = [torch.nn.Parameter(p.double()) for p in start]
    optimizers = [fused_hoad.FusedAdamW(ours, **OPTIONS), torch.optim.AdamW(theirs, **OPTIONS)]
    for step in range(20):
        for a, b, g in zip(ours, theirs, tensors_of([(64, 171), (171,), (1000,)], F32, seed=1000 + 10 * step)):
            a.grad, b.grad = g, g.double()
        for optimizer in optimizers:
            optimizer.step()
    for a, b in zip(ours, theirs):
        assert norm_error(a, b) <= 5e-6
        assert norm_error(optimizers[0].moments(a)[0], optimizers[1].state[b]["exp_avg"]) <= 5e-6
        assert norm_error(optimizers[0].moments(a)[1], optimizers[1].state[b]["exp_avg_sq"]) <= 5e-6


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_unaligned_views_and_strided_gradients(dtype, bits) -> None:
    """Parameters and gradients at odd offsets of a buffer, and gradients that are transposed or
    expanded, give bitwise what aligned contiguous ones give."""
    require_gpu_extension()
    show(f"adamw views {dtype} {bits}")
    shapes = [(33, 17), (300,), (1001,)]
    start, grads = tensors_of(shapes, dtype), tensors_of(shapes, dtype, seed=9)
    grads[1] = grads[1][:1].expand(300)
    results = []
    for moved in (False, True):
        parameters = []
        for p in start:
            storage = torch.zeros(p.numel() + 2, dtype=dtype, device="cuda")
            view = storage[1:-1] if moved else storage[:-2]
            parameters.append(torch.nn.Parameter(view.view(p.shape)))
            parameters[-1].data.copy_(p)
        optimizer = fused_hoad.FusedAdamW(parameters, state_bits=bits, seed=5, **OPTIONS)
        for p, g in zip(parameters, grads):
            p.grad = g if moved else g.clone(memory_format=torch.contiguous_format)
        if moved:
            parameters[0].grad = grads[0].t().contiguous().t()
            storage = torch.empty(grads[2].numel() + 1, dtype=dtype, device="cuda")
            storage[1:].copy_(grads[2])
            parameters[2].grad = storage[1:]
        optimizer.step()
        optimizer.step()
        results.append([p.detach().clone() for p in parameters] + [state_of(optimizer)["exp_avg"]])
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_more_tensors_than_a_launch_takes_and_mixed_types(bits) -> None:
    require_gpu_extension()
    show(f"adamw 250 tensors {bits}")
    shapes = [((37 * k) % 700 + 1,) for k in range(250)]
    dtypes = [BF16 if k % 3 == 0 else F32 for k in range(250)]
    parameters = [torch.nn.Parameter(normal(*s, seed=k, dtype=d)) for k, (s, d) in enumerate(zip(shapes, dtypes))]
    gradients = [normal(*s, seed=1000 + k, dtype=d) for k, (s, d) in enumerate(zip(shapes, dtypes))]
    expected = [p.detach().clone() for p in parameters]
    optimizer = fused_hoad.FusedAdamW(parameters, state_bits=bits, **OPTIONS)
    plain = Plain(parameters, OPTIONS, bits, 0)
    for _ in range(2):
        for p, g in zip(parameters, gradients):
            p.grad = g
        optimizer.step()
        expected = plain.step(expected, gradients)
    assert all(torch.equal(p.detach(), e) for p, e in zip(parameters, expected))
    assert bool((state_of(optimizer)["step"] == 2).all())


@pytest.mark.gpu
def test_rounding_has_no_bias() -> None:
    """The mean of the codes' values over 2^16 equal elements and their steps equals the value rounded,
    within five standard errors: a code's spacing is at most 1/8 (first moment, of the value) or 1/16
    (the root), its standard deviation at most half of that, and the random bits' grid 2^-17."""
    require_gpu_extension()
    count = 1 << 16
    for fraction in (0.011, 0.3, 0.77):
        p = torch.nn.Parameter(torch.zeros(count, device="cuda"))
        p.grad = torch.full((count,), fraction, device="cuda")
        p.grad[::STATE_BLOCK] = 1.0  # the block's largest value
        optimizer = fused_hoad.FusedAdamW([p], lr=0.0, betas=(0.5, 0.75), state_bits=8, seed=3)
        optimizer.step()
        mean, square = optimizer.moments(p)
        rest = torch.arange(count, device="cuda") % STATE_BLOCK != 0
        for got, want, spacing in ((mean[rest], 0.5 * fraction, 1 / 8), (square[rest].sqrt(), 0.5 * fraction, 1 / 16)):
            error = abs(float(got.double().mean()) / want - 1)
            assert error <= spacing * (5 * 0.5 / math.sqrt(count) + 2.0**-17) + 2.0**-20, (fraction, error)
            assert float((got / want - 1).abs().max()) <= spacing


@pytest.mark.gpu
def test_slow_second_moments_decay_and_never_reach_zero() -> None:
    """With beta2 = 0.999 a second moment's root loses 0.05 % a step, a hundredth of a code's spacing.
    After 1,000 steps without gradients in half of a block it has fallen as in 32 bits (to
    0.999^500 = 0.61 of itself), within the random walk of the codes (about 14 % an element, 2 % for
    the mean of 128); rounding to nearest would leave it where it was. No root is zero."""
    require_gpu_extension()
    p = torch.nn.Parameter(torch.zeros(256, device="cuda"))
    optimizer = fused_hoad.FusedAdamW([p], lr=0.0, state_bits=8, seed=11)
    p.grad = torch.ones(256, device="cuda")
    optimizer.step()
    first = optimizer.moments(p)[1].sqrt()
    p.grad[:128] = 0.0
    for _ in range(1000):
        optimizer.step()
    root = optimizer.moments(p)[1].sqrt()
    assert abs(float((root[:128] / first[:128]).mean()) - 0.999**500) <= 0.1
    p.grad.zero_()
    p.grad[0] = 1e6
    optimizer.step()
    assert bool((optimizer.moments(p)[1] > 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_zero_tiny_and_non_finite_gradients(bits) -> None:
    """Zero gradients move a parameter by its decay alone; gradients whose moments are below 2^-100
    leave 8-bit states zero; a non-finite gradient makes its own element non-finite and the state of
    no other block."""
    require_gpu_extension()
    show(f"adamw special {bits}")
    for value in (0.0, 1e-36):
        p = torch.nn.Parameter(torch.ones(600, device="cuda"))
        p.grad = torch.full((600,), value, device="cuda")
        optimizer = fused_hoad.FusedAdamW([p], state_bits=bits, **OPTIONS)
        optimizer.step()
        assert bool(torch.isfinite(p).all())
        if value == 0.0:
            decay = torch.tensor(1 - OPTIONS["lr"] * OPTIONS["weight_decay"])
            assert torch.equal(p.detach().cpu(), decay.expand(600))
        if bits == 8:
            assert not state_of(optimizer)["exp_avg"].any() and not state_of(optimizer)["exp_avg_sq"].any()
    for value in (math.nan, math.inf):
        p = torch.nn.Parameter(torch.ones(600, device="cuda"))
        p.grad = torch.ones(600, device="cuda")
        p.grad[300] = value
        optimizer = fused_hoad.FusedAdamW([p], state_bits=bits, **OPTIONS)
        optimizer.step()
        finite = torch.isfinite(p.detach())
        assert not finite[300] and int((~finite).sum()) == 1
        mean, square = optimizer.moments(p)
        outside = [k for k in range(600) if (k // 256 != 1 if bits == 8 else k != 300)]
        assert bool(torch.isfinite(mean[outside]).all() and torch.isfinite(square[outside]).all())
        assert not torch.isfinite(square[300])


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_state_dicts_copies_and_groups(dtype, bits) -> None:
    """A run that is saved and loaded, or copied, goes on bitwise like one that was not interrupted;
    a second group has its own options and state."""
    require_gpu_extension()
    shapes = [(40, 9), (300,), (7,)]

    def build():
        parameters = [torch.nn.Parameter(p) for p in tensors_of(shapes, dtype)]
        optimizer = fused_hoad.FusedAdamW([{"params": parameters[:2]}, {"params": parameters[2:], "lr": 0.5}],
                                          state_bits=bits, seed=4, **OPTIONS)
        return parameters, optimizer

    def advance(parameters, optimizer, steps):
        for step in steps:
            for p, g in zip(parameters, tensors_of(shapes, dtype, seed=10 * step)):
                p.grad = g
            optimizer.step()

    whole, optimizer = build()
    advance(whole, optimizer, range(1, 7))
    part, first = build()
    advance(part, first, range(1, 4))
    saved = copy.deepcopy(first.state_dict())
    assert set(saved["param_groups"][0]) >= {"lr", "state_bits", "seed"}
    loaded = [torch.nn.Parameter(p.detach().clone()) for p in part]
    second = fused_hoad.FusedAdamW([{"params": loaded[:2]}, {"params": loaded[2:]}], lr=9.0)
    second.load_state_dict(saved)
    assert second.param_groups[0]["lr"] == OPTIONS["lr"] and second.param_groups[1]["lr"] == 0.5
    advance(loaded, second, range(4, 7))
    assert all(torch.equal(a, b) for a, b in zip(whole, loaded))
    assert torch.equal(optimizer.state[whole[0]]["exp_avg"], second.state[loaded[0]]["exp_avg"])
    model = torch.nn.ParameterList(p.detach().clone() for p in part)
    pair = copy.deepcopy((part, first))
    advance(pair[0], pair[1], range(4, 7))
    assert all(torch.equal(a, b) for a, b in zip(whole, pair[0]))
    advance(part, first, range(4, 7))
    assert all(torch.equal(a, b) for a, b in zip(whole, part))
    with pytest.raises(ValueError, match="do not match"):
        fused_hoad.FusedAdamW(model).load_state_dict(saved)
    other = fused_hoad.FusedAdamW([{"params": loaded[:2]}, {"params": loaded[2:]}], state_bits=bits)
    for group in saved["param_groups"]:
        group["state_bits"] = 40 - bits
    with pytest.raises(ValueError, match="does not fit"):
        other.load_state_dict(saved)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_graph_replays(bits) -> None:
    """A captured step, replayed on new gradients with eager work between, equals eager steps bitwise."""
    require_gpu_extension()
    show(f"adamw graph {bits}")
    shapes = [(64, 33), (500,)]
    sets = []
    for _ in range(2):
        parameters = [torch.nn.Parameter(p) for p in tensors_of(shapes, F32)]
        for p in parameters:
            p.grad = torch.zeros_like(p)
        sets.append((parameters, fused_hoad.FusedAdamW(parameters, state_bits=bits, seed=8, **OPTIONS)))

    def feed(parameters, step):
        for p, g in zip(parameters, tensors_of(shapes, F32, seed=10 * step)):
            p.grad.copy_(g)

    for parameters, optimizer in sets:  # the first step allocates the state
        feed(parameters, 1)
        optimizer.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sets[0][1].step()
    for step in range(2, 6):
        feed(sets[0][0], step)
        graph.replay()
        torch.cuda.synchronize()
        feed(sets[1][0], step)
        sets[1][1].step()
        for a, b in zip(sets[0][0], sets[1][0]):
            assert torch.equal(a, b), step
    assert bool((state_of(sets[0][1])["step"] == 5).all())


@pytest.mark.gpu
def test_closure_version_counters_and_schedulers() -> None:
    require_gpu_extension()
    p = torch.nn.Parameter(normal(40, seed=1))
    optimizer = fused_hoad.FusedAdamW([p], lr=1.0)
    scheduler = torch.optim.lr_scheduler.StepLR(optimizer, 1, gamma=0.5)

    def closure():
        optimizer.zero_grad()
        loss = p.square().sum()
        loss.backward()
        return loss

    before = float(p.detach().square().sum())
    assert abs(float(optimizer.step(closure)) - before) <= 1e-4 * before
    scheduler.step()
    assert optimizer.param_groups[0]["lr"] == 0.5
    held = (p * p).sum()
    optimizer.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        held.backward()


@pytest.mark.gpu
def test_large_tensor() -> None:
    """70 million values: places above 2^26, many workgroups; the last values against the plain form."""
    require_gpu_extension()
    show("adamw 70M")
    count = 70_000_001
    p = torch.nn.Parameter(torch.ones(count, device="cuda"))
    p.grad = torch.full((count,), 0.25, device="cuda")
    optimizer = fused_hoad.FusedAdamW([p], state_bits=8, seed=1, **OPTIONS)
    optimizer.step()
    optimizer.step()
    assert bool((p.detach() == p.detach()[0]).float().mean() > 0.0)
    assert bool(torch.isfinite(p).all()) and float((p.detach() - 1).abs().max()) <= 3 * OPTIONS["lr"]
    mean, square = optimizer.moments(p)
    assert abs(float(mean[-256:].double().mean()) / (0.25 * 0.19) - 1) <= 0.05
    assert abs(float(square[-256:].double().mean()) / (0.0625 * 0.0199) - 1) <= 0.1


def test_options_are_checked() -> None:
    p = [torch.nn.Parameter(torch.zeros(3))]
    for options in ({"lr": -1.0}, {"eps": -1.0}, {"weight_decay": -0.1}, {"betas": (1.0, 0.9)}, {"betas": (0.9, -0.1)},
                    {"state_bits": 16}, {"seed": -1}, {"seed": 2**32}):
        with pytest.raises(ValueError):
            fused_hoad.FusedAdamW(p, **options)
    assert fused_hoad.packed_state_size([torch.zeros(1), torch.zeros(256), torch.zeros(257), torch.zeros(0)]) == 1024
    p[0].grad = torch.zeros(3)
    with pytest.raises(RuntimeError, match="parameters must be a CUDA tensor"):
        fused_hoad.FusedAdamW(p).step()


@pytest.mark.gpu
def test_refusals() -> None:
    require_gpu_extension()
    p, g = normal(300, seed=0), normal(300, seed=1)
    m, v = torch.zeros(512, device="cuda"), torch.zeros(512, device="cuda")
    steps = torch.zeros(1, dtype=torch.int32, device="cuda")
    codes, scales = torch.zeros(512, dtype=torch.uint8, device="cuda"), torch.zeros(2, device="cuda")
    step = fused_hoad.adamw_step
    for bad, message in (
        (lambda: step([p], [], m, v, steps, lr=1e-3), "as many"),
        (lambda: step([p.half()], [g.half()], m, v, steps, lr=1e-3), "float32 or bfloat16"),
        (lambda: step([p], [g.bfloat16()], m, v, steps, lr=1e-3), "a gradient must have its parameter's dtype"),
        (lambda: step([p], [g[:299]], m, v, steps, lr=1e-3), "its parameter's shape"),
        (lambda: step([p], [g.cpu()], m, v, steps, lr=1e-3), "a gradient must be a CUDA tensor"),
        (lambda: step([p[::2]], [g[::2]], m, v, steps, lr=1e-3), "parameters must be contiguous"),
        (lambda: step([p], [g], m[:300], v, steps, lr=1e-3), "exp_avg must have 512 values"),
        (lambda: step([p], [g], m, v.bfloat16(), steps, lr=1e-3), "exp_avg_sq must be a contiguous Float"),
        (lambda: step([p], [g], m, v, steps.long(), lr=1e-3), "steps must be a contiguous Int"),
        (lambda: step([p], [g], m, v, steps, lr=-1.0), "non-negative"),
        (lambda: step([p], [g], m, v, steps, lr=1e-3, betas=(0.9, 1.0)), "betas"),
        (lambda: step([p], [g], m, v, steps, lr=1e-3, seed=-1), "seed"),
        (lambda: step([p], [g], codes, codes, steps, lr=1e-3, exp_avg_scale=scales), "scales come together"),
        (lambda: step([p], [g], m, v, steps, lr=1e-3, exp_avg_scale=scales, exp_avg_sq_scale=scales), "Byte"),
        (lambda: step([p], [g], codes, codes, steps, lr=1e-3, exp_avg_scale=scales, exp_avg_sq_scale=scales[:1]),
         "exp_avg_sq_scale must have 2 values"),
        (lambda: fused_hoad.decode_moments(codes[:300], codes, scales, scales), "multiple of 256"),
        (lambda: fused_hoad.decode_moments(codes, codes, scales, m), "exp_avg_sq_scale must have 2 values"),
    ):
        with pytest.raises(RuntimeError, match=message):
            bad()
    assert not steps.any() and not m.any()
    p0 = p.clone()
    step([p], [None], m, v, steps, lr=1e-3)
    assert torch.equal(p, p0) and not steps.any()
    step([], [], m, v, steps, lr=1e-3)


@pytest.mark.gpu
def test_forward_mode_is_refused() -> None:
    """A parameter or gradient with a tangent raises before anything is changed: the update would leave the
    parameter's tangent as it was."""
    from torch.autograd import forward_ad

    require_gpu_extension()
    show("adamw dual tensors")
    p, g = normal(300, seed=0), normal(300, seed=1)
    moments = [torch.zeros(512, device="cuda") for _ in range(2)]
    steps = torch.zeros(1, dtype=torch.int32, device="cuda")
    p0 = p.clone()
    with forward_ad.dual_level():
        for parameter, gradient in ((forward_ad.make_dual(p, g), g), (p, forward_ad.make_dual(g, p))):
            with pytest.raises(RuntimeError, match="adamw_step has no forward-mode derivative"):
                fused_hoad.adamw_step([parameter], [gradient], *moments, steps, lr=1e-3)
    assert torch.equal(p, p0) and not steps.any() and not moments[0].any()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_goes_on_from_a_loaded_state(bits) -> None:
    """A step is captured, a state of an earlier time is loaded, and the graph's replays go on from it
    bitwise as eager steps of another optimizer do that loaded the same; the optimizer's own state, loaded
    into itself, changes nothing; a state that does not fit leaves everything as it was."""
    require_gpu_extension()
    show(f"adamw load and replay {bits}")
    shapes = [(64, 33), (500,)]
    start = tensors_of(shapes, F32)

    def build():
        parameters = [torch.nn.Parameter(p.clone()) for p in start]
        for p in parameters:
            p.grad = torch.zeros_like(p)
        return parameters, fused_hoad.FusedAdamW(parameters, state_bits=bits, seed=8, **OPTIONS)

    def feed(parameters, step):
        for p, g in zip(parameters, tensors_of(shapes, F32, seed=10 * step)):
            p.grad.copy_(g)

    parameters, optimizer = build()
    feed(parameters, 1)
    optimizer.step()
    saved, then = copy.deepcopy(optimizer.state_dict()), [p.detach().clone() for p in parameters]
    held = {name: t.data_ptr() for name, t in state_of(optimizer).items() if t is not None}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        optimizer.step()
    for step in (2, 3):
        feed(parameters, step)
        graph.replay()
    torch.cuda.synchronize()
    before = copy.deepcopy(optimizer.state_dict())
    optimizer.load_state_dict(optimizer.state_dict())
    bad = copy.deepcopy(saved)
    bad["state"][1]["exp_avg"] = bad["state"][1]["exp_avg"][:-1]
    with pytest.raises(ValueError, match="does not fit"):
        optimizer.load_state_dict(bad)
    for k, entry in optimizer.state_dict()["state"].items():
        for name, value in entry.items():
            assert torch.equal(value, before["state"][k][name]), (k, name)

    def load(parameters, optimizer):
        optimizer.load_state_dict(saved)
        with torch.no_grad():
            for p, value in zip(parameters, then):
                p.copy_(value)

    load(parameters, optimizer)
    assert held == {name: t.data_ptr() for name, t in state_of(optimizer).items() if t is not None}
    others, eager = build()
    load(others, eager)
    for step in range(4, 8):
        feed(parameters, step)
        graph.replay()
        torch.cuda.synchronize()
        feed(others, step)
        eager.step()
        assert all(torch.equal(a, b) for a, b in zip(parameters, others)), step
    for p, q in zip(parameters, others):
        assert all(torch.equal(a, b) for a, b in zip(optimizer.moments(p), eager.moments(q)))
    assert bool((state_of(optimizer)["step"] == 5).all())
    # A state without entries is one of zeros, in place as well.
    optimizer.load_state_dict({**saved, "state": {}})
    assert held["exp_avg"] == state_of(optimizer)["exp_avg"].data_ptr()
    assert all(not t.any() for t in state_of(optimizer).values() if t is not None)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_state_and_parameters_changed_from_outside(bits) -> None:
    """After the state was cleared, replaced or partly taken out, after tensors were put in place of the
    views, and after a group's parameters were changed, a step equals that of a new optimizer whose state
    was loaded to be the same. What else the user keeps in the state stays there."""
    require_gpu_extension()
    show(f"adamw changed state {bits}")
    shapes = [(40, 9), (300,), (300,)]

    def build(start):
        parameters = [torch.nn.Parameter(p.detach().clone()) for p in start]
        return parameters, fused_hoad.FusedAdamW(parameters, state_bits=bits, seed=4, **OPTIONS)

    def advance(parameters, optimizer, step):
        for k, p in enumerate(parameters):
            p.grad = normal(*p.shape, seed=10 * step + k)
        optimizer.step()

    def fresh(entry):
        return {name: torch.zeros_like(value) for name, value in entry.items()}

    def clear(optimizer, parameters):
        optimizer.state.clear()
        return {}

    def replace(optimizer, parameters):
        optimizer.state = collections.defaultdict(dict)
        return {}

    def take_out(optimizer, parameters):
        del optimizer.state[parameters[1]]
        return {k: v for k, v in optimizer.state_dict()["state"].items() if k != 1}

    def put_in(optimizer, parameters):
        optimizer.state[parameters[0]] = fresh(optimizer.state[parameters[0]])
        optimizer.state[parameters[2]]["step"] = torch.tensor(7.0, device="cuda")
        return optimizer.state_dict()["state"]

    def keep(optimizer, parameters):
        optimizer.state[parameters[1]]["mine"] = torch.ones(2, device="cuda")
        return {k: {n: t for n, t in v.items() if n != "mine"} for k, v in optimizer.state_dict()["state"].items()}

    for change in (clear, replace, take_out, put_in, keep):
        parameters, optimizer = build(tensors_of(shapes, F32))
        for step in (1, 2):
            advance(parameters, optimizer, step)
        state = copy.deepcopy(change(optimizer, parameters))
        others, other = build(parameters)
        other.load_state_dict({"state": state, "param_groups": copy.deepcopy(other.state_dict()["param_groups"])})
        for step in (3, 4):
            advance(parameters, optimizer, step)
            advance(others, other, step)
            assert all(torch.equal(a, b) for a, b in zip(parameters, others)), (change.__name__, step)
        for a, b in zip(parameters, others):
            assert torch.equal(optimizer.state[a]["exp_avg"], other.state[b]["exp_avg"]), change.__name__
            assert torch.equal(optimizer.state[a]["step"], other.state[b]["step"]), change.__name__
        if change is keep:
            assert torch.equal(optimizer.state[parameters[1]]["mine"], torch.ones(2, device="cuda"))

    # The last two, of one size, change places; then a new parameter takes the first one's.
    parameters, optimizer = build(tensors_of(shapes, F32))
    advance(parameters, optimizer, 1)
    moments = [[t.clone() for t in optimizer.moments(p)] for p in parameters]
    group = optimizer.param_groups[0]
    new = torch.nn.Parameter(normal(40, 9, seed=99))
    group["params"] = [new, parameters[2], parameters[1]]
    for p in group["params"]:
        p.grad = None
    optimizer.step()
    for p, want in ((parameters[1], moments[1]), (parameters[2], moments[2])):
        assert all(torch.equal(a, b) for a, b in zip(optimizer.moments(p), want))
        assert int(optimizer.state[p]["step"]) == 1
    assert not optimizer.moments(new)[0].any() and int(optimizer.state[new]["step"]) == 0


def test_options_of_groups_and_of_loaded_states_are_checked() -> None:
    """As the constructor's: a group's own options, those of a group added later, and those of a state
    that is loaded, another optimizer's among them, which a step would not heed."""
    def parameter():
        return torch.nn.Parameter(torch.zeros(3))

    optimizer = fused_hoad.FusedAdamW([parameter()])
    for options in ({"lr": -1.0}, {"eps": -1.0}, {"weight_decay": -0.1}, {"betas": (1.0, 0.9)}, {"state_bits": 16},
                    {"seed": -1}, {"amsgrad": True}, {"maximize": True}, {"decoupled_weight_decay": False}):
        with pytest.raises(ValueError):
            fused_hoad.FusedAdamW([{"params": [parameter()], **options}])
        with pytest.raises(ValueError):
            optimizer.add_param_group({"params": [parameter()], **options})
        saved = optimizer.state_dict()
        saved["param_groups"] = [{**saved["param_groups"][0], **options}]
        with pytest.raises(ValueError):
            optimizer.load_state_dict(saved)
    assert len(optimizer.param_groups) == 1 and optimizer.param_groups[0]["lr"] == 1e-3
    with pytest.raises(ValueError, match="maximize"):
        optimizer.load_state_dict(torch.optim.AdamW([parameter()], maximize=True).state_dict())
    with pytest.raises(ValueError, match="decoupled"):
        optimizer.load_state_dict(torch.optim.Adam([parameter()], weight_decay=0.1).state_dict())
    optimizer.load_state_dict(torch.optim.AdamW([parameter()], lr=0.5).state_dict())
    assert optimizer.param_groups[0]["lr"] == 0.5 and optimizer.param_groups[0]["state_bits"] == 32
    optimizer.add_param_group({"params": [parameter()], "state_bits": 8})
    assert optimizer.param_groups[1]["state_bits"] == 8 and optimizer.param_groups[1]["betas"] == (0.9, 0.999)


@pytest.mark.gpu
def test_last_blocks_of_a_large_tensor() -> None:
    """70 million equal values and gradients, 8-bit states. After the first step, which the states' rounding
    does not reach, every parameter is the same and moved; the last blocks' codes, scales and parameters,
    the one that the tensor ends in among them, equal the elementary form's after both steps."""
    require_gpu_extension()
    show("adamw 70M, last blocks")
    count, last = 70_000_001, 4 * STATE_BLOCK
    parameter = torch.nn.Parameter(torch.ones(count, device="cuda"))
    parameter.grad = torch.full((count,), 0.25, device="cuda")
    optimizer = fused_hoad.FusedAdamW([parameter], state_bits=8, seed=1, **OPTIONS)
    end = state_span(count)
    places = torch.arange(end - last, end, device="cuda")
    inside = places < count
    beta1, beta2 = OPTIONS["betas"]
    p = torch.ones(last, device="cuda")
    g = torch.where(inside, 0.25, 0.0)
    mean, square = torch.zeros(last, device="cuda"), torch.zeros(last, device="cuda")
    for step in (1, 2):
        optimizer.step()
        size = torch.tensor(OPTIONS["lr"] / (1 - beta1**step), dtype=F32, device="cuda")
        root = torch.tensor(1 / math.sqrt(1 - beta2**step), dtype=F32, device="cuda")
        mean = mean * beta1 + g * (1 - beta1)
        square = square * beta2 + g * g * (1 - beta2)
        deviation = torch.sqrt(square)
        p = p * (1 - OPTIONS["lr"] * OPTIONS["weight_decay"]) - size * (mean / (deviation * root + OPTIONS["eps"]))
        steps = torch.full_like(places, step)
        random = mix(places ^ mix((steps + mix(torch.full_like(steps, 1))) & 0xFFFFFFFF))
        codes = encode(mean, random >> 16, 3) + encode(deviation, random & 0xFFFF, 4)
        pack = state_of(optimizer)
        for name, want in zip(("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale"), codes):
            assert torch.equal(pack[name][-want.numel():], want), (step, name)
        there = int(inside.sum())
        assert torch.equal(parameter.detach()[-there:], p[inside]), step
        if step == 1:
            assert bool((parameter.detach() == p[0]).all()) and float(p[0]) < 1.0 - 0.9 * OPTIONS["lr"]
        mean, square = decode(codes[0], codes[1], 3), decode(codes[2], codes[3], 4) ** 2


def test_hooks_of_load_state_dict_run() -> None:
    """A hook before the load may give another state, and one after it sees the loaded options."""
    def build(lr):
        return fused_hoad.FusedAdamW([torch.nn.Parameter(torch.zeros(3))], lr=lr)

    seen = []

    def before(optimizer, state_dict):
        seen.append(("before", optimizer.param_groups[0]["lr"]))
        groups = [{**group, "lr": 2 * group["lr"]} for group in state_dict["param_groups"]]
        return {**state_dict, "param_groups": groups}

    optimizer = build(0.5)
    optimizer.register_load_state_dict_pre_hook(lambda o, s: seen.append("first"))
    optimizer.register_load_state_dict_pre_hook(before)
    handle = optimizer.register_load_state_dict_post_hook(lambda o: seen.append(("after", o.param_groups[0]["lr"])))
    optimizer.load_state_dict(build(0.25).state_dict())
    assert seen == ["first", ("before", 0.5), ("after", 0.5)]
    handle.remove()
    optimizer.load_state_dict(build(1.0).state_dict())
    assert optimizer.param_groups[0]["lr"] == 2.0 and len(seen) == 5
