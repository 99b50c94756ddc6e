"""Access to the compiled MI355X extension ``fused_hoad._C``.

Mirrors /root/reference/src/fused_hoad/_extension.py:8-65. The extension is the only way into
the kernels: when it is not built, every fused entry point raises; nothing falls back to
another implementation.
"""

from __future__ import annotations

from collections.abc import Sequence
from types import ModuleType

from torch import Tensor

_BUILD_HINT = (
    "The fused_hoad HIP extension is not built. Build it for gfx950 in-tree with "
    "`python -m fused_hoad._build` (run from expanded-gpu-optimization_amd/), the equivalent "
    "of the reference's `pip install -e . --no-build-isolation`."
)


def load_extension() -> ModuleType:
    """Return the compiled extension or raise an actionable ``RuntimeError``."""
    try:
        from fused_hoad import _C
    except ImportError as exc:
        raise RuntimeError(_BUILD_HINT) from exc
    return _C


def extension_available() -> bool:
    """Whether ``fused_hoad._C`` (and the HIP library it links) can be imported."""
    try:
        load_extension()
    except RuntimeError:
        return False
    return True


def fused_forward_laplacian(
    coordinates: Tensor, parameters: Tensor, version: int = 2
) -> tuple[Tensor, Tensor]:
    """``(u, Laplacian u)``, each ``[batch, 1]``, from the gfx950 forward kernel.

    ``version`` 0..5 is accepted for compatibility with the reference's variants; every
    value runs the same kernel.
    """
    output, laplacian = load_extension().fused_forward_laplacian(coordinates, parameters, version)
    return output, laplacian


def fused_forward_laplacian_backward(
    coordinates: Tensor,
    parameters: Tensor,
    grad_output: Tensor,
    grad_laplacian: Tensor,
    version: int = 6,
) -> tuple[Tensor, Tensor]:
    """``(grad_parameters[12737], grad_coordinates[batch, 2])`` from the gfx950 backward.

    Upstream gradients may be ``[batch]`` or ``[batch, 1]``. ``version`` 1..6 is accepted for
    compatibility; every value runs the same deterministic kernels.
    """
    grad_parameters, grad_coordinates = load_extension().fused_forward_laplacian_backward(
        coordinates,
        parameters,
        grad_output.reshape(-1).contiguous(),
        grad_laplacian.reshape(-1).contiguous(),
        version,
    )
    return grad_parameters, grad_coordinates


def poisson_adam_step(
    coordinates: Tensor,
    source: Tensor,
    parameters: Tensor,
    exp_avg: Tensor,
    exp_avg_sq: Tensor,
    step: Tensor,
    *,
    lr: float,
    betas: tuple[float, float],
    eps: float,
    weight_decay: float,
    grad_parameters: Tensor | None = None,
    grad_coordinates: Tensor | None = None,
    boundary: Tensor | None = None,
    boundary_weight: float = 100.0,
) -> Tensor:
    """One fused Poisson PINN + Adam step (two gfx950 kernels); updates ``parameters``,
    ``exp_avg``, ``exp_avg_sq`` and ``step`` in place and returns the loss at entry:
    ``mean((Lap u - f)^2)`` over ``coordinates``, plus ``boundary_weight * mean(u^2)`` over
    ``boundary`` when given."""
    return load_extension().poisson_adam_step(
        coordinates,
        source,
        parameters,
        exp_avg,
        exp_avg_sq,
        step,
        float(lr),
        float(betas[0]),
        float(betas[1]),
        float(eps),
        float(weight_decay),
        grad_parameters,
        grad_coordinates,
        boundary,
        float(boundary_weight),
    )


def gated_linear(
    x: Tensor,
    gate_weight: Tensor,
    up_weight: Tensor,
    gate_bias: Tensor | None = None,
    up_bias: Tensor | None = None,
    *,
    activation: str = "silu",
) -> Tensor:
    """``activation(x gate_weight^T + gate_bias) * (x up_weight^T + up_bias)``, ``[..., hidden]``
    for ``x [..., width]`` and weights ``[hidden, width]``, all float32 or all bfloat16, with both
    projections, the activation (``"silu"``, ``"tanh"``, ``"gelu"``, ``"sigmoid"``) and the product
    in one gfx950 kernel.

    Differentiable once in every tensor, in reverse mode, with gradients that are bitwise reproducible;
    for the backward it keeps both projections in float32. float32 products are good to 2^-24 of themselves
    and 2^-126 of their operands' values; in the larger layers to 2^-21, and to 2^-51 of the largest value in
    an operand's row along the contraction. A non-finite operand makes the projections and gradients formed
    from it non-finite (NaN where float32 arithmetic could give an infinity).
    """
    return load_extension().gated_linear(x, gate_weight, up_weight, gate_bias, up_bias, activation)


def residual_norm(
    residual: Tensor,
    block: Tensor | None = None,
    gate: Tensor | None = None,
    *,
    weight: Tensor,
    bias: Tensor | None = None,
    post_weight: Tensor | None = None,
    post_bias: Tensor | None = None,
    residual_scale: float = 1.0,
    kind: str = "rms",
    eps: float = 1e-6,
) -> tuple[Tensor, Tensor]:
    """``(hidden, normed)`` between two blocks of a residual network, one gfx950 kernel::

        n = norm(block) * post_weight + post_bias      (block itself without post_weight)
        hidden = residual_scale * residual + gate * n
        normed = norm(hidden) * weight + bias

    over the last dimension (at most 16,384 wide) of ``residual`` and ``block``, float32 or
    bfloat16 with everything of one type. ``kind`` is ``"rms"`` or ``"layer"``. ``gate`` has the
    residual's first dimensions and one (or nothing) for the others before the last: ``[width]``
    for each channel, ``[samples, 1, width]`` for each of several problems, or the residual's own
    shape. Without a block, ``(residual, norm(residual) * weight + bias)``.

    Differentiable once in every tensor, in reverse mode, with gradients that are bitwise reproducible;
    sums and statistics are float32, and ``normed`` is formed from ``hidden`` before its rounding.
    """
    hidden, normed = load_extension().residual_norm(
        residual, block, gate, weight, bias, post_weight, post_bias, float(residual_scale), kind, float(eps)
    )
    return hidden, normed


def adamw_step(
    parameters: Sequence[Tensor],
    gradients: Sequence[Tensor | None],
    exp_avg: Tensor,
    exp_avg_sq: Tensor,
    steps: Tensor,
    *,
    lr: float,
    betas: tuple[float, float] = (0.9, 0.999),
    eps: float = 1e-8,
    weight_decay: float = 1e-2,
    exp_avg_scale: Tensor | None = None,
    exp_avg_sq_scale: Tensor | None = None,
    seed: int = 0,
) -> None:
    """One AdamW step (decoupled weight decay) over many tensors at once, in place: two gfx950
    kernels for every 108 tensors. Parameters are float32 or bfloat16; those whose gradient is
    ``None`` stay as they are and do not count a step.

    The moments are packed: tensor ``k``'s start at the sum of the sizes before it, each rounded
    up to 256 (``packed_state_size``). With the scales ``None`` they are float32; with scales
    (float32, one for every 256 values) they are bytes, the first moment and the second's square
    root as small floating-point numbers over the scale, rounded stochastically by bits mixed from
    ``seed``, the step and the place (``decode_moments`` gives the values). ``steps`` is int32, one
    for each tensor, counted on the device, so a step can be captured in a HIP graph.
    """
    load_extension().adamw_step(
        list(parameters),
        list(gradients),
        exp_avg,
        exp_avg_sq,
        steps,
        float(lr),
        float(betas[0]),
        float(betas[1]),
        float(eps),
        float(weight_decay),
        exp_avg_scale,
        exp_avg_sq_scale,
        int(seed),
    )


def decode_moments(
    exp_avg: Tensor, exp_avg_sq: Tensor, exp_avg_scale: Tensor, exp_avg_sq_scale: Tensor
) -> tuple[Tensor, Tensor]:
    """The first and second moments, float32, that packed 8-bit states stand for."""
    mean, square = load_extension().decode_moments(exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale)
    return mean, square
