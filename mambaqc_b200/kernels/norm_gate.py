"""The norms after and before a block, fused with its output gate and residual.

    out = x + scale * sigmoid(z) * P(y)        n = Q(out)

P normalises the block's output, ``scale`` [D] weighs what it adds to the residual
stream x, and Q is the norm in front of the next block; P and Q are both LayerNorm
or both RMSNorm, each with its own weight and bias. The reference block adds
``sigmoid(z) * y`` with no norm on either side
(mambaqc/models/quaternion_mamba2_block.py:154-164; ``gate_residual`` here); deep
stacks of blocks want both. The kernels are in ``csrc/norm_gate.cu``.
"""

from __future__ import annotations

import torch

from .. import _lib

__all__ = ["norm_gate_residual", "residual_norm"]

_KINDS = {"layer": _lib.MQC_NORM_LAYER, "rms": _lib.MQC_NORM_RMS}
_TYPES = (torch.float32, torch.bfloat16)


def _fits(x, tensors, vectors, norm, eps) -> bool:
    """Whether ``_check`` would pass, without building its messages."""
    shape, dev = x.shape, x.get_device()
    if dev < 0 or norm not in _KINDS or not eps >= 0 or not shape or \
            x.dtype not in _TYPES or shape[-1] > _lib.MQC_NORM_GATE_MAX_WIDTH:
        return False
    width = shape[-1]
    for t in tensors:
        if t.shape != shape or t.dtype not in _TYPES or t.get_device() != dev:
            return False
    for t in vectors:
        if t is not None and (t.dim() != 1 or t.numel() != width or t.get_device() != dev):
            return False
    return True


def _check(what, x, tensors, vectors, norm, eps):
    assert norm in _KINDS, f"{what}: norm must be 'layer' or 'rms', got {norm!r}"
    assert eps >= 0, f"{what}: eps must not be negative"
    assert x.dim() >= 1, f"{what}: x must have at least one dimension"
    shape, dev = x.shape, x.get_device()
    width = shape[-1]
    assert width <= _lib.MQC_NORM_GATE_MAX_WIDTH, \
        f"{what}: width {width} (at most {_lib.MQC_NORM_GATE_MAX_WIDTH})"
    for name, t in tensors:
        assert t.shape == shape, f"{what}: {name} must have x's shape"
        if t.dtype not in _TYPES:
            _lib.dtype_code(t)
        assert t.get_device() == dev, f"{what}: tensors on different devices"
    for name, t in vectors:
        if t is not None:
            assert t.dim() == 1 and t.numel() == width, f"{what}: {name} must be [{width}]"
            assert t.get_device() == dev, f"{what}: tensors on different devices"
    if dev < 0:
        _lib.require_cuda(x, what=what)


def norm_gate_residual(x: torch.Tensor, y: torch.Tensor, z: torch.Tensor, weight: torch.Tensor,
                       scale: torch.Tensor, bias: torch.Tensor | None = None,
                       next_weight: torch.Tensor | None = None,
                       next_bias: torch.Tensor | None = None, *, norm: str = "rms",
                       eps: float = 1e-5):
    """out = x + scale * sigmoid(z) * P(y), and with ``next_weight`` also n = Q(out).

    x, y, z [..., D], D <= 4096: the residual stream, the block's output and its gate
    (a column slice of a wider tensor is read in place); weight, scale, bias,
    next_weight, next_bias [D]. x may be fp32 with bf16 y and z; an fp32 y takes a
    bf16 x to fp32. out is in x's dtype, n in y's. Computed in fp32 and rounded once:
    n is Q of out before it is rounded. Differentiable in every tensor (once)."""
    if not _fits(x, (y, z), (weight, scale, bias, next_weight, next_bias), norm, eps):
        _check("norm_gate_residual", x, (("x", x), ("y", y), ("z", z)),
               (("weight", weight), ("scale", scale), ("bias", bias),
                ("next_weight", next_weight), ("next_bias", next_bias)), norm, eps)
    assert next_bias is None or next_weight is not None, "next_bias needs next_weight"
    if x.dtype == torch.bfloat16 and y.dtype == torch.float32:
        x = x.float()
    if z.dtype != y.dtype:
        z = z.to(y.dtype)
    out, n = _lib.torch_ops().norm_gate(x, y, z, weight, bias, scale, next_weight, next_bias,
                                        _KINDS[norm], float(eps), y.dtype is torch.float32)
    return out if next_weight is None else (out, n)


def residual_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                  norm: str = "rms", eps: float = 1e-5,
                  dtype: torch.dtype | None = None) -> torch.Tensor:
    """Q(x) alone, the norm in front of the first block: x [..., D], D <= 4096, weight
    and bias [D]. Returned in ``dtype`` (x's if None; bf16 from an fp32 x for a block
    that computes in bf16). Differentiable."""
    assert weight is not None, "residual_norm needs a weight"
    if not _fits(x, (), (weight, bias), norm, eps):
        _check("residual_norm", x, (("x", x),), (("weight", weight), ("bias", bias)), norm, eps)
    dtype = x.dtype if dtype is None else dtype
    assert dtype in (torch.float32, torch.bfloat16), "dtype must be float32 or bfloat16"
    if x.dtype == torch.bfloat16 and dtype == torch.float32:
        x = x.float()
    return _lib.torch_ops().norm_gate(x, None, None, None, None, None, weight, bias,
                                      _KINDS[norm], float(eps), dtype is torch.float32)[1]
