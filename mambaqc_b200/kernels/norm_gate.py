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

import ctypes

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from .block_fused import _rows

__all__ = ["norm_gate_residual", "residual_norm"]

_KINDS = {"layer": _lib.MQC_NORM_LAYER, "rms": _lib.MQC_NORM_RMS}


_F32 = torch.float32
_CODES = {torch.float32: _lib.MQC_DTYPE_F32, torch.bfloat16: _lib.MQC_DTYPE_BF16}


def _param(t: torch.Tensor | None) -> torch.Tensor | None:
    """Contiguous fp32 (the tensor itself where it is that already)."""
    if t is None or (t.dtype is _F32 and t.is_contiguous()):
        return t
    return t.detach().to(_F32).contiguous()


def _forward(x, y, z, params, kind, eps, out_dtype, keep):
    """(out, n, x, y, z, z_row, stats); out is None without y, n without a next weight."""
    width = x.shape[-1]
    rows = x.numel() // width if width else 0
    x = x.contiguous()
    weight, bias, scale, next_weight, next_bias = params
    out = n = stats = None
    z_row = width
    if y is not None:
        y = y.contiguous()
        if not z.is_contiguous():
            z, z_row = _rows(z)
            z_row = max(z_row, width)
        out = torch.empty_like(x)
    if next_weight is not None:
        n = torch.empty_like(x, dtype=out_dtype)
    if keep:
        stats = torch.empty((rows, 4), dtype=_F32, device=x.device)
    ptr = _lib.ptr
    a = _lib.NormGateArgs(rows, width, z_row, _CODES[x.dtype], _CODES[out_dtype], kind, eps,
                          x.data_ptr(), ptr(y), ptr(z), ptr(weight), ptr(bias), ptr(scale),
                          ptr(next_weight), ptr(next_bias), ptr(out), ptr(n), ptr(stats))
    _lib.call_on(x.get_device(), "mqc_norm_gate_fwd", ctypes.byref(a))
    return out, n, x, y, z, z_row, stats


class _NormGate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, z, weight, bias, scale, next_weight, next_bias, kind, eps, out_dtype):
        raw = (weight, bias, scale, next_weight, next_bias)
        params = tuple(map(_param, raw))
        out, n, x, y, z, z_row, stats = _forward(x, y, z, params, kind, eps, out_dtype, True)
        ctx.save_for_backward(x, y, z, stats, *params)
        ctx.meta = (kind, eps, out_dtype, z_row,
                    tuple(None if t is None else t.dtype for t in raw))
        ctx.set_materialize_grads(False)
        return out, n

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dn):
        x, y, z, stats, *params = ctx.saved_tensors
        kind, eps, out_dtype, z_row, dtypes = ctx.meta
        width = x.shape[-1]
        rows = stats.shape[0]
        dev = x.device
        if dout is not None:
            dout = (dout if dout.dtype is x.dtype else dout.to(x.dtype)).contiguous()
        if dn is not None:
            dn = (dn if dn.dtype is out_dtype else dn.to(out_dtype)).contiguous()
        dx = torch.empty_like(x)
        dy = dz = None
        if y is not None:
            dy, dz = torch.empty_like(y), torch.empty_like(y)
        # needs_input_grad of weight, bias, scale, next_weight, next_bias
        sums = [torch.empty_like(t) if t is not None and w else None
                for t, w in zip(params, ctx.needs_input_grad[3:8])]
        nbytes = _lib.load().mqc_norm_gate_bwd_workspace_size(rows, width)
        ws = torch.empty(max(1, nbytes // 4), dtype=_F32, device=dev)
        ptr = _lib.ptr
        weight, bias, scale, next_weight, next_bias = map(ptr, params)
        dweight, dbias, dscale, dnext_weight, dnext_bias = map(ptr, sums)
        a = _lib.NormGateArgs(rows, width, z_row, _CODES[x.dtype], _CODES[out_dtype], kind, eps,
                              x.data_ptr(), ptr(y), ptr(z), weight, bias, scale, next_weight,
                              next_bias, None, None, stats.data_ptr(), ptr(dout), ptr(dn),
                              dx.data_ptr(), ptr(dy), ptr(dz), dweight, dscale, dbias,
                              dnext_weight, dnext_bias)
        _lib.call_on(dev.index, "mqc_norm_gate_bwd", ctypes.byref(a), ws.data_ptr(), nbytes)
        sums = [t if t is None or d is _F32 else t.to(d) for t, d in zip(sums, dtypes)]
        return (dx, dy, dz, *sums, None, None, None)


def _run(x, y, z, weight, bias, scale, next_weight, next_bias, norm, eps, out_dtype):
    if torch.is_grad_enabled():
        for t in (x, y, z, weight, bias, scale, next_weight, next_bias):
            if t is not None and t.requires_grad:
                return _NormGate.apply(x, y, z, weight, bias, scale, next_weight, next_bias,
                                       _KINDS[norm], eps, out_dtype)
    params = tuple(map(_param, (weight, bias, scale, next_weight, next_bias)))
    return _forward(x, y, z, params, _KINDS[norm], eps, out_dtype, False)[:2]


def _fits(x, tensors, vectors, norm, eps) -> bool:
    """Whether ``_check`` would pass, without building its messages."""
    shape, dev = x.shape, x.get_device()
    if dev < 0 or norm not in _KINDS or not eps >= 0 or not shape or \
            x.dtype not in _CODES or shape[-1] > _lib.MQC_NORM_GATE_MAX_WIDTH:
        return False
    width = shape[-1]
    for t in tensors:
        if t.shape != shape or t.dtype not in _CODES or t.get_device() != dev:
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
        if t.dtype not in _CODES:
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
    n is Q of out before it is rounded. Differentiable in every tensor."""
    if not _fits(x, (y, z), (weight, scale, bias, next_weight, next_bias), norm, eps):
        _check("norm_gate_residual", x, (("x", x), ("y", y), ("z", z)),
               (("weight", weight), ("scale", scale), ("bias", bias),
                ("next_weight", next_weight), ("next_bias", next_bias)), norm, eps)
    assert next_bias is None or next_weight is not None, "next_bias needs next_weight"
    if x.dtype == torch.bfloat16 and y.dtype == torch.float32:
        x = x.float()
    if z.dtype != y.dtype:
        z = z.to(y.dtype)
    out, n = _run(x, y, z, weight, bias, scale, next_weight, next_bias, norm, float(eps), y.dtype)
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
    return _run(x, None, None, None, None, None, weight, bias, norm, float(eps), dtype)[1]
