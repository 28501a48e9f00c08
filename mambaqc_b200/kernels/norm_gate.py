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

from .. import _lib
from .block_fused import _rows

__all__ = ["norm_gate_residual", "residual_norm"]

_KINDS = {"layer": _lib.MQC_NORM_LAYER, "rms": _lib.MQC_NORM_RMS}


def _param(t: torch.Tensor | None) -> torch.Tensor | None:
    return None if t is None else t.detach().to(torch.float32).contiguous()


def _forward(x, y, z, params, kind, eps, out_dtype, keep):
    """(out, n, x, y, z, z_row, stats); out is None without y, n without a next weight."""
    width = x.shape[-1]
    rows = x.numel() // width if width else 0
    xc = x.contiguous()
    dev = x.device
    weight, bias, scale, next_weight, next_bias = params
    yc = zs = out = n = stats = None
    z_row = width
    if y is not None:
        yc = y.contiguous()
        zs, z_row = _rows(z)
        out = torch.empty(x.shape, dtype=x.dtype, device=dev)
    if next_weight is not None:
        n = torch.empty(x.shape, dtype=out_dtype, device=dev)
    if keep:
        stats = torch.empty(rows, 4, dtype=torch.float32, device=dev)
    a = _lib.NormGateArgs()
    a.rows, a.width, a.z_row = rows, width, max(z_row, width)
    a.x_dtype = _lib.dtype_code(xc)
    a.y_dtype = _lib.MQC_DTYPE_F32 if out_dtype == torch.float32 else _lib.MQC_DTYPE_BF16
    a.norm, a.eps = kind, eps
    a.x, a.y, a.z = xc.data_ptr(), _lib.ptr(yc), _lib.ptr(zs)
    a.weight, a.bias, a.scale = _lib.ptr(weight), _lib.ptr(bias), _lib.ptr(scale)
    a.next_weight, a.next_bias = _lib.ptr(next_weight), _lib.ptr(next_bias)
    a.out, a.n, a.stats = _lib.ptr(out), _lib.ptr(n), _lib.ptr(stats)
    _lib.call_on(dev, "mqc_norm_gate_fwd", ctypes.byref(a))
    return out, n, xc, yc, zs, z_row, stats


class _NormGate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, z, weight, bias, scale, next_weight, next_bias, kind, eps, out_dtype):
        raw = (weight, bias, scale, next_weight, next_bias)
        params = tuple(_param(t) for t in raw)
        out, n, xc, yc, zs, z_row, stats = _forward(x, y, z, params, kind, eps, out_dtype, True)
        ctx.save_for_backward(xc, yc, zs, stats, *params)
        ctx.meta = (kind, eps, out_dtype, z_row,
                    tuple(None if t is None else t.dtype for t in raw))
        ctx.set_materialize_grads(False)
        return out, n

    @staticmethod
    def backward(ctx, dout, dn):
        xc, yc, zs, stats, weight, bias, scale, next_weight, next_bias = ctx.saved_tensors
        kind, eps, out_dtype, z_row, dtypes = ctx.meta
        width = xc.shape[-1]
        rows = xc.numel() // width if width else 0
        dev = xc.device
        dout = None if dout is None else dout.to(xc.dtype).contiguous()
        dn = None if dn is None else dn.to(out_dtype).contiguous()
        dx = torch.empty(xc.shape, dtype=xc.dtype, device=dev)
        dy = dz = None
        if yc is not None:
            dy = torch.empty(xc.shape, dtype=out_dtype, device=dev)
            dz = torch.empty(xc.shape, dtype=out_dtype, device=dev)
        # needs_input_grad of weight, bias, scale, next_weight, next_bias
        want = ctx.needs_input_grad[3:8]
        sums = [torch.empty(width, dtype=torch.float32, device=dev)
                if t is not None and w else None
                for t, w in zip((weight, bias, scale, next_weight, next_bias), want)]
        nbytes = _lib.load().mqc_norm_gate_bwd_workspace_size(rows, width)
        ws = torch.empty(max(1, nbytes // 4), dtype=torch.float32, device=dev)
        a = _lib.NormGateArgs()
        a.rows, a.width, a.z_row = rows, width, max(z_row, width)
        a.x_dtype = _lib.dtype_code(xc)
        a.y_dtype = _lib.MQC_DTYPE_F32 if out_dtype == torch.float32 else _lib.MQC_DTYPE_BF16
        a.norm, a.eps = kind, eps
        a.x, a.y, a.z = xc.data_ptr(), _lib.ptr(yc), _lib.ptr(zs)
        a.weight, a.bias, a.scale = _lib.ptr(weight), _lib.ptr(bias), _lib.ptr(scale)
        a.next_weight, a.next_bias = _lib.ptr(next_weight), _lib.ptr(next_bias)
        a.stats, a.dout, a.dn = stats.data_ptr(), _lib.ptr(dout), _lib.ptr(dn)
        a.dx, a.dy, a.dz = dx.data_ptr(), _lib.ptr(dy), _lib.ptr(dz)
        a.dweight, a.dbias, a.dscale, a.dnext_weight, a.dnext_bias = map(_lib.ptr, sums)
        _lib.call_on(dev, "mqc_norm_gate_bwd", ctypes.byref(a), ws.data_ptr(), nbytes)
        sums = [None if t is None else t.to(d) for t, d in zip(sums, dtypes)]
        return (dx, dy, dz, *sums, None, None, None)


def _run(x, y, z, weight, bias, scale, next_weight, next_bias, norm, eps, out_dtype):
    if torch.is_grad_enabled() and any(
            t is not None and t.requires_grad
            for t in (x, y, z, weight, bias, scale, next_weight, next_bias)):
        return _NormGate.apply(x, y, z, weight, bias, scale, next_weight, next_bias,
                               _KINDS[norm], eps, out_dtype)
    params = tuple(_param(t) for t in (weight, bias, scale, next_weight, next_bias))
    return _forward(x, y, z, params, _KINDS[norm], eps, out_dtype, False)[:2]


def _check(what, x, tensors, vectors, norm, eps):
    assert norm in _KINDS, f"{what}: norm must be 'layer' or 'rms', got {norm!r}"
    assert eps >= 0, f"{what}: eps must not be negative"
    width = x.shape[-1]
    assert width <= _lib.MQC_NORM_GATE_MAX_WIDTH, \
        f"{what}: width {width} (at most {_lib.MQC_NORM_GATE_MAX_WIDTH})"
    _lib.dtype_code(x)
    for name, t in tensors.items():
        assert t.shape == x.shape, f"{what}: {name} must have x's shape"
        _lib.dtype_code(t)
    for name, t in vectors.items():
        assert t is None or tuple(t.shape) == (width,), f"{what}: {name} must be [{width}]"
    for t in (*tensors.values(), *vectors.values()):
        assert t is None or t.device == x.device, f"{what}: tensors on different devices"
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
    assert x.dim() >= 1, "x must have at least one dimension"
    _check("norm_gate_residual", x, {"y": y, "z": z},
           {"weight": weight, "scale": scale, "bias": bias, "next_weight": next_weight,
            "next_bias": next_bias}, norm, eps)
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
    assert x.dim() >= 1, "x must have at least one dimension"
    _check("residual_norm", x, {}, {"weight": weight, "bias": bias}, norm, eps)
    assert weight is not None, "residual_norm needs a weight"
    dtype = x.dtype if dtype is None else dtype
    assert dtype in (torch.float32, torch.bfloat16), "dtype must be float32 or bfloat16"
    if x.dtype == torch.bfloat16 and dtype == torch.float32:
        x = x.float()
    return _run(x, None, None, None, None, None, weight, bias, norm, float(eps), dtype)[1]
