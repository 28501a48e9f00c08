"""Gated linear recurrence: a real-valued sequence mixer next to the quaternion scan.

With s = sigmoid and, per channel, a rate ``sharpness * softplus(Lambda)``:

    a[t] = exp(-sharpness softplus(Lambda) s(r[t]))
    h[t] = a[t] h[t-1] + sqrt(1 - a[t]^2) s(i[t]) x[t]          y = h

``gated_linear_scan`` runs a whole sequence and is differentiable;
``gated_linear_step`` advances the state of a batch by one token. The kernels
are in ``csrc/gated_scan.cu``. The reference has no real-valued recurrence: its
block mixes time with the quaternion scan alone
(mambaqc/models/quaternion_mamba2_block.py:166-230).
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from .block_fused import _rows

__all__ = ["gated_linear_scan", "gated_linear_step"]

_F32 = torch.float32
_CODES = {torch.float32: _lib.MQC_DTYPE_F32, torch.bfloat16: _lib.MQC_DTYPE_BF16}


def _f32(t: torch.Tensor | None) -> torch.Tensor | None:
    """Contiguous fp32 (the tensor itself where it is that already)."""
    if t is None or (t.dtype is _F32 and t.is_contiguous()):
        return t
    return t.detach().to(_F32).contiguous()


def _placed(t: torch.Tensor, dm: int):
    """(tensor, row stride) of a tensor whose rows the kernel can read in place."""
    if t.is_contiguous():
        return t, dm
    t, row = _rows(t)
    return t, max(row, dm)


def _like(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _forward(x, r, i, lam, h0, reset, sharpness, want_state, keep):
    """(y, hT, saved): ``keep`` leaves the states that the backward pass starts from."""
    bsz, seqlen, dm = x.shape
    xs, x_row = _placed(x, dm)
    rs, r_row = _placed(r, dm)
    si, i_row = _placed(i, dm)
    dev = x.device
    y = _like(x)
    hT = ckpt = None
    if want_state:
        hT = torch.empty((bsz, dm), dtype=_F32, device=dev)
    if keep:
        tiles = -(-seqlen // _lib.MQC_GATED_SCAN_TILE)
        ckpt = torch.empty((bsz, tiles, dm), dtype=_F32, device=dev)
    ptr = _lib.ptr
    a = _lib.GatedScanArgs(bsz, seqlen, dm, _CODES[x.dtype], sharpness, xs.data_ptr(),
                           rs.data_ptr(), si.data_ptr(), x_row, r_row, i_row, lam.data_ptr(),
                           ptr(h0), ptr(reset), y.data_ptr(), ptr(hT), ptr(ckpt))
    a.status = _lib.status_ptr(dev.index)
    _lib.call_on(dev.index, "mqc_gated_scan_fwd", ctypes.byref(a))
    return y, hT, (xs, rs, si, ckpt)


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, r, i, Lambda, h0, reset, sharpness, want_state):
        lam = _f32(Lambda)
        y, hT, (xs, rs, si, ckpt) = _forward(x, r, i, lam, _f32(h0), reset, sharpness, want_state,
                                             True)
        ctx.save_for_backward(xs, rs, si, lam, reset, ckpt)
        ctx.meta = (sharpness, Lambda.dtype, None if h0 is None else h0.dtype)
        ctx.set_materialize_grads(False)
        return y, hT

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dhT):
        xs, rs, si, lam, reset, ckpt = ctx.saved_tensors
        bsz, seqlen, dm = xs.shape
        sharpness, lam_dtype, h0_dtype = ctx.meta
        dev = xs.device
        dy_row = dm
        if dy is not None:
            dy, dy_row = _placed(dy if dy.dtype is xs.dtype else dy.to(xs.dtype), dm)
        dhT = _f32(dhT)
        dx, dr, di = _like(xs), _like(xs), _like(xs)
        nbytes = _lib.load().mqc_gated_scan_bwd_workspace_size(bsz, seqlen, dm)
        ws = torch.empty(max(1, nbytes // 4), dtype=_F32, device=dev)
        dlam = torch.empty_like(lam)
        dh0 = None
        if h0_dtype is not None and ctx.needs_input_grad[4]:
            dh0 = torch.empty((bsz, dm), dtype=_F32, device=dev)
        ptr = _lib.ptr
        a = _lib.GatedScanArgs(bsz, seqlen, dm, _CODES[xs.dtype], sharpness, xs.data_ptr(),
                               rs.data_ptr(), si.data_ptr(), _placed(xs, dm)[1],
                               _placed(rs, dm)[1], _placed(si, dm)[1], lam.data_ptr(), None,
                               ptr(reset), None, None, ckpt.data_ptr(), ptr(dy), ptr(dhT), dy_row,
                               dx.data_ptr(), dr.data_ptr(), di.data_ptr(), dlam.data_ptr(),
                               ptr(dh0), _lib.status_ptr(dev.index))
        _lib.call_on(dev.index, "mqc_gated_scan_bwd", ctypes.byref(a), ws.data_ptr(), nbytes)
        if lam_dtype is not _F32:
            dlam = dlam.to(lam_dtype)
        if dh0 is not None and h0_dtype is not _F32:
            dh0 = dh0.to(h0_dtype)
        return dx, dr, di, dlam, dh0, None, None, None


def _check(what, x, r, i, Lambda, h):
    shape, dtype, dev = x.shape, x.dtype, x.get_device()
    assert r.shape == shape and i.shape == shape, f"{what}: x, r and i must have one shape"
    assert r.dtype is dtype and i.dtype is dtype, f"{what}: x, r and i must have one dtype"
    assert Lambda.dim() == 1 and Lambda.numel() == shape[-1], f"{what}: Lambda must be [D]"
    assert h is None or (h.dim() == 2 and h.shape[0] == shape[0] and h.shape[1] == shape[-1]), \
        f"{what}: state must be [B, D]"
    if dtype not in _CODES:
        _lib.dtype_code(x)
    if dev < 0:
        _lib.require_cuda(x, what=what)
    assert r.get_device() == dev and i.get_device() == dev and Lambda.get_device() == dev and \
        (h is None or h.get_device() == dev), f"{what}: tensors on different devices"


def gated_linear_scan(x: torch.Tensor, r: torch.Tensor, i: torch.Tensor, Lambda: torch.Tensor,
                      h0: torch.Tensor | None = None, reset: torch.Tensor | None = None, *,
                      sharpness: float = 8.0, return_final_state: bool = False):
    """The recurrence over x, r, i [B, T, D] (fp32 or bf16, one dtype; the recurrence
    and input gates r and i before their sigmoid; column slices of wider tensors are
    read in place), Lambda [D], start state h0 [B, D] (zero if None).

    ``reset`` [B, T] bool marks steps that drop the state (the first token of each
    document of a packed sequence): there h = s(i) x. Returns y [B, T, D] in x's
    dtype, and with ``return_final_state`` also h_T [B, D] fp32. The state is fp32
    throughout. Differentiable in x, r, i, Lambda, h0, from y and h_T; the backward
    pass recomputes the states from fp32 ones kept every 64 steps."""
    assert x.dim() == 3, f"x must be [B, T, D], got {tuple(x.shape)}"
    _check("gated_linear_scan", x, r, i, Lambda, h0)
    assert sharpness > 0, "sharpness must be positive"
    if reset is not None:
        assert reset.dtype == torch.bool and reset.shape == x.shape[:2], \
            "reset must be bool [B, T]"
        assert reset.device == x.device, "gated_linear_scan: tensors on different devices"
        reset = reset.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or r.requires_grad or i.requires_grad or
                                    Lambda.requires_grad or
                                    (h0 is not None and h0.requires_grad)):
        y, hT = _GatedScan.apply(x, r, i, Lambda, h0, reset, float(sharpness),
                                 return_final_state)
    else:
        y, hT, _ = _forward(x, r, i, _f32(Lambda), _f32(h0), reset, float(sharpness),
                            return_final_state, False)
    return (y, hT) if return_final_state else y


def gated_linear_step(x: torch.Tensor, r: torch.Tensor, i: torch.Tensor, Lambda: torch.Tensor,
                      h: torch.Tensor, *, sharpness: float = 8.0,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """One token of B sequences: x, r, i [B, D]; the state h [B, D] fp32 is advanced
    in place. Returns y [B, D] in x's dtype (``out`` if given). Has no gradient: what
    requires one is read as it stands."""
    assert x.dim() == 2, f"x must be [B, D], got {tuple(x.shape)}"
    _check("gated_linear_step", x, r, i, Lambda, h)
    assert sharpness > 0, "sharpness must be positive"
    assert h is not None and h.dtype == torch.float32 and h.is_contiguous(), \
        "h must be a contiguous float32 [B, D] state"
    if out is None:
        out = _like(x.detach() if x.requires_grad else x)
    else:
        assert out.shape == x.shape and out.dtype == x.dtype and out.is_contiguous() and \
            out.device == x.device, "out must be a contiguous tensor like x"
    bsz, dm = x.shape
    x, x_row = _placed(x, dm)
    r, r_row = _placed(r, dm)
    i, i_row = _placed(i, dm)
    _lib.call_on(x.get_device(), "mqc_gated_scan_step", x.data_ptr(), x_row, r.data_ptr(), r_row,
                 i.data_ptr(), i_row, _f32(Lambda).data_ptr(), h.data_ptr(), out.data_ptr(), bsz,
                 dm, float(sharpness), _CODES[x.dtype])
    return out
