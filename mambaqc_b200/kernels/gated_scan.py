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

from .. import _lib
from .block_fused import _rows

__all__ = ["gated_linear_scan", "gated_linear_step"]


def _f32(t: torch.Tensor | None) -> torch.Tensor | None:
    """Contiguous fp32 (the tensor itself where it is that already)."""
    return None if t is None else t.detach().to(torch.float32).contiguous()


def _forward(x, r, i, lam, h0, reset, sharpness, want_state, keep):
    """(y, hT, saved): ``keep`` leaves the states that the backward pass starts from."""
    bsz, seqlen, dm = x.shape
    xs, x_row = _rows(x)
    rs, r_row = _rows(r)
    si, i_row = _rows(i)
    dev = x.device
    y = torch.empty(bsz, seqlen, dm, dtype=x.dtype, device=dev)
    hT = torch.empty(bsz, dm, dtype=torch.float32, device=dev) if want_state else None
    ckpt = None
    if keep:
        tiles = -(-seqlen // _lib.MQC_GATED_SCAN_TILE)
        ckpt = torch.empty(bsz, tiles, dm, dtype=torch.float32, device=dev)
    a = _lib.GatedScanArgs()
    a.batch, a.seq_len, a.channels = bsz, seqlen, dm
    a.dtype, a.sharpness = _lib.dtype_code(x), sharpness
    a.x, a.r, a.i = xs.data_ptr(), rs.data_ptr(), si.data_ptr()
    a.x_row, a.r_row, a.i_row = max(x_row, dm), max(r_row, dm), max(i_row, dm)
    a.lambda_, a.h0, a.reset = lam.data_ptr(), _lib.ptr(h0), _lib.ptr(reset)
    a.y, a.hT, a.ckpt = y.data_ptr(), _lib.ptr(hT), _lib.ptr(ckpt)
    a.status = _lib.status_word(dev).data_ptr()
    _lib.call_on(dev, "mqc_gated_scan_fwd", ctypes.byref(a))
    return y, hT, (xs, rs, si, ckpt)


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, r, i, Lambda, h0, reset, sharpness, want_state):
        lam = _f32(Lambda)
        y, hT, (xs, rs, si, ckpt) = _forward(x, r, i, lam, _f32(h0), reset, sharpness, want_state,
                                             True)
        ctx.save_for_backward(xs, rs, si, lam, reset, ckpt)
        ctx.sharpness = sharpness
        ctx.meta = (Lambda.dtype, None if h0 is None else h0.dtype)
        ctx.set_materialize_grads(False)
        return y, hT

    @staticmethod
    def backward(ctx, dy, dhT):
        xs, rs, si, lam, reset, ckpt = ctx.saved_tensors
        bsz, seqlen, dm = xs.shape
        lam_dtype, h0_dtype = ctx.meta
        dev = xs.device
        x_row, r_row, i_row = (_rows(t)[1] for t in (xs, rs, si))
        dys, dy_row = (None, 0) if dy is None else _rows(dy.to(xs.dtype))
        dhT = _f32(dhT)
        dx, dr, di = (torch.empty(bsz, seqlen, dm, dtype=xs.dtype, device=dev) for _ in range(3))
        dlam = torch.empty(dm, dtype=torch.float32, device=dev)
        dh0 = None
        if h0_dtype is not None and ctx.needs_input_grad[4]:
            dh0 = torch.empty(bsz, dm, dtype=torch.float32, device=dev)
        nbytes = _lib.load().mqc_gated_scan_bwd_workspace_size(bsz, seqlen, dm)
        ws = torch.empty(max(1, nbytes // 4), dtype=torch.float32, device=dev)
        a = _lib.GatedScanArgs()
        a.batch, a.seq_len, a.channels = bsz, seqlen, dm
        a.dtype, a.sharpness = _lib.dtype_code(xs), ctx.sharpness
        a.x, a.r, a.i = xs.data_ptr(), rs.data_ptr(), si.data_ptr()
        a.x_row, a.r_row, a.i_row = max(x_row, dm), max(r_row, dm), max(i_row, dm)
        a.lambda_, a.reset, a.ckpt = lam.data_ptr(), _lib.ptr(reset), ckpt.data_ptr()
        a.dy, a.dy_row, a.dhT = _lib.ptr(dys), max(dy_row, dm), _lib.ptr(dhT)
        a.dx, a.dr, a.di = dx.data_ptr(), dr.data_ptr(), di.data_ptr()
        a.dlambda, a.dh0 = dlam.data_ptr(), _lib.ptr(dh0)
        a.status = _lib.status_word(dev).data_ptr()
        _lib.call_on(dev, "mqc_gated_scan_bwd", ctypes.byref(a), ws.data_ptr(), nbytes)
        return (dx, dr, di, dlam.to(lam_dtype), None if dh0 is None else dh0.to(h0_dtype),
                None, None, None)


def _check(what, x, r, i, Lambda, h):
    assert r.shape == x.shape and i.shape == x.shape, f"{what}: x, r and i must have one shape"
    assert r.dtype == x.dtype and i.dtype == x.dtype, f"{what}: x, r and i must have one dtype"
    assert tuple(Lambda.shape) == (x.shape[-1],), f"{what}: Lambda must be [D]"
    assert h is None or tuple(h.shape) == (x.shape[0], x.shape[-1]), f"{what}: state must be [B, D]"
    _lib.dtype_code(x)
    _lib.require_cuda(x, r, i, Lambda, h, what=what)
    for t in (r, i, Lambda, h):
        assert t is None or t.device == x.device, f"{what}: tensors on different devices"


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
    if torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (x, r, i, Lambda, h0)):
        y, hT = _GatedScan.apply(x, r, i, Lambda, h0, reset, float(sharpness),
                                 return_final_state)
    else:
        y, hT, _ = _forward(x, r, i, _f32(Lambda), _f32(h0), reset, float(sharpness),
                            return_final_state, False)
    return (y, hT) if return_final_state else y


@torch.no_grad()
def gated_linear_step(x: torch.Tensor, r: torch.Tensor, i: torch.Tensor, Lambda: torch.Tensor,
                      h: torch.Tensor, *, sharpness: float = 8.0,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """One token of B sequences: x, r, i [B, D]; the state h [B, D] fp32 is advanced
    in place. Returns y [B, D] in x's dtype (``out`` if given). No gradient."""
    assert x.dim() == 2, f"x must be [B, D], got {tuple(x.shape)}"
    _check("gated_linear_step", x, r, i, Lambda, h)
    assert sharpness > 0, "sharpness must be positive"
    assert h is not None and h.dtype == torch.float32 and h.is_contiguous(), \
        "h must be a contiguous float32 [B, D] state"
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    else:
        assert out.shape == x.shape and out.dtype == x.dtype and out.is_contiguous() and \
            out.device == x.device, "out must be a contiguous tensor like x"
    bsz, dm = x.shape
    x, x_row = _rows(x)
    r, r_row = _rows(r)
    i, i_row = _rows(i)
    _lib.call_on(x.device, "mqc_gated_scan_step", x.data_ptr(), max(x_row, dm), r.data_ptr(),
                 max(r_row, dm), i.data_ptr(), max(i_row, dm), _f32(Lambda).data_ptr(),
                 h.data_ptr(), out.data_ptr(), bsz, dm, float(sharpness), _lib.dtype_code(x))
    return out
