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

import torch

from .. import _lib

__all__ = ["gated_linear_scan", "gated_linear_step"]

_TYPES = (torch.float32, torch.bfloat16)


def _check(what, x, r, i, Lambda, h):
    shape, dtype, dev = x.shape, x.dtype, x.get_device()
    assert r.shape == shape and i.shape == shape, f"{what}: x, r and i must have one shape"
    assert r.dtype is dtype and i.dtype is dtype, f"{what}: x, r and i must have one dtype"
    assert Lambda.dim() == 1 and Lambda.numel() == shape[-1], f"{what}: Lambda must be [D]"
    assert h is None or (h.dim() == 2 and h.shape[0] == shape[0] and h.shape[1] == shape[-1]), \
        f"{what}: state must be [B, D]"
    if dtype not in _TYPES:
        _lib.dtype_code(x)
    if dev < 0:
        _lib.require_cuda(x, what=what)
    assert r.get_device() == dev and i.get_device() == dev and Lambda.get_device() == dev and \
        (h is None or h.get_device() == dev), f"{what}: tensors on different devices"


def gated_linear_scan(x: torch.Tensor, r: torch.Tensor, i: torch.Tensor, Lambda: torch.Tensor,
                      h0: torch.Tensor | None = None, reset: torch.Tensor | None = None, *,
                      sharpness: float = 8.0, return_final_state: bool = False,
                      wait_poll_limit: int = -1):
    """The recurrence over x, r, i [B, T, D] (fp32 or bf16, one dtype; the recurrence
    and input gates r and i before their sigmoid; column slices of wider tensors are
    read in place), Lambda [D], start state h0 [B, D] (zero if None).

    ``reset`` [B, T] bool marks steps that drop the state (the first token of each
    document of a packed sequence): there h = s(i) x. Returns y [B, T, D] in x's
    dtype, and with ``return_final_state`` also h_T [B, D] fp32. The state is fp32
    throughout. Differentiable in x, r, i, Lambda, h0, from y and h_T; the backward
    pass recomputes the states from fp32 ones kept every 32 steps (once: it has no
    second derivative).

    A device-side wait, forward or backward, that is not over after about a second gives up
    and reports to the device's status word, which ``_lib.check_device_status`` turns into
    an error, and each call by itself where MAMBAQC_B200_SYNC_CHECK is 1.
    ``wait_poll_limit`` 0 makes it give up at once (for tests)."""
    assert x.dim() == 3, f"x must be [B, T, D], got {tuple(x.shape)}"
    _check("gated_linear_scan", x, r, i, Lambda, h0)
    assert sharpness > 0, "sharpness must be positive"
    assert wait_poll_limit in (-1, 0), "wait_poll_limit must be -1 (default) or 0"
    if reset is not None:
        assert reset.dtype == torch.bool and reset.shape == x.shape[:2], \
            "reset must be bool [B, T]"
        assert reset.device == x.device, "gated_linear_scan: tensors on different devices"
    y, hT = _lib.torch_ops().gated_scan(x, r, i, Lambda, h0, reset, float(sharpness),
                                        return_final_state, _lib.status_ptr(x.get_device()),
                                        wait_poll_limit == 0)
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
    assert out is None or (out.shape == x.shape and out.dtype == x.dtype and
                           out.is_contiguous() and out.device == x.device), \
        "out must be a contiguous tensor like x"
    return _lib.torch_ops().gated_step(x, r, i, Lambda, h, float(sharpness), out)
