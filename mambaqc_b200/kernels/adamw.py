"""AdamW over a list of tensors in a few launches, moments in 32 or in 8 bits.

``adamw_step`` is the update of ``mambaqc_b200.optim.AdamW`` on plain tensors;
``grad_norm`` the global gradient norm that its clipping uses; ``adamw_moments``
the values that 8-bit moments stand for. The kernels are in ``csrc/adamw.cu``.

8-bit moments: 256 consecutive values of a tensor share one power of two (a byte,
the biased fp32 exponent of the largest). A byte of ``exp_avg`` is sign, 4 exponent
and 3 fraction bits of m under it, a byte of ``exp_avg_sq`` 4 exponent and 4
fraction bits of sqrt(v). Both, and bf16 parameters, are rounded up or down by a
hash of (seed, step, tensor, element) that makes the rounding unbiased: v moves by
1 - beta2 = 0.1 % a step, which rounding to nearest would lose every time.
"""

from __future__ import annotations

import torch

from .. import _lib

__all__ = ["adamw_step", "adamw_moments", "grad_norm"]


_FLOATS = (torch.float32, torch.bfloat16)


def _check_list(what, name, tensors, sizes, dev, dtypes):
    """Contiguous tensors of the given element counts and types on one device."""
    assert len(tensors) == len(sizes), f"{what}: {len(sizes)} tensors, but {len(tensors)} of {name}"
    for k, t in enumerate(tensors):
        if t.dtype not in dtypes:
            raise TypeError(f"{what}: {name}[{k}] is {t.dtype}, "
                            f"not one of {', '.join(map(str, dtypes))}")
        assert t.is_contiguous(), f"{what}: {name}[{k}] must be contiguous"
        assert t.numel() == sizes[k], \
            f"{what}: {name}[{k}] has {t.numel()} elements, not {sizes[k]}"
        assert t.get_device() == dev, f"{what}: tensors on different devices"


def _blocks(sizes):
    return [-(-n // _lib.MQC_ADAMW_BLOCK) for n in sizes]


@torch.no_grad()
def grad_norm(grads: list[torch.Tensor], max_norm: float | None = None) -> torch.Tensor:
    """[norm, factor] fp32 on the device: the Euclidean norm of all of ``grads``
    together (contiguous fp32 or bf16, mixed as they come), and what clipping to
    ``max_norm`` multiplies them by, min(1, max_norm / (norm + 1e-6)) (1 if None)."""
    grads = list(grads)
    if not grads:
        return torch.tensor([0.0, 1.0])
    _lib.require_cuda(grads[0], what="grad_norm")
    _check_list("grad_norm", "grads", grads, [g.numel() for g in grads], grads[0].get_device(),
                _FLOATS)
    assert max_norm is None or max_norm >= 0, "max_norm must not be negative"
    return _lib.torch_ops().grad_norm(grads, -1.0 if max_norm is None else float(max_norm))


@torch.no_grad()
def adamw_step(params: list[torch.Tensor], grads: list[torch.Tensor],
               exp_avgs: list[torch.Tensor], exp_avg_sqs: list[torch.Tensor], *, step: int,
               lr: float, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 1e-2, max_grad_norm: float | None = None,
               exponents: tuple[list[torch.Tensor], list[torch.Tensor]] | None = None,
               seed: int = 0, carry: bool = False, clip: torch.Tensor | None = None,
               ordinals: list[int] | None = None) -> torch.Tensor | None:
    """One AdamW step, in place, of contiguous fp32 or bf16 ``params`` with contiguous
    fp32 or bf16 ``grads``; ``step`` is 1 for the first.

    32-bit moments: ``exp_avgs`` and ``exp_avg_sqs`` are fp32. 8-bit moments: they are
    uint8 codes and ``exponents`` the two lists of uint8 block exponents
    [ceil(numel / 256)]; all zero is the zero state. A block's largest value is held at
    the last code below the next power of two; with ``carry`` it may be rounded up to
    that power, which a moment that grows slowly over many steps needs (the optimizer
    sets it; for a single step the two differ by one code at most). ``max_grad_norm`` clips by the
    global norm of ``grads`` without a pass that rewrites them, and returns that norm
    (a device scalar); ``clip`` (a device fp32 scalar, from ``grad_norm``) is for
    callers that split one clipped step over several calls. ``ordinals`` are the
    tensors' places in such a caller's whole list (default 0, 1, ...): with ``seed``
    and ``step`` they choose the rounding of 8-bit moments and bf16 parameters."""
    params, grads = list(params), list(grads)
    exp_avgs, exp_avg_sqs = list(exp_avgs), list(exp_avg_sqs)
    assert step >= 1, "step counts from 1"
    assert max_grad_norm is None or clip is None, "max_grad_norm and clip exclude each other"
    if not params:
        return None if max_grad_norm is None else torch.zeros(())
    ops = _lib.torch_ops()
    bits8 = exponents is not None
    em, ev = (list(exponents[0]), list(exponents[1])) if bits8 else ([], [])
    if not ops.lists_fit(params, grads, exp_avgs, exp_avg_sqs, em, ev, bits8):
        _refuse_lists(params, grads, exp_avgs, exp_avg_sqs, em, ev, bits8)
    if ordinals is None:
        ordinals = range(len(params))
    assert len(ordinals) == len(params), "adamw_step: one ordinal a tensor"
    norm = None
    if max_grad_norm is not None:
        assert max_grad_norm >= 0, "max_norm must not be negative"
        got = ops.grad_norm(grads, float(max_grad_norm))
        norm, clip = got[0], got[1]
    elif clip is not None:
        assert clip.numel() == 1 and clip.dtype == torch.float32 and \
            clip.get_device() == params[0].get_device(), \
            "clip must be one float32 on the parameters' device"
    ops.adamw_step(params, grads, exp_avgs, exp_avg_sqs, em, ev, ordinals, clip, step, lr, betas[0],
                   betas[1], eps, weight_decay, bits8, carry, seed & 0xFFFFFFFF)
    return norm


def _refuse_lists(params, grads, exp_avgs, exp_avg_sqs, em, ev, bits8):
    """Says what does not fit about the lists of a step."""
    what = "adamw_step"
    _lib.require_cuda(params[0], what=what)
    state = (torch.uint8,) if bits8 else (torch.float32,)
    sizes, dev = [p.numel() for p in params], params[0].get_device()
    _check_list(what, "params", params, sizes, dev, _FLOATS)
    _check_list(what, "grads", grads, sizes, dev, _FLOATS)
    _check_list(what, "exp_avgs", exp_avgs, sizes, dev, state)
    _check_list(what, "exp_avg_sqs", exp_avg_sqs, sizes, dev, state)
    if bits8:
        _check_list(what, "exponents[0]", em, _blocks(sizes), dev, state)
        _check_list(what, "exponents[1]", ev, _blocks(sizes), dev, state)
    raise AssertionError(f"{what}: the lists do not fit together")


@torch.no_grad()
def adamw_moments(exp_avgs: list[torch.Tensor], exp_avg_sqs: list[torch.Tensor],
                  exponents: tuple[list[torch.Tensor], list[torch.Tensor]]):
    """(m, sqrt(v)) of 8-bit moments, two lists of bf16 tensors shaped like the codes
    (exact: a value has at most 5 significant bits)."""
    exp_avgs, exp_avg_sqs = list(exp_avgs), list(exp_avg_sqs)
    if not exp_avgs:
        return [], []
    what = "adamw_moments"
    _lib.require_cuda(exp_avgs[0], what=what)
    em, ev = list(exponents[0]), list(exponents[1])
    ops = _lib.torch_ops()
    if not ops.lists_fit(exp_avgs, exp_avgs, exp_avgs, exp_avg_sqs, em, ev, True):
        sizes, dev = [t.numel() for t in exp_avgs], exp_avgs[0].get_device()
        for name, part, count in (("exp_avgs", exp_avgs, sizes),
                                  ("exp_avg_sqs", exp_avg_sqs, sizes),
                                  ("exponents[0]", em, _blocks(sizes)),
                                  ("exponents[1]", ev, _blocks(sizes))):
            _check_list(what, name, part, count, dev, (torch.uint8,))
    return ops.adamw_moments(exp_avgs, exp_avg_sqs, em, ev)
