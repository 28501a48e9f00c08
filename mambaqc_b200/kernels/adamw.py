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

import ctypes

import torch

from .. import _lib

__all__ = ["adamw_step", "adamw_moments", "grad_norm"]


_Tensor = torch.Tensor


def _pointers(tensors):
    return (ctypes.c_void_p * len(tensors))(*map(_Tensor.data_ptr, tensors))


def _check_list(what, name, tensors, sizes, dev, dtypes):
    """Contiguous tensors of the given element counts and types on one device."""
    if (list(map(_Tensor.numel, tensors)) == sizes and
            set(map(_Tensor.get_device, tensors)) == {dev} and
            all(map(_Tensor.is_contiguous, tensors)) and
            all([t.dtype in dtypes for t in tensors])):
        return
    assert len(tensors) == len(sizes), f"{what}: {len(sizes)} tensors, but {len(tensors)} of {name}"
    for k, t in enumerate(tensors):
        if t.dtype not in dtypes:
            raise TypeError(f"{what}: {name}[{k}] is {t.dtype}, "
                            f"not one of {', '.join(map(str, dtypes))}")
        assert t.is_contiguous(), f"{what}: {name}[{k}] must be contiguous"
        assert t.numel() == sizes[k], \
            f"{what}: {name}[{k}] has {t.numel()} elements, not {sizes[k]}"
        assert t.get_device() == dev, f"{what}: tensors on different devices"


_CODES = {torch.float32: _lib.MQC_DTYPE_F32, torch.bfloat16: _lib.MQC_DTYPE_BF16}
_FLOATS = tuple(_CODES)


@torch.no_grad()
def grad_norm(grads: list[torch.Tensor], max_norm: float | None = None) -> torch.Tensor:
    """[norm, factor] fp32 on the device: the Euclidean norm of all of ``grads``
    together (contiguous fp32 or bf16, mixed as they come), and what clipping to
    ``max_norm`` multiplies them by, min(1, max_norm / (norm + 1e-6)) (1 if None)."""
    grads = list(grads)
    if not grads:
        return torch.tensor([0.0, 1.0])
    _lib.require_cuda(grads[0], what="grad_norm")
    sizes = list(map(_Tensor.numel, grads))
    _check_list("grad_norm", "grads", grads, sizes, grads[0].get_device(), _FLOATS)
    assert max_norm is None or max_norm >= 0, "max_norm must not be negative"
    return _grad_norm(grads, sizes, max_norm)


def _grad_norm(grads, sizes, max_norm):
    dev, n = grads[0].device, len(grads)
    # 4-byte words: the partial sums (8-byte aligned), then the two results
    nbytes = _lib.load().mqc_grad_norm_workspace_size(n)
    out = torch.empty(nbytes // 4 + 2, dtype=torch.float32, device=dev)
    _lib.call_on(dev.index, "mqc_grad_norm", n, (ctypes.c_int64 * n)(*sizes), _pointers(grads),
                 (ctypes.c_int32 * n)(*[_CODES[g.dtype] for g in grads]),
                 -1.0 if max_norm is None else float(max_norm), out.data_ptr() + nbytes,
                 out.data_ptr(), nbytes)
    return out[nbytes // 4:]


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
    what = "adamw_step"
    _lib.require_cuda(params[0], what=what)
    bits = 32 if exponents is None else 8
    state = (torch.float32,) if bits == 32 else (torch.uint8,)
    sizes = list(map(_Tensor.numel, params))
    idx = params[0].get_device()
    _check_list(what, "params", params, sizes, idx, _FLOATS)
    _check_list(what, "grads", grads, sizes, idx, _FLOATS)
    _check_list(what, "exp_avgs", exp_avgs, sizes, idx, state)
    _check_list(what, "exp_avg_sqs", exp_avg_sqs, sizes, idx, state)
    lists = [params, grads, exp_avgs, exp_avg_sqs]
    if bits == 8:
        blocks = [-(-n // _lib.MQC_ADAMW_BLOCK) for n in sizes]
        for name, part in zip(("exponents[0]", "exponents[1]"), exponents):
            _check_list(what, name, part, blocks, idx, state)
        lists += [list(exponents[0]), list(exponents[1])]
    if ordinals is None:
        ordinals = range(len(params))
    assert len(ordinals) == len(params), f"{what}: one ordinal a tensor"
    norm = None
    a = _lib.AdamwArgs()
    if max_grad_norm is not None:
        assert max_grad_norm >= 0, "max_norm must not be negative"
        got = _grad_norm(grads, sizes, max_grad_norm)
        norm, a.clip = got[0], got.data_ptr() + 4
    elif clip is not None:
        assert clip.numel() == 1 and clip.dtype == torch.float32 and clip.get_device() == idx, \
            "clip must be one float32 on the parameters' device"
        a.clip = clip.data_ptr()
    a.lr, (a.beta1, a.beta2), a.eps, a.weight_decay = lr, betas, eps, weight_decay
    a.step, a.state_bits, a.seed = step, bits, seed & 0xFFFFFFFF
    a.flags = _lib.MQC_ADAMW_CARRY if carry else 0
    # one call for each pair of parameter and gradient types
    kinds: dict[tuple, list[int] | range] = {}
    pairs = [(p.dtype, g.dtype) for p, g in zip(params, grads)]
    if len(set(pairs)) == 1:
        kinds[pairs[0]] = range(len(params))
    else:
        for k, pair in enumerate(pairs):
            kinds.setdefault(pair, []).append(k)
    for (p_dtype, g_dtype), members in kinds.items():
        n = len(members)
        part, count, place = lists, sizes, ordinals
        if n < len(params):
            part = [[t[k] for k in members] for t in lists]
            count, place = [sizes[k] for k in members], [ordinals[k] for k in members]
        numel = (ctypes.c_int64 * n)(*count)
        places = (ctypes.c_int64 * n)(*place)
        arrays = [_pointers(t) for t in part]
        a.count, a.param_dtype, a.grad_dtype = n, _CODES[p_dtype], _CODES[g_dtype]
        a.numel, a.ordinal = ctypes.addressof(numel), ctypes.addressof(places)
        for field, arr in zip(("param", "grad", "exp_avg", "exp_avg_sq", "exp_avg_exponent",
                               "exp_avg_sq_exponent"), arrays):
            setattr(a, field, ctypes.addressof(arr))
        _lib.call_on(idx, "mqc_adamw_step", ctypes.byref(a))
    return norm


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
    sizes = list(map(_Tensor.numel, exp_avgs))
    idx, n = exp_avgs[0].get_device(), len(exp_avgs)
    _check_list(what, "exp_avgs", exp_avgs, sizes, idx, (torch.uint8,))
    _check_list(what, "exp_avg_sqs", exp_avg_sqs, sizes, idx, (torch.uint8,))
    blocks = [-(-k // _lib.MQC_ADAMW_BLOCK) for k in sizes]
    for name, part in zip(("exponents[0]", "exponents[1]"), exponents):
        _check_list(what, name, part, blocks, idx, (torch.uint8,))
    m = [torch.empty_like(t, dtype=torch.bfloat16) for t in exp_avgs]
    root = [torch.empty_like(t, dtype=torch.bfloat16) for t in exp_avgs]
    _lib.call_on(idx, "mqc_adamw_moments", n, (ctypes.c_int64 * n)(*sizes), _pointers(exp_avgs),
                 _pointers(exp_avg_sqs), _pointers(exponents[0]), _pointers(exponents[1]),
                 _pointers(m), _pointers(root))
    return m, root
