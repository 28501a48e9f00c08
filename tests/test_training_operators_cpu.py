"""C-ABI checks of the gated recurrence, norm + gate + residual and AdamW that need no
GPU: struct layouts against the header, and refusals before anything is launched."""

import ctypes

import pytest
import torch

from mambaqc_b200 import _lib
from tests.test_capi_cpu import INVALID, MISALIGNED, UNSUPPORTED, _c_offsets, no_gpu

FAKE = 0x10000  # never dereferenced: validation fails before any launch


@pytest.mark.parametrize("cstruct,pystruct", [("mqc_gated_scan_args", "GatedScanArgs"),
                                              ("mqc_norm_gate_args", "NormGateArgs"),
                                              ("mqc_adamw_args", "AdamwArgs")])
def test_struct_layout_matches_header(cstruct, pystruct, tmp_path):
    py = getattr(_lib, pystruct)
    got = _c_offsets(cstruct, [f for f, _ in py._fields_], tmp_path)
    assert got[0] == ctypes.sizeof(py)
    assert got[1:] == [getattr(py, f).offset for f, _ in py._fields_]


def _args(cls, base, changed):
    a = cls()
    for k, v in {**base, **changed}.items():
        setattr(a, k, v)
    return ctypes.byref(a)


SCAN = dict(batch=2, seq_len=8, channels=4, dtype=0, sharpness=8.0, x=FAKE, r=FAKE, i=FAKE,
            x_row=4, r_row=4, i_row=4, lambda_=FAKE, y=FAKE)


@no_gpu
@pytest.mark.parametrize("changed,want", [
    (dict(dtype=7), INVALID), (dict(batch=-1), INVALID), (dict(sharpness=0.0), INVALID),
    (dict(x=None), INVALID), (dict(lambda_=None), INVALID), (dict(y=None), INVALID),
    (dict(r_row=3), INVALID), (dict(x=FAKE + 2), MISALIGNED), (dict(hT=FAKE + 1), MISALIGNED),
    (dict(seq_len=1 << 31), UNSUPPORTED), (dict(batch=0), 0), (dict(channels=0), 0),
])
def test_scan_forward_refusals(changed, want):
    lib = _lib.load()
    assert lib.mqc_gated_scan_fwd(_args(_lib.GatedScanArgs, SCAN, changed), None) == want
    assert lib.mqc_gated_scan_fwd(None, None) == INVALID


@no_gpu
@pytest.mark.parametrize("changed,ws,want", [
    (dict(), 1 << 20, 0), (dict(dlambda=None), 1 << 20, INVALID), (dict(ckpt=None), 1 << 20, INVALID),
    (dict(dx=None), 1 << 20, INVALID), (dict(), 16, INVALID), (dict(dy_row=1), 1 << 20, INVALID),
    (dict(dr=FAKE + 1), 1 << 20, MISALIGNED),
])
def test_scan_backward_refusals(changed, ws, want):
    base = {**SCAN, **dict(ckpt=FAKE, dy=FAKE, dy_row=4, dx=FAKE, dr=FAKE, di=FAKE, dlambda=FAKE)}
    if want == 0:
        base["channels"] = 0
    got = _lib.load().mqc_gated_scan_bwd(_args(_lib.GatedScanArgs, base, changed), FAKE, ws, None)
    assert got == want


@no_gpu
def test_step_refusals():
    lib = _lib.load()

    def call(x=FAKE, row=8, h=FAKE, batch=2, channels=8, sharpness=8.0, dtype=0):
        return lib.mqc_gated_scan_step(x, row, FAKE, 8, FAKE, 8, FAKE, h, FAKE, batch, channels,
                                       sharpness, dtype, None)

    assert call(x=None) == INVALID and call(row=7) == INVALID and call(dtype=3) == INVALID
    assert call(sharpness=-1.0) == INVALID and call(batch=-1) == INVALID
    assert call(h=FAKE + 2) == MISALIGNED
    assert call(batch=0) == 0 and call(channels=0) == 0


NORM = dict(rows=4, width=32, z_row=32, x_dtype=0, y_dtype=0, norm=0, eps=1e-5, x=FAKE, y=FAKE,
            z=FAKE, weight=FAKE, scale=FAKE, next_weight=FAKE, out=FAKE, n=FAKE)


@no_gpu
@pytest.mark.parametrize("changed,want", [
    (dict(x_dtype=5), INVALID), (dict(x_dtype=1), UNSUPPORTED), (dict(width=4097), UNSUPPORTED),
    (dict(norm=2), INVALID), (dict(eps=-1.0), INVALID), (dict(rows=-1), INVALID),
    (dict(x=None), INVALID), (dict(z=None), INVALID), (dict(scale=None), INVALID),
    (dict(z_row=31), INVALID), (dict(y=None, next_weight=None), INVALID), (dict(out=None), INVALID),
    (dict(n=None), INVALID), (dict(weight=FAKE + 2), MISALIGNED), (dict(stats=FAKE + 4), MISALIGNED),
    (dict(rows=0), 0), (dict(width=0), 0),
])
def test_norm_forward_refusals(changed, want):
    lib = _lib.load()
    assert lib.mqc_norm_gate_fwd(_args(_lib.NormGateArgs, NORM, changed), None) == want
    assert lib.mqc_norm_gate_fwd(None, None) == INVALID


@no_gpu
@pytest.mark.parametrize("changed,ws,want", [
    (dict(stats=None), 1 << 26, INVALID), (dict(dx=None), 1 << 26, INVALID),
    (dict(dz=None), 1 << 26, INVALID), (dict(), 16, INVALID), (dict(dy=FAKE + 1), 1 << 26, MISALIGNED),
])
def test_norm_backward_refusals(changed, ws, want):
    base = {**NORM, **dict(stats=FAKE, dout=FAKE, dn=FAKE, dx=FAKE, dy=FAKE, dz=FAKE)}
    got = _lib.load().mqc_norm_gate_bwd(_args(_lib.NormGateArgs, base, changed), FAKE, ws, None)
    assert got == want


def _adamw(**changed):
    one = (ctypes.c_void_p * 2)(FAKE, FAKE)
    sizes = (ctypes.c_int64 * 2)(8, 8)
    base = dict(count=2, numel=ctypes.addressof(sizes), param=ctypes.addressof(one),
                grad=ctypes.addressof(one), exp_avg=ctypes.addressof(one),
                exp_avg_sq=ctypes.addressof(one), lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8,
                weight_decay=0.0, step=1, param_dtype=0, grad_dtype=0, state_bits=32)
    for k, v in changed.items():
        if isinstance(v, ctypes.Array):
            changed[k] = ctypes.addressof(v)
    return _lib.load().mqc_adamw_step(_args(_lib.AdamwArgs, base, changed), None)


@no_gpu
def test_adamw_refusals():
    assert _lib.load().mqc_adamw_step(None, None) == INVALID
    for bad in (dict(count=-1), dict(step=0), dict(beta1=1.0), dict(beta2=-0.1),
                dict(state_bits=16), dict(flags=2), dict(param_dtype=9), dict(grad=None), dict(state_bits=8),
                dict(numel=None), dict(numel=(ctypes.c_int64 * 2)(8, -1)),
                dict(param=(ctypes.c_void_p * 2)(FAKE, None))):
        assert _adamw(**bad) == INVALID, bad
    assert _adamw(param=(ctypes.c_void_p * 2)(FAKE, FAKE + 2)) == MISALIGNED
    assert _adamw(count=0) == 0
    none = (ctypes.c_void_p * 2)(None, None)
    empty = (ctypes.c_int64 * 2)(0, 0)
    assert _adamw(numel=empty, param=none, grad=none, exp_avg=none, exp_avg_sq=none) == 0


@no_gpu
def test_grad_norm_and_moments_refusals():
    lib = _lib.load()
    sizes = (ctypes.c_int64 * 1)(8)
    ptrs = (ctypes.c_void_p * 1)(FAKE)
    odd = (ctypes.c_void_p * 1)(FAKE + 1)
    types = (ctypes.c_int32 * 1)(0)
    wrong = (ctypes.c_int32 * 1)(4)
    need = lib.mqc_grad_norm_workspace_size(1)
    assert need > 0 and lib.mqc_grad_norm_workspace_size(0) == 0
    assert lib.mqc_grad_norm(1, sizes, ptrs, types, 1.0, None, FAKE, need, None) == INVALID
    assert lib.mqc_grad_norm(1, sizes, odd, types, 1.0, FAKE, FAKE, need, None) == INVALID
    assert lib.mqc_grad_norm(1, sizes, ptrs, wrong, 1.0, FAKE, FAKE, need, None) == INVALID
    assert lib.mqc_grad_norm(1, sizes, ptrs, types, 1.0, FAKE, None, need, None) == INVALID
    assert lib.mqc_grad_norm(1, sizes, ptrs, types, 1.0, FAKE, FAKE, 0, None) == INVALID
    args = [sizes, ptrs, ptrs, ptrs, ptrs, ptrs, ptrs, None]
    assert lib.mqc_adamw_moments(0, *args) == 0
    for k in range(1, 7):
        bad = list(args)
        bad[k] = None
        assert lib.mqc_adamw_moments(1, *bad) == INVALID
    assert lib.mqc_adamw_moments(1, sizes, ptrs, ptrs, ptrs, ptrs, odd, ptrs, None) == MISALIGNED


def test_optimizer_refuses_without_a_gpu():
    from mambaqc_b200.kernels import adamw_step, gated_linear_scan, residual_norm
    from mambaqc_b200.models import HybridMamba2
    t = torch.zeros(2, 3, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        gated_linear_scan(t, t, t, t[0, 0])
    with pytest.raises(RuntimeError, match="CUDA"):
        residual_norm(t, torch.ones(4))
    with pytest.raises(RuntimeError, match="CUDA"):
        adamw_step([t], [t], [t.clone()], [t.clone()], step=1, lr=1e-3)
    lm = HybridMamba2(10, d_model=16, n_layers=3, pattern="gq", d_state=4)
    kinds = [type(b).__name__ for b in lm.layers]
    assert kinds == ["GatedRecurrentBlock", "QuaternionMamba2Block", "GatedRecurrentBlock"]
    assert len(lm.pre_norm) == 4 and len(lm.post_norm) == 3


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_survives_copy_and_pickle(bits):
    import copy
    import pickle

    from mambaqc_b200.optim import AdamW
    p = torch.nn.Parameter(torch.ones(300))
    opt = AdamW([p], lr=1e-2, state_bits=bits, seed=9)
    opt.state[p] = {"step": 3, "exp_avg": torch.ones(300), "exp_avg_sq": torch.ones(300)}
    opt.grad_norm = torch.tensor(2.0)
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert other.state_bits == bits and other.seed == 9 and other.grad_norm == 2.0
        q = other.param_groups[0]["params"][0]
        assert q is not p and other.state[q]["step"] == 3
        assert other.param_groups[0]["lr"] == 1e-2
        assert other.state_dict()["state_bits"] == bits


def test_state_of_torch_adamw_loads():
    """Steps as numbers (parameters that share one are stepped in one call), moments
    flat in the parameters' order and fp32; what has no counterpart is refused."""
    from mambaqc_b200.optim import AdamW

    def params():
        g = torch.Generator().manual_seed(3)
        return [torch.nn.Parameter(torch.randn(5, 7, generator=g)),
                torch.nn.Parameter(torch.randn(6, 4, generator=g).t()),
                torch.nn.Parameter(torch.randn(9, generator=g).bfloat16())]

    theirs = params()
    opt = torch.optim.AdamW(theirs, lr=1e-2, betas=(0.8, 0.9))
    for _ in range(3):
        for p in theirs:
            p.grad = torch.randn(p.shape).to(p.dtype)
        opt.step()
    ours = params()
    got = AdamW(ours)
    got.load_state_dict(opt.state_dict())
    assert got.param_groups[0]["lr"] == 1e-2 and tuple(got.param_groups[0]["betas"]) == (0.8, 0.9)
    for p, q in zip(theirs, ours):
        s, want = got.state[q], opt.state[p]
        assert type(s["step"]) is int and s["step"] == 3
        for name in ("exp_avg", "exp_avg_sq"):
            assert s[name].dtype == torch.float32 and s[name].is_contiguous()
            assert torch.equal(s[name], want[name].float().reshape(-1))
    again = AdamW(params())
    again.load_state_dict(got.state_dict())
    assert all(type(again.state[q]["step"]) is int for q in again.param_groups[0]["params"])
    with pytest.raises(ValueError, match="32-bit"):
        AdamW(params(), state_bits=8).load_state_dict(opt.state_dict())
    odd = torch.optim.AdamW(params(), amsgrad=True)
    with pytest.raises(ValueError, match="amsgrad"):
        AdamW(params()).load_state_dict(odd.state_dict())


def test_refused_step_is_not_counted():
    from mambaqc_b200.optim import AdamW
    p = torch.nn.Parameter(torch.ones(4))
    p.grad = torch.ones(4)
    opt = AdamW([p])
    for _ in range(2):
        with pytest.raises(RuntimeError, match="CUDA"):
            opt.step()
    assert opt.state[p]["step"] == 0


def test_extension_is_built_again_for_another_torch(monkeypatch, tmp_path, capsys):
    """An extension newer than its source, but for another torch, is compiled again;
    without torch's headers or g++ the C library is built alone."""
    import shutil
    import subprocess

    from mambaqc_b200.csrc import build
    _lib.torch_ops()                                        # this one loads
    lib = tmp_path / "_torch_ops.so"
    shutil.copy(build.OPS_LIB, lib)
    monkeypatch.setattr(build, "OPS_LIB", lib)
    ran = []

    def run(cmd, **_):
        ran.append(cmd)
        lib.with_suffix(".so.tmp").write_bytes(b"new")
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build.subprocess, "run", run)
    assert build.build_torch_ops(quiet=True) == lib and not ran
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    assert build.build_torch_ops(quiet=True) == lib and len(ran) == 1
    assert lib.read_bytes() == b"new"
    monkeypatch.setattr(build.shutil, "which", lambda name: None)
    assert build.build_torch_ops(force=True, quiet=True) is None and len(ran) == 1
    assert "no g++" in capsys.readouterr().err
