"""Norm + gate + residual on the GPU against the formulas in 64 bits, with gradients
from torch's autograd through those and from differences.

Tolerances (relative L2): fp32 results are a few dozen roundings of 6e-8 at most:
1e-5. A bf16 result is rounded once, by at most half of 2^-7 of each value: 2^-8 + 1e-5.
Column sums over the rows cancel by chance; they are fp32 and get 1e-5 too, as a sum
of n terms grows like sqrt(n) and so does its error. Rows that are the same number
throughout are judged on their own."""

import pytest
import torch

from tests.gpu_util import DEV, RTOL_F32, gen, rel_l2

pytestmark = pytest.mark.gpu

from mambaqc_b200.kernels import norm_gate_residual, residual_norm  # noqa: E402

TOL_BF16 = 2.0 ** -8 + 1e-5
EPS = 1e-5
F32, BF16 = torch.float32, torch.bfloat16


def _tol(dt):
    return RTOL_F32 if dt == F32 else TOL_BF16


def _norm(u, w, b, kind):
    if kind == "layer":
        u = u - u.mean(-1, keepdim=True)
    u = u / torch.sqrt(u.square().mean(-1, keepdim=True) + EPS) * w
    return u if b is None else u + b


def _ref(q, kind):
    out = q["x"] + q["scale"] * torch.sigmoid(q["z"]) * _norm(q["y"], q["weight"], q.get("bias"),
                                                               kind)
    if "next_weight" not in q:
        return (out,)
    return out, _norm(out, q["next_weight"], q.get("next_bias"), kind)


def _call(q, kind):
    got = norm_gate_residual(q["x"], q["y"], q["z"], q["weight"], q["scale"], q.get("bias"),
                             q.get("next_weight"), q.get("next_bias"), norm=kind, eps=EPS)
    return got if isinstance(got, tuple) else (got,)


def _inputs(rows, d, xt, yt, bias, nxt, seed=0):
    g = gen(seed + rows + 3 * d)
    q = {"x": torch.randn(rows, d, generator=g).to(xt),
         "y": (2 * torch.randn(rows, d, generator=g) + 0.5).to(yt),
         "z": torch.randn(rows, d, generator=g).to(yt),
         "weight": 1 + 0.2 * torch.randn(d, generator=g),
         "scale": 0.7 + 0.2 * torch.randn(d, generator=g)}
    if bias:
        q["bias"] = 0.2 * torch.randn(d, generator=g)
    if nxt:
        q["next_weight"] = 1 + 0.2 * torch.randn(d, generator=g)
        if bias:
            q["next_bias"] = 0.2 * torch.randn(d, generator=g)
    return q


def _check(q, kind, xt, yt, grads=None):
    """Outputs and gradients of one set of inputs against 64 bits."""
    dev = {k: v.to(DEV).requires_grad_() for k, v in q.items()}
    ref = {k: v.double().requires_grad_() for k, v in q.items()}
    outs, refs = _call(dev, kind), _ref(ref, kind)
    g = gen(5)
    if grads is None:
        grads = [torch.randn(o.shape, generator=g).to(o.dtype) for o in outs]
    torch.autograd.backward(outs, [v.to(DEV) for v in grads])
    torch.autograd.backward(refs, [v.double() for v in grads])
    assert outs[0].dtype == xt and rel_l2(outs[0], refs[0]) < _tol(xt)
    if len(outs) == 2:
        assert outs[1].dtype == yt and rel_l2(outs[1], refs[1]) < _tol(yt)
    for k, v in dev.items():
        tol = _tol(v.dtype)
        assert rel_l2(v.grad, ref[k].grad) < tol, (k, rel_l2(v.grad, ref[k].grad))


TYPES = [(F32, F32), (F32, BF16), (BF16, BF16)]
SHAPES = [(2, 3), (3, 5), (2, 32), (7, 33), (5, 128), (300, 100), (9, 515), (64, 768),
          (33, 1024), (1000, 257), (4, 2048), (3, 2050), (5, 4096), (3, 4095), (2, 1025)]


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kind,bias,nxt", [("layer", True, True), ("rms", False, True),
                                           ("layer", False, False), ("rms", True, False)])
def test_matches_64_bits(shape, types, kind, bias, nxt):
    _check(_inputs(*shape, *types, bias, nxt), kind, *types)


def test_many_rows():
    """More row groups than the grid holds: every CTA walks several."""
    for types in TYPES:
        _check(_inputs(20000, 64, *types, True, True), "layer", *types)
        _check(_inputs(7001, 100, *types, True, True), "rms", *types)


@pytest.mark.parametrize("kind,d", [("rms", 1), ("layer", 2), ("layer", 1)])
def test_narrow_rows(kind, d):
    """Rows whose norm leaves no freedom (one value under RMSNorm is its sign, two under
    LayerNorm are +1 and -1, one is zero): the gradients through the norm are eps-sized
    differences of numbers of the size of 1/std (up to 100 here), so they are judged to
    an absolute 1e-4, a few roundings of those."""
    q = _inputs(40, d, F32, F32, True, True)
    q["y"] = q["y"].sign() * (0.2 + q["y"].abs())
    dev = {k: v.to(DEV).requires_grad_() for k, v in q.items()}
    ref = {k: v.double().requires_grad_() for k, v in q.items()}
    outs, refs = _call(dev, kind), _ref(ref, kind)
    (outs[0].sum() + outs[1].sum()).backward()
    (refs[0].sum() + refs[1].sum()).backward()
    for o, r in zip(outs, refs):
        torch.testing.assert_close(o.double().cpu(), r, rtol=0, atol=1e-4)
    for k, v in dev.items():
        scale = 40 if v.dim() == 1 else 1   # the column sums add 40 rows
        torch.testing.assert_close(v.grad.double().cpu(), ref[k].grad, rtol=0, atol=scale * 1e-4)


def test_constant_and_zero_rows():
    """A row of one number has no variance: LayerNorm gives its bias; a zero row gives
    its bias under either norm. Gradients are finite."""
    q = _inputs(4, 96, F32, F32, True, True)
    q["y"][0] = 0.0
    q["y"][1] = 3.0
    q["x"][2] = 0.0
    for kind in ("layer", "rms"):
        dev = {k: v.to(DEV).requires_grad_() for k, v in q.items()}
        out, n = _call(dev, kind)
        (out.sum() + n.square().sum()).backward()
        gate = (q["scale"] * torch.sigmoid(q["z"].double()))
        assert rel_l2(out[0], q["x"][0].double() + gate[0] * q["bias"].double()) < RTOL_F32
        if kind == "layer":
            assert rel_l2(out[1], q["x"][1].double() + gate[1] * q["bias"].double()) < RTOL_F32
        for v in dev.values():
            assert torch.isfinite(v.grad).all()


def test_large_mean_and_scale():
    """A mean of 1000 standard deviations: the mean is taken off before the squares are
    summed, so the error stays the mean's own rounding, 1000 * 6e-8 of the result."""
    q = _inputs(16, 768, F32, F32, True, True)
    q["y"] = 1000.0 + q["y"]
    ref = _ref({k: v.double() for k, v in q.items()}, "layer")
    got = _call({k: v.to(DEV) for k, v in q.items()}, "layer")
    assert rel_l2(got[0], ref[0]) < 1e-4 and rel_l2(got[1], ref[1]) < 1e-4
    q = _inputs(16, 768, F32, F32, True, True)
    q["y"] = q["y"] * 1e12
    ref = _ref({k: v.double() for k, v in q.items()}, "rms")
    got = _call({k: v.to(DEV) for k, v in q.items()}, "rms")
    assert rel_l2(got[1], ref[1]) < RTOL_F32


def test_saturated_gates_and_nan():
    q = _inputs(8, 64, F32, F32, True, True)
    q["z"][:, 0], q["z"][:, 1], q["z"][:, 2] = 200.0, -200.0, -90.0
    _check(q, "layer", F32, F32)
    q["z"][:, 3], q["z"][:, 4] = float("inf"), float("-inf")
    dev = {k: v.to(DEV).requires_grad_() for k, v in q.items()}
    out, n = _call(dev, "layer")
    refs = _ref({k: v.double() for k, v in q.items()}, "layer")
    assert rel_l2(out, refs[0]) < RTOL_F32 and rel_l2(n, refs[1]) < RTOL_F32
    for where in ("x", "y", "z"):
        p = {k: v.clone() for k, v in q.items()}
        p[where][3, 7] = float("nan")
        o, m = _call({k: v.to(DEV) for k, v in p.items()}, "layer")
        assert torch.isnan(m[3]).all() and torch.isnan(o[3, 7])
        keep = [k for k in range(8) if k != 3]
        assert torch.equal(o[keep], out[keep]) and torch.equal(m[keep], n[keep])


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("d,offset", [(64, 64), (64, 1), (30, 30), (515, 515)])
def test_strided_gate_and_views(types, d, offset):
    """z as a slice of a wider projection (also at an odd offset), x and y transposed or
    with leading dimensions, and an expanded gradient."""
    xt, yt = types
    q = _inputs(12, d, xt, yt, True, True)
    wide = torch.randn(3, 4, d + offset, generator=gen(2)).to(yt)
    dev = {k: v.to(DEV) for k, v in q.items()}
    ref = {k: v.double() for k, v in q.items()}
    wd, wr = wide.to(DEV).requires_grad_(), wide.double().requires_grad_()
    yd = dev["y"].view(3, 4, d).transpose(0, 1).contiguous().transpose(0, 1).requires_grad_()
    yr = ref["y"].view(3, 4, d).requires_grad_()
    dev.update(x=dev["x"].view(3, 4, d), y=yd, z=wd[..., offset:])
    ref.update(x=ref["x"].view(3, 4, d), y=yr, z=wr[..., offset:])
    outs, refs = _call(dev, "layer"), _ref(ref, "layer")
    (outs[0].sum() + outs[1][..., :1].sum()).backward()
    (refs[0].sum() + refs[1][..., :1].sum()).backward()
    assert rel_l2(outs[0], refs[0]) < _tol(xt) and rel_l2(outs[1], refs[1]) < _tol(yt)
    assert rel_l2(wd.grad, wr.grad) < _tol(yt)
    assert rel_l2(yd.grad, yr.grad) < _tol(yt)


def test_one_of_two_gradients():
    """Only out, or only n, is used further on; parameters without a gradient."""
    for use in (0, 1):
        q = _inputs(50, 100, F32, F32, True, True)
        dev = {k: v.to(DEV).requires_grad_(k not in ("scale", "next_bias")) for k, v in q.items()}
        ref = {k: v.double().requires_grad_(k not in ("scale", "next_bias")) for k, v in q.items()}
        w = torch.randn(50, 100, generator=gen(4))
        (_call(dev, "layer")[use] * w.to(DEV)).sum().backward()
        (_ref(ref, "layer")[use] * w.double()).sum().backward()
        for k, v in dev.items():
            if v.requires_grad:
                e = ref[k].grad if ref[k].grad is not None else torch.zeros(v.shape)
                if torch.count_nonzero(e) == 0:
                    assert torch.count_nonzero(v.grad) == 0, k
                else:
                    assert rel_l2(v.grad, e) < RTOL_F32, k
        assert dev["scale"].grad is None and dev["next_bias"].grad is None


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("types", TYPES)
def test_residual_norm(kind, bias, types):
    xt, nt = types
    for rows, d in [(1, 7), (40, 96), (9, 1030), (3000, 64)]:
        q = _inputs(rows, d, xt, nt, bias, True)
        w, b = q["next_weight"], q.get("next_bias")
        x = q["x"].to(DEV).requires_grad_()
        wd = w.to(DEV).requires_grad_()
        bd = None if b is None else b.to(DEV).requires_grad_()
        n = residual_norm(x, wd, bd, norm=kind, eps=EPS, dtype=nt)
        xr, wr = q["x"].double().requires_grad_(), w.double().requires_grad_()
        br = None if b is None else b.double().requires_grad_()
        nr = _norm(xr, wr, br, kind)
        g = torch.randn(rows, d, generator=gen(1)).to(nt)
        n.backward(g.to(DEV))
        nr.backward(g.double())
        assert n.dtype == nt and rel_l2(n, nr) < _tol(nt)
        assert rel_l2(x.grad, xr.grad) < _tol(xt)
        assert rel_l2(wd.grad, wr.grad) < RTOL_F32
        if b is not None:
            assert rel_l2(bd.grad, br.grad) < RTOL_F32


def test_types_meet():
    """bf16 parameters get bf16 gradients; a bf16 residual under an fp32 branch is taken
    to fp32; the gate takes the branch's type."""
    q = {k: v.to(DEV) for k, v in _inputs(8, 64, BF16, F32, True, True).items()}
    out, n = _call(q, "rms")
    assert out.dtype == F32 and n.dtype == F32
    q = _inputs(8, 64, F32, BF16, True, True)
    q["z"] = q["z"].float()
    w = q["weight"].to(BF16)
    dev = {k: v.to(DEV) for k, v in q.items()}
    dev["weight"] = w.to(DEV).requires_grad_()
    dev["z"] = dev["z"].requires_grad_()
    out, n = _call(dev, "rms")
    (out.sum() + n.float().sum()).backward()
    assert dev["weight"].grad.dtype == BF16 and dev["z"].grad.dtype == F32


def test_gradient_against_differences():
    """Central differences with step e = 0.01 along each gradient's signs: truncation
    e^2 / 6 of the third derivative and 1e-6 / (2 e) of rounding: 2e-3."""
    for kind in ("layer", "rms"):
        base = {k: v.to(DEV) for k, v in _inputs(6, 40, F32, F32, True, True).items()}
        w = [torch.randn(6, 40, generator=gen(8 + k)).to(DEV) for k in range(2)]

        def loss(q):
            return sum((o.double() * v.double()).sum() for o, v in zip(_call(q, kind), w))

        leaves = {k: v.clone().requires_grad_() for k, v in base.items()}
        loss(leaves).backward()
        for k, v in leaves.items():
            step, way = 0.01, torch.sign(v.grad)
            got = (loss({**base, k: base[k] + step * way})
                   - loss({**base, k: base[k] - step * way})).item() / (2 * step)
            want = (v.grad.double() * way.double()).sum().item()
            assert abs(got - want) < 2e-3 * abs(want), (kind, k, got, want)


def test_second_derivative_is_refused():
    q = {k: v.to(DEV).requires_grad_() for k, v in _inputs(4, 32, F32, F32, True, True).items()}
    outs = _call(q, "layer")
    grads = [torch.ones_like(o, requires_grad=True) for o in outs]
    first = torch.autograd.grad(outs, list(q.values()), grads, create_graph=True)
    plain = torch.autograd.grad(_call(q, "layer"), list(q.values()), [g.detach() for g in grads])
    for a, b in zip(first, plain):
        assert torch.equal(a.detach(), b)
    with pytest.raises(RuntimeError, match="differentiable once"):
        first[1].sum().backward()


def test_empty_rows():
    q = {k: v.to(DEV).requires_grad_() for k, v in _inputs(4, 32, F32, F32, True, True).items()}
    for k in "xyz":
        q[k] = q[k].detach()[:0].requires_grad_()
    out, n = _call(q, "layer")
    assert out.shape == (0, 32) and n.shape == (0, 32)
    (out.sum() + n.sum()).backward()
    for k in ("weight", "bias", "scale", "next_weight", "next_bias"):
        assert torch.count_nonzero(q[k].grad) == 0


def test_same_bits_on_every_run_and_on_another_stream():
    q = _inputs(5000, 96, F32, BF16, True, True)
    dev = {k: v.to(DEV).requires_grad_() for k, v in q.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    runs = []
    for k in range(3):
        with torch.cuda.stream(side if k == 2 else torch.cuda.current_stream()):
            outs = _call(dev, "layer")
            runs.append([*outs, *torch.autograd.grad([o.float().square().sum() for o in outs],
                                                     list(dev.values()))])
    torch.cuda.synchronize()
    for other in runs[1:]:
        for a, b in zip(runs[0], other):
            assert torch.equal(a, b)


def test_refusals():
    q = {k: v.to(DEV) for k, v in _inputs(4, 32, F32, F32, True, True).items()}

    def call(**changed):
        p = {**q, **changed}
        return norm_gate_residual(p["x"], p["y"], p["z"], p["weight"], p["scale"], p["bias"],
                                  p["next_weight"], p["next_bias"], norm=p.get("norm", "rms"),
                                  eps=p.get("eps", 1e-5))

    with pytest.raises(AssertionError, match="y must have x's shape"):
        call(y=q["y"][:2])
    with pytest.raises(AssertionError, match="scale must be"):
        call(scale=q["scale"][:5])
    with pytest.raises(AssertionError, match="norm must be"):
        call(norm="batch")
    with pytest.raises(AssertionError, match="eps"):
        call(eps=-1.0)
    with pytest.raises(AssertionError, match="next_weight"):
        call(next_weight=None)
    with pytest.raises(TypeError, match="float16"):
        call(y=q["y"].half())
    with pytest.raises(AssertionError, match="devices"):
        call(scale=q["scale"].cpu())
    wide = torch.zeros(2, 4097, device=DEV)
    one = torch.ones(4097, device=DEV)
    with pytest.raises(AssertionError, match="at most 4096"):
        residual_norm(wide, one)
    with pytest.raises(AssertionError, match="dtype"):
        residual_norm(q["x"], q["weight"], dtype=torch.float16)


def test_forward_mode_derivatives_are_refused():
    """A tangent must not vanish without a word: the operators have no forward mode."""
    import torch.autograd.forward_ad as fwad
    q = {k: v.to(DEV) for k, v in _inputs(4, 16, F32, F32, True, True).items()}
    for name in q:
        for needs in (False, True):
            with fwad.dual_level():
                args = dict(q)
                if needs:
                    args["x"] = q["x"].clone().requires_grad_()
                args[name] = fwad.make_dual(args[name], torch.ones_like(args[name]))
                with pytest.raises(RuntimeError, match="forward"):
                    _call(args, "rms")
    with fwad.dual_level():
        dual = fwad.make_dual(q["x"], torch.ones_like(q["x"]))
        with pytest.raises(RuntimeError, match="forward"):
            residual_norm(dual, q["weight"])
    assert torch.isfinite(residual_norm(q["x"], q["weight"])).all()
