"""Gated linear recurrence on the GPU against the recurrence stepped in 64 bits,
with gradients from torch's autograd through that and from differences.

Tolerances (relative L2): every fp32 operation rounds by at most 2^-24 = 6e-8 and
the sigmoids, root and exponential are within a few of those; an error in a step's
decay acts over 1/(1 - a) steps and is random from step to step, so it grows by the
root of that, 32 at a = 0.999: 1e-5 holds with room. bf16 results are rounded once,
by at most half of 2^-7 of each value: 2^-8 + 1e-5 (their inputs are exact in 64 bits)."""

import math

import pytest
import torch

from tests.gpu_util import DEV, RTOL_F32, gen, rel_l2

pytestmark = pytest.mark.gpu

from mambaqc_b200 import _lib  # noqa: E402
from mambaqc_b200.kernels import gated_linear_scan, gated_linear_step  # noqa: E402

TOL_BF16 = 2.0 ** -8 + 1e-5
C = 8.0


def _tol(dt):
    return RTOL_F32 if dt == torch.float32 else TOL_BF16


def _ref(x, r, i, lam, h0=None, reset=None, sharpness=C):
    """The definition, step by step (torch autograd goes through it)."""
    log_a = -sharpness * torch.nn.functional.softplus(lam, threshold=200.0) * torch.sigmoid(r)
    h = torch.zeros_like(x[:, 0]) if h0 is None else h0
    ys = []
    for t in range(x.shape[1]):
        a = torch.exp(log_a[:, t])
        u = torch.sigmoid(i[:, t]) * x[:, t]
        new = a * h + torch.sqrt(-torch.expm1(2 * log_a[:, t])) * u
        if reset is not None:
            new = torch.where(reset[:, t, None], u, new)
        h = new
        ys.append(h)
    return torch.stack(ys, 1), h


def _inputs(b, t, d, dt, seed=0, with_h0=True, resets=0.0):
    g = gen(seed + 7 * b + 13 * t + 31 * d)
    x, r, i = (torch.randn(b, t, d, generator=g).to(dt) for _ in range(3))
    decay = 0.9 + 0.099 * torch.rand(d, generator=g)
    lam = torch.log(torch.expm1(-torch.log(decay) / C))
    h0 = torch.randn(b, d, generator=g) if with_h0 else None
    reset = torch.rand(b, t, generator=g) < resets if resets else None
    return x, r, i, lam, h0, reset


def _dev(t):
    return None if t is None else t.to(DEV)


SHAPES = [(1, 1, 1), (2, 3, 5), (1, 63, 64), (1, 64, 64), (2, 65, 66), (3, 130, 33),
          (1, 1025, 64), (2, 700, 100), (1, 2300, 7), (5, 257, 128), (1, 128, 1)]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("resets", [0.0, 0.05])
def test_forward_and_backward_match_64_bits(shape, dt, resets):
    b, t, d = shape
    args = _inputs(b, t, d, dt, with_h0=sum(shape) % 2 == 0, resets=resets)
    x, r, i, lam, h0, reset = args
    g = gen(3)
    dy = torch.randn(b, t, d, generator=g).to(dt)
    dhT = torch.randn(b, d, generator=g)

    leaves = [_dev(v).requires_grad_() for v in (x, r, i, lam)]
    h0d = None if h0 is None else _dev(h0).requires_grad_()
    y, hT = gated_linear_scan(*leaves, h0d, _dev(reset), return_final_state=True)
    torch.autograd.backward([y, hT], [_dev(dy), _dev(dhT)])

    ref = [v.double().requires_grad_() for v in (x, r, i, lam)]
    h0r = None if h0 is None else h0.double().requires_grad_()
    yr, hr = _ref(*ref, h0r, reset)
    torch.autograd.backward([yr, hr], [dy.double(), dhT.double()])

    assert y.dtype == dt and hT.dtype == torch.float32
    assert rel_l2(y, yr) < _tol(dt)
    assert rel_l2(hT, hr) < RTOL_F32
    for name, a, e in zip("xri", leaves, ref):
        assert rel_l2(a.grad, e.grad) < _tol(dt), name
    # a sum of b t terms that cancel by chance: judged against the terms' own size
    assert rel_l2(leaves[3].grad, ref[3].grad) < 10 * RTOL_F32, "Lambda"
    if h0 is not None:
        assert rel_l2(h0d.grad, h0r.grad) < RTOL_F32, "h0"
    # without a gradient the same kernel runs without keeping states: the same bits
    with torch.no_grad():
        y2 = gated_linear_scan(*[v.detach() for v in leaves], _dev(h0), _dev(reset))
    assert torch.equal(y, y2)


def test_many_channel_tiles_and_long_sequences():
    """More channel tiles than SMs, and a sequence of many tiles for one channel tile
    (each cluster size in turn: 1 .. 16 CTAs)."""
    for b, t, d in [(4, 70, 2600), (1, 20000, 40), (2, 400, 640), (40, 130, 512)]:
        x, r, i, lam, h0, _ = _inputs(b, t, d, torch.float32, seed=5)
        y, hT = gated_linear_scan(*map(_dev, (x, r, i, lam, h0)), return_final_state=True)
        yr, hr = _ref(*(v.to(DEV).double() for v in (x, r, i, lam, h0)))
        assert rel_l2(y, yr) < RTOL_F32, (b, t, d)
        assert rel_l2(hT, hr) < RTOL_F32, (b, t, d)


def test_long_memory():
    """Decay 0.99995: an error in a acts over 20000 steps. Half a unit in the last
    place of a (3e-8), random over the steps, gives sqrt(20000) 3e-8 = 4e-6; ten times
    that is allowed."""
    b, t, d = 1, 16384, 64
    g = gen(11)
    x, r, i = (torch.randn(b, t, d, generator=g) for _ in range(3))
    lam = torch.log(torch.expm1(torch.full((d,), 1e-4 / C)))
    y = gated_linear_scan(*map(_dev, (x, r, i, lam)))
    yr, _ = _ref(*(v.to(DEV).double() for v in (x, r, i, lam)))
    assert rel_l2(y, yr) < 4e-5


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_saturated_gates(dt):
    """Gates far out on both sides and rates from nothing to immediate forgetting:
    finite, and equal to 64 bits where those have a value."""
    vals = torch.tensor([-200.0, -90.0, -30.0, -3.0, 0.0, 3.0, 30.0, 90.0, 200.0])
    r, i = torch.meshgrid(vals, vals, indexing="ij")
    d = r.numel()
    t = 70
    r = r.reshape(1, 1, d).expand(1, t, d).to(dt).contiguous()
    i = i.reshape(1, 1, d).expand(1, t, d).to(dt).contiguous()
    x = torch.randn(1, t, d, generator=gen(1)).to(dt)
    for level in (-40.0, -5.0, 0.0, 40.0):
        lam = torch.full((d,), level)
        leaves = [_dev(v).requires_grad_() for v in (x, r, i, lam)]
        y, hT = gated_linear_scan(*leaves, return_final_state=True)
        y.float().sum().backward()
        yr, _ = _ref(*(v.double() for v in (x, r, i, lam)))
        assert rel_l2(y, yr) < _tol(dt), level
        for v in leaves:
            assert torch.isfinite(v.grad).all(), level


def test_infinities_and_nan():
    x, r, i, lam, h0, _ = _inputs(2, 150, 66, torch.float32, seed=2)
    clean = gated_linear_scan(*map(_dev, (x, r, i, lam, h0)))
    # +inf and -inf gates are the saturated ones
    r2, i2 = r.clone(), i.clone()
    r2[0, 10], r2[0, 11], i2[0, 12], i2[0, 13] = math.inf, -math.inf, math.inf, -math.inf
    y = gated_linear_scan(*map(_dev, (x, r2, i2, lam, h0)))
    yr, _ = _ref(*(v.double() for v in (x, r2, i2, lam, h0)))
    assert rel_l2(y, yr) < RTOL_F32
    # a NaN spoils its channel from its step on, nothing else; a reset ends that
    for which in range(3):
        v = [x.clone(), r.clone(), i.clone()]
        v[which][1, 40, 5] = math.nan
        y = gated_linear_scan(*map(_dev, v), _dev(lam), _dev(h0))
        bad = torch.isnan(y)
        want = torch.zeros_like(bad)
        want[1, 40:, 5] = True
        assert torch.equal(bad, want), which
        assert torch.equal(y[~bad], clean[~bad])
        reset = torch.zeros(2, 150, dtype=torch.bool)
        reset[1, 100] = True
        y = gated_linear_scan(*map(_dev, v), _dev(lam), _dev(h0), _dev(reset))
        want[1, 100:, 5] = False
        assert torch.equal(torch.isnan(y), want), which


def test_resets_split_a_packed_sequence():
    """Two documents packed in one sequence: as if each were run alone (the state at a
    reset is dropped, and with it the input's decay factor)."""
    x, r, i, lam, _, _ = _inputs(1, 200, 32, torch.float32, with_h0=False)
    for cut in (1, 63, 64, 65, 199):
        reset = torch.zeros(1, 200, dtype=torch.bool)
        reset[0, cut] = True
        y = gated_linear_scan(*map(_dev, (x, r, i, lam)), None, _dev(reset))
        first = gated_linear_scan(*(_dev(v[:, :cut]) for v in (x, r, i)), _dev(lam))
        alone = torch.zeros(1, 200 - cut, dtype=torch.bool)
        alone[0, 0] = True
        second = gated_linear_scan(*(_dev(v[:, cut:]) for v in (x, r, i)), _dev(lam), None,
                                   _dev(alone))
        assert rel_l2(y[:, :cut], first) < RTOL_F32
        assert rel_l2(y[:, cut:], second) < RTOL_F32
    every = torch.ones(1, 200, dtype=torch.bool)
    leaves = [_dev(v).requires_grad_() for v in (x, r, i, lam)]
    y = gated_linear_scan(*leaves, None, _dev(every))
    assert rel_l2(y, torch.sigmoid(i.double()) * x.double()) < RTOL_F32
    y.sum().backward()
    assert torch.count_nonzero(leaves[1].grad) == 0 and torch.count_nonzero(leaves[3].grad) == 0


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d,offset", [(64, 0), (64, 1), (33, 0), (50, 2)])
def test_strided_inputs_and_gradients(dt, d, offset):
    """x, r, i as column slices of one projection (odd offsets and widths leave the
    pair loads' alignment), every second sequence, and a gradient that is expanded."""
    b, t = 4, 90
    wide = torch.randn(b, t, 3 * d + offset, generator=gen(d)).to(dt)
    lam = torch.randn(d, generator=gen(1)) - 4

    def parts(w):
        w = w[::2]
        return [w[..., offset + k * d: offset + (k + 1) * d] for k in range(3)]

    w = _dev(wide).requires_grad_()
    lv = _dev(lam).requires_grad_()
    y = gated_linear_scan(*parts(w), lv)
    y.sum().backward()
    wr = wide.double().requires_grad_()
    lr = lam.double().requires_grad_()
    yr, _ = _ref(*parts(wr), lr)
    yr.sum().backward()
    assert rel_l2(y, yr) < _tol(dt)
    # dx, dr, di are rounded once, then summed into the slice's own place: no more
    assert rel_l2(w.grad, wr.grad) < _tol(dt)
    assert rel_l2(lv.grad, lr.grad) < 10 * RTOL_F32


def test_only_some_gradients():
    x, r, i, lam, h0, _ = map(_dev, _inputs(2, 100, 40, torch.float32))
    xr = x.clone().requires_grad_()
    y, hT = gated_linear_scan(xr, r, i, lam, h0, return_final_state=True)
    hT.sum().backward()                         # from the last state alone
    ref = [v.cpu().double() for v in (x, r, i, lam, h0)]
    ref[0].requires_grad_()
    _, hr = _ref(*ref)
    hr.sum().backward()
    assert rel_l2(xr.grad, ref[0].grad) < RTOL_F32
    hv = h0.clone().to(torch.bfloat16).requires_grad_()   # a bf16 start state
    lb = lam.to(torch.bfloat16).requires_grad_()
    y = gated_linear_scan(x, r, i, lb, hv)
    y.sum().backward()
    assert hv.grad.dtype == torch.bfloat16 and lb.grad.dtype == torch.bfloat16
    assert torch.isfinite(hv.grad).all() and torch.isfinite(lb.grad).all()


def test_gradient_against_differences():
    """Directional derivatives by central differences with step e in fp32: the
    truncation is e^2 / 6 of the third derivative (of order one here: 2e-5 at e =
    0.01), the outputs' rounding 1e-6 / (2 e) = 5e-5 of the loss's scale; 2e-3."""
    x, r, i, lam, h0, _ = _inputs(2, 150, 34, torch.float32)
    base = [_dev(v) for v in (x, r, i, lam, h0)]
    weight = _dev(torch.randn(x.shape, generator=gen(9)))

    def loss(v):
        return (gated_linear_scan(*v).double() * weight.double()).sum()

    leaves = [v.clone().requires_grad_() for v in base]
    (gated_linear_scan(*leaves) * weight).sum().backward()
    for k, v in enumerate(leaves):
        direction = torch.sign(v.grad)
        step = 0.01
        up = [u + step * direction if j == k else u for j, u in enumerate(base)]
        down = [u - step * direction if j == k else u for j, u in enumerate(base)]
        got = (loss(up) - loss(down)).item() / (2 * step)
        want = (v.grad.double() * direction.double()).sum().item()
        assert abs(got - want) < 2e-3 * abs(want), (k, got, want)


def test_second_derivative_is_refused():
    """The first derivative under create_graph is right; taking another from it raises."""
    x, r, i, lam, h0, _ = map(_dev, _inputs(2, 70, 8, torch.float32))
    leaves = [v.clone().requires_grad_() for v in (x, r, i, lam, h0)]
    plain = torch.autograd.grad(gated_linear_scan(*leaves).sum(), leaves)
    y = gated_linear_scan(*leaves)
    g = torch.ones_like(y, requires_grad=True)
    first = torch.autograd.grad(y, leaves, g, create_graph=True)
    for a, b in zip(first, plain):
        assert torch.equal(a.detach(), b)
    with pytest.raises(RuntimeError, match="differentiable once"):
        first[0].sum().backward()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,d", [(1, 1), (3, 33), (8, 64), (64, 1536)])
def test_step_matches_scan(dt, b, d):
    t = 5
    x, r, i, lam, h0, _ = map(_dev, _inputs(b, t, d, dt))
    y, hT = gated_linear_scan(x, r, i, lam, h0, return_final_state=True)
    h = h0.clone()
    for k in range(t):
        out = gated_linear_step(x[:, k], r[:, k], i[:, k], lam, h)
        assert out.dtype == dt
        # the same formulas in fp32, the products of a tile in another order
        assert rel_l2(out, y[:, k]) < (RTOL_F32 if dt == torch.float32 else 2.0 ** -8)
    assert rel_l2(h, hT) < RTOL_F32
    keep = torch.empty_like(x[:, 0].contiguous())
    got = gated_linear_step(x[:, 0], r[:, 0], i[:, 0], lam, h0.clone(), out=keep)
    assert got is keep


def test_empty_and_single_steps():
    lam = torch.zeros(8, device=DEV)
    h0 = torch.randn(2, 8, device=DEV)
    e = torch.empty(2, 0, 8, device=DEV)
    y, hT = gated_linear_scan(e, e, e, lam, h0, return_final_state=True)
    assert y.shape == (2, 0, 8) and torch.equal(hT, h0)
    _, hT = gated_linear_scan(e, e, e, lam, return_final_state=True)
    assert torch.count_nonzero(hT) == 0
    hv, lv = h0.clone().requires_grad_(), lam.clone().requires_grad_()
    _, hT = gated_linear_scan(e, e, e, lv, hv, return_final_state=True)
    (hT * 3).sum().backward()
    assert torch.equal(hv.grad, torch.full_like(hv, 3.0)) and torch.count_nonzero(lv.grad) == 0
    e = torch.empty(0, 5, 8, device=DEV)
    y, hT = gated_linear_scan(e, e, e, lam, return_final_state=True)
    assert y.shape == (0, 5, 8) and hT.shape == (0, 8)
    assert gated_linear_step(e[:, 0], e[:, 0], e[:, 0], lam, e[:, 0].contiguous()).shape == (0, 8)


def test_same_bits_on_every_run_and_on_another_stream():
    args = [_dev(v) for v in _inputs(3, 500, 130, torch.bfloat16)[:4]]
    leaves = [v.requires_grad_() for v in args]
    runs = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for k in range(3):
        with torch.cuda.stream(side if k == 2 else torch.cuda.current_stream()):
            y = gated_linear_scan(*leaves)
            runs.append([y.detach(), *torch.autograd.grad(y.float().square().sum(), leaves)])
    torch.cuda.synchronize()
    for other in runs[1:]:
        for a, b in zip(runs[0], other):
            assert torch.equal(a, b)


def test_refusals():
    x, r, i, lam, h0, _ = map(_dev, _inputs(2, 6, 8, torch.float32))
    with pytest.raises(AssertionError, match="one shape"):
        gated_linear_scan(x, r[:, :5], i, lam)
    with pytest.raises(AssertionError, match="one dtype"):
        gated_linear_scan(x, r.bfloat16(), i, lam)
    with pytest.raises(AssertionError, match="Lambda"):
        gated_linear_scan(x, r, i, lam[:4])
    with pytest.raises(AssertionError, match="state"):
        gated_linear_scan(x, r, i, lam, h0[:1])
    with pytest.raises(AssertionError, match="reset"):
        gated_linear_scan(x, r, i, lam, h0, torch.zeros(2, 6, device=DEV))
    with pytest.raises(AssertionError, match="sharpness"):
        gated_linear_scan(x, r, i, lam, sharpness=0.0)
    with pytest.raises(TypeError, match="float16"):
        gated_linear_scan(x.half(), r.half(), i.half(), lam)
    with pytest.raises(RuntimeError, match="CUDA"):
        gated_linear_scan(x.cpu(), r.cpu(), i.cpu(), lam.cpu())
    with pytest.raises(AssertionError, match="contiguous float32"):
        gated_linear_step(x[:, 0], r[:, 0], i[:, 0], lam, h0.bfloat16())
    with pytest.raises(AssertionError, match="out"):
        gated_linear_step(x[:, 0], r[:, 0], i[:, 0], lam, h0, out=h0[:1])


# (batch, channels) whose sequences go one CTA each, and to clusters of CTAs
ONE_CTA, CLUSTERS = (160, 256), (1, 8)


@pytest.mark.parametrize("b,d", [ONE_CTA, CLUSTERS])
@pytest.mark.parametrize("t_nan,t_reset", [(70, 100), (72, 75), (75, 72), (74, 74), (100, 70), (30, 190)])
def test_reset_and_nan_in_one_tile(b, d, t_nan, t_reset):
    """A NaN gate and a reset, in one run of steps or two runs of a tile: the NaN
    reaches from its step to the next reset in y, and the gradients of the other
    document and of other channels are those of clean inputs, bit for bit."""
    t, ch = 200, 5
    x, r, i, lam, h0, _ = _inputs(b, t, d, torch.float32, seed=4)
    reset = torch.zeros(b, t, dtype=torch.bool)
    reset[:, t_reset] = True

    def run(gate):
        leaves = [_dev(v).requires_grad_() for v in (x, gate, i, lam, h0)]
        y, hT = gated_linear_scan(*leaves, _dev(reset), return_final_state=True)
        return y.detach(), hT.detach(), torch.autograd.grad([y.sum() + hT.sum()], leaves)

    y, hT, grads = run(r)
    bad_r = r.clone()
    bad_r[0, t_nan, ch] = math.nan
    y2, hT2, grads2 = run(bad_r)
    bad = torch.zeros(b, t, d, dtype=torch.bool, device=DEV)
    last = t_reset if t_reset >= t_nan else t
    bad[0, t_nan:last, ch] = True
    assert torch.equal(torch.isnan(y2), bad)
    assert torch.equal(y2[~bad], y[~bad])
    assert torch.isnan(hT2).sum() == (t_reset < t_nan)
    # the document without the NaN, in this channel; every other channel whole
    clean = torch.ones(b, t, d, dtype=torch.bool, device=DEV)
    clean[0, :, ch] = False
    other = slice(t_reset, t) if t_nan < t_reset else slice(0, t_reset)
    clean[0, other, ch] = True
    if t_nan == t_reset:        # the step's own decay is not used at all
        clean[:] = True
        assert torch.isnan(grads2[1][0, t_nan, ch]) or grads2[1][0, t_nan, ch] == 0
        clean[0, t_nan, ch] = False
    for a, e in zip(grads2[:3], grads[:3]):
        assert torch.equal(a[clean], e[clean])
    keep = torch.arange(d, device=DEV) != ch
    assert torch.equal(grads2[3][keep], grads[3][keep])
    h0_clean = torch.ones(b, d, dtype=torch.bool, device=DEV)
    h0_clean[0, ch] = t_nan >= t_reset
    assert torch.equal(grads2[4][h0_clean], grads[4][h0_clean])


@pytest.mark.parametrize("b,d", [ONE_CTA, CLUSTERS])
def test_nan_outlives_vanishing_decays(b, d):
    """Decays that multiply to nothing over a run are no reset: a NaN state stays one
    in a call with ``reset``, and a call whose resets are all False has the bits of one
    without."""
    t = 200
    x, r, i, _, h0, reset = _inputs(b, t, d, torch.float32, seed=6, resets=1e-9)
    assert not reset.any()
    for rate in (0.1, 2.0, 30.0):
        lam = torch.log(torch.expm1(torch.full((d,), rate / C)))
        h0 = h0.clone()
        h0[0, 3] = math.nan
        args = [_dev(v) for v in (x, r, i, lam, h0)]
        y = gated_linear_scan(*args)
        y2, hT = gated_linear_scan(*args, _dev(reset), return_final_state=True)
        assert torch.isnan(y2[0, :, 3]).all() and torch.isnan(hT[0, 3]), rate
        clean = torch.ones(b, t, d, dtype=torch.bool, device=DEV)
        clean[0, :, 3] = False
        assert torch.equal(y[clean], y2[clean])
        # backward: a NaN that arrives from the end reaches the start
        leaves = [v.clone().requires_grad_() for v in args[:4]] + [_dev(torch.zeros(b, d)).requires_grad_()]
        _, hT = gated_linear_scan(*leaves, _dev(reset), return_final_state=True)
        dhT = torch.ones_like(hT)
        dhT[0, 3] = math.nan
        dh0 = torch.autograd.grad(hT, leaves[4], dhT)[0]
        assert torch.isnan(dh0[0, 3]) and torch.isnan(dh0).sum() == 1, rate


# Products of decays far from 1. Every step's -log a is a product of three fp32 factors:
# the rate's softplus (log1pf and expf: 3 units of 6e-8), the sigmoid (its exponential's
# argument and value, its reciprocal: 5) and two roundings; added up over the steps with
# a rounding each, its relative error is below 1e-6. So a product exp(-S) is within
# 1e-6 S of its value, and each of up to one join for every 8 steps rounds by 1e-7 more.
def _decay_bound(total, steps):
    return 1e-6 * total + 1e-7 * (steps / 8 + 10)


@pytest.mark.parametrize("b,d", [ONE_CTA, CLUSTERS])
@pytest.mark.parametrize("t", [1, 40, 200, 1500])
@pytest.mark.parametrize("decay", [0.999, 0.9, 0.7, 0.6, 0.5, 0.1, 3e-7])
def test_forgotten_state_keeps_its_digits(b, d, t, decay):
    """With x = 0 the state is h0 times the product of the decays: each y and the last
    state against 64 bits as long as fp32 has the value, and the gradient of h0 from the
    last state alone, which is the product itself."""
    if b > 1 and t > 200:
        t = 300
    g = gen(t)
    rate = -math.log(decay)
    lam = torch.full((d,), math.log(math.expm1(rate / C)))
    r = 3.0 + torch.rand(b, t, d, generator=g)
    x = torch.zeros(b, t, d)
    h0 = 1e6 * (1 + torch.rand(b, d, generator=g))
    leaf = _dev(h0).requires_grad_()
    y, hT = gated_linear_scan(_dev(x), _dev(r), _dev(x), _dev(lam), leaf, return_final_state=True)
    dh0 = torch.autograd.grad(hT.sum(), leaf)[0]
    soft = torch.nn.functional.softplus(lam.to(DEV).double(), threshold=200.0)
    total = torch.cumsum(C * soft * torch.sigmoid(r.to(DEV).double()), 1)
    want = torch.exp(-total) * h0.to(DEV).double()[:, None]
    steps = torch.arange(1, t + 1, device=DEV)[None, :, None]
    bound = _decay_bound(total, steps)
    held = want > 1e-30             # well inside fp32; below it only "next to nothing"
    off = (y.double() - want).abs()
    assert (off <= bound * want)[held].all(), (off / want / bound)[held].max()
    assert (y.abs()[~held] <= 1.1e-30).all()
    last = want[:, -1]
    off = (hT.double() - last).abs()
    assert torch.where(last > 1e-30, off <= bound[:, -1] * last, hT.abs() <= 1.1e-30).all()
    last = torch.exp(-total[:, -1])
    off = (dh0.double() - last).abs()
    assert torch.where(last > 1e-30, off <= bound[:, -1] * last, dh0.abs() <= 1.1e-30).all()


@pytest.mark.parametrize("shape", [(1, 150, 64), (2, 700, 100), (160, 90, 256)])
def test_gradients_under_fast_decay(shape):
    """Rates up to 18 a step (decays down to 1e-8), a large start state, resets: every
    channel's gradients against 64 bits. An error of 1e-6 of -log a is 1e-6 L of the
    decay that dr, dLambda and the carried gradient are proportional to."""
    b, t, d = shape
    x, r, i, _, h0, reset = _inputs(b, t, d, torch.float32, seed=8, resets=0.02)
    rates = torch.tensor([0.2, 1.0, 2.5, 5.0, 10.0, 15.0, 18.0, 30.0])[torch.arange(d) % 8]
    lam = torch.where(rates / C > 0.1, torch.log(torch.expm1(rates / C)), torch.log(rates / C))
    h0 = 1e4 * h0
    g = gen(2)
    dy, dhT = torch.randn(b, t, d, generator=g), torch.randn(b, d, generator=g)
    out = []
    for to in (lambda v: v.to(DEV), lambda v: v.to(DEV).double()):
        leaves = [to(v).requires_grad_() for v in (x, r, i, lam, h0)]
        f = gated_linear_scan if to(x).dtype == torch.float32 else None
        if f is not None:
            y, hT = f(*leaves, _dev(reset), return_final_state=True)
        else:
            y, hT = _ref(*leaves, _dev(reset))
        out.append([y, hT, *torch.autograd.grad([y, hT], leaves, [to(dy), to(dhT)])])
    soft = C * torch.nn.functional.softplus(lam.to(DEV).double(), threshold=200.0)
    bound = 1e-5 + 2e-6 * soft
    for name, got, want in zip(("y", "hT", "x", "r", "i", "Lambda", "h0"), *out):
        got, want = got.double().reshape(-1, d), want.reshape(-1, d)
        size = want.square().sum(0).sqrt()
        off = (got - want).square().sum(0).sqrt()
        # dLambda is one cancelling sum a channel, as in the test of slow decays: ten times
        room = bound * size * (10 if name == "Lambda" else 1) + 1e-30
        assert (off <= room).all(), (name, (off / room).max().item(), (off / room).argmax().item())


@pytest.mark.parametrize("b,d", [ONE_CTA, CLUSTERS])
@pytest.mark.parametrize("rate", [0.05, 0.9, 6.0, 18.0])
@pytest.mark.parametrize("masked", [False, True])
def test_infinite_states_stay_infinite(b, d, rate, masked):
    """An infinite start state or input keeps its sign over runs and tiles, becomes NaN
    where it meets the other infinity, and ends at a reset: the places of infinities
    and NaN are those of 64 bits. An infinite gradient reaches the start state."""
    t = 200
    x, r, i, _, h0, _ = _inputs(b, t, d, torch.float32, seed=9)
    lam = torch.log(torch.expm1(torch.full((d,), rate / C)))
    h0[0, 0], h0[0, 1] = math.inf, -math.inf
    x[0, 70, 2], x[0, 3, 3] = math.inf, -math.inf
    x[0, 20, 4], x[0, 150, 4] = math.inf, -math.inf
    reset = torch.zeros(b, t, dtype=torch.bool) if masked else None
    if masked:
        reset[:, 120] = True
    leaf = _dev(h0).requires_grad_()
    y, hT = gated_linear_scan(*map(_dev, (x, r, i, lam)), leaf, _dev(reset), return_final_state=True)
    yr, hr = _ref(*(v.to(DEV).double() for v in (x, r, i, lam, h0)), _dev(reset))
    for got, want in ((y, yr), (hT, hr)):
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.isposinf(got), torch.isposinf(want))
        assert torch.equal(torch.isneginf(got), torch.isneginf(want))
    dhT = torch.ones_like(hT)
    dhT[0, 6], dhT[0, 7] = math.inf, -math.inf
    dh0 = torch.autograd.grad(hT, leaf, dhT)[0]
    if not masked:
        assert torch.isposinf(dh0[0, 6]) and torch.isneginf(dh0[0, 7])
        assert torch.isfinite(dh0).sum() == dh0.numel() - 2
    else:
        assert torch.count_nonzero(dh0) == 0


@pytest.mark.parametrize("rate", [0.3, 2.0, 10.0, 15.0, 30.0])
def test_step_keeps_the_digits_of_a_fast_decay(rate):
    d = 37
    lam = torch.log(torch.expm1(torch.full((d,), rate / C)))
    r = torch.linspace(-2, 8, d)[None]
    h0 = torch.full((1, d), 1e6)
    h, zero = _dev(h0), torch.zeros(1, d, device=DEV)
    gated_linear_step(zero, _dev(r), zero, _dev(lam), h)
    total = C * torch.nn.functional.softplus(lam.double(), threshold=200.0) * torch.sigmoid(r.double())
    want = 1e6 * torch.exp(-total)
    assert ((h.cpu().double() / want - 1).abs() <= _decay_bound(total, 1)).all()


def test_device_timeout_is_reported_and_context_survives(monkeypatch):
    """A wait for the cluster's other CTAs that is made to give up (no polls) reports to
    the status word, forward and backward, and each call raises by itself under
    MAMBAQC_B200_SYNC_CHECK=1; calls after it are right."""
    monkeypatch.delenv("MAMBAQC_B200_SYNC_CHECK", raising=False)
    x, r, i, lam, h0, _ = _inputs(1, 300, 8, torch.float32)     # one sequence: a cluster
    dev = torch.device(DEV)
    _lib.check_device_status(dev)
    leaves = [_dev(v).requires_grad_() for v in (x, r, i, lam, h0)]

    def scan(**kw):
        return gated_linear_scan(*leaves, **kw)

    y = scan(wait_poll_limit=0)
    with pytest.raises(RuntimeError, match="timed out"):
        _lib.check_device_status(dev)
    torch.autograd.grad(y.sum(), leaves)
    with pytest.raises(RuntimeError, match="timed out"):
        _lib.check_device_status(dev)
    late = scan(wait_poll_limit=0)
    with pytest.raises(RuntimeError, match="timed out"):
        _lib.check_device_status(dev)
    monkeypatch.setenv("MAMBAQC_B200_SYNC_CHECK", "1")
    with pytest.raises(RuntimeError, match="timed out"):
        torch.autograd.grad(late.sum(), leaves)
    with pytest.raises(RuntimeError, match="timed out"):
        scan(wait_poll_limit=0)
    with torch.no_grad(), pytest.raises(RuntimeError, match="timed out"):
        scan(wait_poll_limit=0)
    with pytest.raises(AssertionError, match="wait_poll_limit"):
        scan(wait_poll_limit=7)
    y = scan()                                                  # the check itself passes
    grads = torch.autograd.grad(y.sum(), leaves)
    ref = [v.double().requires_grad_() for v in (x, r, i, lam, h0)]
    yr, _ = _ref(*ref)
    want = torch.autograd.grad(yr.sum(), ref)
    assert rel_l2(y, yr) < RTOL_F32
    for a, e in zip(grads, want):
        assert rel_l2(a, e) < 10 * RTOL_F32
    _lib.check_device_status(dev)


def test_forward_mode_derivatives_are_refused():
    """A tangent must not vanish without a word: the operator has no forward mode."""
    import torch.autograd.forward_ad as fwad
    x, r, i, lam, h0, _ = map(_dev, _inputs(2, 6, 8, torch.float32))
    for k in range(5):
        for needs in (False, True):
            with fwad.dual_level():
                args = [x, r, i, lam, h0]
                if needs:
                    args[0] = x.clone().requires_grad_()
                args[k] = fwad.make_dual(args[k], torch.ones_like(args[k]))
                with pytest.raises(RuntimeError, match="forward"):
                    gated_linear_scan(*args, return_final_state=True)
                if k < 4 and not needs:
                    with pytest.raises(RuntimeError, match="forward"):
                        step = [x[:, 0], r[:, 0], i[:, 0], lam]
                        step[k] = fwad.make_dual(step[k], torch.ones_like(step[k]))
                        gated_linear_step(*step, h0.clone())
    # outside a level nothing changes
    assert torch.isfinite(gated_linear_scan(x, r, i, lam, h0)).all()


def test_step_advances_the_version_counters():
    """A backward through a graph that saved the state before a step raises, as after
    torch's own operations in place."""
    x, r, i, lam, h0, _ = map(_dev, _inputs(2, 1, 8, torch.float32))
    x, r, i = x[:, 0], r[:, 0], i[:, 0]
    w = torch.ones_like(h0, requires_grad=True)
    out = torch.empty_like(x)
    loss = (w * h0).sum() + (w * out).sum()
    before = h0._version, out._version, x._version
    gated_linear_step(x, r, i, lam, h0, out=out)
    assert (h0._version, out._version, x._version) == (before[0] + 1, before[1] + 1, before[2])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():                    # states of inference mode have no count
        state = h0.clone()
        gated_linear_step(x.detach(), r, i, lam, state)
    gated_linear_step(x, r, i, lam, state)
