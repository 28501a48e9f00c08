"""AdamW over a list of tensors on the GPU, moments in 32 and in 8 bits, against the
update in 64 bits and against torch.optim.AdamW.

Tolerances. 32 bits: a step rounds each of p, m, v a handful of times by 6e-8:
relative L2 1e-6 a step. 8 bits: the rounded moments are a function with steps, so a
last-place difference before rounding (6e-8 of the value against a rounding step of
1/32 or 1/16 of it) lands on the other side in about 4e-6 of the values: codes may
differ in 1e-4 of them, by one step each. bf16 parameters: the same, with a
rounding step of 2^-8."""

import pytest
import torch

from tests.gpu_util import DEV, gen, rel_l2

pytestmark = pytest.mark.gpu

from mambaqc_b200.kernels import adamw_moments, adamw_step, grad_norm  # noqa: E402
from mambaqc_b200.models import QuaternionMamba2  # noqa: E402
from mambaqc_b200.optim import AdamW  # noqa: E402
from mambaqc_b200.training import train_step  # noqa: E402

F32, BF16, U8 = torch.float32, torch.bfloat16, torch.uint8
BLOCK = 256
HYPER = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


# ---------------------------------------------------------------- 64-bit oracle

def _mix(h):
    h = h * 0x6A09E667 & 0xFFFFFFFF
    h = h ^ (h >> 15)
    h = h * 0xBB67AE85 & 0xFFFFFFFF
    return h ^ (h >> 13)


def _noise(n, seed, step, ordinal):
    key = _mix(_mix(_mix(seed) ^ step) ^ ordinal)
    return _mix(torch.arange(n, dtype=torch.int64) ^ key)


def _values(code, e, fraction):
    c = code.cpu().long()
    e = e.cpu().double().repeat_interleave(BLOCK)[: c.numel()]
    mag = c % 128 if fraction == 3 else c
    v = torch.exp2(e - 142 + (mag >> fraction)) * (1 + (mag % (1 << fraction)) / (1 << fraction))
    v = torch.where(mag > 0, v, 0.0)
    return torch.where(c > 127, -v, v) if fraction == 3 else v


def _rounded(x, noise, fraction, e, carry):
    """Values of x as 8 bits hold them under the block exponents e, which have to be
    those of the blocks' largest values (to 1e-6: at a power of two the fp32 value may
    lie on its other side)."""
    n = x.numel()
    blocks = -(-n // BLOCK)
    pad = torch.zeros(blocks * BLOCK, dtype=torch.float64)
    pad[:n] = x.abs()
    top = pad.view(blocks, BLOCK).amax(1)
    e = e.cpu().double()
    least, last = 1 + 2.0 ** -fraction, 2 - 2.0 ** -fraction
    high = torch.exp2(e - 127) * (last if carry else 2.0)
    assert (top <= high * (1 + 1e-6)).all()
    assert ((top >= high / 2 * (1 - 1e-6)) | (e == 16)).all()
    unit = torch.exp2(e - 142).repeat_interleave(BLOCK)[:n]
    w, r = x.abs() / unit, noise.double() / 65536
    grid = torch.exp2(torch.floor(torch.log2(w.clamp(min=least))) - fraction)
    big = torch.floor(w / grid + r) * grid
    big = big.clamp(max=2.0 ** 15 * last)
    small = least * ((w > 0) if fraction == 4 else (w > r * least)).double()
    return torch.where(w < least, small, big) * unit * torch.sign(x)


def _oracle(p, g, m, v, step, clip=1.0, lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1):
    b1, b2 = betas
    g = g.double() * clip
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    hat = m / (1 - b1 ** step) / ((v / (1 - b2 ** step)).sqrt() + eps)
    return p.double() * (1 - lr * weight_decay) - lr * hat, m, v


def _state(sizes, bits):
    if bits == 32:
        return [torch.zeros(n, device=DEV) for n in sizes], \
               [torch.zeros(n, device=DEV) for n in sizes], None
    m = [torch.zeros(n, dtype=U8, device=DEV) for n in sizes]
    v = [torch.zeros(n, dtype=U8, device=DEV) for n in sizes]
    e = [[torch.zeros(-(-n // BLOCK), dtype=U8, device=DEV) for n in sizes] for _ in range(2)]
    return m, v, tuple(e)


SIZES = [1, 2, 3, 5, 31, 255, 256, 257, 1000, 2047, 2048, 2049, 70001]


# ----------------------------------------------------------------- 32-bit moments

@pytest.mark.parametrize("pt,gt", [(F32, F32), (F32, BF16), (BF16, BF16), (BF16, F32)])
def test_32_bit_steps_match_64_bits(pt, gt):
    g = gen(1)
    params = [torch.randn(n, generator=g).to(pt) for n in SIZES]
    m, v, _ = _state(SIZES, 32)
    dev = [p.to(DEV) for p in params]
    rp = [p.double() for p in params]
    rm = [torch.zeros(n, dtype=torch.float64) for n in SIZES]
    rv = [torch.zeros(n, dtype=torch.float64) for n in SIZES]
    for step in range(1, 4):
        grads = [(10.0 ** (-k % 5) * torch.randn(n, generator=g)).to(gt)
                 for k, n in enumerate(SIZES)]
        before = [p.cpu().double() for p in dev]
        adamw_step(dev, [x.to(DEV) for x in grads], m, v, step=step, seed=3, **HYPER)
        for k in range(len(SIZES)):
            start = rp[k] if pt == F32 else before[k]   # bf16: from what the step read
            rp[k], rm[k], rv[k] = _oracle(start, grads[k], rm[k], rv[k], step)
            assert rel_l2(m[k], rm[k]) < step * 1e-6 and rel_l2(v[k], rv[k]) < step * 1e-6
            if pt == F32:
                assert rel_l2(dev[k], rp[k]) < step * 1e-6
            else:   # one of the two bf16 neighbours of the exact value
                got = dev[k].cpu().double()
                assert ((got - rp[k]).abs() <= rp[k].abs() * 2.0 ** -7).all()


def test_matches_torch_adamw_over_many_steps():
    g = gen(2)
    ours = [torch.nn.Parameter(torch.randn(s, generator=g).to(DEV)) for s in ((33, 7), (5,), (300,))]
    theirs = [torch.nn.Parameter(p.detach().clone()) for p in ours]
    a = AdamW([{"params": ours[:1]}, {"params": ours[1:], "lr": 3e-3, "weight_decay": 0.0}],
              lr=1e-2, weight_decay=0.2)
    b = torch.optim.AdamW([{"params": theirs[:1]},
                           {"params": theirs[1:], "lr": 3e-3, "weight_decay": 0.0}],
                          lr=1e-2, weight_decay=0.2)
    for step in range(30):
        for p, q in zip(ours, theirs):
            p.grad = torch.randn(p.shape, generator=g).to(DEV)
            q.grad = p.grad.clone()
        if step % 7 == 3:           # a tensor without a gradient now and then
            ours[1].grad = theirs[1].grad = None
        a.step(max_grad_norm=5.0)
        want = torch.nn.utils.clip_grad_norm_(theirs, 5.0)
        b.step()
        assert abs(a.grad_norm.item() - want.item()) < 1e-6 * want.item()
    for p, q in zip(ours, theirs):
        assert rel_l2(p, q) < 30e-6
    assert a.state[ours[1]]["step"] == 26


# ------------------------------------------------------------------ 8-bit moments

def _close_codes(got, want, noise_scale):
    """Equal but for 1e-4 of the values (at least one), those within one step."""
    differ = got != want
    assert differ.sum().item() <= max(1, 1e-4 * got.numel()), differ.sum()
    assert ((got - want).abs() <= want.abs() * noise_scale + 1e-300)[differ].all()


@pytest.mark.parametrize("carry", [False, True])
@pytest.mark.parametrize("pt,gt", [(F32, F32), (F32, BF16), (BF16, BF16)])
def test_8_bit_steps_match_64_bits(pt, gt, carry):
    """Each step from the state the step before left, so that a value that landed on
    the other side does not add up."""
    g = gen(4)
    dev = [torch.randn(n, generator=g).to(pt).to(DEV) for n in SIZES]
    m, v, e = _state(SIZES, 8)
    spread = [torch.exp(3 * torch.randn(n, generator=g)) for n in SIZES]  # within a block too
    for step in range(1, 5):
        grads = [(s * torch.randn(n, generator=g)).to(gt) for s, n in zip(spread, SIZES)]
        before = [(p.cpu().double(), _values(a, b, 3), _values(c, d, 4).square())
                  for p, a, b, c, d in zip(dev, m, e[0], v, e[1])]
        adamw_step(dev, [x.to(DEV) for x in grads], m, v, step=step, exponents=e, seed=77,
                   carry=carry, **HYPER)
        ms, roots = adamw_moments(m, v, e)
        for k, n in enumerate(SIZES):
            p0, m0, v0 = before[k]
            rp, rm, rv = _oracle(p0, grads[k], m0, v0, step)
            if pt == F32:
                assert rel_l2(dev[k], rp) < 1e-6
            noise = _noise(n, 77, step, k)
            got_m, got_r = _values(m[k], e[0][k], 3), _values(v[k], e[1][k], 4)
            _close_codes(got_m, _rounded(rm, noise >> 16, 3, e[0][k], carry), 2.0 ** -3)
            _close_codes(got_r, _rounded(rv.sqrt(), noise & 0xFFFF, 4, e[1][k], carry), 2.0 ** -4)
            # the values handed out are the codes' own
            assert torch.equal(ms[k].cpu().double(), got_m)
            assert torch.equal(roots[k].cpu().double(), got_r)


def test_8_bit_rounding_is_unbiased_where_nearest_would_freeze():
    """Under a constant gradient v goes from 0.25 g^2 to g^2; a step moves it by less
    than half a rounding step, so rounding to nearest would leave it at its start.
    Over n = 65536 elements the mean of v is within 5 standard errors of the 32-bit
    value; a root's spread is at most 1/16 of it a step and 15 % in all."""
    n, steps = 65536, 1500
    grad = torch.full((n,), 0.02, device=DEV)
    p = torch.zeros(n, device=DEV)
    m, v, e = _state([n], 8)
    # roots of 0.01: exponent of 0.01, code 15 << 4 | fraction
    e[1][0].fill_(127 - 7)
    v[0].fill_((15 << 4) | 4)                      # 2^-7 * 1.25 = 0.009766
    start = adamw_moments(m, v, e)[1][0].float()[0].item()
    assert abs(start - 0.009766) < 1e-5
    for step in range(1, steps + 1):
        adamw_step([p], [grad], m, v, step=step, lr=0.0, weight_decay=0.0, exponents=e, seed=5,
                   carry=True)
    want = 0.02 ** 2 - (0.02 ** 2 - start ** 2) * 0.999 ** steps
    root = adamw_moments(m, v, e)[1][0].double()
    # sqrt is concave: the mean of the roots, each unbiased, follows sqrt(v) step by step
    assert abs(root.mean().item() / want ** 0.5 - 1) < 0.02
    assert root.std().item() / want ** 0.5 < 0.2
    mean = adamw_moments(m, v, e)[0][0].double().mean().item()
    assert abs(mean / 0.02 - 1) < 5 * 0.07 / n ** 0.5 + 1e-3


def test_8_bit_root_above_zero_stays_above_zero():
    """One large value in the block: the small ones' roots keep a code, so their step
    stays bounded where m is kept."""
    n = 256
    grad = torch.full((n,), 1e-9, device=DEV)
    grad[7] = 1e3
    p = torch.zeros(n, device=DEV)
    m, v, e = _state([n], 8)
    for step in range(1, 6):
        adamw_step([p], [grad], m, v, step=step, lr=1e-3, weight_decay=0.0, exponents=e, seed=1)
    assert (adamw_moments(m, v, e)[1][0] > 0).all()
    assert torch.isfinite(p).all() and p.abs().max().item() < 5 * 1e-3 * 1.2


def test_8_bit_zero_and_extreme_gradients():
    n = 300
    for size in (0.0, 1e-38, 1e-30, 1e18, 3e38):
        p = torch.ones(n, device=DEV)
        grad = torch.full((n,), size, device=DEV)
        m, v, e = _state([n], 8)
        adamw_step([p], [grad], m, v, step=1, lr=1e-3, weight_decay=0.0, exponents=e, seed=1)
        if size == 0.0:
            assert torch.equal(p, torch.ones_like(p)) and torch.count_nonzero(m[0]) == 0
        if size <= 1e18:
            assert torch.isfinite(p).all()
            assert torch.isfinite(torch.cat(sum(adamw_moments(m, v, e), []))).all()


def test_8_bit_block_with_nan_is_marked():
    n = 600
    p = torch.ones(n, device=DEV)
    m, v, e = _state([n], 8)
    grad = torch.ones(n, device=DEV)
    grad[300], grad[599] = float("nan"), float("inf")
    adamw_step([p], [grad], m, v, step=1, lr=1e-3, exponents=e)
    bad = torch.isnan(p)
    assert bad[300] and bad[599] and bad.sum() == 2
    assert e[0][0].tolist()[1:] == [255, 255] and e[0][0][0] != 255
    roots = adamw_moments(m, v, e)[1][0]
    assert torch.isfinite(roots[:256]).all() and torch.isnan(roots[256:]).all()
    adamw_step([p], [torch.ones_like(p)], m, v, step=2, lr=1e-3, exponents=e)
    assert torch.isfinite(p[:256]).all() and torch.isnan(p[256:]).all()


# ------------------------------------------------------------- lists and layouts

@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_equal_one_at_a_time(bits):
    """More tensors than one launch takes, empty ones among them, one call or one each:
    the same bits."""
    sizes = [(37 * k) % 1500 for k in range(150)] + [70000]
    g = gen(6)
    start = [torch.randn(n, generator=g).to(DEV) for n in sizes]
    grads = [torch.randn(n, generator=g).to(DEV) for n in sizes]
    runs = []
    for together in (True, False):
        p = [t.clone() for t in start]
        m, v, e = _state(sizes, bits)
        for step in (1, 2):
            if together:
                adamw_step(p, grads, m, v, step=step, exponents=e, seed=9, **HYPER)
                continue
            for k in range(len(sizes)):
                one = None if e is None else ([e[0][k]], [e[1][k]])
                adamw_step([p[k]], [grads[k]], [m[k]], [v[k]], step=step, exponents=one, seed=9,
                           ordinals=[k], **HYPER)
        runs.append(p + m + v + ([] if e is None else e[0] + e[1]))
    for a, b in zip(*runs):
        assert torch.equal(a, b)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("pt", [F32, BF16])
def test_misaligned_views_give_the_same_bits(bits, pt):
    """Tensors that start one element off their alignment take the scalar path."""
    n = 5000
    g = gen(7)
    p0, g0 = torch.randn(n, generator=g).to(pt), torch.randn(n, generator=g).to(pt)
    runs = []
    for off in (0, 1):
        def place(t, dtype=None):
            room = torch.zeros(n + 8, dtype=dtype or t.dtype, device=DEV)
            room[off: off + n] = t.to(DEV)
            return room[off: off + n]
        p, grad = place(p0), place(g0)
        state = F32 if bits == 32 else U8
        m, v = place(torch.zeros(n), state), place(torch.zeros(n), state)
        e = None if bits == 32 else _state([n], 8)[2]
        for step in (1, 2, 3):
            adamw_step([p], [grad], [m], [v], step=step, exponents=e, seed=2, **HYPER)
        runs.append([p, m, v])
    for a, b in zip(*runs):
        assert torch.equal(a, b)


def test_mixed_types_in_one_list():
    g = gen(8)
    kinds = [(F32, F32), (BF16, BF16), (F32, BF16), (F32, F32), (BF16, BF16)]
    params = [torch.randn(500 + k, generator=g).to(a).to(DEV) for k, (a, _) in enumerate(kinds)]
    grads = [torch.randn(500 + k, generator=g).to(b).to(DEV) for k, (_, b) in enumerate(kinds)]
    sizes = [p.numel() for p in params]
    got = [p.clone() for p in params]
    m, v, e = _state(sizes, 8)
    norm = adamw_step(got, grads, m, v, step=1, exponents=e, max_grad_norm=1.0, seed=4, **HYPER)
    want = torch.sqrt(sum(x.double().square().sum() for x in grads))
    assert abs(norm.item() / want.item() - 1) < 1e-6
    clip = grad_norm(grads, 1.0)[1]
    for k in range(len(kinds)):
        one = params[k].clone()
        mk, vk, ek = _state([sizes[k]], 8)
        adamw_step([one], [grads[k]], mk, vk, step=1, exponents=ek, clip=clip, seed=4,
                   ordinals=[k], **HYPER)
        assert torch.equal(one, got[k]) and torch.equal(mk[0], m[k])


# ------------------------------------------------------------------ gradient norm

def test_grad_norm():
    g = gen(10)
    for sizes in ([1], [3, 5], [2048, 2049, 1], [1000003], [17] * 200, [0, 4, 0]):
        for dt in (F32, BF16):
            grads = [torch.randn(n, generator=g).to(dt).to(DEV) for n in sizes]
            want = torch.sqrt(sum(x.double().square().sum() for x in grads)).item()
            norm, factor = grad_norm(grads, 0.5).tolist()
            assert abs(norm / want - 1) < 1e-6
            assert abs(factor / min(1.0, 0.5 / (want + 1e-6)) - 1) < 2e-6
            assert grad_norm(grads)[1].item() == 1.0
    big = torch.full((5000,), 1e25, device=DEV)     # squares above fp32's range
    assert grad_norm([big], 1.0)[0].item() == float("inf")
    assert grad_norm([torch.zeros(9, device=DEV)], 1.0).tolist() == [0.0, 1.0]
    bad = torch.tensor([1.0, float("nan")], device=DEV)
    assert all(torch.isnan(grad_norm([bad], 1.0)))
    one, two = (grad_norm([torch.randn(300000, generator=gen(1)).to(DEV)], 1.0) for _ in range(2))
    assert torch.equal(one, two)


def test_another_stream():
    n = 100000
    grad = torch.randn(n, generator=gen(3)).to(DEV)
    runs = []
    side = torch.cuda.Stream()
    for st in (torch.cuda.current_stream(), side):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            p = torch.ones(n, device=DEV)
            m, v, e = _state([n], 8)
            adamw_step([p], [grad], m, v, step=1, exponents=e, max_grad_norm=1.0, **HYPER)
        torch.cuda.synchronize()
        runs.append([p, m[0], v[0]])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


# --------------------------------------------------------------------- optimizer

@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("pt", [F32, BF16])
def test_state_dict_continues_with_the_same_bits(bits, pt):
    def build():
        g = gen(12)
        return [torch.nn.Parameter(torch.randn(s, generator=g).to(DEV, pt))
                for s in ((40, 30), (7,))]

    def steps(opt, params, which):
        for k in which:
            g = gen(100 + k)
            for p in params:
                p.grad = torch.randn(p.shape, generator=g).to(DEV, pt)
            opt.step(max_grad_norm=1.0)

    a = build()
    oa = AdamW(a, lr=1e-2, state_bits=bits, seed=6)
    steps(oa, a, range(3))
    saved = oa.state_dict()
    b = build()
    for p, q in zip(a, b):
        q.data.copy_(p.data)
    ob = AdamW(b, lr=1.0, state_bits=bits)
    ob.load_state_dict(saved)
    assert ob.seed == 6 and ob.param_groups[0]["lr"] == 1e-2
    steps(oa, a, range(3, 6))
    steps(ob, b, range(3, 6))
    for p, q in zip(a, b):
        assert torch.equal(p, q)
        assert ob.state[q]["exp_avg"].dtype == (F32 if bits == 32 else U8)
    with pytest.raises(ValueError, match="moments"):
        AdamW(build(), state_bits=40 - bits).load_state_dict(saved)


def test_transposed_parameters_and_gradients():
    g = gen(13)
    base = torch.randn(20, 30, generator=g).to(DEV)
    p = torch.nn.Parameter(base.t())                   # not contiguous
    q = torch.nn.Parameter(base.t().contiguous())
    grad = torch.randn(20, 30, generator=g).to(DEV).t()
    a, b = AdamW([p], lr=1e-2), AdamW([q], lr=1e-2)
    p.grad, q.grad = grad, grad.contiguous()
    a.step()
    b.step()
    assert torch.equal(p.detach().contiguous(), q.detach())


def test_moments_and_closure():
    p = torch.nn.Parameter(torch.ones(10, 3, device=DEV))
    opt = AdamW([p], lr=1e-2, state_bits=8)
    loss = opt.step(lambda: _backward(p))
    assert loss.item() == 30.0
    m, root = opt.moments(p)
    assert m.shape == p.shape and root.shape == p.shape
    # g = 2: m = 0.2 and sqrt(v) = 2 sqrt(0.001), within a rounding step
    assert ((m.float() / 0.2 - 1).abs() <= 2.0 ** -3).all()
    assert ((root.float() / (2 * 0.001 ** 0.5) - 1).abs() <= 2.0 ** -4).all()


def _backward(p):
    loss = p.square().sum()
    loss.backward()
    return loss.detach()


@pytest.mark.parametrize("pt", [F32, BF16])
def test_8_bit_training_follows_32_bit_training(pt):
    """The LM harness on one repeated batch: the loss falls as it does with 32-bit
    moments (both are held to the bound of the 32-bit harness test)."""
    last = {}
    for bits in (32, 8):
        torch.manual_seed(0)
        lm = QuaternionMamba2(61, d_model=32, n_layers=2, d_state=8).to(DEV, pt)
        opt = AdamW(lm.parameters(), lr=3e-3, state_bits=bits)
        seq = torch.randint(0, 61, (4, 65), generator=gen(5)).to(DEV)
        losses = [train_step(lm, opt, seq[:, :-1], seq[:, 1:]).item() for _ in range(30)]
        assert all(torch.isfinite(torch.tensor(losses)))
        assert losses[-1] < 0.8 * losses[0], (bits, losses)
        last[bits] = losses[-1]
        assert opt.grad_norm is not None and opt.grad_norm.item() > 0


def test_refusals():
    p, g = torch.ones(300, device=DEV), torch.ones(300, device=DEV)
    m, v, e = _state([300], 8)
    f = [torch.zeros(300, device=DEV)]
    with pytest.raises(AssertionError, match="step"):
        adamw_step([p], [g], f, f, step=0, lr=1e-3)
    with pytest.raises(AssertionError, match="grads"):
        adamw_step([p], [], f, f, step=1, lr=1e-3)
    with pytest.raises(TypeError, match="float16"):
        adamw_step([p], [g.half()], f, f, step=1, lr=1e-3)
    with pytest.raises(TypeError, match="exp_avgs"):
        adamw_step([p], [g], m, v, step=1, lr=1e-3)
    with pytest.raises(AssertionError, match="elements"):
        adamw_step([p], [g[:200].clone()], f, f, step=1, lr=1e-3)
    with pytest.raises(AssertionError, match="exponents"):
        adamw_step([p], [g], m, v, step=1, lr=1e-3, exponents=([e[0][0][:1]], e[1]))
    with pytest.raises(AssertionError, match="contiguous"):
        adamw_step([torch.ones(30, 20, device=DEV).t()], [torch.ones(30, 20, device=DEV).t()],
                   [torch.zeros(600, device=DEV)], [torch.zeros(600, device=DEV)], step=1, lr=1e-3)
    with pytest.raises(RuntimeError, match="betas"):
        adamw_step([p], [g], f, [torch.zeros(300, device=DEV)], step=1, lr=1e-3, betas=(1.0, 0.9))
    with pytest.raises(AssertionError, match="exclude"):
        adamw_step([p], [g], f, f, step=1, lr=1e-3, max_grad_norm=1.0, clip=p[:1])
    with pytest.raises(RuntimeError, match="CUDA"):
        adamw_step([p.cpu()], [g.cpu()], [f[0].cpu()], [f[0].cpu()], step=1, lr=1e-3)
    for bad in (dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(state_bits=16)):
        with pytest.raises(ValueError):
            AdamW([torch.nn.Parameter(p)], **bad)
    sparse = torch.nn.Parameter(torch.ones(4, 2, device=DEV))
    sparse.grad = torch.sparse_coo_tensor([[1]], [[1.0, 1.0]], (4, 2)).to(DEV)
    with pytest.raises(RuntimeError, match="sparse"):
        AdamW([sparse]).step()


def test_moments_have_the_bits_of_elementary_operations():
    """No sum of products is fused: an 8-bit code follows from a moment's last bits."""
    n = 100003
    p, g, m, v = (torch.randn(n, generator=gen(k)).to(DEV) for k in range(4))
    v = v.square()
    want_m = m * 0.9 + g * (1 - 0.9)
    want_v = v * 0.999 + (g * g) * (1 - 0.999)
    adamw_step([p], [g], [m], [v], step=3, lr=1e-3, betas=(0.9, 0.999))
    assert torch.equal(m, want_m)
    assert torch.equal(v, want_v)


@pytest.mark.parametrize("bits", [32, 8])
def test_step_advances_the_version_counters(bits):
    """What a step writes in place counts as written: a second backward through a graph
    from before the step raises instead of using the new weights."""
    p = torch.nn.Parameter(torch.randn(300, generator=gen(1)).to(DEV))
    opt = AdamW([p], lr=1e-2, state_bits=bits)
    loss = p.square().sum()
    loss.backward(retain_graph=True)
    opt.step()
    states = [v for v in opt.state[p].values() if torch.is_tensor(v)]
    before = [v._version for v in (p, *states)]
    opt.step(max_grad_norm=1.0)
    assert [v._version for v in (p, *states)] == [k + 1 for k in before]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("pt", [F32, BF16])
@pytest.mark.parametrize("size", [3e19, 1e25, 3e38])
def test_finite_gradient_whose_square_overflows(bits, pt, size):
    """v is infinite, so the update is m over infinity, nothing: the parameter moves by
    its decay alone, as in the formula (and torch.optim.AdamW); elements beside it step
    as they would without it. In 32 bits that holds for the steps after it too."""
    n = 2500
    lr, wd = 1e-2, 0.0
    grad = torch.ones(n, device=DEV)
    runs = []
    for value in (1.0, size):
        p = torch.ones(n, device=DEV, dtype=pt)
        g = grad.clone()
        g[[5, 300, 2499]] = value
        g[301] = -value
        m, v, e = _state([n], bits)
        adamw_step([p], [g], m, v, step=1, lr=lr, weight_decay=wd, exponents=e, seed=1)
        if bits == 32:
            assert torch.isinf(v[0]).sum() == (0 if value == 1.0 else 4)
            runs.append(p.clone())
            adamw_step([p], [grad], m, v, step=2, lr=lr, weight_decay=wd, exponents=e, seed=1)
        runs.append(p.clone())
    half = len(runs) // 2
    big = torch.zeros(n, dtype=torch.bool, device=DEV)
    big[[5, 300, 301, 2499]] = True
    for ones, got in zip(runs[:half], runs[half:]):
        assert torch.equal(got[big], torch.ones_like(got[big]))
        assert torch.equal(got[~big], ones[~big])


@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("size", [1e-15, 1e-17, 2e-18, 1e-19, 1e-20, 3e-21])
def test_tiny_second_moments_32_bits(size, off):
    """v down to fp32's smallest numbers, with an eps below their roots: the update is
    the formula's of the moments as stored (their roots and quotient are within a few
    units of 6e-8)."""
    n = 3000
    room = [torch.zeros(n + 1, device=DEV) for _ in range(4)]
    p, g, m, v = (t[off: off + n] for t in room)
    g.copy_(size * (1 + torch.rand(n, generator=gen(2))))
    adamw_step([p], [g], [m], [v], step=1, lr=1.0, betas=(0.9, 0.999), eps=1e-30, weight_decay=0.0)
    m64, v64 = m.double(), v.double()
    want = -10.0 * m64 / (v64.sqrt() / 0.001 ** 0.5 + 1e-30)
    assert (v64 > 0).all()
    assert ((p.double() / want - 1).abs() <= 1e-6).all()


@pytest.mark.parametrize("size", [1e-15, 1e-17, 2e-18, 1e-19, 1e-20])
def test_tiny_second_moments_8_bits(size):
    """The codes of small roots are those of sqrt(v), v as fp32 has it."""
    n = 3000
    p = torch.zeros(n, device=DEV)
    g = (size * (1 + torch.rand(n, generator=gen(2)))).to(DEV)
    m, v, e = _state([n], 8)
    adamw_step([p], [g], m, v, step=1, lr=1.0, betas=(0.9, 0.999), eps=1e-30, weight_decay=0.0,
               exponents=e, seed=7)
    g32 = g.cpu()
    v32 = (g32 * g32) * torch.tensor(1 - 0.999)
    got = _values(v[0], e[1][0], 4)
    noise = _noise(n, 7, 1, 0)
    _close_codes(got, _rounded(v32.double().sqrt(), noise & 0xFFFF, 4, e[1][0], False), 2.0 ** -4)
    want = -10.0 * (0.1 * g32.double()) / (v32.double().sqrt() / 0.001 ** 0.5 + 1e-30)
    assert ((p.cpu().double() / want - 1).abs() <= 1e-6).all()


def test_clipping_factor_is_rounded_once():
    """Gradients of whole numbers, whose squares add up exactly: the norm is the root
    of a whole number, and the factor max_norm / (norm + 1e-6) has one rounding from 64
    bits, max_norm being what the caller gave."""
    g = gen(20)
    for k in range(200):
        grads = [torch.randint(-9, 10, (50 + k,), generator=g).float() for _ in range(3)]
        norm = sum(t.double().square().sum() for t in grads).sqrt()
        max_norm = (0.1, 1.0, 1 / 3, 0.7)[k % 4]
        got = grad_norm([t.to(DEV) for t in grads], max_norm).cpu()
        assert got[0] == norm.float(), k
        assert got[1] == (max_norm / (norm + 1e-6)).float(), k


def test_continues_a_state_of_torch_adamw(monkeypatch):
    """The steps after the switch are those of torch's optimizer, one call each."""
    from mambaqc_b200 import optim

    def params():
        g = gen(31)
        return [torch.nn.Parameter(torch.randn(s, generator=g).to(DEV)) for s in ((20, 30), (7,))] \
            + [torch.nn.Parameter(torch.randn(8, 5, generator=g).to(DEV).t())]

    def steps(opt, which, ps):
        for k in which:
            g = gen(200 + k)
            for p in ps:
                p.grad = torch.randn(p.shape, generator=g).to(DEV)
            opt.step()

    a = params()
    oa = torch.optim.AdamW(a, lr=1e-2, weight_decay=0.1)
    steps(oa, range(4), a)
    b = params()
    for p, q in zip(a, b):
        q.data.copy_(p.data)
    ob = AdamW(b)
    ob.load_state_dict(oa.state_dict())
    calls = []
    monkeypatch.setattr(optim, "adamw_step", lambda *x, **k: calls.append(1) or adamw_step(*x, **k))
    steps(oa, range(4, 8), a)
    steps(ob, range(4, 8), b)
    assert len(calls) == 4
    for p, q in zip(a, b):
        assert rel_l2(q, p) < 8e-6


@pytest.mark.parametrize("bits", [32, 8])
def test_smallest_eps(bits):
    """An eps that has no fp32 reciprocal: parameters whose gradients are all zero stay
    where they are, the others step by the formula."""
    n = 700
    grad = torch.zeros(n, device=DEV)
    grad[1::2] = 3.0
    p = torch.ones(n, device=DEV)
    m, v, e = _state([n], bits)
    adamw_step([p], [grad], m, v, step=1, lr=1e-2, eps=1e-40, weight_decay=0.0, exponents=e)
    assert torch.equal(p[0::2], torch.ones_like(p[0::2]))
    assert ((p[1::2] - 0.99).abs() < 1e-6).all()
