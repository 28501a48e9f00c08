"""What the operators of a gated-recurrent training stack compute, and the cases they are timed at.

Three operators, each in a plain form of elementary torch operations (``own`` false) and through
the calls a user makes of this package (``own`` true):

* ``scan``  -- the gated linear recurrence over a sequence, with its gradient, and its one-token form
* ``norm``  -- norm of a block's output, gate, residual scale and the next block's norm, with its gradient
* ``adamw`` -- one AdamW step over a list of tensors, moments in 32 or in 8 bits, with gradient clipping

Formulas, with s = sigmoid:

scan    a[t] = exp(-c softplus(Lambda) s(r[t])), h[t] = a[t] h[t-1] + sqrt(1 - a[t]^2) s(i[t]) x[t];
        where reset[t] is set the state is dropped: h[t] = s(i[t]) x[t].
norm    out = x + scale s(z) P(y), n = Q(out), P and Q LayerNorm or RMSNorm over the last axis.
adamw   m <- b1 m + (1 - b1) g, v <- b2 v + (1 - b2) g^2,
        p <- (1 - lr wd) p - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps), g clipped by the global norm.
        In 8 bits a block of 256 values shares a power of two; m is held in sign, 4 exponent and 3 fraction
        bits, sqrt(v) in 4 exponent and 4 fraction bits, both rounded up or down by a hash of the element's
        index and the step (so that a change smaller than a rounding step is not lost step after step).
        bfloat16 parameters are rounded by the same hash.
"""

import math

import torch

own = False

SHARPNESS = 8.0   # c of the recurrence
BLOCK = 256       # values that share one power of two in the 8-bit moments
EPS = 1e-5        # of the norms

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ cases

def listed():
    return [
        # training step of a layer as wide as the base preset's d_inner (768 x 2), batch 4 x 2048 under bf16 autocast
        dict(name="scan_train_base_bf16", op="scan", mode="train", batch=4, seq=2048, width=1536,
             dtype="bf16", h0=False, reset=False),
        # fp32 training on packed documents (the state is dropped where one starts), odd width and length
        dict(name="scan_train_packed_f32", op="scan", mode="train", batch=3, seq=1001, width=515,
             dtype="f32", h0=True, reset=True),
        # prefill of one long prompt: few channels, so the time axis has to carry the parallelism
        dict(name="scan_prefill_long_bf16", op="scan", mode="forward", batch=1, seq=32768, width=1024,
             dtype="bf16", h0=True, reset=False),
        # one token for each of 64 sequences, the smallest call: latency
        dict(name="scan_step_b64_bf16", op="scan", mode="step", batch=64, seq=1, width=1536,
             dtype="bf16", h0=True, reset=False),
        # residual epilogue of the base preset in training: fp32 residual stream, bf16 block output and gate
        dict(name="norm_train_base_mixed", op="norm", mode="train", rows=8192, width=768,
             stream="f32", dtype="bf16", norm="layer", bias=True, next=True),
        # large preset, all bf16, rms
        dict(name="norm_train_large_bf16", op="norm", mode="train", rows=16384, width=1024,
             stream="bf16", dtype="bf16", norm="rms", bias=False, next=True),
        # odd rows and width in fp32, no norm of the next block (the last layer before a different head)
        dict(name="norm_train_odd_f32", op="norm", mode="train", rows=1731, width=515,
             stream="f32", dtype="f32", norm="rms", bias=True, next=False),
        # decoding: 8 sequences, one token each
        dict(name="norm_decode_b8_bf16", op="norm", mode="forward", rows=8, width=1024,
             stream="bf16", dtype="bf16", norm="layer", bias=True, next=True),
        # every tensor of a one-layer small-preset LM (d_model 512, N 32) without its two largest: 16 tensors, clipped
        dict(name="adamw32_small_tensors", op="adamw", bits=32, tensors="small", elements=0, count=16,
             param="f32", grad="f32", clip=True),
        # one B projection of the small preset (1024 x 131072), moments in 32 bits
        dict(name="adamw32_projection", op="adamw", bits=32, tensors="equal", elements=134217728, count=1,
             param="f32", grad="f32", clip=False),
        # the same projection with moments in 8 bits
        dict(name="adamw8_projection", op="adamw", bits=8, tensors="equal", elements=134217728, count=1,
             param="f32", grad="f32", clip=True),
        # bf16 parameters and gradients, 8-bit moments, ragged sizes from one element up
        dict(name="adamw8_ragged_bf16", op="adamw", bits=8, tensors="ragged", elements=9000001, count=18,
             param="bf16", grad="bf16", clip=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["scan", "scan", "norm", "norm", "adamw", "adamw"])
    if op == "scan":
        mode = rng.choice(["train", "train", "forward", "step"])
        width = _log_int(rng, 33, 2048)
        if rng.random() < 0.5:
            width = -(-width // 64) * 64
        batch = _log_int(rng, 1, 256 if mode == "step" else 8)
        seq = 1 if mode == "step" else _log_int(rng, 16, max(16, min(32768, 12582912 // (batch * width))))
        return dict(op="scan", mode=mode, batch=batch, seq=seq, width=width, dtype=rng.choice(["f32", "bf16"]),
                    h0=True if mode == "step" else rng.random() < 0.5,
                    reset=False if mode == "step" else rng.random() < 0.3)
    if op == "norm":
        mode = rng.choice(["train", "train", "forward"])
        width = _log_int(rng, 65, 4096)
        if rng.random() < 0.5:
            width = -(-width // 64) * 64
        dtype = rng.choice(["f32", "bf16"])
        return dict(op="norm", mode=mode, rows=_log_int(rng, 1, max(2, 16777216 // width)), width=width,
                    stream="f32" if dtype == "f32" else rng.choice(["f32", "bf16"]), dtype=dtype,
                    norm=rng.choice(["rms", "layer"]), bias=rng.random() < 0.5, next=rng.random() < 0.7)
    bits = rng.choice([8, 32])
    param, grad = rng.choice([("f32", "f32"), ("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16")])
    kind = rng.choice(["equal", "ragged"])
    return dict(op="adamw", bits=bits, tensors=kind, elements=_log_int(rng, 2000, 60000000),
                count=rng.randint(1, 20) if kind == "ragged" else rng.randint(1, 3),
                param=param, grad=grad, clip=rng.random() < 0.5)


def _sizes(case):
    """Element counts of an adamw case's tensors."""
    if case["tensors"] == "small":
        d, di, ds, vocab = 512, 1024, 32, 10000
        return [2 * di * d, di * 4, di, di * ds, di * ds * 3, di * di, di, di, di * di, di, di * 4,
                4 * di * d, vocab * d, d, d, vocab * d][: case["count"]]
    n, k = case["elements"], case["count"]
    if case["tensors"] == "equal":
        return [max(1, n // k)] * k
    # ragged: each tensor about twice the one before it, odd, the first of one element
    total, out = float(2 ** k - 1), []
    for i in range(k):
        out.append(max(1, int(n * (2 ** i) / total)) | 1)
    out[0] = 1
    return out


# ------------------------------------------------------------------ inputs

def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=dev).to(dtype)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device=dev)

    s = dict(case=case)
    if case["op"] == "scan":
        dt = _DTYPES[case["dtype"]]
        b, t, d = case["batch"], case["seq"], case["width"]
        shape = (b, d) if case["mode"] == "step" else (b, t, d)
        s["x"], s["r"], s["i"] = (randn(*shape, dtype=dt) for _ in range(3))
        # decay a^c between 0.9 and 0.999 where the recurrence gate is open
        decay = 0.9 + 0.099 * rand(d)
        s["Lambda"] = torch.log(torch.expm1(-torch.log(decay) / SHARPNESS))
        s["h0"] = randn(b, d) if case["h0"] else None
        s["reset"] = None
        if case["reset"]:
            s["reset"] = rand(b, t) < 1 / 256
        if case["mode"] == "train":
            s["dy"], s["dhT"] = randn(*shape, dtype=dt), randn(b, d)
            for k in ("x", "r", "i", "Lambda", "h0"):
                if s[k] is not None:
                    s[k].requires_grad_()
    elif case["op"] == "norm":
        st, dt = _DTYPES[case["stream"]], _DTYPES[case["dtype"]]
        rows, d = case["rows"], case["width"]
        s["x"], s["y"] = randn(rows, d, dtype=st), randn(rows, d, dtype=dt)
        wide = randn(rows, 2 * d, dtype=dt)   # the gate is the right half of a block's input projection
        s["z"] = wide[:, d:]
        s["weight"], s["scale"] = 1 + 0.1 * randn(d), 0.5 + 0.1 * randn(d)
        s["bias"] = 0.1 * randn(d) if case["bias"] else None
        s["next_weight"] = 1 + 0.1 * randn(d) if case["next"] else None
        s["next_bias"] = 0.1 * randn(d) if case["next"] and case["bias"] else None
        if case["mode"] == "train":
            s["dout"] = randn(rows, d, dtype=st)
            s["dn"] = randn(rows, d, dtype=dt) if case["next"] else None
            s["z"] = s["z"].detach()
            for k in ("x", "y", "z", "weight", "scale", "bias", "next_weight", "next_bias"):
                if s[k] is not None:
                    s[k].requires_grad_()
    else:
        pd, gd = _DTYPES[case["param"]], _DTYPES[case["grad"]]
        for k in ("params", "grads", "m", "v", "m_exp", "v_exp"):
            s[k] = []
        for n in _sizes(case):
            s["params"].append(0.02 * randn(n, dtype=torch.float32).to(pd))
            size = 10.0 ** (-3 - 2 * rand(1))        # gradients of one tensor are of one size
            s["grads"].append((size * randn(n)).to(gd))
            m, root = 0.3 * size * randn(n), size * (0.5 + rand(n))
            if case["bits"] == 32:
                s["m"].append(m)
                s["v"].append(root * root)
                continue
            blocks = -(-n // BLOCK)
            for key, value, bits in (("m", m, 3), ("v", root, 4)):
                # codes of the values, rounded down, under the block's largest
                full = torch.zeros(blocks * BLOCK, device=dev)
                full[:n] = value
                raw = full.abs().view(blocks, BLOCK).view(torch.int32)
                e = (raw.amax(1, keepdim=True) >> 23).clamp(16, 254)
                code = ((raw - ((e - 15) << 23)) >> (23 - bits)).clamp(0, (16 << bits) - 1)
                if key == "m":
                    code = code | (full.view(blocks, BLOCK) < 0).int() * 128
                s[key].append(code.to(torch.uint8).view(-1)[:n].clone())
                s[key + "_exp"].append(e.to(torch.uint8).view(-1))
                del full, raw, code
        s["step"] = 100
        # active: about half of the gradients' norm
        norm = math.sqrt(sum(float(t.float().square().sum()) for t in s["grads"]))
        s["max_norm"] = 0.5 * norm if case["clip"] else None
    return s


_LR, _BETAS, _ADAM_EPS, _WD, _SEED = 1e-3, (0.9, 0.999), 1e-8, 0.1, 1234


# ------------------------------------------------------------------ plain forms

def _scan_plain(a, b, h0, backward=False):
    """h[t] = a[t] h[t-1] + b[t] along dim 1 by doubling; ``backward`` runs from the end."""
    a, b = (a.flip(1), b.flip(1)) if backward else (a.clone(), b.clone())
    if h0 is not None:
        b[:, 0] += a[:, 0] * h0
    k = 1
    while k < a.shape[1]:
        b = torch.cat([b[:, :k], b[:, k:] + a[:, k:] * b[:, :-k]], dim=1)
        a = torch.cat([a[:, :k], a[:, k:] * a[:, :-k]], dim=1)
        k *= 2
    return b.flip(1) if backward else b


def _gates_plain(s):
    x, r, i = (s[k].detach().float() for k in ("x", "r", "i"))
    sr, si = torch.sigmoid(r), torch.sigmoid(i)
    rate = SHARPNESS * torch.log1p(torch.exp(s["Lambda"].detach()))
    lam = rate * sr                                # -log a
    a = torch.exp(-lam)
    beta = torch.sqrt(-torch.expm1(-2 * lam))
    return x, sr, si, lam, a, beta


def _run_scan_plain(s):
    case = s["case"]
    dt = s["x"].dtype
    x, sr, si, lam, a, beta = _gates_plain(s)
    if case["mode"] == "step":
        h = a * s["h0"] + beta * si * x
        s["h0"].copy_(h)
        return h.to(dt), s["h0"]
    h0 = s["h0"].detach() if s["h0"] is not None else torch.zeros_like(x[:, 0])
    if s["reset"] is not None:
        keep = ~s["reset"][..., None]
        a, beta_r = a * keep, torch.where(keep, beta, torch.ones_like(beta))
    else:
        keep, beta_r = torch.ones_like(a, dtype=torch.bool), beta
    h = _scan_plain(a, beta_r * si * x, h0)
    y, hT = h.to(dt), h[:, -1].clone()
    if case["mode"] == "forward":
        return y, hT
    dy = s["dy"].float()
    dy = torch.cat([dy[:, :-1], (dy[:, -1] + s["dhT"])[:, None]], dim=1)
    a_next = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], dim=1)
    gh = _scan_plain(a_next, dy, None, backward=True)
    before = torch.cat([h0[:, None], h[:, :-1]], dim=1)
    dx = gh * beta_r * si
    di = gh * beta_r * x * si * (1 - si)
    # d/dlam of a is -a, of beta a^2 / beta; where the state is dropped neither depends on lam
    slope = torch.where(lam > 0, a * a / beta, torch.zeros_like(a))
    dlam = torch.where(keep, gh * (slope * si * x - a * before), torch.zeros_like(a))
    dr = dlam * lam * (1 - sr)
    dLambda = (dlam * sr).sum((0, 1)) * SHARPNESS * torch.sigmoid(s["Lambda"].detach())
    out = [y, hT, dx.to(dt), dr.to(dt), di.to(dt), dLambda]
    if s["h0"] is not None:
        out.append(gh[:, 0] * a[:, 0])
    return out


def _norm_plain(u, kind):
    if kind == "layer":
        u = u - u.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((u * u).mean(-1, keepdim=True) + EPS)
    return u * rstd, rstd


def _norm_grad_plain(dhat, hat, rstd, kind):
    d = dhat - hat * (dhat * hat).mean(-1, keepdim=True)
    if kind == "layer":
        d = d - dhat.mean(-1, keepdim=True)
    return d * rstd


def _run_norm_plain(s):
    case, kind = s["case"], s["case"]["norm"]
    w, scale = s["weight"].detach(), s["scale"].detach()
    x, y, z = (s[k].detach().float() for k in ("x", "y", "z"))
    gate = torch.sigmoid(z)
    yhat, yr = _norm_plain(y, kind)
    p = yhat * w if s["bias"] is None else yhat * w + s["bias"].detach()
    out = x + scale * gate * p
    result = [out.to(s["x"].dtype)]
    if case["next"]:
        w2 = s["next_weight"].detach()
        nhat, nr = _norm_plain(out, kind)
        n = nhat * w2 if s["next_bias"] is None else nhat * w2 + s["next_bias"].detach()
        result.append(n.to(s["y"].dtype))
    if case["mode"] == "forward":
        return result
    d = s["dout"].float()
    if case["next"]:
        dn = s["dn"].float()
        d = d + _norm_grad_plain(dn * w2, nhat, nr, kind)
    dp = d * scale * gate
    result += [d.to(s["x"].dtype), _norm_grad_plain(dp * w, yhat, yr, kind).to(s["y"].dtype),
               (d * scale * p * gate * (1 - gate)).to(s["z"].dtype), (dp * yhat).sum(0), (d * gate * p).sum(0)]
    if s["bias"] is not None:
        result.append(dp.sum(0))
    if case["next"]:
        result.append((dn * nhat).sum(0))
        if s["next_bias"] is not None:
            result.append(dn.sum(0))
    return result


def _hash(index, key):
    """32 well-mixed bits of an element's index and a 32-bit key, in int64."""
    h = (index & 0xFFFFFFFF) ^ key ^ ((index >> 32) * 0x9E3779B9 & 0xFFFFFFFF)
    h = h * 0x6A09E667 & 0xFFFFFFFF
    h = h ^ h >> 15
    h = h * 0xBB67AE85 & 0xFFFFFFFF
    return h ^ h >> 13


def _key(seed, step, tensor):
    """The key of one tensor's step: the same mixing, over seed, step and the tensor's place in the list."""
    def mix(h):
        h = h * 0x6A09E667 & 0xFFFFFFFF
        h ^= h >> 15
        h = h * 0xBB67AE85 & 0xFFFFFFFF
        return h ^ h >> 13
    return mix(mix(mix(seed & 0xFFFFFFFF) ^ step & 0xFFFFFFFF) ^ tensor)


def _decode_plain(code, e, fraction, n):
    """Values of 8-bit codes: sign (3 fraction bits) or none (4), exponent under the block's, fraction."""
    blocks = e.numel()
    c = torch.zeros(blocks * BLOCK, dtype=torch.int32, device=code.device)
    c[:n] = code
    c = c.view(blocks, BLOCK)
    mag = c & 127 if fraction == 3 else c
    value = (((e.int()[:, None] - 15) << 23) + (mag << (23 - fraction))).view(torch.float32)
    value = torch.where(mag == 0, torch.zeros_like(value), value)
    if fraction == 3:
        value = torch.where(c > 127, -value, value)
    value = torch.where((e == 255)[:, None], torch.full_like(value, float("nan")), value)
    return value.view(-1)[:n]


def _encode_plain(value, noise, fraction):
    """(codes, exponents) of values under each block's largest; ``noise``: 16 bits that say up or down."""
    n = value.numel()
    blocks = -(-n // BLOCK)
    v = torch.zeros(blocks * BLOCK, device=value.device)
    v[:n] = value
    v = v.view(blocks, BLOCK)
    r = torch.zeros(blocks * BLOCK, dtype=torch.int32, device=value.device)
    r[:n] = noise
    r = r.view(blocks, BLOCK)
    raw = v.abs().view(torch.int32)
    e = raw.amax(1, keepdim=True) >> 23
    bad = e == 255
    e = e.clamp(16, 254)
    shift = 23 - fraction
    least = 1 + 2.0 ** -fraction                            # code 1, in units of 2^(e - 142)
    code = (raw - ((e - 15) << 23) + (r << (shift - 16))) >> shift
    w = v.abs() * ((269 - e) << 23).view(torch.float32)
    small = w < least
    up = w > r.float() * (least / 65536)
    if fraction == 4:
        up = w > 0                                          # a root above zero stays above zero
    code = torch.where(small, up.int(), code.clamp(0, (16 << fraction) - 1))
    if fraction == 3:
        code = code | (v < 0).int() * 128
    code = torch.where(bad, torch.zeros_like(code), code)
    e = torch.where(bad, torch.full_like(e, 255), e)
    return code.to(torch.uint8).view(-1)[:n], e.to(torch.uint8).view(-1)


def _run_adamw_plain(s):
    case = s["case"]
    t = s["step"]
    b1, b2 = _BETAS
    step_size = _LR / (1 - b1 ** t)
    root_scale = 1 / math.sqrt(1 - b2 ** t)
    norm = clip = None
    if s["max_norm"] is not None:
        norm = torch.sqrt(torch.stack([g.float().square().sum() for g in s["grads"]]).sum())
        clip = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    moments = []
    for k, (p, g) in enumerate(zip(s["params"], s["grads"])):
        n = p.numel()
        g = g.float()
        if clip is not None:
            g = g * clip
        if case["bits"] == 32:
            m, v = s["m"][k], s["v"][k]
        else:
            m = _decode_plain(s["m"][k], s["m_exp"][k], 3, n)
            root = _decode_plain(s["v"][k], s["v_exp"][k], 4, n)
            v = root * root
        m = m * b1 + g * (1 - b1)
        v = v * b2 + (g * g) * (1 - b2)
        root = torch.sqrt(v)
        new = p.float() * (1 - _LR * _WD) - step_size * (m / (root * root_scale + _ADAM_EPS))
        h = None
        if case["bits"] == 8 or p.dtype == torch.bfloat16:
            h = _hash(torch.arange(n, device=p.device), _key(_SEED, t, k))
        if p.dtype == torch.bfloat16:
            r = (h * 0x9E3779B9 & 0xFFFFFFFF) >> 16
            bits = new.view(torch.int32)
            new = torch.where(torch.isfinite(new), ((bits + r.int()) & -65536).view(torch.float32), new)
        p.copy_(new)
        if case["bits"] == 32:
            s["m"][k].copy_(m)
            s["v"][k].copy_(v)
            moments += [s["m"][k], s["v"][k]]
            continue
        for key, value, noise, fraction in (("m", m, h >> 16, 3), ("v", root, h & 0xFFFF, 4)):
            code, e = _encode_plain(value, noise.int(), fraction)
            s[key][k].copy_(code)
            s[key + "_exp"][k].copy_(e)
            moments.append(_decode_plain(code, e, fraction, n).to(torch.bfloat16))
    s["step"] = t + 1
    return ([] if norm is None else [norm]) + s["params"] + moments


# ------------------------------------------------------------------ the package's calls

def _run_scan_own(s):
    from mambaqc_b200.kernels import gated_linear_scan, gated_linear_step
    mode = s["case"]["mode"]
    if mode == "step":
        y = gated_linear_step(s["x"], s["r"], s["i"], s["Lambda"], s["h0"], sharpness=SHARPNESS)
        return y, s["h0"]
    y, hT = gated_linear_scan(s["x"], s["r"], s["i"], s["Lambda"], s["h0"], s["reset"],
                              sharpness=SHARPNESS, return_final_state=True)
    if mode == "forward":
        return y, hT
    leaves = [s[k] for k in ("x", "r", "i", "Lambda", "h0") if s[k] is not None]
    return [y.detach(), hT.detach(), *torch.autograd.grad([y, hT], leaves, [s["dy"], s["dhT"]])]


def _run_norm_own(s):
    from mambaqc_b200.kernels import norm_gate_residual
    case = s["case"]
    got = norm_gate_residual(s["x"], s["y"], s["z"], s["weight"], s["scale"], s["bias"],
                             s["next_weight"], s["next_bias"], norm=case["norm"], eps=EPS)
    outs = list(got) if case["next"] else [got]
    if case["mode"] == "forward":
        return outs
    grads = [s["dout"]] + ([s["dn"]] if case["next"] else [])
    leaves = [s[k] for k in ("x", "y", "z", "weight", "scale", "bias", "next_weight", "next_bias")
              if s[k] is not None]
    return [o.detach() for o in outs] + list(torch.autograd.grad(outs, leaves, grads))


def _run_adamw_own(s):
    from mambaqc_b200.kernels import adamw_moments, adamw_step
    bits8 = s["case"]["bits"] == 8
    exponents = (s["m_exp"], s["v_exp"]) if bits8 else None
    norm = adamw_step(s["params"], s["grads"], s["m"], s["v"], step=s["step"], lr=_LR, betas=_BETAS,
                      eps=_ADAM_EPS, weight_decay=_WD, max_grad_norm=s["max_norm"], exponents=exponents,
                      seed=_SEED)
    s["step"] += 1
    moments = []
    if bits8:
        for m, root in zip(*adamw_moments(s["m"], s["v"], exponents)):
            moments += [m, root]
    else:
        for m, v in zip(s["m"], s["v"]):
            moments += [m, v]
    return ([] if norm is None else [norm]) + s["params"] + moments


def run(state):
    op = state["case"]["op"]
    if own:
        return {"scan": _run_scan_own, "norm": _run_norm_own, "adamw": _run_adamw_own}[op](state)
    return {"scan": _run_scan_plain, "norm": _run_norm_plain, "adamw": _run_adamw_plain}[op](state)


# ------------------------------------------------------------------ least work

def work(case):
    if case["op"] == "scan":
        es = 4 if case["dtype"] == "f32" else 2
        rows, d = case["batch"] * case["seq"], case["width"]
        n = rows * d
        states = case["batch"] * d * 4 * (2 if case["h0"] else 1)
        marks = rows if case["reset"] else 0
        if case["mode"] == "train":
            # x, r, i, dy in; y, dx, dr, di out; states and their gradients
            return dict(bytes=8 * n * es + 2 * states + marks + 8 * d, flops=60 * n)
        return dict(bytes=4 * n * es + states + marks + 4 * d, flops=24 * n)
    if case["op"] == "norm":
        ss, es = (4 if case[k] == "f32" else 2 for k in ("stream", "dtype"))
        n = case["rows"] * case["width"]
        nx = 1 if case["next"] else 0
        vectors = (2 + (1 if case["bias"] else 0) * (1 + nx) + nx) * 4 * case["width"]
        moved = 2 * ss + (2 + nx) * es                     # x, y, z in; out, n out
        flops = 16 + 8 * nx
        if case["mode"] == "train":
            moved += 2 * ss + (2 + nx) * es                # dout, dn in; dx, dy, dz out
            flops += 30 + 12 * nx
            vectors *= 2
        return dict(bytes=n * moved + vectors, flops=flops * n)
    n = sum(_sizes(case))
    ps, gs = (4 if case[k] == "f32" else 2 for k in ("param", "grad"))
    moved = 2 * ps + gs + (16 if case["bits"] == 32 else 4 + 4)   # 8 bits: codes in and out, values out
    return dict(bytes=n * moved, flops=18 * n)


# ------------------------------------------------------------------ the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"scan": _exact_scan, "norm": _exact_norm, "adamw": _exact_adamw}[case["op"]](case, s)


def _exact_scan(case, s):
    x, r, i = (s[k].detach().double() for k in ("x", "r", "i"))
    big = s["Lambda"].detach().double()
    soft = torch.nn.functional.softplus(big, threshold=100.0)
    if case["mode"] == "step":
        x, r, i = x[:, None], r[:, None], i[:, None]
    batch, seq, d = x.shape
    h0 = torch.zeros(batch, d, dtype=torch.float64, device=x.device) if s["h0"] is None else s["h0"].detach().double()
    log_a = -SHARPNESS * soft * r.sigmoid()
    drop = torch.zeros(batch, seq, 1, dtype=torch.bool, device=x.device) if s["reset"] is None else s["reset"][..., None]
    a = log_a.exp().masked_fill(drop, 0.0)
    beta = (-(2 * log_a).expm1()).sqrt()
    beta_or_one = beta.masked_fill(drop, 1.0)
    u = beta_or_one * i.sigmoid() * x
    h = torch.empty_like(x)
    state = h0
    for t in range(seq):
        state = torch.addcmul(u[:, t], a[:, t], state)
        h[:, t] = state
    if case["mode"] == "step":
        return [h[:, 0], state]
    if case["mode"] == "forward":
        return [h, state]
    dy = s["dy"].double()
    grad = torch.empty_like(x)
    g = s["dhT"].double()
    for t in range(seq - 1, -1, -1):
        g = g + dy[:, t]
        grad[:, t] = g
        g = g * a[:, t]
    dh0 = g
    prev = torch.cat([h0.unsqueeze(1), h[:, :-1]], 1)
    dx = grad * beta_or_one * i.sigmoid()
    di = dx * x * (1 - i.sigmoid())
    # derivative in log a: of a it is a, of sqrt(1 - a^2) it is -a^2 / sqrt(1 - a^2)
    dlog = grad * (a * prev - a * a / beta * i.sigmoid() * x)
    dlog = dlog.masked_fill(drop, 0.0)
    dr = dlog * log_a * (1 - r.sigmoid())
    dbig = (dlog * r.sigmoid()).sum(1).sum(0) * -SHARPNESS * big.sigmoid()
    return [h, state, dx, dr, di, dbig] + ([dh0] if s["h0"] is not None else [])


def _exact_norm(case, s):
    keys = [k for k in ("x", "y", "z", "weight", "scale", "bias", "next_weight", "next_bias") if s[k] is not None]
    q = {k: s[k].detach().double().requires_grad_() for k in keys}

    def normed(u, w, b):
        d = u - u.mean(-1, keepdim=True) if case["norm"] == "layer" else u
        d = d * torch.rsqrt(d.pow(2).mean(-1, keepdim=True) + EPS) * w
        return d if b is None else d + b

    outs = [q["x"] + q["scale"] * q["z"].sigmoid() * normed(q["y"], q["weight"], q.get("bias"))]
    if case["next"]:
        outs.append(normed(outs[0], q["next_weight"], q.get("next_bias")))
    if case["mode"] == "forward":
        return [o.detach() for o in outs]
    grads = [s["dout"].double()] + ([s["dn"].double()] if case["next"] else [])
    return [o.detach() for o in outs] + list(torch.autograd.grad(outs, [q[k] for k in keys], grads))


def _exact_adamw(case, s):
    t = s["step"]
    b1, b2 = _BETAS
    norm = torch.sqrt(sum(g.double().square().sum() for g in s["grads"]))
    clip = 1.0 if s["max_norm"] is None else torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)

    def values(code, e, fraction):
        c = code.long()
        e = e.double().repeat_interleave(BLOCK)[: c.numel()]
        mag = c % 128 if fraction == 3 else c
        size = torch.exp2(e - 142 + (mag >> fraction)) * (1 + (mag % (1 << fraction)).double() / (1 << fraction))
        size = size * (mag > 0)
        return torch.where(c > 127, -size, size) if fraction == 3 else size

    def rounded(value, noise, fraction):
        n = value.numel()
        at = torch.arange(n, device=value.device) // BLOCK
        top = torch.zeros(-(-n // BLOCK), dtype=torch.float64, device=value.device)
        top.scatter_reduce_(0, at, value.abs(), "amax")
        e = torch.where(top > 0, torch.floor(torch.log2(top.clamp(min=1e-300))) + 127, 0 * top).clamp(16, 254)
        unit = torch.exp2(e - 142)[at]
        w = value.abs() / unit
        r = noise.double() / 65536
        least = 1 + 2.0 ** -fraction
        grid = torch.exp2(torch.floor(torch.log2(w.clamp(min=least))) - fraction)
        up = torch.floor(w / grid + r) * grid
        up = torch.minimum(up, torch.full_like(up, 2.0 ** 15 * (2 - 2.0 ** -fraction)))
        low = least * ((w > 0) if fraction == 4 else (w > r * least)).double()
        return torch.where(w < least, low, up) * unit * torch.sign(value)

    params, moments = [], []
    for k, (p, g) in enumerate(zip(s["params"], s["grads"])):
        g = g.double() * clip
        if case["bits"] == 32:
            m, v = s["m"][k].double(), s["v"][k].double()
        else:
            m = values(s["m"][k], s["m_exp"][k], 3)
            v = values(s["v"][k], s["v_exp"][k], 4).square()
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g.square()
        del g
        hat = (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + _ADAM_EPS)
        params.append(p.double() * (1 - _LR * _WD) - _LR * hat)
        del hat
        if case["bits"] == 32:
            moments += [m, v]
            continue
        bits = _hash(torch.arange(p.numel(), device=p.device), _key(_SEED, t, k))
        moments += [rounded(m, bits >> 16, 3), rounded(v.sqrt(), bits & 0xFFFF, 4)]
    return ([] if s["max_norm"] is None else [norm]) + params + moments
