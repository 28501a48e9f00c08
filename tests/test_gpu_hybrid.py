"""The normed stack of gated recurrent and quaternion blocks on the GPU: loss and
gradients against a 64-bit composition of its formulas, checkpointing, recurrent
decoding, and training steps with the package's optimizer."""

import pytest
import torch
import torch.nn.functional as F

from tests.gpu_util import DEV, RTOL_F32, gen, rel_l2

pytestmark = pytest.mark.gpu

from mambaqc_b200.kernels import (gate_residual, gated_linear_scan, gated_linear_step,  # noqa: E402
                                  norm_gate_residual, residual_norm)
from mambaqc_b200.models import (GatedRecurrentBlock, HybridMamba2,  # noqa: E402
                                 QuaternionMamba2Block)
from mambaqc_b200.optim import AdamW  # noqa: E402
from mambaqc_b200.training import data_parallel, train_step  # noqa: E402

V, DM = 61, 32


@pytest.fixture(autouse=True)
def _full_precision_products():
    prev = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    yield
    torch.backends.cuda.matmul.allow_tf32 = prev


def _block_ref(p, n, sharpness=8.0):
    """(y, z) of GatedRecurrentBlock from its parameters, step by step."""
    di = p["Lambda"].shape[0]
    xz = F.linear(n, p["in_proj.weight"])
    w = p["conv1d.conv.weight"]
    conv = F.conv1d(F.pad(xz[..., :di].transpose(1, 2), (w.shape[-1] - 1, 0)), w,
                    p["conv1d.conv.bias"], groups=di).transpose(1, 2)
    u = F.silu(conv)
    r, i = F.linear(u, p["gate_proj.weight"], p["gate_proj.bias"]).chunk(2, -1)
    log_a = -sharpness * F.softplus(p["Lambda"]) * torch.sigmoid(r)
    h, hs = torch.zeros_like(u[:, 0]), []
    for t in range(u.shape[1]):
        h = torch.exp(log_a[:, t]) * h + \
            torch.sqrt(-torch.expm1(2 * log_a[:, t])) * torch.sigmoid(i[:, t]) * u[:, t]
        hs.append(h)
    return F.linear(torch.stack(hs, 1), p["out_proj.weight"]), xz[..., di:]


def _norm_ref(u, w, kind):
    if kind == "layer":
        u = u - u.mean(-1, keepdim=True)
    return u / torch.sqrt(u.square().mean(-1, keepdim=True) + 1e-5) * w


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_loss_and_gradients_match_64_bits(kind):
    """Two recurrent blocks; 1e-4 as for the quaternion LM's gradients (fp32 products
    summed in another order, through two layers)."""
    torch.manual_seed(0)
    lm = HybridMamba2(V, d_model=DM, n_layers=2, pattern="g", norm=kind)
    g = gen(1)
    ids, labels = (torch.randint(0, V, (2, 75), generator=g) for _ in range(2))
    q = {k: v.detach().double().requires_grad_() for k, v in lm.state_dict().items()}
    x = F.embedding(ids, q["embedding.weight"])
    n = _norm_ref(x, q["pre_norm.0"], kind)
    for k in range(2):
        pre = f"layers.{k}."
        y, z = _block_ref({a[len(pre):]: b for a, b in q.items() if a.startswith(pre)}, n)
        x = x + q[f"scale.{k}"] * torch.sigmoid(z) * _norm_ref(y, q[f"post_norm.{k}"], kind)
        n = _norm_ref(x, q[f"pre_norm.{k + 1}"], kind)
    logits = F.linear(n, q["lm_head.weight"])[..., :V]
    loss_ref = F.cross_entropy(logits.reshape(-1, V), labels.reshape(-1))
    loss_ref.backward()
    lm = lm.to(DEV)
    out = lm(ids.to(DEV), labels=labels.to(DEV))
    out["loss"].backward()
    assert out["logits"].shape == (2, 75, V)
    assert abs(out["loss"].item() - loss_ref.item()) < RTOL_F32 * loss_ref.item()
    for name, p in lm.named_parameters():
        assert rel_l2(p.grad, q[name].grad) < 1e-4, name


def test_quaternion_block_parts_join_to_its_forward():
    torch.manual_seed(0)
    blk = QuaternionMamba2Block(DM, d_state=8).to(DEV)
    x = torch.randn(2, 30, DM, generator=gen(2)).to(DEV)
    with torch.no_grad():
        y, z, h = blk.mix(x)
        out, h2 = blk(x, return_ssm_state=True)
        assert torch.equal(gate_residual(x, z, y), out) and torch.equal(h, h2)


def test_checkpointing_matches_plain_backward():
    torch.manual_seed(0)
    lm = HybridMamba2(V, d_model=DM, n_layers=3, pattern="gq", d_state=8).to(DEV)
    ids = torch.randint(0, V, (2, 40), generator=gen(3)).to(DEV)
    grads = []
    for on in (False, True):
        lm.zero_grad(set_to_none=True)
        lm.gradient_checkpointing = on
        lm.train()
        lm(ids, labels=ids)["loss"].backward()
        grads.append({n: p.grad.clone() for n, p in lm.named_parameters()})
    for n in grads[0]:
        assert rel_l2(grads[1][n], grads[0][n]) < RTOL_F32, n


def test_block_step_matches_forward():
    torch.manual_seed(0)
    blk = GatedRecurrentBlock(DM).to(DEV)
    x = torch.randn(2, 20, DM, generator=gen(7)).to(DEV)
    with torch.no_grad():
        full_y, full_z = blk(x)
        for start in (1, 2, 5):
            _, _, cache = blk.mix_prefill(x[:, :start])
            for t in range(start, 20):
                y, z = blk.mix_step(x[:, t], cache)
                assert rel_l2(y, full_y[:, t]) < 2 * RTOL_F32, t
                assert rel_l2(z, full_z[:, t]) < RTOL_F32, t


def test_cached_generation_matches_full_recompute():
    torch.manual_seed(0)
    lm = HybridMamba2(V, d_model=DM, n_layers=3, pattern="gq", d_state=8).to(DEV)
    prompt = torch.randint(0, V, (2, 6), generator=gen(8)).to(DEV)
    a = lm.generate(prompt, max_new_tokens=12, top_k=1)
    b = lm.generate(prompt, max_new_tokens=12, top_k=1, use_cache=True)
    assert torch.equal(a, b)


@pytest.mark.parametrize("pattern", ["g", "gq"])
@pytest.mark.parametrize("bits", [32, 8])
def test_training_steps_reduce_the_loss(pattern, bits):
    """The harness on one repeated batch (bf16 autocast, checkpointed blocks, clipping in
    the optimizer's step): the loss falls, as the quaternion LM's test asks."""
    torch.manual_seed(0)
    lm = data_parallel(HybridMamba2(V, d_model=DM, n_layers=2, pattern=pattern,
                                    d_state=8).to(DEV))
    opt = AdamW(lm.parameters(), lr=3e-3, state_bits=bits)
    seq = torch.randint(0, V, (4, 65), generator=gen(5)).to(DEV)
    losses = [train_step(lm, opt, seq[:, :-1], seq[:, 1:]).item() for _ in range(30)]
    assert all(torch.isfinite(torch.tensor(losses)))
    assert losses[-1] < 0.8 * losses[0], losses


def test_refusals():
    with pytest.raises(AssertionError, match="pattern"):
        HybridMamba2(V, d_model=DM, n_layers=2, pattern="gx")
    with pytest.raises(AssertionError, match="norm"):
        HybridMamba2(V, d_model=DM, n_layers=2, norm="batch")


def test_prefill_projects_the_prompt_once():
    torch.manual_seed(0)
    block = GatedRecurrentBlock(DM).to(DEV)
    x = torch.randn(2, 9, DM, generator=gen(3)).to(DEV)
    calls = []
    block.in_proj.register_forward_hook(lambda *_: calls.append(1))
    with torch.no_grad():
        y, z, cache = block.mix_prefill(x)
        assert len(calls) == 1
        want = block.mix(x)
        x_in = block.in_proj(x)[..., : block.d_inner]
    for a, b in zip((y, z, cache["h"]), want):
        assert torch.equal(a, b)
    assert torch.equal(cache["conv"], x_in[:, -(block.d_conv - 1):])


def test_operators_in_a_captured_graph():
    """Recurrence, its one-token form and the norms, forward, replay on new inputs from a
    CUDA graph with the bits of the calls."""
    b, t, d = 2, 300, 64
    g = gen(17)
    lam = torch.randn(d, generator=g).to(DEV) - 4
    w = torch.rand(d, generator=g).to(DEV) + 0.5
    x, r, i, z = (torch.randn(b, t, d, generator=g).to(DEV) for _ in range(4))
    h = torch.zeros(b, d, device=DEV)

    def run(state):
        y, h_T = gated_linear_scan(x, r, i, lam, return_final_state=True)
        out, n = norm_gate_residual(x, y, z, w, w, next_weight=w)
        state.copy_(h_T)
        step = gated_linear_step(x[:, 0], r[:, 0], i[:, 0], lam, state)
        return y, out, n, residual_norm(out, w), step

    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(h)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = run(h)
        for k in range(2):
            for v in (x, r, i, z):
                v.copy_(torch.randn(b, t, d, generator=g))
            graph.replay()
            want = run(torch.zeros(b, d, device=DEV))
            for a, e in zip(got, want):
                assert torch.equal(a, e), k
