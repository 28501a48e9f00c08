"""A normed stack of gated recurrent and quaternion blocks, and its recurrent block.

``GatedRecurrentBlock`` mixes time with the real-valued gated linear recurrence
(``kernels.gated_linear_scan``) where ``QuaternionMamba2Block`` uses the quaternion
scan. Its projections have 5 d_inner d_model + 2 d_inner^2 weights or so, against the
8 d_state d_inner^2 of the quaternion block's B and C projections alone.

``HybridMamba2`` stacks both kinds by a pattern, with a norm in front of and behind
each block, the output gate and a learned residual scale in one kernel
(``kernels.norm_gate_residual``): the last block's call also applies the final norm.
The residual stream stays in the embedding's type (fp32 under bf16 autocast). The
reference has neither the block nor the norms; its LM is ``QuaternionMamba2``.
"""

from __future__ import annotations

import math

import torch
import torch.nn as nn
import torch.utils.checkpoint as ckpt

from mambaqc_b200.kernels.block_fused import causal_conv1d_silu
from mambaqc_b200.kernels.gated_scan import gated_linear_scan, gated_linear_step
from mambaqc_b200.kernels.norm_gate import norm_gate_residual, residual_norm
from mambaqc_b200.layers.causal_conv1d import CausalConv1d
from mambaqc_b200.models.quaternion_mamba2 import QuaternionMamba2
from mambaqc_b200.models.quaternion_mamba2_block import QuaternionMamba2Block

__all__ = ["GatedRecurrentBlock", "HybridMamba2"]


class GatedRecurrentBlock(nn.Module):
    """[batch, seq_len, d_model] -> (y, z), both [batch, seq_len, d_model]: the block's
    output and its gate, for ``norm_gate_residual``.

    in_proj -> causal conv + SiLU -> gates r, i -> gated linear recurrence -> out_proj.
    """

    def __init__(self, d_model: int, d_conv: int = 4, expand_factor: int = 2,
                 sharpness: float = 8.0, bias: bool = False):
        super().__init__()
        self.d_model = d_model
        self.d_conv = d_conv
        self.d_inner = d_model * expand_factor
        self.sharpness = sharpness
        self.in_proj = nn.Linear(d_model, self.d_inner + d_model, bias=bias)
        self.conv1d = CausalConv1d(self.d_inner, kernel_size=d_conv, bias=True)
        self.gate_proj = nn.Linear(self.d_inner, 2 * self.d_inner, bias=True)
        # decay between 0.9 and 0.999 a step where the recurrence gate is open
        decay = 0.9 + 0.099 * torch.rand(self.d_inner)
        self.Lambda = nn.Parameter(torch.log(torch.expm1(-torch.log(decay) / sharpness)))
        self.out_proj = nn.Linear(self.d_inner, d_model, bias=bias)

    def _project(self, x: torch.Tensor):
        xz = self.in_proj(x)
        return xz[..., : self.d_inner], xz[..., self.d_inner:]

    def mix(self, x: torch.Tensor, reset: torch.Tensor | None = None):
        """(y, z, h_T). ``reset`` [B, T] marks the first token of each document of a
        packed sequence (the recurrence drops its state there; the conv still sees up
        to d_conv - 1 tokens before it)."""
        x_in, z = self._project(x)
        y, h_T = self._recur(x_in, reset)
        return y, z, h_T

    def _recur(self, x_in: torch.Tensor, reset: torch.Tensor | None = None):
        """(y, h_T) from the projected input."""
        conv = self.conv1d.conv
        x_act = causal_conv1d_silu(x_in, conv.weight, conv.bias)
        r, i = self.gate_proj(x_act).to(x_act.dtype).chunk(2, dim=-1)
        h, h_T = gated_linear_scan(x_act, r, i, self.Lambda, None, reset,
                                   sharpness=self.sharpness, return_final_state=True)
        return self.out_proj(h), h_T

    def forward(self, x: torch.Tensor, reset: torch.Tensor | None = None):
        return self.mix(x, reset)[:2]

    @torch.no_grad()
    def mix_prefill(self, x: torch.Tensor):
        """``mix`` over a prompt with the cache a continuation needs: the last d_conv - 1
        conv inputs and the fp32 state."""
        x_in, z = self._project(x)
        y, h_T = self._recur(x_in)
        k1 = self.d_conv - 1
        hist = x_in.new_zeros(x.shape[0], k1, self.d_inner)
        take = min(k1, x.shape[1])
        if take > 0:
            hist[:, k1 - take:] = x_in[:, -take:]
        return y, z, {"conv": hist, "h": h_T}

    @torch.no_grad()
    def mix_step(self, x_t: torch.Tensor, cache: dict):
        """(y, z) of one token, x_t [B, d_model], from and into ``cache``."""
        x_in, z = self._project(x_t)
        window = torch.cat([cache["conv"].to(x_in.dtype), x_in[:, None]], dim=1)
        conv = self.conv1d.conv
        x_act = causal_conv1d_silu(window, conv.weight, conv.bias)[:, -1]
        cache["conv"] = window[:, 1:].contiguous()
        r, i = self.gate_proj(x_act).to(x_act.dtype).chunk(2, dim=-1)
        h = gated_linear_step(x_act, r, i, self.Lambda, cache["h"], sharpness=self.sharpness)
        return self.out_proj(h), z

    def extra_repr(self) -> str:
        return (f"d_model={self.d_model}, d_inner={self.d_inner}, d_conv={self.d_conv}, "
                f"sharpness={self.sharpness}")


class HybridMamba2(QuaternionMamba2):
    """An LM of ``n_layers`` blocks by ``pattern``, repeated as needed: "g" a
    ``GatedRecurrentBlock``, "q" a ``QuaternionMamba2Block``. ``forward``,
    ``generate`` and the training harness are those of ``QuaternionMamba2``."""

    def __init__(self, vocab_size: int, d_model: int = 768, n_layers: int = 12,
                 pattern: str = "ggq", d_state: int = 64, d_conv: int = 4,
                 expand_factor: int = 2, norm: str = "rms", eps: float = 1e-5,
                 pad_vocab_size_multiple: int = 8, bias: bool = False, dropout: float = 0.0):
        assert pattern and set(pattern) <= {"g", "q"}, f"pattern of 'g' and 'q', got {pattern!r}"
        assert norm in ("rms", "layer"), f"norm must be 'layer' or 'rms', got {norm!r}"
        nn.Module.__init__(self)
        self.vocab_size = vocab_size
        self.d_model = d_model
        self.n_layers = n_layers
        m = pad_vocab_size_multiple
        self.vocab_size_padded = -(-vocab_size // m) * m if m > 1 else vocab_size
        self.norm, self.eps = norm, eps
        self.embedding = nn.Embedding(self.vocab_size_padded, d_model)
        self.dropout = nn.Dropout(dropout) if dropout > 0.0 else nn.Identity()
        self.layers = nn.ModuleList([
            QuaternionMamba2Block(d_model=d_model, d_state=d_state, d_conv=d_conv,
                                  expand_factor=expand_factor, bias=bias)
            if pattern[k % len(pattern)] == "q" else
            GatedRecurrentBlock(d_model=d_model, d_conv=d_conv, expand_factor=expand_factor,
                                bias=bias)
            for k in range(n_layers)])
        # pre_norm[k] is in front of layer k, pre_norm[n_layers] in front of the head
        self.pre_norm = nn.ParameterList([nn.Parameter(torch.ones(d_model))
                                          for _ in range(n_layers + 1)])
        self.post_norm = nn.ParameterList([nn.Parameter(torch.ones(d_model))
                                           for _ in range(n_layers)])
        self.scale = nn.ParameterList([
            nn.Parameter(torch.full((d_model,), 1 / math.sqrt(max(1, n_layers))))
            for _ in range(n_layers)])
        self.lm_head = nn.Linear(d_model, self.vocab_size_padded, bias=False)
        self.gradient_checkpointing = False
        self.apply(self._init_weights)

    def _first_norm(self, x: torch.Tensor) -> torch.Tensor:
        dtype = x.dtype
        if x.is_cuda and torch.is_autocast_enabled("cuda"):
            dtype = torch.get_autocast_dtype("cuda")
        return residual_norm(x, self.pre_norm[0], norm=self.norm, eps=self.eps, dtype=dtype)

    def _join(self, k: int, x, y, z):
        return norm_gate_residual(x, y, z.to(y.dtype), self.post_norm[k], self.scale[k],
                                  next_weight=self.pre_norm[k + 1], norm=self.norm, eps=self.eps)

    def _layer(self, k: int, x: torch.Tensor, n: torch.Tensor):
        y, z = self.layers[k].mix(n)[:2]
        return self._join(k, x, y, z)

    def _features(self, input_ids: torch.Tensor) -> torch.Tensor:
        x = self.dropout(self.embedding(input_ids))
        n = self._first_norm(x)
        for k in range(self.n_layers):
            if self.gradient_checkpointing and self.training and torch.is_grad_enabled():
                x, n = ckpt.checkpoint(self._layer, k, x, n, use_reentrant=False)
            else:
                x, n = self._layer(k, x, n)
        return n

    @torch.no_grad()
    def _next_logits_cached(self, input_ids: torch.Tensor, caches: list | None):
        prompt = caches is None
        x = self.embedding(input_ids if prompt else input_ids[:, -1])
        n = self._first_norm(x)
        if prompt:
            caches = []
        for k, layer in enumerate(self.layers):
            if prompt:
                y, z, c = layer.mix_prefill(n)
                caches.append(c)
            else:
                y, z = layer.mix_step(n, caches[k])
            x, n = self._join(k, x, y, z)
        if prompt:
            n = n[:, -1]
        return self.lm_head(n)[..., : self.vocab_size], caches
