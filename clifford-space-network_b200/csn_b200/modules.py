"""nn.Module front ends of the block kernels, parameter-compatible with torch.nn, and the gated
recurrent and linear-attention blocks."""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import ops


class LayerNorm(nn.LayerNorm):
    """nn.LayerNorm (same parameters, state_dict keys and eps) computed by the CUDA LayerNorm
    kernels (ops.layer_norm) for one normalised axis of C % 4 == 0, C <= 1024 features with affine
    weight and bias; other shapes go to F.layer_norm, and keep what only that has: second
    derivatives, forward-mode tangents, tracing, and a float32 result under autocast."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        C = x.shape[-1]
        if (len(self.normalized_shape) == 1 and self.weight is not None and self.bias is not None
                and ops.layer_norm_supported(C)):
            return ops.layer_norm(x, self.weight, self.bias, self.eps)
        return F.layer_norm(x, self.normalized_shape, self.weight, self.bias, self.eps)


class BlockLayerNorm(LayerNorm):
    """LayerNorm of the gated recurrent and linear-attention blocks, whose other operators are
    differentiable once and not traced either: bfloat16 and float16 features on CUDA go to
    ops.layer_norm at every width."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if (x.is_cuda and x.dtype in (torch.bfloat16, torch.float16) and len(self.normalized_shape) == 1
                and self.weight is not None and self.bias is not None):
            return ops.layer_norm(x, self.weight, self.bias, self.eps)
        return super().forward(x)


def causal_conv_input(ln: nn.LayerNorm, conv: nn.Conv1d, x: torch.Tensor) -> torch.Tensor:
    """x_conv = silu(conv(ln(x).transpose(1, 2))[:, :, :T].transpose(1, 2)) of the blocks
    (python/clifford_cl6.py:140-142), as the fused CUDA kernels when the layers have the blocks'
    form (affine LayerNorm over C; depthwise, bias, stride 1, dilation 1, left padding K - 1
    conv) and the sizes fit them; otherwise the same chain of library layers."""
    T = x.shape[1]
    C = x.shape[-1]
    K = conv.kernel_size[0]
    if (x.dim() == 3 and len(ln.normalized_shape) == 1 and ln.weight is not None and ln.bias is not None
            and conv.groups == C == conv.in_channels == conv.out_channels and conv.bias is not None
            and conv.stride == (1,) and conv.dilation == (1,) and conv.padding == (K - 1,)
            and conv.padding_mode == "zeros" and ops.ln_conv_silu_supported(C, K)):
        return ops.ln_conv_silu(x, ln.weight, ln.bias, ln.eps, conv.weight, conv.bias)
    return F.silu(conv(ln(x).transpose(1, 2))[:, :, :T].transpose(1, 2))


def generator_inputs(x: torch.Tensor, biv_proj: nn.Linear, gamma_proj: nn.Linear, time_proj: nn.Linear,
                     omega_scale: torch.Tensor, dt_base: float):
    """(biv [..., N*K], gamma [..., N], dt [..., HT]) of the blocks' projections
    (python/clifford_cl6.py:144-155: biv_proj(x) * omega_scale, softplus(gamma_proj(x)),
    softplus(time_head.proj(x)) * dt_base) as ONE GEMM over the concatenated weights and the
    CUDA projection epilogue; the parameters stay the three nn.Linear layers'."""
    N = gamma_proj.out_features
    HT = time_proj.out_features
    K = biv_proj.out_features // N
    W = torch.cat([biv_proj.weight, gamma_proj.weight, time_proj.weight], 0)
    b = torch.cat([biv_proj.bias, gamma_proj.bias, time_proj.bias], 0)
    raw = ops.linear(x, W, b)
    return ops.projection_epilogue(raw, omega_scale, dt_base, N, K, HT)


# ------------------------------------------------------------- gated recurrent block
class DropoutAdd(nn.Module):
    """residual + dropout(x, p) in training, residual + x otherwise (residual None: without it), by
    ops.dropout_add.  Each call in training draws its (seed, offset) from torch's generator of x's
    device, as nn.Dropout draws its mask: it follows torch.manual_seed, a captured training step draws
    a new mask at every replay, and a forward pass that is run again for activation checkpointing,
    which puts the generator back first, has the mask of the first run."""

    def __init__(self, p: float = 0.1):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"DropoutAdd: 0 <= p <= 1 expected, got {p}")
        self.p = p

    @staticmethod
    def numbers(device) -> torch.Tensor:
        """(seed, offset) of a call, from the device's generator."""
        return torch.randint(1 << 62, (2,), device=device)

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        if not self.training or self.p == 0.0:
            return x if residual is None else residual + x
        return ops.dropout_add(x, residual, self.p, self.numbers(x.device))


class GatedRecurrence(nn.Module):
    """The mixer of a gated recurrent block: one projection of x gives forget logits, inputs and output
    gates, ops.gated_scan runs the recurrence over them as they lie, and a projection goes back.  The
    channels' forget biases spread their memory from 2 steps to about 1000."""

    def __init__(self, d_model: int, d_inner: Optional[int] = None):
        super().__init__()
        self.d_inner = d_model if d_inner is None else d_inner
        self.in_proj = nn.Linear(d_model, 3 * self.d_inner)
        self.out_proj = nn.Linear(self.d_inner, d_model)
        with torch.no_grad():
            self.in_proj.bias[:self.d_inner] = torch.linspace(0.0, 7.0, self.d_inner)

    def init_state(self, batch_size: int, device=None) -> torch.Tensor:
        device = device if device is not None else self.in_proj.weight.device
        return torch.zeros(batch_size, self.d_inner, device=device, dtype=torch.float32)

    def forward(self, x: torch.Tensor, h0: Optional[torch.Tensor] = None, cu_seqlens: Optional[torch.Tensor] = None):
        """x [B, T, d_model], or [L, d_model] packed with cu_seqlens -> (out, float32 states [B, d_inner])."""
        f, v, gate = ops.linear(x, self.in_proj.weight, self.in_proj.bias).split(self.d_inner, -1)
        y, h = ops.gated_scan(f, v, h0=h0, gate=gate, cu_seqlens=cu_seqlens)
        return ops.linear(y, self.out_proj.weight, self.out_proj.bias), h

    @torch.no_grad()
    def step(self, x_t: torch.Tensor, h: torch.Tensor) -> torch.Tensor:
        """One token for each stream: x_t [B, d_model]; the state h [B, d_inner] is advanced in place."""
        f, v, gate = self.in_proj(x_t).split(self.d_inner, -1)
        return self.out_proj(ops.gated_step(f, v, h, gate=gate))


class GatedFeedForward(nn.Module):
    """w_down(silu(w_gate x) * w_up x) with the parameters of GeometricGatedLinearUnit
    (python/clifford_model.py:29-43): 16-bit layers by ops.silu_gated_linear, float32 ones as that
    module computes them."""

    def __init__(self, d_model: int, d_ffn: Optional[int] = None):
        super().__init__()
        d_ffn = 2 * d_model if d_ffn is None else d_ffn
        self.w_gate = nn.Linear(d_model, d_ffn, bias=False)
        self.w_up = nn.Linear(d_model, d_ffn, bias=False)
        self.w_down = nn.Linear(d_ffn, d_model, bias=False)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.dtype == torch.float32:
            y = ops.silu_gate(ops.linear(x, torch.cat([self.w_gate.weight, self.w_up.weight], 0)))
        else:
            y = ops.silu_gated_linear(x, self.w_gate.weight, self.w_up.weight)
        return ops.linear(y, self.w_down.weight)


class GatedRecurrentBlock(nn.Module):
    """x + drop(mixer(ln_1(x))), then + drop(ffn(ln_2(.))): the channelwise recurrence and the gated
    feed-forward product as a residual block, trained with forward() and advanced one token at a time
    with step()."""

    def __init__(self, d_model: int, d_inner: Optional[int] = None, d_ffn: Optional[int] = None, dropout: float = 0.0):
        super().__init__()
        self.ln_1, self.ln_2 = BlockLayerNorm(d_model), BlockLayerNorm(d_model)
        self.mixer = GatedRecurrence(d_model, d_inner)
        self.ffn = GatedFeedForward(d_model, d_ffn)
        self.drop_1, self.drop_2 = DropoutAdd(dropout), DropoutAdd(dropout)

    def init_state(self, batch_size: int, device=None) -> torch.Tensor:
        return self.mixer.init_state(batch_size, device)

    def forward(self, x: torch.Tensor, h0: Optional[torch.Tensor] = None, cu_seqlens: Optional[torch.Tensor] = None):
        """x [B, T, d_model], or [L, d_model] packed with cu_seqlens -> (out, states after the last steps)."""
        mixed, h = self.mixer(self.ln_1(x), h0, cu_seqlens)
        x = self.drop_1(mixed, x)
        return self.drop_2(self.ffn(self.ln_2(x)), x), h

    @torch.no_grad()
    def step(self, x_t: torch.Tensor, h: torch.Tensor) -> torch.Tensor:
        """One token, without dropout: x_t [B, d_model] -> out [B, d_model]; h is advanced in place."""
        x_t = x_t + self.mixer.step(self.ln_1(x_t), h)
        return x_t + self.ffn(self.ln_2(x_t))


# ------------------------------------------------------------- linear-attention block
class LinearAttention(nn.Module):
    """The mixer of a linear-attention block: one projection of x gives queries, keys and values, ops.linear_attention
    runs over them as they lie, each head's output is normalised, and a projection goes back.  The heads'
    memories run from 2^5 to 2^12 steps and are not trained (a buffer, float32 whatever the layer's type)."""

    def __init__(self, d_model: int, num_heads: int, num_kv_heads: Optional[int] = None, head_dim: Optional[int] = None):
        super().__init__()
        self.num_heads = num_heads
        self.num_kv_heads = num_heads if num_kv_heads is None else num_kv_heads
        self.head_dim = d_model // num_heads if head_dim is None else head_dim
        if num_heads < 1 or self.num_kv_heads < 1 or num_heads % self.num_kv_heads or not 1 <= self.head_dim <= 128:
            raise ValueError(f"LinearAttention: num_kv_heads has to divide num_heads and heads have 1 to 128 places, got "
                             f"{self.num_kv_heads}, {num_heads} and {self.head_dim}")
        self.in_proj = nn.Linear(d_model, (num_heads + 2 * self.num_kv_heads) * self.head_dim, bias=False)
        self.norm = BlockLayerNorm(self.head_dim)
        self.out_proj = nn.Linear(num_heads * self.head_dim, d_model, bias=False)
        self.register_buffer("log_decay", self._decays(), persistent=False)

    def _decays(self, **kw) -> torch.Tensor:
        return torch.log1p(-torch.exp2(-torch.linspace(5.0, 12.0, self.num_heads, dtype=torch.float32, **kw)))

    def _apply(self, fn, *args, **kwargs):
        decay = self.log_decay
        super()._apply(fn, *args, **kwargs)
        # .bfloat16() and the like change the layer's type, not the decays': 16 bits have no number next to 1 - 2^-12.
        # .to_empty() leaves them as well, and makes those of a module that had no memory: no state_dict brings them.
        device = self.log_decay.device
        if decay.is_meta and device.type != "meta":
            decay = self._decays(device="cpu")
        self.log_decay = decay.to(device)
        return self

    def init_state(self, batch_size: int, device=None) -> torch.Tensor:
        device = device if device is not None else self.in_proj.weight.device
        return torch.zeros(batch_size, self.num_heads, self.head_dim, self.head_dim, device=device, dtype=torch.float32)

    def _heads(self, x: torch.Tensor):
        h, hk, d = self.num_heads, self.num_kv_heads, self.head_dim
        q, k, v = ops.linear(x, self.in_proj.weight).split([h * d, hk * d, hk * d], -1)
        return q.unflatten(-1, (h, d)), k.unflatten(-1, (hk, d)), v.unflatten(-1, (hk, d))

    def forward(self, x: torch.Tensor, s0: Optional[torch.Tensor] = None, cu_seqlens: Optional[torch.Tensor] = None):
        """x [B, T, d_model], or [L, d_model] packed with cu_seqlens -> (out, float32 states [B, H, D, D])."""
        o, s = ops.linear_attention(*self._heads(x), self.log_decay, s0=s0, cu_seqlens=cu_seqlens)
        return ops.linear(self.norm(o).flatten(-2), self.out_proj.weight), s

    @torch.no_grad()
    def step(self, x_t: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
        """One token for each stream: x_t [B, d_model]; the states s [B, H, D, D] are advanced in place."""
        o = ops.linear_attention_step(*self._heads(x_t), self.log_decay, s)
        return ops.linear(self.norm(o).flatten(-2), self.out_proj.weight)


class LinearAttentionBlock(nn.Module):
    """x + drop(mixer(ln_1(x))), then + drop(ffn(ln_2(.))): linear attention and the gated feed-forward product as a residual
    block, trained with forward() and advanced one token at a time with step()."""

    def __init__(self, d_model: int, num_heads: int, num_kv_heads: Optional[int] = None, head_dim: Optional[int] = None,
                 d_ffn: Optional[int] = None, dropout: float = 0.0):
        super().__init__()
        self.ln_1, self.ln_2 = BlockLayerNorm(d_model), BlockLayerNorm(d_model)
        self.mixer = LinearAttention(d_model, num_heads, num_kv_heads, head_dim)
        self.ffn = GatedFeedForward(d_model, d_ffn)
        self.drop_1, self.drop_2 = DropoutAdd(dropout), DropoutAdd(dropout)

    def init_state(self, batch_size: int, device=None) -> torch.Tensor:
        return self.mixer.init_state(batch_size, device)

    def forward(self, x: torch.Tensor, s0: Optional[torch.Tensor] = None, cu_seqlens: Optional[torch.Tensor] = None):
        """x [B, T, d_model], or [L, d_model] packed with cu_seqlens -> (out, states after the last steps)."""
        mixed, s = self.mixer(self.ln_1(x), s0, cu_seqlens)
        x = self.drop_1(mixed, x)
        return self.drop_2(self.ffn(self.ln_2(x)), x), s

    @torch.no_grad()
    def step(self, x_t: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
        """One token, without dropout: x_t [B, d_model] -> out [B, d_model]; s is advanced in place."""
        x_t = x_t + self.mixer.step(self.ln_1(x_t), s)
        return x_t + self.ffn(self.ln_2(x_t))
