"""The memory sublayer of MemoryTransformerBlock (memory_transformer/memory_block.py:549-558,
variant A; variant B runs the same lines at :578-587):

    residual = hidden_states
    hidden_states = self.memory_layernorm(hidden_states)
    mem_output, _ = self.memory_attn(hidden_states, memory, token_routing_state=..., ...)
    hidden_states = residual + mem_output

Here the norm (RMSNorm of memory_block.py:18-28, or nn.LayerNorm) is one HIP row kernel that
writes its output straight in the q projection's dtype, and the residual add is the
accumulator input of the o_proj GEMM.  Parameter names are the block's:
``memory_layernorm.weight`` (``.bias`` for LayerNorm) and ``memory_attn.{q,k,v,o}_proj.weight``.
"""

from __future__ import annotations

from typing import Any, Dict, Optional

import torch
import torch.nn as nn

from . import ops
from .memory_attention import MemoryCrossAttention
from ._half import float16_via_float32


class RMSNorm(nn.Module):
    """memory_block.py:18-28: y = x / sqrt(mean(x^2) + eps) * weight, on the HIP row kernel."""

    def __init__(self, dim: int, eps: float = 1e-6):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim))

    def forward(self, x: torch.Tensor, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        return ops.row_norm(x, self.weight, None, self.eps, "rms", out_dtype)


def _norm_of(norm: nn.Module):
    """(weight, bias, eps, kind) of a block's norm."""
    if isinstance(norm, RMSNorm):
        return norm.weight, None, norm.eps, "rms"
    if isinstance(norm, nn.LayerNorm) and norm.weight is not None and len(norm.normalized_shape) == 1:
        return norm.weight, norm.bias, norm.eps, "layer"
    raise ValueError(f"expected RMSNorm or nn.LayerNorm with a weight over the last dim, got {norm}")


class MemorySublayer(nn.Module):
    """``residual + memory_attn(memory_layernorm(hidden_states))`` of MemoryTransformerBlock.

    Constructor arguments follow the block's (memory_block.py:431-499): ``hidden_dim``,
    ``num_heads``, ``num_kv_heads``, ``use_rms_norm``, ``norm_eps``, ``memory_dim``,
    ``wo_init_zero``, ``gradient_checkpointing``.  ``forward`` takes the memory arguments of
    MemoryCrossAttention.forward (dense ``memory``, ``token_routing_state`` or the fused
    ``routed_memory_state``) and returns the new hidden states.

    Options without a reference counterpart: ``post_norm`` puts a norm (``post_layernorm``) behind the attention,
    ``gate`` a learned gate ("scalar" or "channel", parameter ``gate``, starting at ``gate_init``) on what is added, and
    ``residual_scale`` scales the stream it is added to: hidden = residual_scale * hidden + gate * norm(attention).
    ``forward(..., next_norm=module)`` also returns the next sublayer's norm of the new hidden states, (hidden, normed),
    from the same pass; ``normed=`` takes such rows in place of this sublayer's own norm, and ``gate=`` a gate of
    the caller's own, one per row (..., 1) or per element, in place of the parameter."""

    def __init__(self, hidden_dim: int, num_heads: int, num_kv_heads: Optional[int] = None,
                 use_rms_norm: bool = True, norm_eps: float = 1e-6, memory_dim: Optional[int] = None,
                 wo_init_zero: bool = True, gradient_checkpointing: bool = False, post_norm: bool = False,
                 gate: Optional[str] = None, gate_init: float = 1.0, residual_scale: float = 1.0):
        super().__init__()
        if gate not in (None, "scalar", "channel"):
            raise ValueError(f"gate must be None, 'scalar' or 'channel', got {gate!r}")
        self.residual_scale = float(residual_scale)
        self.post_layernorm = None
        if post_norm:
            self.post_layernorm = (RMSNorm(hidden_dim, norm_eps) if use_rms_norm
                                   else nn.LayerNorm(hidden_dim, eps=norm_eps))
        self.gate = None if gate is None else nn.Parameter(torch.full((1 if gate == "scalar" else hidden_dim,),
                                                                      float(gate_init)))
        self.use_rms_norm = bool(use_rms_norm)
        self.memory_layernorm = RMSNorm(hidden_dim, norm_eps) if use_rms_norm else nn.LayerNorm(hidden_dim,
                                                                                                  eps=norm_eps)
        self.memory_attn = MemoryCrossAttention(hidden_dim, num_heads, num_kv_heads, memory_dim=memory_dim,
                                                wo_init_zero=wo_init_zero,
                                                gradient_checkpointing=gradient_checkpointing)
        # memory_layernorm folded into the q projection's GEMM where the shapes allow it
        # (ops.norm_linear_supported); False runs the norm kernel ahead of the projection
        self.fuse_norm = True

    @float16_via_float32
    def forward(self, hidden_states: torch.Tensor, memory: Optional[torch.Tensor] = None,
                token_routing_state: Optional[Dict[str, Any]] = None, token_routing_kernel_version: str = "v2",
                routed_memory_state: Optional[Dict[str, Any]] = None, *, normed: Optional[torch.Tensor] = None,
                next_norm: Optional[nn.Module] = None, gate: Optional[torch.Tensor] = None):
        attn = self.memory_attn
        cdt = attn.q_proj.weight.dtype
        if cdt not in (torch.float32, torch.bfloat16):
            raise ValueError(f"memory projections in {cdt}: the HIP kernels take float32 or bfloat16")
        ln = self.memory_layernorm
        kind = "rms" if self.use_rms_norm else "layer"
        bias = None if self.use_rms_norm else ln.bias
        if normed is not None:
            pre = attn.attention_preproj(normed.to(cdt), memory, token_routing_state, token_routing_kernel_version,
                                         routed_memory_state)
        elif self.fuse_norm and ops.norm_linear_supported(hidden_states, attn.q_proj.weight):
            # only the q projection reads the normalised rows: the norm runs inside its GEMM
            pre = attn.attention_preproj(hidden_states, memory, token_routing_state, token_routing_kernel_version,
                                         routed_memory_state, query_norm=(ln.weight, bias, ln.eps, kind))
        else:
            x = ops.row_norm(hidden_states, ln.weight, bias, ln.eps, kind, cdt)
            pre = attn.attention_preproj(x, memory, token_routing_state, token_routing_kernel_version,
                                         routed_memory_state)
        gate = self.gate if gate is None else gate
        if self.post_layernorm is None and gate is None and next_norm is None and self.residual_scale == 1.0:
            return ops.linear_residual(pre, attn.o_proj.weight, hidden_states)
        return self.join(ops.linear(pre, attn.o_proj.weight), hidden_states, next_norm, gate)

    def join(self, mem_output: torch.Tensor, hidden_states: torch.Tensor, next_norm: Optional[nn.Module] = None,
             gate: Optional[torch.Tensor] = None):
        """What follows the attention's output projection (``ops.gated_residual_norm``): the new hidden states, or
        with ``next_norm`` (hidden, normed).  A decode step calls it on ``memory_decode_step``'s result."""
        gate = self.gate if gate is None else gate
        w1, b1, eps, kind = (None, None, 1e-6, "rms") if self.post_layernorm is None else _norm_of(self.post_layernorm)
        w2, b2, eps2, kind2 = (None, None, eps, kind) if next_norm is None else _norm_of(next_norm)
        h, n = ops.gated_residual_norm(mem_output, hidden_states, post_weight=w1, post_bias=b1, gate=gate,
                                       residual_scale=self.residual_scale, pre_weight=w2, pre_bias=b2, eps=eps, norm=kind,
                                       pre_eps=eps2, pre_norm=kind2, out_dtype=self.memory_attn.q_proj.weight.dtype)
        return h if next_norm is None else (h, n)
