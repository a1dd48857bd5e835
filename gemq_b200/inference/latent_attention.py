"""DeepSeek-V2's attention on the latent operators, beside ``QuantFusedDeepseekV2MoEBlock``.

The reference leaves this part of the layer to the host model (gemq/inference/patch.py:104-124); its linears are what the loader makes
of them: ``nn.Linear`` or ``QuantLinear`` (gemq/quantize.py:333-343 quantises attention linears).
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
from torch import Tensor

from ..kernels import dequantize
from ..kernels.latent_attention import NOPE, ROPE, VALUE, latent_append, latent_decode, latent_decode_shared, latent_prefill
from .latent_cache import LatentPlan, PagedLatentCache
from .quant_linear import QuantLinear


def _weight(linear, dtype: torch.dtype) -> Tensor:
    """``[out, in]`` of a linear, de-quantised if it is quantised."""
    if isinstance(linear, QuantLinear):
        return dequantize(linear.W_q, linear.scales, linear.zeros, linear.W_nbits, linear.group_size)[:linear.in_features].t().to(dtype)
    return linear.weight.to(dtype)


def _refresh(layer: "LatentAttention", _) -> None:  # a function of the module: the layer can be pickled
    layer.refresh()


class LatentAttention(nn.Module):
    """``q_proj`` (any module from hidden states to ``heads * 192``), ``kv_a_proj`` (to ``rank + 64``), the latent's norm weight and ``kv_b_proj``
    (from ``rank`` to ``heads * 256``), ``o_proj`` (from ``heads * 128``).  Prompts are attended to in the expanded form, decoded tokens
    in the absorbed one, which needs the two halves of ``kv_b_proj``'s weight by themselves: they are made of it here, and again when a
    state is loaded (``refresh`` after any other change)."""

    def __init__(self, q_proj: nn.Module, kv_a_proj: nn.Module, norm_weight: Tensor, eps: float, kv_b_proj: nn.Module, o_proj: nn.Module,
                 heads: int, inv_freq: Tensor, scale: Optional[float] = None, rope_scale: float = 1.0):
        super().__init__()
        self.q_proj, self.kv_a_proj, self.kv_b_proj, self.o_proj = q_proj, kv_a_proj, kv_b_proj, o_proj
        self.heads, self.eps, self.rope_scale = heads, eps, rope_scale
        self.scale = (NOPE + ROPE) ** -0.5 if scale is None else scale
        rank = norm_weight.shape[0]
        if getattr(kv_b_proj, "bias", None) is not None:
            raise ValueError("the absorbed form has no place for a bias of kv_b_proj")
        if tuple(inv_freq.shape) != (ROPE // 2,):
            raise ValueError(f"inv_freq must be [32], not {list(inv_freq.shape)}")
        self.norm_weight = nn.Parameter(norm_weight.detach().contiguous(), requires_grad=False)
        self.inv_freq = inv_freq.detach().float().contiguous()  # no buffer: a change of the module's type leaves it in 32 bits
        self.rank = rank
        self.refresh()
        self.register_load_state_dict_post_hook(_refresh)

    def refresh(self) -> None:
        """The halves of ``kv_b_proj``'s weight as it is now."""
        w = _weight(self.kv_b_proj, self.norm_weight.dtype)
        if tuple(w.shape) != (self.heads * (NOPE + VALUE), self.rank):
            raise ValueError(f"kv_b_proj must have a weight of {[self.heads * (NOPE + VALUE), self.rank]}, not {list(w.shape)}")
        w = w.reshape(self.heads, NOPE + VALUE, self.rank)
        self.register_buffer("w_keys", w[:, :NOPE].detach().contiguous(), persistent=False)                    # [heads, 128, rank]
        self.register_buffer("w_values", w[:, NOPE:].detach().transpose(1, 2).contiguous(), persistent=False)  # [heads, rank, 128]

    @classmethod
    def from_hf(cls, config, attn, inv_freq: Optional[Tensor] = None, scale: Optional[float] = None,
                rope_scale: float = 1.0) -> "LatentAttention":
        """From a Hugging Face ``DeepseekV2Attention``.  Where the configuration scales its rotation (yarn), the frequencies, the scale of the
        scores and that of the rotation are the caller's to give."""
        if (config.qk_nope_head_dim, config.qk_rope_head_dim, config.v_head_dim) != (NOPE, ROPE, VALUE):
            raise ValueError("the kernels take heads of 128 + 64 numbers and values of 128")
        rope = getattr(config, "rope_parameters", None) or getattr(config, "rope_scaling", None) or {}
        if rope.get("rope_type", rope.get("type", "default" if "rope_theta" in rope or not rope else None)) != "default" and (
                inv_freq is None or scale is None):
            raise ValueError("the configuration scales its rotation: give inv_freq and scale (and rope_scale)")
        norm = attn.kv_a_layernorm
        if inv_freq is None:
            theta = getattr(config, "rope_theta", None) or rope["rope_theta"]
            inv_freq = 1.0 / theta ** (torch.arange(0, ROPE, 2, dtype=torch.float32, device=norm.weight.device) / ROPE)
        q_proj = attn.q_proj if getattr(config, "q_lora_rank", None) is None else nn.Sequential(attn.q_a_proj, attn.q_a_layernorm, attn.q_b_proj)
        eps = getattr(norm, "variance_epsilon", getattr(norm, "eps", None))
        return cls(q_proj, attn.kv_a_proj_with_mqa, norm.weight, eps, attn.kv_b_proj, attn.o_proj, config.num_attention_heads, inv_freq, scale,
                   rope_scale)

    @torch.no_grad()
    def forward(self, hidden: Tensor, cache: PagedLatentCache, layer: int, plan: LatentPlan) -> Tensor:
        """``hidden [tokens, D]`` in the order of the plan -> ``[tokens, D]``; their rows are stored in the cache's layer."""
        tokens, H, rank = hidden.shape[0], self.heads, self.rank
        pages = cache.layer(layer)
        if self.inv_freq.device != hidden.device:
            self.inv_freq = self.inv_freq.to(hidden.device)
        q = self.q_proj(hidden).view(tokens, H, NOPE + ROPE)
        q_rope, rows = latent_append(self.kv_a_proj(hidden), q[..., NOPE:], self.norm_weight, self.eps, self.inv_freq, plan.positions, plan.slots,
                                     pages, self.rope_scale)
        q_nope = q[..., :NOPE]
        if not plan.steps:
            if plan.rows is not None:  # rows from before this step come from their pages
                rows = pages.view(-1, rank + ROPE)[plan.rows]
            kv = self.kv_b_proj(rows[:, :rank]).view(-1, H, NOPE + VALUE)
            out, _ = latent_prefill(q_nope, q_rope, kv, rows[:, rank:], plan.cu_q, plan.cu_k, self.scale)
            return self.o_proj(out.reshape(tokens, H * VALUE))
        # absorbed: one [tokens, rank] block a head, seen as [sequences, steps, heads, rank]
        batch = plan.lens.shape[0]
        q_latent = torch.matmul(q_nope.transpose(0, 1), self.w_keys).view(H, batch, plan.steps, rank).permute(1, 2, 0, 3)
        q_rope = q_rope.view(batch, plan.steps, H, ROPE)
        if plan.starts is None:
            out, _ = latent_decode(q_latent, q_rope, pages, plan.table, plan.lens, self.scale)
        else:
            out, _ = latent_decode_shared(q_latent, q_rope, pages, plan.table, plan.lens, plan.prefix_table, plan.prefix_lens, plan.starts,
                                          self.scale)
        out = torch.matmul(out.view(tokens, H, rank).transpose(0, 1), self.w_values)
        return self.o_proj(out.transpose(0, 1).reshape(tokens, H * VALUE))
