"""The decoder with its projections in 8-bit integers, for inference and evaluation.

Weights are quantised once, one scale for each output channel; the input of every
projection is quantised as it is made, one scale for each token:

* the norms write their output in 8 bits (``rms_norm_q8``, ``residual_rms_norm_q8``),
* the attention output and the SwiGLU output go through ``quantize_rows``,
* QKV, o_proj, gate_up, down and the LM head are ``linear_q8`` products.

The residual stream, QK-norm + RoPE, the attention core and SwiGLU stay in bf16 on the
operators of :mod:`hackable_lm_b200.kernels`.  No counterpart in the reference, whose
model runs in bf16 only.
"""
from __future__ import annotations

import copy

import torch
import torch.nn.functional as F
from torch import nn

from . import kernels


class Int8Linear(nn.Module):
    """A bias-free projection [N, K] as int8 codes and a scale for each output channel."""

    def __init__(self, weight: torch.Tensor) -> None:
        super().__init__()
        q, scale = kernels.quantize_rows(weight.detach())
        self.register_buffer("weight", q)
        self.register_buffer("weight_scale", scale)

    def _apply(self, fn, recurse=True):
        """Moves to another device; a move to another type (``.half()``, ``.to(torch.bfloat16)``) is for
        the floating tensors around the codes, whose scales stay as they are, in fp32."""
        scale = self.weight_scale
        super()._apply(fn, recurse)
        if self.weight_scale.dtype != torch.float32:
            self.weight_scale = scale.to(self.weight_scale.device)
        return self

    def forward(self, q: torch.Tensor, scale: torch.Tensor, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        return kernels.linear_q8(q, scale, self.weight, self.weight_scale, out_dtype)

    def dequantized(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The weight that the codes stand for."""
        return kernels.dequantize_rows(self.weight, self.weight_scale, dtype)


class QuantizedBlock(nn.Module):
    def __init__(self, block: nn.Module) -> None:
        super().__init__()
        qkv = block.attn.qkv
        self.n_head, self.n_kv_head, self.head_dim = qkv.n_head, qkv.n_kv_head, qkv.head_dim
        self.eps = block.mlp.down.norm_eps
        self.rope = copy.deepcopy(qkv.rope)
        self.attention = copy.deepcopy(block.attn.attention)
        self.qkv_proj = Int8Linear(qkv.qkv_proj.weight)
        self.o_proj = Int8Linear(block.attn.out.o_proj.weight)
        self.gate_up_proj = Int8Linear(block.mlp.gate_up.gate_up_proj.weight)
        self.down_proj = Int8Linear(block.mlp.down.down_proj.weight)

    def forward(self, x: torch.Tensor, q8: torch.Tensor, scale: torch.Tensor):
        """x [B, T, C] bf16 and its norm in 8 bits -> the same after the block."""
        B, T, _ = x.shape
        qkv = self.qkv_proj(q8, scale, x.dtype)
        q, k, v = qkv.view(B, T, -1, self.head_dim).split((self.n_head, self.n_kv_head, self.n_kv_head), dim=2)
        cos, sin = self.rope(T, x.device, x.dtype)
        q, k = kernels.qk_norm_rope_triton(q, k, cos, sin, self.eps)
        y = self.attention(q, k, v).reshape(B, T, self.n_head * self.head_dim)
        branch = self.o_proj(*kernels.quantize_rows(y), x.dtype)
        x, q8, scale = kernels.residual_rms_norm_q8(x, branch, self.eps)
        h = kernels.swiglu_triton(self.gate_up_proj(q8, scale, x.dtype))
        branch = self.down_proj(*kernels.quantize_rows(h), x.dtype)
        return kernels.residual_rms_norm_q8(x, branch, self.eps)


class QuantizedLanguageModel(nn.Module):
    """``model.LanguageModel`` on 8-bit integer projections.  ``forward(idx, targets)`` returns
    what the model returns: (logits, None) without targets, else (None, mean loss over the
    targets within the vocabulary; -100 and any other are left out).  No gradients.  It holds copies: training the model
    further, or moving it, changes nothing here."""

    def __init__(self, model: nn.Module) -> None:
        super().__init__()
        for p in model.parameters():
            if not (p.is_cuda or p.is_meta):
                raise RuntimeError("quantize_int8: the 8-bit operators run only on CUDA (sm_100a) tensors")
        self.config = copy.deepcopy(model.config)
        self.tok_emb = nn.Embedding.from_pretrained(model.tok_emb.weight.detach().clone(), freeze=True)
        self.blocks = nn.ModuleList([QuantizedBlock(b) for b in model.blocks])
        self.lm_head = Int8Linear(model.lm_head.lm_head.weight)
        self.loss_rows = model.lm_head.chunk_size or 4096
        if self.loss_rows < 0:  # as the model's own loss refuses it
            raise RuntimeError(f"loss_chunk_size must be nonnegative, got {self.loss_rows}")

    @torch.no_grad()
    def forward(self, idx: torch.Tensor, targets: torch.Tensor | None = None):
        x = self.tok_emb(idx)
        q8, scale = kernels.rms_norm_q8(x, None, self.config.norm_eps)
        for block in self.blocks:
            x, q8, scale = block(x, q8, scale)
        if targets is None:
            return self.lm_head(q8, scale, x.dtype), None
        q8, scale, t = q8.reshape(-1, q8.shape[-1]), scale.reshape(-1), targets.reshape(-1).to(torch.int64)
        # as the fused LM-head loss: targets outside the vocabulary are left out (F.cross_entropy
        # would stop the process's GPU work at one)
        counted = (t >= 0) & (t < self.config.vocab_size)
        t = torch.where(counted, t, -100)
        total = torch.zeros((), dtype=torch.float32, device=x.device)
        for s in range(0, t.numel(), self.loss_rows):  # logits of a chunk of tokens at a time, in fp32
            e = s + self.loss_rows
            logits = self.lm_head(q8[s:e], scale[s:e], torch.float32)
            total = total + F.cross_entropy(logits, t[s:e], reduction="sum")
        return None, total / counted.sum()

    def dequantized_weights(self, dtype: torch.dtype = torch.bfloat16) -> dict[str, torch.Tensor]:
        """The weights that the codes stand for, by module name."""
        return {name: m.dequantized(dtype) for name, m in self.named_modules() if isinstance(m, Int8Linear)}
