"""DiT inference with 8-bit integer products.

``DiTInt8`` runs the blocks of a trained DiT with every weight matrix in int8 (a
scale for each output channel) and every product's input in int8 (a scale for
each token), half the weight bytes and the int8 tensor-core rate:

    mod        = c8 Wada8^T + b                     gemm_s8 (M = B; c8 is quantised once for all blocks)
    x, h8      = x + g2' a', rms(x)*(1+sc1)+sh1     rmsnorm_mod_quant (the previous block's gated residual)
    qkv        = h8 Wqkv8^T + b                     gemm_s8
    o          = attention(rope(rms_h(q)), ...)     as in DiTBlock, bf16
    a          = o8 Wo8^T + bo                      quant_rows, gemm_s8
    x1, h8     = x + g1 a, rms(x1)*(1+sc2)+sh2      rmsnorm_mod_quant
    gu         = h8 [W1;W3]8^T                      gemm_s8
    a'         = silu(g)*u in 8 bits, W2            swiglu_quant, gemm_s8

The residual stream, attention, embedders and final layer stay in the model's
type.  Sums, norms and scales are fp32 or exact integers; no gradients.  It is
called as the DiT is, and batch_image_inference takes it in the DiT's place.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.nn as nn

from ..ops import functional as Fn
from ..ops.modules import Int8Linear
from ..parallel.sequence import SPContext, qkv_attention_forward
from .dit import DiT, DiTBlock, _w13


class DiTInt8Block(nn.Module):
    def __init__(self, blk: DiTBlock):
        super().__init__()
        self.cfg = blk.cfg
        ada_w, ada_b, qkv_w, qkv_b, qn_w, kn_w, proj_w, proj_b, w1, w3, w2, w2_b = blk.block_params()
        self.ada = Int8Linear.from_weight(ada_w, ada_b)
        self.qkv = Int8Linear.from_weight(qkv_w, qkv_b)
        self.proj = Int8Linear.from_weight(proj_w, proj_b)
        self.w13 = Int8Linear.from_weight(_w13(w1, w3), None)
        self.w2 = Int8Linear.from_weight(w2, w2_b)
        self.register_buffer("q_norm", qn_w.detach().clone() if qn_w is not None else None)
        self.register_buffer("k_norm", kn_w.detach().clone() if kn_w is not None else None)

    def forward(self, a: torch.Tensor, x: Optional[torch.Tensor], gate: Optional[torch.Tensor], c8, freqs, B: int, S: int,
                sp: SPContext) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """(a, x, gate): the stream as x + gate * a (x None: a itself), rows [B*S, D].  Returns the
        block's output in the same form."""
        cfg = self.cfg
        D, H, Dh = cfg.hidden, cfg.heads, cfg.head_dim
        mod = self.ada.rows(*c8)  # [B, 6D]
        sh1, sc1, g1, sh2, sc2, g2 = (mod[:, i * D:(i + 1) * D] for i in range(6))
        q, s, x = Fn.rmsnorm_mod_quant(a, None, sc1, sh1, S, cfg.norm_eps, residual=x, gate=gate)
        qkv = self.qkv.rows(q, s)
        o = qkv_attention_forward(qkv, B, S, H, Dh, self.q_norm, self.k_norm, freqs, 1e-6, cfg.qk_norm, sp)[0]
        a = self.proj(o)
        q, s, x = Fn.rmsnorm_mod_quant(a, None, sc2, sh2, S, cfg.norm_eps, residual=x, gate=g1)
        a = self.w2.rows(*Fn.swiglu_quant(self.w13.rows(q, s), cfg.ffn_hidden))
        return a, x, g2


class DiTInt8(DiT):
    """A DiT whose blocks multiply in int8.  Built from a DiT in bf16; the DiT's embedders and
    final layer are used as they are, its blocks are read once and nothing of them is kept."""

    def __init__(self, model: DiT):
        nn.Module.__init__(self)
        if any(p.dtype != torch.bfloat16 for p in model.parameters()):
            raise ValueError("DiTInt8 needs a DiT in bf16")
        self.cfg = model.cfg
        self.x_embedder, self.t_embedder, self.text_embedder = model.x_embedder, model.t_embedder, model.text_embedder
        with torch.no_grad():
            self.blocks = nn.ModuleList([DiTInt8Block(b) for b in model.blocks])
        self.final_layer = model.final_layer
        self._freq_cache = {}

    def initialize_weights(self, seed: int = 0):
        raise NotImplementedError("DiTInt8 takes its weights from a DiT")

    def int8(self) -> "DiTInt8":
        return self

    def run_blocks(self, h: torch.Tensor, c_silu: torch.Tensor, freqs: torch.Tensor, sp: SPContext) -> torch.Tensor:
        B, S, D = h.shape
        c8 = Fn.quant_rows(c_silu)
        a, x, gate = h.reshape(B * S, D), None, None
        for blk in self.blocks:
            a, x, gate = blk(a, x, gate, c8, freqs, B, S, sp)
        if x is None:
            return h
        return torch.addcmul(x.view(B, S, D), gate.unsqueeze(1), a.view(B, S, D))

    @torch.no_grad()
    def forward_local(self, x_img: torch.Tensor, text: torch.Tensor, t: torch.Tensor, h_tok: int, w_tok: int,
                      sp: SPContext):
        return super().forward_local(x_img, text, t, h_tok, w_tok, sp)
